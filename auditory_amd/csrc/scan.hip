// Selective state space scan over frames: every channel d carries N states through a recurrence whose step size, input and
// output vectors come with each frame (the PrevSmooth recurrence of the spectrum has one state and a fixed gain).
//
//   dt = softplus(delta + bias) or delta + bias,  a = exp(dt A_n),  h_t = a h_{t-1} + dt u B_n,  v = sum_n C_n h + D u,
//   y = v silu(z) or v
//
// Gradients, with f = dy silu(z) (or dy) and carry_t = a_{t+1} g_{t+1}:
//   g_t = f C_n + carry_t,  du = dt sum_n g B + D f,  ddt = u sum_n g B + sum_n A a h_{t-1} g,  dz = dy v silu'(z)
//   dB_n = sum_d g dt u,  dC_n = sum_d f h,  dA_n = sum_t dt a h_{t-1} g,  dD = sum f u,  dstate = carry_0
//
// A workgroup owns 64 channels of an item: a lane is a channel, a wave a share of the states.  Tiles of 16 steps go through
// LDS: all threads turn u and delta into (dt, dt u), each wave runs its states over the tile, all threads add the waves'
// partial sums up and store.  What a step's B and C hold is the same for all lanes of a wave: a small kernel lays them out in
// float32 first, and the waves read them as scalars, beside the vector pipe and LDS.
//
// Where items x channels leave the card idle, the time axis is cut into chunks: (1) every chunk but the last is scanned, the
// first from the true state, the others from zero, for its final state and its sum of dt; (3) every chunk works its true
// state out from those, h' = exp(A sum dt) h + (final state) chunk by chunk, and is scanned from there.
//
// Steps at and behind lengths[b] have dt = 0: the state stays, y is zero, and what the inputs hold there has no effect.
//
// The vector pipe bounds it, not memory: a state and step is one exponential (8 cycles of a SIMD) and four products and fused
// products (4 cycles each), a channel and step about 50 more instructions (softplus, gate, conversions, the sum over the waves).
// 8 x 2048 x 1536, 16 states, bfloat16: 178 us, 204 MB (floor 40 us); 192 workgroups, one a CU, whose SIMDs issue vector
// instructions 75 % of the time.  Gradients, 4 x 2048 x 1024: 41 us the first scan, 126 the second (82 %), of 255 for values and
// gradients.  What was measured on the way there: B and C broadcast from LDS 243 us; scalar loads without a group in hand 638, as
// runs of 64 bytes a group ahead 207; one barrier a tile instead of two 190; both elements of a thread side by side 186; addresses
// moved on by a tile, a turn of the loop for each LDS buffer 178.  Not taken: the steps' LDS reads a group ahead 182, the output of
// a tile behind the next one's scan 192, groups of half the size 194; inputs that lie still in the caches change nothing.
#include <type_traits>

#include "frame_ops.h"

namespace aud {
namespace {

constexpr int kNT = 256, kT = kScanTile, kCh = 64;
constexpr int kMaxChunks = 64, kJoinThreads = 64;
// Up to 8 chunks (16 where the card is not full) a workgroup walks the ones in front of its own; with more that reads too much
// (16 chunks, 64 workgroups of channels: 9 us more in the second scan) and a kernel between the scans (5 us) joins them.
constexpr int kFoldChunks = 8;

#if defined(__clang__)
typedef const float __attribute__((address_space(4)))* ScalarTable;  // read by scalar loads: nothing writes it meanwhile
#else
typedef const float* ScalarTable;
#endif

// B and C of GS steps for this wave's NW states, in scalar registers.  The scalar loads of the next group are sent off in front of
// a group's arithmetic and the LDS reads it needs are done by then: scalar loads come back out of order, so any wait for
// LDS would wait for them too.
template <int NW>
struct Vectors {
    static constexpr int GS = NW >= 8 ? 2 : 16 / NW < 8 ? 16 / NW : 8;
    float b[GS][NW], c[GS][NW];
    template <bool WITH_B, bool WITH_C>
    __device__ __forceinline__ void load(ScalarTable p) {
#pragma unroll
        for (int k = 0; k < GS; ++k)
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                if (WITH_B) b[k][i] = p[k * 2 * NW + i];
                if (WITH_C) c[k][i] = p[(k * 2 + 1) * NW + i];
            }
    }
};

__device__ __forceinline__ void wait_lds() {  // this wave's LDS reads (and scalar loads) have arrived
#if defined(__clang__)
    __builtin_amdgcn_s_waitcnt(0xC07F);
#endif
    __builtin_amdgcn_sched_barrier(0);
}
// Everything loaded so far has arrived.  In front of a loop: a register that is still on its way there would be waited for in
// every turn, and the loads that the turn has sent off with it.
__device__ __forceinline__ void wait_loads() {
#if defined(__clang__)
    __builtin_amdgcn_s_waitcnt(0x0F70);
#endif
}
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

struct Where {  // which channels, chunk and item a workgroup has
    int b, chunk, g, d0, dn, block;  // first channel, channels (<= 64), block within the group
    // (the first pass leaves the last chunk out, the gradients' first pass the first one)
    __device__ __forceinline__ Where(const ScanArgs& a, int blocks, int skip_last, int skip_first) {
        int id = blockIdx.x;
        block = id % blocks;
        id /= blocks;
        g = id % a.G;
        id /= a.G;
        const int chunks = a.chunks - skip_last - skip_first;
        chunk = id % chunks + skip_first;
        b = id / chunks;
        const int dg = a.Dn / a.G;
        d0 = g * dg + block * kCh;
        dn = dg - block * kCh < kCh ? dg - block * kCh : kCh;
    }
};

// E neighbouring floats of LDS at once
template <int E>
struct alignas(E * 4) Floats {
    float v[E];
};
template <int E>
__device__ __forceinline__ void lds_read(const float* p, float (&f)[E]) {
    const Floats<E> q = *reinterpret_cast<const Floats<E>*>(p);
#pragma unroll
    for (int i = 0; i < E; ++i) f[i] = q.v[i];
}
template <int E>
__device__ __forceinline__ void lds_write(float* p, const float (&f)[E]) {
    constexpr int M = E > 4 ? 4 : E;
#pragma unroll
    for (int j = 0; j < E; j += M) {
        Floats<M> q;
#pragma unroll
        for (int i = 0; i < M; ++i) q.v[i] = f[j + i];
        *reinterpret_cast<Floats<M>*>(p + j) = q;
    }
}
// E neighbouring channels of one step as stored, in whole registers: nothing touches them before the step they are wanted in, so
// the loads stay in flight until then.  Loads are unconditional: the caller gives an address that is there.
template <int DT, int E, bool VEC>
struct Raw {
    static constexpr int S = int(sizeof(typename Elem<DT>::raw));
    static constexpr bool WHOLE = VEC && E * S >= 4;
    static constexpr int WORDS = WHOLE ? E * S / 4 : E;
    struct alignas(WHOLE ? E * S : 4) Words {
        uint32_t w[WORDS];
    } r;
    // p: the first of the channels, `left` of them are there (one at least)
    __device__ __forceinline__ void load(const typename Elem<DT>::raw* p, int left) {
        if constexpr (WHOLE) r = *reinterpret_cast<const Words*>(p);
        else
#pragma unroll
            for (int i = 0; i < E; ++i) {
                if constexpr (S == 4) r.w[i] = __float_as_uint(p[i < left ? i : 0]);
                else r.w[i] = p[i < left ? i : 0];
            }
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (S == 4) return __uint_as_float(r.w[i]);
        else if constexpr (WHOLE) return Elem<DT>::up(typename Elem<DT>::raw(i & 1 ? r.w[i / 2] >> 16 : r.w[i / 2] & 0xFFFFu));
        else return Elem<DT>::up(typename Elem<DT>::raw(r.w[i]));
    }
};
template <int DT, int E, bool VEC>
__device__ __forceinline__ void store_some(void* base, int64_t at, int c, int dn, const float (&f)[E]) {
    if constexpr (VEC) {
        if (c < dn) store_pack<DT, E>(base, at + c, f);
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (c + i < dn) static_cast<typename Elem<DT>::raw*>(base)[at + c + i] = Elem<DT>::down(f[i]);
    }
}

__device__ __forceinline__ float step_size(float raw, int softp) { return softp ? softplus(raw) : raw; }
// (one branch for all of a thread's elements, so that their chains run side by side)
template <int E>
__device__ __forceinline__ void step_sizes(float (&dt)[E], int softp) {
    if (softp)
#pragma unroll
        for (int i = 0; i < E; ++i) dt[i] = softplus(dt[i]);
}

// B and C in float32 -> table [B, G, tiles, waves, 16 steps, B or C, NW states]: what a wave reads of a tile is one run.  States
// past N and steps at and behind the item's length are 0.
template <int DT>
__global__ void __launch_bounds__(kNT) k_scan_table(ScanArgs a, int NP, int NW, int tiles) {
    const int64_t i = int64_t(blockIdx.x) * kNT + threadIdx.x;
    const unsigned per = 2 * kT * NP, r = unsigned(i % per);
    const int n = int(r / (2 * kT * NW) * NW + r % NW), which = int(r / NW % 2);
    int64_t q = i / per;
    const int t = int(q % tiles) * kT + int(r / (2 * NW) % kT);
    q /= tiles;
    const int g = int(q % a.G);
    const int64_t b = q / a.G;
    if (b >= a.B) return;
    float v = 0.f;
    if (n < a.N && t < item_rows(a.lengths, int(b), a.L))
        v = which ? Elem<DT>::up(static_cast<const typename Elem<DT>::raw*>(a.Cm)[b * a.ci + int64_t(t) * a.cr + g * a.N + n])
                  : Elem<DT>::up(static_cast<const typename Elem<DT>::raw*>(a.Bm)[b * a.bi + int64_t(t) * a.br + g * a.N + n]);
    a.table[i] = v;
}

// What a chunk starts from, worked out from the table `sums` of the first pass.  Forward: slot 0 holds the first state, slot c + 1
// the state behind chunk c as far as the chunk knows it (chunk 0: the true one).  BACK, from the end: slot c + 1 holds what chunk
// c + 1 hands back (the last one: truly).  Several slots are read at once, so that their loads wait for one another once.
template <int NW, bool BACK>
__device__ __forceinline__ void chunk_state(const ScanArgs& a, const Where& at, int n0, int d, bool live, const float (&A2)[NW], float (&h)[NW]) {
    constexpr int kAhead = NW <= 8 ? kFoldChunks : 4;
    const int64_t per = int64_t(a.N) * a.Dn;
    const float* s = a.sums + int64_t(at.b) * a.chunks * per + d;
    const float* dt = a.sums + int64_t(a.B) * a.chunks * per + int64_t(at.b) * a.chunks * a.Dn + d;
    if (!live) return;
    if (!a.fold) {  // k_scan_join has been over the table
        const int64_t slot = BACK ? at.chunk + 1 : at.chunk;
#pragma unroll
        for (int i = 0; i < NW; ++i)
            if (n0 + i < a.N) h[i] = s[slot * per + int64_t(n0 + i) * a.Dn];
        return;
    }
    // forward: slots 1 .. chunk (slot 0 alone for chunk 0); back: slots chunks - 1 down to chunk + 1
    const int count = BACK ? a.chunks - 1 - at.chunk : (at.chunk > 0 ? at.chunk : 1);
    for (int k = 0; k < count; k += kAhead) {
        float part[kAhead][NW], sum[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int kk = k + j < count ? k + j : count - 1;
            const int slot = BACK ? a.chunks - 1 - kk : (at.chunk > 0 ? 1 + kk : 0);
            const int chunk = BACK ? slot : (slot > 0 ? slot - 1 : 0);
            sum[j] = dt[int64_t(chunk) * a.Dn];
#pragma unroll
            for (int i = 0; i < NW; ++i) part[j][i] = n0 + i < a.N ? s[slot * per + int64_t(n0 + i) * a.Dn] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (k + j >= count) break;
#pragma unroll
            for (int i = 0; i < NW; ++i) h[i] = k + j == 0 ? part[j][i] : fmaf(exp2_hw(sum[j] * A2[i]), h[i], part[j][i]);
        }
    }
}

// ---- values.  PASS 1: a chunk's final state from zero and its sum of dt; PASS 3: y.  W waves of NW states each ---------------
// One barrier a tile: between two of them a wave runs its states over tile k, turns the inputs of tile k + 1 (on their way
// while it ran) into steps and, at the next one's start, adds up and stores tile k.  Eight waves of two states (16 states)
// against four of four, when the whole took 190 us: 275 us at 8 x 2048 x 1536, 16 waves of one: 199.
template <int DT, int NW, int W, bool VEC, int PASS>
__global__ void __launch_bounds__(64 * W) k_scan(ScanArgs a, int blocks) {
    constexpr int NP = W * NW, E = 16 / W, ROW = kCh / E;  // elements a thread loads and stores, threads a step
    float* lds = reinterpret_cast<float*>(dyn_lds());
    float2* s_step = reinterpret_cast<float2*>(lds);  // [2][16][64] (dt, dt u)
    float* s_y = lds + 4 * kT * kCh;                  // [2][W][16][64]
    const Where at(a, blocks, PASS == 1, 0);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int pt = tid / ROW, c = (tid % ROW) * E;    // this thread's step and channels when a tile is loaded and stored
    const int len = item_rows(a.lengths, at.b, a.L), tiles = (a.L + kT - 1) / kT;
    const int64_t u0 = at.b * a.ui + at.d0, e0 = at.b * a.ei + at.d0, z0 = at.b * a.zi + at.d0, y0 = int64_t(at.b) * a.L * a.Dn + at.d0;
    const int d = at.d0 + lane;
    const bool live = lane < at.dn;
    float A2[NW], h[NW], sum_dt = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        const int n = wave * NW + i;
        const bool there = live && n < a.N;
        A2[i] = there ? a.A[int64_t(d) * a.N + n] * kLog2e : 0.f;
        h[i] = 0.f;
        if (there && at.chunk == 0 && (PASS == 1 || a.chunks == 1) && a.state) h[i] = a.state[(int64_t(at.b) * a.Dn + d) * a.N + n];
        // (a copy for the first chunk's second scan: state_out, written by the last chunk, may be the state itself)
        if (there && at.chunk == 0 && PASS == 1) a.sums[(int64_t(at.b) * a.chunks * a.N + n) * a.Dn + d] = h[i];
    }
    if (PASS == 3 && a.chunks > 1) chunk_state<NW, false>(a, at, wave * NW, d, live, A2, h);
    float skip[E], bias[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const bool there = c + i < at.dn;
        skip[i] = there && a.D ? a.D[at.d0 + c + i] : 0.f;
        bias[i] = there && a.delta_bias ? a.delta_bias[at.d0 + c + i] : 0.f;
    }
    const int first = at.chunk * a.chunk_tiles, end = first + a.chunk_tiles < tiles ? first + a.chunk_tiles : tiles;
    Raw<DT, E, VEC> ru{}, rd{}, rz{};
    // addresses of this thread's channels in its row of the tile, moved on by 16 rows a tile (rows behind the last one: the last)
    typedef typename Elem<DT>::raw raw;
    const int cc = c < at.dn ? c : 0, left = at.dn - cc;
    const int64_t row = first * kT + pt;
    const raw* pu = static_cast<const raw*>(a.u) + u0 + row * a.ur + cc;
    const raw* pd = static_cast<const raw*>(a.delta) + e0 + row * a.er + cc;
    const raw* pz = a.z ? static_cast<const raw*>(a.z) + z0 + row * a.zr + cc : pu;  // (no gate: read and not used)
    const int64_t su = kT * a.ur, sd = kT * a.er, sz = a.z ? kT * a.zr : su;
    auto fetch = [&](int tile) {
        if ((tile + 1) * kT > a.L) {  // (the last tile: the addresses are not moved on from here)
            const int64_t over = tile * kT + pt < a.L ? 0 : tile * kT + pt - (a.L - 1);
            pu -= over * a.ur, pd -= over * a.er, pz -= over * (a.z ? a.zr : a.ur);
        }
        ru.load(pu, left);
        rd.load(pd, left);
        if (PASS == 3) rz.load(pz, left);
    };
    float* pk = a.kept ? a.kept + ((int64_t(at.b) * tiles + first) * a.N + wave * NW) * a.Dn + d : nullptr;
    raw* py = PASS == 3 ? static_cast<raw*>(a.y) + y0 + int64_t(first * kT + pt) * a.Dn : nullptr;
    float u[2][E], z[2][E];  // of the tile that is being scanned, and of the next one
    auto stage = [&](int tile, int buf) {
        float step[2 * E], dt[E];
        const bool row_on = tile * kT + pt < len;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            u[buf][i] = ru.get(i);
            z[buf][i] = rz.get(i);
            dt[i] = rd.get(i) + bias[i];
        }
        step_sizes(dt, a.softplus);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const bool on = row_on && c + (VEC ? 0 : i) < at.dn;
            step[2 * i] = on ? dt[i] : 0.f;
            step[2 * i + 1] = on ? dt[i] * u[buf][i] : 0.f;
        }
        lds_write(lds + 2 * ((buf * kT + pt) * kCh + c), step);
    };
    if (first < end) {
        fetch(first);
        stage(first, 0);
    }
    __syncthreads();
    ScalarTable bc = (ScalarTable)(a.table + ((int64_t(at.b) * a.G + at.g) * tiles + first) * kT * 2 * NP + wave * kT * 2 * NW);
    typedef Vectors<NW> Vec;
    constexpr int GS = Vec::GS;
    Vec next{};
    wait_loads();
    if (first < end) next.template load<true, PASS == 3>(bc);
    auto scan_tile = [&](int tile, auto which) {  // (a turn of the loop for each buffer: what belongs to one stays in its registers)
        constexpr int buf = decltype(which)::value;
        const bool more = tile + 1 < end;
        if (more) {
            pu += su, pd += sd, pz += sz;
            fetch(tile + 1);
        }
        if (PASS == 3 && a.kept) {
#pragma unroll
            for (int i = 0; i < NW; ++i)
                if (live && wave * NW + i < a.N) pk[int64_t(i) * a.Dn] = h[i];
            pk += int64_t(a.N) * a.Dn;
        }
#pragma unroll
        for (int k0 = 0; k0 < kT; k0 += GS) {
            const Vec now = next;
            float2 st[GS];
#pragma unroll
            for (int k = 0; k < GS; ++k) st[k] = s_step[(buf * kT + k0 + k) * kCh + lane];
            ScalarTable ahead = bc + (k0 + GS) * 2 * NW;
            if (k0 + GS == kT) ahead = more ? bc + kT * 2 * NP : bc;  // (nothing behind the last tile: any address of the table)
            wait_lds();
            next.template load<true, PASS == 3>(ahead);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < GS; ++k) {
                float y = 0.f;
#pragma unroll
                for (int i = 0; i < NW; ++i) {
                    h[i] = fmaf(exp2_hw(st[k].x * A2[i]), h[i], st[k].y * now.b[k][i]);
                    if (PASS == 3) y = fmaf(now.c[k][i], h[i], y);
                }
                if (PASS == 3) s_y[((buf * W + wave) * kT + k0 + k) * kCh + lane] = y;
                else sum_dt += st[k].x;
            }
        }
        bc += kT * 2 * NP;
        if (more) stage(tile + 1, buf ^ 1);
        __syncthreads();
        const int t = tile * kT + pt;
        if (PASS == 3 && t < a.L) {
            float y[E];
#pragma unroll
            for (int i = 0; i < E; ++i) y[i] = skip[i] * u[buf][i];
#pragma unroll
            for (int w = 0; w < W; ++w) {
                float part[E];
                lds_read(s_y + ((buf * W + w) * kT + pt) * kCh + c, part);
#pragma unroll
                for (int i = 0; i < E; ++i) y[i] += part[i];
            }
            if (a.z)
#pragma unroll
                for (int i = 0; i < E; ++i) y[i] *= z[buf][i] * fast_sigmoid(z[buf][i]);
#pragma unroll
            for (int i = 0; i < E; ++i) y[i] = t < len ? y[i] : 0.f;
            store_some<DT, E, VEC>(py, 0, c, at.dn, y);
        }
        if (PASS == 3) py += kT * a.Dn;
    };
    for (int tile = first; tile < end; tile += 2) {
        scan_tile(tile, std::integral_constant<int, 0>{});
        if (tile + 1 < end) scan_tile(tile + 1, std::integral_constant<int, 1>{});
    }
    if (!live) return;
    float* dt_sums = a.sums + int64_t(a.B) * a.chunks * a.N * a.Dn;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        const int n = wave * NW + i;
        if (n >= a.N) continue;
        if (PASS == 1) a.sums[((int64_t(at.b) * a.chunks + at.chunk + 1) * a.N + n) * a.Dn + d] = h[i];
        else if (at.chunk == a.chunks - 1 && a.state_out) a.state_out[(int64_t(at.b) * a.Dn + d) * a.N + n] = h[i];
    }
    if (PASS == 1 && wave == 0) dt_sums[(int64_t(at.b) * a.chunks + at.chunk) * a.Dn + d] = sum_dt;
}

// many chunks: the same once for all of them, slot by slot in place (sixteen at once)
template <bool BACK>
__global__ void __launch_bounds__(kJoinThreads) k_scan_join(ScanArgs a) {
    constexpr int kAhead = 16;
    const int64_t id = int64_t(blockIdx.x) * kJoinThreads + threadIdx.x, per = int64_t(a.N) * a.Dn;
    if (id >= a.B * per) return;
    const int64_t b = id / per;
    const int n = int(id % per / a.Dn), d = int(id % a.Dn);
    const float A2 = a.A[int64_t(d) * a.N + n] * kLog2e;
    float* s = a.sums + b * a.chunks * per + int64_t(n) * a.Dn + d;
    const float* dt = a.sums + int64_t(a.B) * a.chunks * per + b * a.chunks * a.Dn + d;
    // slots 1 .. chunks - 1, forward from 1 or back from the last; the first of them is true already
    float h = 0.f;
    for (int k = 0; k < a.chunks - 1; k += kAhead) {
        float mine[kAhead], sum[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int kk = k + j < a.chunks - 1 ? k + j : a.chunks - 2, slot = BACK ? a.chunks - 1 - kk : 1 + kk;
            mine[j] = s[slot * per];
            sum[j] = dt[int64_t(BACK ? slot : slot - 1) * a.Dn];
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (k + j >= a.chunks - 1) break;
            const int slot = BACK ? a.chunks - 1 - (k + j) : 1 + k + j;
            h = k + j == 0 ? mine[j] : fmaf(exp2_hw(sum[j] * A2), h, mine[j]);
            s[slot * per] = h;
        }
    }
}

// ---- one frame: four lanes a channel, a quarter of its states each ----------------------------------------------------
template <int DT>
__global__ void __launch_bounds__(kNT) k_scan_step(ScanArgs a) {
    const int64_t id = int64_t(blockIdx.x) * kNT + threadIdx.x, ch = id >> 2;
    const int part = int(id & 3);
    const bool on = ch < int64_t(a.B) * a.Dn;  // (all lanes of a wave reach the exchange below)
    const int64_t b = on ? ch / a.Dn : 0;
    const int d = on ? int(ch % a.Dn) : 0, g = d / (a.Dn / a.G);
    typedef typename Elem<DT>::raw raw;
    const bool live = on && item_rows(a.lengths, int(b), 1) > 0;
    const float u = Elem<DT>::up(static_cast<const raw*>(a.u)[b * a.ui + d]);
    const float dt_raw = Elem<DT>::up(static_cast<const raw*>(a.delta)[b * a.ei + d]) + (a.delta_bias ? a.delta_bias[d] : 0.f);
    const float dt = step_size(dt_raw, a.softplus);
    float v = 0.f;
    if (on)
        for (int n = part; n < a.N; n += 4) {
            const int64_t at = ch * a.N + n;
            float h = a.state ? a.state[at] : 0.f;
            if (a.kept) a.kept[(b * a.N + n) * a.Dn + d] = h;
            if (live) {
                const float bn = Elem<DT>::up(static_cast<const raw*>(a.Bm)[b * a.bi + g * a.N + n]);
                const float cn = Elem<DT>::up(static_cast<const raw*>(a.Cm)[b * a.ci + g * a.N + n]);
                h = fmaf(exp2_hw(dt * (a.A[int64_t(d) * a.N + n] * kLog2e)), h, dt * u * bn);
                v = fmaf(cn, h, v);
            }
            if (a.state_out) a.state_out[at] = h;
        }
    v += __shfl_xor(v, 1);
    v += __shfl_xor(v, 2);
    if (on && part == 0) {
        if (a.D) v = fmaf(a.D[d], u, v);
        if (a.z) {
            const float z = Elem<DT>::up(static_cast<const raw*>(a.z)[b * a.zi + d]);
            v *= z * fast_sigmoid(z);
        }
        static_cast<raw*>(a.y)[ch] = Elem<DT>::down(live ? v : 0.f);
    }
}

// ---- gradients ------------------------------------------------------------------------------------------------------------
// Sums over the 64 lanes of many values at once: two values are joined into one register, each half of the lanes going on
// with one of them, so 64 values cost 63 additions and leave lane l with the sum of one.  LEVEL 0 .. 5 splits by lane bit
// 5 - LEVEL; lanes with the bit clear keep `a`.
template <int LEVEL>
__device__ __forceinline__ float lane_partner(float v) {
    constexpr int ctrl = LEVEL == 2 ? 0x140 : LEVEL == 3 ? 0x141 : LEVEL == 4 ? 0x4E : 0xB1;  // l ^ 15, l ^ 7, l ^ 2, l ^ 1
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xF, 0xF, true));
}
template <int LEVEL>
__device__ __forceinline__ float lane_join(float a, float b, int lane) {
#if defined(__clang__)
    if constexpr (LEVEL == 0) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
        return __uint_as_float(r[0]) + __uint_as_float(r[1]);
    } else if constexpr (LEVEL == 1) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
        return __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
#else
    if constexpr (LEVEL < 2) return ((lane >> (5 - LEVEL)) & 1 ? b : a) + __shfl_xor((lane >> (5 - LEVEL)) & 1 ? a : b, 32 >> LEVEL);
#endif
    else {
        const bool up = (lane >> (5 - LEVEL)) & 1;
        return (up ? b : a) + lane_partner<LEVEL>(up ? a : b);
    }
}
__device__ __forceinline__ float lane_join_at(int level, float a, float b, int lane) {  // (level is a constant where it is called)
    switch (level) {
        case 0: return lane_join<0>(a, b, lane);
        case 1: return lane_join<1>(a, b, lane);
        case 2: return lane_join<2>(a, b, lane);
        case 3: return lane_join<3>(a, b, lane);
        case 4: return lane_join<4>(a, b, lane);
        default: return lane_join<5>(a, b, lane);
    }
}
constexpr int log2_of(int v) { return v <= 1 ? 0 : 1 + log2_of(v / 2); }
// The sums over the lanes of v[step][state] for TS steps of NW states, handed in step by step from the last to the first.
// When step 0 is in, lane l has the sum of state i, step k:  bit q of i = bit 5 - q of l,  bit j of k = bit 5 - log2 NW - j.
template <int NW, int TS>
struct LaneSums {
    static constexpr int LI = log2_of(NW), LK = log2_of(TS), USED = LI + LK;
    static_assert(USED <= 6, "at most 64 values");
    float stack[LK > 0 ? LK : 1];
    float total;
    __device__ __forceinline__ void add(int k, float (&v)[NW], int lane) {
#pragma unroll
        for (int q = 0; q < LI; ++q)
#pragma unroll
            for (int i = 0; i < (NW >> (q + 1)); ++i) v[i] = lane_join_at(q, v[2 * i], v[2 * i + 1], lane);
        float x = v[0];
#pragma unroll
        for (int j = 0; j < LK; ++j) {
            if ((k >> j) & 1) {
                stack[j] = x;
                return;
            }
            x = lane_join_at(LI + j, x, stack[j], lane);
        }
        if constexpr (USED <= 4) x += lane_partner<4>(x);
        if constexpr (USED <= 5) x += lane_partner<5>(x);
        total = x;
    }
    static __device__ __forceinline__ int state_of(int lane) {
        int i = 0;
#pragma unroll
        for (int q = 0; q < LI; ++q) i |= ((lane >> (5 - q)) & 1) << q;
        return i;
    }
    static __device__ __forceinline__ int step_of(int lane) {
        int k = 0;
#pragma unroll
        for (int j = 0; j < LK; ++j) k |= ((lane >> (5 - LI - j)) & 1) << j;
        return k;
    }
    static __device__ __forceinline__ bool first_of(int lane) { return (lane & ((1 << (6 - USED)) - 1)) == 0; }
};

// PASS 1: what a chunk hands to the one in front of it, from a zero carry, and its sum of dt; PASS 3: everything.  W waves of NW
// states each.
template <int DT, int NW, int W, bool VEC, int PASS>
__global__ void __launch_bounds__(64 * W, 2) k_scan_grad(ScanArgs a, int blocks) {
    constexpr int NP = W * NW, E = 16 / W, ROW = kCh / E;
    constexpr int TS = NW <= 4 ? 16 : 64 / NW, SUBS = kT / TS;  // steps whose states are in registers at once
    float* lds = reinterpret_cast<float*>(dyn_lds());
    float* s_dt = lds;                      // [16][64] each
    float* s_f = s_dt + kT * kCh;
    float* s_du = s_f + kT * kCh;           // dt u
    float* s_db = s_du + kT * kCh;          // [16][NP] each
    float* s_dc = s_db + kT * NP;
    float* s_sum = s_dc + kT * NP;          // [3][W][16][64]: sum_n g B, sum_n A a h g, sum_n C h of each wave
    const Where at(a, blocks, 0, PASS == 1);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int pt = tid / ROW, c = (tid % ROW) * E;
    const int len = item_rows(a.lengths, at.b, a.L), tiles = (a.L + kT - 1) / kT;
    const int64_t u0 = at.b * a.ui + at.d0, e0 = at.b * a.ei + at.d0, z0 = at.b * a.zi + at.d0, g0 = at.b * a.yi + at.d0;
    const int64_t o0 = int64_t(at.b) * a.L * a.Dn + at.d0;
    const int d = at.d0 + lane;
    const bool live = lane < at.dn;
    float A2[NW], An[NW], carry[NW], dA[NW], sum_dt = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        const int n = wave * NW + i;
        const bool there = live && n < a.N;
        An[i] = there ? a.A[int64_t(d) * a.N + n] : 0.f;
        A2[i] = An[i] * kLog2e;
        carry[i] = dA[i] = 0.f;
        if (there && at.chunk == a.chunks - 1 && a.dstate_out) carry[i] = a.dstate_out[(int64_t(at.b) * a.Dn + d) * a.N + n];
    }
    if (PASS == 3 && at.chunk < a.chunks - 1) chunk_state<NW, true>(a, at, wave * NW, d, live, A2, carry);
    float skip[E], bias[E], sum_fu[E], sum_dd[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const bool there = c + i < at.dn;
        skip[i] = there && a.D ? a.D[at.d0 + c + i] : 0.f;
        bias[i] = there && a.delta_bias ? a.delta_bias[at.d0 + c + i] : 0.f;
        sum_fu[i] = sum_dd[i] = 0.f;
    }
    const int first = at.chunk * a.chunk_tiles, end = first + a.chunk_tiles < tiles ? first + a.chunk_tiles : tiles;
    Raw<DT, E, VEC> ru{}, rd{}, rz{}, ry{};
    // addresses of this thread's channels in its row of the tile, moved back by 16 rows a tile (rows behind the last one: the last)
    typedef typename Elem<DT>::raw raw;
    const int cc = c < at.dn ? c : 0, left = at.dn - cc;
    const int64_t row = (end - 1) * kT + pt, over = row < a.L ? 0 : row - (a.L - 1);
    const raw* pu = static_cast<const raw*>(a.u) + u0 + (row - over) * a.ur + cc;
    const raw* pd = static_cast<const raw*>(a.delta) + e0 + (row - over) * a.er + cc;
    const raw* pg = static_cast<const raw*>(a.dy) + g0 + (row - over) * a.yr + cc;
    const raw* pz = a.z ? static_cast<const raw*>(a.z) + z0 + (row - over) * a.zr + cc : pg;  // (no gate: read and not used)
    const int64_t su = kT * a.ur, sd = kT * a.er, sg = kT * a.yr, sz = a.z ? kT * a.zr : sg;
    const int64_t step_o = int64_t(kT) * a.Dn;
    const int lane_in = live ? lane : 0;
    // (the same for all lanes: states in front of the tile, results of its first row)
    const float* pk = PASS == 3 ? a.kept + ((int64_t(at.b) * tiles + (end - 1)) * a.N + wave * NW) * a.Dn + at.d0 : nullptr;
    const unsigned lane_o = unsigned((int64_t(pt) * a.Dn + c) * int(sizeof(raw)));  // bytes: 16 rows of 2^24 channels at most
    int64_t o_tile = o0 + int64_t(end - 1) * step_o;
    const int64_t gn = int64_t(a.G) * a.N, table_bc = int64_t(a.B) * a.L * gn;
    int64_t o_bc = (int64_t(at.b) * a.L + int64_t(end - 1) * kT) * gn + int64_t(at.g) * a.N;
    float h0[NW];  // the state in front of the tile
#pragma unroll
    for (int i = 0; i < NW; ++i) h0[i] = 0.f;
    auto fetch = [&] {
        if (PASS == 3) ru.load(pu, left);
        rd.load(pd, left);
        rz.load(pz, left);
        ry.load(pg, left);
        if (PASS == 3)
#pragma unroll
            for (int i = 0; i < NW; ++i)
                if (wave * NW + i < a.N) h0[i] = pk[int64_t(i) * a.Dn + lane_in];
    };
    wait_loads();
    if (first < end) {
        fetch();
        pu += over * a.ur, pd += over * a.er, pg += over * a.yr, pz += over * (a.z ? a.zr : a.yr);
    }
    ScalarTable bc = (ScalarTable)(a.table + ((int64_t(at.b) * a.G + at.g) * tiles + (end - 1)) * kT * 2 * NP + wave * kT * 2 * NW);
    for (int tile = end - 1; tile >= first; --tile, bc -= kT * 2 * NP) {
        const int t0 = tile * kT, t = t0 + pt;
        const bool on = t < len;
        float u[E], z[E], dy[E], arg[E], dt[E], f[E], dtu[E], hs0[NW];
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const bool there = on && c + (VEC ? 0 : i) < at.dn;
            u[i] = there ? ru.get(i) : 0.f;
            z[i] = there ? rz.get(i) : 0.f;
            dy[i] = there ? ry.get(i) : 0.f;
            arg[i] = (there ? rd.get(i) : 0.f) + bias[i];
            dt[i] = arg[i];
            f[i] = dy[i];
        }
        step_sizes(dt, a.softplus);
        if (a.z)
#pragma unroll
            for (int i = 0; i < E; ++i) f[i] *= z[i] * fast_sigmoid(z[i]);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            if (!(on && c + (VEC ? 0 : i) < at.dn)) dt[i] = 0.f;
            dtu[i] = dt[i] * u[i];
        }
        lds_write(s_dt + pt * kCh + c, dt);
        lds_write(s_f + pt * kCh + c, f);
        if (PASS == 3) lds_write(s_du + pt * kCh + c, dtu);
#pragma unroll
        for (int i = 0; i < NW; ++i) hs0[i] = live ? h0[i] : 0.f;
        __syncthreads();
        if (tile > first) {
            pu -= su, pd -= sd, pg -= sg, pz -= sz;
            if (PASS == 3) pk -= int64_t(a.N) * a.Dn;
            fetch();
        }
        typedef Vectors<NW> Vec;
        constexpr int GS = Vec::GS;
        if constexpr (PASS == 1) {
            Vec next;
            next.template load<false, true>(bc + (kT - GS) * 2 * NW);
#pragma unroll
            for (int k0 = kT - GS; k0 >= 0; k0 -= GS) {
                const Vec now = next;
                float s[GS], fk[GS];
#pragma unroll
                for (int k = 0; k < GS; ++k) s[k] = s_dt[(k0 + k) * kCh + lane], fk[k] = s_f[(k0 + k) * kCh + lane];
                wait_lds();
                if (k0 > 0) next.template load<false, true>(bc + (k0 - GS) * 2 * NW);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int k = GS - 1; k >= 0; --k) {
                    sum_dt += s[k];
#pragma unroll
                    for (int i = 0; i < NW; ++i) carry[i] = exp2_hw(s[k] * A2[i]) * fmaf(fk[k], now.c[k][i], carry[i]);
                }
            }
        } else {
            // (a loop where a part is less than the tile: its steps are then not constants, but the tables' offsets stay small)
#pragma unroll 1
            for (int sub = SUBS - 1; sub >= 0; --sub) {
                const int k0 = sub * TS;
                float h[NW], hs[TS][NW], as[TS][NW];  // states behind and decays of the steps of this part of the tile
#pragma unroll
                for (int i = 0; i < NW; ++i) h[i] = hs0[i];
                Vec next;
                next.template load<true, true>(bc);
                if constexpr (SUBS > 1) {  // up to this part: once more from the tile's first state
#pragma unroll 1
                    for (int q = 0; q < k0; q += GS) {
                        const Vec now = next;
                        float s[GS], x[GS];
#pragma unroll
                        for (int k = 0; k < GS; ++k) s[k] = s_dt[(q + k) * kCh + lane], x[k] = s_du[(q + k) * kCh + lane];
                        wait_lds();
                        next.template load<true, true>(bc + (q + GS) * 2 * NW);
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int k = 0; k < GS; ++k)
#pragma unroll
                            for (int i = 0; i < NW; ++i) h[i] = fmaf(exp2_hw(s[k] * A2[i]), h[i], x[k] * now.b[k][i]);
                    }
                }
                float before[NW];
#pragma unroll
                for (int i = 0; i < NW; ++i) before[i] = h[i];
#pragma unroll
                for (int q = 0; q < TS; q += GS) {
                    const Vec now = next;
                    float s[GS], x[GS];
#pragma unroll
                    for (int k = 0; k < GS; ++k) s[k] = s_dt[(k0 + q + k) * kCh + lane], x[k] = s_du[(k0 + q + k) * kCh + lane];
                    wait_lds();
                    if (q + GS < TS) next.template load<true, true>(bc + (k0 + q + GS) * 2 * NW);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int k = 0; k < GS; ++k) {
                        float v = 0.f;
#pragma unroll
                        for (int i = 0; i < NW; ++i) {
                            as[q + k][i] = exp2_hw(s[k] * A2[i]);
                            h[i] = fmaf(as[q + k][i], h[i], x[k] * now.b[k][i]);
                            hs[q + k][i] = h[i];
                            v = fmaf(now.c[k][i], h[i], v);
                        }
                        if (a.z) s_sum[((2 * W + wave) * kT + k0 + q + k) * kCh + lane] = v;
                    }
                }
                LaneSums<NW, TS> sum_b, sum_c;
                // (the last group's vectors are still there)
#pragma unroll
                for (int q = TS - GS; q >= 0; q -= GS) {
                    const Vec now = next;
                    float s[GS], x[GS], fk[GS];
#pragma unroll
                    for (int k = 0; k < GS; ++k) {
                        s[k] = s_dt[(k0 + q + k) * kCh + lane], x[k] = s_du[(k0 + q + k) * kCh + lane];
                        fk[k] = s_f[(k0 + q + k) * kCh + lane];
                    }
                    wait_lds();
                    if (q > 0) next.template load<true, true>(bc + (k0 + q - GS) * 2 * NW);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int k = GS - 1; k >= 0; --k) {
                        const int kk = q + k;
                        float gb = 0.f, ahg = 0.f, pb[NW], pc[NW];
#pragma unroll
                        for (int i = 0; i < NW; ++i) {
                            const float g = fmaf(fk[k], now.c[k][i], carry[i]);
                            gb = fmaf(g, now.b[k][i], gb);
                            carry[i] = as[kk][i] * g;
                            const float r = carry[i] * (kk > 0 ? hs[kk > 0 ? kk - 1 : 0][i] : before[i]);
                            ahg = fmaf(An[i], r, ahg);
                            dA[i] = fmaf(s[k], r, dA[i]);
                            pb[i] = g * x[k];
                            pc[i] = fk[k] * hs[kk][i];
                        }
                        sum_b.add(kk, pb, lane);
                        sum_c.add(kk, pc, lane);
                        s_sum[((0 * W + wave) * kT + k0 + kk) * kCh + lane] = gb;
                        s_sum[((1 * W + wave) * kT + k0 + kk) * kCh + lane] = ahg;
                    }
                }
                typedef LaneSums<NW, TS> Sums;
                if (Sums::first_of(lane)) {
                    const int o = (k0 + Sums::step_of(lane)) * NP + wave * NW + Sums::state_of(lane);
                    s_db[o] = sum_b.total;
                    s_dc[o] = sum_c.total;
                }
            }
        }
        __syncthreads();
        if constexpr (PASS == 3) {
            // (the next tile's steps are written beside this: they are read behind the next barrier only)
            if (t < a.L) {
                float du[E], dd[E], dz[E], sums[3][E];
#pragma unroll
                for (int k = 0; k < 3; ++k) {
#pragma unroll
                    for (int i = 0; i < E; ++i) sums[k][i] = 0.f;
                    if (k < 2 || a.z)
#pragma unroll
                        for (int w = 0; w < W; ++w) {
                            float part[E];
                            lds_read(s_sum + ((k * W + w) * kT + pt) * kCh + c, part);
#pragma unroll
                            for (int i = 0; i < E; ++i) sums[k][i] += part[i];
                        }
                }
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    const float ddt = fmaf(u[i], sums[0][i], sums[1][i]);
                    du[i] = fmaf(dt[i], sums[0][i], skip[i] * f[i]);
                    dd[i] = ddt;
                    sum_fu[i] = fmaf(f[i], u[i], sum_fu[i]);
                }
                if (a.softplus)
#pragma unroll
                    for (int i = 0; i < E; ++i) dd[i] *= fast_sigmoid(arg[i]);
                if (a.z)
#pragma unroll
                    for (int i = 0; i < E; ++i) {
                        const float q = fast_sigmoid(z[i]);
                        dz[i] = dy[i] * fmaf(skip[i], u[i], sums[2][i]) * (q * (1.f + z[i] * (1.f - q)));
                    }
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    if (!on) du[i] = dd[i] = dz[i] = 0.f;
                    sum_dd[i] += dd[i];
                }
                auto put = [&](void* base, const float (&f)[E]) {
                    store_some<DT, E, VEC>(reinterpret_cast<char*>(static_cast<raw*>(base) + o_tile) + lane_o, 0, 0, at.dn - c, f);
                };
                put(a.du, du);
                put(a.ddelta, dd);
                if (a.dz) put(a.dz, dz);
            }
            o_tile -= step_o;
            // dB, dC of the tile, summed over this block's channels: partial sums where the group has more blocks
            for (int i = tid; i < kT * NP; i += 64 * W) {
                const int k = i / NP, n = i % NP;
                if (n >= a.N || t0 + k >= a.L) continue;
                const int64_t o = k * gn + n;
                const bool there = t0 + k < len;
                const float vb = there ? s_db[i] : 0.f, vc = there ? s_dc[i] : 0.f;
                if (blocks == 1) {
                    (static_cast<raw*>(a.dB) + o_bc)[o] = Elem<DT>::down(vb);
                    (static_cast<raw*>(a.dC) + o_bc)[o] = Elem<DT>::down(vc);
                } else {
                    (a.part_bc + at.block * table_bc + o_bc)[o] = vb;
                    (a.part_bc + (blocks + at.block) * table_bc + o_bc)[o] = vc;
                }
            }
            o_bc -= kT * gn;
        }
    }
    if constexpr (PASS == 1) {
        if (!live) return;
        float* dt_sums = a.sums + int64_t(a.B) * a.chunks * a.N * a.Dn;
#pragma unroll
        for (int i = 0; i < NW; ++i)
            if (wave * NW + i < a.N) a.sums[((int64_t(at.b) * a.chunks + at.chunk) * a.N + wave * NW + i) * a.Dn + d] = carry[i];
        if (wave == 0) dt_sums[(int64_t(at.b) * a.chunks + at.chunk) * a.Dn + d] = sum_dt;
    } else {
        float* sums_of = a.part + (int64_t(at.b) * a.chunks + at.chunk) * (a.N + 2) * a.Dn;
        if (live) {
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                const int n = wave * NW + i;
                if (n >= a.N) continue;
                sums_of[int64_t(n) * a.Dn + d] = dA[i];
                if (at.chunk == 0 && a.dstate) a.dstate[(int64_t(at.b) * a.Dn + d) * a.N + n] = carry[i];
            }
        }
#pragma unroll
        for (int i = 0; i < E; ++i) {
            s_dt[pt * kCh + c + i] = sum_fu[i];
            s_f[pt * kCh + c + i] = sum_dd[i];
        }
        __syncthreads();
        if (tid < 2 * kCh && lane < at.dn) {
            const float* p = (wave == 0 ? s_dt : s_f) + lane;
            float s = 0.f;
            for (int k = 0; k < kT; ++k) s += p[k * kCh];
            sums_of[int64_t(a.N + wave) * a.Dn + d] = s;
        }
    }
}

// dB, dC: the blocks' partial sums added in order and rounded to the activations' type
template <int DT>
__global__ void __launch_bounds__(kNT) k_scan_bc(ScanArgs a, int blocks) {
    const int64_t n = int64_t(a.B) * a.L * a.G * a.N, i = int64_t(blockIdx.x) * kNT + threadIdx.x;
    if (i >= 2 * n) return;
    const int64_t o = i < n ? i : i - n;
    const float* p = a.part_bc + (i < n ? 0 : blocks * n) + o;
    float s = 0.f;
    for (int k = 0; k < blocks; ++k) s += p[k * n];
    static_cast<typename Elem<DT>::raw*>(i < n ? a.dB : a.dC)[o] = Elem<DT>::down(s);
}


template <int DT>
void run_table(const ScanArgs& a, int NP, int NW, hipStream_t st) {
    const int tiles = (a.L + kT - 1) / kT;
    const int64_t n = int64_t(a.B) * a.G * tiles * kT * 2 * NP;
    if (n > 0) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_table<DT>), dim3(unsigned((n + kNT - 1) / kNT)), dim3(kNT), 0, st, a, NP, NW, tiles);
}
template <int DT, int NW, int W, bool VEC>
hipError_t run(const ScanArgs& a, const ScanRoute& r, hipStream_t st) {
    const dim3 grid(unsigned(int64_t(a.B) * a.chunks * a.G * r.blocks)), wg(64 * W);
    const size_t lds1 = size_t(4) * kT * kCh * 4, lds3 = lds1 + size_t(2) * W * kT * kCh * 4;
    if (hipError_t e = allow_lds<&k_scan<DT, NW, W, VEC, 3>>(lds3)) return e;
    run_table<DT>(a, NW * W, NW, st);
    if (a.chunks > 1) {
        const dim3 first(unsigned(int64_t(a.B) * (a.chunks - 1) * a.G * r.blocks));
        hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan<DT, NW, W, VEC, 1>), first, wg, lds1, st, a, r.blocks);
        if (!a.fold) {
            const unsigned join = unsigned((int64_t(a.B) * a.N * a.Dn + kJoinThreads - 1) / kJoinThreads);
            hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_join<false>), dim3(join), dim3(kJoinThreads), 0, st, a);
        }
    }
    hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan<DT, NW, W, VEC, 3>), grid, wg, lds3, st, a, r.blocks);
    return hipGetLastError();
}
template <int DT, int NW, int W, bool VEC>
hipError_t run_grad(const ScanArgs& a, const ScanRoute& r, hipStream_t st) {
    constexpr int NP = W * NW;
    const dim3 grid(unsigned(int64_t(a.B) * a.chunks * a.G * r.blocks));
    const size_t lds1 = size_t(2) * kT * kCh * 4, lds3 = size_t(3 * kT * kCh + 2 * kT * NP + 3 * W * kT * kCh) * 4;
    if (hipError_t e = allow_lds<&k_scan_grad<DT, NW, W, VEC, 3>>(lds3)) return e;
    run_table<DT>(a, NP, NW, st);
    if (a.chunks > 1) {
        const dim3 first(unsigned(int64_t(a.B) * (a.chunks - 1) * a.G * r.blocks));
        hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_grad<DT, NW, W, VEC, 1>), first, dim3(64 * W), lds1, st, a, r.blocks);
        if (!a.fold) {
            const unsigned join = unsigned((int64_t(a.B) * a.N * a.Dn + kJoinThreads - 1) / kJoinThreads);
            hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_join<true>), dim3(join), dim3(kJoinThreads), 0, st, a);
        }
    }
    hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_grad<DT, NW, W, VEC, 3>), grid, dim3(64 * W), lds3, st, a, r.blocks);
    const int64_t bc = 2 * int64_t(a.B) * a.L * a.G * a.N;
    if (bc > 0 && r.blocks > 1) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_bc<DT>), dim3(unsigned((bc + kNT - 1) / kNT)), dim3(kNT), 0, st, a, r.blocks);
    if (hipError_t e = hipGetLastError()) return e;
    return launch_column_sums(a.part, int64_t(a.B) * a.chunks, a.Dn, a.N, 2, a.dA, a.dD, a.ddelta_bias, st);
}
template <int DT, bool VEC>
hipError_t by_states(const ScanArgs& a, const ScanRoute& r, bool grad, hipStream_t st) {
    const int NP = scan_padded_states(a.N);
    if (grad) {
        switch (NP) {
            case 4: return run_grad<DT, 1, 4, VEC>(a, r, st);
            case 8: return run_grad<DT, 2, 4, VEC>(a, r, st);
            case 16: return run_grad<DT, 4, 4, VEC>(a, r, st);
            case 32: return run_grad<DT, 4, 8, VEC>(a, r, st);
            default: return run_grad<DT, 8, 8, VEC>(a, r, st);
        }
    }
    switch (NP) {
        case 4: return run<DT, 1, 4, VEC>(a, r, st);
        case 8: return run<DT, 1, 8, VEC>(a, r, st);
        case 16: return run<DT, 2, 8, VEC>(a, r, st);
        case 32: return run<DT, 4, 8, VEC>(a, r, st);
        default: return run<DT, 8, 8, VEC>(a, r, st);
    }
}
hipError_t by_type(const ScanArgs& a, const ScanRoute& r, int dtype, bool aligned, bool grad, hipStream_t st) {
    const bool vec = aligned && (a.Dn / a.G) % 4 == 0;
    switch (dtype) {
        case AUD_F32: return vec ? by_states<AUD_F32, true>(a, r, grad, st) : by_states<AUD_F32, false>(a, r, grad, st);
        case AUD_BF16: return vec ? by_states<AUD_BF16, true>(a, r, grad, st) : by_states<AUD_BF16, false>(a, r, grad, st);
        default: return vec ? by_states<AUD_F16, true>(a, r, grad, st) : by_states<AUD_F16, false>(a, r, grad, st);
    }
}

}  // namespace

int scan_padded_states(int N) { return N <= 4 ? 4 : N <= 8 ? 8 : N <= 16 ? 16 : N <= 32 ? 32 : 64; }

// Chunks of the time axis.  A cut axis is scanned twice, which costs 1.7 times the instructions (the first pass has no C, z and
// y); an uncut one keeps one workgroup a CU and needs enough of them.  Measured at 2048 steps of 64-channel workgroups
// (bfloat16, 16 states, MI355X, uncut 190 us then): 192 workgroups 217 / 216 / 220 us in 4 / 8 / 16 chunks; 64 workgroups 44 us of
// kernels in 16 chunks, 46 in 8, 78 in 4.  So: uncut from 170 workgroups on, else about 512 workgroups, chunks of four tiles at
// least.  A tile of the gradients takes three times as long: chunks of two
// tiles there (3 x 501 steps of 2 x 36 channels, values and gradients: 44 us, with four tiles 52).
ScanRoute scan_route(int B, int L, int D, int G, int N, bool grad) {
    ScanRoute r{};
    r.blocks = (D / G + kCh - 1) / kCh;
    const int tiles = L > 0 ? (L + kT - 1) / kT : 1;
    const bool wide = scan_padded_states(N) > 16;
    const int64_t wgs = int64_t(B) * G * r.blocks, want = 512, uncut = !grad ? 170 : wide ? 200 : 400;
    int64_t chunks = wgs >= uncut || wgs == 0 ? 1 : want / wgs;  // (rounded down: one workgroup too many costs a whole round)
    chunks = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(chunks, kMaxChunks), tiles / (grad ? 2 : 4)));
    r.chunk_tiles = int((tiles + chunks - 1) / chunks);
    r.chunks = (tiles + r.chunk_tiles - 1) / r.chunk_tiles;
    r.fold = r.chunks <= kFoldChunks || (r.chunks <= 2 * kFoldChunks && wgs * r.chunks <= 256);
    return r;
}
int64_t scan_sums_floats(const ScanRoute& r, int B, int D, int N) { return r.chunks > 1 ? int64_t(B) * r.chunks * (N + 1) * D : 0; }

hipError_t launch_scan(const ScanArgs& a, const ScanRoute& r, int dtype, bool aligned, hipStream_t st) {
    return by_type(a, r, dtype, aligned, false, st);
}
hipError_t launch_scan_grad(const ScanArgs& a, const ScanRoute& r, int dtype, bool aligned, hipStream_t st) {
    return by_type(a, r, dtype, aligned, true, st);
}
hipError_t launch_scan_step(const ScanArgs& a, int dtype, hipStream_t st) {
    const dim3 grid(unsigned((int64_t(a.B) * a.Dn * 4 + kNT - 1) / kNT));
    switch (dtype) {
        case AUD_F32: hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_step<AUD_F32>), grid, dim3(kNT), 0, st, a); break;
        case AUD_BF16: hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_step<AUD_BF16>), grid, dim3(kNT), 0, st, a); break;
        default: hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_step<AUD_F16>), grid, dim3(kNT), 0, st, a);
    }
    return hipGetLastError();
}

}  // namespace aud
