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
// state out from those, h' = exp(A sum dt) h + (final state) chunk by chunk, and is scanned from there.  The decay of a chunk
// may pass float32 (growing steps); its product with h is taken so that it does not.
//
// Steps at and behind lengths[b] have dt = 0: the state stays, y is zero, and what the inputs hold there has no effect.
//
// The vector pipe bounds it, not memory: a state and step is one exponential (8 cycles of a SIMD) and four products and fused
// products (4 cycles each), a channel and step about 50 more instructions (softplus, gate, conversions, the sum over the waves).
// 8 x 2048 x 1536, 16 states, bfloat16: 178 us, 204 MB (floor 40 us); 192 workgroups, one a CU, whose SIMDs issue vector
// instructions 75 % of the time.  Gradients, 4 x 2048 x 1024: 40 us the first scan, 122 the second (82 %), of 255 for values and
// gradients.  The first scans of a cut axis, 40 us each of values and of gradients there, issue 60 % of the time only; what they wait
// for in the rest (a barrier every 16 steps with little between, 448 workgroups on 256 CUs) was not taken apart.
//
// What was measured on the way to 178: B and C broadcast from LDS 243 us; scalar loads without a group in hand 638, as runs of 64
// bytes a group ahead 207; one barrier a tile instead of two 190; both elements of a thread side by side 186; addresses moved on by a
// tile, a turn of the loop for each LDS buffer 178.  Not taken: the steps' LDS reads a group ahead 182, the output of a tile behind
// the next one's scan 192, groups of half the size 194; inputs that lie still in the caches change nothing.
#include <type_traits>

#include "scan_common.h"

namespace aud {
namespace {

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
    if (tiles == 0) {  // no frame at all: the buffers may be null, so nothing below points into them
#pragma unroll
        for (int i = 0; i < NW; ++i)
            if (PASS == 3 && live && wave * NW + i < a.N && a.state_out) a.state_out[(int64_t(at.b) * a.Dn + d) * a.N + wave * NW + i] = h[i];
        return;
    }
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

// ---- one frame: four lanes a channel, a quarter of its states each ----------------------------------------------------
template <int DT>
__global__ void __launch_bounds__(kNT) k_scan_step(ScanArgs a) {
    const int64_t id = int64_t(a.first + blockIdx.x) * kNT + threadIdx.x, ch = id >> 2;
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

template <int DT, int NW, int W, bool VEC>
hipError_t run(const ScanArgs& a, const ScanRoute& r, hipStream_t st) {
    const int64_t side = int64_t(a.B) * a.G * r.blocks;  // workgroups side by side in a chunk
    const dim3 wg(64 * W);
    const size_t lds1 = size_t(4) * kT * kCh * 4, lds3 = lds1 + size_t(2) * W * kT * kCh * 4;
    if (hipError_t e = allow_lds<&k_scan<DT, NW, W, VEC, 3>>(lds3)) return e;
    if (hipError_t e = run_table<DT>(a, NW * W, NW, st)) return e;
    if (a.chunks > 1) {
        if (hipError_t e = in_slices_of(a, side * (a.chunks - 1), 64 * W, [&](dim3 grid, const ScanArgs& s) {
                hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan<DT, NW, W, VEC, 1>), grid, wg, lds1, st, s, r.blocks);
            }))
            return e;
        if (!a.fold)
            if (hipError_t e = run_join<false>(a, st)) return e;
    }
    return in_slices_of(a, side * a.chunks, 64 * W, [&](dim3 grid, const ScanArgs& s) {
        hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan<DT, NW, W, VEC, 3>), grid, wg, lds3, st, s, r.blocks);
    });
}
template <int DT, bool VEC>
hipError_t by_states(const ScanArgs& a, const ScanRoute& r, hipStream_t st) {
    switch (scan_padded_states(a.N)) {
        case 4: return run<DT, 1, 4, VEC>(a, r, st);
        case 8: return run<DT, 1, 8, VEC>(a, r, st);
        case 16: return run<DT, 2, 8, VEC>(a, r, st);
        case 32: return run<DT, 4, 8, VEC>(a, r, st);
        default: return run<DT, 8, 8, VEC>(a, r, st);
    }
}
hipError_t by_type(const ScanArgs& a, const ScanRoute& r, int dtype, bool aligned, hipStream_t st) {
    const bool vec = aligned && (a.Dn / a.G) % 4 == 0;
    switch (dtype) {
        case AUD_F32: return vec ? by_states<AUD_F32, true>(a, r, st) : by_states<AUD_F32, false>(a, r, st);
        case AUD_BF16: return vec ? by_states<AUD_BF16, true>(a, r, st) : by_states<AUD_BF16, false>(a, r, st);
        default: return vec ? by_states<AUD_F16, true>(a, r, st) : by_states<AUD_F16, false>(a, r, st);
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
    return by_type(a, r, dtype, aligned, st);
}
hipError_t launch_scan_step(const ScanArgs& a, int dtype, hipStream_t st) {
    return in_slices_of(a, (int64_t(a.B) * a.Dn * 4 + kNT - 1) / kNT, kNT, [&](dim3 grid, const ScanArgs& s) {
        switch (dtype) {
            case AUD_F32: hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_step<AUD_F32>), grid, dim3(kNT), 0, st, s); break;
            case AUD_BF16: hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_step<AUD_BF16>), grid, dim3(kNT), 0, st, s); break;
            default: hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_step<AUD_F16>), grid, dim3(kNT), 0, st, s);
        }
    });
}

}  // namespace aud
