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
// A workgroup of four waves owns 64 channels of an item: a lane is a channel, a wave a quarter of the states.  Tiles of 16
// steps go through LDS: all threads turn u and delta into (dt, dt u), each wave runs its states over the tile, all threads
// add the four waves' partial sums up and store.
//
// Where items x channels leave the card idle, the time axis is cut into chunks: (1) every chunk is scanned from a zero state
// for its final state and its sum of dt, (2) the chunks are joined in order, h' = exp(A sum dt) h + (its final state), (3) every
// chunk is scanned from its true state.
//
// Steps at and behind lengths[b] have dt = 0: the state stays, y is zero, and what the inputs hold there has no effect.
#include "frame_ops.h"

namespace aud {
namespace {

constexpr int kNT = 256, kT = kScanTile, kCh = 64;

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

struct Where {  // which channels, chunk and item a workgroup has
    int b, chunk, g, d0, dn, block;  // first channel, channels (<= 64), block within the group
    __device__ __forceinline__ Where(const ScanArgs& a, int blocks) {
        int id = blockIdx.x;
        block = id % blocks;
        id /= blocks;
        g = id % a.G;
        id /= a.G;
        chunk = id % a.chunks;
        b = id / a.chunks;
        const int dg = a.Dn / a.G;
        d0 = g * dg + block * kCh;
        dn = dg - block * kCh < kCh ? dg - block * kCh : kCh;
    }
};

// Four channels (c4 .. c4 + 3 of the block) of one step, as float32; channels past the block read as 0
template <int DT, bool VEC>
__device__ __forceinline__ void load4(const void* base, int64_t at, int c4, int dn, float (&f)[4]) {
    if constexpr (VEC) {
        if (c4 < dn) return unpack<DT, 4>(load_pack<DT, 4>(base, at + c4), f);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = 0.f;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = c4 + i < dn ? Elem<DT>::up(static_cast<const typename Elem<DT>::raw*>(base)[at + c4 + i]) : 0.f;
    }
}
template <int DT, bool VEC>
__device__ __forceinline__ void store4(void* base, int64_t at, int c4, int dn, const float (&f)[4]) {
    if constexpr (VEC) {
        if (c4 < dn) store_pack<DT, 4>(base, at + c4, f);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c4 + i < dn) static_cast<typename Elem<DT>::raw*>(base)[at + c4 + i] = Elem<DT>::down(f[i]);
    }
}

// dt of a step and its slope d dt / d delta
__device__ __forceinline__ float step_size(float raw, int softp) { return softp ? softplus(raw) : raw; }

// B or C of a tile -> dst [16][NP] float32; states past N and steps past the tile read as 0
template <int DT, int NP>
__device__ __forceinline__ void stage_states(const void* base, int64_t item, int64_t row, int N, int t0, int steps, float* dst) {
    for (int i = threadIdx.x; i < kT * NP; i += kNT) {
        const int t = i / NP, n = i % NP;
        dst[i] = t < steps && n < N ? Elem<DT>::up(static_cast<const typename Elem<DT>::raw*>(base)[item + int64_t(t0 + t) * row + n]) : 0.f;
    }
}

// ---- values.  PASS 1: a chunk's final state from zero and its sum of dt; PASS 3: y ------------------------------------
template <int DT, int NW, bool VEC, int PASS>
__global__ void __launch_bounds__(kNT) k_scan(ScanArgs a, int blocks) {
    constexpr int NP = 4 * NW;
    float* lds = reinterpret_cast<float*>(dyn_lds());
    float2* s_step = reinterpret_cast<float2*>(lds);  // [16][64] (dt, dt u)
    float* s_b = lds + 2 * kT * kCh;                  // [16][NP]
    float* s_c = s_b + kT * NP;
    float* s_y = s_c + kT * NP;                       // [4][16][64]
    const Where at(a, blocks);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int pt = tid >> 4, c4 = (tid & 15) * 4;     // this thread's step and channels when the tile is loaded and stored
    const int len = item_rows(a.lengths, at.b, a.L), tiles = (a.L + kT - 1) / kT;
    const int64_t u0 = at.b * a.ui + at.d0, e0 = at.b * a.ei + at.d0, z0 = at.b * a.zi + at.d0;
    const int64_t b0 = at.b * a.bi + at.g * a.N, c0 = at.b * a.ci + at.g * a.N, y0 = int64_t(at.b) * a.L * a.Dn + at.d0;
    const int d = at.d0 + lane;
    const bool live = lane < at.dn;
    float A2[NW], h[NW], sum_dt = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        const int n = wave * NW + i;
        const bool there = live && n < a.N;
        A2[i] = there ? a.A[int64_t(d) * a.N + n] * kLog2e : 0.f;
        h[i] = 0.f;
        if (PASS == 3 && there) {
            if (a.chunks > 1) h[i] = a.sums[((int64_t(at.b) * a.chunks + at.chunk) * a.N + n) * a.Dn + d];
            else if (a.state) h[i] = a.state[(int64_t(at.b) * a.Dn + d) * a.N + n];
        }
    }
    float skip[4], bias[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool there = c4 + i < at.dn;
        skip[i] = there && a.D ? a.D[at.d0 + c4 + i] : 0.f;
        bias[i] = there && a.delta_bias ? a.delta_bias[at.d0 + c4 + i] : 0.f;
    }
    const int first = at.chunk * a.chunk_tiles, end = first + a.chunk_tiles < tiles ? first + a.chunk_tiles : tiles;
    for (int tile = first; tile < end; ++tile) {
        const int t0 = tile * kT, t = t0 + pt;
        float u[4], dl[4], z[4];
        if (t < a.L) {
            load4<DT, VEC>(a.u, u0 + int64_t(t) * a.ur, c4, at.dn, u);
            load4<DT, VEC>(a.delta, e0 + int64_t(t) * a.er, c4, at.dn, dl);
            if (PASS == 3 && a.z) load4<DT, VEC>(a.z, z0 + int64_t(t) * a.zr, c4, at.dn, z);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool on = t < len;
            const float dt = on ? step_size(dl[i] + bias[i], a.softplus) : 0.f;
            s_step[pt * kCh + c4 + i] = float2{dt, on ? dt * u[i] : 0.f};
        }
        const int steps = len - t0;  // (may be negative)
        stage_states<DT, NP>(a.Bm, b0, a.br, a.N, t0, steps, s_b);
        if (PASS == 3) stage_states<DT, NP>(a.Cm, c0, a.cr, a.N, t0, steps, s_c);
        if (PASS == 3 && a.kept && live) {
#pragma unroll
            for (int i = 0; i < NW; ++i)
                if (wave * NW + i < a.N) a.kept[((int64_t(at.b) * tiles + tile) * a.N + wave * NW + i) * a.Dn + d] = h[i];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kT; ++k) {
            const float2 s = s_step[k * kCh + lane];
            float y = 0.f;
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                h[i] = fmaf(exp2_hw(s.x * A2[i]), h[i], s.y * s_b[k * NP + wave * NW + i]);
                if (PASS == 3) y = fmaf(s_c[k * NP + wave * NW + i], h[i], y);
            }
            if (PASS == 3) s_y[(wave * kT + k) * kCh + lane] = y;
            else sum_dt += s.x;
        }
        __syncthreads();
        if (PASS == 3 && t < a.L) {
            float y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float* p = s_y + pt * kCh + c4 + i;
                float v = (p[0] + p[kT * kCh]) + (p[2 * kT * kCh] + p[3 * kT * kCh]);
                v = fmaf(skip[i], u[i], v);
                if (a.z) v *= z[i] * fast_sigmoid(z[i]);
                y[i] = t < len ? v : 0.f;
            }
            store4<DT, VEC>(a.y, y0 + int64_t(t) * a.Dn, c4, at.dn, y);
        }
    }
    if (!live) return;
    float* dt_sums = a.sums + int64_t(a.B) * a.chunks * a.N * a.Dn;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        const int n = wave * NW + i;
        if (n >= a.N) continue;
        if (PASS == 1) a.sums[((int64_t(at.b) * a.chunks + at.chunk) * a.N + n) * a.Dn + d] = h[i];
        else if (a.chunks == 1 && a.state_out) a.state_out[(int64_t(at.b) * a.Dn + d) * a.N + n] = h[i];
    }
    if (PASS == 1 && wave == 0) dt_sums[(int64_t(at.b) * a.chunks + at.chunk) * a.Dn + d] = sum_dt;
}

// the chunks joined in order: sums[chunk] <- the state in front of it.  BACK: from the last chunk to the first, for the
// gradient that a chunk receives from behind
template <bool BACK>
__global__ void __launch_bounds__(kNT) k_scan_join(ScanArgs a) {
    const int64_t i = int64_t(blockIdx.x) * kNT + threadIdx.x, per = int64_t(a.N) * a.Dn;
    if (i >= a.B * per) return;
    const int64_t b = i / per;
    const int n = int(i % per / a.Dn), d = int(i % a.Dn);
    const float A2 = a.A[int64_t(d) * a.N + n] * kLog2e;
    float* s = a.sums + b * a.chunks * per + int64_t(n) * a.Dn + d;
    const float* dt = a.sums + int64_t(a.B) * a.chunks * per + b * a.chunks * a.Dn + d;
    const int64_t own = (b * a.Dn + d) * a.N + n;
    const float* in = BACK ? a.dstate_out : a.state;
    float h = in ? in[own] : 0.f;
    for (int k = 0; k < a.chunks; ++k) {
        const int c = BACK ? a.chunks - 1 - k : k;
        const float mine = s[c * per];
        s[c * per] = h;
        h = fmaf(exp2_hw(dt[int64_t(c) * a.Dn] * A2), h, mine);
    }
    float* out = BACK ? a.dstate : a.state_out;
    if (out) out[own] = h;
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

// ---- gradients.  PASS 1: what a chunk hands to the one in front of it, from a zero carry, and its sum of dt; PASS 3: all ----
template <int DT, int NW, bool VEC, int PASS>
__global__ void __launch_bounds__(kNT) k_scan_grad(ScanArgs a, int blocks) {
    constexpr int NP = 4 * NW, TS = NW <= 4 ? 16 : 64 / NW, SUBS = kT / TS;  // steps whose states are in registers at once
    float* lds = reinterpret_cast<float*>(dyn_lds());
    float* s_dt = lds;                      // [16][64] each
    float* s_du = s_dt + kT * kCh;          // dt u
    float* s_f = s_du + kT * kCh;
    float* s_b = s_f + kT * kCh;            // [16][NP] each
    float* s_c = s_b + kT * NP;
    float* s_db = s_c + kT * NP;
    float* s_dc = s_db + kT * NP;
    float* s_sum = s_dc + kT * NP;          // [3][4][16][64]: sum_n g B, sum_n A a h g, sum_n C h of each wave
    const Where at(a, blocks);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int pt = tid >> 4, c4 = (tid & 15) * 4;
    const int len = item_rows(a.lengths, at.b, a.L), tiles = (a.L + kT - 1) / kT;
    const int64_t u0 = at.b * a.ui + at.d0, e0 = at.b * a.ei + at.d0, z0 = at.b * a.zi + at.d0, g0 = at.b * a.yi + at.d0;
    const int64_t b0 = at.b * a.bi + at.g * a.N, c0 = at.b * a.ci + at.g * a.N, o0 = int64_t(at.b) * a.L * a.Dn + at.d0;
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
        if (PASS == 3 && there) {
            if (a.chunks > 1) carry[i] = a.sums[((int64_t(at.b) * a.chunks + at.chunk) * a.N + n) * a.Dn + d];
            else if (a.dstate_out) carry[i] = a.dstate_out[(int64_t(at.b) * a.Dn + d) * a.N + n];
        }
    }
    float skip[4], bias[4], sum_fu[4] = {0.f, 0.f, 0.f, 0.f}, sum_dd[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool there = c4 + i < at.dn;
        skip[i] = there && a.D ? a.D[at.d0 + c4 + i] : 0.f;
        bias[i] = there && a.delta_bias ? a.delta_bias[at.d0 + c4 + i] : 0.f;
    }
    const int first = at.chunk * a.chunk_tiles, end = first + a.chunk_tiles < tiles ? first + a.chunk_tiles : tiles;
    for (int tile = end - 1; tile >= first; --tile) {
        const int t0 = tile * kT, t = t0 + pt, steps = len - t0;
        const bool on = t < len;
        float u[4], dl[4], z[4], dy[4], dt[4], f[4];
        if (on) {
            if (PASS == 3) load4<DT, VEC>(a.u, u0 + int64_t(t) * a.ur, c4, at.dn, u);
            load4<DT, VEC>(a.delta, e0 + int64_t(t) * a.er, c4, at.dn, dl);
            if (a.z) load4<DT, VEC>(a.z, z0 + int64_t(t) * a.zr, c4, at.dn, z);
            load4<DT, VEC>(a.dy, g0 + int64_t(t) * a.yr, c4, at.dn, dy);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (!on) u[i] = dl[i] = z[i] = dy[i] = 0.f;
            if (PASS == 1) u[i] = 0.f;
            dt[i] = on ? step_size(dl[i] + bias[i], a.softplus) : 0.f;
            f[i] = a.z ? dy[i] * (z[i] * fast_sigmoid(z[i])) : dy[i];
            const int s = pt * kCh + c4 + i;
            s_dt[s] = dt[i];
            if (PASS == 3) s_du[s] = dt[i] * u[i];
            s_f[s] = f[i];
        }
        if (PASS == 3) stage_states<DT, NP>(a.Bm, b0, a.br, a.N, t0, steps, s_b);
        stage_states<DT, NP>(a.Cm, c0, a.cr, a.N, t0, steps, s_c);
        float h0[NW];
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            const int n = wave * NW + i;
            h0[i] = PASS == 3 && live && n < a.N ? a.kept[((int64_t(at.b) * tiles + tile) * a.N + n) * a.Dn + d] : 0.f;
        }
        __syncthreads();
        if constexpr (PASS == 1) {
#pragma unroll
            for (int k = kT - 1; k >= 0; --k) {
                const float s = s_dt[k * kCh + lane], fk = s_f[k * kCh + lane];
                sum_dt += s;
#pragma unroll
                for (int i = 0; i < NW; ++i)
                    carry[i] = exp2_hw(s * A2[i]) * fmaf(fk, s_c[k * NP + wave * NW + i], carry[i]);
            }
        } else {
            for (int sub = SUBS - 1; sub >= 0; --sub) {
                float h[NW], hs[TS][NW], as[TS][NW];  // states behind and decays of the steps of this part of the tile
#pragma unroll
                for (int i = 0; i < NW; ++i) h[i] = h0[i];
                if constexpr (SUBS > 1)
                    for (int k = 0; k < sub * TS; ++k)
#pragma unroll
                        for (int i = 0; i < NW; ++i)
                            h[i] = fmaf(exp2_hw(s_dt[k * kCh + lane] * A2[i]), h[i], s_du[k * kCh + lane] * s_b[k * NP + wave * NW + i]);
                float before[NW];
#pragma unroll
                for (int i = 0; i < NW; ++i) before[i] = h[i];
#pragma unroll
                for (int k = 0; k < TS; ++k) {
                    const int kk = sub * TS + k;
                    const float s = s_dt[kk * kCh + lane], x = s_du[kk * kCh + lane];
                    float v = 0.f;
#pragma unroll
                    for (int i = 0; i < NW; ++i) {
                        as[k][i] = exp2_hw(s * A2[i]);
                        h[i] = fmaf(as[k][i], h[i], x * s_b[kk * NP + wave * NW + i]);
                        hs[k][i] = h[i];
                        v = fmaf(s_c[kk * NP + wave * NW + i], h[i], v);
                    }
                    s_sum[((2 * 4 + wave) * kT + kk) * kCh + lane] = v;
                }
#pragma unroll
                for (int k = TS - 1; k >= 0; --k) {
                    const int kk = sub * TS + k;
                    const float s = s_dt[kk * kCh + lane], x = s_du[kk * kCh + lane], fk = s_f[kk * kCh + lane];
                    float gb = 0.f, ahg = 0.f;
#pragma unroll
                    for (int i = 0; i < NW; ++i) {
                        const float g = fmaf(fk, s_c[kk * NP + wave * NW + i], carry[i]);
                        gb = fmaf(g, s_b[kk * NP + wave * NW + i], gb);
                        carry[i] = as[k][i] * g;
                        const float r = carry[i] * (k > 0 ? hs[k > 0 ? k - 1 : 0][i] : before[i]);
                        ahg = fmaf(An[i], r, ahg);
                        dA[i] = fmaf(s, r, dA[i]);
                        float pb = live ? g * x : 0.f, pc = live ? fk * hs[k][i] : 0.f;
                        for (int m = 1; m < 64; m <<= 1) {
                            pb += __shfl_xor(pb, m);
                            pc += __shfl_xor(pc, m);
                        }
                        if (lane == 0) {
                            s_db[kk * NP + wave * NW + i] = pb;
                            s_dc[kk * NP + wave * NW + i] = pc;
                        }
                    }
                    s_sum[((0 * 4 + wave) * kT + kk) * kCh + lane] = gb;
                    s_sum[((1 * 4 + wave) * kT + kk) * kCh + lane] = ahg;
                }
            }
        }
        __syncthreads();
        if constexpr (PASS == 3) {
            if (t < a.L) {
                float du[4], dd[4], dz[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float sums[3];
#pragma unroll
                    for (int k = 0; k < 3; ++k) {
                        const float* p = s_sum + (k * 4 * kT + pt) * kCh + c4 + i;
                        sums[k] = (p[0] + p[kT * kCh]) + (p[2 * kT * kCh] + p[3 * kT * kCh]);
                    }
                    const float ddt = fmaf(u[i], sums[0], sums[1]);
                    du[i] = fmaf(dt[i], sums[0], skip[i] * f[i]);
                    dd[i] = on ? ddt * (a.softplus ? fast_sigmoid(dl[i] + bias[i]) : 1.f) : 0.f;
                    const float q = fast_sigmoid(z[i]);
                    dz[i] = dy[i] * fmaf(skip[i], u[i], sums[2]) * (q * (1.f + z[i] * (1.f - q)));
                    sum_fu[i] = fmaf(f[i], u[i], sum_fu[i]);
                    sum_dd[i] += dd[i];
                    if (!on) du[i] = dz[i] = 0.f;
                }
                const int64_t o = o0 + int64_t(t) * a.Dn;
                store4<DT, VEC>(a.du, o, c4, at.dn, du);
                store4<DT, VEC>(a.ddelta, o, c4, at.dn, dd);
                if (a.dz) store4<DT, VEC>(a.dz, o, c4, at.dn, dz);
            }
            // dB, dC of the tile, summed over this block's channels
            const int64_t table = int64_t(blocks) * a.B * a.L * a.G * a.N;
            for (int i = tid; i < kT * NP; i += kNT) {
                const int k = i / NP, n = i % NP;
                if (n >= a.N || t0 + k >= a.L) continue;
                const int64_t o = (((int64_t(at.block) * a.B + at.b) * a.L + t0 + k) * a.G + at.g) * a.N + n;
                const bool there = k < steps;
                a.part_bc[o] = there ? s_db[i] : 0.f;
                a.part_bc[table + o] = there ? s_dc[i] : 0.f;
            }
            __syncthreads();
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
        float* row = a.part + (int64_t(at.b) * a.chunks + at.chunk) * (a.N + 2) * a.Dn;
        if (live) {
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                const int n = wave * NW + i;
                if (n >= a.N) continue;
                row[int64_t(n) * a.Dn + d] = dA[i];
                if (a.chunks == 1 && a.dstate) a.dstate[(int64_t(at.b) * a.Dn + d) * a.N + n] = carry[i];
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s_dt[pt * kCh + c4 + i] = sum_fu[i];
            s_du[pt * kCh + c4 + i] = sum_dd[i];
        }
        __syncthreads();
        if (tid < 2 * kCh && lane < at.dn) {
            const float* p = (wave == 0 ? s_dt : s_du) + lane;
            float s = 0.f;
            for (int k = 0; k < kT; ++k) s += p[k * kCh];
            row[int64_t(a.N + wave) * a.Dn + d] = s;
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

template <int DT, int NW, bool VEC>
hipError_t run(const ScanArgs& a, const ScanRoute& r, bool grad, hipStream_t st) {
    constexpr int NP = 4 * NW;
    const dim3 grid(unsigned(int64_t(a.B) * a.chunks * a.G * r.blocks));
    const unsigned join = unsigned((int64_t(a.B) * a.N * a.Dn + kNT - 1) / kNT);
    if (!grad) {
        const size_t lds = size_t(2 * kT * kCh + 2 * kT * NP + 4 * kT * kCh) * 4;
        if (a.chunks > 1) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan<DT, NW, VEC, 1>), grid, dim3(kNT), lds, st, a, r.blocks);
            hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_join<false>), dim3(join), dim3(kNT), 0, st, a);
        }
        hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan<DT, NW, VEC, 3>), grid, dim3(kNT), lds, st, a, r.blocks);
        return hipGetLastError();
    }
    const size_t lds = size_t(3 * kT * kCh + 4 * kT * NP + 12 * kT * kCh) * 4;
    if (lds > 64 * 1024) {
        if (hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&k_scan_grad<DT, NW, VEC, 3>),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024)) return e;
        if (hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&k_scan_grad<DT, NW, VEC, 1>),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024)) return e;
    }
    if (a.chunks > 1) {
        hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_grad<DT, NW, VEC, 1>), grid, dim3(kNT), lds, st, a, r.blocks);
        hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_join<true>), dim3(join), dim3(kNT), 0, st, a);
    }
    hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_grad<DT, NW, VEC, 3>), grid, dim3(kNT), lds, st, a, r.blocks);
    const int64_t bc = 2 * int64_t(a.B) * a.L * a.G * a.N;
    if (bc > 0) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_bc<DT>), dim3(unsigned((bc + kNT - 1) / kNT)), dim3(kNT), 0, st, a, r.blocks);
    if (hipError_t e = hipGetLastError()) return e;
    return launch_column_sums(a.part, int64_t(a.B) * a.chunks, a.Dn, a.N, 2, a.dA, a.dD, a.ddelta_bias, st);
}
template <int DT, bool VEC>
hipError_t by_states(const ScanArgs& a, const ScanRoute& r, bool grad, hipStream_t st) {
    if (a.N <= 4) return run<DT, 1, VEC>(a, r, grad, st);
    if (a.N <= 8) return run<DT, 2, VEC>(a, r, grad, st);
    if (a.N <= 16) return run<DT, 4, VEC>(a, r, grad, st);
    if (a.N <= 32) return run<DT, 8, VEC>(a, r, grad, st);
    return run<DT, 16, VEC>(a, r, grad, st);
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

// chunks of the time axis: until there are about 1024 workgroups, four tiles a chunk at least (a cut axis is scanned twice)
ScanRoute scan_route(int B, int L, int D, int G, int) {
    ScanRoute r{};
    r.blocks = (D / G + kCh - 1) / kCh;
    const int tiles = L > 0 ? (L + kT - 1) / kT : 1;
    const int64_t wgs = int64_t(B) * G * r.blocks;
    int64_t chunks = wgs > 0 ? 1024 / wgs : 1;
    chunks = std::max<int64_t>(1, std::min<int64_t>(chunks, tiles / 4));
    r.chunk_tiles = int((tiles + chunks - 1) / chunks);
    r.chunks = (tiles + r.chunk_tiles - 1) / r.chunk_tiles;
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
