// Gradients of the selective scan (formulas, tiles and chunks: scan.hip).  A tile's states are worked out again from the kept
// ones in front of it and held in registers; then its steps are walked back.  W waves of NW states each.
#include "scan_common.h"

namespace aud {
namespace {

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
    const bool any = first < end;  // (no frame at all: the buffers may be null, nothing is pointed at)
    const int64_t row = (end - 1) * kT + pt, over = row < a.L ? 0 : row - (a.L - 1);
    const raw* pu = any ? static_cast<const raw*>(a.u) + u0 + (row - over) * a.ur + cc : nullptr;
    const raw* pd = any ? static_cast<const raw*>(a.delta) + e0 + (row - over) * a.er + cc : nullptr;
    const raw* pg = any ? static_cast<const raw*>(a.dy) + g0 + (row - over) * a.yr + cc : nullptr;
    const raw* pz = a.z && any ? static_cast<const raw*>(a.z) + z0 + (row - over) * a.zr + cc : pg;  // (no gate: read and not used)
    const int64_t su = kT * a.ur, sd = kT * a.er, sg = kT * a.yr, sz = a.z ? kT * a.zr : sg;
    const int64_t step_o = int64_t(kT) * a.Dn;
    const int lane_in = live ? lane : 0;
    // (the same for all lanes: states in front of the tile, results of its first row)
    const float* pk = PASS == 3 && any ? a.kept + ((int64_t(at.b) * tiles + (end - 1)) * a.N + wave * NW) * a.Dn + at.d0 : nullptr;
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
    if (any) {
        fetch();
        pu += over * a.ur, pd += over * a.er, pg += over * a.yr, pz += over * (a.z ? a.zr : a.yr);
    }
    ScalarTable bc =
        (ScalarTable)(any ? a.table + ((int64_t(at.b) * a.G + at.g) * tiles + (end - 1)) * kT * 2 * NP + wave * kT * 2 * NW : nullptr);
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
    const int64_t n = int64_t(a.B) * a.L * a.G * a.N, i = int64_t(a.first + blockIdx.x) * kNT + threadIdx.x;
    if (i >= 2 * n) return;
    const int64_t o = i < n ? i : i - n;
    const float* p = a.part_bc + (i < n ? 0 : blocks * n) + o;
    float s = 0.f;
    for (int k = 0; k < blocks; ++k) s += p[k * n];
    static_cast<typename Elem<DT>::raw*>(i < n ? a.dB : a.dC)[o] = Elem<DT>::down(s);
}

template <int DT, int NW, int W, bool VEC>
hipError_t run_grad(const ScanArgs& a, const ScanRoute& r, hipStream_t st) {
    constexpr int NP = W * NW;
    const int64_t side = int64_t(a.B) * a.G * r.blocks;  // workgroups side by side in a chunk
    const size_t lds1 = size_t(2) * kT * kCh * 4, lds3 = size_t(3 * kT * kCh + 2 * kT * NP + 3 * W * kT * kCh) * 4;
    if (hipError_t e = allow_lds<&k_scan_grad<DT, NW, W, VEC, 3>>(lds3)) return e;
    if (hipError_t e = run_table<DT>(a, NP, NW, st)) return e;
    if (a.chunks > 1) {
        if (hipError_t e = in_slices_of(a, side * (a.chunks - 1), 64 * W, [&](dim3 grid, const ScanArgs& s) {
                hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_grad<DT, NW, W, VEC, 1>), grid, dim3(64 * W), lds1, st, s, r.blocks);
            }))
            return e;
        if (!a.fold)
            if (hipError_t e = run_join<true>(a, st)) return e;
    }
    if (hipError_t e = in_slices_of(a, side * a.chunks, 64 * W, [&](dim3 grid, const ScanArgs& s) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_grad<DT, NW, W, VEC, 3>), grid, dim3(64 * W), lds3, st, s, r.blocks);
        }))
        return e;
    const int64_t bc = r.blocks > 1 ? 2 * int64_t(a.B) * a.L * a.G * a.N : 0;
    if (hipError_t e = in_slices_of(a, (bc + kNT - 1) / kNT, kNT, [&](dim3 grid, const ScanArgs& s) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_bc<DT>), grid, dim3(kNT), 0, st, s, r.blocks);
        }))
        return e;
    return launch_column_sums(a.part, int64_t(a.B) * a.chunks, a.Dn, a.N, 2, a.dA, a.dD, a.ddelta_bias, st);
}
template <int DT, bool VEC>
hipError_t by_states(const ScanArgs& a, const ScanRoute& r, hipStream_t st) {
    switch (scan_padded_states(a.N)) {
        case 4: return run_grad<DT, 1, 4, VEC>(a, r, st);
        case 8: return run_grad<DT, 2, 4, VEC>(a, r, st);
        case 16: return run_grad<DT, 4, 4, VEC>(a, r, st);
        case 32: return run_grad<DT, 4, 8, VEC>(a, r, st);
        default: return run_grad<DT, 8, 8, VEC>(a, r, st);
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

hipError_t launch_scan_grad(const ScanArgs& a, const ScanRoute& r, int dtype, bool aligned, hipStream_t st) {
    return by_type(a, r, dtype, aligned, st);
}

}  // namespace aud
