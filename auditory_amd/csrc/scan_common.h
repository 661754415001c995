// Shared by the selective scan's values (scan.hip, which states the formulas and the plan) and gradients (scan_grad.hip): the
// tables of B and C and the scalar loads that read them, tiles in LDS, the chunks of the time axis and how they are joined.
#pragma once
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

// 2^x h + part, x the exponent of a whole run of steps.  A run of growing steps can pass float32 where its product with a small h
// does not, and h = 0 stays 0 whatever it is multiplied by: what x has above 120 goes into h first, by powers of two.  (500: more
// than that takes the smallest h there is past float32.)  The joins take the plain form, which ends in an infinity or NaN where this
// one is wanted (neither goes away again), and only then this one: in every step it costs the join of 64 chunks 2 us of 6.
__device__ __forceinline__ float carried(float x, float h, float part) {
    const float y = x > 500.f ? 500.f : x;
    const int n = y > 120.f ? int(ceilf(y - 120.f)) : 0;
    return fmaf(exp2_hw(y - float(n)), ldexpf(h, n), part);
}
__device__ __forceinline__ bool finite(float v) { return fabsf(v) <= 3.402823466e38f; }

struct Where {  // which channels, chunk and item a workgroup has
    int b, chunk, g, d0, dn, block;  // first channel, channels (<= 64), block within the group
    // (the first pass leaves the last chunk out, the gradients' first pass the first one)
    __device__ __forceinline__ Where(const ScanArgs& a, int blocks, int skip_last, int skip_first) {
        int id = a.first + blockIdx.x;
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
    const int64_t i = int64_t(a.first + blockIdx.x) * kNT + threadIdx.x;
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
    auto slot_of = [&](int k) { return BACK ? a.chunks - 1 - k : (at.chunk > 0 ? 1 + k : 0); };
    auto chunk_of = [&](int slot) { return BACK ? slot : (slot > 0 ? slot - 1 : 0); };
    for (int k = 0; k < count; k += kAhead) {
        float part[kAhead][NW], sum[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int slot = slot_of(k + j < count ? k + j : count - 1);
            sum[j] = dt[int64_t(chunk_of(slot)) * a.Dn];
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
    bool plain = true;
#pragma unroll
    for (int i = 0; i < NW; ++i) plain = plain && finite(h[i]);
    if (!plain) {  // once more, slot by slot
        for (int k = 0; k < count; ++k) {
            const int slot = slot_of(k);
            const float sum = dt[int64_t(chunk_of(slot)) * a.Dn];
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                const float part = n0 + i < a.N ? s[slot * per + int64_t(n0 + i) * a.Dn] : 0.f;
                h[i] = k == 0 ? part : carried(sum * A2[i], h[i], part);
            }
        }
    }
}

// many chunks: the same once for all of them, slot by slot in place (sixteen at once)
template <bool BACK>
__global__ void __launch_bounds__(kJoinThreads) k_scan_join(ScanArgs a) {
    constexpr int kAhead = 16;
    const int64_t id = int64_t(a.first + blockIdx.x) * kJoinThreads + threadIdx.x, per = int64_t(a.N) * a.Dn;
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
        const float before = h;
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int kk = k + j < a.chunks - 1 ? k + j : a.chunks - 2, slot = BACK ? a.chunks - 1 - kk : 1 + kk;
            mine[j] = s[slot * per];
            sum[j] = dt[int64_t(BACK ? slot : slot - 1) * a.Dn];
        }
        auto walk = [&](auto join) {
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                if (k + j >= a.chunks - 1) break;
                const int slot = BACK ? a.chunks - 1 - (k + j) : 1 + k + j;
                h = k + j == 0 ? mine[j] : join(sum[j] * A2, h, mine[j]);
                s[slot * per] = h;
            }
        };
        walk([](float x, float v, float part) { return fmaf(exp2_hw(x), v, part); });
        if (finite(h)) continue;
        h = before;
        walk([](float x, float v, float part) { return carried(x, v, part); });
    }
}

template <bool BACK>
hipError_t run_join(const ScanArgs& a, hipStream_t st) {
    return in_slices_of(a, (int64_t(a.B) * a.N * a.Dn + kJoinThreads - 1) / kJoinThreads, kJoinThreads, [&](dim3 grid, const ScanArgs& s) {
        hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_join<BACK>), grid, dim3(kJoinThreads), 0, st, s);
    });
}

template <int DT>
hipError_t run_table(const ScanArgs& a, int NP, int NW, hipStream_t st) {
    const int tiles = (a.L + kT - 1) / kT;
    const int64_t n = int64_t(a.B) * a.G * tiles * kT * 2 * NP;
    return in_slices_of(a, (n + kNT - 1) / kNT, kNT, [&](dim3 grid, const ScanArgs& s) {
        hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_table<DT>), grid, dim3(kNT), 0, st, s, NP, NW, tiles);
    });
}

}  // namespace
}  // namespace aud
