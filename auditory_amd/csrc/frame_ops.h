// Shared by the feature-map and frame-sequence operators (group_norm, causal_conv, scan, scan_grad .hip): the element types of
// their activations (float32, bfloat16, float16 -- parameters, statistics, states and every sum are float32), packed loads
// and stores, the activation functions with their derivatives, and the launch descriptors.
#pragma once
#include <algorithm>
#include <atomic>

#include "kernels.h"

namespace aud {

// an index into a table of LDS: the CPU thread emulator's build ends the process where it is outside
#if defined(__clang__)
#define AUD_IN_TABLE(at, size) ((void)0)
#else
#define AUD_IN_TABLE(at, size) ((at) >= 0 && (at) < (size) ? (void)0 : std::abort())
#endif

// ---- element types: `raw` as stored, up() exact to float32, down() rounds to nearest even ------------------------------
template <int DT>
struct Elem;
template <>
struct Elem<AUD_F32> {
    typedef float raw;
    static __device__ __forceinline__ float up(raw v) { return v; }
    static __device__ __forceinline__ raw down(float v) { return v; }
};
template <>
struct Elem<AUD_BF16> {
    typedef uint16_t raw;
    static __device__ __forceinline__ float up(raw v) { return __uint_as_float(unsigned(v) << 16); }
    static __device__ __forceinline__ raw down(float v) {
#if defined(__clang__)
        return __builtin_bit_cast(raw, static_cast<__bf16>(v));
#else  // (the CPU thread emulator is built with g++)
        unsigned u = __float_as_uint(v);
        if ((u & 0x7FFFFFFFu) > 0x7F800000u) return raw((u >> 16) | 0x40u);
        return raw((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
#endif
    }
};
template <>
struct Elem<AUD_F16> {
    typedef uint16_t raw;
#if defined(__clang__)
    static __device__ __forceinline__ float up(raw v) { return float(__builtin_bit_cast(_Float16, v)); }
    static __device__ __forceinline__ raw down(float v) { return __builtin_bit_cast(raw, static_cast<_Float16>(v)); }
#else
    static float up(raw v) { return aud_emul::half_to_float(v); }
    static raw down(float v) { return aud_emul::float_to_half(v); }
#endif
};

// V consecutive elements moved as one access (V sizeof(raw) bytes, aligned to that)
template <int DT, int V>
struct alignas(V * sizeof(typename Elem<DT>::raw)) Pack {
    typename Elem<DT>::raw v[V];
};
template <int DT, int V>
__device__ __forceinline__ Pack<DT, V> load_pack(const void* base, int64_t element) {
    return *reinterpret_cast<const Pack<DT, V>*>(static_cast<const typename Elem<DT>::raw*>(base) + element);
}
template <int DT, int V>
__device__ __forceinline__ void store_pack(void* base, int64_t element, const float (&f)[V]) {
    Pack<DT, V> p;
#pragma unroll
    for (int i = 0; i < V; ++i) p.v[i] = Elem<DT>::down(f[i]);
    *reinterpret_cast<Pack<DT, V>*>(static_cast<typename Elem<DT>::raw*>(base) + element) = p;
}
template <int DT, int V>
__device__ __forceinline__ void unpack(const Pack<DT, V>& p, float (&f)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = Elem<DT>::up(p.v[i]);
}

// ---- elementary functions on the hardware's base-2 exponential, base-2 logarithm and reciprocal (1 ulp each) -----------
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
__device__ __forceinline__ float fast_sigmoid(float x) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-kLog2e * x)); }
// log(1 + e^x) = max(x, 0) + log1p(e^-|x|); log1p(e) for small e as e log(w) / (w - 1), w = 1 + e rounded: the rounding of w
// cancels in the quotient, so the result is good to a few ulp however small e is
__device__ __forceinline__ float softplus(float x) {
    const float e = __builtin_amdgcn_exp2f(-kLog2e * fabsf(x));
    const float w = 1.f + e, d = w - 1.f;
    const float l = kLn2 * __builtin_amdgcn_logf(w) * (e * __builtin_amdgcn_rcpf(fmaxf(d, 1e-30f)));
    return fmaxf(x, 0.f) + (d > 0.f ? l : e);
}
template <int ACT>
__device__ __forceinline__ float act_value(float p) {
    if constexpr (ACT == AUD_ACT_RELU) return p > 0.f ? p : (p != p ? p : 0.f);  // NaN stays NaN
    else if constexpr (ACT == AUD_ACT_SILU) return p * fast_sigmoid(p);
    else if constexpr (ACT == AUD_ACT_GELU) return 0.5f * p * (1.f + erff(p * 0.70710678118654752f));
    else return p;
}
template <int ACT>
__device__ __forceinline__ float act_slope(float p) {
    if constexpr (ACT == AUD_ACT_RELU) return p > 0.f ? 1.f : 0.f;
    else if constexpr (ACT == AUD_ACT_SILU) {
        const float q = fast_sigmoid(p);
        return q * (1.f + p * (1.f - q));
    } else if constexpr (ACT == AUD_ACT_GELU)
        return 0.5f * (1.f + erff(p * 0.70710678118654752f)) + p * 0.3989422804014327f * __builtin_amdgcn_exp2f(-0.5f * kLog2e * p * p);
    else return 1.f;
}

// more than 64 KB of dynamic LDS has to be allowed, per kernel and device: once
template <auto kernel>
hipError_t allow_lds(size_t bytes) {
    static std::atomic<uint64_t> allowed{0};
    if (bytes <= 64 * 1024) return hipSuccess;
    int device = 0;
    if (hipError_t e = hipGetDevice(&device)) return e;
    const uint64_t bit = uint64_t(1) << (device & 63);
    if (allowed.load(std::memory_order_acquire) & bit) return hipSuccess;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (e == hipSuccess) allowed.fetch_or(bit, std::memory_order_release);
    return e;
}

// A launch holds fewer than 2^32 threads.  A grid of more goes out in slices, in order on the stream: launch(grid, first) for the
// workgroups from `first` on.  What a slice's launch refuses ends the call; nothing is queued behind it.  (The CPU emulator is built
// with a small limit, so that slices are what its tests run.)
#ifndef AUD_LAUNCH_THREADS
#define AUD_LAUNCH_THREADS 0xFFFFFFFFll
#endif
template <typename F>
hipError_t in_slices(int64_t blocks, int threads, F&& launch) {
    const int64_t most = int64_t(AUD_LAUNCH_THREADS) / threads;
    for (int64_t first = 0; first < blocks; first += most) {
        launch(dim3(unsigned(std::min(most, blocks - first))), unsigned(first));
        if (hipError_t e = hipGetLastError()) return e;
    }
    return hipSuccess;
}
// the same for a kernel whose first argument is its descriptor, with the slice's start in it
template <typename A, typename F>
hipError_t in_slices_of(const A& a, int64_t blocks, int threads, F&& launch) {
    return in_slices(blocks, threads, [&](dim3 grid, unsigned first) {
        A s = a;
        s.first = first;
        launch(grid, s);
    });
}

// rows of an item that count: lengths[b] held to [0, rows]; rows where there is no table
__device__ __forceinline__ int item_rows(const int32_t* lengths, int b, int rows) {
    if (!lengths) return rows;
    const int n = lengths[b];
    return n < 0 ? 0 : (n > rows ? rows : n);
}

// elements per access for rows of C elements of e bytes, where all addresses and strides are multiples of `align` bytes
int vector_of(int e, int C, int align);

// ---- launch descriptors ----------------------------------------------------------------------------------------------
struct NormArgs {
    const void* x;            // [B, S, C]: item stride xi, row stride xr (elements), channels contiguous
    const void* dy;           // the same with di, dr (gradients)
    const float *weight, *bias;  // [C] or null (1, 0)
    const int32_t* lengths;   // [B] or null
    void* out;                // y or dx, contiguous
    float* stats;             // [B, G, 2] (mean, 1 / std): out (values; may be null), in (gradients)
    float* part;              // workspace, see group_norm.hip
    float *dweight, *dbias;   // [C] or null
    int B, S, C, G;
    int64_t xi, xr, di, dr;
    float eps;
    int chunks, chunk_rows;
    unsigned first;           // workgroups in front of this launch's (in_slices)
};
struct NormRoute {
    int vec;                 // elements per access
    bool one_wg;             // an item in one workgroup; else in `chunks` of chunk_rows rows
    int chunks, chunk_rows;
    bool join;               // ... whose moments a kernel of its own joins (many groups x chunks)
};
// align: what all addresses and strides are multiples of, bytes
NormRoute norm_route(int dtype, int B, int S, int C, int G, int align, bool grad);
int64_t norm_workspace_floats(const NormRoute& r, int B, int C, int G, bool grad);
hipError_t launch_norm(const NormArgs& a, const NormRoute& r, int dtype, int act, hipStream_t st);
hipError_t launch_norm_grad(const NormArgs& a, const NormRoute& r, int dtype, int act, hipStream_t st);

struct ConvArgs {
    const void *x, *dy;       // [B, L, D], strides as above
    const float *weight, *bias;  // [D, K], [D] or null
    const void* state;        // [B, K - 1, D] contiguous or null (zeros)
    const int32_t* lengths;
    void* out;                // y / dx [B, L, D] contiguous
    void* state_out;          // [B, K - 1, D] or null
    const void* dstate_out;   // gradients: of state_out, or null
    void* dstate;             // ... of state, or null
    float *dweight, *dbias;   // or null
    float* part;              // workspace [B * tiles][K + 1][D]
    int B, L, D;
    int64_t xi, xr, di, dr;
    int T;                    // steps a thread walks
    unsigned first;           // workgroups in front of this launch's
};
int conv_tile(int dtype, int B, int L, int D, int align);
hipError_t launch_conv(const ConvArgs& a, int dtype, int act, int K, int align, hipStream_t st);
hipError_t launch_conv_grad(const ConvArgs& a, int dtype, int act, int K, int align, hipStream_t st);

constexpr int kScanTile = 16;  // steps between kept states; the kernels' unit of work along the time axis
struct ScanArgs {
    const void *u, *delta, *z, *dy;  // [B, L, D]; z null: no gate
    const void *Bm, *Cm;             // [B, L, G, N], (G, N) contiguous
    const float *A, *D, *delta_bias; // [D, N], [D] or null, [D] or null
    const float* state;              // [B, D, N] or null (zeros)
    const int32_t* lengths;
    void* y;                         // [B, L, D] contiguous
    float* state_out;                // [B, D, N] or null
    float* kept;                     // [B, ceil(L / 16), N, D]: the state in front of every tile, or null
    const float* dstate_out;         // gradients: [B, D, N] or null
    void *du, *ddelta, *dz;          // [B, L, D] contiguous (dz null: no gate)
    void *dB, *dC;                   // [B, L, G, N] contiguous
    float *dA, *dD, *ddelta_bias, *dstate;  // dD, ddelta_bias, dstate may be null
    float* table;                    // workspace: B and C in float32 [B, G, 16 tiles, 2, padded states]
    float* sums;                     // workspace: chunk states [B, chunks, N, D] (scan_common.h chunk_state), chunk step sums [B, chunks, D]
    float* part_bc;                  // workspace: [2][blocks of a group][B, L, G, N]
    float* part;                     // workspace: [B * chunks][N + 2][D]
    int B, L, Dn, G, N, softplus;
    int64_t ui, ur, ei, er, zi, zr, yi, yr, bi, br, ci, cr;  // item / row strides of u, delta, z, dy, Bm, Cm
    int chunks, chunk_tiles, fold;
    unsigned first;                  // workgroups in front of this launch's
};
struct ScanRoute {
    int chunks, chunk_tiles;  // the time axis in `chunks` runs of chunk_tiles tiles, scanned side by side and joined
    int blocks;               // blocks of 64 channels a group has
    bool fold;                // few chunks: each walks the ones in front of it, instead of a kernel that joins them
};
int scan_padded_states(int N);
ScanRoute scan_route(int B, int L, int D, int G, int N, bool grad);
int64_t scan_sums_floats(const ScanRoute& r, int B, int D, int N);
hipError_t launch_scan(const ScanArgs& a, const ScanRoute& r, int dtype, bool aligned, hipStream_t st);
hipError_t launch_scan_step(const ScanArgs& a, int dtype, hipStream_t st);
hipError_t launch_scan_grad(const ScanArgs& a, const ScanRoute& r, int dtype, bool aligned, hipStream_t st);

// out[col] = sum over `rows` rows of in[row][col], col = k W + w: k < K goes to out0[w K + k], k = K to out1[w], K + 1 to out2[w]
// (any of them null); a fixed order of additions
hipError_t launch_column_sums(const float* in, int64_t rows, int W, int K, int extra, float* out0, float* out1, float* out2, hipStream_t st);

}  // namespace aud
