// Group norm with an activation, channels last: x [B, S, C] (the gabor maps' own layout: positions, then polarity x filter),
// G groups of C / G neighbouring channels, n = rows of the item x channels of the group values each.
//
//   m = 1/n sum x,  v = 1/n sum (x - m)^2,  r = 1 / sqrt(v + eps),  xh = (x - m) r,  p = xh w_c + b_c,  y = act(p)
//   q = dy act'(p),  dw_c = sum q xh,  db_c = sum q,  t = q w_c,  dx = r (t - 1/n sum t - xh 1/n sum t xh)
//
// Statistics: a thread sums x - k and (x - k)^2 of its rows of a channel, k the first of them, and turns the pair into a mean
// and a sum of squared distances from it; those are joined (rows, channels, chunks of rows) by
//   M2 = sum M2_i + n_i (m_i - m)^2, which has no cancellation, so a level far from zero costs nothing.
// Rows at and behind lengths[b] are not read; their results are zero.
#include "frame_ops.h"

namespace aud {
namespace {

constexpr int kNT = 256;

struct Lanes {  // how a workgroup's threads lie on (rows, packs of channels) for packs [first, first + cols)
    int cols, lanes, r, c;
    __device__ __forceinline__ Lanes(int nt, int n_packs, int first) {
        cols = n_packs - first < nt ? n_packs - first : nt;
        lanes = nt / cols;
        r = int(threadIdx.x) / cols;
        c = first + int(threadIdx.x) % cols;
    }
};

// ---- a chunk of rows: mean and M2 of every group -> part [B, chunks, G, 2] --------------------------------------------
template <int DT, int V>
__global__ void __launch_bounds__(kNT) k_norm_chunk(NormArgs a) {
    float* lds = reinterpret_cast<float*>(dyn_lds());
    float *ch_mean = lds, *ch_m2 = lds + a.C;       // [C] each
    float *ln_mean = lds + 2 * a.C, *ln_m2 = ln_mean + kNT * V;  // [lanes][cols V]
    const int tid = threadIdx.x, chunk = blockIdx.x % a.chunks, b = blockIdx.x / a.chunks;
    const int rows = item_rows(a.lengths, b, a.S);
    const int lo = chunk * a.chunk_rows, hi = lo + a.chunk_rows < rows ? lo + a.chunk_rows : rows;
    const int n = hi > lo ? hi - lo : 0, packs = a.C / V;
    for (int first = 0; first < packs; first += kNT) {
        const Lanes l(kNT, packs, first);
        float k[V], s[V], ss[V];
#pragma unroll
        for (int i = 0; i < V; ++i) k[i] = s[i] = ss[i] = 0.f;
        int cnt = 0;
        if (l.r < l.lanes) {
            const int64_t base = int64_t(b) * a.xi + int64_t(l.c) * V;
            for (int row = lo + l.r; row < hi; row += l.lanes, ++cnt) {
                float x[V];
                unpack<DT, V>(load_pack<DT, V>(a.x, base + int64_t(row) * a.xr), x);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    if (cnt == 0) k[i] = x[i];
                    const float d = x[i] - k[i];
                    s[i] += d;
                    ss[i] = fmaf(d, d, ss[i]);
                }
            }
            const float inv = cnt ? 1.f / float(cnt) : 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int at = l.r * l.cols * V + (l.c - first) * V + i;
                ln_mean[at] = fmaf(s[i], inv, k[i]);
                ln_m2[at] = fmaxf(ss[i] - s[i] * s[i] * inv, 0.f) + 0.f * ss[i];
            }
        }
        __syncthreads();
        for (int c = tid; c < l.cols * V; c += kNT) {
            float m = 0.f;
            for (int r = 0; r < l.lanes; ++r) m += float(n > r ? (n - r + l.lanes - 1) / l.lanes : 0) * ln_mean[r * l.cols * V + c];
            m = n ? m / float(n) : 0.f;
            float m2 = 0.f;
            for (int r = 0; r < l.lanes; ++r) {
                const float d = ln_mean[r * l.cols * V + c] - m;
                m2 += ln_m2[r * l.cols * V + c] + float(n > r ? (n - r + l.lanes - 1) / l.lanes : 0) * d * d;
            }
            ch_mean[first * V + c] = m;
            ch_m2[first * V + c] = m2;
        }
        __syncthreads();
    }
    const int cg = a.C / a.G;
    for (int g = tid; g < a.G; g += kNT) {
        float m = 0.f, m2 = 0.f;
        for (int c = 0; c < cg; ++c) m += ch_mean[g * cg + c];
        m /= float(cg);
        for (int c = 0; c < cg; ++c) {
            const float d = ch_mean[g * cg + c] - m;
            m2 += ch_m2[g * cg + c] + float(n) * d * d;
        }
        float* out = a.part + ((int64_t(b) * a.chunks + chunk) * a.G + g) * 2;
        out[0] = m;
        out[1] = m2;
    }
}

// the chunks of an item joined -> stats [B, G, 2]
__global__ void __launch_bounds__(kNT) k_norm_join(NormArgs a) {
    const int64_t i = int64_t(blockIdx.x) * kNT + threadIdx.x;
    if (i >= int64_t(a.B) * a.G) return;
    const int b = int(i / a.G), g = int(i % a.G), cg = a.C / a.G;
    const int rows = item_rows(a.lengths, b, a.S);
    const float* p = a.part + (int64_t(b) * a.chunks * a.G + g) * 2;
    float m = 0.f, m2 = 0.f;
    for (int c = 0; c < a.chunks; ++c) {
        const int left = rows - c * a.chunk_rows, n = left < 0 ? 0 : (left < a.chunk_rows ? left : a.chunk_rows);
        m += float(n) * p[int64_t(c) * a.G * 2];
    }
    m = rows ? m / float(rows) : 0.f;
    for (int c = 0; c < a.chunks; ++c) {
        const int left = rows - c * a.chunk_rows, n = left < 0 ? 0 : (left < a.chunk_rows ? left : a.chunk_rows);
        const float d = p[int64_t(c) * a.G * 2] - m;
        m2 += p[int64_t(c) * a.G * 2 + 1] + float(n) * float(cg) * d * d;
    }
    a.stats[i * 2] = m;
    a.stats[i * 2 + 1] = 1.f / sqrtf((rows ? m2 / (float(rows) * float(cg)) : 0.f) + a.eps);
}

// y = act((x - m) r w + b)
template <int DT, int V, int ACT>
__global__ void __launch_bounds__(kNT) k_norm_apply(NormArgs a) {
    const int chunk = blockIdx.x % a.chunks, b = blockIdx.x / a.chunks;
    const int rows = item_rows(a.lengths, b, a.S);
    const int lo = chunk * a.chunk_rows, hi = lo + a.chunk_rows < a.S ? lo + a.chunk_rows : a.S;
    const int packs = a.C / V, cg = a.C / a.G;
    for (int first = 0; first < packs; first += kNT) {
        const Lanes l(kNT, packs, first);
        if (l.r >= l.lanes) continue;
        float m[V], sc[V], sh[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = l.c * V + i;
            const float* st = a.stats + (int64_t(b) * a.G + c / cg) * 2;
            m[i] = st[0];
            sc[i] = st[1] * (a.weight ? a.weight[c] : 1.f);
            sh[i] = a.bias ? a.bias[c] : 0.f;
        }
        const int64_t base = int64_t(b) * a.xi + int64_t(l.c) * V, to = int64_t(b) * a.S * a.C + int64_t(l.c) * V;
        for (int row = lo + l.r; row < hi; row += l.lanes) {
            float y[V];
            if (row < rows) {
                unpack<DT, V>(load_pack<DT, V>(a.x, base + int64_t(row) * a.xr), y);
#pragma unroll
                for (int i = 0; i < V; ++i) y[i] = act_value<ACT>(fmaf(y[i] - m[i], sc[i], sh[i]));
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) y[i] = 0.f;
            }
            store_pack<DT, V>(a.out, to + int64_t(row) * a.C, y);
        }
    }
}

// ---- gradients: sums of q and q xh over a chunk of rows, per channel -> part [B, chunks, 2, C] --------------------------
template <int DT, int V, int ACT>
__global__ void __launch_bounds__(kNT) k_norm_grad_chunk(NormArgs a) {
    float* lds = reinterpret_cast<float*>(dyn_lds());  // [2][lanes][cols V]
    const int tid = threadIdx.x, chunk = blockIdx.x % a.chunks, b = blockIdx.x / a.chunks;
    const int rows = item_rows(a.lengths, b, a.S);
    const int lo = chunk * a.chunk_rows, hi = lo + a.chunk_rows < rows ? lo + a.chunk_rows : rows;
    const int packs = a.C / V, cg = a.C / a.G;
    float* out = a.part + (int64_t(b) * a.chunks + chunk) * 2 * a.C;
    for (int first = 0; first < packs; first += kNT) {
        const Lanes l(kNT, packs, first);
        float s0[V], s1[V];
#pragma unroll
        for (int i = 0; i < V; ++i) s0[i] = s1[i] = 0.f;
        if (l.r < l.lanes) {
            float m[V], r[V], w[V], sh[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int c = l.c * V + i;
                const float* st = a.stats + (int64_t(b) * a.G + c / cg) * 2;
                m[i] = st[0];
                r[i] = st[1];
                w[i] = a.weight ? a.weight[c] : 1.f;
                sh[i] = a.bias ? a.bias[c] : 0.f;
            }
            const int64_t xb = int64_t(b) * a.xi + int64_t(l.c) * V, db = int64_t(b) * a.di + int64_t(l.c) * V;
            for (int row = lo + l.r; row < hi; row += l.lanes) {
                float x[V], d[V];
                unpack<DT, V>(load_pack<DT, V>(a.x, xb + int64_t(row) * a.xr), x);
                unpack<DT, V>(load_pack<DT, V>(a.dy, db + int64_t(row) * a.dr), d);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float xh = (x[i] - m[i]) * r[i];
                    const float q = d[i] * act_slope<ACT>(fmaf(xh, w[i], sh[i]));
                    s0[i] = fmaf(q, xh, s0[i]);
                    s1[i] += q;
                }
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int at = l.r * l.cols * V + (l.c - first) * V + i;
                lds[at] = s0[i];
                lds[kNT * V + at] = s1[i];
            }
        }
        __syncthreads();
        for (int c = tid; c < l.cols * V; c += kNT) {
            float t0 = 0.f, t1 = 0.f;
            for (int r = 0; r < l.lanes; ++r) {
                t0 += lds[r * l.cols * V + c];
                t1 += lds[kNT * V + r * l.cols * V + c];
            }
            out[first * V + c] = t0;
            out[a.C + first * V + c] = t1;
        }
        __syncthreads();
    }
}

// 1/n sum t and 1/n sum t xh of every (item, group) -> gsum [B, G, 2] behind the chunk sums
__global__ void __launch_bounds__(kNT) k_norm_grad_join(NormArgs a) {
    const int64_t i = int64_t(blockIdx.x) * kNT + threadIdx.x;
    if (i >= int64_t(a.B) * a.G) return;
    const int b = int(i / a.G), g = int(i % a.G), cg = a.C / a.G;
    const int rows = item_rows(a.lengths, b, a.S);
    float t0 = 0.f, t1 = 0.f;
    for (int c = g * cg; c < (g + 1) * cg; ++c) {
        float s0 = 0.f, s1 = 0.f;
        for (int k = 0; k < a.chunks; ++k) {
            const float* p = a.part + (int64_t(b) * a.chunks + k) * 2 * a.C + c;
            s0 += p[0];
            s1 += p[a.C];
        }
        const float w = a.weight ? a.weight[c] : 1.f;
        t0 = fmaf(w, s0, t0);
        t1 = fmaf(w, s1, t1);
    }
    const float inv = rows ? 1.f / (float(rows) * float(cg)) : 0.f;
    float* out = a.part + int64_t(a.B) * a.chunks * 2 * a.C + i * 2;
    out[0] = t1 * inv;
    out[1] = t0 * inv;
}

template <int DT, int V, int ACT>
__global__ void __launch_bounds__(kNT) k_norm_grad_apply(NormArgs a) {
    const int chunk = blockIdx.x % a.chunks, b = blockIdx.x / a.chunks;
    const int rows = item_rows(a.lengths, b, a.S);
    const int lo = chunk * a.chunk_rows, hi = lo + a.chunk_rows < a.S ? lo + a.chunk_rows : a.S;
    const int packs = a.C / V, cg = a.C / a.G;
    const float* gsum = a.part + int64_t(a.B) * a.chunks * 2 * a.C;
    for (int first = 0; first < packs; first += kNT) {
        const Lanes l(kNT, packs, first);
        if (l.r >= l.lanes) continue;
        float m[V], r[V], w[V], sh[V], u0[V], u1[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = l.c * V + i;
            const int64_t at = (int64_t(b) * a.G + c / cg) * 2;
            m[i] = a.stats[at];
            r[i] = a.stats[at + 1];
            w[i] = a.weight ? a.weight[c] : 1.f;
            sh[i] = a.bias ? a.bias[c] : 0.f;
            u0[i] = gsum[at];
            u1[i] = gsum[at + 1];
        }
        const int64_t xb = int64_t(b) * a.xi + int64_t(l.c) * V, db = int64_t(b) * a.di + int64_t(l.c) * V;
        const int64_t to = int64_t(b) * a.S * a.C + int64_t(l.c) * V;
        for (int row = lo + l.r; row < hi; row += l.lanes) {
            float x[V], d[V];
            if (row < rows) {
                unpack<DT, V>(load_pack<DT, V>(a.x, xb + int64_t(row) * a.xr), x);
                unpack<DT, V>(load_pack<DT, V>(a.dy, db + int64_t(row) * a.dr), d);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float xh = (x[i] - m[i]) * r[i];
                    const float t = d[i] * act_slope<ACT>(fmaf(xh, w[i], sh[i])) * w[i];
                    x[i] = r[i] * ((t - u0[i]) - xh * u1[i]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) x[i] = 0.f;
            }
            store_pack<DT, V>(a.out, to + int64_t(row) * a.C, x);
        }
    }
}

// ---- column sums of a partial-result table ------------------------------------------------------------------------------
constexpr int kCsCols = 64, kCsLanes = 4;
__global__ void __launch_bounds__(kCsCols * kCsLanes) k_column_sums(const float* in, int64_t rows, int W, int K, int extra, float* out0,
                                                                   float* out1, float* out2) {
    float* lds = reinterpret_cast<float*>(dyn_lds());
    const int c = threadIdx.x % kCsCols, lane = threadIdx.x / kCsCols;
    const int64_t width = int64_t(W) * (K + extra), col = int64_t(blockIdx.x) * kCsCols + c;
    float s = 0.f;
    if (col < width)
        for (int64_t r = lane; r < rows; r += kCsLanes) s += in[r * width + col];
    lds[threadIdx.x] = s;
    __syncthreads();
    if (lane == 0 && col < width) {
        for (int k = 1; k < kCsLanes; ++k) s += lds[k * kCsCols + c];
        const int k = int(col / W), w = int(col % W);
        if (k < K) {
            if (out0) out0[int64_t(w) * K + k] = s;
        } else {
            float* out = k == K ? out1 : out2;
            if (out) out[w] = s;
        }
    }
}

template <int DT, int V>
hipError_t run(const NormArgs& a, int act, hipStream_t st) {
    const dim3 grid(unsigned(a.chunks) * unsigned(a.B));
    hipLaunchKernelGGL(HIP_KERNEL_NAME(k_norm_chunk<DT, V>), grid, dim3(kNT), size_t(2 * a.C + 2 * kNT * V) * 4, st, a);
    const unsigned join = unsigned((int64_t(a.B) * a.G + kNT - 1) / kNT);
    hipLaunchKernelGGL(k_norm_join, dim3(join), dim3(kNT), 0, st, a);
    switch (act) {
        case AUD_ACT_RELU: hipLaunchKernelGGL(HIP_KERNEL_NAME(k_norm_apply<DT, V, AUD_ACT_RELU>), grid, dim3(kNT), 0, st, a); break;
        case AUD_ACT_SILU: hipLaunchKernelGGL(HIP_KERNEL_NAME(k_norm_apply<DT, V, AUD_ACT_SILU>), grid, dim3(kNT), 0, st, a); break;
        case AUD_ACT_GELU: hipLaunchKernelGGL(HIP_KERNEL_NAME(k_norm_apply<DT, V, AUD_ACT_GELU>), grid, dim3(kNT), 0, st, a); break;
        default: hipLaunchKernelGGL(HIP_KERNEL_NAME(k_norm_apply<DT, V, AUD_ACT_NONE>), grid, dim3(kNT), 0, st, a);
    }
    return hipGetLastError();
}

template <int DT, int V, int ACT>
hipError_t run_grad(const NormArgs& a, hipStream_t st) {
    const dim3 grid(unsigned(a.chunks) * unsigned(a.B));
    hipLaunchKernelGGL(HIP_KERNEL_NAME(k_norm_grad_chunk<DT, V, ACT>), grid, dim3(kNT), size_t(2 * kNT * V) * 4, st, a);
    const unsigned join = unsigned((int64_t(a.B) * a.G + kNT - 1) / kNT);
    hipLaunchKernelGGL(k_norm_grad_join, dim3(join), dim3(kNT), 0, st, a);
    hipLaunchKernelGGL(HIP_KERNEL_NAME(k_norm_grad_apply<DT, V, ACT>), grid, dim3(kNT), 0, st, a);
    if (hipError_t e = hipGetLastError()) return e;
    if (!a.dweight && !a.dbias) return hipSuccess;
    return launch_column_sums(a.part, int64_t(a.B) * a.chunks, a.C, 0, 2, nullptr, a.dweight, a.dbias, st);
}
template <int DT, int V>
hipError_t run_grad_act(const NormArgs& a, int act, hipStream_t st) {
    switch (act) {
        case AUD_ACT_RELU: return run_grad<DT, V, AUD_ACT_RELU>(a, st);
        case AUD_ACT_SILU: return run_grad<DT, V, AUD_ACT_SILU>(a, st);
        case AUD_ACT_GELU: return run_grad<DT, V, AUD_ACT_GELU>(a, st);
        default: return run_grad<DT, V, AUD_ACT_NONE>(a, st);
    }
}

}  // namespace

hipError_t launch_column_sums(const float* in, int64_t rows, int W, int K, int extra, float* out0, float* out1, float* out2, hipStream_t st) {
    const int64_t width = int64_t(W) * (K + extra);
    hipLaunchKernelGGL(k_column_sums, dim3(unsigned((width + kCsCols - 1) / kCsCols)), dim3(kCsCols * kCsLanes),
                       size_t(kCsCols) * kCsLanes * 4, st, in, rows, W, K, extra, out0, out1, out2);
    return hipGetLastError();
}

NormRoute norm_route(int dtype, int B, int S, int C, bool aligned, bool) {
    NormRoute r{};
    const int e = dtype == AUD_F32 ? 4 : 2;
    r.vec = aligned && C % (16 / e) == 0 ? 16 / e : 1;
    // about a thousand workgroups, at least 16 KB of input each
    const int64_t bytes = int64_t(S) * C * e;
    int64_t chunks = (1024 + B - 1) / B;
    chunks = std::min<int64_t>(chunks, std::max<int64_t>(1, bytes / 16384));
    chunks = std::max<int64_t>(1, std::min<int64_t>(chunks, S));
    r.chunk_rows = int((S + chunks - 1) / chunks);
    r.chunks = r.chunk_rows ? (S + r.chunk_rows - 1) / r.chunk_rows : 1;
    return r;
}

int64_t norm_workspace_floats(const NormRoute& r, int B, int C, int G, bool grad, bool keeps_stats) {
    if (grad) return int64_t(B) * r.chunks * 2 * C + int64_t(B) * G * 2;
    return int64_t(B) * r.chunks * G * 2 + (keeps_stats ? 0 : int64_t(B) * G * 2);
}

#define AUD_BY_TYPE(FN, ...)                                                              \
    switch (dtype) {                                                                      \
        case AUD_F32: return r.vec > 1 ? FN<AUD_F32, 4>(__VA_ARGS__) : FN<AUD_F32, 1>(__VA_ARGS__);   \
        case AUD_BF16: return r.vec > 1 ? FN<AUD_BF16, 8>(__VA_ARGS__) : FN<AUD_BF16, 1>(__VA_ARGS__); \
        default: return r.vec > 1 ? FN<AUD_F16, 8>(__VA_ARGS__) : FN<AUD_F16, 1>(__VA_ARGS__);        \
    }

hipError_t launch_norm(const NormArgs& a, const NormRoute& r, int dtype, int act, hipStream_t st) {
    AUD_BY_TYPE(run, a, act, st)
}
hipError_t launch_norm_grad(const NormArgs& a, const NormRoute& r, int dtype, int act, hipStream_t st) {
    AUD_BY_TYPE(run_grad_act, a, act, st)
}

}  // namespace aud
