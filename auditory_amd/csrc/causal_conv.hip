// Short causal convolution over frames, one filter a channel: x [B, L, D], w [D, K], the K - 1 inputs before x as `state`.
//
//   e = state ++ x,  p_t = b + sum_k w_k e_{t + k},  y = act(p),  state' = the last K - 1 values of e[: K - 1 + len]
//   q = dy act'(p),  de_j = sum_k w_k q_{j - k} + dstate'_{j - len},  dw_k = sum q_t e_{t + k},  db = sum q
//
// A thread owns a pack of channels and walks T steps with the last K - 1 inputs in registers: every input is read once, but
// for the K - 1 in front of a run.  Rows at and behind lengths[b] are not read; their results are zero.
//
// Memory bounds it: 8 x 2048 x 1536 bfloat16, K = 4, 23 us for 101 MB (4.3 TB/s; a copy reaches 5.2).  The loads of eight steps are
// sent off together (one after the other, behind each other's stores: 28.7 us).  Its gradients, without a state: 127 us for 151 MB (floor
// 29), four steps of two inputs in flight; not made faster yet.
#include "frame_ops.h"

namespace aud {
namespace {

constexpr int kNT = 256, kBatch = 8, kGradBatch = 4;  // steps whose loads are in flight together

struct Run {  // the run of steps and the pack of channels of this thread
    int64_t b;
    int c, t0, t1, tile;
    bool on;
    __device__ __forceinline__ Run(const ConvArgs& a, int V, int tiles) {
        const int64_t id = int64_t(a.first + blockIdx.x) * kNT + threadIdx.x;
        const int packs = a.D / V;
        const int64_t q = id / packs;
        c = int(id % packs) * V;
        b = q / tiles;
        tile = int(q % tiles);
        on = b < a.B;
        t0 = tile * a.T;
        t1 = t0 + a.T < a.L ? t0 + a.T : a.L;
    }
};

template <int DT, int V>
__device__ __forceinline__ void load_or_zero(const void* base, int64_t at, bool there, float (&f)[V]) {
    if (there) unpack<DT, V>(load_pack<DT, V>(base, at), f);
    else
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = 0.f;
}

// e_j of item b (j from 0: the first K - 1 are the state)
template <int DT, int V, int K>
__device__ __forceinline__ void load_ext(const ConvArgs& a, int64_t b, int c, int64_t j, float (&f)[V]) {
    if (j < K - 1) load_or_zero<DT, V>(a.state, (b * (K - 1) + j) * a.D + c, a.state != nullptr, f);
    else unpack<DT, V>(load_pack<DT, V>(a.x, b * a.xi + (j - (K - 1)) * a.xr + c), f);
}

template <int DT, int V, int K, int ACT>
__global__ void __launch_bounds__(kNT) k_conv(ConvArgs a, int tiles) {
    const Run r(a, V, tiles);
    if (!r.on) return;
    const int len = item_rows(a.lengths, int(r.b), a.L);
    float w[V][K], bias[V], win[K][V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int k = 0; k < K; ++k) w[i][k] = a.weight[int64_t(r.c + i) * K + k];
        bias[i] = a.bias ? a.bias[r.c + i] : 0.f;
    }
    const int end = r.t1 < len ? r.t1 : len;
    if (r.t0 < end || r.tile == 0) {
#pragma unroll
        for (int j = 0; j < K - 1; ++j) load_ext<DT, V, K>(a, r.b, r.c, int64_t(r.t0) + j, win[j]);
    }
    if (r.tile == 0 && a.state_out && K > 1) {  // by the thread that has read the state: the two may be one buffer
        float keep[K][V];
#pragma unroll
        for (int j = 0; j < K - 1; ++j) {
            if (len + j < K - 1) {
#pragma unroll
                for (int m = 0; m < K - 1; ++m)
                    if (m == len + j)
#pragma unroll
                        for (int i = 0; i < V; ++i) keep[j][i] = win[m][i];
            } else {
                unpack<DT, V>(load_pack<DT, V>(a.x, r.b * a.xi + int64_t(len + j - (K - 1)) * a.xr + r.c), keep[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < K - 1; ++j) store_pack<DT, V>(a.state_out, (r.b * (K - 1) + j) * a.D + r.c, keep[j]);
    }
    const int64_t from = r.b * a.xi + r.c, to = r.b * int64_t(a.L) * a.D + r.c;
    auto step = [&](int t, const Pack<DT, V>& x) {
        unpack<DT, V>(x, win[K - 1]);
        float y[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float p = bias[i];
#pragma unroll
            for (int k = 0; k < K; ++k) p = fmaf(w[i][k], win[k][i], p);
            y[i] = act_value<ACT>(p);
        }
        store_pack<DT, V>(a.out, to + int64_t(t) * a.D, y);
#pragma unroll
        for (int k = 0; k < K - 1; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) win[k][i] = win[k + 1][i];
    };
    int t = r.t0;
    for (; t + kBatch <= end; t += kBatch) {
        Pack<DT, V> x[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) x[j] = load_pack<DT, V>(a.x, from + int64_t(t + j) * a.xr);
#pragma unroll
        for (int j = 0; j < kBatch; ++j) step(t + j, x[j]);
    }
    for (; t < end; ++t) step(t, load_pack<DT, V>(a.x, from + int64_t(t) * a.xr));
    float zero[V];
#pragma unroll
    for (int i = 0; i < V; ++i) zero[i] = 0.f;
    for (int t = r.t0 > end ? r.t0 : end; t < r.t1; ++t) store_pack<DT, V>(a.out, to + int64_t(t) * a.D, zero);
}

// gradients: the run's inputs x_{t0} .. x_{t1 - 1} (and, in the first run, the state) get theirs from q_t, t0 <= t < t1 + K - 1
template <int DT, int V, int K, int ACT>
__global__ void __launch_bounds__(kNT) k_conv_grad(ConvArgs a, int tiles) {
    const Run r(a, V, tiles);
    if (!r.on) return;
    const int len = item_rows(a.lengths, int(r.b), a.L);
    float w[V][K], bias[V], win[K][V], q[K][V], dw[K][V], db[V];  // win[k] = e_{t + k}, q[k] = q_{t - k}
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            w[i][k] = a.weight[int64_t(r.c + i) * K + k];
            dw[k][i] = q[k][i] = 0.f;
        }
        bias[i] = a.bias ? a.bias[r.c + i] : 0.f;
        db[i] = 0.f;
    }
    const int64_t to = r.b * int64_t(a.L) * a.D + r.c;
    const int last = r.t1 + K - 1;  // one behind the last j = t that is written
    if (r.t0 < len) {
#pragma unroll
        for (int j = 0; j < K - 1; ++j) load_ext<DT, V, K>(a, r.b, r.c, int64_t(r.t0) + j, win[j]);
    }
    auto step = [&](int t, const Pack<DT, V>& xt, const Pack<DT, V>& dt) {
#pragma unroll
        for (int k = K - 1; k > 0; --k)
#pragma unroll
            for (int i = 0; i < V; ++i) q[k][i] = q[k - 1][i];
        if (t < len) {
            float d[V];
            unpack<DT, V>(xt, win[K - 1]);
            unpack<DT, V>(dt, d);
            const bool own = t < r.t1;  // (the K - 1 steps behind the run are the next one's to sum)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float p = bias[i];
#pragma unroll
                for (int k = 0; k < K; ++k) p = fmaf(w[i][k], win[k][i], p);
                q[0][i] = d[i] * act_slope<ACT>(p);
            }
            if (own)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    db[i] += q[0][i];
#pragma unroll
                    for (int k = 0; k < K; ++k) dw[k][i] = fmaf(q[0][i], win[k][i], dw[k][i]);
                }
#pragma unroll
            for (int k = 0; k < K - 1; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) win[k][i] = win[k + 1][i];
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) q[0][i] = 0.f;
        }
        // de_t: of the state for t < K - 1, else of x_{t - K + 1}
        float de[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            de[i] = 0.f;
#pragma unroll
            for (int k = 0; k < K; ++k) de[i] = fmaf(w[i][k], q[k][i], de[i]);
        }
        if (a.dstate_out && K > 1 && t >= len && t < len + K - 1) {
            float s[V];
            unpack<DT, V>(load_pack<DT, V>(a.dstate_out, (r.b * (K - 1) + (t - len)) * a.D + r.c), s);
#pragma unroll
            for (int i = 0; i < V; ++i) de[i] += s[i];
        }
        const int at = t - (K - 1);
        if (at >= r.t0) {
            if (at >= len)
#pragma unroll
                for (int i = 0; i < V; ++i) de[i] = 0.f;
            store_pack<DT, V>(a.out, to + int64_t(at) * a.D, de);
        } else if (r.tile == 0 && a.dstate) {
            store_pack<DT, V>(a.dstate, (r.b * (K - 1) + t) * a.D + r.c, de);
        }
    };
    const int64_t xb = r.b * a.xi + r.c, db0 = r.b * a.di + r.c;
    for (int t = r.t0; t < last; t += kGradBatch) {
        Pack<DT, V> xs[kGradBatch], ds[kGradBatch];
#pragma unroll
        for (int j = 0; j < kGradBatch; ++j) {
            const int64_t row = t + j < len ? t + j : (len > 0 ? len - 1 : 0);  // (a row that is there; not used behind the length)
            if (len > 0) {
                xs[j] = load_pack<DT, V>(a.x, xb + row * a.xr);
                ds[j] = load_pack<DT, V>(a.dy, db0 + row * a.dr);
            }
        }
#pragma unroll
        for (int j = 0; j < kGradBatch; ++j)
            if (t + j < last) step(t + j, xs[j], ds[j]);
    }
    float* part = a.part + (r.b * tiles + r.tile) * int64_t(K + 1) * a.D + r.c;
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int k = 0; k < K; ++k) part[int64_t(k) * a.D + i] = dw[k][i];
        part[int64_t(K) * a.D + i] = db[i];
    }
}

inline int tiles_of(const ConvArgs& a) { return a.L > 0 ? (a.L + a.T - 1) / a.T : 1; }

template <int DT, int V, int K, int ACT>
hipError_t run(const ConvArgs& a, bool grad, hipStream_t st) {
    const int tiles = tiles_of(a);
    const int64_t threads = int64_t(a.B) * tiles * (a.D / V);
    const int64_t blocks = (threads + kNT - 1) / kNT;
    if (!grad)
        return in_slices_of(a, blocks, kNT, [&](dim3 grid, const ConvArgs& s) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(k_conv<DT, V, K, ACT>), grid, dim3(kNT), 0, st, s, tiles);
        });
    if (hipError_t e = in_slices_of(a, blocks, kNT, [&](dim3 grid, const ConvArgs& s) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(k_conv_grad<DT, V, K, ACT>), grid, dim3(kNT), 0, st, s, tiles);
        }))
        return e;
    if (!a.dweight && !a.dbias) return hipSuccess;
    return launch_column_sums(a.part, int64_t(a.B) * tiles, a.D, K, 1, a.dweight, a.dbias, nullptr, st);
}
template <int DT, int V, int K>
hipError_t by_act(const ConvArgs& a, int act, bool grad, hipStream_t st) {
    return act == AUD_ACT_SILU ? run<DT, V, K, AUD_ACT_SILU>(a, grad, st) : run<DT, V, K, AUD_ACT_NONE>(a, grad, st);
}
template <int DT, int V>
hipError_t by_taps(const ConvArgs& a, int act, int K, bool grad, hipStream_t st) {
    switch (K) {
        case 1: return by_act<DT, V, 1>(a, act, grad, st);
        case 2: return by_act<DT, V, 2>(a, act, grad, st);
        case 3: return by_act<DT, V, 3>(a, act, grad, st);
        case 4: return by_act<DT, V, 4>(a, act, grad, st);
        default: return hipErrorInvalidValue;
    }
}
hipError_t by_type(const ConvArgs& a, int dtype, int act, int K, int align, bool grad, hipStream_t st) {
    const int v = vector_of(dtype == AUD_F32 ? 4 : 2, a.D, align);
    switch (dtype) {
        case AUD_F32:
            return v == 4   ? by_taps<AUD_F32, 4>(a, act, K, grad, st)
                   : v == 2 ? by_taps<AUD_F32, 2>(a, act, K, grad, st)
                            : by_taps<AUD_F32, 1>(a, act, K, grad, st);
        case AUD_BF16:
            return v == 8   ? by_taps<AUD_BF16, 8>(a, act, K, grad, st)
                   : v >= 2 ? by_taps<AUD_BF16, 2>(a, act, K, grad, st)
                            : by_taps<AUD_BF16, 1>(a, act, K, grad, st);
        default:
            return v == 8   ? by_taps<AUD_F16, 8>(a, act, K, grad, st)
                   : v >= 2 ? by_taps<AUD_F16, 2>(a, act, K, grad, st)
                            : by_taps<AUD_F16, 1>(a, act, K, grad, st);
    }
}

}  // namespace

// steps a thread walks: as many as leave the card about 2048 waves, between 8 and 64
int conv_tile(int dtype, int B, int L, int D, int align) {
    const int v = vector_of(dtype == AUD_F32 ? 4 : 2, D, align), V = dtype != AUD_F32 && v == 4 ? 2 : v;
    int T = 64;
    while (T > 8 && int64_t(B) * (D / V) * ((L + T - 1) / T) < 64 * 2048) T /= 2;
    return T;
}

hipError_t launch_conv(const ConvArgs& a, int dtype, int act, int K, int align, hipStream_t st) {
    return by_type(a, dtype, act, K, align, false, st);
}
hipError_t launch_conv_grad(const ConvArgs& a, int dtype, int act, int K, int align, hipStream_t st) {
    return by_type(a, dtype, act, K, align, true, st);
}

}  // namespace aud
