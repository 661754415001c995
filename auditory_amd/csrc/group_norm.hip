// Group norm with an activation, channels last: x [B, S, C] (the gabor maps' own layout: positions, then polarity x filter),
// G groups of C / G neighbouring channels, n = rows of the item x channels of the group values each.
//
//   m = 1/n sum x,  v = 1/n sum (x - m)^2,  r = 1 / sqrt(v + eps),  xh = (x - m) r,  p = xh w_c + b_c,  y = act(p)
//   q = dy act'(p),  dw_c = sum q xh,  db_c = sum q,  t = q w_c,  dx = r (t - 1/n sum t - xh 1/n sum t xh)
//
// Statistics: a thread sums x - k and (x - k)^2 of its rows of a channel, k the first of them, and turns the pair into a mean
// and a sum of squared distances from it; those are joined (rows, channels, chunks of rows) by
//   M2 = sum M2_i + n_i (m_i - m)^2, which has no cancellation, so a level far from zero costs no more than the mean's own rounding.
// Rows at and behind lengths[b] are not read; their results are zero.
//
// Three routes by the size of an item.  Up to four packs a thread it stays in one workgroup's registers: read once, one launch
// (256 x 352 x 16 float32: 6.6 us, floor 2.2; launch and the two trips through LDS are the rest).  Up to 32 KB (128 KB, 1 MB
// with 256, 1024 items and more) one workgroup reads it twice.  Else chunks of rows in about 512 workgroups: moments of the chunks,
// then every workgroup joins its item's and writes (gradients: channel sums, joined per item, then dx, the parameters' sums by
// workgroups of their own behind them).  Memory bounds that route: 16 x 4096 x 512 bfloat16 forward 15 + 28 us (67 MB read, then 134
// moved), gradients 28 + 5 + 36 us (134, then 201 MB), 109 us a pass on inputs that the Infinity Cache holds, 123 on others, where
// one sweep of everything would be 65.  An item is the unit here, and its 4 MB are more than a CU holds; the statistics need only a
// group of it, 128 KB there, which one or two workgroups' registers would hold.  A route by (item, group) is not built.
#include "frame_ops.h"

namespace aud {
namespace {

constexpr int kItemThreads = 512, kChunkThreads = 256;
constexpr int kMaxChunks = 256;

// How a workgroup's threads lie on (rows, packs of channels) for packs [first, first + cols).  Where the packs take several sweeps
// the last one has threads left over: they may take rows of their own (SPREAD) only if what the lanes of a pack hold is not joined
// behind the sweeps -- the joins know one number of lanes, and their tables have room for NT packs of one sweep or C channels once.
template <int NT, bool SPREAD>
struct Lanes {
    int cols, lanes, r, c;
    __device__ __forceinline__ Lanes(int n_packs, int first) {
        cols = n_packs - first < NT ? n_packs - first : NT;
        lanes = NT / (SPREAD ? cols : n_packs < NT ? n_packs : NT);
        r = int(threadIdx.x) / cols;
        c = first + int(threadIdx.x) - r * cols;
        if (r >= lanes) r = 1 << 30;  // left over: no row is theirs
    }
};
// rows lo + r, lo + r + lanes, ... < hi of the item: fetch(row, j) for four of them, then use(row, j) -- the loads of a batch are
// in flight together
template <int BATCH, typename F, typename U>
__device__ __forceinline__ void walk_rows(int lo, int hi, int r, int lanes, F&& fetch, U&& use) {
    int64_t row = int64_t(lo) + r;
    for (; row + int64_t(BATCH - 1) * lanes < hi; row += int64_t(BATCH) * lanes) {
#pragma unroll
        for (int j = 0; j < BATCH; ++j) fetch(row + int64_t(j) * lanes, j);
#pragma unroll
        for (int j = 0; j < BATCH; ++j) use(row + int64_t(j) * lanes, j);
    }
    for (; row < hi; row += lanes) {
        fetch(row, 0);
        use(row, 0);
    }
}
__device__ __forceinline__ int rows_of_lane(int n, int lanes, int r) { return n > r ? (n - r + lanes - 1) / lanes : 0; }
// lanes that work on a group together: a power of two up to the wave, as many as there are for G groups
template <int NT>
__device__ __forceinline__ int lanes_per_group(int G) {
    int p = 64;
    while (p > 1 && p * G > NT) p >>= 1;
    return p;
}
__device__ __forceinline__ float sum_lanes(float v, int p) {
    for (int m = p >> 1; m > 0; m >>= 1) v += __shfl_xor(v, m);
    return v;
}
// every group of the item by lanes_per_group lanes each: each(group, lane, lanes, there) for all threads the same number of times
template <int NT, typename F>
__device__ __forceinline__ void for_groups(int G, F&& each) {
    const int p = lanes_per_group<NT>(G), lane = int(threadIdx.x) & (p - 1), step = NT / p;
    for (int g0 = 0; g0 < G; g0 += step) {
        const int g = g0 + int(threadIdx.x) / p;
        each(g < G ? g : G - 1, lane, p, g < G);
    }
}

// the channels of a pack: mean, 1 / std x weight, bias (STATS: [G, 2] in LDS or global memory)
template <int V>
struct Affine {
    float m[V], r[V], w[V], sh[V];
    __device__ __forceinline__ void load(const NormArgs& a, const float* stats, int c0) {
        const int cg = a.C / a.G;
        int g = c0 / cg, in = c0 - g * cg;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            m[i] = stats[2 * g];
            r[i] = stats[2 * g + 1];
            w[i] = a.weight ? a.weight[c0 + i] : 1.f;
            sh[i] = a.bias ? a.bias[c0 + i] : 0.f;
            if (++in == cg) in = 0, ++g;
        }
    }
};

// mean and M2 of every group over rows [lo, hi) of item b -> out [G, 2] in LDS; entries: LDS [2][max(NT V, C)]
template <int DT, int V, int NT>
__device__ __forceinline__ void group_moments(const NormArgs& a, int b, int lo, int hi, float* entries, float* out) {
    const int n = hi > lo ? hi - lo : 0, packs = a.C / V, cg = a.C / a.G;
    const int size = NT * V > a.C ? NT * V : a.C;
    float *e_mean = entries, *e_m2 = entries + size;
    int width = a.C, lanes = 1;
    for (int first = 0; first < packs; first += NT) {
        const Lanes<NT, false> l(packs, first);
        lanes = l.lanes;  // (the same in every sweep)
        float k[V], s[V], ss[V];
#pragma unroll
        for (int i = 0; i < V; ++i) k[i] = s[i] = ss[i] = 0.f;
        const int64_t base = int64_t(b) * a.xi + int64_t(l.c) * V;
        if (l.r < n) {
            unpack<DT, V>(load_pack<DT, V>(a.x, base + int64_t(lo + l.r) * a.xr), k);
            Pack<DT, V> p[4];
            walk_rows<4>(lo, hi, l.r, l.lanes, [&](int64_t row, int j) { p[j] = load_pack<DT, V>(a.x, base + row * a.xr); },
                         [&](int64_t, int j) {
                             float x[V];
                             unpack<DT, V>(p[j], x);
#pragma unroll
                             for (int i = 0; i < V; ++i) {
                                 const float d = x[i] - k[i];
                                 s[i] += d;
                                 ss[i] = fmaf(d, d, ss[i]);
                             }
                         });
        }
        if (l.r < l.lanes) {
            const int cnt = rows_of_lane(n, l.lanes, l.r);
            const float inv = cnt ? 1.f / float(cnt) : 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int at = l.r * width + l.c * V + i;
                AUD_IN_TABLE(at, size);
                e_mean[at] = fmaf(s[i], inv, k[i]);
                e_m2[at] = fmaxf(ss[i] - s[i] * s[i] * inv, 0.f) + 0.f * ss[i];  // (NaN stays NaN)
            }
        }
    }
    __syncthreads();
    const float total = n ? 1.f / (float(n) * float(cg)) : 0.f;
    for_groups<NT>(a.G, [&](int g, int lane, int p, bool there) {
        const int dr = p / cg, dc = p - dr * cg, r0 = lane / cg, c0 = lane - r0 * cg;
        float m = 0.f, m2 = 0.f;
        for (int r = r0, c = c0; r < lanes;) {
            m = fmaf(float(rows_of_lane(n, lanes, r)), e_mean[r * width + g * cg + c], m);
            r += dr, c += dc;
            if (c >= cg) c -= cg, ++r;
        }
        m = sum_lanes(m, p) * total;
        for (int r = r0, c = c0; r < lanes;) {
            const float d = e_mean[r * width + g * cg + c] - m;
            m2 += fmaf(float(rows_of_lane(n, lanes, r)) * d, d, e_m2[r * width + g * cg + c]);
            r += dr, c += dc;
            if (c >= cg) c -= cg, ++r;
        }
        m2 = sum_lanes(m2, p);
        if (there && lane == 0) {
            out[2 * g] = m;
            out[2 * g + 1] = m2;
        }
    });
    __syncthreads();
}
__device__ __forceinline__ float inv_std(float m2, int rows, int cg, float eps) {
    return 1.f / sqrtf((rows ? m2 / (float(rows) * float(cg)) : 0.f) + eps);
}

// y of rows [lo, hi) of item b, `rows` of them counting; stats [G, 2] in LDS
template <int DT, int V, int ACT, int NT>
__device__ __forceinline__ void apply_rows(const NormArgs& a, int b, int lo, int hi, int rows, const float* stats) {
    const int packs = a.C / V, live = hi < rows ? hi : rows;
    for (int first = 0; first < packs; first += NT) {
        const Lanes<NT, true> l(packs, first);
        if (l.r >= l.lanes) continue;
        Affine<V> f;
        f.load(a, stats, l.c * V);
#pragma unroll
        for (int i = 0; i < V; ++i) f.w[i] *= f.r[i];
        const int64_t base = int64_t(b) * a.xi + int64_t(l.c) * V, to = int64_t(b) * a.S * a.C + int64_t(l.c) * V;
        Pack<DT, V> p[4];
        walk_rows<4>(lo, live, l.r, l.lanes, [&](int64_t row, int j) { p[j] = load_pack<DT, V>(a.x, base + row * a.xr); },
                     [&](int64_t row, int j) {
                         float y[V];
                         unpack<DT, V>(p[j], y);
#pragma unroll
                         for (int i = 0; i < V; ++i) y[i] = act_value<ACT>(fmaf(y[i] - f.m[i], f.w[i], f.sh[i]));
                         store_pack<DT, V>(a.out, to + row * a.C, y);
                     });
        float zero[V];
#pragma unroll
        for (int i = 0; i < V; ++i) zero[i] = 0.f;
        const int from = lo > live ? lo : live;
        for (int64_t row = int64_t(from) + l.r; row < hi; row += l.lanes) store_pack<DT, V>(a.out, to + row * a.C, zero);
    }
}

// an item in one workgroup: its second sweep finds the rows in the caches
template <int DT, int V, int ACT>
__global__ void __launch_bounds__(kItemThreads) k_norm_item(NormArgs a) {
    float* stats = reinterpret_cast<float*>(dyn_lds());  // [G, 2]
    const int b = a.first + blockIdx.x, rows = item_rows(a.lengths, b, a.S);
    group_moments<DT, V, kItemThreads>(a, b, 0, rows, stats + 2 * a.G, stats);
    for (int g = threadIdx.x; g < a.G; g += kItemThreads) {
        const float r = inv_std(stats[2 * g + 1], rows, a.C / a.G, a.eps);
        stats[2 * g + 1] = r;
        if (a.stats) {
            a.stats[(int64_t(b) * a.G + g) * 2] = stats[2 * g];
            a.stats[(int64_t(b) * a.G + g) * 2 + 1] = r;
        }
    }
    __syncthreads();
    apply_rows<DT, V, ACT, kItemThreads>(a, b, 0, a.S, rows, stats);
}

// a small item: its values stay in registers (four packs a thread at most), so it is read once, and the variance is summed around
// the mean itself
template <int DT, int V, int ACT>
__global__ void __launch_bounds__(kItemThreads) k_norm_held(NormArgs a) {
    constexpr int NT = kItemThreads, R = 4;
    float* stats = reinterpret_cast<float*>(dyn_lds());  // [G, 2]
    float* entries = stats + 2 * a.G;                    // [lanes][C]
    const int b = a.first + blockIdx.x, rows = item_rows(a.lengths, b, a.S), packs = a.C / V, cg = a.C / a.G;
    const Lanes<NT, false> l(packs, 0);
    const bool mine = l.r < l.lanes;
    const int64_t base = int64_t(b) * a.xi + int64_t(l.c) * V;
    float x[R][V];
    Pack<DT, V> p[R];
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const int row = l.r + j * l.lanes;
        if (mine && row < rows) p[j] = load_pack<DT, V>(a.x, base + int64_t(row) * a.xr);
    }
    float w[V], sh[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        w[i] = mine && a.weight ? a.weight[l.c * V + i] : 1.f;
        sh[i] = mine && a.bias ? a.bias[l.c * V + i] : 0.f;
    }
    int group[V];
    {
        int g = l.c * V / cg, in = l.c * V - g * cg;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            group[i] = g;
            if (++in == cg) in = 0, ++g;
        }
    }
    const float inv = rows ? 1.f / (float(rows) * float(cg)) : 0.f;
    float m[V], part[V];
#pragma unroll
    for (int i = 0; i < V; ++i) part[i] = 0.f;
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const bool on = mine && l.r + j * l.lanes < rows;
        if (on) unpack<DT, V>(p[j], x[j]);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (!on) x[j][i] = 0.f;
            part[i] += x[j][i];
        }
    }
    // twice: the sum of every group, by way of LDS -> stats[2 g + which].  Where the packs of a row divide the wave, its rows are
    // added among the lanes first
    const bool fold = l.cols <= 64 && (l.cols & (l.cols - 1)) == 0;
    const int runs = fold ? NT / 64 : l.lanes, run = fold ? int(threadIdx.x) >> 6 : l.r;
    auto sum_groups = [&](int which) {
        if (fold)
            for (int s = l.cols; s < 64; s <<= 1)
#pragma unroll
                for (int i = 0; i < V; ++i) part[i] += __shfl_xor(part[i], s);
        if (mine && (!fold || int(threadIdx.x & 63) < l.cols)) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                AUD_IN_TABLE(run * a.C + l.c * V + i, NT / packs * a.C);
                entries[run * a.C + l.c * V + i] = part[i];
            }
        }
        __syncthreads();
        for_groups<NT>(a.G, [&](int g, int lane, int q, bool there) {
            const int dr = q / cg, dc = q - dr * cg, r0 = lane / cg;
            float s = 0.f;
            for (int r = r0, c = lane - r0 * cg; r < runs;) {
                s += entries[r * a.C + g * cg + c];
                r += dr, c += dc;
                if (c >= cg) c -= cg, ++r;
            }
            s = sum_lanes(s, q) * inv;
            if (there && lane == 0) stats[2 * g + which] = s;
        });
        __syncthreads();
    };
    sum_groups(0);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        m[i] = mine ? stats[2 * group[i]] : 0.f;
        part[i] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const bool on = mine && l.r + j * l.lanes < rows;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            x[j][i] -= m[i];
            part[i] = on ? fmaf(x[j][i], x[j][i], part[i]) : part[i];
        }
    }
    sum_groups(1);
    if (a.stats)
        for (int g = threadIdx.x; g < a.G; g += NT) {
            a.stats[(int64_t(b) * a.G + g) * 2] = stats[2 * g];
            a.stats[(int64_t(b) * a.G + g) * 2 + 1] = 1.f / sqrtf(stats[2 * g + 1] + a.eps);
        }
    if (!mine) return;
#pragma unroll
    for (int i = 0; i < V; ++i) w[i] *= 1.f / sqrtf(stats[2 * group[i] + 1] + a.eps);
    const int64_t to = int64_t(b) * a.S * a.C + int64_t(l.c) * V;
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const int row = l.r + j * l.lanes;
        if (row >= a.S) continue;
        float y[V];
#pragma unroll
        for (int i = 0; i < V; ++i) y[i] = row < rows ? act_value<ACT>(fmaf(x[j][i], w[i], sh[i])) : 0.f;
        store_pack<DT, V>(a.out, to + int64_t(row) * a.C, y);
    }
}

// an item over several workgroups: moments of a chunk of rows -> part [B, chunks, G, 2]
template <int DT, int V>
__global__ void __launch_bounds__(kChunkThreads) k_norm_chunk(NormArgs a) {
    float* moments = reinterpret_cast<float*>(dyn_lds());
    const int chunk = (a.first + blockIdx.x) % a.chunks, b = (a.first + blockIdx.x) / a.chunks, rows = item_rows(a.lengths, b, a.S);
    const int lo = chunk * a.chunk_rows, hi = lo + a.chunk_rows < rows ? lo + a.chunk_rows : rows;
    group_moments<DT, V, kChunkThreads>(a, b, lo, hi, moments + 2 * a.G, moments);
    float* out = a.part + (int64_t(b) * a.chunks + chunk) * a.G * 2;
    for (int i = threadIdx.x; i < 2 * a.G; i += kChunkThreads) out[i] = moments[i];
}
// ... joined: (mean, 1 / std) of group g of item b from `chunks` moments, by p lanes
__device__ __forceinline__ void join_chunks(const NormArgs& a, int b, int g, int rows, int lane, int p, float& mean, float& r) {
    const float* q = a.part + (int64_t(b) * a.chunks * a.G + g) * 2;
    const int cg = a.C / a.G;
    float m = 0.f, m2 = 0.f;
    for (int c = lane; c < a.chunks; c += p) {
        const int left = rows - c * a.chunk_rows, n = left < 0 ? 0 : (left < a.chunk_rows ? left : a.chunk_rows);
        m = fmaf(float(n), q[int64_t(c) * a.G * 2], m);
    }
    m = rows ? sum_lanes(m, p) / float(rows) : 0.f;
    for (int c = lane; c < a.chunks; c += p) {
        const int left = rows - c * a.chunk_rows, n = left < 0 ? 0 : (left < a.chunk_rows ? left : a.chunk_rows);
        const float d = q[int64_t(c) * a.G * 2] - m;
        m2 += fmaf(float(n) * float(cg) * d, d, q[int64_t(c) * a.G * 2 + 1]);
    }
    mean = m;
    r = inv_std(sum_lanes(m2, p), rows, cg, a.eps);
}
__global__ void __launch_bounds__(kChunkThreads) k_norm_join(NormArgs a) {  // many groups: a thread each
    const int64_t i = int64_t(a.first + blockIdx.x) * kChunkThreads + threadIdx.x;
    if (i >= int64_t(a.B) * a.G) return;
    const int b = int(i / a.G), g = int(i % a.G);
    float m, r;
    join_chunks(a, b, g, item_rows(a.lengths, b, a.S), 0, 1, m, r);
    a.stats[i * 2] = m;
    a.stats[i * 2 + 1] = r;
}
// JOIN: the chunks' moments are joined here, by every workgroup of the item for itself; else a.stats holds them
template <int DT, int V, int ACT, bool JOIN>
__global__ void __launch_bounds__(kChunkThreads) k_norm_apply(NormArgs a) {
    float* stats = reinterpret_cast<float*>(dyn_lds());
    const int chunk = (a.first + blockIdx.x) % a.chunks, b = (a.first + blockIdx.x) / a.chunks, rows = item_rows(a.lengths, b, a.S);
    const int lo = chunk * a.chunk_rows, hi = lo + a.chunk_rows < a.S ? lo + a.chunk_rows : a.S;
    if constexpr (JOIN) {
        for_groups<kChunkThreads>(a.G, [&](int g, int lane, int p, bool there) {
            float m, r;
            join_chunks(a, b, g, rows, lane, p, m, r);
            if (!there || lane) return;
            stats[2 * g] = m;
            stats[2 * g + 1] = r;
            if (a.stats && chunk == 0) {
                a.stats[(int64_t(b) * a.G + g) * 2] = m;
                a.stats[(int64_t(b) * a.G + g) * 2 + 1] = r;
            }
        });
    } else {
        for (int i = threadIdx.x; i < 2 * a.G; i += kChunkThreads) stats[i] = a.stats[int64_t(b) * a.G * 2 + i];
    }
    __syncthreads();
    apply_rows<DT, V, ACT, kChunkThreads>(a, b, lo, hi, rows, stats);
}

// ---- gradients --------------------------------------------------------------------------------------------------------
// sums of q xh and q over rows [lo, hi) of item b, per channel -> LDS out [2][C]; entries: LDS [2][max(NT V, C)]
template <int DT, int V, int ACT, int NT>
__device__ __forceinline__ void channel_sums(const NormArgs& a, int b, int lo, int hi, const float* stats, float* entries, float* out) {
    const int packs = a.C / V, size = NT * V > a.C ? NT * V : a.C;
    int lanes = 1;
    for (int first = 0; first < packs; first += NT) {
        const Lanes<NT, false> l(packs, first);
        lanes = l.lanes;
        if (l.r >= l.lanes) continue;
        Affine<V> f;
        f.load(a, stats, l.c * V);
        float s0[V], s1[V];
#pragma unroll
        for (int i = 0; i < V; ++i) s0[i] = s1[i] = 0.f;
        const int64_t xb = int64_t(b) * a.xi + int64_t(l.c) * V, db = int64_t(b) * a.di + int64_t(l.c) * V;
        Pack<DT, V> px[2], pd[2];
        walk_rows<2>(lo, hi, l.r, l.lanes,
                     [&](int64_t row, int j) {
                         px[j] = load_pack<DT, V>(a.x, xb + row * a.xr);
                         pd[j] = load_pack<DT, V>(a.dy, db + row * a.dr);
                     },
                     [&](int64_t, int j) {
                         float x[V], d[V];
                         unpack<DT, V>(px[j], x);
                         unpack<DT, V>(pd[j], d);
#pragma unroll
                         for (int i = 0; i < V; ++i) {
                             const float xh = (x[i] - f.m[i]) * f.r[i];
                             const float q = d[i] * act_slope<ACT>(fmaf(xh, f.w[i], f.sh[i]));
                             s0[i] = fmaf(q, xh, s0[i]);
                             s1[i] += q;
                         }
                     });
#pragma unroll
        for (int i = 0; i < V; ++i) {
            AUD_IN_TABLE(l.r * a.C + l.c * V + i, size);
            entries[l.r * a.C + l.c * V + i] = s0[i];
            entries[size + l.r * a.C + l.c * V + i] = s1[i];
        }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * a.C; c += NT) {
        const float* p = entries + (c < a.C ? c : size + c - a.C);
        float s = 0.f;
        for (int r = 0; r < lanes; ++r) s += p[r * a.C];
        out[c] = s;
    }
    __syncthreads();
}
// 1/n sum t, 1/n sum t xh of every group from an item's channel sums [2][C] -> LDS out [G, 2]
template <int NT>
__device__ __forceinline__ void group_sums(const NormArgs& a, int rows, const float* sums, float* out) {
    const int cg = a.C / a.G;
    const float inv = rows ? 1.f / (float(rows) * float(cg)) : 0.f;
    for_groups<NT>(a.G, [&](int g, int lane, int p, bool there) {
        float t0 = 0.f, t1 = 0.f;
        for (int c = g * cg + lane; c < (g + 1) * cg; c += p) {
            const float w = a.weight ? a.weight[c] : 1.f;
            t0 = fmaf(w, sums[a.C + c], t0);
            t1 = fmaf(w, sums[c], t1);
        }
        t0 = sum_lanes(t0, p) * inv;
        t1 = sum_lanes(t1, p) * inv;
        if (there && lane == 0) {
            out[2 * g] = t0;
            out[2 * g + 1] = t1;
        }
    });
    __syncthreads();
}
template <int DT, int V, int ACT, int NT>
__device__ __forceinline__ void grad_rows(const NormArgs& a, int b, int lo, int hi, int rows, const float* stats, const float* gsum) {
    const int packs = a.C / V, live = hi < rows ? hi : rows;
    for (int first = 0; first < packs; first += NT) {
        const Lanes<NT, true> l(packs, first);
        if (l.r >= l.lanes) continue;
        Affine<V> f;
        f.load(a, stats, l.c * V);
        float u0[V], u1[V];
        const int cg = a.C / a.G;
        int g = l.c * V / cg, in = l.c * V - g * cg;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            u0[i] = gsum[2 * g];
            u1[i] = gsum[2 * g + 1];
            if (++in == cg) in = 0, ++g;
        }
        const int64_t xb = int64_t(b) * a.xi + int64_t(l.c) * V, db = int64_t(b) * a.di + int64_t(l.c) * V;
        const int64_t to = int64_t(b) * a.S * a.C + int64_t(l.c) * V;
        Pack<DT, V> px[2], pd[2];
        walk_rows<2>(lo, live, l.r, l.lanes,
                     [&](int64_t row, int j) {
                         px[j] = load_pack<DT, V>(a.x, xb + row * a.xr);
                         pd[j] = load_pack<DT, V>(a.dy, db + row * a.dr);
                     },
                     [&](int64_t row, int j) {
                         float x[V], d[V];
                         unpack<DT, V>(px[j], x);
                         unpack<DT, V>(pd[j], d);
#pragma unroll
                         for (int i = 0; i < V; ++i) {
                             const float xh = (x[i] - f.m[i]) * f.r[i];
                             const float t = d[i] * act_slope<ACT>(fmaf(xh, f.w[i], f.sh[i])) * f.w[i];
                             x[i] = f.r[i] * ((t - u0[i]) - xh * u1[i]);
                         }
                         store_pack<DT, V>(a.out, to + row * a.C, x);
                     });
        float zero[V];
#pragma unroll
        for (int i = 0; i < V; ++i) zero[i] = 0.f;
        const int from = lo > live ? lo : live;
        for (int64_t row = int64_t(from) + l.r; row < hi; row += l.lanes) store_pack<DT, V>(a.out, to + row * a.C, zero);
    }
}

// an item in one workgroup -> dx and its channel sums, part [B, 2, C] (one item: the parameters' gradients themselves)
template <int DT, int V, int ACT>
__global__ void __launch_bounds__(kItemThreads) k_norm_grad_item(NormArgs a) {
    float* stats = reinterpret_cast<float*>(dyn_lds());  // [G, 2]
    float *gsum = stats + 2 * a.G, *sums = gsum + 2 * a.G, *entries = sums + 2 * a.C;
    const int b = a.first + blockIdx.x, rows = item_rows(a.lengths, b, a.S);
    for (int i = threadIdx.x; i < 2 * a.G; i += kItemThreads) stats[i] = a.stats[int64_t(b) * a.G * 2 + i];
    __syncthreads();
    channel_sums<DT, V, ACT, kItemThreads>(a, b, 0, rows, stats, entries, sums);
    for (int c = threadIdx.x; c < 2 * a.C; c += kItemThreads) {
        if (a.B > 1) a.part[int64_t(b) * 2 * a.C + c] = sums[c];
        else if (c < a.C && a.dweight) a.dweight[c] = sums[c];
        else if (c >= a.C && a.dbias) a.dbias[c - a.C] = sums[c];
    }
    group_sums<kItemThreads>(a, rows, sums, gsum);
    grad_rows<DT, V, ACT, kItemThreads>(a, b, 0, a.S, rows, stats, gsum);
}

// an item over several workgroups: channel sums of a chunk -> part [B, chunks, 2, C]
template <int DT, int V, int ACT>
__global__ void __launch_bounds__(kChunkThreads) k_norm_grad_chunk(NormArgs a) {
    float* stats = reinterpret_cast<float*>(dyn_lds());
    float *sums = stats + 2 * a.G, *entries = sums + 2 * a.C;
    const int chunk = (a.first + blockIdx.x) % a.chunks, b = (a.first + blockIdx.x) / a.chunks, rows = item_rows(a.lengths, b, a.S);
    const int lo = chunk * a.chunk_rows, hi = lo + a.chunk_rows < rows ? lo + a.chunk_rows : rows;
    for (int i = threadIdx.x; i < 2 * a.G; i += kChunkThreads) stats[i] = a.stats[int64_t(b) * a.G * 2 + i];
    __syncthreads();
    channel_sums<DT, V, ACT, kChunkThreads>(a, b, lo, hi, stats, entries, sums);
    float* out = a.part + (int64_t(b) * a.chunks + chunk) * 2 * a.C;
    for (int c = threadIdx.x; c < 2 * a.C; c += kChunkThreads) out[c] = sums[c];
}
// ... its chunks added -> [B, 2, C] behind them
constexpr int kJoinCols = 64, kJoinLanes = 4;
__global__ void __launch_bounds__(kJoinCols * kJoinLanes) k_norm_grad_join(NormArgs a) {
    float* lds = reinterpret_cast<float*>(dyn_lds());
    const int blocks = (2 * a.C + kJoinCols - 1) / kJoinCols, b = (a.first + blockIdx.x) / blocks;
    const int c = (a.first + blockIdx.x) % blocks * kJoinCols + threadIdx.x % kJoinCols, lane = threadIdx.x / kJoinCols;
    float s = 0.f;
    if (c < 2 * a.C)
#pragma unroll 4
        for (int k = lane; k < a.chunks; k += kJoinLanes) s += a.part[(int64_t(b) * a.chunks + k) * 2 * a.C + c];
    lds[threadIdx.x] = s;
    __syncthreads();
    if (lane == 0 && c < 2 * a.C) {
        for (int k = 1; k < kJoinLanes; ++k) s += lds[k * kJoinCols + threadIdx.x];
        a.part[(int64_t(a.B) * a.chunks + b) * 2 * a.C + c] = s;
    }
}
// dx of a chunk of rows; the workgroups behind them add the items' channel sums up for the parameters
template <int DT, int V, int ACT>
__global__ void __launch_bounds__(kChunkThreads) k_norm_grad_apply(NormArgs a) {
    const float* sums = a.part + int64_t(a.B) * a.chunks * 2 * a.C;
    const int64_t work = int64_t(a.B) * a.chunks;
    if (a.first + blockIdx.x >= work) {
        const int c = int(a.first + blockIdx.x - work) * kChunkThreads + int(threadIdx.x);
        if (c >= 2 * a.C) return;
        float s = 0.f;
#pragma unroll 8
        for (int b = 0; b < a.B; ++b) s += sums[int64_t(b) * 2 * a.C + c];
        if (c < a.C && a.dweight) a.dweight[c] = s;
        if (c >= a.C && a.dbias) a.dbias[c - a.C] = s;
        return;
    }
    float* stats = reinterpret_cast<float*>(dyn_lds());
    float* gsum = stats + 2 * a.G;
    const int chunk = (a.first + blockIdx.x) % a.chunks, b = (a.first + blockIdx.x) / a.chunks, rows = item_rows(a.lengths, b, a.S);
    const int lo = chunk * a.chunk_rows, hi = lo + a.chunk_rows < a.S ? lo + a.chunk_rows : a.S;
    for (int i = threadIdx.x; i < 2 * a.G; i += kChunkThreads) stats[i] = a.stats[int64_t(b) * a.G * 2 + i];
    group_sums<kChunkThreads>(a, rows, sums + int64_t(b) * 2 * a.C, gsum);
    grad_rows<DT, V, ACT, kChunkThreads>(a, b, lo, hi, rows, stats, gsum);
}

// ---- column sums of a partial-result table ------------------------------------------------------------------------------
constexpr int kCsCols = 32, kCsLanes = 32;
__global__ void __launch_bounds__(kCsCols * kCsLanes) k_column_sums(const float* in, int64_t rows, int W, int K, int extra, float* out0,
                                                                   float* out1, float* out2, unsigned first) {
    float* lds = reinterpret_cast<float*>(dyn_lds());
    const int c = threadIdx.x % kCsCols, lane = threadIdx.x / kCsCols;
    const int64_t width = int64_t(W) * (K + extra), col = int64_t(first + blockIdx.x) * kCsCols + c;
    float s = 0.f;
    if (col < width)
#pragma unroll 4
        for (int64_t r = lane; r < rows; r += kCsLanes) s += in[r * width + col];
    lds[threadIdx.x] = s;
    __syncthreads();
    for (int k = kCsLanes / 2; k > 0; k >>= 1) {
        if (lane < k) lds[threadIdx.x] += lds[threadIdx.x + k * kCsCols];
        __syncthreads();
    }
    if (lane == 0 && col < width) {
        s = lds[c];
        const int k = int(col / W), w = int(col % W);
        if (k < K) {
            if (out0) out0[int64_t(w) * K + k] = s;
        } else {
            float* out = k == K ? out1 : out2;
            if (out) out[w] = s;
        }
    }
}

inline size_t entries_of(int nt, int V, int C) { return size_t(2) * size_t(std::max(nt * V, C)); }

template <int DT, int V, int ACT>
hipError_t run(const NormArgs& a, const NormRoute& r, hipStream_t st) {
    const int packs = a.C / V;
    if (r.one_wg && packs <= kItemThreads && int64_t(a.S) <= 4 * (kItemThreads / packs)) {
        const size_t lds = (2 * size_t(a.G) + size_t(kItemThreads / packs) * a.C) * 4;
        if (hipError_t e = allow_lds<&k_norm_held<DT, V, ACT>>(lds)) return e;
        return in_slices_of(a, a.B, kItemThreads, [&](dim3 grid, const NormArgs& s) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(k_norm_held<DT, V, ACT>), grid, dim3(kItemThreads), lds, st, s);
        });
    }
    if (r.one_wg) {
        const size_t lds = (2 * size_t(a.G) + entries_of(kItemThreads, V, a.C)) * 4;
        if (hipError_t e = allow_lds<&k_norm_item<DT, V, ACT>>(lds)) return e;
        return in_slices_of(a, a.B, kItemThreads, [&](dim3 grid, const NormArgs& s) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(k_norm_item<DT, V, ACT>), grid, dim3(kItemThreads), lds, st, s);
        });
    }
    const int64_t work = int64_t(a.chunks) * a.B;
    const dim3 wg(kChunkThreads);
    const size_t lds = (2 * size_t(a.G) + entries_of(kChunkThreads, V, a.C)) * 4;
    if (hipError_t e = allow_lds<&k_norm_chunk<DT, V>>(lds)) return e;
    if (hipError_t e = in_slices_of(a, work, kChunkThreads, [&](dim3 grid, const NormArgs& s) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(k_norm_chunk<DT, V>), grid, wg, lds, st, s);
        }))
        return e;
    if (!r.join)
        return in_slices_of(a, work, kChunkThreads, [&](dim3 grid, const NormArgs& s) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(k_norm_apply<DT, V, ACT, true>), grid, wg, size_t(s.G) * 8, st, s);
        });
    const int64_t join = (int64_t(a.B) * a.G + kChunkThreads - 1) / kChunkThreads;
    if (hipError_t e = in_slices_of(a, join, kChunkThreads,
                                    [&](dim3 grid, const NormArgs& s) { hipLaunchKernelGGL(k_norm_join, grid, wg, 0, st, s); }))
        return e;
    return in_slices_of(a, work, kChunkThreads, [&](dim3 grid, const NormArgs& s) {
        hipLaunchKernelGGL(HIP_KERNEL_NAME(k_norm_apply<DT, V, ACT, false>), grid, wg, size_t(s.G) * 8, st, s);
    });
}

template <int DT, int V, int ACT>
hipError_t run_grad(const NormArgs& a, const NormRoute& r, hipStream_t st) {
    if (r.one_wg) {
        const size_t lds = (4 * size_t(a.G) + 2 * size_t(a.C) + entries_of(kItemThreads, V, a.C)) * 4;
        if (hipError_t e = allow_lds<&k_norm_grad_item<DT, V, ACT>>(lds)) return e;
        if (hipError_t e = in_slices_of(a, a.B, kItemThreads, [&](dim3 grid, const NormArgs& s) {
                hipLaunchKernelGGL(HIP_KERNEL_NAME(k_norm_grad_item<DT, V, ACT>), grid, dim3(kItemThreads), lds, st, s);
            }))
            return e;
        if (a.B == 1 || (!a.dweight && !a.dbias)) return hipSuccess;
        return launch_column_sums(a.part, a.B, a.C, 0, 2, nullptr, a.dweight, a.dbias, st);
    }
    const int64_t work = int64_t(a.chunks) * a.B;
    const size_t lds = (2 * size_t(a.G) + 2 * size_t(a.C) + entries_of(kChunkThreads, V, a.C)) * 4;
    if (hipError_t e = allow_lds<&k_norm_grad_chunk<DT, V, ACT>>(lds)) return e;
    if (hipError_t e = in_slices_of(a, work, kChunkThreads, [&](dim3 grid, const NormArgs& s) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(k_norm_grad_chunk<DT, V, ACT>), grid, dim3(kChunkThreads), lds, st, s);
        }))
        return e;
    const int64_t join = int64_t(a.B) * ((2 * a.C + kJoinCols - 1) / kJoinCols);
    if (hipError_t e = in_slices_of(a, join, kJoinCols * kJoinLanes, [&](dim3 grid, const NormArgs& s) {
            hipLaunchKernelGGL(k_norm_grad_join, grid, dim3(kJoinCols * kJoinLanes), size_t(kJoinCols) * kJoinLanes * 4, st, s);
        }))
        return e;
    const int64_t more = a.dweight || a.dbias ? (2 * a.C + kChunkThreads - 1) / kChunkThreads : 0;
    return in_slices_of(a, work + more, kChunkThreads, [&](dim3 grid, const NormArgs& s) {
        hipLaunchKernelGGL(HIP_KERNEL_NAME(k_norm_grad_apply<DT, V, ACT>), grid, dim3(kChunkThreads), size_t(s.G) * 16, st, s);
    });
}

template <int DT, int V>
hipError_t by_act(const NormArgs& a, const NormRoute& r, int act, bool grad, hipStream_t st) {
    switch (act) {
        case AUD_ACT_RELU: return grad ? run_grad<DT, V, AUD_ACT_RELU>(a, r, st) : run<DT, V, AUD_ACT_RELU>(a, r, st);
        case AUD_ACT_SILU: return grad ? run_grad<DT, V, AUD_ACT_SILU>(a, r, st) : run<DT, V, AUD_ACT_SILU>(a, r, st);
        case AUD_ACT_GELU: return grad ? run_grad<DT, V, AUD_ACT_GELU>(a, r, st) : run<DT, V, AUD_ACT_GELU>(a, r, st);
        default: return grad ? run_grad<DT, V, AUD_ACT_NONE>(a, r, st) : run<DT, V, AUD_ACT_NONE>(a, r, st);
    }
}
hipError_t by_type(const NormArgs& a, const NormRoute& r, int dtype, int act, bool grad, hipStream_t st) {
    switch (dtype) {
        case AUD_F32:
            return r.vec == 4   ? by_act<AUD_F32, 4>(a, r, act, grad, st)
                   : r.vec == 2 ? by_act<AUD_F32, 2>(a, r, act, grad, st)
                                : by_act<AUD_F32, 1>(a, r, act, grad, st);
        case AUD_BF16:
            return r.vec == 8   ? by_act<AUD_BF16, 8>(a, r, act, grad, st)
                   : r.vec == 4 ? by_act<AUD_BF16, 4>(a, r, act, grad, st)
                   : r.vec == 2 ? by_act<AUD_BF16, 2>(a, r, act, grad, st)
                                : by_act<AUD_BF16, 1>(a, r, act, grad, st);
        default:
            return r.vec == 8   ? by_act<AUD_F16, 8>(a, r, act, grad, st)
                   : r.vec == 4 ? by_act<AUD_F16, 4>(a, r, act, grad, st)
                   : r.vec == 2 ? by_act<AUD_F16, 2>(a, r, act, grad, st)
                                : by_act<AUD_F16, 1>(a, r, act, grad, st);
    }
}

}  // namespace

hipError_t launch_column_sums(const float* in, int64_t rows, int W, int K, int extra, float* out0, float* out1, float* out2, hipStream_t st) {
    const int64_t width = int64_t(W) * (K + extra);
    return in_slices((width + kCsCols - 1) / kCsCols, kCsCols * kCsLanes, [&](dim3 grid, unsigned first) {
        hipLaunchKernelGGL(k_column_sums, grid, dim3(kCsCols * kCsLanes), size_t(kCsCols) * kCsLanes * 4, st, in, rows, W, K, extra, out0,
                           out1, out2, first);
    });
}

int vector_of(int e, int C, int align) {
    for (int v = 16 / e; v > 1; v /= 2)
        if (align >= v * e && C % v == 0) return v;
    return 1;
}

NormRoute norm_route(int dtype, int B, int S, int C, int G, int align, bool) {
    NormRoute r{};
    const int e = dtype == AUD_F32 ? 4 : 2;
    r.vec = vector_of(e, C, align);
    const int64_t bytes = int64_t(S) * C * e;
    r.one_wg = bytes <= 32 * 1024 || (B >= 256 && bytes <= 128 * 1024) || (B >= 1024 && bytes <= 1024 * 1024);
    r.chunks = 1;
    r.chunk_rows = S;
    if (!r.one_wg) {
        // about 512 workgroups, two a CU, at least 8 KB of input each (16 x 4096 x 512 bfloat16, values and gradients: 110 us;
        // 256 workgroups 116, 768 114, 1024 118, 2048 145)
        int64_t chunks = std::min<int64_t>((512 + B - 1) / B, kMaxChunks);
        chunks = std::max<int64_t>(1, std::min<int64_t>(chunks, std::min<int64_t>(S, bytes / 8192)));
        r.chunk_rows = int((S + chunks - 1) / chunks);
        r.chunks = (S + r.chunk_rows - 1) / r.chunk_rows;
    }
    r.join = int64_t(r.chunks) * G > 8192;
    return r;
}

int64_t norm_workspace_floats(const NormRoute& r, int B, int C, int G, bool grad) {
    if (grad) return r.one_wg ? (B > 1 ? int64_t(B) * 2 * C : 0) : int64_t(B) * (r.chunks + 1) * 2 * C;
    // the chunks' moments, and the statistics where they are joined by a kernel of their own and the caller keeps none
    return r.one_wg ? 0 : int64_t(B) * r.chunks * G * 2 + (r.join ? int64_t(B) * G * 2 : 0);
}

hipError_t launch_norm(const NormArgs& a, const NormRoute& r, int dtype, int act, hipStream_t st) {
    return by_type(a, r, dtype, act, false, st);
}
hipError_t launch_norm_grad(const NormArgs& a, const NormRoute& r, int dtype, int act, hipStream_t st) {
    return by_type(a, r, dtype, act, true, st);
}

}  // namespace aud
