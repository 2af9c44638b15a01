// Group norm with an activation on channels-last data: x [n][rows][c], groups of c / groups neighbouring channels.
//
//   xhat = (x - mean) rstd,  z = gamma xhat + beta,  y = act(z)        mean, var over the rows and channels of (sample, group)
//   dz = dy act'(z);  dbeta = sum dz, dgamma = sum dz xhat over samples and rows
//   dx = rstd (gamma dz - s1 - xhat s2),   s1, s2 = means over the group of gamma dz and of gamma dz xhat
//
// The sums of the statistics are in fp64, and mean and rstd are kept as fp64: their rounding moves every element of a group
// together, an fp32 sum of squares loses a small variance under a large mean, and ReLU's border in the backward pass (is z
// over zero?) is decided by a threshold on x that is worked out in fp64 and rounded so that no fp32 x lies between it and the
// true one.  The rest is fp32; the gradient sums are fp32 within a workgroup's rows and fp64 across workgroups, always in the
// same order.
//
// What bounds it: HBM, and the launches at small sizes.  Three launches each way: sums over a chunk of rows, one value per
// (sample, group) from the chunks' sums, and the pass that writes.  The second read of x (and dy) comes from the 256 MB cache
// where the tensors fit in it.  A thread keeps to one vector of neighbouring channels, so that its gamma, beta and statistics
// stay in registers, and a workgroup's accesses cover whole rows, contiguous in memory.
#include "common.h"
#include "../../include/geomae_hip.h"
#include <math.h>
#include <type_traits>

namespace geomae {

constexpr int kGnThreads = 256;
constexpr int kGnUnroll = 4;                       // rows in flight per thread
constexpr int kGnMaxGroups = 1024;
constexpr int kGnBlocks = 1024;                    // workgroups of a pass: four per CU
constexpr int kGnFold = 64;                        // samples whose sums one thread adds up for the parameters' gradients

enum { kGnNone = 0, kGnRelu = 1, kGnSilu = 2, kGnGelu = 3 };

struct GnShape {
    int64_t rows;                                  // of a sample
    int32_t n, c, groups, cg;
    int32_t chunks;                                // of a sample's rows
    int64_t chunk_rows;
};

template <typename T> __device__ __forceinline__ float gn_float(T x) { return (float)x; }
template <> __device__ __forceinline__ float gn_float<uint16_t>(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }   // bf16
template <typename T> __device__ __forceinline__ T gn_narrow(float x) { return (T)x; }
template <> __device__ __forceinline__ uint16_t gn_narrow<uint16_t>(float x) {
    const uint32_t b = __float_as_uint(x);
    return x != x ? (uint16_t)((b >> 16) | 0x40) : (uint16_t)((b + 0x7fff + ((b >> 16) & 1)) >> 16);
}
// (element-aligned: a tensor may start anywhere, and global memory takes wide accesses at any element's address)
template <typename T, int V> struct __attribute__((packed, aligned(sizeof(T)))) GnPack { T v[V]; };
template <typename T, int V> __device__ __forceinline__ GnPack<T, V> gn_read(const T* p) { return *reinterpret_cast<const GnPack<T, V>*>(p); }

template <int ACT> __device__ __forceinline__ float gn_act(float z) {
    if constexpr (ACT == kGnRelu) return z < 0.f ? 0.f : z;            // NaN stays
    if constexpr (ACT == kGnSilu) return z / (1.0f + expf(-z));
    if constexpr (ACT == kGnGelu) return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
    return z;
}
template <int ACT> __device__ __forceinline__ float gn_slope(float z) {     // (ReLU's: gn_threshold)
    if constexpr (ACT == kGnSilu) {
        const float s = 1.0f / (1.0f + expf(-z));
        return s * (1.0f + z * (1.0f - s));
    }
    if constexpr (ACT == kGnGelu)
        return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) + z * 0.39894228040143268f * expf(-0.5f * z * z);
    return 1.0f;
}
// z > 0 as a comparison of sign * x with a threshold
__device__ __forceinline__ void gn_threshold(double mean, double scale, double beta, float& sign, float& thr) {
    sign = scale < 0.0 ? -1.0f : 1.0f;
    if (scale == 0.0) {
        thr = beta > 0.0 ? -INFINITY : INFINITY;
        return;
    }
    const double t = (mean - beta / scale) * (double)sign;
    float f = (float)t;
    if ((double)f > t) f = nextafterf(f, -INFINITY);
    thr = f;
}

__device__ __forceinline__ float gn_weight(const void* w, int dtype, int c, float none) {
    if (!w) return none;
    if (dtype == GEOMAE_DTYPE_F32) return static_cast<const float*>(w)[c];
    if (dtype == GEOMAE_DTYPE_BF16) return gn_float(static_cast<const uint16_t*>(w)[c]);
    return gn_float(static_cast<const _Float16*>(w)[c]);
}

// ------------------------------------------------------------------------------------------------ sums of x
// the workgroup's lanes as tx columns (vectors of V channels) x ty rows; c > 256 V is walked in tiles of 256 V channels
struct GnLanes {
    int tx, ty, col, row;
    bool live;
};
template <int V> __device__ __forceinline__ GnLanes gn_lanes(int c, int tile) {
    GnLanes l;
    const int cv = (c - tile * kGnThreads * V) / V;
    l.tx = cv < kGnThreads ? cv : kGnThreads;
    l.ty = kGnThreads / l.tx;
    l.row = threadIdx.x / l.tx;
    l.col = (tile * kGnThreads + (int)threadIdx.x - l.row * l.tx) * V;
    l.live = l.row < l.ty;
    return l;
}

// a[2 V] of every lane summed over the lanes of its column into slot (column) of the LDS array; fixed order
template <typename S, int W>
__device__ __forceinline__ void gn_sum_rows(S (&a)[W], const GnLanes& l, S* lds) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) lds[i * kGnThreads + threadIdx.x] = a[i];
    for (int have = l.ty; have > 1;) {
        const int half = (have + 1) >> 1;
        __syncthreads();
        if (l.live && l.row + half < have) {
#pragma unroll
            for (int i = 0; i < W; ++i) lds[i * kGnThreads + threadIdx.x] += lds[i * kGnThreads + threadIdx.x + half * l.tx];
        }
        have = half;
    }
    __syncthreads();
}

template <typename T, int V>
__global__ __launch_bounds__(kGnThreads) void gn_sums_kernel(const T* __restrict__ x, GnShape s, double2* __restrict__ partial) {
    __shared__ double lds[2 * V * kGnThreads];
    __shared__ double2 group[kGnMaxGroups];
    const int n = blockIdx.x / s.chunks, chunk = blockIdx.x - n * s.chunks;
    const int64_t r0 = chunk * s.chunk_rows, r1 = r0 + s.chunk_rows < s.rows ? r0 + s.chunk_rows : s.rows;
    x += (int64_t)n * s.rows * s.c;
    for (int g = threadIdx.x; g < s.groups; g += kGnThreads) group[g] = make_double2(0.0, 0.0);
    const int tiles = (s.c + kGnThreads * V - 1) / (kGnThreads * V);
    for (int tile = 0; tile < tiles; ++tile) {
        const GnLanes l = gn_lanes<V>(s.c, tile);
        double a[2 * V];
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) a[i] = 0.0;
        if (l.live) {
            for (int64_t r = r0 + l.row; r < r1; r += kGnUnroll * l.ty) {
                GnPack<T, V> w[kGnUnroll];
#pragma unroll
                for (int u = 0; u < kGnUnroll; ++u)
                    if (r + u * l.ty < r1) w[u] = gn_read<T, V>(x + (r + u * l.ty) * s.c + l.col);
#pragma unroll
                for (int u = 0; u < kGnUnroll; ++u)
                    if (r + u * l.ty < r1) {
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            const double v = (double)gn_float(w[u].v[i]);
                            a[i] += v;
                            a[V + i] = fma(v, v, a[V + i]);
                        }
                    }
            }
        }
        gn_sum_rows<double, 2 * V>(a, l, lds);
        // channels -> groups: a wave per group that begins in or reaches into this tile
        const int c0 = tile * kGnThreads * V, c1 = c0 + l.tx * V;
        for (int g = c0 / s.cg + (int)(threadIdx.x >> 6); g * s.cg < c1 && g < s.groups; g += kGnThreads / kWave) {
            const int b = g * s.cg > c0 ? g * s.cg : c0, e = (g + 1) * s.cg < c1 ? (g + 1) * s.cg : c1;
            double sum = 0.0, sq = 0.0;
            for (int ch = b + lane_id(); ch < e; ch += kWave) {
                const int v = (ch - c0) / V, i = (ch - c0) - v * V;
                sum += lds[i * kGnThreads + v];
                sq += lds[(V + i) * kGnThreads + v];
            }
            sum = wave_sum(sum);
            sq = wave_sum(sq);
            if (lane_id() == 0) group[g] = make_double2(group[g].x + sum, group[g].y + sq);
        }
    }
    __syncthreads();
    for (int g = threadIdx.x; g < s.groups; g += kGnThreads) partial[((int64_t)n * s.chunks + chunk) * s.groups + g] = group[g];
}

// a wave per (sample, group): mean and 1 / sqrt(var + eps)
__global__ __launch_bounds__(kGnThreads) void gn_stats_kernel(const double2* __restrict__ partial, GnShape s, double eps, double2* __restrict__ stats) {
    const int64_t at = (int64_t)blockIdx.x * (kGnThreads / kWave) + (threadIdx.x >> 6);
    if (at >= (int64_t)s.n * s.groups) return;
    const int64_t n = at / s.groups, g = at - n * s.groups;
    double sum = 0.0, sq = 0.0;
    for (int k = lane_id(); k < s.chunks; k += kWave) {
        const double2 p = partial[(n * s.chunks + k) * s.groups + g];
        sum += p.x;
        sq += p.y;
    }
    sum = wave_sum(sum);
    sq = wave_sum(sq);
    if (lane_id() == 0) {
        const double m = (double)s.rows * s.cg, mean = sum / m;
        double var = sq / m - mean * mean;
        var = var < 0.0 ? 0.0 : var;                                   // (NaN stays)
        stats[at] = make_double2(mean, 1.0 / sqrt(var + eps));
    }
}

// ------------------------------------------------------------------------------------------------ y
template <typename T, int V, int ACT>
__global__ __launch_bounds__(kGnThreads) void gn_forward_kernel(const T* __restrict__ x, GnShape s, const double2* __restrict__ stats,
                                                               const void* gamma, const void* beta, int wdtype, T* __restrict__ y) {
    const int n = blockIdx.x / s.chunks, chunk = blockIdx.x - n * s.chunks;
    const int64_t r0 = chunk * s.chunk_rows, r1 = r0 + s.chunk_rows < s.rows ? r0 + s.chunk_rows : s.rows;
    const int64_t base = (int64_t)n * s.rows * s.c;
    const int tiles = (s.c + kGnThreads * V - 1) / (kGnThreads * V);
    for (int tile = 0; tile < tiles; ++tile) {
        const GnLanes l = gn_lanes<V>(s.c, tile);
        if (!l.live) continue;
        float mh[V], ml[V], sc[V], sh[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const double2 st = stats[(int64_t)n * s.groups + (l.col + i) / s.cg];
            mh[i] = (float)st.x;
            ml[i] = (float)(st.x - (double)mh[i]);
            sc[i] = (float)(st.y * (double)gn_weight(gamma, wdtype, l.col + i, 1.f));
            sh[i] = gn_weight(beta, wdtype, l.col + i, 0.f);
        }
        for (int64_t r = r0 + l.row; r < r1; r += kGnUnroll * l.ty) {
            GnPack<T, V> w[kGnUnroll];
#pragma unroll
            for (int u = 0; u < kGnUnroll; ++u)
                if (r + u * l.ty < r1) w[u] = gn_read<T, V>(x + base + (r + u * l.ty) * s.c + l.col);
#pragma unroll
            for (int u = 0; u < kGnUnroll; ++u)
                if (r + u * l.ty < r1) {
                    GnPack<T, V> o;
#pragma unroll
                    for (int i = 0; i < V; ++i) o.v[i] = gn_narrow<T>(gn_act<ACT>(((gn_float(w[u].v[i]) - mh[i]) - ml[i]) * sc[i] + sh[i]));
                    *reinterpret_cast<GnPack<T, V>*>(y + base + (r + u * l.ty) * s.c + l.col) = o;
                }
        }
    }
}

// ------------------------------------------------------------------------------------------------ gradients
// what a lane keeps of its V channels for xhat and dz
template <int V, int ACT> struct GnChannels {
    float mh[V], ml[V], rstd[V], gamma[V], beta[V], sign[V], thr[V];
    __device__ __forceinline__ void load(const GnShape& s, const double2* stats, const void* g, const void* b, int wdtype, int n, int col) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const double2 st = stats[(int64_t)n * s.groups + (col + i) / s.cg];
            mh[i] = (float)st.x;
            ml[i] = (float)(st.x - (double)mh[i]);
            rstd[i] = (float)st.y;
            gamma[i] = gn_weight(g, wdtype, col + i, 1.f);
            beta[i] = gn_weight(b, wdtype, col + i, 0.f);
            if constexpr (ACT == kGnRelu) gn_threshold(st.x, st.y * (double)gamma[i], (double)beta[i], sign[i], thr[i]);
        }
    }
    __device__ __forceinline__ void value(int i, float x, float dy, float& xhat, float& dz) const {
        xhat = ((x - mh[i]) - ml[i]) * rstd[i];
        if constexpr (ACT == kGnRelu) dz = x * sign[i] > thr[i] ? dy : 0.f;
        else dz = dy * gn_slope<ACT>(xhat * gamma[i] + beta[i]);
    }
};

// per (sample, chunk, channel): (sum dz, sum dz xhat)
template <typename T, int V, int ACT>
__global__ __launch_bounds__(kGnThreads) void gn_grad_sums_kernel(const T* __restrict__ x, const T* __restrict__ dy, GnShape s,
                                                                 const double2* __restrict__ stats, const void* gamma, const void* beta,
                                                                 int wdtype, float2* __restrict__ partial) {
    __shared__ float lds[2 * V * kGnThreads];
    const int n = blockIdx.x / s.chunks, chunk = blockIdx.x - n * s.chunks;
    const int64_t r0 = chunk * s.chunk_rows, r1 = r0 + s.chunk_rows < s.rows ? r0 + s.chunk_rows : s.rows;
    const int64_t base = (int64_t)n * s.rows * s.c;
    const int tiles = (s.c + kGnThreads * V - 1) / (kGnThreads * V);
    for (int tile = 0; tile < tiles; ++tile) {
        const GnLanes l = gn_lanes<V>(s.c, tile);
        float a[2 * V];
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) a[i] = 0.f;
        if (l.live) {
            GnChannels<V, ACT> ch;
            ch.load(s, stats, gamma, beta, wdtype, n, l.col);
            for (int64_t r = r0 + l.row; r < r1; r += kGnUnroll * l.ty) {
                GnPack<T, V> w[kGnUnroll], d[kGnUnroll];
#pragma unroll
                for (int u = 0; u < kGnUnroll; ++u)
                    if (r + u * l.ty < r1) {
                        w[u] = gn_read<T, V>(x + base + (r + u * l.ty) * s.c + l.col);
                        d[u] = gn_read<T, V>(dy + base + (r + u * l.ty) * s.c + l.col);
                    }
#pragma unroll
                for (int u = 0; u < kGnUnroll; ++u)
                    if (r + u * l.ty < r1) {
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            float xhat, dz;
                            ch.value(i, gn_float(w[u].v[i]), gn_float(d[u].v[i]), xhat, dz);
                            a[i] += dz;
                            a[V + i] += dz * xhat;
                        }
                    }
            }
        }
        gn_sum_rows<float, 2 * V>(a, l, lds);
        if (l.live && l.row == 0) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                partial[((int64_t)n * s.chunks + chunk) * s.c + l.col + i] =
                    make_float2(lds[i * kGnThreads + threadIdx.x], lds[(V + i) * kGnThreads + threadIdx.x]);
        }
    }
}

// a workgroup per (sample, group): the channels' sums over the chunks, and the group's two means
__global__ __launch_bounds__(kGnThreads) void gn_grad_stats_kernel(const float2* __restrict__ partial, GnShape s, const void* gamma, int wdtype,
                                                                  double2* __restrict__ channel, float2* __restrict__ means) {
    __shared__ double2 lds[kGnThreads];
    const int n = blockIdx.x / s.groups, g = blockIdx.x - n * s.groups;
    double s1 = 0.0, s2 = 0.0;
    for (int c0 = 0; c0 < s.cg; c0 += kGnThreads) {
        const int tx = s.cg - c0 < kGnThreads ? s.cg - c0 : kGnThreads, ty = kGnThreads / tx;
        const int row = threadIdx.x / tx, ch = g * s.cg + c0 + (threadIdx.x - row * tx);
        double2 acc = make_double2(0.0, 0.0);
        if (row < ty)
            for (int k = row; k < s.chunks; k += ty) {
                const float2 p = partial[((int64_t)n * s.chunks + k) * s.c + ch];
                acc.x += p.x;
                acc.y += p.y;
            }
        __syncthreads();
        lds[threadIdx.x] = acc;
        for (int have = ty; have > 1;) {
            const int half = (have + 1) >> 1;
            __syncthreads();
            if (row + half < have) {
                const double2 o = lds[threadIdx.x + half * tx];
                lds[threadIdx.x].x += o.x;
                lds[threadIdx.x].y += o.y;
            }
            have = half;
        }
        if (row == 0) {
            const double2 sum = lds[threadIdx.x];
            channel[(int64_t)n * s.c + ch] = sum;
            const double w = (double)gn_weight(gamma, wdtype, ch, 1.f);
            s1 += w * sum.x;
            s2 += w * sum.y;
        }
    }
    s1 = wave_sum(s1);
    s2 = wave_sum(s2);
    __syncthreads();
    if (lane_id() == 0) lds[threadIdx.x >> 6] = make_double2(s1, s2);
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kGnThreads / kWave; ++w) { s1 += lds[w].x; s2 += lds[w].y; }
        const double m = (double)s.rows * s.cg;
        means[(int64_t)n * s.groups + g] = make_float2((float)(s1 / m), (float)(s2 / m));
    }
}

__device__ __forceinline__ void gn_store_weight(void* w, int dtype, int c, float v) {
    if (!w) return;
    if (dtype == GEOMAE_DTYPE_F32) static_cast<float*>(w)[c] = v;
    else if (dtype == GEOMAE_DTYPE_BF16) static_cast<uint16_t*>(w)[c] = gn_narrow<uint16_t>(v);
    else static_cast<_Float16*>(w)[c] = gn_narrow<_Float16>(v);
}

// d gamma, d beta: the samples' sums of a channel, a channel per thread over the launch's first workgroups
__device__ __forceinline__ void gn_weight_grad(const double2* channel, int rows, int c, int wdtype, void* dgamma, void* dbeta, int block, int blocks) {
    for (int64_t ch = (int64_t)block * kGnThreads + threadIdx.x; ch < c; ch += (int64_t)blocks * kGnThreads) {
        double a = 0.0, b = 0.0;
        for (int n = 0; n < rows; ++n) {
            const double2 p = channel[(int64_t)n * c + ch];
            a += p.x;
            b += p.y;
        }
        gn_store_weight(dbeta, wdtype, (int)ch, (float)a);
        gn_store_weight(dgamma, wdtype, (int)ch, (float)b);
    }
}
__global__ __launch_bounds__(kGnThreads) void gn_weight_grad_kernel(const double2* __restrict__ channel, int rows, int c, int wdtype, void* dgamma, void* dbeta) {
    gn_weight_grad(channel, rows, c, wdtype, dgamma, dbeta, blockIdx.x, gridDim.x);
}
// many samples: first to sums of kGnFold samples each
__global__ __launch_bounds__(kGnThreads) void gn_fold_kernel(const double2* __restrict__ channel, int n, int c, double2* __restrict__ out) {
    const int64_t at = (int64_t)blockIdx.x * kGnThreads + threadIdx.x, rows = (n + kGnFold - 1) / kGnFold;
    if (at >= rows * c) return;
    const int64_t r = at / c, ch = at - r * c;
    double2 acc = make_double2(0.0, 0.0);
    for (int64_t k = r * kGnFold; k < (r + 1) * kGnFold && k < n; ++k) {
        const double2 p = channel[k * c + ch];
        acc.x += p.x;
        acc.y += p.y;
    }
    out[at] = acc;
}

template <typename T, int V, int ACT>
__global__ __launch_bounds__(kGnThreads) void gn_backward_kernel(const T* __restrict__ x, const T* __restrict__ dy, GnShape s,
                                                                const double2* __restrict__ stats, const void* gamma, const void* beta,
                                                                int wdtype, const double2* __restrict__ channel,
                                                                const float2* __restrict__ means, T* __restrict__ dx, void* dgamma, void* dbeta) {
    const int n = blockIdx.x / s.chunks, chunk = blockIdx.x - n * s.chunks;
    const int64_t r0 = chunk * s.chunk_rows, r1 = r0 + s.chunk_rows < s.rows ? r0 + s.chunk_rows : s.rows;
    const int64_t base = (int64_t)n * s.rows * s.c;
    if (dgamma || dbeta) gn_weight_grad(channel, s.n, s.c, wdtype, dgamma, dbeta, blockIdx.x, gridDim.x);
    const int tiles = (s.c + kGnThreads * V - 1) / (kGnThreads * V);
    for (int tile = 0; tile < tiles; ++tile) {
        const GnLanes l = gn_lanes<V>(s.c, tile);
        if (!l.live) continue;
        GnChannels<V, ACT> ch;
        ch.load(s, stats, gamma, beta, wdtype, n, l.col);
        float s1[V], s2[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float2 m = means[(int64_t)n * s.groups + (l.col + i) / s.cg];
            s1[i] = m.x;
            s2[i] = m.y;
        }
        for (int64_t r = r0 + l.row; r < r1; r += kGnUnroll * l.ty) {
            GnPack<T, V> w[kGnUnroll], d[kGnUnroll];
#pragma unroll
            for (int u = 0; u < kGnUnroll; ++u)
                if (r + u * l.ty < r1) {
                    w[u] = gn_read<T, V>(x + base + (r + u * l.ty) * s.c + l.col);
                    d[u] = gn_read<T, V>(dy + base + (r + u * l.ty) * s.c + l.col);
                }
#pragma unroll
            for (int u = 0; u < kGnUnroll; ++u)
                if (r + u * l.ty < r1) {
                    GnPack<T, V> o;
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        float xhat, dz;
                        ch.value(i, gn_float(w[u].v[i]), gn_float(d[u].v[i]), xhat, dz);
                        o.v[i] = gn_narrow<T>(ch.rstd[i] * (ch.gamma[i] * dz - s1[i] - xhat * s2[i]));
                    }
                    *reinterpret_cast<GnPack<T, V>*>(dx + base + (r + u * l.ty) * s.c + l.col) = o;
                }
        }
    }
}

// ------------------------------------------------------------------------------------------------ host
static int gn_vector(int c, int dtype) {           // channels of a lane: 16 bytes where they divide c, else 4 bytes or one
    if (dtype == GEOMAE_DTYPE_F32) return c % 4 == 0 ? 4 : 1;
    return c % 8 == 0 ? 8 : (c % 2 == 0 ? 2 : 1);
}
static GnShape gn_shape(int32_t n, int64_t rows, int32_t c, int32_t groups, int dtype) {
    GnShape s;
    s.n = n; s.rows = rows; s.c = c; s.groups = groups; s.cg = c / groups;
    const int cv = c / gn_vector(c, dtype), ty = cv < kGnThreads ? kGnThreads / cv : 1;
    const int64_t least = (int64_t)ty * kGnUnroll, wanted = kGnBlocks / n > 1 ? kGnBlocks / n : 1;
    s.chunk_rows = (rows + wanted - 1) / wanted;
    s.chunk_rows = s.chunk_rows < least ? least : (s.chunk_rows + least - 1) / least * least;
    s.chunks = (int32_t)((rows + s.chunk_rows - 1) / s.chunk_rows);
    return s;
}
struct GnWorkspace { double2* partial; float2* grad_partial; double2 *channel, *folded; float2* means; int64_t forward_bytes, backward_bytes; };
static GnWorkspace gn_workspace(void* base, const GnShape& s) {
    char* p = static_cast<char*>(base);
    GnWorkspace w;
    w.partial = reinterpret_cast<double2*>(p);
    w.forward_bytes = (int64_t)s.n * s.chunks * s.groups * (int64_t)sizeof(double2);
    w.channel = reinterpret_cast<double2*>(p);
    const int64_t a = (int64_t)s.n * s.c * (int64_t)sizeof(double2);
    w.grad_partial = reinterpret_cast<float2*>(p + a);
    const int64_t b = a + ((int64_t)s.n * s.chunks * s.c * (int64_t)sizeof(float2) + 15) / 16 * 16;
    w.means = reinterpret_cast<float2*>(p + b);
    const int64_t d = b + ((int64_t)s.n * s.groups * (int64_t)sizeof(float2) + 15) / 16 * 16;
    w.folded = reinterpret_cast<double2*>(p + d);                      // two halves, used in turn
    w.backward_bytes = d + (s.n > kGnFold ? 2 * (int64_t)((s.n + kGnFold - 1) / kGnFold) * s.c * (int64_t)sizeof(double2) : 0);
    return w;
}
static int gn_check(const char* what, int32_t n, int64_t rows, int32_t c, int32_t groups, int dtype, int wdtype, int act) {
    GEOMAE_REQUIRE(n >= 0 && rows >= 0 && c > 0 && groups > 0, "%s: bad shape [%d, %lld, %d] in %d groups", what, (int)n,
                   (long long)rows, (int)c, (int)groups);
    GEOMAE_REQUIRE(c % groups == 0, "%s: %d channels do not divide into %d groups", what, (int)c, (int)groups);
    GEOMAE_REQUIRE(groups <= kGnMaxGroups, "%s: at most %d groups, got %d", what, kGnMaxGroups, (int)groups);
    GEOMAE_REQUIRE((int64_t)n * groups <= INT32_MAX && c <= INT32_MAX / 16, "%s: %d samples of %d groups are too many", what, (int)n, (int)groups);
    GEOMAE_REQUIRE(dtype >= 0 && dtype <= 2 && wdtype >= 0 && wdtype <= 2, "%s: unknown dtype", what);
    GEOMAE_REQUIRE(act >= 0 && act <= 3, "%s: unknown activation %d", what, act);
    return GEOMAE_OK;
}

template <typename T, int V, int ACT>
static void gn_launch_forward(const void* x, const GnShape& s, const double2* stats, const void* gamma, const void* beta, int wdtype, void* y, hipStream_t stream) {
    hipLaunchKernelGGL((gn_forward_kernel<T, V, ACT>), dim3(s.chunks * s.n), dim3(kGnThreads), 0, stream, static_cast<const T*>(x), s, stats, gamma, beta,
                       wdtype, static_cast<T*>(y));
}
struct GnBackward { const void *x, *dy, *gamma, *beta; const double2* stats; void *dx, *dgamma, *dbeta; int wdtype; };
template <typename T, int V, int ACT>
static void gn_launch_backward(const GnBackward& b, const GnShape& s, const GnWorkspace& w, hipStream_t stream) {
    hipLaunchKernelGGL((gn_grad_sums_kernel<T, V, ACT>), dim3(s.chunks * s.n), dim3(kGnThreads), 0, stream, static_cast<const T*>(b.x),
                       static_cast<const T*>(b.dy), s, b.stats, b.gamma, b.beta, b.wdtype, w.grad_partial);
    hipLaunchKernelGGL(gn_grad_stats_kernel, dim3(s.groups * s.n), dim3(kGnThreads), 0, stream, w.grad_partial, s, b.gamma, b.wdtype, w.channel, w.means);
    const bool many = s.n > kGnFold;
    hipLaunchKernelGGL((gn_backward_kernel<T, V, ACT>), dim3(s.chunks * s.n), dim3(kGnThreads), 0, stream, static_cast<const T*>(b.x),
                       static_cast<const T*>(b.dy), s, b.stats, b.gamma, b.beta, b.wdtype, w.channel, w.means, static_cast<T*>(b.dx),
                       many ? nullptr : b.dgamma, many ? nullptr : b.dbeta);
    if (!many || !(b.dgamma || b.dbeta)) return;
    const double2* from = w.channel;
    double2* halves[2] = {w.folded, w.folded + (int64_t)((s.n + kGnFold - 1) / kGnFold) * s.c};
    int rows = s.n;
    for (int k = 0; rows > kGnFold; ++k) {
        const int next = (rows + kGnFold - 1) / kGnFold;
        hipLaunchKernelGGL(gn_fold_kernel, dim3(cdiv((int64_t)next * s.c, kGnThreads)), dim3(kGnThreads), 0, stream, from, rows, s.c, halves[k & 1]);
        from = halves[k & 1];
        rows = next;
    }
    hipLaunchKernelGGL(gn_weight_grad_kernel, dim3(cdiv(s.c, kGnThreads)), dim3(kGnThreads), 0, stream, from, rows, s.c, b.wdtype, b.dgamma, b.dbeta);
}
// f(type, vector, activation) for the run-time choice of the three
template <typename F> static void gn_by_act(int act, F f) {
    if (act == kGnRelu) f(std::integral_constant<int, kGnRelu>());
    else if (act == kGnSilu) f(std::integral_constant<int, kGnSilu>());
    else if (act == kGnGelu) f(std::integral_constant<int, kGnGelu>());
    else f(std::integral_constant<int, kGnNone>());
}
template <typename T> struct GnType { typedef T type; };
template <typename F> static void gn_by_type(int dtype, int v, F f) {
    if (dtype == GEOMAE_DTYPE_F32) {
        if (v == 4) f(GnType<float>(), std::integral_constant<int, 4>());
        else f(GnType<float>(), std::integral_constant<int, 1>());
    } else if (dtype == GEOMAE_DTYPE_BF16) {
        if (v == 8) f(GnType<uint16_t>(), std::integral_constant<int, 8>());
        else if (v == 2) f(GnType<uint16_t>(), std::integral_constant<int, 2>());
        else f(GnType<uint16_t>(), std::integral_constant<int, 1>());
    } else {
        if (v == 8) f(GnType<_Float16>(), std::integral_constant<int, 8>());
        else if (v == 2) f(GnType<_Float16>(), std::integral_constant<int, 2>());
        else f(GnType<_Float16>(), std::integral_constant<int, 1>());
    }
}

}  // namespace geomae

using namespace geomae;

extern "C" int64_t geomae_group_norm_workspace_bytes(int32_t n, int64_t rows, int32_t c, int32_t groups, int32_t dtype, int32_t backward) {
    if (gn_check("group_norm_workspace_bytes", n, rows, c, groups, dtype, 0, 0)) return -1;
    if (n == 0 || rows == 0) return 0;
    const GnWorkspace w = gn_workspace(nullptr, gn_shape(n, rows, c, groups, dtype));
    return backward ? w.backward_bytes : w.forward_bytes;
}

extern "C" int geomae_group_norm_forward(const void* x, int32_t dtype, int32_t n, int64_t rows, int32_t c, int32_t groups, const void* gamma,
                                         const void* beta, int32_t weight_dtype, double eps, int32_t activation, void* y, double* stats,
                                         void* workspace, int64_t workspace_bytes, hipStream_t stream) {
    if (int rc = gn_check("group_norm_forward", n, rows, c, groups, dtype, weight_dtype, activation)) return rc;
    GEOMAE_REQUIRE(eps >= 0.0, "group_norm_forward: eps must not be negative");
    if (n == 0 || rows == 0) return GEOMAE_OK;
    GEOMAE_REQUIRE(x && y && stats, "group_norm_forward: null argument");
    const GnShape s = gn_shape(n, rows, c, groups, dtype);
    const GnWorkspace w = gn_workspace(workspace, s);
    if (!workspace || workspace_bytes < w.forward_bytes) {
        set_error("group_norm_forward: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)w.forward_bytes);
        return GEOMAE_ERR_WORKSPACE;
    }
    double2* st = reinterpret_cast<double2*>(stats);
    gn_by_type(dtype, gn_vector(c, dtype), [&](auto t, auto v) {
        typedef typename decltype(t)::type T;
        constexpr int V = decltype(v)::value;
        hipLaunchKernelGGL((gn_sums_kernel<T, V>), dim3(s.chunks * n), dim3(kGnThreads), 0, stream, static_cast<const T*>(x), s, w.partial);
        hipLaunchKernelGGL(gn_stats_kernel, dim3(cdiv((int64_t)n * groups, kGnThreads / kWave)), dim3(kGnThreads), 0, stream, w.partial, s, eps, st);
        gn_by_act(activation, [&](auto a) { gn_launch_forward<T, V, decltype(a)::value>(x, s, st, gamma, beta, weight_dtype, y, stream); });
    });
    return check_launch("gn_forward_kernel");
}

extern "C" int geomae_group_norm_backward(const void* x, const void* dy, int32_t dtype, int32_t n, int64_t rows, int32_t c, int32_t groups,
                                          const void* gamma, const void* beta, int32_t weight_dtype, int32_t activation, const double* stats,
                                          void* dx, void* dgamma, void* dbeta, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
    if (int rc = gn_check("group_norm_backward", n, rows, c, groups, dtype, weight_dtype, activation)) return rc;
    if (n == 0 || rows == 0) return GEOMAE_OK;
    GEOMAE_REQUIRE(x && dy && stats && dx, "group_norm_backward: null argument");
    const GnShape s = gn_shape(n, rows, c, groups, dtype);
    const GnWorkspace w = gn_workspace(workspace, s);
    if (!workspace || workspace_bytes < w.backward_bytes) {
        set_error("group_norm_backward: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)w.backward_bytes);
        return GEOMAE_ERR_WORKSPACE;
    }
    const GnBackward b = {x, dy, gamma, beta, reinterpret_cast<const double2*>(stats), dx, dgamma, dbeta, weight_dtype};
    gn_by_type(dtype, gn_vector(c, dtype), [&](auto t, auto v) {
        typedef typename decltype(t)::type T;
        constexpr int V = decltype(v)::value;
        gn_by_act(activation, [&](auto a) { gn_launch_backward<T, V, decltype(a)::value>(b, s, w, stream); });
    });
    return check_launch("gn_backward_kernel");
}
