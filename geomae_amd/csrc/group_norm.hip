// Group norm with an activation on channels-last data: x [n][rows][c], groups of cg = c / groups neighbouring channels.
//
//   xhat = (x - mean) rstd,  z = gamma xhat + beta,  y = act(z)        mean, var over the rows and channels of (sample, group)
//   dz = dy act'(z);  dbeta = sum dz, dgamma = sum dz xhat over samples and rows
//   dx = rstd (gamma dz - s1 - xhat s2),   s1, s2 = means over the group of gamma dz and of gamma dz xhat
//
// The sums of the statistics are in fp64, of the elements less the group's first one: sums of the squares themselves lose a small
// variance under a large mean, in 64 bits too (a mean of 2^20 spreads leaves 2^-13 of it).  The first element is within sqrt(m var) of the
// mean, m elements, so that the difference of the two sums is good to m 2^-53 of the variance at worst, and to some 2^-53 as a rule.
// Mean and rstd are kept as fp64: their rounding moves every element of a group together, and ReLU's border in the backward pass (is z
// over zero?) is decided by a threshold on x that is worked out in fp64 and rounded so that no fp32 x lies between it and the
// true one.  The rest is fp32; the gradient sums are fp32 within a workgroup's rows, 256 of them one after the other at most, and fp64
// across workgroups, always in the same order.
//
// A thread keeps to one vector of V neighbouring channels of one group (V = 4, 2 or 1, whichever divides cg first), so that its
// statistics, gamma and beta stay in registers.  (8 channels of a 16-bit type, one access of 16 bytes, set up twice as much per
// thread for half as many rows: a quarter longer at 2 x 256 x 128 x 128 bf16 forward, which takes 23 us.)  Two forms:
//  resident  all rows of one or more groups fit a workgroup's registers (128 bytes a thread, 1024 threads: 4096 rows of 32
//            bytes): x and dy are read once and one launch does a pass (the backward pass one more for the parameters'
//            gradients if there is more than one sample).  Bound by launch, load latency and the workgroup's reductions (1 x 256 x
//            25 x 25 fp32 forward 5.5 us; 4 x 256 x 50 x 50 12 us, backward 18: a line fetched for each row's 32 bytes).
//  streamed  three launches a pass: sums over a chunk of rows, one value per (sample, group) from the chunks' sums, and the pass
//            that writes.  Bound by HBM, or the 256 MB cache that the second read of x and dy comes from where they fit in it.
//            Tensors over 64 MB: the writing pass loads and stores past the caches (4 x 128 x 200 x 200 fp32, both passes 132 ->
//            117 us; 61 M bf16 elements forward 84 -> 67 us); smaller ones stay there for whoever comes next.  The launches of 4 x 128 x
//            200 x 200 fp32 (82 MB a tensor): sums 17 us (4.7 TB/s), writing 24 (6.8), gradient sums 31 (5.3), gradients 36 (6.8), the two
//            launches between them 4.6 each.
#include "common.h"
#include "../../include/geomae_hip.h"
#include <math.h>
#include <type_traits>

namespace geomae {

constexpr int kGnThreads = 256;                    // of a streamed workgroup
constexpr int kGnMaxGroups = 1024, kGnMaxChannels = 1 << 22;
constexpr int kGnBlocks = 1024;                    // workgroups of a streamed pass: four per CU
constexpr int kGnSumRows = 256;                    // rows that a thread adds up in fp32 (a multiple of the rows in flight)
constexpr int kGnFold = 64;                        // samples whose sums one thread adds up for the parameters' gradients
constexpr int kGnResidentThreads = 1024;

enum { kGnNone = 0, kGnRelu = 1, kGnSilu = 2, kGnGelu = 3 };

struct GnShape {
    int64_t rows;                                  // of a sample
    int32_t n, c, groups, cg;
    int32_t chunks;                                // of a sample's rows (streamed)
    int64_t chunk_rows;
    int32_t past_cache;                            // streamed: the tensors do not fit the 256 MB cache beside each other
    double inv_m;                                  // 1 / (elements of a group of a sample)
    int32_t v;                                     // channels of a thread
    int32_t cs, threads;                           // channels of a resident workgroup, 0: streamed; its threads ...
    int32_t tx, ty, slabs, slab_groups;            // ... as tx columns x ty rows; workgroups of a sample, groups of a workgroup
    uint32_t tx_inverse;                           // t / tx = (t * this) >> 20 for t < 1024
};

template <typename T> __device__ __forceinline__ float gn_float(T x) { return (float)x; }
template <> __device__ __forceinline__ float gn_float<uint16_t>(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }   // bf16
// (element-aligned: a tensor may start anywhere, and global memory takes wide accesses at any element's address)
template <typename T, int V> struct __attribute__((packed, aligned(sizeof(T)))) GnPack { T v[V]; };
// LAST: the last use of the data for now (GnShape::past_cache): a load and a store that leave the caches to others
template <typename T, int V> struct GnWords { typedef uint32_t type __attribute__((ext_vector_type(V * sizeof(T) / 4), aligned(sizeof(T)))); };
template <typename T, int V, bool LAST = false> __device__ __forceinline__ GnPack<T, V> gn_read(const T* p) {
    if constexpr (LAST && V * sizeof(T) >= 4) {
        typedef typename GnWords<T, V>::type W;
        return __builtin_bit_cast(GnPack<T, V>, __builtin_nontemporal_load(reinterpret_cast<const W*>(p)));
    } else return *reinterpret_cast<const GnPack<T, V>*>(p);
}
// One address for the wave and a lane's 32-bit offset.  (64-bit products per row and lane: 4 x 352 x 90 x 90 in groups of 11, one channel a
// thread, fp32 forward 48 us against 34, bf16 46 against 29; four channels a thread 1 to 3 %.)
template <typename T> __device__ __forceinline__ const T* gn_at(const T* p, uint32_t bytes) { return reinterpret_cast<const T*>(reinterpret_cast<const char*>(p) + bytes); }
template <typename T> __device__ __forceinline__ T* gn_at(T* p, uint32_t bytes) { return reinterpret_cast<T*>(reinterpret_cast<char*>(p) + bytes); }
typedef __bf16 GnBf2 __attribute__((ext_vector_type(2)));
typedef float GnF2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t gn_bf16_pair(float a, float b) {
    const GnBf2 r = __builtin_convertvector((GnF2){a, b}, GnBf2);
    return __builtin_bit_cast(uint32_t, r);
}
template <typename T, int V, bool LAST = false> __device__ __forceinline__ void gn_write(T* p, const float (&x)[V]) {
    GnPack<T, V> w;
    if constexpr (std::is_same<T, uint16_t>::value) {
#pragma unroll
        for (int i = 0; i + 1 < V; i += 2) {
            const uint32_t two = gn_bf16_pair(x[i], x[i + 1]);
            w.v[i] = (uint16_t)two;
            w.v[i + 1] = (uint16_t)(two >> 16);
        }
        if constexpr (V == 1) w.v[0] = (uint16_t)gn_bf16_pair(x[0], 0.f);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) w.v[i] = (T)x[i];
    }
    if constexpr (LAST && V * sizeof(T) >= 4) {
        typedef typename GnWords<T, V>::type W;
        __builtin_nontemporal_store(__builtin_bit_cast(W, w), reinterpret_cast<W*>(p));
    } else *reinterpret_cast<GnPack<T, V>*>(p) = w;
}
// The vector as it is, to the compiler a new one (another one per ACT): its conversions stay where they are used.  Those of all
// activations' loops were moved ahead of the choice between them, 128 values in fp16, which spilled.
template <int ACT, typename T, int V> __device__ __forceinline__ GnPack<T, V> gn_fresh(const GnPack<T, V>& p) {
    if constexpr (V * sizeof(T) >= 4) {
        struct Words { uint32_t w[V * sizeof(T) / 4]; } words = __builtin_bit_cast(Words, p);
#pragma unroll
        for (uint32_t& w : words.w) asm volatile("; %1" : "+v"(w) : "n"(ACT));
        return __builtin_bit_cast(GnPack<T, V>, words);
    } else return p;
}
// vectors that a thread has in flight (streamed) or holds (resident).  8 of four 16-bit channels in flight instead of 4 cost 10 %
// (4 x 128 x 200 x 200 bf16, both passes 91 us against 82), 2 of four fp32 channels nothing and 128 bytes 20 %.
constexpr int gn_rows_in_flight(int v) { return 16 / v; }
template <typename T, int V> constexpr int gn_held() { return V * sizeof(T) == 16 ? 8 : 16; }
static int gn_vectors_held(int v, int item) { return v * item == 16 ? 8 : 16; }

// The hardware's base-2 exponential and reciprocal (1 ulp each): the library's expf and the IEEE division made silu and gelu, not
// memory, the bound (61 M bf16 elements, silu: 85 us).
// gelu: P(normal > a) = exp(-a^2 / 2) R(a) for a = |z|, R(a) = 1/2 - u Q(t) with t = 1 / (1 + 0.3 a), u = a t, Q of degree 7 fitted to
// R's relative error over a <= 14 (6.6e-8 at most; the coefficients are that fit, in fp32).  R is exact at 0 and errors of Q and t count with u there, so that in
// fp32, evaluated with ideal instructions on normal numbers of spread 1, y is off by 2.0e-8 rms and the slope by 2.7e-8, no more
// than 0.5 (1 + erf) in fp32 (2.4e-8 and 2.7e-8); the negative tail keeps its digits (5.5e-6 relative at -10, where 1 + erf is 0).
__device__ __forceinline__ float gn_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504088896341f)); }
__device__ __forceinline__ float gn_normal_ratio(float a, float& density) {     // R; density: exp(-a^2 / 2)
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3f, a, 1.0f));
    density = __builtin_amdgcn_exp2f(a * (a * -0.72134752044448170f));
    float q = 0.0114266658f;
    q = fmaf(q, t, -0.0389440507f);
    q = fmaf(q, t, 0.028955761f);
    q = fmaf(q, t, 0.006710121f);
    q = fmaf(q, t, 0.0490427256f);
    q = fmaf(q, t, 0.0776065477f);
    q = fmaf(q, t, 0.114147519f);
    q = fmaf(q, t, 0.149998063f);
    return fmaf(-a * t, q, 0.5f);
}
template <int ACT> __device__ __forceinline__ float gn_act(float z) {
    if constexpr (ACT == kGnRelu) return z < 0.f ? 0.f : z;            // NaN stays
    if constexpr (ACT == kGnSilu) return z * gn_sigmoid(z);
    if constexpr (ACT == kGnGelu) {                                    // z - z tail above zero, z tail below
        const float a = fabsf(z);
        float density;
        const float ratio = gn_normal_ratio(a, density);
        return fmaf(-a * density, ratio, fmaxf(z, 0.f));
    }
    return z;
}
template <int ACT> __device__ __forceinline__ float gn_slope(float z) {     // (ReLU's: gn_threshold)
    if constexpr (ACT == kGnSilu) {
        const float s = gn_sigmoid(z);
        return s * fmaf(z, 1.0f - s, 1.0f);
    }
    if constexpr (ACT == kGnGelu) {                                    // below zero density (R - a / sqrt(2 pi)), above it 1 less that
        const float a = fabsf(z);
        float density;
        const float ratio = gn_normal_ratio(a, density);
        return fmaf(copysignf(density, z), fmaf(a, 0.39894228040143268f, -ratio), z < 0.f ? 0.f : 1.f);
    }
    return 1.0f;
}
// f(activation), the run-time choice made outside the loops
template <typename F> __host__ __device__ __forceinline__ void gn_by_act(int act, F f) {
    if (act == kGnRelu) f(std::integral_constant<int, kGnRelu>());
    else if (act == kGnSilu) f(std::integral_constant<int, kGnSilu>());
    else if (act == kGnGelu) f(std::integral_constant<int, kGnGelu>());
    else f(std::integral_constant<int, kGnNone>());
}
template <typename F> __device__ __forceinline__ void gn_by_act(int act, int last, F f) {
    gn_by_act(act, [&](auto a) {
        if (last) f(a, std::true_type());
        else f(a, std::false_type());
    });
}
// z > 0 as a comparison of x, its sign turned where gamma is negative, with a threshold
__device__ __forceinline__ float gn_threshold(double mean, double scale, double beta) {
    if (scale == 0.0) return beta > 0.0 ? -INFINITY : INFINITY;
    const double t = scale < 0.0 ? beta / scale - mean : mean - beta / scale;
    float f = (float)t;
    if ((double)f > t) f = nextafterf(f, -INFINITY);
    return f;
}
__device__ __forceinline__ float gn_turned(float x, float gamma) { return __uint_as_float(__float_as_uint(x) ^ (__float_as_uint(gamma) & 0x80000000u)); }

__device__ __forceinline__ float gn_weight(const void* w, int dtype, int c, float none) {
    if (!w) return none;
    if (dtype == GEOMAE_DTYPE_F32) return static_cast<const float*>(w)[c];
    if (dtype == GEOMAE_DTYPE_BF16) return gn_float(static_cast<const uint16_t*>(w)[c]);
    return gn_float(static_cast<const _Float16*>(w)[c]);
}
__device__ __forceinline__ void gn_store_weight(void* w, int dtype, int c, float v) {
    if (!w) return;
    if (dtype == GEOMAE_DTYPE_F32) static_cast<float*>(w)[c] = v;
    else if (dtype == GEOMAE_DTYPE_BF16) static_cast<uint16_t*>(w)[c] = (uint16_t)gn_bf16_pair(v, 0.f);
    else static_cast<_Float16*>(w)[c] = (_Float16)v;
}

struct GnWeights { const void *gamma, *beta; int dtype; };

// what a lane keeps of its V channels, all of one group, for y
template <int V> struct GnScale {
    float mean, scale[V], rest[V], beta[V];
    __device__ __forceinline__ void weights(const GnWeights& w, int col) {          // (scale holds gamma until statistics() is called)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            scale[i] = gn_weight(w.gamma, w.dtype, col + i, 1.f);
            beta[i] = gn_weight(w.beta, w.dtype, col + i, 0.f);
        }
    }
    __device__ __forceinline__ void statistics(double2 stat) {
        mean = (float)stat.x;
        const double lost = stat.x - (double)mean;                     // what mean's rounding lost comes back behind the product
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const double sc = stat.y * (double)scale[i];
            scale[i] = (float)sc;
            rest[i] = (float)(-lost * sc);
        }
    }
    template <int ACT> __device__ __forceinline__ float value(int i, float x) const { return gn_act<ACT>(fmaf(x - mean, scale[i], rest[i]) + beta[i]); }
};
// ... and for xhat and dz
template <int V> struct GnGrad {
    float mean, rstd, rest, gamma[V], other[V];                       // other: beta; ReLU: gn_threshold
    __device__ __forceinline__ void load(double2 stat, const GnWeights& w, int act, int col) {
        mean = (float)stat.x;
        rstd = (float)stat.y;
        rest = (float)(-(stat.x - (double)mean) * stat.y);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            gamma[i] = gn_weight(w.gamma, w.dtype, col + i, 1.f);
            other[i] = gn_weight(w.beta, w.dtype, col + i, 0.f);
            if (act == kGnRelu) other[i] = gn_threshold(stat.x, stat.y * (double)gamma[i], (double)other[i]);
        }
    }
    template <int ACT> __device__ __forceinline__ void value(int i, float x, float dy, float& xhat, float& dz) const {
        xhat = fmaf(x - mean, rstd, rest);
        if constexpr (ACT == kGnRelu) dz = gn_turned(x, gamma[i]) > other[i] ? dy : 0.f;
        else dz = dy * gn_slope<ACT>(fmaf(xhat, gamma[i], other[i]));
    }
    // c1, c2: rstd times the group's two means
    __device__ __forceinline__ float dx(int i, float xhat, float dz, float c1, float c2) const {
        return fmaf(rstd * gamma[i], dz, -fmaf(xhat, c2, c1));
    }
};

// ------------------------------------------------------------------------------------------------ sums over a workgroup
// v summed over the lanes of a wave that are equal modulo tx (a power of two up to 32), in every lane: the halves and rows by
// the swaps, within a row of 16 by rotations (by 8, 4, ...: what is equal modulo 8, 4, ... already makes them exchanges)
template <int CTRL> __device__ __forceinline__ double gn_dpp(double v) {
    return __hiloint2double(dpp_mov<CTRL>(__double2hiint(v)), dpp_mov<CTRL>(__double2loint(v)));
}
template <int CTRL> __device__ __forceinline__ float gn_dpp(float v) { return dpp_mov<CTRL>(v); }
__device__ __forceinline__ float gn_swap32(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}
__device__ __forceinline__ float gn_swap16(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}
__device__ __forceinline__ double gn_swap32(double v) {
    const auto h = __builtin_amdgcn_permlane32_swap((uint32_t)__double2hiint(v), (uint32_t)__double2hiint(v), false, false);
    const auto l = __builtin_amdgcn_permlane32_swap((uint32_t)__double2loint(v), (uint32_t)__double2loint(v), false, false);
    return __hiloint2double((int)h[0], (int)l[0]) + __hiloint2double((int)h[1], (int)l[1]);
}
__device__ __forceinline__ double gn_swap16(double v) {
    const auto h = __builtin_amdgcn_permlane16_swap((uint32_t)__double2hiint(v), (uint32_t)__double2hiint(v), false, false);
    const auto l = __builtin_amdgcn_permlane16_swap((uint32_t)__double2loint(v), (uint32_t)__double2loint(v), false, false);
    return __hiloint2double((int)h[0], (int)l[0]) + __hiloint2double((int)h[1], (int)l[1]);
}
template <typename S> __device__ __forceinline__ S gn_wave_columns(S v, int tx) {
    v = gn_swap32(v);
    if (tx <= 16) v = gn_swap16(v);
    if (tx <= 8) v += gn_dpp<0x128>(v);            // row_ror:8
    if (tx <= 4) v += gn_dpp<0x124>(v);
    if (tx <= 2) v += gn_dpp<0x122>(v);
    if (tx <= 1) v += gn_dpp<0x121>(v);
    return v;
}
__host__ __device__ __forceinline__ bool gn_whole_rows(int tx) { return tx <= kWave / 2 && (tx & (tx - 1)) == 0; }   // a wave holds whole rows
// a[W] of every thread (row, col) of tx columns x ty rows, summed over the rows: res[w * tx + col].  Fixed order.
template <typename S, int W>
__device__ __forceinline__ void gn_sum_rows(S (&a)[W], int tx, int ty, S* res, S* lds) {
    const int threads = blockDim.x, t = threadIdx.x;
    if (gn_whole_rows(tx)) {                                           // a wave's rows first, then the waves
        const int waves = threads / kWave;
#pragma unroll
        for (int w = 0; w < W; ++w) a[w] = gn_wave_columns(a[w], tx);
        if (lane_id() < tx) {
#pragma unroll
            for (int w = 0; w < W; ++w) lds[(w * waves + t / kWave) * tx + lane_id()] = a[w];
        }
        __syncthreads();
        for (int k = t; k < W * tx; k += threads) {
            const int w = k / tx, col = k - w * tx;
            S sum = lds[(w * waves) * tx + col];
#pragma unroll 4
            for (int v = 1; v < waves; ++v) sum += lds[(w * waves + v) * tx + col];
            res[k] = sum;
        }
    } else {
#pragma unroll
        for (int w = 0; w < W; ++w) lds[w * threads + t] = a[w];
        __syncthreads();
        // a row of 16 lanes a column, or a thread if it has few rows
        const int lanes = ty > 16 ? 16 : 1, lane = t & (lanes - 1);
        for (int k = t / lanes; k < W * tx; k += threads / lanes) {
            const int w = k / tx, col = k - w * tx;
            S sum = 0;
#pragma unroll 4
            for (int r = lane; r < ty; r += lanes) sum += lds[w * threads + r * tx + col];
            if (lanes > 1) {
                sum += gn_dpp<0x128>(sum);         // row_ror:8
                sum += gn_dpp<0x124>(sum);
                sum += gn_dpp<0x122>(sum);
                sum += gn_dpp<0x121>(sum);
            }
            if (lane == 0) res[k] = sum;
        }
    }
    __syncthreads();
}
// f(group, b, e, lane, lanes): the entries [b, e) of each of `groups` groups (per of them a group) to be summed by `lanes`
// neighbouring threads; few entries: a thread a group, else a wave
template <typename F> __device__ __forceinline__ void gn_each_group(int groups, int per, F f) {
    if (per <= 16) {
        for (int g = threadIdx.x; g < groups; g += blockDim.x) f(g, 0, 1);
    } else {
        for (int g = threadIdx.x / kWave; g < groups; g += blockDim.x / kWave) f(g, lane_id(), kWave);
    }
}
__device__ __forceinline__ double gn_lanes_sum(double v, int lanes) { return lanes == 1 ? v : wave_sum(v); }

// first: the group's first element, which was taken off the summed ones
__device__ __forceinline__ double2 gn_statistics(double first, double sum, double sq, double inv_m, double eps) {
    const double mean = sum * inv_m;
    double var = sq * inv_m - mean * mean;
    var = var < 0.0 ? 0.0 : var;                                       // (NaN stays)
    return make_double2(first + mean, 1.0 / sqrt(var + eps));
}

// ------------------------------------------------------------------------------------------------ resident
// Workgroup -> (sample, first channel): neighbours in memory go to one XCD (workgroup b runs on XCD b mod 8), whose L2 then
// serves the lines that the channel ranges share.
__device__ __forceinline__ int gn_spread(int b, int total) {
    const int each = total / 8, more = total - each * 8, x = b & 7;
    return x * each + (x < more ? x : more) + (b >> 3);
}
struct GnSlab {
    int tx, ty, row, col;                          // col: this thread's first channel within the slab
    int n, c0, groups;
    bool live;
    template <int V> __device__ __forceinline__ void set(const GnShape& s) {
        const int b = gn_spread(blockIdx.x, gridDim.x);
        n = b / s.slabs;
        c0 = (b - n * s.slabs) * s.cs;
        groups = s.slab_groups;
        tx = s.tx;
        ty = s.ty;
        row = (int)((threadIdx.x * s.tx_inverse) >> 20);
        col = (threadIdx.x - row * tx) * V;
        live = row < ty;
    }
};
extern __shared__ __align__(16) char gn_lds[];

template <typename T, int V>
__global__ __launch_bounds__(kGnResidentThreads) void gn_resident_forward_kernel(const T* __restrict__ x, GnShape s, GnWeights w, double eps, int act,
                                                                                T* __restrict__ y, double2* __restrict__ stats) {
    constexpr int R = gn_held<T, V>();
    GnSlab l;
    l.set<V>(s);
    double2* group = reinterpret_cast<double2*>(gn_lds);
    double* res = reinterpret_cast<double*>(group + l.groups);
    double* lds = res + 2 * l.tx;
    const int64_t base = (int64_t)l.n * s.rows * s.c + l.c0 + l.col;
    const int rows = (int)s.rows;
    GnPack<T, V> v[R];
#pragma unroll
    for (int u = 0; u < R; ++u) {
        const int r = l.row + u * l.ty;
        if (l.live && r < rows) v[u] = gn_read<T, V>(x + base + (int64_t)r * s.c);
    }
    const int mine = (l.live ? l.col : 0) / s.cg;                      // this thread's group of the workgroup's
    const T* const row0 = x + (int64_t)l.n * s.rows * s.c + l.c0;      // the sample's first row
    const double first = (double)gn_float(row0[mine * s.cg]);
    GnScale<V> ch;
    ch.weights(w, l.c0 + (l.live ? l.col : 0));
    double a[2] = {0.0, 0.0};
#pragma unroll
    for (int u = 0; u < R; ++u)
        if (l.live && l.row + u * l.ty < rows) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const double d = (double)gn_float(v[u].v[i]) - first;
                a[0] += d;
                a[1] = fma(d, d, a[1]);
            }
        }
    gn_sum_rows<double, 2>(a, l.tx, l.ty, res, lds);
    const int per = s.cg / V;
    gn_each_group(l.groups, per, [&](int g, int lane, int lanes) {
        double sum = 0.0, sq = 0.0;
        for (int k = lane; k < per; k += lanes) {
            sum += res[g * per + k];
            sq += res[l.tx + g * per + k];
        }
        sum = gn_lanes_sum(sum, lanes);
        sq = gn_lanes_sum(sq, lanes);
        if (lane == 0) {
            group[g] = gn_statistics((double)gn_float(row0[g * s.cg]), sum, sq, s.inv_m, eps);
            stats[(int64_t)l.n * s.groups + l.c0 / s.cg + g] = group[g];
        }
    });
    __syncthreads();
    if (!l.live) return;
    ch.statistics(group[mine]);
    gn_by_act(act, [&](auto A) {
#pragma unroll
        for (int u = 0; u < R; ++u) {
            const int r = l.row + u * l.ty;
            if (r < rows) {
                float o[V];
                const GnPack<T, V> xv = gn_fresh<decltype(A)::value>(v[u]);
#pragma unroll
                for (int i = 0; i < V; ++i) o[i] = ch.template value<decltype(A)::value>(i, gn_float(xv.v[i]));
                gn_write<T, V>(y + base + (int64_t)r * s.c, o);
            }
        }
    });
}

// channel [n][c] receives the samples' (sum dz, sum dz xhat); one sample: dgamma, dbeta themselves
template <typename T, int V>
__global__ __launch_bounds__(kGnResidentThreads) void gn_resident_backward_kernel(const T* __restrict__ x, const T* __restrict__ dy, GnShape s,
                                                                                 const double2* __restrict__ stats, GnWeights w, int act,
                                                                                 T* __restrict__ dx, double2* __restrict__ channel, void* dgamma, void* dbeta) {
    constexpr int R = gn_held<T, V>();
    GnSlab l;
    l.set<V>(s);
    float2* group = reinterpret_cast<float2*>(gn_lds);
    float* res = reinterpret_cast<float*>(group + l.groups);           // [2 V][tx]
    float* gamma = res + 2 * V * l.tx;                                 // [V][tx], whole rows
    float* lds = gamma + (gn_whole_rows(l.tx) ? V * l.tx : 0);
    const int64_t base = (int64_t)l.n * s.rows * s.c + l.c0 + l.col;
    const int rows = (int)s.rows;
    GnPack<T, V> v[R], d[R];
#pragma unroll
    for (int u = 0; u < R; ++u) {
        const int r = l.row + u * l.ty;
        if (l.live && r < rows) {
            v[u] = gn_read<T, V>(x + base + (int64_t)r * s.c);
            d[u] = gn_read<T, V>(dy + base + (int64_t)r * s.c);
        }
    }
    GnGrad<V> ch;
    const int mine = l.live ? l.col : 0;
    ch.load(stats[(int64_t)l.n * s.groups + (l.c0 + mine) / s.cg], w, act, l.c0 + mine);
    float ab[2 * V];
#pragma unroll
    for (int i = 0; i < 2 * V; ++i) ab[i] = 0.f;
    gn_by_act(act, [&](auto A) {
#pragma unroll
        for (int u = 0; u < R; ++u)
            if (l.live && l.row + u * l.ty < rows) {
                const GnPack<T, V> xv = gn_fresh<decltype(A)::value>(v[u]), dv = gn_fresh<decltype(A)::value>(d[u]);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    float xhat, dz;
                    ch.template value<decltype(A)::value>(i, gn_float(xv.v[i]), gn_float(dv.v[i]), xhat, dz);
                    ab[i] += dz;
                    ab[V + i] = fmaf(dz, xhat, ab[V + i]);
                }
            }
    });
    if (gn_whole_rows(l.tx) && l.live && l.row == 0) {
#pragma unroll
        for (int i = 0; i < V; ++i) gamma[i * l.tx + l.col / V] = ch.gamma[i];
    }
    if (l.tx <= kGnResidentThreads / 2) gn_sum_rows<float, 2 * V>(ab, l.tx, l.ty, res, lds);
    else {                                                             // (64 KB of LDS: half of the sums at a time)
        gn_sum_rows<float, V>(*reinterpret_cast<float(*)[V]>(&ab[0]), l.tx, l.ty, res, lds);
        gn_sum_rows<float, V>(*reinterpret_cast<float(*)[V]>(&ab[V]), l.tx, l.ty, res + V * l.tx, lds);
    }
    for (int c = threadIdx.x; c < s.cs; c += blockDim.x) {
        const int k = c / V, i = c - k * V;
        const float sa = res[i * l.tx + k], sb = res[(V + i) * l.tx + k];
        if (channel) channel[(int64_t)l.n * s.c + l.c0 + c] = make_double2((double)sa, (double)sb);
        else {
            gn_store_weight(dbeta, w.dtype, l.c0 + c, sa);
            gn_store_weight(dgamma, w.dtype, l.c0 + c, sb);
        }
    }
    gn_each_group(l.groups, s.cg, [&](int g, int lane, int lanes) {
        double s1 = 0.0, s2 = 0.0;
        for (int c = g * s.cg + lane; c < (g + 1) * s.cg; c += lanes) {
            const int k = c / V, i = c - k * V;
            const double gm = (double)(gn_whole_rows(l.tx) ? gamma[i * l.tx + k] : gn_weight(w.gamma, w.dtype, l.c0 + c, 1.f));
            s1 += gm * (double)res[i * l.tx + k];
            s2 += gm * (double)res[(V + i) * l.tx + k];
        }
        s1 = gn_lanes_sum(s1, lanes);
        s2 = gn_lanes_sum(s2, lanes);
        if (lane == 0) group[g] = make_float2((float)(s1 * s.inv_m), (float)(s2 * s.inv_m));
    });
    __syncthreads();
    if (!l.live) return;
    const float2 mean = group[l.col / s.cg];
    const float c1 = ch.rstd * mean.x, c2 = ch.rstd * mean.y;
    gn_by_act(act, [&](auto A) {
#pragma unroll
        for (int u = 0; u < R; ++u) {
            const int r = l.row + u * l.ty;
            if (r < rows) {
                float o[V];
                const GnPack<T, V> xv = gn_fresh<4 + decltype(A)::value>(v[u]), dv = gn_fresh<4 + decltype(A)::value>(d[u]);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    float xhat, dz;
                    ch.template value<decltype(A)::value>(i, gn_float(xv.v[i]), gn_float(dv.v[i]), xhat, dz);
                    o[i] = ch.dx(i, xhat, dz, c1, c2);
                }
                gn_write<T, V>(dx + base + (int64_t)r * s.c, o);
            }
        }
    });
}

// ------------------------------------------------------------------------------------------------ streamed
// the workgroup's threads as tx columns (vectors of V channels) x ty rows; c > 256 V is walked in tiles of 256 V channels
struct GnLanes {
    int tx, ty, col, row;
    bool live;
    // of this lane's first vector from the workgroup's first row, in bytes; below 2^32: 256 rows of kGnMaxChannels at most
    template <typename T> __device__ __forceinline__ uint32_t offset(int c) const { return ((uint32_t)row * (uint32_t)c + (uint32_t)col) * (uint32_t)sizeof(T); }
};
template <int V> __device__ __forceinline__ GnLanes gn_lanes(int c, int tile) {
    GnLanes l;
    const int cv = (c - tile * kGnThreads * V) / V;
    l.tx = cv < kGnThreads ? cv : kGnThreads;
    l.ty = __builtin_amdgcn_readfirstlane(kGnThreads / l.tx);
    l.row = threadIdx.x / l.tx;
    l.col = (tile * kGnThreads + (int)threadIdx.x - l.row * l.tx) * V;
    l.live = l.row < l.ty;
    return l;
}
// f(vector, offset of its row's first element from x): the lane's rows of [r0, r1), U loads at a time, unguarded but for the last
template <typename T, int V, int U, bool LAST = false, typename F> __device__ __forceinline__ void gn_rows(const T* x, int c, const GnLanes& l, int64_t r0, int64_t r1, F f) {
    const uint32_t lane = l.template offset<T>(c);
    const int64_t step = (int64_t)l.ty * c;
    const int all = U * l.ty;
    int64_t r = r0;
    GnPack<T, V> w[U];
    for (; r + all <= r1; r += all) {
#pragma unroll
        for (int u = 0; u < U; ++u) w[u] = gn_read<T, V, LAST>(gn_at(x + r * c + u * step, lane));
#pragma unroll
        for (int u = 0; u < U; ++u) f(w[u], r * c + u * step);
    }
    const int left = (int)(r1 - r);
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (l.row + u * l.ty < left) w[u] = gn_read<T, V, LAST>(gn_at(x + r * c + u * step, lane));
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (l.row + u * l.ty < left) f(w[u], r * c + u * step);
}

// partial [n][groups][chunks]: (sum, sum of squares) of the elements less their group's first one
template <typename T, int V>
__global__ __launch_bounds__(kGnThreads) void gn_sums_kernel(const T* __restrict__ x, GnShape s, double2* __restrict__ partial) {
    __shared__ double lds[2 * kGnThreads], res[2 * kGnThreads];
    double2* group = reinterpret_cast<double2*>(gn_lds);
    const int n = blockIdx.x / s.chunks, chunk = blockIdx.x - n * s.chunks;
    const int64_t r0 = chunk * s.chunk_rows, r1 = r0 + s.chunk_rows < s.rows ? r0 + s.chunk_rows : s.rows;
    x += (int64_t)n * s.rows * s.c;
    for (int g = threadIdx.x; g < s.groups; g += kGnThreads) group[g] = make_double2(0.0, 0.0);
    const int tiles = (s.c + kGnThreads * V - 1) / (kGnThreads * V);
    for (int tile = 0; tile < tiles; ++tile) {
        const GnLanes l = gn_lanes<V>(s.c, tile);
        double a[2] = {0.0, 0.0};
        if (l.live) {
            const double first = (double)gn_float(x[l.col / s.cg * s.cg]);
            gn_rows<T, V, gn_rows_in_flight(V)>(x, s.c, l, r0, r1, [&](const GnPack<T, V>& w, int64_t) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const double d = (double)gn_float(w.v[i]) - first;
                    a[0] += d;
                    a[1] = fma(d, d, a[1]);
                }
            });
        }
        gn_sum_rows<double, 2>(a, l.tx, l.ty, res, lds);
        // columns -> the groups that begin in or reach into this tile
        const int per = s.cg / V, k0 = tile * kGnThreads, k1 = k0 + l.tx, g0 = k0 / per;
        gn_each_group((k1 - 1) / per - g0 + 1, per, [&](int j, int lane, int lanes) {
            const int g = g0 + j, b = g * per > k0 ? g * per : k0, e = (g + 1) * per < k1 ? (g + 1) * per : k1;
            double sum = 0.0, sq = 0.0;
            for (int k = b + lane; k < e; k += lanes) {
                sum += res[k - k0];
                sq += res[l.tx + k - k0];
            }
            sum = gn_lanes_sum(sum, lanes);
            sq = gn_lanes_sum(sq, lanes);
            if (lane == 0) group[g] = make_double2(group[g].x + sum, group[g].y + sq);
        });
        __syncthreads();
    }
    for (int g = threadIdx.x; g < s.groups; g += kGnThreads) partial[((int64_t)n * s.groups + g) * s.chunks + chunk] = group[g];
}

// a wave per (sample, group): mean and 1 / sqrt(var + eps)
template <typename T>
__global__ __launch_bounds__(kGnThreads) void gn_stats_kernel(const T* __restrict__ x, const double2* __restrict__ partial, GnShape s, double eps,
                                                             double2* __restrict__ stats) {
    const int64_t at = (int64_t)blockIdx.x * (kGnThreads / kWave) + (threadIdx.x >> 6);
    if (at >= (int64_t)s.n * s.groups) return;
    double sum = 0.0, sq = 0.0;
#pragma unroll 4
    for (int k = lane_id(); k < s.chunks; k += kWave) {
        const double2 p = partial[at * s.chunks + k];
        sum += p.x;
        sq += p.y;
    }
    sum = wave_sum(sum);
    sq = wave_sum(sq);
    if (lane_id() == 0) {
        const int64_t n = at / s.groups;
        const double first = (double)gn_float(x[n * s.rows * s.c + (at - n * s.groups) * s.cg]);
        stats[at] = gn_statistics(first, sum, sq, s.inv_m, eps);
    }
}

template <typename T, int V>
__global__ __launch_bounds__(kGnThreads) void gn_forward_kernel(const T* __restrict__ x, GnShape s, const double2* __restrict__ stats, GnWeights w,
                                                               int act, T* __restrict__ y) {
    const int n = blockIdx.x / s.chunks, chunk = blockIdx.x - n * s.chunks;
    const int64_t r0 = chunk * s.chunk_rows, r1 = r0 + s.chunk_rows < s.rows ? r0 + s.chunk_rows : s.rows;
    const int64_t base = (int64_t)n * s.rows * s.c;
    const int tiles = (s.c + kGnThreads * V - 1) / (kGnThreads * V);
    for (int tile = 0; tile < tiles; ++tile) {
        const GnLanes l = gn_lanes<V>(s.c, tile);
        if (!l.live) continue;
        const uint32_t lane = l.template offset<T>(s.c);
        GnScale<V> ch;
        ch.weights(w, l.col);
        ch.statistics(stats[(int64_t)n * s.groups + l.col / s.cg]);
        gn_by_act(act, s.past_cache, [&](auto A, auto last) {
            constexpr bool LAST = decltype(last)::value;
            gn_rows<T, V, gn_rows_in_flight(V), LAST>(x + base, s.c, l, r0, r1, [&](const GnPack<T, V>& v, int64_t r) {
                float o[V];
#pragma unroll
                for (int i = 0; i < V; ++i) o[i] = ch.template value<decltype(A)::value>(i, gn_float(v.v[i]));
                gn_write<T, V, LAST>(gn_at(y + base + r, lane), o);
            });
        });
    }
}

// two tensors at once, half the rows in flight of each
template <typename T, int V, int U, bool LAST = false, typename F>
__device__ __forceinline__ void gn_rows2(const T* x, const T* dy, int c, const GnLanes& l, int64_t r0, int64_t r1, F f) {
    const uint32_t lane = l.template offset<T>(c);
    const int64_t step = (int64_t)l.ty * c;
    const int all = U * l.ty;
    int64_t r = r0;
    GnPack<T, V> w[U], d[U];
    for (; r + all <= r1; r += all) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            w[u] = gn_read<T, V, LAST>(gn_at(x + r * c + u * step, lane));
            d[u] = gn_read<T, V, LAST>(gn_at(dy + r * c + u * step, lane));
        }
#pragma unroll
        for (int u = 0; u < U; ++u) f(w[u], d[u], r * c + u * step);
    }
    const int left = (int)(r1 - r);
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (l.row + u * l.ty < left) {
            w[u] = gn_read<T, V, LAST>(gn_at(x + r * c + u * step, lane));
            d[u] = gn_read<T, V, LAST>(gn_at(dy + r * c + u * step, lane));
        }
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (l.row + u * l.ty < left) f(w[u], d[u], r * c + u * step);
}

// per (sample, chunk, channel): (sum dz, sum dz xhat)
template <typename T, int V>
__global__ __launch_bounds__(kGnThreads) void gn_grad_sums_kernel(const T* __restrict__ x, const T* __restrict__ dy, GnShape s,
                                                                 const double2* __restrict__ stats, GnWeights w, int act, float2* __restrict__ partial) {
    __shared__ float lds[V * kGnThreads], res[2 * V * kGnThreads];
    const int n = blockIdx.x / s.chunks, chunk = blockIdx.x - n * s.chunks;
    const int64_t r0 = chunk * s.chunk_rows, r1 = r0 + s.chunk_rows < s.rows ? r0 + s.chunk_rows : s.rows;
    const int64_t base = (int64_t)n * s.rows * s.c;
    const int tiles = (s.c + kGnThreads * V - 1) / (kGnThreads * V);
    for (int tile = 0; tile < tiles; ++tile) {
        const GnLanes l = gn_lanes<V>(s.c, tile);
        float a[V], b[V];
#pragma unroll
        for (int i = 0; i < V; ++i) a[i] = b[i] = 0.f;
        if (l.live) {
            GnGrad<V> ch;
            ch.load(stats[(int64_t)n * s.groups + l.col / s.cg], w, act, l.col);
            gn_by_act(act, [&](auto A) {
                gn_rows2<T, V, gn_rows_in_flight(V) / 2>(x + base, dy + base, s.c, l, r0, r1, [&](const GnPack<T, V>& v, const GnPack<T, V>& d, int64_t) {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        float xhat, dz;
                        ch.template value<decltype(A)::value>(i, gn_float(v.v[i]), gn_float(d.v[i]), xhat, dz);
                        a[i] += dz;
                        b[i] = fmaf(dz, xhat, b[i]);
                    }
                });
            });
        }
        gn_sum_rows<float, V>(a, l.tx, l.ty, res, lds);
        gn_sum_rows<float, V>(b, l.tx, l.ty, res + V * l.tx, lds);
        for (int c = threadIdx.x; c < l.tx * V; c += kGnThreads) {
            const int k = c / V, i = c - k * V;
            partial[((int64_t)n * s.chunks + chunk) * s.c + tile * kGnThreads * V + c] = make_float2(res[i * l.tx + k], res[(V + i) * l.tx + k]);
        }
        __syncthreads();
    }
}

// a workgroup per (sample, group): the channels' sums over the chunks, and the group's two means
constexpr int kGnStatThreads = 512;
__global__ __launch_bounds__(kGnStatThreads) void gn_grad_stats_kernel(const float2* __restrict__ partial, GnShape s, GnWeights w,
                                                                      double2* __restrict__ channel, float2* __restrict__ means) {
    __shared__ double2 lds[kGnStatThreads];
    const int n = blockIdx.x / s.groups, g = blockIdx.x - n * s.groups;
    double s1 = 0.0, s2 = 0.0;
    for (int c0 = 0; c0 < s.cg; c0 += kGnStatThreads) {
        const int tx = s.cg - c0 < kGnStatThreads ? s.cg - c0 : kGnStatThreads, ty = kGnStatThreads / tx;
        const int row = threadIdx.x / tx, ch = g * s.cg + c0 + (threadIdx.x - row * tx);
        double2 acc = make_double2(0.0, 0.0);
        if (row < ty) {
#pragma unroll 8
            for (int k = row; k < s.chunks; k += ty) {
                const float2 p = partial[((int64_t)n * s.chunks + k) * s.c + ch];
                acc.x += p.x;
                acc.y += p.y;
            }
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
            const double gm = (double)gn_weight(w.gamma, w.dtype, ch, 1.f);
            s1 += gm * sum.x;
            s2 += gm * sum.y;
        }
    }
    s1 = wave_sum(s1);
    s2 = wave_sum(s2);
    __syncthreads();
    if (lane_id() == 0) lds[threadIdx.x >> 6] = make_double2(s1, s2);
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < kGnStatThreads / kWave; ++k) { s1 += lds[k].x; s2 += lds[k].y; }
        means[(int64_t)n * s.groups + g] = make_float2((float)(s1 * s.inv_m), (float)(s2 * s.inv_m));
    }
}

// d gamma, d beta: the samples' sums of a channel, a channel per thread over the launch's first workgroups
__device__ __forceinline__ void gn_weight_grad(const double2* channel, int rows, int c, int wdtype, void* dgamma, void* dbeta, int block, int blocks) {
    for (int64_t ch = (int64_t)block * kGnThreads + threadIdx.x; ch < c; ch += (int64_t)blocks * kGnThreads) {
        double a = 0.0, b = 0.0;
#pragma unroll 4
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

template <typename T, int V>
__global__ __launch_bounds__(kGnThreads) void gn_backward_kernel(const T* __restrict__ x, const T* __restrict__ dy, GnShape s,
                                                                const double2* __restrict__ stats, GnWeights w, int act,
                                                                const double2* __restrict__ channel, const float2* __restrict__ means,
                                                                T* __restrict__ dx, void* dgamma, void* dbeta) {
    const int n = blockIdx.x / s.chunks, chunk = blockIdx.x - n * s.chunks;
    const int64_t r0 = chunk * s.chunk_rows, r1 = r0 + s.chunk_rows < s.rows ? r0 + s.chunk_rows : s.rows;
    const int64_t base = (int64_t)n * s.rows * s.c;
    if (dgamma || dbeta) gn_weight_grad(channel, s.n, s.c, w.dtype, dgamma, dbeta, blockIdx.x, gridDim.x);
    const int tiles = (s.c + kGnThreads * V - 1) / (kGnThreads * V);
    for (int tile = 0; tile < tiles; ++tile) {
        const GnLanes l = gn_lanes<V>(s.c, tile);
        if (!l.live) continue;
        const uint32_t lane = l.template offset<T>(s.c);
        GnGrad<V> ch;
        ch.load(stats[(int64_t)n * s.groups + l.col / s.cg], w, act, l.col);
        const float2 mean = means[(int64_t)n * s.groups + l.col / s.cg];
        const float c1 = ch.rstd * mean.x, c2 = ch.rstd * mean.y;
        gn_by_act(act, s.past_cache, [&](auto A, auto last) {
            constexpr bool LAST = decltype(last)::value;
            gn_rows2<T, V, gn_rows_in_flight(V) / 2, LAST>(x + base, dy + base, s.c, l, r0, r1, [&](const GnPack<T, V>& v, const GnPack<T, V>& d, int64_t r) {
                float o[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    float xhat, dz;
                    ch.template value<decltype(A)::value>(i, gn_float(v.v[i]), gn_float(d.v[i]), xhat, dz);
                    o[i] = ch.dx(i, xhat, dz, c1, c2);
                }
                gn_write<T, V, LAST>(gn_at(dx + base + r, lane), o);
            });
        });
    }
}

// ------------------------------------------------------------------------------------------------ host
// Estimates of a pass in us for the choice of its form: linear in what each form does, fitted to 15000 random cases of 1 to 16384 samples,
// 1 to 11600 rows, 16 to 512 channels, all types and activations, at which both forms were timed.  (256 CUs; a 1024-thread workgroup of
// 128 registers fills one.)
struct GnEstimate {
    double one;                                    // a pass
    // resident: a round of workgroups over the CUs, in it 1000 elements of a workgroup (silu, gelu: more), 1000 lines of 128 bytes that its
    // rows touch, and columns that no wave holds whole; 10^6 lines, MB and 1000 waves of all
    double round, elements, silu, gelu, lines, ragged, all_lines, mb, waves;
    // streamed: MB, 10^6 elements (silu, gelu, one channel a thread: more), KB of a row, 1000 groups and 10^6 channels of all samples
    double s_one, s_mb, s_elements, s_silu, s_gelu, s_single, s_row, s_groups, s_channels;
};
static const GnEstimate kGnEstimate[2] = {
    {2.8, 1.7, 0.11, 0.029, 0.097, 0.71, 0.51, 3.2, 0.10, 0.35, 10.0, 0.28, 0.44, 0.09, 0.42, 0.90, 0.38, 0.3, 8.6},       // forward
    {3.8, 3.3, 0.17, 0.075, 0.20, 0.80, 0.70, 3.3, 0.39, 0.64, 12.0, 0.38, 0.93, 0.24, 0.75, 0.03, 1.6, 4.0, 42.0}};       // backward
static bool gn_streamed_fits(const GnShape& s) { return (int64_t)s.n * s.groups * kGnStatThreads <= UINT32_MAX; }
static bool gn_streamed_is_faster(const GnShape& s, int item, int act, bool backward) {
    const GnEstimate& e = kGnEstimate[backward];
    const double workgroups = (double)s.n * s.slabs, waves = s.threads / kWave, at_once = 256.0 * (16 / (s.threads / kWave));
    const double rounds = ceil(workgroups / at_once), own = 1e-3 * (double)s.rows * s.cs, lines = 1e-3 * (double)s.rows * ((s.cs * item + 127) / 128);
    const double all = 1e-6 * (double)s.n * s.rows * s.c;
    const double resident = e.one + rounds * (e.round + own * (e.elements + (act == kGnSilu ? e.silu : act == kGnGelu ? e.gelu : 0.0)) + lines * e.lines +
                                              (gn_whole_rows(s.tx) ? 0.0 : e.ragged)) +
                            1e-3 * workgroups * (lines * e.all_lines + waves * e.waves) + all * item * e.mb;
    const double streamed = e.s_one + all * (item * e.s_mb + e.s_elements + (act == kGnSilu ? e.s_silu : act == kGnGelu ? e.s_gelu : 0.0) +
                                             (s.v == 1 ? e.s_single : 0.0)) +
                            1e-3 * s.c * item * e.s_row + 1e-3 * s.n * s.groups * e.s_groups + 1e-6 * (double)s.n * s.c * e.s_channels;
    return streamed < resident;
}
static GnShape gn_shape(int32_t n, int64_t rows, int32_t c, int32_t groups, int dtype, int act, bool backward) {
    GnShape s;
    s.n = n; s.rows = rows; s.c = c; s.groups = groups; s.cg = c / groups;
    s.inv_m = 1.0 / ((double)rows * s.cg);
    s.v = s.cg % 4 == 0 ? 4 : (s.cg % 2 == 0 ? 2 : 1);
    const int item = dtype == GEOMAE_DTYPE_F32 ? 4 : 2;
    s.past_cache = (double)n * rows * c * item > 64e6;
    // Resident, if all rows of a group fit and the estimates are for it; more groups to a workgroup while its piece of a row is short of a
    // cache line and there are workgroups for every CU without.  Tensors over 64 MB of more than 1000 rows are streamed (46 cases forward and 46
    // backward: resident 48 and 44 % longer than the better form, streamed 0.1).  Over 5000 random cases that the estimates were
    // not fitted to (profiles/group_norm_forms.txt) the form chosen takes 0.9 % (forward) and 0.8 % (backward) longer than the better
    // one, always resident where it fits 7.0 and 6.5, always streamed 64 and 57.  In us, resident against streamed, fp32 with ReLU: 8 x 512 x 20 x
    // 20 forward 7.0 and 12.4, 4 x 256 x 50 x 50 backward 19.7 and 21.8; 2 x 256 x 64 x 64 backward (64 workgroups) 25.4 and 19.8, 8 x
    // 256 x 90 x 90 in groups of 4 channels (an eighth of each line) forward 59 and 39.
    s.cs = s.threads = s.tx = s.ty = s.slabs = s.slab_groups = 0;
    s.tx_inverse = 0;
    const int held = gn_vectors_held(s.v, item);
    auto fits = [&](int64_t cs) {
        const int64_t tx = cs / s.v;
        return tx <= kGnResidentThreads && rows <= kGnResidentThreads / tx * held;
    };
    if (fits(s.cg)) {
        int k = 1;
        for (int d = 2; d <= groups && (int64_t)k * s.cg * item < 128; ++d)
            if (groups % d == 0 && fits((int64_t)d * s.cg) && (int64_t)n * (groups / d) >= 256) k = d;
        s.cs = k * s.cg;
        const int64_t tx = s.cs / s.v;
        // (two vectors a thread: enough loads in flight, and half the threads to add up)
        int64_t threads = (tx * ((rows + 1) / 2) + kWave - 1) / kWave * kWave;
        threads = threads > kGnResidentThreads ? kGnResidentThreads : threads;
        while (threads < tx || threads / tx * held < rows) threads += kWave;
        s.threads = (int32_t)threads;
        s.tx = (int32_t)tx; s.ty = (int32_t)(threads / tx); s.slabs = c / s.cs; s.slab_groups = s.cs / s.cg;
        s.tx_inverse = (uint32_t)(((1 << 20) + tx - 1) / tx);
        if (gn_streamed_fits(s) && ((s.past_cache && rows > 1000) || gn_streamed_is_faster(s, item, act, backward))) s.cs = 0;
    }
    const int cv = c / s.v, ty = cv < kGnThreads ? kGnThreads / cv : 1, unroll = gn_rows_in_flight(s.v);
    const int64_t least = (int64_t)ty * unroll, wanted = kGnBlocks / n > 1 ? kGnBlocks / n : 1;
    s.chunk_rows = (rows + wanted - 1) / wanted;
    s.chunk_rows = s.chunk_rows < least ? least : (s.chunk_rows + least - 1) / least * least;
    // the gradient sums: a thread adds up at most kGnSumRows rows in fp32, whatever the batch leaves to a workgroup
    if (backward && s.chunk_rows > (int64_t)kGnSumRows * ty) s.chunk_rows = (int64_t)kGnSumRows * ty;
    s.chunks = s.cs ? 0 : (int32_t)((rows + s.chunk_rows - 1) / s.chunk_rows);
    return s;
}
// the threads of a launch are counted in 32 bits
static int gn_check_launches(const char* what, const GnShape& s) {
    const int64_t main = s.cs ? (int64_t)s.n * s.slabs * s.threads : (int64_t)s.n * s.chunks * kGnThreads;
    const int64_t means = s.cs ? 0 : (int64_t)s.n * s.groups * kGnStatThreads, fold = ((int64_t)s.n + kGnFold - 1) / kGnFold * s.c;
    GEOMAE_REQUIRE(main <= UINT32_MAX && means <= UINT32_MAX && fold <= INT32_MAX, "%s: %d samples of %d channels in %d groups are too many", what,
                   (int)s.n, (int)s.c, (int)s.groups);
    return GEOMAE_OK;
}
static int64_t gn_pad(int64_t bytes) { return (bytes + 15) / 16 * 16; }
struct GnWorkspace { double2* partial; float2* grad_partial; double2 *channel, *folded; float2* means; int64_t forward_bytes, backward_bytes; };
static GnWorkspace gn_workspace(void* base, const GnShape& s) {
    char* p = static_cast<char*>(base);
    GnWorkspace w;
    w.partial = reinterpret_cast<double2*>(p);
    w.forward_bytes = (int64_t)s.n * s.chunks * s.groups * (int64_t)sizeof(double2);
    w.channel = reinterpret_cast<double2*>(p);
    int64_t at = s.cs && s.n == 1 ? 0 : (int64_t)s.n * s.c * (int64_t)sizeof(double2);
    w.grad_partial = reinterpret_cast<float2*>(p + at);
    at += gn_pad((int64_t)s.n * s.chunks * s.c * (int64_t)sizeof(float2));
    w.means = reinterpret_cast<float2*>(p + at);
    at += s.cs ? 0 : gn_pad((int64_t)s.n * s.groups * (int64_t)sizeof(float2));
    w.folded = reinterpret_cast<double2*>(p + at);                     // two halves, used in turn
    w.backward_bytes = at + (s.n > kGnFold ? 2 * (int64_t)((s.n + kGnFold - 1) / kGnFold) * s.c * (int64_t)sizeof(double2) : 0);
    return w;
}
// dynamic LDS of the resident kernels: the groups' values, the columns' sums, and what gn_sum_rows works in
static size_t gn_resident_lds(const GnShape& s, bool backward) {
    const int v = s.v;
    const int64_t tx = s.cs / v, item = backward ? 4 : 8;
    if (gn_whole_rows((int)tx)) {
        const int64_t width = backward ? 2 * v : 2, weights = backward ? v : 0;
        return (size_t)(s.cs / s.cg * (backward ? 8 : 16) + (width + weights + width * (s.threads / kWave)) * tx * item);
    }
    const int64_t width = backward ? (tx <= kGnResidentThreads / 2 ? 2 * v : v) : 2;
    return (size_t)(s.cs / s.cg * (backward ? 8 : 16) + ((backward ? 2 * v : 2) * tx + width * s.threads) * item);
}
static int gn_check(const char* what, int32_t n, int64_t rows, int32_t c, int32_t groups, int dtype, int wdtype, int act) {
    GEOMAE_REQUIRE(n >= 0 && rows >= 0 && c > 0 && groups > 0, "%s: bad shape [%d, %lld, %d] in %d groups", what, (int)n,
                   (long long)rows, (int)c, (int)groups);
    GEOMAE_REQUIRE(c % groups == 0, "%s: %d channels do not divide into %d groups", what, (int)c, (int)groups);
    GEOMAE_REQUIRE(groups <= kGnMaxGroups, "%s: at most %d groups, got %d", what, kGnMaxGroups, (int)groups);
    GEOMAE_REQUIRE(c <= kGnMaxChannels, "%s: at most %d channels, got %d", what, kGnMaxChannels, (int)c);
    GEOMAE_REQUIRE((int64_t)n * groups <= INT32_MAX, "%s: %d samples of %d groups are too many", what,
                   (int)n, (int)groups);
    GEOMAE_REQUIRE(dtype >= 0 && dtype <= 2 && wdtype >= 0 && wdtype <= 2, "%s: unknown dtype", what);
    GEOMAE_REQUIRE(act >= 0 && act <= 3, "%s: unknown activation %d", what, act);
    return GEOMAE_OK;
}
static void gn_launch_weight_grad(const double2* channel, int rows, const GnShape& s, const GnWorkspace& w, int wdtype, void* dgamma, void* dbeta, hipStream_t stream) {
    double2* halves[2] = {w.folded, w.folded + (int64_t)((s.n + kGnFold - 1) / kGnFold) * s.c};
    for (int k = 0; rows > kGnFold; ++k) {
        const int next = (rows + kGnFold - 1) / kGnFold;
        hipLaunchKernelGGL(gn_fold_kernel, dim3(cdiv((int64_t)next * s.c, kGnThreads)), dim3(kGnThreads), 0, stream, channel, rows, s.c, halves[k & 1]);
        channel = halves[k & 1];
        rows = next;
    }
    hipLaunchKernelGGL(gn_weight_grad_kernel, dim3(cdiv(s.c, kGnThreads)), dim3(kGnThreads), 0, stream, channel, rows, s.c, wdtype, dgamma, dbeta);
}

// f(type, vector) for the run-time choice of the two
template <typename T> struct GnType { typedef T type; };
template <typename T, typename F> static void gn_by_vector(int v, F f) {
    if (v == 4) f(GnType<T>(), std::integral_constant<int, 4>());
    else if (v == 2) f(GnType<T>(), std::integral_constant<int, 2>());
    else f(GnType<T>(), std::integral_constant<int, 1>());
}
template <typename F> static void gn_by_type(int dtype, int v, F f) {
    if (dtype == GEOMAE_DTYPE_F32) gn_by_vector<float>(v, f);
    else if (dtype == GEOMAE_DTYPE_BF16) gn_by_vector<uint16_t>(v, f);
    else gn_by_vector<_Float16>(v, f);
}

}  // namespace geomae

using namespace geomae;

extern "C" int64_t geomae_group_norm_workspace_bytes(int32_t n, int64_t rows, int32_t c, int32_t groups, int32_t dtype, int32_t backward) {
    if (gn_check("group_norm_workspace_bytes", n, rows, c, groups, dtype, 0, 0)) return -1;
    if (n == 0 || rows == 0) return 0;
    int64_t bytes = 0;
    for (int act : {kGnNone, kGnSilu, kGnGelu}) {                      // (the form may depend on the activation)
        const GnShape s = gn_shape(n, rows, c, groups, dtype, act, backward != 0);
        if (gn_check_launches("group_norm_workspace_bytes", s)) return -1;
        const GnWorkspace w = gn_workspace(nullptr, s);
        const int64_t need = backward ? w.backward_bytes : w.forward_bytes;
        bytes = need > bytes ? need : bytes;
    }
    return bytes;
}

extern "C" int geomae_group_norm_forward(const void* x, int32_t dtype, int32_t n, int64_t rows, int32_t c, int32_t groups, const void* gamma,
                                         const void* beta, int32_t weight_dtype, double eps, int32_t activation, void* y, double* stats,
                                         void* workspace, int64_t workspace_bytes, hipStream_t stream) {
    if (int rc = gn_check("group_norm_forward", n, rows, c, groups, dtype, weight_dtype, activation)) return rc;
    GEOMAE_REQUIRE(eps >= 0.0, "group_norm_forward: eps must not be negative");
    if (n == 0 || rows == 0) return GEOMAE_OK;
    GEOMAE_REQUIRE(x && y && stats, "group_norm_forward: null argument");
    const GnShape s = gn_shape(n, rows, c, groups, dtype, activation, false);
    if (int rc = gn_check_launches("group_norm_forward", s)) return rc;
    const GnWorkspace ws = gn_workspace(workspace, s);
    if (workspace_bytes < ws.forward_bytes || (ws.forward_bytes && !workspace)) {
        set_error("group_norm_forward: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)ws.forward_bytes);
        return GEOMAE_ERR_WORKSPACE;
    }
    double2* st = reinterpret_cast<double2*>(stats);
    const GnWeights w = {gamma, beta, weight_dtype};
    if (s.cs) {
        gn_by_type(dtype, s.v, [&](auto t, auto vec) {
            typedef typename decltype(t)::type T;
            hipLaunchKernelGGL((gn_resident_forward_kernel<T, decltype(vec)::value>), dim3(n * s.slabs), dim3(s.threads), gn_resident_lds(s, false), stream,
                               static_cast<const T*>(x), s, w, eps, activation, static_cast<T*>(y), st);
        });
        return check_launch("gn_resident_forward_kernel");
    }
    gn_by_type(dtype, s.v, [&](auto t, auto vec) {
        typedef typename decltype(t)::type T;
        constexpr int V = decltype(vec)::value;
        const T* in = static_cast<const T*>(x);
        hipLaunchKernelGGL((gn_sums_kernel<T, V>), dim3(s.chunks * n), dim3(kGnThreads), groups * sizeof(double2), stream, in, s, ws.partial);
        hipLaunchKernelGGL(gn_stats_kernel<T>, dim3(cdiv((int64_t)n * groups, kGnThreads / kWave)), dim3(kGnThreads), 0, stream, in, ws.partial, s, eps, st);
        hipLaunchKernelGGL((gn_forward_kernel<T, V>), dim3(s.chunks * n), dim3(kGnThreads), 0, stream, in, s, st, w, activation, static_cast<T*>(y));
    });
    return check_launch("gn_forward_kernel");
}

extern "C" int geomae_group_norm_backward(const void* x, const void* dy, int32_t dtype, int32_t n, int64_t rows, int32_t c, int32_t groups,
                                          const void* gamma, const void* beta, int32_t weight_dtype, int32_t activation, const double* stats,
                                          void* dx, void* dgamma, void* dbeta, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
    if (int rc = gn_check("group_norm_backward", n, rows, c, groups, dtype, weight_dtype, activation)) return rc;
    if (n == 0 || rows == 0) {                                          // sums of nothing
        if (!dgamma && !dbeta) return GEOMAE_OK;
        hipLaunchKernelGGL(gn_weight_grad_kernel, dim3(cdiv(c, kGnThreads)), dim3(kGnThreads), 0, stream, nullptr, 0, c, weight_dtype, dgamma, dbeta);
        return check_launch("gn_weight_grad_kernel");
    }
    GEOMAE_REQUIRE(x && dy && stats && dx, "group_norm_backward: null argument");
    const GnShape s = gn_shape(n, rows, c, groups, dtype, activation, true);
    if (int rc = gn_check_launches("group_norm_backward", s)) return rc;
    const GnWorkspace ws = gn_workspace(workspace, s);
    if (workspace_bytes < ws.backward_bytes || (ws.backward_bytes && !workspace)) {
        set_error("group_norm_backward: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)ws.backward_bytes);
        return GEOMAE_ERR_WORKSPACE;
    }
    const double2* st = reinterpret_cast<const double2*>(stats);
    const GnWeights w = {gamma, beta, weight_dtype};
    const bool weights = dgamma || dbeta, many = n > kGnFold;
    gn_by_type(dtype, s.v, [&](auto t, auto vec) {
        typedef typename decltype(t)::type T;
        constexpr int V = decltype(vec)::value;
        const T *in = static_cast<const T*>(x), *grad = static_cast<const T*>(dy);
        if (s.cs) {
            hipLaunchKernelGGL((gn_resident_backward_kernel<T, V>), dim3(n * s.slabs), dim3(s.threads), gn_resident_lds(s, true), stream, in, grad, s,
                               st, w, activation, static_cast<T*>(dx), n == 1 ? nullptr : ws.channel, dgamma, dbeta);
            if (weights && n > 1) gn_launch_weight_grad(ws.channel, n, s, ws, weight_dtype, dgamma, dbeta, stream);
            return;
        }
        hipLaunchKernelGGL((gn_grad_sums_kernel<T, V>), dim3(s.chunks * n), dim3(kGnThreads), 0, stream, in, grad, s, st, w, activation, ws.grad_partial);
        hipLaunchKernelGGL(gn_grad_stats_kernel, dim3(groups * n), dim3(kGnStatThreads), 0, stream, ws.grad_partial, s, w, ws.channel, ws.means);
        hipLaunchKernelGGL((gn_backward_kernel<T, V>), dim3(s.chunks * n), dim3(kGnThreads), 0, stream, in, grad, s, st, w, activation, ws.channel,
                           ws.means, static_cast<T*>(dx), many ? nullptr : dgamma, many ? nullptr : dbeta);
        if (weights && many) gn_launch_weight_grad(ws.channel, n, s, ws, weight_dtype, dgamma, dbeta, stream);
    });
    return check_launch("gn_backward_kernel");
}
