// AdamW over many tensors where they lie (geomae_amd.optim.MultiTensorAdamW), moments in 32 or in 8 bits.
//
//   g' = g * grad_scale * min(1, max_norm / (norm + 1e-6)),   norm = grad_scale * sqrt(sum over all tensors of g^2)
//   p *= 1 - lr wd ;  m += (1 - b1) (g' - m) ;  v = b2 v + (1 - b2) g'^2
//   p -= lr / (1 - b1^s) * m / (sqrt(v) / sqrt(1 - b2^s) + eps)               s = steps this tensor has taken, kept on the device
//
// all in fp32 (the norm's sums in fp64: its rounding would reach every element), operation by operation as in optim.hip.
//
// 8-bit moments: 32 consecutive elements share an exponent byte E (value = code value * 2^(E - 135); a power of two, so that
// scaling is exact and a block's re-scaling never re-rounds its other elements).  m: sign, 4 exponent and 3 fraction bits
// (e4m3, largest 448, 0x7f = NaN); r = sqrt(v), not v: half the binades for the same range: 4 exponent and 4 fraction bits,
// no sign (largest code 254 = 480, 255 = NaN).  E is the exponent field of the block's largest magnitude, one more where that
// is above the largest code.
// Rounding is STOCHASTIC: k = floor(y / step + (u + 1/2) / 65536).  To the nearest, r would freeze: with b2 = 0.999 a step
// moves it by 0.05 % at most, half a code step is 3 %.  u: 16 bits (low half m, high half r) of a hash of (seed, tensor index,
// step, element), so that a run is reproducible and graph replays draw anew.  r > 0 never becomes code 0: m over a zero root
// would be an unbounded update; the smallest code bounds it by the block's own largest ratio.
//
// What bounds it: HBM.  Bytes per element: fp32 parameters 28 with 32-bit moments (p, m, v in and out, g in) and 16 1/8 with
// 8-bit ones.  A workgroup takes a chunk of 4096 elements of one tensor, found through a table built once; the gradients'
// addresses, which change from step to step, ride in the launch's arguments, so that no copy to the device and no state of the
// call's own stands between two steps or inside a captured graph.
#include "common.h"
#include "../../include/geomae_hip.h"
#include <math.h>

namespace geomae {

constexpr int kMaThreads = 256, kMaVec = 4, kMaIters = 4;
constexpr int kMaChunk = kMaThreads * kMaVec * kMaIters;             // elements of a workgroup
constexpr int kMaTensors = 256;                                      // gradient addresses of a launch (2 KB of arguments)
constexpr int kMaHypers = 16;                                        // distinct hyper-parameter sets of a launch
constexpr int kMaNormGrid = 1024;                                    // workgroups (= partial sums) of a norm launch

struct MaScalars { float decay, w1, b2, omb2, bc2_sqrt, eps, step_size; uint32_t key; };
struct MaControl { float coef; int32_t skip; };

__host__ __device__ __forceinline__ uint32_t ma_mix(uint32_t x) {
    x = (x ^ (x >> 15)) * 0xBB67AE85u;
    x = (x ^ (x >> 13)) * 0x243F6A89u;
    return x ^ (x >> 16);
}

// ------------------------------------------------------------------------------------------------ typed loads and stores
// Parameters and gradients are views at any element offset: the packed types tell the compiler no more than the element's own
// alignment (global memory takes 8- and 16-byte accesses at any 2- or 4-byte address).
template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) MaPack { T v[N]; };

template <typename T> __device__ __forceinline__ float ma_float(T x) { return (float)x; }
template <> __device__ __forceinline__ float ma_float<uint16_t>(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }   // bf16
template <typename T> __device__ __forceinline__ T ma_narrow(float x) { return (T)x; }
template <> __device__ __forceinline__ uint16_t ma_narrow<uint16_t>(float x) {                                               // to nearest even
    const uint32_t b = __float_as_uint(x);
    return x != x ? (uint16_t)((b >> 16) | 0x40) : (uint16_t)((b + 0x7fff + ((b >> 16) & 1)) >> 16);
}

template <typename T>
__device__ __forceinline__ void ma_load(const T* p, int64_t e, int64_t n, float (&out)[kMaVec]) {
    if (e + kMaVec <= n) {
        const MaPack<T, kMaVec> w = *reinterpret_cast<const MaPack<T, kMaVec>*>(p + e);
#pragma unroll
        for (int i = 0; i < kMaVec; ++i) out[i] = ma_float<T>(w.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < kMaVec; ++i) out[i] = e + i < n ? ma_float<T>(p[e + i]) : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void ma_store(T* p, int64_t e, int64_t n, const float (&x)[kMaVec]) {
    if (e + kMaVec <= n) {
        MaPack<T, kMaVec> w;
#pragma unroll
        for (int i = 0; i < kMaVec; ++i) w.v[i] = ma_narrow<T>(x[i]);
        *reinterpret_cast<MaPack<T, kMaVec>*>(p + e) = w;
    } else {
#pragma unroll
        for (int i = 0; i < kMaVec; ++i)
            if (e + i < n) p[e + i] = ma_narrow<T>(x[i]);
    }
}

// ------------------------------------------------------------------------------------------------ 8-bit moments
// largest finite magnitude of the 8 lanes x 4 elements of a block
__device__ __forceinline__ float ma_block_max(const float (&x)[kMaVec]) {
    float a = 0.f;
#pragma unroll
    for (int i = 0; i < kMaVec; ++i) {
        const float y = fabsf(x[i]);
        a = fmaxf(a, y < INFINITY ? y : 0.f);
    }
    a = fmaxf(a, dpp_mov<kDppXor1>(a));
    a = fmaxf(a, dpp_mov<kDppXor2>(a));
    return fmaxf(a, dpp_mov<kDppHalfMirror>(a));
}
template <bool SIGNED>
__device__ __forceinline__ int ma_exponent(float largest) {          // + 0x1fffff / 0x0fffff: carries above 1.75 / 1.875
    const int e = (int)((__float_as_uint(largest) + (SIGNED ? 0x1fffffu : 0x0fffffu)) >> 23);
    return e < 16 ? 16 : (e > 254 ? 254 : e);
}
__device__ __forceinline__ float ma_unscale(int e) { return __uint_as_float((uint32_t)(e - 8) << 23); }     // 2^(E - 135)
__device__ __forceinline__ float ma_scale(int e) { return __uint_as_float((uint32_t)(262 - e) << 23); }     // 2^(135 - E)

// y >= 0 in units of the block's scale -> the code value it is held as
template <int DIGITS>
__device__ __forceinline__ float ma_round(float y, uint32_t u16) {
    int place = (int)(__float_as_uint(y) >> 23);
    place = place < 121 ? 121 : place;                               // below 2^-6 the codes are evenly spaced
    const float inv_step = __uint_as_float((uint32_t)(254 + DIGITS - place) << 23);
    const float step = __uint_as_float((uint32_t)(place - DIGITS) << 23);
    return floorf(__fadd_rn(y * inv_step, ((float)u16 + 0.5f) * 0x1p-16f)) * step;
}
__device__ __forceinline__ uint32_t ma_code_signed(const float (&x)[kMaVec], float scale, const uint32_t (&draw)[kMaVec]) {
    float q[kMaVec];
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < kMaVec; ++i) {
        const float y = fabsf(x[i]) * scale;
        q[i] = copysignf(ma_round<3>(y, draw[i] & 0xffffu), x[i]);
        if (!(fabsf(x[i]) < INFINITY)) bad |= 0x7fu << (8 * i), q[i] = 0.f;
    }
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);   // exact: q is a code's value already
    w = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w, true);
    return (uint32_t)w | bad;
}
__device__ __forceinline__ uint32_t ma_code_root(const float (&x)[kMaVec], float scale, const uint32_t (&draw)[kMaVec]) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < kMaVec; ++i) {
        const float y = x[i] * scale;
        float q = ma_round<4>(y, draw[i] >> 16);
        if (q == 0.f && x[i] > 0.f) q = 0x1p-10f;
        uint32_t c = q >= 0x1p-6f ? (__float_as_uint(q) >> 19) - 1920u : (uint32_t)(q * 0x1p10f);
        if (!(x[i] < INFINITY)) c = 255u;
        w |= c << (8 * i);
    }
    return w;
}
__device__ __forceinline__ void ma_value_signed(uint32_t w, float unscale, float (&out)[kMaVec]) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    out[0] = a[0] * unscale; out[1] = a[1] * unscale; out[2] = b[0] * unscale; out[3] = b[1] * unscale;
}
__device__ __forceinline__ void ma_value_root(uint32_t w, float unscale, float (&out)[kMaVec]) {
#pragma unroll
    for (int i = 0; i < kMaVec; ++i) {
        const uint32_t c = (w >> (8 * i)) & 255u;
        const float f = c == 255u ? NAN : __uint_as_float(c << 19) * 0x1p120f;     // 4 + 4 bits as an fp32 with that exponent bias
        out[i] = f * unscale;
    }
}

// ------------------------------------------------------------------------------------------------ norm
struct MaNormArgs {
    const GeomaeAdamwTensor* rows;
    const int32_t* chunks;              // [num chunks][2] = (tensor, chunk of that tensor)
    double* partial;                    // one per workgroup
    int32_t first_tensor, first_chunk, num_chunks;
    const void* grads[kMaTensors];
};

template <typename T>
__device__ __forceinline__ double ma_sumsq(const T* g, int64_t start, int64_t n) {
    double acc = 0.0;
    float x[kMaIters][kMaVec];
#pragma unroll
    for (int it = 0; it < kMaIters; ++it) {
        const int64_t e = start + (it * kMaThreads + threadIdx.x) * kMaVec;
        ma_load<T>(g, e < n ? e : n, n, x[it]);
    }
#pragma unroll
    for (int it = 0; it < kMaIters; ++it)
#pragma unroll
        for (int i = 0; i < kMaVec; ++i) acc += (double)x[it][i] * (double)x[it][i];
    return acc;
}

__global__ __launch_bounds__(kMaThreads) void multi_sumsq_kernel(MaNormArgs a) {
    __shared__ double red[kMaThreads / kWave];
    double acc = 0.0;
    for (int c = blockIdx.x; c < a.num_chunks; c += gridDim.x) {
        const int32_t* at = a.chunks + 2 * ((int64_t)a.first_chunk + c);
        const int t = at[0];
        const int64_t start = (int64_t)at[1] * kMaChunk;
        const void* g = a.grads[t - a.first_tensor];
        if (!g) continue;
        const int64_t n = a.rows[t].numel;
        const int dtype = a.rows[t].dtype;
        if (dtype == GEOMAE_DTYPE_F32) acc += ma_sumsq(static_cast<const float*>(g), start, n);
        else if (dtype == GEOMAE_DTYPE_BF16) acc += ma_sumsq(static_cast<const uint16_t*>(g), start, n);
        else acc += ma_sumsq(static_cast<const _Float16*>(g), start, n);
    }
    acc = wave_sum(acc);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
    __syncthreads();
    if (threadIdx.x == 0) a.partial[blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

// ------------------------------------------------------------------------------------------------ per-tensor scalars
struct MaPrepareArgs {
    const GeomaeAdamwTensor* rows;
    const double* partial;
    MaScalars* scalars;
    MaControl* control;
    float* grad_norm;
    const float* grad_scale_ptr;
    double grad_scale, max_norm;
    int32_t want_norm, num_partial, first_tensor, num_tensors, skip_nonfinite;
    uint32_t seed;
    GeomaeAdamwHyper hypers[kMaHypers];
    uint8_t hyper_of[kMaTensors];       // 255: no gradient, the tensor is left as it is
};

// one workgroup: the norm of all tensors from its partial sums (in a fixed order), the factor of the gradients, and what each
// tensor's update needs of its own step count
__global__ __launch_bounds__(kMaThreads) void multi_prepare_kernel(MaPrepareArgs a) {
    __shared__ double red[kMaThreads / kWave];
    __shared__ int32_t skip_s;
    double acc = 0.0;
    for (int i = threadIdx.x; i < a.num_partial; i += kMaThreads) acc += a.partial[i];
    acc = wave_sum(acc);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
    __syncthreads();
    if (threadIdx.x == 0) {
        const float scale = a.grad_scale_ptr ? (float)((double)*a.grad_scale_ptr * a.grad_scale) : (float)a.grad_scale;
        float coef = scale;
        int32_t skip = 0;
        if (a.want_norm) {
            const float norm = (float)(sqrt(red[0] + red[1] + red[2] + red[3]) * fabs((double)scale));
            if (a.grad_norm) *a.grad_norm = norm;
            if (a.max_norm > 0.0 && a.max_norm < INFINITY) {
                const float c = (float)a.max_norm / (norm + 1e-6f);
                coef *= c > 1.0f ? 1.0f : c;                         // NaN stays NaN
            }
            skip = a.skip_nonfinite && !(norm < INFINITY);
        }
        a.control->coef = coef;
        a.control->skip = skip;
        skip_s = skip;
    }
    __syncthreads();
    const int t = threadIdx.x;
    if (skip_s || t >= a.num_tensors || a.hyper_of[t] == 255) return;
    const GeomaeAdamwTensor row = a.rows[a.first_tensor + t];
    const GeomaeAdamwHyper h = a.hypers[a.hyper_of[t]];
    const int64_t step = *row.step + 1;
    *row.step = step;
    const double lr = h.lr_ptr ? (double)*h.lr_ptr : h.lr;
    const double bc1 = 1.0 - pow(h.beta1, (double)step), bc2 = 1.0 - pow(h.beta2, (double)step);
    MaScalars s;
    s.decay = (float)(1.0 - lr * h.weight_decay);
    s.w1 = (float)(1.0 - h.beta1);
    s.b2 = (float)h.beta2;
    s.omb2 = (float)(1.0 - h.beta2);
    s.bc2_sqrt = (float)sqrt(bc2);
    s.eps = (float)h.eps;
    s.step_size = (float)(lr / bc1);
    s.key = ma_mix(ma_mix(a.seed + 0x9E3779B9u * (uint32_t)row.index) ^ (uint32_t)step);
    a.scalars[a.first_tensor + t] = s;
}

// ------------------------------------------------------------------------------------------------ update
struct MaStepArgs {
    const GeomaeAdamwTensor* rows;
    const int32_t* chunks;
    const MaScalars* scalars;
    const MaControl* control;
    int32_t first_tensor, first_chunk;
    const void* grads[kMaTensors];
};

template <typename T, bool MASTER, int BITS>
__device__ __forceinline__ void ma_update(const GeomaeAdamwTensor& row, const T* g, int64_t start, const MaScalars& s, float coef) {
    const int64_t n = row.numel, padded = (n + 31) & ~(int64_t)31;   // the moments' and masters' own length
    T* param = static_cast<T*>(row.param);
    float gv[kMaIters][kMaVec], pv[kMaIters][kMaVec], mv[kMaIters][kMaVec], vv[kMaIters][kMaVec];
    uint32_t mw[kMaIters], rw[kMaIters];
    int me[kMaIters], re[kMaIters];
#pragma unroll
    for (int it = 0; it < kMaIters; ++it) {
        const int64_t e = start + (it * kMaThreads + (int)threadIdx.x) * kMaVec;
        if (e >= padded) continue;                                   // whole groups of 8 lanes
        ma_load<T>(g, e < n ? e : n, n, gv[it]);
        if constexpr (MASTER) {
            const float4 w = *reinterpret_cast<const float4*>(row.master + e);
            pv[it][0] = w.x; pv[it][1] = w.y; pv[it][2] = w.z; pv[it][3] = w.w;
        } else ma_load<T>(param, e < n ? e : n, n, pv[it]);
        if constexpr (BITS == 32) {
            const float4 m = *reinterpret_cast<const float4*>(static_cast<const float*>(row.exp_avg) + e);
            const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(row.exp_avg_sq) + e);
            mv[it][0] = m.x; mv[it][1] = m.y; mv[it][2] = m.z; mv[it][3] = m.w;
            vv[it][0] = v.x; vv[it][1] = v.y; vv[it][2] = v.z; vv[it][3] = v.w;
        } else {
            mw[it] = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(row.exp_avg) + e);
            rw[it] = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(row.exp_avg_sq) + e);
            me[it] = row.exp_avg_exponent[e >> 5];
            re[it] = row.exp_avg_sq_exponent[e >> 5];
        }
    }
#pragma unroll
    for (int it = 0; it < kMaIters; ++it) {
        const int64_t e = start + (it * kMaThreads + (int)threadIdx.x) * kMaVec;
        if (e >= padded) continue;
        float r[kMaVec];
        if constexpr (BITS == 8) {
            ma_value_signed(mw[it], ma_unscale(me[it]), mv[it]);
            ma_value_root(rw[it], ma_unscale(re[it]), r);
#pragma unroll
            for (int i = 0; i < kMaVec; ++i) vv[it][i] = __fmul_rn(r[i], r[i]);
        }
#pragma unroll
        for (int i = 0; i < kMaVec; ++i) {
            const float x = __fmul_rn(gv[it][i], coef);
            float& m = mv[it][i];
            float& v = vv[it][i];
            const float d = __fsub_rn(x, m);
            m = s.w1 < 0.5f ? __fadd_rn(m, __fmul_rn(s.w1, d)) : __fsub_rn(x, __fmul_rn(d, __fsub_rn(1.0f, s.w1)));
            v = __fadd_rn(__fmul_rn(v, s.b2), __fmul_rn(__fmul_rn(s.omb2, x), x));
            r[i] = __fsqrt_rn(v);
            float p = __fmul_rn(pv[it][i], s.decay);
            const float denom = __fadd_rn(__fdiv_rn(r[i], s.bc2_sqrt), s.eps);
            pv[it][i] = __fadd_rn(p, __fmul_rn(-s.step_size, __fdiv_rn(m, denom)));
        }
        if (e < n) ma_store<T>(param, e, n, pv[it]);
        if constexpr (MASTER) {
#pragma unroll
            for (int i = 0; i < kMaVec; ++i) pv[it][i] = e + i < n ? pv[it][i] : 0.f;             // (0 / 0 where eps is 0)
            *reinterpret_cast<float4*>(row.master + e) = make_float4(pv[it][0], pv[it][1], pv[it][2], pv[it][3]);
        }
        if constexpr (BITS == 32) {
            *reinterpret_cast<float4*>(static_cast<float*>(row.exp_avg) + e) = make_float4(mv[it][0], mv[it][1], mv[it][2], mv[it][3]);
            *reinterpret_cast<float4*>(static_cast<float*>(row.exp_avg_sq) + e) = make_float4(vv[it][0], vv[it][1], vv[it][2], vv[it][3]);
        } else {
            uint32_t draw[kMaVec];
#pragma unroll
            for (int i = 0; i < kMaVec; ++i) draw[i] = ma_mix(s.key + (uint32_t)(e + i));
            const int em = ma_exponent<true>(ma_block_max(mv[it])), er = ma_exponent<false>(ma_block_max(r));
            *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(row.exp_avg) + e) = ma_code_signed(mv[it], ma_scale(em), draw);
            *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(row.exp_avg_sq) + e) = ma_code_root(r, ma_scale(er), draw);
            if ((threadIdx.x & 7) == 0) {
                row.exp_avg_exponent[e >> 5] = (uint8_t)em;
                row.exp_avg_sq_exponent[e >> 5] = (uint8_t)er;
            }
        }
    }
}

template <int BITS>
__global__ __launch_bounds__(kMaThreads) void multi_adamw_kernel(MaStepArgs a) {
    const int32_t* at = a.chunks + 2 * (a.first_chunk + (int64_t)blockIdx.x);
    const int t = at[0];
    const int64_t start = (int64_t)at[1] * kMaChunk;
    const void* g = a.grads[t - a.first_tensor];
    if (!g || a.control->skip) return;
    const float coef = a.control->coef;
    const GeomaeAdamwTensor row = a.rows[t];
    const MaScalars s = a.scalars[t];
    if (row.dtype == GEOMAE_DTYPE_F32) ma_update<float, false, BITS>(row, static_cast<const float*>(g), start, s, coef);
    else if (row.dtype == GEOMAE_DTYPE_BF16) {
        if (row.master) ma_update<uint16_t, true, BITS>(row, static_cast<const uint16_t*>(g), start, s, coef);
        else ma_update<uint16_t, false, BITS>(row, static_cast<const uint16_t*>(g), start, s, coef);
    } else {
        if (row.master) ma_update<_Float16, true, BITS>(row, static_cast<const _Float16*>(g), start, s, coef);
        else ma_update<_Float16, false, BITS>(row, static_cast<const _Float16*>(g), start, s, coef);
    }
}

// ------------------------------------------------------------------------------------------------ codes -> values
__global__ __launch_bounds__(256) void adamw_moments8_kernel(const uint32_t* m, const uint8_t* me, const uint32_t* r, const uint8_t* re,
                                                            int64_t words, uint2* m_out, uint2* r_out) {
    auto put = [](uint2* out, int64_t i, const float (&x)[kMaVec]) {
        uint32_t h[kMaVec];
#pragma unroll
        for (int k = 0; k < kMaVec; ++k) h[k] = ma_narrow<uint16_t>(x[k]);
        out[i] = make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
    };
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) {
        float x[kMaVec];
        ma_value_signed(m[i], ma_unscale(me[i >> 3]), x);
        put(m_out, i, x);
        ma_value_root(r[i], ma_unscale(re[i >> 3]), x);
        put(r_out, i, x);
    }
}

struct MaWorkspace { double* partial; MaScalars* scalars; MaControl* control; int64_t bytes; };
static MaWorkspace ma_workspace(void* base, int32_t num_tensors) {
    const int64_t slices = (num_tensors + kMaTensors - 1) / kMaTensors;
    char* p = static_cast<char*>(base);
    MaWorkspace w;
    w.partial = reinterpret_cast<double*>(p);
    const int64_t scal = slices * kMaNormGrid * (int64_t)sizeof(double);
    w.scalars = reinterpret_cast<MaScalars*>(p + scal);
    const int64_t ctl = scal + (int64_t)num_tensors * (int64_t)sizeof(MaScalars);
    w.control = reinterpret_cast<MaControl*>(p + ctl);
    w.bytes = ctl + 256;
    return w;
}

}  // namespace geomae

using namespace geomae;

extern "C" int32_t geomae_multi_adamw_chunk(void) { return kMaChunk; }

extern "C" int64_t geomae_multi_adamw_workspace_bytes(int32_t num_tensors) {
    return num_tensors < 0 ? -1 : ma_workspace(nullptr, num_tensors).bytes;
}

extern "C" int geomae_multi_adamw_step(const GeomaeAdamwTensor* table, const int32_t* chunks, const int64_t* first_chunk,
                                       int32_t num_tensors, const void* const* grads, const int32_t* hyper_of,
                                       const GeomaeAdamwHyper* hypers, int32_t num_hypers, int32_t state_bits, double max_norm,
                                       double grad_scale, const float* grad_scale_ptr, int32_t skip_nonfinite, uint32_t seed,
                                       float* grad_norm_out, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
    GEOMAE_REQUIRE(num_tensors >= 0, "multi_adamw_step: negative tensor count");
    if (num_tensors == 0) return GEOMAE_OK;
    GEOMAE_REQUIRE(table && chunks && first_chunk && grads && hyper_of && hypers && num_hypers > 0, "multi_adamw_step: null argument");
    GEOMAE_REQUIRE(state_bits == 32 || state_bits == 8, "multi_adamw_step: state_bits must be 8 or 32, got %d", state_bits);
    const MaWorkspace w = ma_workspace(workspace, num_tensors);
    if (!workspace || workspace_bytes < w.bytes) {
        set_error("multi_adamw_step: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)w.bytes);
        return GEOMAE_ERR_WORKSPACE;
    }
    for (int32_t t = 0; t < num_tensors; ++t) {
        GEOMAE_REQUIRE(first_chunk[t + 1] >= first_chunk[t] && first_chunk[t + 1] <= INT32_MAX, "multi_adamw_step: bad chunk table");
        GEOMAE_REQUIRE(!grads[t] || (hyper_of[t] >= 0 && hyper_of[t] < num_hypers), "multi_adamw_step: hyper-parameter set %d of tensor %d out of range",
                       (int)hyper_of[t], (int)t);
    }
    const bool norm = max_norm > 0.0 || skip_nonfinite || grad_norm_out;
    int32_t num_partial = 0;
    if (norm) {
        MaNormArgs a;
        a.rows = table; a.chunks = chunks;
        for (int32_t t0 = 0; t0 < num_tensors; t0 += kMaTensors) {
            const int32_t t1 = t0 + kMaTensors < num_tensors ? t0 + kMaTensors : num_tensors;
            a.first_tensor = t0; a.first_chunk = (int32_t)first_chunk[t0]; a.num_chunks = (int32_t)(first_chunk[t1] - first_chunk[t0]);
            if (a.num_chunks == 0) continue;
            for (int32_t t = t0; t < t1; ++t) a.grads[t - t0] = grads[t];
            const int grid = a.num_chunks < kMaNormGrid ? a.num_chunks : kMaNormGrid;
            a.partial = w.partial + num_partial;
            hipLaunchKernelGGL(multi_sumsq_kernel, dim3(grid), dim3(kMaThreads), 0, stream, a);
            num_partial += grid;
        }
        if (int rc = check_launch("multi_sumsq_kernel")) return rc;
    }
    MaPrepareArgs pa;
    pa.rows = table; pa.partial = w.partial; pa.scalars = w.scalars; pa.control = w.control;
    pa.grad_norm = grad_norm_out; pa.grad_scale_ptr = grad_scale_ptr; pa.grad_scale = grad_scale; pa.max_norm = max_norm;
    pa.want_norm = norm; pa.num_partial = num_partial; pa.skip_nonfinite = skip_nonfinite; pa.seed = seed;
    MaStepArgs sa;
    sa.rows = table; sa.chunks = chunks; sa.scalars = w.scalars; sa.control = w.control;
    for (int32_t t0 = 0; t0 < num_tensors;) {        // slices of at most kMaTensors tensors and kMaHypers distinct hyper-parameter sets
        int32_t slot_of[kMaHypers], used = 0, t = t0;
        for (; t < num_tensors && t - t0 < kMaTensors; ++t) {
            sa.grads[t - t0] = grads[t];
            pa.hyper_of[t - t0] = 255;
            if (!grads[t]) continue;
            int32_t k = 0;
            while (k < used && slot_of[k] != hyper_of[t]) ++k;
            if (k == used) {
                if (used == kMaHypers) break;
                slot_of[used] = hyper_of[t];
                pa.hypers[used++] = hypers[hyper_of[t]];
            }
            pa.hyper_of[t - t0] = (uint8_t)k;
        }
        pa.first_tensor = t0; pa.num_tensors = t - t0;
        sa.first_tensor = t0; sa.first_chunk = (int32_t)first_chunk[t0];
        const int64_t num_chunks = first_chunk[t] - first_chunk[t0];
        hipLaunchKernelGGL(multi_prepare_kernel, dim3(1), dim3(kMaThreads), 0, stream, pa);
        if (num_chunks > 0) {
            if (state_bits == 32) hipLaunchKernelGGL(multi_adamw_kernel<32>, dim3((uint32_t)num_chunks), dim3(kMaThreads), 0, stream, sa);
            else hipLaunchKernelGGL(multi_adamw_kernel<8>, dim3((uint32_t)num_chunks), dim3(kMaThreads), 0, stream, sa);
        }
        t0 = t;
    }
    return check_launch("multi_adamw_kernel");
}

extern "C" int geomae_adamw_moments8(const uint8_t* exp_avg, const uint8_t* exp_avg_exponent, const uint8_t* exp_avg_sq,
                                     const uint8_t* exp_avg_sq_exponent, int64_t num_elems, void* exp_avg_out, void* root_out,
                                     hipStream_t stream) {
    GEOMAE_REQUIRE(num_elems >= 0 && num_elems % 32 == 0, "adamw_moments8: a multiple of 32 elements is wanted, got %lld", (long long)num_elems);
    if (num_elems == 0) return GEOMAE_OK;
    GEOMAE_REQUIRE(exp_avg && exp_avg_exponent && exp_avg_sq && exp_avg_sq_exponent && exp_avg_out && root_out, "adamw_moments8: null argument");
    GEOMAE_REQUIRE((((uintptr_t)exp_avg | (uintptr_t)exp_avg_sq) & 3) == 0 && (((uintptr_t)exp_avg_out | (uintptr_t)root_out) & 7) == 0,
                   "adamw_moments8: codes must be 4-byte, outputs 8-byte aligned");
    const int64_t words = num_elems / 4;
    hipLaunchKernelGGL(adamw_moments8_kernel, dim3(stream_grid(words, 256)), dim3(256), 0, stream, reinterpret_cast<const uint32_t*>(exp_avg),
                       exp_avg_exponent, reinterpret_cast<const uint32_t*>(exp_avg_sq), exp_avg_sq_exponent, words,
                       static_cast<uint2*>(exp_avg_out), static_cast<uint2*>(root_out));
    return check_launch("adamw_moments8_kernel");
}
