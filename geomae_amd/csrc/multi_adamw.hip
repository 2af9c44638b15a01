// AdamW over many tensors where they lie (geomae_amd.optim.MultiTensorAdamW), moments in 32 or in 8 bits.
//
//   g' = g * grad_scale * min(1, max_norm / (norm + 1e-6)),   norm = grad_scale * sqrt(sum over all tensors of g^2)
//   p *= 1 - lr wd ;  m += (1 - b1) (g' - m) ;  v = b2 v + (1 - b2) g'^2
//   p -= lr / (1 - b1^s) * m / (sqrt(v) / sqrt(1 - b2^s) + eps)               s = steps this tensor has taken, kept on the device
//
// all in fp32 (the norm's sums in fp64: its rounding would reach every element), operation by operation as
// torch.optim.AdamW rounds it.
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
// call's own stands between two steps or inside a captured graph.  Measured on two cards: 40 M fp32 elements, 32-bit moments 200 and 215 us
// (1.12 GB, 5.6 and 5.2 TB/s, as a copy of as many bytes); 48 M bf16 elements with masters, 8-bit moments 163 us (0.77 GB, 4.7 TB/s; VALU is
// not far behind) and 32 us for the norm before it (96 MB, 3.0 TB/s).
#include "common.h"
#include "../../include/geomae_hip.h"
#include <math.h>

namespace geomae {

constexpr int kMaThreads = 256, kMaVec = 4, kMaIters = 4;
constexpr int kMaChunk = kMaThreads * kMaVec * kMaIters;             // elements of a workgroup
constexpr int kMaTensors = 384;                                      // gradient addresses of a launch (3 of its 4 KB of arguments)
constexpr int kMaHypers = 8;                                         // distinct hyper-parameter sets of a launch
constexpr int kMaNormGrid = 1024;                                    // workgroups (= partial sums) of a norm, over all launches

struct MaScalars { float decay, w1, b2, omb2, bc2_sqrt, inv_bc2_sqrt, eps, step_size; uint32_t key; };

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
template <> __device__ __forceinline__ uint16_t ma_narrow<uint16_t>(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }

// kMaVec elements at offset o of a chunk that has `left` of them; FULL: all of the workgroup's
template <bool FULL, typename T>
__device__ __forceinline__ void ma_load(const T* p, int o, int left, float (&out)[kMaVec]) {
    if (FULL || o + kMaVec <= left) {
        const MaPack<T, kMaVec> w = *reinterpret_cast<const MaPack<T, kMaVec>*>(p + o);
#pragma unroll
        for (int i = 0; i < kMaVec; ++i) out[i] = ma_float<T>(w.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < kMaVec; ++i) out[i] = o + i < left ? ma_float<T>(p[o + i]) : 0.f;
    }
}
template <bool FULL, typename T>
__device__ __forceinline__ void ma_store(T* p, int o, int left, const float (&x)[kMaVec]) {
    if (FULL || o + kMaVec <= left) {
        MaPack<T, kMaVec> w;
#pragma unroll
        for (int i = 0; i < kMaVec; ++i) w.v[i] = ma_narrow<T>(x[i]);
        *reinterpret_cast<MaPack<T, kMaVec>*>(p + o) = w;
    } else {
#pragma unroll
        for (int i = 0; i < kMaVec; ++i)
            if (o + i < left) p[o + i] = ma_narrow<T>(x[i]);
    }
}

// ------------------------------------------------------------------------------------------------ 8-bit moments
// A magnitude in units of its block's scale, times 2^-120, has the codes' exponent field and digits at the top of its fp32 bits,
// the even spacing below 2^-6 as fp32's own subnormal numbers.  Decoding is a shift and an exponent, encoding a shift too: the
// draw, (2 u + 1) in units of 2^-17 of a step, is added below the code's last digit and carries into it.  (The largest code and
// above, infinity and NaN end at or over the NaN code and are clamped to it.)
__device__ __forceinline__ uint32_t ma_magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }
// largest finite magnitude (its bits) of the 8 lanes x 4 elements of a block
__device__ __forceinline__ uint32_t ma_block_max(const float (&x)[kMaVec]) {
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < kMaVec; ++i) a = max(a, ma_magnitude(x[i]));
    if (__builtin_expect(a >= 0x7f800000u, 0)) {
        a = 0;
#pragma unroll
        for (int i = 0; i < kMaVec; ++i) a = max(a, ma_magnitude(x[i]) < 0x7f800000u ? ma_magnitude(x[i]) : 0u);
    }
    a = max(a, (uint32_t)dpp_mov<kDppXor1>((int)a));
    a = max(a, (uint32_t)dpp_mov<kDppXor2>((int)a));
    return max(a, (uint32_t)dpp_mov<kDppHalfMirror>((int)a));
}
template <bool SIGNED>
__device__ __forceinline__ int ma_exponent(uint32_t largest) {       // + 0x1fffff / 0x0fffff: carries above 1.75 / 1.875
    const int e = (int)((largest + (SIGNED ? 0x1fffffu : 0x0fffffu)) >> 23);
    return e < 16 ? 16 : (e > 254 ? 254 : e);
}
__device__ __forceinline__ float ma_scale(int e) { return __uint_as_float((uint32_t)(262 - e) << 23); }     // 2^(135 - E)

__device__ __forceinline__ uint32_t ma_code_signed(const float (&x)[kMaVec], float scale, const uint32_t (&draw)[kMaVec]) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < kMaVec; ++i) {
        const uint32_t z = __float_as_uint(fabsf(x[i]) * scale * 0x1p-120f);
        const uint32_t c = min((z + (((draw[i] & 0xffffu) << 4) | 8u)) >> 20, 0x7fu);
        w |= (c | ((__float_as_uint(x[i]) >> 24) & 0x80u)) << (8 * i);
    }
    return w;
}
__device__ __forceinline__ uint32_t ma_code_root(const float (&x)[kMaVec], float scale, const uint32_t (&draw)[kMaVec]) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < kMaVec; ++i) {
        const uint32_t z = __float_as_uint(fabsf(x[i]) * scale * 0x1p-120f);               // (a NaN may have a sign)
        const uint32_t c = min(max((z + ((draw[i] >> 13 & ~7u) | 4u)) >> 19, min(__float_as_uint(x[i]), 1u)), 255u);
        w |= c << (8 * i);
    }
    return w;
}
__device__ __forceinline__ void ma_value_signed(uint32_t w, int e, float (&out)[kMaVec]) {
    const float unscale = __uint_as_float((uint32_t)(e - 8) << 23);  // 2^(E - 135)
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    out[0] = a[0] * unscale; out[1] = a[1] * unscale; out[2] = b[0] * unscale; out[3] = b[1] * unscale;
}
__device__ __forceinline__ void ma_value_root(uint32_t w, int e, float (&out)[kMaVec]) {
#pragma unroll
    for (int i = 0; i < kMaVec; ++i) out[i] = ldexpf(__uint_as_float(((w >> (8 * i)) & 255u) << 19), e - 15);
    if (__builtin_expect((((w & 0x7f7f7f7fu) + 0x01010101u) & w & 0x80808080u) != 0, 0)) {
#pragma unroll
        for (int i = 0; i < kMaVec; ++i)
            if (((w >> (8 * i)) & 255u) == 255u) out[i] = NAN;
    }
}

// ------------------------------------------------------------------------------------------------ norm, per-tensor scalars
template <bool FULL, typename T>
__device__ __forceinline__ double ma_sumsq(const T* g, int left) {
    double acc = 0.0;
    float x[kMaIters][kMaVec];
#pragma unroll
    for (int it = 0; it < kMaIters; ++it) ma_load<FULL, T>(g, (it * kMaThreads + (int)threadIdx.x) * kMaVec, left, x[it]);
#pragma unroll
    for (int it = 0; it < kMaIters; ++it)
#pragma unroll
        for (int i = 0; i < kMaVec; ++i) acc = fma((double)x[it][i], (double)x[it][i], acc);
    return acc;
}
template <typename T>
__device__ __forceinline__ double ma_sumsq(const void* g, int64_t start, int64_t n) {
    const T* p = static_cast<const T*>(g) + start;
    return n - start >= kMaChunk ? ma_sumsq<true, T>(p, kMaChunk) : ma_sumsq<false, T>(p, (int)(n - start));
}

// the sum of squares of all gradients from its partial sums, in a fixed order, in every thread
constexpr int kMaHeld = 4;              // partial sums that a thread loads ahead
__device__ __forceinline__ void ma_load_partials(const double* partial, int count, double (&held)[kMaHeld]) {
#pragma unroll
    for (int k = 0; k < kMaHeld; ++k) {
        const int i = k * kMaThreads + (int)threadIdx.x;
        held[k] = i < count ? partial[i] : 0.0;
    }
}
__device__ __forceinline__ double ma_sum_partials(const double* partial, int count, const double (&held)[kMaHeld]) {
    __shared__ double red[kMaThreads / kWave];
    double acc = 0.0;
#pragma unroll
    for (int k = 0; k < kMaHeld; ++k) acc += held[k];
    for (int i = kMaHeld * kMaThreads + (int)threadIdx.x; i < count; i += kMaThreads) acc += partial[i];
    acc = wave_sum(acc);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
    __syncthreads();
    return red[0] + red[1] + red[2] + red[3];
}

// the factor of the gradients: scale and clipping
struct MaFactor {
    const double* partial;              // of the norm
    int32_t num_partial, skip_nonfinite;
    double grad_scale;
    const float* grad_scale_ptr;
    float max_norm;
    float* grad_norm;                   // of the first launch: receives the norm
};
// false: the step is skipped
__device__ __forceinline__ bool ma_factor(const MaFactor& f, const double (&held)[kMaHeld], float& coef) {
    const float scale = f.grad_scale_ptr ? (float)((double)*f.grad_scale_ptr * f.grad_scale) : (float)f.grad_scale;
    coef = scale;
    if (f.num_partial == 0) return true;
    const float norm = (float)(sqrt(ma_sum_partials(f.partial, f.num_partial, held)) * fabs((double)scale));
    if (f.grad_norm && blockIdx.x == 0 && threadIdx.x == 0) *f.grad_norm = norm;
    if (f.max_norm > 0.f && f.max_norm < INFINITY) {
        const float c = f.max_norm / (norm + 1e-6f);
        coef *= c > 1.0f ? 1.0f : c;                                 // NaN stays NaN
    }
    return !(f.skip_nonfinite && !(norm < INFINITY));
}

struct MaPrepareArgs {
    const GeomaeAdamwTensor* rows;
    const int32_t* chunks;              // [num chunks][2] = (tensor, chunk of that tensor)
    MaScalars* scalars;
    double* partial;                    // one per norm workgroup of this launch
    MaFactor factor;                    // skip_nonfinite: decides over the step (no partial sums: nothing to decide yet)
    float* grad_norm;                   // set where there is no element at all: 0
    int32_t first_tensor, num_tensors, first_chunk, num_chunks, with_scalars;
    uint32_t seed;
    GeomaeAdamwHyper hypers[kMaHypers];
    const void* grads[kMaTensors];
    uint8_t hyper_of[kMaTensors];       // 255: no gradient, the tensor is left as it is
};

// what each tensor's update needs of its own step count, which it advances
__device__ __forceinline__ void ma_tensor_scalars(const MaPrepareArgs& a) {
    double held[kMaHeld];
    float coef;
    ma_load_partials(a.factor.partial, a.factor.num_partial, held);
    if (!ma_factor(a.factor, held, coef)) return;
    if (a.grad_norm && threadIdx.x == 0) *a.grad_norm = 0.f;
    for (int t = threadIdx.x; t < a.num_tensors; t += kMaThreads) {
        if (a.hyper_of[t] == 255) continue;
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
        s.inv_bc2_sqrt = (float)(1.0 / (double)s.bc2_sqrt);
        s.eps = (float)h.eps;
        s.step_size = (float)(lr / bc1);
        s.key = ma_mix(ma_mix(a.seed + 0x9E3779B9u * (uint32_t)row.index) ^ (uint32_t)step);
        a.scalars[a.first_tensor + t] = s;
    }
}

// Workgroup 0: the scalars (two powers in fp64 per tensor: started first, hidden behind the others).  The rest: partial sums of
// the squares, the next chunk's table entries loaded ahead of this chunk's data (three dependent loads a chunk otherwise).  The
// update's workgroups add the partial sums themselves, while their own data is on its way: a last workgroup that collects
// them here has to order its reads behind the others' writes, and the cache write-back of that, once per workgroup, made this
// launch six times as long (48 M elements: 269 us against 43).
__global__ __launch_bounds__(kMaThreads) void multi_prepare_kernel(MaPrepareArgs a) {
    if (a.with_scalars && blockIdx.x == 0) {
        ma_tensor_scalars(a);
        return;
    }
    __shared__ double red[kMaThreads / kWave];
    const int blocks = gridDim.x - a.with_scalars, block = blockIdx.x - a.with_scalars;
    double acc = 0.0;
    const int2* chunks = reinterpret_cast<const int2*>(a.chunks) + a.first_chunk;
    int2 at = chunks[block];
    int64_t n = a.rows[at.x].numel;
    int dtype = a.rows[at.x].dtype;
    for (int c = block; c < a.num_chunks; c += blocks) {
        const void* g = a.grads[at.x - a.first_tensor];
        const int64_t start = (int64_t)at.y * kMaChunk, left = n;
        const int now = dtype;
        if (c + blocks < a.num_chunks) {
            at = chunks[c + blocks];
            n = a.rows[at.x].numel;
            dtype = a.rows[at.x].dtype;
        }
        if (!g) continue;
        if (now == GEOMAE_DTYPE_F32) acc += ma_sumsq<float>(g, start, left);
        else if (now == GEOMAE_DTYPE_BF16) acc += ma_sumsq<uint16_t>(g, start, left);
        else acc += ma_sumsq<_Float16>(g, start, left);
    }
    acc = wave_sum(acc);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
    __syncthreads();
    if (threadIdx.x == 0) a.partial[block] = red[0] + red[1] + red[2] + red[3];
}

// ------------------------------------------------------------------------------------------------ update
struct MaStepArgs {
    const GeomaeAdamwTensor* rows;
    const int32_t* chunks;
    const MaScalars* scalars;
    MaFactor factor;
    int32_t first_tensor, first_chunk;
    const void* grads[kMaTensors];
};

// m / (sqrt(v) / c + eps) of four elements, operation by operation as torch.optim.AdamW rounds it; r receives the roots.
__device__ __forceinline__ void ma_quotients(const float (&m)[kMaVec], const float (&v)[kMaVec], const MaScalars& s, float (&r)[kMaVec], float (&q)[kMaVec]) {
#pragma unroll
    for (int i = 0; i < kMaVec; ++i) {
        r[i] = sqrtf(v[i]);                                            // (correctly rounded; __fsqrt_rn is good to an ulp)
        q[i] = __fdiv_rn(m[i], __fadd_rn(__fdiv_rn(r[i], s.bc2_sqrt), s.eps));
    }
}
// The same from the hardware's 1-ulp reciprocals, each result corrected by its remainder, which a fused multiply-add has exactly: within
// 0.5000003 units of the last place, which is the rounded value but for one in a million.  For 8-bit moments, whose step moves half the
// bytes of a 32-bit one: the update of 48 M bf16 elements with masters takes about 160 us, with the above in its place 175 and more, with
// uncorrected 1-ulp results 148.  v is 0 or in [2^-96, 2^96), |m| 0 or in [2^-100, 2^27), eps in [2^-100, 2^100]: nothing over- or
// underflows, no remainder either.
__device__ __forceinline__ void ma_quotients_in_range(const float (&m)[kMaVec], const float (&v)[kMaVec], const MaScalars& s, float (&r)[kMaVec],
                                                      float (&q)[kMaVec]) {
#pragma unroll
    for (int i = 0; i < kMaVec; ++i) {
        const float y = __builtin_amdgcn_rsqf(fmaxf(v[i], 0x1p-96f)), r0 = v[i] * y;
        r[i] = fmaf(fmaf(-r0, r0, v[i]), 0.5f * y, r0);
        const float h0 = r[i] * s.inv_bc2_sqrt, denom = fmaf(fmaf(-h0, s.bc2_sqrt, r[i]), s.inv_bc2_sqrt, h0) + s.eps;
        const float inv = __builtin_amdgcn_rcpf(denom), q0 = m[i] * inv;
        q[i] = fmaf(fmaf(-q0, denom, m[i]), inv, q0);
    }
}
__device__ __forceinline__ bool ma_in_range(const float (&m)[kMaVec], const float (&v)[kMaVec], const MaScalars& s) {
    constexpr uint32_t kLow = 31u << 23, kHigh = 223u << 23, kLowM = 27u << 24;      // 2^-96, 2^96; 2^-100 without the sign
    uint32_t least = ~0u, most = 0, least_m = ~0u;                     // (least: of the bits less one, zero is the largest)
    float most_m = 0.f;
#pragma unroll
    for (int i = 0; i < kMaVec; ++i) {
        least = min(least, __float_as_uint(v[i]) - 1u);
        most = max(most, __float_as_uint(v[i]));
        least_m = min(least_m, (__float_as_uint(m[i]) << 1) - 1u);
        most_m = fmaxf(most_m, fabsf(m[i]));                           // (NaN stays NaN either way)
    }
    return least >= kLow - 1u && most < kHigh && least_m >= kLowM - 1u && most_m < 0x1p27f && s.eps >= 0x1p-100f && s.eps <= 0x1p100f;
}

template <typename T, bool MASTER, int BITS, bool FULL>
__device__ __forceinline__ void ma_update(const GeomaeAdamwTensor& row, const T* g, int64_t start, int left, const MaScalars& s, const MaFactor& factor) {
    const int padded = (left + 31) & ~31;                            // the moments' and masters' own length
    T* param = static_cast<T*>(row.param) + start;
    float* master = MASTER ? row.master + start : nullptr;
    float *m32 = static_cast<float*>(row.exp_avg) + start, *v32 = static_cast<float*>(row.exp_avg_sq) + start;
    uint8_t *m8 = static_cast<uint8_t*>(row.exp_avg) + start, *r8 = static_cast<uint8_t*>(row.exp_avg_sq) + start;
    uint8_t *me8 = row.exp_avg_exponent + (start >> 5), *re8 = row.exp_avg_sq_exponent + (start >> 5);
    float gv[kMaIters][kMaVec], pv[kMaIters][kMaVec], mv[kMaIters][kMaVec], vv[kMaIters][kMaVec];
    uint32_t mw[kMaIters], rw[kMaIters];
    int me[kMaIters], re[kMaIters];
    double held[kMaHeld];
    ma_load_partials(factor.partial, factor.num_partial, held);      // (first: loads complete in order)
#pragma unroll
    for (int it = 0; it < kMaIters; ++it) {
        const int o = (it * kMaThreads + (int)threadIdx.x) * kMaVec;
        if (!FULL && o >= padded) continue;                          // whole groups of 8 lanes
        ma_load<FULL, T>(g, o, left, gv[it]);
        if constexpr (MASTER) {
            const float4 w = *reinterpret_cast<const float4*>(master + o);
            pv[it][0] = w.x; pv[it][1] = w.y; pv[it][2] = w.z; pv[it][3] = w.w;
        } else ma_load<FULL, T>(param, o, left, pv[it]);
        if constexpr (BITS == 32) {
            const float4 m = *reinterpret_cast<const float4*>(m32 + o), v = *reinterpret_cast<const float4*>(v32 + o);
            mv[it][0] = m.x; mv[it][1] = m.y; mv[it][2] = m.z; mv[it][3] = m.w;
            vv[it][0] = v.x; vv[it][1] = v.y; vv[it][2] = v.z; vv[it][3] = v.w;
        } else {
            mw[it] = *reinterpret_cast<const uint32_t*>(m8 + o);
            rw[it] = *reinterpret_cast<const uint32_t*>(r8 + o);
            me[it] = me8[o >> 5];
            re[it] = re8[o >> 5];
        }
    }
    float coef;
    if (!ma_factor(factor, held, coef)) return;
#pragma unroll
    for (int it = 0; it < kMaIters; ++it) {
        const int o = (it * kMaThreads + (int)threadIdx.x) * kMaVec;
        if (!FULL && o >= padded) continue;
        float r[kMaVec];
        if constexpr (BITS == 8) {
            ma_value_signed(mw[it], me[it], mv[it]);
            ma_value_root(rw[it], re[it], r);
#pragma unroll
            for (int i = 0; i < kMaVec; ++i) vv[it][i] = __fmul_rn(r[i], r[i]);
        }
#pragma unroll
        for (int i = 0; i < kMaVec; ++i) {
            const float x = __fmul_rn(gv[it][i], coef);
            float& m = mv[it][i];
            float& v = vv[it][i];
            const float d = __fsub_rn(x, m);
            if (BITS == 8 || s.w1 < 0.5f) m = __fadd_rn(m, __fmul_rn(s.w1, d));
            else m = __fsub_rn(x, __fmul_rn(d, __fsub_rn(1.0f, s.w1)));
            v = __fadd_rn(__fmul_rn(v, s.b2), __fmul_rn(__fmul_rn(s.omb2, x), x));
            pv[it][i] = __fmul_rn(pv[it][i], s.decay);
        }
        float q[kMaVec];
        if (BITS == 8 && __builtin_expect(ma_in_range(mv[it], vv[it], s), 1)) ma_quotients_in_range(mv[it], vv[it], s, r, q);
        else ma_quotients(mv[it], vv[it], s, r, q);                     // (32 bits: HBM hides them)
#pragma unroll
        for (int i = 0; i < kMaVec; ++i) pv[it][i] = __fadd_rn(pv[it][i], __fmul_rn(-s.step_size, q[i]));
        ma_store<FULL, T>(param, o, left, pv[it]);
        if constexpr (MASTER) {
            if constexpr (!FULL) {
#pragma unroll
                for (int i = 0; i < kMaVec; ++i) pv[it][i] = o + i < left ? pv[it][i] : 0.f;         // (0 / 0 where eps is 0)
            }
            *reinterpret_cast<float4*>(master + o) = make_float4(pv[it][0], pv[it][1], pv[it][2], pv[it][3]);
        }
        if constexpr (BITS == 32) {
            *reinterpret_cast<float4*>(m32 + o) = make_float4(mv[it][0], mv[it][1], mv[it][2], mv[it][3]);
            *reinterpret_cast<float4*>(v32 + o) = make_float4(vv[it][0], vv[it][1], vv[it][2], vv[it][3]);
        } else {
            const uint32_t first = s.key + (uint32_t)start + (uint32_t)o;
            uint32_t draw[kMaVec];
#pragma unroll
            for (int i = 0; i < kMaVec; ++i) draw[i] = ma_mix(first + (uint32_t)i);
            const int em = ma_exponent<true>(ma_block_max(mv[it])), er = ma_exponent<false>(ma_block_max(r));
            *reinterpret_cast<uint32_t*>(m8 + o) = ma_code_signed(mv[it], ma_scale(em), draw);
            *reinterpret_cast<uint32_t*>(r8 + o) = ma_code_root(r, ma_scale(er), draw);
            if ((threadIdx.x & 7) == 0) {
                me8[o >> 5] = (uint8_t)em;
                re8[o >> 5] = (uint8_t)er;
            }
        }
    }
}
template <typename T, bool MASTER, int BITS>
__device__ __forceinline__ void ma_update(const GeomaeAdamwTensor& row, const void* g, int64_t start, const MaScalars& s, const MaFactor& factor) {
    const T* p = static_cast<const T*>(g) + start;
    if (row.numel - start >= kMaChunk) ma_update<T, MASTER, BITS, true>(row, p, start, kMaChunk, s, factor);
    else ma_update<T, MASTER, BITS, false>(row, p, start, (int)(row.numel - start), s, factor);
}

template <int BITS>
__global__ __launch_bounds__(kMaThreads) void multi_adamw_kernel(MaStepArgs a) {
    const int32_t* at = a.chunks + 2 * (a.first_chunk + (int64_t)blockIdx.x);
    const int t = at[0];
    const int64_t start = (int64_t)at[1] * kMaChunk;
    const void* g = a.grads[t - a.first_tensor];
    if (!g) {
        // (it may be the one that writes the norm)
        double held[kMaHeld];
        float coef;
        if (!(a.factor.grad_norm && blockIdx.x == 0)) return;
        ma_load_partials(a.factor.partial, a.factor.num_partial, held);
        ma_factor(a.factor, held, coef);
        return;
    }
    const GeomaeAdamwTensor row = a.rows[t];
    const MaScalars s = a.scalars[t];
    if (row.dtype == GEOMAE_DTYPE_F32) ma_update<float, false, BITS>(row, g, start, s, a.factor);
    else if (row.dtype == GEOMAE_DTYPE_BF16) {
        if (row.master) ma_update<uint16_t, true, BITS>(row, g, start, s, a.factor);
        else ma_update<uint16_t, false, BITS>(row, g, start, s, a.factor);
    } else {
        if (row.master) ma_update<_Float16, true, BITS>(row, g, start, s, a.factor);
        else ma_update<_Float16, false, BITS>(row, g, start, s, a.factor);
    }
}

// ------------------------------------------------------------------------------------------------ codes -> values
// HBM: 2 1/16 bytes in and 4 out per element; 48 M elements 61 us (291 MB, 4.8 TB/s).
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
        ma_value_signed(m[i], me[i >> 3], x);
        put(m_out, i, x);
        ma_value_root(r[i], re[i >> 3], x);
        put(r_out, i, x);
    }
}

static_assert(sizeof(MaPrepareArgs) <= 4096 && sizeof(MaStepArgs) <= 4096, "a launch takes 4 KB of arguments");
struct MaWorkspace { double* partial; MaScalars* scalars; int64_t bytes; };
static MaWorkspace ma_workspace(void* base, int32_t num_tensors) {
    char* p = static_cast<char*>(base);
    MaWorkspace w;
    // a launch of few tensors (one for every kMaHypers hyper-parameter sets at worst) has one norm workgroup at least
    const int64_t partial = (kMaNormGrid + (int64_t)num_tensors) * (int64_t)sizeof(double);
    w.partial = reinterpret_cast<double*>(p);
    w.scalars = reinterpret_cast<MaScalars*>(p + partial);
    w.bytes = partial + (int64_t)num_tensors * (int64_t)sizeof(MaScalars);
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
    GEOMAE_REQUIRE(table && first_chunk && grads && hyper_of && hypers && num_hypers > 0, "multi_adamw_step: null argument");
    GEOMAE_REQUIRE(chunks || first_chunk[num_tensors] == 0, "multi_adamw_step: null argument");
    GEOMAE_REQUIRE(max_norm >= 0.0, "multi_adamw_step: max_norm must not be negative");
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
    // slices of at most kMaTensors tensors and kMaHypers distinct hyper-parameter sets
    MaPrepareArgs pa;
    auto slice = [&](int32_t t0) {
        int32_t slot_of[kMaHypers], used = 0, t = t0;
        for (; t < num_tensors && t - t0 < kMaTensors; ++t) {
            pa.grads[t - t0] = grads[t];
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
        pa.first_tensor = t0;
        pa.num_tensors = t - t0;
        pa.first_chunk = (int32_t)first_chunk[t0];
        pa.num_chunks = (int32_t)(first_chunk[t] - first_chunk[t0]);
        return t;
    };
    const int64_t chunks_all = first_chunk[num_tensors];
    const bool norm = (max_norm > 0.0 || skip_nonfinite || grad_norm_out) && chunks_all > 0;
    pa.rows = table; pa.chunks = chunks; pa.scalars = w.scalars; pa.seed = seed;
    // (a norm below fp32's numbers is not "no clipping")
    const float limit = max_norm > 0.0 && (float)max_norm == 0.f ? 0x1p-149f : (float)max_norm;
    pa.factor = {w.partial, 0, skip_nonfinite, grad_scale, grad_scale_ptr, limit, nullptr};
    pa.grad_norm = chunks_all == 0 ? grad_norm_out : nullptr;
    int32_t num_partial = 0;
    // skip_nonfinite: the scalars wait for the whole norm, a launch of their own
    for (int pass = 0; pass < 2; ++pass) {
        if (pass == 1 && !(norm && skip_nonfinite)) break;
        pa.with_scalars = !(norm && skip_nonfinite) || pass == 1;
        pa.factor.num_partial = pass == 1 ? num_partial : 0;
        for (int32_t t0 = 0; t0 < num_tensors;) {
            const int32_t t1 = slice(t0);
            int grid = 0;
            if (norm && pass == 0 && pa.num_chunks > 0) {            // a share of kMaNormGrid by size
                grid = (int)((int64_t)kMaNormGrid * pa.num_chunks / chunks_all);
                grid = grid < 1 ? 1 : (grid > pa.num_chunks ? pa.num_chunks : grid);
            }
            pa.partial = w.partial + num_partial;
            num_partial += grid;
            if (grid + pa.with_scalars > 0)
                hipLaunchKernelGGL(multi_prepare_kernel, dim3(grid + pa.with_scalars), dim3(kMaThreads), 0, stream, pa);
            t0 = t1;
        }
    }
    MaStepArgs sa;
    sa.rows = table; sa.chunks = chunks; sa.scalars = w.scalars;
    sa.factor = pa.factor;
    sa.factor.num_partial = num_partial;
    sa.factor.grad_norm = grad_norm_out;
    for (int32_t t0 = 0; t0 < num_tensors;) {
        const int32_t t1 = t0 + kMaTensors < num_tensors ? t0 + kMaTensors : num_tensors;
        for (int32_t t = t0; t < t1; ++t) sa.grads[t - t0] = grads[t];
        sa.first_tensor = t0; sa.first_chunk = (int32_t)first_chunk[t0];
        const int64_t num_chunks = first_chunk[t1] - first_chunk[t0];
        if (num_chunks > 0) {
            if (state_bits == 32) hipLaunchKernelGGL(multi_adamw_kernel<32>, dim3((uint32_t)num_chunks), dim3(kMaThreads), 0, stream, sa);
            else hipLaunchKernelGGL(multi_adamw_kernel<8>, dim3((uint32_t)num_chunks), dim3(kMaThreads), 0, stream, sa);
            sa.factor.grad_norm = nullptr;
        }
        t0 = t1;
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
