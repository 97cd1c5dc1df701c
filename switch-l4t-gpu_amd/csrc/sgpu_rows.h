// sgpu_rows.h -- device helpers of the operators on rows of heads (sgpu_score.hip, sgpu_paged.hip): vector
// types, angles, sums of the wave's halves, and fp32 values as fp16 pieces.
#pragma once
#include "sgpu_device.h"

namespace {

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_a2 __attribute__((ext_vector_type(8), aligned(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) void lds_void;

// sin and cos of 2 pi u, u in turns: u is reduced to the nearest quarter turn in 64 bits (a far
// position's angle has no fp32 digits left), the rest, at most an eighth of a turn, goes through
// the Taylor series of both (first term left out below 2e-9 of 1).
__device__ __forceinline__ void sincos_turns(double u, float& sn, float& cs) {
    const double quarters = rint(4.0 * u);
    const float x = (float)((u - 0.25 * quarters) * 6.283185307179586476925), x2 = x * x;
    float s = __builtin_fmaf(x2, 2.7557319e-6f, -1.98412698e-4f);
    s = __builtin_fmaf(s, x2, 8.33333333e-3f);
    s = __builtin_fmaf(s, x2, -0.166666667f);
    s = __builtin_fmaf(s * x2, x, x);
    float c = __builtin_fmaf(x2, -2.75573192e-7f, 2.48015873e-5f);
    c = __builtin_fmaf(c, x2, -1.38888889e-3f);
    c = __builtin_fmaf(c, x2, 4.16666667e-2f);
    c = __builtin_fmaf(c, x2, -0.5f);
    c = __builtin_fmaf(c, x2, 1.0f);
    const int q = (int)(quarters - 4.0 * floor(0.25 * quarters));       // 0..3
    sn = q & 1 ? c : s;
    cs = q & 1 ? s : c;
    if (q & 2) sn = -sn;
    if (q == 1 || q == 2) cs = -cs;
}

template <typename O> __device__ __forceinline__ void put4(O* p, const float (&v)[4]);
template <> __device__ __forceinline__ void put4<float>(float* p, const float (&v)[4]) {
    *reinterpret_cast<sgpu_f32x4*>(p) = sgpu_f32x4{v[0], v[1], v[2], v[3]};
}
template <> __device__ __forceinline__ void put4<_Float16>(_Float16* p, const float (&v)[4]) {
    *reinterpret_cast<f16x4*>(p) = f16x4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
}

__device__ __forceinline__ void lds_sync() {      // the wave's own LDS writes are seen by its other lanes
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Both halves of the wave: f(lane, lane ^ 32).
__device__ __forceinline__ float half_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float pow2(int e) { return __builtin_amdgcn_ldexpf(1.0f, e); }

// The exponent e that brings values of magnitude bits m below 2^15, and the largest to 2^11 or more, as x * 2^-e:
// a multiple of 4, so that it seldom changes from tile to tile (0 for zero; -124 at least: 2^-e stays a number).
__device__ __forceinline__ int scale_of(uint32_t m) { return m ? max(((int)(m >> 23) - 138) & ~3, -124) : 0; }

// y (two values below 2^15) as two fp16 pieces of 11 bits each, rounded to nearest: off by at most
// 2^-22 of the value, or 2^-25 where that is more.
__device__ __forceinline__ void split2(float y0, float y1, f16x2& hi, f16x2& lo) {
    hi = __builtin_convertvector((f32x2{y0, y1}), f16x2);
    float minus = -1.0f;               // opaque: one v_fma_mix_f32 each, not a conversion and a subtraction
    __asm__("" : "+s"(minus));
    lo = __builtin_convertvector((f32x2{__builtin_fmaf((float)hi[0], minus, y0), __builtin_fmaf((float)hi[1], minus, y1)}), f16x2);
}

}  // namespace
