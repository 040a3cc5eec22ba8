// Row work shared by the kernels of the feed-forward half: 8 consecutive elements at any address, and fp32 column sums.
#pragma once
#include "hstu_device.h"
#include "../../include/hstu_ffn.h"

namespace hstu {

typedef __attribute__((ext_vector_type(4))) unsigned int ffn_u4;
typedef __attribute__((ext_vector_type(2))) unsigned int ffn_u2;
// 16 and 8 bytes at any address: global memory takes unaligned vector accesses, so rows of an odd width need no other path
typedef ffn_u4 __attribute__((aligned(1))) ffn_u4_any;
typedef ffn_u2 __attribute__((aligned(1))) ffn_u2_any;

// the first min(n, 8) of 8 consecutive elements, zero behind them.  The rows are streamed: nontemporal
template <typename T> __device__ __forceinline__ void load8_any(const T* p, int n, float* v) {
    if (n >= 8) {
        T t[8];
#pragma unroll
        for (int q = 0; q < (int)(8 * sizeof(T) / 16); q++) {
            const ffn_u4 x = __builtin_nontemporal_load(reinterpret_cast<const ffn_u4_any*>(p) + q);
            __builtin_memcpy(reinterpret_cast<char*>(t) + 16 * q, &x, 16);
        }
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = to_float(t[k]);
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = k < n ? to_float(p[k]) : 0.f;
    }
}
template <typename T> __device__ __forceinline__ void store8_any(T* p, int n, const float* v) {
    T t[8];
#pragma unroll
    for (int k = 0; k < 8; k++) t[k] = from_float<T>(v[k]);
    if (n >= 8) {
#pragma unroll
        for (int q = 0; q < (int)(8 * sizeof(T) / 16); q++) {
            ffn_u4 x;
            __builtin_memcpy(&x, reinterpret_cast<char*>(t) + 16 * q, 16);
            __builtin_nontemporal_store(x, reinterpret_cast<ffn_u4_any*>(p) + q);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (k < n) p[k] = t[k];
    }
}

// ---- the gated product's activation ------------------------------------------------------------------------------------
// silu(z) = z / (1 + e^-z); e^-z by the base-2 exponential instruction: the rounding of its argument costs |z| 2^-24 relative
__device__ __forceinline__ float sigmoid_of(float z) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * z)); }
__device__ __forceinline__ float act_of(float z, int act) {
    if (act == HSTU_ACT_SILU) return z * sigmoid_of(z);
    return 0.5f * z * erfcf(-0.70710678f * z);
}
// act and its derivative
__device__ __forceinline__ void act_and_grad(float z, int act, float& a, float& d) {
    if (act == HSTU_ACT_SILU) {
        const float s = sigmoid_of(z);
        a = z * s;
        d = s * (1.0f + z * (1.0f - s));
    } else {
        const float phi = 0.5f * erfcf(-0.70710678f * z);
        a = z * phi;
        d = phi + z * 0.39894228f * __builtin_amdgcn_exp2f(-0.72134752f * z * z);
    }
}

// ---- 8-bit activations ---------------------------------------------------------------------------------------------------
// exponent byte of a group whose finite values reach `top` (>= 0): 448 = 1.75 * 2^8, so E = floor(log2 top) - 8, one more
// where the mantissa is above 1.75
__device__ __forceinline__ int pack8_exponent(float top) {
    const unsigned b = __builtin_bit_cast(unsigned, top);
    const int e = (int)(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < 1 ? 1 : e;
}
__device__ __forceinline__ float pack8_scale(int byte) { return __builtin_bit_cast(float, (unsigned)byte << 23); }           // 2^E
__device__ __forceinline__ float pack8_inv_scale(int byte) { return __builtin_bit_cast(float, (unsigned)(254 - byte) << 23); } // 2^-E
__device__ __forceinline__ float pack8_finite_abs(float v) {
    const float a = __builtin_fabsf(v);
    return a < __builtin_inff() ? a : 0.f;   // NaN compares false
}
// four values to four codes; what is not finite becomes a NaN code
__device__ __forceinline__ unsigned pack8_codes(float a, float b, float c, float d, float inv) {
    const float nan = __builtin_nanf("");
    a = __builtin_fabsf(a) < __builtin_inff() ? a * inv : nan;
    b = __builtin_fabsf(b) < __builtin_inff() ? b * inv : nan;
    c = __builtin_fabsf(c) < __builtin_inff() ? c * inv : nan;
    d = __builtin_fabsf(d) < __builtin_inff() ? d * inv : nan;
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}

// the values of the first min(n, 8) of 8 consecutive codes of one group, brought into [-top, top]; zero behind them
__device__ __forceinline__ void unpack8_any(const uint8_t* p, int n, int byte, float top, float* v) {
    ffn_u2 q = {0u, 0u};
    if (n >= 8) q = __builtin_nontemporal_load(reinterpret_cast<const ffn_u2_any*>(p));
    else {
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (k < n) q[k >> 2] |= (unsigned)p[k] << (8 * (k & 3));
    }
    const float scale = pack8_scale(byte);
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[h], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[h], true);
        const float w[4] = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float x = w[k] * scale;
            v[4 * h + k] = __builtin_isnan(x) ? x : fminf(fmaxf(x, -top), top);
        }
    }
}
template <typename T> __device__ __forceinline__ constexpr float largest_finite();
template <> __device__ __forceinline__ constexpr float largest_finite<float>() { return 3.40282347e38f; }
template <> __device__ __forceinline__ constexpr float largest_finite<_Float16>() { return 65504.f; }
template <> __device__ __forceinline__ constexpr float largest_finite<__bf16>() { return 3.38953139e38f; }

// Column sums in a fixed order: sum over r < rows of partial[r, c] for c < 2 * half, the first half to out0 and the second to
// out1 (either may be NULL), rounded once to out_dtype.  Defined in hstu_norm.hip.
hipError_t launch_colsum(const float* partial, int rows, int half, void* out0, void* out1, int32_t out_dtype, hipStream_t st);

}  // namespace hstu
