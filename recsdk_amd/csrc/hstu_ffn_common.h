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

typedef unsigned int __attribute__((aligned(1))) ffn_u1_any;
typedef unsigned short __attribute__((aligned(1))) ffn_h1_any;

// the first min(n, 8) of 8 consecutive elements, zero behind them: as they lie in memory, so that a row can be under way while
// another is worked on, and as floats.  The rows are streamed: nontemporal.  The end of a row goes in pieces of four, two and
// one elements, in registers
template <typename T> struct Raw8 { ffn_u4 q[8 * sizeof(T) / 16]; };
template <typename T> __device__ __forceinline__ Raw8<T> load8_raw(const T* p, int n) {
    Raw8<T> r;
    if (n >= 8) {
#pragma unroll
        for (int q = 0; q < (int)(8 * sizeof(T) / 16); q++) r.q[q] = __builtin_nontemporal_load(reinterpret_cast<const ffn_u4_any*>(p) + q);
        return r;
    }
#pragma unroll
    for (int q = 0; q < (int)(8 * sizeof(T) / 16); q++) r.q[q] = ffn_u4{0u, 0u, 0u, 0u};
    if (n <= 0) return r;
    const bool four = n & 4, two = n & 2;
    if constexpr (sizeof(T) == 2) {
        unsigned w0 = 0, w1 = 0, w2 = 0, w3 = 0;
        if (four) {
            const ffn_u2 x = *reinterpret_cast<const ffn_u2_any*>(p);
            w0 = x[0];
            w1 = x[1];
        }
        if (two) {
            const unsigned x = *reinterpret_cast<const ffn_u1_any*>(p + (four ? 4 : 0));
            w0 = four ? w0 : x;
            w2 = four ? x : 0u;
        }
        if (n & 1) {
            const unsigned x = *reinterpret_cast<const ffn_h1_any*>(p + (four ? 4 : 0) + (two ? 2 : 0));
            w0 = !four && !two ? x : w0;
            w1 = !four && two ? x : w1;
            w2 = four && !two ? x : w2;
            w3 = four && two ? x : w3;
        }
        r.q[0] = ffn_u4{w0, w1, w2, w3};
    } else {
        ffn_u4 lo = {0u, 0u, 0u, 0u}, hi = lo;
        if (four) lo = *reinterpret_cast<const ffn_u4_any*>(p);
        if (two) {
            const ffn_u2 x = *reinterpret_cast<const ffn_u2_any*>(p + (four ? 4 : 0));
            if (four) { hi[0] = x[0]; hi[1] = x[1]; }
            else { lo[0] = x[0]; lo[1] = x[1]; }
        }
        if (n & 1) {
            const unsigned x = *reinterpret_cast<const ffn_u1_any*>(p + (four ? 4 : 0) + (two ? 2 : 0));
            if (four) { hi[0] = two ? hi[0] : x; hi[2] = two ? x : 0u; }
            else { lo[0] = two ? lo[0] : x; lo[2] = two ? x : 0u; }
        }
        r.q[0] = lo;
        r.q[sizeof(T) == 4 ? 1 : 0] = hi;
    }
    return r;
}
template <typename T> __device__ __forceinline__ void to_floats(const Raw8<T>& r, float* v) {
    T t[8];
    __builtin_memcpy(t, &r, sizeof(r));
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = to_float(t[k]);
}
template <typename T> __device__ __forceinline__ void load8_any(const T* p, int n, float* v) { to_floats(load8_raw(p, n), v); }
template <bool STREAM = true, typename T> __device__ __forceinline__ void store8_any(T* p, int n, const float* v) {
    T t[8];
#pragma unroll
    for (int k = 0; k < 8; k++) t[k] = from_float<T>(v[k]);
    Raw8<T> r;
    __builtin_memcpy(&r, t, sizeof(r));
    if (n >= 8) {
#pragma unroll
        for (int q = 0; q < (int)(8 * sizeof(T) / 16); q++) {
            if (STREAM) __builtin_nontemporal_store(r.q[q], reinterpret_cast<ffn_u4_any*>(p) + q);
            else *(reinterpret_cast<ffn_u4_any*>(p) + q) = r.q[q];
        }
        return;
    }
    if (n <= 0) return;
    const bool four = n & 4, two = n & 2;
    if constexpr (sizeof(T) == 2) {
        const ffn_u4 w = r.q[0];
        if (four) *reinterpret_cast<ffn_u2_any*>(p) = ffn_u2{w[0], w[1]};
        if (two) *reinterpret_cast<ffn_u1_any*>(p + (four ? 4 : 0)) = four ? w[2] : w[0];
        if (n & 1) *reinterpret_cast<ffn_h1_any*>(p + (four ? 4 : 0) + (two ? 2 : 0)) = (unsigned short)(four ? (two ? w[3] : w[2]) : (two ? w[1] : w[0]));
    } else {
        const ffn_u4 lo = r.q[0], hi = r.q[sizeof(T) == 4 ? 1 : 0];
        if (four) *reinterpret_cast<ffn_u4_any*>(p) = lo;
        if (two) *reinterpret_cast<ffn_u2_any*>(p + (four ? 4 : 0)) = four ? ffn_u2{hi[0], hi[1]} : ffn_u2{lo[0], lo[1]};
        if (n & 1) *reinterpret_cast<ffn_u1_any*>(p + (four ? 4 : 0) + (two ? 2 : 0)) = four ? (two ? hi[2] : hi[0]) : (two ? lo[2] : lo[0]);
    }
}

// ---- the gated product's activation ------------------------------------------------------------------------------------
// silu(z) = z / (1 + e^-z); e^-z by the base-2 exponential instruction: the rounding of its argument costs |z| 2^-24 relative
__device__ __forceinline__ float sigmoid_of(float z) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * z)); }
// N values at a time: one branch, and the exponentials and reciprocals of all of them under way together
template <int N> __device__ __forceinline__ void act_of(const float* z, int act, float* a) {
    if (act == HSTU_ACT_SILU) {
#pragma unroll
        for (int k = 0; k < N; k++) a[k] = z[k] * sigmoid_of(z[k]);
    } else {
#pragma unroll
        for (int k = 0; k < N; k++) a[k] = 0.5f * z[k] * erfcf(-0.70710678f * z[k]);
    }
}
// act and its derivative
template <int N> __device__ __forceinline__ void act_and_grad(const float* z, int act, float* a, float* d) {
    if (act == HSTU_ACT_SILU) {
#pragma unroll
        for (int k = 0; k < N; k++) {
            const float s = sigmoid_of(z[k]);
            a[k] = z[k] * s;
            d[k] = __builtin_fmaf(a[k], 1.0f - s, s);   // s (1 + z (1 - s))
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; k++) {
            const float phi = 0.5f * erfcf(-0.70710678f * z[k]);
            a[k] = z[k] * phi;
            d[k] = phi + z[k] * 0.39894228f * __builtin_amdgcn_exp2f(-0.72134752f * z[k] * z[k]);
            __builtin_amdgcn_sched_barrier(0);   // (one erfc at a time: side by side they cost the row work its occupancy)
        }
    }
}

// ---- z in 24 bits: the upper 16 bits of an fp32 value in one plane, the next 8 in another -------------------------------------
// (the rest is cut off: 2^-15 of the value at most, and a NaN of the arithmetic stays one)
__device__ __forceinline__ unsigned upper_pair(float a, float b) { return __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, b), __builtin_bit_cast(unsigned, a), 0x07060302u); }
__device__ __forceinline__ unsigned lower_quad(float a, float b, float c, float d) {
    const unsigned lo = __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, b), __builtin_bit_cast(unsigned, a), 0x0c0c0501u);
    const unsigned hi = __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, d), __builtin_bit_cast(unsigned, c), 0x05010c0cu);
    return lo | hi;
}
// 8 values from 8 upper parts and 8 lower ones
__device__ __forceinline__ void join24(const ffn_u4& up, const ffn_u2& low, float* v) {
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const unsigned u = k & 1 ? up[k >> 1] & 0xffff0000u : up[k >> 1] << 16, l = (low[k >> 2] >> (8 * (k & 3))) & 0xffu;
        v[k] = __builtin_bit_cast(float, u | (l << 8));
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

// the first min(n, 8) of 8 consecutive codes of one group with its exponent byte, and the values they stand for, brought into
// [-top, top] (zero codes behind them)
struct Codes8 { ffn_u2 q; int byte; };
__device__ __forceinline__ Codes8 codes8_raw(const uint8_t* p, int n, int byte) {
    Codes8 r = {{0u, 0u}, byte};
    if (n >= 8) r.q = __builtin_nontemporal_load(reinterpret_cast<const ffn_u2_any*>(p));
    else if (n > 0) {
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (k < n) r.q[k >> 2] |= (unsigned)p[k] << (8 * (k & 3));
    }
    return r;
}
__device__ __forceinline__ void code_values(const Codes8& c, float top, float* v) {
    const float scale = pack8_scale(c.byte);
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.q[h], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.q[h], true);
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
