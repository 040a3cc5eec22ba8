// The gated projection for few rows (single tokens, the candidates of a request): act(x Wg^T + bg) * (x Wu^T + bu) with m <= 64.
//
// The weights are read once and there is nothing to share between workgroups but a few rows of x, so nothing goes through LDS on
// the way in: a workgroup owns 16 FB columns f (their gate and their value rows), its eight waves take pieces of 128 bytes of k in
// turn, and a lane's 16-byte loads of W and x are MFMA fragments as they come (16 x 16 blocks, W as the A operand).  Rows of any
// alignment are read in place; the last piece of a row goes by elements.  The waves' fp32 sums meet in LDS and are added in order.
// Bounded by reading W: 16 FB columns a workgroup make f / 16 workgroups, and every wave has a whole piece per operand in flight.
// One row, 1024 -> 4096: 3.3 us (16.8 MB of W; 5.1 TB/s, part of it out of the cache), with 32 columns a workgroup 6.2, with the next
// piece under way 4.0.  48 rows: 7.1 to 7.7 us, in which each workgroup reads all of x.
#pragma once
#include "hstu_gemm.h"

namespace hstu {

struct RowsArgs {
    const void* x;
    const void* weight;
    const void* bias;
    void* out;
    void* z;
    uint8_t* z_aux;
    int64_t x_stride;
    int32_t m, k, f, bias_f32, act, keep;
};
constexpr int ROWS_MAX_M = 64;
constexpr int ROWS_WAVES = 8;

// 16 bytes of consecutive elements at any address, zero from element n on
template <typename T> __device__ __forceinline__ typename GM<T>::frag load_frag(const T* p, int n) {
    typedef typename GM<T>::frag frag;
    constexpr int EC = 16 / sizeof(T);
    if (n >= EC) return __builtin_bit_cast(frag, *reinterpret_cast<const gm_u4_any*>(p));
    T e[EC];
#pragma unroll
    for (int i = 0; i < EC; i++) e[i] = i < n ? p[i] : from_float<T>(0.f);
    frag v;
    __builtin_memcpy(&v, e, 16);
    return v;
}
__device__ __forceinline__ gm_f32x4 mfma16(gm_bf16x8 a, gm_bf16x8 b, gm_f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ gm_f32x4 mfma16(gm_f16x8 a, gm_f16x8 b, gm_f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ gm_f32x4 mfma16(gm_f32x4 a, gm_f32x4 b, gm_f32x4 c) {
#pragma unroll
    for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
}

template <typename T, int MB, int FB>
__global__ __launch_bounds__(64 * ROWS_WAVES) void hstu_gated_rows_kernel(const RowsArgs a) {
    typedef typename GM<T>::frag frag;
    constexpr int EC = 16 / sizeof(T), PIECE = 8 * EC, W = ROWS_WAVES;
    constexpr int VALS = 2 * FB * MB * 256;            // fp32 sums of a wave
    __shared__ float red[W * VALS];
    __shared__ float zs[2][16 * MB][16 * FB + 1];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r16 = lane & 15, q = lane >> 4;
    const int f0 = blockIdx.x * (16 * FB);
    const T* x = reinterpret_cast<const T*>(a.x);
    const T* wt = reinterpret_cast<const T*>(a.weight);
    // rows behind the last one repeat it: their products are never stored
    const T* wrow[2][FB];
    const T* xrow[MB];
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
        for (int b = 0; b < FB; b++) wrow[h][b] = wt + ((int64_t)h * a.f + min(f0 + 16 * b + r16, a.f - 1)) * a.k + q * EC;
#pragma unroll
    for (int j = 0; j < MB; j++) xrow[j] = x + (int64_t)min(16 * j + r16, a.m - 1) * a.x_stride + q * EC;
    gm_f32x4 acc[2][FB][MB];
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
        for (int b = 0; b < FB; b++)
#pragma unroll
            for (int j = 0; j < MB; j++) acc[h][b][j] = gm_f32x4{0.f, 0.f, 0.f, 0.f};
    // whole pieces without a branch between their loads; only a row's last piece may be shorter
    struct Piece { frag w[2][2][FB], x[2][MB]; };
    auto multiply = [&](const Piece& p) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int b = 0; b < FB; b++)
#pragma unroll
                    for (int j = 0; j < MB; j++) acc[h][b][j] = mfma16(p.w[s][h][b], p.x[s][j], acc[h][b][j]);
    };
    int k0 = w * PIECE;
#pragma unroll 2
    for (; k0 + PIECE <= a.k; k0 += W * PIECE) {
        Piece p;
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const int at = k0 + 4 * EC * s;
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int b = 0; b < FB; b++) p.w[s][h][b] = __builtin_bit_cast(frag, *reinterpret_cast<const gm_u4_any*>(wrow[h][b] + at));
#pragma unroll
            for (int j = 0; j < MB; j++) p.x[s][j] = __builtin_bit_cast(frag, *reinterpret_cast<const gm_u4_any*>(xrow[j] + at));
        }
        multiply(p);
    }
    if (k0 < a.k) {
        Piece p;
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const int at = k0 + 4 * EC * s, n = a.k - (at + q * EC), o = n > 0 ? at : 0;
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int b = 0; b < FB; b++) p.w[s][h][b] = load_frag(wrow[h][b] + o, n);
#pragma unroll
            for (int j = 0; j < MB; j++) p.x[s][j] = load_frag(xrow[j] + o, n);
        }
        multiply(p);
    }
    // a lane holds f = 16 b + 4 q + e of row m = 16 j + r16
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
        for (int b = 0; b < FB; b++)
#pragma unroll
            for (int j = 0; j < MB; j++)
                *reinterpret_cast<gm_f32x4*>(red + w * VALS + (((h * FB + b) * MB + j) * 64 + lane) * 4) = acc[h][b][j];
    __syncthreads();
    for (int v = threadIdx.x * 4; v < VALS; v += 64 * W * 4) {
        gm_f32x4 s = *reinterpret_cast<const gm_f32x4*>(red + v);
#pragma unroll
        for (int i = 1; i < W; i++) s += *reinterpret_cast<const gm_f32x4*>(red + i * VALS + v);
        const int l = (v >> 2) & 63, j = (v >> 8) % MB, hb = (v >> 8) / MB, h = hb / FB, b = hb % FB;
        const int c = 16 * b + 4 * (l >> 4);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            float z = s[e];
            if (a.bias && f0 + c + e < a.f) {
                const int64_t at = (int64_t)h * a.f + f0 + c + e;
                z += a.bias_f32 ? reinterpret_cast<const float*>(a.bias)[at] : to_float(reinterpret_cast<const T*>(a.bias)[at]);
            }
            // columns behind f repeat the last one: zero, they must not set a group's exponent
            zs[h][16 * j + (l & 15)][c + e] = f0 + c + e < a.f ? z : 0.f;
        }
    }
    __syncthreads();
    for (int v = threadIdx.x; v < a.m * 16 * FB; v += 64 * W) {
        const int m = v / (16 * FB), c = v % (16 * FB), f = f0 + c;
        const float zg = zs[0][m][c], zu = zs[1][m][c];
        float act;
        act_of<1>(&zg, a.act, &act);
        if (f < a.f) reinterpret_cast<T*>(a.out)[(int64_t)m * a.f + f] = from_float<T>(act * zu);
        if (a.keep == HSTU_KEEP_FULL) {
            const int kept = HSTU_GATED_KEPT(a.f);   // (the grid covers the kept columns, and only those)
            const int64_t at = (int64_t)m * 2 * kept + f;
            if constexpr (sizeof(T) == 4) {
                reinterpret_cast<T*>(a.z)[at] = zg;
                reinterpret_cast<T*>(a.z)[at + kept] = zu;
            } else {
                const unsigned bg = __builtin_bit_cast(unsigned, zg), bu = __builtin_bit_cast(unsigned, zu);
                uint16_t* up = reinterpret_cast<uint16_t*>(a.z) + at + f - (f & 31);   // blocks of 32: the gate's, the values'
                up[0] = (uint16_t)(bg >> 16);
                up[32] = (uint16_t)(bu >> 16);
                a.z_aux[at] = (uint8_t)(bg >> 8);
                a.z_aux[at + kept] = (uint8_t)(bu >> 8);
            }
        }
    }
    if constexpr (FB == 2) {
        if (a.keep == HSTU_KEEP_8BIT && threadIdx.x < 2 * a.m) {
            const int m = threadIdx.x >> 1, h = threadIdx.x & 1;
            float top = 0.f;
            for (int c = 0; c < 32; c++) top = fmaxf(top, pack8_finite_abs(zs[h][m][c]));
            const int e = pack8_exponent(top);
            const float inv = pack8_inv_scale(e);
            const int64_t at = ((int64_t)m * 2 + h) * HSTU_GATED_KEPT(a.f) + f0;
            a.z_aux[at / HSTU_PACK8_GROUP] = (uint8_t)e;
            uint8_t* z = reinterpret_cast<uint8_t*>(a.z) + at;
            for (int c = 0; c < 32; c += 4) {
                const unsigned u = pack8_codes(zs[h][m][c], zs[h][m][c + 1], zs[h][m][c + 2], zs[h][m][c + 3], inv);
#pragma unroll
                for (int i = 0; i < 4; i++) z[c + i] = (uint8_t)(u >> (8 * i));
            }
        }
    }
}

hipError_t launch_gated_rows_bf16(const RowsArgs& a, hipStream_t st);
hipError_t launch_gated_rows_f16(const RowsArgs& a, hipStream_t st);
hipError_t launch_gated_rows_f32(const RowsArgs& a, hipStream_t st);

template <typename T> hipError_t launch_gated_rows_t(const RowsArgs& a, hipStream_t st) {
    // 8-bit groups of 32 columns stay within a workgroup
    const bool wide = a.keep == HSTU_KEEP_8BIT;
    const int cols = a.keep == HSTU_KEEP_NONE ? a.f : HSTU_GATED_KEPT(a.f);
    const dim3 grid((unsigned)((cols + (wide ? 31 : 15)) / (wide ? 32 : 16))), nt(64 * ROWS_WAVES);
#define GR_GO(MB)                                                                                              \
    do {                                                                                                       \
        if (wide) hipLaunchKernelGGL((hstu_gated_rows_kernel<T, MB, 2>), grid, nt, 0, st, a);                  \
        else hipLaunchKernelGGL((hstu_gated_rows_kernel<T, MB, 1>), grid, nt, 0, st, a);                       \
    } while (0)
    if (a.m <= 16) GR_GO(1);
    else if (a.m <= 32) GR_GO(2);
    else if (a.m <= 48) GR_GO(3);
    else GR_GO(4);
#undef GR_GO
    return hipGetLastError();
}

}  // namespace hstu
