// The gated projection for few rows (single tokens, the candidates of a request): act(x Wg^T + bg) * (x Wu^T + bu) with m <= 64.
//
// The weights are read once and there is nothing to share between workgroups but a few rows of x, so nothing goes through LDS on
// the way in: a workgroup owns 16 FB columns f (their gate and their value rows), its eight waves take pieces of 256 bytes of k in
// turn.  Four neighbouring lanes load 64 bytes of a row, and a transpose over them makes MFMA fragments (16 x 16 blocks, W as the A
// operand); loaded as fragments, 16 rows to 16 neighbouring lanes, a load brings 16 bytes a cycle into a CU for 64.  Rows of any
// alignment are read in place; what the last piece of a row has of them is cut out of the row's last 16 bytes.  The waves' fp32 sums
// meet in LDS and are added in order.
// Bounded by reading W, for more rows by each workgroup's reading of all of x: at 48 rows of 1024 -> 4096 the 256 workgroups fetch 25 MB of
// x from the L2s beside 16.8 MB of W.  1024 -> 4096 bf16: one row 3.4 us (part of W out of the caches; 4.2 loaded as fragments), 48 rows
// 4.7 (7.0); 4096 -> 1024: one row 6.0 (10.3), 64 rows 11.5 (24).  32 columns a workgroup, half the readers of x, are slower at one row (6.2
// for 4.3; more rows were not measured), and so is a second piece under way.
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

// the last n elements (all of them where n is larger, zeros where it is not positive) moved to the front, zeros behind
template <typename T> __device__ __forceinline__ gm_u4 last_elements(gm_u4 v, int n) {
    const int bytes = 16 - max(min(n * (int)sizeof(T), 16), 0);
    if constexpr (sizeof(T) == 2) {
        const bool half = bytes & 2;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const unsigned moved = __builtin_amdgcn_alignbit(i < 3 ? v[i < 3 ? i + 1 : 3] : 0u, v[i], 16);
            v[i] = half ? moved : v[i];
        }
    }
    if (bytes & 4) v = (gm_u4){v[1], v[2], v[3], 0u};
    if (bytes & 8) v = (gm_u4){v[2], v[3], 0u, 0u};
    if (bytes & 16) v = (gm_u4){0u, 0u, 0u, 0u};
    return v;
}
__device__ __forceinline__ gm_f32x4 mfma16(gm_bf16x8 a, gm_bf16x8 b, gm_f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ gm_f32x4 mfma16(gm_f16x8 a, gm_f16x8 b, gm_f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ gm_f32x4 mfma16(gm_f32x4 a, gm_f32x4 b, gm_f32x4 c) {
#pragma unroll
    for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
}

// 4 x 4 transpose of 16-byte fragments over four neighbouring lanes: v[j] of lane s becomes v[s] of lane j
template <int CTRL> __device__ __forceinline__ void exchange(unsigned& a, unsigned& b, bool upper) {
    const unsigned from_b = (unsigned)__builtin_amdgcn_mov_dpp((int)b, CTRL, 0xf, 0xf, true), from_a = (unsigned)__builtin_amdgcn_mov_dpp((int)a, CTRL, 0xf, 0xf, true);
    a = upper ? from_b : a;
    b = upper ? b : from_a;
}
template <typename F> __device__ __forceinline__ void quad_transpose(F (&v)[4], int lane) {
    gm_u4 u[4];
#pragma unroll
    for (int i = 0; i < 4; i++) u[i] = __builtin_bit_cast(gm_u4, v[i]);
#pragma unroll
    for (int t = 0; t < 4; t++) {
        unsigned a = u[0][t], b = u[1][t], c = u[2][t], d = u[3][t];
        exchange<0xB1>(a, b, lane & 1);   // quad_perm 1 0 3 2
        exchange<0xB1>(c, d, lane & 1);
        exchange<0x4E>(a, c, lane & 2);   // quad_perm 2 3 0 1
        exchange<0x4E>(b, d, lane & 2);
        u[0][t] = a;
        u[1][t] = b;
        u[2][t] = c;
        u[3][t] = d;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = __builtin_bit_cast(F, u[i]);
}

template <typename T, int MB, int FB>
__global__ __launch_bounds__(64 * ROWS_WAVES) void hstu_gated_rows_kernel(const RowsArgs a) {
    typedef typename GM<T>::frag frag;
    constexpr int ES = sizeof(T), EC = 16 / ES, PIECE = 16 * EC, W = ROWS_WAVES;
    constexpr int VALS = 2 * FB * MB * 256;            // fp32 sums of a wave
    __shared__ float red[W * VALS];
    __shared__ float zs[2][16 * MB][16 * FB + 1];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, q = lane >> 4;
    const int f0 = blockIdx.x * (16 * FB);
    const T* x = reinterpret_cast<const T*>(a.x);
    const T* wt = reinterpret_cast<const T*>(a.weight);
    // Load i of a block: lane l takes chunk (l & 3) + 4 (l >> 4) of row 4 (l >> 2 & 3) + i.  After the transpose load j holds chunk
    // j + 4 (l >> 4) of row l & 15, a fragment.  Rows behind the last one repeat it: their products are never stored
    const int chunk = ((lane & 3) + 4 * q) * EC, fb = min(f0, a.f - 1);
    const char* wb[2] = {reinterpret_cast<const char*>(wt + (int64_t)fb * a.k), reinterpret_cast<const char*>(wt + ((int64_t)a.f + fb) * a.k)};
    const char* xb[MB];
    unsigned wo[FB][4], xo[MB][4];   // bytes from there to the lane's row
#pragma unroll
    for (int j = 0; j < MB; j++) xb[j] = reinterpret_cast<const char*>(x + (int64_t)(16 * j) * a.x_stride);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = (lane & 12) + i;
#pragma unroll
        for (int b = 0; b < FB; b++) wo[b][i] = (unsigned)(min(f0 + 16 * b + r, a.f - 1) - fb) * (unsigned)a.k * ES;
#pragma unroll
        for (int j = 0; j < MB; j++) xo[j][i] = (unsigned)(min(16 * j + r, a.m - 1) - 16 * j) * (unsigned)a.x_stride * ES;
    }
    auto load = [](const char* at, unsigned off) __attribute__((always_inline)) { return *reinterpret_cast<const gm_u4_any*>(at + off); };
    gm_f32x4 acc[2][FB][MB];
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
        for (int b = 0; b < FB; b++)
#pragma unroll
            for (int j = 0; j < MB; j++) acc[h][b][j] = gm_f32x4{0.f, 0.f, 0.f, 0.f};
    // whole pieces without a branch between their loads; only a row's last piece may be shorter
    struct Piece { frag w[2][FB][4], x[MB][4]; };
    auto multiply = [&](Piece& p) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < MB; j++) quad_transpose(p.x[j], lane);
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int b = 0; b < FB; b++) {
                quad_transpose(p.w[h][b], lane);
#pragma unroll
                for (int s = 0; s < 4; s++)
#pragma unroll
                    for (int j = 0; j < MB; j++) acc[h][b][j] = mfma16(p.w[h][b][s], p.x[j][s], acc[h][b][j]);
            }
    };
    int k0 = w * PIECE;
    for (; k0 + PIECE <= a.k; k0 += W * PIECE) {
        const unsigned at = (unsigned)(k0 + chunk) * ES;
        Piece p;
#pragma unroll
        for (int j = 0; j < MB; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) p.x[j][i] = __builtin_bit_cast(frag, load(xb[j], xo[j][i] + at));
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int b = 0; b < FB; b++)
#pragma unroll
                for (int i = 0; i < 4; i++) p.w[h][b][i] = __builtin_bit_cast(frag, load(wb[h], wo[b][i] + at));
        __builtin_amdgcn_sched_barrier(0);
        multiply(p);
    }
    if (k0 < a.k) {
        // a chunk that the row ends in is cut out of the row's last 16 bytes
        const int n = a.k - k0 - chunk;
        const unsigned at = (unsigned)(n >= EC ? k0 + chunk : a.k - EC) * ES;
        Piece p;
#pragma unroll
        for (int i = 0; i < 4; i++) {
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int b = 0; b < FB; b++) p.w[h][b][i] = __builtin_bit_cast(frag, last_elements<T>(load(wb[h], wo[b][i] + at), n));
#pragma unroll
            for (int j = 0; j < MB; j++) p.x[j][i] = __builtin_bit_cast(frag, last_elements<T>(load(xb[j], xo[j][i] + at), n));
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
