// LayerNorm over the last axis, forward and backward (mxrec::layer_norm), any width up to 16384.  HBM-bound row work: a row
// is held in the registers of LPR neighbouring lanes (8 to 64 of a wave, or a workgroup of 256 to 1024), NP pieces of 8
// consecutive columns each, so that it is read once and the variance is taken from the deviations.  Rows of any width and
// alignment take the same path: a lane's 16-byte accesses may start anywhere, a row's last piece goes by four, two and one elements.
//   forward   mean = sum x / C, var = sum (x - mean)^2 / C, rstd = 1 / sqrt(var + eps), y = (x - mean) rstd w + b
//   backward  a = dy w, dx = rstd (a - (sum a + x_hat sum a x_hat) / C), dw = sum_rows dy x_hat, db = sum_rows dy
// The column sums stay in registers over the rows that a lane sees, meet in LDS, leave as one row of partial sums per
// workgroup, and a second kernel adds those in a fixed order: no atomics, reproducible.
// Every finite row is taken: the sum is formed in units of 2^14 (an FMA in place of an addition, the same bits), and a row whose
// squared deviations leave fp32, one that hardly ever comes, takes its variance from deviations in units of 2^90.
// [262144, 512] bf16: forward 101 us (5.3 TB/s; a large copy 4.9), backward 137 to 143 (5.6 to 5.9), column sums 4.8.
// Widths off the 8-column grid pay for accesses that straddle lines: [262144, 257] 88 and 166 us, [262144, 256] 54 and 70.
#include "hstu_ffn_common.h"

namespace hstu {

// sum over groups of N neighbouring lanes, in every lane.  Register moves between lanes instead of LDS permutes: within a quad, then
// mirrored in 8 and 16 lanes (whose halves hold equal sums by then), then the two instructions that exchange rows of 16 and halves
template <int CTRL> __device__ __forceinline__ float ln_moved(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
template <int N> __device__ __forceinline__ float ln_lanes_sum(float x) {
    x += ln_moved<0xB1>(x);                          // quad_perm 1 0 3 2
    x += ln_moved<0x4E>(x);                          // quad_perm 2 3 0 1
    if constexpr (N >= 8) x += ln_moved<0x141>(x);   // mirror of 8
    if constexpr (N >= 16) x += ln_moved<0x140>(x);  // mirror of 16
    if constexpr (N >= 32) {
        const unsigned u = __builtin_bit_cast(unsigned, x);
        const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        x = __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
    }
    if constexpr (N >= 64) {
        const unsigned u = __builtin_bit_cast(unsigned, x);
        const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        x = __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
    }
    return x;
}

// sums of a and b over the LPR lanes of a row; `slot` (0 / 1, alternating) keeps a workgroup-wide sum from meeting the next
// one in LDS
template <int LPR> __device__ __forceinline__ void ln_sum(float& a, float& b, float* red, int slot) {
    a = ln_lanes_sum<(LPR < 64 ? LPR : 64)>(a);
    b = ln_lanes_sum<(LPR < 64 ? LPR : 64)>(b);
    if constexpr (LPR > 64) {
        constexpr int W = LPR / 64;
        float* at = red + slot * 2 * W;
        if ((threadIdx.x & 63) == 0) {
            at[threadIdx.x >> 6] = a;
            at[W + (threadIdx.x >> 6)] = b;
        }
        __syncthreads();
        a = b = 0.f;
#pragma unroll
        for (int i = 0; i < W; i++) {
            a += at[i];
            b += at[W + i];
        }
    }
}

// `def` where the parameter is missing
template <typename T> __device__ __forceinline__ void ln_param(const void* p, bool f32, int c, int n, float def, float* v) {
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = def;
    if (p && n > 0) {
        if (f32) load8_any(reinterpret_cast<const float*>(p) + c, n, v);
        else load8_any(reinterpret_cast<const T*>(p) + c, n, v);
    }
}

// A row's sum is formed in units of this power of two, as many as there can be columns: it stays in fp32 for every row that does
constexpr float LN_SUM_UNIT = (float)HSTU_LN_MAX_COLS;
static_assert(HSTU_LN_MAX_COLS == 1 << 14, "a power of two");

// rstd of a row whose squared deviations `v` leave fp32 (the largest of them then is 2^57 or more): from deviations in units of 2^90,
// and `rest`, their mean.  NaN where one of them is no number
template <int LPR, int NP> __device__ __forceinline__ float ln_far_rstd(const float (&v)[NP][8], int l, int cols, float eps, float* red, float& rest) {
    constexpr float UNIT = 0x1p90f, INV = 0x1p-90f;
    const float count = (float)cols;
    float d1 = 0.f, d2 = 0.f;
#pragma unroll
    for (int q = 0; q < NP; q++)
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const float d = (q * LPR + l) * 8 + k < cols ? v[q][k] * INV : 0.f;
            d1 += d;
            d2 += d * d;
        }
    ln_sum<LPR>(d1, d2, red, 0);
    if constexpr (LPR > 64) __syncthreads();   // (the next row's first sum takes the same place in LDS)
    const float r = d1 / count, t = d2 / count - r * r, var = t < 0.f ? 0.f : t;
    rest = r * UNIT;
    // the variance itself, UNIT^2 var, fits where it is small: only there may eps be all that is left
    return var > 0x1p-100f ? INV / sqrtf(var + eps * INV * INV) : 1.0f / sqrtf(var * UNIT * UNIT + eps);
}

template <typename T, int LPR, int NP>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void hstu_layer_norm_fwd_kernel(const hstu_layer_norm_params p) {
    constexpr int NT = LPR > 256 ? LPR : 256, RPW = NT / LPR;
    __shared__ float red[LPR > 64 ? 4 * (LPR / 64) : 1];
    const int l = threadIdx.x & (LPR - 1);
    const bool f32 = p.param_dtype == HSTU_F32;
    const float count = (float)p.cols;
    float w[NP][8], b[NP][8];
#pragma unroll
    for (int q = 0; q < NP; q++) {
        const int c = (q * LPR + l) * 8;
        ln_param<T>(p.weight, f32, c, p.cols - c, 1.f, w[q]);
        ln_param<T>(p.bias, f32, c, p.cols - c, 0.f, b[q]);
    }
    const int64_t step = (int64_t)gridDim.x * RPW;
    int64_t row = (int64_t)blockIdx.x * RPW + threadIdx.x / LPR;
    Raw8<T> next[NP];   // the row after the one that is worked on is under way
    auto fetch = [&](int64_t r) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < NP; q++) {
            const int c = (q * LPR + l) * 8;
            next[q] = load8_raw(reinterpret_cast<const T*>(p.x) + r * p.x_stride + c, p.cols - c);
        }
    };
    if (row < p.rows) fetch(row);
    for (; row < p.rows; row += step) {
        float v[NP][8], s = 0.f, none = 0.f;
#pragma unroll
        for (int q = 0; q < NP; q++) to_floats(next[q], v[q]);
        if (row + step < p.rows) fetch(row + step);
#pragma unroll
        for (int q = 0; q < NP; q++)
#pragma unroll
            for (int k = 0; k < 8; k++) s = __builtin_fmaf(v[q][k], 1.0f / LN_SUM_UNIT, s);
        ln_sum<LPR>(s, none, red, 0);
        // deviations from the rounded mean, and from them what rounding took from it: rows far from zero keep their accuracy
        // (a constant row has x_hat = 0, not the rounding of its mean times 1 / sqrt(eps))
        const float near = s / count * LN_SUM_UNIT;
        float d1 = 0.f, d2 = 0.f;
#pragma unroll
        for (int q = 0; q < NP; q++)
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float d = v[q][k] - near;
                v[q][k] = d;
                const bool in = (q * LPR + l) * 8 + k < p.cols;
                d1 += in ? d : 0.f;
                d2 += in ? d * d : 0.f;
            }
        ln_sum<LPR>(d1, d2, red, 1);
        float rest = d1 / count, rstd;
        if (d2 <= 3.4e38f) rstd = 1.0f / sqrtf(fmaxf(d2 / count - rest * rest, 0.f) + p.eps);
        else rstd = ln_far_rstd<LPR, NP>(v, l, p.cols, p.eps, red, rest);
        const float mean = near + rest;
        if (l == 0 && p.mean) { p.mean[row] = mean; p.rstd[row] = rstd; }
        T* y = reinterpret_cast<T*>(p.y) + row * p.cols;
#pragma unroll
        for (int q = 0; q < NP; q++) {
            const int c = (q * LPR + l) * 8;
#pragma unroll
            for (int k = 0; k < 8; k++) v[q][k] = (v[q][k] - rest) * rstd * w[q][k] + b[q][k];
            store8_any(y + c, p.cols - c, v[q]);
        }
    }
}

template <typename T, int LPR, int NP>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void hstu_layer_norm_bwd_kernel(const hstu_layer_norm_bwd_params p, float* partial) {
    constexpr int NT = LPR > 256 ? LPR : 256, RPW = NT / LPR, WIDTH = LPR * 8 * NP;
    constexpr int WAVES = NT / 64;
    __shared__ float red[LPR > 64 ? 4 * (LPR / 64) : 1];
    __shared__ float cols[LPR > 64 ? 1 : WAVES * WIDTH];
    const int l = threadIdx.x & (LPR - 1);
    const float inv_c = 1.0f / (float)p.cols;
    float w[NP][8], gw[NP][8], gb[NP][8];
#pragma unroll
    for (int q = 0; q < NP; q++) {
        const int c = (q * LPR + l) * 8;
        ln_param<T>(p.weight, p.param_dtype == HSTU_F32, c, p.cols - c, 1.f, w[q]);
#pragma unroll
        for (int k = 0; k < 8; k++) gw[q][k] = gb[q][k] = 0.f;
    }
    int slot = 0;
    const int64_t step = (int64_t)gridDim.x * RPW;
    int64_t row = (int64_t)blockIdx.x * RPW + threadIdx.x / LPR;
    constexpr bool AHEAD = LPR < 1024;   // (a lane of a 1024-wide workgroup has 128 registers: its row is fetched when it is due)
    Raw8<T> next_x[NP], next_g[NP];      // the row after the one that is worked on is under way
    float next_mean = 0.f, next_rstd = 0.f;
    auto fetch = [&](int64_t r) __attribute__((always_inline)) {
        next_mean = p.mean[r];
        next_rstd = p.rstd[r];
#pragma unroll
        for (int q = 0; q < NP; q++) {
            const int c = (q * LPR + l) * 8;
            next_x[q] = load8_raw(reinterpret_cast<const T*>(p.x) + r * p.x_stride + c, p.cols - c);
            next_g[q] = load8_raw(reinterpret_cast<const T*>(p.d_y) + r * p.dy_stride + c, p.cols - c);
        }
    };
    if (AHEAD && row < p.rows) fetch(row);
    for (; row < p.rows; row += step) {
        if (!AHEAD) fetch(row);
        const float mean = next_mean, rstd = next_rstd;
        float xh[NP][8], g[NP][8];
#pragma unroll
        for (int q = 0; q < NP; q++) {
            to_floats(next_x[q], xh[q]);
            to_floats(next_g[q], g[q]);
        }
        if (AHEAD && row + step < p.rows) fetch(row + step);
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int q = 0; q < NP; q++) {
            const int left = p.cols - (q * LPR + l) * 8;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                // (behind the row both are zero: -mean * rstd may be infinite)
                xh[q][k] = k < left ? (xh[q][k] - mean) * rstd : 0.f;
                gw[q][k] += g[q][k] * xh[q][k];
                gb[q][k] += g[q][k];
                const float a = g[q][k] * w[q][k];
                g[q][k] = a;
                s1 += a;
                s2 += a * xh[q][k];
            }
        }
        if (p.d_x) {
            ln_sum<LPR>(s1, s2, red, slot);
            slot ^= 1;
            s1 *= inv_c;
            s2 *= inv_c;
            T* dx = reinterpret_cast<T*>(p.d_x) + row * p.cols;
#pragma unroll
            for (int q = 0; q < NP; q++) {
                const int c = (q * LPR + l) * 8;
#pragma unroll
                for (int k = 0; k < 8; k++) g[q][k] = (g[q][k] - (s1 + xh[q][k] * s2)) * rstd;
                store8_any(dx + c, p.cols - c, g[q]);
            }
        }
    }
    if (!partial) return;
#pragma unroll
    for (int which = 0; which < 2; which++) {
        float* out = partial + ((int64_t)blockIdx.x * 2 + which) * p.cols;
        if constexpr (LPR > 64) {
#pragma unroll
            for (int q = 0; q < NP; q++)
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const int c = (q * LPR + l) * 8 + k;
                    if (c < p.cols) out[c] = which ? gb[q][k] : gw[q][k];
                }
        } else {
            // lanes of one wave that hold the same columns, then the waves in order
#pragma unroll
            for (int q = 0; q < NP; q++)
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    float s = which ? gb[q][k] : gw[q][k];
#pragma unroll
                    for (int o = LPR; o < 64; o <<= 1) s += __shfl_xor(s, o, 64);
                    if ((threadIdx.x & 63) < LPR) cols[(threadIdx.x >> 6) * WIDTH + (q * LPR + l) * 8 + k] = s;
                }
            __syncthreads();
            for (int c = threadIdx.x; c < p.cols; c += NT) {
                float s = 0.f;
#pragma unroll
                for (int v = 0; v < WAVES; v++) s += cols[v * WIDTH + c];
                out[c] = s;
            }
            __syncthreads();
        }
    }
}

// 32 columns x 32 row slots per workgroup: slot r adds the rows r, r + 32, ..., then the slots are added 0..31
template <typename T> __global__ __launch_bounds__(1024) void hstu_colsum_kernel(const float* partial, int rows, int half, T* out0, T* out1) {
    __shared__ float part[32][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int64_t width = 2 * (int64_t)half, c = (int64_t)blockIdx.x * 32 + tx;
    float s = 0.f;
    if (c < width)
#pragma unroll 8
        for (int r = ty; r < rows; r += 32) s += partial[r * width + c];
    part[ty][tx] = s;
    __syncthreads();
    if (ty == 0 && c < width) {
        float t = 0.f;
#pragma unroll
        for (int r = 0; r < 32; r++) t += part[r][tx];
        T* out = c < half ? out0 : out1;
        if (out) out[c < half ? c : c - half] = from_float<T>(t);
    }
}

hipError_t launch_colsum(const float* partial, int rows, int half, void* out0, void* out1, int32_t out_dtype, hipStream_t st) {
    const dim3 grid((unsigned)((2 * (int64_t)half + 31) / 32));
    if (out_dtype == HSTU_F32) hipLaunchKernelGGL(hstu_colsum_kernel<float>, grid, dim3(1024), 0, st, partial, rows, half, (float*)out0, (float*)out1);
    else if (out_dtype == HSTU_F16) hipLaunchKernelGGL(hstu_colsum_kernel<_Float16>, grid, dim3(1024), 0, st, partial, rows, half, (_Float16*)out0, (_Float16*)out1);
    else hipLaunchKernelGGL(hstu_colsum_kernel<__bf16>, grid, dim3(1024), 0, st, partial, rows, half, (__bf16*)out0, (__bf16*)out1);
    return hipGetLastError();
}

// lanes per row and pieces per lane: the smallest pair that holds the row.  (32, 2) and not (64, 1) up to 512 columns: two rows a wave
// (262144 rows bf16: 512 columns 110 -> 104 us forward, 257 columns 102 -> 87 and 191 -> 161 us backward)
struct LnShape { int lpr, np; };
static LnShape ln_shape(int cols) {
    static const LnShape s[] = {{8, 1}, {16, 1}, {32, 1}, {32, 2}, {64, 2}, {64, 4}, {256, 2}, {512, 2}, {1024, 2}};
    for (const LnShape& x : s)
        if (x.lpr * x.np * 8 >= cols) return x;
    return s[8];
}
static int ln_rows_per_wg(const LnShape& s) { return s.lpr > 256 ? 1 : 256 / s.lpr; }
// Workgroups that walk down the rows with the next one under way.  Forward, narrow rows (one piece a lane): up to 2048 (262144 x 128
// fp16: 38 us with a workgroup for every 16 rows, 27.5 with 2048, 30 with 768).  Wider ones have a row's weight and bias to load before
// their first: 1024 up to 512 columns (262144 x 512 bf16: 104.6 with 2048, 100.6; 16000 x 512: 10.8 and 8.6; 262144 x 257: 87.3 and 85.9, 103
// with 768), 768 beyond (16000 x 1000: 20.1 and 16.6; 30000 x 2048: 55 and 48; 3000 x 16384: 66 and 50).
static unsigned ln_fwd_grid(int64_t rows, const LnShape& s) {
    const int64_t n = (rows + ln_rows_per_wg(s) - 1) / ln_rows_per_wg(s), most = s.np == 1 ? 2048 : s.lpr == 32 ? 1024 : 768;
    return (unsigned)(n < 1 ? 1 : n > most ? most : n);
}
// Backward: each one is a row of the partial-sum table too, so no more than fill the chip and two rows a lane at least, four of wide rows
// (262144 x 128 fp16: 768 38.7 us, 512 41.9; 262144 x 512 bf16: 768 144, 512 137, 256 146; 30000 x 2048: 512 73, 256 69; 8192 x 4096:
// 512 52, 256 48; two rows a lane and four, 500 x 4096: 17.1 and 14.6, 7687 x 1000 fp32: 27.0 and 28.6)
static unsigned ln_bwd_grid(int64_t rows, const LnShape& s) {
    const bool wide = s.lpr >= 256 || s.np == 4;
    const int64_t most = wide ? 256 : s.np > 1 ? 512 : 768, per = (wide ? 4 : 2) * ln_rows_per_wg(s), n = (rows + per - 1) / per;
    return (unsigned)(n < 1 ? 1 : n > most ? most : n);
}

static bool ln_misaligned(const void* p, int32_t dtype) { return (reinterpret_cast<uintptr_t>(p) & (dtype == HSTU_F32 ? 3 : 1)) != 0; }

static int ln_check(int32_t dtype, int32_t param_dtype, int64_t rows, int32_t cols) {
    if (dtype != HSTU_F32 && dtype != HSTU_F16 && dtype != HSTU_BF16)
        return fail(HSTU_ERR_INVALID_ARGUMENT, "dtype expect float32, float16 or bfloat16, but value is %d", dtype);
    if (param_dtype != dtype && param_dtype != HSTU_F32) return fail(HSTU_ERR_INVALID_ARGUMENT, "param_dtype expect float32 or the dtype of x, but value is %d", param_dtype);
    if (rows < 0 || rows > HSTU_FFN_MAX_ROWS) return fail(HSTU_ERR_INVALID_ARGUMENT, "rows must in range:[0,%lld].", HSTU_FFN_MAX_ROWS);
    if (cols < 1 || cols > HSTU_LN_MAX_COLS) return fail(HSTU_ERR_INVALID_ARGUMENT, "cols must in range:[1,%d].", HSTU_LN_MAX_COLS);
    return HSTU_OK;
}

}  // namespace hstu

using namespace hstu;

#define LN_DISPATCH_T(T, KERNEL, s, grid, st, ...)                                                                      \
    do {                                                                                                                  \
        const dim3 nt((unsigned)((s).lpr > 256 ? (s).lpr : 256));                                                         \
        switch ((s).lpr * 8 + (s).np) {                                                                                   \
            case 8 * 8 + 1: hipLaunchKernelGGL((KERNEL<T, 8, 1>), grid, nt, 0, st, __VA_ARGS__); break;                   \
            case 16 * 8 + 1: hipLaunchKernelGGL((KERNEL<T, 16, 1>), grid, nt, 0, st, __VA_ARGS__); break;                 \
            case 32 * 8 + 1: hipLaunchKernelGGL((KERNEL<T, 32, 1>), grid, nt, 0, st, __VA_ARGS__); break;                 \
            case 32 * 8 + 2: hipLaunchKernelGGL((KERNEL<T, 32, 2>), grid, nt, 0, st, __VA_ARGS__); break;                 \
            case 64 * 8 + 2: hipLaunchKernelGGL((KERNEL<T, 64, 2>), grid, nt, 0, st, __VA_ARGS__); break;                 \
            case 64 * 8 + 4: hipLaunchKernelGGL((KERNEL<T, 64, 4>), grid, nt, 0, st, __VA_ARGS__); break;                 \
            case 256 * 8 + 2: hipLaunchKernelGGL((KERNEL<T, 256, 2>), grid, nt, 0, st, __VA_ARGS__); break;               \
            case 512 * 8 + 2: hipLaunchKernelGGL((KERNEL<T, 512, 2>), grid, nt, 0, st, __VA_ARGS__); break;               \
            default: hipLaunchKernelGGL((KERNEL<T, 1024, 2>), grid, nt, 0, st, __VA_ARGS__); break;                       \
        }                                                                                                                 \
    } while (0)
#define LN_DISPATCH(dtype, KERNEL, s, grid, st, ...)                                                                    \
    do {                                                                                                                  \
        if ((dtype) == HSTU_F32) LN_DISPATCH_T(float, KERNEL, s, grid, st, __VA_ARGS__);                                  \
        else if ((dtype) == HSTU_F16) LN_DISPATCH_T(_Float16, KERNEL, s, grid, st, __VA_ARGS__);                          \
        else LN_DISPATCH_T(__bf16, KERNEL, s, grid, st, __VA_ARGS__);                                                     \
    } while (0)

extern "C" int hstu_hip_layer_norm(const hstu_layer_norm_params* p, void* stream) {
    if (!p) return fail(HSTU_ERR_INVALID_ARGUMENT, "params is NULL");
    if (p->struct_size != sizeof(hstu_layer_norm_params))
        return fail(HSTU_ERR_INVALID_ARGUMENT, "hstu_layer_norm_params size mismatch: caller %u, library %zu", p->struct_size, sizeof(hstu_layer_norm_params));
    const int rc = ln_check(p->dtype, p->param_dtype, p->rows, p->cols);
    if (rc != HSTU_OK) return rc;
    if (!(p->eps > 0.f && p->eps <= 3.4e38f)) return fail(HSTU_ERR_INVALID_ARGUMENT, "eps must be positive and finite");
    if (p->x_stride < 0) return fail(HSTU_ERR_INVALID_ARGUMENT, "x_stride must not be negative");
    if (!p->mean != !p->rstd) return fail(HSTU_ERR_INVALID_ARGUMENT, "mean and rstd must both be NULL or neither");
    if (p->rows == 0) return HSTU_OK;
    if (!p->x || !p->y) return fail(HSTU_ERR_INVALID_ARGUMENT, "x and y must not be NULL");
    if (ln_misaligned(p->x, p->dtype) || ln_misaligned(p->y, p->dtype) || ln_misaligned(p->weight, p->param_dtype) || ln_misaligned(p->bias, p->param_dtype))
        return fail(HSTU_ERR_UNSUPPORTED, "x, weight, bias and y must be aligned to their element types");
    const LnShape s = ln_shape(p->cols);
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    LN_DISPATCH(p->dtype, hstu_layer_norm_fwd_kernel, s, dim3(ln_fwd_grid(p->rows, s)), st, *p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(HSTU_ERR_LAUNCH, "kernel launch failed: %s", hipGetErrorString(e));
    return HSTU_OK;
}

static int ln_bwd_validate(const hstu_layer_norm_bwd_params* p) {
    if (!p) return fail(HSTU_ERR_INVALID_ARGUMENT, "params is NULL");
    if (p->struct_size != sizeof(hstu_layer_norm_bwd_params))
        return fail(HSTU_ERR_INVALID_ARGUMENT, "hstu_layer_norm_bwd_params size mismatch: caller %u, library %zu", p->struct_size, sizeof(hstu_layer_norm_bwd_params));
    const int rc = ln_check(p->dtype, p->param_dtype, p->rows, p->cols);
    if (rc != HSTU_OK) return rc;
    if (p->grad_dtype != p->param_dtype && p->grad_dtype != HSTU_F32)
        return fail(HSTU_ERR_INVALID_ARGUMENT, "grad_dtype expect float32 or the dtype of weight, but value is %d", p->grad_dtype);
    if (p->x_stride < 0 || p->dy_stride < 0) return fail(HSTU_ERR_INVALID_ARGUMENT, "x_stride and dy_stride must not be negative");
    if (p->rows && (!p->x || !p->d_y || !p->mean || !p->rstd)) return fail(HSTU_ERR_INVALID_ARGUMENT, "d_y, x, mean and rstd must not be NULL");
    if (ln_misaligned(p->x, p->dtype) || ln_misaligned(p->d_y, p->dtype) || ln_misaligned(p->d_x, p->dtype) || ln_misaligned(p->weight, p->param_dtype) ||
        ln_misaligned(p->d_weight, p->grad_dtype) || ln_misaligned(p->d_bias, p->grad_dtype))
        return fail(HSTU_ERR_UNSUPPORTED, "d_y, x, weight and the gradients must be aligned to their element types");
    return HSTU_OK;
}

static uint64_t ln_bwd_bytes(const hstu_layer_norm_bwd_params* p) {
    if (!p->d_weight && !p->d_bias) return 0;
    return (uint64_t)ln_bwd_grid(p->rows, ln_shape(p->cols)) * 2 * p->cols * sizeof(float);
}

extern "C" int hstu_hip_layer_norm_backward_get_workspace_size(const hstu_layer_norm_bwd_params* p, uint64_t* bytes) {
    if (!bytes) return fail(HSTU_ERR_INVALID_ARGUMENT, "workspace_bytes is NULL");
    const int rc = ln_bwd_validate(p);
    if (rc != HSTU_OK) return rc;
    *bytes = ln_bwd_bytes(p);
    return HSTU_OK;
}

extern "C" int hstu_hip_layer_norm_backward(const hstu_layer_norm_bwd_params* p, void* workspace, uint64_t workspace_bytes, void* stream) {
    const int rc = ln_bwd_validate(p);
    if (rc != HSTU_OK) return rc;
    const uint64_t need = ln_bwd_bytes(p);
    if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)))
        return fail(HSTU_ERR_WORKSPACE, "workspace of %llu bytes (16-byte aligned) needed, got %llu at %p", (unsigned long long)need,
                    (unsigned long long)workspace_bytes, workspace);
    if (!p->d_x && !p->d_weight && !p->d_bias) return HSTU_OK;
    if (p->rows == 0 && !need) return HSTU_OK;
    const LnShape s = ln_shape(p->cols);
    const unsigned grid = ln_bwd_grid(p->rows, s);
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    float* partial = need ? reinterpret_cast<float*>(workspace) : nullptr;
    // without rows the workgroups write zero sums
    LN_DISPATCH(p->dtype, hstu_layer_norm_bwd_kernel, s, dim3(grid), st, *p, partial);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && need) e = launch_colsum(partial, (int)grid, p->cols, p->d_weight, p->d_bias, p->grad_dtype, st);
    if (e != hipSuccess) return fail(HSTU_ERR_LAUNCH, "kernel launch failed: %s", hipGetErrorString(e));
    return HSTU_OK;
}
