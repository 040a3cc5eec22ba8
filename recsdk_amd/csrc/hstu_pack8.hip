// Activations in 8 bits (mxrec::activation_pack8, activation_unpack8): e4m3 codes under one power-of-two exponent per 32
// columns.  A lane holds 8 consecutive columns, four neighbouring lanes a group: its largest magnitude is two lane exchanges.
// Bounded by HBM: 2 + 1 + 1/32 bytes an element of 16 bits in either direction, nothing is read twice.  [16384, 8192] bf16: 67 us to
// pack and 65 to unpack, 6.1 TB/s (a large copy 4.9).
#include "hstu_ffn_common.h"

namespace hstu {

constexpr int P8_NT = 256;
constexpr int P8_ROWS = 4;   // rows of a lane, loaded before the first is worked on

// lanes along a row: a power of two of at least one group, at most a wave
static int p8_lanes(int cols) {
    int l = 4;
    while (l < 64 && l * 8 < cols) l *= 2;
    return l;
}

template <typename T, bool PACK>
__global__ __launch_bounds__(P8_NT) void hstu_pack8_kernel(const hstu_pack8_params p, int lanes, int col_blocks) {
    const int groups = (p.cols + HSTU_PACK8_GROUP - 1) / HSTU_PACK8_GROUP;
    const int tx = threadIdx.x & (lanes - 1), ty = threadIdx.x / lanes, rows_wg = P8_NT / lanes;
    const int cb = blockIdx.x % col_blocks;
    const int64_t r0 = (int64_t)(blockIdx.x / col_blocks) * (rows_wg * P8_ROWS) + ty;
    const int c = (cb * lanes + tx) * 8, n = p.cols - c;   // n <= 0: a lane behind the row, which still takes part in its group
    float v[P8_ROWS][8];
    if constexpr (PACK) {
#pragma unroll
        for (int i = 0; i < P8_ROWS; i++) {
            const int64_t r = r0 + (int64_t)i * rows_wg;
            load8_any(reinterpret_cast<const T*>(p.x) + (r < p.rows && n > 0 ? r * p.x_stride + c : 0), r < p.rows ? n : 0, v[i]);
        }
#pragma unroll
        for (int i = 0; i < P8_ROWS; i++) {
            const int64_t r = r0 + (int64_t)i * rows_wg;
            float top = 0.f;
#pragma unroll
            for (int k = 0; k < 8; k++) top = fmaxf(top, pack8_finite_abs(v[i][k]));
            top = fmaxf(top, __shfl_xor(top, 1, 64));
            top = fmaxf(top, __shfl_xor(top, 2, 64));
            const int e = pack8_exponent(top);
            const float inv = pack8_inv_scale(e);
            const ffn_u2 q = {pack8_codes(v[i][0], v[i][1], v[i][2], v[i][3], inv), pack8_codes(v[i][4], v[i][5], v[i][6], v[i][7], inv)};
            if (r < p.rows && n > 0) {
                uint8_t* dst = p.codes + r * p.cols + c;
                if (n >= 8) __builtin_nontemporal_store(q, reinterpret_cast<ffn_u2_any*>(dst));
                else {
#pragma unroll
                    for (int k = 0; k < 8; k++)
                        if (k < n) dst[k] = (uint8_t)(q[k >> 2] >> (8 * (k & 3)));
                }
                if ((tx & 3) == 0) p.exponents[r * groups + c / HSTU_PACK8_GROUP] = (uint8_t)e;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < P8_ROWS; i++) {
            const int64_t r = r0 + (int64_t)i * rows_wg;
            if (r >= p.rows || n <= 0) continue;
            code_values(codes8_raw(p.codes + r * p.cols + c, n, p.exponents[r * groups + c / HSTU_PACK8_GROUP]), largest_finite<T>(), v[i]);
        }
#pragma unroll
        for (int i = 0; i < P8_ROWS; i++) {
            const int64_t r = r0 + (int64_t)i * rows_wg;
            if (r < p.rows && n > 0) store8_any(reinterpret_cast<T*>(p.x) + r * p.x_stride + c, n, v[i]);
        }
    }
}

static int p8_check(const hstu_pack8_params* p) {
    if (!p) return fail(HSTU_ERR_INVALID_ARGUMENT, "params is NULL");
    if (p->struct_size != sizeof(hstu_pack8_params))
        return fail(HSTU_ERR_INVALID_ARGUMENT, "hstu_pack8_params size mismatch: caller %u, library %zu", p->struct_size, sizeof(hstu_pack8_params));
    if (p->dtype != HSTU_F32 && p->dtype != HSTU_F16 && p->dtype != HSTU_BF16)
        return fail(HSTU_ERR_INVALID_ARGUMENT, "dtype expect float32, float16 or bfloat16, but value is %d", p->dtype);
    if (p->rows < 0 || p->rows > HSTU_FFN_MAX_ROWS) return fail(HSTU_ERR_INVALID_ARGUMENT, "rows must in range:[0,%lld].", HSTU_FFN_MAX_ROWS);
    if (p->cols < 1 || p->cols > HSTU_PACK8_MAX_COLS) return fail(HSTU_ERR_INVALID_ARGUMENT, "cols must in range:[1,%d].", HSTU_PACK8_MAX_COLS);
    if (p->x_stride < 0) return fail(HSTU_ERR_INVALID_ARGUMENT, "x_stride must not be negative");
    if (p->rows && (!p->x || !p->codes || !p->exponents)) return fail(HSTU_ERR_INVALID_ARGUMENT, "x, codes and exponents must not be NULL");
    if (reinterpret_cast<uintptr_t>(p->x) & (p->dtype == HSTU_F32 ? 3 : 1)) return fail(HSTU_ERR_UNSUPPORTED, "x must be aligned to its element type");
    return HSTU_OK;
}

template <bool PACK> static int p8_run(const hstu_pack8_params* p, void* stream) {
    int rc = p8_check(p);
    if (rc != HSTU_OK) return rc;
    if (!PACK && p->x_stride < p->cols && p->rows > 1) return fail(HSTU_ERR_INVALID_ARGUMENT, "x_stride of an output must be at least cols");
    if (p->rows == 0) return HSTU_OK;
    const int lanes = p8_lanes(p->cols), col_blocks = (p->cols + lanes * 8 - 1) / (lanes * 8);
    const int64_t per = (int64_t)(P8_NT / lanes) * P8_ROWS, blocks = (p->rows + per - 1) / per * col_blocks;
    if (blocks > 0xffffff) return fail(HSTU_ERR_UNSUPPORTED, "rows * cols too large for one launch");
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)blocks);
    if (p->dtype == HSTU_F32) hipLaunchKernelGGL((hstu_pack8_kernel<float, PACK>), grid, dim3(P8_NT), 0, st, *p, lanes, col_blocks);
    else if (p->dtype == HSTU_F16) hipLaunchKernelGGL((hstu_pack8_kernel<_Float16, PACK>), grid, dim3(P8_NT), 0, st, *p, lanes, col_blocks);
    else hipLaunchKernelGGL((hstu_pack8_kernel<__bf16, PACK>), grid, dim3(P8_NT), 0, st, *p, lanes, col_blocks);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(HSTU_ERR_LAUNCH, "kernel launch failed: %s", hipGetErrorString(e));
    return HSTU_OK;
}

}  // namespace hstu

extern "C" int hstu_hip_activation_pack8(const hstu_pack8_params* p, void* stream) { return hstu::p8_run<true>(p, stream); }
extern "C" int hstu_hip_activation_unpack8(const hstu_pack8_params* p, void* stream) { return hstu::p8_run<false>(p, stream); }
