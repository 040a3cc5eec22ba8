/*
 * hstu_ffn.h -- C ABI of the feed-forward half of a layer: LayerNorm with its backward (mxrec::layer_norm), the gated
 * projection act(x Wg^T + bg) * (x Wu^T + bu) with its backward (mxrec::gated_linear), and activations kept in 8 bits
 * (mxrec::activation_pack8 / activation_unpack8), which the gated projection's backward also reads.
 *
 * Same conventions as hstu_hip.h: device pointers, asynchronous on `stream`, nothing read on the host, 0 or a negative
 * hstu_status with the message in hstu_hip_last_error().  Pointers need the alignment of their element type only, except
 * workspaces (16 bytes).  Outputs must not overlap inputs or each other.  A workspace needs no initialisation, belongs to one
 * call at a time and is free again when the call's work on the stream is done.  Sums over rows are formed in a fixed order:
 * results are reproducible.  A call whose work would not fit one launch (more elements than the memory holds, unless rows repeat) is
 * refused with HSTU_ERR_UNSUPPORTED.
 */
#ifndef HSTU_FFN_H
#define HSTU_FFN_H

#include "hstu_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define HSTU_LN_MAX_COLS 16384
#define HSTU_FFN_MAX_ROWS (1LL << 30)

/* LayerNorm over the last axis:
 *   y = x_hat * weight + bias     x_hat = (x - mean) * rstd     rstd = 1 / sqrt(var + eps)
 * mean and (biased) variance in fp32, the variance from the deviations; y rounded once.  Finite rows of any size are taken (up to
 * 2^126: beyond it a deviation itself may leave fp32); a row with a NaN or an infinity has NaN for y, mean and rstd.  rows may be 0. */
typedef struct hstu_layer_norm_params {
    uint32_t struct_size;
    int32_t dtype;         /* HSTU_F32 / HSTU_F16 / HSTU_BF16: x, y */
    int32_t param_dtype;   /* weight, bias: dtype or HSTU_F32 */
    int32_t cols;          /* [1, HSTU_LN_MAX_COLS] */
    int64_t rows;          /* [0, HSTU_FFN_MAX_ROWS] */
    int64_t x_stride;      /* elements from a row of x to the next, >= 0 */
    float eps;             /* > 0, finite */
    uint32_t reserved;
    const void* x;         /* [rows, cols] */
    const void* weight;    /* [cols], or NULL: ones */
    const void* bias;      /* [cols], or NULL: zeros */
    void* y;               /* [rows, cols], contiguous */
    float* mean;           /* [rows]; mean and rstd may both be NULL */
    float* rstd;           /* [rows] */
} hstu_layer_norm_params;
int hstu_hip_layer_norm(const hstu_layer_norm_params* p, void* stream);

/* Backward:  a = d_y * weight     d_x = rstd * (a - mean_c(a) - x_hat * mean_c(a * x_hat))
 *            d_weight = sum over rows of d_y * x_hat     d_bias = sum over rows of d_y
 * d_weight and d_bias are summed in fp32 and rounded once to grad_dtype.  Any of the three outputs may be NULL (not wanted). */
typedef struct hstu_layer_norm_bwd_params {
    uint32_t struct_size;
    int32_t dtype;
    int32_t param_dtype;
    int32_t grad_dtype;    /* d_weight, d_bias: param_dtype or HSTU_F32 */
    int64_t rows;
    int32_t cols;
    uint32_t reserved;
    int64_t x_stride;
    int64_t dy_stride;
    const void* d_y;       /* [rows, cols] */
    const void* x;
    const void* weight;    /* or NULL: ones */
    const float* mean;     /* from the forward */
    const float* rstd;
    void* d_x;             /* [rows, cols], contiguous */
    void* d_weight;        /* [cols] */
    void* d_bias;          /* [cols] */
} hstu_layer_norm_bwd_params;
int hstu_hip_layer_norm_backward_get_workspace_size(const hstu_layer_norm_bwd_params* p, uint64_t* workspace_bytes);
int hstu_hip_layer_norm_backward(const hstu_layer_norm_bwd_params* p, void* workspace, uint64_t workspace_bytes, void* stream);

/* Activations in 8 bits.  32 consecutive columns of a row (the last group of a row may be shorter) share an exponent E:
 *   E    = the smallest integer >= -126 with max |v| <= 448 * 2^E over the group's finite values (-126 where there is none)
 *   code = float8_e4m3fn nearest to v * 2^-E (ties to even); NaN for NaN and infinities
 *   exponents[row, group] = E + 127
 * A code stands for code * 2^E, brought into the finite range of the type it is read in.  With power-of-two scales a value is
 * off by at most 2^-4 of itself or 2^-10 * 2^E, whichever is larger, and packing an unpacked tensor again changes no value.  (It may
 * change the codes: a group whose largest value was rounded down to 224 * 2^E comes back with E - 1 and codes twice as large.) */
#define HSTU_PACK8_GROUP 32
#define HSTU_PACK8_MAX_COLS 65536
typedef struct hstu_pack8_params {
    uint32_t struct_size;
    int32_t dtype;         /* HSTU_F32 / HSTU_F16 / HSTU_BF16: x */
    int64_t rows;          /* [0, HSTU_FFN_MAX_ROWS] */
    int32_t cols;          /* [1, HSTU_PACK8_MAX_COLS] */
    uint32_t reserved;
    int64_t x_stride;      /* elements from a row of x to the next (unpack: cols) */
    void* x;               /* [rows, cols]: read by pack, written by unpack */
    uint8_t* codes;        /* [rows, cols] */
    uint8_t* exponents;    /* [rows, ceil(cols / 32)] */
} hstu_pack8_params;
int hstu_hip_activation_pack8(const hstu_pack8_params* p, void* stream);
int hstu_hip_activation_unpack8(const hstu_pack8_params* p, void* stream);

/* Gated projection:
 *   z = x W^T + bias     [m, 2 f], fp32 accumulation; weight rows and z columns [0, f) are the gate, [f, 2 f) the values
 *   out = round(act(z[:, :f]) * z[:, f:])
 * keep says what the backward gets: nothing, z, or z in 8 bits.  z is kept in fp32 for HSTU_F32 and in 24 bits otherwise: the upper
 * 16 bits of the fp32 value in z, the next 8 in z_aux (1 + 8 + 15 bits; rounded to 16 bits, z alone would put as large an error into
 * the gradients as the rounding of dz and of the gradients themselves).  What is kept has rows of 2 fp columns, fp = f rounded up to
 * a multiple of 32 (HSTU_GATED_KEPT(f)): the gate's f, zeros, the values' f, zeros; in 8 bits z_aux has an exponent for each 32 of
 * them, [m, 2, fp / 32].  In the 16-bit upper parts alone, blocks of 32 columns of the gate and of the values take turns, so that a
 * block of both is a line of 128 bytes: [m, fp / 32, 2, 32].  m may be 0. */
#define HSTU_GATED_MAX_K 16384
#define HSTU_GATED_MAX_F 32768
#define HSTU_GATED_KEPT(f) (((f) + 31) / 32 * 32)
enum { HSTU_ACT_SILU = 0, HSTU_ACT_GELU = 1 /* z * Phi(z), with erf */ };
enum { HSTU_KEEP_NONE = 0, HSTU_KEEP_FULL = 1, HSTU_KEEP_8BIT = 2 /* 16-bit dtypes only */ };
typedef struct hstu_gated_params {
    uint32_t struct_size;
    int32_t dtype;         /* HSTU_F32 / HSTU_F16 / HSTU_BF16: x, weight, out */
    int32_t bias_dtype;    /* dtype or HSTU_F32 */
    int32_t act;
    int32_t keep;
    int32_t k;             /* [1, HSTU_GATED_MAX_K] */
    int32_t f;             /* [1, HSTU_GATED_MAX_F] */
    uint32_t reserved;
    int64_t m;             /* [0, HSTU_FFN_MAX_ROWS] */
    int64_t x_stride;      /* elements from a row of x to the next */
    const void* x;         /* [m, k] */
    const void* weight;    /* [2 f, k], contiguous */
    const void* bias;      /* [2 f], or NULL */
    void* out;             /* [m, f], contiguous */
    void* z;               /* HSTU_KEEP_FULL: fp32 [m, 2, fp], or 16-bit upper parts [m, fp / 32, 2, 32]; HSTU_KEEP_8BIT: codes [m, 2, fp] */
    uint8_t* z_aux;        /* HSTU_KEEP_FULL of 16-bit dtypes: lower parts [m, 2, fp]; HSTU_KEEP_8BIT: exponents */
} hstu_gated_params;
int hstu_hip_gated_linear_get_workspace_size(const hstu_gated_params* p, uint64_t* workspace_bytes);
int hstu_hip_gated_linear(const hstu_gated_params* p, void* workspace, uint64_t workspace_bytes, void* stream);

/* Backward:  dz_g = d_out * z_u * act'(z_g)     dz_u = d_out * act(z_g)     (rounded to dtype for the two products,
 *            so in HSTU_F16 within its range)
 *            d_x = dz W  [m, k]     d_weight = dz^T x  [2 f, k]     d_bias = column sums of the unrounded dz  [2 f]
 * Any of the three outputs may be NULL (not wanted). */
typedef struct hstu_gated_bwd_params {
    uint32_t struct_size;
    int32_t dtype;
    int32_t grad_bias_dtype;  /* d_bias: dtype or HSTU_F32 */
    int32_t act;
    int32_t keep;             /* what z holds: HSTU_KEEP_FULL or HSTU_KEEP_8BIT */
    int32_t k;
    int32_t f;
    uint32_t reserved;
    int64_t m;
    int64_t x_stride;
    int64_t dout_stride;
    const void* d_out;        /* [m, f] */
    const void* x;            /* [m, k]; read for d_weight only */
    const void* weight;       /* [2 f, k]; read for d_x only */
    const void* z;
    const uint8_t* z_aux;
    void* d_x;                /* [m, k], contiguous */
    void* d_weight;           /* [2 f, k], contiguous */
    void* d_bias;             /* [2 f] */
} hstu_gated_bwd_params;
int hstu_hip_gated_linear_backward_get_workspace_size(const hstu_gated_bwd_params* p, uint64_t* workspace_bytes);
int hstu_hip_gated_linear_backward(const hstu_gated_bwd_params* p, void* workspace, uint64_t workspace_bytes, void* stream);

/* Which kernels the given arguments select, NUL-terminated into buf; nothing is launched.  Forward: "rows_bf16_48" (few rows: the
 * instance for up to 48) or "tiles_bf16_256x128" (rows x columns of z, "_deep": four buffers).  Backward: both products with the number
 * of shares of their contraction, "dx_f16_256x128_1 dw_f16_128x128_deep_4". */
int hstu_hip_gated_linear_describe_kernel(const hstu_gated_params* p, char* buf, size_t buf_bytes);
int hstu_hip_gated_linear_backward_describe_kernel(const hstu_gated_bwd_params* p, char* buf, size_t buf_bytes);

#ifdef __cplusplus
}
#endif
#endif /* HSTU_FFN_H */
