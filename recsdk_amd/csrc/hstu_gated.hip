// The gated projection act(x Wg^T + bg) * (x Wu^T + bu) and its backward (mxrec::gated_linear): argument checks, the choice of
// tiles, and the row work around the matrix products of hstu_gemm.h.
//   forward   one product kernel whose waves hold a block of the gate and the matching block of the values, so that
//             activation and product happen on the accumulators
//   backward  dz from d_out and the kept z (24 bits; one pass, also the column sums for d_bias), then d_x = dz W and d_weight = dz^T x,
//             which read their operands as they lie in memory (transposing LDS reads; nothing is transposed in HBM)
// dz is rounded to the I/O type between the two, as any training in that type rounds it: the products run on the 16-bit matrix cores.
// A rounding is off by at most 2^-8 (bf16) or 2^-11 (fp16) of the element and independent of the others; over sums of 2 f and of m terms
// it comes out in the norm as large as the rounding of d_x and d_weight themselves.  16384 x 1024 -> 4096 bf16: the gradients are off
// by 0.00234 of their norm, 0.00166 with dz in fp32 (fp16: 0.000293 and 0.000207).  dz in two 16-bit parts would take both products
// twice, 500 us more of 940.
#include <cstdio>

#include "hstu_ffn_common.h"
#include "hstu_gated_rows.h"

namespace hstu {

// ---- rows to 16-byte boundaries ------------------------------------------------------------------------------------------
// The product's copies move aligned 16-byte pieces.  An operand whose rows do not start on such boundaries, or end inside a
// piece, is first copied to rows of `ld` elements, zeros behind each row: x and W of 2789 x 1001 -> 2 * 2731 in fp16, 16.5 MB, in 10 us.
struct PadArgs { const void* src[2]; void* dst[2]; int64_t stride[2], rows[2]; int64_t ld; int32_t cols; };   // up to two operands, one launch
template <typename T>
__global__ __launch_bounds__(256) void hstu_pad_rows_kernel(const PadArgs a) {
    // a wave takes a row, a lane 8 elements at a time
    const int lane = threadIdx.x & 63;
    const int64_t n = a.rows[0] + a.rows[1];
    for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < n; i += (int64_t)gridDim.x * 4) {
        const int which = i >= a.rows[0];
        const int64_t r = which ? i - a.rows[0] : i;
        const T* src = reinterpret_cast<const T*>(a.src[which]) + r * a.stride[which];
        T* dst = reinterpret_cast<T*>(a.dst[which]) + r * a.ld;
        for (int c = lane * 8; c < a.ld; c += 512) {
            float v[8];
            load8_any(src + c, a.cols - c, v);
            store8_any<false>(dst + c, (int)(a.ld - c), v);   // (read again by the next launch)
        }
    }
}

// ---- dz ------------------------------------------------------------------------------------------------------------------
// A lane works on 8 consecutive columns of both halves and walks down its rows; `lanes` lanes side by side, 256 / lanes rows
// at a time.  HBM-bound: reads d_out and z, writes dz.  Columns [2 f, ld) of dz are set to zero (the product reads them).
// [16384, 4096] bf16: 805 MB in 140 to 153 us (5.8 to 5.3 TB/s, a large copy 4.9); with z in 8 bits, [16384, 2048], 52 us.  dz is stored
// through the caches, the products read it next (the whole backward 649 us past them, 635 so).  The next row
// under way while one is worked on was slower (8 bits 45 us for 37 at the time: the registers cost waves).
struct DzArgs {
    const void* d_out;
    const void* z;
    const uint8_t* z_aux;
    void* dz;              // [m, ld], or NULL
    float* partial;        // [row blocks, 2 f] column sums, or NULL
    int64_t m, dout_stride, ld;
    int64_t rows_wg;       // rows of a workgroup
    int32_t f, act, keep, lanes, col_blocks;
};

template <typename T>
__global__ __launch_bounds__(256) void hstu_gated_dz_kernel(const DzArgs a) {
    __shared__ float red[16][256 + 4];   // 16 columns of each of the 256 lanes
    const int lanes = a.lanes, tx = threadIdx.x & (lanes - 1), ty = threadIdx.x / lanes, step = 256 / lanes;
    const int cb = blockIdx.x % a.col_blocks;
    const int64_t rb = blockIdx.x / a.col_blocks;
    const int c = (cb * lanes + tx) * 8, n = a.f - c;
    const int64_t r0 = rb * a.rows_wg, r1 = min(r0 + a.rows_wg, a.m);
    const int64_t kept = HSTU_GATED_KEPT((int64_t)a.f);
    float sg[8], su[8];
#pragma unroll
    for (int k = 0; k < 8; k++) sg[k] = su[k] = 0.f;
    if (n > 0) {
        for (int64_t r = r0 + ty; r < r1; r += step) {
            float d[8], zg[8], zu[8];
            load8_any(reinterpret_cast<const T*>(a.d_out) + r * a.dout_stride + c, n, d);
            if (a.keep == HSTU_KEEP_8BIT) {
                const uint8_t* z = reinterpret_cast<const uint8_t*>(a.z) + r * 2 * kept + c;
                const uint8_t* e = a.z_aux + (r * 2 * kept + c) / HSTU_PACK8_GROUP;
                code_values(codes8_raw(z, 8, e[0]), largest_finite<float>(), zg);
                code_values(codes8_raw(z + kept, 8, e[kept / HSTU_PACK8_GROUP]), largest_finite<float>(), zu);
            } else if constexpr (sizeof(T) == 4) {
                const T* z = reinterpret_cast<const T*>(a.z) + r * 2 * kept + c;
                load8_any(z, 8, zg);
                load8_any(z + kept, 8, zu);
            } else {
                const T* z = reinterpret_cast<const T*>(a.z) + r * 2 * kept + 2 * c - (c & 31);   // blocks of 32: the gate's, the values'
                const uint8_t* low = a.z_aux + r * 2 * kept + c;
                const Raw8<T> ug = load8_raw(z, 8), uu = load8_raw(z + 32, 8);
                const Codes8 lg = codes8_raw(low, 8, 0), lu = codes8_raw(low + kept, 8, 0);
                join24(ug.q[0], lg.q, zg);
                join24(uu.q[0], lu.q, zu);
            }
            float dg[8], du[8], act[8], grad[8];
            act_and_grad<8>(zg, a.act, act, grad);
#pragma unroll
            for (int k = 0; k < 8; k++) {
                dg[k] = d[k] * zu[k] * grad[k];
                du[k] = d[k] * act[k];
                sg[k] += dg[k];
                su[k] += du[k];
            }
            if (a.dz) {
                T* dz = reinterpret_cast<T*>(a.dz) + r * a.ld + c;
                store8_any<false>(dz, n, dg);
                store8_any<false>(dz + a.f, n, du);
                if (n <= 8)
                    for (int64_t k = 2 * (int64_t)a.f; k < a.ld; k++) reinterpret_cast<T*>(a.dz)[r * a.ld + k] = from_float<T>(0.f);
            }
        }
    }
    if (!a.partial) return;
#pragma unroll
    for (int k = 0; k < 8; k++) {
        red[k][threadIdx.x] = sg[k];
        red[8 + k][threadIdx.x] = su[k];
    }
    __syncthreads();
    // column j of lane t: rows of the workgroup in order
    for (int i = threadIdx.x; i < lanes * 16; i += 256) {
        const int t = i >> 4, j = i & 15, col = (cb * lanes + t) * 8 + (j & 7);
        if (col >= a.f) continue;
        float s = 0.f;
        for (int y = 0; y < step; y++) s += red[j][y * lanes + t];
        a.partial[rb * 2 * a.f + (j >= 8 ? a.f : 0) + col] = s;
    }
}

// ---- partial sums ----------------------------------------------------------------------------------------------------------
// What the launches before it left in fp32 parts: shares of d_x and of d_weight, and the row blocks' column sums for d_bias, added
// in order and rounded once, all three in one launch.  A lane adds four neighbouring elements over the parts; where there are
// many (`slots` = 32), lane groups take every 32nd part and meet in LDS.  d_bias, with the most parts, comes first.  Two parts of
// [8192, 1024] with the d_bias of 16384 rows: 15 us.
struct SumArgs {
    const float* part[3];
    void* out[3];
    int64_t n[3];        // elements
    int64_t blocks[3];   // workgroups
    int32_t parts[3];
    int32_t slots[3];    // 1 or 32
    int32_t bias_f32;    // the first output's type
};
template <typename T>
__global__ __launch_bounds__(256) void hstu_sum_parts_kernel(const SumArgs a) {
    __shared__ gm_f32x4 red[256];
    int64_t block = blockIdx.x;
    int w = 0;
    while (w < 2 && block >= a.blocks[w]) block -= a.blocks[w++];
    const int slots = a.slots[w], across = 256 / slots, slot = threadIdx.x / across;
    const int64_t n = a.n[w], i = (block * across + threadIdx.x % across) * 4;
    typedef gm_f32x4 __attribute__((aligned(4))) f4;
    gm_f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if (i + 4 <= n) {
#pragma unroll 8
        for (int k = slot; k < a.parts[w]; k += slots) s += *reinterpret_cast<const f4*>(a.part[w] + k * n + i);
    } else {
        for (int k = slot; k < a.parts[w]; k += slots)
#pragma unroll
            for (int e = 0; e < 3; e++)
                if (i + e < n) s[e] += a.part[w][k * n + i + e];
    }
    if (slots > 1) {
        red[threadIdx.x] = s;
        for (int h = slots / 2; h > 0; h >>= 1) {
            __syncthreads();
            if (slot < h) red[threadIdx.x] += red[threadIdx.x + h * across];
        }
        if (slot) return;
        s = red[threadIdx.x];
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (i + e < n) {
            if (w == 0 && a.bias_f32) reinterpret_cast<float*>(a.out[w])[i + e] = s[e];
            else reinterpret_cast<T*>(a.out[w])[i + e] = from_float<T>(s[e]);
        }
}

// ---- host ------------------------------------------------------------------------------------------------------------------
static int elem_bytes(int32_t dtype) { return dtype == HSTU_F32 ? 4 : 2; }
static uint64_t up256(uint64_t v) { return (v + 255) / 256 * 256; }
static int64_t padded(int64_t cols, int32_t dtype) {
    const int e = 16 / elem_bytes(dtype);
    return (cols + e - 1) / e * e;
}
static bool needs_pad(const void* p, int64_t stride, int64_t cols, int32_t dtype) {
    const int e = 16 / elem_bytes(dtype);
    // (a tile's copies address up to 256 rows with 31 bits: rows further apart than 2^20 elements are brought together too)
    return (reinterpret_cast<uintptr_t>(p) & 15) || stride % e || cols % e || stride > (1 << 20);
}
static bool bad_align(const void* p, int32_t dtype) { return (reinterpret_cast<uintptr_t>(p) & (dtype == HSTU_F32 ? 3 : 1)) != 0; }

static hipError_t launch_gemm(int32_t dtype, const GemmArgs& a, int kind, int tile, hipStream_t st) {
    if (dtype == HSTU_F32) return launch_gemm_f32(a, kind, tile, st);
    if (dtype == HSTU_F16) return launch_gemm_f16(a, kind, tile, st);
    return launch_gemm_bf16(a, kind, tile, st);
}

// a launch holds less than 2^32 threads, a workgroup up to 512
constexpr int64_t GEMM_MAX_TILES = 0x7fffff;
struct Plan { int tile, splits, tiles_n, tiles_m; int64_t c_split; double us; };

// Tiles and shares of the contraction: the cheapest by a model of the launch, in microseconds.  A workgroup takes a start and an
// end (`fixed`) and `piece` for each piece of its share; workgroups come in rounds of what the chip holds at a time; shares
// beyond one cost a second kernel that adds their fp32 sums.
// Measured (bf16, a full chip): a piece of a 256 x 256 tile 1.7, of a 256 x 128 one 1.1, of a 128 x 128 one 0.6 alone on its CU with
// four buffers, 0.65 with two and 1.15 with two workgroups on a CU, of a 64 x 128 one 0.42 and 0.8.  fp32 products are bound by
// their matrix rate: 128 x 128 x 32 in 1.8, 64 x 128 x 32 in 0.95.  Over 129 products of random sizes, each timed in every tile,
// the choice is 0.3 % (forward), 0.8 % (d_x) and 1.5 % (d_weight) slower than the fastest in the mean, 12 % at worst; fp32 0, 3.5 and
// 1.2 %, 16 % at worst.  The times themselves are rough where a launch is short: the fp32 forward of
// 1123 x 240 -> 960 is reckoned 17.4 us in two tiles alike and takes 22 (26 with z kept).
// Each tile has the sizes where it is the fastest (forward, us: 256 x 256, 128 x 128, 256 x 128, 64 x 128):
//   2789 x 1008 x 2736 fp16 37 44 40 55;  16384 x 512 x 2048 bf16 90 91 87 109;  8000 x 128 x 512 bf16 10.4 7.5 7.5 9.0;
//   256 x 1024 x 4096 bf16 26 12.4 16 9.2;  100 x 2000 x 4000 fp32 473 134 245 74
// and 128 x 128 with four buffers where one workgroup per CU is left of a long contraction (d_x of 256 x 1024 x 4096 27.8, with two
// buffers 28.2; d_weight of 4096 x 512 x 2048 51.0 and 56.9).
static Plan gemm_plan(int kind, int32_t dtype, int64_t M, int64_t N, int64_t C) {
    const bool f32 = dtype == HSTU_F32;
    const int64_t bk = 128 / elem_bytes(dtype), pieces = (C + bk - 1) / bk;
    Plan best = {};
    double least = 1e300;
    for (int tile = 0; tile < GEMM_TILES; tile++) {   // (the first one also takes what would be too many tiles of the others)
        if (f32 && tile == TILE_128_DEEP) continue;   // (never the fastest: the copies of two buffers keep ahead of the matrix rate)
        const int64_t tm = (M + gemm_tile_m(tile) - 1) / gemm_tile_m(tile), tn = (N + gemm_tile_n(tile, kind) - 1) / gemm_tile_n(tile, kind);
        for (int splits = 1; splits <= 64; splits *= 2) {
            if (splits > 1 && (kind == GEMM_GATED || pieces < 2 * splits)) break;
            if (tm * tn * splits > GEMM_MAX_TILES && (tile != TILE_256 || splits > 1)) break;
            const double wgs = (double)tm * tn * splits, share = (double)((pieces + splits - 1) / splits);
            const bool pairs = (tile == TILE_128 || tile == TILE_64x128) && wgs > 256;   // two workgroups on a CU
            const double piece16[GEMM_TILES] = {1.7, pairs ? 1.15 : 0.65, 0.6, 1.1, pairs ? 0.8 : 0.42};
            const double piece32[GEMM_TILES] = {7.0, pairs ? 3.6 : 1.8, 0.0, 3.5, pairs ? 1.8 : 0.95};
            const double fixed_us[GEMM_TILES] = {6.0, pairs ? 4.0 : 3.0, 4.0, 4.5, pairs ? 3.0 : 2.5};
            const double piece = f32 ? piece32[tile] : piece16[tile], fixed = fixed_us[tile];
            const double rounds = (double)(int64_t)((wgs + 255) / 256) * (pairs ? 0.5 : 1.0);
            double t = rounds * (fixed + share * piece);
            if (splits > 1) t += 4.0 + (double)splits * M * N * 8 / 4.5e6;
            if (t < least) {
                least = best.us = t;
                best.tile = tile;
                best.tiles_m = (int)tm;
                best.tiles_n = (int)tn;
                best.splits = splits;
            }
        }
    }
    best.c_split = (pieces + best.splits - 1) / best.splits * bk;
    if (C > 0) best.splits = (int)((C + best.c_split - 1) / best.c_split);
    else best.c_split = bk;
    return best;
}

static int gemm_too_large(const Plan& p) {
    if ((int64_t)p.tiles_m * p.tiles_n * p.splits > GEMM_MAX_TILES) return fail(HSTU_ERR_UNSUPPORTED, "m * f too large for one launch");
    return HSTU_OK;
}

static void fill(GemmArgs& a, const Plan& pl, int64_t M, int64_t N, int64_t C) {
    a.M = M; a.N = (int32_t)N; a.C = C;
    a.c_split = pl.c_split; a.splits = pl.splits; a.tiles_m = pl.tiles_m; a.tiles_n = pl.tiles_n;
}

// x (where `x` is given a place) and weight (likewise) to rows of `ld` elements
static hipError_t launch_pad(int32_t dtype, const void* x, int64_t x_stride, int64_t m, void* x_to, const void* w, int64_t f2, void* w_to, int k, int64_t ld, hipStream_t st) {
    PadArgs a = {};
    a.ld = ld;
    a.cols = k;
    a.src[0] = x; a.stride[0] = x_stride; a.dst[0] = x_to; a.rows[0] = x_to ? m : 0;
    a.src[1] = w; a.stride[1] = k; a.dst[1] = w_to; a.rows[1] = w_to ? f2 : 0;
    const int64_t rows = a.rows[0] + a.rows[1];
    if (rows == 0) return hipSuccess;
    const int64_t want = (rows + 3) / 4;
    const dim3 grid((unsigned)(want > 4096 ? 4096 : want));
    if (dtype == HSTU_F32) hipLaunchKernelGGL(hstu_pad_rows_kernel<float>, grid, dim3(256), 0, st, a);
    else if (dtype == HSTU_F16) hipLaunchKernelGGL(hstu_pad_rows_kernel<_Float16>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(hstu_pad_rows_kernel<__bf16>, grid, dim3(256), 0, st, a);
    return hipGetLastError();
}

static int gated_check_sizes(int32_t dtype, int32_t act, int32_t keep, int64_t m, int32_t k, int32_t f) {
    if (dtype != HSTU_F32 && dtype != HSTU_F16 && dtype != HSTU_BF16)
        return fail(HSTU_ERR_INVALID_ARGUMENT, "dtype expect float32, float16 or bfloat16, but value is %d", dtype);
    if (act != HSTU_ACT_SILU && act != HSTU_ACT_GELU) return fail(HSTU_ERR_INVALID_ARGUMENT, "act expect 0 (silu) or 1 (gelu), but value is %d", act);
    if (keep != HSTU_KEEP_NONE && keep != HSTU_KEEP_FULL && keep != HSTU_KEEP_8BIT) return fail(HSTU_ERR_INVALID_ARGUMENT, "keep expect 0, 1 or 2, but value is %d", keep);
    if (keep == HSTU_KEEP_8BIT && dtype == HSTU_F32) return fail(HSTU_ERR_INVALID_ARGUMENT, "8-bit checkpoints need float16 or bfloat16");
    if (m < 0 || m > HSTU_FFN_MAX_ROWS) return fail(HSTU_ERR_INVALID_ARGUMENT, "x dim0 must in range:[0,%lld].", HSTU_FFN_MAX_ROWS);
    if (k < 1 || k > HSTU_GATED_MAX_K) return fail(HSTU_ERR_INVALID_ARGUMENT, "x dim1 must in range:[1,%d].", HSTU_GATED_MAX_K);
    if (f < 1 || f > HSTU_GATED_MAX_F) return fail(HSTU_ERR_INVALID_ARGUMENT, "weight dim0 must be twice a number in range:[1,%d].", HSTU_GATED_MAX_F);
    return HSTU_OK;
}

// Few rows go to the kernel that reads W straight into fragments where a model of both says that it is faster than tiles, most rows
// of which are empty.  A workgroup of that kernel reads 32 rows of W and all of x, at a rate that two on a CU (up to 32 rows) or one have;
// neither kernel reads W faster than memory gives it.  Measured (bf16, us, few rows / tiles):
//   1024 -> 4096: one row 3.4 / 7.9, 48 4.7 / 8.1, 64 5.5 / 8.3;   -> 8192: 32 rows 5.7 / 7.9, 48 8.9 / 8.1, 64 10.8 / 8.3;
//   512 -> 16384: one row 5.0 / 5.4, 32 7.7 / 5.8;   2048 -> 8192: 1 11.4 / 13.0, 48 16.1 / 13.5;   8192 -> 1024: 1 10.1 / 42, 64 20 / 43
// (It takes 16 bytes of a row at a time, at 32-bit offsets within 16 rows.)
static bool few_rows(const hstu_gated_params* p) {
    const double e = elem_bytes(p->dtype);
    if (p->m > ROWS_MAX_M || p->k < 16 / e || (p->m > 1 && p->x_stride > (1 << 20))) return false;
    const int64_t mb = (p->m + 15) / 16, wgs = (p->f + 15) / 16;
    const bool two = mb <= 2;
    const double share = two && wgs > 256 ? 2 : 1, rounds = (double)((wgs + (two ? 511 : 255)) / (two ? 512 : 256));
    const double bytes = (32.0 + 16.0 * mb) * p->k * e * share, fp32 = p->dtype == HSTU_F32 ? 1.9e-3 * share * mb * p->k : 0.0;
    const double rows_us = 1.0 + rounds * (2.0 + bytes / (two ? 95e3 : 58e3) + fp32), least = 2.2 + 2.0 * p->f * p->k * e / 6.9e6;
    const double pad = needs_pad(p->weight, p->k, p->k, p->dtype) ? 4.0 + 2.0 * p->f * p->k * e / 2e6 : 0.0;   // (1001 -> 6001: 24 MB, 16 us)
    const double tiles_us = pad + (p->dtype == HSTU_F32 ? 1.15 : 0.87) * gemm_plan(GEMM_GATED, p->dtype, p->m, p->f, p->k).us;
    return (rows_us > least ? rows_us : least) < (tiles_us > least ? tiles_us : least);
}

struct GatedLayout { uint64_t x, w, bytes; bool pad_x, pad_w; };
static GatedLayout gated_layout(const hstu_gated_params* p) {
    GatedLayout l;
    const uint64_t e = elem_bytes(p->dtype), ld = padded(p->k, p->dtype);
    if (few_rows(p)) { l = {}; return l; }
    l.pad_x = p->m > 0 && needs_pad(p->x, p->m > 1 ? p->x_stride : ld, p->k, p->dtype);
    l.pad_w = p->m > 0 && needs_pad(p->weight, p->k, p->k, p->dtype);
    l.x = 0;
    l.w = l.pad_x ? up256(p->m * ld * e) : 0;
    l.bytes = l.w + (l.pad_w ? up256(2 * (uint64_t)p->f * ld * e) : 0);
    return l;
}

static int gated_validate(const hstu_gated_params* p) {
    if (!p) return fail(HSTU_ERR_INVALID_ARGUMENT, "params is NULL");
    if (p->struct_size != sizeof(hstu_gated_params))
        return fail(HSTU_ERR_INVALID_ARGUMENT, "hstu_gated_params size mismatch: caller %u, library %zu", p->struct_size, sizeof(hstu_gated_params));
    const int rc = gated_check_sizes(p->dtype, p->act, p->keep, p->m, p->k, p->f);
    if (rc != HSTU_OK) return rc;
    if (p->bias_dtype != p->dtype && p->bias_dtype != HSTU_F32) return fail(HSTU_ERR_INVALID_ARGUMENT, "bias_dtype expect float32 or the dtype of x, but value is %d", p->bias_dtype);
    if (p->x_stride < 0) return fail(HSTU_ERR_INVALID_ARGUMENT, "x_stride must not be negative");
    if (p->m == 0) return HSTU_OK;
    if (!p->x || !p->weight || !p->out) return fail(HSTU_ERR_INVALID_ARGUMENT, "x, weight and out must not be NULL");
    if (p->keep != HSTU_KEEP_NONE && (!p->z || (p->dtype != HSTU_F32 && !p->z_aux)))
        return fail(HSTU_ERR_INVALID_ARGUMENT, "z (and z_aux for 16-bit dtypes) must not be NULL when z is kept");
    if (bad_align(p->x, p->dtype) || bad_align(p->weight, p->dtype) || bad_align(p->out, p->dtype) || bad_align(p->bias, p->bias_dtype) ||
        (p->keep == HSTU_KEEP_FULL && bad_align(p->z, p->dtype)))
        return fail(HSTU_ERR_UNSUPPORTED, "x, weight, bias, out and z must be aligned to their element types");
    return HSTU_OK;
}

struct GatedBwdLayout {
    Plan dx, dw;
    int64_t ld, kld;                 // rows of dz, padded rows of x / weight
    bool need_dz, pad_x, pad_w;
    uint64_t dz, x, w, parts_x, parts_w, sums, bytes;
    int lanes, col_blocks;
    int64_t rows_wg, row_blocks;
};

static GatedBwdLayout gated_bwd_layout(const hstu_gated_bwd_params* p) {
    GatedBwdLayout l;
    const uint64_t e = elem_bytes(p->dtype);
    l.ld = padded(2 * (int64_t)p->f, p->dtype);
    l.kld = padded(p->k, p->dtype);
    l.need_dz = p->d_x || p->d_weight;
    l.pad_x = p->d_weight && p->m > 0 && needs_pad(p->x, p->m > 1 ? p->x_stride : l.kld, p->k, p->dtype);
    l.pad_w = p->d_x && p->m > 0 && needs_pad(p->weight, p->k, p->k, p->dtype);
    l.dx = gemm_plan(GEMM_DX, p->dtype, p->m, p->k, 2 * (int64_t)p->f);
    l.dw = gemm_plan(GEMM_DW, p->dtype, 2 * (int64_t)p->f, p->k, p->m);
    // about 2048 workgroups, but at least four rows a lane where there are as many
    l.lanes = 8;
    while (l.lanes < 64 && l.lanes * 8 < p->f) l.lanes *= 2;
    l.col_blocks = (p->f + l.lanes * 8 - 1) / (l.lanes * 8);
    const int64_t step = 256 / l.lanes;
    int64_t rows = (p->m * l.col_blocks + 2047) / 2048;
    rows = (rows + step - 1) / step * step;
    l.rows_wg = rows < 4 * step ? 4 * step : rows;
    l.row_blocks = (p->m + l.rows_wg - 1) / l.rows_wg;
    if (l.row_blocks < 1) l.row_blocks = 1;
    uint64_t at = 0;
    l.dz = at;
    if (l.need_dz) at += up256((uint64_t)p->m * l.ld * e);
    l.x = at;
    if (l.pad_x) at += up256((uint64_t)p->m * l.kld * e);
    l.w = at;
    if (l.pad_w) at += up256(2 * (uint64_t)p->f * l.kld * e);
    l.parts_x = at;
    if (p->d_x && l.dx.splits > 1) at += up256((uint64_t)l.dx.splits * p->m * p->k * 4);
    l.parts_w = at;
    if (p->d_weight && l.dw.splits > 1) at += up256((uint64_t)l.dw.splits * 2 * p->f * p->k * 4);
    l.sums = at;
    if (p->d_bias) at += up256((uint64_t)l.row_blocks * 2 * p->f * 4);
    l.bytes = at;
    return l;
}

static int gated_bwd_validate(const hstu_gated_bwd_params* p) {
    if (!p) return fail(HSTU_ERR_INVALID_ARGUMENT, "params is NULL");
    if (p->struct_size != sizeof(hstu_gated_bwd_params))
        return fail(HSTU_ERR_INVALID_ARGUMENT, "hstu_gated_bwd_params size mismatch: caller %u, library %zu", p->struct_size, sizeof(hstu_gated_bwd_params));
    const int rc = gated_check_sizes(p->dtype, p->act, p->keep, p->m, p->k, p->f);
    if (rc != HSTU_OK) return rc;
    if (p->keep == HSTU_KEEP_NONE) return fail(HSTU_ERR_INVALID_ARGUMENT, "keep expect 1 or 2, but value is 0");
    if (p->grad_bias_dtype != p->dtype && p->grad_bias_dtype != HSTU_F32)
        return fail(HSTU_ERR_INVALID_ARGUMENT, "grad_bias_dtype expect float32 or the dtype of x, but value is %d", p->grad_bias_dtype);
    if (p->x_stride < 0 || p->dout_stride < 0) return fail(HSTU_ERR_INVALID_ARGUMENT, "x_stride and dout_stride must not be negative");
    if (p->m > 0) {
        if (!p->d_out || !p->z || (p->dtype != HSTU_F32 && !p->z_aux))
            return fail(HSTU_ERR_INVALID_ARGUMENT, "d_out and z (and z_aux for 16-bit dtypes) must not be NULL");
        if ((p->d_weight && !p->x) || (p->d_x && !p->weight)) return fail(HSTU_ERR_INVALID_ARGUMENT, "x (for d_weight) and weight (for d_x) must not be NULL");
    }
    if (bad_align(p->d_out, p->dtype) || bad_align(p->x, p->dtype) || bad_align(p->weight, p->dtype) || bad_align(p->d_x, p->dtype) ||
        bad_align(p->d_weight, p->dtype) || bad_align(p->d_bias, p->grad_bias_dtype) || (p->keep == HSTU_KEEP_FULL && bad_align(p->z, p->dtype)))
        return fail(HSTU_ERR_UNSUPPORTED, "d_out, x, weight, z and the gradients must be aligned to their element types");
    return HSTU_OK;
}

static int check_workspace(void* ws, uint64_t have, uint64_t need) {
    if (need && (!ws || have < need || (reinterpret_cast<uintptr_t>(ws) & 15)))
        return fail(HSTU_ERR_WORKSPACE, "workspace of %llu bytes (16-byte aligned) needed, got %llu at %p", (unsigned long long)need, (unsigned long long)have, ws);
    return HSTU_OK;
}

static void add_sum(SumArgs& a, int which, const void* part, int64_t parts, int64_t n, void* out) {
    a.part[which] = reinterpret_cast<const float*>(part);
    a.parts[which] = (int32_t)parts;
    a.n[which] = n;
    a.out[which] = out;
    a.slots[which] = parts > 16 ? 32 : 1;
    const int64_t per = 256 / a.slots[which] * 4;
    a.blocks[which] = (n + per - 1) / per;
}
static hipError_t launch_sums(int32_t dtype, SumArgs& a, hipStream_t st) {
    const int64_t blocks = a.blocks[0] + a.blocks[1] + a.blocks[2];
    if (blocks == 0) return hipSuccess;
    for (int i = 0; i < 3; i++)
        if (!a.slots[i]) a.slots[i] = 1;
    const dim3 grid((unsigned)blocks);
    if (dtype == HSTU_F32) hipLaunchKernelGGL(hstu_sum_parts_kernel<float>, grid, dim3(256), 0, st, a);
    else if (dtype == HSTU_F16) hipLaunchKernelGGL(hstu_sum_parts_kernel<_Float16>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(hstu_sum_parts_kernel<__bf16>, grid, dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace hstu

using namespace hstu;

extern "C" int hstu_hip_gated_linear_get_workspace_size(const hstu_gated_params* p, uint64_t* bytes) {
    if (!bytes) return fail(HSTU_ERR_INVALID_ARGUMENT, "workspace_bytes is NULL");
    const int rc = gated_validate(p);
    if (rc != HSTU_OK) return rc;
    *bytes = gated_layout(p).bytes;
    return HSTU_OK;
}

extern "C" int hstu_hip_gated_linear(const hstu_gated_params* p, void* workspace, uint64_t workspace_bytes, void* stream) {
    int rc = gated_validate(p);
    if (rc != HSTU_OK || p->m == 0) return rc;
    const GatedLayout l = gated_layout(p);
    rc = check_workspace(workspace, workspace_bytes, l.bytes);
    if (rc != HSTU_OK) return rc;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (few_rows(p)) {
        RowsArgs a = {};
        a.x = p->x; a.weight = p->weight; a.bias = p->bias; a.out = p->out; a.z = p->z; a.z_aux = p->z_aux;
        a.x_stride = p->x_stride;
        a.m = (int32_t)p->m; a.k = p->k; a.f = p->f; a.bias_f32 = p->bias_dtype == HSTU_F32; a.act = p->act; a.keep = p->keep;
        const hipError_t e = p->dtype == HSTU_F32 ? launch_gated_rows_f32(a, st) : p->dtype == HSTU_F16 ? launch_gated_rows_f16(a, st) : launch_gated_rows_bf16(a, st);
        if (e != hipSuccess) return fail(HSTU_ERR_LAUNCH, "kernel launch failed: %s", hipGetErrorString(e));
        return HSTU_OK;
    }
    const Plan pl = gemm_plan(GEMM_GATED, p->dtype, p->m, p->f, p->k);
    rc = gemm_too_large(pl);
    if (rc != HSTU_OK) return rc;
    char* ws = reinterpret_cast<char*>(workspace);
    const int64_t ld = padded(p->k, p->dtype);
    hipError_t e = launch_pad(p->dtype, p->x, p->x_stride, p->m, l.pad_x ? ws + l.x : nullptr, p->weight, 2 * (int64_t)p->f, l.pad_w ? ws + l.w : nullptr, p->k, ld, st);
    if (e == hipSuccess) {
        GemmArgs a = {};
        fill(a, pl, p->m, p->f, p->k);
        a.n_op = l.pad_w ? ws + l.w : p->weight;
        a.n_ld = l.pad_w ? ld : p->k;
        a.m_op = l.pad_x ? ws + l.x : p->x;
        a.m_ld = l.pad_x ? ld : p->m > 1 ? p->x_stride : ld;
        a.out = p->out;
        a.bias = p->bias;
        a.bias_f32 = p->bias_dtype == HSTU_F32;
        a.act = p->act;
        a.keep = p->keep;
        a.z = p->z;
        a.z_aux = p->z_aux;
        e = launch_gemm(p->dtype, a, GEMM_GATED, pl.tile, st);
    }
    if (e != hipSuccess) return fail(HSTU_ERR_LAUNCH, "kernel launch failed: %s", hipGetErrorString(e));
    return HSTU_OK;
}

static const char* const TYPE_NAMES[3] = {"f32", "f16", "bf16"};
static const char* const TILE_NAMES[GEMM_TILES] = {"256x256", "128x128", "128x128_deep", "256x128", "64x128"};
static_assert(HSTU_F32 == 0 && HSTU_F16 == 1 && HSTU_BF16 == 2, "in the order of TYPE_NAMES");

extern "C" int hstu_hip_gated_linear_describe_kernel(const hstu_gated_params* p, char* buf, size_t n) {
    if (!buf || n == 0) return fail(HSTU_ERR_INVALID_ARGUMENT, "buf is NULL");
    const int rc = gated_validate(p);
    if (rc != HSTU_OK) return rc;
    if (p->m > 0 && few_rows(p)) snprintf(buf, n, "rows_%s_%d", TYPE_NAMES[p->dtype], (int)(p->m + 15) / 16 * 16);
    else snprintf(buf, n, "tiles_%s_%s", TYPE_NAMES[p->dtype], TILE_NAMES[gemm_plan(GEMM_GATED, p->dtype, p->m, p->f, p->k).tile]);
    return HSTU_OK;
}

extern "C" int hstu_hip_gated_linear_backward_describe_kernel(const hstu_gated_bwd_params* p, char* buf, size_t n) {
    if (!buf || n == 0) return fail(HSTU_ERR_INVALID_ARGUMENT, "buf is NULL");
    const int rc = gated_bwd_validate(p);
    if (rc != HSTU_OK) return rc;
    const GatedBwdLayout l = gated_bwd_layout(p);
    const char* t = TYPE_NAMES[p->dtype];
    snprintf(buf, n, "dx_%s_%s_%d dw_%s_%s_%d", t, TILE_NAMES[l.dx.tile], l.dx.splits, t, TILE_NAMES[l.dw.tile], l.dw.splits);
    return HSTU_OK;
}

extern "C" int hstu_hip_gated_linear_backward_get_workspace_size(const hstu_gated_bwd_params* p, uint64_t* bytes) {
    if (!bytes) return fail(HSTU_ERR_INVALID_ARGUMENT, "workspace_bytes is NULL");
    const int rc = gated_bwd_validate(p);
    if (rc != HSTU_OK) return rc;
    *bytes = gated_bwd_layout(p).bytes;
    return HSTU_OK;
}

extern "C" int hstu_hip_gated_linear_backward(const hstu_gated_bwd_params* p, void* workspace, uint64_t workspace_bytes, void* stream) {
    int rc = gated_bwd_validate(p);
    if (rc != HSTU_OK) return rc;
    const GatedBwdLayout l = gated_bwd_layout(p);
    rc = check_workspace(workspace, workspace_bytes, l.bytes);
    if (rc != HSTU_OK) return rc;
    if (p->d_x && (rc = gemm_too_large(l.dx)) != HSTU_OK) return rc;
    if (p->d_weight && (rc = gemm_too_large(l.dw)) != HSTU_OK) return rc;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    char* ws = reinterpret_cast<char*>(workspace);
    hipError_t e = hipSuccess;
    SumArgs sums = {};
    sums.bias_f32 = p->grad_bias_dtype == HSTU_F32;
    if (l.need_dz || p->d_bias) {
        DzArgs d = {};
        d.d_out = p->d_out; d.z = p->z; d.z_aux = p->z_aux;
        d.dz = l.need_dz ? ws + l.dz : nullptr;
        d.partial = p->d_bias ? reinterpret_cast<float*>(ws + l.sums) : nullptr;
        d.m = p->m; d.dout_stride = p->dout_stride; d.ld = l.ld; d.rows_wg = l.rows_wg;
        d.f = p->f; d.act = p->act; d.keep = p->keep; d.lanes = l.lanes; d.col_blocks = l.col_blocks;
        // without rows the workgroups write zero sums
        const dim3 grid((unsigned)(l.row_blocks * l.col_blocks));
        if (p->dtype == HSTU_F32) hipLaunchKernelGGL(hstu_gated_dz_kernel<float>, grid, dim3(256), 0, st, d);
        else if (p->dtype == HSTU_F16) hipLaunchKernelGGL(hstu_gated_dz_kernel<_Float16>, grid, dim3(256), 0, st, d);
        else hipLaunchKernelGGL(hstu_gated_dz_kernel<__bf16>, grid, dim3(256), 0, st, d);
        e = hipGetLastError();
        // where a product leaves parts too, the column sums are added in the same launch as those; alone, while they are in the L2
        const bool parts = (p->d_x && p->m > 0 && l.dx.splits > 1) || (p->d_weight && l.dw.splits > 1);
        if (p->d_bias && parts) add_sum(sums, 0, d.partial, l.row_blocks, 2 * (int64_t)p->f, p->d_bias);
        else if (e == hipSuccess && p->d_bias) {
            char* db = reinterpret_cast<char*>(p->d_bias);
            e = launch_colsum(d.partial, (int)l.row_blocks, p->f, db, db + (int64_t)p->f * elem_bytes(p->grad_bias_dtype), p->grad_bias_dtype, st);
        }
    }
    if (e == hipSuccess)
        e = launch_pad(p->dtype, p->x, p->x_stride, p->m, l.pad_x ? ws + l.x : nullptr, p->weight, 2 * (int64_t)p->f, l.pad_w ? ws + l.w : nullptr, p->k, l.kld, st);
    if (e == hipSuccess && p->d_x && p->m > 0) {
        GemmArgs a = {};
        fill(a, l.dx, p->m, p->k, 2 * (int64_t)p->f);
        a.n_op = l.pad_w ? ws + l.w : p->weight;
        a.n_ld = l.pad_w ? l.kld : p->k;
        a.m_op = ws + l.dz;
        a.m_ld = l.ld;
        a.out = l.dx.splits > 1 ? ws + l.parts_x : p->d_x;
        e = launch_gemm(p->dtype, a, GEMM_DX, l.dx.tile, st);
        if (l.dx.splits > 1) add_sum(sums, 1, ws + l.parts_x, l.dx.splits, p->m * p->k, p->d_x);
    }
    if (e == hipSuccess && p->d_weight) {
        // without rows the product of empty sums writes zeros
        GemmArgs a = {};
        fill(a, l.dw, 2 * (int64_t)p->f, p->k, p->m);
        a.n_op = l.pad_x ? ws + l.x : p->x;
        a.n_ld = l.pad_x ? l.kld : p->m > 1 ? p->x_stride : l.kld;
        a.m_op = ws + l.dz;
        a.m_ld = l.ld;
        a.out = l.dw.splits > 1 ? ws + l.parts_w : p->d_weight;
        e = launch_gemm(p->dtype, a, GEMM_DW, l.dw.tile, st);
        if (l.dw.splits > 1) add_sum(sums, 2, ws + l.parts_w, l.dw.splits, 2 * (int64_t)p->f * p->k, p->d_weight);
    }
    if (e == hipSuccess) e = launch_sums(p->dtype, sums, st);
    if (e != hipSuccess) return fail(HSTU_ERR_LAUNCH, "kernel launch failed: %s", hipGetErrorString(e));
    return HSTU_OK;
}
