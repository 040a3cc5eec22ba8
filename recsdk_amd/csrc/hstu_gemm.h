// Matrix-core product of the gated projection and of its backward: out[m, n] = sum over c of M[m, c] * N[n, c].
//
// A workgroup owns BM x BN outputs and walks the contraction in pieces of 128 bytes (64 columns of 16 bits, 32 of fp32).
// Both operands of a piece are copied global -> LDS by buffer loads that write LDS directly, into a ring of two to four
// buffers, while the matrix cores work on an older one; one barrier per piece.  The MFMA is issued with the n side as its A
// operand, so that an accumulator register quad holds four consecutive n of one row m and a lane exchange of the two
// half-waves makes 16-byte pieces of an output row.
//
// An operand lies in memory either with the contraction contiguous (KC: element (row, c) at row * ld + c) or with the rows
// contiguous (RC: c * ld + row).  In LDS a KC operand is [rows][128 B], 16-byte chunk c of row r at position
// c ^ ((r >> 1) & 7): a fragment is one 16-byte LDS read, and 16 rows of one chunk cover all 64 banks.  An RC operand is
// [c][rows], read with the transposing LDS load (four c of one row per lane), fp32 four bytes a lane; its chunks are turned
// (line_swizzle) so that the lines that such a load touches lie in different banks.  Counters show no bank conflicts.
// Out-of-range rows and c are never addressed: their loads carry an offset beyond the buffer and return zero.
//
// Bounded by the matrix cores once a product fills the chip: [8192, 8192] outputs over c = 8192 reach 1340 TFLOP/s in bf16, and
// one large library product 1351.  Below that it is the start and the end of a tile that cost, 5 to 7 us per round of tiles: the
// gated forward at 8192 x 1024 -> 2 * 4096, whose contraction is 16 pieces and whose end computes the activation, takes 124 to 134 us
// (1110 to 1025 TFLOP/s; with GELU, whose 16 library erfc a block have nothing beside them there, 150 to 156), and its counters show the
// matrix cores busy for 45 % of it; 16384 rows with kept z take 303 us.
// Tried at that size and slower: four waves of 128 x 128 (263 us against 140 at the time: no second wave covers the end of the
// first), the next lines called into L2 early (143), accumulators that start at the bias (145), workgroups that go on to their
// next tile and start its copies before their end (140, and registers spilled).
#pragma once
#include "hstu_ffn_common.h"

namespace hstu {

typedef __attribute__((ext_vector_type(8))) __bf16 gm_bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 gm_f16x8;
typedef __attribute__((ext_vector_type(2))) __bf16 gm_bf16x2;
typedef __attribute__((ext_vector_type(2))) _Float16 gm_f16x2;
typedef __attribute__((ext_vector_type(4))) short gm_s16x4;
typedef __attribute__((ext_vector_type(8))) short gm_s16x8;
typedef __attribute__((ext_vector_type(16))) float gm_f32x16;
typedef __attribute__((ext_vector_type(4))) float gm_f32x4;
typedef __attribute__((ext_vector_type(2))) float gm_f32x2;
typedef __attribute__((ext_vector_type(4))) unsigned int gm_u4;
typedef __attribute__((ext_vector_type(2))) unsigned int gm_u2;

#define GM_LDS(type, p) ((__attribute__((address_space(3))) type*)(p))

struct GemmArgs {
    const void* n_op;      // n side: [N, C] (KC) or [C, N] (RC)
    const void* m_op;      // m side: [M, C] (KC) or [C, M] (RC)
    int64_t n_ld, m_ld;    // elements; rows of both operands start on 16-byte boundaries
    int64_t M;
    int64_t C;             // length of the contraction
    int64_t c_split;       // length of a workgroup's share of it (a multiple of the piece), C without a split
    int32_t N;             // plain: columns of out; gated: f (the n operand has 2 f rows)
    int32_t splits;
    int32_t tiles_n, tiles_m;
    void* out;             // [M, N] of T; with splits > 1: fp32 [splits, M, N]
    // gated epilogue
    const void* bias;
    int32_t bias_f32;
    int32_t act;
    int32_t keep;
    void* z;
    uint8_t* z_aux;
};

template <typename T> struct GM;
template <> struct GM<__bf16> {
    typedef gm_bf16x8 frag;
    static __device__ __forceinline__ gm_f32x16 mfma(frag a, frag b, gm_f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ unsigned pack2(float x, float y) { gm_bf16x2 r; r[0] = (__bf16)x; r[1] = (__bf16)y; return __builtin_bit_cast(unsigned, r); }
};
template <> struct GM<_Float16> {
    typedef gm_f16x8 frag;
    static __device__ __forceinline__ gm_f32x16 mfma(frag a, frag b, gm_f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ unsigned pack2(float x, float y) { gm_f16x2 r; r[0] = (_Float16)x; r[1] = (_Float16)y; return __builtin_bit_cast(unsigned, r); }
};
template <> struct GM<float> {
    typedef gm_f32x4 frag;   // four consecutive c: four MFMAs of two c each (half-wave g holds c 4 g .. 4 g + 3 of eight)
    static __device__ __forceinline__ gm_f32x16 mfma(frag a, frag b, gm_f32x16 c) {
#pragma unroll
        for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
};

// 16 bytes to an address of any alignment; the first `n` of the elements only where n is smaller
typedef gm_u4 __attribute__((aligned(1))) gm_u4_any;
template <typename T> __device__ __forceinline__ void store16(T* p, gm_u4 v, int n) {
    constexpr int E = 16 / sizeof(T);
    if (n >= E) *reinterpret_cast<gm_u4_any*>(p) = v;
    else {
        T e[E];
        __builtin_memcpy(e, &v, 16);
#pragma unroll
        for (int i = 0; i < E; i++)
            if (i < n) p[i] = e[i];
    }
}

// lane exchange between the half-waves: (a, b) of lane l and of lane l + 32 become (a_l, a_{l+32}) and (b_l, b_{l+32})
__device__ __forceinline__ void swap_halves(unsigned& a, unsigned& b) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0];
    b = r[1];
}

template <int N> struct gm_const { static constexpr int value = N; };

// ---- the kernel -----------------------------------------------------------------------------------------------------------
// GATE: -1 for a plain product, gate_of(act, keep) for the gated projection.  The end of a gated tile is long unrolled code, an
// instance for each of its activations and kept formats: with one for all of them, behind branches, the forward of 1024 x 512 -> 2048
// bf16 took 9.1 us for 8.6, that of 16384 x 1024 -> 4096 with kept z 314 for 309.
constexpr int gate_of(int act, int keep) { return act << 2 | keep; }
template <typename T_, bool NRC_, bool MRC_, int BN_, int BM_, int WN_, int WM_, int STAGES_, int GATE_>
struct GemmShape {
    typedef T_ T;
    static constexpr bool NRC = NRC_, MRC = MRC_, GATED = GATE_ >= 0;
    static constexpr int ACT = GATE_ >> 2, KEEP = GATE_ & 3;      // of a gated one
    static constexpr int ES = sizeof(T), EC = 16 / ES;            // bytes of an element, elements of a 16-byte chunk
    static constexpr int BN = BN_, BM = BM_, BK = 128 / ES;
    static constexpr int WN = WN_, WM = WM_, NW = WN * WM, NT = 64 * NW;
    static constexpr int NB = BN / WN / 32, MB = BM / WM / 32;    // 32 x 32 blocks of a wave
    static constexpr int NI = BN / 8 / NW, MI = BM / 8 / NW;      // 1 KiB copies of a wave per piece and operand
    static constexpr int N_BYTES = BN * 128, STAGE = (BN + BM) * 128, STAGES = STAGES_;
    static constexpr int STEPS = 4;                               // fragment steps per piece: 16 columns c of 16 bits, 8 of fp32
    static_assert(!GATED || (NB % 2 == 0 && !NRC), "a gated wave holds blocks of the gate and the matching ones of the values");
    static_assert(BN % (8 * NW) == 0 && BM % (8 * NW) == 0, "whole copies per wave");
};

// what a chunk's place in line c of an RC operand is turned by: the four lines that a transposing load touches (the two, for
// fp32) lie in different banks
template <int ES, int LINE> __device__ __forceinline__ int line_swizzle(int c) {
    if (ES == 4) return 8 * ((c >> 2) & 1);
    return LINE >= 256 ? 4 * (c & 3) : 4 * ((c >> 1) & 1);
}

// offsets of one operand's copies: 1 KiB piece i of this wave
template <typename S, bool RC, int ROWS, int CNT> struct Stager {
    unsigned voff[CNT];
    int c_of[CNT];   // first c (within the piece) that this lane's chunk of copy i holds

    // `rows`: valid rows from the tile's first one (of each half of a gated n operand)
    __device__ __forceinline__ void init(int w, int lane, int64_t ld, int64_t rows, bool gated) {
        constexpr int ES = S::ES, EC = S::EC;
#pragma unroll
        for (int i = 0; i < CNT; i++) {
            const int p = w + S::NW * i;
            if constexpr (!RC) {
                const int r = 8 * p + (lane >> 3);
                const int chunk = (lane & 7) ^ ((r >> 1) & 7);
                const int row = gated && r >= ROWS / 2 ? r - ROWS / 2 : r;
                c_of[i] = chunk * EC;
                voff[i] = row < rows ? (unsigned)(row * ld * ES + chunk * 16) : 0x80000000u;
            } else {
                constexpr int LINE = ROWS * ES;                 // bytes of a line c in LDS
                constexpr int LPL = LINE / 16;                  // lanes per line
                static_assert(LPL <= 64, "a copy holds whole lines");
                const int c = p * (1024 / LINE) + lane / LPL;
                const int chunk = (lane % LPL) ^ line_swizzle<ES, LINE>(c);
                c_of[i] = c;
                voff[i] = chunk * EC < rows ? (unsigned)((int64_t)c * ld * ES + chunk * 16) : 0x80000000u;
            }
        }
    }
    // copies the piece whose first c is `base`'s into LDS at dst; c_left: columns c from there to the end of the share;
    // half: bytes from the first row of the gate to that of the values (gated n operand)
    __device__ __forceinline__ void issue(const char* base, char* dst, int w, int c_left, int64_t half) const {
#pragma unroll
        for (int i = 0; i < CNT; i++) {
            const char* from = base + (!RC && 8 * (w + S::NW * i) >= ROWS / 2 ? half : 0);
            __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)from, 0, 0x7fffffff, 0x00020000);
            const unsigned o = voff[i] | (c_of[i] < c_left ? 0u : 0x80000000u);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, GM_LDS(void, dst + (w + S::NW * i) * 1024), 16, o, 0, 0, 0);
        }
    }
};

// The transposing LDS load.  The compiler has it wait for every copy into LDS that is under way, whatever part of LDS that
// goes to, unless it knows more of the address: `restrict` is that knowledge (the kernel's own waits and barriers order the two).
__device__ __forceinline__ gm_s16x4 read_tr(const char* __restrict__ at) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16(GM_LDS(gm_s16x4, at)); }

// fragment of 32 rows (block `blk` of the tile) and step s of the piece at `t`
template <typename S, bool RC, int ROWS>
__device__ __forceinline__ typename GM<typename S::T>::frag read_frag(const char* t, int blk, int s, int lane) {
    typedef typename GM<typename S::T>::frag frag;
    const int g = lane >> 5, l32 = lane & 31;
    if constexpr (!RC) {
        const int sw = (l32 >> 1) & 7;
        return *reinterpret_cast<const frag*>(t + (32 * blk + l32) * 128 + (((2 * s + g) ^ sw) << 4));
    } else if constexpr (S::ES == 2) {
        const int rho = (lane >> 2) & 3;
        const int chunk = (4 * blk + 2 * (l32 >> 4) + ((lane & 3) >> 1)) ^ line_swizzle<2, ROWS * 2>(rho);
        const char* at = t + (16 * s + 8 * g + rho) * (ROWS * 2) + (chunk << 4) + 8 * (lane & 1);
        const gm_s16x4 a = read_tr(at);
        const gm_s16x4 b = read_tr(at + 4 * (ROWS * 2));
        const gm_s16x8 v = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        return __builtin_bit_cast(frag, v);
    } else {
        const int chunk = (8 * blk + (l32 >> 2)) ^ line_swizzle<4, ROWS * 4>(4 * g);
        const char* at = t + (8 * s + 4 * g) * (ROWS * 4) + (chunk << 4) + 4 * (l32 & 3);
        frag v;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = *reinterpret_cast<const float*>(at + e * (ROWS * 4));
        return v;
    }
}

// 16 consecutive n-side values of a lane's row m (register r holds n = 8 (r / 4) + 4 g + r % 4) to memory; `n_left` valid columns
// as pairs of 16 bits
template <typename T> __device__ __forceinline__ void store_pairs(T* row, const unsigned* w, int g, int n_left) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
        unsigned a0 = w[4 * h], a1 = w[4 * h + 1], b0 = w[4 * h + 2], b1 = w[4 * h + 3];
        swap_halves(a0, b0);
        swap_halves(a1, b1);
        const int n = 16 * h + 8 * g;
        if (n < n_left) store16<T>(row + n, (gm_u4){a0, a1, b0, b1}, n_left - n);
    }
}
// The upper parts of a row's 32 kept gate columns and of the 32 value columns beside them: pieces change lanes between the rows of a
// block, so that one store covers 8 whole lines of 128 bytes.  Whole lines go past the caches, which leaves those to the operands:
// forward of 16384 x 1024 -> 4096 bf16 334 -> 303 us.  (32-byte pieces of 32 rows, as the lanes have them, 690 past the caches; the lower
// parts and 8-bit codes in lines of their own, 64 bytes, no gain and dz 94 -> 100 and 36 -> 43.)
__device__ __forceinline__ void swap_rows16(unsigned& a, unsigned& b) {   // lanes l (of a) and l - 16 (of b) where l & 16
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0];
    b = r[1];
}
__device__ __forceinline__ void swap_rows8(unsigned& a, unsigned& b) {    // the same with 8
    const int x = __builtin_amdgcn_update_dpp((int)a, (int)b, 0x128, 0xf, 0xc, false);   // rotated by 8 within 16, into the upper 8
    b = (unsigned)__builtin_amdgcn_update_dpp((int)b, (int)a, 0x128, 0xf, 0x3, false);
    a = (unsigned)x;
}
__device__ __forceinline__ void stream16(void* p, unsigned a, unsigned b, unsigned c, unsigned d) {
    __builtin_nontemporal_store((gm_u4){a, b, c, d}, reinterpret_cast<gm_u4_any*>(p));
}
// `block` is where the block's row 0 starts, `ld` from a row to the next, `rows` how many there are
template <typename T> __device__ __forceinline__ void store_kept_pairs(T* block, int64_t ld, unsigned (&w)[2][8], int lane, int rows) {
    unsigned p[2][2][4];
#pragma unroll
    for (int q = 0; q < 2; q++) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            unsigned* v = w[q] + 4 * h;
            swap_halves(v[0], v[2]);
            swap_halves(v[1], v[3]);
#pragma unroll
            for (int i = 0; i < 4; i++) p[q][h][i] = v[i];
        }
#pragma unroll
        for (int i = 0; i < 4; i++) swap_rows16(p[q][0][i], p[q][1][i]);
    }
#pragma unroll
    for (int k = 0; k < 2; k++)
#pragma unroll
        for (int i = 0; i < 4; i++) swap_rows8(p[0][k][i], p[1][k][i]);
    const int at = 32 * ((lane >> 3) & 1) + 16 * ((lane >> 4) & 1) + 8 * (lane >> 5);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = 8 * i + (lane & 7);
        const unsigned* v = p[i & 1][i >> 1];
        if (r < rows) stream16(block + r * ld + at, v[0], v[1], v[2], v[3]);
    }
}
// as quads of bytes
__device__ __forceinline__ void store_quads(uint8_t* row, const unsigned* w, int g, int n_left) {
    unsigned c0 = w[0], c1 = w[1], c2 = w[2], c3 = w[3];
    swap_halves(c0, c2);
    swap_halves(c1, c3);
    const int n = 16 * g;
    if (n < n_left) store16<uint8_t>(row + n, (gm_u4){c0, c2, c1, c3}, n_left - n);
}
template <typename T> __device__ __forceinline__ void store_block(T* row, const float* v, int g, int n_left) {
    if constexpr (sizeof(T) == 2) {
        unsigned w[8];
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = GM<T>::pack2(v[2 * i], v[2 * i + 1]);
        store_pairs(row, w, g, n_left);
    } else {
#pragma unroll
        for (int rr = 0; rr < 4; rr++) {
            const int n = 8 * rr + 4 * g;
            const gm_f32x4 q = {v[4 * rr], v[4 * rr + 1], v[4 * rr + 2], v[4 * rr + 3]};
            if (n < n_left) store16<float>(reinterpret_cast<float*>(row) + n, __builtin_bit_cast(gm_u4, q), n_left - n);
        }
    }
}

template <typename S>
__global__ __launch_bounds__(S::NT) void hstu_gemm_kernel(const GemmArgs a) {
    typedef typename S::T T;
    typedef typename GM<T>::frag frag;
    constexpr int ES = S::ES, BK = S::BK, NB = S::NB, MB = S::MB;
    __shared__ __attribute__((aligned(1024))) char gm_lds[S::STAGES * S::STAGE];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 5, l32 = lane & 31;
    const int wn = w % S::WN, wm = w / S::WN;
    // Workgroup i runs on XCD i % 8: an XCD gets a contiguous run of tiles, in groups of GROUP row tiles by all column tiles,
    // so that the 32 tiles its CUs work on at a time share operands in its L2
    constexpr unsigned GROUP = 4;
    const unsigned per = (unsigned)a.tiles_n * (unsigned)a.tiles_m, total = per * (unsigned)a.splits;
    const unsigned xcd = blockIdx.x & 7, q8 = total >> 3, r8 = total & 7;
    unsigned id = xcd * q8 + (xcd < r8 ? xcd : r8) + (blockIdx.x >> 3);
    const unsigned split = id / per;
    id -= split * per;
    const unsigned grp = id / (GROUP * a.tiles_n), rem = id - grp * GROUP * a.tiles_n;
    const unsigned rows_here = min((unsigned)GROUP, (unsigned)a.tiles_m - grp * GROUP);
    const unsigned tm = grp * GROUP + rem % rows_here, tn = rem / rows_here;
    constexpr int NCOLS = S::GATED ? S::BN / 2 : S::BN;   // output columns of a tile
    const int64_t m0 = (int64_t)tm * S::BM;
    const int n0 = (int)tn * NCOLS;
    const int64_t c0 = (int64_t)split * a.c_split;
    const int64_t c_len = min(a.c_split, a.C - c0);
    const int pieces = (int)((c_len + BK - 1) / BK);

    Stager<S, S::NRC, S::BN, S::NI> sn;
    Stager<S, S::MRC, S::BM, S::MI> sm;
    sn.init(w, lane, a.n_ld, (int64_t)a.N - n0, S::GATED);
    sm.init(w, lane, a.m_ld, a.M - m0, false);
    const char* nb = reinterpret_cast<const char*>(a.n_op) + (S::NRC ? (c0 * a.n_ld + n0) : ((int64_t)n0 * a.n_ld + c0)) * ES;
    const char* mb = reinterpret_cast<const char*>(a.m_op) + (S::MRC ? (c0 * a.m_ld + m0) : (m0 * a.m_ld + c0)) * ES;
    const int64_t n_step = (S::NRC ? a.n_ld : 1) * (int64_t)(BK * ES), m_step = (S::MRC ? a.m_ld : 1) * (int64_t)(BK * ES);

    gm_f32x16 acc[NB][MB];
#pragma unroll
    for (int i = 0; i < NB; i++)
#pragma unroll
        for (int j = 0; j < MB; j++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[i][j][r] = 0.f;

    const int64_t half = S::GATED ? (int64_t)a.N * a.n_ld * ES : 0;
    // piece t into its place of the ring; behind the last one the copies address nothing, so that every turn issues as many
    char* into = gm_lds;
    int64_t c_left = c_len;
    auto copy_in = [&]() __attribute__((always_inline)) {
        const int left = (int)max(min(c_left, (int64_t)BK), (int64_t)0);
        sn.issue(nb, into, w, left, half);
        sm.issue(mb, into + S::N_BYTES, w, left, 0);
        nb += n_step;
        mb += m_step;
        c_left -= BK;
        into = into == gm_lds + (S::STAGES - 1) * S::STAGE ? gm_lds : into + S::STAGE;
    };
    // all but the newest `n` pieces' copies of this wave have landed
    auto landed = [&](auto n) __attribute__((always_inline)) {
        constexpr int left = decltype(n)::value * (S::NI + S::MI);
        static_assert(left < 64, "the counter holds 63");
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(left) : "memory");
    };
    frag nf[2][NB], mf[2][MB];
    auto read_step = [&](const char* cur, int s, frag (&n)[NB], frag (&m)[MB]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NB; i++) {
            const int blk = S::GATED ? (i / (NB / 2)) * (S::BN / 64) + wn * (NB / 2) + i % (NB / 2) : wn * NB + i;
            n[i] = read_frag<S, S::NRC, S::BN>(cur, blk, s, lane);
        }
#pragma unroll
        for (int j = 0; j < MB; j++) m[j] = read_frag<S, S::MRC, S::BM>(cur + S::N_BYTES, wm * MB + j, s, lane);
    };
    auto multiply = [&](const frag (&n)[NB], const frag (&m)[MB]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NB; i++)
#pragma unroll
            for (int j = 0; j < MB; j++) acc[i][j] = GM<T>::mfma(n[i], m[j], acc[i][j]);
    };
    // The fragments of a step are read while the matrix cores work on the step before it, across the pieces too: the barrier
    // that hands a piece over falls between the last reads of one and the first of the next, with a step's products queued.
    if (pieces > 0) {
#pragma unroll
        for (int i = 0; i < S::STAGES; i++) copy_in();
        landed(gm_const<S::STAGES - 1>());
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        read_step(gm_lds, 0, nf[0], mf[0]);
    }
    const char* cur = gm_lds;
    for (int t = 0; t < pieces; t++) {
        const char* nxt = cur == gm_lds + (S::STAGES - 1) * S::STAGE ? gm_lds : cur + S::STAGE;
#pragma unroll
        for (int s = 0; s < S::STEPS; s++) {
            if (s + 1 < S::STEPS) read_step(cur, s + 1, nf[(s + 1) & 1], mf[(s + 1) & 1]);
            else if (t + 1 < pieces) {
                // own reads of this piece and own copies of the next have landed; behind the barrier everybody's have, and
                // this piece's place is free
                landed(gm_const<S::STAGES - 2>());
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                copy_in();
                read_step(nxt, 0, nf[0], mf[0]);
            }
            __builtin_amdgcn_sched_barrier(0);
            multiply(nf[s & 1], mf[s & 1]);
            __builtin_amdgcn_sched_barrier(0);
        }
        cur = nxt;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // copies of nothing may still be under way

    // accumulator register r of block (i, j): row m = 32 j + l32, n = 32 i + 8 (r / 4) + 4 g + r % 4 of the wave's tile
    if constexpr (!S::GATED) {
        const int nw0 = n0 + wn * (32 * NB);
#pragma unroll
        for (int j = 0; j < MB; j++) {
            const int64_t m = m0 + wm * (32 * MB) + 32 * j + l32;
#pragma unroll
            for (int i = 0; i < NB; i++) {
                float v[16];
#pragma unroll
                for (int r = 0; r < 16; r++) v[r] = acc[i][j][r];
                const int n = nw0 + 32 * i, left = m < a.M ? a.N - n : 0;
                if (a.splits > 1) store_block<float>(reinterpret_cast<float*>(a.out) + ((int64_t)split * a.M + m) * a.N + n, v, g, left);
                else store_block<T>(reinterpret_cast<T*>(a.out) + m * a.N + n, v, g, left);
            }
        }
    } else {
#pragma unroll
        for (int gb = 0; gb < NB / 2; gb++) {
        const int n = n0 + (wn * (NB / 2) + gb) * 32;
        float bg[16], bu[16];
#pragma unroll
        for (int r = 0; r < 16; r++) {
            bg[r] = bu[r] = 0.f;
        }
        if (a.bias) {
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int c = n + 8 * (r >> 2) + 4 * g + (r & 3), at = min(c, a.N - 1);
                float vg, vu;
                if (a.bias_f32) { vg = reinterpret_cast<const float*>(a.bias)[at]; vu = reinterpret_cast<const float*>(a.bias)[a.N + at]; }
                else { vg = to_float(reinterpret_cast<const T*>(a.bias)[at]); vu = to_float(reinterpret_cast<const T*>(a.bias)[a.N + at]); }
                bg[r] = c < a.N ? vg : 0.f;
                bu[r] = c < a.N ? vu : 0.f;
            }
        }
#pragma unroll
        for (int j = 0; j < MB; j++) {
            const int64_t m = m0 + wm * (32 * MB) + 32 * j + l32;
            const int left = m < a.M ? a.N - n : 0;
            float zg[16], zu[16], h[16];
#pragma unroll
            for (int r = 0; r < 16; r++) {
                zg[r] = acc[gb][j][r] + bg[r];
                zu[r] = acc[NB / 2 + gb][j][r] + bu[r];
            }
            // kept rows hold whole blocks, with zeros past f: their products are 0 * x, NaN for a row with a NaN or an infinity
            const int64_t kept = HSTU_GATED_KEPT((int64_t)a.N);
            const int whole = left > 0 ? 32 : 0;
            if (S::KEEP != HSTU_KEEP_NONE && n + 32 > a.N) {
#pragma unroll
                for (int r = 0; r < 16; r++)
                    if (n + 8 * (r >> 2) + 4 * g + (r & 3) >= a.N) zg[r] = zu[r] = 0.f;
            }
            if constexpr (S::KEEP == HSTU_KEEP_FULL && S::ES == 4) {
#pragma unroll
                for (int part = 0; part < 2; part++) store_block<T>(reinterpret_cast<T*>(a.z) + (m * 2 + part) * kept + n, part ? zu : zg, g, whole);
            } else if constexpr (S::KEEP == HSTU_KEEP_FULL) {
                unsigned up[2][8];
#pragma unroll
                for (int part = 0; part < 2; part++) {
                    const float* v = part ? zu : zg;
                    unsigned low[4];
#pragma unroll
                    for (int i = 0; i < 8; i++) up[part][i] = upper_pair(v[2 * i], v[2 * i + 1]);
#pragma unroll
                    for (int i = 0; i < 4; i++) low[i] = lower_quad(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                    store_quads(a.z_aux + (m * 2 + part) * kept + n, low, g, whole);
                }
                const int64_t b0 = m - l32;   // row 0 of the block
                store_kept_pairs(reinterpret_cast<T*>(a.z) + b0 * 2 * kept + 2 * n, 2 * kept, up, lane, n < a.N ? (int)min(a.M - b0, (int64_t)32) : 0);
            } else if constexpr (S::KEEP == HSTU_KEEP_8BIT) {
                // the 32 columns of a row lie in the 16 registers of two lanes
#pragma unroll
                for (int part = 0; part < 2; part++) {
                    const float* v = part ? zu : zg;
                    float top = 0.f;
#pragma unroll
                    for (int r = 0; r < 16; r++) top = fmaxf(top, pack8_finite_abs(v[r]));
                    top = fmaxf(top, __shfl_xor(top, 32, 64));
                    const int e = pack8_exponent(top);
                    const float inv = pack8_inv_scale(e);
                    unsigned c[4];
#pragma unroll
                    for (int rr = 0; rr < 4; rr++) c[rr] = pack8_codes(v[4 * rr], v[4 * rr + 1], v[4 * rr + 2], v[4 * rr + 3], inv);
                    store_quads(reinterpret_cast<uint8_t*>(a.z) + (m * 2 + part) * kept + n, c, g, whole);
                    if (g == 0 && left > 0) a.z_aux[((m * 2 + part) * kept + n) / HSTU_PACK8_GROUP] = (uint8_t)e;
                }
            }
            act_of<16>(zg, S::ACT, h);
#pragma unroll
            for (int r = 0; r < 16; r++) h[r] *= zu[r];
            store_block<T>(reinterpret_cast<T*>(a.out) + m * a.N + n, h, g, left);
        }
        }
    }
}

// kinds of products, and the launchers (one translation unit per element type)
enum GemmKind : int { GEMM_GATED = 0 /* KC x KC, gated epilogue */, GEMM_DX = 1 /* n side RC, m side KC */, GEMM_DW = 2 /* both RC */ };
// 256 x 256 outputs by eight waves (one workgroup per CU); 128 x 128 by four, with two buffers (two workgroups per CU) or four (one,
// whose copies run three pieces ahead; 16 bits only); 256 rows m x 128 by eight with three buffers (one); 64 x 128 by four with
// three (two), for products too small for the others
enum GemmTile : int { TILE_256 = 0, TILE_128 = 1, TILE_128_DEEP = 2, TILE_256x128 = 3, TILE_64x128 = 4, GEMM_TILES = 5 };
constexpr int gemm_tile_m(int tile) { return tile == TILE_256 || tile == TILE_256x128 ? 256 : tile == TILE_64x128 ? 64 : 128; }
constexpr int gemm_tile_n(int tile, int kind) { return (tile == TILE_256 ? 256 : 128) / (kind == GEMM_GATED ? 2 : 1); }
hipError_t launch_gemm_bf16(const GemmArgs& a, int kind, int tile, hipStream_t st);
hipError_t launch_gemm_f16(const GemmArgs& a, int kind, int tile, hipStream_t st);
hipError_t launch_gemm_f32(const GemmArgs& a, int kind, int tile, hipStream_t st);

template <typename T, bool NRC, bool MRC, int GATE> void launch_gemm_tile(const GemmArgs& a, int tile, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)a.tiles_n * a.tiles_m * a.splits));
    auto go = [&](auto shape) {
        typedef decltype(shape) S;
        hipLaunchKernelGGL((hstu_gemm_kernel<S>), grid, dim3(S::NT), 0, st, a);
    };
    if (tile == TILE_256) go(GemmShape<T, NRC, MRC, 256, 256, 4, 2, 2, GATE>());
    else if (tile == TILE_128) go(GemmShape<T, NRC, MRC, 128, 128, 2, 2, 2, GATE>());
    else if (tile == TILE_256x128) go(GemmShape<T, NRC, MRC, 128, 256, 2, 4, 3, GATE>());
    else if (tile == TILE_64x128) go(GemmShape<T, NRC, MRC, 128, 64, 2, 2, 3, GATE>());
    else if constexpr (sizeof(T) == 2) go(GemmShape<T, NRC, MRC, 128, 128, 2, 2, 4, GATE>());
}
template <typename T> hipError_t launch_gemm_t(const GemmArgs& a, int kind, int tile, hipStream_t st) {
    if (kind == GEMM_DX) launch_gemm_tile<T, true, false, -1>(a, tile, st);
    else if (kind == GEMM_DW) launch_gemm_tile<T, true, true, -1>(a, tile, st);
    else {
        auto gated = [&](auto act) {
            constexpr int ACT = decltype(act)::value;
            if (a.keep == HSTU_KEEP_NONE) launch_gemm_tile<T, false, false, gate_of(ACT, HSTU_KEEP_NONE)>(a, tile, st);
            else if (sizeof(T) == 4 || a.keep == HSTU_KEEP_FULL) launch_gemm_tile<T, false, false, gate_of(ACT, HSTU_KEEP_FULL)>(a, tile, st);
            else if constexpr (sizeof(T) == 2) launch_gemm_tile<T, false, false, gate_of(ACT, HSTU_KEEP_8BIT)>(a, tile, st);
        };
        if (a.act == HSTU_ACT_SILU) gated(gm_const<HSTU_ACT_SILU>());
        else gated(gm_const<HSTU_ACT_GELU>());
    }
    return hipGetLastError();
}

}  // namespace hstu
