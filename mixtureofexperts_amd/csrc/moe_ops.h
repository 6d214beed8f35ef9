// moe_ops.h -- argument blocks and launchers of the operators on a caller's
// own device tensors (grouped products and their gradients, int8 products,
// block norms), shared by the translation units that hold their kernels.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace moe {

enum OpType { OT_F32 = 0, OT_BF16 = 1, OT_I8 = 2, OT_F8 = 3 };  // (OT_F8: e4m3)
__host__ __device__ constexpr int op_size(int ot) { return ot == OT_F32 ? 4 : (ot == OT_BF16 ? 2 : 1); }

// C[m][n] = sum_k A(m, k) B(n, k) per group.  An operand is held with k
// contiguous ("row": address m ld + k) or with m (n) contiguous ("col":
// address k ld + m).
//
// Ragged rows (ragged_k = 0): group e's rows [offsets[e], offsets[e + 1]) of A
// and C against its own B (b_stride elements apart): the forward product and
// the gradient of the rows.
// Ragged k (ragged_k = 1): A and B are both "col" over the group's rows and C
// is the group's own matrix (c_stride elements apart): the weight gradient.
struct OpGemmArgs {
    const void *A, *B;
    void *C;
    long long lda, ldb, ldc;       // elements
    long long b_stride, c_stride;  // elements per group
    const int *offsets;            // [E + 1] or null: one group of all rows
    int E, rows;                   // groups, rows of the ragged tensors
    int M, N, K;                   // sizes that are not ragged
    int c_f32;                     // C in fp32, else bf16
    int accumulate;                // ragged k: C += (fp32 sums, one rounding)
    const float *sa;               // int8: scale per row of A; e4m3: [rows][kb]
    const float *sb;               // int8: scale per group and column [E][N]; e4m3: [E][ceil(N / 128)][kb]
    int kb;                        // e4m3: blocks of 128 along K
    int exact;                     // e4m3: exact products, whatever the result's type
    float *ws;                     // partial sums (splits > 1), [range][rows][N] or [group][range][M][N]
    int splits;                    // ranges that k is split into over workgroups (1: none)
    int nt, mt;                    // tiles along N, and (ragged k) along M
    // Gated blocks (OpMode), operand and result types as above:
    int act;                       // MOE_ACT_*
    const void *A2, *B2;           // the second rows, the second weight
    long long lda2, ldb2, b2_stride;
    const void *ga, *gb;           // OM_GATE_GRAD: the pre-activations
    long long ldga, ldgb;
    void *C2, *C3;                 // OM_GATED: a and b (or null); OM_GATE_GRAD: db and h
    long long ldc2, ldc3;
    int tail;                      // OM_TWO, 256 x 256 tiles: CUs of an XCD whose last, part round is split (0: none)
};

// What a product of ragged rows computes:
//   OM_PLAIN      C = A B'
//   OM_GATED      a = A B', b = A B2', C = act(a) b
//   OM_GATE_GRAD  dh = A B', C = dh gb act'(ga), C2 = dh act(ga), C3 = act(ga) gb
//   OM_TWO        C = A B' + A2 B2'
enum OpMode { OM_PLAIN = 0, OM_GATED = 1, OM_GATE_GRAD = 2, OM_TWO = 3 };

// The rows of group e, held within [0, rows] whatever the offsets say.
__device__ __forceinline__ void op_group(const int *offsets, int e, int rows, int &lo, int &hi) {
    lo = 0;
    hi = rows;
    if (offsets) {
        lo = min(max(offsets[e], 0), rows);
        hi = min(max(offsets[e + 1], lo), rows);
    }
}

// Grid of kernels with a row (or a few) per workgroup: 2^20 workgroups along x, since
// a dimension's threads have to fit 32 bits, and the workgroup's number in it.
inline dim3 op_row_grid(long long blocks) {
    constexpr long long X = 1 << 20;
    return blocks <= X ? dim3((unsigned)blocks) : dim3((unsigned)X, (unsigned)((blocks + X - 1) / X));
}
__device__ __forceinline__ long long op_row_block() { return (long long)blockIdx.y * gridDim.x + blockIdx.x; }

// Few rows per group and the weights as rows: streamed (moe_ops_stream.h), against 64 x
// 64 tiles of the same product, us.  fp32: up to 16 rows (8 experts of 4096 / 4096, 16
// rows each: 145 / 178, 24: 168 / 162).  bf16 and int8: up to 8 rows, of weights with 4 KB
// and more per row (bf16, 4096 / 14336: 1 row 164 / 183, 4 170 / 204, 8 193 / 191, 16 241 /
// 201; int8 104 / 105, 106 / 122, 109 / 119, 124 / 126; 64 experts of 1408 / 2048, bf16: 1
// row 53 / 51, 8 89 / 77, int8 36 / 30, 57 / 45; 8 of 2048 / 4096: bf16, 8 rows, 37 / 39, int8 17
// / 14) or, shorter, fewer tiles than CUs (2048 / 4096: 12.5 / 15).  Rows that do not end
// on 4 bytes, whose elements' loads bound both: only such few tiles, and of a k too short
// to split or about one row per group (4 rows on each of 3 experts of 1665 / 3000 25 / 26,
// of 16 86 / 52; of 3001 / 3000, 3 experts, 35 / 27, one row 20 / 23).
inline bool op_streamed(int ot, bool b_col, long long rows, long long E, long long N, long long K, int ncu) {
    if (b_col) return false;
    if (ot == OT_F32) return rows <= 16 * E;
    const long long bytes = K * op_size(ot);
    const bool few = (E < rows ? E : rows) * ((N + 63) / 64) < ncu, lengthy = bytes >= 4096;
    return rows <= 8 * E && (bytes % 4 ? few && (!lengthy || rows <= E) : few || lengthy);
}

constexpr int kOpMaxSplits = 16;
// Ranges of k for `tiles` workgroups of a call that could run in `slots`: none
// where half of those have one, no range shorter than `least` (folding the
// ranges is a launch of its own, about 4 us: the streamed form runs 8 KB of k in
// about 10).
inline int op_splits(long long tiles, long long k, long long least, int slots) {
    if (tiles < 1 || 2 * tiles > slots) return 1;
    long long s = (slots + tiles - 1) / tiles;
    if (s > k / least) s = k / least;
    if (s > kOpMaxSplits) s = kOpMaxSplits;
    return s > 1 ? (int)s : 1;
}
// 64 x 64 tiles, three workgroups per CU: as many ranges as have room in one round.
// More than half a tile per CU: the fold writes and reads more than a short k takes, so k
// has to be `lengthy`.
inline int op_tile_splits(long long tiles, long long k, long long least, long long lengthy, int ncu) {
    if (tiles < 1 || (2 * tiles > ncu && k < lengthy)) return 1;
    long long s = 3ll * ncu / tiles;
    if (s > k / least) s = k / least;
    if (s > kOpMaxSplits) s = kOpMaxSplits;
    return s > 1 ? (int)s : 1;
}
// Ragged rows: by 64 x 64 tiles, or the streamed products' 16 columns.  On 256 CUs, one
// range / this many, us: bf16, rows of 16 KB: 64 tiles 61 / 21, 128 56 / 28, 256 61 / 39, 384
// 63 / 51, of 8 KB: 33 / 16, 33 / 20, 33 / 28, 33 / 33; of 4 KB (256 tiles: none) 18 / 22.
// int8 within 1 us of those.  fp32: 16 KB 85 / 29, 83 / 47, 83 / 77, 135 / 111; 8 KB 45 / 20, 45
// / 28, (none) 45 / 47, 70 / 63.
inline int op_rows_splits(int ot, bool b_col, long long rows, long long E, long long N, long long K, int ncu) {
    const long long held = E < rows ? E : rows, bytes = K * op_size(ot);  // groups that may hold rows
    if (op_streamed(ot, b_col, rows, E, N, K, ncu)) return op_splits(held * ((N + 15) / 16), bytes, 8192, ncu);
    const long long mt = (rows + 63) / 64, tiles = (mt > held ? mt : held) * ((N + 63) / 64);
    // a few rows per group read the weights as fast as loads are in flight: four
    // 64 x 64 tiles per CU (4 rows of 3991 on 4 experts of 4970 columns, fp32: 112 us in one
    // range, 86 so)
    if (rows <= 16 * E) return op_splits(tiles, bytes, 2048, 4 * ncu);
    return op_tile_splits(tiles, bytes, 2048, ot == OT_F32 ? 12288 : 8192, ncu);
}
// Ragged k: the rows of each group.  fp32, bound by its products: 8000 rows, 512 / 1024 (128
// tiles) 165 / 77 us, 1000 / 1000 (256) 166 / 141, 4000 rows of 1536 / 1024 (384) 136 / 111, 1900
// of 1000 / 1000 43 / 46 (none).  bf16, bound by its reads: 8000 rows of 512 / 1024 in two
// ranges 41 / 28, but 1000 / 1000 43 / 47: only where half the CUs have no tile.
inline int op_matrix_splits(int ot, long long rows, long long E, long long M, long long N, int ncu) {
    const long long tiles = E * ((M + 63) / 64) * ((N + 63) / 64);
    return ot == OT_F32 ? op_tile_splits(tiles, rows / E, 800, 4000, ncu) : op_splits(tiles, rows / E, 512, ncu);
}

// Few rows per group of a gated forward product: streamed, against tiles, us: 8 bf16 experts of
// 4096 / 14336, 1 row each 354 / 368, 8 333 / 352, 16 377 / 367; of 2048 / 4096, 2 rows 47 / 54, 4 60 / 52; one
// of 4096 / 4096, 8 rows 17 / 33, 16 26 / 20; 64 of 1408 / 2048, 1 row 142 / 142, 8 162 / 146; fp32, 8 of 2048 /
// 4096, 16 rows 112 / 158.
inline bool op_gated_streamed(int ot, bool b_col, long long rows, long long E, long long N, long long K, int ncu) {
    if (b_col) return false;
    if (ot == OT_F32) return rows <= 16 * E;
    const long long bytes = K * op_size(ot);
    const bool few = (E < rows ? E : rows) * ((2 * N + 63) / 64) < ncu;
    if (rows > 8 * E) return false;
    if (bytes % 4) return few && (bytes < 4096 || rows <= E);  // (as op_streamed)
    return few || bytes >= 8192 || (bytes >= 4096 && rows <= 2 * E);
}
// The gated products, by the sizes of the product that they are: 2 hidden columns (two
// weights), one product of dh, 2 hidden elements of k.  The gradients are never streamed.
inline int op_gated_splits(OpMode mode, int ot, bool b_col, long long rows, long long E, long long N, long long K, int ncu) {
    if (mode == OM_GATED && op_gated_streamed(ot, b_col, rows, E, N, K, ncu)) {
        const long long held = E < rows ? E : rows;
        return op_splits(held * ((N + 15) / 16), K * op_size(ot), 8192, ncu);
    }
    return op_rows_splits(ot, true, rows, E, mode == OM_GATED ? 2 * N : N, mode == OM_TWO ? 2 * K : K, ncu);
}

// Tiles of the gated and 8-bit products: 256 x 256 (one workgroup per CU), 128 x 128 (two) or
// 64 x 64 (three), by the rounds that each takes and a round's time, the 128 x 128 one's as
// 100.  N: columns of products.  Measured, us, 256 / 128 / 64 (bf16 gated: a round 165 / 100 / 65):
// forward of 24576 rows on 64 experts 2048 / 1408 367 / 390 / 646, of 2048 rows on 8 of 4096 / 2048
// 117 / 140 / 199, of 512 rows on 8 of 4096 / 4096 122 / 105 / 129; through the down product
// 266 / 247 / 369, 101 / 60 / 75, 101 / 75 / 82; row gradient of 4096 rows on 8 of 2048 / 4096
// 209 / 247 / 300.  8-bit, bf16 result (170 / 100 / 60): 24576 rows 109 / 119 / 192, 4096 rows on 8 of
// 2048 / 4096 64 / 54 / 79, 3102 rows on 64 of 1408 / 2048 48 / 39 / 45; fp32 result (- / 100 / 50): 2048
// rows on 8 of 4096 / 2048 - / 62 / 58, 4096 rows - / 83 / 103.  One cost for a form's three products
// and whole rounds are coarse: of these it takes the slower tile, by 7 to 9 %, for the 24576 rows
// through the down product (256) and in 8 bits (128), the 512 rows through it (64), and the 2048
// rows with an fp32 result (128).
struct OpTileCost {
    int c256, c128, c64;  // 0: none of these
};
constexpr OpTileCost kCostGated = {165, 100, 65}, kCostF8 = {170, 100, 60}, kCostF8Wide = {0, 100, 50};
// tail: the last round of 256 x 256 tiles is split
inline int op_pick_tile(const OpTileCost &c, long long rows, long long E, long long N, int ncu, bool tail) {
    const long long held = E < rows ? E : rows;
    auto tiles = [&](int b) -> long long {  // a group's last tile is half empty on average
        const long long mt = E > 1 ? rows / b + held / 2 : (rows + b - 1) / b;
        return (mt > held ? mt : held) * ((N + b - 1) / b);
    };
    auto rounds = [&](int b, long long slots) { return (tiles(b) + slots - 1) / slots; };
    long long best = rounds(64, 3ll * ncu) * c.c64;
    int pick = 64;
    // (groups of fewer rows leave most of a tile empty)
    if (c.c128 && rows >= 40 * E && N >= 64) {
        const long long t = rounds(128, 2ll * ncu) * c.c128;
        if (t <= best) best = t, pick = 128;
    }
    if (c.c256 && rows >= 96 * E && N >= 192) {
        long long t = rounds(256, ncu) * c.c256;
        if (tail) {
            const long long whole = tiles(256) / ncu, left = tiles(256) - whole * ncu;
            t = whole * c.c256 + (left ? c.c256 / (ncu / left) + c.c256 / 10 : 0);
        }
        if (t <= best) best = t, pick = 256;
    }
    return pick;
}
// bf16 OM_TWO on 256 x 256 tiles: the last round is split where rounds are few and k (of both
// pairs) is long.  8192 rows on 8 skewed experts of 4096 / 14336, 2.25 rounds: 2298 us whole, 1775
// split.
constexpr int kOpTailTile = 256 * 256;  // sums of a split tile in ws
inline bool op_two_tail(int ot, long long rows, long long E, long long N, long long K, int ncu) {
    if (ot != OT_BF16 || 2 * K < 8192 || ncu < 8) return false;
    const long long held = E < rows ? E : rows, tiles = (rows / 256 + held / 2) * ((N + 255) / 256);
    return tiles < 8 * ncu && op_pick_tile(kCostGated, rows, E, N, ncu, true) == 256;
}
// 8-bit products of few rows: streamed where 64 x 64 tiles are fewer than CUs, or of long rows.
// Streamed / tiles, us: 8 experts of 4096 / 14336, a row on two of them 30.5 / 32.7, 1 row each 101 /
// 109, 4 104 / 110, 8 113 / 110; of 2048 / 4096, 1 row 14.5 / 17.0, 4 15.8 / 16.8, 8 17.6 / 16.9; 64 of
// 1408 / 2048 48 / 44.  A group's rows are one workgroup's, 16 at a time, and its weights are read
// again for each 16: 128 experts of 2048 / 2048, 4 rows each 124 us, the same 512 rows by Zipf 107
// to 117, all on one 95; 64 of 1408 / 2048, 4 rows each 34, 64 rows on one and 3 on the others 34.
inline bool op_f8_streamed(long long rows, long long E, long long N, long long K, int ncu) {
    const long long held = E < rows ? E : rows;
    const bool few = held * ((N + 63) / 64) < ncu;
    if (rows > 8 * E) return false;
    if (K % 4) return few && (K < 4096 || rows <= E);  // (as op_streamed)
    return few || (K >= 2048 && rows <= 4 * E);
}
inline int op_f8_splits(long long rows, long long E, long long N, long long K, int ncu) {
    if (!op_f8_streamed(rows, E, N, K, ncu)) return op_rows_splits(OT_F8, true, rows, E, N, K, ncu);
    const long long held = E < rows ? E : rows;
    return op_splits(held * ((N + 15) / 16), K, 8192, ncu);
}

// What a launcher answers to a call of more workgroups than one launch takes.
constexpr hipError_t kOpTooLarge = hipErrorNotSupported;

// b_col as above (ragged k: both operands are); the launchers pick tile and load
// form (op_gemm_plan)
hipError_t launch_op_gemm_f32(bool b_col, bool ragged_k, OpGemmArgs g, int ncu, hipStream_t s);
hipError_t launch_op_gemm_bf16(bool b_col, bool ragged_k, OpGemmArgs g, int ncu, hipStream_t s);
hipError_t launch_op_gemm_i8(OpGemmArgs g, int ncu, hipStream_t s);
// few rows per group, both operands "row": the weights streamed once
hipError_t launch_op_stream(int ot, const OpGemmArgs &g, hipStream_t s);
// C of a call whose k was split: its ranges' sums, in range order
hipError_t launch_op_fold(int ot, bool ragged_k, const OpGemmArgs &g, hipStream_t s);

// OM_GATED, OM_GATE_GRAD and OM_TWO
hipError_t launch_op_gated(int mode, int ot, bool b_col, OpGemmArgs g, int ncu, hipStream_t s);
// the results of the first two where k was split; dh given, not a product: g.A its rows
hipError_t launch_op_gate_fold(int mode, int ot, const OpGemmArgs &g, hipStream_t s);
hipError_t launch_op_gate_rows(int ot, const OpGemmArgs &g, hipStream_t s);

// q[r][k] = rne(127 x[r][k] / max|x[r]|) as int8, scale[r] = max|x[r]| / 127;
// columns [cols, ldq) are not written past pad_to (zeros up to it)
hipError_t launch_quantize_i8(const void *x, long long ldx, int x_bf16, long long rows, int cols, int8_t *q,
                              long long ldq, int pad_to, float *scale, hipStream_t s);

// ---- 8-bit floating point, a scale per block of 128 ---------------------------------
constexpr int kF8Block = 128;
// Blocks of block_rows (1 or 128) x 128: scale = max|block| / 448, q = e4m3(448 x / max|block|).
struct QuantF8Args {
    const void *x;
    long long ldx, x_stride;  // elements
    int x_bf16;
    long long mats, rows;
    int cols, block_rows;
    uint8_t *q;
    long long ldq, q_stride;
    int pad_to;               // zeros in columns [cols, pad_to)
    float *scale;             // [mats][ceil(rows / block_rows)][ceil(cols / 128)]
};
hipError_t launch_quantize_f8(const QuantF8Args &a, hipStream_t s);
hipError_t launch_op_gemm_f8(OpGemmArgs g, int ncu, hipStream_t s);

// ---- norms around a block ----------------------------------------------------------
// z = y (post: y rstd(y) post), r = alpha x + beta gate z (rounded to x's
// type), h = r rstd(r) pre; rstd(v) = 1 / sqrt(mean(v^2) + eps) over a row.
struct NormArgs {
    const void *x, *y;           // [T][D]; y may be null (r = alpha x)
    int x_bf16, y_bf16, h_bf16;
    const void *pre, *post;      // [D] or null
    int w_bf16;
    const void *gate;            // [ceil(T / gate_rows)][D] or null
    int gate_bf16;
    long long gate_rows;         // rows that share a gate row
    float alpha, beta, eps;
    long long T;
    int D;
    void *r, *h;                 // [T][D] or null
    float *stats;                // [T][2] rstd(y), rstd(r), or null
    // gradients
    const void *dr, *dh;         // [T][D] or null
    void *dx, *dy;               // [T][D] or null
    float *dgate, *dpost, *dpre; // [gates][D], [D], [D] or null
    float *ws;                   // partial sums, 3 x [chunks][D]
    // chunks of rows (norm_chunks): rows per chunk; cpg > 0: cpg chunks per
    // gate row, none crossing its rows, their gate sums partial; cpg = 0: a
    // chunk holds whole gate rows
    long long chunk_rows, cpg, chunks;
};
constexpr int kMaxNormDim = 16384;
long long norm_workspace_floats(long long T, int D, long long gate_rows);
hipError_t launch_block_norm(const NormArgs &a, hipStream_t s);
hipError_t launch_block_norm_grad(NormArgs a, hipStream_t s);

}  // namespace moe
