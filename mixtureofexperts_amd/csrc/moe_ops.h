// moe_ops.h -- argument blocks and launchers of the operators on a caller's
// own device tensors (grouped products and their gradients, int8 products,
// block norms), shared by the translation units that hold their kernels.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace moe {

enum OpType { OT_F32 = 0, OT_BF16 = 1, OT_I8 = 2 };
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
    const float *sa;               // int8: scale per row of A
    const float *sb;               // int8: scale per group and column [E][N]
    float *ws;                     // partial sums (splits > 1), [range][rows][N] or [group][range][M][N]
    int splits;                    // ranges that k is split into over workgroups (1: none)
    int nt, mt;                    // tiles along N, and (ragged k) along M
};

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

// q[r][k] = rne(127 x[r][k] / max|x[r]|) as int8, scale[r] = max|x[r]| / 127;
// columns [cols, ldq) are not written past pad_to (zeros up to it)
hipError_t launch_quantize_i8(const void *x, long long ldx, int x_bf16, long long rows, int cols, int8_t *q,
                              long long ldq, int pad_to, float *scale, hipStream_t s);

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
