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

// Few rows per group and the weights as rows: streamed (moe_ops_stream.h).
inline bool op_streamed(bool b_col, long long rows, long long E) { return !b_col && rows <= 16 * E; }

constexpr int kOpMaxSplits = 16;
// Ranges of k for `tiles` workgroups of a call that could run in `slots`: none
// where half of those have one, no range shorter than `least` (folding the
// ranges is a launch of its own, about 4 us: a 64 x 64 tile runs 2 KB of k per
// row in about 16 us, the streamed form 8 KB in about 10).
inline int op_splits(long long tiles, long long k, long long least, int slots) {
    if (tiles < 1 || 2 * tiles > slots) return 1;
    long long s = (slots + tiles - 1) / tiles;
    if (s > k / least) s = k / least;
    if (s > kOpMaxSplits) s = kOpMaxSplits;
    return s > 1 ? (int)s : 1;
}
// Ragged rows: by 64 x 64 tiles, or the streamed products' 16 columns.
inline int op_rows_splits(int ot, bool b_col, long long rows, long long E, long long N, long long K, int ncu) {
    const long long held = E < rows ? E : rows;  // groups that may hold rows
    if (op_streamed(b_col, rows, E)) return op_splits(held * ((N + 15) / 16), K * op_size(ot), 8192, ncu);
    const long long mt = (rows + 63) / 64;
    // a few rows per group read the weights as fast as loads are in flight: four
    // 64 x 64 tiles per CU (4 rows of 3991 on 4 experts of 4970 columns, fp32: 114 us at one)
    const int slots = rows <= 16 * E ? 4 * ncu : ncu;
    return op_splits((mt > held ? mt : held) * ((N + 63) / 64), K * op_size(ot), 2048, slots);
}
// Ragged k: the rows of each group.
inline int op_matrix_splits(long long rows, long long E, long long M, long long N, int ncu) {
    return op_splits(E * ((M + 63) / 64) * ((N + 63) / 64), rows / E, 512, ncu);
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
