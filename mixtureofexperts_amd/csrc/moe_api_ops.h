// moe_api_ops.h -- the C entry points of the operators on a caller's own
// device tensors: argument checks, then one launcher call.  Included by
// moe_api.hip only (it uses that file's fail()).
#pragma once
#include <initializer_list>
#include <mutex>

#include "moe_ops.h"
#include "moe_ops_gated.h"

namespace {
// compute units of the current device (looked up once per device)
int op_cus() {
    static std::mutex mu;
    static int cus[64] = {};
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
    std::lock_guard<std::mutex> lk(mu);
    if (!cus[dev]) {
        int n = 0;
        if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n < 1) n = 256;
        cus[dev] = n;
    }
    return cus[dev];
}

int op_fail(const char *fn, const std::string &why) { return fail(nullptr, MOE_EINVAL, std::string(fn) + ": " + why); }
int op_done(const char *fn, hipError_t e) {
    if (e == hipSuccess) return MOE_OK;
    if (e == kOpTooLarge) return op_fail(fn, "too many tiles for one launch");
    return fail(nullptr, MOE_EHIP, std::string(fn) + ": " + hipGetErrorString(e));
}

// tile counts and byte offsets of a row are formed in 32 bits, with room for a
// part tile past the last element
constexpr int kOpMaxSize = 1 << 30;

// What the grouped products share: groups, sizes, types, the rows' strides.
int op_check_groups(const char *fn, const int32_t *offsets, int32_t groups, int32_t rows, int32_t in_dim,
                    int32_t out_dim) {
    if (groups < 1) return op_fail(fn, "groups must be positive");
    if (rows < 0) return op_fail(fn, "rows must not be negative");
    if (in_dim < 1 || out_dim < 1) return op_fail(fn, "dimensions must be positive");
    if (groups > kOpMaxSize || rows > kOpMaxSize || in_dim > kOpMaxSize || out_dim > kOpMaxSize)
        return op_fail(fn, "sizes above 2^30");
    if (!offsets && groups != 1) return op_fail(fn, "offsets are needed for more than one group");
    return MOE_OK;
}
int op_check_dtypes(const char *fn, int32_t dtype, int32_t out_dtype) {
    if (dtype != MOE_F32 && dtype != MOE_BF16) return op_fail(fn, "dtype must be MOE_F32 or MOE_BF16");
    if (out_dtype != MOE_F32 && out_dtype != MOE_BF16) return op_fail(fn, "the result must be MOE_F32 or MOE_BF16");
    if (dtype == MOE_F32 && out_dtype != MOE_F32) return op_fail(fn, "fp32 operands have an fp32 result");
    return MOE_OK;
}
int op_check_workspace(const char *fn, int64_t need, const void *workspace, int64_t bytes) {
    if (need > 0 && (!workspace || bytes < need || ((uintptr_t)workspace & 15)))
        return op_fail(fn, "the workspace must be 16-byte aligned and hold " + std::to_string(need) + " bytes");
    return MOE_OK;
}
// The bytes that a tensor of `mats` matrices covers: rows of `width` bytes, ld apart.
struct OpRegion {
    int64_t at, width, ld, rows, stride, mats;
    OpRegion(const void *p, int64_t cols, int64_t ld_, int64_t rows_, int64_t stride_, int64_t mats_, int64_t es)
        : at((int64_t)(uintptr_t)p), width(cols * es), ld(ld_ * es), rows(rows_), stride(stride_ * es), mats(mats_) {
        if (rows == 1 || ld == width) width += (rows - 1) * ld, rows = 1, ld = width;  // one piece
        if (rows == 1 && (mats == 1 || stride == width)) width += (mats - 1) * stride, ld = width, mats = 1;
        if (!p) mats = 0;
    }
    OpRegion(const void *p, int64_t bytes) : OpRegion(p, bytes, bytes, 1, 0, 1, 1) {}
    int64_t end() const { return at + (mats - 1) * stride + (rows - 1) * ld + width; }
};
// Whether two matrices (a's ma-th, b's mb-th) share a byte.
bool op_matrices_meet(const OpRegion &a, int64_t ma, const OpRegion &b, int64_t mb) {
    const int64_t pa = a.at + ma * a.stride, pb = b.at + mb * b.stride;
    auto below = [](int64_t x, int64_t d) { return x >= 0 ? x / d : -((-x + d - 1) / d); };  // floor
    if (a.rows == 1 || b.rows == 1 || a.ld == b.ld) {
        // row i of a and row j of b meet where pb - a.width < pa + (i - j) ld < pb + b.width
        const int64_t ld = a.rows > 1 ? a.ld : b.ld;
        const int64_t lo = std::max(below(pb - a.width - pa, ld) + 1, -(b.rows - 1));
        const int64_t hi = std::min(below(pb + b.width - pa - 1, ld), a.rows - 1);
        return lo <= hi;
    }
    // rows of different strides: from one to the next that ends past the other's
    // start.  (So many of them that are interleaved are taken as apart.)
    auto next = [&](int64_t p, const OpRegion &r, int64_t x) { return std::max<int64_t>(0, below(x - p - r.width, r.ld) + 1); };
    int64_t i = 0, j = 0;
    for (int step = 0; step < 1 << 16; ++step) {
        i = next(pa, a, pb + j * b.ld);
        if (i >= a.rows) return false;
        if (pa + i * a.ld < pb + j * b.ld + b.width) return true;
        j = next(pb, b, pa + i * a.ld);
        if (j >= b.rows) return false;
        if (pb + j * b.ld < pa + i * a.ld + a.width) return true;
    }
    return false;
}
bool op_overlap(const OpRegion &a, const OpRegion &b) {
    if (a.mats < 1 || b.mats < 1 || a.end() <= b.at || b.end() <= a.at) return false;
    for (int64_t i = 0; i < a.mats; ++i)
        for (int64_t j = 0; j < b.mats; ++j)
            if (op_matrices_meet(a, i, b, j)) return true;
    return false;
}
int op_check_overlap(const char *fn, const OpRegion &result, std::initializer_list<OpRegion> operands) {
    for (const OpRegion &o : operands)
        if (op_overlap(result, o)) return op_fail(fn, "the result must not overlap an operand");
    return MOE_OK;
}
constexpr int64_t op_bytes(int32_t dtype) { return dtype == MOE_F32 ? 4 : (dtype == MOE_BF16 ? 2 : 1); }
bool op_misaligned(const void *p, int32_t dtype) { return ((uintptr_t)p & (dtype == MOE_F32 ? 3 : 1)) != 0; }

// y[r] = W_e x[r] (grad: dx[r] = W_e^T dy[r]) on rows of k elements -> n
int op_rows_product(const char *fn, bool grad, const void *x, int64_t ldx, const void *w, int64_t ldw,
                    int64_t w_stride, int32_t layout, const int32_t *offsets, int32_t groups, int32_t rows,
                    int32_t in_dim, int32_t out_dim, int32_t dtype, void *y, int64_t ldy, int32_t y_dtype,
                    void *workspace, int64_t workspace_bytes, void *stream) {
    int r = op_check_groups(fn, offsets, groups, rows, in_dim, out_dim);
    if (r == MOE_OK) r = op_check_dtypes(fn, dtype, y_dtype);
    if (r != MOE_OK) return r;
    if (layout != MOE_LAYOUT_FLUX_OUT_IN && layout != MOE_LAYOUT_LLAMA_IN_OUT) return op_fail(fn, "unknown layout");
    const int k = grad ? out_dim : in_dim, n = grad ? in_dim : out_dim;
    const bool flux = layout == MOE_LAYOUT_FLUX_OUT_IN;
    const int wcols = flux ? out_dim : in_dim, wrows = flux ? in_dim : out_dim;
    if (ldx < k || ldy < n || ldw < wcols) return op_fail(fn, "a row stride is smaller than its row");
    if (groups > 1 && w_stride < (wrows - 1) * ldw + wcols) return op_fail(fn, "w_stride is smaller than a matrix");
    if (rows == 0) return MOE_OK;
    if (!x || !w || !y) return op_fail(fn, "null buffer");
    if (op_misaligned(x, dtype) || op_misaligned(w, dtype) || op_misaligned(y, y_dtype))
        return op_fail(fn, "a buffer is not aligned to its elements");
    OpGemmArgs g{};
    g.A = x, g.B = w, g.C = y;
    g.lda = ldx, g.ldb = ldw, g.ldc = ldy;
    g.b_stride = groups > 1 ? w_stride : 0;
    g.offsets = offsets, g.E = groups, g.rows = rows;
    g.N = n, g.K = k, g.c_f32 = y_dtype == MOE_F32;
    // the weight is a "row" operand where its contiguous axis is the product's k
    const bool b_col = flux != grad;
    g.splits = op_rows_splits(dtype == MOE_F32 ? OT_F32 : OT_BF16, b_col, rows, groups, n, k, op_cus());
    g.ws = (float *)workspace;
    r = op_check_workspace(fn, g.splits > 1 ? (int64_t)4 * g.splits * rows * n : 0, workspace, workspace_bytes);
    if (r != MOE_OK) return r;
    const int64_t es = op_bytes(dtype);
    r = op_check_overlap(fn, OpRegion(y, n, ldy, rows, 0, 1, op_bytes(y_dtype)),
                         {OpRegion(x, k, ldx, rows, 0, 1, es), OpRegion(w, wcols, ldw, wrows, w_stride, groups, es),
                          OpRegion(offsets, 4 * ((int64_t)groups + 1))});
    if (r != MOE_OK) return r;
    return op_done(fn, dtype == MOE_F32 ? launch_op_gemm_f32(b_col, false, g, op_cus(), (hipStream_t)stream)
                                        : launch_op_gemm_bf16(b_col, false, g, op_cus(), (hipStream_t)stream));
}
}  // namespace

extern "C" {

int moe_grouped_matmul_async(const void *x, int64_t ldx, const void *w, int64_t ldw, int64_t w_stride, int32_t layout,
                             const int32_t *offsets, int32_t groups, int32_t rows, int32_t in_dim, int32_t out_dim,
                             int32_t dtype, void *y, int64_t ldy, int32_t y_dtype, void *workspace,
                             int64_t workspace_bytes, void *stream) {
    return op_rows_product("moe_grouped_matmul_async", false, x, ldx, w, ldw, w_stride, layout, offsets, groups, rows,
                           in_dim, out_dim, dtype, y, ldy, y_dtype, workspace, workspace_bytes, stream);
}

int moe_grouped_matmul_grad_x_async(const void *dy, int64_t lddy, const void *w, int64_t ldw, int64_t w_stride,
                                    int32_t layout, const int32_t *offsets, int32_t groups, int32_t rows,
                                    int32_t in_dim, int32_t out_dim, int32_t dtype, void *dx, int64_t lddx,
                                    int32_t dx_dtype, void *workspace, int64_t workspace_bytes, void *stream) {
    return op_rows_product("moe_grouped_matmul_grad_x_async", true, dy, lddy, w, ldw, w_stride, layout, offsets,
                           groups, rows, in_dim, out_dim, dtype, dx, lddx, dx_dtype, workspace, workspace_bytes, stream);
}

int moe_grouped_matmul_grad_w_workspace(int32_t groups, int32_t rows, int32_t in_dim, int32_t out_dim,
                                        int64_t *bytes) {
    const char *fn = "moe_grouped_matmul_grad_w_workspace";
    if (!bytes) return op_fail(fn, "null bytes");
    int r = op_check_groups(fn, (const int32_t *)bytes, groups, rows, in_dim, out_dim);
    if (r != MOE_OK) return r;
    // enough for either type
    const int splits = std::max(op_matrix_splits(OT_F32, rows, groups, in_dim, out_dim, op_cus()),
                                op_matrix_splits(OT_BF16, rows, groups, in_dim, out_dim, op_cus()));
    *bytes = splits > 1 ? (int64_t)4 * splits * groups * in_dim * out_dim : 0;
    return MOE_OK;
}

int moe_grouped_matmul_workspace(int32_t groups, int32_t rows, int32_t in_dim, int32_t out_dim, int32_t dtype,
                                 int64_t *bytes) {
    const char *fn = "moe_grouped_matmul_workspace";
    if (!bytes) return op_fail(fn, "null bytes");
    int r = op_check_groups(fn, (const int32_t *)bytes, groups, rows, in_dim, out_dim);
    if (r == MOE_OK) r = op_check_dtypes(fn, dtype, MOE_F32);
    if (r != MOE_OK) return r;
    *bytes = 0;
    if (rows == 0) return MOE_OK;
    // enough for either layout, forward or row gradient
    const int ot = dtype == MOE_F32 ? OT_F32 : OT_BF16;
    for (const bool col : {false, true}) {
        const int s = op_rows_splits(ot, col, rows, groups, out_dim, in_dim, op_cus());
        const int t = op_rows_splits(ot, col, rows, groups, in_dim, out_dim, op_cus());
        if (s > 1) *bytes = std::max(*bytes, (int64_t)4 * s * rows * out_dim);
        if (t > 1) *bytes = std::max(*bytes, (int64_t)4 * t * rows * in_dim);
    }
    return MOE_OK;
}

int moe_grouped_matmul_grad_w_async(const void *x, int64_t ldx, const void *dy, int64_t lddy, int32_t layout,
                                    const int32_t *offsets, int32_t groups, int32_t rows, int32_t in_dim,
                                    int32_t out_dim, int32_t dtype, void *dw, int64_t lddw, int64_t dw_stride,
                                    int32_t dw_dtype, int32_t accumulate, void *workspace, int64_t workspace_bytes,
                                    void *stream) {
    const char *fn = "moe_grouped_matmul_grad_w_async";
    int r = op_check_groups(fn, offsets, groups, rows, in_dim, out_dim);
    if (r == MOE_OK) r = op_check_dtypes(fn, dtype, dw_dtype);
    if (r != MOE_OK) return r;
    if (layout != MOE_LAYOUT_FLUX_OUT_IN && layout != MOE_LAYOUT_LLAMA_IN_OUT) return op_fail(fn, "unknown layout");
    const bool flux = layout == MOE_LAYOUT_FLUX_OUT_IN;
    const int m = flux ? in_dim : out_dim, n = flux ? out_dim : in_dim;
    if (ldx < in_dim || lddy < out_dim || lddw < n) return op_fail(fn, "a row stride is smaller than its row");
    if (groups > 1 && dw_stride < (m - 1) * lddw + n) return op_fail(fn, "dw_stride is smaller than a matrix");
    if (!dw || (rows > 0 && (!x || !dy))) return op_fail(fn, "null buffer");
    if (op_misaligned(x, dtype) || op_misaligned(dy, dtype) || op_misaligned(dw, dw_dtype))
        return op_fail(fn, "a buffer is not aligned to its elements");
    if (rows == 0 && accumulate) return MOE_OK;
    int64_t need = 0;
    r = moe_grouped_matmul_grad_w_workspace(groups, rows, in_dim, out_dim, &need);
    if (r != MOE_OK) return r;
    r = op_check_workspace(fn, need, workspace, workspace_bytes);
    if (r != MOE_OK) return r;
    if (rows > 0) {
        const int64_t es = op_bytes(dtype);
        r = op_check_overlap(fn, OpRegion(dw, n, lddw, m, dw_stride, groups, op_bytes(dw_dtype)),
                             {OpRegion(x, in_dim, ldx, rows, 0, 1, es), OpRegion(dy, out_dim, lddy, rows, 0, 1, es),
                              OpRegion(offsets, 4 * ((int64_t)groups + 1))});
        if (r != MOE_OK) return r;
    }
    OpGemmArgs g{};
    g.A = flux ? x : dy, g.B = flux ? dy : x, g.C = dw;
    g.lda = flux ? ldx : lddy, g.ldb = flux ? lddy : ldx, g.ldc = lddw;
    g.c_stride = groups > 1 ? dw_stride : 0;
    g.offsets = offsets, g.E = groups, g.rows = rows;
    g.M = m, g.N = n, g.c_f32 = dw_dtype == MOE_F32, g.accumulate = accumulate != 0;
    g.splits = op_matrix_splits(dtype == MOE_F32 ? OT_F32 : OT_BF16, rows, groups, m, n, op_cus());
    g.ws = (float *)workspace;
    return op_done(fn, dtype == MOE_F32 ? launch_op_gemm_f32(true, true, g, op_cus(), (hipStream_t)stream)
                                        : launch_op_gemm_bf16(true, true, g, op_cus(), (hipStream_t)stream));
}

// ---- gated blocks --------------------------------------------------------------------
static int op_check_gated(const char *fn, const int32_t *offsets, int32_t groups, int32_t rows, int32_t in_dim,
                          int32_t out_dim, int32_t dtype, int32_t out_dtype, int32_t layout, int32_t activation) {
    int r = op_check_groups(fn, offsets, groups, rows, in_dim, out_dim);
    if (r == MOE_OK) r = op_check_dtypes(fn, dtype, out_dtype);
    if (r != MOE_OK) return r;
    if (layout != MOE_LAYOUT_FLUX_OUT_IN && layout != MOE_LAYOUT_LLAMA_IN_OUT) return op_fail(fn, "unknown layout");
    if (activation < MOE_ACT_GELU || activation > MOE_ACT_IDENTITY) return op_fail(fn, "unknown activation");
    return MOE_OK;
}
static int64_t gated_workspace(OpMode mode, int32_t groups, int32_t rows, int32_t n, int32_t k, int32_t dtype) {
    int64_t bytes = 0;
    if (rows == 0) return 0;
    for (const bool col : {false, true}) {  // enough for either layout
        const int s = op_gated_splits(mode, dtype == MOE_F32 ? OT_F32 : OT_BF16, col, rows, groups, n, k, op_cus());
        if (s > 1) bytes = std::max(bytes, (int64_t)4 * (mode == OM_GATED ? 2 : 1) * s * rows * n);
    }
    if (mode == OM_TWO && op_two_tail(dtype == MOE_F32 ? OT_F32 : OT_BF16, rows, groups, n, k, op_cus()))
        bytes = std::max(bytes, (int64_t)4 * kOpTailTile * 8 * (op_cus() / 8));
    return bytes;
}
static int gated_workspace_of(const char *fn, OpMode mode, int32_t groups, int32_t rows, int32_t n, int32_t k,
                              int32_t dtype, int64_t *bytes) {
    if (!bytes) return op_fail(fn, "null bytes");
    int r = op_check_groups(fn, (const int32_t *)bytes, groups, rows, n, k);
    if (r == MOE_OK) r = op_check_dtypes(fn, dtype, MOE_F32);
    if (r != MOE_OK) return r;
    *bytes = gated_workspace(mode, groups, rows, n, k, dtype);
    return MOE_OK;
}
// No result may share a byte with an operand or with another result.
static int op_check_results(const char *fn, std::initializer_list<OpRegion> results,
                            std::initializer_list<OpRegion> operands) {
    for (const OpRegion *a = results.begin(); a != results.end(); ++a) {
        const int r = op_check_overlap(fn, *a, operands);
        if (r != MOE_OK) return r;
        for (const OpRegion *b = results.begin(); b != a; ++b)
            if (op_overlap(*a, *b)) return op_fail(fn, "results must not overlap each other");
    }
    return MOE_OK;
}
static bool op_any_misaligned(int32_t dtype, std::initializer_list<const void *> ps) {
    for (const void *p : ps)
        if (op_misaligned(p, dtype)) return true;
    return false;
}

int moe_gated_matmul_workspace(int32_t groups, int32_t rows, int32_t in_dim, int32_t hidden_dim, int32_t dtype,
                               int64_t *bytes) {
    return gated_workspace_of("moe_gated_matmul_workspace", OM_GATED, groups, rows, hidden_dim, in_dim, dtype, bytes);
}

int moe_gated_matmul_async(const void *x, int64_t ldx, const void *w1, int64_t ldw1, int64_t w1_stride, const void *w3,
                           int64_t ldw3, int64_t w3_stride, int32_t layout, int32_t activation, const int32_t *offsets,
                           int32_t groups, int32_t rows, int32_t in_dim, int32_t hidden_dim, int32_t dtype, void *h,
                           int64_t ldh, int32_t h_dtype, void *a, int64_t lda, void *b, int64_t ldb, void *workspace,
                           int64_t workspace_bytes, void *stream) {
    const char *fn = "moe_gated_matmul_async";
    int r = op_check_gated(fn, offsets, groups, rows, in_dim, hidden_dim, dtype, h_dtype, layout, activation);
    if (r != MOE_OK) return r;
    const bool flux = layout == MOE_LAYOUT_FLUX_OUT_IN;
    const int wcols = flux ? hidden_dim : in_dim, wrows = flux ? in_dim : hidden_dim;
    if ((a != nullptr) != (b != nullptr)) return op_fail(fn, "a and b come together");
    if (ldx < in_dim || ldh < hidden_dim || ldw1 < wcols || ldw3 < wcols || (a && (lda < hidden_dim || ldb < hidden_dim)))
        return op_fail(fn, "a row stride is smaller than its row");
    if (groups > 1 && (w1_stride < (wrows - 1) * ldw1 + wcols || w3_stride < (wrows - 1) * ldw3 + wcols))
        return op_fail(fn, "a weight's stride is smaller than a matrix");
    if (rows == 0) return MOE_OK;
    if (!x || !w1 || !w3 || !h) return op_fail(fn, "null buffer");
    if (op_any_misaligned(dtype, {x, w1, w3, a, b}) || op_misaligned(h, h_dtype))
        return op_fail(fn, "a buffer is not aligned to its elements");
    r = op_check_workspace(fn, gated_workspace(OM_GATED, groups, rows, hidden_dim, in_dim, dtype), workspace, workspace_bytes);
    if (r != MOE_OK) return r;
    const int64_t es = op_bytes(dtype);
    r = op_check_results(fn,
                         {OpRegion(h, hidden_dim, ldh, rows, 0, 1, op_bytes(h_dtype)), OpRegion(a, hidden_dim, lda, rows, 0, 1, es),
                          OpRegion(b, hidden_dim, ldb, rows, 0, 1, es)},
                         {OpRegion(x, in_dim, ldx, rows, 0, 1, es), OpRegion(w1, wcols, ldw1, wrows, w1_stride, groups, es),
                          OpRegion(w3, wcols, ldw3, wrows, w3_stride, groups, es),
                          OpRegion(offsets, 4 * ((int64_t)groups + 1))});
    if (r != MOE_OK) return r;
    OpGemmArgs g{};
    g.A = x, g.lda = ldx;
    g.B = w1, g.ldb = ldw1, g.b_stride = groups > 1 ? w1_stride : 0;
    g.B2 = w3, g.ldb2 = ldw3, g.b2_stride = groups > 1 ? w3_stride : 0;
    g.C = h, g.ldc = ldh, g.c_f32 = h_dtype == MOE_F32;
    g.C2 = a, g.ldc2 = lda, g.C3 = b, g.ldc3 = ldb;
    g.offsets = offsets, g.E = groups, g.rows = rows, g.N = hidden_dim, g.K = in_dim, g.act = activation;
    const int ot = dtype == MOE_F32 ? OT_F32 : OT_BF16;
    g.splits = op_gated_splits(OM_GATED, ot, flux, rows, groups, hidden_dim, in_dim, op_cus());
    g.ws = (float *)workspace;
    return op_done(fn, launch_op_gated(OM_GATED, ot, flux, g, op_cus(), (hipStream_t)stream));
}

int moe_gated_matmul_grad_workspace(int32_t groups, int32_t rows, int32_t hidden_dim, int32_t out_dim, int32_t dtype,
                                    int64_t *bytes) {
    return gated_workspace_of("moe_gated_matmul_grad_workspace", OM_GATE_GRAD, groups, rows, hidden_dim, out_dim, dtype, bytes);
}

int moe_gated_matmul_grad_async(const void *dy, int64_t lddy, const void *w2, int64_t ldw2, int64_t w2_stride,
                                int32_t layout, int32_t activation, const void *a, int64_t lda, const void *b, int64_t ldb,
                                const int32_t *offsets, int32_t groups, int32_t rows, int32_t hidden_dim, int32_t out_dim,
                                int32_t dtype, void *da, int64_t ldda, void *db, int64_t lddb, void *h, int64_t ldh,
                                void *workspace, int64_t workspace_bytes, void *stream) {
    const char *fn = "moe_gated_matmul_grad_async";
    int r = op_check_gated(fn, offsets, groups, rows, hidden_dim, out_dim, dtype, dtype, layout, activation);
    if (r != MOE_OK) return r;
    const bool flux = layout == MOE_LAYOUT_FLUX_OUT_IN;
    const int wcols = flux ? out_dim : hidden_dim, wrows = flux ? hidden_dim : out_dim;
    if (!w2 && out_dim != hidden_dim) return op_fail(fn, "without w2 dy is the gradient of h: out_dim must be hidden_dim");
    if (lddy < out_dim || (w2 && ldw2 < wcols) || std::min({lda, ldb, ldda, lddb, ldh}) < hidden_dim)
        return op_fail(fn, "a row stride is smaller than its row");
    if (w2 && groups > 1 && w2_stride < (wrows - 1) * ldw2 + wcols) return op_fail(fn, "w2_stride is smaller than a matrix");
    if (rows == 0) return MOE_OK;
    if (!dy || !a || !b || !da || !db || !h) return op_fail(fn, "null buffer");
    if (op_any_misaligned(dtype, {dy, w2, a, b, da, db, h})) return op_fail(fn, "a buffer is not aligned to its elements");
    if (w2) {
        r = op_check_workspace(fn, gated_workspace(OM_GATE_GRAD, groups, rows, hidden_dim, out_dim, dtype), workspace,
                               workspace_bytes);
        if (r != MOE_OK) return r;
    }
    const int64_t es = op_bytes(dtype);
    auto rows_of = [&](const void *p, int64_t cols, int64_t ld) { return OpRegion(p, cols, ld, rows, 0, 1, es); };
    r = op_check_results(fn, {rows_of(da, hidden_dim, ldda), rows_of(db, hidden_dim, lddb), rows_of(h, hidden_dim, ldh)},
                         {rows_of(dy, out_dim, lddy), rows_of(a, hidden_dim, lda), rows_of(b, hidden_dim, ldb),
                          OpRegion(w2, wcols, ldw2, wrows, w2_stride, groups, es),
                          OpRegion(offsets, 4 * ((int64_t)groups + 1))});
    if (r != MOE_OK) return r;
    OpGemmArgs g{};
    g.A = dy, g.lda = lddy;
    g.B = w2, g.ldb = ldw2, g.b_stride = groups > 1 ? w2_stride : 0;
    g.ga = a, g.ldga = lda, g.gb = b, g.ldgb = ldb;
    g.C = da, g.ldc = ldda, g.C2 = db, g.ldc2 = lddb, g.C3 = h, g.ldc3 = ldh;
    g.offsets = offsets, g.E = groups, g.rows = rows, g.N = hidden_dim, g.K = out_dim, g.act = activation;
    g.c_f32 = dtype == MOE_F32, g.splits = 1;
    const int ot = dtype == MOE_F32 ? OT_F32 : OT_BF16;
    if (!w2) return op_done(fn, launch_op_gate_rows(ot, g, (hipStream_t)stream));
    // dh = W2' dy: the weight's k is its out_dim, contiguous in the flux order
    g.splits = op_gated_splits(OM_GATE_GRAD, ot, !flux, rows, groups, hidden_dim, out_dim, op_cus());
    g.ws = (float *)workspace;
    return op_done(fn, launch_op_gated(OM_GATE_GRAD, ot, !flux, g, op_cus(), (hipStream_t)stream));
}

int moe_gated_matmul_grad_x_workspace(int32_t groups, int32_t rows, int32_t in_dim, int32_t hidden_dim, int32_t dtype,
                                      int64_t *bytes) {
    return gated_workspace_of("moe_gated_matmul_grad_x_workspace", OM_TWO, groups, rows, in_dim, hidden_dim, dtype, bytes);
}

int moe_gated_matmul_grad_x_async(const void *da, int64_t ldda, const void *db, int64_t lddb, const void *w1,
                                  int64_t ldw1, int64_t w1_stride, const void *w3, int64_t ldw3, int64_t w3_stride,
                                  int32_t layout, const int32_t *offsets, int32_t groups, int32_t rows, int32_t in_dim,
                                  int32_t hidden_dim, int32_t dtype, void *dx, int64_t lddx, int32_t dx_dtype,
                                  void *workspace, int64_t workspace_bytes, void *stream) {
    const char *fn = "moe_gated_matmul_grad_x_async";
    int r = op_check_gated(fn, offsets, groups, rows, in_dim, hidden_dim, dtype, dx_dtype, layout, MOE_ACT_IDENTITY);
    if (r != MOE_OK) return r;
    const bool flux = layout == MOE_LAYOUT_FLUX_OUT_IN;
    const int wcols = flux ? hidden_dim : in_dim, wrows = flux ? in_dim : hidden_dim;
    if (ldda < hidden_dim || lddb < hidden_dim || lddx < in_dim || ldw1 < wcols || ldw3 < wcols)
        return op_fail(fn, "a row stride is smaller than its row");
    if (groups > 1 && (w1_stride < (wrows - 1) * ldw1 + wcols || w3_stride < (wrows - 1) * ldw3 + wcols))
        return op_fail(fn, "a weight's stride is smaller than a matrix");
    if (rows == 0) return MOE_OK;
    if (!da || !db || !w1 || !w3 || !dx) return op_fail(fn, "null buffer");
    if (op_any_misaligned(dtype, {da, db, w1, w3}) || op_misaligned(dx, dx_dtype))
        return op_fail(fn, "a buffer is not aligned to its elements");
    r = op_check_workspace(fn, gated_workspace(OM_TWO, groups, rows, in_dim, hidden_dim, dtype), workspace, workspace_bytes);
    if (r != MOE_OK) return r;
    const int64_t es = op_bytes(dtype);
    r = op_check_overlap(fn, OpRegion(dx, in_dim, lddx, rows, 0, 1, op_bytes(dx_dtype)),
                         {OpRegion(da, hidden_dim, ldda, rows, 0, 1, es), OpRegion(db, hidden_dim, lddb, rows, 0, 1, es),
                          OpRegion(w1, wcols, ldw1, wrows, w1_stride, groups, es),
                          OpRegion(w3, wcols, ldw3, wrows, w3_stride, groups, es),
                          OpRegion(offsets, 4 * ((int64_t)groups + 1))});
    if (r != MOE_OK) return r;
    OpGemmArgs g{};
    g.A = da, g.lda = ldda, g.A2 = db, g.lda2 = lddb;
    g.B = w1, g.ldb = ldw1, g.b_stride = groups > 1 ? w1_stride : 0;
    g.B2 = w3, g.ldb2 = ldw3, g.b2_stride = groups > 1 ? w3_stride : 0;
    g.C = dx, g.ldc = lddx, g.c_f32 = dx_dtype == MOE_F32;
    g.offsets = offsets, g.E = groups, g.rows = rows, g.N = in_dim, g.K = hidden_dim;
    const int ot = dtype == MOE_F32 ? OT_F32 : OT_BF16;
    g.splits = op_gated_splits(OM_TWO, ot, !flux, rows, groups, in_dim, hidden_dim, op_cus());
    g.tail = op_two_tail(ot, rows, groups, in_dim, hidden_dim, op_cus()) ? op_cus() / 8 : 0;
    g.ws = (float *)workspace;
    return op_done(fn, launch_op_gated(OM_TWO, ot, !flux, g, op_cus(), (hipStream_t)stream));
}

int moe_quantize_int8_async(const void *x, int64_t ldx, int32_t x_dtype, int64_t rows, int32_t cols, void *q,
                            int64_t ldq, float *scale, void *stream) {
    const char *fn = "moe_quantize_int8_async";
    if (x_dtype != MOE_F32 && x_dtype != MOE_BF16) return op_fail(fn, "x_dtype must be MOE_F32 or MOE_BF16");
    if (rows < 0 || cols < 1) return op_fail(fn, "rows must not be negative and cols positive");
    if (cols > kOpMaxSize) return op_fail(fn, "sizes above 2^30");
    if (rows > kOpMaxSize) return op_fail(fn, "too many rows (above 2^30)");
    if (ldx < cols || ldq < cols) return op_fail(fn, "a row stride is smaller than its row");
    if (rows == 0) return MOE_OK;
    if (!x || !q || !scale) return op_fail(fn, "null buffer");
    if (op_misaligned(x, x_dtype) || op_misaligned(scale, MOE_F32))
        return op_fail(fn, "a buffer is not aligned to its elements");
    const OpRegion from(x, cols, ldx, rows, 0, 1, op_bytes(x_dtype)), codes(q, cols, ldq, rows, 0, 1, 1), scales(scale, 4 * rows);
    int r = op_check_overlap(fn, codes, {from, scales});
    if (r == MOE_OK) r = op_check_overlap(fn, scales, {from});
    if (r != MOE_OK) return r;
    return op_done(fn, launch_quantize_i8(x, ldx, x_dtype == MOE_BF16, rows, cols, (int8_t *)q, ldq, cols, scale,
                                          (hipStream_t)stream));
}

// Workspace of the int8 product: partial sums, then the rows' scales and codes
// (padded to 16 bytes) where the call quantises them.
static int64_t int8_partial_bytes(int32_t groups, int32_t rows, int32_t in_dim, int32_t out_dim) {
    const int s = op_rows_splits(OT_I8, false, rows, groups, out_dim, in_dim, op_cus());
    return s > 1 ? round_up((int64_t)4 * s * rows * out_dim, 16) : 0;
}

int moe_int8_matmul_workspace(int32_t groups, int32_t rows, int32_t in_dim, int32_t out_dim, int32_t x_dtype,
                              int64_t *bytes) {
    const char *fn = "moe_int8_matmul_workspace";
    if (!bytes) return op_fail(fn, "null bytes");
    const int r = op_check_groups(fn, (const int32_t *)bytes, groups, rows, in_dim, out_dim);
    if (r != MOE_OK) return r;
    *bytes = rows > 0 ? int8_partial_bytes(groups, rows, in_dim, out_dim) : 0;
    if (x_dtype != MOE_INT8) *bytes += round_up((int64_t)rows * 4, 16) + (int64_t)rows * round_up(in_dim, 16);
    return MOE_OK;
}

int moe_int8_matmul_async(const void *x, int64_t ldx, int32_t x_dtype, const float *x_scale, const void *w,
                          int64_t ldw, int64_t w_stride, const float *w_scale, const int32_t *offsets, int32_t groups,
                          int32_t rows, int32_t in_dim, int32_t out_dim, void *y, int64_t ldy, int32_t y_dtype,
                          void *workspace, int64_t workspace_bytes, void *stream) {
    const char *fn = "moe_int8_matmul_async";
    int r = op_check_groups(fn, offsets, groups, rows, in_dim, out_dim);
    if (r != MOE_OK) return r;
    const bool codes = x_dtype == MOE_INT8;
    if (!codes && x_dtype != MOE_F32 && x_dtype != MOE_BF16)
        return op_fail(fn, "x_dtype must be MOE_INT8, MOE_BF16 or MOE_F32");
    if (y_dtype != MOE_F32 && y_dtype != MOE_BF16) return op_fail(fn, "the result must be MOE_F32 or MOE_BF16");
    if (in_dim > 131071) return op_fail(fn, "in_dim above 131071 (the int32 sums could overflow)");
    if (ldx < in_dim || ldy < out_dim || ldw < in_dim) return op_fail(fn, "a row stride is smaller than its row");
    if (groups > 1 && w_stride < (out_dim - 1) * ldw + in_dim) return op_fail(fn, "w_stride is smaller than a matrix");
    if (rows == 0) return MOE_OK;
    if (!x || !w || !w_scale || !y) return op_fail(fn, "null buffer");
    if (codes && !x_scale) return op_fail(fn, "int8 rows need x_scale");
    if ((!codes && op_misaligned(x, x_dtype)) || op_misaligned(y, y_dtype) || op_misaligned(w_scale, MOE_F32) ||
        (codes && op_misaligned(x_scale, MOE_F32)))
        return op_fail(fn, "a buffer is not aligned to its elements");
    int64_t need = 0;
    r = moe_int8_matmul_workspace(groups, rows, in_dim, out_dim, x_dtype, &need);
    if (r == MOE_OK) r = op_check_workspace(fn, need, workspace, workspace_bytes);
    if (r != MOE_OK) return r;
    r = op_check_overlap(fn, OpRegion(y, out_dim, ldy, rows, 0, 1, op_bytes(y_dtype)),
                         {OpRegion(x, in_dim, ldx, rows, 0, 1, op_bytes(x_dtype)),
                          OpRegion(w, in_dim, ldw, out_dim, w_stride, groups, 1), OpRegion(codes ? x_scale : nullptr, 4 * (int64_t)rows),
                          OpRegion(w_scale, 4 * (int64_t)groups * out_dim), OpRegion(offsets, 4 * ((int64_t)groups + 1))});
    if (r != MOE_OK) return r;
    if (!codes) {
        float *sx = (float *)((uint8_t *)workspace + int8_partial_bytes(groups, rows, in_dim, out_dim));
        int8_t *q = (int8_t *)sx + round_up((int64_t)rows * 4, 16);
        const int64_t ldq = round_up(in_dim, 16);
        r = op_done(fn, launch_quantize_i8(x, ldx, x_dtype == MOE_BF16, rows, in_dim, q, ldq, (int)ldq, sx,
                                           (hipStream_t)stream));
        if (r != MOE_OK) return r;
        x = q, ldx = ldq, x_scale = sx;
    }
    OpGemmArgs g{};
    g.A = x, g.B = w, g.C = y;
    g.lda = ldx, g.ldb = ldw, g.ldc = ldy;
    g.b_stride = groups > 1 ? w_stride : 0;
    g.offsets = offsets, g.E = groups, g.rows = rows;
    g.N = out_dim, g.K = in_dim, g.c_f32 = y_dtype == MOE_F32;
    g.splits = op_rows_splits(OT_I8, false, rows, groups, out_dim, in_dim, op_cus());
    g.ws = (float *)workspace;
    g.sa = x_scale, g.sb = w_scale;
    return op_done(fn, launch_op_gemm_i8(g, op_cus(), (hipStream_t)stream));
}

// ---- 8-bit floating point ------------------------------------------------------------
int moe_quantize_fp8_async(const void *x, int64_t ldx, int64_t x_stride, int32_t x_dtype, int64_t matrices, int64_t rows,
                           int32_t cols, int32_t block_rows, void *q, int64_t ldq, int64_t q_stride, float *scale,
                           void *stream) {
    const char *fn = "moe_quantize_fp8_async";
    if (x_dtype != MOE_F32 && x_dtype != MOE_BF16) return op_fail(fn, "x_dtype must be MOE_F32 or MOE_BF16");
    if (block_rows != 1 && block_rows != kF8Block) return op_fail(fn, "block_rows must be 1 or 128");
    if (matrices < 0 || rows < 0 || cols < 1) return op_fail(fn, "matrices and rows must not be negative and cols positive");
    if (matrices > kOpMaxSize || rows > kOpMaxSize || cols > kOpMaxSize) return op_fail(fn, "sizes above 2^30");
    if (ldx < cols || ldq < cols) return op_fail(fn, "a row stride is smaller than its row");
    if (matrices > 1 && (x_stride < (rows - 1) * ldx + cols || q_stride < (rows - 1) * ldq + cols))
        return op_fail(fn, "a matrix stride is smaller than a matrix");
    if (matrices == 0 || rows == 0) return MOE_OK;
    if (!x || !q || !scale) return op_fail(fn, "null buffer");
    if (op_misaligned(x, x_dtype) || op_misaligned(scale, MOE_F32))
        return op_fail(fn, "a buffer is not aligned to its elements");
    const int64_t scales = matrices * ((rows + block_rows - 1) / block_rows) * ((cols + kF8Block - 1) / kF8Block);
    const OpRegion from(x, cols, ldx, rows, x_stride, matrices, op_bytes(x_dtype));
    const int r = op_check_results(fn, {OpRegion(q, cols, ldq, rows, q_stride, matrices, 1), OpRegion(scale, 4 * scales)}, {from});
    if (r != MOE_OK) return r;
    const QuantF8Args a{x, ldx, matrices > 1 ? x_stride : 0, x_dtype == MOE_BF16, matrices, rows, cols, block_rows,
                        (uint8_t *)q, ldq, matrices > 1 ? q_stride : 0, cols, scale};
    return op_done(fn, launch_quantize_f8(a, (hipStream_t)stream));
}

// Workspace of the product: partial sums, then the rows' scales and codes (padded to 16
// bytes) where the call quantises them.
static int64_t fp8_partial_bytes(int32_t groups, int32_t rows, int32_t in_dim, int32_t out_dim) {
    const int s = op_f8_splits(rows, groups, out_dim, in_dim, op_cus());
    return s > 1 ? round_up((int64_t)4 * s * rows * out_dim, 16) : 0;
}
static int64_t fp8_blocks(int64_t n) { return (n + kF8Block - 1) / kF8Block; }

int moe_fp8_matmul_workspace(int32_t groups, int32_t rows, int32_t in_dim, int32_t out_dim, int32_t x_dtype,
                             int64_t *bytes) {
    const char *fn = "moe_fp8_matmul_workspace";
    if (!bytes) return op_fail(fn, "null bytes");
    const int r = op_check_groups(fn, (const int32_t *)bytes, groups, rows, in_dim, out_dim);
    if (r != MOE_OK) return r;
    *bytes = rows > 0 ? fp8_partial_bytes(groups, rows, in_dim, out_dim) : 0;
    if (x_dtype != MOE_FP8_E4M3)
        *bytes += round_up((int64_t)rows * fp8_blocks(in_dim) * 4, 16) + (int64_t)rows * round_up((int64_t)in_dim, 16);
    return MOE_OK;
}

static int fp8_matmul(const char *fn, bool exact, const void *x, int64_t ldx, int32_t x_dtype, const float *x_scale,
                      const void *w, int64_t ldw, int64_t w_stride, const float *w_scale, const int32_t *offsets,
                      int32_t groups, int32_t rows, int32_t in_dim, int32_t out_dim, void *y, int64_t ldy, int32_t y_dtype,
                      void *workspace, int64_t workspace_bytes, void *stream) {
    int r = op_check_groups(fn, offsets, groups, rows, in_dim, out_dim);
    if (r != MOE_OK) return r;
    const bool codes = x_dtype == MOE_FP8_E4M3;
    if (!codes && x_dtype != MOE_F32 && x_dtype != MOE_BF16)
        return op_fail(fn, "x_dtype must be MOE_FP8_E4M3, MOE_BF16 or MOE_F32");
    if (y_dtype != MOE_F32 && y_dtype != MOE_BF16) return op_fail(fn, "the result must be MOE_F32 or MOE_BF16");
    if (ldx < in_dim || ldy < out_dim || ldw < in_dim) return op_fail(fn, "a row stride is smaller than its row");
    if (groups > 1 && w_stride < (out_dim - 1) * ldw + in_dim) return op_fail(fn, "w_stride is smaller than a matrix");
    if (rows == 0) return MOE_OK;
    if (!x || !w || !w_scale || !y) return op_fail(fn, "null buffer");
    if (codes && !x_scale) return op_fail(fn, "coded rows need x_scale");
    if ((!codes && op_misaligned(x, x_dtype)) || op_misaligned(y, y_dtype) || op_misaligned(w_scale, MOE_F32) ||
        (codes && op_misaligned(x_scale, MOE_F32)))
        return op_fail(fn, "a buffer is not aligned to its elements");
    int64_t need = 0;
    r = moe_fp8_matmul_workspace(groups, rows, in_dim, out_dim, x_dtype, &need);
    if (r == MOE_OK) r = op_check_workspace(fn, need, workspace, workspace_bytes);
    if (r != MOE_OK) return r;
    const int64_t kb = fp8_blocks(in_dim);
    r = op_check_overlap(fn, OpRegion(y, out_dim, ldy, rows, 0, 1, op_bytes(y_dtype)),
                         {OpRegion(x, in_dim, ldx, rows, 0, 1, op_bytes(x_dtype)),
                          OpRegion(w, in_dim, ldw, out_dim, w_stride, groups, 1),
                          OpRegion(codes ? x_scale : nullptr, 4 * (int64_t)rows * kb),
                          OpRegion(w_scale, 4 * (int64_t)groups * fp8_blocks(out_dim) * kb),
                          OpRegion(offsets, 4 * ((int64_t)groups + 1))});
    if (r != MOE_OK) return r;
    if (!codes) {
        float *sx = (float *)((uint8_t *)workspace + fp8_partial_bytes(groups, rows, in_dim, out_dim));
        uint8_t *q = (uint8_t *)sx + round_up((int64_t)rows * kb * 4, 16);
        const int64_t ldq = round_up((int64_t)in_dim, 16);
        const QuantF8Args a{x, ldx, 0, x_dtype == MOE_BF16, 1, rows, in_dim, 1, q, ldq, 0, (int)ldq, sx};
        r = op_done(fn, launch_quantize_f8(a, (hipStream_t)stream));
        if (r != MOE_OK) return r;
        x = q, ldx = ldq, x_scale = sx;
    }
    OpGemmArgs g{};
    g.A = x, g.B = w, g.C = y;
    g.lda = ldx, g.ldb = ldw, g.ldc = ldy;
    g.b_stride = groups > 1 ? w_stride : 0;
    g.offsets = offsets, g.E = groups, g.rows = rows;
    g.N = out_dim, g.K = in_dim, g.c_f32 = y_dtype == MOE_F32;
    g.splits = op_f8_splits(rows, groups, out_dim, in_dim, op_cus());
    g.ws = (float *)workspace;
    g.sa = x_scale, g.sb = w_scale, g.kb = (int)kb, g.exact = exact;
    return op_done(fn, launch_op_gemm_f8(g, op_cus(), (hipStream_t)stream));
}

int moe_fp8_matmul_async(const void *x, int64_t ldx, int32_t x_dtype, const float *x_scale, const void *w, int64_t ldw,
                         int64_t w_stride, const float *w_scale, const int32_t *offsets, int32_t groups, int32_t rows,
                         int32_t in_dim, int32_t out_dim, void *y, int64_t ldy, int32_t y_dtype, void *workspace,
                         int64_t workspace_bytes, void *stream) {
    return fp8_matmul("moe_fp8_matmul_async", false, x, ldx, x_dtype, x_scale, w, ldw, w_stride, w_scale, offsets, groups,
                      rows, in_dim, out_dim, y, ldy, y_dtype, workspace, workspace_bytes, stream);
}

int moe_fp8_matmul_exact_async(const void *x, int64_t ldx, int32_t x_dtype, const float *x_scale, const void *w,
                               int64_t ldw, int64_t w_stride, const float *w_scale, const int32_t *offsets, int32_t groups,
                               int32_t rows, int32_t in_dim, int32_t out_dim, void *y, int64_t ldy, int32_t y_dtype,
                               void *workspace, int64_t workspace_bytes, void *stream) {
    return fp8_matmul("moe_fp8_matmul_exact_async", true, x, ldx, x_dtype, x_scale, w, ldw, w_stride, w_scale, offsets,
                      groups, rows, in_dim, out_dim, y, ldy, y_dtype, workspace, workspace_bytes, stream);
}

static int op_check_norm(const char *fn, int64_t T, int32_t D, int32_t x_dtype, int32_t y_dtype, int32_t h_dtype,
                         int32_t w_dtype, int32_t gate_dtype, const void *gate, int64_t gate_rows) {
    for (const int32_t t : {x_dtype, y_dtype, h_dtype, w_dtype, gate_dtype})
        if (t != MOE_F32 && t != MOE_BF16) return op_fail(fn, "dtypes must be MOE_F32 or MOE_BF16");
    if (T < 0) return op_fail(fn, "T must not be negative");
    if (D < 1 || D > kMaxNormDim) return op_fail(fn, "D must be 1 to " + std::to_string(kMaxNormDim));
    if (T > kOpMaxSize) return op_fail(fn, "too many rows (above 2^30)");
    if (gate && gate_rows < 1) return op_fail(fn, "gate_rows must be positive");
    return MOE_OK;
}

int moe_block_norm_async(const void *x, int32_t x_dtype, const void *y, int32_t y_dtype, const void *post_weight,
                         const void *pre_weight, int32_t w_dtype, const void *gate, int32_t gate_dtype,
                         int64_t gate_rows, float alpha, float beta, float eps, int64_t T, int32_t D, void *r, void *h,
                         int32_t h_dtype, float *stats, void *stream) {
    const char *fn = "moe_block_norm_async";
    int rc = op_check_norm(fn, T, D, x_dtype, y_dtype, h_dtype, w_dtype, gate_dtype, gate, gate_rows);
    if (rc != MOE_OK) return rc;
    if (!(eps >= 0.0f)) return op_fail(fn, "eps must not be negative");
    if (T == 0) return MOE_OK;
    if ((h != nullptr) != (pre_weight != nullptr)) return op_fail(fn, "h and pre_weight come together");
    if (!y && (post_weight || gate)) return op_fail(fn, "post_weight and gate need y");
    if (!x || (!r && !h)) return op_fail(fn, "null buffer");
    if (op_misaligned(x, x_dtype) || op_misaligned(r, x_dtype) || op_misaligned(y, y_dtype) ||
        op_misaligned(h, h_dtype) || op_misaligned(pre_weight, w_dtype) || op_misaligned(post_weight, w_dtype) ||
        op_misaligned(gate, gate_dtype) || op_misaligned(stats, MOE_F32))
        return op_fail(fn, "a buffer is not aligned to its elements");
    NormArgs a{};
    a.x = x, a.y = y, a.x_bf16 = x_dtype == MOE_BF16, a.y_bf16 = y_dtype == MOE_BF16, a.h_bf16 = h_dtype == MOE_BF16;
    a.pre = pre_weight, a.post = post_weight, a.w_bf16 = w_dtype == MOE_BF16;
    a.gate = gate, a.gate_bf16 = gate_dtype == MOE_BF16, a.gate_rows = gate_rows;
    a.alpha = alpha, a.beta = beta, a.eps = eps, a.T = T, a.D = D;
    a.r = r, a.h = h, a.stats = stats;
    return op_done(fn, launch_block_norm(a, (hipStream_t)stream));
}

int moe_block_norm_grad_workspace(int64_t T, int32_t D, int64_t gate_rows, int64_t *bytes) {
    const char *fn = "moe_block_norm_grad_workspace";
    if (!bytes) return op_fail(fn, "null bytes");
    if (T < 0 || T > kOpMaxSize || D < 1 || D > kMaxNormDim || gate_rows < 0) return op_fail(fn, "bad sizes");
    *bytes = T == 0 ? 0 : 4 * (int64_t)norm_workspace_floats(T, D, gate_rows);
    return MOE_OK;
}

int moe_block_norm_grad_async(const void *dr, const void *dh, const void *r, int32_t x_dtype, const void *y,
                              int32_t y_dtype, int32_t h_dtype, const float *stats, const void *post_weight,
                              const void *pre_weight, int32_t w_dtype, const void *gate, int32_t gate_dtype,
                              int64_t gate_rows, float alpha, float beta, int64_t T, int32_t D, void *dx, void *dy,
                              float *dgate, float *dpost, float *dpre, void *workspace, int64_t workspace_bytes,
                              void *stream) {
    const char *fn = "moe_block_norm_grad_async";
    int rc = op_check_norm(fn, T, D, x_dtype, y_dtype, h_dtype, w_dtype, gate_dtype, gate, gate_rows);
    if (rc != MOE_OK) return rc;
    if (T > 0) {
        if (!y && (post_weight || gate || dy)) return op_fail(fn, "post_weight, gate and dy need y");
        if (dgate && !gate) return op_fail(fn, "dgate needs gate");
        if (dpost && !post_weight) return op_fail(fn, "dpost needs post_weight");
        if (dh && !pre_weight) return op_fail(fn, "dh needs pre_weight");
        if (dpre && !dh) return op_fail(fn, "dpre needs dh");
        if (!dr && !dh) return op_fail(fn, "dr or dh is needed");
        if ((dh && !r) || ((dh || post_weight) && !stats)) return op_fail(fn, "null buffer");
    }
    if (op_misaligned(dr, x_dtype) || op_misaligned(r, x_dtype) || op_misaligned(dx, x_dtype) ||
        op_misaligned(y, y_dtype) || op_misaligned(dy, y_dtype) || op_misaligned(dh, h_dtype) ||
        op_misaligned(pre_weight, w_dtype) || op_misaligned(post_weight, w_dtype) || op_misaligned(gate, gate_dtype) ||
        op_misaligned(stats, MOE_F32) || op_misaligned(dgate, MOE_F32) || op_misaligned(dpost, MOE_F32) ||
        op_misaligned(dpre, MOE_F32))
        return op_fail(fn, "a buffer is not aligned to its elements");
    int64_t need = 0;
    rc = moe_block_norm_grad_workspace(T, D, gate ? gate_rows : 0, &need);
    if (rc != MOE_OK) return rc;
    if ((dgate || dpost || dpre) && need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)))
        return op_fail(fn, "the workspace must be 16-byte aligned and hold " + std::to_string(need) + " bytes");
    NormArgs a{};
    a.y = y, a.x_bf16 = x_dtype == MOE_BF16, a.y_bf16 = y_dtype == MOE_BF16, a.h_bf16 = h_dtype == MOE_BF16;
    a.pre = pre_weight, a.post = post_weight, a.w_bf16 = w_dtype == MOE_BF16;
    a.gate = gate, a.gate_bf16 = gate_dtype == MOE_BF16, a.gate_rows = gate_rows;
    a.alpha = alpha, a.beta = beta, a.T = T, a.D = D;
    a.r = (void *)r, a.stats = (float *)stats;
    a.dr = dr, a.dh = dh, a.dx = dx, a.dy = dy, a.dgate = dgate, a.dpost = dpost, a.dpre = dpre;
    a.ws = (float *)workspace;
    return op_done(fn, launch_block_norm_grad(a, (hipStream_t)stream));
}

}  // extern "C"
