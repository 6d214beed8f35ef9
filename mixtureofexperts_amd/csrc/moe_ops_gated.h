// moe_ops_gated.h -- what the gated blocks need beside the tiles of
// moe_ops_gemm.h: the streamed form of a few rows, the folds of calls whose k was
// split, and the gate alone.
#pragma once
#include "moe_ops_gemm.h"
#include "moe_ops_stream.h"

namespace moe {
namespace ops {

// h (and a, b) at columns n .. n + 3 of a row from the sums of a and b.
template <bool BF16>
__device__ __forceinline__ void gated_put4(const OpGemmArgs &g, long long row, int n, const float *a, const float *b) {
    float f[4];
    const Gate gate(g.act);
    gate_form<BF16>(gate, g.c_f32, [&](auto SMOOTH, auto FAST) {
#pragma unroll
        for (int c = 0; c < 4; ++c) f[c] = gate.value<decltype(SMOOTH)::value, decltype(FAST)::value>(a[c]).f * b[c];
    });
    put4(g, row * g.ldc + n, n, f[0], f[1], f[2], f[3], vec_ok(g));
    if (g.C2) {
        OpGemmArgs t = g;
        t.c_f32 = !BF16, t.c_stride = 0;
        t.C = g.C2, t.ldc = g.ldc2;
        put4(t, row * t.ldc + n, n, a[0], a[1], a[2], a[3], vec_ok(t));
        t.C = g.C3, t.ldc = g.ldc3;
        put4(t, row * t.ldc + n, n, b[0], b[1], b[2], b[3], vec_ok(t));
    }
}

// As stream_rows, of both weights at once: a workgroup owns 16 columns of each.
template <int OT, int MT>
__device__ __forceinline__ void stream_gated_rows(const OpGemmArgs &g, int e, int n0, int lo, int rows, int ks,
                                                  lds_u8 *red) {
    constexpr int ES = op_size(OT), KE = 128 / ES, CE = 16 / ES;
    constexpr int U = MT <= 2 ? 2 : 1;
    const int lane = threadIdx.x & 63, r16 = lane & 15, q4 = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int k0, klen;
    k_range(g, ks, KE, k0, klen);
    // rows past the last one repeat it (their results are not stored)
    const long long col = min(n0 + r16, g.N - 1);
    const uint8_t *b[2] = {(const uint8_t *)g.B + ((long long)e * g.b_stride + col * g.ldb + k0) * ES,
                           (const uint8_t *)g.B2 + ((long long)e * g.b2_stride + col * g.ldb2 + k0) * ES};
    const uint8_t *a[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
        a[m] = (const uint8_t *)g.A + ((long long)(lo + min(m * 16 + r16, rows - 1)) * g.lda + k0) * ES;
    f32x4 acc[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m][0] = acc[m][1] = f32x4{0, 0, 0, 0};
    const int pieces = (klen + KE - 1) / KE, whole = klen / KE;
    // UU pieces, all loads in flight before the first product
    auto piece = [&](auto UU_, int p) {
        constexpr int UU = decltype(UU_)::value;
        u32x4 fb[2][UU][2], fa[MT][UU][2];
#pragma unroll
        for (int u = 0; u < UU; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const long long o = (long long)(p + u * kStreamWaves) * 128 + h * 64 + q4 * 16;
                __builtin_memcpy(&fb[0][u][h], b[0] + o, 16);
                __builtin_memcpy(&fb[1][u][h], b[1] + o, 16);
#pragma unroll
                for (int m = 0; m < MT; ++m) __builtin_memcpy(&fa[m][u][h], a[m] + o, 16);
            }
#pragma unroll
        for (int u = 0; u < UU; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    acc[m][0] = fma16<OT>(fb[0][u][h], fa[m][u][h], acc[m][0]);
                    acc[m][1] = fma16<OT>(fb[1][u][h], fa[m][u][h], acc[m][1]);
                }
    };
    int p = w;
    for (; p + (U - 1) * kStreamWaves < whole; p += U * kStreamWaves) piece(num<U>{}, p);
    for (; p < whole; p += kStreamWaves) piece(num<1>{}, p);
    for (; p < pieces; p += kStreamWaves) {  // the last, part piece
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = p * KE + (h * 4 + q4) * CE;
            const u32x4 f0 = load_chunk<ES>(b[0] + (long long)k * ES, klen - k);
            const u32x4 f1 = load_chunk<ES>(b[1] + (long long)k * ES, klen - k);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const u32x4 x = load_chunk<ES>(a[m] + (long long)k * ES, klen - k);
                acc[m][0] = fma16<OT>(f0, x, acc[m][0]);
                acc[m][1] = fma16<OT>(f1, x, acc[m][1]);
            }
        }
    }
    // red: [wave][MT][2][64 lanes] 16 bytes
    typedef __attribute__((address_space(3))) f32x4 lds_acc;
    lds_acc *ra = (lds_acc *)red;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) ra[((w * MT + m) * 2 + h) * 64 + lane] = acc[m][h];
    __syncthreads();
    if (w < MT) {
        f32x4 v[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            v[h] = ra[(w * 2 + h) * 64 + lane];
            for (int x = 1; x < kStreamWaves; ++x) v[h] += ra[((x * MT + w) * 2 + h) * 64 + lane];
        }
        const int ml = w * 16 + r16, n = n0 + 4 * q4;
        if (ml < rows && g.splits > 1) {  // a range's sums, folded by op_gate_fold_kernel
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float *ws = g.ws + ((long long)(2 * ks + h) * g.rows + lo + ml) * g.N;
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (n + c < g.N) ws[n + c] = v[h][c];
            }
        } else if (ml < rows && n < g.N) {
            const float fa[4] = {v[0][0], v[0][1], v[0][2], v[0][3]}, fb[4] = {v[1][0], v[1][1], v[1][2], v[1][3]};
            gated_put4<OT == OT_BF16>(g, lo + ml, n, fa, fb);
        }
    }
    __syncthreads();
}

// MOST rows at a time.  Bound by reading both weights: 32 rows on 8 bf16 experts of 4096 /
// 14336 (1.88 GB) 281 to 370 us by where the two weights lie (12 placements; at most of them
// 326 to 343, 5.6 TB/s; each workgroup starting at another k: 358 to 377).  64 rows take the
// registers of three workgroups per CU.  32 rows leave room for five, which fp32 rows of up to
// 4 KB gain by, having few loads each: 64 / 32, us, 8 experts of 512 / 2048, 2 rows each 16.0 /
// 13.2, 16 17.3 / 14.8, 64 rows on one and 9 on the others 17.7 / 19.9; 64 of 512 / 1408 82 / 72; 8 of
// 1024 / 4096, 8 rows 60.0 / 59.1.  Longer rows lose: 8 of 2048 / 4096, 16 rows 113 / 115, uneven
// ones 122 / 131; bf16 with four workgroups per CU, 8 of 2048 / 14336, 1 row 186 / 201, 128 of
// 2048 / 768 161 / 175.
template <int OT, int MOST>
__global__ __launch_bounds__(kStreamWaves * 64) __attribute__((amdgpu_waves_per_eu(MOST == 32 ? 5 : 1))) void
op_gated_stream_kernel(OpGemmArgs g) {
    __shared__ __attribute__((aligned(16))) uint8_t red_[kStreamWaves * (MOST / 16) * 2 * 64 * 16];
    lds_u8 *red = (lds_u8 *)red_;
    const int r = blockIdx.x / g.nt, n0 = (blockIdx.x - r * g.nt) * 16;
    int e, lo, hi;
    held_group(g, r, e, lo, hi);
    if (e < 0) return;
    while (lo < hi) {
        const int rows = min(hi - lo, MOST);
        if (rows <= 16) stream_gated_rows<OT, 1>(g, e, n0, lo, rows, blockIdx.y, red);
        else if (rows <= 32) stream_gated_rows<OT, 2>(g, e, n0, lo, rows, blockIdx.y, red);
        else stream_gated_rows<OT, MOST / 16>(g, e, n0, lo, rows, blockIdx.y, red);
        lo += rows;
    }
}

// Results of a call whose k was split, from the ranges' sums in range order: four
// columns of a row per thread.  ws [range][a, b][rows][N] (OM_GATE_GRAD:
// [range][rows][N]), rows of the groups only.
template <int OT, int MODE>
__global__ __launch_bounds__(256) void op_gate_fold_kernel(OpGemmArgs g) {
    constexpr bool BF16 = OT == OT_BF16;
    constexpr int CE = MODE == OM_GATED ? 4 : GateChunk<BF16>::CE;
    const int per = (g.N + CE - 1) / CE;
    const long long i = op_row_block() * 256 + threadIdx.x;
    const long long row = i / per;
    const int n = (int)(i - row * per) * CE;
    if (row >= g.rows) return;
    if (g.offsets) {
        int lo, hi, unused;
        op_group(g.offsets, 0, g.rows, lo, unused);
        op_group(g.offsets, g.E - 1, g.rows, unused, hi);
        if (row < lo || row >= hi) return;
    }
    const long long all = (long long)g.rows * g.N;
    const float *ws = g.ws + row * g.N + n;
    if constexpr (MODE == OM_GATED) {
        float a[4] = {0, 0, 0, 0}, b[4] = {0, 0, 0, 0};
        for (int s = 0; s < g.splits; ++s) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                if (n + c >= g.N) continue;
                a[c] += ws[2 * s * all + c];
                b[c] += ws[(2 * s + 1) * all + c];
            }
        }
        gated_put4<BF16>(g, row, n, a, b);
    } else {
        GateChunk<BF16> dh;
#pragma unroll
        for (int c = 0; c < CE; ++c) dh.v[c] = 0.0f;
        for (int s = 0; s < g.splits; ++s) {
#pragma unroll
            for (int c = 0; c < CE; ++c)
                if (n + c < g.N) dh.v[c] += ws[s * all + c];
        }
        GateRaw a, b;
        gate_load_ab<BF16>(g, row, n, a, b);
        gate_store<BF16>(g, row, n, dh, a, b);
    }
}

// The gate's gradients where dh is given (g.A): bound by its three reads and three
// writes.  256 threads of 16 bytes each, 2^lx of them along a row.  8192 x 14336 bf16 (1.41 GB):
// 243 us, 5.8 TB/s.
template <int OT>
__global__ __launch_bounds__(256) void op_gate_rows_kernel(OpGemmArgs g, int lx) {
    constexpr bool BF16 = OT == OT_BF16;
    constexpr int CE = GateChunk<BF16>::CE, ES = op_size(OT);
    int lo = 0, hi = g.rows, unused;
    if (g.offsets) {
        op_group(g.offsets, 0, g.rows, lo, unused);
        op_group(g.offsets, g.E - 1, g.rows, unused, hi);
    }
    const long long n = (((long long)blockIdx.x << lx) + (threadIdx.x & ((1 << lx) - 1))) * CE;
    if (n >= g.N) return;
    const long long step = (long long)gridDim.y << (8 - lx);
    for (long long r = lo + ((long long)blockIdx.y << (8 - lx)) + (threadIdx.x >> lx); r < hi; r += step) {
        GateRaw a, b;
        const GateRaw dh = gate_load<BF16>((const uint8_t *)g.A + r * g.lda * ES, (int)n, g.N);
        gate_load_ab<BF16>(g, r, (int)n, a, b);
        gate_store<BF16>(g, r, (int)n, GateChunk<BF16>(dh), a, b);
    }
}

}  // namespace ops

hipError_t launch_op_gate_fold(int mode, int ot, const OpGemmArgs &g, hipStream_t s) {
    const int ce = mode == OM_GATED || ot == OT_F32 ? 4 : 8;
    const long long blocks = ((long long)g.rows * ((g.N + ce - 1) / ce) + 255) / 256;
    if (blocks > 0x7fffffffll / 256) return kOpTooLarge;
    const dim3 gr = op_row_grid(blocks);
    if (mode == OM_GATED && ot == OT_F32) ops::op_gate_fold_kernel<OT_F32, OM_GATED><<<gr, 256, 0, s>>>(g);
    else if (mode == OM_GATED) ops::op_gate_fold_kernel<OT_BF16, OM_GATED><<<gr, 256, 0, s>>>(g);
    else if (ot == OT_F32) ops::op_gate_fold_kernel<OT_F32, OM_GATE_GRAD><<<gr, 256, 0, s>>>(g);
    else ops::op_gate_fold_kernel<OT_BF16, OM_GATE_GRAD><<<gr, 256, 0, s>>>(g);
    return hipGetLastError();
}

hipError_t launch_op_gate_rows(int ot, const OpGemmArgs &g, hipStream_t s) {
    const long long chunks = ((long long)g.N + (ot == OT_F32 ? 3 : 7)) / (ot == OT_F32 ? 4 : 8);
    int lx = 0;
    while (lx < 8 && (1 << lx) < chunks) ++lx;
    const long long gx = (chunks + (1 << lx) - 1) >> lx;
    long long gy = ((long long)g.rows + (256 >> lx) - 1) >> (8 - lx);
    if (gy > 16384) gy = 16384;
    const dim3 gr((unsigned)gx, (unsigned)gy);
    if (ot == OT_F32) ops::op_gate_rows_kernel<OT_F32><<<gr, 256, 0, s>>>(g, lx);
    else ops::op_gate_rows_kernel<OT_BF16><<<gr, 256, 0, s>>>(g, lx);
    return hipGetLastError();
}

static hipError_t launch_gated_stream(int ot, OpGemmArgs g, hipStream_t s) {
    g.nt = (g.N + 15) / 16;
    const long long grid = (long long)(g.E < g.rows ? g.E : g.rows) * g.nt;  // the groups that can hold rows
    if (grid * g.splits > 0x7fffffffll / (ops::kStreamWaves * 64)) return kOpTooLarge;
    const dim3 gr((unsigned)grid, g.splits), b(ops::kStreamWaves * 64);
    if (ot != OT_F32) ops::op_gated_stream_kernel<OT_BF16, 64><<<gr, b, 0, s>>>(g);
    else if (g.K <= 1024) ops::op_gated_stream_kernel<OT_F32, 32><<<gr, b, 0, s>>>(g);
    else ops::op_gated_stream_kernel<OT_F32, 64><<<gr, b, 0, s>>>(g);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess && g.splits > 1 ? launch_op_gate_fold(OM_GATED, ot, g, s) : e;
}

template <int OT, int MODE>
static hipError_t gated_plan(bool b_col, const OpGemmArgs &g, int ncu, hipStream_t s) {
    if (b_col) return ops::op_gemm_plan<OT, false, true, false, MODE>(g, ncu, s);
    return ops::op_gemm_plan<OT, false, false, false, MODE>(g, ncu, s);
}

hipError_t launch_op_gated(int mode, int ot, bool b_col, OpGemmArgs g, int ncu, hipStream_t s) {
    if (mode == OM_GATED && op_gated_streamed(ot, b_col, g.rows, g.E, g.N, g.K, ncu)) return launch_gated_stream(ot, g, s);
    if (ot == OT_F32) {
        if (mode == OM_GATED) return gated_plan<OT_F32, OM_GATED>(b_col, g, ncu, s);
        if (mode == OM_GATE_GRAD) return gated_plan<OT_F32, OM_GATE_GRAD>(b_col, g, ncu, s);
        return gated_plan<OT_F32, OM_TWO>(b_col, g, ncu, s);
    }
    if (mode == OM_GATED) return gated_plan<OT_BF16, OM_GATED>(b_col, g, ncu, s);
    if (mode == OM_GATE_GRAD) return gated_plan<OT_BF16, OM_GATE_GRAD>(b_col, g, ncu, s);
    return gated_plan<OT_BF16, OM_TWO>(b_col, g, ncu, s);
}

}  // namespace moe
