// moe_ops_stream.h -- products of a few rows per group (a decode step): the
// weights are the traffic, so they go from global memory straight into MFMA
// fragments, each read once per 16 MT rows of a group.
//
// A workgroup owns 16 columns of one group; its four waves take interleaved
// 128-byte pieces of k, U of them in flight, and their partial 16 x 16 blocks
// are added in wave order through LDS.  Bound by HBM reads: 32 rows on 8 bf16
// experts of 4096 / 14336 154 to 166 us (5.6 to 6 TB/s), two int8 rows on two of them
// 26 us (4.4 TB/s).  64 fp32 rows on 8 experts of 512 / 2048 10 us (3.4 TB/s, one round of
// workgroups).  Up to 8 or 16 rows per group on average (op_streamed): a group of more
// than 64 is walked 64 rows at a time, its weights read again each time.
#pragma once
#include "moe_ops_gemm.h"

namespace moe {
namespace ops {

constexpr int kStreamWaves = 4;

template <int OT, int MT>
__device__ __forceinline__ void stream_rows(const OpGemmArgs &g, int e, int n0, int lo, int rows, int ks, lds_u8 *red) {
    constexpr int ES = op_size(OT), KE = 128 / ES, CE = 16 / ES;
    constexpr int U = MT == 1 ? 4 : 2;
    const int lane = threadIdx.x & 63, r16 = lane & 15, q4 = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int k0, klen;
    k_range(g, ks, KE, k0, klen);
    // rows past the last one repeat it (their results are not stored)
    const uint8_t *b =
        (const uint8_t *)g.B + ((long long)e * g.b_stride + (long long)min(n0 + r16, g.N - 1) * g.ldb + k0) * ES;
    const uint8_t *a[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
        a[m] = (const uint8_t *)g.A + ((long long)(lo + min(m * 16 + r16, rows - 1)) * g.lda + k0) * ES;
    acc_t<OT> acc[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m] = acc_t<OT>{0, 0, 0, 0};
    const int pieces = (klen + KE - 1) / KE;
    const int whole = klen / KE;
    int p = w;
    for (; p + (U - 1) * kStreamWaves < whole; p += U * kStreamWaves) {
        u32x4 fb[U][2], fa[MT][U][2];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const long long o = (long long)(p + u * kStreamWaves) * 128 + h * 64 + q4 * 16;
                __builtin_memcpy(&fb[u][h], b + o, 16);
#pragma unroll
                for (int m = 0; m < MT; ++m) __builtin_memcpy(&fa[m][u][h], a[m] + o, 16);
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int m = 0; m < MT; ++m) acc[m] = fma16<OT>(fb[u][h], fa[m][u][h], acc[m]);
    }
    for (; p < whole; p += kStreamWaves) {
        u32x4 fb[2], fa[MT][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const long long o = (long long)p * 128 + h * 64 + q4 * 16;
            __builtin_memcpy(&fb[h], b + o, 16);
#pragma unroll
            for (int m = 0; m < MT; ++m) __builtin_memcpy(&fa[m][h], a[m] + o, 16);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[m] = fma16<OT>(fb[h], fa[m][h], acc[m]);
    }
    for (; p < pieces; p += kStreamWaves) {  // the last, part piece
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = p * KE + (h * 4 + q4) * CE;
            const u32x4 fb = load_chunk<ES>(b + (long long)k * ES, klen - k);
#pragma unroll
            for (int m = 0; m < MT; ++m)
                acc[m] = fma16<OT>(fb, load_chunk<ES>(a[m] + (long long)k * ES, klen - k), acc[m]);
        }
    }
    // red: [wave][MT][64 lanes] 16 bytes
    typedef __attribute__((address_space(3))) acc_t<OT> lds_acc;
    lds_acc *ra = (lds_acc *)red;
#pragma unroll
    for (int m = 0; m < MT; ++m) ra[(w * MT + m) * 64 + lane] = acc[m];
    __syncthreads();
    if (w < MT) {
        acc_t<OT> v = ra[w * 64 + lane];
        for (int x = 1; x < kStreamWaves; ++x) v += ra[(x * MT + w) * 64 + lane];
        const int ml = w * 16 + r16, n = n0 + 4 * q4;
        if (ml < rows && g.splits > 1) {  // a range's sums, folded by op_fold_kernel
            acc_elem<OT> *ws = (acc_elem<OT> *)g.ws + ((long long)ks * g.rows + lo + ml) * g.N;
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (n + c < g.N) ws[n + c] = v[c];
        } else if (ml < rows) {
            float o[4];
            RowScale sa;
            if constexpr (OT == OT_I8) sa = RowScale(g.sa[lo + ml]);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                if constexpr (OT == OT_I8) o[c] = sa(v[c], n + c < g.N ? g.sb[(long long)e * g.N + n + c] : 0.0f);
                else o[c] = v[c];
            }
            put4(g, (long long)(lo + ml) * g.ldc + n, n, o[0], o[1], o[2], o[3], vec_ok(g));
        }
    }
    __syncthreads();
}

template <int OT>
__global__ __launch_bounds__(kStreamWaves * 64) void op_stream_kernel(OpGemmArgs g) {
    __shared__ __attribute__((aligned(16))) uint8_t red_[kStreamWaves * 4 * 64 * 16];
    lds_u8 *red = (lds_u8 *)red_;
    // workgroup (r, n): the r-th group that holds rows, 16 columns
    int r = blockIdx.x / g.nt;
    const int n0 = (blockIdx.x - r * g.nt) * 16, lane = threadIdx.x & 63;
    int e = -1, lo = 0, hi = 0;
    for (int base = 0; base < g.E && e < 0; base += 64) {
        int a = 0, b = 0;
        if (base + lane < g.E) op_group(g.offsets, base + lane, g.rows, a, b);
        unsigned long long held = __ballot(a < b);
        const int n = __popcll(held);
        if (r < n) {
            for (int i = 0; i < r; ++i) held &= held - 1;
            const int src = __ffsll((long long)held) - 1;
            e = base + src;
            lo = __shfl(a, src);
            hi = __shfl(b, src);
        }
        r -= n;
    }
    e = __builtin_amdgcn_readfirstlane(e);
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    if (e < 0) return;
    while (lo < hi) {
        const int rows = min(hi - lo, 64);
        if (rows <= 16) stream_rows<OT, 1>(g, e, n0, lo, rows, blockIdx.y, red);
        else if (rows <= 32) stream_rows<OT, 2>(g, e, n0, lo, rows, blockIdx.y, red);
        else stream_rows<OT, 4>(g, e, n0, lo, rows, blockIdx.y, red);
        lo += rows;
    }
}

// Results of a call whose k was split: the ranges' sums in range order.  One
// element per thread.  Ragged rows: ws [range][rows][N], rows of the groups
// only; ragged k: ws [group][range][M][N].
template <int OT, bool RAGK>
__global__ __launch_bounds__(256) void op_fold_kernel(OpGemmArgs g) {
    const acc_elem<OT> *ws = (const acc_elem<OT> *)g.ws;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long per = RAGK ? (long long)g.M * g.N : (long long)g.rows * g.N;
    long long e = 0, at = i, row = 0, n;
    if constexpr (RAGK) {
        e = i / per;
        if (e >= g.E) return;
        at = i - e * per;
        ws += e * g.splits * per;
        row = at / g.N;
        n = at - row * g.N;
    } else {
        if (i >= per) return;
        row = i / g.N;
        n = i - row * g.N;
        if (g.offsets) {
            int lo, hi, unused;
            op_group(g.offsets, 0, g.rows, lo, unused);
            op_group(g.offsets, g.E - 1, g.rows, unused, hi);
            if (row < lo || row >= hi) return;
        }
    }
    acc_elem<OT> sum = 0;
    for (int s = 0; s < g.splits; ++s) sum += ws[s * per + at];
    float v;
    if constexpr (OT == OT_I8) {
        int a = 0;
        if (g.offsets) {  // the last group that starts at or before the row
            int b = g.E - 1;
            while (a < b) {
                const int mid = (a + b + 1) >> 1;
                if (g.offsets[mid] <= row) a = mid; else b = mid - 1;
            }
        }
        v = RowScale(g.sa[row])(sum, g.sb[(long long)a * g.N + n]);
    } else {
        v = sum;
    }
    const long long c = e * g.c_stride + row * g.ldc + n;
    if (g.c_f32) {
        float *d = (float *)g.C + c;
        *d = RAGK && g.accumulate ? *d + v : v;
    } else {
        uint16_t *d = (uint16_t *)g.C + c;
        *d = f32_to_bf16(RAGK && g.accumulate ? bf16_to_f32(*d) + v : v);
    }
}

// One row's codes: the largest magnitude, then rne(127 x / max).  A code's
// border is an odd multiple of max / 254: 127 x is formed before the division,
// so that a border divides exactly.  x and max are scaled by 2^-64 where 127 x
// could overflow.  A row of zeros has scale 0 and codes 0; a row that holds an
// infinity or a NaN has scale NaN (and codes 0), so that its products are NaN.
struct RowMax {
    float m = 0.0f;
    bool bad = false;
    __device__ __forceinline__ void take(float x) {
        const float v = fabsf(x);
        bad |= !(v <= 3.402823466e38f);
        m = fmaxf(m, v);
    }
    // over the 256 threads of a workgroup; NaN has to survive the maximum
    __device__ __forceinline__ float all(float *part) {
        auto larger = [](float a, float b) { return (a != a || b != b) ? __builtin_nanf("") : fmaxf(a, b); };
        float v = bad ? __builtin_nanf("") : m;
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) v = larger(v, __shfl_xor(v, d));
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
        __syncthreads();
        return larger(larger(part[0], part[1]), larger(part[2], part[3]));
    }
};
struct RowCode {
    float down, ms, inv;
    bool live;
    __device__ __forceinline__ explicit RowCode(float m)
        : down(m > 1.0e36f ? 5.421010862427522e-20f : 1.0f), ms(m * down), inv(127.0f / ms),
          live(m > 0.0f) {}  // (false for 0 and NaN)
    // The product with 127 / max is off by less than 127 * 2^-22: the division
    // itself runs only where that could cross a border, or max is so small that
    // 127 / max overflows.
    __device__ __forceinline__ int operator()(float x) const {
        const float y = x * down;
        float r = y * inv;
        const float t = fabsf(r) - floorf(fabsf(r));
        if (!(fabsf(t - 0.5f) > 1.0e-4f) || !(inv < 1.0e38f)) r = y * 127.0f / ms;
        return live ? (int)rintf(r) : 0;
    }
};

// Bound by HBM: 8192 x 4096 bf16 rows 24 us (100 MB, 4.2 TB/s).
// Rows of up to 2048 NV columns, in registers: 256 threads with NV groups of 8
// columns each (VEC: 16-byte loads of x, 8-byte stores of the codes).
template <int XB, int NV, bool VEC>
__global__ __launch_bounds__(256) void quantize_i8_kernel(const void *x_, long long ldx, long long rows, int cols,
                                                          int8_t *q_, long long ldq, int pad_to, float *scale) {
    __shared__ float part[4];
    const long long r = op_row_block();
    if (r >= rows) return;
    int8_t *q = q_ + r * ldq;
    float v[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = VEC ? ((int)threadIdx.x + i * 256) * 8 : (int)threadIdx.x + i * 2048;
        if constexpr (VEC && XB) {
            uint4 u = make_uint4(0u, 0u, 0u, 0u);
            if (c < cols) u = *(const uint4 *)((const uint16_t *)x_ + r * ldx + c);
            const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[i][2 * k] = __uint_as_float(w[k] << 16);
                v[i][2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
            }
        } else if constexpr (VEC) {
            float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f), b = a;
            if (c < cols) {
                a = *(const float4 *)((const float *)x_ + r * ldx + c);
                b = *(const float4 *)((const float *)x_ + r * ldx + c + 4);
            }
            v[i][0] = a.x, v[i][1] = a.y, v[i][2] = a.z, v[i][3] = a.w;
            v[i][4] = b.x, v[i][5] = b.y, v[i][6] = b.z, v[i][7] = b.w;
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int ck = c + k * 256;
                v[i][k] = 0.0f;
                if (ck < cols)
                    v[i][k] = XB ? bf16_to_f32(((const uint16_t *)x_)[r * ldx + ck]) : ((const float *)x_)[r * ldx + ck];
            }
        }
    }
    RowMax mx;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) mx.take(v[i][k]);
    const float m = mx.all(part);
    if (threadIdx.x == 0) scale[r] = m / 127.0f;
    const RowCode code(m);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = VEC ? ((int)threadIdx.x + i * 256) * 8 : (int)threadIdx.x + i * 2048;
        if constexpr (VEC) {
            if (c >= pad_to) continue;
            unsigned w[2] = {0u, 0u};
#pragma unroll
            for (int k = 0; k < 8; ++k) w[k >> 2] |= (unsigned)(code(v[i][k]) & 255) << (8 * (k & 3));
            *(uint2 *)(q + c) = make_uint2(w[0], w[1]);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (c + k * 256 < pad_to) q[c + k * 256] = (int8_t)code(v[i][k]);
        }
    }
}
// Longer rows, read twice.
template <int XB>
__global__ __launch_bounds__(256) void quantize_i8_long_kernel(const void *x_, long long ldx, long long rows, int cols,
                                                               int8_t *q_, long long ldq, int pad_to, float *scale) {
    __shared__ float part[4];
    const long long r = op_row_block();
    if (r >= rows) return;
    int8_t *q = q_ + r * ldq;
    auto at = [&](int c) -> float {
        if constexpr (XB) return bf16_to_f32(((const uint16_t *)x_)[r * ldx + c]);
        else return ((const float *)x_)[r * ldx + c];
    };
    RowMax mx;
    for (int c = threadIdx.x; c < cols; c += 256) mx.take(at(c));
    const float m = mx.all(part);
    if (threadIdx.x == 0) scale[r] = m / 127.0f;
    const RowCode code(m);
    for (int c = threadIdx.x; c < pad_to; c += 256) q[c] = (int8_t)(c < cols ? code(at(c)) : 0);
}

}  // namespace ops
}  // namespace moe
