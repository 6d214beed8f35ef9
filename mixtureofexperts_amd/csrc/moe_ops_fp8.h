// moe_ops_fp8.h -- 8-bit floating point (e4m3) with a scale for each block of 128:
// codes of rows (1 x 128) and of weights (128 x 128), and the products
//
//   y[r][n] = sum over blocks kb of xs[r][kb] ws[n / 128][kb] (sum over k in kb of q[r][k] w[n][k])
//
// A stage of k is one block: the matrix unit gives a block's sum of 128 products, the
// vector unit multiplies it with its two scales and adds it to the fp32 sum.
//
// The matrix unit's 8-bit instructions (16x16x128_f8f6f4 and 16x16x32_fp8_fp8 alike) cut
// each product to a multiple of 2^-13 of the largest of its eight neighbours along k.  Any sum
// is off by less than 7 * 2^-13 of its magnitudes, however little is left of them; measured,
// sums of N(0, 1) codes by 1.4e-5 of themselves, of codes of all magnitudes by 5e-5, a
// hundredth of a bf16 result's rounding.  The instruction is twice as fast (4040 TFLOP/s in a
// loop, 16x16x32_bf16 1960), so tiles with bf16 results take it unless the caller asks for
// exact products (codes of 8192 rows, 8 even groups of 4096 / 14336: 490 and 870 us).
// Those, fp32 results, split sums, and few rows, where the weights' bytes bind, have the codes
// widened to bf16, which is exact, and products that are exact and summed in fp32 (1e-8 and
// 8e-8).
#pragma once
#include "moe_ops_gemm.h"
#include "moe_ops_stream.h"

namespace moe {
namespace ops {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// ---- codes --------------------------------------------------------------------------
// 448 x / m rounded to e4m3, to the bit: m a block's largest magnitude.  The product with
// 448 rcp(m) in fp32 is off by at most 2^-21.6 of itself (the reciprocal 2^-23, three
// products 2^-24).
//   bf16: 448 |x| (11 bits) and a border between two codes times m (13 bits) are equal or at
//     least 2^-13 apart, and a third of all waves hold an equal one: the product, rounded to 15
//     bits of fraction, is the border where the quotient is, and on its side elsewhere.
//   fp32: where 2^-21 less and 2^-21 more round to the same code, so does the quotient.
//     Else 448 |x| and border * m are compared in fp64, where both are exact (27 and 29 bits),
//     x and m moved by 2^64 where m is small or large.
struct F8Code {
    float a;          // m
    float mid, low, high;  // 448 / m, less and more
    bool live;        // (false for 0, infinity and NaN: codes 0)
    bool plain;       // they are normal numbers
    __device__ __forceinline__ explicit F8Code(unsigned bits) {
        a = __uint_as_float(bits);
        live = bits != 0u && bits < 0x7f800000u;
        plain = a >= 0x1p-100f && a <= 0x1p100f;
        mid = 448.0f * __builtin_amdgcn_rcpf(a);
        low = mid * (1.0f - 0x1p-21f), high = mid * (1.0f + 0x1p-21f);
    }
    static __device__ __forceinline__ float snapped(float y) {
        return __uint_as_float((__float_as_uint(y) + 0x80u) & 0xffffff00u);
    }
    __device__ __forceinline__ float decided(float x) const {
        const float adj = a > 0x1p64f ? 0x1p-64f : (a < 0x1p-64f ? 0x1p64f : 1.0f), m = a * adj;
        const float y = x * adj * (448.0f / m);  // off by 2^-22 at most
        // 20 bits below e4m3's three; of |y| below 2^-6, whose codes are 2^-9 apart, those
        // of |y| + 2^-6
        const float off = fabsf(y) < 0x1p-6f ? 0x1p-6f : 0.0f, z = fabsf(y) + off;
        const unsigned t = __float_as_uint(z) & 0xfffffu;
        if (t - 0x7fff8u > 16u) return y;  // no border within y's roundings
        const unsigned mid = (__float_as_uint(z) & 0xfff00000u) | 0x80000u;
        const double border = ((double)__uint_as_float(mid) - (double)off) * (double)m;
        const double v = 448.0 * (double)fabsf(x * adj);
        const unsigned r = v > border ? mid + 64u : (v < border ? mid - 64u : mid);
        return copysignf(__uint_as_float(r) - off, x);
    }
};
__device__ __forceinline__ unsigned f8_pack(float a, float b, float c, float d) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// Eight columns from c on of a row (those past cols are 0), as they are in memory.
template <int XB>
struct F8Raw {
    unsigned w[XB ? 4 : 8];
    __device__ __forceinline__ F8Raw() {
#pragma unroll
        for (unsigned &x : w) x = 0u;
    }
    __device__ __forceinline__ float at(int k) const {
        if constexpr (XB) return __uint_as_float(k & 1 ? w[k / 2] & 0xffff0000u : w[k / 2] << 16);
        else return __uint_as_float(w[k]);
    }
    // bits of the largest magnitude (infinities and NaNs above all numbers)
    __device__ __forceinline__ unsigned largest() const {
        if constexpr (XB) {
            typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
            u16x2 m = __builtin_bit_cast(u16x2, w[0] & 0x7fff7fffu);
#pragma unroll
            for (int k = 1; k < 4; ++k) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[k] & 0x7fff7fffu));
            return (unsigned)max(m[0], m[1]) << 16;
        } else {
            unsigned m = 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) m = max(m, w[k] & 0x7fffffffu);
            return m;
        }
    }
};
template <int XB, bool VEC>
__device__ __forceinline__ F8Raw<XB> f8_load(const void *row, int c, int cols) {
    F8Raw<XB> r;
    if constexpr (VEC) {
        if (c >= cols) return r;
        const uint4 *p = (const uint4 *)((const uint8_t *)row + (long long)c * (XB ? 2 : 4));
#pragma unroll
        for (int h = 0; h < (XB ? 1 : 2); ++h) {
            const uint4 u = p[h];
            r.w[4 * h] = u.x, r.w[4 * h + 1] = u.y, r.w[4 * h + 2] = u.z, r.w[4 * h + 3] = u.w;
        }
    } else if (c + 8 <= cols) {  // at any alignment
        __builtin_memcpy(r.w, (const uint8_t *)row + (long long)c * (XB ? 2 : 4), sizeof(r.w));
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (c + k >= cols) continue;
            if constexpr (XB) r.w[k / 2] |= (unsigned)((const uint16_t *)row)[c + k] << (16 * (k & 1));
            else r.w[k] = ((const unsigned *)row)[c + k];
        }
    }
    return r;
}
template <int XB>
__device__ __forceinline__ void f8_codes8(const F8Code &code, const F8Raw<XB> &raw, unsigned (&w)[2]) {
    unsigned lo[2], hi[2];
    bool sure = code.plain;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float v[4];
        if constexpr (XB) {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = F8Code::snapped(raw.at(4 * h + k) * code.mid);
            lo[h] = f8_pack(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = raw.at(4 * h + k);
            lo[h] = f8_pack(v[0] * code.low, v[1] * code.low, v[2] * code.low, v[3] * code.low);
            hi[h] = f8_pack(v[0] * code.high, v[1] * code.high, v[2] * code.high, v[3] * code.high);
            sure &= lo[h] == hi[h];
        }
    }
    if (!sure && code.live) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = code.decided(raw.at(4 * h + k));
            lo[h] = f8_pack(v[0], v[1], v[2], v[3]);
        }
    }
    w[0] = code.live ? lo[0] : 0u;
    w[1] = code.live ? lo[1] : 0u;
}
template <bool VEC>
__device__ __forceinline__ void f8_store(uint8_t *row, int c, int pad_to, const unsigned (&w)[2]) {
    if constexpr (VEC) {
        if (c < pad_to) *(uint2 *)(row + c) = make_uint2(w[0], w[1]);
    } else if (c + 8 <= pad_to) {
        __builtin_memcpy(row + c, w, 8);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (c + k < pad_to) row[c + k] = (uint8_t)(w[k >> 2] >> (8 * (k & 3)));
    }
}
// over the 16 lanes of a block's row (a DPP row, rotated)
__device__ __forceinline__ unsigned f8_over_row(unsigned m) {
    m = max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x128, 0xf, 0xf, false));
    m = max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x124, 0xf, 0xf, false));
    m = max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x122, 0xf, 0xf, false));
    return max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x121, 0xf, 0xf, false));
}
// m / 448, correctly rounded: a product with 1 / 448 and one step on its remainder, which
// an fma gives exactly (but where the quotient is subnormal, or 448 q overflows).
__device__ __forceinline__ float f8_scale(unsigned bits) {
    const float m = __uint_as_float(bits), q = m * (1.0f / 448.0f);
    float s = fmaf(fmaf(-448.0f, q, m), 1.0f / 448.0f, q);
    if (!(m > 0x1p-90f && m < 0x1p120f)) s = bits < 0x7f800000u ? m / 448.0f : __builtin_nanf("");
    return s;
}

// Blocks of a row: 16 lanes each, 2^lx of a workgroup's 16 along the row; R rows of a lane
// on their way at once.  8192 x 4096 bf16: 21 us (4.9 TB/s; as many workgroups as CUs, each
// loading its next rows under the codes of the last: 32).
template <int XB, bool VEC>
__global__ __launch_bounds__(256) void quantize_f8_rows_kernel(QuantF8Args a, int lx) {
    constexpr int R = 4, XS = XB ? 2 : 4;
    const int group = threadIdx.x >> 4, l = threadIdx.x & 15;
    const int kbs = (a.cols + 127) >> 7;
    const long long kb = ((long long)blockIdx.x << lx) + (group & ((1 << lx) - 1));
    if (kb >= kbs) return;
    const int c = (int)kb * 128 + l * 8;
    const long long step = (long long)gridDim.y << (4 - lx);
    for (long long e = blockIdx.z; e < a.mats; e += gridDim.z) {
        const uint8_t *x = (const uint8_t *)a.x + e * a.x_stride * XS;
        for (long long r0 = ((long long)blockIdx.y << (4 - lx)) + (group >> lx); r0 < a.rows; r0 += R * step) {
            F8Raw<XB> v[R];
#pragma unroll
            for (int i = 0; i < R; ++i) v[i] = f8_load<XB, VEC>(x + min(r0 + i * step, a.rows - 1) * a.ldx * XS, c, a.cols);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const long long r = r0 + i * step;
                if (r >= a.rows) continue;  // (the same for a block's 16 lanes)
                const unsigned m = f8_over_row(v[i].largest());
                if (l == 0) a.scale[(e * a.rows + r) * kbs + kb] = f8_scale(m);
                unsigned w[2];
                f8_codes8(F8Code(m), v[i], w);
                f8_store<VEC>(a.q + e * a.q_stride + r * a.ldq, c, a.pad_to, w);
            }
        }
    }
}

// Blocks of 128 x 128, one per workgroup: held in registers between the maximum and the
// codes, read once.  64 matrices of 1408 x 2048 bf16: 105 us (5.2 TB/s, a copy's rate; 141 with
// a division per value).
template <int XB, bool VEC>
__global__ __launch_bounds__(256) void quantize_f8_tiles_kernel(QuantF8Args a) {
    __shared__ unsigned part[4];
    const int kbs = (a.cols + 127) >> 7;
    const long long rbs = (a.rows + 127) >> 7;
    const long long tile = op_row_block();
    if (tile >= a.mats * rbs * kbs) return;
    const long long e = tile / (rbs * kbs), t = tile - e * (rbs * kbs);
    const long long rb = t / kbs;
    const int kb = (int)(t - rb * kbs);
    constexpr int XS = XB ? 2 : 4;
    const int c = kb * 128 + ((int)threadIdx.x & 15) * 8;
    const long long r0 = rb * 128 + (threadIdx.x >> 4);
    const uint8_t *x = (const uint8_t *)a.x + e * a.x_stride * XS;
    F8Raw<XB> v[8];
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long long r = r0 + i * 16;
        if (r < a.rows) v[i] = f8_load<XB, VEC>(x + r * a.ldx * XS, c, a.cols);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, v[i].largest());
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, d));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
    __syncthreads();
    m = max(max(part[0], part[1]), max(part[2], part[3]));
    if (threadIdx.x == 0) a.scale[tile] = f8_scale(m);
    const F8Code code(m);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long long r = r0 + i * 16;
        if (r >= a.rows) continue;
        unsigned w[2];
        f8_codes8(code, v[i], w);
        f8_store<VEC>(a.q + e * a.q_stride + r * a.ldq, c, a.pad_to, w);
    }
}

// ---- products -----------------------------------------------------------------------
struct F8Frag {
    u32x4 h[2];  // 32 codes of a row
};
struct F8Wide {
    bf16x8_t v[4];  // the same in bf16
    __device__ __forceinline__ F8Wide() {}
    __device__ __forceinline__ explicit F8Wide(const F8Frag &f) {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = widen_fp8x8(f.h[k / 2][k % 2 * 2], f.h[k / 2][k % 2 * 2 + 1]);
    }
};
// A block's products: rows of `b` become the 16 x 16 block's rows (4 (lane / 16) + c), rows of
// `a` its columns (lane % 16).  The order of k within a lane's 32 codes is free, as
// long as both operands have the same.
__device__ __forceinline__ f32x4 f8_block(const F8Frag &b, const F8Frag &a) {
    union { u32x4 h[2]; i32x8 v; } fb, fa;
    fb.h[0] = b.h[0], fb.h[1] = b.h[1], fa.h[0] = a.h[0], fa.h[1] = a.h[1];
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb.v, fa.v, f32x4{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ f32x4 f8_block(const F8Wide &b, const F8Wide &a) {
    f32x4 c = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < 4; ++k) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b.v[k], a.v[k], c, 0, 0, 0);
    return c;
}

// 16 rows x 16 columns by a wave, straight from global memory: pieces p, p + step, ...
// of the range [k0, k0 + klen).  Sums in fp64, which scales of any size cannot leave.
__device__ __forceinline__ void f8_direct(const OpGemmArgs &g, int e, int n0, int lo, int rows, int k0, int klen, int p,
                                          int step, double (&acc)[4]) {
    constexpr int U = 2;
    const int lane = threadIdx.x & 63, r16 = lane & 15, q4 = lane >> 4;
    // rows past the last one repeat it (their results are not stored)
    const long long row = lo + min(r16, rows - 1);
    const uint8_t *b = (const uint8_t *)g.B + (long long)e * g.b_stride + (long long)min(n0 + r16, g.N - 1) * g.ldb + k0;
    const uint8_t *a = (const uint8_t *)g.A + row * g.lda + k0;
    const float *sb = g.sb + ((long long)e * ((g.N + 127) >> 7) + (n0 >> 7)) * g.kb + (k0 >> 7);
    const float *sa = g.sa + row * g.kb + (k0 >> 7);
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[c] = 0.0;
    auto add = [&](const F8Frag &fb, const F8Frag &fa, float x, float w) {
        const f32x4 v = f8_block(F8Wide(fb), F8Wide(fa));
        const double f = (double)x * (double)w;
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[c] += (double)v[c] * f;
    };
    const int pieces = (klen + 127) >> 7, whole = klen >> 7;
    // UU pieces, all loads in flight before the first product
    auto some = [&](auto UU_) {
        constexpr int UU = decltype(UU_)::value;
        F8Frag fb[UU], fa[UU];
        float w[UU], x[UU];
#pragma unroll
        for (int u = 0; u < UU; ++u) {
            const int q = p + u * step;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const long long o = (long long)q * 128 + h * 64 + q4 * 16;
                __builtin_memcpy(&fb[u].h[h], b + o, 16);
                __builtin_memcpy(&fa[u].h[h], a + o, 16);
            }
            w[u] = sb[q];
            x[u] = sa[q];
        }
#pragma unroll
        for (int u = 0; u < UU; ++u) add(fb[u], fa[u], x[u], w[u]);
        p += UU * step;
    };
    while (p + (U - 1) * step < whole) some(num<U>{});
    while (p < whole) some(num<1>{});
    if (p < pieces) {  // the last, part piece
        F8Frag fb, fa;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = p * 128 + h * 64 + q4 * 16;
            fb.h[h] = load_chunk<1>(b + k, klen - k);
            fa.h[h] = load_chunk<1>(a + k, klen - k);
        }
        add(fb, fa, sa[p], sb[p]);
    }
}

// Results of row lo + ml at columns n .. n + 3, or a range's sums of them.
__device__ __forceinline__ void f8_put4(const OpGemmArgs &g, long long row, int n, int ks, const float (&v)[4]) {
    if (g.splits > 1) {
        float *ws = g.ws + ((long long)ks * g.rows + row) * g.N;
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (n + c < g.N) ws[n + c] = v[c];
    } else {
        put4(g, row * g.ldc + n, n, v[0], v[1], v[2], v[3], vec_ok(g));
    }
}

// Few rows: as op_stream_kernel, 16 rows at a time.  Bound by reading the weights: a row on
// two experts of 4096 / 14336 28 us (117 MB, one wave of workgroups), on all eight 101 (4.7 TB/s).
__global__ __launch_bounds__(kStreamWaves * 64) void op_f8_stream_kernel(OpGemmArgs g) {
    __shared__ double red[kStreamWaves][4][64];
    const int r = blockIdx.x / g.nt, n0 = (blockIdx.x - r * g.nt) * 16, ks = blockIdx.y;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int e, lo, hi, k0, klen;
    held_group(g, r, e, lo, hi);
    if (e < 0) return;
    k_range(g, ks, 128, k0, klen);
    for (; lo < hi; lo += 16) {
        double acc[4];
        f8_direct(g, e, n0, lo, min(hi - lo, 16), k0, klen, w, kStreamWaves, acc);
#pragma unroll
        for (int c = 0; c < 4; ++c) red[w][c][lane] = acc[c];
        __syncthreads();
        if (w == 0) {
            float v[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                double s = red[0][c][lane];
                for (int x = 1; x < kStreamWaves; ++x) s += red[x][c][lane];
                v[c] = (float)s;
            }
            const int ml = lane & 15, n = n0 + 4 * (lane >> 4);
            if (ml < hi - lo && n < g.N) f8_put4(g, lo + ml, n, ks, v);
        }
        __syncthreads();
    }
}

// Tiles sum in units of 2^-48.  A product of two scales is then a normal number from 2^-174 on,
// and a smaller one's rounding, 2^-150 in these units, changes a sum of 2^23 blocks (each below
// 128 * 448^2 < 2^25) by less than 2^-149, fp32's last place.  Up to 2^31 no such sum
// overflows, so that an infinity in one is the result's own.
constexpr float kF8Unit = 0x1p48f, kF8Most = 0x1p79f, kF8Normal = 0x1p-78f;  // 2^31, 2^-126 in it
// The largest and the smallest non-zero product (in magnitude) that a lane multiplies with.
struct F8Range {
    unsigned most = 0, least = ~0u;  // bits; twice the bits less one (0: ~0)
    __device__ __forceinline__ void take(float f) {
        const unsigned u = __float_as_uint(f);
        most = max(most, u & 0x7fffffffu);
        least = min(least, (u << 1) - 1u);
    }
    // some row may have to be summed in fp64 (f8_far_row)
    __device__ __forceinline__ bool far() const {
        return most > __float_as_uint(kF8Most) || least < 2u * __float_as_uint(kF8Normal) - 1u;
    }
};
// Rows that are: one product too large, or all below fp32's normal range, whose results would
// be rounded twice.  (With a NaN among them the row's are NaN already.)  most: the bits of the
// row's largest.
__device__ __forceinline__ bool f8_far_row(unsigned most) {
    return (most > __float_as_uint(kF8Most) && most <= 0x7f800000u) || (most > 0u && most < __float_as_uint(kF8Normal));
}

// The tile loop: as op_gemm_tile, a stage one block of k, the wave's columns taken one
// 16-column block at a time.  Step j of a stage:
//   MFMAs of column block j: the block's sums, MI x 4 registers
//   the sums of block j - 1 (of the stage before: its last) times the scales, into acc
//   reads of column block j + 1; in the last step the wait for stage s + 1, the barrier
//   and the reads of its scales, first columns and rows, and the loads of stage s + 2
// so that the vector unit's part runs under the next MFMAs.  The scales of a stage, one
// for each row and column of the tile, come into the ring with it.
// WIDE: the codes in bf16.
// 8192 rows, 8 even groups of 4096 / 14336, codes given, 256 x 256 tiles: 481 to 499 us (2.0
// PFLOP/s; the scaling after the products instead of under them 553); skewed groups 526 to 550,
// of whose cycles the matrix units are busy 42 % and other vector instructions, mostly the
// scaling's four multiply-adds per product instruction, take 34 %: three quarters if neither ran
// under the other; in 35 % of their time waves wait.  Widened, 128 x 128 tiles: bf16 870 and 930 us,
// fp32 890 and 960.
template <int BM, int BN, int WM, int WN, int NS, int VB, bool WIDE>
__device__ __forceinline__ void f8_gemm_tile(const OpGemmArgs &g, uint8_t *ring_) {
    constexpr int NT = WM * WN * 64, KE = 128;
    constexpr int MI = BM / WM / 16, NJ = BN / WN / 16;
    constexpr bool DIRECT = VB > 0;
    static_assert(NS == 2 && NJ % 2 == 0 && BM + BN <= NT && 128 % (BN / WN) == 0, "slots, scales, one block of columns per wave");
    using TA = Tile<1, BM, false, NT, 2, VB>;
    using TB = Tile<1, BN, false, NT, 2, VB>;
    constexpr int RING = NS * (TA::BYTES + TB::BYTES), SCALES = RING;  // then NS x NT scales

    OpJob jb;
    if (!ragged_job<BM>(g, jb, BN)) return;
    const int lane = threadIdx.x & 63, r16 = lane & 15, q4 = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = w % WM, wn = w / WM;
    const int mrows = jb.len - jb.m0;
    int k0, klen;
    k_range(g, jb.ks, KE, k0, klen);
    TA ta;
    TB tb;
    ta.init((const uint8_t *)g.A + (long long)(jb.lo + jb.m0) * g.lda + k0, g.lda, mrows, klen);
    tb.init((const uint8_t *)g.B + (long long)jb.e * g.b_stride + (long long)jb.n0 * g.ldb + k0, g.ldb, g.N - jb.n0, klen);
    // this thread's scale: of tile row t (t < BM), of tile column t - BM
    const float *sbase = w * 64 < BM ? g.sa + (long long)(jb.lo + jb.m0) * g.kb + (k0 >> 7)
                                     : g.sb + ((long long)jb.e * ((g.N + 127) >> 7) + (jb.n0 >> 7)) * g.kb + (k0 >> 7);
    const unsigned sb_lo = __builtin_amdgcn_readfirstlane((unsigned)(unsigned long long)sbase);
    const unsigned sb_hi = __builtin_amdgcn_readfirstlane((unsigned)((unsigned long long)sbase >> 32));
    unsigned soff = kOutOfRange;
    if constexpr (DIRECT) {
        const int t = threadIdx.x;
        if (t < BM) {
            if (t < mrows) soff = (unsigned)(t * g.kb * 4);
        } else if (t < BM + BN) {
            if (t - BM < g.N - jb.n0) soff = (unsigned)(((t - BM) >> 7) * g.kb * 4);
        }
    }
    const int S = (klen + KE - 1) / KE;
    lds_u8 *ring = (lds_u8 *)ring_;
    constexpr int A0 = 0, B0 = NS * TA::BYTES;  // all slots of A, all of B, all scales
    auto a_slot = [](auto SLOT) { return A0 + decltype(SLOT)::value * TA::BYTES; };
    auto b_slot = [](auto SLOT) { return B0 + decltype(SLOT)::value * TB::BYTES; };
    auto s_slot = [](auto SLOT) { return SCALES + decltype(SLOT)::value * NT * 4; };
    // The lane's places in the images, of the first slot and block: the others are within
    // a DS instruction's offset of them.  (Opaque: the compiler would otherwise keep an
    // address for each read, more than there are registers.)
    auto place = [&](int at) {
        unsigned v = (unsigned)(uintptr_t)ring + at;
        asm("" : "+v"(v));
        return v;
    };
    auto chunk = [&](int half) { return ((half * 4 + q4) ^ TA::row_swz(r16)) << 4; };
    const unsigned a_at[2] = {place(A0 + (wm * 16 + r16) * 128 + chunk(0)), place(A0 + (wm * 16 + r16) * 128 + chunk(1))};
    const unsigned b_at[2] = {place(B0 + (wn * NJ * 16 + r16) * 128 + chunk(0)), place(B0 + (wn * NJ * 16 + r16) * 128 + chunk(1))};
    const unsigned x_at = place(SCALES + (wm * 16 + r16) * 4), w_at = place(SCALES + (BM + wn * (BN / WN)) * 4);
    using FragA = std::conditional_t<WIDE, F8Wide, F8Frag>;
    auto read_a = [&](auto SLOT, int i) {
        F8Frag f;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            f.h[h] = *(const __attribute__((address_space(3))) u32x4 *)(uintptr_t)(a_at[h] + decltype(SLOT)::value * TA::BYTES + i * WM * 2048);
        return FragA(f);
    };
    auto read_b = [&](auto SLOT, int j) {
        F8Frag f;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            f.h[h] = *(const __attribute__((address_space(3))) u32x4 *)(uintptr_t)(b_at[h] + decltype(SLOT)::value * TB::BYTES + j * 2048);
        return f;
    };
    typedef __attribute__((address_space(3))) float lds_f32;
    F8Range range;
    auto read_scales = [&](auto SLOT, float (&f)[MI]) {
        // one for all columns of the wave
        const float sw = __uint_as_float(__builtin_amdgcn_readfirstlane(
            *(const __attribute__((address_space(3))) unsigned *)(uintptr_t)(w_at + decltype(SLOT)::value * NT * 4)));
        const float unit = sw * kF8Unit;
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            const float sx = *(const lds_f32 *)(uintptr_t)(x_at + decltype(SLOT)::value * NT * 4 + i * WM * 64);
            f[i] = sx * unit;
            range.take(f[i]);
        }
    };
    f32x4 acc[MI][NJ];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    FragA fa[MI];
    F8Frag fb[2];
    f32x4 part[2][MI];
    float f[2][MI];
#pragma unroll
    for (int i = 0; i < MI; ++i) part[1][i] = f32x4{0, 0, 0, 0}, f[1][i] = 0.0f;
    // NI: the wave's row blocks that hold rows
    auto scaled = [&](auto NI, int j, const f32x4 (&p)[MI], const float (&by)[MI]) {
#pragma unroll
        for (int i = 0; i < decltype(NI)::value; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[i][j][c] = fmaf(p[i][c], by[i], acc[i][j][c]);
    };
    // P: the parity of the stage
    auto step = [&](auto NI, auto P, int j) {
        constexpr int p = decltype(P)::value;
        const FragA b(fb[j & 1]);
#pragma unroll
        for (int i = 0; i < decltype(NI)::value; ++i) part[j & 1][i] = f8_block(b, fa[i]);
        if (j == 0) scaled(NI, NJ - 1, part[1], f[1 - p]);
        else scaled(NI, j - 1, part[1 - (j & 1)], f[p]);
    };
    // the order of a step: reads first, then after each MFMA what fits under it
    auto mixed = [](auto NI) {
        if constexpr (!WIDE) {
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
            for (int i = 0; i < decltype(NI)::value; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x2, 4, 0);
            }
        }
    };
    if (S > 0) {
        if constexpr (DIRECT) {
            constexpr int NL = TA::NC + TB::NC + 1;
            const unsigned l0 = (unsigned)(uintptr_t)ring;
            auto load_scales = [&](auto SLOT, int s) {
                const unsigned long long at = ((unsigned long long)sb_hi << 32 | sb_lo) + 4ull * s;
                u32x4 rs;
                rs[0] = __builtin_amdgcn_readfirstlane((unsigned)at);
                rs[1] = __builtin_amdgcn_readfirstlane((unsigned)(at >> 32) & 0xffffu);
                rs[2] = 0x7fffffffu;
                rs[3] = 0x00027000u;
                const unsigned v = s < S ? soff : kOutOfRange;
                const unsigned m0 = __builtin_amdgcn_readfirstlane(l0 + s_slot(SLOT) + w * 256);
                asm volatile("s_nop 4\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds" ::"v"(v),
                             "s"(rs), "s"(m0)
                             : "m0");
            };
            auto load = [&](auto SLOT, int s) {
                ta.load_lds(s, l0 + a_slot(SLOT), w);
                tb.load_lds(s, l0 + b_slot(SLOT), w);
                load_scales(SLOT, s);
            };
            load(num<0>{}, 0);
            load(num<1>{}, 1);
            wait_loads<NL>();
            lds_barrier();
            read_scales(num<0>{}, f[0]);
            auto run = [&](auto NI_) {
                constexpr int NI = decltype(NI_)::value;
#pragma unroll
                for (int i = 0; i < NI; ++i) fa[i] = read_a(num<0>{}, i);
                if constexpr (NI > 0) fb[0] = read_b(num<0>{}, 0);
                auto stage = [&](auto SLOT, int s) {
                    constexpr int P = decltype(SLOT)::value;
                    using Next = num<1 - P>;
#pragma unroll
                    for (int j = 0; j < NJ; ++j) {
                        if (j < NJ - 1) {
                            if constexpr (NI > 0) {
                                fb[1 - (j & 1)] = read_b(SLOT, j + 1);
                                step(NI_, SLOT, j);
                                mixed(NI_);
                            }
                        } else {
                            wait_loads<0>();
                            lds_barrier();
                            const F8Frag last = fb[1];
                            if constexpr (NI > 0) fb[0] = read_b(Next{}, 0);
                            const FragA b(last);
#pragma unroll
                            for (int i = 0; i < MI; ++i) {
                                if (i < NI) {
                                    part[1][i] = f8_block(b, fa[i]);
                                    fa[i] = read_a(Next{}, i);
#pragma unroll
                                    for (int c = 0; c < 4; ++c)
                                        acc[i][j - 1][c] = fmaf(part[0][i][c], f[P][i], acc[i][j - 1][c]);
                                }
                                if (i == 0) ta.load_lds(s + NS, l0 + a_slot(SLOT), w);
                                if (i == 1) tb.load_lds(s + NS, l0 + b_slot(SLOT), w);
                                if (i == MI - 1) load_scales(SLOT, s + NS);
                                __builtin_amdgcn_sched_barrier(0);
                            }
                            read_scales(Next{}, f[1 - P]);
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                };
                int s = 0;
                for (; s + 2 <= S; s += 2) {
                    stage(num<0>{}, s);
                    stage(num<1>{}, s + 1);
                }
                if (s < S) stage(num<0>{}, s);
#pragma unroll
                for (int i = 0; i < NI; ++i) f[1][i] = (S & 1) ? f[0][i] : f[1][i];
                scaled(NI_, NJ - 1, part[1], f[1]);
            };
            if constexpr (MI < 4) {
                run(num<MI>{});
            } else {
                const int ni = (mrows - wm * 16 + WM * 16 - 1) / (WM * 16);
                if (ni >= MI) run(num<MI>{});
                else if (ni == 3) run(num<3>{});
                else if (ni == 2) run(num<2>{});
                else if (ni == 1) run(num<1>{});
                else run(num<0>{});
            }
            wait_loads<0>();  // no load may still be writing LDS when the workgroup ends
        } else {
            float sreg = 0.0f;
            auto load = [&](int s) {
                ta.load_regs(s);
                tb.load_regs(s);
                const int t = threadIdx.x;  // (rows may be too far apart for 32 bits here)
                const bool row = t < BM, ok = row ? t < mrows : t < BM + BN && t - BM < g.N - jb.n0;
                sreg = ok ? sbase[(row ? (long long)t : (long long)((t - BM) >> 7)) * g.kb + s] : 0.0f;
            };
            auto keep = [&](auto SLOT) {
                ta.store_regs(ring + a_slot(SLOT));
                tb.store_regs(ring + b_slot(SLOT));
                ((lds_f32 *)(ring + s_slot(SLOT)))[threadIdx.x] = sreg;
            };
            auto stage = [&](auto SLOT, int s) {
                lds_barrier();
                if (s + 1 < S) load(s + 1);
                read_scales(SLOT, f[decltype(SLOT)::value]);
#pragma unroll
                for (int i = 0; i < MI; ++i) fa[i] = read_a(SLOT, i);
                fb[0] = read_b(SLOT, 0);
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    if (j < NJ - 1) fb[1 - (j & 1)] = read_b(SLOT, j + 1);
                    step(num<MI>{}, SLOT, j);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (s + 1 < S) keep(num<1 - decltype(SLOT)::value>{});
            };
            load(0);
            keep(num<0>{});
            int s = 0;
            for (; s + 2 <= S; s += 2) {
                stage(num<0>{}, s);
                stage(num<1>{}, s + 1);
            }
            if (s < S) stage(num<0>{}, s);
#pragma unroll
            for (int i = 0; i < MI; ++i) f[1][i] = (S & 1) ? f[0][i] : f[1][i];
            scaled(num<MI>{}, NJ - 1, part[1], f[1]);
        }
    }
    const bool far = __any(range.far());
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] *= 1.0f / kF8Unit;
    bool split = false;
    if constexpr (WIDE && BM <= 64) split = g.splits > 1;  // (split calls run the smallest tiles, widened)
    if (split) {
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            const int ml = (i * WM + wm) * 16 + r16;
            if (ml >= mrows) continue;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int n = jb.n0 + (wn * NJ + j) * 16 + 4 * q4;
                const float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
                f8_put4(g, jb.lo + jb.m0 + ml, n, jb.ks, v);
            }
        }
    } else {
        const long long at0 = (long long)(jb.lo + jb.m0) * g.ldc;
        auto val = [&](int i, int j, int c) -> float { return acc[i][j][c]; };
        bool f32 = false;
        if constexpr (WIDE) f32 = g.c_f32;  // (fp32 results are of widened codes)
        if (f32) store_tile_rows<4, BM, BN, WM, WN, RING, false>(g, ring, at0, mrows, jb.n0, wm, wn, lane, val);
        else store_tile_rows<2, BM, BN, WM, WN, RING, false>(g, ring, at0, mrows, jb.n0, wm, wn, lane, val);
    }
    // Far rows' results again, in fp64, over those just stored (every wave's stores are done
    // at the barrier).  A row's depend on its own scales alone.  8192 rows on 8 experts of 4096 /
    // 14336, even and skewed groups: with one such row 1094 and 708 us, 490 and 545 without (skewed
    // ones on a slower box: one row 978, 101 rows 2500, all of them 9800, none 640); with
    // one block's scale of 1e-36 in a row or a weight of otherwise ordinary ones, where this only
    // looks, 500 and 550.
    wait_loads<0>();
    lds_barrier();
    if (!far) return;
    // (opaque: addresses formed from them before the loop would be kept through it)
    int e = jb.e, row0 = jb.lo + jb.m0;
    asm("" : "+s"(e), "+s"(row0));
    const int nw = jb.n0 + wn * (BN / WN);
    if (nw >= g.N) return;
    const float *sb = g.sb + ((long long)e * ((g.N + 127) >> 7) + (nw >> 7)) * g.kb + (k0 >> 7);
    for (int i = 0; i < MI; ++i) {
        const int r0 = (i * WM + wm) * 16;
        if (r0 >= mrows) continue;
        const float *sa = g.sa + (long long)(row0 + min(r0 + r16, mrows - 1)) * g.kb + (k0 >> 7);
        unsigned most = 0;
        for (int s = q4; s < S; s += 4) most = max(most, __float_as_uint(sa[s] * (sb[s] * kF8Unit)) & 0x7fffffffu);
        most = max(most, (unsigned)__shfl_xor((int)most, 16));
        most = max(most, (unsigned)__shfl_xor((int)most, 32));
        const bool again = f8_far_row(most);
        if (!__any(again)) continue;
        for (int j = 0; j < NJ; ++j) {
            const int n0 = nw + j * 16;
            if (n0 >= g.N) continue;
            double d[4];
            f8_direct(g, e, n0, row0 + r0, min(16, mrows - r0), k0, klen, 0, 1, d);
            const int n = n0 + 4 * q4;
            if (again && r0 + r16 < mrows && n < g.N) {
                const float v[4] = {(float)d[0], (float)d[1], (float)d[2], (float)d[3]};
                f8_put4(g, row0 + r0 + r16, n, jb.ks, v);
            }
        }
    }
}

template <int BM, int BN, int WM, int WN, int NS, int WPE, int VB, bool WIDE>
__global__ __launch_bounds__(WM * WN * 64) __attribute__((amdgpu_waves_per_eu(WPE, WPE))) void op_f8_kernel(OpGemmArgs g) {
    __shared__ __attribute__((aligned(1024))) uint8_t ring[NS * ((BM + BN) * 128 + WM * WN * 64 * 4)];
    f8_gemm_tile<BM, BN, WM, WN, NS, VB, WIDE>(g, ring);
}

}  // namespace ops

template <int BM, int BN, int WM, int WN, int WPE, bool WIDE>
static hipError_t launch_f8_tiles(OpGemmArgs g, int vb, hipStream_t s) {
    g.nt = (g.N + BN - 1) / BN;
    const long long mtiles = (long long)(g.rows / BM) + (g.E < g.rows ? g.E : g.rows);
    const long long grid = (mtiles * g.nt * g.splits + 7) / 8 * 8;
    if (grid > 0x7fffffffll / (WM * WN * 64)) return kOpTooLarge;
    const dim3 gr((unsigned)grid), b(WM * WN * 64);
    if (vb == 16) {
        ops::op_f8_kernel<BM, BN, WM, WN, 2, WPE, 16, WIDE><<<gr, b, 0, s>>>(g);
    } else if constexpr (BN != 64) {
        return hipErrorInvalidValue;
    } else if (vb == 4) {
        ops::op_f8_kernel<BM, BN, WM, WN, 2, WIDE ? 2 : WPE, 4, WIDE><<<gr, b, 0, s>>>(g);
    } else {
        ops::op_f8_kernel<BM, BN, WM, WN, 2, WIDE ? 2 : WPE, 0, WIDE><<<gr, b, 0, s>>>(g);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess && g.splits > 1 ? launch_op_fold(OT_BF16, false, g, s) : e;
}

hipError_t launch_op_gemm_f8(OpGemmArgs g, int ncu, hipStream_t s) {
    if (op_f8_streamed(g.rows, g.E, g.N, g.K, ncu)) {
        g.nt = (g.N + 15) / 16;
        const long long grid = (long long)(g.E < g.rows ? g.E : g.rows) * g.nt;
        if (grid * g.splits > 0x7fffffffll / (ops::kStreamWaves * 64)) return kOpTooLarge;
        ops::op_f8_stream_kernel<<<dim3((unsigned)grid, g.splits), ops::kStreamWaves * 64, 0, s>>>(g);
        const hipError_t e = hipGetLastError();
        return e == hipSuccess && g.splits > 1 ? launch_op_fold(OT_BF16, false, g, s) : e;
    }
    int vb = 0;
    if (ops::tile_offsets_ok(g.lda, 1) && ops::tile_offsets_ok(g.ldb, 1)) {
        auto pieces = [&](int bytes) {
            return ops::whole_pieces(g.A, g.lda, 0, g.K, 1, bytes) && ops::whole_pieces(g.B, g.ldb, g.b_stride, g.K, 1, bytes);
        };
        if (pieces(16)) vb = 16;
        else if (g.lda >= 16 && g.ldb >= 16 && pieces(4)) vb = 4;
    }
    // fp32 results, sums that are folded, and where the caller asks for it: the codes
    // widened (above)
    const bool wide = g.c_f32 || g.splits > 1 || g.exact;
    OpTileCost c = wide ? kCostF8Wide : kCostF8;
    if (vb != 16) c.c256 = c.c128 = 0;  // (the other loads' registers do not fit beside these tiles)
    const int t = g.splits > 1 ? 64 : op_pick_tile(c, g.rows, g.E, g.N, ncu, false);
    if (t == 256) return launch_f8_tiles<256, 256, 4, 2, 2, false>(g, vb, s);
    if (t == 128 && wide) return launch_f8_tiles<128, 128, 2, 2, 2, true>(g, vb, s);
    if (t == 128) return launch_f8_tiles<128, 128, 2, 2, 2, false>(g, vb, s);
    if (wide) return launch_f8_tiles<64, 64, 2, 2, 3, true>(g, vb, s);
    return launch_f8_tiles<64, 64, 2, 2, 3, false>(g, vb, s);
}

template <int XB, bool VEC>
static void quantize_f8(const QuantF8Args &a, hipStream_t s) {
    const long long kbs = (a.cols + 127) / 128;
    if (a.block_rows != 1) {
        ops::quantize_f8_tiles_kernel<XB, VEC><<<op_row_grid(a.mats * ((a.rows + 127) / 128) * kbs), 256, 0, s>>>(a);
        return;
    }
    int lx = 0;
    while (lx < 4 && (1 << lx) < kbs) ++lx;
    const long long gy = (((a.rows + (16 >> lx) - 1) >> (4 - lx)) + 3) / 4;
    const dim3 gr((unsigned)((kbs + (1 << lx) - 1) >> lx), (unsigned)(gy < 16384 ? gy : 16384),
                  (unsigned)(a.mats < 1024 ? a.mats : 1024));
    ops::quantize_f8_rows_kernel<XB, VEC><<<gr, 256, 0, s>>>(a, lx);
}

hipError_t launch_quantize_f8(const QuantF8Args &a, hipStream_t s) {
    const int es = a.x_bf16 ? 2 : 4;
    const bool vec = (((uintptr_t)a.x | (uintptr_t)(a.ldx * es) | (uintptr_t)(a.x_stride * es)) & 15) == 0 &&
                     (((uintptr_t)a.q | (uintptr_t)a.ldq | (uintptr_t)a.q_stride) & 7) == 0 && (a.cols & 7) == 0 &&
                     (a.pad_to & 7) == 0;
    if (a.x_bf16 && vec) quantize_f8<1, true>(a, s);
    else if (a.x_bf16) quantize_f8<1, false>(a, s);
    else if (vec) quantize_f8<0, true>(a, s);
    else quantize_f8<0, false>(a, s);
    return hipGetLastError();
}

}  // namespace moe
