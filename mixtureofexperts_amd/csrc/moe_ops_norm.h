// moe_ops_norm.h -- the norms before and after a block with its gate and
// residual scale, and their gradients: one pass over the data, a row held in
// registers by TPR threads (8 consecutive channels per thread and vector), so
// that every tensor is read and written once.  Bound by HBM: 8192 x 4096, a bf16
// stream and fp32 y with both norms and a gate 67 us (336 MB, 5.0 TB/s; 51 with
// the inputs in the last-level cache), the gradients 115 (537 MB, 4.7 TB/s); one
// row of 512 2.2 us of kernel.
#pragma once
#include "moe_internal.h"
#include "moe_ops.h"

namespace moe {
namespace ops {

// Eight channels of a row.
struct Row8 {
    float v[8];
};
// The same as they are loaded: fp32, or bf16 pairs in the first four words.  A
// load and its widening are apart so that loads of several tensors are in
// flight together, whatever their types (the branches are uniform).  Without
// VEC (odd D or unaligned rows) the elements are widened as they are read.
struct Raw8 {
    unsigned u[8];
};
// channels from c of a row; those past D read as 0.  ANY (without VEC): whole vectors
// by loads that need not be aligned, all but a row's last (8190 x 4092, bf16: the norm
// 77 us, by elements 262; the gradient's largest form has no registers left for it).
template <bool VEC, bool ANY = false>
__device__ __forceinline__ Raw8 load_raw(const void *p, int bf16, long long row, int c, int D) {
    Raw8 o{};
    if (bf16) {
        const uint16_t *q = (const uint16_t *)p + row * D + c;
        if constexpr (VEC) {
            if (c < D) {
                const uint4 w = *(const uint4 *)q;
                o.u[0] = w.x, o.u[1] = w.y, o.u[2] = w.z, o.u[3] = w.w;
            }
        } else if (ANY && c + 8 <= D) {
            unsigned w[4];
            __builtin_memcpy(w, q, 16);
#pragma unroll
            for (int i = 0; i < 8; ++i) o.u[i] = i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) o.u[i] = c + i < D ? (unsigned)q[i] << 16 : 0u;
        }
    } else {
        const unsigned *q = (const unsigned *)p + row * D + c;
        if constexpr (VEC) {
            if (c < D) {
                const uint4 w = *(const uint4 *)q, x = *(const uint4 *)(q + 4);
                o.u[0] = w.x, o.u[1] = w.y, o.u[2] = w.z, o.u[3] = w.w;
                o.u[4] = x.x, o.u[5] = x.y, o.u[6] = x.z, o.u[7] = x.w;
            }
        } else if (ANY && c + 8 <= D) {
            __builtin_memcpy(o.u, q, 32);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) o.u[i] = c + i < D ? q[i] : 0u;
        }
    }
    return o;
}
template <bool VEC>
__device__ __forceinline__ Row8 widen(const Raw8 &r, int bf16) {
    Row8 o;
    if (VEC && bf16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            o.v[2 * i] = __uint_as_float(r.u[i] << 16);
            o.v[2 * i + 1] = __uint_as_float(r.u[i] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) o.v[i] = __uint_as_float(r.u[i]);
    }
    return o;
}
template <bool VEC, bool ANY = false>
__device__ __forceinline__ Row8 load8(const void *p, int bf16, long long row, int c, int D) {
    return widen<VEC>(load_raw<VEC, ANY>(p, bf16, row, c, D), bf16);
}
__device__ __forceinline__ unsigned pack_bf16(float a, float b) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(unsigned, v);
}
template <bool VEC, bool ANY = false>
__device__ __forceinline__ void store8(void *p, int bf16, long long row, int c, int D, const Row8 &o) {
    if (c >= D) return;
    if (bf16) {
        uint16_t *q = (uint16_t *)p + row * D + c;
        unsigned w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack_bf16(o.v[2 * i], o.v[2 * i + 1]);
        if constexpr (VEC) {
            *(uint4 *)q = make_uint4(w[0], w[1], w[2], w[3]);
        } else if (ANY && c + 8 <= D) {
            __builtin_memcpy(q, w, 16);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < D) q[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
        }
    } else {
        float *q = (float *)p + row * D + c;
        if constexpr (VEC) {
            *(float4 *)q = make_float4(o.v[0], o.v[1], o.v[2], o.v[3]);
            *(float4 *)(q + 4) = make_float4(o.v[4], o.v[5], o.v[6], o.v[7]);
        } else if (ANY && c + 8 <= D) {
            __builtin_memcpy(q, o.v, 32);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < D) q[i] = o.v[i];
        }
    }
}

// The same around the caches (16-byte rows, as the type has them).
__device__ __forceinline__ void store8_past(void *p, int bf16, long long row, int c, int D, const Row8 &o) {
    typedef unsigned u32x4v __attribute__((ext_vector_type(4)));
    if (c >= D) return;
    if (bf16) {
        typedef __bf16 bf16x8v __attribute__((ext_vector_type(8)));
        bf16x8v b;
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = (__bf16)o.v[i];
        __builtin_nontemporal_store(__builtin_bit_cast(u32x4v, b), (u32x4v *)((uint16_t *)p + row * D + c));
    } else {
        u32x4v *q = (u32x4v *)((float *)p + row * D + c);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            __builtin_nontemporal_store(u32x4v{__float_as_uint(o.v[4 * i]), __float_as_uint(o.v[4 * i + 1]),
                                               __float_as_uint(o.v[4 * i + 2]), __float_as_uint(o.v[4 * i + 3])},
                                        q + i);
    }
}

// Sum over the TPR threads of a row, the same bits in each of them.  Every sum
// of a workgroup uses another `part` than the one before it: the barrier of a
// sum then also separates the reads of the sum before from the writes of the
// one after.
// A wave's part runs on DPP (four steps inside rows of 16 lanes, then the four
// rows' sums by lane reads): no LDS round trips.
template <int CTRL>
__device__ __forceinline__ float add_dpp(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float wave_sum(float v) {
    v = add_dpp<0xB1>(v);   // lane ^ 1
    v = add_dpp<0x4E>(v);   // lane ^ 2
    v = add_dpp<0x141>(v);  // the other quad of 8 lanes
    v = add_dpp<0x140>(v);  // the other half of 16 lanes
    auto row = [&](int l) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l)); };
    return (row(0) + row(16)) + (row(32) + row(48));
}
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float *part) {
    v = wave_sum(v);
    if constexpr (TPR > 64) {
        constexpr int NW = TPR / 64;
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
        __syncthreads();
        v = part[0];
#pragma unroll
        for (int w = 1; w < NW; ++w) v += part[w];
    }
    return v;
}

// The same with its last steps in fp64: those of the few largest partial sums,
// whose roundings would be the sum's (the others' average out).
template <int TPR>
__device__ __forceinline__ double row_sum_wide(float v, double *part) {
    v = add_dpp<0x140>(add_dpp<0x141>(add_dpp<0x4E>(add_dpp<0xB1>(v))));
    auto row = [&](int l) {
        return (double)__builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l));
    };
    double d = (row(0) + row(16)) + (row(32) + row(48));
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = d;
        __syncthreads();
        d = part[0];
#pragma unroll
        for (int w = 1; w < TPR / 64; ++w) d += part[w];
    }
    return d;
}

// WIDE: a bf16 stream that a gate or a post norm is added to.  An r that a few fp32
// roundings put on the other side of a bf16 border (one in 30000) would be 2^-8 off
// in an fp32 h, far more than all else there, and whether h is wanted, and in which
// type, may not decide r.  So r is always the fp64 formula's value rounded by way of
// fp32 (one in 290000 on the other side then; 2000 x 4096: an fp32 h off by 2e-6 of its
// norm, 1.3e-5 by fp32 steps): it is formed in fp32, and again in fp64 where a border
// lies within what the fp32 steps may be off (about an element in 8000).  Each rounds
// by 2^-24 of its value: y's term at rstd beta, its product with y, the weight and the
// gate, the sum at the addition and on the way by fp32.  8192 x 4096, fp32 y, both
// norms, a gate: 67 to 68 us, 67 all in fp32, 81 all in fp64 (117 registers instead of 66).
template <int TPR, int NV, bool VEC, bool WIDE>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void block_norm_kernel(NormArgs a) {
    constexpr int RPB = TPR < 256 ? 256 / TPR : 1;
    __shared__ float part[2][16];
    __shared__ double wpart[WIDE ? 16 : 1];
    const long long row = op_row_block() * RPB + threadIdx.x / TPR;
    if (row >= a.T) return;  // whole waves; no barrier below when RPB > 1, the whole workgroup otherwise
    const int tid = threadIdx.x % TPR, D = a.D;
    Row8 r[NV], y[NV];
    Raw8 rx[NV];
    {
        Raw8 ry[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (tid + i * TPR) * 8;
            rx[i] = load_raw<VEC, true>(a.x, WIDE ? 1 : a.x_bf16, row, c, D);
            ry[i] = a.y ? load_raw<VEC, true>(a.y, a.y_bf16, row, c, D) : Raw8{};
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if constexpr (!WIDE) r[i] = widen<VEC>(rx[i], a.x_bf16);
            y[i] = widen<VEC>(ry[i], a.y_bf16);
        }
    }
    float iy = 1.0f;
    double iyw = 1.0;
    if (a.y && a.post) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int q = 0; q < 8; ++q) s += y[i].v[q] * y[i].v[q];
        if constexpr (WIDE) {
            const double m = row_sum_wide<TPR>(s, wpart) / (double)D + (double)a.eps;
            if (m > 1e-30 && m < 1e30) {  // a Newton step of 1 / sqrt(m) from its fp32 value
                const double v = 1.0f / sqrtf((float)m);
                iyw = v * (1.5 - 0.5 * m * v * v);
            } else {
                iyw = 1.0 / sqrt(m);
            }
            iy = (float)iyw;
        } else {
            iy = 1.0f / sqrtf(row_sum<TPR>(s, part[0]) / (float)D + a.eps);
        }
    }
    const long long grow = a.gate ? row / a.gate_rows : 0;
    float s = 0.0f;
    if constexpr (WIDE) {
        const float f = (float)((double)a.beta * iyw);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (tid + i * TPR) * 8;
            const Row8 p = a.post ? load8<VEC, true>(a.post, a.w_bf16, 0, c, D) : Row8{};
            const Row8 t = a.gate ? load8<VEC, true>(a.gate, a.gate_bf16, grow, c, D) : Row8{};
            r[i] = widen<VEC>(rx[i], 1);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                float z = y[i].v[q] * f;
                if (a.post) z *= p.v[q];
                if (a.gate) z *= t.v[q];
                float v = __builtin_fmaf(a.alpha, r[i].v[q], z);
                const float border = __uint_as_float((__float_as_uint(v) & 0xffff0000u) | 0x8000u);
                if (!(fabsf(v - border) > __builtin_fmaf(fabsf(z), 4.1f * 0x1p-24f, fabsf(v) * (2.1f * 0x1p-24f)))) {
                    double w = (double)a.beta * iyw * (double)y[i].v[q];
                    if (a.post) w *= (double)p.v[q];
                    if (a.gate) w *= (double)t.v[q];
                    v = (float)((double)a.alpha * (double)r[i].v[q] + w);
                }
                r[i].v[q] = v;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (tid + i * TPR) * 8;
        if constexpr (!WIDE) {
#pragma unroll
            for (int q = 0; q < 8; ++q) r[i].v[q] *= a.alpha;
        }
        if (!WIDE && a.y) {
            Row8 z = y[i];
            if (a.post) {
                const Row8 p = load8<VEC, true>(a.post, a.w_bf16, 0, c, D);
#pragma unroll
                for (int q = 0; q < 8; ++q) z.v[q] = z.v[q] * iy * p.v[q];
            }
            if (a.gate) {
                const Row8 p = load8<VEC, true>(a.gate, a.gate_bf16, grow, c, D);
#pragma unroll
                for (int q = 0; q < 8; ++q) z.v[q] *= p.v[q];
            }
#pragma unroll
            for (int q = 0; q < 8; ++q) r[i].v[q] += a.beta * z.v[q];
        }
        // the norm is taken of the residual stream as it is stored, which is what
        // the next block and the gradient read
        if (WIDE || a.x_bf16) {
#pragma unroll
            for (int q = 0; q < 8; q += 2) {
                const unsigned w = pack_bf16(r[i].v[q], r[i].v[q + 1]);
                r[i].v[q] = __uint_as_float(w << 16), r[i].v[q + 1] = __uint_as_float(w & 0xffff0000u);
            }
        }
#pragma unroll
        for (int q = 0; q < 8; ++q) s += r[i].v[q] * r[i].v[q];
        // h is what the next block reads at once, r waits until that block is done:
        // it leaves the caches to h and to the inputs (8192 x 4096, a bf16 stream and
        // fp32 y: 63 -> 51 us alone; y written, this, h read, y written and the norm of
        // r and y: 245 -> 232; only where r is read at once does it cost: five norms in
        // a row 233 -> 250)
        if (VEC && a.r && a.h) store8_past(a.r, a.x_bf16, row, c, D, r[i]);
        else if (a.r) store8<VEC, true>(a.r, a.x_bf16, row, c, D, r[i]);
    }
    float ir = 1.0f;
    if (a.h) {
        ir = 1.0f / sqrtf(row_sum<TPR>(s, part[1]) / (float)D + a.eps);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (tid + i * TPR) * 8;
            const Row8 p = load8<VEC, true>(a.pre, a.w_bf16, 0, c, D);
#pragma unroll
            for (int q = 0; q < 8; ++q) r[i].v[q] = r[i].v[q] * ir * p.v[q];
            store8<VEC, true>(a.h, a.h_bf16, row, c, D, r[i]);
        }
    }
    if (a.stats && tid == 0) {
        a.stats[2 * row] = iy;
        a.stats[2 * row + 1] = ir;
    }
}

// With rhat = r rstd(r), a = dh pre, b = dz post, yhat = y rstd(y) (y without
// the post norm):
//   G = dr + rstd(r) (a - rhat mean(a rhat)),   dpre = sum_t dh rhat
//   dx = alpha G,  dgate = sum beta G yhat post,  dz = beta G gate
//   dy = rstd(y) (b - yhat mean(b yhat)),       dpost = sum_t dz yhat
// A workgroup takes a chunk of rows and keeps its columns' sums in registers;
// norm_fold_kernel adds the chunks' in order.
template <int TPR, int NV, bool VEC, int XB, int YB, int HB>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void block_norm_grad_kernel(NormArgs a) {
    constexpr int RPB = TPR < 256 ? 256 / TPR : 1;
    // types known at compile time, or (2) at run time
    const int xb = XB == 2 ? a.x_bf16 : XB, yb = YB == 2 ? a.y_bf16 : YB, hb = HB == 2 ? a.h_bf16 : HB;
    __shared__ float part[2][16];
    // two vectors of 1024 threads leave too few registers for every sum: the
    // weights' go to LDS, each slot its own thread's
    constexpr bool SL = TPR == 1024 && NV == 2;
    __shared__ float4 lsum[SL ? 4 * NV * TPR : 1];
    const long long chunk = (long long)blockIdx.x * RPB + threadIdx.x / TPR;
    if (RPB > 1 && chunk >= a.chunks) return;  // whole waves when TPR = 64 (no barrier then)
    const int tid = threadIdx.x % TPR, D = a.D;
    long long row, end;
    if (a.cpg > 0) {
        const long long grp = chunk / a.cpg, first = grp * a.gate_rows;
        row = first + (chunk - grp * a.cpg) * a.chunk_rows;
        end = min(min(row + a.chunk_rows, first + a.gate_rows), a.T);
    } else {
        row = chunk * a.chunk_rows;
        end = min(row + a.chunk_rows, a.T);
    }
    Row8 spre[SL ? 1 : NV], spost[SL ? 1 : NV], sgate[NV];
    // sums += t * u, which = 0: pre, 1: post
    auto slot = [&](int which, int i, int half) -> float4 & { return lsum[((which * NV + i) * 2 + half) * TPR + tid]; };
    auto add = [&](Row8 *reg, int which, int i, const Row8 &t, const Row8 &u) {
        if constexpr (SL) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float4 f = slot(which, i, half);
                f.x += t.v[4 * half] * u.v[4 * half], f.y += t.v[4 * half + 1] * u.v[4 * half + 1];
                f.z += t.v[4 * half + 2] * u.v[4 * half + 2], f.w += t.v[4 * half + 3] * u.v[4 * half + 3];
                slot(which, i, half) = f;
            }
        } else {
#pragma unroll
            for (int q = 0; q < 8; ++q) reg[i].v[q] += t.v[q] * u.v[q];
        }
    };
    auto total = [&](const Row8 *reg, int which, int i) -> Row8 {
        if constexpr (SL) {
            const float4 f = slot(which, i, 0), h = slot(which, i, 1);
            return Row8{{f.x, f.y, f.z, f.w, h.x, h.y, h.z, h.w}};
        } else {
            return reg[i];
        }
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        sgate[i] = Row8{};
        if constexpr (SL) {
#pragma unroll
            for (int j = 0; j < 4; ++j) slot(j >> 1, i, j & 1) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        } else {
            spre[i] = spost[i] = Row8{};
        }
    }
    // One vector per thread: the weights stay in registers over the rows, and
    // the next row's loads are in flight while a row is worked on.
    constexpr bool AHEAD = NV == 1 && !SL;
    struct RowData {
        Raw8 r[NV], h[NV], g[NV], y[NV];
        float iy, ir;
    };
    auto load_row = [&](long long rw, RowData &d) {
        d.iy = a.post ? a.stats[2 * rw] : 1.0f;
        d.ir = a.dh ? a.stats[2 * rw + 1] : 1.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (tid + i * TPR) * 8;
            if (!SL) {  // (SL: loaded where they are used, fewer registers live)
                d.r[i] = a.dh ? load_raw<VEC>(a.r, xb, rw, c, D) : Raw8{};
                d.h[i] = a.dh ? load_raw<VEC>(a.dh, hb, rw, c, D) : Raw8{};
                d.g[i] = a.dr ? load_raw<VEC>(a.dr, xb, rw, c, D) : Raw8{};
                d.y[i] = a.y ? load_raw<VEC>(a.y, yb, rw, c, D) : Raw8{};
            }
        }
    };
    Row8 kpre, kpost, kgate;  // AHEAD: the weights and the current gate row
    long long kgrow = -1;
    if constexpr (AHEAD) {
        if (a.dh) kpre = load8<VEC>(a.pre, a.w_bf16, 0, tid * 8, D);
        if (a.post) kpost = load8<VEC>(a.post, a.w_bf16, 0, tid * 8, D);
    }
    int turn = 0;  // the part of the next sum
    auto work = [&](RowData &d) {
        const float iy = d.iy, ir = d.ir;
        int wrow = 0;  // the weights' row; opaque where keeping them in registers over the rows would spill
        if constexpr (!AHEAD) asm volatile("" : "+s"(wrow));
        Row8 g[NV], y[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) g[i] = Row8{};
        if (a.dh) {
            Row8 rh[NV], t[NV];
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (tid + i * TPR) * 8;
                if constexpr (SL) {
                    d.r[i] = load_raw<VEC>(a.r, xb, row, c, D);
                    d.h[i] = load_raw<VEC>(a.dh, hb, row, c, D);
                }
                rh[i] = widen<VEC>(d.r[i], xb);
                t[i] = widen<VEC>(d.h[i], hb);
                const Row8 p = AHEAD ? kpre : load8<VEC>(a.pre, a.w_bf16, wrow, c, D);
#pragma unroll
                for (int q = 0; q < 8; ++q) rh[i].v[q] *= ir;
                add(spre, 0, i, t[i], rh[i]);
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    t[i].v[q] *= p.v[q];
                    s += t[i].v[q] * rh[i].v[q];
                }
            }
            s = row_sum<TPR>(s, part[turn]) / (float)D;
            turn ^= 1;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int q = 0; q < 8; ++q) g[i].v[q] = ir * (t[i].v[q] - rh[i].v[q] * s);
            if constexpr (SL) __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (tid + i * TPR) * 8;
            if constexpr (SL) {
                d.g[i] = a.dr ? load_raw<VEC>(a.dr, xb, row, c, D) : Raw8{};
                d.y[i] = a.y ? load_raw<VEC>(a.y, yb, row, c, D) : Raw8{};
            }
            const Row8 o = widen<VEC>(d.g[i], xb);
#pragma unroll
            for (int q = 0; q < 8; ++q) g[i].v[q] += o.v[q];
            y[i] = widen<VEC>(d.y[i], yb);
        }
        const long long grow = a.gate ? row / a.gate_rows : 0;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (tid + i * TPR) * 8;
            if (a.dx) {
                Row8 o;
#pragma unroll
                for (int q = 0; q < 8; ++q) o.v[q] = a.alpha * g[i].v[q];
                store8<VEC>(a.dx, xb, row, c, D, o);
            }
            if (a.y) {
                Row8 po;
                if (a.post) {
                    po = AHEAD ? kpost : load8<VEC>(a.post, a.w_bf16, wrow, c, D);
#pragma unroll
                    for (int q = 0; q < 8; ++q) y[i].v[q] *= iy;  // yhat
                }
#pragma unroll
                for (int q = 0; q < 8; ++q) g[i].v[q] *= a.beta;
                if (a.gate) {
                    Row8 gt;
                    if constexpr (AHEAD) {
                        if (grow != kgrow) kgate = load8<VEC>(a.gate, a.gate_bf16, grow, c, D);
                        kgrow = grow;
                        gt = kgate;
                    } else {
                        gt = load8<VEC>(a.gate, a.gate_bf16, grow, c, D);
                    }
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        sgate[i].v[q] += g[i].v[q] * (a.post ? y[i].v[q] * po.v[q] : y[i].v[q]);
                        g[i].v[q] *= gt.v[q];
                    }
                }
                if (a.post) {
                    add(spost, 1, i, g[i], y[i]);
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        g[i].v[q] *= po.v[q];
                        s += g[i].v[q] * y[i].v[q];
                    }
                }
            }
        }
        if (a.y && a.post) {
            s = row_sum<TPR>(s, part[turn]) / (float)D;
            turn ^= 1;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int q = 0; q < 8; ++q) g[i].v[q] = iy * (g[i].v[q] - y[i].v[q] * s);
        }
        if (a.y && a.dy) {
#pragma unroll
            for (int i = 0; i < NV; ++i) store8<VEC>(a.dy, yb, row, (tid + i * TPR) * 8, D, g[i]);
        }
        // a gate row that ends inside the chunk is complete
        if (a.dgate && a.cpg == 0 && (row + 1 == a.T || (row + 1) % a.gate_rows == 0)) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                store8<VEC>(a.dgate, 0, grow, (tid + i * TPR) * 8, D, sgate[i]);
#pragma unroll
                for (int q = 0; q < 8; ++q) sgate[i].v[q] = 0.0f;
            }
        }
    };
    RowData even, odd;
    if constexpr (AHEAD) {
        if (row < end) load_row(row, even);
        while (row < end) {
            if (row + 1 < end) load_row(row + 1, odd);
            work(even);
            if (++row >= end) break;
            if (row + 1 < end) load_row(row + 1, even);
            work(odd);
            ++row;
        }
    } else {
        for (; row < end; ++row) {
            load_row(row, even);
            work(even);
        }
    }
    // partial sums: [pre | post | gate][chunk][D]
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (tid + i * TPR) * 8;
        if (a.dpre) store8<VEC>(a.ws, 0, chunk, c, D, total(spre, 0, i));
        if (a.dpost) store8<VEC>(a.ws, 0, a.chunks + chunk, c, D, total(spost, 1, i));
        if (a.dgate && a.cpg > 0) store8<VEC>(a.ws, 0, 2 * a.chunks + chunk, c, D, sgate[i]);
    }
}

// Adds the chunks' sums in a fixed order: 64 columns per workgroup, 16 slices
// of the chunks.  blockIdx.y: 0 dpre, 1 dpost, 2 + g gate row g.
__global__ __launch_bounds__(1024) void norm_fold_kernel(NormArgs a) {
    __shared__ float part[16][64];
    const int what = blockIdx.y;
    float *out = what == 0 ? a.dpre : (what == 1 ? a.dpost : a.dgate + (long long)(what - 2) * a.D);
    if ((what == 0 && !a.dpre) || (what == 1 && !a.dpost)) return;
    const long long first = what < 2 ? what * a.chunks : 2 * a.chunks + (what - 2) * a.cpg;
    const long long n = what < 2 ? a.chunks : a.cpg;
    const int col = blockIdx.x * 64 + (threadIdx.x & 63), sl = threadIdx.x >> 6;
    float v = 0.0f;
    if (col < a.D) {
        const float *p = a.ws + first * a.D + col;
        long long i = sl;
        for (; i + 7 * 16 < n; i += 8 * 16) {  // eight loads in flight
            float w[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) w[q] = p[(i + q * 16) * a.D];
#pragma unroll
            for (int q = 0; q < 8; ++q) v += w[q];
        }
        for (; i < n; i += 16) v += p[i * a.D];
    }
    part[sl][threadIdx.x & 63] = v;
    __syncthreads();
    if (sl == 0 && col < a.D) {
#pragma unroll
        for (int i = 1; i < 16; ++i) v += part[i][threadIdx.x];
        out[col] = v;
    }
}

}  // namespace ops

// Waves per row of the gradient kernel for D channels.
static int norm_grad_threads(int D) {
    return D <= 512 ? 64 : (D <= 2048 ? 256 : (D <= 8192 ? 512 : 1024));
}

// Chunks of the gradient's rows: about eight waves per CU, at least four rows
// each (their sums are written once per chunk); a few thousand at most, whatever T.
static void norm_chunks(long long T, int D, long long gate_rows, long long &chunk_rows, long long &cpg,
                        long long &chunks) {
    const long long target = 2048 / (norm_grad_threads(D) / 64);
    long long R = (T + target - 1) / target;
    if (R < 4) R = 4;
    cpg = 0;
    if (gate_rows > 0 && gate_rows <= R) {
        chunk_rows = R / gate_rows * gate_rows;  // whole gate rows
        chunks = (T + chunk_rows - 1) / chunk_rows;
    } else {
        const long long per = gate_rows > 0 ? gate_rows : T, groups = (T + per - 1) / per;
        chunk_rows = R < per ? R : per;
        cpg = (per + chunk_rows - 1) / chunk_rows;
        chunks = groups * cpg;
    }
}

long long norm_workspace_floats(long long T, int D, long long gate_rows) {
    long long r, c, n;
    if (gate_rows > T) gate_rows = T;
    norm_chunks(T, D, gate_rows, r, c, n);
    return 3 * n * D;
}

#define MOE_NORM(N, TPR, ...)                                                            \
    {                                                                                    \
        const long long rpb = TPR < 256 ? 256 / TPR : 1, blocks = ((N) + rpb - 1) / rpb; \
        __VA_ARGS__<<<op_row_grid(blocks), TPR < 256 ? 256 : TPR, 0, s>>>(a);            \
    }
template <bool VEC, bool WIDE>
static hipError_t norm_launch(const NormArgs &a, hipStream_t s) {
    using namespace ops;
    if (a.D <= 512) MOE_NORM(a.T, 64, block_norm_kernel<64, 1, VEC, WIDE>)
    else if (a.D <= 2048) MOE_NORM(a.T, 256, block_norm_kernel<256, 1, VEC, WIDE>)
    else if (a.D <= 4096) MOE_NORM(a.T, 256, block_norm_kernel<256, 2, VEC, WIDE>)
    else if (a.D <= 8192) MOE_NORM(a.T, 1024, block_norm_kernel<1024, 1, VEC, WIDE>)
    else MOE_NORM(a.T, 1024, block_norm_kernel<1024, 2, VEC, WIDE>)
    return hipGetLastError();
}
template <bool VEC, int XB, int YB, int HB>
static hipError_t norm_grad_launch(const NormArgs &a, hipStream_t s) {
    using namespace ops;
    if (a.D <= 512) MOE_NORM(a.chunks, 64, block_norm_grad_kernel<64, 1, VEC, XB, YB, HB>)
    else if (a.D <= 2048) MOE_NORM(a.chunks, 256, block_norm_grad_kernel<256, 1, VEC, XB, YB, HB>)
    else if (a.D <= 4096) MOE_NORM(a.chunks, 512, block_norm_grad_kernel<512, 1, VEC, XB, YB, HB>)
    else if (a.D <= 8192) MOE_NORM(a.chunks, 512, block_norm_grad_kernel<512, 2, VEC, XB, YB, HB>)
    else MOE_NORM(a.chunks, 1024, block_norm_grad_kernel<1024, 2, VEC, XB, YB, HB>)
    return hipGetLastError();
}
#undef MOE_NORM

// whole 16-byte vectors in every tensor of the call
static bool norm_vec(const NormArgs &a) {
    if (a.D & 7) return false;
    for (const void *p : {a.x, a.y, a.pre, a.post, a.gate, (const void *)a.r, (const void *)a.h, a.dr, a.dh,
                          (const void *)a.dx, (const void *)a.dy, (const void *)a.dgate, (const void *)a.ws})
        if ((uintptr_t)p & 15) return false;
    return true;
}
static hipError_t norm_run(const NormArgs &a, bool grad, hipStream_t s) {
    if (!grad) {
        const bool wide = a.x_bf16 && a.y && (a.post || a.gate);
        if (wide) return norm_vec(a) ? norm_launch<true, true>(a, s) : norm_launch<false, true>(a, s);
        return norm_vec(a) ? norm_launch<true, false>(a, s) : norm_launch<false, false>(a, s);
    }
    if (!norm_vec(a)) return norm_grad_launch<false, 2, 2, 2>(a, s);
    // the gradient is bound by its instructions as much as by its bytes: types
    // known at compile time, and the weights and the next row held in registers
    // (8192 x 4096, bf16 stream, fp32 y: 152 -> 114 us)
    switch ((a.x_bf16 ? 4 : 0) | (a.y_bf16 ? 2 : 0) | (a.h_bf16 ? 1 : 0)) {
    case 0: return norm_grad_launch<true, 0, 0, 0>(a, s);
    case 1: return norm_grad_launch<true, 0, 0, 1>(a, s);
    case 2: return norm_grad_launch<true, 0, 1, 0>(a, s);
    case 3: return norm_grad_launch<true, 0, 1, 1>(a, s);
    case 4: return norm_grad_launch<true, 1, 0, 0>(a, s);
    case 5: return norm_grad_launch<true, 1, 0, 1>(a, s);
    case 6: return norm_grad_launch<true, 1, 1, 0>(a, s);
    default: return norm_grad_launch<true, 1, 1, 1>(a, s);
    }
}

hipError_t launch_block_norm(const NormArgs &a, hipStream_t s) {
    if (a.T <= 0) return hipSuccess;
    if (a.D < 1 || a.D > kMaxNormDim) return hipErrorInvalidValue;
    return norm_run(a, false, s);
}

hipError_t launch_block_norm_grad(NormArgs a, hipStream_t s) {
    if (a.D < 1 || a.D > kMaxNormDim) return hipErrorInvalidValue;
    if (a.gate && a.gate_rows > a.T) a.gate_rows = a.T;
    long long gr = a.gate ? a.gate_rows : 0;
    if (a.T > 0) {
        norm_chunks(a.T, a.D, gr, a.chunk_rows, a.cpg, a.chunks);
        if (gr == 0) a.gate_rows = a.T;  // the chunks' one group
        hipError_t e = norm_run(a, true, s);
        if (e != hipSuccess) return e;
    } else {
        a.chunks = a.cpg = 0;  // no rows: the weights' gradients are zeros
    }
    const long long gates = a.dgate && a.cpg > 0 ? (a.T + a.gate_rows - 1) / a.gate_rows : 0;
    if (!a.dpre && !a.dpost && gates == 0) return hipSuccess;
    if (gates > 65000) return kOpTooLarge;  // (a few thousand at most: norm_chunks)
    ops::norm_fold_kernel<<<dim3((a.D + 63) / 64, (unsigned)(2 + gates)), 1024, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace moe
