// moe_ops_gate.h -- the gate of a gated feed-forward block, h = act(a) b, and
// its gradients: da = dh b act'(a), db = dh act(a).
//
//   silu, gelu: act = a s, s = 1 / (1 + e^-z), z = r (a + c a^3); silu: r = 1, c = 0;
//     gelu: r = 2 sqrt(2 / pi), c = 0.044715 (its tanh form: 0.5 (1 + tanh(z / 2)) = s);
//     act' = s + a s (1 - s) r (1 + 3 c a^2)
//   relu, identity: act = a, act' = 1 but where a <= floor: 0; floor = 0 or NaN
// so that a kernel holds two forms, not four.  (With a four-way choice by the activation
// around a tile's results one value of 16 was wrong for the identity; why was not found out.)
#pragma once
#include <type_traits>

#include "moe_internal.h"
#include "moe_ops.h"

namespace moe {
namespace ops {

// FAST: the hardware's exp and reciprocal, for results that are rounded to bf16.  e^-z is
// 2^(-z log2 e) there, whose rounded exponent costs some 2^-24 |z| of it: act is off by up to
// 57 * 2^-24 of itself for |z| up to 80 (2.6 * 2^-24 otherwise), a 1000th of a bf16 half step.
// Else expf and an IEEE division: the forward product of 8192 rows, one bf16 expert of 4096 /
// 14336, fp32 result, 1580 us, 1530 with the hardware's.
template <bool FAST>
__device__ __forceinline__ float gate_sigmoid(float z) {
    if constexpr (FAST) return __builtin_amdgcn_rcpf(1.0f + __expf(-z));
    else return 1.0f / (1.0f + expf(-z));
}

struct GateValue {
    float f, d;  // act(a), act'(a)
};

struct Gate {
    float r, c, floor;
    bool smooth;
    __device__ __forceinline__ explicit Gate(int act)
        : r(act == MOE_ACT_GELU ? 1.5957691216057308f : 1.0f), c(act == MOE_ACT_GELU ? 0.044715f : 0.0f),
          floor(act == MOE_ACT_RELU ? 0.0f : __builtin_nanf("")), smooth(act == MOE_ACT_SILU || act == MOE_ACT_GELU) {}

    template <bool SMOOTH, bool FAST>
    __device__ __forceinline__ GateValue value(float a) const {
        if constexpr (SMOOTH) {
            // past |a| = 32 gelu's s is 0 or 1 in 32 bits: the powers of a stop there, where
            // they could overflow (and 0 times infinity would be NaN)
            const float q = __builtin_amdgcn_fmed3f(a, -32.0f, 32.0f), q2 = q * q;
            const float s = gate_sigmoid<FAST>(r * (a + c * q2 * q)), f = a * s;
            // (an infinite f, where 1 - s is 0, is kept from being NaN; a NaN, at a = -infinity
            // too, stays one, which fminf would not let it)
            const float most = f > 3e38f ? 3e38f : f;
            return {f, s + most * (1.0f - s) * (r * (1.0f + 3.0f * c * q2))};
        } else {
            const bool zero = a <= floor;
            return {zero ? 0.0f : a, zero ? 0.0f : 1.0f};
        }
    }
};

// f(SMOOTH, FAST) of the gate's form; f32: results that stay in 32 bits.
template <bool BF16, typename F>
__device__ __forceinline__ void gate_form(const Gate &gate, bool f32, F f) {
    if (!gate.smooth) {
        f(std::false_type{}, std::false_type{});
    } else if constexpr (BF16) {
        if (f32) f(std::true_type{}, std::false_type{});
        else f(std::true_type{}, std::true_type{});
    } else {
        f(std::true_type{}, std::false_type{});
    }
}

struct GateBack {
    float da, db, h;
};
template <bool SMOOTH, bool FAST>
__device__ __forceinline__ GateBack gate_back(const Gate &g, float dh, float a, float b) {
    const GateValue v = g.value<SMOOTH, FAST>(a);
    return {dh * b * v.d, dh * v.f, v.f * b};
}

// CE elements of a row from column n on, N its columns: 16 bytes at any alignment,
// element by element past the end.  Raw: as they are in memory.
struct GateRaw {
    uint4 u;
};
template <bool BF16>
__device__ __forceinline__ GateRaw gate_load(const void *row, int n, int N) {
    constexpr int CE = BF16 ? 8 : 4, ES = BF16 ? 2 : 4;
    GateRaw r;
    if (n + CE <= N) {
        __builtin_memcpy(&r.u, (const uint8_t *)row + (long long)n * ES, 16);
    } else {
        unsigned w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int q = 0; q < CE; ++q) {
            if (n + q >= N) continue;
            if constexpr (BF16) w[q / 2] |= (unsigned)((const uint16_t *)row)[n + q] << (16 * (q & 1));
            else w[q] = ((const unsigned *)row)[n + q];
        }
        r.u = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return r;
}
template <bool BF16>
struct GateChunk {
    static constexpr int CE = BF16 ? 8 : 4;
    float v[CE];
    __device__ __forceinline__ GateChunk() {}
    __device__ __forceinline__ explicit GateChunk(const GateRaw &r) {
        const unsigned w[4] = {r.u.x, r.u.y, r.u.z, r.u.w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if constexpr (BF16) {
                v[2 * q] = __uint_as_float(w[q] << 16);
                v[2 * q + 1] = __uint_as_float(w[q] & 0xffff0000u);
            } else {
                v[q] = __uint_as_float(w[q]);
            }
        }
    }
    // PAST: around the caches
    template <bool PAST>
    __device__ __forceinline__ void store(void *row, int n, int N) const {
        typedef unsigned u32x4_u __attribute__((ext_vector_type(4), aligned(2)));
        auto put = [&](auto &whole, void *at) {
            const u32x4_u t = __builtin_bit_cast(u32x4_u, whole);
            if constexpr (PAST) __builtin_nontemporal_store(t, (u32x4_u *)at);
            else *(u32x4_u *)at = t;
        };
        if constexpr (BF16) {
            typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
            bf16x8 o;
#pragma unroll
            for (int q = 0; q < CE; ++q) o[q] = (__bf16)v[q];
            if (n + CE <= N) {
                put(o, (uint16_t *)row + n);
            } else {
#pragma unroll
                for (int q = 0; q < CE; ++q)
                    if (n + q < N) ((uint16_t *)row)[n + q] = f32_to_bf16(v[q]);
            }
        } else {
            if (n + CE <= N) {
                put(v, (float *)row + n);
            } else {
#pragma unroll
                for (int q = 0; q < CE; ++q)
                    if (n + q < N) ((float *)row)[n + q] = v[q];
            }
        }
    }
};

// The pre-activations at a chunk of row `row`.
template <bool BF16>
__device__ __forceinline__ void gate_load_ab(const OpGemmArgs &g, long long row, int n, GateRaw &a, GateRaw &b) {
    constexpr int ES = BF16 ? 2 : 4;
    a = gate_load<BF16>((const uint8_t *)g.ga + row * g.ldga * ES, n, g.N);
    b = gate_load<BF16>((const uint8_t *)g.gb + row * g.ldgb * ES, n, g.N);
}
// da, db and h there from dh.
template <bool BF16, bool PAST = false>
__device__ __forceinline__ void gate_store(const OpGemmArgs &g, long long row, int n, const GateChunk<BF16> &dh,
                                           const GateRaw &ra, const GateRaw &rb) {
    constexpr int ES = BF16 ? 2 : 4;
    const GateChunk<BF16> a(ra), b(rb);
    GateChunk<BF16> da, db, h;
    const Gate gate(g.act);
    gate_form<BF16>(gate, !BF16, [&](auto SMOOTH, auto FAST) {
#pragma unroll
        for (int q = 0; q < GateChunk<BF16>::CE; ++q) {
            const GateBack r = gate_back<decltype(SMOOTH)::value, decltype(FAST)::value>(gate, dh.v[q], a.v[q], b.v[q]);
            da.v[q] = r.da, db.v[q] = r.db, h.v[q] = r.h;
        }
    });
    da.template store<PAST>((uint8_t *)g.C + row * g.ldc * ES, n, g.N);
    db.template store<PAST>((uint8_t *)g.C2 + row * g.ldc2 * ES, n, g.N);
    h.template store<PAST>((uint8_t *)g.C3 + row * g.ldc3 * ES, n, g.N);
}

}  // namespace ops
}  // namespace moe
