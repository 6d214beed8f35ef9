// moe_ops_gemm.h -- grouped products on a caller's own row-major tensors: no
// packing, any strides, groups of any length whose bounds stay on the device.
//
// Per group C = A B^T with fp32 (int8: int32) sums.  The three products of a
// linear layer are one kernel with three operand orders (OpGemmArgs):
//   forward / row gradient: A "row", B "row" or "col" by the weight's layout;
//   weight gradient: A and B "col", k running over the group's rows.
//
// LDS.  A stage is KSUB pieces of 64 bytes of k per "row" operand row (32 bf16,
// 16 fp32, 64 int8) and the same number of k rows of a "col" operand.  KSUB is 2
// where an operand is "row", so that whole 128-byte lines are read (8192 rows,
// 8 bf16 experts of 4096 / 14336: 902 us, 954 at 1), else 1.  A lane's fragment
// is 16 bytes of consecutive k of one row for every type, so one loop serves
// bf16 (one MFMA per fragment pair), int8 (one) and fp32 (four, element j of
// each lane's four: the k order inside a fragment is free as long as both
// operands use the same).
//   row operand: row r's 16-byte chunk c at slot c ^ (-(r >> 2) & 3), KSUB 2: c ^
//     ((r >> 1) & 7): the sixteen lanes that a ds_read_b128 serves at a time
//     (rows 0-3 and 12-15 of one k group, 4-7 and 8-11 of the next) lie in all 64
//     banks once;
//   col operand: k row kr, its 16-element unit u at unit u ^ col_swz(kr).
//     bf16 fragments come through ds_read_b64_tr_b16 (16 lanes read 4 k rows
//     x 16 columns and each receives one column), fp32 ones through four
//     ds_read_b32.
#pragma once
#include <type_traits>

#include "moe_internal.h"
#include "moe_ops.h"

namespace moe {
namespace ops {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) uint8_t lds_u8;

template <int N>
using num = std::integral_constant<int, N>;

template <int OT>
using acc_t = std::conditional_t<OT == OT_I8, i32x4, f32x4>;

template <int OT>
using acc_elem = std::conditional_t<OT == OT_I8, int, float>;

template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// One 16-byte fragment pair into the 16 x 16 block: rows of `b` become the
// block's rows (4 (lane / 16) + c), rows of `a` its columns (lane % 16).
template <int OT>
__device__ __forceinline__ acc_t<OT> fma16(const u32x4 &b, const u32x4 &a, acc_t<OT> c) {
    if constexpr (OT == OT_BF16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, b),
                                                       __builtin_bit_cast(bf16x8_t, a), c, 0, 0, 0);
    } else if constexpr (OT == OT_I8) {
        return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, b), __builtin_bit_cast(i32x4, a), c, 0,
                                                     0, 0);
    } else {
        const f32x4 fb = __builtin_bit_cast(f32x4, b), fa = __builtin_bit_cast(f32x4, a);
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[j], fa[j], c, 0, 0, 0);
        return c;
    }
}

// 16 bytes at p of which the first n elements exist (the others read as 0).
// p need only have the element's alignment.
template <int ES>
__device__ __forceinline__ u32x4 load_chunk(const uint8_t *p, int n) {
    constexpr int CE = 16 / ES;
    u32x4 v = {0u, 0u, 0u, 0u};
    if (n >= CE) {
        __builtin_memcpy(&v, p, 16);
    } else if (n > 0) {
        // element by element into a 128-bit value (no indexed register array)
        unsigned long long lo = 0, hi = 0;
#pragma unroll
        for (int i = 0; i < CE; ++i) {
            unsigned long long x = 0;
            if (i < n) {
                if constexpr (ES == 4) x = *(const uint32_t *)(p + 4 * i);
                else if constexpr (ES == 2) x = *(const uint16_t *)(p + 2 * i);
                else x = p[i];
            }
            if (i * ES < 8) lo |= x << (8 * (i * ES)); else hi |= x << (8 * (i * ES - 8));
        }
        v = u32x4{(unsigned)lo, (unsigned)(lo >> 32), (unsigned)hi, (unsigned)(hi >> 32)};
    }
    return v;
}

// Unit swizzle of a "col" operand's k row: the fragment reads of half a wave
// (8 k rows x 32 bytes, bf16; 4 k rows x 64 bytes per instruction, fp32) fall
// into different banks.  NU: 16-element units per k row.
template <int ES, int NU>
__device__ __forceinline__ int col_swz(int kr) {
    if constexpr (ES == 2) {
        if constexpr (NU >= 8) return (kr & 3) | (((kr >> 3) & 1) << 2);
        else if constexpr (NU == 4) return ((kr >> 1) & 1) | (((kr >> 3) & 1) << 1);
        else return (kr >> 3) & 1;
    } else {
        return (kr >> 2) & (NU >= 4 ? 3 : NU - 1);
    }
}

constexpr unsigned kOutOfRange = 0x80000000u;  // past every buffer's num_records: reads as 0

// One operand's tile of ROWS rows: its LDS stage image and how NT threads fill
// it.  VB 16 or 4: by buffer loads of 16 bytes a lane straight into LDS, a lane
// whose bytes lie outside reads zeros by the buffer's own range check.  16: rows
// of whole, aligned chunks.  4: rows of whole, aligned dwords (fp32: any; at least
// a chunk apart), whose last chunk may hold elements of the next row: of a "col" operand they only
// reach results that are not stored, and the next row is there except in the
// last stage; of a "row" operand they would be summed.  Such a last stage is
// loaded by dwords (weight gradient, 12 groups of 259 rows: fp32, 1001 / 2731, 169 us,
// by dwords alone 210; bf16, 1002 / 2730, 47 us, through registers 75).  VB 0: through registers, any alignment.
template <int ES, int ROWS, bool COL, int NT, int KSUB, int VB>
struct Tile {
    static constexpr bool DIRECT = VB > 0;
    static_assert(VB == 0 || VB == 16 || VB == 4, "alignment of the rows");
    static constexpr int CE = 16 / ES;           // elements per chunk
    static constexpr int KE = KSUB * 64 / ES;     // k per stage
    static constexpr int NC = KSUB * ROWS * 4 / NT;  // chunks per thread
    static constexpr int ROWB = COL ? ROWS * ES : 64 * KSUB;
    static constexpr int CPR = ROWB / 16;        // chunks per LDS row
    static constexpr int NU = ROWS / 16;         // 16-element units per k row (COL)
    static constexpr int UC = ES;                // chunks per unit
    static constexpr int BYTES = ROWS * 64 * KSUB;
    static_assert(NC >= 1 && KSUB * ROWS * 4 % NT == 0, "threads cover the tile");

    const uint8_t *base;  // element (row 0, first k) of the tile
    long long ldb;        // bytes between rows (COL: between k)
    int lim;              // valid rows (COL: valid elements of a k row)
    int klen;             // k range
    unsigned base_lo, base_hi;  // DIRECT: base, in scalar registers
    unsigned voff[DIRECT ? NC : 1];
    u32x4 reg[DIRECT ? 1 : NC];

    static __device__ __forceinline__ int row_swz(int row) {
        return KSUB == 2 ? (row >> 1) & 7 : -(row >> 2) & 3;
    }
    // chunk i of the image -> its LDS row and source chunk within the row
    static __device__ __forceinline__ void place(int i, int &row, int &chunk) {
        row = i / CPR;
        const int q = i % CPR;
        if constexpr (COL) chunk = (((q / UC) ^ col_swz<ES, NU>(row)) * UC) + q % UC;
        else chunk = q ^ row_swz(row);
    }
    // DIRECT: wave w's load j fills the 1 KB from chunk (j NW + w) 64
    static __device__ __forceinline__ int chunk_of(int j) { return j * NT + (int)threadIdx.x; }

    // load j of this thread: its LDS row and its first element within the row
    static __device__ __forceinline__ void place_load(int j, int &row, int &elem) {
        int chunk;
        place(chunk_of(j), row, chunk);
        elem = chunk * CE;
    }
    // a stage whose last chunks may not be read whole (krem: what is left of k)
    __device__ __forceinline__ bool part_chunks(int krem) const {
        if constexpr (COL) return krem > 0 && krem <= KE && lim < ROWS && lim % CE != 0;
        else return krem > 0 && krem < KE && krem % CE != 0;
    }
    // such a stage, by dwords
    __device__ __forceinline__ void load_dwords(const u32x4 &rs, int krem, unsigned lds, int w) const {
        constexpr int STEP = NT * 4, DE = 4 / ES;  // elements per dword
        const unsigned m0 = __builtin_amdgcn_readfirstlane(lds + w * 256);
#pragma unroll
        for (int j = 0; j < 4 * NC; j += 4) {
            unsigned v[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int i = (j + q) * NT + (int)threadIdx.x;
                int row, chunk;
                place(i / 4, row, chunk);
                const int elem = chunk * CE + i % 4 * DE;
                const bool ok = COL ? elem < lim && row < krem : row < lim && elem < krem;
                v[q] = ok ? (unsigned)(row * (int)ldb + elem * ES) : kOutOfRange;
            }
            asm volatile(
                "s_nop 4\n\ts_mov_b32 m0, %5\n\ts_nop 0\n\tbuffer_load_dword %0, %4, 0 offen lds\n\t"
                "s_add_u32 m0, m0, %6\n\ts_nop 0\n\tbuffer_load_dword %1, %4, 0 offen lds\n\t"
                "s_add_u32 m0, m0, %6\n\ts_nop 0\n\tbuffer_load_dword %2, %4, 0 offen lds\n\t"
                "s_add_u32 m0, m0, %6\n\ts_nop 0\n\tbuffer_load_dword %3, %4, 0 offen lds" ::"v"(v[0]),
                "v"(v[1]), "v"(v[2]), "v"(v[3]), "s"(rs), "s"(m0 + j * STEP), "n"(STEP)
                : "m0", "scc");
        }
    }

    __device__ __forceinline__ void init(const uint8_t *b, long long ld_bytes, int limit, int k) {
        base = b;
        ldb = ld_bytes;
        lim = limit;
        klen = k;
        if constexpr (DIRECT) {
            base_lo = __builtin_amdgcn_readfirstlane((unsigned)(unsigned long long)b);
            base_hi = __builtin_amdgcn_readfirstlane((unsigned)((unsigned long long)b >> 32));
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                int row, elem;
                place_load(j, row, elem);
                const bool ok = COL ? elem < lim : row < lim;
                voff[j] = ok ? (unsigned)(row * (int)ldb + elem * ES) : kOutOfRange;
            }
        }
    }
    // Stage s straight into the LDS image at byte offset lds (DIRECT).  Inline
    // assembly that the compiler does not see as a memory access: its wait
    // insertion would otherwise make every later LDS read wait for all loads in
    // flight.  Order is kept by the kernel's own waits and barriers.  The
    // compiler's hazard handling does not look inside either: a VMEM
    // instruction needs five wait states after a VALU instruction
    // (v_readfirstlane) wrote a scalar register that it reads, one after a
    // scalar write of M0.
    __device__ __forceinline__ void load_lds(int s, unsigned lds, int w) const {
        const int k0 = s * KE;
        const unsigned long long a =
            ((unsigned long long)base_hi << 32 | base_lo) + (COL ? (long long)k0 * ldb : (long long)k0 * ES);
        u32x4 rs;
        rs[0] = __builtin_amdgcn_readfirstlane((unsigned)a);
        rs[1] = __builtin_amdgcn_readfirstlane((unsigned)(a >> 32) & 0xffffu);
        rs[2] = 0x7fffffffu;
        rs[3] = 0x00027000u;
        const int krem = klen - k0;
        if constexpr (VB == 4) {
            if (part_chunks(krem)) {
                load_dwords(rs, krem, lds, w);
                return;
            }
        }
        unsigned v[NC];
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            v[j] = voff[j];
            if (krem < KE) {  // the last stage: what lies past the k range reads as 0
                int row, elem;
                place_load(j, row, elem);
                if (COL ? row >= krem : elem >= krem) v[j] = kOutOfRange;
            }
        }
        const unsigned m0 = __builtin_amdgcn_readfirstlane(lds + w * 1024);
        constexpr int STEP = NT * 16;  // LDS bytes between a thread's loads
        if constexpr (NC == 1) {
            asm volatile("s_nop 4\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(v[0]),
                         "s"(rs), "s"(m0)
                         : "m0");
        } else if constexpr (NC == 2) {
            asm volatile(
                "s_nop 4\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %2, 0 offen lds\n\t"
                "s_add_u32 m0, m0, %4\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"v"(v[0]),
                "v"(v[1]), "s"(rs), "s"(m0), "n"(STEP)
                : "m0", "scc");
        } else {
            static_assert(NC <= 4 && NC != 3, "loads per thread");
            asm volatile(
                "s_nop 4\n\ts_mov_b32 m0, %5\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %4, 0 offen lds\n\t"
                "s_add_u32 m0, m0, %6\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %4, 0 offen lds\n\t"
                "s_add_u32 m0, m0, %6\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %4, 0 offen lds\n\t"
                "s_add_u32 m0, m0, %6\n\ts_nop 0\n\tbuffer_load_dwordx4 %3, %4, 0 offen lds" ::"v"(v[0]),
                "v"(v[1]), "v"(v[NC > 2 ? 2 : 0]), "v"(v[NC > 3 ? 3 : 0]), "s"(rs), "s"(m0), "n"(STEP)
                : "m0", "scc");
        }
    }
    // Stage s into registers.  Whole chunks are loaded without a branch, so that
    // they are in flight together: rows past the last one repeat it (their
    // products are not stored); chunks that cross an edge element by element.
    __device__ __forceinline__ void load_regs(int s) {
        const int k0 = s * KE, krem = klen - k0;
        const bool whole = krem >= KE && (!COL || lim >= ROWS);
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            int row, chunk;
            place(chunk_of(j), row, chunk);
            if (!COL) row = min(row, lim - 1);
            const uint8_t *p = COL ? base + (long long)(k0 + row) * ldb + chunk * 16
                                   : base + (long long)row * ldb + (long long)k0 * ES + chunk * 16;
            if (whole) {
                __builtin_memcpy(&reg[j], p, 16);
            } else {
                const int n = COL ? (row < krem ? lim - chunk * CE : 0) : krem - chunk * CE;
                reg[j] = load_chunk<ES>(p, n);
            }
        }
    }
    __device__ __forceinline__ void store_regs(lds_u8 *lds) const {
#pragma unroll
        for (int j = 0; j < NC; ++j)
            *(__attribute__((address_space(3))) u32x4 *)(lds + chunk_of(j) * 16) = reg[j];
    }

    // fragment of the 16 rows from 16 * blk, 64-byte piece ks of the stage
    static __device__ __forceinline__ u32x4 frag(const lds_u8 *lds, int blk, int ks, int lane) {
        const int r16 = lane & 15, q4 = lane >> 4;
        if constexpr (!COL) {
            const lds_u8 *p = lds + (blk * 16 + r16) * ROWB + (((ks * 4 + q4) ^ row_swz(r16)) << 4);
            return *(const __attribute__((address_space(3))) u32x4 *)p;
        } else if constexpr (ES == 2) {
            union { s16x4 h[2]; u32x4 v; } f;
            const int kr = ks * 32 + q4 * 8 + (r16 >> 2);
            const lds_u8 *p = lds + kr * ROWB + (blk ^ col_swz<ES, NU>(kr)) * 32 + (r16 & 3) * 8;
            const lds_u8 *p1 = p + 4 * ROWB;  // k rows kr + 4: bit 2 of kr is clear and not part of the swizzle
            f.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)p);
            f.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)p1);
            return f.v;
        } else {
            u32x4 v;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int kr = ks * 16 + q4 * 4 + j;
                const lds_u8 *p = lds + kr * ROWB + (blk ^ col_swz<ES, NU>(kr)) * 64 + r16 * 4;
                v[j] = *(const __attribute__((address_space(3))) unsigned *)p;
            }
            return v;
        }
    }
    static constexpr int READS = !COL ? 1 : (ES == 2 ? 2 : 4);  // LDS reads per fragment
};

// ---- work list -------------------------------------------------------------------
struct OpJob {
    int e;         // group
    int m0, n0;    // tile origin (ragged rows: m0 counted from the group's first row)
    int lo, len;   // the group's first row and rows
    int ks;        // range of k (of g.splits)
};

// M tiles per block of the order (block, n tile, M tile): a group of many M
// tiles re-reads neither its rows for every n tile nor its matrix for every M tile.
constexpr int kOpMBlock = 8;

// Item `item` of the tiles of all groups, group-major; false past the last.
// Every wave scans the groups' lengths, 64 groups at a time.
template <int BM>
__device__ __forceinline__ bool ragged_job(const OpGemmArgs &g, OpJob &jb, int BN) {
    const int lane = threadIdx.x & 63, NT = g.nt;
    // tiles of the group of this lane, summed over the lanes up to it
    auto scan = [&](int base, int &lo, int &len) {
        lo = 0;
        len = 0;
        if (base + lane < g.E) {
            int hi;
            op_group(g.offsets, base + lane, g.rows, lo, hi);
            len = hi - lo;
        }
        int t = (len + BM - 1) / BM;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int u = __shfl_up(t, d);
            if (lane >= d) t += u;
        }
        return t;
    };
    int lo, len, W = 0, t = 0;
    for (int base = 0; base < g.E; base += 64) {
        t = scan(base, lo, len);
        W += __shfl(t, 63);
    }
    W *= NT * g.splits;
    // contiguous per-XCD ranges (block L runs on XCD L mod 8)
    const int per = (W + 7) >> 3, slot = blockIdx.x >> 3;
    int item = (blockIdx.x & 7) * per + slot;
    if (slot >= per || item >= W) return false;
    jb.ks = __builtin_amdgcn_readfirstlane(item % g.splits);
    item = __builtin_amdgcn_readfirstlane(item / g.splits);
    for (int base = 0; base < g.E; base += 64) {
        if (g.E > 64) t = scan(base, lo, len);
        const unsigned long long past = __ballot(t * NT > item);
        if (past) {
            const int src = __ffsll((long long)past) - 1;
            const int before = src > 0 ? __shfl(t, src - 1) : 0;
            const int nte = __shfl(t, src) - before;
            jb.e = base + src;
            jb.lo = __shfl(lo, src);
            jb.len = __shfl(len, src);
            item -= before * NT;
            int m, n;
            const int nfb = nte / kOpMBlock, infull = nfb * kOpMBlock * NT;
            if (item < infull) {
                const int b = item / (kOpMBlock * NT), q = item - b * (kOpMBlock * NT);
                n = q / kOpMBlock;
                m = b * kOpMBlock + (q - n * kOpMBlock);
            } else {
                const int ml = nte - nfb * kOpMBlock, q = item - infull;
                n = q / ml;
                m = nfb * kOpMBlock + (q - n * ml);
            }
            jb.m0 = __builtin_amdgcn_readfirstlane(m * BM);
            jb.n0 = __builtin_amdgcn_readfirstlane(n * BN);
            jb.e = __builtin_amdgcn_readfirstlane(jb.e);
            jb.lo = __builtin_amdgcn_readfirstlane(jb.lo);
            jb.len = __builtin_amdgcn_readfirstlane(jb.len);
            return true;
        }
        item -= __shfl(t, 63) * NT;
    }
    return false;
}

// The group of the r-th longest length (ties by index), with its rows.  Up to
// 512 groups, held eight to a lane: the length is found by bisection over the
// count of groups at least that long; more groups are taken in their order.
__device__ __forceinline__ int longest_group(const OpGemmArgs &g, int r, int &lo, int &hi) {
    int e = r;
    if (g.E > 1 && g.E <= 512) {
        const int lane = threadIdx.x & 63, n = (g.E + 63) >> 6;
        int len[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            len[q] = -1;
            if (q < n && q * 64 + lane < g.E) {
                int a, b;
                op_group(g.offsets, q * 64 + lane, g.rows, a, b);
                len[q] = b - a;
            }
        }
        auto count = [&](int t) {  // groups of at least t rows
            int c = 0;
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (q < n) c += __popcll(__ballot(len[q] >= t));
            return c;
        };
        int t = 0;
        for (int bit = 1 << (31 - __clz(g.rows | 1)); bit > 0; bit >>= 1)
            if (count(t | bit) > r) t |= bit;
        int skip = r - count(t + 1);  // among the groups of exactly t rows
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            if (q >= n) break;
            unsigned long long m = __ballot(len[q] == t);
            const int c = __popcll(m);
            if (skip >= 0 && skip < c) {
                for (int k = 0; k < skip; ++k) m &= m - 1;
                e = q * 64 + __ffsll((long long)m) - 1;
            }
            skip -= c;
        }
    }
    op_group(g.offsets, e, g.rows, lo, hi);
    return e;
}

// Weight gradient: tiles of the groups' matrices, the longest group first (a
// tile's time is its group's rows).  A group's tiles are dealt to the 8 XCDs
// in contiguous parts, so that every XCD has its share of every group: with
// whole groups per XCD one long group kept one XCD busy while the others were
// done (64 groups of 2048 x 1408 over 49152 rows, Zipf lengths: 1000 us).
// Within a group: ranges of its rows, blocks of kOpMBlock M tiles, n tile, M tile.
__device__ __forceinline__ bool matrix_job(const OpGemmArgs &g, OpJob &jb, int BM, int BN, int KE) {
    const int T = g.mt * g.nt * g.splits, part = (T + 7) >> 3;
    const int slot = blockIdx.x >> 3, r = slot / part;
    if (r >= g.E) return false;
    int item = (((int)blockIdx.x + r) & 7) * part + slot - r * part;
    if (item >= T) return false;
    int lo, hi;
    jb.e = __builtin_amdgcn_readfirstlane(longest_group(g, r, lo, hi));
    jb.ks = item / (g.mt * g.nt);
    item -= jb.ks * (g.mt * g.nt);
    const int nfb = g.mt / kOpMBlock, infull = nfb * kOpMBlock * g.nt;
    int m, n;
    if (item < infull) {
        const int b = item / (kOpMBlock * g.nt), q = item - b * (kOpMBlock * g.nt);
        n = q / kOpMBlock;
        m = b * kOpMBlock + (q - n * kOpMBlock);
    } else {
        const int ml = g.mt - nfb * kOpMBlock, q = item - infull;
        n = q / ml;
        m = nfb * kOpMBlock + (q - n * ml);
    }
    jb.m0 = m * BM;
    jb.n0 = n * BN;
    if (g.splits > 1) {  // equal ranges of whole stages
        const int chunk = ((hi - lo + g.splits - 1) / g.splits + KE - 1) / KE * KE;
        const int b = min(lo + jb.ks * chunk, hi);
        hi = min(b + chunk, hi);
        lo = b;
    }
    jb.lo = __builtin_amdgcn_readfirstlane(lo);
    jb.len = __builtin_amdgcn_readfirstlane(hi - lo);
    return true;
}

// Range ks of k, in whole stages of KE (the last ones may be empty).
__device__ __forceinline__ void k_range(const OpGemmArgs &g, int ks, int KE, int &k0, int &klen) {
    k0 = 0;
    klen = g.K;
    if (g.splits > 1) {
        const int chunk = ((g.K + g.splits - 1) / g.splits + KE - 1) / KE * KE;
        k0 = __builtin_amdgcn_readfirstlane(min(ks * chunk, g.K));
        klen = __builtin_amdgcn_readfirstlane(min(chunk, g.K - k0));
    }
}

// ---- results ---------------------------------------------------------------------
// int8: a row's scale, applied before its channel's.  A sum, up to 2^31, times a
// scale past 2^96 or a subnormal one would overflow or lose bits where the
// channel's scale brings the result back, so such a scale is moved by 2^64 and
// the result moved back; a factor of 1 leaves every other result as it is.
struct RowScale {
    float s = 0.0f, back = 1.0f;
    __device__ __forceinline__ RowScale() {}
    __device__ __forceinline__ explicit RowScale(float x) {
        const float m = fabsf(x);
        const bool big = m > 0x1p96f, tiny = m < 0x1p-126f && m > 0.0f;
        s = x * (big ? 0x1p-64f : (tiny ? 0x1p64f : 1.0f));
        back = big ? 0x1p64f : (tiny ? 0x1p-64f : 1.0f);
    }
    __device__ __forceinline__ float operator()(int sum, float channel) const {
        return (float)sum * s * channel * back;
    }
};

__device__ __forceinline__ uint32_t pack2(float a, float b) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
}

// four results at columns n .. n + 3 of a row of C (element index at), N the
// row's columns; vec: a whole aligned store is possible
__device__ __forceinline__ void put4(const OpGemmArgs &g, long long at, int n, float v0, float v1, float v2, float v3,
                                     bool vec) {
    float v[4] = {v0, v1, v2, v3};
    if (g.c_f32) {
        float *c = (float *)g.C + at;
        if (vec && n + 3 < g.N) {
            float4 o = make_float4(v0, v1, v2, v3);
            if (g.accumulate) {
                const float4 p = *(const float4 *)c;
                o = make_float4(p.x + v0, p.y + v1, p.z + v2, p.w + v3);
            }
            *(float4 *)c = o;
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (n + q < g.N) c[q] = g.accumulate ? c[q] + v[q] : v[q];
        }
    } else {
        uint16_t *c = (uint16_t *)g.C + at;
        if (vec && n + 3 < g.N) {
            if (g.accumulate) {
                const uint2 p = *(const uint2 *)c;
                v[0] += bf16_to_f32((uint16_t)p.x), v[1] += bf16_to_f32((uint16_t)(p.x >> 16));
                v[2] += bf16_to_f32((uint16_t)p.y), v[3] += bf16_to_f32((uint16_t)(p.y >> 16));
            }
            *(uint2 *)c = make_uint2(pack2(v[0], v[1]), pack2(v[2], v[3]));
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (n + q < g.N) c[q] = f32_to_bf16(g.accumulate ? bf16_to_f32(c[q]) + v[q] : v[q]);
        }
    }
}

__device__ __forceinline__ bool vec_ok(const OpGemmArgs &g) {
    const int es = g.c_f32 ? 4 : 2;
    return (((uintptr_t)g.C | (uintptr_t)(g.ldc * es) | (uintptr_t)(g.c_stride * es)) & (4 * es - 1)) == 0;
}

// A tile's results through LDS, so that whole rows are stored: a wave's own
// stores are 16 rows x 32 (fp32: 64) bytes each.  Row r's 16-byte chunk c is
// kept at chunk c ^ (r mod CH): the column-wise writes and the row-wise reads
// both spread over the banks.  The chunks are stored whole at whatever alignment
// their rows have (12 groups of 259 rows of 1001 / 2731, weight gradient: 169 us, by
// elements 175; bf16 69, by elements 75).  PAST: around the caches (weight gradients,
// which the optimizer reads when all of them are done: 64 Zipf groups of 2048 / 1408
// 383 us, 404 through the caches; results of row products gain nothing).  EO:
// bytes of a result; PR rows at a time.  val(i, j, c): the lane's result in row
// block i, column block j, column 4 (lane / 16) + c.
template <int EO, int BM, int BN, int WM, int WN, int RING, bool PAST, typename Val>
__device__ __forceinline__ void store_tile_rows(const OpGemmArgs &g, lds_u8 *ring, long long at0, int mrows, int n0,
                                                int wm, int wn, int lane, Val val) {
    constexpr int NT = WM * WN * 64, NJ = BN / WN / 16;
    constexpr int CW = BN * EO, CH = CW / 16, CE = 16 / EO;
    constexpr int FIT = RING / CW;
    constexpr int PR = FIT >= BM ? BM : (FIT >= BM / 2 ? BM / 2 : BM / 4);  // rows per pass
    static_assert(PR % (WM * 16) == 0 && BM % PR == 0 && NT % CH == 0 && PR % (NT / CH) == 0, "passes");
    constexpr int IP = PR / (WM * 16);  // row blocks of a wave per pass
    const int r16 = lane & 15, q4 = lane >> 4;
#pragma unroll
    for (int p = 0; p < BM / PR; ++p) {
        if (p * PR >= mrows) break;
        __syncthreads();  // the ring (the previous pass) is no longer read
#pragma unroll
        for (int ii = 0; ii < IP; ++ii) {
            const int i = p * IP + ii, r = (ii * WM + wm) * 16 + r16;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int b = ((wn * NJ + j) * 16 + 4 * q4) * EO, c = b / 16;
                lds_u8 *q = ring + r * CW + ((c ^ (r & (CH - 1))) << 4) + (b & 15);
                if constexpr (EO == 4) {
                    typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
                    *(lds_f32x4 *)q = f32x4{val(i, j, 0), val(i, j, 1), val(i, j, 2), val(i, j, 3)};
                } else {
                    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
                    *(__attribute__((address_space(3))) u32x2 *)q =
                        u32x2{pack2(val(i, j, 0), val(i, j, 1)), pack2(val(i, j, 2), val(i, j, 3))};
                }
            }
        }
        __syncthreads();
        const int ch = (int)threadIdx.x % CH, n = n0 + ch * CE;
        const int rows = min(PR, mrows - p * PR);
        if (n < g.N) {
            for (int r = (int)threadIdx.x / CH; r < rows; r += NT / CH) {
                u32x4 v = *(const __attribute__((address_space(3))) u32x4 *)(ring + r * CW + ((ch ^ (r & (CH - 1))) << 4));
                uint8_t *dst = (uint8_t *)g.C + (at0 + (long long)(p * PR + r) * g.ldc + n) * EO;
                if (n + CE <= g.N) {
                    if (g.accumulate) {
                        u32x4 o;
                        __builtin_memcpy(&o, dst, 16);
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            if constexpr (EO == 4)
                                v[q] = __float_as_uint(__uint_as_float(o[q]) + __uint_as_float(v[q]));
                        }
                    }
                    typedef u32x4 __attribute__((aligned(2))) u32x4_u;
                    if constexpr (PAST) __builtin_nontemporal_store(v, (u32x4_u *)dst);
                    else *(u32x4_u *)dst = v;
                } else {
#pragma unroll
                    for (int q = 0; q < CE; ++q) {
                        if (n + q >= g.N) continue;
                        if constexpr (EO == 4) {
                            float *d = (float *)dst + q;
                            const float x = __uint_as_float(v[q]);
                            *d = g.accumulate ? *d + x : x;
                        } else {
                            ((uint16_t *)dst)[q] = (uint16_t)(v[q / 2] >> (16 * (q & 1)));
                        }
                    }
                }
            }
        }
    }
}

// ---- the kernel --------------------------------------------------------------------
// Bound by the matrix units at the clock that their load leaves: 8192 rows, 8
// bf16 experts of 4096 / 14336 in 835 to 862 us (1140 TFLOP/s, units 56 % busy; one 8192
// cubed product 1325), their row gradient the same, int8 485 (2000 TOP/s); fp32, 4096
// cubed, 142 TFLOP/s of 154.  The weight gradient of 64 groups of 2048 / 1408 over
// 49152 rows (383 us) is bound by its 738 MB result, stored after each tile.
//
// WM x WN waves; wave (wm, wn) owns the 16-row blocks wm, wm + WM, ... (so that
// the blocks of a part-filled tile are spread over the SIMDs, and a wave skips
// those past the last row) and BN / WN adjacent columns.
//
// DIRECT: a ring of NS stages in LDS.  The wave's columns are taken in two
// halves.  Stage s:
//   half 0: MFMAs of the first columns | reads of the stage's second columns
//   wait until stage s + 1 landed; barrier (nothing of slot s is read any more)
//   half 1: MFMAs of the second columns | reads of stage s + 1's rows and first
//           columns | loads of stage s + NS into slot s
// Loads past the last stage read zeros without touching memory, which keeps
// the count of loads in flight exact (a stage loaded by dwords counts for more
// and is waited for earlier).
template <int OT, bool ACOL, bool BCOL, bool RAGK, int BM, int BN, int WM, int WN, int KSUB, int NS, int VB>
__device__ __forceinline__ void op_gemm_tile(const OpGemmArgs &g, uint8_t *ring_) {
    constexpr int ES = op_size(OT), NT = WM * WN * 64, KE = KSUB * 64 / ES;
    constexpr int MI = BM / WM / 16, NJ = BN / WN / 16, JH = NJ / 2;
    constexpr bool DIRECT = VB > 0;
    using TA = Tile<ES, BM, ACOL, NT, KSUB, VB>;
    using TB = Tile<ES, BN, BCOL, NT, KSUB, VB>;

    OpJob jb;
    if constexpr (RAGK) {
        if (!matrix_job(g, jb, BM, BN, KE)) return;
    } else {
        if (!ragged_job<BM>(g, jb, BN)) return;
    }
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = w % WM, wn = w / WM;

    TA ta;
    TB tb;
    int klen;
    {
        const uint8_t *A = (const uint8_t *)g.A, *B = (const uint8_t *)g.B;
        if constexpr (RAGK) {
            klen = jb.len;
            ta.init(A + ((long long)jb.lo * g.lda + jb.m0) * ES, g.lda * ES, g.M - jb.m0, klen);
            tb.init(B + ((long long)jb.lo * g.ldb + jb.n0) * ES, g.ldb * ES, g.N - jb.n0, klen);
        } else {
            static_assert(!ACOL || RAGK, "ragged rows: A is a row operand");
            int k0;
            k_range(g, jb.ks, KE, k0, klen);
            ta.init(A + ((long long)(jb.lo + jb.m0) * g.lda + k0) * ES, g.lda * ES, jb.len - jb.m0, klen);
            B += (long long)jb.e * g.b_stride * ES;
            tb.init(B + (BCOL ? (long long)k0 * g.ldb + jb.n0 : (long long)jb.n0 * g.ldb + k0) * ES, g.ldb * ES,
                    g.N - jb.n0, klen);
        }
    }
    // int8: the scales of the tile's rows, the same in every wave, on their way under
    // the products (7101 rows, 10 experts of 256 / 6912: 61.8 us, 62.5 loaded after them)
    const int mrows = RAGK ? g.M - jb.m0 : jb.len - jb.m0;
    constexpr int RS = OT == OT_I8 ? BM / 64 : 1;
    float rscale[RS];
    if constexpr (OT == OT_I8) {
#pragma unroll
        for (int i = 0; i < RS; ++i) rscale[i] = i * 64 + lane < mrows ? g.sa[jb.lo + jb.m0 + i * 64 + lane] : 0.0f;
    }
    acc_t<OT> acc[MI][NJ];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = acc_t<OT>{0, 0, 0, 0};

    lds_u8 *ring = (lds_u8 *)ring_;
    // all slots of A, then all of B: the slots of an operand are within a DS
    // instruction's 16-bit offset of each other
    auto a_slot = [](auto SLOT) { return decltype(SLOT)::value * TA::BYTES; };
    auto b_slot = [](auto SLOT) { return NS * TA::BYTES + decltype(SLOT)::value * TB::BYTES; };
    const int S = (klen + KE - 1) / KE;
    auto read_a = [&](auto SLOT, int i, int ks) { return TA::frag(ring + a_slot(SLOT), i * WM + wm, ks, lane); };
    auto read_b = [&](auto SLOT, int j, int ks) { return TB::frag(ring + b_slot(SLOT), wn * NJ + j, ks, lane); };
    if (S > 0) {
        if constexpr (DIRECT) {
            constexpr int NL = TA::NC + TB::NC;
            const unsigned l0 = (unsigned)(uintptr_t)ring;
            auto load = [&](auto SLOT, int s) {
                ta.load_lds(s, l0 + a_slot(SLOT), w);
                tb.load_lds(s, l0 + b_slot(SLOT), w);
            };
            load(num<0>{}, 0);
            load(num<1>{}, 1);
            if constexpr (NS > 2) load(num<2 % NS>{}, 2);
            if constexpr (NS > 3) load(num<3 % NS>{}, 3);
            wait_loads<(NS - 1) * NL>();
            lds_barrier();
            // NI: the wave's row blocks that hold rows
            auto run = [&](auto NI_) {
                constexpr int NI = decltype(NI_)::value;
                u32x4 fa[MI], fb[2][JH];
#pragma unroll
                for (int i = 0; i < NI; ++i) fa[i] = read_a(num<0>{}, i, 0);
                if constexpr (NI > 0) {
#pragma unroll
                    for (int j = 0; j < JH; ++j) fb[0][j] = read_b(num<0>{}, j, 0);
                }
                auto stage = [&](auto SLOT, int s) {
                    using Next = num<(decltype(SLOT)::value + 1) % NS>;
#pragma unroll
                    for (int ks = 0; ks < KSUB; ++ks) {
                        if constexpr (NI > 0) {
#pragma unroll
                            for (int j = 0; j < JH; ++j) fb[1][j] = read_b(SLOT, JH + j, ks);
#pragma unroll
                            for (int i = 0; i < NI; ++i)
#pragma unroll
                                for (int j = 0; j < JH; ++j) acc[i][j] = fma16<OT>(fb[0][j], fa[i], acc[i][j]);
                        }
                        const bool last = ks == KSUB - 1;
                        if (last) {
                            wait_loads<(NS - 2) * NL>();
                            lds_barrier();
                        }
                        if constexpr (NI > 0) {
#pragma unroll
                            for (int j = 0; j < JH; ++j)
                                fb[0][j] = last ? read_b(Next{}, j, 0) : read_b(SLOT, j, ks + 1);
                        }
                        if (last) load(SLOT, s + NS);
#pragma unroll
                        for (int i = 0; i < NI; ++i) {
#pragma unroll
                            for (int j = 0; j < JH; ++j) acc[i][JH + j] = fma16<OT>(fb[1][j], fa[i], acc[i][JH + j]);
                            fa[i] = last ? read_a(Next{}, i, 0) : read_a(SLOT, i, ks + 1);
                        }
                    }
                };
                int s = 0;
                for (; s + NS <= S; s += NS) {
                    stage(num<0>{}, s);
                    stage(num<1>{}, s + 1);
                    if constexpr (NS > 2) stage(num<2 % NS>{}, s + 2);
                    if constexpr (NS > 3) stage(num<3 % NS>{}, s + 3);
                }
                if (s < S) stage(num<0>{}, s);
                if (s + 1 < S) stage(num<1>{}, s + 1);
                if constexpr (NS > 3)
                    if (s + 2 < S) stage(num<2 % NS>{}, s + 2);
            };
            if constexpr (RAGK || MI < 4) {
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
            auto step = [&](auto SLOT, int s) {
                lds_barrier();
                if (s + 1 < S) {
                    ta.load_regs(s + 1);
                    tb.load_regs(s + 1);
                }
#pragma unroll
                for (int ks = 0; ks < KSUB; ++ks) {
                    u32x4 fa[MI], fb[NJ];
#pragma unroll
                    for (int i = 0; i < MI; ++i) fa[i] = read_a(SLOT, i, ks);
#pragma unroll
                    for (int j = 0; j < NJ; ++j) fb[j] = read_b(SLOT, j, ks);
#pragma unroll
                    for (int i = 0; i < MI; ++i)
#pragma unroll
                        for (int j = 0; j < NJ; ++j) acc[i][j] = fma16<OT>(fb[j], fa[i], acc[i][j]);
                }
                if (s + 1 < S) {
                    using Other = num<1 - decltype(SLOT)::value>;
                    ta.store_regs(ring + a_slot(Other{}));
                    tb.store_regs(ring + b_slot(Other{}));
                }
            };
            ta.load_regs(0);
            tb.load_regs(0);
            ta.store_regs(ring + a_slot(num<0>{}));
            tb.store_regs(ring + b_slot(num<0>{}));
            int s = 0;
            for (; s + 2 <= S; s += 2) {
                step(num<0>{}, s);
                step(num<1>{}, s + 1);
            }
            if (s < S) step(num<0>{}, s);
        }
    }

    const int r16 = lane & 15, q4 = lane >> 4;
    if constexpr (BM <= 64) {  // (split calls run the smallest tiles)
        if (g.splits > 1) {    // a range's sums, folded by op_fold_kernel
            const long long first = RAGK ? (long long)(jb.e * g.splits + jb.ks) * g.M + jb.m0
                                         : (long long)jb.ks * g.rows + jb.lo + jb.m0;
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                const int ml = (i * WM + wm) * 16 + r16;
                if (ml >= mrows) continue;
                acc_elem<OT> *ws = (acc_elem<OT> *)g.ws + (first + ml) * g.N;
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const int n = jb.n0 + (wn * NJ + j) * 16 + 4 * q4;
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        if (n + c < g.N) ws[n + c] = acc[i][j][c];
                }
            }
            return;
        }
    }
    const long long at0 = RAGK ? (long long)jb.e * g.c_stride + (long long)jb.m0 * g.ldc
                               : (long long)(jb.lo + jb.m0) * g.ldc;  // the tile's first row in C
    // int8: the lane's scales, of its row blocks and its columns
    float sa[MI], sb[NJ][4];
    bool far = false;
    if constexpr (OT == OT_I8) {
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            const int ml = (i * WM + wm) * 16 + r16;
            sa[i] = ml < mrows ? g.sa[jb.lo + jb.m0 + ml] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int n = jb.n0 + (wn * NJ + j) * 16 + 4 * q4 + c;
                sb[j][c] = n < g.N ? g.sb[(long long)jb.e * g.N + n] : 0.0f;
            }
        // every wave looks at all rows of the tile: the answer is the workgroup's
#pragma unroll
        for (int i = 0; i < RS; ++i) far |= RowScale(rscale[i]).back != 1.0f;
        far = __any(far);
    }
    constexpr int RING = NS * (TA::BYTES + TB::BYTES);
    auto store = [&](auto val) {
        if (g.c_f32) store_tile_rows<4, BM, BN, WM, WN, RING, RAGK>(g, ring, at0, mrows, jb.n0, wm, wn, lane, val);
        else store_tile_rows<2, BM, BN, WM, WN, RING, RAGK>(g, ring, at0, mrows, jb.n0, wm, wn, lane, val);
    };
    auto val = [&](int i, int j, int c) -> float {
        if constexpr (OT == OT_I8) return (float)acc[i][j][c] * sa[i] * sb[j][c];
        else return acc[i][j][c];
    };
    if constexpr (OT == OT_I8) {
        // (the factor that moves a result back on every one: 8192 rows on 8 experts of
        // 4096 / 14336 2 % longer)
        if (far) {
            store([&](int i, int j, int c) -> float { return RowScale(sa[i])(acc[i][j][c], sb[j][c]); });
            return;
        }
    }
    if (g.c_f32 || !g.accumulate) {
        store(val);
        return;
    }
    // a bf16 sum that is added to stays in fp32 until its one rounding
    const bool vec = vec_ok(g);
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        const int ml = (i * WM + wm) * 16 + r16;
        if (ml >= mrows) continue;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int n = jb.n0 + (wn * NJ + j) * 16 + 4 * q4;
            put4(g, at0 + (long long)ml * g.ldc + n, n, val(i, j, 0), val(i, j, 1), val(i, j, 2), val(i, j, 3), vec);
        }
    }
}

template <int OT, bool ACOL, bool BCOL, bool RAGK, int BM, int BN, int WM, int WN, int KSUB, int NS, int WPE, int VB>
__global__ __launch_bounds__(WM * WN * 64) __attribute__((amdgpu_waves_per_eu(WPE, WPE))) void op_gemm_kernel(
    OpGemmArgs g) {
    __shared__ __attribute__((aligned(1024))) uint8_t ring[NS * (BM + BN) * 64 * KSUB];
    op_gemm_tile<OT, ACOL, BCOL, RAGK, BM, BN, WM, WN, KSUB, NS, VB>(g, ring);
}

// Rows of whole, aligned pieces of `bytes`.
inline bool whole_pieces(const void *p, long long ld, long long stride, int contiguous, int es, int bytes) {
    return (((uintptr_t)p | (uintptr_t)(ld * es) | (uintptr_t)(stride * es)) & (bytes - 1)) == 0 &&
           (long long)contiguous * es % bytes == 0;
}
// A tile's byte offsets (up to 255 rows) within 31 bits.
inline bool tile_offsets_ok(long long ld, int es) { return ld * es < (1ll << 22); }

template <int OT, bool ACOL, bool BCOL, bool RAGK, int BM, int BN, int WM, int WN, int KSUB, int NS, int WPE>
hipError_t launch_tiles(OpGemmArgs g, int vb, hipStream_t s) {
    g.nt = (g.N + BN - 1) / BN;
    g.mt = RAGK ? (g.M + BM - 1) / BM : 0;
    // ragged rows: sum of ceil(rows_e / BM) <= rows / BM + the groups that can hold a row
    // ragged k: every XCD's part of every group
    const long long mtiles = (long long)(g.rows / BM) + (g.E < g.rows ? g.E : g.rows);
    const long long grid =
        RAGK ? ((long long)g.mt * g.nt * g.splits + 7) / 8 * 8 * g.E : (mtiles * g.nt * g.splits + 7) / 8 * 8;
    if (grid > 0x7fffffffll / (WM * WN * 64)) return kOpTooLarge;
    const dim3 b(WM * WN * 64);
    // (bf16 pairs by dwords: the registers of three waves per SIMD are too few)
    constexpr int W4 = WPE == 3 && BM == 128 && OT == OT_BF16 ? 2 : WPE;
#define MOE_OP_TILES(KS_, NS_, VB_)                                                                       \
    op_gemm_kernel<OT, ACOL, BCOL, RAGK, BM, BN, WM, WN, KS_, NS_, VB_ == 4 ? W4 : WPE, VB_><<<(unsigned)grid, b, 0, \
                                                                                              s>>>(g)
    if (vb == 16) {
        MOE_OP_TILES(KSUB, NS, 16);
    } else if constexpr (BN == 256) {
        return hipErrorInvalidValue;  // (staging through registers leaves too few for these tiles)
    } else if (vb == 4) {
        MOE_OP_TILES(KSUB, NS, 4);
    } else if constexpr (OT == OT_F32) {
        if constexpr (BM == 64) {
            MOE_OP_TILES(1, 2, 0);  // row strides of 4 MB and more
        } else {
            return hipErrorInvalidValue;
        }
    } else {
        MOE_OP_TILES(2, 2, 0);
    }
#undef MOE_OP_TILES
    const hipError_t e = hipGetLastError();
    return e == hipSuccess && g.splits > 1 ? launch_op_fold(OT, RAGK, g, s) : e;
}

// Tile and load form of a call.  256 x 256 tiles where there are two rounds of
// them (ragged rows: and groups average enough rows to fill them), else 128 x
// 128, and 64 x 64 for short groups or few tiles.  Measured on 8192 rows, 8 bf16
// experts of 4096 / 14336, 256 x 256 against 128 x 256 with two workgroups per
// CU: forward 874 / 1055 us, row gradient 852 / 926, int8 563 / 627; the weight
// gradient of 64 Zipf groups of 2048 / 1408, 256 x 256 against 128 x 128 with three
// workgroups per CU: 411 / 453 us.  Where even 64 x 64 tiles are few, k is split into
// ranges (op_rows_splits, op_matrix_splits).
template <int OT, bool ACOL, bool BCOL, bool RAGK>
hipError_t op_gemm_plan(OpGemmArgs g, int ncu, hipStream_t s) {
    constexpr int ES = op_size(OT);
    // row operands are loaded in whole 128-byte lines
    constexpr int KSUB = ACOL && BCOL ? 1 : 2;
    // alignment of the rows that are loaded straight into LDS; 0: through registers
    int vb = 0;
    if (tile_offsets_ok(g.lda, ES) && tile_offsets_ok(g.ldb, ES)) {
        auto pieces = [&](int bytes) {
            return whole_pieces(g.A, g.lda, 0, ACOL ? g.M : g.K, ES, bytes) &&
                   whole_pieces(g.B, g.ldb, g.b_stride, BCOL ? g.N : g.K, ES, bytes);
        };
        if (pieces(16)) vb = 16;
        else if (g.lda >= 16 / ES && g.ldb >= 16 / ES && pieces(4)) vb = 4;
    }
    auto tiles = [&](int b) -> long long {
        const long long nt = (g.N + b - 1) / b;
        if (RAGK) return nt * ((g.M + b - 1) / b) * g.E;
        const long long few = (long long)g.rows / b > g.E ? (long long)g.rows / b : (g.E < g.rows ? g.E : g.rows);
        return nt * few;
    };
    const long long avg = RAGK ? g.M : (long long)g.rows / g.E;
    if (g.splits > 1) return launch_tiles<OT, ACOL, BCOL, RAGK, 64, 64, 2, 2, KSUB, 4 / KSUB, 3>(g, vb, s);
    if constexpr (OT != OT_F32) {
        const bool large = RAGK ? tiles(256) >= 2 * ncu : avg >= 192 && g.N >= 192 && tiles(256) >= 2 * ncu;
        if (vb == 16 && large)
            return launch_tiles<OT, ACOL, BCOL, RAGK, 256, 256, 4, 2, KSUB, 4 / KSUB, 2>(g, vb, s);
    }
    bool medium = avg >= 64 && g.N >= 64 && tiles(128) >= ncu;
    if constexpr (OT == OT_F32) {
        // fp32 is bound by its matrix rate: the CU with the most tiles decides, a 128 x 128
        // tile taking as long as 3.8 of 64 x 64 (weight gradient, whose stores it spares:
        // 3.4).  A group's last tile is half empty on average.  us, 128 / 64: row products
        // of 4096 cubed 964 / 1000, 3000 cubed 536 / 424, 8 groups of 1024 rows 2048 / 2048 605 /
        // 545, 44114 rows 2240 / 192 409 / 326; weight gradients of 4096 cubed 957 / 1009, 12 groups
        // of 259 rows 1001 / 2731 164 / 194, 3 of 1325 rows 12810 / 69 176 / 135.
        auto per_cu = [&](int b) -> long long {
            const long long nt = (g.N + b - 1) / b;
            const long long mt = RAGK ? (g.M + b - 1) / b * (long long)g.E
                                      : (g.E > 1 ? g.rows / b + (g.E < g.rows ? g.E : g.rows) / 2 + 1 : (g.rows + b - 1) / b);
            return (nt * mt + ncu - 1) / ncu;
        };
        // (a weight gradient of fewer rows than 64 is bound by its stores: 71 groups of one
        // row at most, 6193 / 257, 158 / 181)
        if (vb == 0) medium = false;
        else if (!RAGK || g.rows >= 64ll * g.E) medium = (RAGK ? 34 : 38) * per_cu(128) < 10 * per_cu(64);
    }
    if (medium)
        return launch_tiles<OT, ACOL, BCOL, RAGK, 128, 128, 2, 2, KSUB, RAGK ? 3 : 4 / KSUB, RAGK ? 3 : 2>(g, vb, s);
    return launch_tiles<OT, ACOL, BCOL, RAGK, 64, 64, 2, 2, KSUB, 4 / KSUB, 3>(g, vb, s);
}

}  // namespace ops
}  // namespace moe
