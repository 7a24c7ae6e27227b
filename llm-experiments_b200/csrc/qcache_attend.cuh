// Attention of a few new tokens over a quantised key / value cache (the form is in b2kv.h).
//
// What bounds it: HBM.  A cached token of a head is D * (k_bits + v_bits) / 8 + D / 8 bytes for 4 * D * (query heads) flops, so the
// arithmetic has to be hidden behind 23 bytes per clock and SM, and with 4 bits 46 elements per clock have to be widened.  Plain
// fp32 arithmetic cannot (128 FMAs per clock and SM, one per element and query head); the tensor cores can, if widening is cheap:
//
//   * Keys' codes become fp16 numbers by masking alone: a code c in bits 2 .. 5 or 6 .. 9 of a 16-bit half is the fp16 subnormal c * 2^-22 or c * 2^-18, two
//     codes per instruction, and tensor cores take subnormals at full speed.  They add products by the exponents as they stand, so
//     that a number whose first bit is k places below the tenth loses k bits of the sum: at most 4 here, which is why units of 4-bit codes are kept
//     turned by two bits (bits 0 .. 3 and 4 .. 7 would lose 7 and 3).  Codes stay uncentred (c + 8, c + 128): what the centre comes to is a small product of
//     the key scales and the query's sums over the groups, which the scores start from.  A group's sum is multiplied by its key scale in fp32.
//   * Values' codes are put behind the exponent of 1024 by the mask's instruction, and the centre is taken off by a second one (a row of ones in the
//     product does that too, but moving its operand into place costs as much, and over thousands of tokens the sums of uncentred codes grow far
//     beyond what is left in the end).
//   * Both products have the cache's rows as the operand of many rows: S[token, column] = K q (16 tokens by 8 columns per MMA, m16n8k16)
//     and O[element, column] += V^T P.  A column is one (new token, query head) pair of the key / value head.  The cache's
//     layout gives a lane the codes that it needs as one piece, the query is permuted to match, and P goes from the accumulator's
//     layout to the operand's by an 8 x 8 transpose within the warp.  The rows go through tcgen05 only if they were first widened into
//     shared memory at 16 bits per element, which is four times the traffic of reading them; as register operands they are widened in place.
//   * A probability is rounded to fp16, multiplied by its value scale there and rounded again (11 bits; the output has 8).  fp16 has room for that as
//     long as a group's scales are of a size: each group (of a warp's tokens of a pair) has a reference exponent, and a scale goes this way if it lies within
//     2^-8 .. 2 of it.  The weight is 2^14 at most and 2^10 where it is the largest, so that products stay below 2^15, and a product below 2^-14, where
//     bits are lost, is one whose weight is below 2^-16 of the largest.
//   * What lies outside (a group whose tokens differ by more, a large value that no query gives any weight) is seldom there and goes another way: weight times
//     scale in fp32, as a sum of bfloat16 parts, which have fp32's range, by as many more products.  So no element depends on what lies in other groups, nor on
//     tokens that it does not see.  The reference moves, and the accumulators with it, where more than half of a group's scales in a stage lie outside; it
//     stays within 2^64 of the largest, so that sums are finite.
//   * fp32 queries and weights are sums of two fp16 numbers (22 bits), in columns of their own (four pairs of them to a tile of eight); keys are centred like values; and only 16 tokens'
//     products are added up in the tensor core, whose sums are cut off and not rounded.
//   * Softmax: scores in the log2 domain, references that move only when a score has outgrown its own by more than 2^4 (one vote per stage), sums per
//     lane until the end, all in fp32.
#pragma once

#include <cuda_fp16.h>

#include <atomic>
#include <type_traits>

#include "qcache.cuh"

namespace b2kv {
namespace qcache {

struct AttendParams {
    b2kv_qcache c;
    Divisor by_block;
    const void* q;
    void* out;
    const float* slopes;
    float* ws_o;    // [2 * CTAs, kCols, D]: what a CTA has of its first (sequence, head) and of its last, normalised
    float* ws_lse;  // [2 * CTAs, kCols]: log2 of the sum of exponentials
    unsigned long long* tickets;  // [pairs]: (number of the call << 24) | pieces of the pair that are there
    unsigned long long call;      // 40 bits, another for each call and never 0
    int32_t* dev_status;
    int64_t ld_q, ld_out;
    int R, m, col_tiles, T_upper, len_bias, window;
    int cluster;      // > 0: a cluster of this many CTAs per (sequence, head, column tile); 0: all tokens laid end to end and cut into gridDim.x pieces
    float scale;        // scale * log2 e = scale * 2^scale_exp
    int scale_exp;
    float cap;          // times log2 e; 0 without one
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_huge_valf();
constexpr float kLowest = -3.0e38f;  // a reference where nothing was seen yet: any score has outgrown it, and differences stay finite

__device__ __forceinline__ int lane_id() {
    int lane;
    asm("mov.u32 %0, %%laneid;" : "=r"(lane));
    return lane;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// d = the product alone
__device__ __forceinline__ void mma_new(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t half_sub(uint32_t a, uint32_t b) {
    uint32_t y;
    asm("sub.f16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
    return y;
}
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {  // one instruction
    uint32_t y;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "r"(mask), "r"(bits));
    return y;
}
__device__ __forceinline__ uint32_t half_mul(uint32_t a, uint32_t b) {
    uint32_t y;
    asm("mul.f16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
    return y;
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    uint32_t y;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
    return y;
}
__device__ __forceinline__ float2 unpack_half(uint32_t x) { return __half22float2(*reinterpret_cast<__half2*>(&x)); }

// 16 / 8 / 4 bytes into shared memory, zeros where `there` is false (nothing is read then).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void copy_small(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(there ? BYTES : 0) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void copy_small(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <int BYTES>
struct Words {
    uint32_t w[(BYTES + 3) / 4];
    // BYTES bytes at a shared address that is a multiple of the largest power of two in BYTES (up to 16)
    __device__ __forceinline__ void load(uint32_t at) {
        if constexpr (BYTES % 16 == 0) {
#pragma unroll
            for (int i = 0; i < BYTES / 16; ++i) load16(at + 16 * i, 4 * i);
        } else if constexpr (BYTES % 8 == 0) {
#pragma unroll
            for (int i = 0; i < BYTES / 8; ++i) load8(at + 8 * i, 2 * i);
        } else if constexpr (BYTES % 4 == 0) {
#pragma unroll
            for (int i = 0; i < BYTES / 4; ++i) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[i]) : "r"(at + 4 * i) : "memory");
        } else {
#pragma unroll
            for (int i = 0; i < (BYTES + 3) / 4; ++i) {
                uint16_t lo, hi = 0;
                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(lo) : "r"(at + 4 * i) : "memory");
                if (4 * i + 2 < BYTES) asm volatile("ld.shared.u16 %0, [%1];" : "=h"(hi) : "r"(at + 4 * i + 2) : "memory");
                w[i] = lo | static_cast<uint32_t>(hi) << 16;
            }
        }
    }
    __device__ __forceinline__ void store(uint32_t at) const {
#pragma unroll
        for (int i = 0; i < BYTES / 4; ++i) asm volatile("st.shared.u32 [%0], %1;" ::"r"(at + 4 * i), "r"(w[i]) : "memory");
    }
    __device__ __forceinline__ void load16(uint32_t at, int i) {
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]) : "r"(at) : "memory");
    }
    __device__ __forceinline__ void load8(uint32_t at, int i) {
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[i]), "=r"(w[i + 1]) : "r"(at) : "memory");
    }
};

// The first token that any query of a sequence of n tokens sees.
__device__ __forceinline__ int first_seen(const AttendParams& p, int n) { return p.window > 0 ? max(n - p.m + 1 - p.window, 0) : 0; }

// What a warp's ring holds with two CTAs per SM: at least two stages, one in the arithmetic and one on its way, of 32 tokens where that many fit, else 16.
// What a stage costs beside its products (copies, masks, references, the scales' exponents) is a quarter of 32 tokens' time, so two long stages beat
// four short ones (8 and 4 bits, heads of 128, the benchmark's batch: 286 against 340 us); 64 tokens run out of registers (4 bits: 292 against 276 us).
template <int NG, int KB, int VB, int NT>
struct Ring {
    static constexpr int kWarps = NT == 1 && NG <= 4 ? 6 : 4;  // of 168 or 255 registers per thread
    static constexpr int kCtas = 2;
    static constexpr int kToken = NG * 4 * (KB + VB) + 4 * scale_row(NG);
    // Half of what an SM has for two CTAs, less the queries, what is kept per column, and 1 KB of small things.
    static constexpr int kRoom = (113 * 1024 - 1024 - NG * NT * 512 - NT * (640 + kWarps * 64) - 64) / kWarps;
    static constexpr int kTokens = 2 * 32 * kToken <= kRoom ? 32 : 16;
    static constexpr int kFit = kRoom / (kTokens * kToken);
    static constexpr int kStages = kFit > 4 ? 4 : kFit;
    static_assert(kStages >= 2, "");
};

// T: type of queries and outputs; NG groups of 32 elements; KB, VB bits; NT tiles of 8 columns (fp32: one, of 4 columns and of what fp16 leaves of each).
template <typename T, int NG, int KB, int VB, int NT>
struct Attend {
    using R = Ring<NG, KB, VB, NT>;
    static constexpr int WARPS = R::kWarps, STAGES = R::kStages, kTok = R::kTokens, MT = kTok / 16;
    static constexpr bool kF32 = std::is_same<T, float>::value;
    static_assert(!kF32 || NT == 1, "");
    static constexpr int D = NG * kGroup, kCols = kF32 ? 4 : 8 * NT, kThreads = WARPS * 32;
    static constexpr int kKRow = D * KB / 8, kVRow = D * VB / 8, kSRow = scale_row(NG) * 2;
    static constexpr int kKBytes = kTok * kKRow, kVBytes = kTok * kVRow, kSBytes = kTok * kSRow;
    static constexpr int kStage = (kKBytes + kVBytes + 2 * kSBytes + 15) / 16 * 16;
    static constexpr int kRing = WARPS * STAGES * kStage;
    // Results are put together in a stage of each warp's ring, as many columns at a time as go into one.
    static constexpr int kRoundCols = kCols * D * 4 <= kStage ? kCols : kCols * D * 2 <= kStage ? kCols / 2 : kCols / 4;
    static constexpr int kRounds = kCols / kRoundCols;
    static_assert(kRoundCols * D * 4 <= kStage && kRoundCols % 2 == 0, "");
    static constexpr int kMl = WARPS * kCols * 2 * 4;
        // The centre of the keys costs -kKOff * sum over groups of (key scale) * (sum of the group's query): a product over the groups, the sums
    // in three bfloat16 parts (16 places: part k / kSG of group k % kSG; with 8 groups in two products).
    static constexpr int kSG = scale_row(NG), kOffs = kF32 ? 1 : kSG == 8 ? 4 : 2;
    static constexpr int kKOff = KB == 4 ? 8 : 128;  // what is added to a key's code
    // A code of one in a score's sum, as a power of two: codes' own (fp16 numbers or subnormals), and in fp32, where that would let sums of large keys
    // overflow, another 2^-16 that the key scales are multiplied by (a scale of 8 bits stays exact).
    static constexpr int kKeyUnitExp = (KB == 4 ? 2 : 0) - (kF32 ? 16 : 24);
    static constexpr float kKeyUnit = (KB == 4 ? 4.0f : 1.0f) * (kF32 ? 0x1p-16f : 0x1p-24f);
    // Weights are probabilities (relative to the largest) times 2^kShift, up to 2^(kLag + kShift); value scales relative to their reference are below 2: products
    // below 2^15.
    static constexpr int kShift = 10, kLag = 4;
    // Scales from 2^-kSpan of the reference to twice the reference go through fp16; a new reference is kHeadroom above the scales that it was made for; one
    // is never more than kReach below the largest scale: sums stay below 2^(kReach + 15 + kHeadroom) * 127 * 2^30 tokens.
    static constexpr int kSpan = 8, kHeadroom = 2, kReach = 64;
    static constexpr float kValueUnit = VB == 4 ? 4.0f : 1.0f;  // of a code of one; every other row of 4 bits has 16 times that

    // Where 16-byte piece ch of row r lies in a stage: moved about so that the lanes that read together meet different banks.
    __device__ static __forceinline__ int k_place(int r, int ch) {
        if constexpr (kKRow == 128) ch ^= r & 1;
        if constexpr (kKRow == 256) ch ^= ((ch >> 3) & 1) ^ ((r & 1) << 1);
        return r * kKRow + ch * 16;
    }
    __device__ static __forceinline__ int v_place(int r, int ch) {
        if constexpr (kVRow == 32) return (r >> 2) * 128 + ((((r & 3) << 1 | ch) ^ (((r >> 2) & 1) << 1)) << 4);
        if constexpr (kVRow == 64) return (r >> 1) * 128 + ((((r & 1) << 2 | ch) ^ (((r >> 1) & 3) << 1)) << 4);
        if constexpr (kVRow == 128) ch ^= ((r >> 1) & 3) << 1;
        if constexpr (kVRow == 256) ch ^= ((r >> 1) & 1) | ((r >> 2) & 1) << 2;
        return r * kVRow + ch * 16;
    }

    // Where a lane reads and copies within a stage, from one row or piece to the next.  The rows 8 further on lie 8 rows further on, whatever
    // the moving about.
    struct Lane {
        uint32_t k;         // its piece of row gid of the keys
        uint32_t v;         // its piece of row 2 tig of the values
        uint32_t put_k, put_v;  // its first 16-byte piece of a copy
        // Its piece of row 2 tig + 1: the rows in between were moved about alike.
        __device__ __forceinline__ uint32_t v_next() const { return NG == 3 ? v + kVRow : v ^ kVRow; }
        __device__ __forceinline__ void set() {
            const int lane = lane_id(), gid = lane >> 2, tig = lane & 3;
            k = NG == 3 ? gid * kKRow + tig * NG * KB : k_place(gid, tig * NG * KB / 16) + tig * NG * KB % 16;
            const int at = gid * (NG * VB / 2);
            v = NG == 3 ? 2 * tig * kVRow + at : v_place(2 * tig, at / 16) + at % 16;
            put_k = k_place(lane / (kKRow / 16), lane % (kKRow / 16));
            put_v = kKBytes + v_place(lane / (kVRow / 16), lane % (kVRow / 16));
        }
    };
    // Piece i * 32 + lane lies at (the lane's first) ^ this + i * 512.
    __device__ static __forceinline__ uint32_t moved_v(int i) {
        return kVRow == 128 ? (i & 1) * 64 : kVRow == 256 ? (i & 1) * 16 + ((i >> 1) & 1) * 64 : 0;
    }

    // What is seldom asked for, in shared memory: of a column of the CTA's present pair.
    struct Column {
        int lo, lim;  // it sees tokens lo <= t < lim
        float slope;  // log2 e times its slope
        float f;      // a score is the product's sum times this (before a cap and a bias), and times Prepared::rest
    };

    struct Warp {
        uint32_t off[NT][kOffs];   // what the key's centre comes to, as the second operand of a product with the key scales (not for fp32)
        float f[NT][2];            // Column::f where a score is the product's sum times it, else 1
        int apart;                 // bits: 1 - scores are made apart from that (a cap, a bias, a factor beyond fp32), 2 - a factor beyond fp32
        int all_lo, all_lim;       // tokens that every used column sees
        float o[NT][NG * 2][4];    // elements 32 (j / 2) + 4 gid + 2 (j & 1) (+1 in the last two), columns 2 tig, 2 tig + 1
        float ref[NT][2];          // scores are taken relative to this: what was the largest so far, less kShift
        float sum[NT][2];          // of 2^(score - ref), this lane's tokens
        bool fresh;                // some column may not have seen anything yet
    };

    // What value scales of the warp's present pair are relative to, in shared memory: one over the reference of each group (a power of two; 0 where no stage has
    // been seen yet), and the largest (biased) exponent that has gone into the accumulators.
    struct Refs {
        float by[kSG];
        int most[kSG];
        __device__ __forceinline__ int exponent(int u) const { return 254 - (__float_as_int(by[u]) >> 23); }
        __device__ __forceinline__ void set(int u, int e, int m) { by[u] = __int_as_float((254 - e) << 23), most[u] = m; }
    };

    // fp32: the second half of a tile is for the same columns as the first, and lanes 2 apart (in tig) have the same scores.
    __device__ static __forceinline__ int col_of(int nt, int c) { return kF32 ? c & 3 : nt * 8 + c; }

    // The queries of a pair are prepared by the CTA's warps together: unit i, group i % NG of the columns of tile i / NG, is warp i % WARPS's.
    static constexpr int kUnits = NT * NG, kUnitsEach = (kUnits + WARPS - 1) / WARPS;
    struct Prepared {
        uint32_t most[kUnits / NG][8][NG];  // largest magnitude of a column's group, as a whole number (NaN above infinity above all others)
        float sum[kUnits / NG][8][kSG];     // what the centre of its keys comes to
        Column columns[kCols];
        float rest[kCols];                  // what the factor of a column's scores has beyond 2^-100 .. 2^100 (a power of two, nearly always 1)
        uint4 queries[NG * NT * 32];        // the second operand of S = K q, both steps of a group in one
    };
    static constexpr int kSmem = kRing + kMl + 16 * ((WARPS * 4 + 15) / 16) + static_cast<int>(sizeof(Prepared));
    static_assert(kSmem <= 112 * 1024, "two CTAs per SM, and 1 KB for what has a fixed size");
    // A lane's part of them as they lie in memory: octet tig of its warp's groups, of column gid.
    struct Query {
        uint4 w[kUnitsEach][sizeof(T) / 2];
    };
    __device__ static __forceinline__ void load_query(const AttendParams& p, Query& raw, int b, int g, int ct) {
        const int lane = lane_id(), gid = lane >> 2, tig = lane & 3, warp = threadIdx.x >> 5;
#pragma unroll
        for (int i = 0; i < kUnitsEach; ++i) {
            const int unit = warp + i * WARPS, nt = unit / NG, u = unit - nt * NG;
            const int col = ct * kCols + col_of(nt, gid), row = col / p.R, h = g * p.R + col - row * p.R;
            const bool is = (kUnits % WARPS == 0 || unit < kUnits) && col < p.m * p.R;
            const T* const src = static_cast<const T*>(p.q) + (static_cast<int64_t>(b) * p.m + row) * p.ld_q + static_cast<int64_t>(h) * D + u * kGroup + tig * 8;
#pragma unroll
            for (int k = 0; k < static_cast<int>(sizeof(T) / 2); ++k)
                raw.w[i][k] = is ? reinterpret_cast<const uint4*>(src)[k] : make_uint4(0, 0, 0, 0);
        }
    }

    // The CTA's part in it (two barriers), then the warp's own.  n: tokens of the sequence.
    __device__ static __forceinline__ void begin(const AttendParams& p, Warp& w, Refs& refs, const Query& raw, Prepared& q, int g, int ct, int n) {
        const int lane = lane_id(), gid = lane >> 2, tig = lane & 3, warp = threadIdx.x >> 5;
        float x[kUnitsEach][8];
#pragma unroll
        for (int i = 0; i < kUnitsEach; ++i) {
            const int unit = warp + i * WARPS, nt = unit / NG, u = unit - nt * NG;
#pragma unroll
            for (int k = 0; k < static_cast<int>(sizeof(T) / 2); ++k) Elt<T>::widen(raw.w[i][k], x[i] + k * Elt<T>::kPerChunk);
            uint32_t most = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(x[i][e]) & 0x7fffffffu);
            most = max(most, __shfl_xor_sync(~0u, most, 1));
            most = max(most, __shfl_xor_sync(~0u, most, 2));
            if (tig == 0 && (kUnits % WARPS == 0 || unit < kUnits)) q.most[nt][gid][u] = most;
        }
        __syncthreads();
        // q = qn * 2^e with the largest |qn| of a column in [2^14, 2^15): exact, and no fp16 overflow.  The exponent, biased:
        const auto exponent = [&](int nt, int c) {
            uint32_t most = q.most[nt][c][0];
#pragma unroll
            for (int u = 1; u < NG; ++u) most = max(most, q.most[nt][c][u]);
            return most == 0 ? 127 : min(max(static_cast<int>(most >> 23), 15), 254);
        };
#pragma unroll
        for (int i = 0; i < kUnitsEach; ++i) {
            const int unit = warp + i * WARPS, nt = unit / NG, u = unit - nt * NG;
            if (kUnits % WARPS != 0 && unit >= kUnits) break;  // (a warp's lanes all the same)
            const float down = __int_as_float((254 + 14 - exponent(nt, gid)) << 23);
            uint32_t high[4], low[4] = {};
            float sum = 0.0f;  // of what the products see
            // elements in the order of the codes in a word's halves: 4 bits (0,4) (1,5) (2,6) (3,7), the odd ones 16 times too
            // large there; 8 bits (0,1) (2,3) (4,5) (6,7)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float by = KB == 4 && (j & 1) ? 0.0625f : 1.0f;
                const float a = x[i][KB == 4 ? j : 2 * j] * (down * by), c = x[i][KB == 4 ? j + 4 : 2 * j + 1] * (down * by);
                high[j] = pack_half(a, c);
                const float2 got = unpack_half(high[j]);
                sum += (got.x + got.y) * (1.0f / by);
                if constexpr (kF32) low[j] = pack_half(a - got.x, c - got.y);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) high[j] = kF32 && gid >= 4 ? low[j] : high[j];
            q.queries[unit * 32 + lane] = make_uint4(high[0], high[1], high[2], high[3]);
            sum += __shfl_xor_sync(~0u, sum, 1);
            sum += __shfl_xor_sync(~0u, sum, 2);
            if (tig == 0) {
                q.sum[nt][gid][u] = sum * (-static_cast<float>(kKOff) * kKeyUnit);
                if (u == NG - 1)
                    for (int v = NG; v < kSG; ++v) q.sum[nt][gid][v] = 0.0f;
            }
        }
        bool beyond = false;
        if (threadIdx.x < kCols) {
            const int c = threadIdx.x, col = ct * kCols + c, i = col / p.R, place = n - p.m + i;
            const bool is = col < p.m * p.R;
            // a score is scale * 2^(e - 14) over what a code of one is in the product: queries, keys and scales of any size can make scores of an
            // ordinary one, so this may be no fp32 number
            const int power = p.scale_exp + exponent(c / 8, c % 8) - 127 - 14 - kKeyUnitExp, within = min(max(power, -100), 100);
            const float f = p.scale * __int_as_float((127 + within) << 23);
            q.rest[c] = __int_as_float((127 + min(max(power - within, -126), 127)) << 23);
            beyond = is && power != within;
            q.columns[c] = Column{is && p.window > 0 ? max(place + 1 - p.window, 0) : 0, is ? place + 1 : 0,
                                  is && p.slopes != nullptr ? p.slopes[g * p.R + col - i * p.R] * kLog2e : 0.0f, f};
        }
        beyond = __syncthreads_or(beyond);

        const Column c = q.columns[lane & (kCols - 1)];
        const bool is = ct * kCols + (lane & (kCols - 1)) < p.m * p.R;
        w.all_lim = __reduce_min_sync(~0u, is ? c.lim : 0x7fffffff);
        w.all_lo = __reduce_max_sync(~0u, is ? c.lo : 0);
        w.apart = (beyond ? 2 : 0) | (beyond || p.cap > 0.0f || p.slopes != nullptr ? 1 : 0);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) w.f[nt][e] = w.apart == 0 ? q.columns[col_of(nt, 2 * tig + e)].f : 1.0f;
            if constexpr (!kF32) {
                // places 2 tig and 2 tig + 1 of every eight: two neighbouring groups, one of their three parts
                constexpr int kPairs = kSG / 2;
                uint32_t parts[3];
                float s[2] = {q.sum[nt][gid][tig % kPairs * 2], q.sum[nt][gid][tig % kPairs * 2 + 1]};
#pragma unroll
                for (int i = 0; i < 3; ++i) {
                    const __nv_bfloat162 both = __floats2bfloat162_rn(s[0], s[1]);
                    parts[i] = *reinterpret_cast<const uint32_t*>(&both);
                    s[0] -= __uint_as_float(parts[i] << 16), s[1] -= __uint_as_float(parts[i] & 0xffff0000u);
                }
#pragma unroll
                for (int i = 0; i < kOffs; ++i) {
                    const int which = (tig + 4 * i) / kPairs;
                    w.off[nt][i] = which == 0 ? parts[0] : which == 1 ? parts[1] : which == 2 ? parts[2] : 0u;
                }
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int j = 0; j < NG * 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) w.o[nt][j][e] = 0.0f;
#pragma unroll
            for (int e = 0; e < 2; ++e) w.ref[nt][e] = kLowest, w.sum[nt][e] = 0.0f;
        }
        w.fresh = true;
        if (lane < kSG) refs.by[lane] = 0.0f;
    }

    // Where a lane's token of a tile lies: its row, -1 where there is none or no query sees it.
    __device__ static __forceinline__ int64_t find(const AttendParams& p, int b, int g, int t0, int seen, int n) {
        const int lane = lane_id(), t = t0 + (lane & (kTok - 1));
        return t < n && t >= seen ? row_of(p.c, p.by_block, b, g, t, p.dev_status) : -1;
    }

    // Starts the copies of a tile whose rows `find` gave (zeros where there is none); a bit for each token that is there.
    __device__ static __forceinline__ uint32_t copy_paged(const AttendParams& p, const Lane& l, uint32_t stage, int64_t row) {
        const int lane = lane_id();
        const uint32_t there = __ballot_sync(~0u, row >= 0);
        const int64_t at = row >= 0 ? row : 0;
        const uint32_t ks = stage + kKBytes + kVBytes;
        if (kTok == 32 || lane < kTok) {
            copy_small<kSRow>(ks + lane * kSRow, static_cast<const uint8_t*>(p.c.k_scales) + at * kSRow, row >= 0);
            copy_small<kSRow>(ks + kSBytes + lane * kSRow, static_cast<const uint8_t*>(p.c.v_scales) + at * kSRow, row >= 0);
        }
        const uint8_t* const k = static_cast<const uint8_t*>(p.c.k_codes);
        const uint8_t* const v = static_cast<const uint8_t*>(p.c.v_codes);
        if (there == ~0u && p.c.block_size % 16 == 0) {  // tiles begin at multiples of 16: every 16 tokens lie one behind the other
            const int64_t first = __shfl_sync(~0u, at, 0), second = kTok == 32 ? __shfl_sync(~0u, at, 16) - 16 : first;
            pieces_halves<kKRow>(stage + l.put_k, k + first * kKRow, k + second * kKRow, [](int) { return 0u; });
            pieces_halves<kVRow>(stage + l.put_v, v + first * kVRow, v + second * kVRow, moved_v);
        } else {
            pieces_paged<kKRow>(stage + l.put_k, k, at, there, [](int) { return 0u; });
            pieces_paged<kVRow>(stage + l.put_v, v, at, there, moved_v);
        }
        return there;
    }
    // first, second: where row 0 would lie for the first 16 rows and for the others
    template <int ROW, typename F>
    __device__ static __forceinline__ void pieces_halves(uint32_t dst, const uint8_t* first, const uint8_t* second, F&& moved) {
        constexpr int kCh = ROW / 16, kPieces = kCh * kTok, kPer = (kPieces + 31) / 32, kHalf = kCh * 16;
        const int lane = lane_id();
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const bool front = i * 32 + 31 < kHalf || (i * 32 < kHalf && i * 32 + lane < kHalf);
            if (kPieces % 32 == 0 || i * 32 + lane < kPieces) copy16((dst ^ moved(i)) + i * 512, (front ? first : second) + (i * 32 + lane) * 16);
        }
    }
    template <int ROW, typename F>
    __device__ static __forceinline__ void pieces_paged(uint32_t dst, const uint8_t* src, int64_t mine, uint32_t there, F&& moved) {
        constexpr int kCh = ROW / 16, kPieces = kCh * kTok, kPer = (kPieces + 31) / 32;
        const int lane = lane_id();
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int idx = i * 32 + lane, r = idx / kCh, ch = idx - r * kCh;
            const int64_t row = __shfl_sync(~0u, mine, r & 31);
            if (kPieces % 32 == 0 || idx < kPieces) copy16((dst ^ moved(i)) + i * 512, src + row * ROW + ch * 16, (there >> r) & 1u);
        }
    }

    // The same for rows that follow one another, the sequence's first one at row `row`: tokens t0 .., those from `seen` to n - 1.
    __device__ static __forceinline__ uint32_t copy_run(const AttendParams& p, const Lane& l, uint32_t stage, int64_t row, int t0, int seen, int n) {
        const int lane = lane_id();
        const int64_t at = row + t0;
        const uint32_t ks = stage + kKBytes + kVBytes + lane * kSRow;
        const uint8_t* const k = static_cast<const uint8_t*>(p.c.k_codes) + at * kKRow;
        const uint8_t* const v = static_cast<const uint8_t*>(p.c.v_codes) + at * kVRow;
        const uint8_t* const k_scale = static_cast<const uint8_t*>(p.c.k_scales) + (at + lane) * kSRow;
        const uint8_t* const v_scale = static_cast<const uint8_t*>(p.c.v_scales) + (at + lane) * kSRow;
        uint32_t there = ~0u;
        if (t0 >= seen && t0 + kTok <= n) {  // nearly always
            if (kTok == 32 || lane < kTok) {
                copy_small<kSRow>(ks, k_scale);
                copy_small<kSRow>(ks + kSBytes, v_scale);
            }
            pieces_run<kKRow, true>(stage + l.put_k, k, there, [](int) { return 0u; });
            pieces_run<kVRow, true>(stage + l.put_v, v, there, moved_v);
        } else {
            const int t = t0 + (lane & (kTok - 1));
            const bool is = t >= seen && t < n;
            there = __ballot_sync(~0u, is);
            if (kTok == 32 || lane < kTok) {
                copy_small<kSRow>(ks, is ? k_scale : static_cast<const uint8_t*>(p.c.k_scales), is);
                copy_small<kSRow>(ks + kSBytes, is ? v_scale : static_cast<const uint8_t*>(p.c.v_scales), is);
            }
            pieces_run<kKRow, false>(stage + l.put_k, k, there, [](int) { return 0u; });
            pieces_run<kVRow, false>(stage + l.put_v, v, there, moved_v);
        }
        return there;
    }
    template <int ROW, bool kAll, typename F>
    __device__ static __forceinline__ void pieces_run(uint32_t dst, const uint8_t* src, uint32_t there, F&& moved) {
        constexpr int kCh = ROW / 16, kPieces = kCh * kTok, kPer = (kPieces + 31) / 32;
        const int lane = lane_id();
        const uint8_t* const from = src + lane * 16;
        const uint8_t* const some = src + (there != 0 ? __ffs(there) - 1 : 0) * ROW;  // a row that is there, for the address of those that are not
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int idx = i * 32 + lane, r = idx / kCh;
            if (kPieces % 32 == 0 || idx < kPieces) {
                if constexpr (kAll) {
                    copy16((dst ^ moved(i)) + i * 512, from + i * 512);
                } else {
                    const bool is = (there >> r) & 1u;
                    copy16((dst ^ moved(i)) + i * 512, is ? from + i * 512 : some, is);
                }
            }
        }
    }

    // Codes as fp16 numbers, as stored or centred: of bits 2 .. 5 and 6 .. 9 of 16-bit halves, or of two bytes.
    template <bool kCentred>
    __device__ static __forceinline__ void pieces4(uint32_t x, uint32_t& low, uint32_t& high) {
        if constexpr (kCentred) {
            low = half_sub(and_or(x, 0x003c003cu, 0x64006400u), 0x64206420u);   // 1024 + 4 c less 1024 + 32
            high = half_sub(and_or(x, 0x03c003c0u, 0x64006400u), 0x66006600u);  // 1024 + 64 c less 1024 + 512
        } else {
            low = x & 0x003c003cu;
            high = x & 0x03c003c0u;
        }
    }
    template <bool kCentred>
    __device__ static __forceinline__ uint32_t piece8(uint32_t x, int sel) {
        return kCentred ? half_sub(__byte_perm(x, 0x64646464u, sel), 0x64806480u) : __byte_perm(x, 0, sel);
    }

    // A row's codes of half a group as operand pieces (a0 and a2, or a1 and a3).
    template <int STEP>
    __device__ static __forceinline__ void k_piece(const uint32_t* w, uint32_t& first, uint32_t& second) {
        if constexpr (KB == 4) {
            pieces4<kF32>(STEP == 0 ? w[0] : __funnelshift_r(w[0], w[0], 8), first, second);
        } else {
            first = piece8<kF32>(w[STEP], 0x4140);
            second = piece8<kF32>(w[STEP], 0x4342);
        }
    }

    // The tokens of a stage, t0 the first.
    __device__ static __forceinline__ void fold(const AttendParams& p, const Lane& l, Warp& w, Refs& refs, const Prepared& prepared, uint32_t stage, int t0,
                                                uint32_t there) {
        const int lane = lane_id(), gid = lane >> 2, tig = lane & 3;
        const uint32_t ks = stage + kKBytes + kVBytes, vs = ks + kSBytes;
        constexpr int kKPiece = NG * KB;   // bytes of a row that a lane reads
        float s[MT][NT][4];
        {
            Words<kKPiece> k[MT][2];
            Words<kSRow> scales[MT][2];
            float acc[MT][NT][4];
#pragma unroll
            for (int h = 0; h < MT; ++h) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    load_k(k[h][i], stage + l.k, h * 16 + i * 8);
                    scales[h][i].load(ks + (h * 16 + i * 8 + gid) * kSRow);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[h][nt][e] = 0.0f;
                if constexpr (!kF32) {
                    uint32_t a0, a1;  // key scales of the two rows, groups 2 tig and 2 tig + 1 of as many as there are
                    const uint32_t at = ks + (h * 16 + gid) * kSRow + tig % (kSG / 2) * 4;
                    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(a0) : "r"(at) : "memory");
                    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(a1) : "r"(at + 8 * kSRow) : "memory");
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = 0; i < kOffs; i += 2) mma_bf16(acc[h][nt], a0, a1, a0, a1, w.off[nt][i], w.off[nt][i + 1]);
                }
            }
#pragma unroll
            for (int u = 0; u < NG; ++u) {
                uint4 q[NT];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) q[nt] = prepared.queries[(nt * NG + u) * 32 + lane];
#pragma unroll
                for (int h = 0; h < MT; ++h) {
                    uint32_t a[2][4];
                    constexpr int kW = KB / 4;  // words of a lane's piece of a group
                    k_piece<0>(k[h][0].w + u * kW, a[0][0], a[0][2]);
                    k_piece<0>(k[h][1].w + u * kW, a[0][1], a[0][3]);
                    k_piece<1>(k[h][0].w + u * kW, a[1][0], a[1][2]);
                    k_piece<1>(k[h][1].w + u * kW, a[1][1], a[1][3]);
                    const uint32_t s0 = scales[h][0].w[u >> 1], s1 = scales[h][1].w[u >> 1];
                    const float down = kF32 ? 0x1p-16f : 1.0f;
                    const float f0 = __uint_as_float(u & 1 ? s0 & 0xffff0000u : s0 << 16) * down;
                    const float f1 = __uint_as_float(u & 1 ? s1 & 0xffff0000u : s1 << 16) * down;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float d[4];
                        mma_new(d, a[0][0], a[0][1], a[0][2], a[0][3], q[nt].x, q[nt].y);
                        mma(d, a[1][0], a[1][1], a[1][2], a[1][3], q[nt].z, q[nt].w);
                        acc[h][nt][0] = fmaf(f0, d[0], acc[h][nt][0]);
                        acc[h][nt][1] = fmaf(f0, d[1], acc[h][nt][1]);
                        acc[h][nt][2] = fmaf(f1, d[2], acc[h][nt][2]);
                        acc[h][nt][3] = fmaf(f1, d[3], acc[h][nt][3]);
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < MT; ++h)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[h][nt][e] = kF32 ? acc[h][nt][e] + __shfl_xor_sync(~0u, acc[h][nt][e], 2) : acc[h][nt][e];
        }
        if (w.apart != 0) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float f = prepared.columns[col_of(nt, 2 * tig + (e & 1))].f;
#pragma unroll
                    for (int h = 0; h < MT; ++h) s[h][nt][e] *= f;
                }
            if (w.apart & 2) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float rest = prepared.rest[col_of(nt, 2 * tig + (e & 1))];
#pragma unroll
                        for (int h = 0; h < MT; ++h) s[h][nt][e] *= rest;
                    }
            }
            if (p.cap > 0.0f) {
                const float down = 1.0f / p.cap;
#pragma unroll
                for (int h = 0; h < MT; ++h)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[h][nt][e] = tanhf(s[h][nt][e] * down) * p.cap;
            }
            if (p.slopes != nullptr) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const Column c = prepared.columns[col_of(nt, 2 * tig + (e & 1))];
#pragma unroll
                        for (int h = 0; h < MT; ++h) s[h][nt][e] -= c.slope * static_cast<float>(c.lim - 1 - (t0 + h * 16 + (e >> 1) * 8 + gid));
                    }
            }
        }
        // Relative to the references, which move where a score has outgrown its own by more than 2^8 (or may be the first one seen).
        const bool masked = there != ~0u || t0 < w.all_lo || t0 + kTok > w.all_lim;  // the stage has a token that some column does not see
        uint32_t hidden = 0;                                                         // then: a bit per score of this lane
        bool move = masked || w.fresh;
        if (!move) {
            float most = kNegInf;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int h = 0; h < MT; ++h) {
                        s[h][nt][e] = fmaf(s[h][nt][e], w.f[nt][e & 1], -w.ref[nt][e & 1]);
                        most = fmaxf(most, s[h][nt][e]);
                    }
            move = __any_sync(~0u, most > static_cast<float>(kLag + kShift));
            if (move) {
#pragma unroll
                for (int h = 0; h < MT; ++h)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[h][nt][e] += w.ref[nt][e & 1];
            }
        } else {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const Column c = prepared.columns[col_of(nt, 2 * tig + (e & 1))];
#pragma unroll
                    for (int h = 0; h < MT; ++h) {
                        const int r = h * 16 + (e >> 1) * 8 + gid, t = t0 + r;
                        s[h][nt][e] *= w.f[nt][e & 1];
                        if (!((there >> r) & 1u) || t < c.lo || t >= c.lim) {
                            s[h][nt][e] = kNegInf;
                            hidden |= 1u << ((h * NT + nt) * 4 + e);
                        }
                    }
                }
            w.fresh = w.fresh && masked;
        }
        if (move) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float top = kNegInf;
#pragma unroll
                    for (int h = 0; h < MT; ++h) top = fmaxf(top, fmaxf(s[h][nt][e], s[h][nt][e + 2]));
#pragma unroll
                    for (int d = 4; d <= 16; d <<= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
                    top = fmaxf(top - kShift, w.ref[nt][e]);
                    const float by = top == w.ref[nt][e] ? 1.0f : ex2(w.ref[nt][e] - top);
                    w.ref[nt][e] = top;
                    w.sum[nt][e] *= by;
#pragma unroll
                    for (int j = 0; j < NG * 2; ++j) w.o[nt][j][e] *= by, w.o[nt][j][e + 2] *= by;
#pragma unroll
                    for (int h = 0; h < MT; ++h) s[h][nt][e] -= top, s[h][nt][e + 2] -= top;
                }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int h = 0; h < MT; ++h) {
                    s[h][nt][e] = ex2(s[h][nt][e]);
                    s[h][nt][e + 2] = ex2(s[h][nt][e + 2]);
                    w.sum[nt][e] += s[h][nt][e] + s[h][nt][e + 2];
                }
        // Value scales relative to their references; one vote on whether there are references yet and all scales lie where fp16 holds them (zeros do).
        Words<kSRow> mine;
        mine.load(vs + (lane & (kTok - 1)) * kSRow);
        float x[kSG];
        const bool first = refs.by[0] == 0.0f;
        if (__builtin_expect(__any_sync(~0u, relative(refs, mine, x) || first), 0)) {
            bool far = true;
            if (first) {
                first_refs(refs, mine);
                far = __any_sync(~0u, relative(refs, mine, x));
            }
            if (far) {
                far_scales(w, refs, stage, s, hidden, mine);
                relative(refs, mine, x);
            }
        }
        if constexpr (kF32)
            values_f32(l, w, stage, s, x);
        else
            values_bf16(l, w, stage, s, x);
    }

    // x = a token's scales relative to their references (exact); whether one lies outside 2^-kSpan .. 2 and is not zero.
    __device__ static __forceinline__ bool relative(const Refs& refs, const Words<kSRow>& mine, float (&x)[kSG]) {
        constexpr uint32_t kLeast = (127 - kSpan) << 23, kMost = 128 << 23;
        uint32_t least = ~0u, most = 0;
#pragma unroll
        for (int u = 0; u < kSG; ++u) {
            x[u] = __uint_as_float(u & 1 ? mine.w[u >> 1] & 0xffff0000u : mine.w[u >> 1] << 16) * refs.by[u];
            least = min(least, __float_as_uint(x[u]) - 1);
            most = max(most, __float_as_uint(x[u]));
        }
        return least < kLeast - 1 || most >= kMost;
    }

    // The references of a pair's first stage: a little above its largest scales.  (All lanes write the same.)
    __device__ static __forceinline__ void first_refs(Refs& refs, const Words<kSRow>& mine) {
        __syncwarp();
#pragma unroll
        for (int u = 0; u < kSG; ++u) {
            const uint32_t y = u & 1 ? mine.w[u >> 1] >> 16 : mine.w[u >> 1] & 0xffffu;
            const int e = static_cast<int>(__reduce_max_sync(~0u, y < 0x7f80u ? y : 0u) >> 7) + kHeadroom;
            refs.set(u, min(max(e, 1), 253), e);
        }
        __syncwarp();
    }

    // A stage with scales outside their references' range, or NaN ones.  References move where most of a group's scales lie outside; what lies outside all
    // the same is multiplied here, and `mine` keeps the rest.  Groups of NaN spoil their elements of the columns that see their token.
    // (A loop over the groups that is not unrolled: it is run seldom, and should take neither registers nor instruction cache.)
    __device__ static __forceinline__ void far_scales(Warp& w, Refs& refs, uint32_t stage, const float (&weight)[MT][NT][4], uint32_t hidden, Words<kSRow>& mine) {
        const int lane = lane_id(), gid = lane >> 2, tig = lane & 3;
#pragma unroll 1
        for (int u = 0; u < NG; ++u) {
            uint32_t y = mine.w[0];
#pragma unroll
            for (int i = 1; i < kSG / 2; ++i) y = (u >> 1) == i ? mine.w[i] : y;
            y = u & 1 ? y >> 16 : y & 0xffffu;
            const uint32_t bad = __ballot_sync(~0u, y >= 0x7f80u);  // a bit per token, like those below
            y = y >= 0x7f80u ? 0u : y;
            const int e = y != 0 ? max(static_cast<int>(y >> 7), 1) : 0, old = refs.exponent(u);
            const auto outside = [&](int ref) { return e != 0 && (e > ref || e + kSpan < ref); };
            const int largest = static_cast<int>(__reduce_max_sync(~0u, static_cast<uint32_t>(e)));
            const int largest_outside = static_cast<int>(__reduce_max_sync(~0u, outside(old) ? static_cast<uint32_t>(e) : 0u));
            const bool moves = 2 * __popc(__ballot_sync(~0u, outside(old))) > __popc(__ballot_sync(~0u, e != 0));
            const int most = max(max(refs.most[u], old), largest);
            const int now = max(moves ? min(largest_outside + kHeadroom, 253) : old, most - kReach);
            const uint32_t far = __ballot_sync(~0u, outside(now));
            const float x = outside(now) ? __uint_as_float(y << 16) * __int_as_float((254 - now) << 23) : 0.0f;
            __syncwarp();
            refs.set(u, now, most);
            __syncwarp();
            float add[NT][2][4] = {};
            if (far != 0) far_products(stage, weight, u, x, add);
            if (bad != 0) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        bool spoilt = false;
#pragma unroll
                        for (int h = 0; h < MT; ++h)
#pragma unroll
                            for (int i = 0; i < 2; ++i)
                                spoilt = spoilt || (((bad >> (h * 16 + i * 8 + gid)) & 1u) && !((hidden >> ((h * NT + nt) * 4 + i * 2 + c)) & 1u));
                        const uint32_t lanes = __ballot_sync(~0u, spoilt);
                        const float nan = ((lanes >> tig) & 0x11111111u) != 0 ? __int_as_float(0x7fc00000) : 0.0f;
#pragma unroll
                        for (int j = 0; j < 2; ++j) add[nt][j][c] += nan, add[nt][j][c + 2] += nan;
                    }
            }
            // 2^(old - now) in two factors, each of them a normal number
            const int half = (old - now) / 2;
            const float by0 = __int_as_float((127 + half) << 23), by1 = __int_as_float((127 + old - now - half) << 23);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < NG * 2; ++j)
#pragma unroll
                    for (int c = 0; c < 4; ++c) w.o[nt][j][c] = (j >> 1) == u ? fmaf(w.o[nt][j][c] * by0, by1, add[nt][j & 1][c]) : w.o[nt][j][c];
            y = outside(now) ? 0u : y;
#pragma unroll
            for (int i = 0; i < kSG / 2; ++i)
                mine.w[i] = (u >> 1) != i ? mine.w[i] : u & 1 ? (mine.w[i] & 0xffffu) | y << 16 : (mine.w[i] & 0xffff0000u) | y;
        }
    }

    // add = the products of group u's codes with weights times x, a scale per lane's token (0: no part in this): bfloat16 numbers, which hold codes as they
    // are, and weights times scales as sums of two (fp32: three, the second in the tile's other half and the third in a product of its own).
    __device__ static __forceinline__ void far_products(uint32_t stage, const float (&weight)[MT][NT][4], int u, float x, float (&add)[NT][2][4]) {
        const int lane = lane_id(), gid = lane >> 2, tig = lane & 3;
        const float rest = kF32 && tig >= 2 ? 1.0f : 0.0f;  // (a number and no branch, as below)
        const auto pack = [](float lo, float hi) {
            const __nv_bfloat162 both = __floats2bfloat162_rn(lo, hi);
            return *reinterpret_cast<const uint32_t*>(&both);
        };
        const auto less = [](uint32_t y, float by, float& lo, float& hi) {
            lo = fmaf(-by, __uint_as_float(y << 16), lo), hi = fmaf(-by, __uint_as_float(y & 0xffff0000u), hi);
        };
        const int at = gid * (NG * VB / 2) + u * (VB / 2);
#pragma unroll
        for (int h = 0; h < MT; ++h) {
            struct Piece {
                uint32_t w[1];
            } v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = h * 16 + (i >> 1) * 8 + 2 * tig + (i & 1);
                const uint32_t from = stage + kKBytes + (NG == 3 ? r * kVRow + at : v_place(r, at / 16) + at % 16);
                if constexpr (VB == 4) {
                    uint16_t y;
                    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(y) : "r"(from) : "memory");
                    v[i].w[0] = y;
                } else {
                    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[i].w[0]) : "r"(from) : "memory");
                }
            }
            uint32_t a[2][4];
            v_pieces(v, 0, a);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 y = unpack_half(a[j][i]);
                    a[j][i] = pack(y.x, y.y);
                }
            const float f0 = __shfl_sync(~0u, x, h * 16 + gid), f1 = __shfl_sync(~0u, x, h * 16 + 8 + gid);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float y[4] = {weight[h][nt][0] * f0, weight[h][nt][1] * f0, weight[h][nt][2] * f1, weight[h][nt][3] * f1};
                uint32_t b[2][2];  // [part][tokens gid or gid + 8]
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t first = pack(y[2 * i], y[2 * i + 1]);
                    if constexpr (kF32) {
                        less(first, rest, y[2 * i], y[2 * i + 1]);
                        b[0][i] = pack(y[2 * i], y[2 * i + 1]);
                        less(first, 1.0f - rest, y[2 * i], y[2 * i + 1]);
                        less(pack(y[2 * i], y[2 * i + 1]), 1.0f, y[2 * i], y[2 * i + 1]);
                        b[1][i] = pack(y[2 * i] * (1.0f - rest), y[2 * i + 1] * (1.0f - rest));
                    } else {
                        b[0][i] = first;
                        less(first, 1.0f, y[2 * i], y[2 * i + 1]);
                        b[1][i] = pack(y[2 * i], y[2 * i + 1]);
                    }
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    b[k][0] = transpose8x8(b[k][0]), b[k][1] = transpose8x8(b[k][1]);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float d[4] = {};
                        mma_bf16(d, a[j][0], a[j][1], a[j][2], a[j][3], b[k][0], b[k][1]);
#pragma unroll
                        for (int c = 0; c < 4; ++c) add[nt][j][c] += d[c];
                    }
                }
            }
        }
    }

    // O += V^T P for fp32: weights times value scales in 32 bits, then as two fp16 numbers.
    __device__ static __forceinline__ void values_f32(const Lane& l, Warp& w, uint32_t stage, const float (&weight)[MT][NT][4], const float (&x)[kSG]) {
        const int lane = lane_id(), gid = lane >> 2, tig = lane & 3;
        // (A number, and no branch on the lane: the compiler may lay such a branch around what follows, and instructions of the whole warp are among it.)
        const float rest = tig >= 2 ? 1.0f : 0.0f;
        // scales relative to their references, bfloat16 numbers as before, in place
        Words<kSRow> mine;
#pragma unroll
        for (int i = 0; i < kSG / 2; ++i) mine.w[i] = __byte_perm(__float_as_uint(x[2 * i]), __float_as_uint(x[2 * i + 1]), 0x7632);
        __syncwarp();
        mine.store(stage + kKBytes + kVBytes + kSBytes + (lane & (kTok - 1)) * kSRow);
        __syncwarp();
        const uint32_t vs = stage + kKBytes + kVBytes + kSBytes;
        const uint32_t values_at[2] = {stage + kKBytes + l.v, stage + kKBytes + l.v_next()};
#pragma unroll
        for (int h = 0; h < MT; ++h) {
            const int r = h * 16 + gid;
            Words<kSRow> s0, s1;
            s0.load(vs + r * kSRow);
            s1.load(vs + (r + 8) * kSRow);
            Words<NG * VB / 2> v[4];  // tokens 2 tig, 2 tig + 1, 2 tig + 8, 2 tig + 9
#pragma unroll
            for (int i = 0; i < 4; ++i) load_v(v[i], values_at[i & 1], h * 16 + (i >> 1) * 8);
#pragma unroll
            for (int u = 0; u < NG; ++u) {
                const float f0 = __uint_as_float(u & 1 ? s0.w[u >> 1] & 0xffff0000u : s0.w[u >> 1] << 16);
                const float f1 = __uint_as_float(u & 1 ? s1.w[u >> 1] & 0xffff0000u : s1.w[u >> 1] << 16);
                const float y[4] = {weight[h][0][0] * f0, weight[h][0][1] * f0, weight[h][0][2] * f1, weight[h][0][3] * f1};
                // lanes of the second half have what fp16 leaves: less `rest` times the rounded number, and rounded again
                const float2 g0 = unpack_half(pack_half(y[0], y[1])), g1 = unpack_half(pack_half(y[2], y[3]));
                const uint32_t b0 = transpose8x8(pack_half(fmaf(-rest, g0.x, y[0]), fmaf(-rest, g0.y, y[1])));
                const uint32_t b1 = transpose8x8(pack_half(fmaf(-rest, g1.x, y[2]), fmaf(-rest, g1.y, y[3])));
                uint32_t a[2][4];
                v_pieces(v, u, a);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float d[4];
                    mma_new(d, a[j][0], a[j][1], a[j][2], a[j][3], b0, b1);
#pragma unroll
                    for (int e = 0; e < 4; ++e) w.o[0][2 * u + j][e] += d[e];
                }
            }
        }
    }

    // O += V^T P for bfloat16: weights go to the operand's layout as fp16 numbers and meet the value scales there, two per instruction.  The scales
    // are made fp16 (relative to their references, which is exact) and brought into that order by the lane that has the token, in place.
    __device__ static __forceinline__ void values_bf16(const Lane& l, Warp& w, uint32_t stage, const float (&weight)[MT][NT][4], const float (&x)[kSG]) {
        const int lane = lane_id(), gid = lane >> 2, tig = lane & 3;
        constexpr int kWords = kSG / 2;
        const uint32_t vs = stage + kKBytes + kVBytes + kSBytes;
        const uint32_t values_at[2] = {stage + kKBytes + l.v, stage + kKBytes + l.v_next()};
        {
            uint32_t c[kWords];
#pragma unroll
            for (int i = 0; i < kWords; ++i) c[i] = pack_half(x[2 * i], x[2 * i + 1]);
            const bool odd = lane & 1;
            const int r = lane & (kTok - 1);
            const uint32_t to = vs + (((r >> 4) * 4 + ((r & 7) >> 1)) * 2 + ((r >> 3) & 1)) * (kSG * 4);
            __syncwarp();  // every lane has its row
            if constexpr (kWords == 1) {
                const uint32_t other = __shfl_xor_sync(~0u, c[0], 1);
                const uint32_t y = odd ? __byte_perm(other, c[0], 0x7632) : __byte_perm(c[0], other, 0x5410);
                if (kTok == 32 || lane < kTok) asm volatile("st.shared.u32 [%0], %1;" ::"r"(to + odd * 4), "r"(y) : "memory");
            } else {
                uint32_t y[kWords];
#pragma unroll
                for (int i = 0; i < kWords / 2; ++i) {
                    const uint32_t other = __shfl_xor_sync(~0u, odd ? c[i] : c[i + kWords / 2], 1);
                    const uint32_t own = odd ? c[i + kWords / 2] : c[i];
                    const uint32_t first = odd ? other : own, second = odd ? own : other;
                    y[2 * i] = __byte_perm(first, second, 0x5410);
                    y[2 * i + 1] = __byte_perm(first, second, 0x7632);
                }
                if (kTok == 32 || lane < kTok) {
#pragma unroll
                    for (int i = 0; i < kWords; i += 2)
                        asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(to + odd * kWords * 4 + i * 4), "r"(y[i]), "r"(y[i + 1]) : "memory");
                }
            }
            __syncwarp();
        }
#pragma unroll
        for (int h = 0; h < MT; ++h) {
            Words<2 * kSG * 4> sv;  // groups of tokens 2 tig and 2 tig + 1, then of 2 tig + 8 and 2 tig + 9
            sv.load(vs + (h * 4 + tig) * (2 * kSG * 4));
            Words<NG * VB / 2> v[4];  // tokens 2 tig, 2 tig + 1, 2 tig + 8, 2 tig + 9
#pragma unroll
            for (int i = 0; i < 4; ++i) load_v(v[i], values_at[i & 1], h * 16 + (i >> 1) * 8);
            uint32_t weights[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 2; ++i) weights[nt][i] = transpose8x8(pack_half(weight[h][nt][2 * i], weight[h][nt][2 * i + 1]));
#pragma unroll
            for (int u = 0; u < NG; ++u) {
                uint32_t b[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 2; ++i) b[nt][i] = half_mul(weights[nt][i], sv.w[i * kSG + u]);
                uint32_t a[2][4];
                v_pieces(v, u, a);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    mma(w.o[nt][2 * u], a[0][0], a[0][1], a[0][2], a[0][3], b[nt][0], b[nt][1]);
                    mma(w.o[nt][2 * u + 1], a[1][0], a[1][1], a[1][2], a[1][3], b[nt][0], b[nt][1]);
                }
            }
        }
    }

    // a[j]: elements 4 gid + 2 j (pieces 0 and 2) and + 1 (pieces 1 and 3) of the group, of tokens 2 tig, + 1 (0 and 1), 2 tig + 8, + 9.
    template <typename W>
    __device__ static __forceinline__ void v_pieces(const W (&v)[4], int u, uint32_t (&a)[2][4]) {
        if constexpr (VB == 4) {
            const int sel = u & 1 ? 0x7632 : 0x5410;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t x = __byte_perm(v[2 * i].w[u >> 1], v[2 * i + 1].w[u >> 1], sel), y = __byte_perm(x, 0, 0x2301);
                pieces4<true>(x, a[0][2 * i], a[0][2 * i + 1]);
                pieces4<true>(y, a[1][2 * i], a[1][2 * i + 1]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t x = __byte_perm(v[2 * i].w[u], v[2 * i + 1].w[u], 0x5410), y = __byte_perm(v[2 * i].w[u], v[2 * i + 1].w[u], 0x7632);
                a[0][2 * i] = piece8<true>(x, 0x4240);
                a[0][2 * i + 1] = piece8<true>(x, 0x4341);
                a[1][2 * i] = piece8<true>(y, 0x4240);
                a[1][2 * i + 1] = piece8<true>(y, 0x4341);
            }
        }
    }

    // A lane's piece of a row `rows` (a multiple of 8) behind the one at `at`: whole 16-byte pieces, which were moved about, or a part of one.
    template <typename W>
    __device__ static __forceinline__ void load_k(W& k, uint32_t at, int rows) {
        if constexpr (NG * KB > 16 && NG != 3) {
#pragma unroll
            for (int i = 0; i < NG * KB / 16; ++i) k.load16((at ^ (i * 16)) + rows * kKRow, 4 * i);
        } else {
            k.load(at + rows * kKRow);
        }
    }
    template <typename W>
    __device__ static __forceinline__ void load_v(W& v, uint32_t at, int rows) {
        if constexpr (NG * VB / 2 > 16) {
#pragma unroll
            for (int i = 0; i < NG * VB / 32; ++i) v.load16((at ^ (i * 16)) + rows * kVRow, 4 * i);
        } else {
            v.load(at + rows * kVRow);
        }
    }

    // This warp's reference and sum of each column into ml [kCols][2]; sums of all lanes are left in w.sum.
    __device__ static __forceinline__ void leave_sums(Warp& w, float* ml) {
        const int lane = lane_id(), gid = lane >> 2, tig = lane & 3;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int d = 4; d <= 16; d <<= 1) w.sum[nt][e] += __shfl_xor_sync(~0u, w.sum[nt][e], d);
                if (gid == 0 && (!kF32 || tig < 2)) {
                    float* const to = ml + col_of(nt, 2 * tig + e) * 2;
                    to[0] = w.ref[nt][e], to[1] = w.sum[nt][e];
                }
            }
    }
    // Its normalised result for columns c0 .. c0 + kRoundCols - 1 into o [kRoundCols][D].
    __device__ static __forceinline__ void leave(const Warp& w, const Refs& refs, uint32_t o, int c0) {
        const int lane = lane_id(), gid = lane >> 2, tig = lane & 3;
        // the accumulators are in units of their group's reference times kValueUnit, and of 2^-kShift like the sums
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int col = col_of(nt, 2 * tig + e) - c0;
                const float sum = w.sum[nt][e], by = sum == 0.0f ? 0.0f : __frcp_rn(sum) * (1.0f / kValueUnit);
#pragma unroll
                for (int u = 0; u < NG; ++u) {
                    const float up = __int_as_float(refs.exponent(u) << 23);
                    float x[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int j = 2 * u + (i >> 1), at = (i & 1) * 2 + e;
                        const float times = VB == 4 && (i & 1) ? 16.0f : 1.0f;
                        const float y = kF32 ? w.o[nt][j][at] + __shfl_xor_sync(~0u, w.o[nt][j][at], 2) : w.o[nt][j][at];
                        x[i] = y * (by / times) * up;
                    }
                    if (col >= 0 && col < kRoundCols && (!kF32 || tig < 2))
                        asm volatile("st.shared.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(o + (col * D + u * kGroup + gid * 4) * 4), "f"(x[0]), "f"(x[1]),
                                     "f"(x[2]), "f"(x[3])
                                     : "memory");
                }
            }
    }

    __device__ static __forceinline__ void store(T* out, const float (&x)[4]) {
        if constexpr (kF32) {
            *reinterpret_cast<float4*>(out) = make_float4(x[0], x[1], x[2], x[3]);
        } else {
            __nv_bfloat162 h[2] = {__floats2bfloat162_rn(x[0], x[1]), __floats2bfloat162_rn(x[2], x[3])};
            *reinterpret_cast<uint2*>(out) = *reinterpret_cast<uint2*>(h);
        }
    }
    __device__ static __forceinline__ T* out_row(const AttendParams& p, int b, int g, int mine) {
        const int i = mine / p.R, h = g * p.R + mine - i * p.R;
        return static_cast<T*>(p.out) + (static_cast<int64_t>(b) * p.m + i) * p.ld_out + static_cast<int64_t>(h) * D;
    }
};

// Tokens of sequence b, and the first one that any query of it sees, rounded down to a whole number of tiles.
template <int TOK>
__device__ __forceinline__ int attended(const AttendParams& p, int b, int& first) {
    const int n = min(max(tokens_held(p.c, b) + p.len_bias, 0), p.T_upper);
    first = first_seen(p, n) / TOK * TOK;
    return n;
}
template <int TOK>
__device__ __forceinline__ int tiles_of(const AttendParams& p, int b) {  // at least one: an empty sequence's rows are written too
    int first;
    const int n = attended<TOK>(p, b, first);
    return max(1, (n - first + TOK - 1) / TOK);
}

// How the tiles of all (sequence, head, column tile) pairs, laid end to end, are cut into pieces of the same cost.  A pair costs what kPairCost tiles do on
// top of its tiles: the units before its first tile are nobody's work, but count.  (Without them a CTA whose sequences are short had several times
// the work of one whose sequences are long: 359 -> 286 us for 64 sequences of 512 .. 8192 tokens.)
constexpr uint32_t kPairCost = 24;
struct Cut {
    uint32_t total, each, more;  // units; of a piece (the first `more` have one more)
    __device__ __forceinline__ Cut(uint32_t units, uint32_t pieces) : total(units), each(units / pieces), more(units - units / pieces * pieces) {}
    __device__ __forceinline__ uint32_t start(uint32_t i) const { return each * i + min(i, more); }
    __device__ __forceinline__ uint32_t piece_of(uint32_t u) const {
        return u < more * (each + 1) ? u / (each + 1) : more + (u - more * (each + 1)) / each;
    }
};

// A place in a CTA's run of tiles: tiles tile .. end - 1 of the pair (b, g, ct), whose first is token `first` of the sequence's n, are its next ones, and `left`
// more units follow in other pairs.  In shared memory, one for each warp (all lanes write the same): it is needed from pair to pair only.
template <int TOK>
struct Place {
    int b, g, ct, n, first, tiles, tile, end, left;
    uint32_t unit;  // the pair's first unit

    __device__ __forceinline__ void sequence(const AttendParams& p) {
        n = attended<TOK>(p, b, first);
        tiles = max(1, (n - first + TOK - 1) / TOK);
    }
    __device__ __forceinline__ void whole() { tile = 0, end = tiles, left = 0; }
    // The pair's tiles from its unit `from` on, of a run of `run` units; maybe none.
    __device__ __forceinline__ void take(int from, int run) {
        const int cost = static_cast<int>(kPairCost), to = min(from + run, tiles + cost);
        tile = max(from - cost, 0), end = max(to - cost, 0);
        left = run - (to - from);
    }
    // The same of the run's next pair that has tiles for it; false where there is none.
    __device__ __forceinline__ bool next(const AttendParams& p) {
        Place at = *this;
        do {
            if (at.left <= 0) return false;
            at.unit += at.tiles + kPairCost;
            if (++at.ct == p.col_tiles) {
                at.ct = 0;
                if (++at.g == p.c.G) at.g = 0, ++at.b, at.sequence(p);
            }
            at.take(0, at.left);
        } while (at.tile >= at.end);
        __syncwarp();
        *this = at;
        __syncwarp();
        return true;
    }

    // The CTA's run: a piece of all units.  Every thread adds up a stretch of sequences; the one in whose stretch the piece begins knows where.
    template <int THREADS>
    __device__ static __forceinline__ uint32_t find_run(const AttendParams& p, Place* found) {
        __shared__ uint32_t sums[THREADS / 32];
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, stretch = (p.c.B + THREADS - 1) / THREADS;
        const int from = threadIdx.x * stretch, to = min(from + stretch, p.c.B);
        const uint32_t each = p.c.G * p.col_tiles;
        uint32_t mine = 0;
        for (int b = from; b < to; ++b) mine += (tiles_of<TOK>(p, b) + kPairCost) * each;
        uint32_t sum = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t other = __shfl_up_sync(~0u, sum, d);
            if (lane >= d) sum += other;
        }
        if (lane == 31) sums[warp] = sum;
        if (threadIdx.x == 0) found->left = -1;
        __syncthreads();
        uint32_t total = 0, before = sum - mine;
#pragma unroll
        for (int i = 0; i < THREADS / 32; ++i) {
            if (i < warp) before += sums[i];
            total += sums[i];
        }
        const Cut cut(total, gridDim.x);
        const uint32_t start = cut.start(blockIdx.x);
        const int run = static_cast<int>(cut.start(blockIdx.x + 1) - start);
        if (start >= before && start < before + mine && run > 0) {
            Place at;
            uint32_t first = before;
            for (at.b = from;; ++at.b) {
                at.sequence(p);
                const uint32_t next = first + (at.tiles + kPairCost) * each;
                if (start < next) break;
                first = next;
            }
            const uint32_t per = at.tiles + kPairCost, pair = (start - first) / per;
            at.g = static_cast<int>(pair) / p.col_tiles, at.ct = static_cast<int>(pair) - at.g * p.col_tiles;
            at.unit = first + pair * per;
            at.take(static_cast<int>(start - at.unit), run);
            *found = at;
        }
        __syncthreads();
        return total;
    }
};

template <typename T, int NG, int KB, int VB, int NT>
__global__ void __launch_bounds__(Ring<NG, KB, VB, NT>::kWarps * 32, Ring<NG, KB, VB, NT>::kCtas) attend_kernel(const AttendParams p) {
    using A = Attend<T, NG, KB, VB, NT>;
    constexpr int kTok = A::kTok, S = A::STAGES, W = A::WARPS, kThreads = A::kThreads, D = A::D;
    extern __shared__ __align__(128) uint8_t smem[];
    float* const ml = reinterpret_cast<float*>(smem + A::kRing);
    uint32_t* const left_at = reinterpret_cast<uint32_t*>(smem + A::kRing + A::kMl);
    auto& prepared = *reinterpret_cast<typename A::Prepared*>(smem + A::kRing + A::kMl + 16 * ((W * 4 + 15) / 16));
    __shared__ Place<kTok> now[W], ahead[W];
    __shared__ uint32_t there[W][S];  // which tokens of a stage are there
    __shared__ typename A::Refs refs[W];
    __shared__ int pieces[3];
    const int warp = threadIdx.x >> 5;
    const uint32_t ring = smem_u32(smem) + warp * S * A::kStage;
    if (p.cluster > 0) grid_launch_dependents();  // (a launch of long runs fills the SMs to its end)
    grid_dependency_wait();

    // This CTA's run of tiles, and which of a pair's tokens are this warp's: kTok from `skip` on, `step` further on the next ones.
    int step = W * kTok, skip = warp * kTok;
    typename A::Query raw;
    uint32_t total = 0;  // units of all pairs
    if (p.cluster > 0) {
        Place<kTok> at;
        const int in_all = blockIdx.x / p.cluster, each = p.c.G * p.col_tiles;
        at.b = in_all / each;
        const int pair = in_all - at.b * each;
        at.g = pair / p.col_tiles, at.ct = pair - at.g * p.col_tiles;
        A::load_query(p, raw, at.b, at.g, at.ct);
        at.sequence(p);
        at.whole();
        skip += step * (blockIdx.x - in_all * p.cluster);
        step *= p.cluster;
        now[warp] = ahead[warp] = at;
        __syncwarp();
    } else {
        __shared__ Place<kTok> found;
        total = Place<kTok>::template find_run<kThreads>(p, &found);
        if (found.left < 0) return;
        now[warp] = ahead[warp] = found;
        __syncwarp();
        if (found.tile >= found.end) {  // (the run begins with units of a pair's cost alone)
            const bool any = now[warp].next(p);
            ahead[warp].next(p);
            if (!any) return;
        }
        A::load_query(p, raw, now[warp].b, now[warp].g, now[warp].ct);  // (ahead of the copies, which would hold it up)
    }

    // Copies run ahead of the arithmetic, across pairs too: the next one is of tokens copy_t .. of the pair at ahead[warp], whose copies end at copy_end, and
    // of whose tokens those from `seen` to held - 1 are seen; `row`: where this lane's token of it lies (contiguous: the pair's first row).
    const bool paged = p.c.block_table != nullptr;
    int copy_t, copy_end, seen, held;
    int64_t row = 0;
    const auto enter = [&] {
        const Place<kTok>& at = ahead[warp];
        copy_t = at.first + at.tile * kTok + skip;
        copy_end = at.first + at.end * kTok;
        held = at.n;
        seen = first_seen(p, held);
        if (!paged) row = row_of(p.c, p.by_block, at.b, at.g, 0, nullptr);
    };
    const auto look = [&] {
        while (copy_t >= copy_end) {
            if (!ahead[warp].next(p)) return;
            enter();
        }
        if (paged) row = A::find(p, ahead[warp].b, ahead[warp].g, copy_t, seen, held);
    };
    typename A::Lane l;
    l.set();
    const auto copy = [&](int slot) {
        if (copy_t < copy_end) {
            const uint32_t to = ring + slot * A::kStage;
            const uint32_t is = paged ? A::copy_paged(p, l, to, row) : A::copy_run(p, l, to, row, copy_t, seen, held);
            there[warp][slot] = is;
            copy_t += step;
            look();
        }
        copy_commit();
    };
    enter();
    look();
#pragma unroll
    for (int i = 0; i < S - 1; ++i) copy(i);

    typename A::Warp q;
    int slot = 0;
    bool first_of_run = true;
    for (;;) {
        int t = now[warp].first + now[warp].tile * kTok + skip;
        const int end = now[warp].first + now[warp].end * kTok;
        A::begin(p, q, refs[warp], raw, prepared, now[warp].g, now[warp].ct, now[warp].n);
        for (; t < end; t += step) {
            copy_wait<S - 2>();
            __syncwarp();
            copy(slot == 0 ? S - 1 : slot - 1);
            A::fold(p, l, q, refs[warp], prepared, ring + slot * A::kStage, t, there[warp][slot]);
            slot = slot == S - 1 ? 0 : slot + 1;
        }
        if (p.cluster > 1) {
            copy_wait<0>();
            cluster_arrive();  // this CTA's ring is free for the others' results
        }
        // The pair, and on to the next one, whose queries are on their way while the warps' results are put together.
        const int b = now[warp].b, g = now[warp].g, ct = now[warp].ct, tile = now[warp].tile, tiles = now[warp].tiles;
        const uint32_t unit = now[warp].unit;
        const bool whole = p.cluster == 1 || (p.cluster == 0 && tile == 0 && now[warp].end == tiles);
        const bool on = p.cluster == 0 && now[warp].next(p);
        if (on) A::load_query(p, raw, now[warp].b, now[warp].g, now[warp].ct);

        // The warps' results, in the stage of each ring that the next copy goes to (clusters: in the first one, all are free).
        const uint32_t mine = static_cast<uint32_t>((warp * S + (p.cluster > 1 ? 0 : slot == 0 ? S - 1 : slot - 1)) * A::kStage);
        A::leave_sums(q, ml + warp * A::kCols * 2);
        if ((threadIdx.x & 31) == 0) left_at[warp] = mine;
        const int used = min(p.m * p.R - ct * A::kCols, A::kCols);
        constexpr int kQuads = A::kRoundCols * D / 4, kPer = (kQuads + kThreads - 1) / kThreads;
        float kept[A::kRounds * kPer][4];
        float kept_lse[A::kRounds * kPer];
#pragma unroll
        for (int r = 0; r < A::kRounds; ++r) {
            A::leave(q, refs[warp], smem_u32(smem) + mine, r * A::kRoundCols);
            __syncthreads();
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                const int i = threadIdx.x + k * kThreads;
                const int in_round = i / (D / 4), col = r * A::kRoundCols + in_round, d = (i - in_round * (D / 4)) * 4;
                float (&x)[4] = kept[r * kPer + k];
                x[0] = x[1] = x[2] = x[3] = 0.0f;
                kept_lse[r * kPer + k] = kNegInf;
                if ((kQuads % kThreads == 0 || i < kQuads) && col < used) {
                    // (shares of 1 are what results are multiplied by: sums of exponentials times the type's largest values are not finite)
                    float top = kNegInf, total = 0.0f, share[W];
#pragma unroll
                    for (int j = 0; j < W; ++j) top = fmaxf(top, ml[(j * A::kCols + col) * 2]);
#pragma unroll
                    for (int j = 0; j < W; ++j) {
                        share[j] = ml[(j * A::kCols + col) * 2 + 1] * ex2(ml[(j * A::kCols + col) * 2] - top);
                        total += share[j];
                    }
                    const float by = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
                    for (int j = 0; j < W; ++j) {
                        const float l = share[j] * by;
                        const float4 y = *reinterpret_cast<const float4*>(smem + left_at[j] + (in_round * D + d) * 4);
                        x[0] += l * y.x, x[1] += l * y.y, x[2] += l * y.z, x[3] += l * y.w;
                    }
                    kept_lse[r * kPer + k] = total == 0.0f ? kNegInf : top + log2f(total);
                    if (whole) {
                        A::store(A::out_row(p, b, g, ct * A::kCols + col) + d, x);
                    } else if (p.cluster == 0) {
                        const int64_t at = 2ll * blockIdx.x + (first_of_run ? 0 : 1);
                        *reinterpret_cast<float4*>(p.ws_o + (at * A::kCols + col) * D + d) = make_float4(x[0], x[1], x[2], x[3]);
                        if (d == 0) p.ws_lse[at * A::kCols + col] = kept_lse[r * kPer + k];
                    }
                }
            }
            if (r + 1 < A::kRounds || p.cluster == 0) __syncthreads();
        }
        if (p.cluster > 1) {
            // One pair per cluster.  Every CTA has a share of the columns' elements, quads rank, rank + cluster, ... of them, and gets all CTAs' results for
            // it, each behind the other, into the rings (all but the first stages), and their sums to where the queries were.
            constexpr int kRoom = (S - 1) * A::kStage / 16;  // quads in a warp's ring
            static_assert(A::kCols * D / 4 + 7 <= W * kRoom && 8 * A::kCols * 4 <= NG * NT * 512, "");
            const auto where = [](int quad) { return static_cast<uint32_t>(quad / kRoom * (S * A::kStage) + A::kStage + quad % kRoom * 16); };
            const uint32_t their_lse = smem_u32(prepared.queries);
            const int rank = static_cast<int>(cluster_rank()), each = (A::kCols * D / 4 + p.cluster - 1) / p.cluster;
            cluster_wait();
#pragma unroll
            for (int k = 0; k < A::kRounds * kPer; ++k) {
                const int i = threadIdx.x + k % kPer * kThreads;
                const int quad = k / kPer * kQuads + i, col = quad / (D / 4);
                if ((kQuads % kThreads == 0 || i < kQuads) && col < used) {
                    peer_store4(peer_address(smem_u32(smem) + where(rank * each + quad / p.cluster), quad % p.cluster), kept[k]);
                    if (quad % (D / 4) == 0)
                        for (int j = 0; j < p.cluster; ++j) peer_store_u32(their_lse + (rank * A::kCols + col) * 4, j, __float_as_uint(kept_lse[k]));
                }
            }
            cluster_sync();
            const float* const lse = reinterpret_cast<const float*>(prepared.queries);
            for (int i = threadIdx.x; i * p.cluster + rank < used * (D / 4); i += kThreads) {
                const int quad = i * p.cluster + rank, col = quad / (D / 4), d = (quad - col * (D / 4)) * 4;
                float top = kNegInf, total = 0.0f, x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                for (int j = 0; j < p.cluster; ++j) top = fmaxf(top, lse[j * A::kCols + col]);
                const float ref = (top == kNegInf ? 0.0f : top) + 3.0f;  // (weights of 1 / 8 at most: sums of up to 8 results are finite)
                for (int j = 0; j < p.cluster; ++j) {
                    const float l = ex2(lse[j * A::kCols + col] - ref);
                    const float4 y = *reinterpret_cast<const float4*>(smem + where(j * each + i));
                    total += l;
                    x[0] += l * y.x, x[1] += l * y.y, x[2] += l * y.z, x[3] += l * y.w;
                }
                const float by = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] *= by;
                A::store(A::out_row(p, b, g, ct * A::kCols + col) + d, x);
            }
        } else if (p.cluster == 0 && !whole) {
            // A pair that was cut: the CTA that brings its last piece puts them together.  (The rounds' last barrier has ordered this CTA's stores.)
            if (threadIdx.x == 0) {
                const Cut cut(total, gridDim.x);
                const uint32_t first = unit;
                const int c0 = static_cast<int>(cut.piece_of(first + kPairCost)), c1 = static_cast<int>(cut.piece_of(first + kPairCost + tiles - 1));
                __threadfence();
                unsigned long long* const word = p.tickets + (static_cast<int64_t>(b) * p.c.G + g) * p.col_tiles + ct;
                // the word may hold anything: the first piece to come makes it this call's
                const unsigned long long old = *reinterpret_cast<volatile unsigned long long*>(word), own = p.call << 24;
                if (old >> 24 != p.call) atomicCAS(word, old, own);
                const int before = static_cast<int>(atomicAdd(word, 1ull) & 0xffffffu);
                const bool last = before == c1 - c0;
                if (last) {
                    atomicExch(word, 0ull);  // (a launch replayed from a graph has the same number)
                    __threadfence();
                }
                // the first piece is its CTA's last pair, unless it is its first one too
                pieces[0] = last ? c1 - c0 + 1 : 0;
                pieces[1] = 2 * c0 + (cut.start(c0) < first ? 1 : 0);
                pieces[2] = 2 * (c0 + 1);
            }
            __syncthreads();
            const int n = pieces[0], piece0 = pieces[1], piece1 = pieces[2];
            const auto place = [&](int i, int col) { return static_cast<int64_t>(i == 0 ? piece0 : piece1 + 2 * (i - 1)) * A::kCols + col; };
            if (n > 0) {
                for (int i = threadIdx.x; i < used * (D / 4); i += kThreads) {
                    const int col = i / (D / 4), d = (i - col * (D / 4)) * 4;
                    // the pieces' results in the order of the tokens, each taken relative to the largest so far; weights are 2^-kDown at most, so that sums
                    // of up to 2^kDown results are finite
                    constexpr float kDown = 12.0f;
                    float top = kLowest, total_weight = 0.0f, x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    for (int j0 = 0; j0 < n; j0 += 4) {
                        float lse[4];
                        float4 y[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int64_t at = place(min(j0 + j, n - 1), col);
                            lse[j] = j0 + j < n ? __ldcg(p.ws_lse + at) : kNegInf;
                            y[j] = __ldcg(reinterpret_cast<const float4*>(p.ws_o + at * D + d));
                        }
                        float most = fmaxf(fmaxf(lse[0], lse[1]), fmaxf(lse[2], lse[3]));
                        most = fmaxf(most, top);
                        const float by = ex2(top - most);
                        top = most;
                        total_weight *= by;
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] *= by;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float l = ex2(lse[j] - top - kDown);
                            total_weight += l;
                            if (j0 + j < n) x[0] += l * y[j].x, x[1] += l * y[j].y, x[2] += l * y[j].z, x[3] += l * y[j].w;
                        }
                    }
                    const float by = total_weight == 0.0f ? 0.0f : 1.0f / total_weight;
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] *= by;
                    A::store(A::out_row(p, b, g, ct * A::kCols + col) + d, x);
                }
            }
            __syncthreads();  // (pieces)
        }
        first_of_run = false;
        if (!on) break;
    }
    copy_wait<0>();
}

struct Plan {
    int cols, col_tiles, cluster, ctas;
    int64_t pairs;
    size_t workspace;
};

template <typename T, int NG, int KB, int VB, int NT>
int launch_attend(const AttendParams& p, const Plan& plan, void* stream) {
    using A = Attend<T, NG, KB, VB, NT>;
    auto kernel = attend_kernel<T, NG, KB, VB, NT>;
    static std::atomic<bool> ready[64];
    int device = 0;
    B2KV_CUDA_TRY(cudaGetDevice(&device));
    if (device >= 64 || !ready[device].load(std::memory_order_relaxed)) {
        B2KV_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, A::kSmem));
        if (device < 64) ready[device].store(true, std::memory_order_relaxed);
    }
    OverlapLaunch launch(dim3(static_cast<unsigned>(plan.ctas)), A::kThreads, A::kSmem, stream, plan.cluster > 1 ? plan.cluster : 1);
    B2KV_CUDA_TRY(cudaLaunchKernelEx(&launch.cfg, kernel, p));
    return B2KV_OK;
}

// Clusters of `size` CTAs that run at the same time on the current device; 0 without one.
template <typename T, int NG, int KB, int VB, int NT>
int count_clusters(int size) {
    using A = Attend<T, NG, KB, VB, NT>;
    auto kernel = attend_kernel<T, NG, KB, VB, NT>;
    int count = 0;
    OverlapLaunch launch(dim3(static_cast<unsigned>(size)), A::kThreads, A::kSmem, nullptr, static_cast<unsigned>(size));
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, A::kSmem) == cudaSuccess &&
        cudaOccupancyMaxActiveClusters(&count, kernel, &launch.cfg) == cudaSuccess)
        return count;
    cudaGetLastError();
    return 0;
}
int clusters_at_once(int size);

template <int NG, int KB, int VB>
int attend_sized(const AttendParams& p, const Plan& plan, void* stream) {
    if (p.c.dtype == B2KV_DTYPE_F32) return launch_attend<float, NG, KB, VB, 1>(p, plan, stream);
    constexpr bool kWide = NG != 8 || KB == VB;  // tiles of 16 columns (make_plan asks for none elsewhere)
    if constexpr (kWide)
        if (plan.cols == 16) return launch_attend<__nv_bfloat16, NG, KB, VB, 2>(p, plan, stream);
    return launch_attend<__nv_bfloat16, NG, KB, VB, 1>(p, plan, stream);
}

// One file each, so that they compile side by side.
int attend_32(const AttendParams& p, const Plan& plan, void* stream);
int attend_64(const AttendParams& p, const Plan& plan, void* stream);
int attend_96(const AttendParams& p, const Plan& plan, void* stream);
int attend_128(const AttendParams& p, const Plan& plan, void* stream);
int attend_256(const AttendParams& p, const Plan& plan, void* stream);

template <int NG>
int attend_bits(const AttendParams& p, const Plan& plan, void* stream) {
    if (p.c.k_bits == 4) return attend_sized<NG, 4, 4>(p, plan, stream);
    if (p.c.v_bits == 4) return attend_sized<NG, 8, 4>(p, plan, stream);
    return attend_sized<NG, 8, 8>(p, plan, stream);
}

}  // namespace qcache
}  // namespace b2kv
