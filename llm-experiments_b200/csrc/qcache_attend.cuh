// Attention of a few new tokens over a quantised key / value cache (the form is in b2kv.h).
//
// What bounds it: HBM.  A cached token of a head is D * (k_bits + v_bits) / 8 + D / 8 bytes for 4 * D * (query heads) flops, so the
// arithmetic has to be hidden behind 23 bytes per clock and SM, and with 4 bits 46 elements per clock have to be widened.  Plain
// fp32 arithmetic cannot (128 FMAs per clock and SM, one per element and query head); the tensor cores can, if widening is cheap:
//
//   * Codes become fp16 numbers by masking alone: a code c in the low bits of a 16-bit half is the fp16 subnormal c * 2^-24, one in
//     the next four bits is c * 2^-20, and tensor cores and half-precision adds take subnormals at full speed.  Two codes per
//     instruction, no conversion.
//   * Both products have the cache's rows as the operand of many rows: S[token, column] = K q (16 tokens by 8 columns per MMA, m16n8k16)
//     and O[element, column] += V^T P.  A column is one (new token, query head) pair of the key / value head.  The cache's
//     layout gives a lane the codes that it needs as one piece, the query is permuted to match, and P goes from the accumulator's
//     layout to the operand's by an 8 x 8 transpose within the warp.  The rows go through tcgen05 only if they were first widened into
//     shared memory at 16 bits per element, which is four times the traffic of reading them; as register operands they are widened in place.
//   * Key codes are taken as stored (c + 8, c + 128); the accumulator of a group starts at minus 8 (128) times the group's sum of the query.
//     A group's sum is multiplied by its key scale in fp32.  Value codes are centred (one half-precision add per two), because over thousands
//     of tokens the sum of uncentred ones grows far beyond what is left when the centre is taken off.
//   * A probability times a value scale is rounded to fp16 (11 bits; the output has 8).  To keep it in range whatever the scales
//     are, it is taken relative to the largest scale's exponent so far, and the accumulators are rescaled when that grows: below 2^15
//     always, and full precision down to scales 2^20 below the largest.
//   * fp32 queries and probabilities are sums of two fp16 numbers (22 bits), in columns of their own.
//   * Softmax: scores in the log2 domain, reference maxima that move only when a score has outgrown its reference by more than 2^8 (one vote
//     per 32 tokens), sums per lane until the end, all in fp32.
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "qcache.cuh"

namespace b2kv {
namespace qcache {

struct AttendParams {
    b2kv_qcache c;
    const void* q;
    void* out;
    const float* slopes;
    float* ws_o;   // [slots, kCols, D]: normalised
    float* ws_lse; // [slots, kCols]: log2 of the sum of exponentials
    int32_t* dev_status;
    int64_t ld_q, ld_out;
    int R, m, col_tiles, T_upper, len_bias, window;
    int n_splits, share;  // pieces of a (sequence, head) and tokens in one
    float scale, softcap;
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_huge_valf();
constexpr int kStageTokens = 32;
constexpr int kScaleExpMin = 17;  // (biased) smaller exponents of value scales are taken for this one: 2^-110

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
    __device__ __forceinline__ void load16(uint32_t at, int i) {
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]) : "r"(at) : "memory");
    }
    __device__ __forceinline__ void load8(uint32_t at, int i) {
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[i]), "=r"(w[i + 1]) : "r"(at) : "memory");
    }
};

// T: type of queries and outputs; NG groups of 32 elements; KB, VB bits; NT tiles of 8 columns (fp32: 2, the second for what fp16 leaves
// of the first); WARPS per CTA, STAGES of 32 tokens in each warp's ring.
template <typename T, int NG, int KB, int VB, int NT, int WARPS, int STAGES>
struct Attend {
    static constexpr bool kF32 = std::is_same<T, float>::value;
    static_assert(!kF32 || NT == 2, "");
    static constexpr int D = NG * kGroup, kCols = kF32 ? 8 : 8 * NT, kThreads = WARPS * 32;
    static constexpr int kKRow = D * KB / 8, kVRow = D * VB / 8, kSRow = scale_row(NG) * 2;
    static constexpr int kKBytes = kStageTokens * kKRow, kVBytes = kStageTokens * kVRow, kSBytes = kStageTokens * kSRow;
    static constexpr int kStage = (kKBytes + kVBytes + 2 * kSBytes + 15) / 16 * 16;
    static constexpr int kRing = WARPS * STAGES * kStage;
    static constexpr int kMerge = WARPS * kCols * (D + 2) * 4;
    static constexpr int kSmem = kRing > kMerge ? kRing : kMerge;
    static constexpr int kKOff = KB == 4 ? 8 : 128;  // what is added to a key's code

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

    struct Warp {
        uint32_t q[NT][NG][2][2];  // the query as the second operand of S = K q
        float off[NT][NG][2];      // what a group's accumulator starts at, columns 2 tig and 2 tig + 1
        float f[NT][2];            // score = sum * f
        float slope[NT][2];        // log2 e times the column's slope
        int lo[NT][2], lim[NT][2]; // the column sees tokens lo <= t < lim
        int all_lo, all_lim;       // tokens that every used column sees
        float o[NT][NG * 2][4];    // elements 32 (j / 2) + 4 gid + 2 (j & 1) (+1 in the last two), columns 2 tig, 2 tig + 1
        float top[NT][2], sum[NT][2];
        int scale_exp;
    };

    // fp32: both tiles are the same columns.
    __device__ static __forceinline__ int col_of(int nt, int c) { return kF32 ? c : nt * 8 + c; }

    __device__ static void load8(const float* p, float (&x)[8]) {
        const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    }
    __device__ static void load8(const __nv_bfloat16* p, float (&x)[8]) { Elt<__nv_bfloat16>::widen(*reinterpret_cast<const uint4*>(p), x); }

    // Queries of sequence b, head g, column tile ct, and what goes with them.  n: tokens of the sequence.
    __device__ static __forceinline__ void begin(const AttendParams& p, Warp& w, int b, int g, int ct, int n) {
        const int lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
        const int used = p.m * p.R;
        w.all_lo = 0, w.all_lim = 0x7fffffff;
#pragma unroll
        for (int nt = 0; nt < (kF32 ? 1 : NT); ++nt) {
            const int col = ct * kCols + col_of(nt, gid);  // the column whose query this lane loads
            float x[NG][8];
            float most = 0.0f;
            if (col < used) {
                const int i = col / p.R, h = g * p.R + col - i * p.R;
                const T* src = static_cast<const T*>(p.q) + (static_cast<int64_t>(b) * p.m + i) * p.ld_q + static_cast<int64_t>(h) * D;
#pragma unroll
                for (int u = 0; u < NG; ++u) {
                    load8(src + u * kGroup + tig * 8, x[u]);
#pragma unroll
                    for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[u][e]));
                }
            } else {
#pragma unroll
                for (int u = 0; u < NG; ++u)
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[u][e] = 0.0f;
            }
            most = fmaxf(most, __shfl_xor_sync(~0u, most, 1));
            most = fmaxf(most, __shfl_xor_sync(~0u, most, 2));
            // q = qn * 2^e with the largest |qn| in [2^14, 2^15): exact, and no fp16 overflow
            const int biased = min(max(__float_as_int(most) >> 23, 27), 254);
            const float down = __int_as_float((254 + 14 - biased) << 23);
            // 2^(e - 14 + 24) * scale, the 24 for the codes' 2^-24
            const float f = p.scale * kLog2e * 1024.0f * __int_as_float(biased << 23);
            float part[2][NG];
#pragma unroll
            for (int u = 0; u < NG; ++u) {
                part[0][u] = part[1][u] = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) x[u][e] *= down;
                // elements in the order of the codes in a word's halves: 4 bits (0,4) (1,5) (2,6) (3,7), the odd ones 16 times too
                // large there; 8 bits (0,1) (2,3) (4,5) (6,7)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float by = KB == 4 && (j & 1) ? 0.0625f : 1.0f;
                    const float a = x[u][KB == 4 ? j : 2 * j] * by, c = x[u][KB == 4 ? j + 4 : 2 * j + 1] * by;
                    const uint32_t h = pack_half(a, c);
                    const float2 got = unpack_half(h);
                    w.q[nt][u][j >> 1][j & 1] = h;
                    part[0][u] += (got.x + got.y) / by;
                    if constexpr (kF32) {
                        const uint32_t l = pack_half(a - got.x, c - got.y);
                        const float2 low = unpack_half(l);
                        w.q[1][u][j >> 1][j & 1] = l;
                        part[1][u] += (low.x + low.y) / by;
                    }
                }
            }
            const int from0 = 8 * tig, from1 = 8 * tig + 4;  // lanes that loaded columns 2 tig and 2 tig + 1
#pragma unroll
            for (int l = 0; l < (kF32 ? 2 : 1); ++l)
#pragma unroll
                for (int u = 0; u < NG; ++u) {
                    float s = part[l][u];
                    s += __shfl_xor_sync(~0u, s, 1);
                    s += __shfl_xor_sync(~0u, s, 2);
                    s *= -static_cast<float>(kKOff) * 0x1p-24f;
                    w.off[nt + l][u][0] = __shfl_sync(~0u, s, from0);
                    w.off[nt + l][u][1] = __shfl_sync(~0u, s, from1);
                }
            w.f[nt][0] = __shfl_sync(~0u, f, from0);
            w.f[nt][1] = __shfl_sync(~0u, f, from1);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int mine = ct * kCols + col_of(nt, 2 * tig + e);
                const int i = mine / p.R, place = n - p.m + i;
                const bool is = mine < used;
                w.lim[nt][e] = is ? place + 1 : 0;
                w.lo[nt][e] = is && p.window > 0 ? max(place + 1 - p.window, 0) : 0;
                w.slope[nt][e] = is && p.slopes != nullptr ? p.slopes[g * p.R + mine - i * p.R] * kLog2e : 0.0f;
                if (is) w.all_lim = min(w.all_lim, w.lim[nt][e]), w.all_lo = max(w.all_lo, w.lo[nt][e]);
            }
        }
#pragma unroll
        for (int d = 1; d <= 2; d <<= 1) {  // (used columns differ from lane to lane)
            w.all_lim = min(w.all_lim, __shfl_xor_sync(~0u, w.all_lim, d));
            w.all_lo = max(w.all_lo, __shfl_xor_sync(~0u, w.all_lo, d));
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int j = 0; j < NG * 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) w.o[nt][j][e] = 0.0f;
#pragma unroll
            for (int e = 0; e < 2; ++e) w.top[nt][e] = kNegInf, w.sum[nt][e] = 0.0f;
        }
        w.scale_exp = kScaleExpMin;
    }

    // Starts the copies of tokens t0 .. t0 + 31 (below t1) of a sequence and head; a bit for each token that is there.
    __device__ static __forceinline__ uint32_t issue(const AttendParams& p, uint32_t stage, int b, int g, int t0, int t1) {
        const int lane = threadIdx.x & 31, t = t0 + lane;
        const int64_t row = t < t1 ? row_of(p.c, b, g, t, p.dev_status) : -1;
        const uint32_t there = __ballot_sync(~0u, row >= 0);
        const int64_t at = row >= 0 ? row : 0;
        const uint32_t ks = stage + kKBytes + kVBytes;
        copy_small<kSRow>(ks + lane * kSRow, static_cast<const uint8_t*>(p.c.k_scales) + at * kSRow, row >= 0);
        copy_small<kSRow>(ks + kSBytes + lane * kSRow, static_cast<const uint8_t*>(p.c.v_scales) + at * kSRow, row >= 0);
        copy_rows<kKRow>(stage, static_cast<const uint8_t*>(p.c.k_codes), at, there, [](int r, int ch) { return k_place(r, ch); });
        copy_rows<kVRow>(stage + kKBytes, static_cast<const uint8_t*>(p.c.v_codes), at, there, [](int r, int ch) { return v_place(r, ch); });
        return there;
    }
    template <int ROW, typename F>
    __device__ static __forceinline__ void copy_rows(uint32_t dst, const uint8_t* src, int64_t mine, uint32_t there, F&& place) {
        constexpr int kCh = ROW / 16;
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int i = 0; i < kCh; ++i) {
            const int idx = i * 32 + lane, r = idx / kCh, ch = idx - r * kCh;
            const int64_t row = __shfl_sync(~0u, mine, r);
            copy16(dst + place(r, ch), src + row * ROW + ch * 16, (there >> r) & 1u);
        }
    }

    // Two rows' codes of half a group as operand pieces (a0 and a1 of two rows; a2 and a3 likewise).
    template <int STEP>
    __device__ static __forceinline__ void k_piece(const uint32_t* w, uint32_t& first, uint32_t& second) {
        if constexpr (KB == 4) {
            const uint32_t x = STEP == 0 ? w[0] : w[0] >> 8;
            first = x & 0x000f000fu;
            second = x & 0x00f000f0u;
        } else {
            first = __byte_perm(w[STEP], 0, 0x4140);
            second = __byte_perm(w[STEP], 0, 0x4342);
        }
    }

    // The 32 tokens of a stage.
    __device__ static __forceinline__ void fold(const AttendParams& p, Warp& w, uint32_t stage, int t0, uint32_t there) {
        const int lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
        const uint32_t ks = stage + kKBytes + kVBytes, vs = ks + kSBytes, vc = stage + kKBytes;
        constexpr int kKPiece = NG * KB, kVPiece = NG * VB / 2;  // bytes of a row that a lane reads
        constexpr int NS = kF32 ? 1 : NT;                        // tiles of scores
        float s[2][NS][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = h * 16 + gid;
            Words<kKPiece> k0, k1;
            load_k(k0, stage, r, tig);
            load_k(k1, stage, r + 8, tig);
            Words<kSRow> s0, s1;
            s0.load(ks + r * kSRow);
            s1.load(ks + (r + 8) * kSRow);
            float acc[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[nt][e] = 0.0f;
#pragma unroll
            for (int u = 0; u < NG; ++u) {
                uint32_t a[2][4];
                constexpr int kW = KB / 4;  // words of a lane's piece of a group
                k_piece<0>(k0.w + u * kW, a[0][0], a[0][2]);
                k_piece<0>(k1.w + u * kW, a[0][1], a[0][3]);
                k_piece<1>(k0.w + u * kW, a[1][0], a[1][2]);
                k_piece<1>(k1.w + u * kW, a[1][1], a[1][3]);
                const float f0 = __uint_as_float(u & 1 ? s0.w[u >> 1] & 0xffff0000u : s0.w[u >> 1] << 16);
                const float f1 = __uint_as_float(u & 1 ? s1.w[u >> 1] & 0xffff0000u : s1.w[u >> 1] << 16);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float d[4] = {w.off[nt][u][0], w.off[nt][u][1], w.off[nt][u][0], w.off[nt][u][1]};
                    mma(d, a[0][0], a[0][1], a[0][2], a[0][3], w.q[nt][u][0][0], w.q[nt][u][0][1]);
                    mma(d, a[1][0], a[1][1], a[1][2], a[1][3], w.q[nt][u][1][0], w.q[nt][u][1][1]);
                    acc[nt][0] = fmaf(f0, d[0], acc[nt][0]);
                    acc[nt][1] = fmaf(f0, d[1], acc[nt][1]);
                    acc[nt][2] = fmaf(f1, d[2], acc[nt][2]);
                    acc[nt][3] = fmaf(f1, d[3], acc[nt][3]);
                }
            }
#pragma unroll
            for (int nt = 0; nt < NS; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[h][nt][e] = (kF32 ? acc[0][e] + acc[NT - 1][e] : acc[nt][e]) * w.f[nt][e & 1];
        }
        if (p.softcap > 0.0f) {
            const float down = 1.0f / (p.softcap * kLog2e), up = p.softcap * kLog2e;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int nt = 0; nt < NS; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[h][nt][e] = tanhf(s[h][nt][e] * down) * up;
        }
        if (p.slopes != nullptr) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int nt = 0; nt < NS; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        s[h][nt][e] -= w.slope[nt][e & 1] * static_cast<float>(w.lim[nt][e & 1] - 1 - (t0 + h * 16 + (e >> 1) * 8 + gid));
        }
        // Masks, where the stage has a token that some column does not see.
        const bool masked = there != ~0u || t0 < w.all_lo || t0 + kStageTokens > w.all_lim;
        uint32_t hidden = 0;  // a bit per score of this lane
        if (masked) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int nt = 0; nt < NS; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = h * 16 + (e >> 1) * 8 + gid, t = t0 + r;
                        if (!((there >> r) & 1u) || t < w.lo[nt][e & 1] || t >= w.lim[nt][e & 1]) {
                            s[h][nt][e] = kNegInf;
                            hidden |= 1u << (h * 8 + nt * 4 + e);
                        }
                    }
        }
        // The references, where a score has outgrown its own by more than 2^8.
        bool grown = false;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int nt = 0; nt < NS; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) grown = grown || s[h][nt][e] > w.top[nt][e & 1] + 8.0f;
        if (__any_sync(~0u, grown)) {
#pragma unroll
            for (int nt = 0; nt < NS; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float top = fmaxf(fmaxf(s[0][nt][e], s[0][nt][e + 2]), fmaxf(s[1][nt][e], s[1][nt][e + 2]));
#pragma unroll
                    for (int d = 4; d <= 16; d <<= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
                    top = fmaxf(top, w.top[nt][e]);
                    const float by = top == w.top[nt][e] ? 1.0f : ex2(w.top[nt][e] - top);
                    w.top[nt][e] = top;
                    w.sum[nt][e] *= by;
#pragma unroll
                    for (int l = 0; l < (kF32 ? 2 : 1); ++l)
#pragma unroll
                        for (int j = 0; j < NG * 2; ++j) w.o[nt + l][j][e] *= by, w.o[nt + l][j][e + 2] *= by;
                }
        }
#pragma unroll
        for (int nt = 0; nt < NS; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float top = w.top[nt][e] == kNegInf ? 0.0f : w.top[nt][e];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    s[h][nt][e] = ex2(s[h][nt][e] - top);
                    s[h][nt][e + 2] = ex2(s[h][nt][e + 2] - top);
                    w.sum[nt][e] += s[h][nt][e] + s[h][nt][e + 2];
                }
            }
        // The largest exponent of a value scale (NaN groups have none).
        {
            Words<kSRow> mine;
            mine.load(vs + lane * kSRow);
            uint32_t most = 0;
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                const uint32_t x = i & 1 ? mine.w[i >> 1] >> 16 : mine.w[i >> 1] & 0xffffu;
                most = max(most, x >= 0x7f80u ? 0u : x);
            }
            const int now = static_cast<int>(__reduce_max_sync(~0u, most) >> 7);
            if (now > w.scale_exp) {
                const float by = w.scale_exp - now < -126 ? 0.0f : __int_as_float((127 + w.scale_exp - now) << 23);
                w.scale_exp = now;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < NG * 2; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) w.o[nt][j][e] *= by;
            }
        }
        const float vf = __int_as_float((260 - w.scale_exp) << 23);  // 2^(6 - exponent)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = h * 16 + gid;
            Words<kSRow> s0, s1;
            s0.load(vs + r * kSRow);
            s1.load(vs + (r + 8) * kSRow);
            Words<kVPiece> v[4];  // tokens 2 tig, 2 tig + 1, 2 tig + 8, 2 tig + 9
#pragma unroll
            for (int i = 0; i < 4; ++i) load_v(v[i], vc, h * 16 + 2 * tig + (i & 1) + (i >> 1) * 8, gid);
#pragma unroll
            for (int u = 0; u < NG; ++u) {
                const float f0 = vf * __uint_as_float(u & 1 ? s0.w[u >> 1] & 0xffff0000u : s0.w[u >> 1] << 16);
                const float f1 = vf * __uint_as_float(u & 1 ? s1.w[u >> 1] & 0xffff0000u : s1.w[u >> 1] << 16);
                uint32_t b[NT][2];
#pragma unroll
                for (int nt = 0; nt < NS; ++nt) {
                    float x[4] = {s[h][nt][0] * f0, s[h][nt][1] * f0, s[h][nt][2] * f1, s[h][nt][3] * f1};
                    if (masked) {  // (0 times a NaN scale)
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] = (hidden >> (h * 8 + nt * 4 + e)) & 1u ? 0.0f : x[e];
                    }
                    const uint32_t p0 = pack_half(x[0], x[1]), p1 = pack_half(x[2], x[3]);
                    b[nt][0] = transpose8x8(p0);
                    b[nt][1] = transpose8x8(p1);
                    if constexpr (kF32) {
                        const float2 g0 = unpack_half(p0), g1 = unpack_half(p1);
                        b[1][0] = transpose8x8(pack_half(x[0] - g0.x, x[1] - g0.y));
                        b[1][1] = transpose8x8(pack_half(x[2] - g1.x, x[3] - g1.y));
                    }
                }
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
                const uint32_t x = __byte_perm(v[2 * i].w[u >> 1], v[2 * i + 1].w[u >> 1], sel);
                a[0][2 * i] = half_sub(x & 0x000f000fu, 0x00080008u);
                a[0][2 * i + 1] = half_sub(x & 0x00f000f0u, 0x00800080u);
                a[1][2 * i] = half_sub((x >> 8) & 0x000f000fu, 0x00080008u);
                a[1][2 * i + 1] = half_sub((x >> 8) & 0x00f000f0u, 0x00800080u);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t x = __byte_perm(v[2 * i].w[u], v[2 * i + 1].w[u], 0x5410), y = __byte_perm(v[2 * i].w[u], v[2 * i + 1].w[u], 0x7632);
                a[0][2 * i] = half_sub(x & 0x00ff00ffu, 0x00800080u);
                a[0][2 * i + 1] = half_sub(__byte_perm(x, 0, 0x4341), 0x00800080u);
                a[1][2 * i] = half_sub(y & 0x00ff00ffu, 0x00800080u);
                a[1][2 * i + 1] = half_sub(__byte_perm(y, 0, 0x4341), 0x00800080u);
            }
        }
    }

    // A lane's pieces of a row, which lie in one 16-byte piece or are whole ones.
    template <typename W>
    __device__ static __forceinline__ void load_k(W& k, uint32_t stage, int r, int tig) {
        constexpr int kBytes = NG * KB;
        if constexpr (kBytes > 16 && kBytes % 16 == 0) {
#pragma unroll
            for (int i = 0; i < kBytes / 16; ++i) k.load16(stage + k_place(r, tig * (kBytes / 16) + i), 4 * i);
        } else if constexpr (NG == 3) {
            k.load(stage + r * kKRow + tig * kBytes);
        } else {
            k.load(stage + k_place(r, tig * kBytes / 16) + tig * kBytes % 16);
        }
    }
    template <typename W>
    __device__ static __forceinline__ void load_v(W& v, uint32_t codes, int r, int gid) {
        constexpr int kBytes = NG * VB / 2;
        if constexpr (kBytes > 16 && kBytes % 16 == 0) {
#pragma unroll
            for (int i = 0; i < kBytes / 16; ++i) v.load16(codes + v_place(r, gid * (kBytes / 16) + i), 4 * i);
        } else if constexpr (NG == 3) {
            v.load(codes + r * kVRow + gid * kBytes);
        } else {
            v.load(codes + v_place(r, gid * kBytes / 16) + gid * kBytes % 16);
        }
    }

    // This warp's result into `o` [kCols][D] (normalised) and `ml` [kCols][2] (reference, sum).
    __device__ static __forceinline__ void leave(Warp& w, float* o, float* ml) {
        const int lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
        constexpr int NS = kF32 ? 1 : NT;
        // the accumulators are in units of 2^-24 * 2^(6 - exponent)
        const float up = __int_as_float(w.scale_exp << 23);
#pragma unroll
        for (int nt = 0; nt < NS; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float sum = w.sum[nt][e];
#pragma unroll
                for (int d = 4; d <= 16; d <<= 1) sum += __shfl_xor_sync(~0u, sum, d);
                const int col = col_of(nt, 2 * tig + e);
                const float by = sum == 0.0f ? 0.0f : 0x1p18f / sum;
                if (gid == 0) ml[col * 2] = w.top[nt][e], ml[col * 2 + 1] = sum;
#pragma unroll
                for (int u = 0; u < NG; ++u) {
                    float x[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int j = 2 * u + (i >> 1), at = (i & 1) * 2 + e;
                        const float y = kF32 ? w.o[0][j][at] + w.o[NT - 1][j][at] : w.o[nt][j][at];
                        x[i] = y * by * (VB == 4 && (i & 1) ? 0.0625f : 1.0f) * up;
                    }
                    *reinterpret_cast<float4*>(o + col * D + u * kGroup + gid * 4) = make_float4(x[0], x[1], x[2], x[3]);
                }
            }
    }

    __device__ static __forceinline__ void store(T* out, float x) { *out = Elt<T>::from_float(x); }

    // The warps' results put together: into the output rows, or into the workspace as piece `slot`.
    __device__ static __forceinline__ void merge(const AttendParams& p, const float* o, const float* ml, int b, int g, int ct, int slot) {
        for (int idx = threadIdx.x; idx < kCols * D; idx += kThreads) {
            const int col = idx / D, d = idx - col * D;
            const int mine = ct * kCols + col;
            if (mine >= p.m * p.R) break;
            float top = kNegInf;
#pragma unroll
            for (int i = 0; i < WARPS; ++i) top = fmaxf(top, ml[(i * kCols + col) * 2]);
            const float ref = top == kNegInf ? 0.0f : top;
            float sum = 0.0f, x = 0.0f;
#pragma unroll
            for (int i = 0; i < WARPS; ++i) {
                const float l = ml[(i * kCols + col) * 2 + 1] * ex2(ml[(i * kCols + col) * 2] - ref);
                sum += l;
                x += l * o[(i * kCols + col) * D + d];
            }
            x = sum == 0.0f ? 0.0f : x / sum;
            if (slot >= 0) {
                p.ws_o[(static_cast<int64_t>(slot) * kCols + col) * D + d] = x;
                if (d == 0) p.ws_lse[static_cast<int64_t>(slot) * kCols + col] = sum == 0.0f ? kNegInf : ref + log2f(sum);
            } else {
                const int i = mine / p.R, h = g * p.R + mine - i * p.R;
                store(static_cast<T*>(p.out) + (static_cast<int64_t>(b) * p.m + i) * p.ld_out + static_cast<int64_t>(h) * D + d, x);
            }
        }
    }
};

// Tokens of sequence b, and the first one that any query of it sees.
__device__ __forceinline__ int attended(const AttendParams& p, int b, int& first) {
    const int n = min(max(tokens_held(p.c, b) + p.len_bias, 0), p.T_upper);
    first = p.window > 0 ? max(n - p.m + 1 - p.window, 0) : 0;
    return n;
}

// One CTA per (sequence, head, column tile) and share of its tokens; the warps take its stages in turn.
template <typename T, int NG, int KB, int VB, int NT, int WARPS, int STAGES>
__global__ void __launch_bounds__(WARPS * 32) attend_kernel(const AttendParams p) {
    using A = Attend<T, NG, KB, VB, NT, WARPS, STAGES>;
    extern __shared__ __align__(128) uint8_t smem[];
    grid_dependency_wait();
    const int pair = blockIdx.x, split = blockIdx.y, warp = threadIdx.x >> 5;
    const int ct = pair % p.col_tiles, bg = pair / p.col_tiles, b = bg / p.c.G, g = bg - b * p.c.G;
    int first;
    const int n = attended(p, b, first);
    const int t_begin = first + split * p.share, t_end = min(n, t_begin + p.share);
    typename A::Warp w;
    A::begin(p, w, b, g, ct, n);
    const uint32_t ring = smem_u32(smem) + warp * STAGES * A::kStage;
    uint32_t there[STAGES];
    const int stages = t_end > t_begin ? (t_end - t_begin + kStageTokens - 1) / kStageTokens : 0;
    for (int i = warp; i < stages; i += WARPS) {
        const int t0 = t_begin + i * kStageTokens;
        there[0] = A::issue(p, ring, b, g, t0, t_end);
        copy_commit();
        copy_wait<0>();
        __syncwarp();
        A::fold(p, w, ring, t0, there[0]);
        __syncwarp();
    }
    __syncthreads();
    float* const o = reinterpret_cast<float*>(smem);
    float* const ml = o + WARPS * A::kCols * A::D;
    A::leave(w, o + warp * A::kCols * A::D, ml + warp * A::kCols * 2);
    __syncthreads();
    A::merge(p, o, ml, b, g, ct, p.n_splits > 1 ? pair * p.n_splits + split : -1);
}

// One CTA per column: its pieces put together.
template <typename T, int D, int COLS>
__global__ void __launch_bounds__(D < 64 ? 64 : D) merge_kernel(const AttendParams p) {
    grid_dependency_wait();
    const int pair = blockIdx.x, col = blockIdx.y, d = threadIdx.x;
    const int ct = pair % p.col_tiles, bg = pair / p.col_tiles, b = bg / p.c.G, g = bg - b * p.c.G;
    const int mine = ct * COLS + col;
    if (mine >= p.m * p.R || d >= D) return;
    const int64_t slot0 = static_cast<int64_t>(pair) * p.n_splits;
    float top = kNegInf;
    for (int i = 0; i < p.n_splits; ++i) top = fmaxf(top, p.ws_lse[(slot0 + i) * COLS + col]);
    const float ref = top == kNegInf ? 0.0f : top;
    float sum = 0.0f, x = 0.0f;
    for (int i = 0; i < p.n_splits; ++i) {
        const float l = ex2(p.ws_lse[(slot0 + i) * COLS + col] - ref);
        sum += l;
        x += l * p.ws_o[((slot0 + i) * COLS + col) * D + d];
    }
    x = sum == 0.0f ? 0.0f : x / sum;
    const int i = mine / p.R, h = g * p.R + mine - i * p.R;
    static_cast<T*>(p.out)[(static_cast<int64_t>(b) * p.m + i) * p.ld_out + static_cast<int64_t>(h) * D + d] = Elt<T>::from_float(x);
}

struct Plan {
    int cols, col_tiles, n_splits, share;
    int64_t pairs;
    size_t workspace;
};

template <typename T, int NG, int KB, int VB, int NT>
int launch_attend(const AttendParams& p, const Plan& plan, void* stream) {
    constexpr int kWarps = 8, kStages = 1;
    using A = Attend<T, NG, KB, VB, NT, kWarps, kStages>;
    auto kernel = attend_kernel<T, NG, KB, VB, NT, kWarps, kStages>;
    B2KV_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, A::kSmem));
    OverlapLaunch launch(dim3(static_cast<unsigned>(plan.pairs), plan.n_splits), kWarps * 32, A::kSmem, stream);
    B2KV_CUDA_TRY(cudaLaunchKernelEx(&launch.cfg, kernel, p));
    if (plan.n_splits > 1) {
        OverlapLaunch second(dim3(static_cast<unsigned>(plan.pairs), A::kCols), A::D < 64 ? 64 : A::D, 0, stream);
        B2KV_CUDA_TRY(cudaLaunchKernelEx(&second.cfg, merge_kernel<T, A::D, A::kCols>, p));
    }
    return B2KV_OK;
}

template <int NG, int KB, int VB>
int attend_sized(const AttendParams& p, const Plan& plan, void* stream) {
    if (p.c.dtype == B2KV_DTYPE_F32) return launch_attend<float, NG, KB, VB, 2>(p, plan, stream);
    return plan.cols == 8 ? launch_attend<__nv_bfloat16, NG, KB, VB, 1>(p, plan, stream) : launch_attend<__nv_bfloat16, NG, KB, VB, 2>(p, plan, stream);
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
