// Quantised key / value cache: rows into it and out of it.
//
// Both are streams: a row of D elements comes in at D * (2 or 4) bytes and leaves at D * bits / 8 + D / 16, or the other way round.  A thread has
// octet o (8 neighbouring elements) of every group of a row, as the cache keeps them one behind the other: its codes are one piece of memory
// (16 bytes for 4 bits and heads of 128), what it reads or writes of the row in full width are D / 32 pieces of 16 bytes, 64 bytes apart, which the
// four threads of the row fill between them; and a group's largest magnitude is two shuffles away.  That keeps 64 bytes per thread on their way and
// finds a row's place once for all of it (one octet per thread with its own divisions: 2.2 TB/s into the cache, 2.8 out of it).
//
// A code is the quotient rounded to the nearest whole number, ties to even, as if it had been computed exactly.  The correctly rounded fp32
// quotient gives that: x / scale lies exactly on a border n + 1/2 only if it is one.  (A border times the scale has at most 8 + 8
// bits, so it is a float; the next float away from it, a step u, moves the quotient by u / scale, which is more than half a step of
// the quotient, because the scale's mantissa is below 2.  So no other quotient rounds onto the border.)  The same holds for max / L.  Scales
// of ordinary size take the quotient from their reciprocal and one correction by the remainder, which an FMA gives exactly: a border comes out as
// itself, and anything else is right to a small part of a step.
#include "qcache.cuh"

#include <type_traits>

namespace b2kv {
namespace qcache {

int check(const b2kv_qcache* c) {
    if (c == nullptr) return B2KV_ERR_BAD_ARG;
    if (elt_bytes(c->dtype) == 0 || b2kv_qcache_scale_row(c->D) == 0) return B2KV_ERR_UNSUPPORTED;
    const bool bits = (c->k_bits == 4 && c->v_bits == 4) || (c->k_bits == 8 && (c->v_bits == 4 || c->v_bits == 8));
    if (!bits) return B2KV_ERR_UNSUPPORTED;
    if (!c->k_codes || !c->v_codes || !c->k_scales || !c->v_scales) return B2KV_ERR_BAD_ARG;
    if (c->B <= 0 || c->G <= 0 || c->T_max <= 0) return B2KV_ERR_BAD_ARG;
    if (c->T_max > 1 << 30) return B2KV_ERR_UNSUPPORTED;  // (places are counted in 32 bits)
    if (c->block_table != nullptr) {
        if (c->max_blocks <= 0 || c->block_size <= 0 || c->n_blocks <= 0) return B2KV_ERR_BAD_ARG;
        if (static_cast<int64_t>(c->max_blocks) * c->block_size < c->T_max) return B2KV_ERR_BAD_ARG;
    }
    if (!aligned16(c->k_codes) || !aligned16(c->v_codes) || !aligned16(c->k_scales) || !aligned16(c->v_scales)) return B2KV_ERR_ALIGN;
    return B2KV_OK;
}

namespace {

constexpr int kThreads = 256;

// Eight elements as they lie in memory.
template <typename T>
struct Octet {
    uint4 w[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
    }
    __device__ __forceinline__ void widen(float (&f)[8]) const;
    __device__ __forceinline__ uint32_t largest() const;  // magnitude, as a whole number: in the same order, NaN above infinity above all others
};
template <>
__device__ __forceinline__ void Octet<float>::widen(float (&f)[8]) const {
    Elt<float>::widen(w[0], f);
    Elt<float>::widen(w[1], f + 4);
}
template <>
__device__ __forceinline__ void Octet<__nv_bfloat16>::widen(float (&f)[8]) const {
    Elt<__nv_bfloat16>::widen(w[0], f);
}
template <>
__device__ __forceinline__ uint32_t Octet<float>::largest() const {
    const uint32_t a = max(max(w[0].x & 0x7fffffffu, w[0].y & 0x7fffffffu), max(w[0].z & 0x7fffffffu, w[0].w & 0x7fffffffu));
    const uint32_t b = max(max(w[1].x & 0x7fffffffu, w[1].y & 0x7fffffffu), max(w[1].z & 0x7fffffffu, w[1].w & 0x7fffffffu));
    return max(a, b);
}
template <>
__device__ __forceinline__ uint32_t Octet<__nv_bfloat16>::largest() const {
    const uint32_t x = __vmaxu2(__vmaxu2(w[0].x & 0x7fff7fffu, w[0].y & 0x7fff7fffu), __vmaxu2(w[0].z & 0x7fff7fffu, w[0].w & 0x7fff7fffu));
    return max(x & 0xffff0000u, x << 16);
}

// Two numbers in one instruction.
struct Two {
    unsigned long long v;
    __device__ __forceinline__ Two() {}
    __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
    __device__ __forceinline__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
    __device__ __forceinline__ Two operator*(const Two& o) const {
        Two r;
        asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(v), "l"(o.v));
        return r;
    }
    __device__ __forceinline__ Two operator+(const Two& o) const {
        Two r;
        asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(v), "l"(o.v));
        return r;
    }
    __device__ __forceinline__ static Two fma(const Two& a, const Two& b, const Two& c) {
        Two r;
        asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
        return r;
    }
};

__device__ __forceinline__ void store4(float* p, const float* f) { *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]); }
__device__ __forceinline__ void store4(__nv_bfloat16* p, const float* f) {
    __nv_bfloat162 h[2] = {__floats2bfloat162_rn(f[0], f[1]), __floats2bfloat162_rn(f[2], f[3])};
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(h);
}
__device__ __forceinline__ void store8(float* p, const float* f) { store4(p, f), store4(p + 4, f + 4); }
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float* f) {
    __nv_bfloat162 h[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = __floats2bfloat162_rn(f[2 * e], f[2 * e + 1]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(h);
}

// Eight codes as numbers code + 8 or code + 128, lowest first, of a group's elements, `most` their largest magnitude; all four lanes of the group get
// its scale.
template <int BITS>
__device__ __forceinline__ uint2 quantise(const float (&f)[8], uint32_t most, uint32_t& scale) {
    constexpr int kTop = BITS == 4 ? 7 : 127;
    constexpr uint32_t kTimes = BITS == 4 ? 16 : 256;
    most = max(most, __shfl_xor_sync(~0u, most, 1));
    most = max(most, __shfl_xor_sync(~0u, most, 2));
    const __nv_bfloat16 rounded = __float2bfloat16_rn(most < 0x7f800000u ? __uint_as_float(most) / kTop : __int_as_float(0x7fc00000));
    scale = __bfloat16_as_ushort(rounded);
    const float s = __bfloat162float(rounded);
    uint32_t n[8];
    if (s >= 0x1p-100f) {
        const float inverse = 1.0f / s, magic = 12582912.0f + (kTop + 1);  // 1.5 * 2^23: the sum's last bits are the rounded number's
        const Two by(inverse, inverse), less(-s, -s), up(magic, magic);
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const Two x(f[e], f[e + 1]), q = x * by;
            const Two right = Two::fma(Two::fma(q, less, x), by, q) + up;
            float a, b;
            right.get(a, b);
            n[e] = __float_as_uint(a), n[e + 1] = __float_as_uint(b);
        }
    } else {  // (no scale, or a NaN, or one so small that remainders would be cut off)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float q = s > 0.0f ? fminf(fmaxf(f[e] / s, -kTop), kTop) : 0.0f;
            n[e] = __float_as_uint(q + (12582912.0f + (kTop + 1)));
        }
    }
    constexpr int kPer = 32 / BITS;
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 8 / kPer; ++i) {
        // all but the last code leave nothing above them but the same bits each time, which come off at the end
        uint32_t x = n[i * kPer + kPer - 1], off = 0x4b400000u;
#pragma unroll
        for (int e = kPer - 2; e >= 0; --e) x = x * kTimes + n[i * kPer + e], off = off * kTimes + 0x4b400000u;
        w[i] = x - off;
    }
    return make_uint2(w[0], w[8 / kPer - 1]);
}

// What a row's thread keeps of it: octet o of all NG groups.
template <int NG, int BITS>
struct Codes {
    static constexpr int kBytes = NG * BITS;
    uint32_t w[(kBytes + 3) / 4];
    __device__ __forceinline__ void load(const uint8_t* p) { each([&](auto* to, auto* from) { *to = *from; }, reinterpret_cast<uint8_t*>(w), p); }
    __device__ __forceinline__ void store(uint8_t* p) const { each([&](auto* to, auto* from) { *to = *from; }, p, reinterpret_cast<const uint8_t*>(w)); }
    // in pieces of the largest power of two that divides the whole, which is what the place is a multiple of
    template <typename F>
    __device__ static __forceinline__ void each(F&& copy, uint8_t* to, const uint8_t* from) {
        using Piece = typename std::conditional<kBytes % 16 == 0, uint4, typename std::conditional<kBytes % 8 == 0, uint2, uint32_t>::type>::type;
#pragma unroll
        for (int i = 0; i < kBytes / static_cast<int>(sizeof(Piece)); ++i) copy(reinterpret_cast<Piece*>(to) + i, reinterpret_cast<const Piece*>(from) + i);
    }

    // Octets to and from units of 8 codes (keys) or of 4, those of the octet's first half for all groups before those of its second (values).
    template <bool kValues>
    __device__ __forceinline__ void put(int u, uint2 c) {
        if constexpr (BITS == 8) {
            w[kValues ? u : 2 * u] = c.x, w[kValues ? NG + u : 2 * u + 1] = c.y;
        } else if constexpr (!kValues) {
            w[u] = __funnelshift_l(c.x, c.x, 2);
        } else {
            const uint32_t x = ((c.x << 2) & 0xfffcfffcu) | ((c.x >> 14) & 0x00030003u);
            put16(u, x & 0xffffu);
            put16(NG + u, x >> 16);
        }
    }
    template <bool kValues>
    __device__ __forceinline__ uint2 get(int u) const {
        if constexpr (BITS == 8) {
            return make_uint2(w[kValues ? u : 2 * u], w[kValues ? NG + u : 2 * u + 1]);
        } else if constexpr (!kValues) {
            return make_uint2(__funnelshift_r(w[u], w[u], 2), 0);
        } else {
            const uint32_t x = get16(u) | get16(NG + u) << 16;
            return make_uint2(((x >> 2) & 0x3fff3fffu) | ((x << 14) & 0xc000c000u), 0);
        }
    }
    __device__ __forceinline__ void put16(int i, uint32_t x) { w[i / 2] = i & 1 ? (w[i / 2] & 0xffffu) | x << 16 : (w[i / 2] & 0xffff0000u) | x; }
    __device__ __forceinline__ uint32_t get16(int i) const { return i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu; }
};

template <typename T, int NG, int BITS, bool kValues>
__device__ __forceinline__ void write_row(const b2kv_qcache& c, const T* src, int o, int64_t row) {
    Octet<T> in[NG];
#pragma unroll
    for (int u = 0; u < NG; ++u) in[u].load(src + u * kGroup + o * 8);
    Codes<NG, BITS> codes = {};
    uint32_t scales[scale_row(NG) / 2] = {};
#pragma unroll
    for (int u = 0; u < NG; ++u) {
        float f[8];
        in[u].widen(f);
        uint32_t scale;
        codes.template put<kValues>(u, quantise<BITS>(f, in[u].largest(), scale));
        scales[u / 2] |= u & 1 ? scale << 16 : scale;
    }
    if (row < 0) return;
    codes.store(static_cast<uint8_t*>(kValues ? c.v_codes : c.k_codes) + row * (NG * 4 * BITS) + o * (NG * BITS));
    if (o == 0) {  // the row of scales; what lies behind the last takes part in products, with zeros
        uint32_t* const to = static_cast<uint32_t*>(kValues ? c.v_scales : c.k_scales) + row * (scale_row(NG) / 2);
        if constexpr (scale_row(NG) == 2) *to = scales[0];
        if constexpr (scale_row(NG) == 4) *reinterpret_cast<uint2*>(to) = make_uint2(scales[0], scales[1]);
        if constexpr (scale_row(NG) == 8) *reinterpret_cast<uint4*>(to) = make_uint4(scales[0], scales[1], scales[2], scales[3]);
    }
}

// Thread = (row of a head, octet); grid.y 0 keys, 1 values.
template <typename T, int NG, int KB, int VB>
__global__ void __launch_bounds__(kThreads) write_kernel(const b2kv_qcache c, const T* k, int64_t ld_k, const T* v, int64_t ld_v, Divisor by_heads,
                                                         Divisor by_rows, Divisor by_block, uint32_t rows, int32_t* dev_status) {
    grid_launch_dependents();
    grid_dependency_wait();
    const uint32_t at = blockIdx.x * (kThreads / 4) + threadIdx.x / 4, o = threadIdx.x & 3;
    const uint32_t i = min(at, rows - 1);  // (lanes behind the end go along with the shuffles)
    const uint32_t src = by_heads.quotient(i), g = i - src * by_heads.d, b = by_rows.quotient(src);
    const int64_t place = static_cast<int64_t>(tokens_held(c, b)) + (src - b * by_rows.d);
    int64_t row = -1;
    if (place < 0 || place >= c.T_max)
        report_status(dev_status, B2KV_DEV_BAD_POSITION);
    else
        row = row_of(c, by_block, b, g, static_cast<int>(place), dev_status);
    if (at >= rows) row = -1;
    if (blockIdx.y == 0)
        write_row<T, NG, KB, false>(c, k + src * ld_k + static_cast<int64_t>(g) * (NG * kGroup), o, row);
    else
        write_row<T, NG, VB, true>(c, v + src * ld_v + static_cast<int64_t>(g) * (NG * kGroup), o, row);
}

// Thread = (row of a head of the output, octet).
template <typename T, int NG, int BITS, bool kValues>
__global__ void __launch_bounds__(kThreads) read_kernel(const b2kv_qcache c, T* out, int n, int last, int len_bias, Divisor by_heads, Divisor by_rows,
                                                        Divisor by_block, uint32_t rows, int32_t* dev_status) {
    grid_launch_dependents();
    grid_dependency_wait();
    const uint32_t i = blockIdx.x * (kThreads / 4) + threadIdx.x / 4, o = threadIdx.x & 3;
    if (i >= rows) return;
    const uint32_t dst = by_heads.quotient(i), g = i - dst * by_heads.d, b = by_rows.quotient(dst);
    const int64_t held = min(static_cast<int64_t>(tokens_held(c, b)) + len_bias, static_cast<int64_t>(c.T_max));
    const int64_t place = static_cast<int64_t>(dst - b * by_rows.d) + (last ? held - n : 0);
    const int64_t row = place >= 0 && place < held ? row_of(c, by_block, b, g, static_cast<int>(place), dev_status) : -1;
    Codes<NG, BITS> codes;
    uint32_t scales[scale_row(NG) / 2] = {};
    if (row >= 0) {
        codes.load(static_cast<const uint8_t*>(kValues ? c.v_codes : c.k_codes) + row * (NG * 4 * BITS) + o * (NG * BITS));
        const uint32_t* const from = static_cast<const uint32_t*>(kValues ? c.v_scales : c.k_scales) + row * (scale_row(NG) / 2);
#pragma unroll
        for (int u = 0; u < (NG + 1) / 2; ++u) scales[u] = from[u];
    }
    T* const to = out + static_cast<int64_t>(i) * (NG * kGroup) + o * 8;
#pragma unroll
    for (int u = 0; u < NG; ++u) {
        float f[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (row >= 0) {
            const float s = __uint_as_float(u & 1 ? scales[u / 2] & 0xffff0000u : scales[u / 2] << 16);
            const uint2 x = codes.template get<kValues>(u);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t code = BITS == 4 ? (x.x >> (4 * e)) & 15u : ((e < 4 ? x.x : x.y) >> (8 * (e & 3))) & 255u;
                f[e] = (__uint_as_float(0x4b000000u | code) - (8388608.0f + (1 << (BITS - 1)))) * s;  // exact: 2^23 + code less that, 8 bits by 8
            }
        }
        store8(to + u * kGroup, f);
    }
}

template <typename T, int NG, int KB, int VB>
int launch_write(const b2kv_qcache& c, const void* k, int64_t ld_k, const void* v, int64_t ld_v, int n, int32_t* dev_status, void* stream) {
    const int64_t rows = static_cast<int64_t>(c.B) * n * c.G;
    if (rows > 0x7fffffff) return B2KV_ERR_UNSUPPORTED;
    OverlapLaunch launch(dim3(static_cast<unsigned>((rows + kThreads / 4 - 1) / (kThreads / 4)), 2), kThreads, 0, stream);
    B2KV_CUDA_TRY(cudaLaunchKernelEx(&launch.cfg, write_kernel<T, NG, KB, VB>, c, static_cast<const T*>(k), ld_k, static_cast<const T*>(v), ld_v,
                                     Divisor(c.G), Divisor(n), by_block(c), static_cast<uint32_t>(rows), dev_status));
    return B2KV_OK;
}

template <typename T, int NG, int BITS, bool kValues>
int launch_read(const b2kv_qcache& c, void* out, int n, int last, int len_bias, int32_t* dev_status, void* stream) {
    const int64_t rows = static_cast<int64_t>(c.B) * n * c.G;
    if (rows > 0x7fffffff) return B2KV_ERR_UNSUPPORTED;
    OverlapLaunch launch(static_cast<unsigned>((rows + kThreads / 4 - 1) / (kThreads / 4)), kThreads, 0, stream);
    B2KV_CUDA_TRY(cudaLaunchKernelEx(&launch.cfg, read_kernel<T, NG, BITS, kValues>, c, static_cast<T*>(out), n, last, len_bias, Divisor(c.G), Divisor(n),
                                     by_block(c), static_cast<uint32_t>(rows), dev_status));
    return B2KV_OK;
}

// fn(NG as a type) for the cache's head size.
template <int N>
struct Groups {
    static constexpr int value = N;
};
template <typename F>
int by_size(int D, F&& fn) {
    switch (D) {
        case 32: return fn(Groups<1>());
        case 64: return fn(Groups<2>());
        case 96: return fn(Groups<3>());
        case 128: return fn(Groups<4>());
        default: return fn(Groups<8>());
    }
}

template <typename T>
int write_typed(const b2kv_qcache& c, const void* k, int64_t ld_k, const void* v, int64_t ld_v, int n, int32_t* dev_status, void* stream) {
    return by_size(c.D, [&](auto groups) {
        constexpr int NG = decltype(groups)::value;
        if (c.k_bits == 4) return launch_write<T, NG, 4, 4>(c, k, ld_k, v, ld_v, n, dev_status, stream);
        if (c.v_bits == 4) return launch_write<T, NG, 8, 4>(c, k, ld_k, v, ld_v, n, dev_status, stream);
        return launch_write<T, NG, 8, 8>(c, k, ld_k, v, ld_v, n, dev_status, stream);
    });
}

template <typename T>
int read_typed(const b2kv_qcache& c, int which, void* out, int n, int last, int len_bias, int32_t* dev_status, void* stream) {
    return by_size(c.D, [&](auto groups) {
        constexpr int NG = decltype(groups)::value;
        if (which == 0)
            return c.k_bits == 4 ? launch_read<T, NG, 4, false>(c, out, n, last, len_bias, dev_status, stream)
                                 : launch_read<T, NG, 8, false>(c, out, n, last, len_bias, dev_status, stream);
        return c.v_bits == 4 ? launch_read<T, NG, 4, true>(c, out, n, last, len_bias, dev_status, stream)
                             : launch_read<T, NG, 8, true>(c, out, n, last, len_bias, dev_status, stream);
    });
}

}  // namespace
}  // namespace qcache
}  // namespace b2kv

using namespace b2kv;

extern "C" {

int b2kv_qcache_scale_row(int D) {
    return D == 32 || D == 64 || D == 96 || D == 128 || D == 256 ? qcache::scale_row(D / qcache::kGroup) : 0;
}

int b2kv_qcache_write(const b2kv_qcache* cache, const void* k, int64_t ld_k, const void* v, int64_t ld_v, int n, int32_t* dev_status, void* stream) {
    const int rc = qcache::check(cache);
    if (rc != B2KV_OK) return rc;
    if (!k || !v || n <= 0 || n > cache->T_max) return B2KV_ERR_BAD_ARG;
    const int64_t cols = static_cast<int64_t>(cache->G) * cache->D;
    if (ld_k < cols || ld_v < cols) return B2KV_ERR_BAD_ARG;
    if (cache->seq_lens == nullptr && (cache->len < 0 || cache->len > cache->T_max - n)) return B2KV_ERR_BAD_ARG;
    const int es = elt_bytes(cache->dtype);
    if (!aligned16(k) || !aligned16(v) || !stride_ok(ld_k, es) || !stride_ok(ld_v, es)) return B2KV_ERR_ALIGN;
    return cache->dtype == B2KV_DTYPE_F32 ? qcache::write_typed<float>(*cache, k, ld_k, v, ld_v, n, dev_status, stream)
                                          : qcache::write_typed<__nv_bfloat16>(*cache, k, ld_k, v, ld_v, n, dev_status, stream);
}

int b2kv_qcache_read(const b2kv_qcache* cache, int which, void* out, int n, int last, int len_bias, int32_t* dev_status, void* stream) {
    const int rc = qcache::check(cache);
    if (rc != B2KV_OK) return rc;
    if (!out || n <= 0 || (which != 0 && which != 1)) return B2KV_ERR_BAD_ARG;
    if (!aligned16(out)) return B2KV_ERR_ALIGN;
    return cache->dtype == B2KV_DTYPE_F32 ? qcache::read_typed<float>(*cache, which, out, n, last, len_bias, dev_status, stream)
                                          : qcache::read_typed<__nv_bfloat16>(*cache, which, out, n, last, len_bias, dev_status, stream);
}

}  // extern "C"
