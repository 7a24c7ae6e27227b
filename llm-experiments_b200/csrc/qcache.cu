// Quantised key / value cache: rows into it and out of it.
//
// Both are streams: a row of D elements comes in at D * (2 or 4) bytes and leaves at D * bits / 8 + D / 16, or the other way round.
// One thread has 8 neighbouring elements (16 bytes of bfloat16), four threads next to one another a group: its largest
// magnitude is two shuffles away.
//
// A code is the quotient rounded to the nearest whole number, ties to even, as if it had been computed exactly.  The fp32 division
// gives that: x / scale lies exactly on a border n + 1/2 only if it is one.  (A border times the scale has at most 8 + 8
// bits, so it is a float; the next float away from it, a step u, moves the quotient by u / scale, which is more than half a step of
// the quotient, because the scale's mantissa is below 2.  So no other quotient rounds onto the border.)  The same holds for max / L.
#include "qcache.cuh"

#include <algorithm>

namespace b2kv {
namespace qcache {

int check(const b2kv_qcache* c) {
    if (c == nullptr) return B2KV_ERR_BAD_ARG;
    if (elt_bytes(c->dtype) == 0 || b2kv_qcache_scale_row(c->D) == 0) return B2KV_ERR_UNSUPPORTED;
    const bool bits = (c->k_bits == 4 && c->v_bits == 4) || (c->k_bits == 8 && (c->v_bits == 4 || c->v_bits == 8));
    if (!bits) return B2KV_ERR_UNSUPPORTED;
    if (!c->k_codes || !c->v_codes || !c->k_scales || !c->v_scales) return B2KV_ERR_BAD_ARG;
    if (c->B <= 0 || c->G <= 0 || c->T_max <= 0) return B2KV_ERR_BAD_ARG;
    if (c->block_table != nullptr) {
        if (c->max_blocks <= 0 || c->block_size <= 0 || c->n_blocks <= 0) return B2KV_ERR_BAD_ARG;
        if (static_cast<int64_t>(c->max_blocks) * c->block_size < c->T_max) return B2KV_ERR_BAD_ARG;
    }
    if (!aligned16(c->k_codes) || !aligned16(c->v_codes) || !aligned16(c->k_scales) || !aligned16(c->v_scales)) return B2KV_ERR_ALIGN;
    return B2KV_OK;
}

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ void load8(const float* p, float (&f)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&f)[8]) {
    Elt<__nv_bfloat16>::widen(*reinterpret_cast<const uint4*>(p), f);
}
__device__ __forceinline__ void store8(float* p, const float (&f)[8]) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&f)[8]) {
    __nv_bfloat162 h[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = __floats2bfloat162_rn(f[2 * e], f[2 * e + 1]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(h);
}

// Eight stored codes of a group from its elements; every lane of the four that hold the group gets the scale.
template <int BITS>
__device__ __forceinline__ uint2 quantise(const float (&f)[8], __nv_bfloat16& scale) {
    constexpr int kTop = BITS == 4 ? 7 : 127;
    float most = 0.0f;
    bool finite = true;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        most = fmaxf(most, fabsf(f[e]));
        finite = finite && fabsf(f[e]) <= 3.402823466e38f;
    }
    most = finite ? most : __int_as_float(0x7f800000);
    most = fmaxf(most, __shfl_xor_sync(~0u, most, 1));
    most = fmaxf(most, __shfl_xor_sync(~0u, most, 2));
    finite = most <= 3.402823466e38f;
    scale = __float2bfloat16_rn(finite ? most / static_cast<float>(kTop) : __int_as_float(0x7fc00000));
    const float s = __bfloat162float(scale);
    uint2 w = make_uint2(0, 0);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float q = s > 0.0f ? fminf(fmaxf(rintf(f[e] / s), -kTop), kTop) : 0.0f;
        const uint32_t c = static_cast<uint32_t>(static_cast<int>(q) + kTop + 1);
        if (BITS == 4)
            w.x |= c << (4 * e);
        else
            (e < 4 ? w.x : w.y) |= c << (8 * (e & 3));
    }
    return w;
}

// Octet o of group u of a row of `groups` groups; values are units of half an octet.
template <int BITS, bool kValues>
__device__ __forceinline__ void store_codes(uint8_t* row, int groups, int u, int o, uint2 w) {
    if (!kValues && BITS == 4) {
        reinterpret_cast<uint32_t*>(row)[o * groups + u] = __funnelshift_l(w.x, w.x, 2);
    } else if (!kValues) {
        reinterpret_cast<uint2*>(row)[o * groups + u] = w;
    } else if (BITS == 4) {
        w.x = ((w.x << 2) & 0xfffcfffcu) | ((w.x >> 14) & 0x00030003u);
        reinterpret_cast<uint16_t*>(row)[2 * o * groups + u] = static_cast<uint16_t>(w.x);
        reinterpret_cast<uint16_t*>(row)[(2 * o + 1) * groups + u] = static_cast<uint16_t>(w.x >> 16);
    } else {
        reinterpret_cast<uint32_t*>(row)[2 * o * groups + u] = w.x;
        reinterpret_cast<uint32_t*>(row)[(2 * o + 1) * groups + u] = w.y;
    }
}
template <int BITS, bool kValues>
__device__ __forceinline__ uint2 load_codes(const uint8_t* row, int groups, int u, int o) {
    if (!kValues && BITS == 4) {
        const uint32_t w = reinterpret_cast<const uint32_t*>(row)[o * groups + u];
        return make_uint2(__funnelshift_r(w, w, 2), 0);
    }
    if (!kValues) return reinterpret_cast<const uint2*>(row)[o * groups + u];
    if (BITS == 4) {
        const uint32_t w = reinterpret_cast<const uint16_t*>(row)[2 * o * groups + u] |
                           static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(row)[(2 * o + 1) * groups + u]) << 16;
        return make_uint2(((w >> 2) & 0x3fff3fffu) | ((w << 14) & 0xc000c000u), 0);
    }
    return make_uint2(reinterpret_cast<const uint32_t*>(row)[2 * o * groups + u], reinterpret_cast<const uint32_t*>(row)[(2 * o + 1) * groups + u]);
}

// Thread = octet; grid.y 0 keys, 1 values.  `octets` is B * n * G * D / 8, a multiple of four: the lanes of a group are all inside or all outside.
template <typename T, int KB, int VB>
__global__ void __launch_bounds__(kThreads) write_kernel(b2kv_qcache c, const T* k, int64_t ld_k, const T* v, int64_t ld_v, int n, int64_t octets,
                                                         int32_t* dev_status) {
    grid_launch_dependents();
    grid_dependency_wait();
    const int64_t at = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    const bool inside = at < octets;
    const int groups = c.D / kGroup, per_row = c.D / 8;
    const int64_t i = inside ? at : 0;  // (lanes behind the end go along with the shuffles)
    const int64_t head_row = i / per_row;
    const int j = static_cast<int>(i - head_row * per_row), u = j >> 2, o = j & 3;
    const int64_t src = head_row / c.G;
    const int g = static_cast<int>(head_row - src * c.G), b = static_cast<int>(src / n);
    const int64_t place = static_cast<int64_t>(tokens_held(c, b)) + (src - static_cast<int64_t>(b) * n);
    int64_t row = -1;
    if (place < 0 || place >= c.T_max)
        report_status(dev_status, B2KV_DEV_BAD_POSITION);
    else
        row = row_of(c, b, g, static_cast<int>(place), dev_status);
    float f[8];
    __nv_bfloat16 scale;
    const bool values = blockIdx.y != 0;
    load8((values ? v + src * ld_v : k + src * ld_k) + static_cast<int64_t>(g) * c.D + j * 8, f);
    const uint2 w = (values ? VB : KB) == 4 ? quantise<4>(f, scale) : quantise<8>(f, scale);
    if (!inside || row < 0) return;
    if (values)
        store_codes<VB, true>(static_cast<uint8_t*>(c.v_codes) + row * (c.D * VB / 8), groups, u, o, w);
    else
        store_codes<KB, false>(static_cast<uint8_t*>(c.k_codes) + row * (c.D * KB / 8), groups, u, o, w);
    if (o == 0) {
        __nv_bfloat16* const to = static_cast<__nv_bfloat16*>(values ? c.v_scales : c.k_scales) + row * scale_row(groups);
        to[u] = scale;
        if (u == groups - 1)  // the rest takes part in products, with zeros
            for (int r = groups; r < scale_row(groups); ++r) to[r] = __float2bfloat16_rn(0.0f);
    }
}

// Thread = octet of the output.
template <typename T, int BITS, bool kValues>
__global__ void __launch_bounds__(kThreads) read_kernel(b2kv_qcache c, T* out, int n, int last, int len_bias, int64_t octets, int32_t* dev_status) {
    grid_launch_dependents();
    grid_dependency_wait();
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    if (i >= octets) return;
    const int groups = c.D / kGroup, per_row = c.D / 8;
    const int64_t head_row = i / per_row;
    const int j = static_cast<int>(i - head_row * per_row), u = j >> 2, o = j & 3;
    const int64_t dst = head_row / c.G;
    const int g = static_cast<int>(head_row - dst * c.G), b = static_cast<int>(dst / n);
    const int64_t held = min(static_cast<int64_t>(tokens_held(c, b)) + len_bias, static_cast<int64_t>(c.T_max));
    const int64_t place = dst - static_cast<int64_t>(b) * n + (last ? held - n : 0);
    float f[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    const int64_t row = place >= 0 && place < held ? row_of(c, b, g, static_cast<int>(place), dev_status) : -1;
    if (row >= 0) {
        const float s = __bfloat162float(static_cast<const __nv_bfloat16*>(kValues ? c.v_scales : c.k_scales)[row * scale_row(groups) + u]);
        const uint2 w = load_codes<BITS, kValues>(static_cast<const uint8_t*>(kValues ? c.v_codes : c.k_codes) + row * (c.D * BITS / 8), groups, u, o);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t code = BITS == 4 ? (w.x >> (4 * e)) & 15u : ((e < 4 ? w.x : w.y) >> (8 * (e & 3))) & 255u;
            f[e] = static_cast<float>(static_cast<int>(code) - (1 << (BITS - 1))) * s;  // exact: 8 bits by 8
        }
    }
    store8(out + i * 8, f);
}

template <typename T, int KB, int VB>
int launch_write(const b2kv_qcache& c, const void* k, int64_t ld_k, const void* v, int64_t ld_v, int n, int32_t* dev_status, void* stream) {
    const int64_t octets = static_cast<int64_t>(c.B) * n * c.G * (c.D / 8);
    const int64_t blocks = (octets + kThreads - 1) / kThreads;
    if (blocks > 0x7fffffff) return B2KV_ERR_UNSUPPORTED;
    OverlapLaunch launch(dim3(static_cast<unsigned>(blocks), 2), kThreads, 0, stream);
    B2KV_CUDA_TRY(cudaLaunchKernelEx(&launch.cfg, write_kernel<T, KB, VB>, c, static_cast<const T*>(k), ld_k, static_cast<const T*>(v), ld_v, n, octets,
                                     dev_status));
    return B2KV_OK;
}

template <typename T, int BITS, bool kValues>
int launch_read(const b2kv_qcache& c, void* out, int n, int last, int len_bias, int32_t* dev_status, void* stream) {
    const int64_t octets = static_cast<int64_t>(c.B) * n * c.G * (c.D / 8);
    const int64_t blocks = (octets + kThreads - 1) / kThreads;
    if (blocks > 0x7fffffff) return B2KV_ERR_UNSUPPORTED;
    OverlapLaunch launch(static_cast<unsigned>(blocks), kThreads, 0, stream);
    B2KV_CUDA_TRY(cudaLaunchKernelEx(&launch.cfg, read_kernel<T, BITS, kValues>, c, static_cast<T*>(out), n, last, len_bias, octets, dev_status));
    return B2KV_OK;
}

template <typename T>
int write_typed(const b2kv_qcache& c, const void* k, int64_t ld_k, const void* v, int64_t ld_v, int n, int32_t* dev_status, void* stream) {
    if (c.k_bits == 4) return launch_write<T, 4, 4>(c, k, ld_k, v, ld_v, n, dev_status, stream);
    if (c.v_bits == 4) return launch_write<T, 8, 4>(c, k, ld_k, v, ld_v, n, dev_status, stream);
    return launch_write<T, 8, 8>(c, k, ld_k, v, ld_v, n, dev_status, stream);
}

template <typename T>
int read_typed(const b2kv_qcache& c, int which, void* out, int n, int last, int len_bias, int32_t* dev_status, void* stream) {
    if (which == 0)
        return c.k_bits == 4 ? launch_read<T, 4, false>(c, out, n, last, len_bias, dev_status, stream)
                             : launch_read<T, 8, false>(c, out, n, last, len_bias, dev_status, stream);
    return c.v_bits == 4 ? launch_read<T, 4, true>(c, out, n, last, len_bias, dev_status, stream)
                         : launch_read<T, 8, true>(c, out, n, last, len_bias, dev_status, stream);
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
