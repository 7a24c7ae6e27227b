// Quantised key / value cache: what its kernels share.  The form is in b2kv.h.
#pragma once

#include "b2kv_common.cuh"

namespace b2kv {
namespace qcache {

constexpr int kGroup = 32;  // elements that share a scale

// bfloat16 per row of scales: the groups of a row, rounded up so that a row is 4, 8 or 16 bytes, which cp.async takes whole.
__host__ __device__ constexpr int scale_row(int groups) { return groups <= 2 ? 2 : groups <= 4 ? 4 : 8; }

// Checks that every entry makes: pointers, sizes and types of the cache.
int check(const b2kv_qcache* c);

__device__ __forceinline__ int tokens_held(const b2kv_qcache& c, int b) { return c.seq_lens ? c.seq_lens[b] : c.len; }

// Quotients by a divisor that the host knows, of numbers below 2^31: m / 2^(31 + l) is above 1 / d by less than 2^-31 / d.
struct Divisor {
    uint32_t d, m;
    int shift;
    explicit Divisor(uint32_t by = 1) : d(by) {
        int l = 0;
        while ((1ull << l) < by) ++l;
        shift = 31 + l;
        m = static_cast<uint32_t>(((1ull << shift) + by - 1) / by);
    }
    __device__ __forceinline__ uint32_t quotient(uint32_t n) const { return static_cast<uint32_t>((static_cast<uint64_t>(n) * m) >> shift); }
};
inline Divisor by_block(const b2kv_qcache& c) { return Divisor(c.block_table != nullptr ? c.block_size : 1); }

// Row of token t (0 <= t < T_max) of sequence b, head g; -1 for a table entry outside the pool, which is recorded.
__device__ __forceinline__ int64_t row_of(const b2kv_qcache& c, const Divisor& by_block, int b, int g, int t, int32_t* dev_status) {
    if (c.block_table == nullptr) return (static_cast<int64_t>(b) * c.G + g) * c.T_max + t;
    const int j = static_cast<int>(by_block.quotient(t));
    const int blk = c.block_table[static_cast<int64_t>(b) * c.max_blocks + j];
    if (blk < 0 || blk >= c.n_blocks) {
        report_status(dev_status, B2KV_DEV_BAD_BLOCK);
        return -1;
    }
    return (static_cast<int64_t>(blk) * c.G + g) * c.block_size + (t - j * c.block_size);
}

}  // namespace qcache
}  // namespace b2kv
