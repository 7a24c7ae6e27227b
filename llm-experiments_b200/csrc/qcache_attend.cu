// Attention over a quantised cache: checks, how the work is cut, and which instance runs.
#include "qcache_attend.cuh"

#include <math.h>

#include <algorithm>
#include <atomic>
#include <chrono>

namespace b2kv {
namespace qcache {
namespace {

int check_attend(const b2kv_qcache* c, const b2kv_qcache_attend_args* a) {
    const int rc = check(c);
    if (rc != B2KV_OK) return rc;
    if (a == nullptr || !a->q || !a->out) return B2KV_ERR_BAD_ARG;
    if (a->H <= 0 || a->H % c->G != 0 || a->m <= 0 || a->T_upper < 0 || a->T_upper > c->T_max || a->window < 0) return B2KV_ERR_BAD_ARG;
    if (a->m > B2KV_QCACHE_MAX_ROWS) return B2KV_ERR_UNSUPPORTED;
    if (!isfinite(a->scale) || !isfinite(a->softcap) || !(a->softcap == 0.0f || a->softcap >= 1e-30f)) return B2KV_ERR_BAD_ARG;  // (its reciprocal is taken)
    const int64_t cols = static_cast<int64_t>(a->H) * c->D;
    if (a->ld_q < cols || a->ld_out < cols) return B2KV_ERR_BAD_ARG;
    const int es = elt_bytes(c->dtype);
    if (!aligned16(a->q) || !aligned16(a->out) || !stride_ok(a->ld_q, es) || !stride_ok(a->ld_out, es)) return B2KV_ERR_ALIGN;
    return B2KV_OK;
}

// Results of two pairs per CTA, their sums, and a ticket per pair.
size_t tickets_at(const Plan& plan, const b2kv_qcache& c) { return static_cast<size_t>(plan.ctas) * 2 * plan.cols * (c.D + 1) * sizeof(float); }

constexpr int kMostCluster = 8;

// Clusters of that many CTAs that a launch gets going together.  A cluster lies within one group of SMs, so there are fewer than there are places for
// its CTAs (sizes 2 - 8: 148, 93, 71, 56, 45, 37, 33 for 296 CTAs), and the last of them wait for what an earlier launch leaves behind: one
// in sixteen is not counted on (1024 tokens, 32 pairs: 8.0 us in clusters of 7, 10.5 of 8; 36 pairs: 8.0 of 6, 9.3 of 7, 14.2 of 8; 73 pairs: 9.5 of 3, 14.9 of 4).
int64_t cluster_places(int size) {
    static std::atomic<int> known[64][kMostCluster + 1];
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess) device = 64;
    int count = device < 64 ? known[device][size].load(std::memory_order_relaxed) : 0;
    if (count == 0) {
        count = size == 1 ? device_sm_count() * 2 : clusters_at_once(size);
        if (count <= 0) count = std::max(1, device_sm_count() * 2 / size);
        if (size > 2) count -= count / 16;
        if (device < 64) known[device][size].store(count, std::memory_order_relaxed);
    }
    return count;
}

bool make_plan(const b2kv_qcache& c, const b2kv_qcache_attend_args& a, Plan& plan) {
    const int columns = a.m * (a.H / c.G);
    const int most = a.window > 0 ? static_cast<int>(std::min<int64_t>(a.T_upper, static_cast<int64_t>(a.window) + a.m - 1)) : a.T_upper;
    const int64_t heads = static_cast<int64_t>(c.B) * c.G;
    const int at_once = device_sm_count() * 2;  // CTAs that run at the same time
    // Columns (new token, query head) of a key / value head that are taken together: 16 share the widening of the codes (4 sequences of 131072
    // tokens, 16 heads to one: 198 against 242 us), 8 make more pairs where there are few tokens to a CTA (40 columns over 2048 tokens: 22.1 against 25.5 us).
    // Keys of 8 and values of 4 bits in heads of 256 have no form of 16 (kWide): it took 261.5 -> 296.8 us for 4 sequences of 65536 tokens and 16 heads to one,
    // 212.2 -> 248.0 for 64 of 2048 .. 4096, 108.5 -> 140.9 for 16 columns over 32 of 4096 .. 8192.  With the same bits for both it pays at length
    // ((4, 4) 227.3 -> 200.4 us and 198.1 -> 183.8, (8, 8) 359.5 -> 275.1 and 257.5 -> 251.6) and costs up to 8 and 18 % in the last case.
    const int forced_columns = tune_get("qcache_columns");
    const bool wide = c.dtype != B2KV_DTYPE_F32 && (c.D != 256 || c.k_bits == c.v_bits) &&
                      (forced_columns != 0 ? forced_columns == 16 : columns > 8 && heads * ((columns + 15) / 16) * most >= at_once * 1024ll);
    plan.cols = c.dtype == B2KV_DTYPE_F32 ? 4 : wide ? 16 : 8;
    plan.col_tiles = (columns + plan.cols - 1) / plan.cols;
    plan.pairs = heads * plan.col_tiles;
    if (plan.pairs > 0x7fffffff) return false;
    // A cluster of 1 - 8 CTAs for each pair, or one run of tiles per CTA that is there.  In tokens that a CTA gets through in the time (bf16 rows, heads of 128): setting
    // up and finishing a CTA is about 430, putting a cluster's results together 150, finding and cutting a run 1000 and each piece of a pair, which one CTA
    // puts together, another 10: so few pairs are cut into no more pieces than pay (one pair of 131072 tokens: 27 us in 115 pieces, 43 in 296; of
    // 8192: 12.5 in 29, 35.6 in 296; 320 pairs of 400: 18.8 in runs, 14.4 as they are).
    const int64_t pieces = static_cast<int64_t>(sqrt(most / 10.0)) + 1;
    const int run_ctas = static_cast<int>(std::min<int64_t>(at_once, plan.pairs * pieces));
    const int64_t runs = 1000 + plan.pairs * (most + 16 * kPairCost) / run_ctas + 10 * run_ctas / plan.pairs;
    int64_t best = 0;
    for (int size = 1; size <= kMostCluster; ++size) {
        const int64_t places = cluster_places(size), waves = (plan.pairs + places - 1) / places;
        const int64_t cost = waves * (430 + (size > 1 ? 150 : 0) + (most + size - 1) / size);
        if (size == 1 || cost < best) best = cost, plan.cluster = size;
    }
    // (a run counts units in 32 bits)
    const bool countable = plan.pairs * (most / 16 + 1 + kPairCost) < (1ll << 31);
    if (runs < best && countable) plan.cluster = 0;
    const int forced = tune_get("qcache_cluster");
    if (forced >= 1 && forced <= kMostCluster) plan.cluster = forced;
    if (forced < 0 && countable) plan.cluster = 0;
    plan.workspace = 0;
    if (plan.cluster == 0) {
        plan.ctas = run_ctas;
        plan.workspace = tickets_at(plan, c) + static_cast<size_t>(plan.pairs) * sizeof(unsigned long long);
    } else {
        if (plan.pairs * plan.cluster > 0x7fffffff) return false;
        plan.ctas = static_cast<int>(plan.pairs) * plan.cluster;
    }
    return true;
}

}  // namespace
}  // namespace qcache
}  // namespace b2kv

using namespace b2kv;

extern "C" {

size_t b2kv_qcache_attend_workspace_bytes(const b2kv_qcache* cache, const b2kv_qcache_attend_args* args) {
    qcache::Plan plan;
    return qcache::check_attend(cache, args) == B2KV_OK && qcache::make_plan(*cache, *args, plan) ? plan.workspace : 0;
}

int b2kv_qcache_attend(const b2kv_qcache* cache, const b2kv_qcache_attend_args* args, void* workspace, size_t workspace_bytes, int32_t* dev_status,
                       void* stream) {
    using namespace qcache;
    const int rc = check_attend(cache, args);
    if (rc != B2KV_OK) return rc;
    const b2kv_qcache& c = *cache;
    const b2kv_qcache_attend_args& a = *args;
    Plan plan;
    if (!make_plan(c, a, plan)) return B2KV_ERR_UNSUPPORTED;
    if (plan.workspace > 0) {
        if (workspace == nullptr || workspace_bytes < plan.workspace) return B2KV_ERR_WORKSPACE;
        if (!aligned16(workspace)) return B2KV_ERR_ALIGN;
    }
    AttendParams p{};
    p.c = c;
    p.by_block = by_block(c);
    p.q = a.q, p.out = a.out, p.slopes = a.slopes, p.dev_status = dev_status;
    p.ld_q = a.ld_q, p.ld_out = a.ld_out;
    p.R = a.H / c.G, p.m = a.m, p.col_tiles = plan.col_tiles, p.T_upper = a.T_upper, p.len_bias = a.len_bias;
    p.window = static_cast<int>(std::min<int64_t>(a.window, static_cast<int64_t>(a.T_upper) + a.m));  // (no sum with it overflows)
    p.cluster = plan.cluster;
    p.scale = static_cast<float>(frexp(static_cast<double>(a.scale) * M_LOG2E, &p.scale_exp));
    // A cap beyond 2^126 is taken for that, whose inverse is a normal number, and its product with log2 e is finite.  (Scores that would show the difference lie
    // above 2^114, where the next fp32 number is 2^91 away.)
    p.cap = static_cast<float>(std::min(a.softcap * M_LOG2E, 0x1p126));
    p.ws_o = static_cast<float*>(workspace);
    p.ws_lse = p.ws_o + static_cast<size_t>(plan.ctas) * 2 * plan.cols * c.D;
    p.tickets = reinterpret_cast<unsigned long long*>(static_cast<char*>(workspace) + tickets_at(plan, c));
    static std::atomic<unsigned long long> calls{static_cast<unsigned long long>(std::chrono::steady_clock::now().time_since_epoch().count())};
    do p.call = calls.fetch_add(1, std::memory_order_relaxed) & 0xffffffffffull;
    while (p.call == 0);
    switch (c.D) {
        case 32: return attend_32(p, plan, stream);
        case 64: return attend_64(p, plan, stream);
        case 96: return attend_96(p, plan, stream);
        case 128: return attend_128(p, plan, stream);
        default: return attend_256(p, plan, stream);
    }
}

}  // extern "C"
