// Attention over a quantised cache, heads of 128 elements.
#include "qcache_attend.cuh"

int b2kv::qcache::attend_128(const AttendParams& p, const Plan& plan, void* stream) { return attend_bits<4>(p, plan, stream); }

// (All instances are two CTAs to an SM: one speaks for them all.)
int b2kv::qcache::clusters_at_once(int size) { return count_clusters<__nv_bfloat16, 4, 4, 4, 1>(size); }
