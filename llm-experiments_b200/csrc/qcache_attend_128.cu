// Attention over a quantised cache, heads of 128 elements.
#include "qcache_attend.cuh"

int b2kv::qcache::attend_128(const AttendParams& p, const Plan& plan, void* stream) { return attend_bits<4>(p, plan, stream); }
