// Attention over a quantised cache, heads of 64 elements.
#include "qcache_attend.cuh"

int b2kv::qcache::attend_64(const AttendParams& p, const Plan& plan, void* stream) { return attend_bits<2>(p, plan, stream); }
