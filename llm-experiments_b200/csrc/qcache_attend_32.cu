// Attention over a quantised cache, heads of 32 elements.
#include "qcache_attend.cuh"

int b2kv::qcache::attend_32(const AttendParams& p, const Plan& plan, void* stream) { return attend_bits<1>(p, plan, stream); }
