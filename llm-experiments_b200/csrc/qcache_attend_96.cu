// Attention over a quantised cache, heads of 96 elements.
#include "qcache_attend.cuh"

int b2kv::qcache::attend_96(const AttendParams& p, const Plan& plan, void* stream) { return attend_bits<3>(p, plan, stream); }
