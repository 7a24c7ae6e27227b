// Attention over a quantised cache, heads of 256 elements.
#include "qcache_attend.cuh"

int b2kv::qcache::attend_256(const AttendParams& p, const Plan& plan, void* stream) { return attend_bits<8>(p, plan, stream); }
