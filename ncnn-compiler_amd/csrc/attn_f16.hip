// The attention kernels for f16 queries.
#include "attention.h"

namespace nhip {

int attn_run_f16(const AttnArgs& a, int src, hipStream_t s) { return attn::run<f16>(a, src, s); }
int attn_prefix_f16(const AttnArgs& prefix, const AttnArgs& own, hipStream_t s) { return attn::run_prefix<f16>(prefix, own, s); }

}  // namespace nhip
