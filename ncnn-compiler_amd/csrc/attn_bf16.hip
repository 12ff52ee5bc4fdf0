// The attention kernels for bf16 queries.
#include "attention.h"

namespace nhip {

int attn_run_bf16(const AttnArgs& a, int src, hipStream_t s) { return attn::run<bf16>(a, src, s); }
int attn_prefix_bf16(const AttnArgs& prefix, const AttnArgs& own, hipStream_t s) { return attn::run_prefix<bf16>(prefix, own, s); }

}  // namespace nhip
