// The attention kernels for bf16 queries.
#include "attention.h"

namespace nhip {

int attn_run_bf16(const AttnArgs& a, int src, hipStream_t s) { return attn::run<bf16>(a, src, s); }

}  // namespace nhip
