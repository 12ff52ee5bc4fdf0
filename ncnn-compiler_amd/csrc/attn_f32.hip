// The attention kernels for f32 queries.
#include "attention.h"

namespace nhip {

int attn_run_f32(const AttnArgs& a, int src, hipStream_t s) { return attn::run<float>(a, src, s); }

}  // namespace nhip
