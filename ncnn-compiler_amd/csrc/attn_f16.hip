// The attention kernels for f16 queries.
#include "attention.h"

namespace nhip {

int attn_run_f16(const AttnArgs& a, int src, hipStream_t s) { return attn::run<f16>(a, src, s); }

}  // namespace nhip
