// paged_attn_kernel on FP16 pages.
#include "paged_attn.h"

namespace jitnn {

void paged_attn_launch_f16(int D, unsigned blocks, hipStream_t s, const AttnArgs &a) { paged_attn_pick<_Float16>(D, blocks, s, a); }

}  // namespace jitnn
