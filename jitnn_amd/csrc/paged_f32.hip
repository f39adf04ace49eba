// paged_attn_kernel on FP32 pages.
#include "paged_attn.h"

namespace jitnn {

void paged_attn_launch_f32(int D, unsigned blocks, hipStream_t s, const AttnArgs &a) { paged_attn_pick<float>(D, blocks, s, a); }

}  // namespace jitnn
