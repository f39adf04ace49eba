// Launches of the router of a mixture of experts.
#include "router.h"

#include <algorithm>

namespace jitnn {

// One launch for logits and choice: few experts, and few enough tokens for a workgroup each.
static bool one_launch(int tokens, int experts, int d, bool lists) { return !lists && (long long)experts * d <= 131072 && tokens <= 64; }

bool router_needs_logits(int tokens, int experts, int d, bool lists) { return !one_launch(tokens, experts, d, lists); }

void router_launch(const RouterArgs &a, hipStream_t s) {
    const bool lists = a.lists.list != nullptr;
    if (one_launch(a.tokens, a.experts, a.d, lists)) {
        hipLaunchKernelGGL(router_one_kernel, dim3(a.tokens), dim3(1024), 0, s, a);
        return;
    }
    if (a.tokens <= 8) hipLaunchKernelGGL(router_logits_kernel, dim3((a.experts + 3) / 4, a.tokens), dim3(256), 0, s, a);
    else hipLaunchKernelGGL(router_tiles_kernel, dim3((a.tokens + 15) / 16, (a.experts + 15) / 16), dim3(256), 0, s, a);
    if (lists && a.tokens <= CHOOSE_FEW) {
        const int waves = std::max(1, std::min(16, 2048 / a.experts));  // (at most 32 KiB for the logits and their order)
        hipLaunchKernelGGL(choose_few_kernel, dim3(1), dim3(1024), (size_t)waves * 16 * a.experts, s, a, waves);
        return;
    }
    hipLaunchKernelGGL(choose_kernel, dim3((a.tokens + 3) / 4), dim3(256), (size_t)64 * a.experts, s, a);
    if (lists) expert_lists_launch(a.ids, a.tokens * a.used, a.experts, a.lists, s);
}

void expert_lists_launch(const int *ids, int slots, int experts, const ExpertLists &lists, hipStream_t s) {
    hipLaunchKernelGGL(expert_lists_kernel, dim3(1), dim3(1024), 0, s, ids, slots, experts, lists);
}

}  // namespace jitnn
