// attention_bf16.hip — the attention kernels (attention_impl.h) for bf16 cache and activations
#include "attention_impl.h"

namespace mi355x {

hipError_t attn_launch_bf16(const AttnArgs &a, const AttnPlan &pl, void *work, hipStream_t st) {
    return launch_attn_any<__bf16, __bf16>(a, pl, work, st);
}

}  // namespace mi355x
