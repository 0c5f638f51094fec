// attention_f32.hip — the attention kernels (attention_impl.h) for f16 cache, f32 activations
#include "attention_impl.h"

namespace mi355x {

hipError_t attn_launch_f16_f32(const AttnArgs &a, const AttnPlan &pl, void *work, hipStream_t st) {
    return launch_attn_any<_Float16, float>(a, pl, work, st);
}

}  // namespace mi355x
