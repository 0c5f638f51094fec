// attention_kernels.hip — the attention kernels (attention_impl.h) for one pair of types and one head size,
// compiled once for each: ATTN_CACHE and ATTN_IO are the types of the cache and of the activations, ATTN_DIM the
// largest head size, ATTN_NAME the launch function
#include "attention_impl.h"

namespace mi355x {

hipError_t ATTN_NAME(const AttnArgs &a, const AttnPlan &pl, void *work, hipStream_t st) {
    return launch_attn_any<ATTN_CACHE, ATTN_IO, ATTN_DIM>(a, pl, work, st);
}

}  // namespace mi355x
