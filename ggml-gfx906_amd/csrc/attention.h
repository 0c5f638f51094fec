// attention.h — what the attention kernels (attention_impl.h) and their host side (attention.cpp) share
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mi355x {

// n / d for 0 <= n < 2^31: the divisors are the same for a whole launch, a division takes some 40 instructions
struct Div {
    uint32_t d, mul, shift;
    __host__ __device__ Div(uint32_t by = 1) : d(by), shift(0) {
        while ((1ull << shift) < d) ++shift;
        mul = (uint32_t)((((1ull << shift) - d) << 32) / d + 1);
    }
    __device__ __forceinline__ int of(int n) const { return (int)((__umulhi((uint32_t)n, mul) + (uint32_t)n) >> shift); }
    __device__ __forceinline__ int rest(int n) const { return n - of(n) * (int)d; }
};

struct AttnArgs {
    const char *q; int64_t q_i, q_h, q_b;
    const char *k; int64_t k_j, k_h, k_b;
    const char *v; int64_t v_j, v_h, v_b;
    const char *kp; int64_t kp_j, kp_h;              // the shared prefix, or n_prefix = 0
    const char *vp; int64_t vp_j, vp_h;
    const char *mask; int64_t m_i, m_h, m_b;         // f16, or nullptr
    int m_nh, m_nb;                                  // its head and batch planes
    const float *sinks;
    const char *len; int64_t len_b;                  // i32 [batch], or nullptr: n_kv
    char *o; int64_t o_i, o_h, o_b;
    int D, n_q, n_kv, n_prefix, H, Hk, B;
    Div by_G, by_Hk, by_n_q, by_kv_b;                // G = H / Hk heads a key head; kv_b: batches that share one cache
    int causal;
    float scale, cap;                                // cap = 0: none
    int bias_heads;                                  // slopes: 0 = none, else the power of two of heads
    float m0, m1;
};

constexpr int ATTN_MAX_SLOTS = 256;   // partial results of a row

// what a call launches, by its shapes alone
struct AttnPlan {
    bool tiled;                              // else attn_rows_kernel
    int waves, turns;                        // of a workgroup; groups of its waves that have the same rows
    bool own_rows, pre_rows;                 // row tiles of 32 per wave, or 32 rows whose keys the waves split
    int own_tiles, own_splits, pre_tiles, pre_splits, slots;
};

// the launches of one call, by cache and activation type and by the head size the kernels are built for (D up
// to it; attention_kernels.hip). `work`: the partial results of pl.slots > 1
#define ATTN_LAUNCH(NAME) hipError_t NAME(const AttnArgs &a, const AttnPlan &pl, void *work, hipStream_t st);
ATTN_LAUNCH(attn_launch_f16_64)
ATTN_LAUNCH(attn_launch_f16_96)
ATTN_LAUNCH(attn_launch_f16_128)
ATTN_LAUNCH(attn_launch_f16_192)
ATTN_LAUNCH(attn_launch_f16_256)
ATTN_LAUNCH(attn_launch_bf16_64)
ATTN_LAUNCH(attn_launch_bf16_96)
ATTN_LAUNCH(attn_launch_bf16_128)
ATTN_LAUNCH(attn_launch_bf16_192)
ATTN_LAUNCH(attn_launch_bf16_256)
ATTN_LAUNCH(attn_launch_f32_64)
ATTN_LAUNCH(attn_launch_f32_96)
ATTN_LAUNCH(attn_launch_f32_128)
ATTN_LAUNCH(attn_launch_f32_192)
ATTN_LAUNCH(attn_launch_f32_256)
#undef ATTN_LAUNCH

}  // namespace mi355x
