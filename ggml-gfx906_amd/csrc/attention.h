// attention.h — what the attention kernels (attention_impl.h) and their host side (attention.cpp) share
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mi355x {

struct AttnArgs {
    const char *q; int64_t q_i, q_h, q_b;
    const char *k; int64_t k_j, k_h, k_b;
    const char *v; int64_t v_j, v_h, v_b;
    const char *kp; int64_t kp_j, kp_h;              // the shared prefix, or n_prefix = 0
    const char *vp; int64_t vp_j, vp_h;
    const char *mask; int64_t m_i, m_h, m_b;         // f16, or nullptr
    int m_nh, m_nb;                                  // its head and batch planes
    bool m_vec;                                      // rows of 8-byte aligned groups of four
    const float *sinks;
    const char *len; int64_t len_b;                  // i32 [batch], or nullptr: n_kv
    char *o; int64_t o_i, o_h, o_b;
    int D, n_q, n_kv, n_prefix, H, Hk, B, kv_b;      // kv_b: batches that share one cache
    int causal;
    float scale, cap;                                // cap = 0: none
    int bias_heads;                                  // slopes: 0 = none, else the power of two of heads
    float m0, m1;
};

constexpr int ATTN_MAX_SLOTS = 256;   // partial results of a row

// what a call launches, by its shapes alone
struct AttnPlan {
    bool tiled;                              // else attn_rows_kernel
    bool own_rows, pre_rows;                 // row tiles of 128 (4 waves of 32), or 32 rows with split keys
    int own_tiles, own_splits, pre_tiles, pre_splits, slots;
};

// the launches of one call: cache type, then activation type (attention_f16.hip, attention_bf16.hip,
// attention_f32.hip). `work`: the partial results of pl.slots > 1
hipError_t attn_launch_f16(const AttnArgs &a, const AttnPlan &pl, void *work, hipStream_t st);
hipError_t attn_launch_bf16(const AttnArgs &a, const AttnPlan &pl, void *work, hipStream_t st);
hipError_t attn_launch_f16_f32(const AttnArgs &a, const AttnPlan &pl, void *work, hipStream_t st);

}  // namespace mi355x
