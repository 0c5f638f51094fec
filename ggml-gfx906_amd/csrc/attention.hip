// attention.hip — softmax(scale * Q K^T + mask) V over a key / value cache (GGML_OP_FLASH_ATTN_EXT),
// and the same for sequences that share one long prefix.
//
// Per (batch b, head h, query i), with hk = h / (H / Hk) the shared key / value head:
//     x_j = cap * tanh(scale * q.k_j / cap)  [or scale * q.k_j]  + slope_h * mask_ij
//     o   = sum_j exp(x_j - m) v_j / (sum_j exp(x_j - m) + exp(sink_h - m)),  m = max(x, sink)
// over the keys j < len_b that the mask leaves (not -inf) and, when causal, j <= len_b - n_q + i.
// A row that sees nothing is zeros. A key that a row does not see takes no part in it, whatever its
// bytes hold: caches are not cleared, and a NaN times a weight of 0 would be NaN.
#include "../../include/ggml-mi355x.h"
#include "dispatch.h"
#include "qcommon.h"

#include <algorithm>
#include <cmath>

namespace mi355x {

namespace {

constexpr float LOG2E = 1.44269504088896340736f;

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
    int D, n_q, n_kv, n_prefix, H, Hk, B, kv_b;      // kv_b: batches that share one cache
    int causal;
    float scale, cap;                                // cap = 0: none
    int bias_heads;                                  // slopes: 0 = none, else the power of two of heads
    float m0, m1;
};

__device__ __forceinline__ float wave_add(float v) {
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) v += __shfl_xor(v, s, 64);
    return v;
}

__device__ __forceinline__ float slope_of(const AttnArgs &a, int h) {
    if (a.bias_heads == 0) return 1.0f;
    return h < a.bias_heads ? powf(a.m0, (float)(h + 1)) : powf(a.m1, (float)(2 * (h - a.bias_heads) + 1));
}

// a score in units of log 2: the cap and the factor log2(e), so that exp is one exp2
__device__ __forceinline__ float scaled(const AttnArgs &a, float s) {
    s *= a.scale;
    if (a.cap != 0.0f) s = a.cap * tanhf(s / a.cap);
    return s * LOG2E;
}

__device__ __forceinline__ int own_len(const AttnArgs &a, int b) {
    if (!a.len) return a.n_kv;
    return min(max(*reinterpret_cast<const int32_t *>(a.len + b * a.len_b), 0), a.n_kv);
}

// running softmax of one row, in one wave: lane l holds values l, l + 64, ... of the row
struct RowState {
    float m, l, o[4];
};

// keys [j0, j1) in steps of `step` of one segment (k, v: its first key for this head), in one wave
template <typename TQ, typename TK>
__device__ void row_keys(const AttnArgs &a, const float (&q)[4], const char *k, int64_t k_j, const char *v, int64_t v_j,
                         const _Float16 *mask, float slope, int j0, int j1, int step, RowState &r) {
    const int lane = threadIdx.x & 63;
    for (int j = j0; j < j1; j += step) {
        float add = 0.0f;
        if (mask) {
            add = (float)mask[j];
            if (add == -INFINITY) continue;
            add *= slope * LOG2E;
        }
        const TK *kr = reinterpret_cast<const TK *>(k + j * k_j), *vr = reinterpret_cast<const TK *>(v + j * v_j);
        float s = 0.0f;
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (lane + 64 * c < a.D) s = fmaf(q[c], (float)kr[lane + 64 * c], s);
        const float x = scaled(a, wave_add(s)) + add;
        const float m = fmaxf(r.m, x);
        // (-inf less -inf: a score of -inf has the weight 0 also where nothing greater was met yet; a
        // NaN score, which no maximum keeps, does reach the sum)
        const float p = x == -INFINITY ? 0.0f : exp2f(x - m), f = r.m == -INFINITY ? 1.0f : exp2f(r.m - m);
        r.m = m;
        r.l = r.l * f + p;
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (lane + 64 * c < a.D) r.o[c] = r.o[c] * f + p * (float)vr[lane + 64 * c];
    }
}

// one workgroup per (query, head, batch): its waves take every fourth key
template <typename TQ, typename TK>
__global__ __launch_bounds__(256) void attn_rows_kernel(const AttnArgs a) {
    __shared__ RowState part[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int i = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
    const int hk = h / (a.H / a.Hk), bk = b / a.kv_b;
    float q[4];
    const TQ *qr = reinterpret_cast<const TQ *>(a.q + i * a.q_i + h * a.q_h + b * a.q_b);
#pragma unroll
    for (int c = 0; c < 4; ++c) q[c] = lane + 64 * c < a.D ? (float)qr[lane + 64 * c] : 0.0f;
    RowState r{-INFINITY, 0.0f, {0.0f, 0.0f, 0.0f, 0.0f}};
    row_keys<TQ, TK>(a, q, a.kp + hk * a.kp_h, a.kp_j, a.vp + hk * a.vp_h, a.vp_j, nullptr, 0.0f, wave, a.n_prefix, 4, r);
    int end = own_len(a, b);
    if (a.causal) end = end - a.n_q + i + 1;
    const _Float16 *mask = nullptr;
    if (a.mask) mask = reinterpret_cast<const _Float16 *>(a.mask + i * a.m_i + (h % a.m_nh) * a.m_h + (b % a.m_nb) * a.m_b);
    row_keys<TQ, TK>(a, q, a.k + hk * a.k_h + bk * a.k_b, a.k_j, a.v + hk * a.v_h + bk * a.v_b, a.v_j, mask, slope_of(a, h), wave, end, 4, r);
    part[wave][lane] = r;
    __syncthreads();
    if (wave != 0) return;
    float m = a.sinks ? a.sinks[h] * LOG2E : -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) m = fmaxf(m, part[w][lane].m);
    float l = a.sinks && m != -INFINITY ? exp2f(a.sinks[h] * LOG2E - m) : 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const RowState &s = part[w][lane];
        const float f = m == -INFINITY ? 0.0f : exp2f(s.m - m);
        if (s.m == -INFINITY && s.l == 0.0f) continue;   // (a wave without keys)
        l += s.l * f;
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] += s.o[c] * f;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    TQ *out = reinterpret_cast<TQ *>(a.o + i * a.o_i + h * a.o_h + b * a.o_b);
#pragma unroll
    for (int c = 0; c < 4; ++c)
        if (lane + 64 * c < a.D) out[lane + 64 * c] = (TQ)(o[c] * inv);
}

int elem(int t) { return t == T_F32 ? 4 : 2; }

// data and the strides of the dims that have more than one index: multiples of `to`
bool aligned_to(const TensorView &t, size_t to) {
    if ((uintptr_t)t.data % to != 0) return false;
    for (int i = 1; i < 4; ++i)
        if (t.ne[i] > 1 && t.nb[i] % to != 0) return false;
    return true;
}

// 16-byte aligned rows of contiguous values (an empty tensor has no rows to look at)
bool rows_fit(const TensorView &t) {
    if (t.ne[0] == 0 || t.ne[1] == 0 || t.ne[2] == 0 || t.ne[3] == 0) return true;
    return (int64_t)t.nb[0] == elem(t.type) && aligned_to(t, 16);
}

bool dims_fit(const TensorView &t) {
    for (int i = 0; i < 4; ++i)
        if (t.ne[i] < 0 || t.ne[i] > (1 << 30)) return false;
    return true;
}

}  // namespace

// shapes, types and layouts of flash_attn (kp / vp: nullptr) and flash_attn_prefix
static int check_attn(const AttnTensors &t, const AttnSpec &p) {
    const TensorView &q = t.q, &k = t.k, &v = t.v, &d = t.dst;
    if (k.type != v.type || !(k.type == T_F16 || k.type == T_BF16)) return GGML_MI355X_EINVAL;
    if (q.type != d.type || !(q.type == k.type || (q.type == T_F32 && k.type == T_F16))) return GGML_MI355X_EINVAL;
    for (const TensorView *x : {&q, &k, &v, &d})
        if (!dims_fit(*x) || !rows_fit(*x)) return GGML_MI355X_EINVAL;
    const int64_t D = q.ne[0], n_q = q.ne[1], H = q.ne[2], B = q.ne[3];
    if (D < 8 || D > ATTN_MAX_D || D % 8 != 0 || k.ne[0] != D || v.ne[0] != D) return GGML_MI355X_EINVAL;
    for (int i = 1; i < 4; ++i)
        if (k.ne[i] != v.ne[i]) return GGML_MI355X_EINVAL;
    if (k.ne[2] <= 0 || H % k.ne[2] != 0 || k.ne[3] <= 0 || B % k.ne[3] != 0) return GGML_MI355X_EINVAL;
    if (H > 65535 || B > 65535 || n_q > (1 << 24)) return GGML_MI355X_EINVAL;
    if (d.ne[0] != D || d.ne[1] != H || d.ne[2] != n_q || d.ne[3] != B) return GGML_MI355X_EINVAL;
    for (int i = 1; i < 4; ++i)
        if (d.ne[i] > 1 && d.nb[i] == 0) return GGML_MI355X_EINVAL;   // two rows in one place
    if (t.kp) {
        const TensorView &kp = *t.kp, &vp = *t.vp;
        if (kp.type != k.type || vp.type != k.type || t.mask) return GGML_MI355X_EINVAL;
        for (const TensorView *x : {&kp, &vp})
            if (!dims_fit(*x) || !rows_fit(*x) || x->ne[0] != D || x->ne[2] != k.ne[2] || x->ne[3] != 1 || x->ne[1] != kp.ne[1])
                return GGML_MI355X_EINVAL;
        if (k.ne[3] != B) return GGML_MI355X_EINVAL;   // every sequence has its own cache
    }
    if (t.mask) {
        const TensorView &m = *t.mask;
        if (m.type != T_F16 || !dims_fit(m) || m.nb[0] != 2 || !aligned_to(m, 2) || m.ne[0] < k.ne[1] || m.ne[1] < n_q) return GGML_MI355X_EINVAL;
        if (m.ne[2] <= 0 || m.ne[3] <= 0 || H % m.ne[2] != 0 || B % m.ne[3] != 0) return GGML_MI355X_EINVAL;
    }
    if (t.sinks && (t.sinks->type != T_F32 || t.sinks->ne[0] < H || t.sinks->nb[0] != 4 || (uintptr_t)t.sinks->data % 4 != 0)) return GGML_MI355X_EINVAL;
    if (t.len) {
        const TensorView &l = *t.len;
        if (l.type != T_I32 || l.ne[0] != B || (B > 1 && l.nb[0] % 4 != 0) || (uintptr_t)l.data % 4 != 0) return GGML_MI355X_EINVAL;
    }
    if (!std::isfinite(p.scale) || !(p.max_bias >= 0.0f) || !std::isfinite(p.max_bias) || !(p.logit_softcap >= 0.0f) ||
        !std::isfinite(p.logit_softcap) || !(p.causal == 0 || p.causal == 1))
        return GGML_MI355X_EINVAL;
    if (p.max_bias > 0.0f && !t.mask) return GGML_MI355X_EINVAL;   // slopes multiply a mask
    return GGML_MI355X_OK;
}

int check_flash_attn(const AttnTensors &t, const AttnSpec &p) { return check_attn(t, p); }

size_t flash_attn_work(const AttnTensors &) { return 0; }

int flash_attn(const AttnTensors &t, const AttnSpec &p, hipStream_t st, Scratch &scratch) {
    const int rc = check_attn(t, p);
    if (rc != GGML_MI355X_OK) return rc;
    const size_t bytes = flash_attn_work(t);
    if (bytes == 0) return flash_attn(t, p, nullptr, st);
    std::lock_guard<std::mutex> hold(scratch.mu);   // until the kernels that use it are queued
    void *work = scratch.get(bytes, st);
    return work ? flash_attn(t, p, work, st) : GGML_MI355X_ENOMEM;
}

int flash_attn(const AttnTensors &t, const AttnSpec &p, void *work, hipStream_t st) {
    const int rc = check_attn(t, p);
    if (rc != GGML_MI355X_OK) return rc;
    const TensorView &q = t.q, &k = t.k, &v = t.v, &d = t.dst;
    if (q.ne[1] == 0 || q.ne[2] == 0 || q.ne[3] == 0) return GGML_MI355X_OK;
    if (!q.data || !d.data || (k.ne[1] > 0 && (!k.data || !v.data)) || (t.kp && t.kp->ne[1] > 0 && (!t.kp->data || !t.vp->data)) ||
        (t.mask && !t.mask->data) || (t.sinks && !t.sinks->data) || (t.len && !t.len->data))
        return GGML_MI355X_EINVAL;
    AttnArgs a{};
    a.q = static_cast<const char *>(q.data);
    a.q_i = (int64_t)q.nb[1]; a.q_h = (int64_t)q.nb[2]; a.q_b = (int64_t)q.nb[3];
    a.k = static_cast<const char *>(k.data);
    a.k_j = (int64_t)k.nb[1]; a.k_h = (int64_t)k.nb[2]; a.k_b = (int64_t)k.nb[3];
    a.v = static_cast<const char *>(v.data);
    a.v_j = (int64_t)v.nb[1]; a.v_h = (int64_t)v.nb[2]; a.v_b = (int64_t)v.nb[3];
    if (t.kp) {
        a.kp = static_cast<const char *>(t.kp->data);
        a.kp_j = (int64_t)t.kp->nb[1]; a.kp_h = (int64_t)t.kp->nb[2];
        a.vp = static_cast<const char *>(t.vp->data);
        a.vp_j = (int64_t)t.vp->nb[1]; a.vp_h = (int64_t)t.vp->nb[2];
        a.n_prefix = (int)t.kp->ne[1];
    }
    if (t.mask) {
        a.mask = static_cast<const char *>(t.mask->data);
        a.m_i = (int64_t)t.mask->nb[1]; a.m_h = (int64_t)t.mask->nb[2]; a.m_b = (int64_t)t.mask->nb[3];
        a.m_nh = (int)t.mask->ne[2]; a.m_nb = (int)t.mask->ne[3];
    }
    if (t.sinks) a.sinks = static_cast<const float *>(t.sinks->data);
    if (t.len) {
        a.len = static_cast<const char *>(t.len->data);
        a.len_b = (int64_t)t.len->nb[0];
    }
    a.o = static_cast<char *>(d.data);
    a.o_h = (int64_t)d.nb[1]; a.o_i = (int64_t)d.nb[2]; a.o_b = (int64_t)d.nb[3];
    a.D = (int)q.ne[0]; a.n_q = (int)q.ne[1]; a.n_kv = (int)k.ne[1];
    a.H = (int)q.ne[2]; a.Hk = (int)k.ne[2]; a.B = (int)q.ne[3]; a.kv_b = (int)(q.ne[3] / k.ne[3]);
    a.causal = p.causal;
    a.scale = p.scale;
    a.cap = p.logit_softcap;
    if (p.max_bias > 0.0f) {
        a.bias_heads = 1 << (int)std::floor(std::log2((double)a.H));
        a.m0 = std::pow(2.0f, -p.max_bias / a.bias_heads);
        a.m1 = std::pow(2.0f, -p.max_bias / 2.0f / a.bias_heads);
    }
    const dim3 grid(a.n_q, a.H, a.B);
    if (q.type == T_F32) hipLaunchKernelGGL((attn_rows_kernel<float, _Float16>), grid, dim3(256), 0, st, a);
    else if (q.type == T_F16) hipLaunchKernelGGL((attn_rows_kernel<_Float16, _Float16>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((attn_rows_kernel<__bf16, __bf16>), grid, dim3(256), 0, st, a);
    return hipGetLastError() == hipSuccess ? GGML_MI355X_OK : GGML_MI355X_EHIP;
}

}  // namespace mi355x
