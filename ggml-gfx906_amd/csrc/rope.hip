// rope.hip — rotary positions (GGML_OP_ROPE) and their gradient (GGML_OP_ROPE_BACK).
//
// Every pair (a, b) of a head's first n_dims values turns by t = pos * f_i:
//     a' = (a cos t - b sin t) * size,   b' = (a sin t + b cos t) * size
// with f_i = base^(-2i/n_dims), stretched for long contexts (below), divided by the pair's frequency
// factor. Pairs are neighbours (2i, 2i+1) or the two halves (i, i + n_dims/2); the values behind
// n_dims are copied. The gradient turns by -t: a turn's transpose is its inverse, and `size` stays.
//
// Angles are formed in 64 bits as turns: pos * f_i / 2pi less its nearest whole number, and only
// that remainder (|.| <= 1/2) is rounded to 32 bits: 2^-26 of a turn, beside the roundings of the
// 64-bit frequency and product (2^-53 each of the turns made, together 2^-23.6 of a turn at position
// 2^31; a third one where a factor divides). A 32-bit angle of 1e6 radians would be off by up to 0.03.
#include "../../include/ggml-mi355x.h"
#include "dispatch.h"
#include "qcommon.h"

#include <cmath>

namespace mi355x {

namespace {

struct RopeArgs {
    const char *src;
    char *dst;
    const int32_t *pos;
    const float *factors;             // per pair, or nullptr
    int64_t s_h, s_t, s_b;            // byte strides: head, token, batch
    int64_t d_h, d_t, d_b;
    int64_t pos_b;                    // elements from one batch's positions to the next (0: shared)
    int64_t rows;                     // ne1 * ne2 * ne3
    int ne0, ne1, ne2, n_dims;
    int halves;                       // pairs (i, i + n_dims/2), else (2i, 2i+1)
    float size;                       // factor of the turned values
    float way;                        // +1, or -1 for the gradient
    double turns[ROPE_MAX_DIMS / 2];  // f_i / 2pi
};

// cosine and sine of pair p at position `pos`, times the factor
__device__ __forceinline__ void turn(const RopeArgs &a, int p, double pos, float &cs, float &sn) {
    double t = pos * a.turns[p];
    if (a.factors) t /= (double)a.factors[p];
    t -= rint(t);
    sincospif(2.0f * (float)t, &sn, &cs);
    cs *= a.size;
    sn *= a.size * a.way;
}

// any layout: one thread per pair, then one per copied value
template <typename TS, typename TD>
__global__ __launch_bounds__(256) void rope_kernel(const RopeArgs a) {
    const int half = a.n_dims / 2, units = half + (a.ne0 - a.n_dims);
    const int64_t n = a.rows * units;
    for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < n; u += (int64_t)gridDim.x * 256) {
        const int64_t row = u / units;
        const int p = (int)(u % units);
        const int64_t h = row % a.ne1, t = row / a.ne1 % a.ne2, b = row / a.ne1 / a.ne2;
        const TS *s = reinterpret_cast<const TS *>(a.src + h * a.s_h + t * a.s_t + b * a.s_b);
        TD *d = reinterpret_cast<TD *>(a.dst + h * a.d_h + t * a.d_t + b * a.d_b);
        if (p >= half) {
            d[p + half] = (TD)(float)s[p + half];
            continue;
        }
        float cs, sn;
        turn(a, p, (double)a.pos[b * a.pos_b + t], cs, sn);
        const int ia = a.halves ? p : 2 * p, ib = a.halves ? p + half : 2 * p + 1;
        const float x = (float)s[ia], y = (float)s[ib];
        d[ia] = (TD)(x * cs - y * sn);
        d[ib] = (TD)(x * sn + y * cs);
    }
}

// Rows of whole groups of 2 W values at the places of W: a thread turns the same W pairs of HEADS heads of one
// token, so their sines are formed once, and all its loads are issued before them.
// Bound by memory: 4096 tokens x 32 heads x 128 f32 values, 134 MB in 24.4 us, 5.5 TB/s; 8192 x 8 x 128 f32
// into f16 12.4 us, 4.1 TB/s; a token's 32 heads 3.5 us, the launch.
template <typename T, int W> struct RopeVec { typedef T v __attribute__((ext_vector_type(W))); };

template <typename TS, typename TD, bool HALVES, int HEADS, int W>
__global__ __launch_bounds__(256) void rope_vec_kernel(const RopeArgs a) {
    typedef typename RopeVec<TS, W>::v SV;
    typedef typename RopeVec<TD, W>::v DV;
    const uint32_t units = (uint32_t)a.ne0 / (2 * W), at = blockIdx.x * 256 + threadIdx.x;
    const uint32_t t = at / units, u = at % units;
    if (t >= (uint32_t)a.ne2) return;
    const int h0 = blockIdx.y * HEADS, b = blockIdx.z;
    const bool turns = u < (uint32_t)a.n_dims / (2 * W);
    // the two groups of W values
    const int i0 = HALVES && turns ? W * u : 2 * W * u, i1 = HALVES && turns ? W * u + a.n_dims / 2 : 2 * W * u + W;
    const char *s = a.src + (int64_t)t * a.s_t + b * a.s_b;
    char *d = a.dst + (int64_t)t * a.d_t + b * a.d_b;
    SV x[HEADS], y[HEADS];
#pragma unroll
    for (int k = 0; k < HEADS; ++k) {
        const TS *r = reinterpret_cast<const TS *>(s + min(h0 + k, a.ne1 - 1) * a.s_h);
        x[k] = *reinterpret_cast<const SV *>(r + i0);
        y[k] = *reinterpret_cast<const SV *>(r + i1);
    }
    float cs[W] = {}, sn[W] = {};
    if (turns) {
        const double pos = (double)a.pos[b * a.pos_b + t];
#pragma unroll
        for (int e = 0; e < W; ++e) turn(a, W * u + e, pos, cs[e], sn[e]);
    }
#pragma unroll
    for (int k = 0; k < HEADS; ++k) {
        if (h0 + k >= a.ne1) break;
        TD *r = reinterpret_cast<TD *>(d + (h0 + k) * a.d_h);
        float v[2 * W];
        TD w[2 * W];
#pragma unroll
        for (int e = 0; e < W; ++e) {
            v[e] = (float)x[k][e];
            v[W + e] = (float)y[k][e];
        }
        DV lo, hi;
#pragma unroll
        for (int e = 0; e < W; ++e) {
            const int ia = HALVES ? e : 2 * e, ib = HALVES ? e + W : 2 * e + 1;
            w[ia] = (TD)(turns ? v[ia] * cs[e] - v[ib] * sn[e] : v[ia]);
            w[ib] = (TD)(turns ? v[ia] * sn[e] + v[ib] * cs[e] : v[ib]);
        }
#pragma unroll
        for (int e = 0; e < W; ++e) {
            lo[e] = w[e];
            hi[e] = w[W + e];
        }
        *reinterpret_cast<DV *>(r + i0) = lo;
        *reinterpret_cast<DV *>(r + i1) = hi;
    }
}

// f_i / 2pi for every pair, and the turned values' factor. Stretching (YaRN): a pair that turns
// more than beta_fast times over the trained context keeps its frequency, one that turns less than
// beta_slow times is scaled by freq_scale, with a ramp over the pairs between; ext_factor mixes the
// two rules. base^(-2i/n) comes as products of two tables (some 30 roundings) in the host's 80-bit
// format, so that the stored frequency is off by one 64-bit rounding.
void rope_turns(const RopeSpec &p, double *turns, float *size) {
    const int n = p.n_dims, half = n / 2;
    const long double log_base = std::log((long double)p.freq_base), step = std::exp(-2.0L * log_base / n);
    const long double pi = 3.14159265358979323846264338327950288L;
    long double small[16], big = 1.0L / (2.0L * pi);
    small[0] = 1.0L;
    for (int i = 1; i < 16; ++i) small[i] = small[i - 1] * step;
    long double low = 0, high = 0, sz = p.attn_factor;
    if (p.ext_factor != 0.0f) {
        auto turning = [&](long double beta) { return n * std::log(p.n_ctx_orig / (beta * 2.0L * pi)) / (2.0L * log_base); };
        low = std::max(0.0L, std::floor(turning(p.beta_fast)));
        high = std::min((long double)(n - 1), std::ceil(turning(p.beta_slow)));
        sz *= 1.0L + 0.1L * std::log(1.0L / p.freq_scale);
    }
    for (int i = 0; i < half; ++i) {
        if (i && i % 16 == 0) big *= small[15] * step;
        long double keep = 0.0L;
        if (p.ext_factor != 0.0f) {
            const long double ramp = std::min(1.0L, std::max(0.0L, (i - low) / std::max(0.001L, high - low)));
            keep = (1.0L - ramp) * p.ext_factor;
        }
        turns[i] = (double)(big * small[i % 16] * (p.freq_scale * (1.0L - keep) + keep));
    }
    *size = (float)sz;
}

bool rope_type(int t) { return t == T_F32 || t == T_F16 || t == T_BF16; }
int rope_bytes(int t) { return t == T_F32 ? 4 : 2; }

template <typename TS, typename TD>
void rope_launch(const RopeArgs &g, int64_t batches, hipStream_t st) {
    auto fits = [](const void *p, int64_t h, int64_t t, int64_t b, int to) { return (uintptr_t)p % to == 0 && h % to == 0 && t % to == 0 && b % to == 0; };
    auto groups = [&](int w) {
        return g.ne0 % (2 * w) == 0 && g.n_dims % (2 * w) == 0 && fits(g.src, g.s_h, g.s_t, g.s_b, w * (int)sizeof(TS)) &&
               fits(g.dst, g.d_h, g.d_t, g.d_b, w * (int)sizeof(TD)) && (int64_t)(g.ne0 / (2 * w)) * g.ne2 < (1LL << 31) && batches <= 65535 &&
               g.ne1 <= 65535;
    };
    const int w = groups(4) ? 4 : groups(2) ? 2 : groups(1) ? 1 : 0;
    const int64_t threads = w ? (int64_t)(g.ne0 / (2 * w)) * g.ne2 : 0;
    // One head a thread until that makes 4 waves for each SIMD of the 256 CUs; from there on the sines cost
    // more than further waves hide, and a thread takes 8 heads (4 where there are fewer): 4096 x 32 x 128 f32
    // 42.9 us with a pair a thread, 30.9 / 25.4 / 24.4 / 23.4 with 2 / 4 / 8 / 16 heads; 4 x 1000 x 20 x 80
    // bf16 12.9 with one, 9.8 / 8.6 / 8.0 / 9.9. Rows that only fall into groups of 4 or of 2 values, 4 heads a thread:
    // 3 x 3707 x 40 x 204 f16, 52 of them turned, 120 us (a pair a thread 354), 2000 x 32 x 102 f32 10.8 (18.0).
    const int heads = threads * g.ne1 * batches < 4LL * 4 * 256 * 64 || g.ne1 == 1 ? 1 : g.ne1 < 8 || w < 4 ? 4 : 8;
    if (w == 0 || (w < 4 && heads == 1)) {
        const int64_t n = g.rows * (g.n_dims / 2 + g.ne0 - g.n_dims);
        hipLaunchKernelGGL((rope_kernel<TS, TD>), dim3((unsigned)std::min<int64_t>((n + 255) / 256, 1 << 20)), dim3(256), 0, st, g);
        return;
    }
    const dim3 grid((unsigned)((threads + 255) / 256), (unsigned)((g.ne1 + heads - 1) / heads), (unsigned)batches);
#define ROPE_CASE(N, W)                                                                                              \
    if (heads == N && w == W) {                                                                                      \
        if (g.halves) hipLaunchKernelGGL((rope_vec_kernel<TS, TD, true, N, W>), grid, dim3(256), 0, st, g);           \
        else hipLaunchKernelGGL((rope_vec_kernel<TS, TD, false, N, W>), grid, dim3(256), 0, st, g);                   \
    }
    ROPE_CASE(1, 4)
    ROPE_CASE(4, 4)
    ROPE_CASE(8, 4)
    ROPE_CASE(4, 2)
    ROPE_CASE(4, 1)
#undef ROPE_CASE
}

template <typename TS>
void rope_pick(int td, const RopeArgs &g, int64_t batches, hipStream_t st) {
    if (td == T_F32) rope_launch<TS, float>(g, batches, st);
    else if (td == T_F16) rope_launch<TS, _Float16>(g, batches, st);
    else rope_launch<TS, __bf16>(g, batches, st);
}

}  // namespace

int check_rope(const TensorView &s, const TensorView &pos, const TensorView *ff, const TensorView &d, const RopeSpec &p) {
    if (!rope_type(s.type) || !rope_type(d.type) || pos.type != T_I32 || (ff && ff->type != T_F32)) return GGML_MI355X_EINVAL;
    for (int i = 0; i < 4; ++i)
        if (s.ne[i] != d.ne[i] || s.ne[i] < 0) return GGML_MI355X_EINVAL;
    if ((int64_t)s.nb[0] != rope_bytes(s.type) || (int64_t)d.nb[0] != rope_bytes(d.type)) return GGML_MI355X_EINVAL;
    // whole values: an odd byte offset would split one; and no two results in one place
    for (int i = 1; i < 4; ++i)
        if ((d.ne[i] > 1 && d.nb[i] == 0) || (s.ne[i] > 1 && s.nb[i] % rope_bytes(s.type) != 0) || (d.ne[i] > 1 && d.nb[i] % rope_bytes(d.type) != 0)) return GGML_MI355X_EINVAL;
    if ((uintptr_t)s.data % rope_bytes(s.type) != 0 || (uintptr_t)d.data % rope_bytes(d.type) != 0) return GGML_MI355X_EINVAL;
    if (p.mode != GGML_MI355X_ROPE_NEIGHBOURS && p.mode != GGML_MI355X_ROPE_HALVES) return GGML_MI355X_EINVAL;
    if (p.n_dims < 2 || p.n_dims % 2 != 0 || p.n_dims > ROPE_MAX_DIMS || p.n_dims > s.ne[0]) return GGML_MI355X_EINVAL;
    if (s.ne[0] > (1 << 24) || s.ne[1] > (1 << 30) || s.ne[2] > (1 << 30) || s.ne[3] > (1 << 30)) return GGML_MI355X_EINVAL;
    if (s.ne[1] > 0 && s.ne[2] > 0 && s.ne[3] > 0 && (double)s.ne[1] * s.ne[2] * s.ne[3] * s.ne[0] > (double)(1LL << 46)) return GGML_MI355X_EINVAL;
    // one position per token, the same for every batch or a row of them for each
    if (pos.ne[0] != s.ne[2] || !(pos.ne[1] == 1 || pos.ne[1] == s.ne[3]) || pos.ne[2] != 1 || pos.ne[3] != 1) return GGML_MI355X_EINVAL;
    if (pos.nb[0] != 4 || (pos.ne[1] > 1 && pos.nb[1] % 4 != 0) || (uintptr_t)pos.data % 4 != 0) return GGML_MI355X_EINVAL;
    if (ff && (ff->ne[0] < p.n_dims / 2 || ff->nb[0] != 4 || (uintptr_t)ff->data % 4 != 0)) return GGML_MI355X_EINVAL;
    if (!(p.freq_base > 0.0f) || !std::isfinite(p.freq_base) || !std::isfinite(p.freq_scale) || !std::isfinite(p.ext_factor) ||
        !std::isfinite(p.attn_factor))
        return GGML_MI355X_EINVAL;
    if (p.ext_factor != 0.0f && !(p.n_ctx_orig > 0 && p.freq_base > 1.0f && p.freq_scale > 0.0f && p.beta_fast > 0.0f && p.beta_slow > 0.0f &&
                                  std::isfinite(p.beta_fast) && std::isfinite(p.beta_slow)))
        return GGML_MI355X_EINVAL;
    return GGML_MI355X_OK;
}

int rope(const TensorView &s, const TensorView &pos, const TensorView *ff, const TensorView &d, const RopeSpec &p, bool back,
         hipStream_t st) {
    const int rc = check_rope(s, pos, ff, d, p);
    if (rc != GGML_MI355X_OK) return rc;
    RopeArgs g;
    g.rows = s.ne[1] * s.ne[2] * s.ne[3];
    if (g.rows == 0) return GGML_MI355X_OK;
    if (!s.data || !d.data || !pos.data || (ff && !ff->data)) return GGML_MI355X_EINVAL;
    g.src = static_cast<const char *>(s.data);
    g.dst = static_cast<char *>(d.data);
    g.pos = static_cast<const int32_t *>(pos.data);
    g.factors = ff ? static_cast<const float *>(ff->data) : nullptr;
    g.s_h = (int64_t)s.nb[1]; g.s_t = (int64_t)s.nb[2]; g.s_b = (int64_t)s.nb[3];
    g.d_h = (int64_t)d.nb[1]; g.d_t = (int64_t)d.nb[2]; g.d_b = (int64_t)d.nb[3];
    // (a dim of one index has any stride: none, so that it is aligned)
    if (s.ne[1] == 1) g.s_h = g.d_h = 0;
    if (s.ne[2] == 1) g.s_t = g.d_t = 0;
    if (s.ne[3] == 1) g.s_b = g.d_b = 0;
    g.pos_b = pos.ne[1] > 1 ? (int64_t)pos.nb[1] / 4 : 0;
    g.ne0 = (int)s.ne[0]; g.ne1 = (int)s.ne[1]; g.ne2 = (int)s.ne[2];
    g.n_dims = p.n_dims;
    g.halves = p.mode == GGML_MI355X_ROPE_HALVES;
    g.way = back ? -1.0f : 1.0f;
    rope_turns(p, g.turns, &g.size);
    if (s.type == T_F32) rope_pick<float>(d.type, g, s.ne[3], st);
    else if (s.type == T_F16) rope_pick<_Float16>(d.type, g, s.ne[3], st);
    else rope_pick<__bf16>(d.type, g, s.ne[3], st);
    return hipGetLastError() == hipSuccess ? GGML_MI355X_OK : GGML_MI355X_EHIP;
}

}  // namespace mi355x
