// attention.cpp — checks, plan and launch of attention over a key / value cache and behind a shared prefix
// (kernels: attention_impl.h)
#include "../../include/ggml-mi355x.h"
#include "attention.h"
#include "dispatch.h"
#include "qcommon.h"

#include <algorithm>
#include <cmath>

namespace mi355x {

namespace {

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
    // (no heads or no batches have a cache of none)
    auto shared = [](int64_t n, int64_t by) { return by > 0 ? n % by == 0 : n == 0 && by == 0; };
    if (!shared(H, k.ne[2]) || !shared(B, k.ne[3])) return GGML_MI355X_EINVAL;
    // (a grid has less than 2^32 threads: 256 for every row's join or problem, 512 for 256 rows of a prompt)
    if (H > 65535 || B > 65535 || n_q >= (1 << 24) || H * B > (1 << 22) || H * B * n_q > (t.kp ? 1 << 25 : 1 << 28)) return GGML_MI355X_EINVAL;
    if (d.ne[0] != D || d.ne[1] != H || d.ne[2] != n_q || d.ne[3] != B) return GGML_MI355X_EINVAL;
    for (int i = 1; i < 4; ++i)
        if (d.ne[i] > 1 && d.nb[i] == 0 && H * B * n_q > 0) return GGML_MI355X_EINVAL;   // two rows in one place
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
        if (!shared(H, m.ne[2]) || !shared(B, m.ne[3])) return GGML_MI355X_EINVAL;
    }
    if (t.sinks && (t.sinks->type != T_F32 || t.sinks->ne[0] < H || t.sinks->nb[0] != 4 || (uintptr_t)t.sinks->data % 4 != 0)) return GGML_MI355X_EINVAL;
    if (t.len) {
        const TensorView &l = *t.len;
        if (l.type != T_I32 || l.ne[0] != B || (B > 1 && l.nb[0] % 4 != 0) || (uintptr_t)l.data % 4 != 0) return GGML_MI355X_EINVAL;
    }
    if (!std::isfinite(p.scale) || !(p.max_bias >= 0.0f) || !std::isfinite(p.max_bias) || !(p.logit_softcap >= 0.0f) ||
        !(p.logit_softcap <= 0x1p64f) ||   // (its product with log2(e), and the scale over it, stay normal numbers)
        !(p.causal == 0 || p.causal == 1))
        return GGML_MI355X_EINVAL;
    if (p.max_bias > 0.0f && !t.mask) return GGML_MI355X_EINVAL;   // slopes multiply a mask
    return GGML_MI355X_OK;
}

int check_flash_attn(const AttnTensors &t, const AttnSpec &p) { return check_attn(t, p); }

static AttnPlan plan_attn(const AttnTensors &t) {
    AttnPlan p{};
    const int64_t n_q = t.q.ne[1], H = t.q.ne[2], B = t.q.ne[3], Hk = t.k.ne[2], G = H / Hk;
    // the tile kernel's offsets inside a tile are 32-bit: positions up to 16 MiB apart
    p.tiled = true;
    for (const TensorView *x : {&t.k, &t.v, t.kp, t.vp})
        if (x && x->nb[1] >= (1u << 24)) p.tiled = false;
    if (!p.tiled) return p;
    // Splits of the keys, and workgroups of 4 or of 8 waves: the fewest us by a model of the launch.
    //   a workgroup of row tiles with heads of 128 values: 4 waves, 128 rows 7 us, and per tile of 64 keys 1.4 alone
    //     on its CU, 2.0 beside another one, 2.3 beside split keys; 8 waves, 256 rows 9 and 1.92; 8 waves, 128 rows,
    //     two tiles at a time 8 and 1.85 for both, 2.05 where there are more workgroups than CUs. Of a tile's time
    //     0.55 (8 waves: 0.65) up to 64 values, 0.83 up to 96; 1.8 for f32 activations. The rows of a causal call (the
    //     rule is not known here: taken for one) see fewer keys, the last tiles the most
    //   a workgroup of split keys: 5 us, and per 128 keys what one CU draws from HBM, 1.6 (1.1 up to 64 values); all
    //     of them no less than their bytes at 5.5 TB/s, which fewer than 256 workgroups do not reach
    //   a prefix's workgroups are dealt first, then the batches' own, 512 (256 wide ones) at a time
    //   more than one partial result a row: 5 for the second launch, and their trip through memory
    // Measured / by the model, us: one token, 8 key heads of 128 values, 8192 keys, 1 / 4 / 16 / 32 / 64 splits 85.7,
    // 30.9, 17.2, 16.9, 19.2 / 107, 35, 17, 18, 21; 131072 keys, 16 / 24 / 32 / 64 splits 122, 116, 105, 106 / 131, 119,
    // 110, 116; 64 sequences behind 8192 shared keys, 6 / 8 / 16 splits of them 54, 46, 53 / 65, 52, 58; 16 x 4 draft
    // tokens behind 32768, 24 / 28 / 32 splits 62, 58, 68 / 72, 72, 79. Row tiles, 4 waves / 8 / two tiles at a time: 32
    // causal heads of 8192 tokens 547, 533, 588 / 526, 510, 557; of 2048 60, 61, 50 / 71, 70, 41; 16 of 512 behind 512
    // 27.9, 33.2, 22.8 / 29, 40, 23, the latter's 2 and 4 splits 23.9, 24.9 / 24, 23.
    const int64_t D = t.q.ne[0], rows = n_q * G;
    const double size = t.q.type == T_F32 ? 1.8 : 1.0, size4 = size * (D <= 64 ? 0.55 : D <= 96 ? 0.83 : D <= 128 || D > 192 ? 1.0 : 0.75),
                 size8 = size * (D <= 64 ? 0.65 : D <= 96 ? 0.83 : 1.0);
    // workgroups, us of each alone on its CU and not, bytes of split keys
    struct Part { double groups, alone, beside, bytes; int tiles; };
    auto part = [&](int64_t rows, int64_t problems, int64_t keys, bool by_rows, int waves, int turns, int s) {
        const int64_t per_tile = by_rows ? waves / turns * 32 : 32, step = by_rows ? (D <= 128 ? 64 * turns : 32) : 128;
        const int tiles = (int)((rows + per_tile - 1) / per_tile);
        const double groups = (double)problems * tiles * s, n = std::ceil(std::ceil((double)keys / s) / step);
        if (!by_rows) return Part{groups, 5.0 + n * (D <= 64 ? 1.1 : 1.6), 0.0, (double)problems * keys * D * 4, tiles};
        if (turns == 2) return Part{groups, 8.0 + n * 1.85 * size8, 8.0 + n * 2.05 * size8, 0.0, tiles};
        if (waves == 8) return Part{groups, 9.0 + n * 1.92 * size8, 9.0 + n * 1.92 * size8, 0.0, tiles};
        return Part{groups, 7.0 + n * 1.4 * size4, 7.0 + n * (t.kp ? 2.3 : 2.0) * size4, 0.0, tiles};
    };
    const double fewer = t.k.ne[1] > 0 ? std::min(1.0, (double)n_q / (double)t.k.ne[1]) : 0.0;   // of the first rows, causal
    auto launch = [&](const Part &pre, const Part &own, int waves) {
        // (over 128 values: split keys' LDS, over 192 and f32 ones the accumulators leave room for one)
        const bool one = waves == 8 || D > 192 || (D > 128 && (!p.own_rows || t.q.type == T_F32));
        const double at_once = one ? 256.0 : 512.0, all = pre.groups + own.groups;
        auto us = [&](const Part &x) { return x.bytes == 0.0 && all > 256.0 ? x.beside : x.alone; };
        const double own_us = us(own), pre_us = us(pre);
        // what split keys draw from memory, beside the time that row tiles hold the CUs
        const double bytes = pre.bytes + own.bytes, rate = 5.5e6 * std::min(1.0, 0.6 + 0.4 * all / 256.0);
        const double memory = bytes == 0.0 ? 0.0
                                           : 5.0 + bytes / rate + 3.0 * ((pre.bytes > 0.0 ? pre.groups : 0.0) + (own.bytes > 0.0 ? own.groups : 0.0)) / 512.0 +
                                                 (pre.groups > 0.0 && pre.bytes == 0.0 ? pre.groups * pre_us / at_once : 0.0);
        if (pre.groups == 0.0) {
            const double rounds = own.groups / at_once;
            if (own.bytes != 0.0) return std::max(memory, own_us);
            return std::max(own_us, own_us * ((1.0 - fewer / 2) * rounds + (1.0 - fewer) * (std::ceil(rounds) - rounds)));
        }
        // the prefix's whole rounds, the rest of it with own ones beside it, then the others wherever one ends first
        const double before = std::floor(pre.groups / at_once) * pre_us, left = std::fmod(pre.groups, at_once), beside = at_once - left;
        const double end = before + (left > 0.0 ? pre_us : 0.0), rest = own.groups - beside;
        if (rest <= 0.0) return std::max({memory, end, before + own_us});
        return std::max({memory, end, std::min(before + own_us * (1.0 + std::ceil(rest / beside)), end + own_us * std::ceil(rest / at_once))});
    };
    auto join = [&](int slots) { return slots > 1 ? 5.0 + (double)B * H * n_q * slots * D * 8 / 5e6 : 0.0; };
    static const int SPLITS[] = {1, 2, 3, 4, 6, 8, 12, 16, 20, 24, 28, 32, 48, 64, 96, 128};
    static const int PREFIX_SPLITS[] = {1, 2, 3, 4, 6, 8, 10, 12, 14, 16, 18, 20, 22, 24, 26, 28, 30, 32, 48, 64, 96, 128};
    static_assert(128 <= ATTN_MAX_SLOTS / 2, "a prefix's splits and the batches' own");
    p.own_rows = rows > 32;
    p.pre_rows = t.kp && B * rows > 32;
    const int64_t n_kv = t.k.ne[1], n_pre = t.kp ? t.kp->ne[1] : 0;
    double best = 0.0;
    // (row tiles may gain by the wide workgroups; split keys do not, and beside them two smaller ones do better)
    struct Kind { int waves, turns; };
    static const Kind KINDS[] = {{4, 1}, {8, 1}, {8, 2}};
    for (const Kind &w : KINDS) {
        const bool wide = w.waves == 8;
        if (wide && (!p.own_rows || D > 128)) continue;
        if (t.kp && (w.turns > 1 || (p.own_rows && D <= 128 && !wide))) continue;
        auto consider = [&](int so, int sp) {
            if ((so > 1 && (so - 1) * 32 >= n_kv) || (sp > 1 && (sp - 1) * 32 >= n_pre)) return false;
            const Part own = part(rows, B * Hk, n_kv, p.own_rows, w.waves, w.turns, so);
            const Part pre = t.kp ? part(B * rows, Hk, n_pre, p.pre_rows, w.waves, 1, sp) : Part{};
            const double us = launch(pre, own, w.waves) + join(so + sp);
            if (p.slots != 0 && us >= best) return true;
            best = us;
            p.waves = w.waves;
            p.turns = w.turns;
            p.own_splits = so;
            p.own_tiles = own.tiles;
            p.pre_splits = sp;
            p.pre_tiles = pre.tiles;
            p.slots = so + sp;
            return true;
        };
        if (!t.kp) {
            for (int so : SPLITS)
                if (!consider(so, 0)) break;
            continue;
        }
        // the prefix's splits, then the own keys', and the prefix's again beside those
        for (int sp : PREFIX_SPLITS)
            if (!consider(1, sp)) break;
        const int sp = p.pre_splits;
        for (int so : SPLITS)
            if (so > 1 && !consider(so, sp)) break;
        if (p.own_splits == 1) continue;
        const int so = p.own_splits;
        for (int again : PREFIX_SPLITS)
            if (!consider(so, again)) break;
    }
    return p;
}

size_t flash_attn_work(const AttnTensors &t) {
    if (t.q.ne[1] == 0 || t.q.ne[2] == 0 || t.q.ne[3] == 0) return 0;
    const AttnPlan p = plan_attn(t);
    return p.slots > 1 ? (size_t)t.q.ne[1] * t.q.ne[2] * t.q.ne[3] * p.slots * (t.q.ne[0] + 2) * sizeof(float) : 0;
}

static bool has_data(const AttnTensors &t) {
    return t.q.data && t.dst.data && (t.k.ne[1] == 0 || (t.k.data && t.v.data)) && (!t.kp || t.kp->ne[1] == 0 || (t.kp->data && t.vp->data)) &&
           (!t.mask || t.mask->data) && (!t.sinks || t.sinks->data) && (!t.len || t.len->data);
}

int flash_attn(const AttnTensors &t, const AttnSpec &p, hipStream_t st, Scratch &scratch) {
    const int rc = check_attn(t, p);
    if (rc != GGML_MI355X_OK) return rc;
    const size_t bytes = flash_attn_work(t);
    if (bytes == 0 || !has_data(t)) return flash_attn(t, p, nullptr, st);
    std::lock_guard<std::mutex> hold(scratch.mu);   // until the kernels that use it are queued
    void *work = scratch.get(bytes, st);
    return work ? flash_attn(t, p, work, st) : GGML_MI355X_ENOMEM;
}

int flash_attn(const AttnTensors &t, const AttnSpec &p, void *work, hipStream_t st) {
    const int rc = check_attn(t, p);
    if (rc != GGML_MI355X_OK) return rc;
    const TensorView &q = t.q, &k = t.k, &v = t.v, &d = t.dst;
    if (q.ne[1] == 0 || q.ne[2] == 0 || q.ne[3] == 0) return GGML_MI355X_OK;
    if (!has_data(t)) return GGML_MI355X_EINVAL;
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
    a.H = (int)q.ne[2]; a.Hk = (int)k.ne[2]; a.B = (int)q.ne[3];
    a.by_G = Div((uint32_t)(a.H / a.Hk)); a.by_Hk = Div((uint32_t)a.Hk); a.by_n_q = Div((uint32_t)a.n_q);
    a.by_kv_b = Div((uint32_t)(q.ne[3] / k.ne[3]));
    a.causal = p.causal;
    a.scale = p.scale;
    a.cap = p.logit_softcap;
    if (p.max_bias > 0.0f) {
        a.bias_heads = 1 << (int)std::floor(std::log2((double)a.H));
        a.m0 = std::pow(2.0f, -p.max_bias / a.bias_heads);
        a.m1 = std::pow(2.0f, -p.max_bias / 2.0f / a.bias_heads);
    }
    const AttnPlan pl = plan_attn(t);
    typedef hipError_t (*Launch)(const AttnArgs &, const AttnPlan &, void *, hipStream_t);
    static const Launch launch[3][5] = {{attn_launch_f16_64, attn_launch_f16_96, attn_launch_f16_128, attn_launch_f16_192, attn_launch_f16_256},
                                        {attn_launch_bf16_64, attn_launch_bf16_96, attn_launch_bf16_128, attn_launch_bf16_192, attn_launch_bf16_256},
                                        {attn_launch_f32_64, attn_launch_f32_96, attn_launch_f32_128, attn_launch_f32_192, attn_launch_f32_256}};
    const int type = q.type == T_F32 ? 2 : q.type == T_BF16 ? 1 : 0;
    const hipError_t e = launch[type][a.D <= 64 ? 0 : a.D <= 96 ? 1 : a.D <= 128 ? 2 : a.D <= 192 ? 3 : 4](a, pl, work, st);
    return e == hipSuccess ? GGML_MI355X_OK : GGML_MI355X_EHIP;
}

}  // namespace mi355x
