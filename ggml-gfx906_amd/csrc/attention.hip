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

// one workgroup per (query, head, batch): its waves take every fourth key. For layouts whose positions
// lie too far apart for the tile kernel's 32-bit offsets
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
        const float f = m == -INFINITY ? 1.0f : exp2f(s.m - m);
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

// ------------------------------------------------------------------------------------------
// the tile kernel
//
// A row is one (query, head of a group) pair: the G = H / Hk heads that share a key / value head are
// rows of one problem, r = i * G + g, so its keys and values are read once for all of them (for a
// shared prefix the sequences are too: r = (b * n_q + i) * G + g). A wave holds 32 rows and takes
// tiles of keys:
//     S^T = K Q^T   (MFMA 32x32x16: A = keys from LDS, B = the rows' queries in registers)
//     p   = exp2(S^T c - m)
//     O^T += V^T P^T (A = values from LDS by the transposing read, B = p)
// With both products transposed a lane's 16 results of S^T belong to one row (lane & 31), so the
// running maximum and sum are the lane's own scalars, and they are the very values that O^T's B operand
// wants from that lane once the keys are taken in the order the MFMA returned them: the weights never
// leave the registers. Tiles come by LDS DMA, one tile ahead.
//   BY_ROWS: 4 waves of 32 rows each share tiles of KT keys (prompts, shared prefixes)
//   else:    4 waves share 32 rows and take tiles of 32 keys in turn, joined at the end (tokens)
// 16-byte pieces of a tile's rows are permuted (swz_k, swz_v) so that neither read meets an LDS bank
// twice; the DMA writes LDS in order, so the permutation is in the addresses it reads from.
//
// m moves only when a tile exceeds it by more than 2^LAZY, so the 16 DP/32 accumulators are rarely
// rescaled; weights are kept 2^BIAS times larger, up to 2^(BIAS + LAZY) = 2^15, which f16 still holds, so
// that small ones stay clear of f16's subnormals.
// F32 queries: q (scaled by a power of two per row) and p are each carried as a sum of two f16 values
// (2^-22), two MFMAs per product.
// ------------------------------------------------------------------------------------------
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef const __attribute__((address_space(3))) char *lds_const;

constexpr float BIAS = 8.0f, LAZY = 7.0f;
constexpr int MAX_SLOTS = 256;   // partial results of a row

template <typename T> struct Vec;
template <> struct Vec<_Float16> { typedef f16x8 x8; };
template <> struct Vec<__bf16> { typedef bf16x8 x8; };

__device__ __forceinline__ f32x16 mma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

// the permuted place of 16-byte piece c of row r of a tile with DP values a row
template <int DP> __device__ __forceinline__ int swz_k(int r) { return DP == 64 ? (r >> 1) & 7 : r & 15; }
template <int DP> __device__ __forceinline__ int swz_v(int r) { return DP == 64 ? ((r >> 1) & 1) << 2 : (r & 3) << 2; }

// which keys and rows a launch works on
struct AttnPart {
    float *part_o, *part_ml;   // partial results, or nullptr: the call's result
    int slot0, n_split;        // this launch's splits among
    int slots;                 // all partial results of a row
    int n_bh;                  // (batch,) key / value head problems
    int rows, row_tiles;       // of each
};

// 16 bytes per lane from base + voff + soff into LDS at dst + 16 * lane (dst, soff wave-uniform). Written out
// because the compiler, which can not tell the stages apart, makes every LDS read wait for each DMA that it
// knows of; the kernel waits itself. No result registers; the address registers are read at issue. The
// nops are the wait states from a scalar's write by a vector instruction and from m0's to their use.
typedef int i32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ i32x4 buffer_at(const char *p) {   // a raw buffer of 2 GiB
    const uint64_t at = (uint64_t)(uintptr_t)p;
    return i32x4{(int)__builtin_amdgcn_readfirstlane((uint32_t)at), (int)__builtin_amdgcn_readfirstlane((uint32_t)(at >> 32) & 0xffff), 0x7fffffff, 0x00020000};
}
__device__ __forceinline__ void dma16(i32x4 r, const char *dst, uint32_t voff, uint32_t soff) {
    const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_const)dst);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 :: "s"(at), "v"(voff), "s"(r), "s"(soff) : "memory");
}

template <typename TK, typename TQ, int DP, bool BY_ROWS, bool PREFIX>
struct AttnTile {
    static constexpr bool SPLIT = sizeof(TQ) == 4;
    static constexpr int KT = BY_ROWS && DP <= 128 ? 64 : 32;   // keys of a tile
    static constexpr int CPR = DP / 8;                          // 16-byte pieces of a row
    static constexpr int WAVES = !BY_ROWS && DP == 256 ? 2 : 4; // (two stages of every wave's tiles fit the 160 KB)
    static constexpr int LOADERS = BY_ROWS ? 256 : 64;          // threads that load a tile together
    static constexpr int RPI = LOADERS / CPR;                   // rows of one DMA round
    static constexpr int ROUNDS = KT / RPI;
    static constexpr int BYTES = KT * DP * 2;                   // of a tile of keys, and of values
    static constexpr int LDS = (BY_ROWS ? 1 : WAVES) * 4 * BYTES;   // keys and values, two stages
    typedef typename Vec<TK>::x8 x8;
};

// a finished row's place: the call's result, or this launch's partial result (sum, maximum, weighted values)
struct RowOut {
    int b, i, head;
    int64_t slot;   // of the partial results
};
template <bool PREFIX>
__device__ __forceinline__ RowOut row_out(const AttnArgs &a, const AttnPart &p, int row, int bh, int split) {
    const int G = a.H / a.Hk, hk = bh % a.Hk, g = row % G, bi = row / G;
    RowOut r;
    r.i = PREFIX ? bi % a.n_q : bi;
    r.b = PREFIX ? bi / a.n_q : bh / a.Hk;
    r.head = hk * G + g;
    r.slot = (((int64_t)r.b * a.Hk + hk) * a.n_q * G + r.i * G + g) * p.slots + p.slot0 + split;
    return r;
}

// the sink joins a row's sum: the factor of its weighted values, 0 for a row without weight
__device__ __forceinline__ float finish(const AttnArgs &a, int head, float m, float l) {
    float f = 1.0f;
    if (a.sinks) {
        const float s = a.sinks[head] * LOG2E, top = fmaxf(m, s);
        if (top != -INFINITY) {
            f = exp2f(m - top);
            l = l * f + exp2f(s - top);
        }
    }
    return l == 0.0f ? 0.0f : f / l;
}

// A weight of 0 times a NaN or an infinity in a key that a row does not see, but another row of its tile
// or the DMA's filling does, makes the row's sums NaN. Such a row is done again by its wave, key by key,
// without the keys that it does not see; a NaN that it does see comes out again.
template <typename TK, typename TQ, bool PREFIX>
__device__ void redo_row(const AttnArgs &a, const AttnPart &p, int row, int bh, int split, int j_begin, int j_end) {
    const int lane = threadIdx.x & 63;
    const RowOut w = row_out<PREFIX>(a, p, row, bh, split);
    const int hk = bh % a.Hk, bk = PREFIX ? 0 : (bh / a.Hk) / a.kv_b;
    float q[4];
    const TQ *qr = reinterpret_cast<const TQ *>(a.q + w.i * a.q_i + w.head * a.q_h + w.b * a.q_b);
#pragma unroll
    for (int c = 0; c < 4; ++c) q[c] = lane + 64 * c < a.D ? (float)qr[lane + 64 * c] : 0.0f;
    RowState r{-INFINITY, 0.0f, {0.0f, 0.0f, 0.0f, 0.0f}};
    if constexpr (PREFIX) {
        row_keys<TQ, TK>(a, q, a.kp + hk * a.kp_h, a.kp_j, a.vp + hk * a.vp_h, a.vp_j, nullptr, 0.0f, j_begin, j_end, 1, r);
    } else {
        const int seen = a.causal ? own_len(a, w.b) - a.n_q + w.i + 1 : j_end;
        const _Float16 *mask = nullptr;
        if (a.mask) mask = reinterpret_cast<const _Float16 *>(a.mask + w.i * a.m_i + (w.head % a.m_nh) * a.m_h + (w.b % a.m_nb) * a.m_b);
        row_keys<TQ, TK>(a, q, a.k + hk * a.k_h + bk * a.k_b, a.k_j, a.v + hk * a.v_h + bk * a.v_b, a.v_j, mask, slope_of(a, w.head), j_begin,
                         min(j_end, seen), 1, r);
    }
    if (p.part_o) {
        if (lane == 0) {
            p.part_ml[2 * w.slot] = r.m;
            p.part_ml[2 * w.slot + 1] = r.l;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (lane + 64 * c < a.D) p.part_o[w.slot * a.D + lane + 64 * c] = r.o[c];
    } else {
        const float f = finish(a, w.head, r.m, r.l);
        TQ *out = reinterpret_cast<TQ *>(a.o + w.i * a.o_i + w.head * a.o_h + w.b * a.o_b);
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (lane + 64 * c < a.D) out[lane + 64 * c] = (TQ)(r.o[c] * f);
    }
}

template <typename TQ> __device__ __forceinline__ void store4(TQ *p, f32x4 x);
template <> __device__ __forceinline__ void store4(float *p, f32x4 x) { *reinterpret_cast<f32x4 *>(p) = x; }
template <> __device__ __forceinline__ void store4(_Float16 *p, f32x4 x) {
    *reinterpret_cast<f16x4 *>(p) = f16x4{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
}
template <> __device__ __forceinline__ void store4(__bf16 *p, f32x4 x) {
    *reinterpret_cast<bf16x4 *>(p) = bf16x4{(__bf16)x[0], (__bf16)x[1], (__bf16)x[2], (__bf16)x[3]};
}

// a wave's 32 rows out of the accumulators: lane (row, h) holds values 32 d + 8 r4 + 4 h .. + 3
template <typename TK, typename TQ, int DP, bool PREFIX>
__device__ __forceinline__ void store_rows(const AttnArgs &a, const AttnPart &p, const f32x16 (&o)[DP / 32], float m, float l, int row,
                                           bool row_ok, int bh, int split, int j_begin, int j_end) {
    const int lane = threadIdx.x & 63, h = lane >> 5;
    bool bad = l != l;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) bad |= o[d][r] != o[d][r];
    const uint64_t votes = __ballot(bad && row_ok);
    uint32_t again = (uint32_t)votes | (uint32_t)(votes >> 32);
    if (row_ok && !(again >> (lane & 31) & 1)) {
        const RowOut w = row_out<PREFIX>(a, p, row, bh, split);
        if (p.part_o && h == 0) {
            p.part_ml[2 * w.slot] = m;
            p.part_ml[2 * w.slot + 1] = l;
        }
        const float f = p.part_o ? 1.0f : finish(a, w.head, m, l);
        float *po = p.part_o + w.slot * a.D;
        TQ *out = reinterpret_cast<TQ *>(a.o + w.i * a.o_i + w.head * a.o_h + w.b * a.o_b);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                const int at = 32 * d + 8 * r4 + 4 * h;
                if (at >= a.D) continue;
                const f32x4 x = f32x4{o[d][4 * r4], o[d][4 * r4 + 1], o[d][4 * r4 + 2], o[d][4 * r4 + 3]} * f;
                if (p.part_o) *reinterpret_cast<f32x4 *>(po + at) = x;
                else store4<TQ>(out + at, x);
            }
    }
    while (again) {
        const int at = __builtin_ctz(again);
        again &= again - 1;
        redo_row<TK, TQ, PREFIX>(a, p, __builtin_amdgcn_readlane(row, at), bh, split, j_begin, j_end);
    }
}

// 32 rows that `waves` waves hold parts of, each in its stretch of LDS (values [row][DP], then the
// maxima and the sums): THREADS / 32 threads a row
template <typename TK, typename TQ, int DP, int WAVES, bool PREFIX>
__device__ __forceinline__ void join_waves(const AttnArgs &a, const AttnPart &p, const char *lds, int stretch, int tops, int row0, int bh,
                                           int split, int j_begin, int j_end) {
    constexpr int TPR = WAVES * 2, N = DP / TPR;
    const int r = threadIdx.x / TPR, d0 = threadIdx.x % TPR * N, row = row0 + r;
    const bool ok = row < p.rows;
    float m = -INFINITY, l = 0.0f, f[WAVES];
    f32x4 x[N / 4];
#pragma unroll
    for (int w = 0; w < WAVES; ++w) m = fmaxf(m, reinterpret_cast<const float *>(lds + w * stretch + tops)[r]);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        const float *ml = reinterpret_cast<const float *>(lds + w * stretch + tops);
        f[w] = m == -INFINITY ? 1.0f : exp2f(ml[r] - m);
        l += ml[32 + r] * f[w];
    }
#pragma unroll
    for (int e = 0; e < N / 4; ++e) {
        x[e] = f32x4{};
#pragma unroll
        for (int w = 0; w < WAVES; ++w) x[e] += *reinterpret_cast<const f32x4 *>(lds + w * stretch + (r * DP + d0 + 4 * e) * 4) * f[w];
    }
    bool bad = l != l;
#pragma unroll
    for (int e = 0; e < N / 4; ++e)
#pragma unroll
        for (int c = 0; c < 4; ++c) bad |= x[e][c] != x[e][c];
    // a row's threads are neighbours in one wave: any of their votes counts
    uint64_t again = __ballot(bad && ok);
#pragma unroll
    for (int sft = 1; sft < TPR; sft <<= 1) again |= again >> sft;
    uint64_t firsts = 0;
#pragma unroll
    for (int t = 0; t < 64; t += TPR) firsts |= 1ull << t;
    again &= firsts;
    const int lane = threadIdx.x & 63;
    if (ok && !(again >> (lane / TPR * TPR) & 1)) {
        const RowOut w = row_out<PREFIX>(a, p, row, bh, split);
        if (p.part_o && d0 == 0) {
            p.part_ml[2 * w.slot] = m;
            p.part_ml[2 * w.slot + 1] = l;
        }
        const float s = p.part_o ? 1.0f : finish(a, w.head, m, l);
        float *po = p.part_o + w.slot * a.D;
        TQ *out = reinterpret_cast<TQ *>(a.o + w.i * a.o_i + w.head * a.o_h + w.b * a.o_b);
#pragma unroll
        for (int e = 0; e < N / 4; ++e) {
            const int at = d0 + 4 * e;
            if (at >= a.D) continue;
            if (p.part_o) *reinterpret_cast<f32x4 *>(po + at) = x[e];
            else store4<TQ>(out + at, x[e] * s);
        }
    }
    while (again) {
        const int at = __builtin_ctzll(again);
        again &= again - 1;
        redo_row<TK, TQ, PREFIX>(a, p, __builtin_amdgcn_readlane(row, at), bh, split, j_begin, j_end);
    }
}

// the splits' partial results of a row, in their order: one wave a row, groups of DP / 4 lanes take
// every other split
template <typename TQ, int DP>
__global__ __launch_bounds__(256) void attn_join_kernel(const AttnArgs a, const AttnPart p) {
    __shared__ float weight[4][MAX_SLOTS];
    constexpr int LPR = DP / 4, GROUPS = 64 / LPR;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t rr = (int64_t)blockIdx.x * 4 + wave;
    const int G = a.H / a.Hk, per = a.n_q * G;
    if (rr >= (int64_t)a.B * a.Hk * per) return;
    const int r = (int)(rr % per), hk = (int)(rr / per % a.Hk), b = (int)(rr / per / a.Hk), i = r / G, head = hk * G + r % G;
    const float *ml = p.part_ml + 2 * rr * p.slots;
    float m = -INFINITY;
    for (int s = lane; s < p.slots; s += 64) m = fmaxf(m, ml[2 * s]);
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor(m, s, 64));
    float l = 0.0f;
    for (int s = lane; s < p.slots; s += 64) {
        const float f = m == -INFINITY ? 1.0f : exp2f(ml[2 * s] - m);
        weight[wave][s] = f;
        l += ml[2 * s + 1] * f;
    }
    l = wave_add(l);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (the wave's own weights)
    const int d = lane % LPR * 4, grp = lane / LPR;
    f32x4 x{};
    if (d < a.D)
        for (int s = grp; s < p.slots; s += GROUPS) x += *reinterpret_cast<const f32x4 *>(p.part_o + (rr * p.slots + s) * a.D + d) * weight[wave][s];
#pragma unroll
    for (int s = LPR; s < 64; s <<= 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] += __shfl_xor(x[e], s, 64);
    if (grp != 0 || d >= a.D) return;
    TQ *out = reinterpret_cast<TQ *>(a.o + i * a.o_i + head * a.o_h + b * a.o_b);
    store4<TQ>(out + d, x * finish(a, head, m, l));
}

// one round of pieces: LDS place `slot` (row slot / CPR, place slot % CPR) takes row `row` of the tensor's tile
template <int DP>
__device__ __forceinline__ uint32_t piece_off(int place, int swz, int D) { return (uint32_t)(min(place ^ swz, D / 8 - 1) * 16); }

template <typename TK, typename TQ, int DP, bool BY_ROWS, bool PREFIX>
__global__ __launch_bounds__((AttnTile<TK, TQ, DP, BY_ROWS, PREFIX>::WAVES * 64), (BY_ROWS && DP <= 128 ? 2 : 1)) void attn_tile_kernel(const AttnArgs a, const AttnPart p) {
    using T = AttnTile<TK, TQ, DP, BY_ROWS, PREFIX>;
    typedef typename T::x8 x8;
    constexpr bool SPLIT = T::SPLIT;
    constexpr int KT = T::KT, CPR = T::CPR, RPI = T::RPI, ROUNDS = T::ROUNDS, BYTES = T::BYTES, NT = DP / 16, NB = DP / 32;
    __shared__ __align__(16) char lds[T::LDS];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    // problem, row tile (the last ones first: with a causal rule they see the most keys), split of the keys
    int id = blockIdx.x;
    const int bh = id % p.n_bh;
    id /= p.n_bh;
    const int split = id % p.n_split, tile = p.row_tiles - 1 - id / p.n_split;
    const int G = a.H / a.Hk, hk = bh % a.Hk, pb = bh / a.Hk;

    // this lane's row
    const int row0 = BY_ROWS ? tile * 128 + wave * 32 : tile * 32;
    const int row = min(row0 + (lane & 31), p.rows - 1);
    const bool row_ok = row0 + (lane & 31) < p.rows;
    const int g = row % G, bi = row / G;
    const int i = PREFIX ? bi % a.n_q : bi, b = PREFIX ? bi / a.n_q : pb;
    const int head = hk * G + g;

    // keys of this split, and how many of them the lane's row sees
    const int n = PREFIX ? a.n_prefix : own_len(a, b);
    int end = n;                                    // of the workgroup's rows
    if (!PREFIX && a.causal) {
        const int last = min(BY_ROWS ? tile * 128 + 127 : row0 + 31, p.rows - 1) / G;
        end = max(0, n - a.n_q + last + 1);
    }
    int j_begin = 0, j_end = end;
    if (p.n_split > 1) {
        const int per = ((end + p.n_split - 1) / p.n_split + 127) & ~127;
        j_begin = min(end, split * per);
        j_end = min(end, j_begin + per);
    }
    j_begin = __builtin_amdgcn_readfirstlane(j_begin);
    j_end = __builtin_amdgcn_readfirstlane(j_end);
    const int seen = min(j_end, !PREFIX && a.causal ? n - a.n_q + i + 1 : n);

    const bool masked = !PREFIX && a.mask != nullptr;
    const char *mrow = nullptr;
    float slope = 0.0f;
    if (masked) {
        mrow = a.mask + i * a.m_i + (head % a.m_nh) * a.m_h + (b % a.m_nb) * a.m_b;
        slope = slope_of(a, head) * LOG2E;
    }

    const char *kb = PREFIX ? a.kp + hk * a.kp_h : a.k + hk * a.k_h + (int64_t)(pb / a.kv_b) * a.k_b;
    const char *vb = PREFIX ? a.vp + hk * a.vp_h : a.v + hk * a.v_h + (int64_t)(pb / a.kv_b) * a.v_b;
    const int64_t k_j = PREFIX ? a.kp_j : a.k_j, v_j = PREFIX ? a.vp_j : a.v_j;

    // the tile at key j into stage `st` of this wave's (BY_ROWS: the workgroup's) LDS
    const int ltid = BY_ROWS ? tid : lane, lrow = ltid / CPR, place = ltid % CPR;
    char *stage0 = lds + (BY_ROWS ? 0 : wave * 4 * BYTES);
    const uint32_t k_row = (uint32_t)lrow * (uint32_t)k_j, v_row = (uint32_t)lrow * (uint32_t)v_j;
    auto load = [&](int j, int st) {
        char *kd = stage0 + st * 2 * BYTES + (BY_ROWS ? wave * 1024 : 0), *vd = kd + BYTES;
        const i32x4 kr = buffer_at(kb + j * k_j), vr = buffer_at(vb + j * v_j);
        const int last = j_end - 1 - j;
        if (last >= KT - 1) {
#pragma unroll
            for (int u = 0; u < ROUNDS; ++u) {
                const int r = u * RPI + lrow;
                dma16(kr, kd + u * T::LOADERS * 16, k_row + piece_off<DP>(place, swz_k<DP>(r), a.D), (uint32_t)(u * RPI) * (uint32_t)k_j);
                dma16(vr, vd + u * T::LOADERS * 16, v_row + piece_off<DP>(place, swz_v<DP>(r), a.D), (uint32_t)(u * RPI) * (uint32_t)v_j);
            }
        } else {   // rows behind the keys: the last key again
#pragma unroll
            for (int u = 0; u < ROUNDS; ++u) {
                const int r = u * RPI + lrow;
                const uint32_t rr = (uint32_t)min(r, last);
                dma16(kr, kd + u * T::LOADERS * 16, rr * (uint32_t)k_j + piece_off<DP>(place, swz_k<DP>(r), a.D), 0);
                dma16(vr, vd + u * T::LOADERS * 16, rr * (uint32_t)v_j + piece_off<DP>(place, swz_v<DP>(r), a.D), 0);
            }
        }
    };

    // the first tile's DMA, then the queries, then one wait for both: the compiler, which knows of the
    // latter only, would otherwise wait inside the loop, and there for the tile ahead too
    const int j0 = BY_ROWS ? j_begin : j_begin + wave * 32;
    if (j0 < j_end) load(j0, 0);

    // queries: lane (row, h) holds values 16 t + 8 h .. + 7 of its row
    x8 qf[NT], ql[SPLIT ? NT : 1];
    float c = a.scale;
    {
        const char *qr = a.q + i * a.q_i + head * a.q_h + b * a.q_b;
        if constexpr (SPLIT) {
            float v[NT][8], top = 0.0f;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int d = 16 * t + 8 * h;
                f32x4 x0{}, x1{};
                if (d < a.D) {
                    x0 = *reinterpret_cast<const f32x4 *>(qr + 4 * d);
                    x1 = *reinterpret_cast<const f32x4 *>(qr + 4 * d + 16);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[t][e] = x0[e];
                    v[t][4 + e] = x1[e];
                    top = fmaxf(top, fmaxf(fabsf(x0[e]), fabsf(x1[e])));
                }
            }
            top = fmaxf(top, swap32_f(top));
            // 2^-e * q below 1: no f16 overflows, and the second term keeps its bits
            int e2 = 0;
            if (top > 0.0f && top < INFINITY) (void)frexpf(top, &e2);
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float x = ldexpf(v[t][e], -e2);
                    const _Float16 hi = (_Float16)x;
                    qf[t][e] = hi;
                    ql[t][e] = (_Float16)(x - (float)hi);
                }
            c = ldexpf(c, e2);
        } else {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                x8 z{};
                qf[t] = 16 * t + 8 * h < a.D ? *reinterpret_cast<const x8 *>(qr + 2 * (16 * t + 8 * h)) : z;
            }
        }
    }
    const bool capped = a.cap != 0.0f;
    const float c_cap = capped ? c / a.cap : 0.0f, cap2 = a.cap * LOG2E;
    c *= LOG2E;
    // the maximum is taken of the bare products, so their factor must be above 0: its sign goes into
    // the queries, and for 0 a factor that leaves nothing of any product of f16 values
    if (c < 0.0f) {
        c = -c;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            qf[t] = -qf[t];
            if constexpr (SPLIT) ql[t] = -ql[t];
        }
    }
    c = fmaxf(c, 0x1p-126f);
    __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0)

    f32x16 o[NB];
#pragma unroll
    for (int d = 0; d < NB; ++d) o[d] = f32x16{};
    float m = -INFINITY, l = 0.0f;   // (l: of the lane's own keys)

    // the mask's values at the tile's keys, in the order of the scores
    auto fetch = [&](int j, f16x4 (&w)[KT / 8]) {
        const int left = seen - j - 4 * h;
#pragma unroll
        for (int r = 0; r < KT / 8; ++r) {
            const _Float16 *mp = reinterpret_cast<const _Float16 *>(mrow) + j + 8 * r + 4 * h;
            w[r] = f16x4{};
            if (a.m_vec && 8 * r + 4 <= left) {
                w[r] = *reinterpret_cast<const f16x4 *>(mp);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (8 * r + e < left) w[r][e] = mp[e];
            }
        }
    };

    auto compute = [&](int j, int st, const f16x4 (&w)[KT / 8]) {
        const char *kt = stage0 + st * 2 * BYTES, *vt = kt + BYTES;
        f32x16 s[KT / 32];
        const int krow = lane & 31, ksw = swz_k<DP>(krow);
#pragma unroll
        for (int u = 0; u < KT / 32; ++u) {
            s[u] = f32x16{};
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const x8 kf = *reinterpret_cast<const x8 *>(kt + (u * 32 + krow) * DP * 2 + (((2 * t + h) ^ ksw) * 16));
                s[u] = mma(kf, qf[t], s[u]);
                if constexpr (SPLIT) s[u] = mma(kf, ql[t], s[u]);
            }
        }
        // s[u][r] is the product of key j + 32 u + 8 (r / 4) + 4 h + r % 4; f times it is the score in units
        // of log 2
        const int left = seen - j - 4 * h;
        float f = c;
        if (capped || masked) {
            f = 1.0f;
#pragma unroll
            for (int u = 0; u < KT / 32; ++u)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    float x = s[u][r];
                    x = capped ? cap2 * tanhf(x * c_cap) : x * c;
                    if (masked) {
                        const float add = (float)w[4 * u + r / 4][r % 4];
                        x = add == -INFINITY ? -INFINITY : fmaf(slope, add, x);
                    }
                    s[u][r] = x;
                }
        }
        if (__any(seen - j < KT)) {
#pragma unroll
            for (int u = 0; u < KT / 32; ++u)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (32 * u + 8 * (r / 4) + r % 4 >= left) s[u][r] = -INFINITY;
        }
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < KT / 32; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, s[u][r]);
        top = fmaxf(top, swap32_f(top)) * f;
        if (__any(top > m + LAZY)) {
            const float m1 = top > m + LAZY ? top : m;
            const float drop = m == m1 ? 1.0f : exp2f(m - m1);   // (m = -inf: nothing is summed yet)
            m = m1;
            l *= drop;
#pragma unroll
            for (int d = 0; d < NB; ++d) o[d] *= drop;
        }
        const float ref = BIAS - (m == -INFINITY ? 0.0f : m);
        float sum = 0.0f;
#pragma unroll
        for (int u = 0; u < KT / 32; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[u][r] = __builtin_amdgcn_exp2f(fmaf(s[u][r], f, ref));
                sum += s[u][r];
            }
        l += sum;
        // O^T += V^T P^T, 16 keys a step: the lane's weights 8 (t % 2) .. + 7 of block t / 2
        const int vi = lane & 15, vrow = 4 * h + (vi >> 2), vch = 2 * ((lane >> 4) & 1) + ((vi & 3) >> 1), vsw = swz_v<DP>(vrow);
#pragma unroll
        for (int t = 0; t < KT / 16; ++t) {
            x8 pf, pl;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = s[t / 2][8 * (t % 2) + e];
                pf[e] = (TK)x;
                if constexpr (SPLIT) pl[e] = (TK)(x - (float)pf[e]);
            }
#pragma unroll
            for (int d = 0; d < NB; ++d) {
                const char *vp = vt + (16 * t + vrow) * DP * 2 + (((4 * d + vch) ^ vsw) * 16) + 8 * (vi & 1);
                const i16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4 *)vp);
                const i16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4 *)(vp + 8 * DP * 2));
                const i16x8 vv = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
                const x8 vf = __builtin_bit_cast(x8, vv);
                o[d] = mma(vf, pf, o[d]);
                if constexpr (SPLIT) o[d] = mma(vf, pl, o[d]);
            }
        }
    };

    if constexpr (BY_ROWS) {
        // (a later row sees no fewer keys)
        const int seen_most = row0 < p.rows ? __builtin_amdgcn_readlane(seen, 31) : 0;
        f16x4 w[KT / 8], ahead[KT / 8];
        if (masked && j_begin < j_end) fetch(j_begin, ahead);
        int st = 0;
        for (int j = j_begin; j < j_end; j += KT, st ^= 1) {
            // this wave's share of the tile has come; behind the barrier everyone's has, and the other stage is read
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (masked) {   // (moved here, so that the compiler's wait for them comes before the next DMA)
#pragma unroll
                for (int r = 0; r < KT / 8; ++r) {
                    w[r] = ahead[r];
                    asm volatile("" : "+v"(w[r]));
                }
            }
            if (j + KT < j_end) {
                load(j + KT, st ^ 1);
                if (masked) fetch(j + KT, ahead);
            }
            if (j < seen_most) compute(j, st, w);
        }
    } else {
        constexpr int STEP = T::WAVES * 32;
        int j = j0, st = 0;
        f16x4 w[KT / 8];
        if (j + STEP < j_end) load(j + STEP, 1);
        for (; j < j_end; j += STEP, st ^= 1) {
            if (masked) fetch(j, w);
            if (j + STEP < j_end) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * ROUNDS) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            compute(j, st, w);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the stage is read
            if (j + 2 * STEP < j_end) load(j + 2 * STEP, st);
        }
    }
    l += swap32_f(l);
    const float me = m - BIAS;   // (-inf: no key)

    if constexpr (!BY_ROWS) {
        // join the waves: each leaves its rows in its own stages, wave w then joins values w * DP/4 ..
        asm volatile("" ::: "memory");
        float *po = reinterpret_cast<float *>(lds + wave * 4 * BYTES);   // [row][DP], DP * 128 bytes = 2 BYTES
        float *pm = reinterpret_cast<float *>(lds + wave * 4 * BYTES + 2 * BYTES);
#pragma unroll
        for (int d = 0; d < NB; ++d)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                const f32x4 x = {o[d][4 * r4], o[d][4 * r4 + 1], o[d][4 * r4 + 2], o[d][4 * r4 + 3]};
                *reinterpret_cast<f32x4 *>(po + (lane & 31) * DP + 32 * d + 8 * r4 + 4 * h) = x;
            }
        if (h == 0) {
            pm[lane] = me;
            pm[32 + lane] = l;
        }
        __syncthreads();
        join_waves<TK, TQ, DP, T::WAVES, PREFIX>(a, p, lds, 4 * BYTES, 2 * BYTES, row0, bh, split, j_begin, j_end);
    } else {
        store_rows<TK, TQ, DP, PREFIX>(a, p, o, me, l, row, row_ok, bh, split, j_begin, j_end);
    }
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

// what a call launches, by its shapes alone
struct AttnPlan {
    bool tiled;                              // else attn_rows_kernel
    bool own_rows, pre_rows;                 // row tiles of 128 (4 waves of 32), or 32 rows with split keys
    int own_tiles, own_splits, pre_tiles, pre_splits, slots;
};

static AttnPlan plan_attn(const AttnTensors &t) {
    AttnPlan p{};
    const int64_t n_q = t.q.ne[1], H = t.q.ne[2], B = t.q.ne[3], Hk = t.k.ne[2], G = H / Hk;
    // the tile kernel's offsets inside a tile are 32-bit: positions up to 16 MiB apart
    p.tiled = true;
    for (const TensorView *x : {&t.k, &t.v, t.kp, t.vp})
        if (x && x->nb[1] >= (1u << 24)) p.tiled = false;
    if (!p.tiled) return p;
    auto pick = [](int64_t rows, int64_t problems, int64_t keys, bool &by_rows, int &tiles, int &splits) {
        by_rows = rows > 32;
        tiles = (int)((rows + (by_rows ? 127 : 31)) / (by_rows ? 128 : 32));
        const int64_t groups = std::max<int64_t>(1, problems * tiles);
        splits = (int)std::max<int64_t>(1, std::min({(512 + groups - 1) / groups, (keys + 127) / 128, (int64_t)MAX_SLOTS / 2}));
        if (groups >= 256) splits = 1;
    };
    pick(n_q * G, B * Hk, t.k.ne[1], p.own_rows, p.own_tiles, p.own_splits);
    p.slots = p.own_splits;
    if (t.kp) {
        pick(B * n_q * G, Hk, t.kp->ne[1], p.pre_rows, p.pre_tiles, p.pre_splits);
        p.slots += p.pre_splits;
    }
    return p;
}

size_t flash_attn_work(const AttnTensors &t) {
    const AttnPlan p = plan_attn(t);
    return p.slots > 1 ? (size_t)t.q.ne[1] * t.q.ne[2] * t.q.ne[3] * p.slots * (t.q.ne[0] + 2) * sizeof(float) : 0;
}

template <typename TK, typename TQ, int DP, bool BY_ROWS, bool PREFIX>
static void launch_tiles(const AttnArgs &a, const AttnPart &p, hipStream_t st) {
    const dim3 grid((unsigned)(p.n_bh * p.row_tiles * p.n_split));
    hipLaunchKernelGGL((attn_tile_kernel<TK, TQ, DP, BY_ROWS, PREFIX>), grid, dim3(AttnTile<TK, TQ, DP, BY_ROWS, PREFIX>::WAVES * 64), 0, st, a, p);
}

template <typename TK, typename TQ, int DP>
static void launch_attn(const AttnArgs &a, const AttnPlan &pl, void *work, hipStream_t st) {
    const int G = a.H / a.Hk;
    AttnPart p{};
    p.slots = pl.slots;
    if (pl.slots > 1) {
        const size_t rows = (size_t)a.B * a.H * a.n_q * pl.slots;
        p.part_o = static_cast<float *>(work);
        p.part_ml = p.part_o + rows * a.D;
    }
    if (pl.pre_splits) {
        p.slot0 = 0;
        p.n_split = pl.pre_splits;
        p.n_bh = a.Hk;
        p.rows = a.B * a.n_q * G;
        p.row_tiles = pl.pre_tiles;
        if (pl.pre_rows) launch_tiles<TK, TQ, DP, true, true>(a, p, st);
        else launch_tiles<TK, TQ, DP, false, true>(a, p, st);
    }
    p.slot0 = pl.slots - pl.own_splits;
    p.n_split = pl.own_splits;
    p.n_bh = a.B * a.Hk;
    p.rows = a.n_q * G;
    p.row_tiles = pl.own_tiles;
    if (pl.own_rows) launch_tiles<TK, TQ, DP, true, false>(a, p, st);
    else launch_tiles<TK, TQ, DP, false, false>(a, p, st);
    if (pl.slots > 1) {
        const int64_t rows = (int64_t)a.B * a.H * a.n_q;
        hipLaunchKernelGGL((attn_join_kernel<TQ, DP>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a, p);
    }
}

template <typename TK, typename TQ>
static void launch_attn_d(const AttnArgs &a, const AttnPlan &pl, void *work, hipStream_t st) {
    if (a.D <= 64) launch_attn<TK, TQ, 64>(a, pl, work, st);
    else if (a.D <= 128) launch_attn<TK, TQ, 128>(a, pl, work, st);
    else launch_attn<TK, TQ, 256>(a, pl, work, st);
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
        a.m_vec = aligned_to(*t.mask, 8);
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
    const AttnPlan pl = plan_attn(t);
    if (pl.tiled) {
        if (q.type == T_F32) launch_attn_d<_Float16, float>(a, pl, work, st);
        else if (q.type == T_F16) launch_attn_d<_Float16, _Float16>(a, pl, work, st);
        else launch_attn_d<__bf16, __bf16>(a, pl, work, st);
    } else {
        const dim3 grid(a.n_q, a.H, a.B);
        if (q.type == T_F32) hipLaunchKernelGGL((attn_rows_kernel<float, _Float16>), grid, dim3(256), 0, st, a);
        else if (q.type == T_F16) hipLaunchKernelGGL((attn_rows_kernel<_Float16, _Float16>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((attn_rows_kernel<__bf16, __bf16>), grid, dim3(256), 0, st, a);
    }
    return hipGetLastError() == hipSuccess ? GGML_MI355X_OK : GGML_MI355X_EHIP;
}

}  // namespace mi355x
