// attention_impl.h — softmax(scale * Q K^T + mask) V over a key / value cache (GGML_OP_FLASH_ATTN_EXT),
// and the same for sequences that share one long prefix.
//
// Per (batch b, head h, query i), with hk = h / (H / Hk) the shared key / value head:
//     x_j = cap * tanh(scale * q.k_j / cap)  [or scale * q.k_j]  + slope_h * mask_ij
//     o   = sum_j exp(x_j - m) v_j / (sum_j exp(x_j - m) + exp(sink_h - m)),  m = max(x, sink)
// over the keys j < len_b that the mask leaves (not -inf) and, when causal, j <= len_b - n_q + i.
// A row that sees nothing is zeros. A key that a row does not see takes no part in it, whatever its
// bytes hold: caches are not cleared, and a NaN times a weight of 0 would be NaN.
#pragma once

#include "attention.h"
#include "qcommon.h"

#include <type_traits>

namespace mi355x {

namespace {

constexpr float LOG2E = 1.44269504088896340736f;

__device__ __forceinline__ float wave_add(float v) {
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) v += __shfl_xor(v, s, 64);
    return v;
}

// tanh without a branch: below 1/4 the odd Taylor polynomial to x^9 (the next term is 2^-26 of x there), above
// (1 - t) / (1 + t), t = exp(-2 |x|); off by some 3 units in the last place
__device__ __forceinline__ float tanh_of(float x) {
    const float y = fabsf(x), t = __builtin_amdgcn_exp2f(-2.0f * LOG2E * y), q = x * x;
    const float big = copysignf((1.0f - t) * __builtin_amdgcn_rcpf(1.0f + t), x);
    const float odd = fmaf(q, fmaf(q, fmaf(q, fmaf(q, 62.0f / 2835.0f, -17.0f / 315.0f), 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
    return y < 0.25f ? x * odd : big;   // (a NaN fails the comparison and comes out of `big`)
}

__device__ __forceinline__ float slope_of(const AttnArgs &a, int h) {
    if (a.bias_heads == 0) return 1.0f;
    return h < a.bias_heads ? powf(a.m0, (float)(h + 1)) : powf(a.m1, (float)(2 * (h - a.bias_heads) + 1));
}

// a score in units of log 2: the cap and the factor log2(e), so that exp is one exp2
__device__ __forceinline__ float scaled(const AttnArgs &a, float s) {
    s *= a.scale;
    if (a.cap != 0.0f) s = a.cap * tanh_of(s / a.cap);
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
        // a row that is NaN throughout stays it: NaN weights of a whole model must not cost every key for every row
        bool lost = true;
#pragma unroll
        for (int c = 0; c < 4; ++c) lost &= lane + 64 * c >= a.D || r.o[c] != r.o[c];
        if (__all(lost)) return;
    }
}

// one workgroup per (query, head, batch): its waves take every fourth key. For layouts whose positions
// lie too far apart for the tile kernel's 32-bit offsets
template <typename TQ, typename TK>
__global__ __launch_bounds__(256) void attn_rows_kernel(const AttnArgs a) {
    __shared__ RowState part[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int i = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
    const int hk = a.by_G.of(h), bk = a.by_kv_b.of(b);
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
//   BY_ROWS: 4 or 8 waves of 32 rows each share tiles of KT keys (prompts, shared prefixes)
//   else:    the waves share 32 rows and take tiles of 32 keys in turn, joined at the end (tokens)
// 16-byte pieces of a tile's rows are permuted (swz_k, swz_v) so that neither read meets an LDS bank
// twice; the DMA writes LDS in order, so the permutation is in the addresses it reads from.
//
// m moves only when a tile exceeds it by more than 2^LAZY, so the 16 DP/32 accumulators are rarely
// rescaled; weights are kept 2^BIAS times larger: f16 ones up to 2^(BIAS + LAZY) = 2^15, which f16 still holds,
// so that small ones stay clear of its subnormals (f16 values times them stay far below f32's end); bf16 ones
// up to 1, since a bf16 value may lie anywhere in f32's range and its product must too.
// F32 queries: q (scaled by a power of two per row) and p are each carried as a sum of two f16 values, two MFMAs per
// product: to 2^-22 of the value, or of q 2^-40 of its row's largest, of p 2^-33 of the largest weight. 16-bit ones: p
// so too where keys are split (bf16: to 2^-16), else rounded to their type; its sum is of the unrounded weights.
//
// Bound by the matrix cores and, beside them, the vector units' exponentials, maxima and sums where a key
// meets many rows: 8192 causal tokens, 32 heads on 8 of 128 bf16 values 531 us, 1.04 PFLOP/s (a large library product
// reaches 1.2). By memory where it meets few: 64 tokens, the same heads in f16, ragged to 8192 keys 291 us,
// 5.5 TB/s; one token behind 131072 keys 101 us, 5.3. By latency in small calls: one token's 12 heads of 64
// values, 1000 keys 6.0 us and 3.3 for the join. A mask's rows lie across a load's lanes: 16 heads of 80 values,
// 2 x 777 queries, 1900 keys, f32, 58 us, 46 without a mask.
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

constexpr float LAZY = 7.0f;

template <typename T> struct Vec;
template <> struct Vec<_Float16> {
    typedef f16x8 x8;
    static constexpr float BIAS = 8.0f;
};
template <> struct Vec<__bf16> {
    typedef bf16x8 x8;
    static constexpr float BIAS = -LAZY;
};

__device__ __forceinline__ f32x16 mma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

// the permuted place of 16-byte piece c of row r of a tile with DP values a row
template <int DP> __device__ __forceinline__ int swz_k(int r) { return DP == 64 ? (r >> 1) & 7 : r & 15; }
template <int DP> __device__ __forceinline__ int swz_v(int r) { return DP == 64 ? ((r >> 1) & 1) << 2 : (r & 3) << 2; }

// which keys and rows some of a launch's workgroups work on
struct AttnPart {
    float *part_o, *part_ml;   // partial results, or nullptr: the call's result
    int slot0;                 // these splits among
    int slots;                 // all partial results of a row
    Div by_split, by_bh;       // splits; (batch,) key / value head problems
    int rows, row_tiles;       // of each
    int blocks;
};

// LDS DMA: 16 bytes per lane from the buffer into LDS, the wave's 1 KiB at dst + 1024 * u. Written out because the
// compiler, which can not tell the stages apart, makes every LDS read wait for each DMA that it knows of; the
// kernel waits itself. No result registers; the address registers are read at issue; m0, the LDS address, is a
// reserved register, which the compiler sets right before an own use (these kernels have none). A change of m0
// costs a DMA some 40 cycles, so four of them share one: the instruction's offset moves both addresses, and
// the buffer begins DMA_BACK bytes early to give its share back. The nops are the wait states from a scalar's
// write by a vector instruction and from m0's to their use.
typedef int i32x4 __attribute__((ext_vector_type(4)));
constexpr int DMA_BACK = 4096;
__device__ __forceinline__ i32x4 buffer_at(const char *p) {   // a raw buffer of 2 GiB, from DMA_BACK bytes before p
    const uint64_t at = (uint64_t)(uintptr_t)p - DMA_BACK;
    return i32x4{(int)__builtin_amdgcn_readfirstlane((uint32_t)at), (int)__builtin_amdgcn_readfirstlane((uint32_t)(at >> 32) & 0xffff), 0x7fffffff, 0x00020000};
}
// number u of a wave's DMAs in a row (dst: of the first), from byte voff (the lane's) + soff behind the buffer's p
__device__ __forceinline__ void dma16(int u, i32x4 buf, const char *dst, uint32_t voff, uint32_t soff) {
    const uint32_t s = soff + DMA_BACK - u % 4 * 1024;
    switch (u % 4) {
        case 0: {
            const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_const)dst + (uint32_t)u * 1024);
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(at), "v"(voff), "s"(buf), "s"(s) : "memory");
            break;
        }
        case 1: asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, %2 offen offset:0x400 lds" ::"v"(voff), "s"(buf), "s"(s) : "memory"); break;
        case 2: asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, %2 offen offset:0x800 lds" ::"v"(voff), "s"(buf), "s"(s) : "memory"); break;
        default: asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, %2 offen offset:0xc00 lds" ::"v"(voff), "s"(buf), "s"(s) : "memory");
    }
}

// DC: the head size that the products are formed for; DP: the next power of two, a row's place in LDS (what lies
// behind the row is a copy of its last piece, and no product reads it beyond DC)
constexpr int row_place(int DC) { return DC <= 64 ? 64 : DC <= 128 ? 128 : 256; }

template <typename TK, typename TQ, int DC, int WAVES, bool BY_ROWS, int TURNS = 1>
struct AttnTile {
    static constexpr bool SPLIT = sizeof(TQ) == 4;
    static constexpr int DP = row_place(DC);
    static constexpr int KT = BY_ROWS && DP <= 128 ? 64 : 32;   // keys of a tile
    static constexpr int CPR = DP / 8;                          // 16-byte pieces of a row
    static constexpr int RPD = 64 / CPR;                        // rows of a DMA
    static constexpr int ROUNDS = KT / RPD / (BY_ROWS ? WAVES / TURNS : 1);   // a wave's DMAs of a tile of keys, or of values
    static constexpr int BYTES = KT * DP * 2;                   // of a tile of keys, and of values
    // BY_ROWS: two stages of keys and values; else one of each per wave, whose 32 rows also fit it as f32,
    // and those rows' maxima and sums
    static constexpr int STRETCH = BY_ROWS ? 4 * BYTES : 2 * BYTES + 256;
    static constexpr int LDS = (BY_ROWS ? TURNS : WAVES) * STRETCH;
    static constexpr int STEP = BY_ROWS ? TURNS * KT : WAVES * 32;   // keys that a workgroup takes at a time
    typedef typename Vec<TK>::x8 x8;
};

// F32 queries as two f16 terms. A row is scaled to below 2^15, so that no f16 overflows and the second terms lie as far
// above f16's subnormals as they can; infinities are no measure of the others, and have no second term
__device__ __forceinline__ float size_of(float x) { return fabsf(x) < INFINITY ? fabsf(x) : 0.0f; }
__device__ __forceinline__ int shift_of(float top) {
    if (top == 0.0f) return 0;
    int e;
    (void)frexpf(top, &e);
    return 15 - e;
}
__device__ __forceinline__ void query_terms(float q, int up, _Float16 &hi, _Float16 &lo) {
    const float x = ldexpf(q, up);
    hi = (_Float16)x;
    lo = fabsf(x) < INFINITY ? (_Float16)(x - (float)hi) : (_Float16)0.0f;
}

// a finished row's place: the call's result, or this launch's partial result (sum, maximum, weighted values)
struct RowOut {
    int b, i, head;
    int64_t slot;   // of the partial results
};
template <bool PREFIX>
__device__ __forceinline__ RowOut row_out(const AttnArgs &a, const AttnPart &p, int row, int bh, int split) {
    const int G = (int)a.by_G.d, pb = a.by_Hk.of(bh), hk = bh - pb * a.Hk, bi = a.by_G.of(row), g = row - bi * G;
    RowOut r;
    r.b = PREFIX ? a.by_n_q.of(bi) : pb;
    r.i = PREFIX ? bi - r.b * a.n_q : bi;
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

template <typename TQ> __device__ __forceinline__ void store4(TQ *p, f32x4 x);
template <> __device__ __forceinline__ void store4(float *p, f32x4 x) { *reinterpret_cast<f32x4 *>(p) = x; }
template <> __device__ __forceinline__ void store4(_Float16 *p, f32x4 x) {
    *reinterpret_cast<f16x4 *>(p) = f16x4{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
}
template <> __device__ __forceinline__ void store4(__bf16 *p, f32x4 x) {
    *reinterpret_cast<bf16x4 *>(p) = bf16x4{(__bf16)x[0], (__bf16)x[1], (__bf16)x[2], (__bf16)x[3]};
}

// a row out of the accumulators: lane (row, h) holds values 32 d + 8 r4 + 4 h .. + 3
template <typename TQ, int NB>
__device__ __forceinline__ void put_row(const AttnArgs &a, const AttnPart &p, const RowOut &w, const f32x16 (&o)[NB], float m, float l) {
    const int h = (threadIdx.x & 63) >> 5;
    if (p.part_o && h == 0) {
        p.part_ml[2 * w.slot] = m;
        p.part_ml[2 * w.slot + 1] = l;
    }
    const float f = p.part_o ? 1.0f : finish(a, w.head, m, l);
    float *po = p.part_o + w.slot * a.D;
    TQ *out = reinterpret_cast<TQ *>(a.o + w.i * a.o_i + w.head * a.o_h + w.b * a.o_b);
#pragma unroll
    for (int d = 0; d < NB; ++d)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            if (32 * d + 8 * r4 >= a.D) continue;   // (D is a multiple of 8)
            const int at = 32 * d + 8 * r4 + 4 * h;
            const f32x4 x = f32x4{o[d][4 * r4], o[d][4 * r4 + 1], o[d][4 * r4 + 2], o[d][4 * r4 + 3]} * f;
            if (p.part_o) *reinterpret_cast<f32x4 *>(po + at) = x;
            else store4<TQ>(out + at, x);
        }
}

// A weight of 0 times a NaN or an infinity in a key that a row does not see, but another row of its tile
// or the DMA's filling does, makes the row's sums NaN. Such rows (bits of `again`) are formed again by a wave, all at
// once: the scores of 32 keys by the same products, out of operands read straight from memory, then the keys' values one
// key at a time, for the rows that see it; a NaN that a row does see comes out again. It ends where the weights of all rows
// have become NaN, which makes them NaN throughout. Rolled loops and few registers, so that the tiles' loop,
// which nearly always is all there is, keeps its own (values by MFMA out of unrolled loads held 200 more scalars and cost
// 64-value heads a wave a SIMD). Bound by the vector units and the loads' latency, 0.8 us a key: 8192 causal tokens, 32
// heads on 8 of 128 bf16 values, 0.54 ms, with one NaN value that every row sees 17 (500 a row and a key at a
// time); 2048 masked f32 queries 0.12, with a NaN in one hidden key 2.0.
template <typename TK, typename TQ, int DC, bool PREFIX>
__device__ __forceinline__ void redo_rows(const AttnArgs &a, const AttnPart &p, int row0, uint32_t again, int bh, int split, int j_begin, int j_end) {
    typedef typename Vec<TK>::x8 x8;
    constexpr bool SPLIT = sizeof(TQ) == 4;
    constexpr int NT = DC / 16, NB = DC / 32;
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));   // (or the compiler keeps the caller's addresses of the row through its loop)
    const int h = lane >> 5;
    const RowOut w = row_out<PREFIX>(a, p, min(row0 + (lane & 31), p.rows - 1), bh, split);
    const int pb = a.by_Hk.of(bh), hk = bh - pb * a.Hk, bk = PREFIX ? 0 : a.by_kv_b.of(pb);
    const char *kb = PREFIX ? a.kp + hk * a.kp_h : a.k + hk * a.k_h + bk * a.k_b;
    const char *vb = PREFIX ? a.vp + hk * a.vp_h : a.v + hk * a.v_h + bk * a.v_b;
    const int64_t k_j = PREFIX ? a.kp_j : a.k_j, v_j = PREFIX ? a.vp_j : a.v_j;
    const int seen = min(j_end, PREFIX ? a.n_prefix : a.causal ? own_len(a, w.b) - a.n_q + w.i + 1 : own_len(a, w.b));
    const _Float16 *mask = nullptr;
    if (!PREFIX && a.mask) mask = reinterpret_cast<const _Float16 *>(a.mask + w.i * a.m_i + (w.head % a.m_nh) * a.m_h + (w.b % a.m_nb) * a.m_b);
    const float slope = mask ? slope_of(a, w.head) * LOG2E : 0.0f;
    const TQ *q = reinterpret_cast<const TQ *>(a.q + w.i * a.q_i + w.head * a.q_h + w.b * a.q_b);
    int up = 0;
    if constexpr (SPLIT) {
        float size = 0.0f;
        for (int d = 0; d < a.D; ++d) size = fmaxf(size, size_of(q[d]));
        up = shift_of(size);
    }
    const float c = ldexpf(a.scale, -up);

    f32x16 o[NB];
#pragma unroll
    for (int d = 0; d < NB; ++d) o[d] = f32x16{};
    float m = -INFINITY, l = 0.0f;
    for (int j = j_begin; j < j_end && __any(j < seen); j += 32) {
        f32x16 s{};
        const TK *kr = reinterpret_cast<const TK *>(kb + min(j + (lane & 31), j_end - 1) * k_j);
#pragma unroll 2
        for (int t = 0; t < NT; ++t) {
            const int d = 16 * t + 8 * h;
            x8 kf{}, qf{}, ql{};
            if (d < a.D) {
                kf = *reinterpret_cast<const x8 *>(kr + d);
                if constexpr (SPLIT) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        _Float16 hi, lo;
                        query_terms(q[d + e], up, hi, lo);
                        qf[e] = hi;
                        ql[e] = lo;
                    }
                } else {
                    qf = *reinterpret_cast<const x8 *>(q + d);
                }
            }
            s = mma(kf, qf, s);
            if constexpr (SPLIT) s = mma(kf, ql, s);
        }
        // s[r] belongs to key j + 8 (r / 4) + 4 h + r % 4
        uint32_t sees = 0;
        float top = m;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int key = j + 8 * (r / 4) + 4 * h + r % 4;
            bool see = key < seen;
            float x = s[r] * c;
            if (a.cap != 0.0f) x = a.cap * tanh_of(x / a.cap);
            x *= LOG2E;
            if (mask) {
                const float add = see ? (float)mask[key] : -INFINITY;
                see &= add != -INFINITY;
                x = fmaf(slope, add, x);
            }
            s[r] = see ? x : -INFINITY;
            sees |= see ? 1u << r : 0u;
            top = fmaxf(top, s[r]);
        }
        if (!__any(sees)) continue;
        top = fmaxf(top, swap32_f(top));
        const float drop = m == top ? 1.0f : exp2f(m - top), ref = top == -INFINITY ? 0.0f : top;
        m = top;
        l *= drop;
#pragma unroll
        for (int d = 0; d < NB; ++d) o[d] *= drop;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(s[r] - ref);
        // two keys (one of the largest heads) on their way at a time
        constexpr int AT_ONCE = NB <= 4 ? 2 : 1;
        typedef TK x4 __attribute__((ext_vector_type(4)));
        for (int r = 0; r < 16; ++r) {
#pragma unroll
            for (int half0 = 0; half0 < 2; half0 += AT_ONCE) {
                x4 x[AT_ONCE][4 * NB];
#pragma unroll
                for (int u = 0; u < AT_ONCE; ++u) {
                    const int key = min(j + 8 * (r / 4) + 4 * (half0 + u) + r % 4, j_end - 1);
                    const TK *vr = reinterpret_cast<const TK *>(vb + key * v_j) + 4 * h;
#pragma unroll
                    for (int e = 0; e < 4 * NB; ++e) x[u][e] = 8 * e < a.D ? *reinterpret_cast<const x4 *>(vr + 8 * e) : x4{};
                }
#pragma unroll
                for (int u = 0; u < AT_ONCE; ++u) {
                    const int from = (lane & 31) + 32 * (half0 + u);
                    const float weight = __shfl(s[0], from, 64);
                    const bool see = __shfl(sees, from, 64) & 1;
                    if (see) {
                        l += weight;
#pragma unroll
                        for (int e = 0; e < 16 * NB; ++e) o[e / 16][e % 16] = fmaf(weight, (float)x[u][e / 4][e % 4], o[e / 16][e % 16]);
                    }
                }
            }
            // (the next weight and its bit, in the same registers)
            sees >>= 1;
#pragma unroll
            for (int e = 0; e < 15; ++e) s[e] = s[e + 1];
        }
        const uint64_t lost = __ballot(l != l);
        if (((uint32_t)lost & again) == again) break;
    }
    if (again >> (lane & 31) & 1) put_row<TQ, NB>(a, p, w, o, m, l);
}

// a wave's 32 rows, of which this lane's is `row`
template <typename TK, typename TQ, int DC, bool PREFIX>
__device__ __forceinline__ void store_rows(const AttnArgs &a, const AttnPart &p, const f32x16 (&o)[DC / 32], float m, float l, int row0, int row,
                                           bool row_ok, int bh, int split, int j_begin, int j_end) {
    // (a sum of infinities of both signs is NaN too: such a row is formed again for nothing, to the same result)
    float all = l;
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
        for (int d = 0; d < DC / 32; ++d) all += o[d][r];
    const bool bad = all != all;
    const uint64_t votes = __ballot(bad && row_ok);
    const uint32_t again = (uint32_t)votes | (uint32_t)(votes >> 32);
    // (such rows too, under their new values: registers enough for a branch less, 2000 masked queries of 64-value heads 90.9 us
    // and 88.0)
    if (row_ok) put_row<TQ, DC / 32>(a, p, row_out<PREFIX>(a, p, row, bh, split), o, m, l);
    if (again) redo_rows<TK, TQ, DC, PREFIX>(a, p, row0, again, bh, split, j_begin, j_end);
}

// the place of piece c (four values) of row r in a wave's stretch of LDS: permuted by the row, against bank conflicts
template <int DP> __device__ __forceinline__ int piece_at(int r, int c) { return (r * (DP / 4) + (c ^ (r & (DP / 4 - 1)))) * 16; }

// up to 32 rows that the waves hold parts of, each in its stretch of LDS (pieces of the rows, then the maxima and
// the sums): a thread a piece, so that a token's few rows are spread over all threads
template <typename TK, typename TQ, int DC, int WAVES, bool PREFIX>
__device__ __forceinline__ void join_waves(const AttnArgs &a, const AttnPart &p, const char *lds, int stretch, int tops, int row0, int bh,
                                           int split, int j_begin, int j_end) {
    constexpr int DP = row_place(DC), PIECES = DP / 4, AT_ONCE = WAVES * 64 / PIECES;   // of a row; rows
    const int lane = threadIdx.x & 63, c = threadIdx.x % PIECES, n = min(32, p.rows - row0);
    uint32_t bad_rows = 0;
    for (int r0 = 0; r0 < n; r0 += AT_ONCE) {
        const int r = r0 + threadIdx.x / PIECES, row = row0 + min(r, n - 1);
        const bool ok = r < n;
        float m = -INFINITY, l = 0.0f;
        f32x4 x{};
        if (ok) {
            float mw[WAVES];
            f32x4 xw[WAVES];
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                mw[w] = reinterpret_cast<const float *>(lds + w * stretch + tops)[r];
                xw[w] = *reinterpret_cast<const f32x4 *>(lds + w * stretch + piece_at<DP>(r, c));
                m = fmaxf(m, mw[w]);
            }
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const float f = m == -INFINITY ? 1.0f : exp2f(mw[w] - m);
                l += reinterpret_cast<const float *>(lds + w * stretch + tops)[32 + r] * f;
                x += xw[w] * f;
            }
        }
        // a row's threads are neighbours in one wave: any of their votes counts
        const float all = (x[0] + x[1]) + (x[2] + x[3]) + l;
        uint64_t again = __ballot(ok && 4 * c < a.D && all != all);
        if (again) {
#pragma unroll
            for (int sft = 1; sft < PIECES; sft <<= 1) again |= again >> sft;
            uint64_t firsts = 0;
#pragma unroll
            for (int t = 0; t < 64; t += PIECES) firsts |= 1ull << t;
            again &= firsts;
        }
        if (ok && 4 * c < a.D && !(again >> (lane / PIECES * PIECES) & 1)) {
            const RowOut w = row_out<PREFIX>(a, p, row, bh, split);
            if (p.part_o) {
                if (c == 0) {
                    p.part_ml[2 * w.slot] = m;
                    p.part_ml[2 * w.slot + 1] = l;
                }
                *reinterpret_cast<f32x4 *>(p.part_o + w.slot * a.D + 4 * c) = x;
            } else {
                TQ *out = reinterpret_cast<TQ *>(a.o + w.i * a.o_i + w.head * a.o_h + w.b * a.o_b);
                store4<TQ>(out + 4 * c, x * finish(a, w.head, m, l));
            }
        }
        while (again) {
            const int at = __builtin_ctzll(again);
            again &= again - 1;
            bad_rows |= 1u << __builtin_amdgcn_readlane(r, at);
        }
    }
    if (bad_rows) redo_rows<TK, TQ, DC, PREFIX>(a, p, row0, bad_rows, bh, split, j_begin, j_end);
}

// the splits' partial results of a row, joined in a fixed order: GROUPS groups of DP / 4 threads a row take
// every GROUPS-th split
template <typename TQ, int DP, int GROUPS>
__global__ __launch_bounds__(256) void attn_join_kernel(const AttnArgs a, const AttnPart p) {
    constexpr int LPR = DP / 4, TPR = LPR * GROUPS, ROWS = 256 / TPR;
    __shared__ f32x4 part[ROWS][GROUPS == 1 ? 1 : GROUPS][GROUPS == 1 ? 1 : LPR];
    const int tid = threadIdx.x, row = tid / TPR, grp = tid % TPR / LPR, d = tid % LPR * 4;
    // rows lie by batch, key head, query, head of the group
    const int rows = a.B * a.H * a.n_q, rr = min((int)blockIdx.x * ROWS + row, rows - 1);
    const int G = (int)a.by_G.d, ri = a.by_G.of(rr), bhk = a.by_n_q.of(ri), b = a.by_Hk.of(bhk), i = ri - bhk * a.n_q;
    const int head = (bhk - b * a.Hk) * G + rr - ri * G;
    const float *po = p.part_o + (int64_t)rr * p.slots * a.D + d, *ml = p.part_ml + (int64_t)2 * rr * p.slots;
    const bool has = d < a.D;
    // (the first two of the thread's splits are on their way while the maximum forms)
    f32x4 x0{}, x1{};
    if (has && grp < p.slots) x0 = *reinterpret_cast<const f32x4 *>(po + (int64_t)grp * a.D);
    if (has && grp + GROUPS < p.slots) x1 = *reinterpret_cast<const f32x4 *>(po + (int64_t)(grp + GROUPS) * a.D);
    float m = -INFINITY, l = 0.0f;
    auto weight_of = [&](int s) { return m == -INFINITY ? 1.0f : exp2f(ml[2 * s] - m); };
    __shared__ float weights[GROUPS == 1 ? 1 : ATTN_MAX_SLOTS];
    if constexpr (GROUPS == 1) {   // a few splits
        for (int s = 0; s < p.slots; ++s) m = fmaxf(m, ml[2 * s]);
        for (int s = 0; s < p.slots; ++s) l += ml[2 * s + 1] * weight_of(s);
    } else {                       // one row a workgroup: every wave looks at all of them
        const int lane = tid & 63;
        for (int s = lane; s < p.slots; s += 64) m = fmaxf(m, ml[2 * s]);
#pragma unroll
        for (int s = 32; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor(m, s, 64));
        for (int s = lane; s < p.slots; s += 64) {
            const float f = weight_of(s);
            if (tid < 64) weights[s] = f;
            l += ml[2 * s + 1] * f;
        }
        l = wave_add(l);
        __syncthreads();
    }
    auto weight = [&](int s) { return GROUPS == 1 ? weight_of(s) : weights[s]; };
    f32x4 x{};
    if (grp < p.slots) x += x0 * weight(grp);
    if (grp + GROUPS < p.slots) x += x1 * weight(grp + GROUPS);
    if (has) {
#pragma unroll 4
        for (int s = grp + 2 * GROUPS; s < p.slots; s += GROUPS) x += *reinterpret_cast<const f32x4 *>(po + (int64_t)s * a.D) * weight(s);
    }
    if constexpr (GROUPS > 1) {
        part[row][grp][tid % LPR] = x;
        __syncthreads();
    }
    if (grp != 0 || !has || (int)blockIdx.x * ROWS + row >= rows) return;
#pragma unroll
    for (int g = 1; g < GROUPS; ++g) x += part[row][g][tid % LPR];   // (by the row's first group, in order)
    TQ *out = reinterpret_cast<TQ *>(a.o + i * a.o_i + head * a.o_h + b * a.o_b);
    store4<TQ>(out + d, x * finish(a, head, m, l));
}

// one round of pieces: LDS place `slot` (row slot / CPR, place slot % CPR) takes row `row` of the tensor's tile
__device__ __forceinline__ uint32_t piece_off(int place, int swz, int D) { return (uint32_t)(min(place ^ swz, D / 8 - 1) * 16); }

// a batch's own keys without a mask or a cap, with either; behind a shared prefix; the prefix (the last two
// have no mask, and may have a cap)
enum AttnKind { OWN, OWN_GENERAL, OWN_BEHIND, PREFIX_KEYS };

template <typename TK, typename TQ, int DC, int WAVES, bool BY_ROWS, AttnKind KIND, int TURNS>
__device__ __forceinline__ void attn_tiles(const AttnArgs &a, const AttnPart &p, char *lds, int id) {
    using T = AttnTile<TK, TQ, DC, WAVES, BY_ROWS, TURNS>;
    typedef typename T::x8 x8;
    constexpr bool SPLIT = T::SPLIT, PREFIX = KIND == PREFIX_KEYS;
    constexpr float BIAS = Vec<TK>::BIAS;
    constexpr int DP = T::DP, KT = T::KT, CPR = T::CPR, RPD = T::RPD, ROUNDS = T::ROUNDS, BYTES = T::BYTES, NT = DC / 16, NB = DC / 32;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    // problem, row tile (the last ones first: with a causal rule they see the most keys), split of the keys
    const int bh = p.by_bh.rest(id), at = p.by_bh.of(id), behind = p.by_split.of(at);
    const int split = at - behind * (int)p.by_split.d, tile = p.row_tiles - 1 - behind;
    const int G = (int)a.by_G.d, pb = a.by_Hk.of(bh), hk = bh - pb * a.Hk;

    // this lane's row (TURNS groups of RW waves have the same rows, and take turns at the tiles of keys)
    constexpr int RW = WAVES / TURNS;
    const int turn = BY_ROWS ? wave / RW : 0, rwave = BY_ROWS ? wave % RW : wave;
    const int row0 = (BY_ROWS ? tile * RW + rwave : tile) * 32;
    const int row = min(row0 + (lane & 31), p.rows - 1);
    const bool row_ok = row0 + (lane & 31) < p.rows;
    const int bi = a.by_G.of(row), head = hk * G + row - bi * G;
    const int b = PREFIX ? a.by_n_q.of(bi) : pb, i = PREFIX ? bi - b * a.n_q : bi;

    // queries: lane (row, h) holds values 16 t + 8 h .. + 7 of its row. They are asked for before anything that waits for
    // the batch's length, and the first tile's DMA follows; one wait covers both (the compiler, which knows of
    // the queries only, would otherwise wait inside the loop, and there for the tile ahead too)
    x8 qf[NT], ql[SPLIT ? NT : 1];
    f32x4 qx[SPLIT ? 2 * NT : 1];
    {
        const char *qr = a.q + i * a.q_i + head * a.q_h + b * a.q_b;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int d = 16 * t + 8 * h;
            if constexpr (SPLIT) {
                qx[2 * t] = qx[2 * t + 1] = f32x4{};
                if (d < a.D && row_ok) {
                    qx[2 * t] = *reinterpret_cast<const f32x4 *>(qr + 4 * d);
                    qx[2 * t + 1] = *reinterpret_cast<const f32x4 *>(qr + 4 * d + 16);
                }
            } else {
                x8 z{};
                qf[t] = d < a.D && row_ok ? *reinterpret_cast<const x8 *>(qr + 2 * d) : z;
            }
        }
    }
    __builtin_amdgcn_sched_barrier(0);

    // keys of this split, and how many of them the lane's row sees
    const int n = PREFIX ? a.n_prefix : own_len(a, b);
    int end = n;                                    // of the workgroup's rows
    if (!PREFIX && a.causal) {
        const int last = min((BY_ROWS ? (tile + 1) * RW : tile + 1) * 32 - 1, p.rows - 1);
        end = max(0, n - a.n_q + a.by_G.of(last) + 1);
    }
    int j_begin = 0, j_end = end;
    if (p.by_split.d > 1) {
        const int per = (p.by_split.of(end + (int)p.by_split.d - 1) + T::STEP - 1) / T::STEP * T::STEP;
        j_begin = min(end, split * per);
        j_end = min(end, j_begin + per);
    }
    j_begin = __builtin_amdgcn_readfirstlane(j_begin);
    j_end = __builtin_amdgcn_readfirstlane(j_end);
    const int seen = min(j_end, !PREFIX && a.causal ? n - a.n_q + i + 1 : n);

    const bool masked = KIND == OWN_GENERAL && a.mask != nullptr;
    const char *mrow = nullptr;
    float slope = 0.0f;
    if (masked) {
        mrow = a.mask + i * a.m_i + (head % a.m_nh) * a.m_h + (b % a.m_nb) * a.m_b;
        // (above 0, so that -inf stays -inf; a hidden key whose product is not finite makes the row NaN, and the
        // row is done again)
        slope = fmaxf(slope_of(a, head) * LOG2E, 0x1p-100f);
    }

    const char *kb = PREFIX ? a.kp + hk * a.kp_h : a.k + hk * a.k_h + (int64_t)a.by_kv_b.of(pb) * a.k_b;
    const char *vb = PREFIX ? a.vp + hk * a.vp_h : a.v + hk * a.v_h + (int64_t)a.by_kv_b.of(pb) * a.v_b;
    const int64_t k_j = PREFIX ? a.kp_j : a.k_j, v_j = PREFIX ? a.vp_j : a.v_j;

    // the tile at key j into `dst`, this wave's (BY_ROWS: the workgroup's) LDS
    // (its waves take ROUNDS pieces of RPD rows each)
    const int lrow = lane / CPR, place = lane % CPR, first = BY_ROWS ? rwave * ROUNDS : 0;
    char *stage0 = lds + (BY_ROWS ? turn : wave) * T::STRETCH;
    const uint32_t k_row = lrow * (uint32_t)k_j, v_row = lrow * (uint32_t)v_j;
    auto load = [&](const char *base, int64_t stride, uint32_t row0, int j, char *dst, auto swz) {
        const char *to = dst + first * 1024;
        const i32x4 buf = buffer_at(base + j * stride);
        const uint32_t step = (uint32_t)stride;
        const int last = j_end - 1 - j;
        if (last >= KT - 1) {
#pragma unroll
            for (int u = 0; u < ROUNDS; ++u)
                dma16(u, buf, to, row0 + piece_off(place, swz((first + u) * RPD + lrow), a.D), (uint32_t)((first + u) * RPD) * step);
        } else {   // rows behind the keys: the last key again
#pragma unroll
            for (int u = 0; u < ROUNDS; ++u) {
                const int r = (first + u) * RPD + lrow;
                dma16(u, buf, to, (uint32_t)min(r, last) * step + piece_off(place, swz(r), a.D), 0);
            }
        }
    };
    auto load_k = [&](int j, char *dst) { load(kb, k_j, k_row, j, dst, [](int r) { return swz_k<DP>(r); }); };
    auto load_v = [&](int j, char *dst) { load(vb, v_j, v_row, j, dst, [](int r) { return swz_v<DP>(r); }); };

    const int j0 = j_begin + (BY_ROWS ? turn * KT : wave * 32);
    if (j0 < j_end) {
        load_k(j0, stage0);
        load_v(j0, stage0 + BYTES);
    }

    float c = a.scale;
    if constexpr (SPLIT) {
        float top = 0.0f;
#pragma unroll
        for (int t = 0; t < 2 * NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(qx[t][e]));
        const bool infinite = __any(top == INFINITY);   // (hardly ever)
        if (infinite) {
            top = 0.0f;
#pragma unroll
            for (int t = 0; t < 2 * NT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) top = fmaxf(top, size_of(qx[t][e]));
        }
        top = fmaxf(top, swap32_f(top));
        const int up = shift_of(top);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = ldexpf(qx[2 * t + e / 4][e % 4], up);
                qf[t][e] = (_Float16)x;
                ql[t][e] = (_Float16)(x - (float)qf[t][e]);
            }
        if (infinite) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 8; ++e) ql[t][e] = fabsf((float)qf[t][e]) < INFINITY ? ql[t][e] : (_Float16)0.0f;
        }
        c = ldexpf(c, -up);
    }
    const bool capped = KIND != OWN && a.cap != 0.0f;
    const float cap2 = a.cap * LOG2E;
    // the maximum is taken of the bare products, so their factor must be above 0: its sign goes into
    // the queries, and for 0 a factor that leaves nothing of any product
    if (c < 0.0f) {
        c = -c;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            qf[t] = -qf[t];
            if constexpr (SPLIT) ql[t] = -ql[t];
        }
    }
    if constexpr (std::is_same<TK, __bf16>::value) {
        // (bf16 products reach 2^128: beside such a factor 2^64 of it goes over to it; a query that this brings below
        // bf16's range is below 2^-62, and its products times the factor below 2^-34)
        if (c < 0x1p-100f) {
            c *= 0x1p64f;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 8; ++e) qf[t][e] = (TK)((float)qf[t][e] * 0x1p-64f);
        }
    }
    const float c_cap = capped ? c / a.cap : 0.0f;
    c = fmaxf(c * LOG2E, 0x1p-126f);
    // a mask alone joins the bare products, by the slope over their factor, where that is no extreme number
    const bool scaled = capped || (masked && __any(!(c > 0x1p-60f && c < 0x1p20f)));
    if (masked && !scaled) slope /= c;
    __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0)

    f32x16 o[NB];
#pragma unroll
    for (int d = 0; d < NB; ++d) o[d] = f32x16{};
    float m = -INFINITY, l = 0.0f;   // (l: of the lane's own keys)

    // the mask's values at the tile's keys, 8 in a row from one load: half the cache lines that 4 at a time ask for
    // (rows of a mask begin at any multiple of 2 bytes; the card's loads may)
    auto fetch = [&](int j, f16x8 (&w)[KT / 16]) {
        typedef f16x8 f16x8_any __attribute__((aligned(2)));
        const _Float16 *mp = reinterpret_cast<const _Float16 *>(mrow) + j + 8 * h;
        if (__all(seen - j >= KT)) {
#pragma unroll
            for (int r = 0; r < KT / 16; ++r) w[r] = *reinterpret_cast<const f16x8_any *>(mp + 16 * r);
        } else {
            const int left = seen - j - 8 * h;
#pragma unroll
            for (int r = 0; r < KT / 16; ++r)
#pragma unroll
                for (int e = 0; e < 8; ++e) w[r][e] = 16 * r + e < left ? mp[16 * r + e] : (_Float16)-INFINITY;
        }
    };
    // and in the order of the scores: the row's two lanes trade halves
    auto arrange = [&](const f16x8 (&from)[KT / 16], f16x4 (&w)[KT / 8]) {
        typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
        typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int r = 0; r < KT / 16; ++r) {
            const u32x4 x = __builtin_bit_cast(u32x4, from[r]);
            const auto a0 = __builtin_amdgcn_permlane32_swap(x[0], x[2], false, false), a1 = __builtin_amdgcn_permlane32_swap(x[1], x[3], false, false);
            w[2 * r] = __builtin_bit_cast(f16x4, u32x2{a0[0], a1[0]});
            w[2 * r + 1] = __builtin_bit_cast(f16x4, u32x2{a0[1], a1[1]});
        }
#pragma unroll
        for (int r = 0; r < KT / 8; ++r) asm volatile("" : "+v"(w[r]));   // here, behind the loads' wait and before the next DMA
    };

    // whether the mask hides the tile from all of the wave's rows
    auto hidden = [&](const f16x4 (&w)[KT / 8]) {
        typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
        if (!__all(__builtin_bit_cast(u32x2, w[0])[0] == 0xfc00fc00u)) return false;   // (most tiles end here)
        uint32_t other = 0;
#pragma unroll
        for (int r = 0; r < KT / 8; ++r) {
            const u32x2 v = __builtin_bit_cast(u32x2, w[r]);
            other |= (v[0] ^ 0xfc00fc00u) | (v[1] ^ 0xfc00fc00u);
        }
        return __all(other == 0) != 0;
    };

    // LDS reads run AHEAD operands ahead of the MFMAs that take them: left to itself the compiler, short of
    // registers, reads each operand right before its use
    constexpr int AHEAD = 4, PER = SPLIT ? 2 : 1;   // (MFMAs an operand)
    f32x16 s[KT / 32];
    auto products = [&](const char *kt) {
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
        __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
        for (int n = AHEAD; n < KT / 32 * NT; ++n) {
            __builtin_amdgcn_sched_group_barrier(0x008, PER, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, PER * AHEAD, 0);
    };
    // the same with the next tile's DMA (a whole one, into `to`) dealt out among the MFMAs: issued in a row it holds a
    // wave up for hundreds of cycles, a tenth of a tile's time
    auto products_and_load = [&](const char *kt, int j, char *to) {
        constexpr int NQK = KT / 32 * NT, EVERY = NQK / (2 * ROUNDS) > 0 ? NQK / (2 * ROUNDS) : 1;
        static_assert(!BY_ROWS || 2 * ROUNDS * EVERY <= NQK, "every DMA has its step");
        const int krow = lane & 31, ksw = swz_k<DP>(krow);
        const i32x4 kbuf = buffer_at(kb + j * k_j), vbuf = buffer_at(vb + j * v_j);
        auto read = [&](int n) { return *reinterpret_cast<const x8 *>(kt + (n / NT * 32 + krow) * DP * 2 + (((2 * (n % NT) + h) ^ ksw) * 16)); };
        x8 kf[AHEAD];
#pragma unroll
        for (int n = 0; n < AHEAD; ++n) kf[n] = read(n);
#pragma unroll
        for (int n = 0; n < NQK; ++n) {
            __builtin_amdgcn_sched_barrier(0);
            const f32x16 from = n % NT == 0 ? f32x16{} : s[n / NT];
            s[n / NT] = mma(kf[n % AHEAD], qf[n % NT], from);
            if constexpr (SPLIT) s[n / NT] = mma(kf[n % AHEAD], ql[n % NT], s[n / NT]);
            if (n + AHEAD < NQK) kf[n % AHEAD] = read(n + AHEAD);
            if (n % EVERY == 0 && n / EVERY < 2 * ROUNDS) {
                const int u = n / EVERY % ROUNDS, r = (first + u) * RPD + lrow;
                const uint32_t rows = (uint32_t)((first + u) * RPD);
                if (n / EVERY < ROUNDS) dma16(u, kbuf, to + first * 1024, k_row + piece_off(place, swz_k<DP>(r), a.D), rows * (uint32_t)k_j);
                else dma16(u, vbuf, to + BYTES + first * 1024, v_row + piece_off(place, swz_v<DP>(r), a.D), rows * (uint32_t)v_j);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    // the weights of the tile's keys from their products: s[u][r] belongs to key j + 32 u + 8 (r / 4) + 4 h +
    // r % 4, f times it is the score in units of log 2
    auto weights = [&](int j, const f16x4 (&w)[KT / 8]) {
        const int left = seen - j - 4 * h;
        float f = c;
        if (scaled) {
            const float by = capped ? c_cap : c;
            f = 1.0f;
#pragma unroll
            for (int u = 0; u < KT / 32; ++u)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[u][r] *= by;
        }
        if (capped) {
#pragma unroll
            for (int u = 0; u < KT / 32; ++u)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[u][r] = cap2 * tanh_of(s[u][r]);
        }
        if (masked) {
#pragma unroll
            for (int u = 0; u < KT / 32; ++u)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[u][r] = fmaf(slope, (float)w[4 * u + r / 4][r % 4], s[u][r]);
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
    };
    // (-1 that the compiler does not see: a second term is then one mixed fma, not a conversion, a difference and
    // another conversion)
    // Weights of 16-bit activations are two terms as well where the waves split the keys: bound by memory, the second
    // product costs next to nothing (64 x 8192 f16 keys of 8 heads of 128 values 303 and 302 us, of 64 values 201 and
    // 203), and the result is off by its own rounding alone, rms 2.1e-4 of it, with rounded weights 2.9e-4 (bf16 1.6e-3,
    // 2.3e-3). Row tiles round them: two terms take 8192 causal tokens from 513 to 681 us, 64 sequences behind 8192
    // shared keys from 36 to 39.
    constexpr bool TWO = SPLIT || !BY_ROWS;
    constexpr int PV = TWO ? 2 : 1;
    float minus = -1.0f;
    asm("" : "+s"(minus));
    auto values = [&](const char *vt) {
        // O^T += V^T P^T, 16 keys a step: the lane's weights 8 (t % 2) .. + 7 of block t / 2
        const int vi = lane & 15, vrow = 4 * h + (vi >> 2), vch = 2 * ((lane >> 4) & 1) + ((vi & 3) >> 1), vsw = swz_v<DP>(vrow);
#pragma unroll
        for (int t = 0; t < KT / 16; ++t) {
            x8 pf, pl;
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                typedef float f32x2 __attribute__((ext_vector_type(2)));
                typedef TK x2 __attribute__((ext_vector_type(2)));
                const f32x2 x = {s[t / 2][8 * (t % 2) + e], s[t / 2][8 * (t % 2) + e + 1]};
                const x2 hi = __builtin_convertvector(x, x2);
                pf[e] = hi[0];
                pf[e + 1] = hi[1];
                if constexpr (TWO) {
                    pl[e] = (TK)fmaf(minus, (float)hi[0], x[0]);
                    pl[e + 1] = (TK)fmaf(minus, (float)hi[1], x[1]);
                }
            }
#pragma unroll
            for (int d = 0; d < NB; ++d) {
                const char *vp = vt + (16 * t + vrow) * DP * 2 + (((4 * d + vch) ^ vsw) * 16) + 8 * (vi & 1);
                const i16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4 *)vp);
                const i16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4 *)(vp + 8 * DP * 2));
                const i16x8 vv = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
                const x8 vf = __builtin_bit_cast(x8, vv);
                o[d] = mma(vf, pf, o[d]);
                if constexpr (TWO) o[d] = mma(vf, pl, o[d]);
            }
        }
        __builtin_amdgcn_sched_group_barrier(0x100, 2 * AHEAD, 1);
#pragma unroll
        for (int n = AHEAD; n < KT / 16 * NB; ++n) {
            __builtin_amdgcn_sched_group_barrier(0x008, PV, 1);
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, PV * AHEAD, 1);
    };

    if constexpr (BY_ROWS) {
        // (a later row sees no fewer keys)
        const int seen_most = row0 < p.rows ? __builtin_amdgcn_readlane(seen, 31) : 0;
        f16x4 w[KT / 8];
        f16x8 ahead[KT / 16];
        if (masked && j0 < j_end) fetch(j0, ahead);
        char *now = stage0, *next = stage0 + 2 * BYTES;
        for (int j = j0; j - turn * KT < j_end; j += T::STEP) {   // (as often for every wave)
            // this wave's share of the tile has come; behind the barrier everyone's has, and the other stage is read
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (masked) arrange(ahead, w);
            // (8 waves that share a tile have half the DMA each, and lose 3 % by dealing it out, as do loads of a mask before
            // it; but a wave alone on its SIMD gains 11 % with a mask too)
            const bool mine = j < seen_most && !(masked && hidden(w)), among = RW == 4 && !(masked && DP < 256) && mine && j + T::STEP + KT <= j_end;
            if (j + T::STEP < j_end && !among) {
                load_k(j + T::STEP, next);
                load_v(j + T::STEP, next + BYTES);
            }
            if (masked && j + T::STEP < j_end) fetch(j + T::STEP, ahead);
            if (mine) {
                // (a wave that feeds the matrix cores goes before one that forms weights)
                __builtin_amdgcn_s_setprio(1);
                if (among) products_and_load(now, j + T::STEP, next);
                else products(now);
                __builtin_amdgcn_s_setprio(0);
                weights(j, w);
                __builtin_amdgcn_s_setprio(1);
                values(now + BYTES);
                __builtin_amdgcn_s_setprio(0);
            }
            char *t = now;
            now = next;
            next = t;
        }
    } else {
        // a tile's keys are refilled once their products are formed, its values behind those, so that either
        // is on its way while the other is worked on
        constexpr int STEP = T::STEP;
        f16x4 w[KT / 8];
        f16x8 ahead[KT / 16];
        if (masked && j0 < j_end) fetch(j0, ahead);
        for (int j = j0; j < j_end; j += STEP) {
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(ROUNDS) : "memory");   // the keys
            if (masked) {
                arrange(ahead, w);
                if (j + STEP < j_end) fetch(j + STEP, ahead);
            }
            const bool idle = masked && hidden(w);
            if (!idle) products(stage0);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (j + STEP < j_end) load_k(j + STEP, stage0);
            if (!idle) weights(j, w);
            if (j + STEP < j_end) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(ROUNDS) : "memory");   // the values
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if (!idle) values(stage0 + BYTES);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (j + STEP < j_end) load_v(j + STEP, stage0 + BYTES);
        }
    }
    l += swap32_f(l);

    if constexpr (!BY_ROWS) {
        // join the waves: each leaves its rows in its own stretch
        asm volatile("" ::: "memory");
        if (row_ok) {
            float *pm = reinterpret_cast<float *>(stage0 + 2 * BYTES);
#pragma unroll
            for (int d = 0; d < NB; ++d)
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4)
                    *reinterpret_cast<f32x4 *>(stage0 + piece_at<DP>(lane & 31, 8 * d + 2 * r4 + h)) =
                        f32x4{o[d][4 * r4], o[d][4 * r4 + 1], o[d][4 * r4 + 2], o[d][4 * r4 + 3]};
            if (h == 0) {
                pm[lane] = m - BIAS;   // (-inf: no key)
                pm[32 + lane] = l;
            }
        }
        __syncthreads();
        join_waves<TK, TQ, DC, WAVES, PREFIX>(a, p, lds, T::STRETCH, 2 * BYTES, row0, bh, split, j_begin, j_end);
    } else {
        if constexpr (TURNS > 1) {
            // the second group leaves its part to the first one, in LDS that no DMA is on its way to: the rows' maxima
            // and sums, and its accumulators in order of the lanes
            static_assert(TURNS == 2 && RW * (NB * 4096 + 512) <= T::LDS, "a wave's accumulators, maxima and sums");
            char *mine = lds + rwave * (NB * 4096 + 512);
            __syncthreads();
            if (turn == 1) {
                float *ml = reinterpret_cast<float *>(mine + NB * 4096);
                ml[lane] = m;
                ml[64 + lane] = l;
#pragma unroll
                for (int d = 0; d < NB; ++d)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        reinterpret_cast<f32x4 *>(mine)[(4 * d + r) * 64 + lane] = f32x4{o[d][4 * r], o[d][4 * r + 1], o[d][4 * r + 2], o[d][4 * r + 3]};
            }
            __syncthreads();
            if (turn == 1) return;
            const float *ml = reinterpret_cast<const float *>(mine + NB * 4096);
            const float m1 = ml[lane], top = fmaxf(m, m1);
            const float f0 = m == top ? 1.0f : exp2f(m - top), f1 = m1 == top ? 1.0f : exp2f(m1 - top);
            l = l * f0 + ml[64 + lane] * f1;
#pragma unroll
            for (int d = 0; d < NB; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const f32x4 x = reinterpret_cast<const f32x4 *>(mine)[(4 * d + r) * 64 + lane];
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[d][4 * r + e] = o[d][4 * r + e] * f0 + x[e] * f1;
                }
            m = top;
        }
        store_rows<TK, TQ, DC, PREFIX>(a, p, o, m - BIAS, l, row0, row, row_ok, bh, split, j_begin, j_end);
    }
}

// One launch: the workgroups of a shared prefix (PRE: 0 none, 1 split keys, 2 row tiles), which are bound
// by the matrix cores, then those of the batches' own keys, bound by memory, on the same CUs. 8 waves on a
// CU: two workgroups of 4, which take turns at the matrix cores, or one of 8, which loads each tile of keys
// for twice the rows, or (TURNS = 2) whose halves have the same rows, work on two tiles of keys and join what they have
// in LDS: half the splits, or none, where row tiles are few. 4 where the largest heads' accumulators leave room for
// no more. Causal heads of 128 values, 32 on 8, 2048 tokens: 60 us by 4 waves, 61 by 8, 50 in turns; 8192: 547, 533, 588.
template <typename TK, typename TQ, int DC, int WAVES, int PRE, bool OWN_ROWS, bool GENERAL, int TURNS>
__global__ __launch_bounds__(WAVES * 64, DC == 256 || (DC == 192 && sizeof(TQ) == 4) ? 1 : 2) void attn_tile_kernel(const AttnArgs a, const AttnPart pre, const AttnPart own) {
    constexpr int L0 = AttnTile<TK, TQ, DC, WAVES, OWN_ROWS, TURNS>::LDS, L1 = AttnTile<TK, TQ, DC, WAVES, PRE == 2>::LDS;
    __shared__ __align__(16) char lds[PRE && L1 > L0 ? L1 : L0];
    if constexpr (PRE != 0) {
        if ((int)blockIdx.x < pre.blocks) {
            attn_tiles<TK, TQ, DC, WAVES, PRE == 2, PREFIX_KEYS, 1>(a, pre, lds, blockIdx.x);
            return;
        }
    }
    attn_tiles<TK, TQ, DC, WAVES, OWN_ROWS, PRE ? OWN_BEHIND : GENERAL ? OWN_GENERAL : OWN, TURNS>(a, own, lds, blockIdx.x - (PRE ? pre.blocks : 0));
}

template <typename TK, typename TQ, int DC>
static void launch_attn(const AttnArgs &a, const AttnPlan &pl, void *work, hipStream_t st) {
    const int G = (int)a.by_G.d;
    AttnPart own{}, pre{};
    own.slots = pl.slots;
    if (pl.slots > 1) {
        own.part_o = static_cast<float *>(work);
        own.part_ml = own.part_o + (size_t)a.B * a.H * a.n_q * pl.slots * a.D;
    }
    pre = own;
    if (pl.pre_splits) {
        pre.by_split = Div((uint32_t)pl.pre_splits);
        pre.by_bh = Div((uint32_t)a.Hk);
        pre.rows = a.B * a.n_q * G;
        pre.row_tiles = pl.pre_tiles;
        pre.blocks = a.Hk * pre.row_tiles * pl.pre_splits;
    }
    own.slot0 = pl.pre_splits;
    own.by_split = Div((uint32_t)pl.own_splits);
    own.by_bh = Div((uint32_t)(a.B * a.Hk));
    own.rows = a.n_q * G;
    own.row_tiles = pl.own_tiles;
    own.blocks = a.B * a.Hk * own.row_tiles * pl.own_splits;
    const bool general = a.mask != nullptr || a.cap != 0.0f;
    const dim3 grid((unsigned)(pre.blocks + own.blocks));
    constexpr int DP = row_place(DC), WIDE = DP == 256 ? 4 : 8;
#define ATTN_CASE(WAVES, PRE, ROWS, GENERAL, TURNS) \
    hipLaunchKernelGGL((attn_tile_kernel<TK, TQ, DC, WAVES, PRE, ROWS, GENERAL, TURNS>), grid, dim3(WAVES * 64), 0, st, a, pre, own)
    if (pl.pre_splits) {
        if (!pl.pre_rows) ATTN_CASE(4, 1, false, false, 1);
        else if (!pl.own_rows) ATTN_CASE(4, 2, false, false, 1);
        else ATTN_CASE(WIDE, 2, true, false, 1);
    } else if (pl.waves == 4) {
        if (pl.own_rows && general) ATTN_CASE(4, 0, true, true, 1);
        else if (pl.own_rows) ATTN_CASE(4, 0, true, false, 1);
        else if (general) ATTN_CASE(4, 0, false, true, 1);
        else ATTN_CASE(4, 0, false, false, 1);
    } else if (pl.turns == 2) {
        if (general) ATTN_CASE(WIDE, 0, true, true, WIDE / 4);
        else ATTN_CASE(WIDE, 0, true, false, WIDE / 4);
    } else {
        if (general) ATTN_CASE(WIDE, 0, true, true, 1);
        else ATTN_CASE(WIDE, 0, true, false, 1);
    }
#undef ATTN_CASE
    if (pl.slots > 1) {
        // a workgroup a row, its splits side by side, where rows are few; one group of threads a row where it has a
        // few splits and the rows fill the CUs by themselves (6400 rows of 4 splits: 11.6 us and 5.7)
        const int64_t rows = (int64_t)a.B * a.H * a.n_q;
        constexpr int ALL = 1024 / DP;
        if (pl.slots <= 2 || (pl.slots <= 8 && rows >= 2048)) {
            const unsigned grid = (unsigned)((rows * (DP / 4) + 255) / 256);
            hipLaunchKernelGGL((attn_join_kernel<TQ, DP, 1>), dim3(grid), dim3(256), 0, st, a, own);
        } else {
            hipLaunchKernelGGL((attn_join_kernel<TQ, DP, ALL>), dim3((unsigned)rows), dim3(256), 0, st, a, own);
        }
    }
}

template <typename TK, typename TQ, int DC>
static hipError_t launch_attn_any(const AttnArgs &a, const AttnPlan &pl, void *work, hipStream_t st) {
    if (pl.tiled) launch_attn<TK, TQ, DC>(a, pl, work, st);
    else hipLaunchKernelGGL((attn_rows_kernel<TQ, TK>), dim3(a.n_q, a.H, a.B), dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace

}  // namespace mi355x
