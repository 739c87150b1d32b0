// hrs_attention: o_i = sum_j softmax_j(f(scale q_i . k_j) + bias(j - p_i)) v_j over the keys j that query i sees.
//
// Documents lie back to back (offsets) or in padded rows (lengths); a query sees keys of its own document only.  With
// p_i = i + lk - lq (the last query stands at the last key), causal order and a prefix that everyone sees both come down
// to one number per query: it sees j < lim_i, lim_i = max(p_i + 1, prefix) cut to [0, lk], or lk without causal order.
// f caps scores, f(s) = cap tanh(s / cap); bias is -slope_h |j - p_i| or a row of a table clamped at +-reach.
//
// The query heads that share a key head are rows of one matrix: row r of a document is token r / G, head r % G (G = query
// heads per key head), so one pass over the keys serves all of them and a single token still fills G rows.
//
// One pass over the keys with the running maximum m and sum l of every row (all in base 2: scores are multiplied by
// log2 e once).  S^T = K Q^T puts the query on the lane: maximum and sum are in-lane, with one exchange between the
// wave's halves.  The accumulator of S^T leaves a lane with keys 8 g + 4 h .. + 3 (g = 0 .. 3) of 32; as the second
// operand of O^T = V^T P^T its register order defines the order of the contraction, and V's operand is read in that same
// order with transposing LDS reads, so the weights never change lanes.
#include "hrs_ops.h"

struct AttnArgs {
    const void *q, *k, *v;
    void* out;
    const int32_t *q_offs, *k_offs, *q_lens, *k_lens, *prefix;
    const float *slopes, *table;
    int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh;  // strides in elements: document, token, head
    int64_t q_rows, k_rows;  // tokens per document, or of all documents where offsets are given
    int batch, heads, kv_heads, group, dim, tiles;
    int b0;  // first document of this launch
    int causal, reach;
    float scale2;        // scale log2 e
    float cap2, cap_in, cap_u;  // cap log2 e; 2 log2 e scale / cap; scale / cap
    // long documents: `chunk` keys per workgroup, unnormalised sums [chunks][rows][dim] and (m, l) [chunks][rows]
    int chunk, chunks;
    int64_t part_rows;
    float* part;
    float2* part_ml;
};

enum { BIAS_NONE = 0, BIAS_SLOPE = 1, BIAS_TABLE = 2 };
#define LOG2E 1.44269504088896f
#define TABLE_EDGE 96  // 64 keys of a tile and 32 rows of a wave

struct DocRange {
    int64_t q0, k0;  // first token, from the start of the tensor
    int lq, lk, q_total;
};
__device__ __forceinline__ int64_t clamp64(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : v > hi ? hi : v; }
// Lengths and offsets are cut to the tensors they point into: whatever they hold, nothing outside is read or written.
__device__ __forceinline__ DocRange doc_range(const AttnArgs& a, int b) {
    DocRange d;
    if (a.q_offs) {
        d.q0 = clamp64(a.q_offs[b], 0, a.q_rows);
        d.lq = (int)(clamp64(a.q_offs[b + 1], d.q0, a.q_rows) - d.q0);
        d.q_total = d.lq;
    } else {
        d.q0 = 0;
        d.q_total = (int)a.q_rows;
        d.lq = d.q_total;
    }
    if (a.q_lens) d.lq = (int)clamp64(a.q_lens[b], 0, d.lq);
    if (a.k_offs) {
        d.k0 = clamp64(a.k_offs[b], 0, a.k_rows);
        d.lk = (int)(clamp64(a.k_offs[b + 1], d.k0, a.k_rows) - d.k0);
    } else {
        d.k0 = 0;
        d.lk = (int)a.k_rows;
    }
    if (a.k_lens) d.lk = (int)clamp64(a.k_lens[b], 0, d.lk);
    return d;
}

// Piece p of row i lies at piece p ^ swizzle of its row of DP elements.  K: 8 consecutive rows, same piece -> 8 bank groups.
// V: 4 consecutive rows, two pieces -> 8 bank groups.
template <int DP>
__device__ __forceinline__ int swizzle_k(int i) { return DP == 32 ? (i >> 1) & 3 : i & 7; }
template <int DP>
__device__ __forceinline__ int swizzle_v(int i) { return DP == 32 ? i & 2 : (i & 3) << 1; }

typedef short s16x4 __attribute__((ext_vector_type(4)));
// Four rows of 16 elements, one row per four lanes (each lane names 8 bytes); lane l of 16 receives column l of the four.
__device__ __forceinline__ s16x4 lds_read_tr(const char* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
}

__device__ __forceinline__ float swap_halves(float v) {
    const unsigned u = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

// cap tanh(scale s / cap) in base 2.  tanh u = 1 - 2 / (1 + e^2u) is off by 2^-22 or so of 1 whatever u is: up to a cap of
// 64 that is less than 2e-5 of a score.  Larger caps would lose small scores that way, so below |u| = 0.4 capped takes tanh's
// series up to u^11 (next term 3.6e-3 u^12 < 7e-8), above it the same quotient, there within 2^-21 of its result.  Kernels
// of their own (CAP_ANY), as a branch in the others it would cost them registers: two documents of 8192 tokens, 16 heads of
// 64: 1085 us with a cap of 100, 912 with 60; 8 tokens over 32768 keys, 32 / 8 heads of 128: 229 and 207.
enum { CAP_NONE = 0, CAP_TO_64 = 1, CAP_ANY = 2 };
#define CAP_DIRECT (64.f * LOG2E)
__device__ __forceinline__ float capped_direct(const AttnArgs& a, float s) { return fmaf(-2.f * a.cap2, rcp_hw(1.f + exp2_hw(s * a.cap_in)), a.cap2); }
__device__ __forceinline__ float capped(const AttnArgs& a, float s) {
    const float u = s * a.cap_u, t = u * u;
    float p = fmaf(t, -0.0088632355f, 0.0218694885f);
    p = fmaf(t, p, -0.0539682540f);
    p = fmaf(t, p, 0.1333333333f);
    p = fmaf(t, p, -0.3333333333f);
    p = fmaf(t, p, 1.f);
    return t < 0.16f ? s * a.scale2 * p : capped_direct(a, s);
}

// A table's entry in base 2.  A finite one stays finite, also the type's lowest and largest values (log2 e times them would
// be infinite): beyond +-1e30 entries count as they are.  NaN stays NaN.
__device__ __forceinline__ float table2(float t) {
    const float x = t * LOG2E;
    return fabsf(x) < 1e30f || t != t ? x : t < 0.f ? fminf(t, -1e30f) : fmaxf(t, 1e30f);
}

// Weights are 2^(x - base) up to a factor that cancels in the quotient.  In fp16, where 2^-25 rounds to nothing, the largest
// is put near the top of its range instead of at 1, or many keys of 2^-26 each would be mass lost (1.6 % for a million of them).
template <typename T>
constexpr float top_weight(float largest) { return __is_same(T, _Float16) ? 15.f - largest : 0.f; }

// Score of one (query, key) pair in base 2: s is q . k, d = j - p_i.
template <int BIAS, bool CAP>
__device__ __forceinline__ float score2(const AttnArgs& a, float s, float slope2, const float* table, int d) {
    float x = !CAP ? s * a.scale2 : a.cap2 > CAP_DIRECT ? capped(a, s) : capped_direct(a, s);
    if constexpr (BIAS == BIAS_SLOPE) x = fmaf(-slope2, fabsf((float)d), x);
    if constexpr (BIAS == BIAS_TABLE) {
        const int at = d < -a.reach ? -a.reach : d > a.reach ? a.reach : d;
        x += table2(table[at]);
    }
    return x;
}

// ---- any alignment, any table ------------------------------------------------------------------------
// 128 rows per workgroup, 32 per wave; pieces of K and V pass through registers one by one and the table is read from
// memory.  Two to four times slower than the kernels below (two documents of 8192 tokens, 16 heads of 64, slope: 1.57 ms
// against 0.74): the way for operands that cannot be fetched in aligned 16-byte pieces.
template <typename T, int DP, int BIAS, bool CAP>
__global__ __launch_bounds__(256) void k_attend_any(AttnArgs a) {
    typedef typename vec_of<T>::x8 x8;
    constexpr int KT = DP <= 128 ? 64 : 32, PPR = DP / 8, NB = KT / 32, ND = DP / 32, NS = DP / 16;
    __shared__ __attribute__((aligned(16))) char kl[KT * DP * 2];
    __shared__ __attribute__((aligned(16))) char vl[KT * DP * 2];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, h = lane >> 5, c32 = lane & 31;
    int id = blockIdx.x;
    const int t0 = id % a.tiles;
    id /= a.tiles;
    const int hk = id % a.kv_heads, b = a.b0 + id / a.kv_heads;
    const DocRange dr = doc_range(a, b);
    const int64_t rows = (int64_t)dr.lq * a.group, rows_all = (int64_t)dr.q_total * a.group;
    const T* kbase = (const T*)a.k + b * a.k_sb + dr.k0 * a.k_st + hk * a.k_sh;
    const T* vbase = (const T*)a.v + b * a.v_sb + dr.k0 * a.v_st + hk * a.v_sh;
    const int prefix = a.prefix ? a.prefix[b] : 0;

    for (int64_t row0 = (int64_t)t0 * 128; row0 < rows_all; row0 += (int64_t)a.tiles * 128) {
        const int64_t row = row0 + wv * 32 + c32;
        const bool live = row < rows;
        const int token = (int)(row / a.group), head = hk * a.group + (int)(row % a.group);
        const T* qp = (const T*)a.q + b * a.q_sb + (dr.q0 + token) * a.q_st + head * a.q_sh;
        x8 qf[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) qf[s] = load8_any<T>(qp + s * 16 + h * 8, live ? a.dim - (s * 16 + h * 8) : 0);
        const int pos = token + dr.lk - dr.lq;
        int lim = dr.lk;
        if (a.causal) {
            lim = pos + 1 > prefix ? pos + 1 : prefix;
            lim = lim < 0 ? 0 : lim > dr.lk ? dr.lk : lim;
        }
        if (!live) lim = 0;
        // keys that any row of the workgroup sees
        int64_t last = row0 + 127 < rows - 1 ? row0 + 127 : rows - 1;
        int need = dr.lk;
        if (a.causal) {
            const int p = (int)(last / a.group) + dr.lk - dr.lq + 1;
            need = p > prefix ? p : prefix;
            need = need > dr.lk ? dr.lk : need;
        }
        if (row0 >= rows) need = 0;
        const float slope2 = BIAS == BIAS_SLOPE && live ? a.slopes[head] * LOG2E : 0.f;
        const float* table = BIAS == BIAS_TABLE ? a.table + (int64_t)(live ? head : 0) * (2 * a.reach + 1) + a.reach : nullptr;

        f32x16 acc[ND];
#pragma unroll
        for (int i = 0; i < ND; ++i) acc[i] = (f32x16)(0.f);
        float m = -INFINITY, l = 0.f;
        for (int j0 = 0; j0 < need; j0 += KT) {
            __syncthreads();
            for (int id2 = tid; id2 < KT * PPR; id2 += 256) {
                const int i = id2 / PPR, p = id2 % PPR;
                const int64_t j = j0 + i;
                const int left = j < dr.lk ? a.dim - p * 8 : 0;  // what stands behind the document is never read: zeros
                *(x8*)(kl + i * (DP * 2) + (p ^ swizzle_k<DP>(i)) * 16) = load8_any<T>(kbase + j * a.k_st + p * 8, left);
                *(x8*)(vl + i * (DP * 2) + (p ^ swizzle_v<DP>(i)) * 16) = load8_any<T>(vbase + j * a.v_st + p * 8, left);
            }
            __syncthreads();
            f32x16 s[NB];
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                s[n] = (f32x16)(0.f);
                const int i = n * 32 + c32;
#pragma unroll
                for (int t = 0; t < NS; ++t) s[n] = mfma32(*(const x8*)(kl + i * (DP * 2) + ((2 * t + h) ^ swizzle_k<DP>(i)) * 16), qf[t], s[n]);
            }
            float top = -INFINITY;
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int j = j0 + n * 32 + 8 * (r >> 2) + 4 * h + (r & 3);
                    const float x = score2<BIAS, CAP>(a, s[n][r], slope2, table, j - pos);
                    s[n][r] = j < lim ? x : -INFINITY;
                    top = fmaxf(top, s[n][r]);
                }
            top = fmaxf(top, swap_halves(top));
            const float m_new = fmaxf(m, top);
            const float keep = exp2_hw(m - (m_new == -INFINITY ? 0.f : m_new));
            const float base = m_new == -INFINITY ? 0.f : m_new - top_weight<T>(0.f);  // nothing seen so far: every weight is exp2(-inf) = 0
            m = m_new;
#pragma unroll
            for (int i = 0; i < ND; ++i) acc[i] *= keep;
            x8 pf[2 * NB];
            float part = 0.f;  // (a tile's weights are summed before they meet the running sum, beside which single ones may be nothing)
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const T w = (T)exp2_hw(s[n][r] - base);
                    part += (float)w;  // (the rounded weight: numerator and denominator round alike)
                    pf[2 * n + (r >> 3)][r & 7] = w;
                }
            l = fmaf(l, keep, part);
            // step t: keys 16 t + 8 e + 4 h + (0 .. 3) of the tile, e = 0, 1
#pragma unroll
            for (int t = 0; t < 2 * NB; ++t)
#pragma unroll
                for (int i = 0; i < ND; ++i) {
                    union {
                        s16x4 half[2];
                        x8 all;
                    } vf;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int key = t * 16 + e * 8 + 4 * h + ((lane & 15) >> 2), col = i * 32 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
                        vf.half[e] = lds_read_tr(vl + key * (DP * 2) + ((col >> 3) ^ swizzle_v<DP>(key)) * 16 + (col & 7) * 2);
                    }
                    acc[i] = mfma32(vf.all, pf[t], acc[i]);
                }
        }
        l += swap_halves(l);
        const float inv = l > 0.f || l != l ? 1.f / l : 0.f;  // a row that sees nothing is zero; NaN stays NaN
        if (row < rows_all) {
            T* op = (T*)a.out + ((b * (a.q_offs ? 0 : a.q_rows) + dr.q0 + token) * a.heads + head) * a.dim;
#pragma unroll
            for (int i = 0; i < ND; ++i)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int d = i * 32 + g * 8 + h * 4;
                    if (d < a.dim) {
                        T o[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[e] = live ? (T)(acc[i][4 * g + e] * inv) : (T)0.f;
                        __builtin_memcpy(op + d, o, 8);
                    }
                }
        }
    }
}

// ---- aligned operands: K and V by LDS-DMA --------------------------------------------------------------
// A row of the tile and what it is allowed to see.
struct RowPlace {
    int row;  // row / group: token, row % group: head of this key head's group
    bool live;
    int token, head, pos, lim;
};
// (a division costs some 30 instructions even in 32 bits)
__device__ __forceinline__ int token_of(const AttnArgs& a, int row) { return a.group == 1 ? row : (int)((unsigned)row / (unsigned)a.group); }
__device__ __forceinline__ int limit_of(const AttnArgs& a, const DocRange& d, int pos, int prefix) {
    if (!a.causal) return d.lk;
    const int lim = pos + 1 > prefix ? pos + 1 : prefix;
    return lim < 0 ? 0 : lim > d.lk ? d.lk : lim;
}
__device__ __forceinline__ RowPlace row_place(const AttnArgs& a, const DocRange& d, int hk, int prefix, int row) {
    RowPlace r;
    r.row = row;
    r.live = row < d.lq * a.group;
    r.token = token_of(a, row);
    r.head = hk * a.group + (row - r.token * a.group);
    r.pos = r.token + d.lk - d.lq;
    r.lim = r.live ? limit_of(a, d, r.pos, prefix) : 0;
    return r;
}

// The state of one lane's row (query c = lane % 32 of the wave; the wave's halves hold different keys and dimensions).
template <typename T, int DP, int NB, int BIAS, int CAP, bool FIXED>
struct Attend {
    typedef typename vec_of<T>::x8 x8;
    static constexpr int ND = DP / 32, NS = DP / 16, KT = NB * 32;
    // With a slope the bias of a tile wholly before (or behind) all positions of the wave is linear in j: its part that
    // varies over the tile enters as the initial value of the products, so it costs no instruction.
    static constexpr bool RAMP = BIAS == BIAS_SLOPE && !CAP && DP <= 64;
    x8 qf[NS];
    f32x16 acc[ND];
    f32x16 ramp;  // before the positions; negated once the tiles have come behind them (tiles are taken in order)
    bool flipped;
    float m, l, slope2, edge_lo, edge_hi;
    int pos, lim;
    int pos_min, pos_max, lim_min, lim_max;  // over the wave's live rows
    int table_at;                            // of the row's head in the LDS copy, at distance 0
    bool tame;                               // biases are of a size that scores do not vanish beside

    __device__ __forceinline__ void open(const AttnArgs& a, const DocRange& d, int b, int hk, int prefix, int row0, const RowPlace& r, const float* table) {
        const int lane = threadIdx.x & 63, h = lane >> 5;
        const T* qp = (const T*)a.q + b * a.q_sb + (d.q0 + r.token) * a.q_st + r.head * a.q_sh + h * 8;
#pragma unroll
        for (int s = 0; s < NS; ++s) qf[s] = (r.live && s * 16 + h * 8 < a.dim) ? *(const x8*)(qp + s * 16) : (x8)((T)0.f);
        const int rows = d.lq * a.group, last = row0 + 31 < rows - 1 ? row0 + 31 : rows - 1;
        const bool any = row0 < rows;
        pos_min = token_of(a, row0) + d.lk - d.lq;
        pos_max = (any ? token_of(a, last) : 0) + d.lk - d.lq;
        lim_min = any ? limit_of(a, d, pos_min, prefix) : 0;
        lim_max = any ? limit_of(a, d, pos_max, prefix) : 0;
        pos_min = __builtin_amdgcn_readfirstlane(pos_min);
        pos_max = __builtin_amdgcn_readfirstlane(pos_max);
        lim_min = __builtin_amdgcn_readfirstlane(lim_min);
        lim_max = __builtin_amdgcn_readfirstlane(lim_max);
        pos = r.live ? r.pos : pos_max;  // (rows behind the last one are computed along, inside the table, and dropped)
        lim = r.lim;
        m = FIXED ? 0.f : -INFINITY;
        l = 0.f;
#pragma unroll
        for (int i = 0; i < ND; ++i) acc[i] = (f32x16)(0.f);
        if constexpr (BIAS == BIAS_SLOPE) slope2 = r.live ? a.slopes[r.head] * LOG2E : 0.f;
        if constexpr (RAMP) {
            const float per = slope2 / a.scale2;
            tame = !__any(!(fabsf(per) < 1e15f));
#pragma unroll
            for (int e = 0; e < 16; ++e) ramp[e] = per * (float)(8 * (e >> 2) + (e & 3));
            flipped = false;
        }
        if constexpr (BIAS == BIAS_TABLE) {
            table_at = (r.head - hk * a.group) * (2 * (a.reach + TABLE_EDGE) + 1) + a.reach + TABLE_EDGE;
            edge_lo = table[table_at - a.reach];
            edge_hi = table[table_at + a.reach];
            tame = !__any(!(fabsf(edge_lo) < 1e30f && fabsf(edge_hi) < 1e30f));
        }
    }

    // The row's sum over both halves of the wave; a row that is none has nothing.
    __device__ __forceinline__ void close(bool live) {
        l += swap_halves(l);
        if (!live) {
            l = 0.f;
            m = FIXED ? 0.f : -INFINITY;
#pragma unroll
            for (int i = 0; i < ND; ++i) acc[i] = (f32x16)(0.f);
        }
    }

    // Keys j0 .. j0 + KT - 1, of which those below lim are seen; kl, vl: their tile in LDS.
    __device__ __forceinline__ void tile(const AttnArgs& a, const char* kl, const char* vl, const float* table, int j0) {
        const int lane = threadIdx.x & 63, h = lane >> 5, c32 = lane & 31;
        const bool before = tame && j0 + KT - 1 <= pos_min, behind = tame && !before && j0 >= pos_max;  // (of a slope)
        if constexpr (RAMP) {
            if (behind && !flipped) {
                ramp = -ramp;
                flipped = true;
            }
        }
        f32x16 s[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            const int i = n * 32 + c32;
            if constexpr (RAMP) {
                if (before || behind)
                    s[n] = mfma32(*(const x8*)(kl + i * (DP * 2) + ((h ^ swizzle_k<DP>(i)) << 4)), qf[0], ramp);
                else
                    s[n] = mfma32(*(const x8*)(kl + i * (DP * 2) + ((h ^ swizzle_k<DP>(i)) << 4)), qf[0], (f32x16)(0.f));
            } else {
                s[n] = mfma32(*(const x8*)(kl + i * (DP * 2) + ((h ^ swizzle_k<DP>(i)) << 4)), qf[0], (f32x16)(0.f));
            }
#pragma unroll
            for (int t = 1; t < NS; ++t) s[n] = mfma32(*(const x8*)(kl + i * (DP * 2) + (((2 * t + h) ^ swizzle_k<DP>(i)) << 4)), qf[t], s[n]);
        }
        if constexpr (RAMP) {
            // The scores are read behind a branch here, and the compiler has left a read too close behind the last product
            // on such a path (three of the twelve wait states that the result of a 32 x 32 product needs).
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("s_nop 11");
            __builtin_amdgcn_sched_barrier(0);
        }
        // x = s mul + add + n more is the score in base 2 (n: the tile's 32 keys)
        float mul = CAP ? 1.f : a.scale2, add = 0.f, more = 0.f;
        const int d0 = j0 + 4 * h - pos;  // distance of this lane's first key
        if constexpr (CAP) {
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[n][e] = CAP == CAP_ANY ? capped(a, s[n][e]) : capped_direct(a, s[n][e]);
        }
        if constexpr (BIAS == BIAS_SLOPE) {
            if (RAMP && before) {
                add = slope2 * (float)d0;
                more = slope2 * 32.f;
            } else if (RAMP && behind) {
                add = -slope2 * (float)d0;
                more = slope2 * -32.f;
            } else {
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[n][e] = fmaf(-slope2, fabsf((float)(d0 + n * 32 + 8 * (e >> 2) + (e & 3))), CAP ? s[n][e] : s[n][e] * a.scale2);
                mul = 1.f;
            }
        }
        if constexpr (BIAS == BIAS_TABLE) {
            if (tame && j0 + KT - 1 <= pos_min - a.reach) {
                add = edge_lo;
            } else if (tame && j0 >= pos_max + a.reach) {
                add = edge_hi;
            } else {
                // a tile that reaches into the table is at most KT + 30 past its ends, which the copy in LDS repeats
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        int d = d0 + n * 32 + 8 * (e >> 2) + (e & 3);
                        if (!tame) d = d < -a.reach ? -a.reach : d > a.reach ? a.reach : d;
                        s[n][e] = (CAP ? s[n][e] : s[n][e] * a.scale2) + table[table_at + d];
                    }
                mul = 1.f;
            }
        }
        if (j0 + KT > lim_min) {  // (else every row of the wave sees the whole tile)
            const int left = lim - (j0 + 4 * h);
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[n][e] = n * 32 + 8 * (e >> 2) + (e & 3) < left ? s[n][e] : -INFINITY;
        }
        float off[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) off[n] = RAMP ? fmaf((float)n, more, add) : add;
        if constexpr (!FIXED) {
            float top = -INFINITY;
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                float t[4] = {s[n][0], s[n][1], s[n][2], s[n][3]};  // (four chains: a maximum waits for the one before)
#pragma unroll
                for (int e = 4; e < 16; e += 4)
#pragma unroll
                    for (int i = 0; i < 4; ++i) t[i] = fmaxf(t[i], s[n][e + i]);
                top = fmaxf(top, fmaf(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])), mul, off[n]));
            }
            top = fmaxf(top, swap_halves(top));
            // The base m of a row's weights follows its maximum only when that is 2^8 ahead: weights up to 2^8 (in fp16 from
            // 2^7 to 2^15; its largest is 65504) are as exact as those up to 1, and the sums need not be rescaled each time some row of the
            // wave finds a new maximum, which over 8192 keys of random scores is in three tiles of five.
            if (__any(top > m + 8.f)) {
                const float m_new = fmaxf(m, top);
                const float keep = exp2_hw(m - (m_new == -INFINITY ? 0.f : m_new));
                m = m_new;
                l *= keep;
#pragma unroll
                for (int i = 0; i < ND; ++i) acc[i] *= keep;
            }
            const float base = m == -INFINITY ? 0.f : m - top_weight<T>(8.f);  // nothing seen so far: every weight is exp2(-inf) = 0
#pragma unroll
            for (int n = 0; n < NB; ++n) off[n] -= base;
        }
        // The sum of weights is that of the rounded ones, two per instruction: numerator and denominator round alike.  A tile's
        // are summed before they meet the running sum, beside which single ones may be nothing.
        x8 pf[2 * NB];
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                const float w0 = FIXED ? exp2_hw(s[n][e]) : exp2_hw(fmaf(s[n][e], mul, off[n]));
                const float w1 = FIXED ? exp2_hw(s[n][e + 1]) : exp2_hw(fmaf(s[n][e + 1], mul, off[n]));
                const typename vec_of<T>::x2 w = {(T)w0, (T)w1};
                part[(e >> 1) & 3] = add_pair(w, part[(e >> 1) & 3]);
                pf[2 * n + (e >> 3)][e & 7] = w[0];
                pf[2 * n + (e >> 3)][(e & 7) + 1] = w[1];
            }
        l += (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
        for (int t = 0; t < 2 * NB; ++t)
#pragma unroll
            for (int i = 0; i < ND; ++i) {
                union {
                    s16x4 half[2];
                    x8 all;
                } vf;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int key = t * 16 + e * 8 + 4 * h + ((lane & 15) >> 2), col = i * 32 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
                    vf.half[e] = lds_read_tr(vl + key * (DP * 2) + (((col >> 3) ^ swizzle_v<DP>(key)) << 4) + (col & 7) * 2);
                }
                acc[i] = mfma32(vf.all, pf[t], acc[i]);
            }
    }
};

// glds16_asm for the lanes of `mask` alone.
__device__ __forceinline__ void glds16_masked_asm(const void* sbase, int voff, uint32_t lds_addr, uint64_t mask) {
    unsigned keep;
    uint64_t lanes;
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b64 %1, exec\n\ts_mov_b32 m0, %4\n\ts_and_b64 exec, exec, %5\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3\n\ts_mov_b64 exec, %1\n\ts_mov_b32 m0, %0"
        : "=&s"(keep), "=&s"(lanes)
        : "v"(voff), "s"(sbase), "s"(lds_addr), "s"(mask)
        : "memory", "scc");
}

// The wave's share of the DMA of one tile: KT rows of K and of V, NI instructions of 1 KB each.
template <int DP, int KT, int NWAVES>
struct TileLoad {
    static constexpr int PPR = DP / 8, RPI = 64 / PPR, NI = KT / RPI / NWAVES;
    int kof[NI], vof[NI], row0;  // this lane's row of instruction j is row0 + j RPI
    int piece;                   // of K that instruction 0 fetches for this lane
    // Whether instruction j fetches a piece of the head (its rows are j RPI further, a multiple of 8 or below it).
    __device__ __forceinline__ bool in_head(const AttnArgs& a, int j) const { return (piece ^ (DP == 32 ? 0 : j * RPI & 7)) * 8 < a.dim; }
    __device__ __forceinline__ void open(const AttnArgs& a, int wave) {
        const int lane = threadIdx.x & 63;
        row0 = wave * NI * RPI + lane / PPR;
#pragma unroll
        for (int j = 0; j < NI; ++j) {
            const int row = row0 + j * RPI, pk = (lane % PPR) ^ swizzle_k<DP>(row), pv = (lane % PPR) ^ swizzle_v<DP>(row);
            // (a piece of V behind the head's dimension repeats the first: it ends in columns not stored)
            kof[j] = row * (int)(a.k_st * 2) + pk * 16;
            if (j == 0) piece = pk;
            vof[j] = row * (int)(a.v_st * 2) + (pv * 8 < a.dim ? pv * 16 : 0);
        }
    }
    // Pieces of K behind the head's dimension are never fetched and meet zeros of q: zero (0 times whatever stood there could
    // be NaN), in the tile's first `rows` rows of one buffer or of both.
    __device__ __forceinline__ void blank_pads(const AttnArgs& a, uint32_t kl, int rows, int buffers, int next, int wave) const {
        if (a.dim == DP) return;
        for (int b = 0; b < buffers; ++b)
#pragma unroll
            for (int j = 0; j < NI; ++j)
                if ((wave * NI + j) * RPI < rows && !in_head(a, j)) *(__attribute__((address_space(3))) u32x4*)(uintptr_t)(kl + b * next + (wave * NI + j) * 1024 + (threadIdx.x & 63) * 16) = (u32x4)(0u);
    }
    // The wave's rows of V behind the last key become zero (0 times a V that is infinite there would be NaN).
    __device__ __forceinline__ void blank_behind(int j0, int lk, uint32_t vl, int wave) const {
        const int rows = lk - j0 - wave * NI * RPI, from = rows < 0 ? 0 : rows, lane = threadIdx.x & 63;  // rows of the wave that hold keys
        uint32_t at = vl + (wave * NI + from / RPI) * 1024 + lane * 16;
        if (from < NI * RPI && lane / PPR >= from % RPI) *(__attribute__((address_space(3))) u32x4*)(uintptr_t)at = (u32x4)(0u);
        for (int j = from / RPI + 1; j < NI; ++j) *(__attribute__((address_space(3))) u32x4*)(uintptr_t)(at += 1024) = (u32x4)(0u);
    }
    // Rows j0 .. of K and V to LDS.  What stands behind the last key is never read: rows there repeat it, or (ZERO) those of V
    // are zero and not fetched.  (Some instructions then fetch nothing, so a wave that counts its requests blanks them once
    // they have landed instead.)  Whole tiles have a path of their own: single tokens over long keys gain 11 %.
    template <bool ZERO, typename T>
    __device__ __forceinline__ void issue(const AttnArgs& a, const T* k, const T* v, int j0, int lk, uint32_t kl, uint32_t vl, int wave) {
        const char* kb = uniform_ptr(k + j0 * a.k_st);
        const char* vb = uniform_ptr(v + j0 * a.v_st);
        const bool whole = j0 + KT <= lk;
        const int behind = row0 - (lk - 1 - j0);  // rows from the last key to row0
        auto back = [&](int j) __attribute__((always_inline)) { return behind + j * RPI > 0 ? behind + j * RPI : 0; };
        if (whole) {
            if (a.dim == DP) {
#pragma unroll
                for (int j = 0; j < NI; ++j) glds16_asm(kb, kof[j], kl + (wave * NI + j) * 1024);
            } else {
#pragma unroll
                for (int j = 0; j < NI; ++j) glds16_masked_asm(kb, kof[j], kl + (wave * NI + j) * 1024, __ballot(in_head(a, j)));
            }
#pragma unroll
            for (int j = 0; j < NI; ++j) glds16_asm(vb, vof[j], vl + (wave * NI + j) * 1024);
        } else {
#pragma unroll
            for (int j = 0; j < NI; ++j) glds16_masked_asm(kb, kof[j] - back(j) * (int)(a.k_st * 2), kl + (wave * NI + j) * 1024, __ballot(in_head(a, j)));
#pragma unroll
            for (int j = 0; j < NI; ++j) {
                if (ZERO)
                    glds16_masked_asm(vb, vof[j], vl + (wave * NI + j) * 1024, __ballot(behind + j * RPI <= 0));
                else
                    glds16_asm(vb, vof[j] - back(j) * (int)(a.v_st * 2), vl + (wave * NI + j) * 1024);
            }
            if (ZERO) blank_behind(j0, lk, vl, wave);
        }
    }
};

// Table rows of a key head's group, in base 2, each with its first and last entry repeated TABLE_EDGE times.
__device__ __forceinline__ void stage_table(const AttnArgs& a, int hk, float* dst) {
    const int width = 2 * a.reach + 1, wide = width + 2 * TABLE_EDGE;
    for (int g = 0; g < a.group; ++g) {
        const float* src = a.table + (int64_t)(hk * a.group + g) * width;
        for (int i = threadIdx.x; i < wide; i += blockDim.x) {
            const int at = i - TABLE_EDGE;
            dst[g * wide + i] = table2(src[at < 0 ? 0 : at < width ? at : width - 1]);
        }
    }
}

__device__ __forceinline__ int64_t out_row(const AttnArgs& a, const DocRange& d, int b, int token, int head) {
    return ((a.q_offs ? 0 : b * a.q_rows) + d.q0 + token) * a.heads + head;
}

// One lane's row of O^T: registers 4 g .. 4 g + 3 are dimensions 8 g + 4 h .. + 3 of 32.  One exchange between the wave's
// halves per two pieces gives either half whole 16-byte pieces.
template <typename T, int ND>
__device__ __forceinline__ void store_row(const AttnArgs& a, const f32x16 (&acc)[ND], float inv, int64_t orow, bool write) {
    const int h = (threadIdx.x >> 5) & 1;
    T* op = (T*)a.out + orow * a.dim;
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int g = 0; g < 4; g += 2) {
            union {
                T v[4];
                u32x2 u;
            } lo, hi;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                lo.v[e] = (T)(acc[i][4 * g + e] * inv);
                hi.v[e] = (T)(acc[i][4 * g + 4 + e] * inv);
            }
            const auto r0 = __builtin_amdgcn_permlane32_swap(lo.u.x, hi.u.x, false, false);
            const auto r1 = __builtin_amdgcn_permlane32_swap(lo.u.y, hi.u.y, false, false);
            u32x4 o;
            o.x = r0[0];
            o.y = r1[0];
            o.z = r0[1];
            o.w = r1[1];
            const int d = i * 32 + (g + h) * 8;
            if (write && d < a.dim) __builtin_memcpy(op + d, &o, 16);
        }
}
template <int ND>
__device__ __forceinline__ void store_part(const AttnArgs& a, const f32x16 (&acc)[ND], float m, float l, int chunk, int64_t orow, bool write) {
    const int h = (threadIdx.x >> 5) & 1;
    const int64_t at = chunk * a.part_rows + orow;
    if (!write) return;
    float* op = a.part + at * a.dim;
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = i * 32 + g * 8 + h * 4;
            const f32x4 o = {acc[i][4 * g], acc[i][4 * g + 1], acc[i][4 * g + 2], acc[i][4 * g + 3]};
            if (d < a.dim) *(f32x4*)(op + d) = o;
        }
    if (h == 0) a.part_ml[at] = make_float2(m, l);
}
// 1 / l; a row that sees nothing is zero, NaN stays NaN.
__device__ __forceinline__ float inverse(float l) { return l > 0.f || l != l ? 1.f / l : 0.f; }

// ---- many rows: 128 per workgroup, 32 per wave ---------------------------------------------------------
// All four waves read the tiles of 64 keys (32 for heads wider than 128) that they fetch together, two buffers deep.
// Two documents of 8192 tokens, 16 heads of 64: 0.63 ms, 0.87 PFLOP/s; with a slope 0.74 (0.86 where the inputs are not
// those of the call before, still in the caches); causal 0.35; 8 heads of 128: 0.555 ms, 0.99 PFLOP/s, capped 0.60.  Bound by the sum of matrix and vector work: per 64 keys x 32 rows x 64 a SIMD spends 512
// cycles on products and about 900 on weights (32 exponentials of a quarter of the vector rate, 110 other operations), takes
// 1190, and what one side saves the clock (1.9 GHz under this load) or the other side eats.  Built and not kept, all
// within 3 %: 64 rows per wave (half the LDS reads, two independent softmax chains), four waves per SIMD, three tiles in
// flight, independent chains for maximum and sum.
template <typename T, int DP, int BIAS, int CAP, bool FIXED>
__global__ __launch_bounds__(256, DP <= 64 && !(BIAS == BIAS_SLOPE && !CAP) && CAP != CAP_ANY ? 3 : DP <= 128 ? 2 : 1) void k_attend_rows(AttnArgs a) {
    constexpr int NB = DP <= 128 ? 2 : 1, KT = NB * 32, TILE = KT * DP * 2;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const float* table = (const float*)(lds + 4 * TILE);
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int id = spread_over_xcds((int)blockIdx.x, (int)gridDim.x);
    const int chunk = id % a.chunks;
    id /= a.chunks;
    const int t0 = a.tiles - 1 - id % a.tiles;  // causal: the longest rows first
    id /= a.tiles;
    const int hk = id % a.kv_heads, b = a.b0 + id / a.kv_heads;
    const DocRange dr = doc_range(a, b);
    const int rows = dr.lq * a.group, rows_all = dr.q_total * a.group;
    const T* kbase = (const T*)a.k + b * a.k_sb + dr.k0 * a.k_st + hk * a.k_sh;
    const T* vbase = (const T*)a.v + b * a.v_sb + dr.k0 * a.v_st + hk * a.v_sh;
    const int prefix = a.prefix ? a.prefix[b] : 0;
    const int from = chunk * a.chunk;
    if (from > 0 && from >= dr.lk) return;
    TileLoad<DP, KT, 4> load;
    load.open(a, wv);
    const uint32_t l0 = lds_addr_of(lds);
    load.blank_pads(a, l0, KT, 2, 2 * TILE, wv);
    // keys that any of the workgroup's rows from row0 on sees, in this chunk; the first tile of them is requested at once
    auto begin = [&](int row0) __attribute__((always_inline)) {
        if (row0 >= rows) return 0;
        const int last = row0 + 127 < rows - 1 ? row0 + 127 : rows - 1;
        int need = limit_of(a, dr, token_of(a, last) + dr.lk - dr.lq, prefix);
        if (need > from + a.chunk) need = from + a.chunk;
        if (from < need) load.template issue<true>(a, kbase, vbase, from, dr.lk, l0, l0 + TILE, wv);
        return need;
    };
    int need = begin(t0 * 128);
    if constexpr (BIAS == BIAS_TABLE) {
        stage_table(a, hk, (float*)(lds + 4 * TILE));
        __syncthreads();
    }

    // (a row number stays below 2^31: at most 2^29 rows, and steps of at most 2^29 + 128)
    for (int row0 = t0 * 128; row0 < rows_all; row0 += a.tiles * 128) {
        const RowPlace r = row_place(a, dr, hk, prefix, row0 + wv * 32 + (lane & 31));
        Attend<T, DP, NB, BIAS, CAP, FIXED> st;
        st.open(a, dr, b, hk, prefix, row0 + wv * 32, r, table);
        int buf = 0;
        for (int j0 = from; j0 < need; j0 += KT, buf ^= 1) {
            wait_all_barrier();  // the tile has landed; everyone has read the one before
            if (j0 + KT < need) load.template issue<true>(a, kbase, vbase, j0 + KT, dr.lk, l0 + (buf ^ 1) * 2 * TILE, l0 + (buf ^ 1) * 2 * TILE + TILE, wv);
            if (j0 < st.lim_max) st.tile(a, lds + buf * 2 * TILE, lds + buf * 2 * TILE + TILE, table, j0);
        }
        st.close(r.live);
        const bool write = r.row < rows_all;
        const int64_t orow = out_row(a, dr, b, r.token, r.head);
        if (a.chunks == 1)
            store_row<T>(a, st.acc, inverse(st.l), orow, write);
        else
            store_part(a, st.acc, st.m, st.l, chunk, orow, write);
        if (row0 + a.tiles * 128 < rows_all) {
            __syncthreads();  // (the next rows fetch over the last tile)
            need = begin(row0 + a.tiles * 128);
        }
    }
}

// ---- few rows: up to 32 per document and key head --------------------------------------------------------
// The waves of a workgroup share the keys instead of the rows: wave w takes tiles w, w + NW, .. of 32 keys through an LDS
// ring of its own, without a barrier, and the waves' sums meet at the end in a fixed order.
// Bound by HBM: 8 documents of 32768 keys, 8 key heads of 128, 4 query heads each: 204 us, 5.2 TB/s, the rate of a copy;
// lengths of 1 .. 32768 164 us (4.5 TB/s; the longest document's chunks end last), with a cap and a slope 183 us.
template <typename T, int DP, int NW, int BIAS, int CAP, bool FIXED>
__global__ __launch_bounds__(64 * NW) void k_attend_few(AttnArgs a) {
    constexpr int KT = 32, TILE = KT * DP * 2, ND = DP / 32, RING = 4 * TILE;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const float* table = (const float*)(lds + NW * RING);
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int id = spread_over_xcds((int)blockIdx.x, (int)gridDim.x);
    const int hk = id % a.kv_heads;
    id /= a.kv_heads;
    const int chunk = id % a.chunks, b = a.b0 + id / a.chunks;
    const DocRange dr = doc_range(a, b);
    const int rows_all = dr.q_total * a.group;
    const T* kbase = (const T*)a.k + b * a.k_sb + dr.k0 * a.k_st + hk * a.k_sh;
    const T* vbase = (const T*)a.v + b * a.v_sb + dr.k0 * a.v_st + hk * a.v_sh;
    const int prefix = a.prefix ? a.prefix[b] : 0;
    const int from = chunk * a.chunk;
    if (from > 0 && from >= dr.lk) return;
    if constexpr (BIAS == BIAS_TABLE) {
        stage_table(a, hk, (float*)(lds + NW * RING));
        __syncthreads();
    }
    TileLoad<DP, KT, 1> load;
    load.open(a, 0);
    char* mine = lds + wv * RING;
    const uint32_t l0 = lds_addr_of(lds) + wv * RING;

    for (int row0 = 0; row0 < rows_all; row0 += 32) {
        const RowPlace r = row_place(a, dr, hk, prefix, row0 + (lane & 31));
        Attend<T, DP, 1, BIAS, CAP, FIXED> st;
        st.open(a, dr, b, hk, prefix, row0, r, table);
        int need = st.lim_max;
        if (need > from + a.chunk) need = from + a.chunk;
        int buf = 0;
        const int first = from + wv * KT;
        if (first < need) {
            const bool more = first + NW * KT < need;
            load.blank_pads(a, l0, more ? KT : dr.lk - first, more ? 2 : 1, 2 * TILE, 0);
            load.template issue<false>(a, kbase, vbase, first, dr.lk, l0, l0 + TILE, 0);
        }
        for (int j0 = first; j0 < need; j0 += NW * KT, buf ^= 1) {
            // this wave's reads of the other buffer are done (the products that needed them are under way)
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (j0 + NW * KT < need) {
                load.template issue<false>(a, kbase, vbase, j0 + NW * KT, dr.lk, l0 + (buf ^ 1) * 2 * TILE, l0 + (buf ^ 1) * 2 * TILE + TILE, 0);
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * TileLoad<DP, KT, 1>::NI) : "memory");
            } else {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            }
            if (j0 + KT > dr.lk) {
                load.blank_behind(j0, dr.lk, l0 + buf * 2 * TILE + TILE, 0);
                asm volatile("" ::: "memory");  // (a wave's LDS accesses are done in order)
            }
            st.tile(a, mine + buf * 2 * TILE, mine + buf * 2 * TILE + TILE, table, j0);
        }
        st.close(r.live);
        // join: wave 0 takes the others' (m, l, O) in order
        __syncthreads();
        float* sum = (float*)lds;  // [NW - 1][ND * 16 + 2][64]
        constexpr int EACH = (ND * 16 + 2) * 64;
        static_assert((NW - 1) * EACH * 4 <= NW * RING, "the sums fit where the tiles were");
        if (wv > 0) {
            float* to = sum + (wv - 1) * EACH + lane;
            to[0] = st.m;
            to[64] = st.l;
#pragma unroll
            for (int i = 0; i < ND; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) to[(2 + i * 16 + e) * 64] = st.acc[i][e];
        }
        __syncthreads();
        if (wv == 0) {
#pragma unroll 1
            for (int w = 0; w < NW - 1; ++w) {
                const float* of = sum + w * EACH + lane;
                const float m2 = of[0], l2 = of[64], top = fmaxf(st.m, m2), base = top == -INFINITY ? 0.f : top;
                const float f1 = FIXED ? 1.f : exp2_hw(st.m - base), f2 = FIXED ? 1.f : exp2_hw(m2 - base);
                st.m = top;
                st.l = st.l * f1 + l2 * f2;
#pragma unroll
                for (int i = 0; i < ND; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) st.acc[i][e] = st.acc[i][e] * f1 + of[(2 + i * 16 + e) * 64] * f2;
            }
            const bool write = r.row < rows_all;
            const int64_t orow = out_row(a, dr, b, r.token, r.head);
            if (a.chunks == 1)
                store_row<T>(a, st.acc, inverse(st.l), orow, write);
            else
                store_part(a, st.acc, st.m, st.l, chunk, orow, write);
        }
        if (row0 + 32 < rows_all) __syncthreads();
    }
}

// ---- the chunks of a row joined --------------------------------------------------------------------------
// One workgroup per row: o = sum_c o_c 2^(m_c - m) / sum_c l_c 2^(m_c - m).  Thread (phase, piece) adds the chunks phase,
// phase + phases, .. of its 4 dimensions; the phases meet in LDS in order.  256 rows of 8 chunks: 4.8 us.
template <typename T>
__global__ __launch_bounds__(256) void k_attend_join(AttnArgs a, int rows_hint) {
    __shared__ float factor[256], wave_top[4], wave_sum[4];
    __shared__ f32x4 sums[256];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int b = a.b0 + blockIdx.x / rows_hint;
    const DocRange dr = doc_range(a, b);
    const int64_t rows_all = (int64_t)dr.q_total * a.heads;
    const int n = dr.lk <= a.chunk ? 1 : (dr.lk + a.chunk - 1) / a.chunk;  // at most 256
    const int pieces = a.dim / 4, phases = 256 / pieces, ph = tid / pieces, d = (tid - ph * pieces) * 4;
    for (int64_t row = blockIdx.x % rows_hint; row < rows_all; row += rows_hint) {
        const int64_t at = ((a.q_offs ? 0 : b * a.q_rows) + dr.q0) * a.heads + row;
        const float2 ml = tid < n ? a.part_ml[tid * a.part_rows + at] : make_float2(-INFINITY, 0.f);
        float m = ml.x;
#pragma unroll
        for (int x = 32; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
        if (lane == 0) wave_top[wv] = m;
        __syncthreads();
        m = fmaxf(fmaxf(wave_top[0], wave_top[1]), fmaxf(wave_top[2], wave_top[3]));
        const float f = exp2_hw(ml.x - (m == -INFINITY ? 0.f : m));
        factor[tid] = f;
        float l = ml.y * f;
#pragma unroll
        for (int x = 32; x > 0; x >>= 1) l += __shfl_xor(l, x);
        if (lane == 0) wave_sum[wv] = l;
        __syncthreads();
        l = (wave_sum[0] + wave_sum[1]) + (wave_sum[2] + wave_sum[3]);
        f32x4 o = (f32x4)(0.f);
        if (ph < phases) {
#pragma unroll 4
            for (int c = ph; c < n; c += phases) o += *(const f32x4*)(a.part + (c * a.part_rows + at) * a.dim + d) * factor[c];
        }
        sums[tid] = o;
        __syncthreads();
        if (ph == 0) {
            for (int p = 1; p < phases; ++p) o += sums[p * pieces + tid];
            const float inv = inverse(l);
            T v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (T)(o[e] * inv);
            __builtin_memcpy((T*)a.out + at * a.dim + d, v, 8);
        }
        __syncthreads();
    }
}

// ---- host side ---------------------------------------------------------------------------------------
#define ATTN_TABLE_LDS 16384  // bytes of table rows that a workgroup keeps in LDS; larger ones are read from memory

struct AttnPlan {
    bool fast = false, few = false;
    int64_t longest_q = 0, part_rows = 0;
    size_t bytes = 0;  // of workspace
};

template <typename K>
static int launch_attend(hrs_ctx* ctx, hrs_per_device_once& attr, K kernel, int threads, int lds, int64_t grid, const AttnArgs& a, hipStream_t st) {
    HRS_REQUIRE(grid < (1 << 24), "hrs_attention: %lld workgroups for one document", (long long)grid);
    if (lds > 65536 && attr.need(ctx->device)) {
        HRS_CHECK_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
        attr.done(ctx->device);
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(threads), lds, st, a);
    HRS_CHECK_HIP(hipGetLastError());
    return HRS_OK;
}
template <typename T, int DP, int BIAS, int CAP, bool FIXED>
static int launch_fast(hrs_ctx* ctx, const AttnArgs& a, const AttnPlan& p, hipStream_t st) {
    static hrs_per_device_once once_few, once_rows;
    const int table = BIAS == BIAS_TABLE ? a.group * (2 * (a.reach + TABLE_EDGE) + 1) * 4 : 0;
    const int64_t pairs = (int64_t)a.batch * a.kv_heads;
    if (p.few) {
        constexpr int NW = DP == 256 ? 2 : 4;
        return launch_attend(ctx, once_few, k_attend_few<T, DP, NW, BIAS, CAP, FIXED>, 64 * NW, NW * 4 * 32 * DP * 2 + table, pairs * a.chunks, a, st);
    }
    constexpr int KT = DP <= 128 ? 64 : 32;
    return launch_attend(ctx, once_rows, k_attend_rows<T, DP, BIAS, CAP, FIXED>, 256, 4 * KT * DP * 2 + table, pairs * a.tiles * a.chunks, a, st);
}
template <typename T, int DP, int BIAS, bool CAP>
static int launch_form(hrs_ctx* ctx, const AttnArgs& a, const AttnPlan& p, hipStream_t st) {
    if (!p.fast) {
        static hrs_per_device_once once;
        return launch_attend(ctx, once, k_attend_any<T, DP, BIAS, CAP>, 256, 0, (int64_t)a.batch * a.kv_heads * a.tiles, a, st);
    }
    // Capped scores without a bias lie within +-cap: in bf16, whose range is that of fp32, the weights need no running
    // maximum.  They are 2^+-80 at most, so that |v| times the number of keys may reach 2^48 and |v| may fall to 2^-46 before
    // the sums leave fp32 (documented).  Two documents of 8192 tokens, 16 heads of 64: 795 us, 912 with the maximum; 8 heads
    // of 128, 4096 tokens, causal: 172 and 184.
    if constexpr (CAP && BIAS == BIAS_NONE && __is_same(T, __bf16)) {
        if (a.cap2 <= 80.f) return launch_fast<T, DP, BIAS, CAP_TO_64, true>(ctx, a, p, st);
    }
    if (CAP && a.cap2 > CAP_DIRECT) return launch_fast<T, DP, BIAS, CAP ? CAP_ANY : CAP_NONE, false>(ctx, a, p, st);
    return launch_fast<T, DP, BIAS, CAP ? CAP_TO_64 : CAP_NONE, false>(ctx, a, p, st);
}
template <typename T, int DP>
static int launch_dim(hrs_ctx* ctx, const AttnArgs& a, const AttnPlan& p, hipStream_t st) {
    const bool cap = a.cap2 > 0.f;
    if (a.table) return cap ? launch_form<T, DP, BIAS_TABLE, true>(ctx, a, p, st) : launch_form<T, DP, BIAS_TABLE, false>(ctx, a, p, st);
    if (a.slopes) return cap ? launch_form<T, DP, BIAS_SLOPE, true>(ctx, a, p, st) : launch_form<T, DP, BIAS_SLOPE, false>(ctx, a, p, st);
    return cap ? launch_form<T, DP, BIAS_NONE, true>(ctx, a, p, st) : launch_form<T, DP, BIAS_NONE, false>(ctx, a, p, st);
}
template <typename T>
static int launch_type(hrs_ctx* ctx, const AttnArgs& a, const AttnPlan& p, hipStream_t st) {
    int rc;
    if (a.dim <= 32)
        rc = launch_dim<T, 32>(ctx, a, p, st);
    else if (a.dim <= 64)
        rc = launch_dim<T, 64>(ctx, a, p, st);
    else if (a.dim <= 128)
        rc = launch_dim<T, 128>(ctx, a, p, st);
    else
        rc = launch_dim<T, 256>(ctx, a, p, st);
    if (rc || a.chunks == 1) return rc;
    int64_t rows = p.longest_q * a.heads;  // workgroups per document
    if (rows > (1 << 20) / a.batch + 1) rows = (1 << 20) / a.batch + 1;  // (each takes further rows in turn)
    hipLaunchKernelGGL(k_attend_join<T>, dim3((unsigned)(rows * a.batch)), dim3(256), 0, st, a, (int)rows);
    HRS_CHECK_HIP(hipGetLastError());
    return HRS_OK;
}

static int attention_args(const hrs_attention_args* p, AttnArgs& a) {
    HRS_REQUIRE(p->dtype == HRS_TYPE_BF16 || p->dtype == HRS_TYPE_FP16, "hrs_attention: type %d is neither bf16 nor fp16", p->dtype);
    HRS_REQUIRE(p->batch >= 0 && p->q_heads >= 1 && p->kv_heads >= 1 && p->q_heads % p->kv_heads == 0,
                "hrs_attention: batch=%d, q_heads=%d, kv_heads=%d (query heads must be a multiple of key heads)", p->batch, p->q_heads, p->kv_heads);
    HRS_REQUIRE(p->head_dim >= 8 && p->head_dim <= 256 && p->head_dim % 8 == 0, "hrs_attention: head_dim=%d must be a multiple of 8 in [8, 256]", p->head_dim);
    HRS_REQUIRE(p->q_rows >= 0 && p->k_rows >= 0 && p->q_rows < (1ll << 30) && p->k_rows < (1ll << 30), "hrs_attention: q_rows=%lld, k_rows=%lld",
                (long long)p->q_rows, (long long)p->k_rows);
    HRS_REQUIRE(p->q_rows * (p->q_heads / p->kv_heads) <= (1ll << 29), "hrs_attention: q_rows=%lld with %d query heads per key head", (long long)p->q_rows, p->q_heads / p->kv_heads);
    HRS_REQUIRE(p->scale > 0.f && p->scale < INFINITY, "hrs_attention: scale=%g must be positive and finite", (double)p->scale);
    HRS_REQUIRE(p->softcap >= 0.f && p->softcap < INFINITY, "hrs_attention: softcap=%g must be finite, 0 for none", (double)p->softcap);
    HRS_REQUIRE(!(p->slopes && p->bias_table), "hrs_attention: slopes and bias_table exclude each other");
    HRS_REQUIRE(!p->bias_table || (p->bias_reach >= 0 && p->bias_reach < (1 << 24)), "hrs_attention: bias_reach=%d", p->bias_reach);
    HRS_REQUIRE(!p->prefix_lens || p->causal, "hrs_attention: a prefix needs causal order (without it every key is seen)");
    HRS_REQUIRE(!(p->q_offs && p->q_lens), "hrs_attention: q_offs and q_lens exclude each other");
    for (int i = 0; i < 3; ++i)
        HRS_REQUIRE(p->q_stride[i] >= 0 && p->k_stride[i] >= 0 && p->v_stride[i] >= 0, "hrs_attention: negative stride");
    memset(&a, 0, sizeof(a));
    a.q = p->q;
    a.k = p->k;
    a.v = p->v;
    a.out = p->out;
    a.q_offs = p->q_offs;
    a.k_offs = p->k_offs;
    a.q_lens = p->q_lens;
    a.k_lens = p->k_lens;
    a.prefix = p->prefix_lens;
    a.slopes = p->slopes;
    a.table = p->bias_table;
    a.q_sb = p->q_offs ? 0 : p->q_stride[0];
    a.q_st = p->q_stride[1];
    a.q_sh = p->q_stride[2];
    a.k_sb = p->k_offs ? 0 : p->k_stride[0];
    a.k_st = p->k_stride[1];
    a.k_sh = p->k_stride[2];
    a.v_sb = p->k_offs ? 0 : p->v_stride[0];
    a.v_st = p->v_stride[1];
    a.v_sh = p->v_stride[2];
    a.q_rows = p->q_rows;
    a.k_rows = p->k_rows;
    a.batch = p->batch;
    a.heads = p->q_heads;
    a.kv_heads = p->kv_heads;
    a.group = p->q_heads / p->kv_heads;
    a.dim = p->head_dim;
    a.causal = p->causal != 0;
    a.reach = p->bias_reach;
    a.scale2 = p->scale * LOG2E;
    if (p->softcap > 0.f) {
        a.cap2 = p->softcap * LOG2E;
        a.cap_in = 2.f * LOG2E * p->scale / p->softcap;
        a.cap_u = p->scale / p->softcap;
    }
    HRS_REQUIRE(a.scale2 < 1e30f && a.cap2 < 1e30f && a.cap_in < 1e30f, "hrs_attention: scale=%g with softcap=%g leaves the range of fp32", (double)p->scale, (double)p->softcap);
    return HRS_OK;
}

// How the work is cut, from the arguments alone (never from device data).  A call whose addresses are not 16-byte aligned
// needs no workspace; the size of one is asked for as if they were.
static AttnPlan plan_attention(hrs_ctx* ctx, const hrs_attention_args* p, AttnArgs& a, bool aligned) {
    AttnPlan plan;
    // without a hint for packed documents: twice their mean
    const int64_t mean_q = a.q_offs && a.batch ? (2 * a.q_rows + a.batch - 1) / a.batch : a.q_rows;
    const int64_t mean_k = a.k_offs && a.batch ? (2 * a.k_rows + a.batch - 1) / a.batch : a.k_rows;
    auto hint = [](int64_t given, int64_t otherwise, int64_t all) {
        const int64_t v = given > 0 ? given : otherwise;
        return v < 1 ? (int64_t)1 : v < all ? v : all;
    };
    plan.longest_q = hint(p->max_q, mean_q, a.q_rows);
    const int64_t longest_k = hint(p->max_k, mean_k, a.k_rows), rows = plan.longest_q * a.group;
    a.tiles = (int)((rows + 127) / 128);
    a.chunks = 1;
    a.chunk = 1 << 30;
    // 16-byte pieces, and 64 rows of K or V within the 2^31 bytes that a DMA's lane offset spans
    const int64_t strides = a.q_sb | a.q_st | a.q_sh | a.k_sb | a.k_st | a.k_sh | a.v_sb | a.v_st | a.v_sh;
    plan.fast = aligned && strides % 8 == 0 && a.k_st < (1 << 23) && a.v_st < (1 << 23) &&
                (!a.table || (int64_t)a.group * (2 * (a.reach + TABLE_EDGE) + 1) * 4 <= ATTN_TABLE_LDS);
    if (!plan.fast) return plan;
    plan.few = rows <= 32;
    // Many documents: one workgroup takes all rows of a document (it walks on while there are rows), since most would find
    // none or few: 1024 ragged documents of up to 256 tokens, 16 heads of 64: 358 us with two workgroups for each, 320 with one;
    // 600 of up to 512: 577 and 488; 2048 of up to 128, 12 heads, without a hint: 397 and 219; but 400 of up to 1000, 12 heads of
    // 32: 547 and 560.
    const int64_t pairs = (int64_t)a.batch * a.kv_heads, enough = 16 * (int64_t)ctx->num_cu;
    if (!plan.few && pairs * a.tiles > enough && (a.q_offs || a.q_lens)) {
        const int64_t t = (enough + pairs - 1) / pairs;
        if (t < a.tiles) a.tiles = (int)t;
    }
    // Too few workgroups for the card: long documents are cut into chunks of keys, joined by a second launch.  Few rows
    // (one workgroup fills a CU): two per CU, of 1024 keys at least; more chunks only add to the join.  8 documents of
    // up to 32768 keys, 8 key heads of 128: 151 us with 4 chunks, 164 with 8, 183 with 16, 215 with 32; 13 documents: 382 with
    // 2, 373 with 4, 380 with 9, and of 32768 keys each 595, 473, 480.
    const int64_t groups = pairs * (plan.few ? 1 : a.tiles), cus = ctx->num_cu;
    if (groups < 2 * cus && longest_k > 1024) {
        int64_t chunks = (plan.few ? 2 : 4) * cus / groups, most = longest_k / (plan.few ? 1024 : 512);
        if (chunks < 2) chunks = 2;
        if (chunks > most) chunks = most;
        if (chunks > 64) chunks = 64;
        if (chunks > 1) {
            a.chunk = (int)(((longest_k + chunks - 1) / chunks + 127) / 128 * 128);
            // every key of every document has its chunk, whatever the hint said
            a.chunks = (int)((a.k_rows + a.chunk - 1) / a.chunk);
            if (a.chunks > 256) {  // (a hint far below the documents' room)
                a.chunks = 256;
                a.chunk = (int)((a.k_rows / 256 + 128) / 128 * 128);
            }
            a.chunks = (int)((a.k_rows + a.chunk - 1) / a.chunk);
        }
        if (a.chunks > 1) {
            plan.part_rows = (a.q_offs ? a.q_rows : a.batch * a.q_rows) * a.heads;
            plan.bytes = (size_t)a.chunks * plan.part_rows * (a.dim * sizeof(float) + sizeof(float2));
        } else {
            a.chunks = 1;
            a.chunk = 1 << 30;
        }
    }
    a.part_rows = plan.part_rows;
    return plan;
}

static bool nothing_to_do(const AttnArgs& a) { return a.batch == 0 || a.q_rows == 0; }
static int operands_given(const AttnArgs& a) {
    HRS_REQUIRE(a.q && a.out && (a.k_rows == 0 || (a.k && a.v)), "hrs_attention: null operand");
    return HRS_OK;
}

extern "C" int hrs_attention_workspace(hrs_ctx* ctx, const hrs_attention_args* p, size_t* bytes) {
    HRS_REQUIRE(ctx && p && bytes, "hrs_attention_workspace: null argument");
    *bytes = 0;
    AttnArgs a;
    int rc = attention_args(p, a);
    if (rc || nothing_to_do(a) || (rc = operands_given(a))) return rc;
    *bytes = plan_attention(ctx, p, a, true).bytes;
    return HRS_OK;
}

extern "C" int hrs_attention(hrs_ctx* ctx, const hrs_attention_args* p, void* stream) {
    HRS_REQUIRE(ctx && p, "hrs_attention: null argument");
    AttnArgs a;
    int rc = attention_args(p, a);
    if (rc || nothing_to_do(a) || (rc = operands_given(a))) return rc;
    HRS_REQUIRE(a.out != a.q && a.out != a.k && a.out != a.v, "hrs_attention: out may not be an input");
    const uintptr_t at = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.out;
    HRS_REQUIRE(at % 2 == 0, "hrs_attention: an operand is not aligned to its elements");
    const AttnPlan plan = plan_attention(ctx, p, a, at % 16 == 0);
    if (plan.bytes) {
        HRS_REQUIRE(p->workspace && p->workspace_bytes >= plan.bytes && (uintptr_t)p->workspace % 16 == 0,
                    "hrs_attention: a workspace of %zu bytes (given: %zu), 16-byte aligned, is needed", plan.bytes, p->workspace ? p->workspace_bytes : (size_t)0);
        a.part = (float*)p->workspace;
        a.part_ml = (float2*)(a.part + (size_t)a.chunks * plan.part_rows * a.dim);
    }
    hrs_device_scope dev(ctx->device);
    HRS_CHECK_HIP(dev.err);
    // as many documents per launch as a grid holds (less than 2^32 threads)
    const int64_t each = (int64_t)a.kv_heads * a.chunks * (plan.few ? 1 : a.tiles), most = each < (1 << 23) ? (1 << 23) / each : 1;
    for (int b0 = 0; b0 < p->batch; b0 += (int)most) {
        a.b0 = b0;
        a.batch = p->batch - b0 < most ? p->batch - b0 : (int)most;
        rc = p->dtype == HRS_TYPE_BF16 ? launch_type<__bf16>(ctx, a, plan, (hipStream_t)stream) : launch_type<_Float16>(ctx, a, plan, (hipStream_t)stream);
        if (rc) return rc;
    }
    return HRS_OK;
}
