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
    int causal, reach;
    float scale2;             // scale log2 e
    float cap2, cap_in;       // cap log2 e; 2 log2 e scale / cap
};

enum { BIAS_NONE = 0, BIAS_SLOPE = 1, BIAS_TABLE = 2 };
#define LOG2E 1.44269504088896f

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

// Where 16-byte piece p of row i lies in its row of DP elements.  K: 8 consecutive rows, same piece -> 8 bank groups.
// V: 4 consecutive rows, two pieces -> 8 bank groups.
template <int DP>
__device__ __forceinline__ int place_k(int i, int p) { return DP == 32 ? p ^ ((i >> 1) & 3) : p ^ (i & 7); }
template <int DP>
__device__ __forceinline__ int place_v(int i, int p) { return DP == 32 ? p ^ (i & 2) : p ^ ((i & 3) << 1); }

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

// Score of one (query, key) pair in base 2: s is q . k, d = j - p_i.
template <int BIAS, bool CAP>
__device__ __forceinline__ float score2(const AttnArgs& a, float s, float slope2, const float* table, int d) {
    float x = CAP ? fmaf(-2.f * a.cap2, rcp_hw(1.f + exp2_hw(s * a.cap_in)), a.cap2) : s * a.scale2;
    if constexpr (BIAS == BIAS_SLOPE) x = fmaf(-slope2, fabsf((float)d), x);
    if constexpr (BIAS == BIAS_TABLE) {
        const int at = d < -a.reach ? -a.reach : d > a.reach ? a.reach : d;
        const float t = table[at];
        // a finite entry stays finite, also the type's lowest value (log2 e times it would be -inf)
        x += fmaxf(t * LOG2E, fminf(t, -1e30f));
    }
    return x;
}

template <typename T, int DP, int BIAS, bool CAP>
__global__ __launch_bounds__(256) void k_attend(AttnArgs a) {
    typedef typename vec_of<T>::x8 x8;
    constexpr int KT = DP <= 128 ? 64 : 32, PPR = DP / 8, NB = KT / 32, ND = DP / 32, NS = DP / 16;
    __shared__ __attribute__((aligned(16))) char kl[KT * DP * 2];
    __shared__ __attribute__((aligned(16))) char vl[KT * DP * 2];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, h = lane >> 5, c32 = lane & 31;
    int id = blockIdx.x;
    const int t0 = id % a.tiles;
    id /= a.tiles;
    const int hk = id % a.kv_heads, b = id / a.kv_heads;
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
                const int64_t j = j0 + i < dr.lk ? j0 + i : dr.lk - 1;  // what stands behind the document is never read
                const int left = a.dim - p * 8;
                *(x8*)(kl + i * (DP * 2) + place_k<DP>(i, p) * 16) = load8_any<T>(kbase + j * a.k_st + p * 8, left);
                *(x8*)(vl + i * (DP * 2) + place_v<DP>(i, p) * 16) = load8_any<T>(vbase + j * a.v_st + p * 8, left);
            }
            __syncthreads();
            f32x16 s[NB];
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                s[n] = (f32x16)(0.f);
                const int i = n * 32 + c32;
#pragma unroll
                for (int t = 0; t < NS; ++t) s[n] = mfma32(*(const x8*)(kl + i * (DP * 2) + place_k<DP>(i, 2 * t + h) * 16), qf[t], s[n]);
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
            const float base = m_new == -INFINITY ? 0.f : m_new;  // nothing seen so far: every weight is exp2(-inf) = 0
            const float keep = exp2_hw(m - base);
            m = m_new;
            l *= keep;
#pragma unroll
            for (int i = 0; i < ND; ++i) acc[i] *= keep;
            x8 pf[2 * NB];
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float w = exp2_hw(s[n][r] - base);
                    l += w;
                    pf[2 * n + (r >> 3)][r & 7] = (T)w;
                }
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
                        vf.half[e] = lds_read_tr(vl + key * (DP * 2) + place_v<DP>(key, col >> 3) * 16 + (col & 7) * 2);
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
                        for (int e = 0; e < 4; ++e) o[e] = (T)(acc[i][4 * g + e] * inv);
                        __builtin_memcpy(op + d, o, 8);
                    }
                }
        }
    }
}

// ---- host side ---------------------------------------------------------------------------------------
template <typename T, int DP, int BIAS, bool CAP>
static int launch_attend(const AttnArgs& a, hipStream_t st) {
    const int64_t grid = (int64_t)a.batch * a.kv_heads * a.tiles;
    HRS_REQUIRE(grid < (1ll << 31), "hrs_attention: %lld workgroups", (long long)grid);
    hipLaunchKernelGGL((k_attend<T, DP, BIAS, CAP>), dim3((unsigned)grid), dim3(256), 0, st, a);
    HRS_CHECK_HIP(hipGetLastError());
    return HRS_OK;
}
template <typename T, int DP>
static int launch_attend_form(const AttnArgs& a, hipStream_t st) {
    const bool cap = a.cap2 > 0.f;
    if (a.table) return cap ? launch_attend<T, DP, BIAS_TABLE, true>(a, st) : launch_attend<T, DP, BIAS_TABLE, false>(a, st);
    if (a.slopes) return cap ? launch_attend<T, DP, BIAS_SLOPE, true>(a, st) : launch_attend<T, DP, BIAS_SLOPE, false>(a, st);
    return cap ? launch_attend<T, DP, BIAS_NONE, true>(a, st) : launch_attend<T, DP, BIAS_NONE, false>(a, st);
}
template <typename T>
static int launch_attend_dim(const AttnArgs& a, hipStream_t st) {
    if (a.dim <= 32) return launch_attend_form<T, 32>(a, st);
    if (a.dim <= 64) return launch_attend_form<T, 64>(a, st);
    if (a.dim <= 128) return launch_attend_form<T, 128>(a, st);
    return launch_attend_form<T, 256>(a, st);
}

static int attention_args(const hrs_attention_args* p, AttnArgs& a) {
    HRS_REQUIRE(p->dtype == HRS_TYPE_BF16 || p->dtype == HRS_TYPE_FP16, "hrs_attention: type %d is neither bf16 nor fp16", p->dtype);
    HRS_REQUIRE(p->batch >= 0 && p->q_heads >= 1 && p->kv_heads >= 1 && p->q_heads % p->kv_heads == 0,
                "hrs_attention: batch=%d, q_heads=%d, kv_heads=%d (query heads must be a multiple of key heads)", p->batch, p->q_heads, p->kv_heads);
    HRS_REQUIRE(p->head_dim >= 8 && p->head_dim <= 256 && p->head_dim % 8 == 0, "hrs_attention: head_dim=%d must be a multiple of 8 in [8, 256]", p->head_dim);
    HRS_REQUIRE(p->q_rows >= 0 && p->k_rows >= 0 && p->q_rows < (1ll << 30) && p->k_rows < (1ll << 30), "hrs_attention: q_rows=%lld, k_rows=%lld",
                (long long)p->q_rows, (long long)p->k_rows);
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
    }
    return HRS_OK;
}

extern "C" int hrs_attention(hrs_ctx* ctx, const hrs_attention_args* p, void* stream) {
    HRS_REQUIRE(ctx && p, "hrs_attention: null argument");
    AttnArgs a;
    int rc = attention_args(p, a);
    if (rc) return rc;
    if (a.batch == 0 || a.q_rows == 0) return HRS_OK;
    HRS_REQUIRE(a.q && a.out && (a.k_rows == 0 || (a.k && a.v)), "hrs_attention: null operand");
    HRS_REQUIRE(a.out != a.q && a.out != a.k && a.out != a.v, "hrs_attention: out may not be an input");
    HRS_REQUIRE(((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.out) % 2 == 0, "hrs_attention: an operand is not aligned to its elements");
    hrs_device_scope dev(ctx->device);
    HRS_CHECK_HIP(dev.err);
    int64_t longest = p->max_q > 0 && p->max_q < a.q_rows ? p->max_q : a.q_rows;
    if (a.q_offs && p->max_q <= 0) longest = (a.q_rows + a.batch - 1) / a.batch;  // without a hint: twice the mean
    a.tiles = (int)((longest * a.group + 127) / 128);
    return p->dtype == HRS_TYPE_BF16 ? launch_attend_dim<__bf16>(a, (hipStream_t)stream) : launch_attend_dim<_Float16>(a, (hipStream_t)stream);
}

extern "C" int hrs_attention_workspace(hrs_ctx* ctx, const hrs_attention_args* p, size_t* bytes) {
    HRS_REQUIRE(ctx && p && bytes, "hrs_attention_workspace: null argument");
    AttnArgs a;
    int rc = attention_args(p, a);
    if (rc) return rc;
    *bytes = 0;
    return HRS_OK;
}
