// Sentence encoders of other widths than the one hrs_encoder.hip is built for, out of the layer's operators (hrs_linear,
// hrs_attention, hrs_layer_norm) with an embedding gather in front and the pooling behind (the same forward pass as there:
// post-LayerNorm blocks, erf-GELU, mean pooling, L2 normalisation; scripts/chromadb_helper.py:58-71).
//
// Tokens are rows; a document is a run of rows, packed back to back (offsets) or in a padded row of S (lengths).  Padded
// rows are computed along and never read by a valid one.  Activations are bf16, sums and statistics fp32.
#include "hrs_ops.h"

struct hrs_encoder_any {
    hrs_encoder_config cfg;
    float *word = nullptr, *pos = nullptr, *type0 = nullptr, *emb_g = nullptr, *emb_b = nullptr;
    struct Layer {
        __bf16 *wqkv = nullptr, *wo = nullptr, *wi = nullptr, *wd = nullptr;
        float *bqkv = nullptr, *bo = nullptr, *bi = nullptr, *bd = nullptr, *ln1g = nullptr, *ln1b = nullptr, *ln2g = nullptr, *ln2b = nullptr;
    };
    std::vector<Layer> layer;
    std::vector<void*> owned;
    hrs_workspace ws;
};

// First row and length of document b, inside the T rows.
struct EncDoc {
    int row, len;
};
__device__ __forceinline__ EncDoc enc_doc(const int* offs, const int* lens, int b, int S, int T) {
    EncDoc d;
    if (offs) {
        const int a = offs[b], e = offs[b + 1];
        d.row = a < 0 ? 0 : a > T ? T : a;
        d.len = (e < d.row ? d.row : e > T ? T : e) - d.row;
    } else {
        const int n = lens[b];
        d.row = b * S;
        d.len = n < 0 ? 0 : n > S ? S : n;
    }
    return d;
}

// x = LayerNorm(word[id] + pos[i] + type), one wave per token, the sum in fp32 registers.  CH pieces of 8 per lane.
template <int CH>
__global__ __launch_bounds__(256) void k_embed_norm(const int* __restrict__ ids, const int* __restrict__ offs, const int* __restrict__ lens, const float* __restrict__ word,
                                                    const float* __restrict__ pos, const float* __restrict__ type0, const float* __restrict__ g, const float* __restrict__ b, int S,
                                                    int T, int H, int vocab, int max_pos, float eps, __bf16* __restrict__ x) {
    typedef vec_of<__bf16>::x8 x8;
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const EncDoc d = enc_doc(offs, lens, blockIdx.y, S, T);
    const int rows = offs ? d.len : S;
    for (int i = blockIdx.x * 4 + wv; i < rows; i += gridDim.x * 4) {
        const int t = d.row + i;
        int id = ids[t];
        if (id < 0 || id >= vocab) id = 0;
        const int p = i < max_pos ? i : max_pos - 1;
        float z[CH][8], s = 0.f;
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            const int c = (j * 64 + lane) * 8;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                z[j][e] = c < H ? word[(size_t)id * H + c + e] + pos[(size_t)p * H + c + e] + type0[c + e] : 0.f;
                s += z[j][e];
            }
        }
        const float mean = wave_sum(s) / (float)H;
        float v = 0.f;
#pragma unroll
        for (int j = 0; j < CH; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float dv = z[j][e] - mean;
                v += (j * 64 + lane) * 8 < H ? dv * dv : 0.f;
            }
        const float rstd = 1.f / sqrtf(wave_sum(v) / (float)H + eps);
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            const int c = (j * 64 + lane) * 8;
            if (c < H) {
                x8 o;
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] = (__bf16)fmaf((z[j][e] - mean) * rstd, g[c + e], b[c + e]);
                *(x8*)(x + (size_t)t * H + c) = o;
            }
        }
    }
}

// Mean over a document's tokens, L2 normalised: one workgroup per document; thread (phase, piece) sums the tokens phase,
// phase + phases, .. of its 8 features, the phases meet in LDS in order.  A document without tokens gives zeros.
__global__ __launch_bounds__(256) void k_pool_rows(const __bf16* __restrict__ x, const int* __restrict__ offs, const int* __restrict__ lens, int S, int T, int H, float* __restrict__ out) {
    typedef vec_of<__bf16>::x8 x8;
    extern __shared__ float sums[];  // [phases][H], then 4 partial norms
    const EncDoc d = enc_doc(offs, lens, blockIdx.x, S, T);
    const int pieces = H / 8, phases = pieces >= 256 ? 1 : 256 / pieces;
    for (int u = threadIdx.x; u < pieces * phases; u += 256) {
        const int ph = u / pieces, c = (u - ph * pieces) * 8;
        float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int i = ph; i < d.len; i += phases) {
            const x8 v = *(const x8*)(x + (size_t)(d.row + i) * H + c);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] += (float)v[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) sums[ph * H + c + e] = s[e];
    }
    __syncthreads();
    const float per = d.len > 0 ? 1.f / (float)d.len : 0.f;
    float q = 0.f;
    for (int c = threadIdx.x; c < H; c += 256) {
        float s = 0.f;
        for (int ph = 0; ph < phases; ++ph) s += sums[ph * H + c];
        s *= per;
        sums[c] = s;  // (own column: nobody else reads it before the next barrier)
        q = fmaf(s, s, q);
    }
    q = wave_sum(q);
    float* norms = sums + phases * H;
    if ((threadIdx.x & 63) == 0) norms[threadIdx.x >> 6] = q;
    __syncthreads();
    const float n = fmaxf(sqrtf((norms[0] + norms[1]) + (norms[2] + norms[3])), 1e-12f);
    for (int c = threadIdx.x; c < H; c += 256) out[(size_t)blockIdx.x * H + c] = sums[c] / n;
}

__global__ void k_round_bf16(const float* __restrict__ in, int64_t n, __bf16* __restrict__ out) {
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) out[i] = (__bf16)in[i];
}

// ---- host side ---------------------------------------------------------------------------------------
static int any_alloc(hrs_encoder_any* e, void** p, size_t bytes) {
    hipError_t err = hipMalloc(p, bytes);
    if (err != hipSuccess) {
        hrs_set_error("encoder allocation of %zu bytes failed: %s", bytes, hipGetErrorString(err));
        return HRS_ERR_NOMEM;
    }
    e->owned.push_back(*p);
    return HRS_OK;
}
static int any_f32(hrs_encoder_any* e, float** dst, std::initializer_list<const float*> parts, size_t n, hipStream_t st) {
    int rc = any_alloc(e, (void**)dst, parts.size() * n * sizeof(float));
    if (rc) return rc;
    size_t at = 0;
    for (const float* p : parts) {
        HRS_CHECK_HIP(hipMemcpyAsync(*dst + at, p, n * sizeof(float), hipMemcpyDeviceToDevice, st));
        at += n;
    }
    return HRS_OK;
}
static int any_bf16(hrs_encoder_any* e, __bf16** dst, std::initializer_list<const float*> parts, size_t n, hipStream_t st) {
    int rc = any_alloc(e, (void**)dst, parts.size() * n * sizeof(__bf16));
    if (rc) return rc;
    size_t at = 0;
    for (const float* p : parts) {
        const size_t blocks = (n + 255) / 256;
        hipLaunchKernelGGL(k_round_bf16, dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(256), 0, st, p, (int64_t)n, *dst + at);
        HRS_CHECK_HIP(hipGetLastError());
        at += n;
    }
    return HRS_OK;
}

void hrs_encoder_any_release(hrs_encoder_any* e) {
    for (void* p : e->owned) (void)hipFree(p);
    if (e->ws.ptr) (void)hipFree(e->ws.ptr);
    delete e;
}

static int any_load(hrs_encoder_any* e, const float* const* w, hipStream_t st) {
    const hrs_encoder_config& c = e->cfg;
    const size_t H = c.hidden, I = c.inter;
    int rc;
    if ((rc = any_f32(e, &e->word, {w[0]}, (size_t)c.vocab * H, st)) || (rc = any_f32(e, &e->pos, {w[1]}, (size_t)c.max_pos * H, st)) || (rc = any_f32(e, &e->type0, {w[2]}, H, st)) ||
        (rc = any_f32(e, &e->emb_g, {w[3]}, H, st)) || (rc = any_f32(e, &e->emb_b, {w[4]}, H, st)))
        return rc;
    for (int l = 0; l < c.layers; ++l) {
        const float* const* p = w + 5 + 16 * l;  // q_w q_b k_w k_b v_w v_b o_w o_b ln1_gamma ln1_beta i_w i_b d_w d_b ln2_gamma ln2_beta
        hrs_encoder_any::Layer& L = e->layer[l];
        if ((rc = any_bf16(e, &L.wqkv, {p[0], p[2], p[4]}, H * H, st)) || (rc = any_f32(e, &L.bqkv, {p[1], p[3], p[5]}, H, st)) || (rc = any_bf16(e, &L.wo, {p[6]}, H * H, st)) ||
            (rc = any_f32(e, &L.bo, {p[7]}, H, st)) || (rc = any_f32(e, &L.ln1g, {p[8]}, H, st)) || (rc = any_f32(e, &L.ln1b, {p[9]}, H, st)) ||
            (rc = any_bf16(e, &L.wi, {p[10]}, I * H, st)) || (rc = any_f32(e, &L.bi, {p[11]}, I, st)) || (rc = any_bf16(e, &L.wd, {p[12]}, H * I, st)) ||
            (rc = any_f32(e, &L.bd, {p[13]}, H, st)) || (rc = any_f32(e, &L.ln2g, {p[14]}, H, st)) || (rc = any_f32(e, &L.ln2b, {p[15]}, H, st)))
            return rc;
    }
    return HRS_OK;
}

int hrs_encoder_any_check(const hrs_encoder_config* cfg) {
    HRS_REQUIRE(cfg->hidden >= 8 && cfg->hidden <= 4096 && cfg->hidden % 8 == 0, "hrs_encoder_load: hidden=%d must be a multiple of 8 in [8, 4096]", cfg->hidden);
    HRS_REQUIRE(cfg->heads >= 1 && cfg->hidden % cfg->heads == 0 && cfg->hidden / cfg->heads % 8 == 0 && cfg->hidden / cfg->heads <= 256,
                "hrs_encoder_load: hidden=%d over heads=%d is not a head width that is a multiple of 8, at most 256", cfg->hidden, cfg->heads);
    HRS_REQUIRE(cfg->inter >= 1 && cfg->inter <= (1 << 20), "hrs_encoder_load: intermediate size %d", cfg->inter);
    HRS_REQUIRE(cfg->layers >= 1 && cfg->layers <= 256, "hrs_encoder_load: layers=%d outside [1, 256]", cfg->layers);
    HRS_REQUIRE(cfg->vocab > 0 && cfg->max_pos > 0, "hrs_encoder_load: bad vocabulary / position table size");
    return HRS_OK;
}

int hrs_encoder_any_load(const hrs_encoder_config* cfg, const float* const* w, void* stream, hrs_encoder_any** out) {
    hrs_encoder_any* e = new hrs_encoder_any();
    e->cfg = *cfg;
    e->layer.resize(cfg->layers);
    const int rc = any_load(e, w, (hipStream_t)stream);
    if (rc) {
        (void)hipStreamSynchronize((hipStream_t)stream);  // copies into what is freed now may be under way
        hrs_encoder_any_release(e);
        return rc;
    }
    *out = e;
    return HRS_OK;
}

// offs_dev (packed, T rows) or lens_dev (padded, T = B S rows); longest: of a document (packed: a hint)
int hrs_encoder_any_run(hrs_ctx* ctx, hrs_encoder_any* e, const int32_t* ids_dev, const int32_t* offs_dev, const int32_t* lens_dev, int B, int S, int64_t T, int64_t longest, float* out_dev,
                        hipStream_t st) {
    const hrs_encoder_config& c = e->cfg;
    const int H = c.hidden, I = c.inter;
    size_t off = 0;
    auto carve = [&](size_t bytes) {
        const size_t o = off;
        off += (bytes + 255) / 256 * 256;
        return o;
    };
    const size_t o_x = carve((size_t)T * H * 2), o_y = carve((size_t)T * H * 2), o_qkv = carve((size_t)T * 3 * H * 2), o_ctx = carve((size_t)T * H * 2), o_h = carve((size_t)T * I * 2);
    hrs_attention_args at;
    memset(&at, 0, sizeof(at));
    at.dtype = HRS_TYPE_BF16;
    at.batch = B;
    at.q_heads = at.kv_heads = c.heads;
    at.head_dim = H / c.heads;
    at.scale = 1.f / sqrtf((float)at.head_dim);
    const int64_t strides[3] = {(int64_t)S * 3 * H, (int64_t)3 * H, at.head_dim};
    for (int i = 0; i < 3; ++i) at.q_stride[i] = at.k_stride[i] = at.v_stride[i] = strides[i];
    at.q_rows = at.k_rows = offs_dev ? T : S;
    at.q_offs = at.k_offs = offs_dev;
    at.q_lens = at.k_lens = lens_dev;
    at.max_q = at.max_k = longest;
    at.q = at.k = at.v = at.out = out_dev;  // (asking for the workspace's size only takes them not to be null)
    size_t need = 0;
    int rc = hrs_attention_workspace(ctx, &at, &need);
    if (rc) return rc;
    const size_t o_att = carve(need);
    if ((rc = hrs_ws_reserve(ctx, &e->ws, off))) return rc;
    char* ws = (char*)e->ws.ptr;
    __bf16 *x = (__bf16*)(ws + o_x), *y = (__bf16*)(ws + o_y), *qkv = (__bf16*)(ws + o_qkv), *cx = (__bf16*)(ws + o_ctx), *hb = (__bf16*)(ws + o_h);
    at.q = qkv;
    at.k = qkv + H;
    at.v = qkv + 2 * H;
    at.out = cx;
    at.workspace = need ? ws + o_att : nullptr;
    at.workspace_bytes = need;

    int64_t gx = (longest + 3) / 4;
    gx = gx < 1 ? 1 : gx > 4096 ? 4096 : gx;
    for (int b0 = 0; b0 < B; b0 += 65535) {  // grid.y holds 65535 documents
        const dim3 grid((unsigned)gx, (unsigned)(B - b0 < 65535 ? B - b0 : 65535));
        const int* ids = offs_dev ? ids_dev : ids_dev + (size_t)b0 * S;
        const int *offs = offs_dev ? offs_dev + b0 : nullptr, *lens = lens_dev ? lens_dev + b0 : nullptr;
        __bf16* to = offs_dev ? x : x + (size_t)b0 * S * H;
        auto embed = H <= 512 ? k_embed_norm<1> : H <= 1024 ? k_embed_norm<2> : H <= 2048 ? k_embed_norm<4> : k_embed_norm<8>;
        hipLaunchKernelGGL(embed, grid, dim3(256), 0, st, ids, offs, lens, e->word, e->pos, e->type0, e->emb_g, e->emb_b, S, (int)T, H, c.vocab, c.max_pos, c.eps, to);
    }
    HRS_CHECK_HIP(hipGetLastError());
    for (int l = 0; l < c.layers; ++l) {
        const hrs_encoder_any::Layer& L = e->layer[l];
        const int bf = HRS_TYPE_BF16;
        if ((rc = hrs_linear(ctx, bf, x, H, L.wqkv, H, L.bqkv, nullptr, 0, HRS_ACT_NONE, qkv, 3 * H, T, 3 * H, H, st)) || (rc = hrs_attention(ctx, &at, st)) ||
            (rc = hrs_linear(ctx, bf, cx, H, L.wo, H, L.bo, x, H, HRS_ACT_NONE, y, H, T, H, H, st)) || (rc = hrs_layer_norm(ctx, bf, y, H, nullptr, 0, L.ln1g, L.ln1b, c.eps, y, H, T, H, st)) ||
            (rc = hrs_linear(ctx, bf, y, H, L.wi, H, L.bi, nullptr, 0, HRS_ACT_GELU, hb, I, T, I, H, st)) ||
            (rc = hrs_linear(ctx, bf, hb, I, L.wd, I, L.bd, y, H, HRS_ACT_NONE, x, H, T, H, I, st)) || (rc = hrs_layer_norm(ctx, bf, x, H, nullptr, 0, L.ln2g, L.ln2b, c.eps, x, H, T, H, st)))
            return rc;
    }
    const int pieces = H / 8, phases = pieces >= 256 ? 1 : 256 / pieces;
    const int most = 1 << 23;  // documents per launch: a grid holds less than 2^32 threads
    for (int b0 = 0; b0 < B; b0 += most) {
        const int *offs = offs_dev ? offs_dev + b0 : nullptr, *lens = lens_dev ? lens_dev + b0 : nullptr;
        hipLaunchKernelGGL(k_pool_rows, dim3(B - b0 < most ? B - b0 : most), dim3(256), (phases * H + 4) * sizeof(float), st, offs_dev ? x : x + (size_t)b0 * S * H, offs, lens, S, (int)T, H,
                           out_dev + (size_t)b0 * H);
    }
    HRS_CHECK_HIP(hipGetLastError());
    return HRS_OK;
}
