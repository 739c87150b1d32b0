// hrs_linear: y = act(x W^T + b) + r, the matrix product of an encoder layer with its whole epilogue.
//
// x [M, K], W [N, K], y and r [M, N], bf16 or fp16, rows at any stride; b fp32 [N].  Products are summed in fp32 on the
// matrix cores, bias, activation and residual are applied to the fp32 sum, and the result is rounded once.
//
// Tiles are computed as W x^T (features on the rows of the matrix instruction, tokens on its columns), so that a lane
// holds consecutive features of one token.  Which feature sits on which row of which instruction is free, and chosen so
// that the 4 NT registers of a lane are 4 NT consecutive features: y leaves in 16-byte pieces straight from the
// accumulators.
#include "hrs_ops.h"

struct LinearArgs {
    const void* x;
    const void* w;
    const float* bias;   // [N], may be null
    const void* resid;   // [M, N], may be null
    void* y;
    int64_t ldx, ldw, ldr, ldy;  // elements
    int64_t M;
    int N, K;
};

// One lane's 4 NT consecutive features n .. of token m: bias, activation, residual, one rounding.
template <typename T, int NT, int ACT>
__device__ __forceinline__ void linear_store(const LinearArgs& a, int64_t m, int n, const f32x4 (&acc)[NT], const float (&bias)[4 * NT]) {
    constexpr int E = 4 * NT;
    if (m >= a.M || n >= a.N) return;
    const int left = a.N - n;
    T* y = (T*)a.y + m * a.ldy + n;
    float v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = activate<ACT>(acc[e / 4][e % 4] + bias[e]);
    const T* r = a.resid ? (const T*)a.resid + m * a.ldr + n : nullptr;
    if (left >= E) {
        T o[E];
        if (r) {
            T rv[E];
            __builtin_memcpy(rv, r, sizeof(rv));
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] += (float)rv[e];
        }
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = (T)v[e];
        __builtin_memcpy(y, o, sizeof(o));
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (e < left) y[e] = (T)(r ? v[e] + (float)r[e] : v[e]);
    }
}

template <int E>
__device__ __forceinline__ void load_bias(const LinearArgs& a, int n, float (&bias)[E]) {
#pragma unroll
    for (int e = 0; e < E; ++e) bias[e] = (a.bias && n + e < a.N) ? a.bias[n + e] : 0.f;
}

// ---- tiles staged through LDS ------------------------------------------------------------------------
// Depth advances by 64: an LDS row is 128 bytes, eight 16-byte pieces, piece p of row i stored at p ^ key(i), so that
// the 8 rows (16 lanes) a fragment read touches together lie in 8 different bank groups.
// Rows of x are read in order: key = i % 8.  Rows of W are read as (r / 4) 4 NT + 4 t + r % 4 for r = 0 .. 15.
__device__ __forceinline__ int key_x(int i) { return i & 7; }
template <int NT>
__device__ __forceinline__ int key_w(int i) { return (i & 3) | (((i / (4 * NT)) & 1) << 2); }

template <typename T, int BM, int BN, int WR, int WC, int ACT>
__global__ __launch_bounds__(64 * WR * WC) void k_linear_any(LinearArgs a) {
    typedef typename vec_of<T>::x8 x8;
    constexpr int NTHR = 64 * WR * WC, MT = BM / WR / 16, NT = BN / WC / 16;
    constexpr int PX = BM * 8 / NTHR, PW = BN * 8 / NTHR;  // pieces a thread moves per stage
    __shared__ __attribute__((aligned(16))) char lds[(BM + BN) * 128];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, qd = lane >> 4, r16 = lane & 15;
    const int64_t m0 = (int64_t)blockIdx.y * BM;
    const int n0 = blockIdx.x * BN;
    const int wm = (wv / WC) * (BM / WR), wn = (wv % WC) * (BN / WC);
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = (f32x4)(0.f);

    for (int k0 = 0; k0 < a.K; k0 += 64) {
        __syncthreads();  // the tile before has been read
#pragma unroll
        for (int j = 0; j < PX + PW; ++j) {
            const bool isx = j < PX;
            const int id = (isx ? j : j - PX) * NTHR + tid, row = id >> 3, p = id & 7;
            const int64_t grow = isx ? m0 + row : n0 + row;
            const int left = grow < (isx ? a.M : (int64_t)a.N) ? a.K - (k0 + p * 8) : 0;
            const T* src = isx ? (const T*)a.x + grow * a.ldx : (const T*)a.w + grow * a.ldw;
            const x8 v = load8_any<T>(src + k0 + p * 8, left);
            const int at = (isx ? row : BM + row) * 128 + ((p ^ (isx ? key_x(row) : key_w<NT>(row))) << 4);
            *(x8*)(lds + at) = v;
        }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            x8 wf[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int row = wn + (r16 >> 2) * (4 * NT) + t * 4 + (r16 & 3);
                wf[t] = *(const x8*)(lds + (BM + row) * 128 + (((s * 4 + qd) ^ key_w<NT>(row)) << 4));
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int row = wm + i * 16 + r16;
                const x8 xf = *(const x8*)(lds + row * 128 + (((s * 4 + qd) ^ key_x(row)) << 4));
#pragma unroll
                for (int t = 0; t < NT; ++t) acc[i][t] = mfma16(wf[t], xf, acc[i][t]);
            }
        }
    }
    const int n = n0 + wn + qd * (4 * NT);
    float bias[4 * NT];
    load_bias(a, n, bias);
#pragma unroll
    for (int i = 0; i < MT; ++i) linear_store<T, NT, ACT>(a, m0 + wm + i * 16 + r16, n, acc[i], bias);
}

// ---- host side ---------------------------------------------------------------------------------------
template <typename T, int ACT>
static int launch_linear(hrs_ctx* ctx, const LinearArgs& a, hipStream_t st) {
    (void)ctx;
    const int64_t gm = (a.M + 63) / 64;
    const int gn = (a.N + 63) / 64;
    for (int64_t g0 = 0; g0 < gm; g0 += 65535) {  // grid.y holds 65535 rows of tiles
        LinearArgs p = a;
        const int64_t m0 = g0 * 64;
        p.x = (const T*)a.x + m0 * a.ldx;
        p.y = (T*)a.y + m0 * a.ldy;
        if (a.resid) p.resid = (const T*)a.resid + m0 * a.ldr;
        p.M = a.M - m0;
        const int64_t rows = gm - g0 < 65535 ? gm - g0 : 65535;
        hipLaunchKernelGGL((k_linear_any<T, 64, 64, 2, 2, ACT>), dim3((unsigned)gn, (unsigned)rows), dim3(256), 0, st, p);
        HRS_CHECK_HIP(hipGetLastError());
    }
    return HRS_OK;
}

template <typename T>
static int launch_linear_act(hrs_ctx* ctx, const LinearArgs& a, int act, hipStream_t st) {
    switch (act) {
        case ACT_RELU: return launch_linear<T, ACT_RELU>(ctx, a, st);
        case ACT_GELU: return launch_linear<T, ACT_GELU>(ctx, a, st);
        case ACT_GELU_TANH: return launch_linear<T, ACT_GELU_TANH>(ctx, a, st);
        case ACT_SILU: return launch_linear<T, ACT_SILU>(ctx, a, st);
        case ACT_TANH: return launch_linear<T, ACT_TANH>(ctx, a, st);
        default: return launch_linear<T, ACT_NONE>(ctx, a, st);
    }
}

extern "C" int hrs_linear(hrs_ctx* ctx, int dtype, const void* x_dev, int64_t ldx, const void* w_dev, int64_t ldw,
                          const float* bias_dev, const void* resid_dev, int64_t ldr, int act, void* y_dev, int64_t ldy,
                          int64_t M, int64_t N, int64_t K, void* stream) {
    HRS_REQUIRE(ctx, "hrs_linear: null ctx");
    HRS_REQUIRE(dtype == HRS_TYPE_BF16 || dtype == HRS_TYPE_FP16, "hrs_linear: type %d is neither bf16 nor fp16", dtype);
    HRS_REQUIRE(act >= ACT_NONE && act <= ACT_TANH, "hrs_linear: unknown activation %d", act);
    HRS_REQUIRE(M >= 0 && N >= 0 && K >= 0 && M < (1ll << 31) && N < (1 << 30) && K < (1 << 30), "hrs_linear: M=%lld, N=%lld, K=%lld", (long long)M, (long long)N, (long long)K);
    if (M == 0 || N == 0) return HRS_OK;
    HRS_REQUIRE(y_dev && (K == 0 || (x_dev && w_dev)), "hrs_linear: null operand");
    HRS_REQUIRE(ldx >= 0 && ldw >= 0 && ldr >= 0, "hrs_linear: negative row stride");
    HRS_REQUIRE(ldy >= N || M == 1, "hrs_linear: rows of y overlap (stride %lld, N=%lld)", (long long)ldy, (long long)N);
    HRS_REQUIRE(y_dev != x_dev && y_dev != w_dev, "hrs_linear: y may not be x or W");
    HRS_REQUIRE(((uintptr_t)x_dev | (uintptr_t)w_dev | (uintptr_t)y_dev | (uintptr_t)resid_dev) % 2 == 0 && (uintptr_t)bias_dev % 4 == 0,
                "hrs_linear: an operand is not aligned to its elements");
    hrs_device_scope dev(ctx->device);
    HRS_CHECK_HIP(dev.err);
    LinearArgs a;
    a.x = x_dev;
    a.w = w_dev;
    a.bias = bias_dev;
    a.resid = resid_dev;
    a.y = y_dev;
    a.ldx = ldx;
    a.ldw = ldw;
    a.ldr = ldr;
    a.ldy = ldy;
    a.M = M;
    a.N = (int)N;
    a.K = (int)K;
    return dtype == HRS_TYPE_BF16 ? launch_linear_act<__bf16>(ctx, a, act, (hipStream_t)stream) : launch_linear_act<_Float16>(ctx, a, act, (hipStream_t)stream);
}
