// hrs_layer_norm: y = (z - mean z) / sqrt(var z + eps) * gamma + beta, z = x + r, row by row.
//
// Bound by HBM: x and r are read once and y written once.  A row stays in the registers of the wave (or of the four
// waves) that loaded it, so the variance is the mean of squared deviations from the finished mean -- two passes over
// registers, one over memory -- and not a difference of two large sums.  All of it in fp32; z is not rounded.
#include "hrs_ops.h"

struct NormArgs {
    const void* x;
    const void* resid;  // may be null
    const float* gamma;
    const float* beta;  // may be null
    void* y;
    int64_t ldx, ldr, ldy;
    int64_t M;
    int N;
    float eps;
};

// 8 elements of z at column c of a row, as fp32 (zero where the row has ended)
template <typename T>
__device__ __forceinline__ void load_z(const T* x, const T* r, int c, int N, float (&z)[8]) {
    typedef T x8 __attribute__((ext_vector_type(8)));
    x8 xv = (x8)((T)0.f), rv = (x8)((T)0.f);
    if (c + 8 <= N) {
        __builtin_memcpy(&xv, x + c, sizeof(x8));
        if (r) __builtin_memcpy(&rv, r + c, sizeof(x8));
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c + e < N) {
                xv[e] = x[c + e];
                if (r) rv[e] = r[c + e];
            }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = (float)xv[e] + (float)rv[e];
}

template <typename T>
__device__ __forceinline__ void store_norm(const NormArgs& a, T* y, int c, const float (&z)[8], float mean, float rstd) {
    typedef T x8 __attribute__((ext_vector_type(8)));
    x8 o;
    if (c + 8 <= a.N) {
        float g[8], b[8] = {};
        __builtin_memcpy(g, a.gamma + c, 32);
        if (a.beta) __builtin_memcpy(b, a.beta + c, 32);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = (T)fmaf((z[e] - mean) * rstd, g[e], b[e]);
        __builtin_memcpy(y + c, &o, sizeof(x8));
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c + e < a.N) y[c + e] = (T)fmaf((z[e] - mean) * rstd, a.gamma[c + e], a.beta ? a.beta[c + e] : 0.f);
    }
}

// WPR waves per row, CH pieces of 8 elements per lane: rows of up to 512 CH WPR elements.  65536 x 1024 bf16 with a
// residual: 70 us, 5.7 TB/s (a copy of 2 GiB reaches 4.96; part of the input is still in the 256 MB cache); 12 x 384: 2.7 us.
template <typename T, int CH, int WPR>
__global__ __launch_bounds__(256) void k_layer_norm(NormArgs a) {
    __shared__ float part[2][4];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int64_t row = (int64_t)blockIdx.x * (4 / WPR) + wv / WPR;
    const int wr = wv % WPR;
    if (WPR == 1 && row >= a.M) return;  // (WPR == 4: one row per workgroup, all of them inside)
    const T* x = (const T*)a.x + row * a.ldx;
    const T* r = a.resid ? (const T*)a.resid + row * a.ldr : nullptr;
    float z[CH][8], s = 0.f;
#pragma unroll
    for (int j = 0; j < CH; ++j) load_z<T>(x, r, ((j * WPR + wr) * 64 + lane) * 8, a.N, z[j]);
#pragma unroll
    for (int j = 0; j < CH; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) s += z[j][e];
    s = wave_sum(s);
    if (WPR > 1) {
        if (lane == 0) part[0][wv] = s;
        __syncthreads();
        s = (part[0][0] + part[0][1]) + (part[0][2] + part[0][3]);
    }
    const float mean = s / (float)a.N;
    float v = 0.f;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        const int c = ((j * WPR + wr) * 64 + lane) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float d = z[j][e] - mean;
            v += c + e < a.N ? d * d : 0.f;
        }
    }
    v = wave_sum(v);
    if (WPR > 1) {
        if (lane == 0) part[1][wv] = v;
        __syncthreads();
        v = (part[1][0] + part[1][1]) + (part[1][2] + part[1][3]);
    }
    const float rstd = 1.f / sqrtf(v / (float)a.N + a.eps);
    T* y = (T*)a.y + row * a.ldy;
#pragma unroll
    for (int j = 0; j < CH; ++j) store_norm<T>(a, y, ((j * WPR + wr) * 64 + lane) * 8, z[j], mean, rstd);
}

// Rows too long for registers: one workgroup per row reads it three times (the second and third time from the caches).
template <typename T>
__global__ __launch_bounds__(256) void k_layer_norm_long(NormArgs a) {
    __shared__ float part[2][4];
    const int64_t row = blockIdx.x;
    const T* x = (const T*)a.x + row * a.ldx;
    const T* r = a.resid ? (const T*)a.resid + row * a.ldr : nullptr;
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    float z[8], s = 0.f, v = 0.f;
    for (int c = threadIdx.x * 8; c < a.N; c += 2048) {
        load_z<T>(x, r, c, a.N, z);
        s += ((z[0] + z[1]) + (z[2] + z[3])) + ((z[4] + z[5]) + (z[6] + z[7]));
    }
    s = wave_sum(s);
    if (lane == 0) part[0][wv] = s;
    __syncthreads();
    const float mean = ((part[0][0] + part[0][1]) + (part[0][2] + part[0][3])) / (float)a.N;
    for (int c = threadIdx.x * 8; c < a.N; c += 2048) {
        load_z<T>(x, r, c, a.N, z);
        for (int e = 0; e < 8; ++e) {
            const float d = z[e] - mean;
            v += c + e < a.N ? d * d : 0.f;
        }
    }
    v = wave_sum(v);
    if (lane == 0) part[1][wv] = v;
    __syncthreads();
    const float rstd = 1.f / sqrtf(((part[1][0] + part[1][1]) + (part[1][2] + part[1][3])) / (float)a.N + a.eps);
    T* y = (T*)a.y + row * a.ldy;
    for (int c = threadIdx.x * 8; c < a.N; c += 2048) {
        load_z<T>(x, r, c, a.N, z);
        store_norm<T>(a, y, c, z, mean, rstd);
    }
}

template <typename T>
static int launch_norm(const NormArgs& a, hipStream_t st) {
    const dim3 four((unsigned)((a.M + 3) / 4)), one((unsigned)a.M), block(256);
    if (a.N <= 512)
        hipLaunchKernelGGL((k_layer_norm<T, 1, 1>), four, block, 0, st, a);
    else if (a.N <= 1024)
        hipLaunchKernelGGL((k_layer_norm<T, 2, 1>), four, block, 0, st, a);
    else if (a.N <= 2048)
        hipLaunchKernelGGL((k_layer_norm<T, 4, 1>), four, block, 0, st, a);
    else if (a.N <= 4096)
        hipLaunchKernelGGL((k_layer_norm<T, 2, 4>), one, block, 0, st, a);
    else if (a.N <= 8192)
        hipLaunchKernelGGL((k_layer_norm<T, 4, 4>), one, block, 0, st, a);
    else
        hipLaunchKernelGGL((k_layer_norm_long<T>), one, block, 0, st, a);
    HRS_CHECK_HIP(hipGetLastError());
    return HRS_OK;
}

int hrs_launch_norm(int dtype, const void* x, int64_t ldx, const void* resid, int64_t ldr, const float* gamma, const float* beta,
                    float eps, void* y, int64_t ldy, int64_t M, int N, hipStream_t st) {
    NormArgs a;
    a.gamma = gamma;
    a.beta = beta;
    a.ldx = ldx;
    a.ldr = ldr;
    a.ldy = ldy;
    a.N = N;
    a.eps = eps;
    const int64_t most = 1 << 22, el = dtype == HRS_TYPE_FP32 ? 4 : 2;  // rows per launch: a grid holds less than 2^32 threads
    for (int64_t m0 = 0; m0 < M; m0 += most) {
        a.x = (const char*)x + m0 * ldx * el;
        a.resid = resid ? (const char*)resid + m0 * ldr * el : nullptr;
        a.y = (char*)y + m0 * ldy * el;
        a.M = M - m0 < most ? M - m0 : most;
        const int rc = dtype == HRS_TYPE_BF16 ? launch_norm<__bf16>(a, st) : dtype == HRS_TYPE_FP16 ? launch_norm<_Float16>(a, st) : launch_norm<float>(a, st);
        if (rc) return rc;
    }
    return HRS_OK;
}

extern "C" int hrs_layer_norm(hrs_ctx* ctx, int dtype, const void* x_dev, int64_t ldx, const void* resid_dev, int64_t ldr,
                              const float* gamma_dev, const float* beta_dev, float eps, void* y_dev, int64_t ldy, int64_t M,
                              int64_t N, void* stream) {
    HRS_REQUIRE(ctx, "hrs_layer_norm: null ctx");
    HRS_REQUIRE(dtype == HRS_TYPE_BF16 || dtype == HRS_TYPE_FP16 || dtype == HRS_TYPE_FP32, "hrs_layer_norm: unknown type %d", dtype);
    HRS_REQUIRE(M >= 0 && M < (1ll << 31) && N >= 0 && N < (1 << 30), "hrs_layer_norm: M=%lld, N=%lld", (long long)M, (long long)N);
    HRS_REQUIRE(eps >= 0.f, "hrs_layer_norm: eps=%g is negative", (double)eps);
    if (M == 0 || N == 0) return HRS_OK;
    HRS_REQUIRE(x_dev && gamma_dev && y_dev, "hrs_layer_norm: null operand");
    HRS_REQUIRE(ldx >= 0 && ldr >= 0, "hrs_layer_norm: negative row stride");
    HRS_REQUIRE(ldy >= N || M == 1, "hrs_layer_norm: rows of y overlap (stride %lld, N=%lld)", (long long)ldy, (long long)N);
    const uintptr_t el = dtype == HRS_TYPE_FP32 ? 4 : 2;
    HRS_REQUIRE(((uintptr_t)x_dev | (uintptr_t)y_dev | (uintptr_t)resid_dev) % el == 0 && ((uintptr_t)gamma_dev | (uintptr_t)beta_dev) % 4 == 0,
                "hrs_layer_norm: an operand is not aligned to its elements");
    HRS_REQUIRE((x_dev != y_dev || ldx == ldy || M == 1) && (resid_dev != y_dev || ldr == ldy || M == 1), "hrs_layer_norm: y in place of x or r needs its row stride");
    hrs_device_scope dev(ctx->device);
    HRS_CHECK_HIP(dev.err);
    return hrs_launch_norm(dtype, x_dev, ldx, resid_dev, ldr, gamma_dev, beta_dev, eps, y_dev, ldy, M, (int)N, (hipStream_t)stream);
}
