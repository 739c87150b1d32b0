// hrs_linear: y = act(x W^T + b) + r, the matrix product of an encoder layer with its whole epilogue.
//
// x [M, K], W [N, K], y and r [M, N], bf16 or fp16, rows at any stride; b fp32 [N].  Products are summed in fp32 on the
// matrix cores, bias, activation and residual are applied to the fp32 sum, and the result is rounded once.
//
// Tiles are computed as W x^T (features on the rows of the matrix instruction, tokens on its columns), so that a lane
// holds features of one token.  Which feature sits on which row of which instruction is free, and chosen so that the
// registers of two instructions are 8 consecutive features and the four lanes of a token have 32 features side by side:
// y leaves in 16-byte pieces straight from the accumulators, 64 bytes next to each other per token and store.
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

// Feature (from the wave's first) on row r of instruction t.
__device__ __forceinline__ int feature_of(int t, int r) { return (t >> 1) * 32 + (r >> 2) * 8 + (t & 1) * 4 + (r & 3); }

// One lane's features of token m, NT / 2 times 8 at n, n + 32, ..: bias, activation, residual, one rounding.
template <typename T, int NT, int ACT>
__device__ __forceinline__ void linear_store(const LinearArgs& a, int64_t m, int n, const f32x4 (&acc)[NT], const float (&bias)[4 * NT]) {
    typedef typename vec_of<T>::x8 x8;
    if (m >= a.M) return;
    T* y = (T*)a.y + m * a.ldy;
    const T* r = a.resid ? (const T*)a.resid + m * a.ldr : nullptr;
#pragma unroll
    for (int u = 0; u < NT / 2; ++u) {
        const int c = n + u * 32, left = a.N - c;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = activate<ACT>(acc[2 * u + e / 4][e % 4] + bias[u * 8 + e]);
        if (left >= 8) {
            if (r) {
                x8 rv;
                __builtin_memcpy(&rv, r + c, 16);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += (float)rv[e];
            }
            x8 o;
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = (T)v[e];
            __builtin_memcpy(y + c, &o, 16);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < left) y[c + e] = (T)(r ? v[e] + (float)r[c + e] : v[e]);
        }
    }
}

template <int NT>
__device__ __forceinline__ void load_bias(const LinearArgs& a, int n, float (&bias)[4 * NT]) {
#pragma unroll
    for (int u = 0; u < NT / 2; ++u) {
        const int c = n + u * 32;
        if (a.bias && c + 8 <= a.N) {
            __builtin_memcpy(bias + u * 8, a.bias + c, 32);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) bias[u * 8 + e] = (a.bias && c + e < a.N) ? a.bias[c + e] : 0.f;
        }
    }
}

// ---- tiles staged through LDS ------------------------------------------------------------------------
// Depth advances by 64: an LDS row is 128 bytes, eight 16-byte pieces, piece p of row i stored at p ^ key(i), so that
// the 8 rows (16 lanes) a fragment read touches together lie in 8 different bank groups.
// Rows of x are read in order: key = i % 8.  Rows of W are read in the order of feature_of.
__device__ __forceinline__ int key_x(int i) { return i & 7; }
__device__ __forceinline__ int key_w(int i) { return (i & 3) | ((i >> 1) & 4); }

// ---- which tile a workgroup takes
struct TilePos {
    int64_t m;  // first token
    int n;      // first feature
};
// Workgroups go round the 8 XCDs, each with an L2 of its own: every XCD gets a consecutive run of tiles, and a run walks
// `deep` tiles of tokens by all features at a time, so that the tiles in flight on an XCD share operand rows.
template <int BM, int BN>
__device__ __forceinline__ TilePos tile_at(int id, int tm, int tn) {
    constexpr int deep = 8;
    const int group = id / (deep * tn), in = id - group * (deep * tn);
    const int rows = tm - group * deep < deep ? tm - group * deep : deep;
    TilePos t;
    t.m = (int64_t)(group * deep + in % rows) * BM;
    t.n = in / rows * BN;
    return t;
}


// Any alignment: pieces pass through registers, those of the next stage while this one is multiplied.  One LDS buffer
// (24 or 32 KB), so that several workgroups of a CU cover each other's barriers.  Bound by the L1's rate for pieces that
// straddle lines and by how the tiles fill the card: 4999 x 1537 x 773 takes 37 us (43 with tanh, a residual and rows of y
// at odd addresses), 4999 x 1536 x 773, whose 128 x 128 tiles fit one round, 24 us.
template <typename T, int BM, int BN, int WR, int WC, int ACT>
__global__ __launch_bounds__(64 * WR * WC, 2) void k_linear_any(LinearArgs a) {
    typedef typename vec_of<T>::x8 x8;
    constexpr int NTHR = 64 * WR * WC, MT = BM / WR / 16, NT = BN / WC / 16;
    constexpr int PX = BM * 8 / NTHR, PW = BN * 8 / NTHR;  // pieces a thread moves per stage
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, qd = lane >> 4, r16 = lane & 15;
    const TilePos tp = tile_at<BM, BN>(spread_over_xcds((int)blockIdx.x, (int)gridDim.x), (int)((a.M + BM - 1) / BM), (a.N + BN - 1) / BN);
    const int wm = (wv / WC) * (BM / WR), wn = (wv % WC) * (BN / WC);
    const T* src[PX + PW];
    int at[PX + PW];
    x8 in[PX + PW];
    const int p = tid & 7;
#pragma unroll
    for (int j = 0; j < PX + PW; ++j) {
        const bool isx = j < PX;
        const int row = (isx ? j : j - PX) * (NTHR / 8) + (tid >> 3);
        const int64_t left = (isx ? a.M - tp.m : (int64_t)a.N - tp.n) - 1;
        const int64_t use = row < left ? row : left;  // behind the last row: the last row again
        src[j] = (isx ? (const T*)a.x + (tp.m + use) * a.ldx : (const T*)a.w + (tp.n + use) * a.ldw) + p * 8;
        at[j] = (isx ? row : BM + row) * 128 + ((p ^ (isx ? key_x(row) : key_w(row))) << 4);
    }
    const int stages = (a.K + 63) >> 6;
    auto fetch = [&](int s) __attribute__((always_inline)) {
        if ((s + 1) * 64 <= a.K) {
#pragma unroll
            for (int j = 0; j < PX + PW; ++j) __builtin_memcpy(&in[j], src[j] + s * 64, 16);
        } else {
#pragma unroll
            for (int j = 0; j < PX + PW; ++j) in[j] = load8_any<T>(src[j] + s * 64, a.K - (s * 64 + p * 8));
        }
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = (f32x4)(0.f);
    if (stages) fetch(0);
    for (int s = 0; s < stages; ++s) {
        __syncthreads();  // the stage before has been read
#pragma unroll
        for (int j = 0; j < PX + PW; ++j) *(x8*)(lds + at[j]) = in[j];
        __syncthreads();
        if (s + 1 < stages) fetch(s + 1);
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
            x8 wf[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int row = wn + feature_of(t, r16);
                wf[t] = *(const x8*)(lds + (BM + row) * 128 + (((t2 * 4 + qd) ^ key_w(row)) << 4));
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int row = wm + i * 16 + r16;
                const x8 xf = *(const x8*)(lds + row * 128 + (((t2 * 4 + qd) ^ key_x(row)) << 4));
#pragma unroll
                for (int t = 0; t < NT; ++t) acc[i][t] = mfma16(wf[t], xf, acc[i][t]);
            }
        }
    }
    const int n = tp.n + wn + qd * 8;
    float bias[4 * NT];
    load_bias<NT>(a, n, bias);
#pragma unroll
    for (int i = 0; i < MT; ++i) linear_store<T, NT, ACT>(a, tp.m + wm + i * 16 + r16, n, acc[i], bias);
}

// ---- tiles by LDS-DMA ----------------------------------------------------------------------------------
// The same tiles for 16-byte aligned operands: pieces go from memory to LDS without passing registers.  A DMA instruction
// fills 8 LDS rows (lane l: row l / 8, place l % 8) and fetches for each place the piece that belongs there.  Rows beyond
// the matrix repeat its last row (their products are not stored).  Behind the depth K, a multiple of 8, the last stage
// fetches its first piece again and overwrites it with zeros once it has landed.
//
// KG groups of WR x WC waves share the depth of one tile: each walks its own run of stages through its own ring, and the
// first adds the sums of the others in order.  That is for products with few tiles, whose time is the latency of one
// stage (about 0.3 us) times their number: 1024 x 1024 x 1024 6.7 us with the depth shared by two (7.8 without),
// 256 x 1024 x 4096 8.7 us with 32 x 32 tiles shared by four (20.5 with 64 x 64 tiles unshared).
template <typename T, int BM, int BN, int RING, int WR, int WC, int KG, int ACT>
__global__ __launch_bounds__(64 * WR * WC * KG) void k_linear_tile(LinearArgs a) {
    typedef typename vec_of<T>::x8 x8;
    constexpr int NW = WR * WC, MT = BM / WR / 16, NT = BN / WC / 16;
    constexpr int PX = BM / 8 / NW, PW = BN / 8 / NW, NP = PX + PW;  // DMA instructions of a wave per stage
    constexpr int STAGE = (BM + BN) * 128;
    extern __shared__ __attribute__((aligned(16))) char lds_all[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), qd = lane >> 4, r16 = lane & 15;
    const int kg = wave / NW, wv = wave % NW;
    char* lds = lds_all + kg * (RING * STAGE);
    const TilePos tp = tile_at<BM, BN>(spread_over_xcds((int)blockIdx.x, (int)gridDim.x), (int)((a.M + BM - 1) / BM), (a.N + BN - 1) / BN);
    const int wm = (wv / WC) * (BM / WR), wn = (wv % WC) * (BN / WC);
    const char* xb = uniform_ptr((const T*)a.x + tp.m * a.ldx);
    const char* wb = uniform_ptr((const T*)a.w + (int64_t)tp.n * a.ldw);
    const uint32_t l0 = lds_addr_of(lds_all) + kg * (RING * STAGE);
    int voff[NP], piece[NP];
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        const bool isx = j < PX;
        const int row = (isx ? wv * PX + j : wv * PW + j - PX) * 8 + (lane >> 3);
        piece[j] = (lane & 7) ^ (isx ? key_x(row) : key_w(row));
        const int64_t left = (isx ? a.M - tp.m : (int64_t)a.N - tp.n) - 1;
        const int64_t use = row < left ? row : left;
        voff[j] = (int)(use * (isx ? a.ldx : a.ldw) * 2) + piece[j] * 16;
    }
    const int stages = (a.K + 63) >> 6, tail = a.K & 63;  // tail: depth of the last stage where it is not full
    const int per = (stages + KG - 1) / KG, s0 = kg * per, s1 = s0 + per < stages ? s0 + per : stages;
    auto place = [&](int slot, int j) __attribute__((always_inline)) { return slot * STAGE + (j < PX ? (wv * PX + j) * 1024 : BM * 128 + (wv * PW + j - PX) * 1024); };
    auto issue = [&](int s, int slot) __attribute__((always_inline)) {
        const int depth = tail && s == stages - 1 ? tail : 64;
#pragma unroll
        for (int j = 0; j < NP; ++j)
            glds16_asm((j < PX ? xb : wb) + (int64_t)s * 128, voff[j] - (piece[j] * 8 >= depth ? piece[j] * 16 : 0), l0 + place(slot, j));
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = (f32x4)(0.f);
#pragma unroll
    for (int i = 0; i < RING - 1; ++i)
        if (s0 + i < s1) issue(s0 + i, i);
    int slot = 0;
    for (int s = s0; s < s0 + per; ++s) {
        // stage s has landed (up to RING - 2 younger stages stay in flight)
        if (RING == 3 && s + 1 < s1) {
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NP) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if (tail && s == stages - 1) {
#pragma unroll
                for (int j = 0; j < NP; ++j)
                    if (piece[j] * 8 >= tail) *(u32x4*)(lds + place(slot, j) + lane * 16) = (u32x4)(0u);
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // everyone's part has landed, everyone has read stage s - 1
        if (s + RING - 1 < s1) issue(s + RING - 1, slot == 0 ? RING - 1 : slot - 1);
        const char* buf = lds + slot * STAGE;
        slot = slot == RING - 1 ? 0 : slot + 1;
        if (KG > 1 && s >= s1) continue;
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
            x8 wf[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int row = wn + feature_of(t, r16);
                wf[t] = *(const x8*)(buf + (BM + row) * 128 + (((t2 * 4 + qd) ^ key_w(row)) << 4));
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int row = wm + i * 16 + r16;
                const x8 xf = *(const x8*)(buf + row * 128 + (((t2 * 4 + qd) ^ key_x(row)) << 4));
#pragma unroll
                for (int t = 0; t < NT; ++t) acc[i][t] = mfma16(wf[t], xf, acc[i][t]);
            }
        }
    }
    if constexpr (KG > 1) {
        static_assert((KG - 1) * BM * BN * 4 <= KG * RING * STAGE, "the sums fit where the stages were");
        f32x4* part = (f32x4*)lds_all;
        __syncthreads();
        if (kg > 0) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int t = 0; t < NT; ++t) part[((((kg - 1) * NW + wv) * MT + i) * NT + t) * 64 + lane] = acc[i][t];
        }
        __syncthreads();
        if (kg > 0) return;
#pragma unroll
        for (int g = 0; g < KG - 1; ++g)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int t = 0; t < NT; ++t) acc[i][t] += part[(((g * NW + wv) * MT + i) * NT + t) * 64 + lane];
    }
    const int n = tp.n + wn + qd * 8;
    float bias[4 * NT];
    load_bias<NT>(a, n, bias);
#pragma unroll
    for (int i = 0; i < MT; ++i) linear_store<T, NT, ACT>(a, tp.m + wm + i * 16 + r16, n, acc[i], bias);
}

// ---- 256 x 256 tiles, two groups of waves in turn ---------------------------------------------------------
// Eight waves, two per SIMD, each 128 tokens x 64 features.  The waves of tokens 0 .. 127 and those of tokens 128 .. 255
// (one of each on every SIMD) run one barrier apart: while one group reads its fragments from LDS and issues DMA, the
// other has the matrix pipe for 32 instructions (512 cycles), then they change places.
// A stage is read in two halves: all of W and tokens 0 .. 63 of either group ("first"), then the other tokens ("second").
// A half's place in LDS is free as soon as both groups have read it, and is filled again for two stages ahead in the
// next phase: a piece has a whole stage (2048 cycles) to arrive, and every phase waits for the half that the next one
// reads with a counted wait, 8 younger requests still in flight.
// 8192^3: 743 us, 1.48 PFLOP/s (a large library product there: 0.69 ms, 1.58); per 1024 of depth a 65536 x 4096 product takes
// 336 us, as the library's does, and 150 us besides: 107 of them are its 537 MB of output at the card's copy rate, which
// nothing here runs under, since all workgroups finish their tiles at about the same time.  Workgroups that stay and fetch
// the next tile under their stores were built and took the same time (486 us either way).  gelu adds 86 us to the 485:
// 13 vector operations per value with the matrix pipe idle.
template <typename T, int ACT>
__global__ __launch_bounds__(512, 2) void k_linear_wide(LinearArgs a) {
    typedef typename vec_of<T>::x8 x8;
    constexpr int BM = 256, BN = 256, NT = 4, STAGE = (BM + BN) * 128;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), qd = lane >> 4, r16 = lane & 15;
    const int group = wv >> 2, wm = group * 128, wn = (wv & 3) * 64;
    const uint32_t l0 = lds_addr_of(lds);
    const int stages = (a.K + 63) >> 6, tail = a.K & 63;
    // DMA instructions of this wave: 0 .. 3 rows of W, 4 .. 5 first tokens, 6 .. 7 second tokens
    auto row_of = [&](int j) __attribute__((always_inline)) { return j < 4 ? wv * 32 + j * 8 : wm + (j >> 1 & 1) * 64 + (wv & 3) * 16 + (j & 1) * 8; };
    auto piece_of = [&](int j) __attribute__((always_inline)) {
        const int row = row_of(j) + (lane >> 3);
        return (lane & 7) ^ (j < 4 ? key_w(row) : key_x(row));
    };
    const TilePos tp = tile_at<BM, BN>(spread_over_xcds((int)blockIdx.x, (int)gridDim.x), (int)((a.M + BM - 1) / BM), (a.N + BN - 1) / BN);
    const char* xb = uniform_ptr((const T*)a.x + tp.m * a.ldx);
    const char* wb = uniform_ptr((const T*)a.w + (int64_t)tp.n * a.ldw);
    int voff[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int row = row_of(j) + (lane >> 3);
        const int64_t left = (j < 4 ? (int64_t)a.N - tp.n : a.M - tp.m) - 1;
        const int64_t use = row < left ? row : left;
        voff[j] = (int)(use * (j < 4 ? a.ldw : a.ldx) * 2) + piece_of(j) * 16;
    }
    auto place = [&](int s, int j) __attribute__((always_inline)) { return (uint32_t)((s & 1) * STAGE + ((j < 4 ? BM : 0) + row_of(j)) * 128); };
    auto issue = [&](int s, int j) __attribute__((always_inline)) {
        const int depth = tail && s == stages - 1 ? tail * 2 : 128;  // bytes of a row in this stage
        const int p16 = piece_of(j) * 16;
        glds16_asm((j < 4 ? wb : xb) + (int64_t)s * 128, voff[j] - (p16 >= depth ? p16 : 0), l0 + place(s, j));
    };
    auto blank = [&](int s, int j) __attribute__((always_inline)) {
        if (piece_of(j) * 8 >= tail) *(u32x4*)(lds + place(s, j) + lane * 16) = (u32x4)(0u);
    };
    auto meet = [&]() __attribute__((always_inline)) {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    f32x4 acc[8][NT];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = (f32x4)(0.f);

#pragma unroll
    for (int j = 0; j < 8; ++j) issue(0, j);
    if (stages > 1) {
#pragma unroll
        for (int j = 0; j < 6; ++j) issue(1, j);
        asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    } else {
        asm volatile("s_waitcnt vmcnt(2)" ::: "memory");
        if (tail) {
#pragma unroll
            for (int j = 0; j < 6; ++j) blank(0, j);
        }
    }
    meet();
    if (group == 1) meet();

    x8 wf[2][NT], xf[2][4];
    auto products = [&](int i0) __attribute__((always_inline)) {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int t = 0; t < NT; ++t) acc[i0 + i][t] = mfma16(wf[t2][t], xf[t2][i], acc[i0 + i][t]);
        __builtin_amdgcn_s_setprio(0);
    };
    for (int s = 0; s < stages; ++s) {
        const char* buf = lds + (s & 1) * STAGE;
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int row = wn + feature_of(t, r16);
                wf[t2][t] = *(const x8*)(buf + (BM + row) * 128 + (((t2 * 4 + qd) ^ key_w(row)) << 4));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = wm + i * 16 + r16;
                xf[t2][i] = *(const x8*)(buf + row * 128 + (((t2 * 4 + qd) ^ key_x(row)) << 4));
            }
        }
        if (s + 1 < stages) {
            issue(s + 1, 6);
            issue(s + 1, 7);
            asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if (tail) {
                blank(s, 6);
                blank(s, 7);
            }
        }
        meet();
        products(0);
        meet();
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = wm + 64 + i * 16 + r16;
                xf[t2][i] = *(const x8*)(buf + row * 128 + (((t2 * 4 + qd) ^ key_x(row)) << 4));
            }
        if (s + 2 < stages) {
#pragma unroll
            for (int j = 0; j < 6; ++j) issue(s + 2, j);
            asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
        } else if (s + 1 < stages) {
            asm volatile("s_waitcnt vmcnt(2)" ::: "memory");
            if (tail) {
#pragma unroll
                for (int j = 0; j < 6; ++j) blank(s + 1, j);
            }
        }
        meet();
        products(4);
        meet();
    }
    if (group == 0) meet();  // both groups have read the last stage
    const int n = tp.n + wn + qd * 8;
    float bias[4 * NT];
    load_bias<NT>(a, n, bias);
#pragma unroll
    for (int i = 0; i < 8; ++i) linear_store<T, NT, ACT>(a, tp.m + wm + i * 16 + r16, n, acc[i], bias);
}

// ---- few tokens -------------------------------------------------------------------------------------------
// Up to 16 tokens: W is read once, straight into the matrix instruction's operand (lane l: feature l % 16, 16 bytes of
// its row), 16 features per workgroup; its 8 or 16 waves share the depth and join their sums in LDS in a fixed order.
// Latency: 12 x 1536 x 384 2.8 us, 16 x 4096 x 1024 4.1 us (2.1 TB/s of W), 16 x 1024 x 4096 9.2 us; 32 x 32 tiles of
// k_linear_tile: 3.5, 4.1 and 8.7 us, but those waste half of the matrix instruction and need aligned operands.
template <typename T, int NW, bool ALIGNED, int ACT>
__global__ __launch_bounds__(64 * NW) void k_linear_few(LinearArgs a) {
    typedef typename vec_of<T>::x8 x8;
    __shared__ float part[NW][4][64];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, qd = lane >> 4, r16 = lane & 15;
    const int n0 = blockIdx.x * 16;
    const int per = ((a.K + NW - 1) / NW + 31) & ~31;  // depth of a wave
    const int k0 = wv * per, k1 = k0 + per < a.K ? k0 + per : a.K;
    const int nrow = n0 + r16 < a.N ? n0 + r16 : a.N - 1;
    const T* wp = (const T*)a.w + (int64_t)nrow * a.ldw + qd * 8;
    const T* xp = (const T*)a.x + (r16 < a.M ? r16 : a.M - 1) * a.ldx + qd * 8;
    auto load = [&](const T* p, int k) __attribute__((always_inline)) {
        const int left = k1 - (k + qd * 8);
        if constexpr (ALIGNED) return left > 0 ? *(const x8*)(p + k) : (x8)((T)0.f);
        return load8_any<T>(p + k, left);
    };
    f32x4 acc = (f32x4)(0.f);
    for (int k = k0; k < k1; k += 128) {
        x8 wf[4], xf[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            wf[u] = load(wp, k + u * 32);
            xf[u] = load(xp, k + u * 32);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) acc = mfma16(wf[u], xf[u], acc);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) part[wv][e][lane] = acc[e];
    __syncthreads();
    const int m = threadIdx.x >> 4, nl = threadIdx.x & 15, n = n0 + nl;
    if (threadIdx.x >= 256 || m >= a.M || n >= a.N) return;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) v += part[w][nl & 3][(nl >> 2) * 16 + m];
    v = activate<ACT>(v + (a.bias ? a.bias[n] : 0.f));
    if (a.resid) v += (float)((const T*)a.resid)[m * a.ldr + n];
    ((T*)a.y)[m * a.ldy + n] = (T)v;
}

// ---- host side ---------------------------------------------------------------------------------------
template <typename T, int BM, int BN, int RING, int WR, int WC, int KG, int ACT>
static int launch_tile(hrs_ctx* ctx, const LinearArgs& a, hipStream_t st) {
    static hrs_per_device_once attr;
    const int lds = KG * RING * (BM + BN) * 128;
    const auto kernel = k_linear_tile<T, BM, BN, RING, WR, WC, KG, ACT>;
    if (attr.need(ctx->device)) {
        HRS_CHECK_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
        attr.done(ctx->device);
    }
    const int64_t tiles = (a.M + BM - 1) / BM * ((a.N + BN - 1) / BN);
    hipLaunchKernelGGL(kernel, dim3((unsigned)tiles), dim3(64 * WR * WC * KG), lds, st, a);
    HRS_CHECK_HIP(hipGetLastError());
    return HRS_OK;
}
template <typename T, int ACT>
static int launch_wide(hrs_ctx* ctx, const LinearArgs& a, hipStream_t st) {
    static hrs_per_device_once attr;
    const int lds = 2 * 512 * 128;
    if (attr.need(ctx->device)) {
        HRS_CHECK_HIP(hipFuncSetAttribute((const void*)k_linear_wide<T, ACT>, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
        attr.done(ctx->device);
    }
    const int64_t tiles = (a.M + 255) / 256 * ((a.N + 255) / 256);
    hipLaunchKernelGGL((k_linear_wide<T, ACT>), dim3((unsigned)tiles), dim3(512), lds, st, a);
    HRS_CHECK_HIP(hipGetLastError());
    return HRS_OK;
}
template <typename T, int ACT>
static int launch_few(const LinearArgs& a, bool aligned, hipStream_t st) {
    const dim3 grid((unsigned)((a.N + 15) / 16));
    if (aligned && a.K >= 2048)
        hipLaunchKernelGGL((k_linear_few<T, 16, true, ACT>), grid, dim3(1024), 0, st, a);
    else if (aligned)
        hipLaunchKernelGGL((k_linear_few<T, 8, true, ACT>), grid, dim3(512), 0, st, a);
    else
        hipLaunchKernelGGL((k_linear_few<T, 8, false, ACT>), grid, dim3(512), 0, st, a);
    HRS_CHECK_HIP(hipGetLastError());
    return HRS_OK;
}
template <typename T, int BM, int BN, int WR, int WC, int ACT>
static int launch_any(hrs_ctx* ctx, const LinearArgs& a, hipStream_t st) {
    static hrs_per_device_once attr;
    const int lds = (BM + BN) * 128;
    const auto kernel = k_linear_any<T, BM, BN, WR, WC, ACT>;
    if (attr.need(ctx->device)) {
        HRS_CHECK_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
        attr.done(ctx->device);
    }
    const int64_t tiles = (a.M + BM - 1) / BM * ((a.N + BN - 1) / BN);
    hipLaunchKernelGGL(kernel, dim3((unsigned)tiles), dim3(64 * WR * WC), lds, st, a);
    HRS_CHECK_HIP(hipGetLastError());
    return HRS_OK;
}

template <typename T, int ACT>
static int launch_linear(hrs_ctx* ctx, const LinearArgs& a, hipStream_t st) {
    // 16-byte pieces; 256 rows of an operand within the 2^31 bytes that a DMA's lane offset spans
    const bool aligned = ((uintptr_t)a.x | (uintptr_t)a.w) % 16 == 0 && (a.ldx | a.ldw | a.K) % 8 == 0 && a.ldx < (1 << 21) && a.ldw < (1 << 21);
    if (a.M <= 16) return launch_few<T, ACT>(a, aligned, st);
    auto tiles = [&](int bm, int bn) { return (a.M + bm - 1) / bm * ((a.N + bn - 1) / bn); };
    const int64_t cus = ctx->num_cu;
    if (!aligned || a.K == 0) {
        // Measured at K = 773 (us): 1000 x 1001: 9.5 with 64 x 64 tiles, 12.6 with 128 x 64, 14.9 with 128 x 128;
        // 4999 x 1537, where 128 x 128 leaves eight tiles for a second round: 43.5, 37.0, 44.6 (4999 x 1536, which does not:
        // 38.9, 31.5, 23.6);  8192 x 2047: 80, 66, 56.
        if (tiles(64, 64) <= 2 * cus) return launch_any<T, 64, 64, 2, 2, ACT>(ctx, a, st);
        const int64_t t = tiles(128, 128), rounds = (t + 2 * cus - 1) / (2 * cus);
        if (10 * t < 6 * rounds * 2 * cus) return launch_any<T, 128, 64, 2, 2, ACT>(ctx, a, st);
        return launch_any<T, 128, 128, 4, 2, ACT>(ctx, a, st);
    }
    // The largest tile of which there is still at most one per CU, and the depth shared by two or four groups of waves:
    // smaller tiles leave less to do one after the other, larger ones read less.  Measured (us, N x K = 1024 x 1024):
    // M = 256: 4.2 with 32 x 32, 5.4 with 32 x 64, 6.2 with 64 x 64;  M = 512: 7.1, 5.8, 6.3;  M = 1024: 12.7, 10.2, 6.7
    // and 8.9 with 128 x 64;  M = 2048: 11.6 with 64 x 64, 9.2 with 128 x 64, 11.0 with 128 x 128;  M = 4096: 21.6, 16.8, 12.5.
    if (tiles(32, 32) <= cus) return launch_tile<T, 32, 32, 3, 2, 1, 4, ACT>(ctx, a, st);
    if (tiles(32, 64) <= cus) return launch_tile<T, 32, 64, 2, 2, 2, 4, ACT>(ctx, a, st);
    if (tiles(64, 64) <= cus) return launch_tile<T, 64, 64, 3, 2, 2, 2, ACT>(ctx, a, st);
    if (tiles(128, 64) <= cus) return launch_tile<T, 128, 64, 3, 2, 2, 2, ACT>(ctx, a, st);
    if (tiles(128, 128) <= cus) return launch_tile<T, 128, 128, 2, 4, 2, 2, ACT>(ctx, a, st);
    // Beyond: 256 x 256 tiles, one per CU at a time, or 128 x 128 tiles, two per CU at a time in 0.70 of the time (depth
    // 1024: 30 us and 21 us a round), whichever needs less for the rounds this product takes.
    const int64_t wide = (tiles(256, 256) + cus - 1) / cus, small = (tiles(128, 128) + 2 * cus - 1) / (2 * cus);
    if (10 * wide <= 7 * small) return launch_wide<T, ACT>(ctx, a, st);
    return launch_tile<T, 128, 128, 2, 4, 2, 1, ACT>(ctx, a, st);
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
    HRS_REQUIRE(resid_dev != y_dev || ldr == ldy || M == 1, "hrs_linear: y in place of the residual needs its row stride (%lld, not %lld)", (long long)ldr, (long long)ldy);
    hrs_device_scope dev(ctx->device);
    HRS_CHECK_HIP(dev.err);
    LinearArgs a;
    a.ldx = ldx;
    a.ldw = ldw;
    a.ldr = ldr;
    a.ldy = ldy;
    a.K = (int)K;
    // Rows and features per launch: a grid holds less than 2^32 threads, of which a kernel takes at most 64 per feature (up to
    // 16 tokens) or one per 32 results.
    const int64_t most_n = 1 << 25;
    for (int64_t n0 = 0; n0 < N; n0 += most_n) {
        a.N = (int)(N - n0 < most_n ? N - n0 : most_n);
        a.w = (const char*)w_dev + n0 * ldw * 2;
        a.bias = bias_dev ? bias_dev + n0 : nullptr;
        int64_t most = (1ll << 36) / a.N;
        if (most > 1 << 22) most = 1 << 22;
        for (int64_t m0 = 0; m0 < M; m0 += most) {
            a.x = (const char*)x_dev + m0 * ldx * 2;
            a.y = (char*)y_dev + (m0 * ldy + n0) * 2;
            a.resid = resid_dev ? (const char*)resid_dev + (m0 * ldr + n0) * 2 : nullptr;
            a.M = M - m0 < most ? M - m0 : most;
            const int rc = dtype == HRS_TYPE_BF16 ? launch_linear_act<__bf16>(ctx, a, act, (hipStream_t)stream) : launch_linear_act<_Float16>(ctx, a, act, (hipStream_t)stream);
            if (rc) return rc;
        }
    }
    return HRS_OK;
}
