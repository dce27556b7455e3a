// Root-mean-square norm over the channels of a row, with the residual's addition in front and an 8-bit output behind it:
//     h = x + r,   rstd = (mean_c h^2 + eps)^(-1/2),   y = h rstd w
//     8-bit output: per row and block of 128 channels  s_b = max(max|y_b| / 448, 2^-126),  q = e4m3(y / s_b)
// backward, with G = dL/dy, D = dL/dh (the gradient that the stored stream h collects behind the norm), xhat = h rstd:
//     dx = dr = D + rstd (G w - xhat mean_c(G w xhat)),     dw = sum over rows of G xhat
// All of it is bound by HBM: a row is read once into registers (16 bytes per lane and access), the sums run over the lanes that
// share the row, and everything that a pass can derive from the row leaves in the same pass.  The square sum and the norm use
// the unrounded fp32 sum x + r; h itself is rounded to the storage type once.  The backward pass takes the two addends rather than
// the rounded h: with bf16 storage the rounding would be as large an error in dw as dw's own (1.5 x together); the price is
// a fifth stream, 50 MB of 250 at 98304 x 256, and that both addends stay alive until then.
#include "dsw_rows_common.h"
#include "../../include/dsw_hip.h"

namespace {

constexpr int RN_THREADS = 256;
enum { RN_NORM = 0, RN_NORM_FP8 = 1, RN_QUANT = 2 };

struct NormArgs {
    const char* X; const char* R; const char* W;
    char* Y; char* H; uint8_t* Q; float* S; float* rstd;
    long rows, ldx, ldr, s_ld;     // element strides between rows; S[block * s_ld + row]
    int C;
    float eps;
};

// TPR threads share a row (a power of two up to one wave, or the whole workgroup), each holds NV vectors of V channels:
// vector t + i * TPR for thread t.  With V * TPR >= 128 a block of 128 channels is 128 / V neighbouring lanes of one i.
template <bool BF16, int TPR, int NV, int MODE>
__global__ __launch_bounds__(RN_THREADS) void rmsnorm_fwd_kernel(const NormArgs P) {
    using Rw = Row<BF16>;
    constexpr int V = Rw::V, E = Rw::E;
    __shared__ float red[2][4];
    const int t = threadIdx.x % TPR;
    int flip = 0;
    for (long r0 = (long)blockIdx.x * (RN_THREADS / TPR); r0 < P.rows; r0 += (long)gridDim.x * (RN_THREADS / TPR), flip ^= 1) {
    const long row = r0 + threadIdx.x / TPR;
    const bool live = row < P.rows;       // (whole waves stay for the shuffles; nothing is loaded or stored for dead rows)
    float v[NV][V];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (t + i * TPR) * V;
        const int n = live ? P.C - c : 0;
        if (n > 0) {
            Rw::load(P.X + (row * P.ldx + c) * E, n, v[i]);
            if (P.R != nullptr) {
                float r[V];
                Rw::load(P.R + (row * P.ldr + c) * E, n, r);
#pragma unroll
                for (int j = 0; j < V; ++j) v[i][j] += r[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) v[i][j] = 0.f;
        }
        if constexpr (MODE != RN_QUANT) {
#pragma unroll
            for (int j = 0; j < V; ++j) ss = fmaf(v[i][j], v[i][j], ss);
        }
    }
    float rstd = 1.f;
    if constexpr (MODE != RN_QUANT) {
        ss = row_sum<TPR>(ss, red, flip);
        rstd = 1.f / sqrtf(ss / (float)P.C + P.eps);
        if (live && t == 0 && P.rstd != nullptr) P.rstd[row] = rstd;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (t + i * TPR) * V;
        const int n = live ? P.C - c : 0;
        if constexpr (MODE != RN_QUANT) {
            if (n > 0) {
                if (P.H != nullptr) Rw::store(P.H + (row * P.C + c) * E, n, v[i]);
                float w[V];
                Rw::load(P.W + (long)c * E, n, w);
#pragma unroll
                for (int j = 0; j < V; ++j) v[i][j] = v[i][j] * rstd * w[j];
            }
        }
        if constexpr (MODE == RN_NORM) {
            if (n > 0) Rw::store(P.Y + (row * P.C + c) * E, n, v[i]);
        } else {
            uint32_t a = 0;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const uint32_t b = __float_as_uint(v[i][j]) & 0x7fffffffu;
                a = j < n && b > a ? b : a;
            }
            a = lanes_umax<128 / V>(a);
            const float s = e4m3_scale(a);
            if (n > 0) {
                float z[V];
                e4m3_quotients(v[i], s, z);
                uint32_t q[V / 4];
#pragma unroll
                for (int j = 0; j < V / 4; ++j) q[j] = e4m3_pack4(z[4 * j], z[4 * j + 1], z[4 * j + 2], z[4 * j + 3]);
                uint8_t* out = P.Q + row * P.C + c;
                if (n >= V) {
                    struct __attribute__((packed, aligned(1))) Bytes { uint32_t q[V / 4]; } b;
#pragma unroll
                    for (int j = 0; j < V / 4; ++j) b.q[j] = q[j];
                    *reinterpret_cast<Bytes*>(out) = b;
                } else {
#pragma unroll
                    for (int j = 0; j < V; ++j) if (j < n) out[j] = (uint8_t)(q[j / 4] >> (8 * (j % 4)));
                }
                if (c % 128 == 0) P.S[(long)(c / 128) * P.s_ld + row] = s;
            }
        }
    }
    }
}

// rows of more channels than the registers of a workgroup hold: the row is read a second time (from the caches) instead
template <bool BF16, int MODE>
__global__ __launch_bounds__(RN_THREADS) void rmsnorm_fwd_long_kernel(const NormArgs P) {
    using Rw = Row<BF16>;
    constexpr int V = Rw::V, E = Rw::E;
    __shared__ float red[2][4];
    const int t = threadIdx.x;
    int flip = 0;
    for (long row = blockIdx.x; row < P.rows; row += gridDim.x, flip ^= 1) {
    auto fetch = [&](int c, float (&v)[V]) {
        const int n = P.C - c;
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = 0.f;
        if (n <= 0) return;
        Rw::load(P.X + (row * P.ldx + c) * E, n, v);
        if (P.R != nullptr) {
            float r[V];
            Rw::load(P.R + (row * P.ldr + c) * E, n, r);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] += r[j];
        }
    };
    float rstd = 1.f;
    if constexpr (MODE != RN_QUANT) {
        float ss = 0.f;
        for (int c = t * V; c < P.C; c += RN_THREADS * V) {
            float v[V];
            fetch(c, v);
#pragma unroll
            for (int j = 0; j < V; ++j) ss = fmaf(v[j], v[j], ss);
        }
        ss = row_sum<RN_THREADS>(ss, red, flip);
        rstd = 1.f / sqrtf(ss / (float)P.C + P.eps);
        if (t == 0 && P.rstd != nullptr) P.rstd[row] = rstd;
    }
    for (int c0 = 0; c0 < P.C; c0 += RN_THREADS * V) {
        const int c = c0 + t * V, n = P.C - c;
        float v[V];
        fetch(c, v);
        if constexpr (MODE != RN_QUANT) {
            if (n > 0) {
                if (P.H != nullptr) Rw::store(P.H + (row * P.C + c) * E, n, v);
                float w[V];
                Rw::load(P.W + (long)c * E, n, w);
#pragma unroll
                for (int j = 0; j < V; ++j) v[j] = v[j] * rstd * w[j];
            }
        }
        if constexpr (MODE == RN_NORM) {
            if (n > 0) Rw::store(P.Y + (row * P.C + c) * E, n, v);
        } else {
            uint32_t a = 0;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const uint32_t b = __float_as_uint(v[j]) & 0x7fffffffu;
                a = j < n && b > a ? b : a;
            }
            a = lanes_umax<128 / V>(a);
            const float s = e4m3_scale(a);
            if (n > 0) {
                uint8_t* out = P.Q + row * P.C + c;
                float z[V];
                e4m3_quotients(v, s, z);
#pragma unroll
                for (int j = 0; j < V; j += 4) {
                    const uint32_t q = e4m3_pack4(z[j], z[j + 1], z[j + 2], z[j + 3]);
#pragma unroll
                    for (int k = 0; k < 4; ++k) if (j + k < n) out[j + k] = (uint8_t)(q >> (8 * k));
                }
                if (c % 128 == 0) P.S[(long)(c / 128) * P.s_ld + row] = s;
            }
        }
    }
    }
}

struct NormBwdArgs {
    const char* G; const char* D; const char* X; const char* R; const char* W; const float* rstd;
    char* dX; float* part;      // part: [blocks][C] column sums, or null when dw is not asked for
    long rows, ldx, ldr;
    int C;
};

// Every workgroup walks rows blockIdx.x, + gridDim.x, ... (in groups of 256 / TPR) and keeps its columns' share of dw in
// registers; the groups of a workgroup join theirs in index order through LDS, the workgroups leave one row each in `part`.
// No atomics: the order of every sum is fixed by the shape.  The streams of a group's next row are on their way while it works on
// the present one.
template <bool BF16, int TPR, int NV>
__global__ __launch_bounds__(RN_THREADS) void rmsnorm_bwd_kernel(const NormBwdArgs P) {
    using Rw = Row<BF16>;
    using u32x4 = typename Rw::u32x4;
    constexpr int V = Rw::V, E = Rw::E, GROUPS = RN_THREADS / TPR;
    __shared__ float red[2][4];
    __shared__ float cols[GROUPS > 1 ? GROUPS * TPR * V : 1];
    const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
    float dw[NV][V];
    u32x4 w[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (t + i * TPR) * V;
        w[i] = Rw::fetch(P.W + (long)c * E, P.C - c);
#pragma unroll
        for (int j = 0; j < V; ++j) dw[i][j] = 0.f;
    }
    u32x4 nx[NV], nr[NV], ng[NV], nd[NV];
    float nrstd = 0.f;
    auto ahead = [&](long row) {
        const bool live = row < P.rows;
        nrstd = live ? P.rstd[row] : 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + i * TPR) * V, n = live ? P.C - c : 0;
            nx[i] = Rw::fetch(P.X + (row * P.ldx + c) * E, n);
            ng[i] = Rw::fetch(P.G + (row * P.C + c) * E, n);
            if (P.R != nullptr) nr[i] = Rw::fetch(P.R + (row * P.ldr + c) * E, n);
            if (P.D != nullptr && P.dX != nullptr) nd[i] = Rw::fetch(P.D + (row * P.C + c) * E, n);
        }
    };
    int flip = 0;
    const long stride = (long)gridDim.x * GROUPS;
    ahead((long)blockIdx.x * GROUPS + group);
    for (long r0 = (long)blockIdx.x * GROUPS; r0 < P.rows; r0 += stride) {
        const long row = r0 + group;
        const bool live = row < P.rows;
        const float rstd = nrstd;
        float h[NV][V], g[NV][V];
        u32x4 d[NV];
        float a = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            Rw::unpack(nx[i], h[i]);
            Rw::unpack(ng[i], g[i]);
            d[i] = nd[i];
            if (P.R != nullptr) {
                float r[V];
                Rw::unpack(nr[i], r);
#pragma unroll
                for (int j = 0; j < V; ++j) h[i][j] += r[j];
            }
        }
        if (r0 + stride < P.rows) ahead(row + stride);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float wv[V];
            Rw::unpack(w[i], wv);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                h[i][j] *= rstd;                                  // xhat
                dw[i][j] = fmaf(g[i][j], h[i][j], dw[i][j]);
                g[i][j] *= wv[j];
                a = fmaf(g[i][j], h[i][j], a);
            }
        }
        if (P.dX == nullptr) continue;                            // (uniform over the grid)
        a = row_sum<TPR>(a, red, flip) / (float)P.C;
        flip ^= 1;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + i * TPR) * V, n = live ? P.C - c : 0;
            if (n > 0) {
                float o[V];
#pragma unroll
                for (int j = 0; j < V; ++j) o[j] = 0.f;
                if (P.D != nullptr) Rw::unpack(d[i], o);
#pragma unroll
                for (int j = 0; j < V; ++j) o[j] = fmaf(rstd, g[i][j] - h[i][j] * a, o[j]);
                Rw::store(P.dX + (row * P.C + c) * E, n, o);
            }
        }
    }
    if (P.part == nullptr) return;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (t + i * TPR) * V;
        if constexpr (GROUPS > 1) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < V; ++j) cols[(group * TPR + t) * V + j] = dw[i][j];
            __syncthreads();
            for (int k = threadIdx.x; k < TPR * V; k += RN_THREADS) {
                float s = 0.f;
#pragma unroll
                for (int q = 0; q < GROUPS; ++q) s += cols[q * TPR * V + k];
                if (i * TPR * V + k < P.C) P.part[(long)blockIdx.x * P.C + i * TPR * V + k] = s;
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) if (c + j < P.C) P.part[(long)blockIdx.x * P.C + c + j] = dw[i][j];
        }
    }
}

// rows beyond the registers of a workgroup: dx row by row (the row is read twice), dw as sums of columns over row ranges
template <bool BF16>
__global__ __launch_bounds__(RN_THREADS) void rmsnorm_bwd_long_dx_kernel(const NormBwdArgs P) {
    using Rw = Row<BF16>;
    constexpr int V = Rw::V, E = Rw::E;
    __shared__ float red[2][4];
    int flip = 0;
    for (long row = blockIdx.x; row < P.rows; row += gridDim.x, flip ^= 1) {
    auto stream = [&](int c, float (&h)[V]) {
        Rw::load(P.X + (row * P.ldx + c) * E, P.C - c, h);
        if (P.R != nullptr) {
            float r[V];
            Rw::load(P.R + (row * P.ldr + c) * E, P.C - c, r);
#pragma unroll
            for (int j = 0; j < V; ++j) h[j] += r[j];
        }
    };
    const float rstd = P.rstd[row];
    float a = 0.f;
    for (int c = threadIdx.x * V; c < P.C; c += RN_THREADS * V) {
        float h[V], g[V], w[V];
        stream(c, h);
        Rw::load(P.G + (row * P.C + c) * E, P.C - c, g);
        Rw::load(P.W + (long)c * E, P.C - c, w);
#pragma unroll
        for (int j = 0; j < V; ++j) a = fmaf(g[j] * w[j], h[j] * rstd, a);
    }
    a = row_sum<RN_THREADS>(a, red, flip) / (float)P.C;
    for (int c = threadIdx.x * V; c < P.C; c += RN_THREADS * V) {
        float h[V], g[V], w[V], d[V];
        stream(c, h);
        Rw::load(P.G + (row * P.C + c) * E, P.C - c, g);
        Rw::load(P.W + (long)c * E, P.C - c, w);
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] = 0.f;
        if (P.D != nullptr) Rw::load(P.D + (row * P.C + c) * E, P.C - c, d);
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] = fmaf(rstd, g[j] * w[j] - h[j] * rstd * a, d[j]);
        Rw::store(P.dX + (row * P.C + c) * E, P.C - c, d);
    }
    }
}
template <bool BF16>
__global__ __launch_bounds__(RN_THREADS) void rmsnorm_bwd_long_dw_kernel(const NormBwdArgs P) {
    using Rw = Row<BF16>;
    constexpr int E = Rw::E;
    const int c = blockIdx.x * RN_THREADS + threadIdx.x;
    if (c >= P.C) return;
    float s = 0.f;
    for (long row = blockIdx.y; row < P.rows; row += gridDim.y)
        s = fmaf(Rw::one(P.G + (row * P.C + c) * E),
                 (Rw::one(P.X + (row * P.ldx + c) * E) + (P.R != nullptr ? Rw::one(P.R + (row * P.ldr + c) * E) : 0.f)) * P.rstd[row], s);
    P.part[(long)blockIdx.y * P.C + c] = s;
}

// dw[c] = sum over the workgroups' rows of part, in a fixed order: 16 columns per workgroup, 16 threads per column, each with
// four chains of its own (a chain of dependent loads is what such a short kernel spends its time on)
template <bool BF16>
__global__ __launch_bounds__(RN_THREADS) void rmsnorm_dw_kernel(const float* part, int nparts, int C, char* dW) {
    __shared__ float red[16][17];
    const int k = threadIdx.x & 15, g = threadIdx.x >> 4, c = blockIdx.x * 16 + k;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < C) {
        int p = g;
#pragma unroll 4
        for (; p + 48 < nparts; p += 64)
#pragma unroll
            for (int q = 0; q < 4; ++q) s[q] += part[(long)(p + 16 * q) * C + c];
        for (int q = 0; p < nparts; p += 16, ++q) s[q & 3] += part[(long)p * C + c];
    }
    red[g][k] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    if (g == 0 && c < C) {
        float v = red[0][k];
#pragma unroll
        for (int q = 1; q < 16; ++q) v += red[q][k];
        Row<BF16>::put(dW + (long)c * Row<BF16>::E, v);
    }
}

// (threads per row, vectors per thread) for a row of nv vectors: one wave per row up to 256 vectors (no barrier), the whole
// workgroup beyond; blocks of 128 channels must not be shared by two i of a thread, hence at least `least` lanes
struct Shape { int tpr, nv; };
static Shape row_shape(long nv, int least) {
    if (nv <= 16 && least <= 16) return {16, 1};
    if (nv <= 32) return {32, 1};
    if (nv <= 64) return {64, 1};
    if (nv <= 128) return {64, 2};
    if (nv <= 256) return {64, 4};
    if (nv <= 512) return {256, 2};
    if (nv <= 1024) return {256, 4};
    if (nv <= 2048) return {256, 8};
    return {0, 0};
}

// workgroups of a forward launch; the kernels walk on from there.  Rows of one wave or less: 8 per CU (16 with the 8-bit output)
// stay and keep their weights' lines (98304 x 256 bf16: 35.4 us = 5.7 TB/s against 41.5 with one group of rows per workgroup; 8-bit
// 34.1 against 36.7); whole-workgroup rows: one each (8192 x 4096: 49.4 against 56.2), up to what a grid may hold.
static unsigned grid_of(long blocks, int tpr, int mode) {
    const long most = tpr > 64 ? 1 << 20 : dsw_device_cus() * (mode == RN_NORM ? 8 : 16);
    return (unsigned)(blocks < most ? blocks : most);
}

#define RN_SHAPES(CASE) CASE(16, 1) CASE(32, 1) CASE(64, 1) CASE(64, 2) CASE(64, 4) CASE(256, 2) CASE(256, 4) CASE(256, 8)

template <bool BF16, int MODE>
static int launch_fwd(const NormArgs& a, hipStream_t s) {
    constexpr int V = Row<BF16>::V;
    const Shape sh = row_shape((a.C + V - 1) / V, MODE == RN_NORM ? 16 : 128 / V);
    if (sh.tpr == 0) {
        DSW_LAUNCH((rmsnorm_fwd_long_kernel<BF16, MODE>), dim3(grid_of(a.rows, RN_THREADS, MODE)), dim3(RN_THREADS), 0, s, a);
        return dsw_check_launch();
    }
    const long blocks = (a.rows + RN_THREADS / sh.tpr - 1) / (RN_THREADS / sh.tpr);
#define CASE(T, N) \
    if (sh.tpr == T && sh.nv == N) { \
        DSW_LAUNCH((rmsnorm_fwd_kernel<BF16, T, N, MODE>), dim3(grid_of(blocks, T, MODE)), dim3(RN_THREADS), 0, s, a); \
        return dsw_check_launch(); \
    }
    RN_SHAPES(CASE)
#undef CASE
    return DSW_ERR_BAD_ARG;
}

// workgroups of the backward pass (= rows of `part`): two per CU with each group's next row in flight, as many as fit where a thread
// holds up to two vectors (98304 x 256 bf16: 768: 48.6, 1024: 52.9, against 47.4; without the next row ahead 52.5 at 1024 and 78.7
// at 512.  8192 x 4096: 69.4, 74.7, 79.8).  Four vectors (279-292 registers) leave room for one workgroup per CU at a time, which costs
// little; eight in bf16 spill.  2^25 elements each, us of this kernel and its five (fp32: four) streams in TB/s:
//   bf16, 256: 64 (5.2)   1024: 61 (5.5)   2048: 65 (5.1)   4096: 64 (5.2)   6144: 82 (4.1)   8192: 73 (4.6)   12288: 215 (1.6)
//   fp32, 256: 111 (4.8)  2048: 109 (4.9)  4096: 115 (4.7)  8192: 115 (4.7)
constexpr int RN_BWD_BLOCKS = 512;
static long bwd_blocks(int64_t rows, int64_t C, int dtype) {
    const int V = dtype == DSW_BF16 ? 8 : 4;
    const Shape sh = row_shape((C + V - 1) / V, 16);
    const long per = sh.tpr == 0 ? 1 : RN_THREADS / sh.tpr;
    const long need = (rows + per - 1) / per;
    return need < 1 ? 1 : need < RN_BWD_BLOCKS ? need : RN_BWD_BLOCKS;
}

template <bool BF16>
static int launch_bwd(const NormBwdArgs& a, char* dW, hipStream_t s) {
    constexpr int V = Row<BF16>::V;
    const Shape sh = row_shape((a.C + V - 1) / V, 16);
    const long blocks = bwd_blocks(a.rows, a.C, BF16 ? DSW_BF16 : DSW_F32);
    if (sh.tpr == 0) {
        if (a.dX != nullptr && a.rows > 0) DSW_LAUNCH(rmsnorm_bwd_long_dx_kernel<BF16>, dim3(grid_of(a.rows, RN_THREADS, RN_NORM)), dim3(RN_THREADS), 0, s, a);
        if (a.part != nullptr)
            DSW_LAUNCH(rmsnorm_bwd_long_dw_kernel<BF16>, dim3((unsigned)((a.C + RN_THREADS - 1) / RN_THREADS), (unsigned)blocks),
                       dim3(RN_THREADS), 0, s, a);
    } else {
#define CASE(T, N) \
        if (sh.tpr == T && sh.nv == N) DSW_LAUNCH((rmsnorm_bwd_kernel<BF16, T, N>), dim3((unsigned)blocks), dim3(RN_THREADS), 0, s, a);
        RN_SHAPES(CASE)
#undef CASE
    }
    if (a.part != nullptr)
        DSW_LAUNCH(rmsnorm_dw_kernel<BF16>, dim3((unsigned)((a.C + 15) / 16)), dim3(RN_THREADS), 0, s, a.part, (int)blocks, a.C, dW);
    return dsw_check_launch();
}

// W [Fin][Fout] (element strides si, so) -> Q [Fout][Fin] e4m3 and one scale per 128 x 128 block, a workgroup each.  A served layer
// quantises its weight in each call, a handful of blocks that no other work hides: so the whole block is in flight at once (16
// values per thread, neighbouring lanes along the smaller stride), is read once, and leaves through LDS as runs of 16 bytes
// (512 x 128 fp32: 5.3 us; 256 threads that read it twice, value after value, 23).
template <bool BF16>
__global__ __launch_bounds__(1024) void quant_weight_kernel(const char* W, long si, long so, uint8_t* Q, float* S, int Fin, int Fout,
                                                            int KB) {
    using Rw = Row<BF16>;
    typedef uint32_t __attribute__((ext_vector_type(4))) u32x4;
    constexpr int EACH = 128 * 128 / 1024, PITCH = 144;       // bytes of a row of the tile: 16-byte places, rows spread over the banks
    __shared__ uint32_t red[16];
    __shared__ __attribute__((aligned(16))) uint8_t tile[128 * PITCH];
    const int k0 = blockIdx.x * 128, n0 = blockIdx.y * 128;
    const int kn = Fin - k0 < 128 ? Fin - k0 : 128, nn = Fout - n0 < 128 ? Fout - n0 : 128;
    const bool along_n = so < si;
    const int lo = threadIdx.x & 127, hi = threadIdx.x >> 7;                  // value i of a thread: (lo, hi + 8 i)
    float v[EACH];
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int n = along_n ? lo : hi + 8 * i, k = along_n ? hi + 8 * i : lo;
        v[i] = n < nn && k < kn ? Rw::one(W + ((k0 + k) * si + (n0 + n) * so) * Rw::E) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
        a = b > a ? b : a;
    }
    a = lanes_umax<64>(a);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 16; ++q) a = red[q] > a ? red[q] : a;
    const float s = e4m3_scale(a);
    if (threadIdx.x == 0) S[(long)blockIdx.y * KB + blockIdx.x] = s;
    float z[EACH];
    e4m3_quotients(v, s, z);
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int n = along_n ? lo : hi + 8 * i, k = along_n ? hi + 8 * i : lo;
        tile[n * PITCH + k] = (uint8_t)e4m3_pack4(z[i], 0.f, 0.f, 0.f);
    }
    __syncthreads();
    const int n = threadIdx.x >> 3, k = (threadIdx.x & 7) * 16;
    if (n >= nn || k >= kn) return;
    uint8_t* const out = Q + (long)(n0 + n) * Fin + k0 + k;
    const uint8_t* const from = tile + n * PITCH + k;
    struct __attribute__((packed, aligned(1))) Any16 { u32x4 v; };
    if (k + 16 <= kn) reinterpret_cast<Any16*>(out)->v = *reinterpret_cast<const u32x4*>(from);
    else for (int j = 0; j < kn - k; ++j) out[j] = from[j];
}

static bool rows_ok(int64_t rows, int64_t C) { return rows >= 0 && C >= 1 && rows <= 0x7fffffff && C <= (1 << 24); }
static bool dtype_ok(int dtype) { return dtype == DSW_F32 || dtype == DSW_BF16; }

}  // namespace

extern "C" {

int dsw_rmsnorm_fwd(const void* X, int64_t ldx, const void* R, int64_t ldr, const void* W, void* Y, void* H, float* rstd,
                    int64_t rows, int64_t C, float eps, int dtype, dsw_stream_t stream) {
    if (!dtype_ok(dtype)) return DSW_ERR_BAD_DTYPE;
    if (!rows_ok(rows, C) || ldx < C || (R && ldr < C) || !(eps >= 0.f)) return DSW_ERR_BAD_ARG;
    if (rows == 0) return DSW_OK;
    if (!X || !W || !Y || ((R != nullptr) != (H != nullptr))) return DSW_ERR_BAD_ARG;
    hipStream_t s = (hipStream_t)stream;
    DswTraceScope trace_(s, DSW_ROLE_RMSNORM, rows, C, 0);
    const NormArgs a{(const char*)X, (const char*)R, (const char*)W, (char*)Y, (char*)H, nullptr, nullptr, rstd,
                     (long)rows, (long)ldx, (long)ldr, 0, (int)C, eps};
    return dtype == DSW_BF16 ? launch_fwd<true, RN_NORM>(a, s) : launch_fwd<false, RN_NORM>(a, s);
}

int dsw_rmsnorm_fwd_fp8(const void* X, int64_t ldx, const void* R, int64_t ldr, const void* W, void* Q, float* S, int64_t s_ld,
                        void* H, int64_t rows, int64_t C, float eps, int dtype, dsw_stream_t stream) {
    if (!dtype_ok(dtype)) return DSW_ERR_BAD_DTYPE;
    if (!rows_ok(rows, C) || ldx < C || (R && ldr < C) || s_ld < rows || !(eps >= 0.f)) return DSW_ERR_BAD_ARG;
    if (rows == 0) return DSW_OK;
    if (!X || !W || !Q || !S || ((R != nullptr) != (H != nullptr))) return DSW_ERR_BAD_ARG;
    hipStream_t s = (hipStream_t)stream;
    DswTraceScope trace_(s, DSW_ROLE_RMSNORM, rows, C, 1);
    const NormArgs a{(const char*)X, (const char*)R, (const char*)W, nullptr, (char*)H, (uint8_t*)Q, S, nullptr,
                     (long)rows, (long)ldx, (long)ldr, (long)s_ld, (int)C, eps};
    return dtype == DSW_BF16 ? launch_fwd<true, RN_NORM_FP8>(a, s) : launch_fwd<false, RN_NORM_FP8>(a, s);
}

int dsw_quant_fp8(const void* X, int64_t ldx, void* Q, float* S, int64_t s_ld, int64_t rows, int64_t C, int dtype,
                  dsw_stream_t stream) {
    if (!dtype_ok(dtype)) return DSW_ERR_BAD_DTYPE;
    if (!rows_ok(rows, C) || ldx < C || s_ld < rows) return DSW_ERR_BAD_ARG;
    if (rows == 0) return DSW_OK;
    if (!X || !Q || !S) return DSW_ERR_BAD_ARG;
    hipStream_t s = (hipStream_t)stream;
    DswTraceScope trace_(s, DSW_ROLE_RMSNORM, rows, C, 2);
    const NormArgs a{(const char*)X, nullptr, nullptr, nullptr, nullptr, (uint8_t*)Q, S, nullptr,
                     (long)rows, (long)ldx, 0, (long)s_ld, (int)C, 0.f};
    return dtype == DSW_BF16 ? launch_fwd<true, RN_QUANT>(a, s) : launch_fwd<false, RN_QUANT>(a, s);
}

int dsw_quant_fp8_weight(const void* W, int64_t stride_in, int64_t stride_out, void* Q, float* S, int64_t Fin, int64_t Fout,
                         int dtype, dsw_stream_t stream) {
    if (!dtype_ok(dtype)) return DSW_ERR_BAD_DTYPE;
    if (Fin < 1 || Fout < 1 || Fin > (1 << 22) || Fout > (1 << 22) || stride_in < 0 || stride_out < 0) return DSW_ERR_BAD_ARG;
    if (!W || !Q || !S) return DSW_ERR_BAD_ARG;
    hipStream_t s = (hipStream_t)stream;
    DswTraceScope trace_(s, DSW_ROLE_RMSNORM, Fout, Fin, 3);
    const dim3 grid((unsigned)((Fin + 127) / 128), (unsigned)((Fout + 127) / 128));
    if (dtype == DSW_BF16)
        DSW_LAUNCH(quant_weight_kernel<true>, grid, dim3(1024), 0, s, (const char*)W, (long)stride_in, (long)stride_out, (uint8_t*)Q, S,
                   (int)Fin, (int)Fout, (int)grid.x);
    else
        DSW_LAUNCH(quant_weight_kernel<false>, grid, dim3(1024), 0, s, (const char*)W, (long)stride_in, (long)stride_out, (uint8_t*)Q, S,
                   (int)Fin, (int)Fout, (int)grid.x);
    return dsw_check_launch();
}

int64_t dsw_rmsnorm_bwd_workspace_bytes(int64_t rows, int64_t C, int dtype) {
    if (!dtype_ok(dtype)) return DSW_ERR_BAD_DTYPE;
    if (!rows_ok(rows, C)) return DSW_ERR_BAD_ARG;
    return bwd_blocks(rows, C, dtype) * C * 4;
}

int dsw_rmsnorm_bwd(const void* G, const void* D, const void* X, int64_t ldx, const void* R, int64_t ldr, const void* W, const float* rstd, void* dX, void* dW,
                    void* workspace, int64_t workspace_bytes, int64_t rows, int64_t C, int dtype, dsw_stream_t stream) {
    if (!dtype_ok(dtype)) return DSW_ERR_BAD_DTYPE;
    if (!rows_ok(rows, C) || ldx < C || (R && ldr < C) || !W) return DSW_ERR_BAD_ARG;
    if (rows > 0 && (!G || !X || !rstd || (!dX && !dW))) return DSW_ERR_BAD_ARG;       // (without rows dX is an empty tensor's null)
    if (dW && (!workspace || workspace_bytes < dsw_rmsnorm_bwd_workspace_bytes(rows, C, dtype))) return DSW_ERR_WORKSPACE;
    if (rows == 0 && !dW) return DSW_OK;
    hipStream_t s = (hipStream_t)stream;
    DswTraceScope trace_(s, DSW_ROLE_RMSNORM, rows, C, 4);
    const NormBwdArgs a{(const char*)G, (const char*)D, (const char*)X, (const char*)R, (const char*)W, rstd, (char*)dX,
                        dW ? (float*)workspace : nullptr, (long)rows, (long)ldx, (long)ldr, (int)C};
    return dtype == DSW_BF16 ? launch_bwd<true>(a, (char*)dW, s) : launch_bwd<false>(a, (char*)dW, s);
}

}  // extern "C"
