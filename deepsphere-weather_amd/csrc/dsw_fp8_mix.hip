// Per-node linear map in 8 bits:  y[m, n] = sum_b xs[m, b] ws[n / 128, b] sum_{k in block b} xq[m, k] wq[n, k] + bias[n]
// with e4m3 rows xq [M][K] (one scale per row and 128 channels) and e4m3 weights wq [N][K] (one scale per 128 x 128).
//
// bf16 output: one 16x16x128 8-bit matrix instruction covers a whole scale block: its result is multiplied by the block's scale and
// added to the running fp32 sum, so no scale is ever applied to an 8-bit value.  Inside the instruction the products of 8
// neighbouring k are aligned to the largest exponent among them and cut 13 bits below it (measured with sums of two products;
// groups of 8 are joined in fp32): a relative 1.5e-5 of a random block, two orders below half a step of bf16.
// fp32 output: the cut would show, so the e4m3 values are widened to bf16 (exact) and multiplied by bf16 instructions (exact
// products, fp32 sums, 1e-8 of a random block), at half the matrix rate.
// The WEIGHT rows are the instruction's row operand and the activation rows its column operand: a lane then holds four
// neighbouring outputs n of ONE activation row m, needs one scale per block, and stores neighbouring outputs.
// (Which k a byte of the operand registers stands for does not matter as long as both operands agree on it.)
#include "dsw_common.h"
#include "../../include/dsw_hip.h"

namespace {

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
struct __attribute__((packed, aligned(1))) Any16 { u32x4 v; };

constexpr int64_t MIX_LD_MAX = (1 << 24) - 1;      // a tile's rows are reached by 32-bit offsets

struct MixArgs {
    const uint8_t* X; const float* XS; const uint8_t* W; const float* WS; const void* bias; void* Y;
    long ldx, ldw, xs_row, xs_blk;      // element strides; XS[m * xs_row + b * xs_blk], WS[nb * KB + b]
    int M, N, K, KB;
};

// a lane's 32 bytes of a row's block, as the operand of the 8-bit instruction or widened to four bf16 operands
typedef __attribute__((ext_vector_type(8))) __bf16 bf16v8;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16v2;
template <bool WIDE> struct Frag { i32x8 v; };
template <> struct Frag<true> { bf16v8 v[4]; };

template <bool WIDE>
static __device__ __forceinline__ Frag<WIDE> make_frag(const u32x4 lo, const u32x4 hi) {
    Frag<WIDE> f;
    if constexpr (WIDE) {
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const uint32_t t = q < 4 ? lo[q] : hi[q - 4];
            const bf16v2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(t, 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(t, 1.f, true);
            const int o = (q & 1) * 4;
            f.v[q >> 1][o] = a[0]; f.v[q >> 1][o + 1] = a[1]; f.v[q >> 1][o + 2] = b[0]; f.v[q >> 1][o + 3] = b[1];
        }
    } else {
        f.v = i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
    }
    return f;
}
template <bool WIDE>
static __device__ __forceinline__ f32x4 block_product(const Frag<WIDE>& a, const Frag<WIDE>& b) {
    f32x4 z = {0.f, 0.f, 0.f, 0.f};
    if constexpr (WIDE) {
#pragma unroll
        for (int q = 0; q < 4; ++q) z = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[q], b.v[q], z, 0, 0, 0);
        return z;
    } else {
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.v, b.v, z, 0, 0, 0, 0, 0, 0);   // (no scales: plain e4m3 x e4m3)
    }
}

static __device__ __forceinline__ u32x4 chunk(const uint8_t* p) { return reinterpret_cast<const Any16*>(p)->v; }
// 16 bytes k .. k + 15 of a row of K bytes; what lies behind the row is zero.  A chunk that the row ends in is read as the row's
// last 16 bytes and shifted down (one load; byte by byte it would be a chain of up to 15).
static __device__ __forceinline__ u32x4 row_chunk(const uint8_t* row, int k, int K) {
    u32x4 t = {0u, 0u, 0u, 0u};
    if (k + 16 <= K) {
        t = chunk(row + k);
    } else if (k < K) {
        if (K >= 16) {
            const u32x4 e = chunk(row + K - 16);
            uint64_t lo = (uint64_t)e[1] << 32 | e[0], hi = (uint64_t)e[3] << 32 | e[2];
            const int cut = 8 * (k + 16 - K);                   // 8 .. 120 bits
            if (cut >= 64) { lo = hi >> (cut - 64); hi = 0; }
            else { lo = lo >> cut | hi << (64 - cut); hi >>= cut; }
            t = u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
        } else {
            for (int j = 0; j < K - k; ++j) t[j >> 2] |= (uint32_t)row[k + j] << (8 * (j & 3));
        }
    }
    return t;
}

template <bool BF16>
static __device__ __forceinline__ float load_out(const void* p, long i) {
    if constexpr (BF16) return bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
    else return static_cast<const float*>(p)[i];
}
template <bool BF16>
static __device__ __forceinline__ void store_out(void* p, long i, float v) {
    if constexpr (BF16) static_cast<uint16_t*>(p)[i] = f32_to_bf16(v);
    else static_cast<float*>(p)[i] = v;
}

// One lane's 16 bytes global memory -> LDS (lane l of the wave writes LDS byte `lds` + 16 l); waited for by hand (vmcnt).
static __device__ __forceinline__ void load_to_lds(const uint8_t* base, uint32_t off, uint32_t lds) {
    uint32_t m0;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0) : "v"(off), "s"(base), "s"(lds) : "memory");
}

// ---- many rows: tiles of (16 NT WN) outputs n x (16 MT WM) rows m per workgroup of WN x WM waves -----------------------------
// Operands travel through LDS, one scale block (128 bytes of every row) per step, two stages: while a block is multiplied the
// next one is on its way.  Row r of a stage is 128 bytes, its 16-byte chunk c sits at place c ^ f(r), so that the 16 rows a
// fragment reads spread over the banks.  Which n a row of the matrix instruction stands for is free: row r of tile t of a wave is
// n = 4 NT (r / 4) + 4 t + r % 4, so that a lane ends with 4 NT neighbouring outputs of one row m and stores whole 16 bytes.
// DMA: 16-byte aligned rows of whole 16-byte chunks go to LDS directly; otherwise through registers.
template <int NT>
static __device__ __forceinline__ int w_place(int row) { return (row & 3) | (((row / (4 * NT)) & 1) << 2); }

template <int NT, int MT, int WN, int WM, bool BF16, bool DMA>
__global__ __launch_bounds__(64 * WN * WM) void fp8_mix_tile_kernel(const MixArgs P, const int tiles_n, const int tiles_m) {
    constexpr bool WIDE = !BF16;
    constexpr int WAVES = WN * WM, BN = 16 * NT * WN, BM = 16 * MT * WM, ROWS = BN + BM, PIECES = ROWS / 8 / WAVES;
    static_assert(ROWS % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0, "a wave's pieces lie in one operand each");
    static_assert(128 % (16 * NT) == 0, "a wave's outputs share a row of weight scales");
    extern __shared__ u32x4 lds[];                     // [2][ROWS][8]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // tiles: each of the 8 dies takes a contiguous run of them (blocks go round the dies), 8 row tiles deep
    const int T = tiles_n * tiles_m, per = (T + 7) >> 3;
    const int t_id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (t_id >= T) return;
    const int deep = 8, band = t_id / (deep * tiles_n), in = t_id - band * deep * tiles_n;
    const int high = tiles_m - band * deep < deep ? tiles_m - band * deep : deep;
    const int n0 = (in / high) * BN, m0 = (band * deep + in % high) * BM;
    const int wn = (wave % WN) * 16 * NT, wm = (wave / WN) * 16 * MT;
    const int r16 = lane & 15, g = lane >> 4;

    // this lane's share of a stage: PIECES chunks, the first BN / 8 pieces are weight rows
    uint32_t off[PIECES];
    const uint8_t* const wbase = P.W + (long)n0 * P.ldw;
    const uint8_t* const xbase = P.X + (long)m0 * P.ldx;
    auto piece_row = [&](int i) { return (wave + i * WAVES) * 8 + (lane >> 3); };
    auto piece_chunk = [&](int i) {
        const int row = piece_row(i);
        return row < BN ? (lane & 7) ^ w_place<NT>(row) : (lane & 7) ^ ((row - BN) & 7);
    };
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int row = piece_row(i);
        if (row < BN) off[i] = (uint32_t)((n0 + row < P.N ? row : P.N - 1 - n0) * P.ldw) + piece_chunk(i) * 16;
        else off[i] = (uint32_t)((m0 + row - BN < P.M ? row - BN : P.M - 1 - m0) * P.ldx) + piece_chunk(i) * 16;
    }
    const int whole = P.K >> 7, tail = P.K & 127;      // whole blocks, bytes of the last one
    u32x4 held[DMA ? 1 : PIECES];
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
    auto fetch = [&](int b, int stage) {
        if constexpr (DMA) {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const bool w = i < BN / 8 / WAVES;
                uint32_t o = off[i];
                if (b == whole) { const int c = piece_chunk(i); o = c * 16 < tail ? o : o - c * 16; }    // (chunks behind the row: cleared below)
                load_to_lds((w ? wbase : xbase) + (long)b * 128, o, lds0 + (uint32_t)((stage * ROWS + (wave + i * WAVES) * 8) * 128));
            }
        } else {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const int at = piece_chunk(i) * 16;
                held[i] = row_chunk((i < BN / 8 / WAVES ? wbase : xbase) + off[i] - at, b * 128 + at, P.K);
            }
        }
    };
    auto store_held = [&](int stage) {
        if constexpr (!DMA) {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) lds[(stage * ROWS + piece_row(i)) * 8 + (lane & 7)] = held[i];
        }
    };

    const float* xs[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        const int m = m0 + wm + 16 * j + r16;
        xs[j] = P.XS + (long)(m < P.M ? m : P.M - 1) * P.xs_row;
    }
    const int nb = (n0 + wn) >> 7, nb_last = (P.N - 1) >> 7;
    const float* const ws = P.WS + (long)(nb < nb_last ? nb : nb_last) * P.KB;

    f32x4 acc[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[t][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    float sx[MT], sw = ws[0];
#pragma unroll
    for (int j = 0; j < MT; ++j) sx[j] = xs[j][0];
    fetch(0, 0);
    store_held(0);
    for (int b = 0; b < P.KB; ++b) {
        const int stage = b & 1;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();                               // the block has landed; the other stage is no longer read
        if (DMA && b == whole) {                       // the last block is short: clear what lies behind the rows
#pragma unroll
            for (int i = 0; i < PIECES; ++i)
                if (piece_chunk(i) * 16 >= tail) lds[(stage * ROWS + piece_row(i)) * 8 + (lane & 7)] = u32x4{0u, 0u, 0u, 0u};
            __syncthreads();
        }
        float s[MT];
#pragma unroll
        for (int j = 0; j < MT; ++j) s[j] = sw * sx[j];
        if (b + 1 < P.KB) {
            sw = ws[b + 1];
#pragma unroll
            for (int j = 0; j < MT; ++j) sx[j] = xs[j][(long)(b + 1) * P.xs_blk];
            fetch(b + 1, stage ^ 1);
        }
        const u32x4* const base = lds + stage * ROWS * 8;
        Frag<WIDE> fx[MT];
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            const int r = BN + wm + 16 * j + r16, f = r16 & 7;
            fx[j] = make_frag<WIDE>(base[r * 8 + (g ^ f)], base[r * 8 + ((g + 4) ^ f)]);
        }
        // products of step t are added while those of step t + 1 are on the matrix cores: a product takes 32 clocks, its four
        // additions 16, and the vector pipe reads a result no sooner than its matrix instruction has ended
        auto weight_frag = [&](int t) {
            const int r = wn + 4 * NT * (r16 >> 2) + 4 * t + (r16 & 3), f = w_place<NT>(r);
            return make_frag<WIDE>(base[r * 8 + (g ^ f)], base[r * 8 + ((g + 4) ^ f)]);
        };
        Frag<WIDE> fw = weight_frag(0);
        f32x4 p[MT];
#pragma unroll
        for (int t = 0; t <= NT; ++t) {
            Frag<WIDE> next = fw;
            if (t + 1 < NT) next = weight_frag(t + 1);
#pragma unroll
            for (int j = 0; j < MT; ++j) {
                f32x4 q = p[j];
                if (t < NT) p[j] = block_product<WIDE>(fw, fx[j]);
                if (t > 0) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) acc[t - 1][j][k] = fmaf(q[k], s[j], acc[t - 1][j][k]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            fw = next;
        }
        if (b + 1 < P.KB) store_held(stage ^ 1);
    }

    const int n = n0 + wn + 4 * NT * g;
    float add[4 * NT];
#pragma unroll
    for (int k = 0; k < 4 * NT; ++k) add[k] = P.bias != nullptr && n + k < P.N ? load_out<BF16>(P.bias, n + k) : 0.f;
    const bool vec = n + 4 * NT <= P.N && P.N % 8 == 0 && ((uintptr_t)P.Y & 15) == 0;
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        const int m = m0 + wm + 16 * j + r16;
        if (m >= P.M) continue;
        const long at = (long)m * P.N + n;
        if (vec) {
            if constexpr (BF16) {
#pragma unroll
                for (int t = 0; t < NT; t += 2) {
                    u32x4 v;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int e = t * 4 + 2 * q;
                        v[q] = f32_to_bf16(acc[e / 4][j][e % 4] + add[e]) | (uint32_t)f32_to_bf16(acc[e / 4][j][e % 4 + 1] + add[e + 1]) << 16;
                    }
                    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(P.Y) + at + 4 * t) = v;
                }
            } else {
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    f32x4 v = acc[t][j];
#pragma unroll
                    for (int q = 0; q < 4; ++q) v[q] += add[4 * t + q];
                    *reinterpret_cast<f32x4*>(static_cast<float*>(P.Y) + at + 4 * t) = v;
                }
            }
        } else {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (n + 4 * t + q < P.N) store_out<BF16>(P.Y, at + 4 * t + q, acc[t][j][q] + add[4 * t + q]);
        }
    }
}

// ---- few rows: 16 outputs n x 16 MT rows m per workgroup; the waves share the blocks of K ------------------------------------
// Bound by reading the weights: every wave reads the 16 weight rows of its blocks straight into registers (16 bytes per lane and
// load, any alignment), U blocks at a time so that their loads are in flight together; the partial sums of the waves are joined in
// wave order through LDS.
constexpr int FEW_WAVES = 8;
template <int MT, int U, bool BF16>
__global__ __launch_bounds__(64 * FEW_WAVES) void fp8_mix_few_kernel(const MixArgs P) {
    constexpr bool WIDE = !BF16;
    __shared__ float part[FEW_WAVES][MT * 4][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MT;
    const int r16 = lane & 15, g = lane >> 4;
    const uint8_t* const w = P.W + (long)(n0 + r16 < P.N ? n0 + r16 : P.N - 1) * P.ldw;
    const uint8_t* x[MT];
    const float* xs[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        const int m = m0 + 16 * j + r16 < P.M ? m0 + 16 * j + r16 : P.M - 1;
        x[j] = P.X + (long)m * P.ldx;
        xs[j] = P.XS + (long)m * P.xs_row;
    }
    const float* const ws = P.WS + (long)(n0 >> 7) * P.KB;
    f32x4 acc[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto add = [&](const u32x4 (&wc)[2], const u32x4 (&xc)[MT][2], float sw, const float (&sx)[MT]) {
        const Frag<WIDE> fw = make_frag<WIDE>(wc[0], wc[1]);
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            const f32x4 p = block_product<WIDE>(fw, make_frag<WIDE>(xc[j][0], xc[j][1]));
            const float s = sw * sx[j];
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[j][q] = fmaf(p[q], s, acc[j][q]);
        }
    };
    const int whole = P.K >> 7;
    for (int b0 = wave; b0 < whole; b0 += FEW_WAVES * U) {
        u32x4 wc[U][2], xc[U][MT][2];
        float sw[U], sx[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int b = b0 + u * FEW_WAVES;
            if (b < whole) {                           // (uniform)
                const long k = (long)b * 128 + g * 16;
                wc[u][0] = chunk(w + k);
                wc[u][1] = chunk(w + k + 64);
                sw[u] = ws[b];
#pragma unroll
                for (int j = 0; j < MT; ++j) {
                    xc[u][j][0] = chunk(x[j] + k);
                    xc[u][j][1] = chunk(x[j] + k + 64);
                    sx[u][j] = xs[j][(long)b * P.xs_blk];
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (b0 + u * FEW_WAVES < whole) add(wc[u], xc[u], sw[u], sx[u]);
    }
    if (whole < P.KB && wave == whole % FEW_WAVES) {   // the short last block, by the wave whose turn it is
        const int k = whole * 128 + g * 16;
        u32x4 wc[2] = {row_chunk(w, k, P.K), row_chunk(w, k + 64, P.K)}, xc[MT][2];
        float sx[MT];
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            xc[j][0] = row_chunk(x[j], k, P.K);
            xc[j][1] = row_chunk(x[j], k + 64, P.K);
            sx[j] = xs[j][(long)whole * P.xs_blk];
        }
        add(wc, xc, ws[whole], sx);
    }
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) part[wave][4 * j + q][lane] = acc[j][q];
    __syncthreads();
    // output (n, m) of the tile: lane 16 (n / 4) + m % 16 of register 4 (m / 16) + n % 4
    for (int e = threadIdx.x; e < 256 * MT; e += 64 * FEW_WAVES) {
        const int n = e & 15, m = e >> 4;
        const int reg = 4 * (m >> 4) + (n & 3), l = 16 * (n >> 2) + (m & 15);
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < FEW_WAVES; ++q) v += part[q][reg][l];
        if (m0 + m < P.M && n0 + n < P.N) {
            if (P.bias != nullptr) v += load_out<BF16>(P.bias, n0 + n);
            store_out<BF16>(P.Y, (long)(m0 + m) * P.N + n0 + n, v);
        }
    }
}

template <int NT, int MT, int WN, int WM, bool BF16, bool DMA>
static int launch_tile(const MixArgs& a, hipStream_t s) {
    constexpr int BN = 16 * NT * WN, BM = 16 * MT * WM;
    const int tn = (a.N + BN - 1) / BN, tm = (a.M + BM - 1) / BM;
    const int lds = 2 * (BN + BM) * 128;
    auto* kernel = fp8_mix_tile_kernel<NT, MT, WN, WM, BF16, DMA>;
    if (lds > 64 * 1024 && hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)
        return DSW_ERR_LAUNCH;
    const long per = ((long)tn * tm + 7) / 8;
    DSW_LAUNCH(kernel, dim3((unsigned)(per * 8)), dim3(64 * WN * WM), lds, s, a, tn, tm);
    return dsw_check_launch();
}
template <bool BF16>
static int launch_few(const MixArgs& a, hipStream_t s) {
    const unsigned gn = (unsigned)((a.N + 15) / 16);
#define FEW(MT_, U_) DSW_LAUNCH((fp8_mix_few_kernel<MT_, U_, BF16>), dim3(gn, (unsigned)((a.M + 16 * MT_ - 1) / (16 * MT_))), dim3(64 * FEW_WAVES), 0, s, a)
    if (a.M <= 16) FEW(1, 4);
    else if (a.M <= 32) FEW(2, 2);
    else if (a.M <= 48) FEW(3, 2);
    else FEW(4, 2);
#undef FEW
    return dsw_check_launch();
}
template <bool BF16>
static int launch_mix(const MixArgs& a, hipStream_t s) {
    const bool dma = a.K % 16 == 0 && a.ldx % 16 == 0 && a.ldw % 16 == 0 && dsw_aligned16(a.X) && dsw_aligned16(a.W);
    if (a.M <= 64 || (long)((a.M + 127) / 128) * ((a.N + 127) / 128) < 64) return launch_few<BF16>(a, s);
    if (!dma) return launch_tile<4, 4, 2, 2, BF16, false>(a, s);
    if constexpr (BF16) {
        if ((long)((a.M + 255) / 256) * ((a.N + 255) / 256) >= 256) return launch_tile<8, 4, 2, 4, BF16, true>(a, s);
    }
    return launch_tile<4, 4, 2, 2, BF16, true>(a, s);
}

}  // namespace

extern "C" {

int64_t dsw_fp8_mix_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (M < 0 || N < 1 || K < 1 || M > 0x7fffffff - 256 || N > (1 << 22) || K > MIX_LD_MAX) return DSW_ERR_BAD_ARG;
    return 0;
}

int dsw_fp8_mix(const void* X, int64_t ldx, const float* XS, int64_t xs_row, int64_t xs_blk, const void* W, int64_t ldw,
                const float* WS, const void* bias, void* Y, int64_t M, int64_t N, int64_t K, int dtype, void* workspace,
                int64_t workspace_bytes, dsw_stream_t stream) {
    if (dtype != DSW_F32 && dtype != DSW_BF16) return DSW_ERR_BAD_DTYPE;
    const int64_t need = dsw_fp8_mix_workspace_bytes(M, N, K);
    if (need < 0 || ldx < K || ldw < K || ldx > MIX_LD_MAX || ldw > MIX_LD_MAX || xs_row < 0 || xs_blk < 0) return DSW_ERR_BAD_ARG;
    if (M == 0) return DSW_OK;
    if (!X || !XS || !W || !WS || !Y) return DSW_ERR_BAD_ARG;
    if (need > 0 && (!workspace || workspace_bytes < need)) return DSW_ERR_WORKSPACE;
    hipStream_t s = (hipStream_t)stream;
    DswTraceScope trace_(s, DSW_ROLE_FP8_MIX, M, K, N);
    const MixArgs a{(const uint8_t*)X, XS, (const uint8_t*)W, WS, bias, Y, (long)ldx, (long)ldw, (long)xs_row, (long)xs_blk,
                    (int)M, (int)N, (int)K, (int)((K + 127) / 128)};
    return dtype == DSW_BF16 ? launch_mix<true>(a, s) : launch_mix<false>(a, s);
}

}  // extern "C"
