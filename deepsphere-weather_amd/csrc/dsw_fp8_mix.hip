// Per-node linear map in 8 bits:  y[m, n] = sum_b xs[m, b] ws[n / 128, b] sum_{k in block b} xq[m, k] wq[n, k] + bias[n]
// with e4m3 rows xq [M][K] (one scale per row and 128 channels) and e4m3 weights wq [N][K] (one scale per 128 x 128).
//
// bf16 output: one 16x16x128 8-bit matrix instruction covers a whole scale block: its result is multiplied by the block's scale and
// added to the running fp32 sum, so no scale is ever applied to an 8-bit value.  Inside the instruction the products of 8
// neighbouring k are aligned to the largest exponent among them and cut 13 bits below it (measured with sums of two products;
// groups of 8 are joined in fp32): a relative 1.5e-5 of a random block, two orders below half a step of bf16.  That is relative to
// the products, not to their sum: where large ones cancel, what is left can be smaller than the loss (fp32 output is for those).
// fp32 output: the cut would show, so the e4m3 values are widened to bf16 (exact) and multiplied by bf16 instructions (exact
// products, fp32 sums, 1e-8 of a random block), at half the matrix rate.
// The two scales of a block are multiplied first, in fp32, and their product scales the block's sum.
// The WEIGHT rows are the instruction's row operand and the activation rows its column operand: a lane then holds four
// neighbouring outputs n of ONE activation row m, needs one scale per block, and stores neighbouring outputs.
// (Which k a byte of the operand registers stands for does not matter as long as both operands agree on it.)
#include "dsw_common.h"
#include "../../include/dsw_hip.h"

namespace {

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
struct __attribute__((packed, aligned(1))) Any16 { u32x4 v; };

constexpr int64_t MIX_LD_MAX = (1 << 23) - 1;      // a tile's 256 rows are reached by offsets below 2^31

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

// Global memory -> LDS without registers: lane l's 16 (4) bytes land at LDS byte `lds` + 16 l (4 l).  The compiler does not count
// these loads: they are waited for by hand.  (m0 holds no value of the compiler's between instructions: it is a reserved register that
// it sets right before an instruction of its own that reads it, of which there is none here.)
static __device__ __forceinline__ void load_to_lds(const uint8_t* base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" :: "v"(off), "s"(base), "s"(lds) : "memory");
}
static __device__ __forceinline__ void load_to_lds4(const float* at, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" :: "v"(at), "s"(lds) : "memory");
}
static __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
static __device__ __forceinline__ uint32_t lds_byte(const void* p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)p; }
// (uniform index: a scalar load, which the counts of vector loads do not see)
static __device__ __forceinline__ float scalar_load(const float* p, int i) {
    return reinterpret_cast<const __attribute__((address_space(4))) float*>(reinterpret_cast<uintptr_t>(p))[i];
}

// ---- many rows: tiles of 16 NT WN outputs n x 16 MT WM rows m per workgroup of WN x WM waves ---------------------------------
// Operands travel through LDS, one scale block (128 bytes of every row) per stage.  Row r of a stage is 128 bytes, its 16-byte
// chunk c sits at place c ^ f(r), so that the 16 rows a fragment reads spread over the banks.  Which n a row of the matrix
// instruction stands for is free: row r of tile t of a wave is n = 4 NT (r / 4) + 4 t + r % 4, so that a lane ends with 4 NT
// neighbouring outputs of one row m and stores whole 16 bytes.
template <int NT>
static __device__ __forceinline__ int w_place(int row) { return (row & 3) | (((row / (4 * NT)) & 1) << 2); }

// tiles of a grid: each of the 8 dies takes a contiguous run of them (blocks go round the dies), 4 row tiles deep, so that the
// tiles that one L2 serves at a time share rows and weights
static __device__ __forceinline__ bool tile_of(int tiles_n, int tiles_m, int& tn, int& tm) {
    const int T = tiles_n * tiles_m, per = (T + 7) >> 3;
    const int id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (id >= T) return false;
    const int deep = 4, band = id / (deep * tiles_n), in = id - band * deep * tiles_n;
    const int high = tiles_m - band * deep < deep ? tiles_m - band * deep : deep;
    tn = in / high;
    tm = band * deep + in % high;
    return true;
}

// A wave's results: lane (r16, g) holds outputs n0 + 4 NT g .. + 4 NT - 1 of the rows m0 + 16 j + r16.  Written as they lie, a store
// would be 64 pieces of 16 bytes in as many lines (measured: 134 MB at 2.4 TB/s); they are turned in the wave's own part of LDS
// (16-byte chunks, chunk c of row m at place c ^ m) and leave as whole runs of a row.
// STREAM: the output is far larger than the caches and leaves past them.
template <int NT, int MT, bool BF16, bool STREAM>
static __device__ __forceinline__ void store_tile(const MixArgs& P, const f32x4 (&acc)[NT][MT], u32x4* own, int n0, int m0, int lane) {
    constexpr int PER = BF16 ? 8 : 4, CH = 16 * NT / PER;        // outputs of a chunk, chunks of a row
    const int r16 = lane & 15, g = lane >> 4;
    const int n = n0 + 4 * NT * g;
    float add[4 * NT];
#pragma unroll
    for (int k = 0; k < 4 * NT; ++k) add[k] = 0.f;
    if (P.bias != nullptr) {
#pragma unroll
        for (int k = 0; k < 4 * NT; ++k) add[k] = n + k < P.N ? load_out<BF16>(P.bias, n + k) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        const int m = 16 * j + r16;
#pragma unroll
        for (int c = 0; c < CH / 4; ++c) {
            u32x4 v;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if constexpr (BF16) {
                    const int e = c * 8 + 2 * q;
                    v[q] = f32x2_to_bf16(acc[e / 4][j][e % 4] + add[e], acc[e / 4][j][e % 4 + 1] + add[e + 1]);
                } else {
                    v[q] = __float_as_uint(acc[c][j][q] + add[4 * c + q]);
                }
            }
            own[m * CH + ((g * (CH / 4) + c) ^ (m & (CH - 1)))] = v;
        }
    }
    const bool whole_chunks = P.N % PER == 0 && ((uintptr_t)P.Y & 15) == 0;
#pragma unroll
    for (int i = 0; i < 16 * MT * CH / 64; ++i) {
        const int e = i * 64 + lane, row = e / CH, c = e % CH;
        const u32x4 v = own[row * CH + (c ^ (row & (CH - 1)))];
        const int m = m0 + row, k = n0 + c * PER;
        if (m >= P.M || k >= P.N) continue;
        const long at = (long)m * P.N + k;
        if (k + PER <= P.N) {
            char* const y = static_cast<char*>(P.Y) + at * (16 / PER);
            if (STREAM && whole_chunks) __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(y));
            else reinterpret_cast<Any16*>(y)->v = v;
        } else {
            for (int q = 0; q < P.N - k; ++q) {
                if constexpr (BF16) static_cast<uint16_t*>(P.Y)[at + q] = (uint16_t)(v[q >> 1] >> (16 * (q & 1)));
                else static_cast<uint32_t*>(P.Y)[at + q] = v[q];
            }
        }
    }
}

// 16-byte aligned rows of whole 16-byte chunks: two stages in LDS, filled without registers.  One meeting per block, before its
// last step t: by then every wave has read its last weights of the block, so its stage takes the loads of the block after next
// (issued at once: they have a whole block's time), and the next block has landed, so its first fragments are read while the
// last step's products are computed.  The matrix cores thus wait neither for the barrier nor for the fragments behind it.
// The products of one step are scaled and added while the next step's are computed: a 16x16x128 product takes 32 clocks, of which
// the vector unit is free for 16, its four additions (measured: 4 additions a product cost 12 %, each further instruction 4
// clocks) - so the loop's addresses are scalars and immediates.
template <int NT, int MT, int WN, int WM, bool BF16>
__global__ __launch_bounds__(64 * WN * WM) void fp8_mix_tile_kernel(const MixArgs P, const int tiles_n, const int tiles_m) {
    constexpr bool WIDE = !BF16;
    constexpr int WAVES = WN * WM, BN = 16 * NT * WN, BM = 16 * MT * WM, ROWS = BN + BM, PIECES = ROWS / 8 / WAVES;
    constexpr int STAGE = ROWS * 8 + WAVES * 16;       // 16-byte units: the rows, then 64 row scales of each wave
    static_assert(ROWS % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0, "a wave's pieces lie in one operand each");
    static_assert(128 % (16 * NT) == 0, "a wave's outputs share a row of weight scales");
    // A block's loads are issued one by one between products (a load costs its wave three scalar instructions; 9 of them behind one
    // another left the matrix cores waiting): GO with each product of the last step of the block before the previous one, the
    // rest from there on.
    constexpr int GO = (PIECES + NT * MT - MT) / (NT * MT - MT), FIRST = MT * GO < PIECES ? MT * GO : PIECES;
    static_assert(MT <= 4 && NT >= 2 && NT % 2 == 0 && FIRST + (NT - 1) * MT * GO > PIECES, "every load is issued before it is waited for");
    extern __shared__ u32x4 lds[];                     // [2][STAGE]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int tn, tm;
    if (!tile_of(tiles_n, tiles_m, tn, tm)) return;
    const int n0 = tn * BN, m0 = tm * BM;
    const int wn = (wave % WN) * 16 * NT, wm = (wave / WN) * 16 * MT;
    const int r16 = lane & 15, g = lane >> 4;

    // this lane's share of a stage: PIECES chunks (the first BN / 8 pieces are weight rows) and one row scale
    uint32_t off[PIECES];
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
    const int ms = m0 + wm + (lane < 16 * MT ? lane : 0);
    const float* xs = P.XS + (long)(ms < P.M ? ms : P.M - 1) * P.xs_row;      // of the next block to be fetched
    const int nb = (n0 + wn) >> 7, nb_last = (P.N - 1) >> 7;
    const float* const ws = P.WS + (long)(nb < nb_last ? nb : nb_last) * P.KB;
    const uint8_t* wk = P.W + (long)n0 * P.ldw;                               // of the next block to be fetched
    const uint8_t* xk = P.X + (long)m0 * P.ldx;
    const uint32_t lds0 = lds_byte(lds);
    const int whole = P.K >> 7, tail = P.K & 127;      // whole blocks, bytes of the last one
    auto fetch_piece = [&](int i, uint32_t o, int stage) {
        load_to_lds(i < BN / 8 / WAVES ? wk : xk, o, lds0 + (uint32_t)(stage * STAGE * 16 + (wave + i * WAVES) * 1024));
    };
    auto fetch_scales = [&](int stage) { load_to_lds4(xs, lds0 + (uint32_t)((stage * STAGE + ROWS * 8 + wave * 16) * 16)); };
    // places of this lane's chunks g and g + 4 in a stage: of row tile 0 (128 apart per tile), of weight tile 0 (32 apart)
    const int x_row = (BN + wm + r16) * 8, x_lo = x_row + (g ^ (r16 & 7)), x_hi = x_row + ((g + 4) ^ (r16 & 7));
    const int w_r = wn + 4 * NT * (r16 >> 2) + (r16 & 3), w_f = w_place<NT>(w_r);
    const int w_lo = w_r * 8 + (g ^ w_f), w_hi = w_r * 8 + ((g + 4) ^ w_f);
    const int s_at = (ROWS * 8 + wave * 16) * 4 + r16;

    f32x4 acc[NT][MT], p[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        p[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (whole > 0) {
        auto advance = [&](bool on) { wk += on ? 128 : 0; xk += on ? 128 : 0; xs += on ? P.xs_blk : 0; };
#pragma unroll
        for (int i = 0; i < PIECES; ++i) fetch_piece(i, off[i], 0);
        fetch_scales(0);
        advance(whole > 1);
#pragma unroll
        for (int i = 0; i < FIRST; ++i) fetch_piece(i, off[i], 1);
        asm volatile("s_waitcnt vmcnt(%0)" :: "n"(FIRST) : "memory");          // block 0 is there, block 1 on its way
        __syncthreads();
        Frag<WIDE> fx[MT], fw = make_frag<WIDE>(lds[w_lo], lds[w_hi]);
        float s[MT], s_old[MT];
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            fx[j] = make_frag<WIDE>(lds[x_lo + 128 * j], lds[x_hi + 128 * j]);
            s[j] = scalar_load(ws, 0) * reinterpret_cast<const float*>(lds)[s_at + 16 * j];
            s_old[j] = 0.f;
        }
        // No branch in the loop (the additions have to stay between the products): behind the last block it fetches that block
        // again, into stages that nobody reads any more.
        int stage = 0;
        for (int b = 0; b < whole; ++b) {
            const u32x4* const here = lds + stage * STAGE;
            const u32x4* const there = lds + (stage ^ 1) * STAGE;
            const float sw = scalar_load(ws, b + 1 < whole ? b + 1 : b);
            float s_next[MT];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                Frag<WIDE> next;
                if (t + 1 < NT) {
                    next = make_frag<WIDE>(here[w_lo + 32 * (t + 1)], here[w_hi + 32 * (t + 1)]);
                } else {
                    wait_loads();
                    __syncthreads();
                    next = make_frag<WIDE>(there[w_lo], there[w_hi]);
#pragma unroll
                    for (int j = 0; j < MT; ++j) s_next[j] = sw * reinterpret_cast<const float*>(there)[s_at + 16 * j];
                }
#pragma unroll
                for (int j = 0; j < MT; ++j) {
                    const f32x4 q = p[j];
                    const float sq = t == 0 ? s_old[j] : s[j];
                    p[j] = block_product<WIDE>(fw, fx[j]);
                    if (t + 1 == NT) {
                        fx[j] = make_frag<WIDE>(there[x_lo + 128 * j], there[x_hi + 128 * j]);
#pragma unroll
                        for (int i = j * GO; i < (j + 1) * GO && i < FIRST; ++i) fetch_piece(i, off[i], stage);      // block b + 2
                    } else {
#pragma unroll
                        for (int i = FIRST + (t * MT + j) * GO; i < FIRST + (t * MT + j + 1) * GO; ++i) {            // block b + 1, the rest
                            if (i < PIECES) fetch_piece(i, off[i], stage ^ 1);
                            else if (i == PIECES) fetch_scales(stage ^ 1);
                        }
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) acc[(t + NT - 1) % NT][j][k] = fmaf(q[k], sq, acc[(t + NT - 1) % NT][j][k]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                fw = next;
                if (t + 2 == NT) advance(b + 2 < whole);                       // block b + 1 is sent for
            }
#pragma unroll
            for (int j = 0; j < MT; ++j) { s_old[j] = s[j]; s[j] = s_next[j]; }
            stage ^= 1;
        }
        wait_loads();
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[NT - 1][j][k] = fmaf(p[j][k], s_old[j], acc[NT - 1][j][k]);
        if (tail) advance(true);
        __syncthreads();
    }
    if (tail) {                                        // the short last block: its chunks behind the rows are cleared in LDS
#pragma unroll
        for (int i = 0; i < PIECES; ++i) { const int c = piece_chunk(i) * 16; fetch_piece(i, c < tail ? off[i] : off[i] - c, 0); }
        fetch_scales(0);
        wait_loads();
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PIECES; ++i)
            if (piece_chunk(i) * 16 >= tail) lds[piece_row(i) * 8 + (lane & 7)] = u32x4{0u, 0u, 0u, 0u};
        __syncthreads();
        const float sw = scalar_load(ws, whole);
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            const Frag<WIDE> fx = make_frag<WIDE>(lds[x_lo + 128 * j], lds[x_hi + 128 * j]);
            const float s = sw * reinterpret_cast<const float*>(lds)[s_at + 16 * j];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const f32x4 q = block_product<WIDE>(make_frag<WIDE>(lds[w_lo + 32 * t], lds[w_hi + 32 * t]), fx);
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[t][j][k] = fmaf(q[k], s, acc[t][j][k]);
            }
        }
    }
    __syncthreads();
    constexpr int OWN = 16 * NT * 16 * MT / (BF16 ? 8 : 4);      // 16-byte chunks of a wave's results
    static_assert(WAVES * OWN <= 2 * STAGE, "the results fit the stages");
    store_tile<NT, MT, BF16, WAVES * NT * MT >= 256>(P, acc, lds + wave * OWN, n0 + wn, m0 + wm, lane);
}

// rows of any alignment and length (M of X, then N of W) -> rows of whole 16-byte chunks, zero behind the row; then the kernels
// above take them
__global__ __launch_bounds__(256) void fp8_align_rows_kernel(const uint8_t* X, long ldx, const uint8_t* W, long ldw, int K, uint8_t* out, long M,
                                                             long rows, int chunks) {
    const long total = rows * chunks;
    for (long e = (long)blockIdx.x * 256 + threadIdx.x; e < total; e += (long)gridDim.x * 256) {
        const long r = e / chunks;
        const int c = (int)(e - r * chunks);
        reinterpret_cast<u32x4*>(out)[e] = row_chunk(r < M ? X + r * ldx : W + (r - M) * ldw, c * 16, K);
    }
}

// ---- few rows: 16 NT outputs n x 16 MT rows m per workgroup; its WV waves share the blocks of K ------------------------------
// Bound by reading the weights: every wave reads the 16 NT weight rows of its blocks straight into registers (16 bytes per lane
// and load, any alignment), U blocks at a time so that their loads are in flight together; the partial sums of the waves are
// joined in wave order through LDS.
template <int MT, int NT, int U, int WV, bool BF16>
__global__ __launch_bounds__(64 * WV) void fp8_mix_few_kernel(const MixArgs P) {
    constexpr bool WIDE = !BF16;
    __shared__ float part[WV][NT * MT * 4][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * 16 * NT, m0 = blockIdx.y * 16 * MT;
    const int r16 = lane & 15, g = lane >> 4;
    const uint8_t* w[NT];
    const uint8_t* x[MT];
    const float* xs[MT];
#pragma unroll
    for (int t = 0; t < NT; ++t) w[t] = P.W + (long)(n0 + 16 * t + r16 < P.N ? n0 + 16 * t + r16 : P.N - 1) * P.ldw;
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        const int m = m0 + 16 * j + r16 < P.M ? m0 + 16 * j + r16 : P.M - 1;
        x[j] = P.X + (long)m * P.ldx;
        xs[j] = P.XS + (long)m * P.xs_row;
    }
    const float* const ws = P.WS + (long)(n0 >> 7) * P.KB;      // (16 NT divides 128: the outputs share a row of scales)
    f32x4 acc[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[t][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto add = [&](const u32x4 (&wc)[NT][2], const u32x4 (&xc)[MT][2], float sw, const float (&sx)[MT]) {
        Frag<WIDE> fw[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) fw[t] = make_frag<WIDE>(wc[t][0], wc[t][1]);
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            const Frag<WIDE> fx = make_frag<WIDE>(xc[j][0], xc[j][1]);
            const float s = sw * sx[j];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const f32x4 p = block_product<WIDE>(fw[t], fx);
#pragma unroll
                for (int q = 0; q < 4; ++q) acc[t][j][q] = fmaf(p[q], s, acc[t][j][q]);
            }
        }
    };
    const int whole = P.K >> 7;
    for (int b0 = wave; b0 < whole; b0 += WV * U) {
        u32x4 wc[U][NT][2], xc[U][MT][2];
        float sw[U], sx[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int b = b0 + u * WV;
            if (b < whole) {                           // (uniform)
                const long k = (long)b * 128 + g * 16;
#pragma unroll
                for (int t = 0; t < NT; ++t) { wc[u][t][0] = chunk(w[t] + k); wc[u][t][1] = chunk(w[t] + k + 64); }
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
            if (b0 + u * WV < whole) add(wc[u], xc[u], sw[u], sx[u]);
    }
    if (whole < P.KB && wave == whole % WV) {          // the short last block, by the wave whose turn it is
        const int k = whole * 128 + g * 16;
        u32x4 wc[NT][2], xc[MT][2];
        float sx[MT];
#pragma unroll
        for (int t = 0; t < NT; ++t) { wc[t][0] = row_chunk(w[t], k, P.K); wc[t][1] = row_chunk(w[t], k + 64, P.K); }
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            xc[j][0] = row_chunk(x[j], k, P.K);
            xc[j][1] = row_chunk(x[j], k + 64, P.K);
            sx[j] = xs[j][(long)whole * P.xs_blk];
        }
        add(wc, xc, ws[whole], sx);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) part[wave][(t * MT + j) * 4 + q][lane] = acc[t][j][q];
    __syncthreads();
    // output (n, m) of the tile: lane 16 (n % 16 / 4) + m % 16 of register 4 (MT (n / 16) + m / 16) + n % 4
    for (int e = threadIdx.x; e < 256 * NT * MT; e += 64 * WV) {
        const int n = e % (16 * NT), m = e / (16 * NT);
        const int reg = 4 * (MT * (n >> 4) + (m >> 4)) + (n & 3), l = 16 * ((n & 15) >> 2) + (m & 15);
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < WV; ++q) v += part[q][reg][l];
        if (m0 + m < P.M && n0 + n < P.N) {
            if (P.bias != nullptr) v += load_out<BF16>(P.bias, n0 + n);
            store_out<BF16>(P.Y, (long)(m0 + m) * P.N + n0 + n, v);
        }
    }
}

// The same split for 16-byte aligned rows of whole 16-byte chunks: a lane's share of a fragment lies in 16
// rows' lines, so reading it straight into registers asks for 64 lines a load (measured: 15 bytes a clock and CU, and the rows m
// are read again by every workgroup); here each wave has its block's rows brought into its own part of LDS, 8 whole lines a
// load, reads its fragments there and sends for its next block before it multiplies.  No wave waits for another until the sums
// are joined.
//
// S = 2: two blocks of a wave under way, with larger tiles in as much LDS: half the round trips, fewer copies of the rows m.
template <int MT, int NT, int WV, int S, bool BF16>
__global__ __launch_bounds__(64 * WV) void fp8_mix_few_lds_kernel(const MixArgs P) {
    constexpr bool WIDE = !BF16;
    constexpr int ROWS = 16 * (NT + MT), LOADS = ROWS / 8;
    constexpr int U = 4;                               // blocks of a wave whose scales are loaded together (S = 2)
    extern __shared__ u32x4 lds[];                     // [WV][S][ROWS][8], then [WV][NT MT 4][64] sums in the same place
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * 16 * NT, m0 = blockIdx.y * 16 * MT;
    const int r16 = lane & 15, g = lane >> 4;
    const uint8_t* const wbase = P.W + (long)n0 * P.ldw;
    const uint8_t* const xbase = P.X + (long)m0 * P.ldx;
    uint32_t off[ROWS / 8];
    const int c16 = ((lane & 7) ^ (lane >> 3)) * 16;   // row r of 8: chunk c at place c ^ r
#pragma unroll
    for (int i = 0; i < ROWS / 8; ++i) {
        const int r = 8 * i + (lane >> 3);
        if (i < 2 * NT) off[i] = (uint32_t)((n0 + r < P.N ? r : P.N - 1 - n0) * P.ldw) + c16;
        else off[i] = (uint32_t)((m0 + r - 16 * NT < P.M ? r - 16 * NT : P.M - 1 - m0) * P.ldx) + c16;
    }
    const float* xs[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) xs[j] = P.XS + (long)(m0 + 16 * j + r16 < P.M ? m0 + 16 * j + r16 : P.M - 1) * P.xs_row;
    const float* const ws = P.WS + (long)(n0 >> 7) * P.KB;
    const uint32_t to = lds_byte(lds) + (uint32_t)(wave * S * ROWS * 128);
    const int whole = P.K >> 7, tail = P.K & 127;
    auto fetch = [&](int b, int stage) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
            load_to_lds((i < 2 * NT ? wbase : xbase) + (long)b * 128, b < whole || c16 < tail ? off[i] : off[i] - c16, to + (stage * ROWS * 8 + 64 * i) * 16);
    };
    f32x4 acc[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[t][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    // block b out of its stage, whose place then takes block `next`
    auto add = [&](int b, int stage, int next, const float (&s)[MT]) {
        u32x4* const own = lds + (wave * S + stage) * ROWS * 8;
        if (b == whole && c16 >= tail) {               // the short last block: clear what lies behind the rows
#pragma unroll
            for (int i = 0; i < LOADS; ++i) own[64 * i + lane] = u32x4{0u, 0u, 0u, 0u};
        }
        const int lo = r16 * 8 + (g ^ (r16 & 7)), hi = r16 * 8 + ((g + 4) ^ (r16 & 7));
        u32x4 wc[NT][2], xc[MT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) { wc[t][0] = own[128 * t + lo]; wc[t][1] = own[128 * t + hi]; }
#pragma unroll
        for (int j = 0; j < MT; ++j) { xc[j][0] = own[128 * (NT + j) + lo]; xc[j][1] = own[128 * (NT + j) + hi]; }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // the fragments are in registers: their place may be filled again
        __builtin_amdgcn_sched_barrier(0);
        if (next < P.KB) fetch(next, stage);
        Frag<WIDE> fw[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) fw[t] = make_frag<WIDE>(wc[t][0], wc[t][1]);
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            const Frag<WIDE> fx = make_frag<WIDE>(xc[j][0], xc[j][1]);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const f32x4 p = block_product<WIDE>(fw[t], fx);
#pragma unroll
                for (int q = 0; q < 4; ++q) acc[t][j][q] = fmaf(p[q], s[j], acc[t][j][q]);
            }
        }
    };
    if constexpr (S == 1) {
        if (wave < P.KB) fetch(wave, 0);
        for (int b = wave; b < P.KB; b += WV) {
            float s[MT];
            const float sw = scalar_load(ws, b);
#pragma unroll
            for (int j = 0; j < MT; ++j) s[j] = xs[j][(long)b * P.xs_blk] * sw;
            wait_loads();
            add(b, 0, b + WV, s);
        }
    } else {
        // The scales of U blocks are loaded in front of everything else: a load that the compiler knows of is waited for with all
        // that was sent for behind it.
        for (int b0 = wave; b0 < P.KB; b0 += U * WV) {
            float s[U][MT];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int b = b0 + u * WV < P.KB ? b0 + u * WV : P.KB - 1;
                const float sw = scalar_load(ws, b);
#pragma unroll
                for (int j = 0; j < MT; ++j) s[u][j] = xs[j][(long)b * P.xs_blk] * sw;
            }
            if (b0 == wave) {
                fetch(b0, 0);
                if (b0 + WV < P.KB) fetch(b0 + WV, 1);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int b = b0 + u * WV;
                if (b >= P.KB) break;                  // (uniform)
                if (b + WV < P.KB) asm volatile("s_waitcnt vmcnt(%0)" :: "n"(LOADS) : "memory");
                else wait_loads();
                add(b, u & 1, b + 2 * WV, s[u]);
            }
        }
    }
    __syncthreads();
    float* const part = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) part[(wave * NT * MT * 4 + (t * MT + j) * 4 + q) * 64 + lane] = acc[t][j][q];
    __syncthreads();
    for (int e = threadIdx.x; e < 256 * NT * MT; e += 64 * WV) {
        const int n = e % (16 * NT), m = e / (16 * NT);
        const int reg = 4 * (MT * (n >> 4) + (m >> 4)) + (n & 3), l = 16 * ((n & 15) >> 2) + (m & 15);
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < WV; ++q) v += part[(q * NT * MT * 4 + reg) * 64 + l];
        if (m0 + m < P.M && n0 + n < P.N) {
            if (P.bias != nullptr) v += load_out<BF16>(P.bias, n0 + n);
            store_out<BF16>(P.Y, (long)(m0 + m) * P.N + n0 + n, v);
        }
    }
}

template <int NT, int MT, int WN, int WM, bool BF16>
static int launch_tile(const MixArgs& a, hipStream_t s) {
    constexpr int BN = 16 * NT * WN, BM = 16 * MT * WM;
    const int tn = (a.N + BN - 1) / BN, tm = (a.M + BM - 1) / BM;
    constexpr int lds = 2 * ((BN + BM) * 128 + WN * WM * 256);
    static_assert(lds <= 160 * 1024, "");
    auto* kernel = fp8_mix_tile_kernel<NT, MT, WN, WM, BF16>;
    if (lds > 64 * 1024 && hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)
        return DSW_ERR_LAUNCH;
    const long per = ((long)tn * tm + 7) / 8;
    DSW_LAUNCH(kernel, dim3((unsigned)(per * 8)), dim3(64 * WN * WM), lds, s, a, tn, tm);
    return dsw_check_launch();
}
template <int MT, int NT, int U, int WV, bool BF16>
static int launch_few(const MixArgs& a, hipStream_t s) {
    DSW_LAUNCH((fp8_mix_few_kernel<MT, NT, U, WV, BF16>), dim3((unsigned)((a.N + 16 * NT - 1) / (16 * NT)), (unsigned)((a.M + 16 * MT - 1) / (16 * MT))),
               dim3(64 * WV), 0, s, a);
    return dsw_check_launch();
}
template <int MT, int NT, int WV, int S, bool BF16>
static int launch_few_lds(const MixArgs& a, hipStream_t s) {
    constexpr int stage = WV * S * 16 * (NT + MT) * 128, sums = WV * NT * MT * 1024, lds = stage > sums ? stage : sums;
    static_assert(lds <= 160 * 1024, "");
    auto* kernel = fp8_mix_few_lds_kernel<MT, NT, WV, S, BF16>;
    if (lds > 64 * 1024 && hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)
        return DSW_ERR_LAUNCH;
    DSW_LAUNCH(kernel, dim3((unsigned)((a.N + 16 * NT - 1) / (16 * NT)), (unsigned)((a.M + 16 * MT - 1) / (16 * MT))), dim3(64 * WV), lds, s, a);
    return dsw_check_launch();
}

static bool rows_aligned(const MixArgs& a) {
    return a.K % 16 == 0 && a.ldx % 16 == 0 && a.ldw % 16 == 0 && dsw_aligned16(a.X) && dsw_aligned16(a.W);
}
// up to here rows of any alignment go through the register kernel; with more rows m aligned copies of both operands are cheaper
constexpr int MIX_FEW_ROWS = 64;
static int64_t mix_ws_bytes(int64_t M, int64_t N, int64_t K, bool aligned) {
    return aligned || M <= MIX_FEW_ROWS ? 0 : (M + N) * ((K + 15) / 16 * 16);
}

// Which kernel, aligned rows (times in us of a replayed graph, bf16 output).  Few rows or outputs: the LDS kernel, named by its row tiles
// m, output tiles n and blocks of a wave under way:
//   rows x K x N          1,1,1  1,1,2  2,1,1  2,1,2  3,1,1  3,1,2  4,1,1  4,1,2  4,2,1
//   16 x 2048 x 4096        3.2    3.2
//   16 x 4096 x 4096        5.1    4.5
//   16 x 8192 x 4096        7.9    6.8
//   16 x 8192 x 6144       10.8   10.6
//   16 x 8192 x 8192       12.8   13.5
//   32 x 2048 x 4096                      3.8    3.8    4.2    4.2    4.5    4.6    6.3
//   32 x 4096 x 4096                      6.1    5.4    6.5    5.8    7.0    6.3    9.0
//   32 x 4096 x 8192                      8.8    9.6    9.5   10.3   10.4   11.2    9.7
//   33 x 4096 x 4096                      7.3    8.4    6.9    6.1    7.4    6.5    9.1
//   48 x 8192 x 4096                     12.0   14.4   11.3   10.1   12.0   10.7   15.1
//   48 x 4096 x 6144                     10.2   12.0    9.3   10.6   10.2   11.4   10.2
//   48 x 8192 x 8192                     23.6   30.1   17.8   19.4   19.0   20.4   20.5
//   64 x 4096 x 4096                      8.8    9.5    9.3   10.7    8.7    7.8   11.1
//   64 x 8192 x 4096                     13.0   15.1   14.3   16.8   13.1   11.9   16.6
//   64 x 8192 x 6144                     17.7   23.1   23.7   25.6   19.4   21.1   22.2
//   64 x 8192 x 8192                     24.9   31.4   29.4   34.1   20.8   22.1   22.0
//   128 x 4096 x 2048                     7.6    8.5    8.0    9.4    6.9    6.7   10.1
//   128 x 2176 x 4096                     9.0   11.6    9.7   11.3    8.5    9.7    8.9
//   128 x 4096 x 4096                    13.7   17.2   14.2   16.1   12.7   13.9   11.4
//   128 x 8192 x 4096                    22.3   28.9   22.6   26.3   19.3   22.0   17.8
// so, from three blocks of K for a wave on (more than 16): two blocks under way and as few row tiles as leave no CU a second workgroup
// (up to 16 rows, whose tiles are small enough to share one: up to three for two CUs); else, from 33 to 64 rows, all of them
// in one tile up to two workgroups a CU (at one and a half, 64 rows would be 9 % faster in tiles of 32; at two they are 16 %
// slower); from 32 blocks on (at 17 it is even) four row tiles and two output tiles where that leaves no CU a second
// workgroup.  With fewer blocks two under way gain nothing: small workgroups of one, four to a CU.
//
// Then tiles by outputs n x rows m ("LDS": 2,1,1):
//   rows x K x N          LDS   32x128  128x128  256x256
//   64 x 8192 x 1024       8.8    32.3     42.9     79.1
//   500 x 2048 x 512       5.2     7.9     10.2     23.5
//   1000 x 256 x 1000      8.2     3.8      4.4      8.6
//   1000 x 4096 x 1000    27.4    19.5     24.2     43.3
//   6000 x 512 x 512      22.2     7.2      6.1     10.9
//   24576 x 256 x 256     37.7    10.4      7.8      8.3
//   98304 x 128 x 256    137      25.4     16.6     17.6
//   98304 x 256 x 64      38.8    10.8     11.2     17.6
//   4096 x 512 x 4096     99.8    30.8     19.1     17.9
//   4096 x 4096 x 4096   294     144       78.1     62.6
// as long as the LDS kernel's workgroups come to four per CU - that; 32 x 128 up to 64 outputs; 128 x 128 as soon as there is such a
// tile for every other CU, 256 x 256 as soon as there is one for every CU (from four blocks of K on: below, its fuller
// epilogue costs more than it saves) and they cover at most a quarter more than 128 x 128 does.  Between them 128 x 64, three to a CU,
// from three for four CUs up to two for each; operands of the call before (in the caches) / of ten calls in turn:
//   rows x K x N          32 x 128      128 x 64     128 x 128       rows x K x N          32 x 128      128 x 64     128 x 128
//   8192 x 512 x 250      5.7 / 7.5     5.0 / 7.4    6.0 / 8.4       30000 x 512 x 128     8.7 / 12.5    6.6 / 8.7    6.2 / 9.2
//   16384 x 512 x 128     5.4 / 7.2     4.8 / 7.4    5.5 / 8.0       24576 x 2048 x 128   17.3 / 24.4   15.0 / 21.2  16.7 / 21.7
//   24576 x 512 x 128     6.7 / 8.4     6.3 / 8.5    5.8 / 8.6       6000 x 512 x 512      6.6 / 8.2     6.2 / 8.2    5.8 / 8.2
//   24576 x 640 x 80      6.8 / 8.5     6.4 / 8.8    5.9 / 9.2       12000 x 1024 x 256      - / 11.0      - / 10.7     - / 10.8
//   4096 x 4096 x 512    24.7 / -      20.4 / -     24.1 / -         22000 x 1024 x 128      - / 11.3      - / 10.7     - / 11.5
//   16384 x 512 x 64      4.3 / 6.2     4.4 / 7.1    5.2 / 7.8       24576 x 1024 x 64     6.9 / 10.4    7.8 / 10.4   7.1 / 11.6
// fp32 output (bf16 matrix instructions): 128 x 128 by four waves instead of eight (4096^3: 139 against 154) from one for every CU
// on (6000 x 512 x 512: 11.3 against 10.1 of the 32 x 128), no larger ones.
template <bool BF16>
static int launch_mix(const MixArgs& a, hipStream_t s) {
    const long cus = dsw_device_cus();
    auto tiles = [&](long n, long m) { return (a.N + n - 1) / n * ((a.M + m - 1) / m); };
    if (!rows_aligned(a)) {                            // (at most MIX_FEW_ROWS: the caller has aligned the others)
        if (a.M <= 16) return launch_few<1, 1, 4, 8, BF16>(a, s);
        if (a.M <= 32) return launch_few<2, 1, 1, 8, BF16>(a, s);
        return launch_few<4, 1, 1, 8, BF16>(a, s);
    }
    if (a.M <= 16) return a.KB > 16 && 2 * tiles(16, 16) <= 3 * cus ? launch_few_lds<1, 1, 8, 2, BF16>(a, s) : launch_few_lds<1, 1, 8, 1, BF16>(a, s);
    if (a.KB > 16) {
        if (tiles(16, 32) <= cus) return launch_few_lds<2, 1, 8, 2, BF16>(a, s);
        if (tiles(16, 48) <= cus) return launch_few_lds<3, 1, 8, 2, BF16>(a, s);
        if (tiles(16, 64) <= cus) return launch_few_lds<4, 1, 8, 2, BF16>(a, s);
        if (a.M > 32 && a.M <= 48 && tiles(16, 48) <= 2 * cus) return launch_few_lds<3, 1, 8, 1, BF16>(a, s);
        if (a.M > 48 && a.M <= 64 && tiles(16, 64) <= 2 * cus) return launch_few_lds<4, 1, 8, 1, BF16>(a, s);
        if (a.M > 64 && a.KB >= 32 && tiles(32, 64) <= cus) return launch_few_lds<4, 2, 8, 1, BF16>(a, s);
    }
    if (tiles(16, 32) <= 4 * cus) return launch_few_lds<2, 1, 8, 1, BF16>(a, s);
    if constexpr (BF16) {
        if (a.KB >= 4 && tiles(256, 256) >= cus && 16 * tiles(256, 256) <= 5 * tiles(128, 128)) return launch_tile<8, 4, 2, 4, BF16>(a, s);
        const long low = tiles(128, 64);
        if (a.N > 64 && 4 * low >= 3 * cus && low <= 2 * cus) return launch_tile<4, 1, 2, 4, BF16>(a, s);
        if (a.N > 64 && tiles(128, 128) >= cus / 2) return launch_tile<4, 2, 2, 4, BF16>(a, s);
    } else {
        if (a.N > 64 && tiles(128, 128) >= cus) return launch_tile<4, 4, 2, 2, BF16>(a, s);
    }
    return launch_tile<2, 2, 1, 4, BF16>(a, s);
}

static int align_rows(const MixArgs& a, uint8_t* out, hipStream_t s) {
    const int chunks = (a.K + 15) / 16;
    const long rows = (long)a.M + a.N, blocks = (rows * chunks + 255) / 256;
    DSW_LAUNCH(fp8_align_rows_kernel, dim3((unsigned)(blocks < 16384 ? blocks : 16384)), dim3(256), 0, s, a.X, a.ldx, a.W, a.ldw, a.K, out, (long)a.M, rows, chunks);
    return dsw_check_launch();
}

}  // namespace

extern "C" {

static bool mix_sizes_ok(int64_t M, int64_t N, int64_t K) {
    return M >= 0 && N >= 1 && K >= 1 && M <= 0x7fffffff - 256 && N <= (1 << 22) && K <= MIX_LD_MAX - 15 &&
           (M + 127) / 128 * ((N + 31) / 32) < (1 << 24) - 8;          // (a grid has less than 2^32 threads)
}

int64_t dsw_fp8_mix_workspace_bytes(int64_t M, int64_t N, int64_t K, int aligned) {
    if (!mix_sizes_ok(M, N, K)) return DSW_ERR_BAD_ARG;
    return mix_ws_bytes(M, N, K, aligned != 0);
}

int dsw_fp8_mix(const void* X, int64_t ldx, const float* XS, int64_t xs_row, int64_t xs_blk, const void* W, int64_t ldw,
                const float* WS, const void* bias, void* Y, int64_t M, int64_t N, int64_t K, int dtype, void* workspace,
                int64_t workspace_bytes, dsw_stream_t stream) {
    if (dtype != DSW_F32 && dtype != DSW_BF16) return DSW_ERR_BAD_DTYPE;
    if (!mix_sizes_ok(M, N, K) || ldx < K || ldw < K || ldx > MIX_LD_MAX || ldw > MIX_LD_MAX || xs_row < 0 || xs_blk < 0) return DSW_ERR_BAD_ARG;
    if (M == 0) return DSW_OK;
    if (!X || !XS || !W || !WS || !Y) return DSW_ERR_BAD_ARG;
    hipStream_t s = (hipStream_t)stream;
    MixArgs a{(const uint8_t*)X, XS, (const uint8_t*)W, WS, bias, Y, (long)ldx, (long)ldw, (long)xs_row, (long)xs_blk,
              (int)M, (int)N, (int)K, (int)((K + 127) / 128)};
    const bool aligned = rows_aligned(a);
    const int64_t need = mix_ws_bytes(M, N, K, aligned);
    if (need > 0 && (!workspace || workspace_bytes < need || !dsw_aligned16(workspace))) return DSW_ERR_WORKSPACE;
    DswTraceScope trace_(s, DSW_ROLE_FP8_MIX, M, K, N);
    if (need > 0) {
        const long ld = (long)((K + 15) / 16 * 16);
        uint8_t* const x = static_cast<uint8_t*>(workspace);
        uint8_t* const w = x + M * ld;
        const int rc = align_rows(a, x, s);
        if (rc != DSW_OK) return rc;
        a.X = x; a.W = w; a.ldx = a.ldw = ld; a.K = (int)ld;       // (zeros behind the rows; the same number of scale blocks)
    }
    return dtype == DSW_BF16 ? launch_mix<true>(a, s) : launch_mix<false>(a, s);
}

}  // extern "C"
