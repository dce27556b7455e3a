// Global norm of many gradient tensors and their clipping:
//     N = (sum over tensors and elements of |g|^p)^(1/p),  p = 1, 2 or inf;      c = min(1, max_norm / (N + 1e-6));      out = c g
// Two launches per batch of tensors, whatever their number and sizes: partial sums of the workgroups, then every workgroup of the
// second launch joins the partials (in index order, the same in each), derives c and scales its share.  Nothing is read back by
// the host, so the pair sits in a captured step.
// The sums are held in 64 bits: squares of fp32 gradients neither overflow nor lose the small tensors, and the kernels
// stay bound by HBM (2 fp64 operations for each 2 or 4 bytes).
#include "dsw_rows_common.h"
#include "../../include/dsw_hip.h"
#include <algorithm>
#include <new>

namespace {

constexpr int GN_THREADS = 256;
constexpr int GN_TENSORS = 144;            // segments per launch: their table travels as a kernel argument (< 4 KB), so a captured
                                           // graph owns its copy and no host buffer has to outlive the call
// elements of a workgroup's step: 4 (bf16) or 8 (fp32) loads of each thread, all in flight (half as many: 9.5 us, 289; a quarter: 10.1,
// 335, against 9.4 and 275 of 7 MB and 500 MB)
constexpr int GN_CHUNK = 256 * 32;
constexpr int GN_BLOCKS = 1024;            // partial sums of one launch at most
constexpr int GN_MAX_PARTS = 16 * 1024;    // partial sums of one call at most

// from here on the results leave past the caches, which keep what the first pass read last for the second, going backwards
// (200 M gradients, 500 MB: 277 us against 314; 7 MB: no difference)
constexpr int64_t GN_STREAM_BYTES = (int64_t)128 << 20;

struct GradTable {
    const char* g[GN_TENSORS];
    char* o[GN_TENSORS];
    long first[GN_TENSORS + 1];            // first chunk of each segment, in chunks of GN_CHUNK elements; [n] = their total
    unsigned short tail[GN_TENSORS];       // elements of the last chunk - 1
    unsigned bf16[(GN_TENSORS + 31) / 32];
    int n;
};

enum { GN_L2 = 0, GN_L1 = 1, GN_INF = 2 };

template <int P>
static __device__ __forceinline__ double fold(double s, float v) {
    if constexpr (P == GN_L2) { const double d = (double)v; return fma(d, d, s); }
    else if constexpr (P == GN_L1) return s + (double)fabsf(v);
    else { const double d = (double)fabsf(v); return d > s || d != d ? d : s; }      // (a NaN sticks: nothing is larger than it)
}
template <int P>
static __device__ __forceinline__ double join(double a, double b) {
    if constexpr (P == GN_INF) return b > a || b != b ? b : a;
    else return a + b;
}

static __device__ __forceinline__ int segment_of(const GradTable& T, long chunk) {
    int lo = 0, hi = T.n - 1;
    while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if (T.first[mid] <= chunk) lo = mid; else hi = mid - 1; }
    return lo;
}

template <int P>
static __device__ __forceinline__ double block_join(double s, double* red) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s = join<P>(s, __shfl_xor(s, off, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    return join<P>(join<P>(red[0], red[1]), join<P>(red[2], red[3]));
}

template <int P, bool BF16>
static __device__ __forceinline__ double chunk_sum(const char* g, int n, double s) {
    using Rw = Row<BF16>;
    constexpr int V = Rw::V, LOADS = GN_CHUNK / (GN_THREADS * V);
    int i = threadIdx.x * V;
    if (n == GN_CHUNK) {
        typename Rw::u32x4 t[LOADS];
#pragma unroll
        for (int q = 0; q < LOADS; ++q) t[q] = Rw::raw(g + (long)(i + q * GN_THREADS * V) * Rw::E);
#pragma unroll
        for (int q = 0; q < LOADS; ++q) {
            float v[V];
            Rw::unpack(t[q], v);
#pragma unroll
            for (int j = 0; j < V; ++j) s = fold<P>(s, v[j]);
        }
        return s;
    }
    for (; i < n; i += GN_THREADS * V) {
        float v[V];
        Rw::load(g + (long)i * Rw::E, n - i, v);
#pragma unroll
        for (int j = 0; j < V; ++j) s = fold<P>(s, v[j]);
    }
    return s;
}

template <int P>
__global__ __launch_bounds__(GN_THREADS) void grad_norm_kernel(const GradTable T, double* part) {
    __shared__ double red[4];
    double s = 0.0;
    for (long chunk = blockIdx.x; chunk < T.first[T.n]; chunk += gridDim.x) {
        const int t = segment_of(T, chunk);
        const long at = (chunk - T.first[t]) * GN_CHUNK;
        const int n = chunk + 1 == T.first[t + 1] ? T.tail[t] + 1 : GN_CHUNK;
        const bool bf16 = T.bf16[t >> 5] >> (t & 31) & 1u;
        s = bf16 ? chunk_sum<P, true>(T.g[t] + at * 2, n, s) : chunk_sum<P, false>(T.g[t] + at * 4, n, s);
    }
    s = block_join<P>(s, red);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

template <int P>
static __device__ __forceinline__ double total_norm(const double* part, int nparts, double* red) {
    double s = 0.0;
    for (int i = threadIdx.x; i < nparts; i += GN_THREADS) s = join<P>(s, part[i]);
    s = block_join<P>(s, red);
    return P == GN_L2 ? sqrt(s) : s;
}

// a whole chunk's loads of this thread, sent for in front of the norm that scales them
template <bool BF16> struct Chunk { typename Row<BF16>::u32x4 t[GN_CHUNK / (GN_THREADS * Row<BF16>::V)]; };
template <bool BF16>
static __device__ __forceinline__ void chunk_load(const char* g, Chunk<BF16>& k) {
    using Rw = Row<BF16>;
#pragma unroll
    for (int q = 0; q < GN_CHUNK / (GN_THREADS * Rw::V); ++q) k.t[q] = Rw::raw(g + (long)((threadIdx.x + q * GN_THREADS) * Rw::V) * Rw::E);
}
template <bool BF16, bool STREAM>
static __device__ __forceinline__ void chunk_store(char* o, const Chunk<BF16>& k, float c) {
    using Rw = Row<BF16>;
    constexpr int V = Rw::V;
#pragma unroll
    for (int q = 0; q < GN_CHUNK / (GN_THREADS * V); ++q) {
        float v[V];
        Rw::unpack(k.t[q], v);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] *= c;
        char* const to = o + (long)((threadIdx.x + q * GN_THREADS) * V) * Rw::E;
        if constexpr (STREAM) Rw::put_raw_stream(to, Rw::pack(v));
        else Rw::put_raw(to, Rw::pack(v));
    }
}
template <bool BF16>
static __device__ __forceinline__ void part_scale(const char* g, char* o, int n, float c) {
    using Rw = Row<BF16>;
    constexpr int V = Rw::V;
    for (int i = threadIdx.x * V; i < n; i += GN_THREADS * V) {
        float v[V];
        Rw::load(g + (long)i * Rw::E, n - i, v);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] *= c;
        Rw::store(o + (long)i * Rw::E, n - i, v);
    }
}

// T.n == 0: the norm alone
template <int P, bool STREAM>
__global__ __launch_bounds__(GN_THREADS) void grad_clip_kernel(const GradTable T, const double* part, int nparts, double max_norm,
                                                               float* norm) {
    __shared__ double red[4];
    struct Place { const char* g; char* o; int n; bool bf16, in_place; };
    auto place = [&](long at_) {
        const long chunk = T.first[T.n] - 1 - at_;             // from the end: what the first pass read last is still in the caches
        const int t = segment_of(T, chunk);
        const bool bf16 = T.bf16[t >> 5] >> (t & 31) & 1u;
        const long at = (chunk - T.first[t]) * GN_CHUNK * (bf16 ? 2 : 4);
        return Place{T.g[t] + at, T.o[t] + at, chunk + 1 == T.first[t + 1] ? T.tail[t] + 1 : GN_CHUNK, bf16, T.g[t] == T.o[t]};
    };
    Chunk<true> half;
    Chunk<false> full;
    // (the first chunk travels while the partials are joined: 7 MB, both launches of a replayed graph 9.7 -> 9.4 us)
    const bool work = T.n > 0 && blockIdx.x < T.first[T.n];
    Place p = work ? place(blockIdx.x) : Place{};
    if (work && p.n == GN_CHUNK) { if (p.bf16) chunk_load<true>(p.g, half); else chunk_load<false>(p.g, full); }
    const double N = total_norm<P>(part, nparts, red);
    if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)N;
    if (!work) return;
    const double q = max_norm / (N + 1e-6);
    const float c = q > 1.0 ? 1.f : (float)q;                  // (a NaN stays one, as in max_norm / norm clamped from above)
    for (long at_ = blockIdx.x;;) {
        if (c == 1.f && p.in_place) {}                         // in place and nothing to clip: g * 1 is g
        else if (p.n < GN_CHUNK) { if (p.bf16) part_scale<true>(p.g, p.o, p.n, c); else part_scale<false>(p.g, p.o, p.n, c); }
        else if (p.bf16) chunk_store<true, STREAM>(p.o, half, c);
        else chunk_store<false, STREAM>(p.o, full, c);
        at_ += gridDim.x;
        if (at_ >= T.first[T.n]) return;
        p = place(at_);
        if (p.n == GN_CHUNK && !(c == 1.f && p.in_place)) { if (p.bf16) chunk_load<true>(p.g, half); else chunk_load<false>(p.g, full); }
    }
}

struct Piece { const char* g; char* o; int64_t n; int bf16; };

// tensors -> segments: empty ones dropped; neighbours in memory (a flat bucket's views) joined, in the order given
static int64_t make_pieces(int n, const void* const* g, void* const* o, const int64_t* numel, const int32_t* dtype, Piece* out) {
    int64_t k = 0;
    for (int i = 0; i < n; ++i) {
        if (numel[i] == 0) continue;
        const int e = dtype[i] == DSW_BF16 ? 2 : 4;
        const Piece p{(const char*)g[i], o ? (char*)o[i] : nullptr, numel[i], dtype[i] == DSW_BF16};
        if (k > 0 && out[k - 1].bf16 == p.bf16 && out[k - 1].g + out[k - 1].n * e == p.g && (!o || out[k - 1].o + out[k - 1].n * e == p.o))
            out[k - 1].n += p.n;
        else if (k > 0 && out[k - 1].bf16 == p.bf16 && p.g + p.n * e == out[k - 1].g && (!o || p.o + p.n * e == out[k - 1].o)) {
            out[k - 1].g = p.g; out[k - 1].o = p.o; out[k - 1].n += p.n;
        } else
            out[k++] = p;
    }
    return k;
}

// whether no written range overlaps another range (two reads of the same memory may)
struct Range { uintptr_t from, to; bool written; };
static bool no_conflict(Range* r, int64_t k) {
    std::sort(r, r + k, [](const Range& a, const Range& b) { return a.from < b.from; });
    uintptr_t any = 0, written = 0;
    for (int64_t i = 0; i < k; ++i) {
        if (r[i].from < (r[i].written ? any : written)) return false;
        if (r[i].to > any) any = r[i].to;
        if (r[i].written && r[i].to > written) written = r[i].to;
    }
    return true;
}

static int kind_of(double p) { return p == 2.0 ? GN_L2 : p == 1.0 ? GN_L1 : p > 1e300 ? GN_INF : -1; }

static void fill_table(GradTable& T, const Piece* p, int n) {
    T.n = n;
    T.first[0] = 0;
    for (unsigned& b : T.bf16) b = 0;
    for (int i = 0; i < n; ++i) {
        const int64_t chunks = (p[i].n + GN_CHUNK - 1) / GN_CHUNK;
        T.g[i] = p[i].g;
        T.o[i] = p[i].o;
        T.first[i + 1] = T.first[i] + (long)chunks;
        T.tail[i] = (unsigned short)(p[i].n - (chunks - 1) * GN_CHUNK - 1);
        if (p[i].bf16) T.bf16[i >> 5] |= 1u << (i & 31);
    }
}

template <int P>
static int run_clip(const Piece* pieces, int64_t k, double* part, double max_norm, bool scale, float* norm, hipStream_t s) {
    const int batches = (int)((k + GN_TENSORS - 1) / GN_TENSORS);
    const int cap = batches <= GN_MAX_PARTS / GN_BLOCKS ? GN_BLOCKS : GN_MAX_PARTS / batches;
    int nparts = 0;
    GradTable T;
    for (int b = 0; b < batches; ++b) {
        const int64_t at = (int64_t)b * GN_TENSORS;
        fill_table(T, pieces + at, (int)(k - at < GN_TENSORS ? k - at : GN_TENSORS));
        const int blocks = (int)(T.first[T.n] < cap ? T.first[T.n] : cap);
        DSW_LAUNCH(grad_norm_kernel<P>, dim3(blocks), dim3(GN_THREADS), 0, s, T, part + nparts);
        nparts += blocks;
    }
    if (!scale || batches == 0) {
        T.n = 0;
        DSW_LAUNCH((grad_clip_kernel<P, false>), dim3(1), dim3(GN_THREADS), 0, s, T, part, nparts, max_norm, norm);
        return dsw_check_launch();
    }
    int64_t bytes = 0;
    for (int64_t i = 0; i < k; ++i) bytes += pieces[i].n * (pieces[i].bf16 ? 2 : 4);
    const bool stream = bytes >= GN_STREAM_BYTES;
    for (int b = batches - 1; b >= 0; --b) {
        const int64_t at = (int64_t)b * GN_TENSORS;
        fill_table(T, pieces + at, (int)(k - at < GN_TENSORS ? k - at : GN_TENSORS));
        const int blocks = (int)(T.first[T.n] < 2 * GN_BLOCKS ? T.first[T.n] : 2 * GN_BLOCKS);
        float* const to = b == 0 ? norm : nullptr;
        if (stream) DSW_LAUNCH((grad_clip_kernel<P, true>), dim3(blocks), dim3(GN_THREADS), 0, s, T, part, nparts, max_norm, to);
        else DSW_LAUNCH((grad_clip_kernel<P, false>), dim3(blocks), dim3(GN_THREADS), 0, s, T, part, nparts, max_norm, to);
    }
    return dsw_check_launch();
}

}  // namespace

extern "C" {

int64_t dsw_grad_norm_workspace_bytes(void) { return (int64_t)GN_MAX_PARTS * 8; }

int dsw_grad_norm_clip(int n, const void* const* grads, void* const* outs, const int64_t* numel, const int32_t* dtypes,
                       double norm_type, double max_norm, float* norm, void* workspace, int64_t workspace_bytes,
                       dsw_stream_t stream) {
    const int kind = kind_of(norm_type);
    if (n < 0 || n > GN_MAX_PARTS * 8 || kind < 0 || !norm || (n > 0 && (!grads || !numel || !dtypes))) return DSW_ERR_BAD_ARG;
    if (outs && !(max_norm >= 0.0)) return DSW_ERR_BAD_ARG;
    if (!workspace || workspace_bytes < dsw_grad_norm_workspace_bytes() || ((uintptr_t)workspace & 7)) return DSW_ERR_WORKSPACE;
    for (int i = 0; i < n; ++i) {
        if (numel[i] < 0 || numel[i] > ((int64_t)1 << 40)) return DSW_ERR_BAD_ARG;
        if (dtypes[i] != DSW_F32 && dtypes[i] != DSW_BF16) return DSW_ERR_BAD_DTYPE;
        if (numel[i] > 0 && (!grads[i] || (outs && !outs[i]))) return DSW_ERR_BAD_ARG;
    }
    Piece* pieces = new (std::nothrow) Piece[n > 0 ? n : 1];
    if (!pieces) return DSW_ERR_WORKSPACE;
    const int64_t k = make_pieces(n, grads, outs, numel, dtypes, pieces);
    int rc = DSW_OK;
    if (outs && k > 0) {
        // no element may be written twice, nor read by one workgroup while another writes it: written ranges overlap nothing
        // but the gradient that they replace in place
        Range* r = new (std::nothrow) Range[2 * k];
        if (!r) rc = DSW_ERR_WORKSPACE;
        else {
            int64_t m = 0;
            for (int64_t i = 0; i < k; ++i) {
                const uintptr_t bytes = (uintptr_t)pieces[i].n * (pieces[i].bf16 ? 2 : 4);
                r[m++] = {(uintptr_t)pieces[i].o, (uintptr_t)pieces[i].o + bytes, true};
                if (pieces[i].g != pieces[i].o) r[m++] = {(uintptr_t)pieces[i].g, (uintptr_t)pieces[i].g + bytes, false};
            }
            if (!no_conflict(r, m)) rc = DSW_ERR_OVERLAP;
            delete[] r;
        }
    }
    if (rc == DSW_OK) {
        hipStream_t s = (hipStream_t)stream;
        DswTraceScope trace_(s, DSW_ROLE_GRAD_NORM, n, k, outs ? 1 : 0);
        double* part = static_cast<double*>(workspace);
        rc = kind == GN_L2 ? run_clip<GN_L2>(pieces, k, part, max_norm, outs != nullptr, norm, s)
           : kind == GN_L1 ? run_clip<GN_L1>(pieces, k, part, max_norm, outs != nullptr, norm, s)
                           : run_clip<GN_INF>(pieces, k, part, max_norm, outs != nullptr, norm, s);
    }
    delete[] pieces;
    return rc;
}

}  // extern "C"
