// Row-wise loads, stores and reductions of the kernels that normalise or quantise rows of channels (dsw_rmsnorm.hip).
#pragma once
#include "dsw_common.h"

namespace {

// 16 bytes of a row: 8 bf16 or 4 fp32 channels, as fp32 values.  Rows may start at any element: the loads are issued as 16-byte
// accesses without an alignment promise (gfx950 takes those in hardware), so that odd channel counts and channel slices take the
// same kernels as aligned rows.
template <bool BF16>
struct Row {
    static constexpr int V = BF16 ? 8 : 4;
    static constexpr int E = BF16 ? 2 : 4;
    typedef uint32_t __attribute__((ext_vector_type(4))) u32x4;
    struct __attribute__((packed, aligned(1))) Any { u32x4 v; };

    static __device__ __forceinline__ float one(const char* p) {
        if constexpr (BF16) return bf16_to_f32(*reinterpret_cast<const uint16_t*>(p));
        else return *reinterpret_cast<const float*>(p);
    }
    static __device__ __forceinline__ void put(char* p, float v) {
        if constexpr (BF16) *reinterpret_cast<uint16_t*>(p) = f32_to_bf16(v);
        else *reinterpret_cast<float*>(p) = v;
    }
    static __device__ __forceinline__ void unpack(const u32x4 t, float (&v)[V]) {
        if constexpr (BF16) {
#pragma unroll
            for (int j = 0; j < 4; ++j) { v[2 * j] = __uint_as_float(t[j] << 16); v[2 * j + 1] = __uint_as_float(t[j] & 0xffff0000u); }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(t[j]);
        }
    }
    static __device__ __forceinline__ u32x4 pack(const float (&v)[V]) {
        u32x4 t;
        if constexpr (BF16) {
#pragma unroll
            for (int j = 0; j < 4; ++j) t[j] = f32x2_to_bf16(v[2 * j], v[2 * j + 1]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) t[j] = __float_as_uint(v[j]);
        }
        return t;
    }
    static __device__ __forceinline__ u32x4 raw(const char* p) { return reinterpret_cast<const Any*>(p)->v; }
    static __device__ __forceinline__ void put_raw(char* p, const u32x4 t) { reinterpret_cast<Any*>(p)->v = t; }
    static __device__ __forceinline__ void put_raw_stream(char* p, const u32x4 t) {            // past the caches
        typedef uint32_t __attribute__((ext_vector_type(4), aligned(1))) any4;
        __builtin_nontemporal_store((any4)t, reinterpret_cast<any4*>(p));
    }
    // channels [0, n) of the 16 bytes at p; the others come back as zero (n >= V: all of them)
    static __device__ __forceinline__ void load(const char* p, int n, float (&v)[V]) {
        if (n >= V) {
            unpack(reinterpret_cast<const Any*>(p)->v, v);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = j < n ? one(p + j * E) : 0.f;
        }
    }
    // the same without the conversion: a lane's 16 bytes with zeros behind channel n (n <= 0: nothing is read)
    static __device__ __forceinline__ u32x4 fetch(const char* p, int n) {
        u32x4 t = {0u, 0u, 0u, 0u};
        if (n >= V) {
            t = reinterpret_cast<const Any*>(p)->v;
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (j < n) {
                    if constexpr (BF16) t[j / 2] |= (uint32_t)*reinterpret_cast<const uint16_t*>(p + j * E) << (16 * (j & 1));
                    else t[j] = *reinterpret_cast<const uint32_t*>(p + j * E);
                }
        }
        return t;
    }
    static __device__ __forceinline__ void store(char* p, int n, const float (&v)[V]) {
        if (n >= V) {
            reinterpret_cast<Any*>(p)->v = pack(v);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) if (j < n) put(p + j * E, v[j]);
        }
    }
};

// sum over the LPR lanes (a power of two, <= 64) that share a row; every lane gets it
template <int LPR>
static __device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int off = LPR / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}
template <int N>
static __device__ __forceinline__ uint32_t lanes_umax(uint32_t v) {
#pragma unroll
    for (int off = N / 2; off > 0; off >>= 1) { const uint32_t o = (uint32_t)__shfl_xor((int)v, off, 64); v = v > o ? v : o; }
    return v;
}

// sum over the TPR threads of a row: within the wave for TPR <= 64, through LDS for whole workgroups of 256 (red: 4 floats per
// use; `flip` alternates between two sets, so that one barrier per sum is enough)
template <int TPR>
static __device__ __forceinline__ float row_sum(float v, float (*red)[4], int flip) {
    if constexpr (TPR <= 64) {
        return lanes_sum<TPR>(v);
    } else {
        v = lanes_sum<64>(v);
        if ((threadIdx.x & 63) == 0) red[flip][threadIdx.x >> 6] = v;
        __syncthreads();
        return (red[flip][0] + red[flip][1]) + (red[flip][2] + red[flip][3]);
    }
}

// e4m3: largest finite value, and the scale of a block from the bit pattern of its largest magnitude.  Magnitudes are compared
// as bit patterns: NaN > inf > finite, so that a NaN of the block reaches its scale.  The floor 2^-126 (the smallest normal
// number) keeps 1 / scale finite and gives blocks of zeros a scale.
constexpr float E4M3_MAX = 448.f;
static __device__ __forceinline__ float e4m3_scale(uint32_t amax_bits) {
    const float s = __uint_as_float(amax_bits) / E4M3_MAX;
    return s < 1.17549435e-38f ? 1.17549435e-38f : s;       // (a NaN compares false and stays)
}
// v / s, rounded once to fp32: a value on the middle between two e4m3 values has to stay there.  The product with 1 / s is corrected
// by its remainder, which the fused multiply-add gives exactly while nothing of it leaves fp32's range (|v| <= 448 s; what is
// smaller than 2^-10 s rounds to zero or not whatever its last bits are); scales far out take the division itself.  Checked for all
// 2^23 significands of s around every middle: equal to the division.  (Three instructions a value instead of eleven.)
template <int V>
static __device__ __forceinline__ void e4m3_quotients(const float (&v)[V], float s, float (&q)[V]) {
    if (s >= 8.27180613e-25f && s <= 1.2676506e30f) {       // 2^-80 .. 2^100
        const float inv = 1.f / s;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float t = v[j] * inv;
            q[j] = fmaf(fmaf(-t, s, v[j]), inv, t);
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) q[j] = v[j] / s;
    }
}
// four values -> four e4m3 bytes, round to nearest even.  |v| <= 448 (1 + 2^-23): what lies above 448 by the rounding of the
// scale rounds to 448.
static __device__ __forceinline__ uint32_t e4m3_pack4(float a, float b, float c, float d) {
    int t = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, t, true);
}

}  // namespace
