// Shared by the block-scaled E4M3 quantizer and product (fp8_quantize.cu, fp8_gemm.cu).
#pragma once

#include "common.cuh"

namespace mixfp4 {

constexpr int kFp8Block = 128;
// Rows that a scale array of activations has room for: the product fetches the scales of up to 128 rows at once.
__host__ __device__ inline int64_t fp8_scale_rows(int64_t m) { return (m + 127) / 128 * 128; }

// Whether a product quantizes a dense x itself, in every CTA: up to 256 row blocks and 48 blocks of K (what shared memory holds
// of it beside the weights' ring).  Itself / by a kernel ahead of it, on the device: 1 x 4096 x 4096 8.3 / 10.1 us, 4 rows
// 8.8 / 10.1, 8 rows (256 blocks) 9.4 / 10.0, 16 rows (512) 10.9 / 10.0, 32 x 4096 x 1024 (256) 8.0 / 7.3; and the host has
// one launch and no workspace for it.
inline bool fp8_quantizes_itself(int64_t m, int64_t k) {
    const int64_t blocks = (k + kFp8Block - 1) / kFp8Block;
    return m <= 64 && blocks <= 48 && m * blocks <= 256;
}

inline int fp8_elem_bytes(int dtype) { return dtype == MIXFP4_F32 ? 4 : 2; }

// Arguments of mixfp4_fp8_quantize_rows, checked before any CUDA call; then the pass itself.
int fp8_check_rows(const void* x, int dtype, int64_t m, int64_t k, int64_t ldx, const uint8_t* codes, int64_t ldq,
                   const float* scales, int64_t lds);
int fp8_quantize_rows(const void* x, int dtype, int64_t m, int64_t k, int64_t ldx, uint8_t* codes, int64_t ldq,
                      float* scales, int64_t lds, cudaStream_t st);

namespace {

constexpr float kFp8Largest = 448.0f;
constexpr int kLaneElems = 16, kLanesPerRow = kFp8Block / kLaneElems;       // a lane holds 16 elements of a row's block

// 16 consecutive elements of a row, as they lie in memory (two to a register where they have 16 bits).
template <typename T>
struct Raw {
    static constexpr int kQuads = sizeof(T);
    uint4 q[kQuads];
};
// From column c on, zero past k.  (Ordinary loads: x may be what a kernel that was still running at this one's start wrote.)
template <typename T>
__device__ __forceinline__ void load16(const T* row, int64_t c, int64_t k, bool vec, Raw<T>& v) {
    if (vec && c + kLaneElems <= k) {
#pragma unroll
        for (int i = 0; i < Raw<T>::kQuads; ++i) v.q[i] = reinterpret_cast<const uint4*>(row + c)[i];
    } else {
        T* e = reinterpret_cast<T*>(v.q);
#pragma unroll
        for (int j = 0; j < kLaneElems; ++j) e[j] = c + j < k ? row[c + j] : Elem<T>::round(0.0f);
    }
}
// Magnitudes compare as integers, and a NaN is the largest of all: two 16-bit ones at once, or one of 32.
template <typename T>
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    if constexpr (sizeof(T) == 2) return __vmaxu2(a, b);
    else return max(a, b);
}
template <typename T>
__device__ __forceinline__ uint32_t largest_of(const Raw<T>& v) {
    constexpr uint32_t kMagnitude = sizeof(T) == 2 ? 0x7fff7fffu : 0x7fffffffu;
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < Raw<T>::kQuads; ++i) {
        a = larger<T>(a, v.q[i].x & kMagnitude);
        a = larger<T>(a, v.q[i].y & kMagnitude);
        a = larger<T>(a, v.q[i].z & kMagnitude);
        a = larger<T>(a, v.q[i].w & kMagnitude);
    }
    return a;
}
template <typename T>
__device__ __forceinline__ float magnitude(uint32_t a) {
    if constexpr (sizeof(T) == 4) {
        return __uint_as_float(a);
    } else {
        const uint16_t bits = (uint16_t)max(a >> 16, a & 0xffffu);
        return Elem<T>::load(reinterpret_cast<const T*>(&bits));
    }
}

__device__ __forceinline__ float block_scale(float largest) {
    const float s = __fdiv_rn(largest, kFp8Largest);
    return s == 0.0f ? 1.0f : s;
}

// x / s rounded once, for the 16 values of a lane.  One reciprocal for all of them and a residual step each:
// q = x r, then q + (x - q s) r, which is the rounded quotient when r is the rounded reciprocal and nothing
// underflows (Markstein 1990, theorem on final rounding).  Scales outside 2^+-100 take the division itself.
template <typename T>
__device__ __forceinline__ uint4 encode16(const Raw<T>& raw, float s) {
    float v[kLaneElems], q[kLaneElems];
#pragma unroll
    for (int j = 0; j < kLaneElems; ++j) v[j] = Elem<T>::load(reinterpret_cast<const T*>(raw.q) + j);
    if (s > 0x1p-100f && s < 0x1p100f) {
        const float r = __frcp_rn(s);
#pragma unroll
        for (int j = 0; j < kLaneElems; ++j) {
            const float q0 = __fmul_rn(v[j], r);
            q[j] = __fmaf_rn(__fmaf_rn(-q0, s, v[j]), r, q0);
        }
    } else {
#pragma unroll
        for (int j = 0; j < kLaneElems; ++j) q[j] = __fdiv_rn(v[j], s);
    }
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(q[4 * i], q[4 * i + 1]), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(q[4 * i + 2], q[4 * i + 3]), __NV_SATFINITE, __NV_E4M3);
        w[i] = lo | (hi << 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

}  // namespace
}  // namespace mixfp4
