// E4M3 codes with one fp32 scale per block of 128: the operands of the block-scaled product (fp8_gemm.cu).
//   activations  s[m, b] = max |x[m, 128 b ..]| / 448, a scale for every row and 128 columns
//   weights      s[i, b] = max |w[128 i .., 128 b ..]| / 448, a scale for every 128 x 128 tile
//   codes        q = e4m3(x / s): the fp32 quotient, then the nearest E4M3 value (ties to even)
// The scale is held in fp32; one that would be zero (a block of zeros, or of magnitudes below 448 times the smallest
// subnormal) becomes 1.  A block that holds a NaN or an infinity has that as its scale, and NaN codes.
//
// Both passes read a block once, keep it in registers and write codes and scale from there.

#include "common.cuh"
#include "fp8.cuh"

namespace mixfp4 {
namespace {

// A group of eight lanes per row and block (4096 x 4096 bf16: 10.5 to 11.4 us, 4.4 to 4.8 TB/s; issue slots 70 % busy, 15 thread
// instructions an element: fewer are possible, by indices that are carried along instead of
// divided and by paired fp32 operations; two blocks a group with their loads ahead 12.1 to 16.4, four 14.3; with 64-bit indices 12.1).
// scales: [block][lds], a row's scales a column of it, so that the product reads the scales of neighbouring rows together.
template <typename T>
__global__ void __launch_bounds__(256) fp8_rows_kernel(const T* x, uint32_t total, uint32_t blocks, int64_t k, int64_t ldx, bool vec,
                                                       uint8_t* codes, int64_t ldq, float* scales, int64_t lds) {
    asm volatile("griddepcontrol.wait;" ::: "memory");                       // x may be the kernel before's output
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int sub = threadIdx.x % kLanesPerRow;
    const uint32_t stride = gridDim.x * (256 / kLanesPerRow);
    for (uint32_t i = blockIdx.x * (256 / kLanesPerRow) + threadIdx.x / kLanesPerRow;; i += stride) {
        const bool in = i < total;
        if (!__any_sync(0xffffffffu, in)) break;
        const uint32_t at = in ? i / blocks : 0;
        const int64_t row = at, b = in ? i - at * blocks : 0;
        const int64_t c = b * kFp8Block + sub * kLaneElems;
        Raw<T> v;
        load16(x + row * ldx, c, in ? k : 0, vec, v);
        uint32_t a = largest_of(v);
#pragma unroll
        for (int d = 1; d < kLanesPerRow; d *= 2) a = larger<T>(a, __shfl_xor_sync(0xffffffffu, a, d));
        if (in) {
            const float s = block_scale(magnitude<T>(a));
            *reinterpret_cast<uint4*>(codes + row * ldq + c) = encode16(v, s);
            if (sub == 0) scales[b * lds + row] = s;
        }
    }
}

// Bound by HBM.  A CTA of 256 threads per 128 x 128 tile: 32 rows a pass, four passes, 64 elements a thread, kept as they were read: in 16 bits
// four CTAs fit an SM, and the loads of one hide behind the arithmetic of the others (14336 x 4096 bf16: 31 us, 5.7 TB/s;
// elements kept in fp32 by 512 threads, two CTAs an SM, 49 us; 512 threads and three CTAs 38 us; five CTAs of 256, 39 us).
// Rows off their 16 bytes are read an element at a time: 14333 x 4095 bf16 61 us, fp32 98 us (aligned 31 and 50).
constexpr int kTileThreads = 256, kTilePasses = 128 * kLanesPerRow / kTileThreads;
template <typename T>
__global__ void __launch_bounds__(kTileThreads, sizeof(T) == 2 ? 4 : 2) fp8_tiles_kernel(const T* w, int64_t n, int64_t k, int64_t ldw,
                                                                                        bool vec, uint8_t* codes, int64_t ldq,
                                                                                        float* scales) {
    __shared__ uint32_t warp_max[kTileThreads / 32];
    const int64_t blocks = (k + kFp8Block - 1) / kFp8Block;
    const int64_t tile = blockIdx.x / blocks, b = blockIdx.x - tile * blocks;
    const int sub = threadIdx.x % kLanesPerRow, first = threadIdx.x / kLanesPerRow;
    const int64_t c = b * kFp8Block + sub * kLaneElems;
    Raw<T> v[kTilePasses];
    uint32_t a = 0;
#pragma unroll
    for (int p = 0; p < kTilePasses; ++p) {
        const int64_t row = tile * kFp8Block + first + p * (kTileThreads / kLanesPerRow);
        load16(w + (row < n ? row : 0) * ldw, c, row < n ? k : 0, vec, v[p]);
    }
#pragma unroll
    for (int p = 0; p < kTilePasses; ++p) a = larger<T>(a, largest_of(v[p]));
#pragma unroll
    for (int d = 1; d < 32; d *= 2) a = larger<T>(a, __shfl_xor_sync(0xffffffffu, a, d));
    if (threadIdx.x % 32 == 0) warp_max[threadIdx.x / 32] = a;
    __syncthreads();
    a = warp_max[threadIdx.x % (kTileThreads / 32)];
#pragma unroll
    for (int d = 1; d < kTileThreads / 32; d *= 2) a = larger<T>(a, __shfl_xor_sync(0xffffffffu, a, d));
    const float s = block_scale(magnitude<T>(a));
    if (threadIdx.x == 0) scales[tile * blocks + b] = s;
#pragma unroll
    for (int p = 0; p < kTilePasses; ++p) {
        const int64_t row = tile * kFp8Block + first + p * (kTileThreads / kLanesPerRow);
        if (row < n) *reinterpret_cast<uint4*>(codes + row * ldq + c) = encode16(v[p], s);
    }
}

// y = code * scale, rounded once.  One thread per 4 columns, an element at a time: a form for checks and exports, simple rather than
// fast (14336 x 4096 to bf16 112 us, 1.6 TB/s, to fp32 123 us; its bytes alone 27 and 45 us at the copy rate; bound by instruction
// issue, 82 % of the slots, 57 thread instructions an element).
template <typename T>
__global__ void __launch_bounds__(256) fp8_dequant_kernel(const uint8_t* codes, int64_t ldq, const float* scales,
                                                          int64_t row_stride, int64_t block_stride, int rows_per_scale,
                                                          int64_t rows, int64_t k, T* y, int64_t ldy) {
    const int64_t quads = (k + 3) / 4, total = rows * quads;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t row = i / quads, c = (i - row * quads) * 4;
        const float s = __ldg(scales + row / rows_per_scale * row_stride + c / kFp8Block * block_stride);
        for (int j = 0; j < 4 && c + j < k; ++j)
            y[row * ldy + c + j] = Elem<T>::round(__fmul_rn(e4m3_to_float(codes[row * ldq + c + j]), s));
    }
}

template <typename F>
int by_type(int dtype, F&& f) {
    switch (dtype) {
        case MIXFP4_BF16: return f(__nv_bfloat16());
        case MIXFP4_F16: return f(__half());
        case MIXFP4_F32: return f(float());
        default: return MIXFP4_E_DTYPE;
    }
}
constexpr int64_t kMaxSide = 0x7fffffff;          // a tensor map's coordinates are 32-bit

}  // namespace

int fp8_check_rows(const void* x, int dtype, int64_t m, int64_t k, int64_t ldx, const uint8_t* codes, int64_t ldq,
                   const float* scales, int64_t lds) {
    if (!x || !codes || !scales) return MIXFP4_E_NULL;
    if (dtype != MIXFP4_BF16 && dtype != MIXFP4_F16 && dtype != MIXFP4_F32) return MIXFP4_E_DTYPE;
    if (m <= 0 || k <= 0 || m > kMaxSide || k > kMaxSide - 128 || ldx < k || ldq < padded_k(k) || lds < fp8_scale_rows(m))
        return MIXFP4_E_SHAPE;
    if (m * ((k + kFp8Block - 1) / kFp8Block) > kMaxSide) return MIXFP4_E_SHAPE;      // 2^38 elements
    if (!aligned(x, fp8_elem_bytes(dtype)) || !aligned(codes, 16) || ldq % 16 != 0 || !aligned(scales, 16) || lds % 4 != 0)
        return MIXFP4_E_ALIGN;
    return MIXFP4_OK;
}

int fp8_quantize_rows(const void* x, int dtype, int64_t m, int64_t k, int64_t ldx, uint8_t* codes, int64_t ldq,
                      float* scales, int64_t lds, cudaStream_t st) {
    return by_type(dtype, [&](auto t) -> int {
        using T = decltype(t);
        const bool vec = aligned(x, 16) && ldx * (int64_t)sizeof(T) % 16 == 0;
        const int64_t blocks = (k + kFp8Block - 1) / kFp8Block, groups = m * blocks, per_cta = 256 / kLanesPerRow;
        const int64_t ctas = (groups + per_cta - 1) / per_cta;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(ctas < 148 * 64 ? ctas : 148 * 64));
        cfg.blockDim = dim3(256);
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        MIXFP4_CUDA_CHECK(cudaLaunchKernelEx(&cfg, fp8_rows_kernel<T>, static_cast<const T*>(x), (uint32_t)groups, (uint32_t)blocks, k, ldx, vec, codes, ldq,
                                             scales, lds));
        return check_launch("fp8_rows_kernel");
    });
}

}  // namespace mixfp4

using namespace mixfp4;

extern "C" int64_t mixfp4_fp8_scale_rows(int64_t m) { return m <= 0 ? 0 : fp8_scale_rows(m); }

extern "C" int mixfp4_fp8_quantize_rows(const void* x, int dtype, int64_t m, int64_t k, int64_t ldx, uint8_t* codes,
                                        int64_t ldq, float* scales, int64_t lds, void* stream) {
    if (const int rc = fp8_check_rows(x, dtype, m, k, ldx, codes, ldq, scales, lds)) return rc;
    return fp8_quantize_rows(x, dtype, m, k, ldx, codes, ldq, scales, lds, static_cast<cudaStream_t>(stream));
}

extern "C" int mixfp4_fp8_quantize_tiles(const void* w, int dtype, int64_t n, int64_t k, int64_t ldw, uint8_t* codes,
                                         int64_t ldq, float* scales, void* stream) {
    if (!w || !codes || !scales) return MIXFP4_E_NULL;
    if (dtype != MIXFP4_BF16 && dtype != MIXFP4_F16 && dtype != MIXFP4_F32) return MIXFP4_E_DTYPE;
    if (n <= 0 || k <= 0 || n > kMaxSide - 128 || k > kMaxSide - 128 || ldw < k || ldq < padded_k(k)) return MIXFP4_E_SHAPE;
    const int64_t tiles = (n + kFp8Block - 1) / kFp8Block * ((k + kFp8Block - 1) / kFp8Block);
    if (tiles > kMaxSide) return MIXFP4_E_SHAPE;
    if (!aligned(w, fp8_elem_bytes(dtype)) || !aligned(codes, 16) || ldq % 16 != 0 || !aligned(scales, 4)) return MIXFP4_E_ALIGN;
    const bool vec = aligned(w, 16) && ldw * fp8_elem_bytes(dtype) % 16 == 0;
    return by_type(dtype, [&](auto t) -> int {
        using T = decltype(t);
        fp8_tiles_kernel<T><<<(unsigned)tiles, kTileThreads, 0, static_cast<cudaStream_t>(stream)>>>(
            static_cast<const T*>(w), n, k, ldw, vec, codes, ldq, scales);
        return check_launch("fp8_tiles_kernel");
    });
}

extern "C" int mixfp4_fp8_dequant(const uint8_t* codes, int64_t ldq, const float* scales, int64_t row_stride,
                                  int64_t block_stride, int rows_per_scale, int64_t rows, int64_t k, void* y, int out_dtype,
                                  int64_t ldy, void* stream) {
    if (!codes || !scales || !y) return MIXFP4_E_NULL;
    if (rows_per_scale != 1 && rows_per_scale != kFp8Block) return MIXFP4_E_MODE;
    if (rows <= 0 || k <= 0 || rows > kMaxSide || k > kMaxSide || ldq < k || ldy < k || row_stride < 0 || block_stride < 0)
        return MIXFP4_E_SHAPE;
    if (out_dtype != MIXFP4_BF16 && out_dtype != MIXFP4_F16 && out_dtype != MIXFP4_F32) return MIXFP4_E_DTYPE;
    if (!aligned(scales, 4) || !aligned(y, fp8_elem_bytes(out_dtype))) return MIXFP4_E_ALIGN;
    return by_type(out_dtype, [&](auto t) -> int {
        using T = decltype(t);
        const int64_t ctas = (rows * ((k + 3) / 4) + 255) / 256;
        fp8_dequant_kernel<T><<<(unsigned)(ctas < 148 * 64 ? ctas : 148 * 64), 256, 0, static_cast<cudaStream_t>(stream)>>>(
            codes, ldq, scales, row_stride, block_stride, rows_per_scale, rows, k, static_cast<T*>(y), ldy);
        return check_launch("fp8_dequant_kernel");
    });
}
