// Microscaled 4-bit floating point (MXFP4): quantisation, dequantisation and the products of 4-bit
// matrices.  The format is that of the Open Compute Project's microscaling specification: 32
// neighbours along K share one power of two, an element is a sign, two bits of exponent and one of
// mantissa (0, 0.5, 1, 1.5, 2, 3, 4, 6).  Declarations and layouts: include/b200gemm.h.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "internal.h"
#include "mxfp4.cuh"

namespace b200 {
namespace {

constexpr int kMxThreads = 256;

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  if constexpr (std::is_same<T, float>::value) return v;
  else if constexpr (std::is_same<T, __half>::value) return __half2float(v);
  else return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  if constexpr (std::is_same<T, float>::value) return v;
  else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}

// Eight neighbours of a row as fp32; elements at or beyond `left` (how many the row still has) are 0.
// VEC: the address is 16-byte aligned.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* __restrict__ src, int64_t left, float (&v)[8]) {
  if (VEC && left >= 8) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(src)), b = __ldg(reinterpret_cast<const float4*>(src) + 1);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(src));
      const T* e = reinterpret_cast<const T*>(&a);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = to_f32(e[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? to_f32(src[i]) : 0.0f;
  }
}

// Blocks along the rows of x [R, C].  Sixteen lanes take one word of four scales (128 elements of a
// row), eight elements a lane: a block's largest magnitude is a maximum over four lanes, its code
// words leave as 64 contiguous bytes, its four scale bytes as one word.  The grid also covers the
// rows that pad the last band of 128, whose scale bytes are zero.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kMxThreads)
mx_quantize_rows_kernel(const T* __restrict__ x, uint8_t* __restrict__ q, uint8_t* __restrict__ scale, int64_t R,
                        int64_t C, int64_t ldx, int64_t words, int64_t units) {
  const int l16 = threadIdx.x & 15;
  const int64_t row_bytes = mx_row_bytes(C);
  const int64_t step = int64_t(gridDim.x) * (kMxThreads / 16);
  // a whole warp stays in the loop together (the shuffles below name all lanes)
  const int64_t first = int64_t(blockIdx.x) * (kMxThreads / 16) + (threadIdx.x >> 4);
  for (int64_t u0 = first - ((threadIdx.x >> 4) & 1); u0 < units; u0 += step) {
    const int64_t u = u0 + ((threadIdx.x >> 4) & 1);
    const int64_t row = u / words, w = u - row * words;
    const int64_t k = w * 128 + l16 * 8;
    const bool live = u < units && row < R;
    float v[8];
    load8<T, VEC>(x + row * ldx + k, live ? C - k : 0, v);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, mx_magnitude(v[i]));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const uint32_t byte = mx_scale_byte(top);
    const uint32_t codes = mx_encode8(v, byte);
    if (live && k < row_bytes * 2) *reinterpret_cast<uint32_t*>(q + row * row_bytes + (k >> 1)) = codes;
    uint32_t word = byte << (8 * (l16 >> 2));
    word |= __shfl_xor_sync(0xffffffffu, word, 4);
    word |= __shfl_xor_sync(0xffffffffu, word, 8);
    if (l16 == 0 && u < units) *reinterpret_cast<uint32_t*>(scale + mx_scale_offset(row, w * 4, words)) = word;
  }
}

// Blocks down the columns of x [R, C]: row c of the result is column c of x.  A thread owns one
// column and four blocks of it (128 rows of x): consecutive lanes read consecutive columns, and what
// a thread writes is 64 contiguous bytes of codes and one word of scales.
template <typename T>
__global__ void __launch_bounds__(kMxThreads)
mx_quantize_cols_kernel(const T* __restrict__ x, uint8_t* __restrict__ q, uint8_t* __restrict__ scale, int64_t R,
                        int64_t C, int64_t ldx, int64_t words, int64_t padded_cols) {
  const int64_t c = int64_t(blockIdx.x) * kMxThreads + threadIdx.x;
  if (c >= padded_cols) return;
  const int64_t row_bytes = mx_row_bytes(R);
  for (int64_t w = blockIdx.y; w < words; w += gridDim.y) {
    uint32_t word = 0;
    for (int b = 0; b < 4; ++b) {
      const int64_t r0 = w * 128 + b * 32;
      float v[32];
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        v[i] = c < C && r0 + i < R ? to_f32(x[(r0 + i) * ldx + c]) : 0.0f;
        top = max(top, mx_magnitude(v[i]));
      }
      const uint32_t byte = mx_scale_byte(top);
      uint32_t codes[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float(&part)[8] = *reinterpret_cast<const float(*)[8]>(v + 8 * i);
        codes[i] = mx_encode8(part, byte);
      }
      if (c < C && r0 < R)
        *reinterpret_cast<uint4*>(q + c * row_bytes + (r0 >> 1)) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
      word |= byte << (8 * b);
    }
    *reinterpret_cast<uint32_t*>(scale + mx_scale_offset(c, w * 4, words)) = word;
  }
}

// A lane takes eight elements: one word of codes in, 16 or 32 bytes of values out.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kMxThreads)
mx_dequantize_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ scale, T* __restrict__ x, int64_t rows,
                     int64_t K, int64_t ldx, int64_t words, int64_t units) {
  const int64_t row_bytes = mx_row_bytes(K);
  const int64_t per_row = row_bytes / 4;
  for (int64_t u = int64_t(blockIdx.x) * kMxThreads + threadIdx.x; u < units; u += int64_t(gridDim.x) * kMxThreads) {
    const int64_t row = u / per_row, k = (u - row * per_row) * 8;
    float v[8];
    mx_decode8(*reinterpret_cast<const uint32_t*>(q + row * row_bytes + (k >> 1)),
               scale[mx_scale_offset(row, k / 32, words)], v);
    T* dst = x + row * ldx + k;
    if (VEC && k + 8 <= K) {
      if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
      } else {
        T h[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = from_f32<T>(v[i]);
        *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(h);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k + i < K) dst[i] = from_f32<T>(v[i]);
    }
  }
}

template <typename T>
int quantize_t(const T* x, uint8_t* q, uint8_t* scale, int64_t R, int64_t C, int64_t ldx, int along, cudaStream_t stream) {
  if (along == 0) {
    const int64_t words = (C + 127) / 128, units = (R + 127) / 128 * 128 * words;
    const int64_t want = (units + kMxThreads / 16 - 1) / (kMxThreads / 16);
    const int grid = int(want < 148 * 32 ? want : 148 * 32);
    const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx * int64_t(sizeof(T)) % 16 == 0;
    if (vec) mx_quantize_rows_kernel<T, true><<<grid, kMxThreads, 0, stream>>>(x, q, scale, R, C, ldx, words, units);
    else mx_quantize_rows_kernel<T, false><<<grid, kMxThreads, 0, stream>>>(x, q, scale, R, C, ldx, words, units);
  } else {
    const int64_t words = (R + 127) / 128, padded = (C + 127) / 128 * 128;
    dim3 grid(unsigned((padded + kMxThreads - 1) / kMxThreads), unsigned(words < 65535 ? words : 65535));
    mx_quantize_cols_kernel<T><<<grid, kMxThreads, 0, stream>>>(x, q, scale, R, C, ldx, words, padded);
  }
  B200_CUDA_TRY(cudaGetLastError());
  return B200_OK;
}

template <typename T>
int dequantize_t(const uint8_t* q, const uint8_t* scale, T* x, int64_t rows, int64_t K, int64_t ldx, cudaStream_t stream) {
  const int64_t words = (K + 127) / 128, units = rows * (mx_row_bytes(K) / 4);
  const int64_t want = (units + kMxThreads - 1) / kMxThreads;
  const int grid = int(want < 148 * 32 ? want : 148 * 32);
  const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx * int64_t(sizeof(T)) % 16 == 0;
  if (vec) mx_dequantize_kernel<T, true><<<grid, kMxThreads, 0, stream>>>(q, scale, x, rows, K, ldx, words, units);
  else mx_dequantize_kernel<T, false><<<grid, kMxThreads, 0, stream>>>(q, scale, x, rows, K, ldx, words, units);
  B200_CUDA_TRY(cudaGetLastError());
  return B200_OK;
}

bool float_dtype(int dtype) { return dtype == B200_F16 || dtype == B200_BF16 || dtype == B200_F32; }
int64_t dtype_bytes(int dtype) { return dtype == B200_F32 ? 4 : 2; }
constexpr int64_t kMxMaxDim = int64_t(1) << 30;

int check_packed(const char* what, const void* q, const void* scale) {
  if (!q || !scale) return fail(B200_ERR_BAD_ARGUMENT, "%s: null pointer", what);
  if (reinterpret_cast<uintptr_t>(q) % 16 || reinterpret_cast<uintptr_t>(scale) % 16)
    return fail(B200_ERR_UNSUPPORTED, "%s: packed elements and scales must be 16-byte aligned", what);
  return B200_OK;
}
int check_float(const char* what, int dtype, const void* p, int64_t rows, int64_t cols, int64_t ld) {
  if (!float_dtype(dtype)) return fail(B200_ERR_BAD_ARGUMENT, "%s: dtype %d is not a floating-point type", what, dtype);
  if (!p) return fail(B200_ERR_BAD_ARGUMENT, "%s: null pointer", what);
  if (rows <= 0 || cols <= 0) return fail(B200_ERR_BAD_ARGUMENT, "%s: sizes must be positive", what);
  if (rows > kMxMaxDim || cols > kMxMaxDim) return fail(B200_ERR_TOO_LARGE, "%s: a dimension exceeds 2^30", what);
  if (ld < cols) return fail(B200_ERR_BAD_ARGUMENT, "%s: a leading dimension is smaller than the row it spans", what);
  if (reinterpret_cast<uintptr_t>(p) % dtype_bytes(dtype))
    return fail(B200_ERR_UNSUPPORTED, "%s: matrix is not aligned to its element size", what);
  return B200_OK;
}

int quantize(int dtype, const void* x, void* q, void* scale, int64_t R, int64_t C, int64_t ldx, int along,
             cudaStream_t stream) {
  uint8_t* q8 = static_cast<uint8_t*>(q);
  uint8_t* s8 = static_cast<uint8_t*>(scale);
  switch (dtype) {
    case B200_F32: return quantize_t(static_cast<const float*>(x), q8, s8, R, C, ldx, along, stream);
    case B200_F16: return quantize_t(static_cast<const __half*>(x), q8, s8, R, C, ldx, along, stream);
    default: return quantize_t(static_cast<const __nv_bfloat16*>(x), q8, s8, R, C, ldx, along, stream);
  }
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" size_t b200_mxfp4_row_bytes(int64_t K) { return K > 0 ? size_t(mx_row_bytes(K)) : 0; }

extern "C" size_t b200_mxfp4_scale_bytes(int64_t rows, int64_t K) {
  return rows > 0 && K > 0 ? size_t((rows + 127) / 128) * size_t((K + 127) / 128) * 512 : 0;
}

extern "C" int b200_quantize_mxfp4(int dtype, const void* x, void* q, void* scale, int64_t R, int64_t C, int64_t ldx,
                                   int along, void* stream) {
  if (along != 0 && along != 1)
    return fail(B200_ERR_BAD_ARGUMENT, "quantize_mxfp4: along must be 0 (blocks in rows) or 1 (blocks in columns)");
  if (ldx == 0) ldx = C;
  int rc = check_float("quantize_mxfp4", dtype, x, R, C, ldx);
  if (!rc) rc = check_packed("quantize_mxfp4", q, scale);
  if (rc) return rc;
  return quantize(dtype, x, q, scale, R, C, ldx, along, static_cast<cudaStream_t>(stream));
}

extern "C" int b200_dequantize_mxfp4(int dtype, const void* q, const void* scale, void* x, int64_t rows, int64_t K,
                                     int64_t ldx, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (ldx == 0) ldx = K;
  int rc = check_float("dequantize_mxfp4", dtype, x, rows, K, ldx);
  if (!rc) rc = check_packed("dequantize_mxfp4", q, scale);
  if (rc) return rc;
  const uint8_t* q8 = static_cast<const uint8_t*>(q);
  const uint8_t* s8 = static_cast<const uint8_t*>(scale);
  switch (dtype) {
    case B200_F32: return dequantize_t(q8, s8, static_cast<float*>(x), rows, K, ldx, stream);
    case B200_F16: return dequantize_t(q8, s8, static_cast<__half*>(x), rows, K, ldx, stream);
    default: return dequantize_t(q8, s8, static_cast<__nv_bfloat16*>(x), rows, K, ldx, stream);
  }
}

extern "C" int b200_gemm_mxfp4(int out_dtype, const void* A, const void* a_scale, const void* B, const void* b_scale,
                               void* C, int64_t M, int64_t N, int64_t K, int64_t ldc, void* stream) {
  if (ldc == 0) ldc = N;
  int rc = check_float("gemm_mxfp4", out_dtype, C, M, N, ldc);
  if (!rc) rc = check_packed("gemm_mxfp4 (A)", A, a_scale);
  if (!rc) rc = check_packed("gemm_mxfp4 (B)", B, b_scale);
  if (rc) return rc;
  if (K <= 0) return fail(B200_ERR_BAD_ARGUMENT, "gemm_mxfp4: sizes must be positive");
  if (K > kMxMaxDim) return fail(B200_ERR_TOO_LARGE, "gemm_mxfp4: a dimension exceeds 2^30");
  MxGemm g;
  g.A = static_cast<const uint8_t*>(A);
  g.a_scale = static_cast<const uint8_t*>(a_scale);
  g.B = static_cast<const uint8_t*>(B);
  g.b_scale = static_cast<const uint8_t*>(b_scale);
  g.C = C;
  g.M = M;
  g.N = N;
  g.K = K;
  g.ldc = ldc;
  return launch_mx_gemm(out_dtype, g, static_cast<cudaStream_t>(stream));
}

extern "C" size_t b200_linear_mxfp4_workspace(int64_t batch, int64_t in_features) {
  if (batch <= 0 || in_features <= 0) return 0;
  return b200_mxfp4_scale_bytes(batch, in_features) + size_t(batch) * b200_mxfp4_row_bytes(in_features);
}

extern "C" int b200_linear_mxfp4(int dtype, const void* X, const void* W, const void* w_scale, const float* bias, void* Y,
                                 int64_t batch, int64_t in_features, int64_t out_features, int flags, void* workspace,
                                 size_t workspace_bytes, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  int rc = check_float("linear_mxfp4 (X)", dtype, X, batch, in_features, in_features);
  if (!rc) rc = check_float("linear_mxfp4 (Y)", dtype, Y, batch, out_features, out_features);
  if (!rc) rc = check_packed("linear_mxfp4 (W)", W, w_scale);
  if (rc) return rc;
  if (flags & ~(B200_LINEAR_RELU | B200_LINEAR_BIAS_FIRST)) return fail(B200_ERR_BAD_ARGUMENT, "unknown flags 0x%x", flags);
  if (bias && reinterpret_cast<uintptr_t>(bias) % 4)
    return fail(B200_ERR_UNSUPPORTED, "linear_mxfp4: bias is not aligned to its element size");
  if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16)
    return fail(B200_ERR_BAD_ARGUMENT, "linear_mxfp4: the workspace must be given, 16-byte aligned");
  const size_t need = b200_linear_mxfp4_workspace(batch, in_features);
  if (workspace_bytes < need)
    return fail(B200_ERR_BAD_ARGUMENT, "linear_mxfp4: the workspace has %zu bytes, %zu are needed", workspace_bytes, need);
  uint8_t* s = static_cast<uint8_t*>(workspace);
  uint8_t* q = s + b200_mxfp4_scale_bytes(batch, in_features);
  rc = quantize(dtype, X, q, s, batch, in_features, in_features, 0, stream);
  if (rc) return rc;
  MxGemm g;
  g.A = q;
  g.a_scale = s;
  g.B = static_cast<const uint8_t*>(W);
  g.b_scale = static_cast<const uint8_t*>(w_scale);
  g.C = Y;
  g.M = batch;
  g.N = out_features;
  g.K = in_features;
  g.ldc = out_features;
  g.tail.bias = bias;
  g.tail.flags = flags;
  return launch_mx_gemm(dtype, g, stream);
}
