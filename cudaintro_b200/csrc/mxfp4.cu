// Microscaled 4-bit floating point (MXFP4): quantisation, dequantisation, and the C entry points of the
// operators (the products' kernels are in gemm_mxfp4.cu).  The format is that of the Open Compute Project's
// microscaling specification: 32 neighbours along K share one power of two, an element is a sign, two bits of
// exponent and one of mantissa (0, 0.5, 1, 1.5, 2, 3, 4, 6).  Declarations and layouts: include/b200gemm.h.
//
// Bound: HBM.  A 16-bit element is read once and 17/32 of a byte written (or the reverse).  Measured, inputs rotated
// through more than L2, calls in a row in a CUDA graph: 8192 x 8192 bf16 along rows 29.5 us = 5.75 TB/s (0.88 of the measured
// copy), fp32 53.3 us = 5.7 TB/s; 4096 x 11008 along columns fp16 21.8 us = 5.25 TB/s, bf16 21.9 us, fp32 32.7 us = 6.2 TB/s; 11008 x
// 4096 back to bf16 20.6 us = 5.5 TB/s, 8192 x 8192 back to fp32 52.5 us = 5.8 TB/s.  Rows aligned to their element only: 4096 x
// 11007 fp16 26.5 us along rows and 27.8 back; 4097 x 11007 along columns fp16 41 us, fp32 37.5.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "internal.h"
#include "mxfp4.cuh"

namespace b200 {
namespace {

constexpr int kMxThreads = 256;

template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  if constexpr (std::is_same<T, float>::value) return v;
  else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}

// Set-up of a kernel in a stream: wait for the one before it, and let the next one (the product that takes what is
// quantised here) begin its own.  Nothing these kernels read is declared read-only for their lifetime (no __ldg, no
// __restrict__): the compiler may move such loads up past this wait.
__device__ __forceinline__ void mx_follow_stream() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// A warp's copy of `n` (at most 512) neighbours that are aligned to their element size only, into aligned shared memory;
// zeros up to 512.  16-bit elements are read as aligned words, the first element on its own where the address asks
// for it: consecutive lanes read consecutive words whatever the alignment.
template <typename T>
__device__ __forceinline__ void stage512(const T* src, int n, T* dst, int lane) {
  if constexpr (sizeof(T) == 4) {
    uint32_t r[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int e = i * 32 + lane;
      r[i] = e < n ? reinterpret_cast<const uint32_t*>(src)[e] : 0u;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) reinterpret_cast<uint32_t*>(dst)[i * 32 + lane] = r[i];
  } else {
    const int odd = int(reinterpret_cast<uintptr_t>(src) >> 1) & 1;
    const uint16_t* s16 = reinterpret_cast<const uint16_t*>(src);
    uint16_t* d16 = reinterpret_cast<uint16_t*>(dst);
    uint32_t r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = odd + 2 * (i * 32 + lane);  // the word holds elements e and e + 1
      r[i] = e + 1 < n ? *reinterpret_cast<const uint32_t*>(s16 + e) : e < n ? uint32_t(s16[e]) : 0u;
    }
    if (odd && lane == 0) d16[0] = n > 0 ? s16[0] : uint16_t(0);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = odd + 2 * (i * 32 + lane);
      d16[e] = uint16_t(r[i]);
      if (e + 1 < 512) d16[e + 1] = uint16_t(r[i] >> 16);
    }
  }
  __syncwarp();
}

// Blocks along the rows of x [R, C].  A warp takes STEPS times eight words of four scales of a row (a word covers 128
// elements): sixteen elements a lane, so a block's largest magnitude is a maximum over two lanes, the codes of a warp
// leave as 256 contiguous bytes, and eight lanes make a word of scales.  A lane has the loads of UNROLL times 16
// elements in flight.  The grid also covers the rows that pad the last band of 128, whose scale bytes are zero.
template <typename T, bool VEC, int STEPS>
__global__ void __launch_bounds__(kMxThreads)
mx_quantize_rows_kernel(const T* x, uint8_t* q, uint8_t* scale, int64_t R,
                        int64_t C, int64_t ldx, int words, int64_t padded_rows) {
  constexpr int chunk = 8 * STEPS;
  constexpr int UNROLL = sizeof(T) == 4 || !VEC ? 1 : 2;
  __shared__ alignas(16) T stage[VEC ? 1 : kMxThreads / 32][VEC ? 1 : 512];
  const int lane = threadIdx.x & 31;
  const int64_t row = int64_t(blockIdx.x) * (kMxThreads / 32) + (threadIdx.x >> 5);
  if (row >= padded_rows) return;  // whole warps
  const int64_t row_bytes = mx_row_bytes(C);
  const bool live = row < R;
  const int end = min(words, (int(blockIdx.y) + 1) * chunk);
  mx_follow_stream();
  for (int w0 = int(blockIdx.y) * chunk; w0 < end; w0 += 4 * UNROLL) {
    Sixteen<T> raw[UNROLL];
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
      const int64_t k = int64_t(w0 + 4 * i) * 128 + lane * 16;
      if constexpr (VEC) {
        load16(x + row * ldx + k, live ? C - k : 0, raw[i]);
      } else {
        const int64_t k0 = int64_t(w0) * 128;
        T* buf = stage[threadIdx.x >> 5];
        __syncwarp();
        stage512(x + row * ldx + k0, live ? int(min(C - k0, int64_t(512))) : 0, buf, lane);
#pragma unroll
        for (int j = 0; j < Sixteen<T>::WORDS; ++j) raw[i].w[j] = reinterpret_cast<const uint32_t*>(buf)[lane * Sixteen<T>::WORDS + j];
      }
    }
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
      const int word = w0 + 4 * i + (lane >> 3);
      const int64_t k = int64_t(w0 + 4 * i) * 128 + lane * 16;
      uint32_t top = top_of<T, Sixteen<T>::WORDS>(raw[i].w);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      const uint32_t byte = mx_scale_byte(top);
      const uint2 codes = encode16(raw[i], byte);
      if (live && k < row_bytes * 2) *reinterpret_cast<uint2*>(q + row * row_bytes + (k >> 1)) = codes;
      uint32_t four = byte << (4 * (lane & 6));
      four |= __shfl_xor_sync(0xffffffffu, four, 2);
      four |= __shfl_xor_sync(0xffffffffu, four, 4);
      if ((lane & 7) == 0 && word < words)
        *reinterpret_cast<uint32_t*>(scale + mx_scale_offset(row, int64_t(word) * 4, words)) = four;
    }
  }
}

// Blocks down the columns of x [R, C]: row c of the result is column c of x.  A CTA takes 256 rows of x (eight
// blocks, one a warp) and 64 columns, two a lane: a warp reads whole 128-byte (fp32: 256-byte) pieces of 32
// rows, a lane then has both of its columns' blocks in registers.  The codes meet in shared memory, from where a
// column's 128 bytes leave as one line, and the scale bytes as words.  VEC: pairs of columns are aligned.
constexpr int kColTileK = 256, kColTileC = 64;
template <typename T, bool VEC>
__global__ void __launch_bounds__(kMxThreads, sizeof(T) == 4 || !VEC ? 2 : 3)
mx_quantize_cols_kernel(const T* x, uint8_t* q, uint8_t* scale, int64_t R,
                        int64_t C, int64_t ldx, int words) {
  constexpr int WORDS = sizeof(T) == 4 ? 64 : 32;   // a word is a pair of 16-bit values or one of two fp32 values
  __shared__ uint4 codes[kColTileC][9];             // 128 bytes of codes a column, and 16 that part the banks
  __shared__ __align__(4) uint8_t bytes[kColTileC][8];  // scale bytes of a column's eight blocks
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row_bytes = mx_row_bytes(R);
  const int64_t c = int64_t(blockIdx.x) * kColTileC + 2 * lane;
  mx_follow_stream();
  for (int64_t k0 = int64_t(blockIdx.y) * kColTileK; k0 < int64_t(words) * 128; k0 += int64_t(gridDim.y) * kColTileK) {
    const int64_t r0 = k0 + warp * 32;
    const T* src = x + r0 * ldx + c;
    uint32_t raw[WORDS];  // fp32: row i's two values at i and 32 + i
    if (VEC && c + 1 < C && r0 + 32 <= R) {
#pragma unroll
      for (int i = 0; i < 32; ++i, src += ldx) {
        if constexpr (sizeof(T) == 4) {
          const uint2 u = __ldcg(reinterpret_cast<const uint2*>(src));
          raw[i] = u.x;
          raw[32 + i] = u.y;
        } else {
          raw[i] = __ldcg(reinterpret_cast<const uint32_t*>(src));
        }
      }
    } else if (!VEC && int64_t(blockIdx.x + 1) * kColTileC <= C && r0 + 32 <= R) {
      // inside x, whatever the alignment: no condition between the loads, so that all of them are in flight (with one
      // each: 156 us for 4097 x 11007 fp16, this 41)
#pragma unroll
      for (int i = 0; i < 32; ++i, src += ldx) {
        if constexpr (sizeof(T) == 4) {
          raw[i] = __float_as_uint(__ldcg(reinterpret_cast<const float*>(src)));
          raw[32 + i] = __float_as_uint(__ldcg(reinterpret_cast<const float*>(src) + 1));
        } else {
          const uint16_t* h = reinterpret_cast<const uint16_t*>(src);
          raw[i] = uint32_t(__ldcg(h)) | (uint32_t(__ldcg(h + 1)) << 16);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i, src += ldx) {
        const bool in = r0 + i < R;
        if constexpr (sizeof(T) == 4) {
          raw[i] = in && c < C ? __float_as_uint(src[0]) : 0u;
          raw[32 + i] = in && c + 1 < C ? __float_as_uint(src[1]) : 0u;
        } else {
          const uint16_t* h = reinterpret_cast<const uint16_t*>(src);
          raw[i] = (in && c < C ? uint32_t(h[0]) : 0u) | (in && c + 1 < C ? uint32_t(h[1]) << 16 : 0u);
        }
      }
    }
    uint32_t top[2];
    if constexpr (sizeof(T) == 4) {
      top[0] = top_of<T, 32>(raw);
      top[1] = top_of<T, 32>(raw + 32);
    } else {
      uint32_t both = 0;
#pragma unroll
      for (int i = 0; i < 32; ++i) both = __vmaxu2(both, raw[i] & 0x7fff7fffu);
      top[0] = __float_as_uint(half_of<T>(both, 0));
      top[1] = __float_as_uint(half_of<T>(both, 1));
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t byte = mx_scale_byte(top[h]);
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if constexpr (sizeof(T) == 4) v[j] = __uint_as_float(raw[32 * h + 8 * i + j]);
          else v[j] = half_of<T>(raw[8 * i + j], h);
        }
        w[i] = mx_encode8(v, byte);
      }
      codes[2 * lane + h][warp] = make_uint4(w[0], w[1], w[2], w[3]);
      bytes[2 * lane + h][warp] = uint8_t(byte);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kColTileC * 8 / kMxThreads; ++i) {
      const int u = i * kMxThreads + threadIdx.x, col = u >> 3, piece = u & 7;
      const int64_t row = int64_t(blockIdx.x) * kColTileC + col, at = (k0 >> 1) + piece * 16;
      if (row < C && at < row_bytes) *reinterpret_cast<uint4*>(q + row * row_bytes + at) = codes[col][piece];
    }
    if (threadIdx.x < 2 * kColTileC) {
      const int col = threadIdx.x >> 1, half = threadIdx.x & 1;
      const int64_t row = int64_t(blockIdx.x) * kColTileC + col, block = k0 / 32 + half * 4;
      if (block < int64_t(words) * 4)
        *reinterpret_cast<uint32_t*>(scale + mx_scale_offset(row, block, words)) =
            *reinterpret_cast<const uint32_t*>(&bytes[col][half * 4]);
    }
    __syncthreads();
  }
}

// A warp takes STEPS times 1024 elements of a row, a lane 16 bytes of values (eight or four elements) at a time.  VEC
// (16-byte aligned rows): they are stored as such.  Otherwise the values of 32 x 16 bytes meet in shared memory and leave
// as words, consecutive lanes consecutive words (stored from the lanes' registers, element by element, rows of 11007 16-bit
// values cost 142 us where these take 28).
template <typename T, bool VEC, int STEPS>
__global__ void __launch_bounds__(kMxThreads)
mx_dequantize_kernel(const uint8_t* q, const uint8_t* scale, T* x, int64_t rows, int64_t K, int64_t ldx, int words) {
  constexpr int chunk = 1024 * STEPS;
  constexpr int N = 16 / int(sizeof(T));  // neighbours a lane takes
  constexpr int UNROLL = 4;
  __shared__ alignas(16) T stage[VEC ? 1 : kMxThreads / 32][VEC ? 1 : 32 * N];
  const int lane = threadIdx.x & 31;
  const int64_t row = int64_t(blockIdx.x) * (kMxThreads / 32) + (threadIdx.x >> 5);
  if (row >= rows) return;  // whole warps
  const uint8_t* qr = q + row * mx_row_bytes(K);
  const uint8_t* sr = scale + mx_scale_offset(row, 0, words);
  T* xr = x + row * ldx;
  const int64_t end = min(K, (int64_t(blockIdx.y) + 1) * chunk);
  mx_follow_stream();
  for (int64_t first = int64_t(blockIdx.y) * chunk; first < end; first += 32 * N * UNROLL) {
    uint32_t codes[UNROLL], byte[UNROLL];
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
      const int64_t k = first + (i * 32 + lane) * N;
      codes[i] = byte[i] = 0;
      if (k < end) {
        if constexpr (N == 8) codes[i] = __ldcg(reinterpret_cast<const uint32_t*>(qr + (k >> 1)));
        else codes[i] = __ldcg(reinterpret_cast<const uint16_t*>(qr + (k >> 1)));
        byte[i] = sr[(k >> 7) * 512 + ((k >> 5) & 3)];
      }
    }
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
      const int64_t k0 = first + i * 32 * N, k = k0 + lane * N;
      if (k0 >= end) break;  // the whole warp
      float v[8];
      mx_decode8(codes[i], byte[i], v);
      alignas(16) T h[N];
#pragma unroll
      for (int j = 0; j < N; ++j) h[j] = from_f32<T>(v[j]);
      if constexpr (VEC) {
        if (k + N <= K) {
          *reinterpret_cast<uint4*>(xr + k) = *reinterpret_cast<const uint4*>(h);
        } else {
#pragma unroll
          for (int j = 0; j < N; ++j)
            if (k + j < K) xr[k + j] = h[j];
        }
      } else {
        T* buf = stage[threadIdx.x >> 5];
        *reinterpret_cast<uint4*>(buf + lane * N) = *reinterpret_cast<const uint4*>(h);
        __syncwarp();
        const int n = int(min(K - k0, int64_t(32 * N)));
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int j = 0; j < N; ++j)
            if (j * 32 + lane < n) xr[k0 + j * 32 + lane] = buf[j * 32 + lane];
        } else {
          const uint16_t* b16 = reinterpret_cast<const uint16_t*>(buf);
          uint16_t* d16 = reinterpret_cast<uint16_t*>(xr + k0);
          const int odd = int(reinterpret_cast<uintptr_t>(d16) >> 1) & 1;
          if (odd && lane == 0) d16[0] = b16[0];
#pragma unroll
          for (int j = 0; j < N / 2; ++j) {
            const int e = odd + 2 * (j * 32 + lane);
            if (e + 1 < n) *reinterpret_cast<uint32_t*>(d16 + e) = uint32_t(b16[e]) | (uint32_t(b16[e + 1]) << 16);
            else if (e < n) d16[e] = b16[e];
          }
        }
        __syncwarp();
      }
    }
  }
}

// A grid that fills the GPU is launched so that its CTAs may take their places before the kernel ahead of it in the stream
// has ended (11008 x 4096 back to bf16, calls in a row in a CUDA graph: 20.2 us, 20.5 plainly).  A smaller one is not: all of it
// would crowd on the SMs that the kernel ahead leaves first (a layer of 2048 x 4096 -> 11008, whose quantiser has 256 CTAs: 46.8 us,
// 44.7 plainly).
template <typename... Args>
int launch_in_stream(void (*kernel)(Args...), dim3 grid, cudaStream_t stream, std::decay_t<Args>... args) {
  constexpr int64_t kFull = 148 * 8;  // CTAs of 256 threads that the GPU holds
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kMxThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent_launch_enabled() && int64_t(grid.x) * grid.y >= kFull ? 1 : 0;
  B200_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, args...));
  return B200_OK;
}

// 1024-element steps of a row that a warp takes: kSteps, or one where kSteps would leave the GPU's warps without work
// (2048 x 4096 with four steps a warp / with one, us: bf16 7.4 / 5.7, fp32 10.9 / 9.1, back to bf16 7.5 / 5.8, to fp32 11.8 / 9.3).
// Where there are warps enough the two are close, but for fp32 along rows: 8192 x 8192 bf16 29.5 / 29.3, fp32 53.3 / 48.4, back to
// bf16 29.5 / 29.3, to fp32 52.5 / 51.9; 11008 x 4096 back to bf16 20.7 / 20.6.  A constant of the kernel: as an argument it
// cost the last of these 3 %.
constexpr int kSteps = 4;
int steps_per_warp(int64_t rows, int64_t steps) {
  return rows * ((steps + kSteps - 1) / kSteps) >= 148 * 48 ? kSteps : 1;
}

template <typename T>
int quantize_t(const T* x, uint8_t* q, uint8_t* scale, int64_t R, int64_t C, int64_t ldx, int along, cudaStream_t stream) {
  if (along == 0) {
    const int64_t words = (C + 127) / 128, padded = (R + 127) / 128 * 128;
    const int steps = steps_per_warp(R, (words + 7) / 8);
    const int64_t chunks = (words + 8 * steps - 1) / (8 * steps);
    if (chunks > 65535) return fail(B200_ERR_TOO_LARGE, "quantize_mxfp4: rows longer than %lld", 65535LL * 1024 * kSteps);
    const dim3 grid(unsigned(padded / (kMxThreads / 32)), unsigned(chunks));
    const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx * int64_t(sizeof(T)) % 16 == 0;
    auto kernel = steps == 1 ? (vec ? mx_quantize_rows_kernel<T, true, 1> : mx_quantize_rows_kernel<T, false, 1>)
                             : (vec ? mx_quantize_rows_kernel<T, true, kSteps> : mx_quantize_rows_kernel<T, false, kSteps>);
    return launch_in_stream(kernel, grid, stream, x, q, scale, R, C, ldx, int(words), padded);
  }
  const int64_t words = (R + 127) / 128, padded = (C + 127) / 128 * 128, tall = (words * 128 + kColTileK - 1) / kColTileK;
  const dim3 grid(unsigned(padded / kColTileC), unsigned(tall < 65535 ? tall : 65535));
  const bool vec = reinterpret_cast<uintptr_t>(x) % (2 * sizeof(T)) == 0 && ldx % 2 == 0;
  return launch_in_stream(vec ? mx_quantize_cols_kernel<T, true> : mx_quantize_cols_kernel<T, false>, grid, stream, x, q,
                          scale, R, C, ldx, int(words));
}

template <typename T>
int dequantize_t(const uint8_t* q, const uint8_t* scale, T* x, int64_t rows, int64_t K, int64_t ldx, cudaStream_t stream) {
  const int64_t words = (K + 127) / 128;
  const int steps = steps_per_warp(rows, (K + 1023) / 1024);
  const int64_t chunks = (K + 1024 * steps - 1) / (1024 * steps);
  if (chunks > 65535) return fail(B200_ERR_TOO_LARGE, "dequantize_mxfp4: rows longer than %lld", 65535LL * 1024 * kSteps);
  const dim3 grid(unsigned((rows + kMxThreads / 32 - 1) / (kMxThreads / 32)), unsigned(chunks));
  const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx * int64_t(sizeof(T)) % 16 == 0;
  auto kernel = steps == 1 ? (vec ? mx_dequantize_kernel<T, true, 1> : mx_dequantize_kernel<T, false, 1>)
                           : (vec ? mx_dequantize_kernel<T, true, kSteps> : mx_dequantize_kernel<T, false, kSteps>);
  return launch_in_stream(kernel, grid, stream, q, scale, x, rows, K, ldx, int(words));
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

extern "C" size_t b200_linear_mxfp4_workspace(int64_t batch, int64_t in_features, int64_t out_features) {
  if (batch <= 0 || in_features <= 0 || out_features <= 0) return 0;
  if (mx_layer_in_one_launch(batch, in_features, out_features)) return 0;
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
  MxGemm g;
  g.X = X;
  g.B = static_cast<const uint8_t*>(W);
  g.b_scale = static_cast<const uint8_t*>(w_scale);
  g.C = Y;
  g.M = batch;
  g.N = out_features;
  g.K = in_features;
  g.ldc = out_features;
  g.tail.bias = bias;
  g.tail.flags = flags;
  const size_t need = b200_linear_mxfp4_workspace(batch, in_features, out_features);
  if (need && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16))
    return fail(B200_ERR_BAD_ARGUMENT, "linear_mxfp4: the workspace must be given, 16-byte aligned");
  if (workspace_bytes < need)
    return fail(B200_ERR_BAD_ARGUMENT, "linear_mxfp4: the workspace has %zu bytes, %zu are needed", workspace_bytes, need);
  if (!need) return launch_mx_layer(dtype, g, stream);
  uint8_t* s = static_cast<uint8_t*>(workspace);
  uint8_t* q = s + b200_mxfp4_scale_bytes(batch, in_features);
  rc = quantize(dtype, X, q, s, batch, in_features, in_features, 0, stream);
  if (rc) return rc;
  g.A = q;
  g.a_scale = s;
  return launch_mx_gemm(dtype, g, stream);
}
