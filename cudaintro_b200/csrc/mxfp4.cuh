// The MXFP4 format on the device: scale bytes, element codes, and where a scale byte lies.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

#include "internal.h"

namespace b200 {

// A product of two 4-bit matrices, C[M,N] = A[M,K] * B[N,K]^T, with the optional tail of a layer.
struct MxGemm {
  const uint8_t* A = nullptr;  // or X, rows that are yet to be quantised (launch_mx_layer)
  const void* X = nullptr;
  const uint8_t* a_scale = nullptr;
  const uint8_t* B = nullptr;
  const uint8_t* b_scale = nullptr;
  void* C = nullptr;
  int64_t M = 0, N = 0, K = 0, ldc = 0;
  Tail tail;
};

// Bytes of one packed row: whole blocks of 32 elements, 16 bytes each.
__host__ __device__ __forceinline__ int64_t mx_row_bytes(int64_t K) { return (K + 31) / 32 * 16; }

// Scale bytes lie in tiles of 128 rows x 4 blocks (512 bytes; `words` tiles along K make a band): in a
// tile, 32 lines of 16 bytes, line l holding the four bytes of rows l, l + 32, l + 64, l + 96.  One
// tcgen05.cp.32x128b moves such a tile into four columns of tensor memory, where the tensor cores
// look for it.
__host__ __device__ __forceinline__ int64_t mx_scale_offset(int64_t row, int64_t block, int64_t words) {
  return ((row >> 7) * words + (block >> 2)) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}

// Scale byte of a block whose largest magnitude has the fp32 bits `top` (taken as an integer maximum, which keeps NaN
// and infinity in sight): the element format's largest power
// of two is 4, so the exponent is floor(log2 max) - 2, kept at -127 and above (zero blocks too).  A block
// with an infinity or a NaN in it gets 255, the scale format's NaN.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t top) {
  const uint32_t e = top >> 23;
  return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}

// Codes of eight elements under a scale byte, element i in bits [4i, 4i + 4): x / 2^E rounded to nearest,
// ties to the even code, magnitudes beyond 6 taken to 6.  1 / 2^E is a normal fp32 number for every
// byte up to 253, so the product is exact wherever it does not vanish.
__device__ __forceinline__ uint32_t mx_encode8(const float* v, uint32_t byte) {
  if (byte == 255u) return 0u;
  const float inv = __uint_as_float((254u - byte) << 23);
  uint32_t pair[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    asm("{\n\t.reg .b8 b;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %1, %2;\n\tcvt.u32.u8 %0, b;\n\t}"
        : "=r"(pair[i])
        : "f"(v[2 * i + 1] * inv), "f"(v[2 * i] * inv));
  return __byte_perm(__byte_perm(pair[0], pair[1], 0x0040), __byte_perm(pair[2], pair[3], 0x0040), 0x5410);
}

// Value of a scale byte: 2^(byte - 127); 0 is a subnormal fp32 number, 255 is NaN.
__device__ __forceinline__ float mx_scale_value(uint32_t byte) {
  return byte == 255u ? __uint_as_float(0x7fffffffu) : byte == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
}

// Values of eight codes, times the scale.
__device__ __forceinline__ void mx_decode8(uint32_t codes, uint32_t byte, float (&v)[8]) {
  const float s = mx_scale_value(byte);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t h;
    asm("{\n\t.reg .b8 b;\n\tcvt.u8.u32 b, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b;\n\t}" : "=r"(h) : "r"(codes >> (8 * i)));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    v[2 * i] = f.x * s;
    v[2 * i + 1] = f.y * s;
  }
}

// Sixteen neighbours of a row, as they lie in memory: words of two 16-bit values, or of one fp32 value.
template <typename T>
struct Sixteen {
  static constexpr int WORDS = 4 * sizeof(T);
  uint32_t w[WORDS];
};
// The address is 16-byte aligned if `vec`; elements at or beyond `left` (how many the row still has) are 0.
template <typename T>
__device__ __forceinline__ void load16(const T* src, int64_t left, Sixteen<T>& v, bool vec = true) {
  if (vec && left >= 16) {
#pragma unroll
    for (int i = 0; i < Sixteen<T>::WORDS / 4; ++i) {
      const uint4 u = __ldcg(reinterpret_cast<const uint4*>(src) + i);
      v.w[4 * i] = u.x; v.w[4 * i + 1] = u.y; v.w[4 * i + 2] = u.z; v.w[4 * i + 3] = u.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if constexpr (sizeof(T) == 4) {
        v.w[i] = i < left ? __float_as_uint(src[i]) : 0u;
      } else {
        const uint32_t e = i < left ? reinterpret_cast<const uint16_t*>(src)[i] : 0u;
        v.w[i / 2] = i & 1 ? v.w[i / 2] | (e << 16) : e;
      }
    }
  }
}

// Low or high 16-bit value of a word as fp32.
template <typename T>
__device__ __forceinline__ float half_of(uint32_t w, int high) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = *reinterpret_cast<const __half2*>(&w);
    return high ? __high2float(h) : __low2float(h);
  } else {
    return __uint_as_float(high ? w & 0xffff0000u : w << 16);
  }
}
// The largest magnitude among `N` words, as fp32 bits (NaN above infinity): of 16-bit types both halves of a word
// are compared at once.
template <typename T, int N>
__device__ __forceinline__ uint32_t top_of(const uint32_t* w) {
  if constexpr (sizeof(T) == 4) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) top = max(top, w[i] & 0x7fffffffu);
    return top;
  } else {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) top = __vmaxu2(top, w[i] & 0x7fff7fffu);
    return max(__float_as_uint(half_of<T>(top, 0)), __float_as_uint(half_of<T>(top, 1)));
  }
}

// Codes of sixteen elements under a scale byte.
template <typename T>
__device__ __forceinline__ uint2 encode16(const Sixteen<T>& x, uint32_t byte) {
  float v[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    if constexpr (sizeof(T) == 4) v[j] = __uint_as_float(x.w[j]);
    else v[j] = half_of<T>(x.w[j / 2], j & 1);
  }
  return make_uint2(mx_encode8(v, byte), mx_encode8(v + 8, byte));
}

}  // namespace b200
