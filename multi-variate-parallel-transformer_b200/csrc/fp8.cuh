// What the 8-bit kernels share: blocks of 128 values in e4m3 with one scale.
//
//   scale = the smallest 2^e, e >= -126, with max|y| <= 448 * 2^e,   q = e4m3(y / scale)
//
// A power of two: y / scale is exact, so the only rounding is the step to e4m3 (to nearest, ties to even), and a value that is
// representable comes back as it was; against a scale of max|y| / 448 a block gives away less than one binade at the bottom
// of e4m3's range, where a value is 2^-15 of the block's largest.  The scale is held as its exponent's byte (e8m0, bias 127).
// A block that holds an infinity or a NaN has the scale NaN (255) and every q NaN: it does not pass unnoticed.
#pragma once
#include "block_rows.cuh"

namespace mvpa {
namespace fp8 {

constexpr int kBlock = 128;

// The byte of the scale from the largest magnitude's bits (the bits of non-negative floats order like the floats do, with
// infinity and then NaN above).  448 = 1.75 * 2^8: above 1.75 in the mantissa (0x600000) the next power is needed.
__device__ __forceinline__ uint32_t scale_byte(uint32_t top_bits) {
  if (top_bits >= 0x7f800000u) return 255u;
  const int b = (int)((top_bits + 0x1fffffu) >> 23) - 8;
  return (uint32_t)(b < 1 ? 1 : b);
}
// 1 / scale, exact; NaN for the byte 255.
__device__ __forceinline__ float inverse_scale(uint32_t byte) {
  return byte == 255u ? __uint_as_float(0x7fffffffu) : __uint_as_float((254u - byte) << 23);
}
// The scale itself (bytes from elsewhere may be 0: 2^-127).
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return byte == 255u ? __uint_as_float(0x7fffffffu) : byte == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
}

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x4(float2 a, float2 b) { return __byte_perm(e4m3x2(a.x, a.y), e4m3x2(b.x, b.y), 0x5410); }

// The largest of the values of eight neighbouring lanes: a block of 128 is eight lanes with sixteen values each.
__device__ __forceinline__ uint32_t max8(uint32_t v) {
  v = max(v, __shfl_xor_sync(0xffffffffu, v, 1));
  v = max(v, __shfl_xor_sync(0xffffffffu, v, 2));
  return max(v, __shfl_xor_sync(0xffffffffu, v, 4));
}

constexpr int kLane = 16;  // values a lane holds of a block: 16 bytes of e4m3, one store

// A lane's sixteen values of its block, as they lie in memory.
template <typename T>
struct Raw {
  static constexpr int kWords = kLane / Vec<T>::N;
  uint4 w[kWords];
  __device__ __forceinline__ void load(const T* __restrict__ row, int col, int width) {
    if (col + kLane <= width) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[i] = *reinterpret_cast<const uint4*>(row + col + i * Vec<T>::N);
    } else {
      float y[kLane];
#pragma unroll
      for (int e = 0; e < kLane; ++e) y[e] = col + e < width ? to_f32<T>(row[col + e]) : 0.f;
      pack(y);
    }
  }
  // Rows at any alignment: the 16-byte pieces that hold the values (and none that holds no value of the row, so that nothing is
  // read from beyond a piece of memory that the row lies in), moved into place by words and then by halves.  Sixteen single loads
  // a lane touch each sector again and again: 2500 x 1027 in fp32 with the residual took 34 us so.
  __device__ __forceinline__ void load_any(const T* __restrict__ row, int col, int width) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(row + col), end = p + min(width - col, kLane) * sizeof(T);
    const uint4* from = reinterpret_cast<const uint4*>(p & ~(uintptr_t)15);
    constexpr int W = 4 * kWords;
    uint32_t v[W + 4];
#pragma unroll
    for (int i = 0; i <= kWords; ++i) {
      uint4 r = make_uint4(0, 0, 0, 0);
      if (reinterpret_cast<uintptr_t>(from + i) < end) r = from[i];
      v[4 * i] = r.x; v[4 * i + 1] = r.y; v[4 * i + 2] = r.z; v[4 * i + 3] = r.w;
    }
    const uint32_t shift = (uint32_t)p & 15;
    if (shift & 8) {
#pragma unroll
      for (int j = 0; j < W + 2; ++j) v[j] = v[j + 2];
    }
    if (shift & 4) {
#pragma unroll
      for (int j = 0; j < W + 1; ++j) v[j] = v[j + 1];
    }
    if constexpr (sizeof(T) == 2) {
      if (shift & 2) {
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] = __funnelshift_r(v[j], v[j + 1], 16);
      }
    }
    if (col + kLane > width) {  // what follows the row
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const int left = width - col - j * (4 / (int)sizeof(T));  // values of the row from this word on
        if (left <= 0) v[j] = 0;
        else if (sizeof(T) == 2 && left == 1) v[j] &= 0xffffu;
      }
    }
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  }
  __device__ __forceinline__ void pack(const float (&y)[kLane]) {  // (values of T)
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      float f[Vec<T>::N];
#pragma unroll
      for (int e = 0; e < Vec<T>::N; ++e) f[e] = y[i * Vec<T>::N + e];
      w[i] = Vec<T>::pack(f);
    }
  }
  __device__ __forceinline__ void get(float (&y)[kLane]) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      float f[Vec<T>::N];
      Vec<T>::unpack(w[i], f);
#pragma unroll
      for (int e = 0; e < Vec<T>::N; ++e) y[i * Vec<T>::N + e] = f[e];
    }
  }
  __device__ __forceinline__ void store(T* __restrict__ row, int col, int width) const {
    if (col + kLane <= width) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) *reinterpret_cast<uint4*>(row + col + i * Vec<T>::N) = w[i];
    } else {
      float y[kLane];
      get(y);
#pragma unroll
      for (int e = 0; e < kLane; ++e)
        if (col + e < width) row[col + e] = from_f32<T>(y[e]);
    }
  }
};

// The same to rows at any alignment, by way of shared memory: the eight lanes of a block write it eight neighbours at a time.  A
// warp's four blocks lie kTurn floats apart and the values of a lane 17: no two lanes of a warp meet in a bank.
constexpr int kTurn = kBlock + kBlock / kLane;
template <typename T>  // (every lane of the warp takes part; `any`: this lane's block exists)
__device__ __forceinline__ void store_any(float* warp_s, int lane, T* __restrict__ row, int block_col, int width, bool any,
                                          const float (&y)[kLane]) {
  float* s = warp_s + (lane >> 3) * kTurn;
  const int l = lane & 7;
#pragma unroll
  for (int e = 0; e < kLane; ++e) s[l * (kLane + 1) + e] = y[e];
  __syncwarp();
#pragma unroll
  for (int j = 0; j < kLane; ++j) {
    const int c = block_col + j * 8 + l;
    if (any && c < width) row[c] = from_f32<T>(s[j * 8 + l + (j >> 1)]);
  }
  __syncwarp();
}

// Sixteen values in e4m3 to a row whose start is on a 16-byte boundary; nothing past `width` is written.
__device__ __forceinline__ void store16(uint8_t* __restrict__ row, int col, int width, const float (&y)[kLane], float inverse) {
  const float2 by = make_float2(inverse, inverse);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = e4m3x4(ptx::fmul2(make_float2(y[4 * i], y[4 * i + 1]), by), ptx::fmul2(make_float2(y[4 * i + 2], y[4 * i + 3]), by));
  if (col + kLane <= width) {
    *reinterpret_cast<uint4*>(row + col) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int e = 0; e < kLane; ++e)
      if (col + e < width) row[col + e] = (uint8_t)(w[e / 4] >> (8 * (e % 4)));
  }
}

// The largest magnitude's bits; a NaN stays one.
__device__ __forceinline__ uint32_t top_of(const float (&y)[kLane]) {
  float top = fabsf(y[0]);
#pragma unroll
  for (int e = 1; e + 1 < kLane; e += 2)
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(top) : "f"(top), "f"(fabsf(y[e])), "f"(fabsf(y[e + 1])));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(top) : "f"(top), "f"(fabsf(y[kLane - 1])));
  return __float_as_uint(top);
}

}  // namespace fp8
}  // namespace mvpa
