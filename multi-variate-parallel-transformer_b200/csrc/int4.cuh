// What the 4-bit kernels share.  A weight (N, K) in 4 bits: q, two values a byte, the first in its low half, rows of bytes on 16-byte
// boundaries; a scale for each group of 32, 64 or 128 neighbours in a row (the last group as long as the row leaves it), fp32 or
// bf16; and, or not, a zero for each group, a byte from 0 to 15.  It stands for (q - zero) * scale, zero = 8 where there are none.
#pragma once
#include "fp8.cuh"

namespace mvpa {
namespace {

struct Int4Weight {
  const uint8_t* q;
  const void* scales;
  const uint8_t* zeros;  // or NULL
  int64_t ld_q, ld_s, ld_z;
  int scale_f32;
  __device__ __forceinline__ float scale(int64_t row, int group) const {
    return scale_f32 ? static_cast<const float*>(scales)[row * ld_s + group]
                     : __bfloat162float(static_cast<const __nv_bfloat16*>(scales)[row * ld_s + group]);
  }
  __device__ __forceinline__ uint32_t zero(int64_t row, int group) const { return zeros != nullptr ? zeros[row * ld_z + group] : 8u; }
};

// Eight values of a word as pairs of bf16, (0, 4), (1, 5), (2, 6), (3, 7), each 2^-11 of q - zero: a nibble in the low bits of the mantissa
// of 128 / 2^11 is (128 + q) / 2^11, from which (128 + zero) / 2^11 (`minus`, twice) is taken.  Whole numbers from -15 to 15 beside a power
// of two: exact.  The power keeps a group's sum, 128 terms of up to 15 |x|, below the largest |x|: only what the scales make of the sums
// can leave fp32, and that where the result does (kInt4Unit takes the power back last).
constexpr float kInt4Unit = 2048.f;
__device__ __forceinline__ uint32_t int4_minus(uint32_t zero) { return 0x3d803d80u | zero | zero << 16; }
__device__ __forceinline__ void int4_pairs(uint32_t w, uint32_t minus, uint32_t (&p)[4]) {
  const __nv_bfloat162 m = *reinterpret_cast<const __nv_bfloat162*>(&minus);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t v;  // (w >> 4 i) & 0x000f000f | 0x3d803d80 in one operation: both constants in registers, or the compiler makes it two
    asm("{\n\t.reg .b32 mask, one;\n\tmov.b32 mask, 0x000f000f;\n\tmov.b32 one, 0x3d803d80;\n\tlop3.b32 %0, %1, mask, one, 0xea;\n\t}" : "=r"(v) : "r"(w >> (4 * i)));
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), m);
    p[i] = *reinterpret_cast<const uint32_t*>(&d);
  }
}

// An fp32 number as three bf16 whose sum it is, exactly (but for what lies below 2^-133): eight bits of the mantissa each, cut off.  An
// infinity or a NaN is the first of them alone.
struct Thirds {
  uint32_t hi, mid, lo;  // bf16 in the upper half of a word
  __device__ __forceinline__ explicit Thirds(float x) {
    const uint32_t b = __float_as_uint(x);
    const bool finite = (b & 0x7fffffffu) < 0x7f800000u;
    hi = (b & 0xffff0000u) | ((b & 0x7fffffffu) > 0x7f800000u ? 0x00400000u : 0u);
    const float r = finite ? x - __uint_as_float(hi) : 0.f;
    mid = __float_as_uint(r) & 0xffff0000u;
    lo = __float_as_uint(r - __uint_as_float(mid)) & 0xffff0000u;
  }
};

}  // namespace
}  // namespace mvpa
