// Weights to 4 bits (int4.cuh) and back.  Bound by memory: a value is read once, and half a byte of it written.
//
//   without zeros   scale = max|y| / 7,            q = 8 + clamp(round(y / scale), -8, 7)
//   with zeros      scale = (hi - lo) / 15,        zero = clamp(round(-lo / scale), 0, 15),   q = clamp(round(y / scale) + zero, 0, 15)
//                   for lo = min(0, min y), hi = max(0, max y)
//
// over the group that y is in; the scale is rounded to the weight's type first, and halves round to even.  A group whose scale rounds to
// zero stands for zeros; one that holds an infinity or a NaN has the scale NaN.  Compiled without approximate arithmetic.
#include "int4.cuh"

namespace mvpa {
namespace {

constexpr int kThreads = 256;
constexpr int kLane = fp8::kLane;  // sixteen values a lane

// Sixteen values are a lane's; a group's lanes are neighbours.  Lanes are numbered along the rows; the row is the number by the lanes of a
// row, for numbers below 2^31 a product with a multiplier that the host forms (n / d = (umulhi(n, m) + n) >> s with s = ceil log2 d and
// m = floor(2^32 (2^s - d) / d) + 1), for more a division.
struct Lanes {
  int64_t rows;
  int per_row, width, groups, each;  // lanes of a row (whole groups); log2 of the lanes of a group
  uint32_t mul, shift;
  bool small;
  Lanes(int64_t r, int w, int group) : rows(r), width(w), groups((w + group - 1) / group), each(group == 32 ? 1 : group == 64 ? 2 : 3), shift(0) {
    per_row = groups << each;
    while (((uint64_t)1 << shift) < (uint64_t)per_row) ++shift;
    mul = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << shift) - per_row)) / per_row + 1);
    small = rows * per_row + kThreads < ((int64_t)1 << 31);
  }
  int64_t ctas() const { return (rows * per_row + kThreads - 1) / kThreads; }
};
struct Place {
  int64_t row;
  int lane, col, group;
  __device__ __forceinline__ explicit Place(const Lanes& g) {
    const int64_t u = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (g.small) {
      const uint32_t r = (__umulhi((uint32_t)u, g.mul) + (uint32_t)u) >> g.shift;
      row = r;
      lane = (int)((uint32_t)u - r * (uint32_t)g.per_row);
    } else {
      row = u / g.per_row;
      lane = (int)(u - row * g.per_row);
    }
    col = lane * kLane;
    group = lane >> g.each;
  }
};

// round(y / s) of the exact quotient, halves to even, for quotients of at most a few hundred.  With the reciprocal rounded to nearest, one
// step from y * inverse gives the quotient rounded to nearest (Markstein), which lies on the side of every half that the exact one lies
// on, or on the half.  On a half the exact one lies too where y and s have bf16's eight bits; in fp32 it may lie 2^-25 beside it, so what
// comes near a half is looked at again: y - (n + 1/2) s, of which the fused operation keeps the sign.  (Instructions are what bounds this
// kernel beside the memory: with that look at every value, and a conversion and a test of its place for each, 15360 x 2048 in bf16 took
// 38 us.)
constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: added to it a number is rounded to a whole one
template <typename T>
__device__ __forceinline__ float nearest(float y, float s, float inverse) {
  float t = y * inverse;
  t = fmaf(fmaf(-t, s, y), inverse, t);
  float n = (t + kMagic) - kMagic;
  if constexpr (sizeof(T) == 4) {
    if (fabsf(fabsf(t - n) - 0.5f) < 0x1p-18f) {
      const float low = floorf(t), d = fmaf(-(low + 0.5f), s, y);
      n = d > 0.f ? low + 1.f : d < 0.f ? low : 2.f * rintf(0.5f * low + 0.25f);  // (a half: the even one of low and low + 1)
    }
  }
  return n;
}

template <typename T, bool VEC, bool ZEROS>
__global__ void __launch_bounds__(kThreads) quantize_int4_kernel(const T* __restrict__ w, int64_t ld_w, uint8_t* __restrict__ q, int64_t ld_q,
                                                                 T* __restrict__ scales, int64_t ld_s, uint8_t* __restrict__ zeros, int64_t ld_z,
                                                                 const Lanes g) {
  ptx::griddep_launch();
  ptx::griddep_wait();
  const Place at(g);
  const int64_t row = at.row;
  const int col = at.col, group = at.group;
  const bool any = row < g.rows;
  float y[kLane];
  fp8::Raw<T> raw = {};
  if (any && col < g.width) {
    if constexpr (VEC) raw.load(w + row * ld_w, col, g.width);
    else raw.load_any(w + row * ld_w, col, g.width);
  }
  raw.get(y);
  uint32_t top = fp8::top_of(y);
  float lo = 0.f, hi = 0.f;
  if constexpr (ZEROS) {
#pragma unroll
    for (int e = 0; e < kLane; ++e) {
      lo = fminf(lo, y[e]);
      hi = fmaxf(hi, y[e]);
    }
  }
  for (int m = 1; m < 1 << g.each; m *= 2) {
    top = max(top, __shfl_xor_sync(0xffffffffu, top, m));
    if constexpr (ZEROS) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, m));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, m));
    }
  }
  if (!any) return;
  const bool finite = top < 0x7f800000u;
  // (in 64 bits where the difference may lose something or leave fp32; max|y| / 7 needs none: its digits repeat, none is next to a half)
  const T rounded = from_f32<T>(ZEROS ? (float)(((double)hi - (double)lo) / 15.0) : __fdiv_rn(__uint_as_float(top), 7.f));
  float s = to_f32<T>(rounded);
  const bool some = finite && s > 0.f;
  const float up = s < 0x1p-60f ? 0x1p64f : 1.f;  // (away from the numbers below the smallest normal one)
  s *= up;
  const float inverse = some ? __frcp_rn(s) : 0.f;
  const float zero = ZEROS && some ? fminf(fmaxf(nearest<T>(-lo * up, s, inverse), 0.f), 15.f) : 0.f;
  if ((at.lane & ((1 << g.each) - 1)) == 0) {
    scales[row * ld_s + group] = finite ? rounded : from_f32<T>(__uint_as_float(0x7fffffffu));
    if constexpr (ZEROS) zeros[row * ld_z + group] = (uint8_t)zero;
  }
  uint32_t word[2] = {};
  const float shift = ZEROS ? zero : 8.f;
  if (some) {
#pragma unroll
    for (int h = 0; h < 4; ++h) {  // four whole numbers from 0 to 15 are one of 16 bits, and stand in the low half of 2^23 + it
      float four = 0.f;
#pragma unroll
      for (int e = 3; e >= 0; --e) {
        const float n = nearest<T>(y[4 * h + e] * up, s, inverse) + shift;
        four = fmaf(four, 16.f, fminf(fmaxf(n, 0.f), 15.f));
      }
      word[h / 2] |= (__float_as_uint(four + 8388608.f) & 0xffffu) << (16 * (h & 1));
    }
  } else {
    word[0] = word[1] = ZEROS ? 0u : 0x88888888u;
  }
  const int left = g.width - col;
  if (left < kLane) {  // what follows the row
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int n = left - 8 * h;
      if (n <= 0) word[h] = 0;
      else if (n < 8) word[h] &= (1u << (4 * n)) - 1;
    }
  }
  uint8_t* to = q + row * ld_q + col / 2;
  if (left >= kLane) {
    *reinterpret_cast<uint2*>(to) = make_uint2(word[0], word[1]);
  } else {
#pragma unroll
    for (int b = 0; b < 8; ++b)
      if (col + 2 * b < g.width) to[b] = (uint8_t)(word[b / 4] >> (8 * (b % 4)));
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) dequantize_int4_kernel(const Int4Weight w, T* __restrict__ out, int64_t ld_out, bool vec, const Lanes g) {
  ptx::griddep_launch();
  ptx::griddep_wait();
  const Place at(g);
  const int64_t row = at.row;
  const int col = at.col, group = at.group;
  if (row >= g.rows || col >= g.width) return;
  const uint8_t* from = w.q + row * w.ld_q + col / 2;
  uint32_t word[2] = {};
  if (col + kLane <= g.width) {
    const uint2 v = *reinterpret_cast<const uint2*>(from);
    word[0] = v.x;
    word[1] = v.y;
  } else {
#pragma unroll
    for (int b = 0; b < 8; ++b)
      if (col + 2 * b < g.width) word[b / 4] |= (uint32_t)from[b] << (8 * (b % 4));
  }
  const float s = w.scale(row, group), zero = __uint_as_float(0x4b000000u | w.zero(row, group));  // (2^23 + zero)
  float y[kLane];
#pragma unroll
  for (int e = 0; e < kLane; ++e) y[e] = (__uint_as_float(0x4b000000u | ((word[e / 8] >> (4 * (e % 8))) & 15u)) - zero) * s;
  T* to = out + row * ld_out;
  if (vec) {
    fp8::Raw<T> raw;
    raw.pack(y);
    raw.store(to, col, g.width);
  } else {
#pragma unroll
    for (int e = 0; e < kLane; ++e)
      if (col + e < g.width) to[col + e] = from_f32<T>(y[e]);
  }
}

template <typename T>
bool vectors(const void* p, int64_t ld) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld * (int64_t)sizeof(T) % 16 == 0;
}

template <typename T>
int run_quantize(const void* w, int64_t ld_w, void* q, int64_t ld_q, void* scales, int64_t ld_s, void* zeros, int64_t ld_z, const Lanes& g,
                 cudaStream_t s) {
  const bool vec = vectors<T>(w, ld_w);
  const auto kernel = zeros != nullptr ? (vec ? quantize_int4_kernel<T, true, true> : quantize_int4_kernel<T, false, true>)
                                       : (vec ? quantize_int4_kernel<T, true, false> : quantize_int4_kernel<T, false, false>);
  MVPA_CUDA_CHECK(launch_dependent(1, kernel, (unsigned)g.ctas(), kThreads, 0, s, (const T*)w, ld_w, (uint8_t*)q, ld_q, (T*)scales, ld_s,
                                   (uint8_t*)zeros, ld_z, g));
  count_launch();
  MVPA_CUDA_CHECK(cudaGetLastError());
  return MVPA_OK;
}

template <typename T>
int run_dequantize(const Int4Weight& w, void* out, int64_t ld_out, const Lanes& g, cudaStream_t s) {
  MVPA_CUDA_CHECK(launch_dependent(1, dequantize_int4_kernel<T>, (unsigned)g.ctas(), kThreads, 0, s, w, (T*)out, ld_out, vectors<T>(out, ld_out), g));
  count_launch();
  MVPA_CUDA_CHECK(cudaGetLastError());
  return MVPA_OK;
}

int check_matrix(const char* what, const char* name, const void* p, int64_t ld, int32_t width, int32_t dtype) {
  if (p == nullptr || ld < width || (reinterpret_cast<uintptr_t>(p) & (dtype == MVPA_F32 ? 3 : 1)) != 0) {
    set_error("%s: %s is NULL, not aligned to its elements, or its leading dimension is shorter than a row", what, name);
    return MVPA_ERR_ALIGNMENT;
  }
  return MVPA_OK;
}

}  // namespace

// What the 4-bit entry points ask of a weight (mvpa_int4_matmul.cu uses it too).
int check_int4(const char* what, int64_t N, int32_t K, int32_t group, int32_t scale_dtype, const mvpa_int4* w) {
  if (N < 0 || K < 0 || (group != 32 && group != 64 && group != 128) || N > 0x7fffffff - 1024 || K > 0x7fffffff - 1024) {
    set_error("%s: rows and columns must not be negative (or exceed 2^31 - 1025), groups are of 32, 64 or 128 (got %lld, %d, %d)", what,
              (long long)N, K, group);
    return MVPA_ERR_SHAPE;
  }
  if (scale_dtype != MVPA_F32 && scale_dtype != MVPA_BF16) {
    set_error("%s: types are MVPA_F32 or MVPA_BF16", what);
    return MVPA_ERR_DTYPE;
  }
  if (N == 0 || K == 0) return MVPA_OK;
  if (w == nullptr) {
    set_error("%s: a weight is NULL", what);
    return MVPA_ERR_ALIGNMENT;
  }
  const int groups = (K + group - 1) / group;
  if (w->q == nullptr || (reinterpret_cast<uintptr_t>(w->q) & 15) != 0 || w->ld_q % 16 != 0 || w->ld_q < (K + 1) / 2 || w->scales == nullptr ||
      (reinterpret_cast<uintptr_t>(w->scales) & (scale_dtype == MVPA_F32 ? 3 : 1)) != 0 || w->ld_s < groups ||
      (w->zeros != nullptr && w->ld_z < groups)) {
    set_error("%s: q must be 16-byte aligned with rows of a multiple of 16 bytes, at least half the columns; scales not NULL and aligned to "
              "their elements; the rows of scales and zeros at least as long as a row has groups", what);
    return MVPA_ERR_ALIGNMENT;
  }
  return MVPA_OK;
}

}  // namespace mvpa

using namespace mvpa;

extern "C" int mvpa_quantize_int4(const void* w, int64_t ld_w, const mvpa_int4* to, int64_t N, int32_t K, int32_t group, int32_t dtype,
                                  void* cuda_stream) {
  int rc = check_int4("mvpa_quantize_int4", N, K, group, dtype, to);
  if (rc != MVPA_OK || N == 0 || K == 0) return rc;
  rc = check_matrix("mvpa_quantize_int4", "w", w, ld_w, K, dtype);
  if (rc != MVPA_OK) return rc;
  const Lanes g(N, K, group);
  if (g.ctas() > 0x7fffffff) {
    set_error("mvpa_quantize_int4: more than 2^31 blocks of 4096 values");
    return MVPA_ERR_UNSUPPORTED;
  }
  void *q = const_cast<void*>(to->q), *scales = const_cast<void*>(to->scales), *zeros = const_cast<void*>(to->zeros);
  cudaStream_t s = (cudaStream_t)cuda_stream;
  return dtype == MVPA_F32 ? run_quantize<float>(w, ld_w, q, to->ld_q, scales, to->ld_s, zeros, to->ld_z, g, s)
                           : run_quantize<__nv_bfloat16>(w, ld_w, q, to->ld_q, scales, to->ld_s, zeros, to->ld_z, g, s);
}

extern "C" int mvpa_dequantize_int4(const mvpa_int4* w, int32_t scale_dtype, void* out, int64_t ld_out, int64_t N, int32_t K, int32_t group,
                                    int32_t out_dtype, void* cuda_stream) {
  int rc = check_int4("mvpa_dequantize_int4", N, K, group, scale_dtype, w);
  if (rc == MVPA_OK && out_dtype != MVPA_F32 && out_dtype != MVPA_BF16) {
    set_error("mvpa_dequantize_int4: out is MVPA_F32 or MVPA_BF16");
    return MVPA_ERR_DTYPE;
  }
  if (rc != MVPA_OK || N == 0 || K == 0) return rc;
  rc = check_matrix("mvpa_dequantize_int4", "out", out, ld_out, K, out_dtype);
  if (rc != MVPA_OK) return rc;
  const Lanes g(N, K, group);
  if (g.ctas() > 0x7fffffff) {
    set_error("mvpa_dequantize_int4: more than 2^31 blocks of 4096 values");
    return MVPA_ERR_UNSUPPORTED;
  }
  const Int4Weight v = {(const uint8_t*)w->q, w->scales, (const uint8_t*)w->zeros, w->ld_q, w->ld_s, w->ld_z, scale_dtype == MVPA_F32};
  cudaStream_t s = (cudaStream_t)cuda_stream;
  return out_dtype == MVPA_F32 ? run_dequantize<float>(v, out, ld_out, g, s) : run_dequantize<__nv_bfloat16>(v, out, ld_out, g, s);
}
