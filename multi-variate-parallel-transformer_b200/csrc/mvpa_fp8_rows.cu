// Rows and weights in 8 bits (fp8.cuh): quantisation, the RMSNorm with the residual's addition, the SwiGLU gate.  Bound by
// memory: every input is read once, and what the unquantised kernels write in 16 bits and a further pass would read again
// leaves as e4m3.  Compiled without approximate arithmetic, so that a value next to a rounding border, and numbers below the
// smallest normal one, come out as the formula says.
#include "fp8.cuh"

namespace mvpa {
namespace {

using namespace fp8;

constexpr int kThreads = 256;

// Row blocks are numbered along the rows; eight lanes take one.  The row is the number by the blocks of a row: for numbers below
// 2^31 a product with a multiplier that the host forms (n / d = (umulhi(n, m) + n) >> s with s = ceil log2 d and
// m = floor(2^32 (2^s - d) / d) + 1), for more a division.
struct Units {
  int64_t rows;
  int width, blocks;
  uint32_t mul, shift;
  bool small;
  Units(int64_t r, int w) : rows(r), width(w), blocks((w + kBlock - 1) / kBlock), shift(0) {
    while ((1u << shift) < (uint32_t)blocks) ++shift;
    mul = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << shift) - blocks)) / blocks + 1);
    small = (r * blocks + kThreads / 8) < ((int64_t)1 << 31);
  }
  unsigned grid() const { return (unsigned)((rows * blocks + kThreads / 8 - 1) / (kThreads / 8)); }
};
struct Unit {
  int64_t row;
  int col;  // of this lane
  int block;
  bool any;
};
__device__ __forceinline__ Unit unit_of(const Units& g) {
  const int64_t u = (int64_t)blockIdx.x * (kThreads / 8) + threadIdx.x / 8;
  Unit t;
  if (g.small) {
    const uint32_t row = (__umulhi((uint32_t)u, g.mul) + (uint32_t)u) >> g.shift;
    t.row = row;
    t.block = (int)((uint32_t)u - row * (uint32_t)g.blocks);
  } else {
    t.row = u / g.blocks;
    t.block = (int)(u - t.row * g.blocks);
  }
  t.col = t.block * kBlock + (threadIdx.x & 7) * kLane;
  t.any = t.row < g.rows;
  return t;
}

// (-> the scale's byte)
__device__ __forceinline__ uint32_t write_unit(const Unit& t, const float (&y)[kLane], uint8_t* q, int64_t ld_q, uint8_t* scales,
                                               int64_t ld_s, int width) {
  const uint32_t byte = scale_byte(max8(top_of(y)));
  if (!t.any) return byte;
  if (t.col < width) store16(q + t.row * ld_q, t.col, width, y, inverse_scale(byte));
  if ((threadIdx.x & 7) == 0) scales[t.row * ld_s + t.block] = (uint8_t)byte;
  return byte;
}

// A lane's values of one block.
template <typename T, bool VEC>
__device__ __forceinline__ void read_unit(const T* __restrict__ x, int64_t ld, const Unit& t, int width, float (&y)[kLane]) {
  Raw<T> raw = {};
  if (t.any && t.col < width) {
    if constexpr (VEC) raw.load(x + t.row * ld, t.col, width);
    else raw.load_any(x + t.row * ld, t.col, width);
  }
  raw.get(y);
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const T* __restrict__ x, int64_t ld_x, uint8_t* __restrict__ q,
                                                                 int64_t ld_q, uint8_t* __restrict__ scales, int64_t ld_s,
                                                                 const Units g) {
  ptx::griddep_launch();
  ptx::griddep_wait();
  const Unit t = unit_of(g);
  float y[kLane];
  read_unit<T, VEC>(x, ld_x, t, g.width, y);
  write_unit(t, y, q, ld_q, scales, ld_s, g.width);
}

// silu(g) u = g / (1 + e^-g) u of two numbers.  e^-g = 2^(-g log2 e): the product in two parts, since 2^x turns an error of x into a
// relative one (log2 e = kHi + kLo), and 2^(hi + lo) = 2^hi (1 + lo ln 2) as |lo| < 2^-16; the reciprocal is an estimate and one
// step of Newton's.  As exact as the quotient by library functions, and the kernel takes 20 instructions a value for 40, since
// most are on pairs: their number is what bounds it beside the memory (32768 x 5632: 155 to 167 us, 86 to 92 % of the copy rate).  It is 8 e^-g that is computed, so that for g < -86.6 it overflows before the reciprocal could
// leave the normal numbers: infinity has no reciprocal by Newton, and the result is NaN (as it is where g log2 e overflows).
// Blocks that come out NaN are looked at again by silu_mul_any.
__device__ __forceinline__ float2 silu_mul(float2 g, float2 u) {
  constexpr float kHi = 1.44269504f, kLo = 1.92596299e-8f, kLn2 = 0.693147181f;
  const auto both = [](float x) { return make_float2(x, x); };
  const float2 hi = ptx::fmul2(g, both(-kHi)), low = ptx::ffma2(g, both(-kHi), make_float2(-hi.x, -hi.y));
  const float2 lo = ptx::ffma2(g, both(-kLo), low);
  const float2 p = ptx::fmul2(make_float2(ptx::ex2(hi.x), ptx::ex2(hi.y)), both(8.f));
  const float2 d = ptx::ffma2(ptx::ffma2(p, ptx::fmul2(lo, both(kLn2)), p), both(0.125f), both(1.f));
  float2 r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(d.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(d.y));
  r = ptx::ffma2(r, ptx::ffma2(make_float2(-d.x, -d.y), r, both(1.f)), r);
  return ptx::fmul2(ptx::fmul2(g, r), u);
}
// The same for any g.  Below -86, 1 / (1 + e^-g) is e^g to more places than fp32 has, as small as it may be beside a large u: in
// four parts, which leave the normal numbers where the product does and not before.  Above 86 it is 1.
__device__ __forceinline__ float silu_mul_any(float g, float u) {
  if (g > 86.f) return g * u;
  if (!(g < -86.f)) return silu_mul(make_float2(g, g), make_float2(u, u)).x;
  const float part = expf(0.25f * g);
  return u * part * part * (g * part) * part;
}

// A warp's units once more, written where `again`: value by value and apart from the kernel, whose registers (32 a thread for aligned
// bf16, which is what lets its warps fill a multiprocessor) it does not add to.
template <typename T>
__device__ __noinline__ void silu_mul_again(bool again, const T* gate, const T* up, int64_t ld_in, uint8_t* q, int64_t ld_q, uint8_t* scales,
                                            int64_t ld_s, const Units g) {
  const Unit t = unit_of(g);
  const int n = again && t.any ? min(g.width - t.col, kLane) : 0;
  gate += t.row * ld_in + t.col;
  up += t.row * ld_in + t.col;
  q += t.row * ld_q + t.col;
  uint32_t top = 0;
#pragma unroll 1
  for (int e = 0; e < n; ++e) top = max(top, __float_as_uint(fabsf(silu_mul_any(to_f32<T>(gate[e]), to_f32<T>(up[e])))));
  const uint32_t byte = scale_byte(max8(top));
  const float inverse = inverse_scale(byte);
#pragma unroll 1
  for (int e = 0; e < n; ++e) q[e] = (uint8_t)e4m3x2(silu_mul_any(to_f32<T>(gate[e]), to_f32<T>(up[e])) * inverse, 0.f);
  if (n > 0 && (threadIdx.x & 7) == 0) scales[t.row * ld_s + t.block] = (uint8_t)byte;
}

// silu(gate) * up, in fp32 from the inputs to the step to e4m3.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) silu_mul_fp8_kernel(const T* __restrict__ gate, const T* __restrict__ up, int64_t ld_in,
                                                                uint8_t* __restrict__ q, int64_t ld_q, uint8_t* __restrict__ scales,
                                                                int64_t ld_s, const Units g) {
  ptx::griddep_launch();
  ptx::griddep_wait();
  const Unit t = unit_of(g);
  float y[kLane], u[kLane];
  read_unit<T, VEC>(gate, ld_in, t, g.width, y);
  read_unit<T, VEC>(up, ld_in, t, g.width, u);
#pragma unroll
  for (int e = 0; e < kLane; e += 2) {
    const float2 v = silu_mul(make_float2(y[e], y[e + 1]), make_float2(u[e], u[e + 1]));
    y[e] = v.x;
    y[e + 1] = v.y;
  }
  const bool again = write_unit(t, y, q, ld_q, scales, ld_s, g.width) == 255u;
  if (__any_sync(0xffffffffu, again)) silu_mul_again<T>(again, gate, up, ld_in, q, ld_q, scales, ld_s, g);
}

// One CTA per block of 128 x 128: eight lanes a row, 32 rows at a time, four times; the values wait in registers for the
// block's largest.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_blocks_kernel(const T* __restrict__ x, int64_t ld_x, uint8_t* __restrict__ q,
                                                                   int64_t ld_q, uint8_t* __restrict__ scales, int64_t ld_s,
                                                                   int64_t rows, int width) {
  constexpr int kTimes = kBlock / (kThreads / 8);
  __shared__ uint32_t s_top[kThreads / 32];
  ptx::griddep_launch();
  ptx::griddep_wait();
  const int64_t row0 = (int64_t)blockIdx.y * kBlock + threadIdx.x / 8;
  Unit t[kTimes];
  float y[kTimes][kLane];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kTimes; ++i) {
    t[i].row = row0 + i * (kThreads / 8);
    t[i].block = blockIdx.x;
    t[i].col = blockIdx.x * kBlock + (threadIdx.x & 7) * kLane;
    t[i].any = t[i].row < rows;
    read_unit<T, VEC>(x, ld_x, t[i], width, y[i]);
  }
#pragma unroll
  for (int i = 0; i < kTimes; ++i) top = max(top, top_of(y[i]));
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) s_top[threadIdx.x / 32] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) top = max(top, s_top[i]);
  const uint32_t byte = scale_byte(top);
#pragma unroll
  for (int i = 0; i < kTimes; ++i)
    if (t[i].any && t[i].col < width) store16(q + t[i].row * ld_q, t[i].col, width, y[i], inverse_scale(byte));
  if (threadIdx.x == 0) scales[(int64_t)blockIdx.y * ld_s + blockIdx.x] = (uint8_t)byte;
}

// y = rmsnorm(h) * w with h = x (+ a, in T as in rmsnorm_kernel); h written out, y to e4m3 without a rounding in between.  A warp
// has a row, NV times sixteen values a lane, which stay in registers in T between the sum of squares and the scaling.  AHEAD, for
// aligned rows of up to 1024 values in fp32: resident warps that load their next row while they work on this one, the weight in
// registers (20000 x 1000 with the residual: 46.5 us for 58.6 with a row a warp).  In bf16, twice the arithmetic a byte, that takes
// registers from too many warps (65536 x 768: 86 us for 65): there and for longer rows each warp has one row.
constexpr int kNormWarps = 4;

// 1 / sqrt(x): the library's, within two units, and a step of Newton's where that is finite and not zero.
__device__ __forceinline__ float inverse_root(float x) {
  const float r = rsqrtf(x), e = fmaf(-x * r, r, 1.f);
  return fabsf(e) < 0.5f ? fmaf(0.5f * r, e, r) : r;
}

template <typename T, int NV, bool VEC>
constexpr bool kNormAhead = VEC && sizeof(T) == 4 && NV <= 2;
template <typename T, int NV, bool VEC>
constexpr int kNormCtas = kNormAhead<T, NV, VEC> ? (NV == 1 ? 5 : 3) : NV * sizeof(T) <= 2 ? 10 : NV * sizeof(T) <= 4 ? 8 : NV * sizeof(T) <= 8 ? 5 : 2;

template <typename T, int NV, bool VEC>
__global__ void __launch_bounds__(kNormWarps * 32, kNormCtas<T, NV, VEC>) rmsnorm_fp8_kernel(const T* __restrict__ x, const T* __restrict__ a,
                                                                                        const T* __restrict__ w, T* __restrict__ h_out,
                                                                                        uint8_t* __restrict__ q, int64_t ld_q,
                                                                                        uint8_t* __restrict__ scales, int64_t ld_s,
                                                                                        int64_t rows, int E, float eps) {
  constexpr bool AHEAD = kNormAhead<T, NV, VEC>;
  __shared__ float s_turn[VEC ? 1 : kNormWarps][VEC ? 1 : 4 * kTurn];
  ptx::griddep_launch();
  ptx::griddep_wait();
  const int lane = threadIdx.x & 31;
  const int64_t step = (int64_t)gridDim.x * kNormWarps;
  const auto col_of = [&](int i) { return (i * 32 + lane) * kLane; };
  const auto load = [&](Raw<T>(&r)[NV], const T* p) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (col_of(i) < E) {
        if constexpr (VEC) r[i].load(p, col_of(i), E);
        else r[i].load_any(p, col_of(i), E);
      }
  };
  int64_t row = (int64_t)blockIdx.x * kNormWarps + (threadIdx.x >> 5);
  Raw<T> raw[NV] = {}, more[NV] = {}, gain[AHEAD ? NV : 1] = {};
  if (row < rows) {
    load(raw, x + row * E);
    if (a != nullptr) load(more, a + row * E);
    if constexpr (AHEAD) load(gain, w);
  }
  for (; row < rows; row += step) {
    const int64_t at = row * E;
    if (a != nullptr) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float v[kLane], b[kLane];
        raw[i].get(v);
        more[i].get(b);
#pragma unroll
        for (int e = 0; e < kLane; ++e) v[e] += b[e];
        raw[i].pack(v);  // (rounds to T)
      }
    }
    float squares = 0.f;  // (short chains: what the sum loses moves every value of the row towards its next step)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float v[kLane], s[4];
      raw[i].get(v);
#pragma unroll
      for (int e = 0; e < kLane; ++e) s[e & 3] = e < 4 ? v[e] * v[e] : fmaf(v[e], v[e], s[e & 3]);
      squares += (s[0] + s[1]) + (s[2] + s[3]);
    }
    Raw<T> mine[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) mine[i] = raw[i];
    if (AHEAD && row + step < rows) {
      load(raw, x + at + step * E);
      if (a != nullptr) load(more, a + at + step * E);
    }
    if (h_out != nullptr) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if constexpr (VEC) {
          if (col_of(i) < E) mine[i].store(h_out + at, col_of(i), E);
        } else {
          if (i * 32 * kLane >= E) break;  // (the same for the whole warp)
          float v[kLane];
          mine[i].get(v);
          store_any(s_turn[threadIdx.x >> 5], lane, h_out + at, (i * 4 + (lane >> 3)) * kBlock, E, col_of(i) / kBlock * kBlock < E, v);
        }
      }
    }
    const float rstd = inverse_root(warp_sum(squares) / (float)E + eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (i * 32 * kLane >= E) break;
      const int col = col_of(i);
      float y[kLane], g[kLane];
      if constexpr (AHEAD) {
        gain[i].get(g);
      } else {
        Raw<T> one = {};
        if (col < E) {
          if constexpr (VEC) one.load(w, col, E);
          else one.load_any(w, col, E);
        }
        one.get(g);
      }
      mine[i].get(y);
      // One rounding on the way to e4m3: the product with the weight is exact in fp32 for bf16; for fp32 its remainder goes along.
#pragma unroll
      for (int e = 0; e < kLane; ++e) {
        const float p = y[e] * g[e];
        if constexpr (sizeof(T) == 2) y[e] = p * rstd;
        else y[e] = fmaf(p, rstd, fmaf(y[e], g[e], -p) * rstd);
      }
      if (col + kLane > E) {  // (past the end 0 * rstd is NaN where rstd is)
#pragma unroll
        for (int e = 0; e < kLane; ++e)
          if (col + e >= E) y[e] = 0.f;
      }
      const uint32_t byte = scale_byte(max8(top_of(y)));
      if (col < E) {
        store16(q + row * ld_q, col, E, y, inverse_scale(byte));
        if ((lane & 7) == 0) scales[row * ld_s + col / kBlock] = (uint8_t)byte;
      }
    }
    if constexpr (!AHEAD) break;
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
template <typename T>
bool vectors(const void* p, int64_t ld) { return aligned16(p) && ld * (int64_t)sizeof(T) % 16 == 0; }

int check(const char* what, int64_t rows, int32_t width, int32_t dtype, const void* q, int64_t ld_q, const void* scales,
          int64_t ld_s) {
  constexpr int kMost = 0x7fffffff - 1024;  // (rows and columns past the last block are still 32-bit numbers)
  if (rows < 0 || width < 0 || width > kMost) {
    set_error("%s: sizes must not be negative and a row at most %d wide (%lld rows of %d)", what, kMost, (long long)rows, width);
    return MVPA_ERR_SHAPE;
  }
  if (dtype != MVPA_F32 && dtype != MVPA_BF16) {
    set_error("%s: element type must be MVPA_F32 or MVPA_BF16", what);
    return MVPA_ERR_DTYPE;
  }
  if (rows == 0 || width == 0) return MVPA_OK;
  if (q == nullptr || scales == nullptr || !aligned16(q) || ld_q % 16 != 0 || ld_q < width) {
    set_error("%s: q must be 16-byte aligned with rows of a multiple of 16 bytes, at least the width; scales not NULL", what);
    return MVPA_ERR_ALIGNMENT;
  }
  if (ld_s < (width + kBlock - 1) / kBlock) {
    set_error("%s: the scales' leading dimension is shorter than a row's blocks", what);
    return MVPA_ERR_SHAPE;
  }
  if (rows > kMost || rows > (int64_t)0x7fffffff * 8 / ((width + kBlock - 1) / kBlock)) {
    set_error("%s: too many rows (%lld)", what, (long long)rows);
    return MVPA_ERR_SHAPE;
  }
  return MVPA_OK;
}
int check_input(const char* what, const void* p, int64_t ld, int32_t width, int32_t dtype) {
  if (p == nullptr || ld < width || (reinterpret_cast<uintptr_t>(p) & (dtype == MVPA_F32 ? 3 : 1)) != 0) {
    set_error("%s: an input is NULL, not aligned to its elements, or its leading dimension is shorter than a row", what);
    return MVPA_ERR_ALIGNMENT;
  }
  return MVPA_OK;
}

template <typename T>
int run_quantize(const void* x, int64_t ld_x, void* q, int64_t ld_q, void* scales, int64_t ld_s, int64_t rows, int width, int tall,
                 cudaStream_t s) {
  const bool vec = vectors<T>(x, ld_x);
  if (tall == 1) {
    const Units g(rows, width);
    MVPA_CUDA_CHECK(launch_dependent(1, vec ? quantize_rows_kernel<T, true> : quantize_rows_kernel<T, false>, g.grid(), kThreads, 0, s,
                                     (const T*)x, ld_x, (uint8_t*)q, ld_q, (uint8_t*)scales, ld_s, g));
  } else {
    const dim3 grid((width + kBlock - 1) / kBlock, (unsigned)((rows + kBlock - 1) / kBlock));
    MVPA_CUDA_CHECK(launch_dependent(1, vec ? quantize_blocks_kernel<T, true> : quantize_blocks_kernel<T, false>, grid, kThreads, 0, s,
                                     (const T*)x, ld_x, (uint8_t*)q, ld_q, (uint8_t*)scales, ld_s, rows, width));
  }
  count_launch();
  MVPA_CUDA_CHECK(cudaGetLastError());
  return MVPA_OK;
}

template <typename T>
int run_silu_mul(const void* gate, const void* up, int64_t ld_in, void* q, int64_t ld_q, void* scales, int64_t ld_s, int64_t rows,
                 int width, cudaStream_t s) {
  const bool vec = vectors<T>(gate, ld_in) && aligned16(up);
  const Units g(rows, width);
  MVPA_CUDA_CHECK(launch_dependent(1, vec ? silu_mul_fp8_kernel<T, true> : silu_mul_fp8_kernel<T, false>, g.grid(), kThreads, 0, s,
                                   (const T*)gate, (const T*)up, ld_in, (uint8_t*)q, ld_q, (uint8_t*)scales, ld_s, g));
  count_launch();
  MVPA_CUDA_CHECK(cudaGetLastError());
  return MVPA_OK;
}

template <typename T, int NV>
int run_rmsnorm(const void* x, const void* add, const void* w, void* h_out, void* q, int64_t ld_q, void* scales, int64_t ld_s,
                int64_t rows, int E, float eps, cudaStream_t s) {
  const bool vec = vectors<T>(x, E) && aligned16(w) && (add == nullptr || aligned16(add)) && (h_out == nullptr || aligned16(h_out));
  const int64_t want = (rows + kNormWarps - 1) / kNormWarps;
  const int64_t most = kNormAhead<T, NV, true> && vec ? (int64_t)device_sm_count() * kNormCtas<T, NV, true> : want;
  MVPA_CUDA_CHECK(launch_dependent(1, vec ? rmsnorm_fp8_kernel<T, NV, true> : rmsnorm_fp8_kernel<T, NV, false>,
                                   (unsigned)(want < most ? want : most), kNormWarps * 32, 0, s, (const T*)x, (const T*)add, (const T*)w, (T*)h_out, (uint8_t*)q, ld_q,
                                   (uint8_t*)scales, ld_s, rows, E, eps));
  count_launch();
  MVPA_CUDA_CHECK(cudaGetLastError());
  return MVPA_OK;
}

template <typename T>
int run_rmsnorm_any(const void* x, const void* add, const void* w, void* h_out, void* q, int64_t ld_q, void* scales, int64_t ld_s,
                    int64_t rows, int E, float eps, cudaStream_t s) {
  const int nv = (E + 32 * kLane - 1) / (32 * kLane);
  if (nv <= 1) return run_rmsnorm<T, 1>(x, add, w, h_out, q, ld_q, scales, ld_s, rows, E, eps, s);
  if (nv <= 2) return run_rmsnorm<T, 2>(x, add, w, h_out, q, ld_q, scales, ld_s, rows, E, eps, s);
  if (nv <= 3) return run_rmsnorm<T, 3>(x, add, w, h_out, q, ld_q, scales, ld_s, rows, E, eps, s);
  if (nv <= 4) return run_rmsnorm<T, 4>(x, add, w, h_out, q, ld_q, scales, ld_s, rows, E, eps, s);
  if constexpr (sizeof(T) == 4) return MVPA_ERR_UNSUPPORTED;  // (refused by the caller: rows of at most 2048)
  else return run_rmsnorm<T, 8>(x, add, w, h_out, q, ld_q, scales, ld_s, rows, E, eps, s);
}

}  // namespace
}  // namespace mvpa

using namespace mvpa;

extern "C" {

int mvpa_quantize_fp8(const void* x, int64_t ld_x, void* q, int64_t ld_q, void* scales, int64_t ld_s, int64_t rows, int32_t width,
                      int32_t block_rows, int32_t dtype, void* cuda_stream) {
  int rc = check("mvpa_quantize_fp8", rows, width, dtype, q, ld_q, scales, ld_s);
  if (rc != MVPA_OK) return rc;
  if (block_rows != 1 && block_rows != kBlock) {
    set_error("mvpa_quantize_fp8: blocks are of 1 or %d rows, got %d", kBlock, block_rows);
    return MVPA_ERR_SHAPE;
  }
  if (rows == 0 || width == 0) return MVPA_OK;
  if (block_rows == kBlock && rows > (int64_t)65535 * kBlock) {
    set_error("mvpa_quantize_fp8: at most %d rows in blocks of %d", 65535 * kBlock, kBlock);
    return MVPA_ERR_SHAPE;
  }
  rc = check_input("mvpa_quantize_fp8", x, ld_x, width, dtype);
  if (rc != MVPA_OK) return rc;
  cudaStream_t s = (cudaStream_t)cuda_stream;
  return dtype == MVPA_F32 ? run_quantize<float>(x, ld_x, q, ld_q, scales, ld_s, rows, width, block_rows, s)
                           : run_quantize<__nv_bfloat16>(x, ld_x, q, ld_q, scales, ld_s, rows, width, block_rows, s);
}

int mvpa_silu_mul_fp8(const void* gate, const void* up, int64_t ld_in, void* q, int64_t ld_q, void* scales, int64_t ld_s,
                      int64_t rows, int32_t width, int32_t dtype, void* cuda_stream) {
  int rc = check("mvpa_silu_mul_fp8", rows, width, dtype, q, ld_q, scales, ld_s);
  if (rc != MVPA_OK || rows == 0 || width == 0) return rc;
  rc = check_input("mvpa_silu_mul_fp8", gate, ld_in, width, dtype);
  if (rc == MVPA_OK) rc = check_input("mvpa_silu_mul_fp8", up, ld_in, width, dtype);
  if (rc != MVPA_OK) return rc;
  cudaStream_t s = (cudaStream_t)cuda_stream;
  return dtype == MVPA_F32 ? run_silu_mul<float>(gate, up, ld_in, q, ld_q, scales, ld_s, rows, width, s)
                           : run_silu_mul<__nv_bfloat16>(gate, up, ld_in, q, ld_q, scales, ld_s, rows, width, s);
}

int mvpa_rmsnorm_fp8(const void* x, const void* add, const void* weight, void* sum_out, void* q, int64_t ld_q, void* scales,
                     int64_t ld_s, int64_t rows, int32_t width, float eps, int32_t dtype, void* cuda_stream) {
  int rc = check("mvpa_rmsnorm_fp8", rows, width, dtype, q, ld_q, scales, ld_s);
  if (rc != MVPA_OK) return rc;
  if (width > (dtype == MVPA_F32 ? 2048 : 4096)) {
    set_error("mvpa_rmsnorm_fp8: rows of at most 4096 (bf16) or 2048 (fp32) elements, got %d", width);
    return MVPA_ERR_UNSUPPORTED;
  }
  if (rows == 0 || width == 0) return MVPA_OK;
  rc = check_input("mvpa_rmsnorm_fp8", x, width, width, dtype);
  if (rc == MVPA_OK) rc = check_input("mvpa_rmsnorm_fp8", weight, width, width, dtype);
  if (rc == MVPA_OK && add != nullptr) rc = check_input("mvpa_rmsnorm_fp8", add, width, width, dtype);
  if (rc == MVPA_OK && sum_out != nullptr) rc = check_input("mvpa_rmsnorm_fp8", sum_out, width, width, dtype);
  if (rc != MVPA_OK) return rc;
  cudaStream_t s = (cudaStream_t)cuda_stream;
  return dtype == MVPA_F32
             ? run_rmsnorm_any<float>(x, add, weight, sum_out, q, ld_q, scales, ld_s, rows, width, eps, s)
             : run_rmsnorm_any<__nv_bfloat16>(x, add, weight, sum_out, q, ld_q, scales, ld_s, rows, width, eps, s);
}

}  // extern "C"
