// Rows and weights in 8 bits (fp8.cuh): quantisation, the RMSNorm with the residual's addition, the SwiGLU gate.  Bound by
// memory: every input is read once, and what the unquantised kernels write in 16 bits and a further pass would read again
// leaves as e4m3.  Compiled without approximate arithmetic, so that a value next to a rounding border, and numbers below the
// smallest normal one, come out as the formula says.
#include "fp8.cuh"

namespace mvpa {
namespace {

using namespace fp8;

constexpr int kThreads = 256;

// Row blocks are numbered along the rows; eight lanes take one.
struct Unit {
  int64_t row;
  int col;  // of this lane
  int block;
  bool any;
};
__device__ __forceinline__ Unit unit_of(int64_t rows, int width) {
  const int blocks = (width + kBlock - 1) / kBlock;
  const int64_t u = (int64_t)blockIdx.x * (kThreads / 8) + threadIdx.x / 8;
  Unit t;
  if (rows * blocks <= 0x7fffffff) {  // (a 32-bit division where that serves)
    t.row = (uint32_t)u / (uint32_t)blocks;
    t.block = (int)((uint32_t)u - (uint32_t)t.row * (uint32_t)blocks);
  } else {
    t.row = u / blocks;
    t.block = (int)(u - t.row * blocks);
  }
  t.col = t.block * kBlock + (threadIdx.x & 7) * kLane;
  t.any = t.row < rows;
  return t;
}

__device__ __forceinline__ void write_unit(const Unit& t, const float (&y)[kLane], uint8_t* q, int64_t ld_q, uint8_t* scales,
                                           int64_t ld_s, int width) {
  const uint32_t byte = scale_byte(max8(top_of(y)));
  if (!t.any) return;
  if (t.col < width) store16(q + t.row * ld_q, t.col, width, y, inverse_scale(byte));
  if ((threadIdx.x & 7) == 0) scales[t.row * ld_s + t.block] = (uint8_t)byte;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const T* __restrict__ x, int64_t ld_x, uint8_t* __restrict__ q,
                                                                 int64_t ld_q, uint8_t* __restrict__ scales, int64_t ld_s,
                                                                 int64_t rows, int width) {
  ptx::griddep_wait();
  const Unit t = unit_of(rows, width);
  float y[kLane] = {};
  if (t.any) load16<T, VEC>(x + t.row * ld_x, t.col, width, y);
  write_unit(t, y, q, ld_q, scales, ld_s, width);
}

// silu(gate) * up, in fp32 from the inputs to the step to e4m3.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) silu_mul_fp8_kernel(const T* __restrict__ gate, const T* __restrict__ up, int64_t ld_in,
                                                                uint8_t* __restrict__ q, int64_t ld_q, uint8_t* __restrict__ scales,
                                                                int64_t ld_s, int64_t rows, int width) {
  ptx::griddep_wait();
  const Unit t = unit_of(rows, width);
  float y[kLane] = {}, u[kLane] = {};
  if (t.any) {
    load16<T, VEC>(gate + t.row * ld_in, t.col, width, y);
    load16<T, VEC>(up + t.row * ld_in, t.col, width, u);
  }
#pragma unroll
  for (int e = 0; e < kLane; ++e) y[e] = y[e] / (1.f + expf(-y[e])) * u[e];
  write_unit(t, y, q, ld_q, scales, ld_s, width);
}

// One CTA per block of 128 x 128: eight lanes a row, 32 rows at a time, four times; the values wait in registers for the
// block's largest.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_blocks_kernel(const T* __restrict__ x, int64_t ld_x, uint8_t* __restrict__ q,
                                                                   int64_t ld_q, uint8_t* __restrict__ scales, int64_t ld_s,
                                                                   int64_t rows, int width) {
  constexpr int kTimes = kBlock / (kThreads / 8);
  __shared__ uint32_t s_top[kThreads / 32];
  ptx::griddep_wait();
  const int col = blockIdx.x * kBlock + (threadIdx.x & 7) * kLane;
  const int64_t row0 = (int64_t)blockIdx.y * kBlock + threadIdx.x / 8;
  float y[kTimes][kLane] = {};
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kTimes; ++i) {
    const int64_t row = row0 + i * (kThreads / 8);
    if (row < rows) load16<T, VEC>(x + row * ld_x, col, width, y[i]);
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
  for (int i = 0; i < kTimes; ++i) {
    const int64_t row = row0 + i * (kThreads / 8);
    if (row < rows && col < width) store16(q + row * ld_q, col, width, y[i], inverse_scale(byte));
  }
  if (threadIdx.x == 0) scales[(int64_t)blockIdx.y * ld_s + blockIdx.x] = (uint8_t)byte;
}

// y = rmsnorm(h) * w with h = x (+ a, in T as in rmsnorm_kernel); h written out, y to e4m3 without a rounding in between.  One
// warp per row, NV times sixteen values a lane, which stay in registers in T.
template <typename T, int NV, bool VEC>
__global__ void __launch_bounds__(kWarpsPerCta * 32) rmsnorm_fp8_kernel(const T* __restrict__ x, const T* __restrict__ a,
                                                                        const T* __restrict__ w, T* __restrict__ h_out,
                                                                        uint8_t* __restrict__ q, int64_t ld_q,
                                                                        uint8_t* __restrict__ scales, int64_t ld_s, int64_t rows,
                                                                        int E, float eps) {
  constexpr int N = Vec<T>::N, P = kLane / N;
  ptx::griddep_wait();
  const int64_t row = (int64_t)blockIdx.x * kWarpsPerCta + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  const int64_t at = row * E;
  uint4 raw[NV][P];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int col = (i * 32 + lane) * kLane;
    float v[kLane] = {};
    if (col < E) load16<T, VEC>(x + at, col, E, v);
    if (a != nullptr && col < E) {
      float b[kLane];
      load16<T, VEC>(a + at, col, E, b);
#pragma unroll
      for (int e = 0; e < kLane; ++e) v[e] = Vec<T>::round(v[e] + b[e]);
    }
#pragma unroll
    for (int e = 0; e < kLane; ++e) ss = fmaf(v[e], v[e], ss);
#pragma unroll
    for (int p = 0; p < P; ++p) {
      float f[N];
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] = v[p * N + e];
      raw[i][p] = Vec<T>::pack(f);
    }
    if (h_out != nullptr && col < E) {
      if (VEC && col + kLane <= E) {
#pragma unroll
        for (int p = 0; p < P; ++p) *reinterpret_cast<uint4*>(h_out + at + col + p * N) = raw[i][p];
      } else {
#pragma unroll
        for (int e = 0; e < kLane; ++e)
          if (col + e < E) h_out[at + col + e] = from_f32<T>(v[e]);
      }
    }
  }
  const float rstd = rsqrtf(warp_sum(ss) / (float)E + eps);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int col = (i * 32 + lane) * kLane;
    if (i * 32 * kLane >= E) break;  // (the same for the whole warp)
    float y[kLane], g[kLane] = {};
    if (col < E) load16<T, VEC>(w, col, E, g);
#pragma unroll
    for (int p = 0; p < P; ++p) {
      float f[N];
      Vec<T>::unpack(raw[i][p], f);
#pragma unroll
      for (int e = 0; e < N; ++e) y[p * N + e] = f[e] * rstd * g[p * N + e];
    }
#pragma unroll
    for (int e = 0; e < kLane; ++e)
      if (col + e >= E) y[e] = 0.f;  // (past the end 0 * rstd would be NaN where rstd is)
    const uint32_t byte = scale_byte(max8(top_of(y)));
    if (col < E) {
      store16(q + row * ld_q, col, E, y, inverse_scale(byte));
      if ((lane & 7) == 0) scales[row * ld_s + col / kBlock] = (uint8_t)byte;
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
template <typename T>
bool vectors(const void* p, int64_t ld) { return aligned16(p) && ld * (int64_t)sizeof(T) % 16 == 0; }

int check(const char* what, int64_t rows, int32_t width, int32_t dtype, const void* q, int64_t ld_q, const void* scales,
          int64_t ld_s) {
  if (rows < 0 || width < 0) {
    set_error("%s: negative sizes (%lld rows of %d)", what, (long long)rows, width);
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
  if (rows > (int64_t)0x7fffffff * 8 / ((width + kBlock - 1) / kBlock)) {
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

unsigned units_grid(int64_t rows, int width) {
  return (unsigned)((rows * ((width + kBlock - 1) / kBlock) + kThreads / 8 - 1) / (kThreads / 8));
}

template <typename T>
int run_quantize(const void* x, int64_t ld_x, void* q, int64_t ld_q, void* scales, int64_t ld_s, int64_t rows, int width, int tall,
                 cudaStream_t s) {
  const bool vec = vectors<T>(x, ld_x);
  if (tall == 1) {
    const unsigned grid = units_grid(rows, width);
    MVPA_CUDA_CHECK(launch_dependent(1, vec ? quantize_rows_kernel<T, true> : quantize_rows_kernel<T, false>, grid, kThreads, 0, s,
                                     (const T*)x, ld_x, (uint8_t*)q, ld_q, (uint8_t*)scales, ld_s, rows, width));
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
  MVPA_CUDA_CHECK(launch_dependent(1, vec ? silu_mul_fp8_kernel<T, true> : silu_mul_fp8_kernel<T, false>, units_grid(rows, width),
                                   kThreads, 0, s, (const T*)gate, (const T*)up, ld_in, (uint8_t*)q, ld_q, (uint8_t*)scales, ld_s, rows,
                                   width));
  count_launch();
  MVPA_CUDA_CHECK(cudaGetLastError());
  return MVPA_OK;
}

template <typename T, int NV>
int run_rmsnorm(const void* x, const void* add, const void* w, void* h_out, void* q, int64_t ld_q, void* scales, int64_t ld_s,
                int64_t rows, int E, float eps, cudaStream_t s) {
  const bool vec = vectors<T>(x, E) && aligned16(w) && (add == nullptr || aligned16(add)) && (h_out == nullptr || aligned16(h_out));
  const unsigned grid = (unsigned)((rows + kWarpsPerCta - 1) / kWarpsPerCta);
  MVPA_CUDA_CHECK(launch_dependent(1, vec ? rmsnorm_fp8_kernel<T, NV, true> : rmsnorm_fp8_kernel<T, NV, false>, grid,
                                   kWarpsPerCta * 32, 0, s, (const T*)x, (const T*)add, (const T*)w, (T*)h_out, (uint8_t*)q, ld_q,
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
