// out = A B^T for e4m3 operands with a scale for each block of 128 along K:
//
//   out[m, n] = sum_kb sa[m, kb] sb[n / 128, kb] sum_{k in block kb} a[m, k] b[n, k]
//
// The inner sums are tcgen05 products (kind::f8f6f4, fp32 accumulators in TMEM); a block's product leaves TMEM once, is scaled
// and added up in fp32 registers, while the tensor cores work on the next block in the other half of TMEM.  Any fp32 scales
// therefore serve, not only powers of two, and no sum is longer than 128 products before it is scaled.
#include "fp8.cuh"
#include "tc_tma_host.cuh"

namespace mvpa {
namespace {

using namespace fp8;

struct MatmulArgs {
  const void *sa, *sb;
  int64_t sa_m, sa_k, sb_n, sb_k;  // strides in elements
  void* out;
  int64_t ld_out, M;
  int N, KB, per;  // blocks along K, blocks per split
  int* status;
};

template <typename S>
__device__ __forceinline__ float load_scale(const void* p, int64_t i) {
  if constexpr (sizeof(S) == 1) return scale_value(static_cast<const uint8_t*>(p)[i]);
  else return static_cast<const float*>(p)[i];
}

template <typename Out>
__device__ __forceinline__ void store_out(void* out, int64_t i, float v) {
  static_cast<Out*>(out)[i] = from_f32<Out>(v);
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The float at `p`'s place in the shared memory of the cluster's CTA `rank`.
__device__ __forceinline__ float peer_load(const float* p, uint32_t rank) {
  uint32_t at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(ptx::smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

enum : int { kGiveUpEmpty = 71, kGiveUpFull = 72, kGiveUpTmemEmpty = 73, kGiveUpTmemFull = 74, kGiveUpDrain = 75 };

// ---- few rows: 128 weight rows x NT tokens a CTA ----------------------------------------------------------------------------
// The weights are the product's M side, so that one token fills 1/16 of a tile and not 1/128; the tile is transposed in TMEM
// (lane = weight row, column = token).  The blocks along K are split over the CTAs of a cluster where there are too few tiles to
// fill the multiprocessors; their sums meet through distributed shared memory in a fixed order.
template <int NT>
struct FewRows {
  static constexpr int kStageBytes = 128 * 128 + NT * 128;
  static constexpr int kStages = 6;
  static constexpr int kTmemCols = 2 * NT < 32 ? 32 : 2 * NT;
  static constexpr size_t kSmem = 1024 + kStages * kStageBytes;
  static_assert(kStages * kStageBytes >= NT * 128 * 4, "the sums of a split wait in the stages' memory");
};

template <int NT, typename Out, typename S>
__global__ void __launch_bounds__(192) matmul_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                                                         const MatmulArgs g) {
  using C = FewRows<NT>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t s_full[C::kStages], s_empty[C::kStages], s_tfull[2], s_tempty[2];
  __shared__ uint32_t s_tmem;
  __shared__ int s_dead;  // a wait ran out: nothing waits any more, and the results are NaN
  __shared__ __align__(16) float s_scale[2][NT];
  uint8_t* stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * 128;
  const int64_t m0 = (int64_t)blockIdx.y * NT;
  const int kb0 = blockIdx.z * g.per, nkb = min(g.KB - kb0, g.per);
  if (warp == 0) {
    ptx::prefetch_tensormap(&map_w);
    ptx::prefetch_tensormap(&map_x);
  } else if (warp == 1) {
    if (lane == 0) {
      for (int i = 0; i < C::kStages; ++i) {
        ptx::mbar_init(&s_full[i], 1);
        ptx::mbar_init(&s_empty[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        ptx::mbar_init(&s_tfull[i], 1);
        ptx::mbar_init(&s_tempty[i], 4);
      }
      ptx::mbar_fence_init();
      s_dead = 0;
    }
    __syncwarp();
    ptx::tmem_alloc(&s_tmem, C::kTmemCols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = s_tmem;
  volatile int* dead = &s_dead;
  const auto wait = [&](uint64_t& bar, int parity, int code) {
    if (*dead) return false;
    if (ptx::mbar_wait(&bar, (uint32_t)parity, g.status, code)) return true;
    *dead = 1;
    return false;
  };
  ptx::griddep_wait();

  float acc[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j] = 0.f;

  if (warp == 0) {
    if (lane == 0) {
      int i = 0;
      for (; i < nkb; ++i) {
        const int st = i % C::kStages;
        if (i >= C::kStages && !wait(s_empty[st], (i / C::kStages + 1) & 1, kGiveUpEmpty)) break;
        uint8_t* w = stages + st * C::kStageBytes;
        ptx::mbar_arrive_expect_tx(&s_full[st], C::kStageBytes);
        ptx::tma_load_2d(w, &map_w, &s_full[st], (kb0 + i) * 128, n0);
        ptx::tma_load_2d(w + 128 * 128, &map_x, &s_full[st], (kb0 + i) * 128, (int)m0);
      }
      for (int k = i < C::kStages ? 0 : i - C::kStages; k < i; ++k)  // no copy is in flight when the CTA ends
        if (!ptx::mbar_wait(&s_full[k % C::kStages], (k / C::kStages) & 1, g.status, kGiveUpDrain)) break;
    }
  } else if (warp == 1) {
    const uint32_t el = ptx::elect_one();
    constexpr uint32_t idesc = ptx::make_idesc_e4m3(128, NT);
    const uint32_t base = ptx::smem_u32(stages);
    int i = 0;
    for (; i < nkb; ++i) {
      const int st = i % C::kStages, buf = i & 1;
      if (!wait(s_tempty[buf], ((i >> 1) & 1) ^ 1, kGiveUpTmemEmpty)) break;
      if (!wait(s_full[st], (i / C::kStages) & 1, kGiveUpFull)) break;
      ptx::tc_fence_after();
      const uint32_t w = base + st * C::kStageBytes;
      ptx::mma_f8_ss_x4_w(el, tmem + buf * NT, ptx::make_desc_halves_sw128(w, 16, 1024),
                          ptx::make_desc_halves_sw128(w + 128 * 128, 16, 1024), idesc);
      ptx::mma_commit_w(el, ptx::smem_u32(&s_empty[st]));
      ptx::mma_commit_w(el, ptx::smem_u32(&s_tfull[buf]));
    }
    if (i > 0) ptx::mbar_wait(&s_empty[(i - 1) % C::kStages], ((i - 1) / C::kStages) & 1, g.status, kGiveUpDrain);
  } else {
    const int quad = warp & 3, t = threadIdx.x - 64;  // a warp reads the TMEM lanes of its place among four
    const uint32_t at = tmem + ((uint32_t)quad << 21);
    const bool mine = t < NT && m0 + t < g.M;
    const int64_t ia = (m0 + t) * g.sa_m, ib = (int64_t)blockIdx.x * g.sb_n;
    const auto scale_of = [&](int i) {
      return mine && i < nkb ? load_scale<S>(g.sa, ia + (kb0 + i) * g.sa_k) * load_scale<S>(g.sb, ib + (kb0 + i) * g.sb_k) : 0.f;
    };
    if (t < NT) s_scale[0][t] = scale_of(0);
    float next = scale_of(1);
    asm volatile("bar.sync 1, 128;" ::: "memory");
    for (int i = 0; i < nkb; ++i) {
      const int buf = i & 1;
      const float after = scale_of(i + 2);
      if (t < NT) s_scale[buf ^ 1][t] = next;
      next = after;
      wait(s_tfull[buf], (i >> 1) & 1, kGiveUpTmemFull);
      ptx::tc_fence_after();
      constexpr int P = NT < 32 ? 16 : 32;
#pragma unroll
      for (int c = 0; c < NT; c += P) {
        uint32_t r[P];
        if constexpr (P == 32) ptx::tmem_ld32(at + buf * NT + c, r);
        else ptx::tmem_ld16(at + buf * NT + c, r);
        ptx::tmem_ld_wait();
        if (c + P == NT) {
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(&s_tempty[buf]);
        }
#pragma unroll
        for (int j = 0; j < P; j += 4) {
          const float4 s = *reinterpret_cast<const float4*>(&s_scale[buf][c + j]);
          acc[c + j] = fmaf(__uint_as_float(r[j]), s.x, acc[c + j]);
          acc[c + j + 1] = fmaf(__uint_as_float(r[j + 1]), s.y, acc[c + j + 1]);
          acc[c + j + 2] = fmaf(__uint_as_float(r[j + 2]), s.z, acc[c + j + 2]);
          acc[c + j + 3] = fmaf(__uint_as_float(r[j + 3]), s.w, acc[c + j + 3]);
        }
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");  // (the next block's scales are there, this one's are read)
    }
  }

  // (warps 2 to 5 hold the sums: thread `row` one weight row, its NT tokens)
  const int row = (warp & 3) * 32 + lane, splits = gridDim.z;
  const bool sums = warp >= 2, inside = sums && n0 + row < g.N;
  const float poison = *dead ? __uint_as_float(0x7fffffffu) : 0.f;
  const int64_t at = m0 * g.ld_out + n0 + row;
  if (splits == 1) {
    if (inside) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
        if (m0 + j < g.M) store_out<Out>(g.out, at + j * g.ld_out, acc[j] + poison);
    }
  } else {
    float* part = reinterpret_cast<float*>(stages);  // (every product that read the stages is finished)
    if (sums) {
#pragma unroll
      for (int j = 0; j < NT; ++j) part[j * 128 + row] = acc[j] + poison;
    }
    __syncwarp();
    cluster_sync();
    if (inside) {
      for (int j = blockIdx.z; j < NT && m0 + j < g.M; j += splits) {
        float v = 0.f;
        for (int z = 0; z < splits; ++z) v += peer_load(part + j * 128 + row, z);
        store_out<Out>(g.out, at + j * g.ld_out, v);
      }
    }
    __syncwarp();
    cluster_sync();  // nobody's memory goes while it is read
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  if (warp == 1) ptx::tmem_dealloc(tmem, C::kTmemCols);
}

template <int NT, typename Out, typename S>
int run_few(const CUtensorMap& map_w, const CUtensorMap& map_x, MatmulArgs g, cudaStream_t s) {
  using C = FewRows<NT>;
  const int tiles_n = (g.N + 127) / 128;
  const int64_t tiles_m = (g.M + NT - 1) / NT;
  if (tiles_m > 65535) {
    set_error("mvpa_matmul_fp8: too many rows (%lld)", (long long)g.M);
    return MVPA_ERR_UNSUPPORTED;
  }
  int splits = 1;
  while (splits < 8 && tiles_n * tiles_m * splits * 2 <= device_sm_count() && g.KB >= 4 * splits) splits *= 2;
  g.per = (g.KB + splits - 1) / splits;
  splits = (g.KB + g.per - 1) / g.per;
  const auto kernel = matmul_few_kernel<NT, Out, S>;
  MVPA_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kSmem));
  MVPA_CUDA_CHECK(launch_dependent(splits, kernel, dim3(tiles_n, (unsigned)tiles_m, splits), 192, C::kSmem, s, map_w, map_x, g));
  count_launch();
  MVPA_CUDA_CHECK(cudaGetLastError());
  return MVPA_OK;
}

int encode_bytes(CUtensorMap* map, const void* base, int64_t rows, int64_t width, int64_t ld, int box_rows) {
  const uint64_t dims[2] = {(uint64_t)width, (uint64_t)rows}, strides[1] = {(uint64_t)ld};
  const uint32_t box[2] = {128, (uint32_t)box_rows};
  return encode_sw128(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, 2, dims, strides, box);
}

template <typename Out, typename S>
int run_matmul(const void* a, int64_t ld_a, const void* b, int64_t ld_b, int K, const MatmulArgs& g, cudaStream_t s) {
  const int nt = g.M <= 16 ? 16 : g.M <= 32 ? 32 : g.M <= 64 ? 64 : 128;
  CUtensorMap map_w, map_x;
  int rc = encode_bytes(&map_w, b, g.N, K, ld_b, 128);
  if (rc == MVPA_OK) rc = encode_bytes(&map_x, a, g.M, K, ld_a, nt);
  if (rc != MVPA_OK) return rc;
  switch (nt) {
    case 16: return run_few<16, Out, S>(map_w, map_x, g, s);
    case 32: return run_few<32, Out, S>(map_w, map_x, g, s);
    case 64: return run_few<64, Out, S>(map_w, map_x, g, s);
    default: return run_few<128, Out, S>(map_w, map_x, g, s);
  }
}

}  // namespace
}  // namespace mvpa

using namespace mvpa;

extern "C" int mvpa_matmul_fp8(const void* a, int64_t ld_a, const void* a_scales, int64_t a_stride_m, int64_t a_stride_k, const void* b,
                               int64_t ld_b, const void* b_scales, int64_t b_stride_n, int64_t b_stride_k, int32_t scale_dtype, void* out,
                               int64_t ld_out, int64_t M, int32_t N, int32_t K, int32_t out_dtype, int32_t* status, void* cuda_stream) {
  if (M < 0 || N < 0 || K < 0 || M > 0x7fffffff) {
    set_error("mvpa_matmul_fp8: M, N and K must not be negative, M below 2^31 (got %lld, %d, %d)", (long long)M, N, K);
    return MVPA_ERR_SHAPE;
  }
  if ((out_dtype != MVPA_F32 && out_dtype != MVPA_BF16) || (scale_dtype != MVPA_F32 && scale_dtype != MVPA_E8M0)) {
    set_error("mvpa_matmul_fp8: out is MVPA_F32 or MVPA_BF16, scales are MVPA_F32 or MVPA_E8M0");
    return MVPA_ERR_DTYPE;
  }
  if (M == 0 || N == 0) return MVPA_OK;
  const int es = out_dtype == MVPA_F32 ? 4 : 2;
  if (out == nullptr || ld_out < N || (reinterpret_cast<uintptr_t>(out) & (es - 1)) != 0) {
    set_error("mvpa_matmul_fp8: out is NULL, not aligned to its elements, or its leading dimension is below N");
    return MVPA_ERR_ALIGNMENT;
  }
  cudaStream_t s = (cudaStream_t)cuda_stream;
  if (K == 0) {  // sums of nothing
    MVPA_CUDA_CHECK(cudaMemset2DAsync(out, (size_t)ld_out * es, 0, (size_t)N * es, (size_t)M, s));
    return MVPA_OK;
  }
  if (a == nullptr || b == nullptr || ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) != 0 || ld_a % 16 != 0 ||
      ld_b % 16 != 0 || ld_a < K || ld_b < K) {
    set_error("mvpa_matmul_fp8: a and b must be 16-byte aligned with rows of a multiple of 16 bytes, at least K");
    return MVPA_ERR_ALIGNMENT;
  }
  if (a_scales == nullptr || b_scales == nullptr ||
      (scale_dtype == MVPA_F32 && ((reinterpret_cast<uintptr_t>(a_scales) | reinterpret_cast<uintptr_t>(b_scales)) & 3) != 0)) {
    set_error("mvpa_matmul_fp8: the scales are NULL or not aligned to their elements");
    return MVPA_ERR_ALIGNMENT;
  }
  MatmulArgs g = {a_scales, b_scales, a_stride_m, a_stride_k, b_stride_n, b_stride_k, out, ld_out, M, N, (int)(((int64_t)K + 127) / 128), 0, status};
  if (out_dtype == MVPA_BF16)
    return scale_dtype == MVPA_E8M0 ? run_matmul<__nv_bfloat16, uint8_t>(a, ld_a, b, ld_b, K, g, s)
                                    : run_matmul<__nv_bfloat16, float>(a, ld_a, b, ld_b, K, g, s);
  return scale_dtype == MVPA_E8M0 ? run_matmul<float, uint8_t>(a, ld_a, b, ld_b, K, g, s)
                                  : run_matmul<float, float>(a, ld_a, b, ld_b, K, g, s);
}
