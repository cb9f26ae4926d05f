// out = A B^T for e4m3 operands with a scale for each block of 128 along K:
//
//   out[m, n] = sum_kb sa[m, kb] sb[n / 128, kb] sum_{k in block kb} a[m, k] b[n, k]
//
// The inner sums are tcgen05 products of e4m3 with fp32 accumulators in TMEM.  Three kernels, by the number of tokens and the type
// of the scales (run_matmul has the rule):
//   few     up to 32 tokens: the weights' rows are the product's M side
//   many    fp32 scales: a block's product leaves TMEM once, is scaled and added up in fp32 registers, so that any numbers serve
//   scaled  scales that are powers of two (e8m0): the tensor cores apply them, and a tile's sum stays in TMEM over the whole of K
#include <type_traits>

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
  int splits;      // pairs of CTAs that share a tile
  int out_tma;     // out's rows start on 16-byte boundaries (1), and end on them too (2)
  int* status;
};

// The two scales of a block as they lie in memory: loaded two blocks ahead, and not touched before they are wanted, since the
// first use is what waits for the load.
template <typename S>
struct Scales {
  S a, b;
  __device__ __forceinline__ float product() const {
    if constexpr (sizeof(S) == 1) return scale_value(a) * scale_value(b);
    else return a * b;
  }
};

template <typename Out>
__device__ __forceinline__ void store_out(void* out, int64_t i, float v) {
  static_cast<Out*>(out)[i] = from_f32<Out>(v);
}

// The float at this place in the shared memory of the cluster's CTA `rank`.
__device__ __forceinline__ float peer_load(uint32_t at, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(ptx::cluster_map(at, rank)) : "memory");
  return v;
}

enum : int { kGiveUpEmpty = 71, kGiveUpFull = 72, kGiveUpTmemEmpty = 73, kGiveUpTmemFull = 74, kGiveUpDrain = 75 };

// The kernel's shared memory is granted once per device (and thread) and not at every call.
template <auto kernel>
cudaError_t grant_smem(size_t bytes) {
  static thread_local uint64_t granted = 0;  // a bit per device
  int device = 0;
  const cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess || (device < 64 && (granted >> device & 1))) return e;
  const cudaError_t set = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (set == cudaSuccess && device < 64) granted |= (uint64_t)1 << device;
  return set;
}

// How many clusters of `ctas` CTAs along x (up to eight) the current device holds at once; asked once per device (and thread).
template <auto kernel>
cudaError_t resident_clusters(int ctas, int threads, size_t smem, int* clusters) {
  static thread_local int known[64][9] = {};  // (one more than the number; 0: not asked yet)
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  if (device < 64 && known[device][ctas] != 0) {
    *clusters = known[device][ctas] - 1;
    return cudaSuccess;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas * 64);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ctas;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  e = cudaOccupancyMaxActiveClusters(clusters, kernel, &cfg);
  if (e == cudaSuccess && device < 64) known[device][ctas] = *clusters + 1;
  return e;
}

// ---- few rows: 128 weight rows x all of up to NT tokens a CTA ----------------------------------------------------------------------------
// The weights are the product's M side, so that one token fills 1/16 of a tile and not 1/128; the tile is transposed in TMEM
// (lane = weight row, column = token).  The blocks along K are split over the CTAs of a cluster where there are too few tiles to
// fill the multiprocessors; their sums meet through distributed shared memory in a fixed order.
template <int NT>
struct FewRows {
  static constexpr int kStageBytes = 128 * 128 + NT * 128;
  static constexpr int kStages = NT == 16 ? 6 : 5;  // (as many as let two CTAs share a multiprocessor)
  static constexpr int kBuffers = 4;  // products on their way home
  static constexpr int kTmemCols = kBuffers * NT;
  static constexpr size_t kSmem = 1024 + kStages * kStageBytes;
  static_assert(kStages * kStageBytes >= NT * 128 * 4, "the sums of a split wait in the stages' memory");
  static_assert(2 * (kSmem + 2048) <= 228 * 1024, "two CTAs, with what the system and the kernel's own variables take of each");
};

template <int NT, typename Out, typename S>
__global__ void __launch_bounds__(192) matmul_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                                                         const MatmulArgs g) {
  using C = FewRows<NT>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t s_full[C::kStages], s_empty[C::kStages], s_tfull[C::kBuffers], s_tempty[C::kBuffers];
  __shared__ uint32_t s_tmem;
  __shared__ int s_dead;  // a wait ran out: nothing waits any more, and the results are NaN
  __shared__ __align__(16) float s_scale[2][NT];
  uint8_t* stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * 128;
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
      for (int i = 0; i < C::kBuffers; ++i) {
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
  const auto wait = [&](uint64_t& bar, uint32_t parity, int code) {
    if (ptx::mbar_test_wait(&bar, parity)) return true;
    if (*dead) return false;
    if (ptx::mbar_wait(&bar, parity, g.status, code)) return true;
    *dead = 1;
    return false;
  };
  ptx::griddep_launch();
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
        ptx::tma_load_2d(w + 128 * 128, &map_x, &s_full[st], (kb0 + i) * 128, 0);
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
      const int st = i % C::kStages, buf = i % C::kBuffers;
      if (!wait(s_tempty[buf], ((i / C::kBuffers) & 1) ^ 1, kGiveUpTmemEmpty)) break;
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
    const bool mine = t < NT && t < g.M;
    const int64_t ia = t * g.sa_m, ib = (int64_t)blockIdx.x * g.sb_n;
    const S *pa = static_cast<const S*>(g.sa) + ia, *pb = static_cast<const S*>(g.sb) + ib;
    const auto scales_of = [&](int i) {
      Scales<S> v = {};
      if (mine && i < nkb) v = {pa[(kb0 + i) * g.sa_k], pb[(kb0 + i) * g.sb_k]};
      return v;
    };
    if (t < NT) s_scale[0][t] = scales_of(0).product();
    Scales<S> next = scales_of(1);
    asm volatile("bar.sync 1, 128;" ::: "memory");
    for (int i = 0; i < nkb; ++i) {
      const int buf = i % C::kBuffers, turn = i & 1;
      const Scales<S> after = scales_of(i + 2);
      if (t < NT) s_scale[turn ^ 1][t] = next.product();
      next = after;
      wait(s_tfull[buf], (i / C::kBuffers) & 1, kGiveUpTmemFull);
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
          const float4 s = *reinterpret_cast<const float4*>(&s_scale[turn][c + j]);
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
  const int64_t at = n0 + row;
  if (splits == 1) {
    if (inside) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
        if (j < g.M) store_out<Out>(g.out, at + j * g.ld_out, acc[j] + poison);
    }
  } else {
    float* part = reinterpret_cast<float*>(stages);  // (every product that read the stages is finished)
    if (sums) {
#pragma unroll
      for (int j = 0; j < NT; ++j) part[j * 128 + row] = acc[j] + poison;
    }
    __syncwarp();
    ptx::cluster_sync();
    if (inside) {
      for (int j = blockIdx.z; j < NT && j < g.M; j += splits) {
        float v = 0.f;
        for (int z = 0; z < splits; ++z) v += peer_load(ptx::smem_u32(part + j * 128 + row), z);
        store_out<Out>(g.out, at + j * g.ld_out, v);
      }
    }
    __syncwarp();
    ptx::cluster_sync();  // nobody's memory goes while it is read
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  if (warp == 1) ptx::tmem_dealloc(tmem, C::kTmemCols);
}

template <int NT, typename Out, typename S>
int run_few(const CUtensorMap& map_w, const CUtensorMap& map_x, MatmulArgs g, cudaStream_t s) {
  using C = FewRows<NT>;
  const int64_t tiles = (g.N + 127) / 128, sms = device_sm_count();
  // Up to two CTAs on a multiprocessor (their stages take half of its memory each), with a few blocks each: one token x 15360 x 2048
  // takes 8.1 us in 120 CTAs and 6.7 in 240, x 2048 x 7680 23.4 in 16 CTAs, 8.8 in 64 and 5.9 in 128.  For 17 to 32 tokens that takes
  // five stages: with six one CTA fits, and what was split for two runs in two turns (22 rows, six / five stages, us: 15360 x 2048
  // 15.9 / 9.6, 2048 x 7680 12.3 / 7.3, 4096 x 4096 14.3 / 6.6, 9500 x 6000 28.0 / 16.6; unsplit in six 8.5 / - / 7.3 / 20.0).
  int splits = 1;
  while (splits < 8 && ((tiles * splits * 2 <= sms && g.KB >= 4 * splits) || (tiles * splits <= sms && g.KB >= 8 * splits))) splits *= 2;
  g.per = (g.KB + splits - 1) / splits;
  splits = (g.KB + g.per - 1) / g.per;
  constexpr auto kernel = matmul_few_kernel<NT, Out, S>;
  MVPA_CUDA_CHECK(grant_smem<kernel>(C::kSmem));
  MVPA_CUDA_CHECK(launch_dependent(splits, kernel, dim3((unsigned)tiles, 1, splits), 192, C::kSmem, s, map_w, map_x, g));
  count_launch();
  MVPA_CUDA_CHECK(cudaGetLastError());
  return MVPA_OK;
}

// ---- many rows: 256 tokens x 256 weight rows a pair of CTAs ------------------------------------------------------------------
// One product over both CTAs' operands (cta_group::2): each CTA loads 128 tokens and 128 weight rows a block and holds its 128
// tokens x 256 sums, so a loaded byte meets twice the operands that it would in one CTA's tile.  The pairs are resident and take
// their tiles one after the other; TMEM holds the products of two blocks, and eight warps a CTA bring them home: a thread has one
// token's 128 columns in registers.
struct ManyRows {
  static constexpr int kStageBytes = 2 * 128 * 128;
  static constexpr int kStages = 5;
  static constexpr int kOutBytes = 8 * 2 * 32 * 128;  // a warp's tokens x 128 bytes of columns, twice
  static constexpr size_t kSmem = 1024 + kStages * kStageBytes + kOutBytes;
  static_assert(256 * 128 * 4 <= kStages * kStageBytes, "the sums of a split wait in the stages' memory");
};
// Four warps that load and issue, eight that add up.  Registers: 384 x 168 at launch, of which the four keep 56 a thread and the
// eight take 216 (128 x 56 + 256 x 216 = 62464 of 64512).
constexpr int kManyThreads = 384;

// Results on their way out: a warp puts 32 tokens x 128 bytes of columns into shared memory (in the 128-byte swizzle: a token's
// 16-byte pieces go to eight different places) and leaves them to the TMA, which writes whole lines, skips rows and pieces of
// 16 bytes past the matrix, and lets the warp go on.  Stored from registers a tile of 256 x 256 held its warps for 4200 cycles of 20000.
struct OutRing {
  uint32_t smem;
  bool two;  // places, or one
  uint32_t which = 0;
  // Where the next 128 bytes of columns go; the store that was there has been read.  (With two places all groups but the newest are
  // waited for, so each use of a place has to be one group: send() commits its store, write() an empty group.)
  __device__ __forceinline__ uint32_t next(int lane) {
    if (lane == 0) {
      if (two) ptx::tma_store_wait_read<1>();
      else ptx::tma_store_wait_read<0>();
    }
    __syncwarp();
    which ^= two ? 1 : 0;
    return smem + which * 4096;
  }
  __device__ __forceinline__ static void put(uint32_t at, int lane, int piece, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + lane * 128 + ((piece ^ (lane & 7)) << 4)), "r"(a), "r"(b), "r"(c), "r"(d)
                 : "memory");
  }
  // Whether the TMA may store `cols` columns from `n` on: it writes whole pieces of 16 bytes, past a row's end too.
  __device__ __forceinline__ static bool whole(const MatmulArgs& g, int n, int cols) { return g.out_tma == 2 || (g.out_tma == 1 && n + cols <= g.N); }
  // The same without the TMA, for other rows and their ends: lanes along the columns, a row at a time.
  template <typename Out>
  __device__ __forceinline__ static void write(uint32_t at, int lane, Out* out, int64_t ld, int rows, int cols) {
    constexpr int kCols = 128 / sizeof(Out);
    using Word = typename std::conditional<sizeof(Out) == 2, uint16_t, uint32_t>::type;
    constexpr int kEach = kCols / 32, kRows = 8;
    __syncwarp();
    for (int r0 = 0; r0 < rows; r0 += kRows) {
      Word v[kRows][kEach];
#pragma unroll
      for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int c = 0; c < kEach; ++c) {
          const int byte = (lane + 32 * c) * (int)sizeof(Out);
          const uint32_t from = at + (r0 + r) * 128 + (((byte >> 4) ^ r) << 4) + (byte & 15);
          if constexpr (sizeof(Out) == 2) asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v[r][c]) : "r"(from));
          else asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[r][c]) : "r"(from));
        }
#pragma unroll
      for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int c = 0; c < kEach; ++c)
          if (r0 + r < rows && lane + 32 * c < cols) reinterpret_cast<Word*>(out)[(r0 + r) * ld + lane + 32 * c] = v[r][c];
    }
    if (lane == 0) ptx::tma_store_commit();
    __syncwarp();
  }
  __device__ __forceinline__ static void send(uint32_t at, int lane, const CUtensorMap* map, int x, int y) {
    ptx::fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      ptx::tma_store_2d(map, at, x, y);
      ptx::tma_store_commit();
    }
  }
};

struct Tile {
  int m0, n0;
};
// Tiles in bands of eight along M: the pairs at work together share few panels of both operands.
template <int kTileN>
__device__ __forceinline__ Tile tile_at(uint32_t t, uint32_t tiles_n, uint32_t tiles_m) {
  constexpr uint32_t kBand = 8;
  const uint32_t band = t / (kBand * tiles_n), rest = t - band * kBand * tiles_n;
  const uint32_t high = min(kBand, tiles_m - band * kBand), n = rest / high;
  return {(int)((band * kBand + rest - n * high) * 256), (int)(n * kTileN)};
}

// A place in a ring of N, and the parity of the pass over it.
template <uint32_t N>
struct Ring {
  uint32_t at = 0, parity = 0;
  __device__ __forceinline__ void step() {
    if (++at == N) {
      at = 0;
      parity ^= 1;
    }
  }
};

// A tile whose blocks several pairs have summed, a token's columns in the shared memory of the CTA of each pair that holds its rows
// (sums[column][row]): each pair has its share of the columns, a thread eight of a token at a time, and adds in the order of the
// blocks.  `group` of `groups`: which 128 threads of the CTA's these are; `turn`: 1 KB of the warp's own, by way of which rows that do
// not start on 16-byte boundaries are written eight columns of four rows at a time.
template <typename Out>
__device__ __forceinline__ void add_splits(uint32_t sums, uint32_t turn, uint32_t splits, uint32_t split, int columns, uint32_t half, int row,
                                           int group, int groups, const Tile& at, const MatmulArgs& g) {
  const int share = columns / (int)splits, lane = row & 31;
  const int64_t m = at.m0 + (int)half * 128 + row;
  for (int c = (int)split * share + group * 8; c < (int)(split + 1) * share; c += groups * 8) {
    const int n = at.n0 + c;
    if (n >= g.N || m - lane >= g.M) break;  // (the same for the whole warp)
    float v[8] = {};
    for (uint32_t z = 0; z < splits; ++z) {
      float p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = peer_load(sums + ((c + j) * 128 + row) * 4, 2 * z + half);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += p[j];
    }
    if (g.out_tma && n + 8 <= g.N) {  // (rows on 16-byte boundaries)
      Out* out = static_cast<Out*>(g.out) + m * g.ld_out + n;
      if (m >= g.M) continue;
      if constexpr (sizeof(Out) == 2) {
        *reinterpret_cast<uint4*>(out) =
            make_uint4(ptx::pack_bf16(v[0], v[1]), ptx::pack_bf16(v[2], v[3]), ptx::pack_bf16(v[4], v[5]), ptx::pack_bf16(v[6], v[7]));
      } else {
        reinterpret_cast<float4*>(out)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(out)[1] = make_float4(v[4], v[5], v[6], v[7]);
      }
      continue;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) asm volatile("st.shared.f32 [%0], %1;" ::"r"(turn + (lane * 8 + ((j + lane) & 7)) * 4), "f"(v[j]) : "memory");
    __syncwarp();
    const int col = lane & 7;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int r = k * 4 + (lane >> 3);
      float w;
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(w) : "r"(turn + (r * 8 + ((col + r) & 7)) * 4) : "memory");
      if (m - lane + r < g.M && n + col < g.N) static_cast<Out*>(g.out)[(m - lane + r) * g.ld_out + n + col] = from_f32<Out>(w);
    }
    __syncwarp();
  }
}

// One operand's tiles on their way in: a warp of each CTA loads its CTA's `rows` rows a block; the loads of both count at the barrier
// of the pair's first CTA, which the tokens' warp there tells how many bytes to expect.  (One lane that issued both operands' loads
// from a branch of its own needed some 450 cycles a block, more than the products of it.)
template <int kStages, int kTileN, int kBytes, typename Wait>
__device__ __forceinline__ void load_operand(const CUtensorMap* map, uint32_t to, bool tokens, int rows, uint64_t* full, uint64_t* empty,
                                             uint32_t pair, uint32_t pairs, uint32_t tiles_n, uint32_t tiles_m, int kb0, int nkb, int* status,
                                             const Wait& wait) {
  const uint32_t el = ptx::elect_one(), rank = ptx::cluster_rank(), half = rank & 1, tiles = tiles_n * tiles_m;
  const uint32_t there = ptx::cluster_map(ptx::smem_u32(full), rank - half);
  Ring<kStages> st;
  uint32_t loads = 0;
  bool on = true;
  for (uint32_t t = pair; t < tiles && on; t += pairs) {
    const Tile at = tile_at<kTileN>(t, tiles_n, tiles_m);
    const int y = (tokens ? at.m0 : at.n0) + (int)half * rows;
    for (int kb = 0; kb < nkb; ++kb, ++loads, st.step()) {
      if (!wait(empty[st.at], st.parity ^ 1, kGiveUpEmpty)) {
        on = false;
        break;
      }
      if (tokens && half == 0 && el) ptx::mbar_arrive_expect_tx(&full[st.at], 2 * kBytes);
      __syncwarp();
      ptx::tma_load_2d_pair_w(el, to + st.at * kBytes, map, there + 8 * st.at, (kb0 + kb) * 128, y);
    }
  }
  if (tokens && half == 0) {  // no copy is in flight when the CTAs end (the other one waits for this one at the end)
    const uint32_t n = min(loads, (uint32_t)kStages);
    for (uint32_t k = loads - n; k != loads; ++k)
      if (!ptx::mbar_wait(&full[k % kStages], (k / kStages) & 1, status, kGiveUpDrain)) break;
  }
}

template <typename Out, typename S, bool SPLIT>
__global__ void __launch_bounds__(kManyThreads, 1) matmul_many_kernel(const __grid_constant__ CUtensorMap map_w,
                                                                      const __grid_constant__ CUtensorMap map_x,
                                                                      const __grid_constant__ CUtensorMap map_o, const MatmulArgs g) {
  using C = ManyRows;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t s_full[C::kStages], s_empty[C::kStages], s_tfull[2], s_tempty[2];
  __shared__ uint32_t s_tmem;
  __shared__ int s_dead;
  const uint32_t stages = (ptx::smem_u32(smem_raw) + 1023) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = ptx::cluster_rank() & 1, first_rank = SPLIT ? ptx::cluster_rank() - rank : 0, split = first_rank >> 1;
  const uint32_t splits = SPLIT ? (uint32_t)g.splits : 1;
  const uint32_t pair = blockIdx.x / (2 * splits), pairs = gridDim.x / (2 * splits);  // (SPLIT: a cluster's pairs have one tile)
  const int kb_first = SPLIT ? (int)split * g.per : 0, nkb = SPLIT ? min(g.KB - kb_first, g.per) : g.KB;
  const uint16_t both = (uint16_t)(3u << first_rank);
  const uint32_t tiles_n = (uint32_t)(g.N + 255) / 256, tiles_m = (uint32_t)((g.M + 255) / 256), tiles = tiles_n * tiles_m;
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
        ptx::mbar_init(&s_tempty[i], 16);
      }
      ptx::mbar_fence_init();
      s_dead = 0;
    }
    __syncwarp();
    ptx::tmem_alloc_pair(&s_tmem, 512);
    ptx::tmem_relinquish_pair();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::cluster_sync();
  ptx::tc_fence_after();
  const uint32_t tmem = s_tmem;
  volatile int* dead = &s_dead;
  const auto wait = [&](uint64_t& bar, uint32_t parity, int code) {
    if (ptx::mbar_test_wait(&bar, parity)) return true;
    if (*dead) return false;
    if (ptx::mbar_wait(&bar, parity, g.status, code)) return true;
    *dead = 1;
    return false;
  };
  ptx::griddep_launch();
  ptx::griddep_wait();

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0 || warp == 2) {  // tokens, weights
      load_operand<C::kStages, 256, C::kStageBytes>(warp == 0 ? &map_x : &map_w, stages + (warp == 0 ? 0 : 128 * 128), warp == 0, 128, s_full,
                                                    s_empty, pair, pairs, tiles_n, tiles_m, kb_first, nkb, g.status, wait);
    } else if (warp == 1 && rank == 0) {
      const uint32_t el = ptx::elect_one();
      constexpr uint32_t idesc = ptx::make_idesc_e4m3(256, 256);
      Ring<C::kStages> st;
      Ring<2> buf;
      uint32_t last = 0, last_parity = 0;
      const uint32_t mine = pair < tiles ? ((tiles - pair + pairs - 1) / pairs) * (uint32_t)nkb : 0;
      uint32_t i = 0;
      for (; i < mine; ++i, st.step(), buf.step()) {
        const uint32_t x = stages + st.at * C::kStageBytes;
        const ptx::DescHalves a = ptx::make_desc_halves_sw128(x, 16, 1024), b = ptx::make_desc_halves_sw128(x + 128 * 128, 16, 1024);
        if (!wait(s_full[st.at], st.parity, kGiveUpFull)) break;
        if (!wait(s_tempty[buf.at], buf.parity ^ 1, kGiveUpTmemEmpty)) break;
        ptx::tc_fence_after();
        ptx::mma_f8_ss_x4_pair_w(el, tmem + buf.at * 256, a, b, idesc);
        ptx::mma_commit_pair_w(el, both, ptx::smem_u32(&s_tfull[buf.at]));
        ptx::mma_commit_pair_w(el, both, ptx::smem_u32(&s_empty[st.at]));
        last = st.at;
        last_parity = st.parity;
      }
      if (i > 0) ptx::mbar_wait(&s_empty[last], last_parity, g.status, kGiveUpDrain);
    }
    if constexpr (SPLIT) {
      __syncwarp();
      ptx::cluster_sync();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int row = (int)rank * 128 + (warp & 3) * 32 + lane, half = (warp - 4) >> 2;
    const uint32_t at_tmem = tmem + ((uint32_t)(warp & 3) << 21) + half * 128;
    const uint32_t tempty[2] = {ptx::cluster_map(ptx::smem_u32(&s_tempty[0]), first_rank), ptx::cluster_map(ptx::smem_u32(&s_tempty[1]), first_rank)};
    OutRing ring = {stages + C::kStages * C::kStageBytes + (warp - 4) * 8192, true};
    Ring<2> buf;
    for (uint32_t t = pair; t < tiles; t += pairs) {
      const Tile at = tile_at<256>(t, tiles_n, tiles_m);
      const int64_t m = at.m0 + row;
      const int n0 = at.n0 + half * 128;
      const bool mine = m < g.M && n0 < g.N;
      const S* pa = static_cast<const S*>(g.sa) + m * g.sa_m + kb_first * g.sa_k;
      const S* pb = static_cast<const S*>(g.sb) + (int64_t)(n0 / 128) * g.sb_n + kb_first * g.sb_k;
      const auto scales_of = [&](int kb) {
        Scales<S> v = {};
        if (mine && kb < nkb) v = {pa[kb * g.sa_k], pb[kb * g.sb_k]};
        return v;
      };
      float2 acc[64];
#pragma unroll
      for (int j = 0; j < 64; ++j) acc[j] = make_float2(0.f, 0.f);
      Scales<S> now = scales_of(0), next = scales_of(1);
#pragma unroll 1
      for (int kb = 0; kb < nkb; ++kb, buf.step()) {
        const Scales<S> after = scales_of(kb + 2);
        wait(s_tfull[buf.at], buf.parity, kGiveUpTmemFull);
        __syncwarp();
        ptx::tc_fence_after();
        const uint32_t from = at_tmem + buf.at * 256;
        uint32_t r0[32], r1[32];
        float2 s2;
        const auto add = [&](int c, const uint32_t (&r)[32]) {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            acc[c * 16 + j] = ptx::ffma2(make_float2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])), s2, acc[c * 16 + j]);
        };
        ptx::tmem_ld32(from, r0);
        ptx::tmem_ld32(from + 32, r1);
        s2.x = s2.y = now.product();
        ptx::tmem_ld_wait();
        add(0, r0);
        ptx::tmem_ld32(from + 64, r0);
        add(1, r1);
        ptx::tmem_ld32(from + 96, r1);
        ptx::tmem_ld_wait();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive_cluster(tempty[buf.at]);
        add(2, r0);
        add(3, r1);
        now = next;
        next = after;
      }
      if (*dead) {
#pragma unroll
        for (int j = 0; j < 64; ++j) acc[j].x = acc[j].y = __uint_as_float(0x7fffffffu);
      }
      if constexpr (SPLIT) {  // (the products that read the stages are finished)
#pragma unroll
        for (int c = 0; c < 128; ++c)
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(stages + ((half * 128 + c) * 128 + (warp & 3) * 32 + lane) * 4),
                       "r"(__float_as_uint(c & 1 ? acc[c / 2].y : acc[c / 2].x))
                       : "memory");
        continue;
      }
      constexpr int kCols = 128 / sizeof(Out);
      const int y = at.m0 + row - lane;
#pragma unroll
      for (int c = 0; c < 128; c += kCols) {
        if (y >= g.M || n0 + c >= g.N) break;  // (the same for the whole warp: a store does not begin past the matrix)
        const uint32_t to = ring.next(lane);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float2* v = acc + c / 2 + k * (16 / sizeof(Out) / 2);
          if constexpr (sizeof(Out) == 2)
            OutRing::put(to, lane, k, ptx::pack_bf16(v[0].x, v[0].y), ptx::pack_bf16(v[1].x, v[1].y), ptx::pack_bf16(v[2].x, v[2].y),
                         ptx::pack_bf16(v[3].x, v[3].y));
          else
            OutRing::put(to, lane, k, __float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
        }
        if (OutRing::whole(g, n0 + c, kCols)) OutRing::send(to, lane, &map_o, n0 + c, y);
        else OutRing::write(to, lane, static_cast<Out*>(g.out) + y * g.ld_out + n0 + c, g.ld_out, (int)min(g.M - y, (int64_t)32), g.N - n0 - c);
      }
    }
    if (lane == 0) ptx::tma_store_wait_all();
    if constexpr (SPLIT) {
      __syncwarp();
      ptx::cluster_sync();
      add_splits<Out>(stages, ring.smem, splits, split, 256, rank, (warp & 3) * 32 + lane, half, 2, tile_at<256>(pair, tiles_n, tiles_m), g);
    }
  }
  __syncwarp();
  ptx::tc_fence_before();
  __syncthreads();
  ptx::cluster_sync();  // neither CTA's memory goes while the other's products or barriers use it
  ptx::tc_fence_after();
  if (warp == 1) ptx::tmem_dealloc_pair(tmem, 512);
}

// ---- many rows, scales that are powers of two: the tensor cores apply them -----------------------------------------------------
// The scales go to TMEM beside the products (kind::mxf8f6f4, which wants one for each 32 along K: a block's serves four times), so
// a tile's sum stays in TMEM over the whole of K and comes home once.  In matmul_many_kernel a block's product has to be fetched
// before the block after the next can start - 512 cycles of products, then some 1400 to hear of them, fetch them in both CTAs and
// say so - which leaves the tensor cores idle half of the time.  Tiles of 256 tokens x 192 weight rows: two of them and the scales
// of three groups of four blocks take 432 of TMEM's 512 columns, and a tile leaves while the next one is summed.
//
// A word of TMEM has room for four scales, and a product names the byte that it wants: they are laid out and copied for four
// blocks at once.  (For each block, four bytes alike, the three copies took the tensor cores' time as well, 100 cycles for 384 of
// products: 470 us for 16384 x 15360 x 2048.)
//
// A long K and so few tiles that most pairs would have none: the pairs of a cluster share the blocks of a tile and add their sums up
// through distributed shared memory, in the order of the blocks.
//
// Where 192 columns a tile would leave pairs without one, tiles of 64: a multiprocessor takes some 150 bytes in a nanosecond, so a
// block of 256 x 64 is there after 0.14 us and one of 256 x 192 after 0.19.
//
// Warps: 0 and 2 load tokens and weights, 1 issues, 3 lays the scales out in shared memory, 4 to 11 take the sums home, every
// other 128 bytes of columns each.
template <int TN>
struct ScaledRows {
  static constexpr int kTileN = TN, kHalfN = kTileN / 2;
  static constexpr int kStages = 6;
  static constexpr int kGroup = 4, kGroups = 3;   // blocks that share a word of scales; such groups on their way
  static constexpr int kOperandBytes = 128 * 128 + kHalfN * 128;
  static constexpr int kScaleBytes = 512 + 1024;  // 128 tokens; two groups of 128 weight rows
  static constexpr int kOutBytes = (8 + 4) * 32 * 128;  // two places for the warps that have more columns, one for the others
  static constexpr uint32_t kTmemScales = 2 * kTileN, kTmemScaleCols = 16;
  static constexpr size_t kSmem = 1024 + kStages * kOperandBytes + kGroups * kScaleBytes + kOutBytes;
  static_assert(kTileN * 128 * 4 <= kStages * kOperandBytes, "the sums of a split wait in the stages' memory");
  static_assert(kTmemScales + kGroups * kTmemScaleCols <= 512 && kOperandBytes % 1024 == 0, "");
};
constexpr int kScaledThreads = 384;

template <typename Out, bool SPLIT, int TN>
__global__ void __launch_bounds__(kScaledThreads, 1) matmul_scaled_kernel(const __grid_constant__ CUtensorMap map_w,
                                                                          const __grid_constant__ CUtensorMap map_x,
                                                                          const __grid_constant__ CUtensorMap map_o, const MatmulArgs g) {
  using C = ScaledRows<TN>;
  constexpr int kWords = TN / 32;  // groups of 32 weight rows
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t s_full[C::kStages], s_empty[C::kStages], s_tfull[2], s_tempty[2], s_sfull[C::kGroups],
      s_sempty[C::kGroups];
  __shared__ uint32_t s_tmem;
  __shared__ int s_dead;
  const uint32_t stages = (ptx::smem_u32(smem_raw) + 1023) & ~1023u;
  const uint32_t outs = stages + C::kStages * C::kOperandBytes, scales = outs + C::kOutBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t half = ptx::cluster_rank() & 1, first_rank = SPLIT ? ptx::cluster_rank() - half : 0, split = first_rank >> 1;
  const uint32_t splits = SPLIT ? (uint32_t)g.splits : 1;
  const uint32_t pair = blockIdx.x / (2 * splits), pairs = gridDim.x / (2 * splits);  // (SPLIT: a cluster's pairs have one tile)
  const int kb_first = SPLIT ? (int)split * g.per : 0, nkb = SPLIT ? min(g.KB - kb_first, g.per) : g.KB;
  const uint16_t both = (uint16_t)(3u << first_rank);
  const uint32_t tiles_n = (uint32_t)(g.N + C::kTileN - 1) / C::kTileN, tiles_m = (uint32_t)((g.M + 255) / 256), tiles = tiles_n * tiles_m;
  if (warp == 0) {
    ptx::prefetch_tensormap(&map_w);
    ptx::prefetch_tensormap(&map_x);
  } else if (warp == 1) {
    if (lane == 0) {
      for (int i = 0; i < C::kStages; ++i) {
        ptx::mbar_init(&s_full[i], 1);
        ptx::mbar_init(&s_empty[i], 1);
      }
      for (int i = 0; i < C::kGroups; ++i) {
        ptx::mbar_init(&s_sfull[i], 2);  // the scales in both CTAs
        ptx::mbar_init(&s_sempty[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        ptx::mbar_init(&s_tfull[i], 1);
        ptx::mbar_init(&s_tempty[i], 16);
      }
      ptx::mbar_fence_init();
      s_dead = 0;
    }
    __syncwarp();
    ptx::tmem_alloc_pair(&s_tmem, 512);
    ptx::tmem_relinquish_pair();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::cluster_sync();
  ptx::tc_fence_after();
  const uint32_t tmem = s_tmem;
  volatile int* dead = &s_dead;
  const auto wait = [&](uint64_t& bar, uint32_t parity, int code) {
    if (ptx::mbar_test_wait(&bar, parity)) return true;
    if (*dead) return false;
    if (ptx::mbar_wait(&bar, parity, g.status, code)) return true;
    *dead = 1;
    return false;
  };
  ptx::griddep_launch();
  ptx::griddep_wait();

  if (warp == 0 || warp == 2) {  // tokens, weights
    load_operand<C::kStages, C::kTileN, C::kOperandBytes>(warp == 0 ? &map_x : &map_w, stages + (warp == 0 ? 0 : 128 * 128), warp == 0,
                                                          warp == 0 ? 128 : C::kHalfN, s_full, s_empty, pair, pairs, tiles_n, tiles_m, kb_first,
                                                          nkb, g.status, wait);
  } else if (warp == 1) {
    if (half == 0) {
      // (The loop has to be shorter than a block's 384 cycles of products: four blocks unrolled, their barriers by address, and each
      // block's barrier looked at while the products of the one before are issued.)
      const uint32_t el = ptx::elect_one();
      constexpr uint32_t idesc = ptx::make_idesc_e4m3_scaled(256, C::kTileN);
      const uint32_t full = ptx::smem_u32(s_full), empty = ptx::smem_u32(s_empty);
      const ptx::DescHalves first = ptx::make_desc_halves_sw128(stages, 16, 1024);
      Ring<C::kStages> st;
      Ring<C::kGroups> group;
      Ring<2> buf;
      uint32_t last = 0, last_parity = 0;
      bool on = true, any = false;
      for (uint32_t t = pair; t < tiles && on; t += pairs, buf.step()) {
        if (!wait(s_tempty[buf.at], buf.parity ^ 1, kGiveUpTmemEmpty)) break;
        const uint32_t d = tmem + buf.at * C::kTileN;
        bool there = false;
        for (int kb0 = 0; kb0 < nkb && on; kb0 += C::kGroup, group.step()) {
          if (!wait(s_sfull[group.at], group.parity, kGiveUpFull)) {
            on = false;
            break;
          }
          ptx::tc_fence_after();
          const uint32_t sa = tmem + C::kTmemScales + group.at * C::kTmemScaleCols, sb = sa + 4, s = scales + group.at * C::kScaleBytes;
          ptx::tmem_copy_scales_pair_w(el, sa, s);
          ptx::tmem_copy_scales_pair_w(el, sb, s + 512);
          if constexpr (TN > 128) ptx::tmem_copy_scales_pair_w(el, sb + 4, s + 1024);
#pragma unroll
          for (uint32_t byte = 0; byte < C::kGroup; ++byte) {
            if (kb0 + (int)byte >= nkb) break;
            if (!there && !wait(s_full[st.at], st.parity, kGiveUpFull)) {
              on = false;
              break;
            }
            ptx::tc_fence_after();
            const ptx::DescHalves a = {first.lo + st.at * (C::kOperandBytes >> 4), first.hi}, b = {a.lo + (128 * 128 >> 4), first.hi};
            ptx::mma_mxf8_ss_x4_pair_w(el, d, a, b, idesc | (byte << 4) | (byte << 29), sa, sb, kb0 > 0 || byte > 0);
            ptx::mma_commit_pair_w(el, both, empty + 8 * st.at);
            last = st.at;
            last_parity = st.parity;
            any = true;
            st.step();
            there = ptx::mbar_test_wait_a(full + 8 * st.at, st.parity);
          }
          ptx::mma_commit_pair_w(el, both, ptx::smem_u32(&s_sempty[group.at]));
        }
        if (on) ptx::mma_commit_pair_w(el, both, ptx::smem_u32(&s_tfull[buf.at]));
      }
      if (any) ptx::mbar_wait(&s_empty[last], last_parity, g.status, kGiveUpDrain);
    }
  } else if (warp == 3) {
    // Word j of lane l: the scales of row 32 j + l over a group of blocks, a byte each.  Four words for this CTA's 128 tokens, and
    // those of the tile's weight rows, whose groups of 32 lie in one block of 128 each (lane j loads the word of rows 32 j).
    const uint8_t *sa = static_cast<const uint8_t*>(g.sa) + kb_first * g.sa_k, *sb = static_cast<const uint8_t*>(g.sb) + kb_first * g.sb_k;
    const auto words = [](const void* p, int64_t rows, int64_t k) {  // four blocks' scales are an aligned word
      return k == 1 && ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)rows) & 3) == 0;
    };
    const bool word_a = words(sa, g.sa_m, g.sa_k), word_b = words(sb, g.sb_n, g.sb_k);
    uint32_t t = pair;
    int kb = 0;
    const uint8_t *row[4], *weights;
    const auto settle = [&]() {  // where the scales of tile t lie
      const Tile at = tile_at<C::kTileN>(t < tiles ? t : pair, tiles_n, tiles_m);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t m = at.m0 + (int)half * 128 + 32 * j + lane;
        row[j] = t < tiles && m < g.M ? sa + m * g.sa_m : nullptr;
      }
      const int n = at.n0 + 32 * lane;
      weights = t < tiles && lane < kWords && n < g.N ? sb + (int64_t)(n / 128) * g.sb_n : nullptr;
    };
    const auto fetch = [&](const uint8_t* p, int64_t k, bool word, uint32_t (&v)[C::kGroup]) {  // (v[0] alone where it is a word)
      if (word && kb + C::kGroup <= nkb) {
        v[0] = p != nullptr ? *reinterpret_cast<const uint32_t*>(p + kb) : 0u;
      } else {
#pragma unroll
        for (int i = 0; i < C::kGroup; ++i) v[i] = p != nullptr && kb + i < nkb ? p[(kb + i) * k] : 0u;
      }
    };
    const auto joined = [&](const uint32_t (&v)[C::kGroup], bool word) { return word ? v[0] : v[0] | v[1] << 8 | v[2] << 16 | v[3] << 24; };
    uint32_t token[4][C::kGroup], weight[C::kGroup];
    const auto load = [&]() {
#pragma unroll
      for (int j = 0; j < 4; ++j) fetch(row[j], g.sa_k, word_a, token[j]);
      fetch(weights, g.sb_k, word_b, weight);
    };
    Ring<C::kGroups> group;
    settle();
    load();
    for (; t < tiles; group.step()) {
      const bool whole = kb + C::kGroup <= nkb;
      uint32_t w[4], v[8] = {};
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = joined(token[j], word_a && whole);
      const uint32_t mine = joined(weight, word_b && whole);
#pragma unroll
      for (int j = 0; j < kWords; ++j) v[j] = __shfl_sync(0xffffffffu, mine, j);
      kb += C::kGroup;
      if (kb >= nkb) {
        kb = 0;
        t += pairs;
        settle();
      }
      load();  // (the next group's, used a group later)
      wait(s_sempty[group.at], group.parity ^ 1, kGiveUpEmpty);
      __syncwarp();
      const uint32_t to = scales + group.at * C::kScaleBytes + lane * 16;
      const auto put = [](uint32_t p, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(p), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
      };
      put(to, w[0], w[1], w[2], w[3]);
      put(to + 512, v[0], v[1], v[2], v[3]);
      if constexpr (TN > 128) put(to + 1024, v[4], v[5], v[6], v[7]);
      ptx::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive_cluster(ptx::cluster_map(ptx::smem_u32(&s_sfull[group.at]), first_rank));
    }
  } else if (warp >= 4) {
    const int quad = warp & 3, group = (warp - 4) >> 2;
    const uint32_t at_tmem = tmem + ((uint32_t)quad << 21);
    OutRing ring = {outs + (group == 0 ? quad * 8192 : 4 * 8192 + quad * 4096), group == 0};
    Ring<2> buf;
    for (uint32_t t = pair; t < tiles; t += pairs, buf.step()) {
      const Tile at = tile_at<C::kTileN>(t, tiles_n, tiles_m);
      wait(s_tfull[buf.at], buf.parity, kGiveUpTmemFull);
      __syncwarp();
      ptx::tc_fence_after();
      const uint32_t from = at_tmem + buf.at * C::kTileN;
      const int y = at.m0 + (int)half * 128 + quad * 32;
      constexpr int kCols = 128 / sizeof(Out);
      if (group * kCols >= C::kTileN && lane == 0)  // (no columns for these warps)
        ptx::mbar_arrive_cluster(ptx::cluster_map(ptx::smem_u32(&s_tempty[buf.at]), first_rank));
#pragma unroll 1
      for (int c = group * kCols; c < C::kTileN; c += 2 * kCols) {
        uint32_t r[kCols];
        if constexpr (kCols == 64) ptx::tmem_ld64(from + c, r);
        else ptx::tmem_ld32(from + c, r);
        ptx::tmem_ld_wait();
        if (c + 2 * kCols >= C::kTileN) {
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive_cluster(ptx::cluster_map(ptx::smem_u32(&s_tempty[buf.at]), first_rank));
        }
        if (*dead) {
#pragma unroll
          for (int j = 0; j < kCols; ++j) r[j] = 0x7fffffffu;
        }
        if constexpr (SPLIT) {  // (the products that read the stages are finished)
#pragma unroll
          for (int j = 0; j < kCols; ++j)
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(stages + ((c + j) * 128 + quad * 32 + lane) * 4), "r"(r[j]) : "memory");
          continue;
        }
        if (y >= g.M || at.n0 + c >= g.N) continue;  // (the same for the whole warp: a store does not begin past the matrix)
        const uint32_t to = ring.next(lane);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t* v = r + k * (kCols / 8);
          if constexpr (sizeof(Out) == 2) {
            const auto two = [&](int i) { return ptx::pack_bf16(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])); };
            OutRing::put(to, lane, k, two(0), two(1), two(2), two(3));
          } else {
            OutRing::put(to, lane, k, v[0], v[1], v[2], v[3]);
          }
        }
        const int n = at.n0 + c;
        if (OutRing::whole(g, n, kCols)) OutRing::send(to, lane, &map_o, n, y);
        else OutRing::write(to, lane, static_cast<Out*>(g.out) + y * g.ld_out + n, g.ld_out, (int)min(g.M - y, (int64_t)32), g.N - n);
      }
    }
    if (lane == 0) ptx::tma_store_wait_all();
  }
  __syncwarp();
  if constexpr (SPLIT) {
    ptx::cluster_sync();
    add_splits<Out>(stages, outs + warp * 4096, splits, split, C::kTileN, half, (warp & 3) * 32 + lane, warp >> 2, kScaledThreads / 128,
                    tile_at<C::kTileN>(pair, tiles_n, tiles_m), g);
    __syncwarp();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::cluster_sync();  // neither CTA's memory goes while the other's products or barriers use it
  ptx::tc_fence_after();
  if (warp == 1) ptx::tmem_dealloc_pair(tmem, 512);
}

int encode_bytes(CUtensorMap* map, const void* base, int64_t rows, int64_t width, int64_t ld, int box_rows) {
  const uint64_t dims[2] = {(uint64_t)width, (uint64_t)rows}, strides[1] = {(uint64_t)ld};
  const uint32_t box[2] = {128, (uint32_t)box_rows};
  return encode_sw128(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, 2, dims, strides, box);
}

template <auto k>
struct Kernel {
  static constexpr auto value = k;
};

template <typename Out, typename S>
int run_many(const void* a, int64_t ld_a, const void* b, int64_t ld_b, int K, MatmulArgs g, cudaStream_t s) {
  constexpr bool kScaled = sizeof(S) == 1;
  constexpr int kLongScaled = 40;  // blocks from which on four pairs may share a tile
  const int64_t pairs = device_sm_count() / 2;
  const auto tiles_of = [&](int width) { return (int64_t)((g.N + width - 1) / width) * ((g.M + 255) / 256); };
  // Narrow tiles where each has a pair of its own, unless K is long and four pairs can share a wide one (on this device 15 clusters of
  // eight CTAs are resident at once).  us, narrow / wide with one, two, four pairs a tile: 300 x 300 x 300 5.2 / 6.3, 9.3, 8.9; 550 x 768 x
  // 2496 7.1 / 8.8, 10.7, 9.9; 550 x 768 x 4096 8.8 / 11.4, 11.9, 10.6; 500 x 2048 x 7680 (22 wide tiles) 13.9 / 17.6, 16.1, -; 132 x 2048
  // x 7680 12.9 / 17.2, 14.8, 12.2; 256 x 1500 x 6000 14.8 / 20.3, 15.8, 12.2; 100 x 500 x 8000 17.5 / 19.4, 15.7, 12.0.
  int fours = 0;  // clusters of four pairs
  if constexpr (kScaled) {
    if (g.KB >= kLongScaled) {
      constexpr auto shared = matmul_scaled_kernel<Out, true, 192>;
      MVPA_CUDA_CHECK(grant_smem<shared>(ScaledRows<192>::kSmem));
      MVPA_CUDA_CHECK(resident_clusters<shared>(8, kScaledThreads, ScaledRows<192>::kSmem, &fours));
    }
  }
  const bool narrow = kScaled && 3 * tiles_of(192) <= pairs && tiles_of(192) > fours;
  const int kTileN = !kScaled ? 256 : narrow ? 64 : 192;
  const int64_t tiles = tiles_of(kTileN);
  if (tiles * g.KB > 0x7fffffff) {
    set_error("mvpa_matmul_fp8: more than 2^31 blocks of 256 x %d x 128", kTileN);
    return MVPA_ERR_UNSUPPORTED;
  }
  CUtensorMap map_w, map_x, map_o = {};
  int rc = encode_bytes(&map_w, b, g.N, K, ld_b, kTileN / 2);
  if (rc == MVPA_OK) rc = encode_bytes(&map_x, a, g.M, K, ld_a, 128);
  g.out_tma = (reinterpret_cast<uintptr_t>(g.out) & 15) == 0 && g.ld_out * (int64_t)sizeof(Out) % 16 == 0;
  if (g.out_tma && (int64_t)g.N * (int)sizeof(Out) % 16 == 0) g.out_tma = 2;
  if (rc == MVPA_OK && g.out_tma) {
    const uint64_t dims[2] = {(uint64_t)g.N, (uint64_t)g.M}, strides[1] = {(uint64_t)g.ld_out * sizeof(Out)};
    const uint32_t box[2] = {128 / sizeof(Out), 32};
    rc = encode_sw128(&map_o, sizeof(Out) == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, g.out, 2, dims, strides, box);
  }
  if (rc != MVPA_OK) return rc;
  const auto run = [&](auto whole, auto parts, int threads, size_t smem, int most4, int most2) {
    // Four or two pairs to a tile, as long as all clusters are resident at once (15 of eight CTAs, 33 of four).  us with 1 / 2 / 4 pairs:
    // scales that are powers of two, above and 550 x 2048 x 7680 (33 tiles) 18.0 / 16.7 / -; others, 300 x 300 x 300 (3 blocks) 6.5 /
    // 11.2 / 9.5, 550 x 768 x 2496 13.1 / 13.4 / 10.7, 132 x 2048 x 7680 30.6 / 21.4 / 15.2, 550 x 768 x 4096 18.5 / 15.8 / 12.0, 64 x
    // 8000 x 8000 (32 tiles) 32.5 / 22.3 / -.
    constexpr auto one = decltype(whole)::value, some = decltype(parts)::value;
    for (int n : {4, 2}) {
      int most = 0;
      if (g.splits > 1 || g.KB < (n == 4 ? most4 : most2)) continue;
      MVPA_CUDA_CHECK(grant_smem<some>(smem));
      MVPA_CUDA_CHECK(resident_clusters<some>(2 * n, threads, smem, &most));
      if (tiles <= most) g.splits = n;
    }
    g.per = (g.KB + g.splits - 1) / g.splits;
    if (g.splits > 1) {
      const dim3 grid(2 * (unsigned)tiles * g.splits);
      MVPA_CUDA_CHECK(launch_dependent(dim3(2 * g.splits), some, grid, threads, smem, s, map_w, map_x, map_o, g));
    } else {
      const dim3 grid(2 * (unsigned)(tiles < pairs ? tiles : pairs));
      MVPA_CUDA_CHECK(grant_smem<one>(smem));
      MVPA_CUDA_CHECK(launch_dependent(dim3(2), one, grid, threads, smem, s, map_w, map_x, map_o, g));
    }
    return MVPA_OK;
  };
  if constexpr (kScaled) {
    if (narrow) {
      constexpr auto kernel = matmul_scaled_kernel<Out, false, 64>;
      MVPA_CUDA_CHECK(grant_smem<kernel>(ScaledRows<64>::kSmem));
      MVPA_CUDA_CHECK(launch_dependent(dim3(2), kernel, dim3(2 * (unsigned)tiles), kScaledThreads, ScaledRows<64>::kSmem, s, map_w, map_x, map_o, g));
    } else {
      rc = run(Kernel<matmul_scaled_kernel<Out, false, 192>>(), Kernel<matmul_scaled_kernel<Out, true, 192>>(), kScaledThreads,
               ScaledRows<192>::kSmem, kLongScaled, 48);
    }
  } else {
    rc = run(Kernel<matmul_many_kernel<Out, S, false>>(), Kernel<matmul_many_kernel<Out, S, true>>(), kManyThreads, ManyRows::kSmem, 16, 24);
  }
  if (rc != MVPA_OK) return rc;
  count_launch();
  MVPA_CUDA_CHECK(cudaGetLastError());
  return MVPA_OK;
}

template <typename Out, typename S>
int run_matmul(const void* a, int64_t ld_a, const void* b, int64_t ld_b, int K, const MatmulArgs& g, cudaStream_t s) {
  // Up to 32 tokens the weights' bytes bound a product, which is what the kernel for few rows is made for.  us, few rows / pairs of
  // CTAs, e8m0 scales: 22 x 15360 x 2048 9.5 / 12.1, 32 x 15360 x 2048 10.4 / 12.0, 32 x 2048 x 7680 7.6 / 10.5, 32 x 768 x 2496 6.0 / 6.7,
  // 32 x 5000 x 2000 7.5 / 7.9, 32 x 4096 x 4096 6.9 / 9.3; where K is short the pairs catch up sooner (4736 x 768: 16 rows 5.1 / 5.6, 32
  // rows 7.1 / 5.6).  Its time grows with the columns that a thread adds up (one row 7.1, 16 rows 8.5, 32 rows 10.4 at 15360 x 2048), so
  // it ends there.
  if (g.M > 32) return run_many<Out, S>(a, ld_a, b, ld_b, K, g, s);
  const int nt = g.M <= 16 ? 16 : 32;
  CUtensorMap map_w, map_x;
  int rc = encode_bytes(&map_w, b, g.N, K, ld_b, 128);
  if (rc == MVPA_OK) rc = encode_bytes(&map_x, a, g.M, K, ld_a, nt);
  if (rc != MVPA_OK) return rc;
  return nt == 16 ? run_few<16, Out, S>(map_w, map_x, g, s) : run_few<32, Out, S>(map_w, map_x, g, s);
}

}  // namespace
}  // namespace mvpa

using namespace mvpa;

extern "C" int mvpa_matmul_fp8(const void* a, int64_t ld_a, const void* a_scales, int64_t a_stride_m, int64_t a_stride_k, const void* b,
                               int64_t ld_b, const void* b_scales, int64_t b_stride_n, int64_t b_stride_k, int32_t scale_dtype, void* out,
                               int64_t ld_out, int64_t M, int32_t N, int32_t K, int32_t out_dtype, int32_t* status, void* cuda_stream) {
  constexpr int kMost = 0x7fffffff - 1024;  // (the first place past the last tile is a 32-bit coordinate)
  if (M < 0 || N < 0 || K < 0 || M > kMost || N > kMost || K > kMost) {
    set_error("mvpa_matmul_fp8: M, N and K must not be negative, and at most %d (got %lld, %d, %d)", kMost, (long long)M, N, K);
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
  MatmulArgs g = {a_scales, b_scales, a_stride_m, a_stride_k, b_stride_n, b_stride_k, out, ld_out, M, N, (int)(((int64_t)K + 127) / 128), 0, 1, 0, status};
  if (out_dtype == MVPA_BF16)
    return scale_dtype == MVPA_E8M0 ? run_matmul<__nv_bfloat16, uint8_t>(a, ld_a, b, ld_b, K, g, s)
                                    : run_matmul<__nv_bfloat16, float>(a, ld_a, b, ld_b, K, g, s);
  return scale_dtype == MVPA_E8M0 ? run_matmul<float, uint8_t>(a, ld_a, b, ld_b, K, g, s)
                                  : run_matmul<float, float>(a, ld_a, b, ld_b, K, g, s);
}
