// out = x W^T, and silu(x Wg^T) * (x Wu^T), for weights in 4 bits (int4.cuh):
//
//   x W^T [m, n] = sum over groups k of scale[n, k] * sum_{j in k} x[m, j] (q[n, j] - zero[n, k])
//
// The whole numbers q - zero are exact in bf16, so the inner sums are products of bf16 on the tensor cores with fp32 sums, and a group's
// sum is scaled in fp32: no weight is rounded.  An fp32 x goes in as the three bf16 that it is the sum of.  Two kernels:
//   few     up to 8 tokens: a warp forms 16 weight rows x 8 tokens from registers alone
//   many    128 weight rows x up to 128 tokens a CTA: the weights are the product's M side, unpacked into TMEM on their way
#include <type_traits>

#include "int4.cuh"
#include "silu.cuh"
#include "tc_pairs.cuh"
#include "tc_tma_host.cuh"

namespace mvpa {

int check_int4(const char* what, int64_t N, int32_t K, int32_t group, int32_t scale_dtype, const mvpa_int4* w);

namespace {

struct Int4Args {
  Int4Weight w[2];
  const void* x;
  int64_t ld_x;
  void* out;
  int64_t ld_out, M;
  int N, K, group, groups, chunks;  // chunks of 128 along K
  int per, splits;                  // many: chunks of a split
  uint32_t tiles_m, tiles_n;
  int vec;                          // few: rows of x on 16-byte boundaries
  int* status;
};

constexpr int kChunk = 128;

template <typename T>
__device__ __forceinline__ float gate_of(float g, float u) {
  if constexpr (sizeof(T) == 4) return silu_mul_f32(g, u);
  else return Sigmoid(g).times(g, u);
}

// ---- few rows ---------------------------------------------------------------------------------------------------------------------------
// Bound by the weights' bytes.  A CTA has 16 weight rows, its warps every kWarps-th chunk of 128 columns; a lane's nibbles go through
// registers straight into the products of mma.sync (m16n8k16: with 8 tokens its rate is far above what the weights' arrival asks for, and
// nothing waits in shared memory).  Which columns stand at which place along K of a product is free as long as both operands agree:
// lane t of a row's four takes 16, 8 or 4 neighbouring bytes, so that all columns of one product lie in one group.
constexpr int kFewWarps = 8;

template <int G>
__device__ __forceinline__ int word_column(int t, int i) {  // the first column, in its chunk, of word i of lane t
  if constexpr (G == 128) return t * 32 + i * 8;
  else if constexpr (G == 64) return (i >> 1) * 64 + t * 16 + (i & 1) * 8;
  else return i * 32 + t * 8;
}

// Four words of a row's chunk; what lies past the row reads as zero.
template <int G>
__device__ __forceinline__ void load_words(const uint8_t* row, int chunk, int t, int bytes, uint32_t (&w)[4]) {
  const uint8_t* p = row + (int64_t)chunk * (kChunk / 2);
  if ((chunk + 1) * (int64_t)(kChunk / 2) <= bytes) {
    if constexpr (G == 128) {
      const uint4 v = *reinterpret_cast<const uint4*>(p + t * 16);
      w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else if constexpr (G == 64) {
      const uint2 a = *reinterpret_cast<const uint2*>(p + t * 8), b = *reinterpret_cast<const uint2*>(p + 32 + t * 8);
      w[0] = a.x; w[1] = a.y; w[2] = b.x; w[3] = b.y;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const uint32_t*>(p + i * 16 + t * 4);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = word_column<G>(t, i) / 2, left = bytes - chunk * (kChunk / 2) - at;
    w[i] = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b)
      if (b < left) w[i] |= (uint32_t)p[at + b] << (8 * b);
  }
}

// Eight neighbouring columns of a token as the right operand of two products, in the order of int4_pairs; in 16 bits, or in three parts.
template <typename T>
struct Columns {
  static constexpr int kParts = sizeof(T) == 4 ? 3 : 1;
  uint32_t b[kParts][4];
  __device__ __forceinline__ void load(const T* row, int64_t col, int K, bool any, bool vec) {
    constexpr int W = 8 * (int)sizeof(T) / 4;
    uint32_t v[W] = {};
    if (any && col < K) {
      if (vec && col + 8 <= K) {
#pragma unroll
        for (int i = 0; i < W; i += 4) {
          const uint4 r = *reinterpret_cast<const uint4*>(row + col + i * 4 / (int)sizeof(T));
          v[i] = r.x; v[i + 1] = r.y; v[i + 2] = r.z; v[i + 3] = r.w;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (col + e >= K) continue;
          if constexpr (sizeof(T) == 4) v[e] = reinterpret_cast<const uint32_t*>(row)[col + e];
          else v[e / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(row)[col + e] << (16 * (e & 1));
        }
      }
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const Thirds a(__uint_as_float(v[i])), c(__uint_as_float(v[i + 4]));
        b[0][i] = __byte_perm(a.hi, c.hi, 0x7632);
        b[kParts - 2][i] = __byte_perm(a.mid, c.mid, 0x7632);
        b[kParts - 1][i] = __byte_perm(a.lo, c.lo, 0x7632);
      }
    } else {
      b[0][0] = __byte_perm(v[0], v[2], 0x5410);
      b[0][1] = __byte_perm(v[0], v[2], 0x7632);
      b[0][2] = __byte_perm(v[1], v[3], 0x5410);
      b[0][3] = __byte_perm(v[1], v[3], 0x7632);
    }
  }
};

__device__ __forceinline__ void mma_16x8x16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <typename T, int G, int W>
__global__ void __launch_bounds__(kFewWarps * 32) int4_few_kernel(const Int4Args g) {
  constexpr int kGroups = kChunk / G;  // of a chunk
  __shared__ float s_sum[kFewWarps][W][128];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, t = lane & 3, token = lane >> 2;
  const int n0 = blockIdx.x * 16, bytes = (g.K + 1) / 2;
  const int row[2] = {min(n0 + (lane >> 2), g.N - 1), min(n0 + (lane >> 2) + 8, g.N - 1)};  // (rows past the last one are not written)
  const T* x = static_cast<const T*>(g.x) + (token < g.M ? token : 0) * g.ld_x;
  ptx::griddep_launch();
  ptx::griddep_wait();
  float acc[W][4] = {};
  uint32_t q[W][2][4];
  const auto fetch = [&](int c) {
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int r = 0; r < 2; ++r) load_words<G>(g.w[w].q + row[r] * g.w[w].ld_q, c, t, bytes, q[w][r]);
  };
  if (warp < g.chunks) fetch(warp);
#pragma unroll 1
  for (int c = warp; c < g.chunks; c += kFewWarps) {
    uint32_t now[W][2][4];
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) now[w][r][i] = q[w][r][i];
    if (c + kFewWarps < g.chunks) fetch(c + kFewWarps);
    float part[W][4];
    float scale[W][2];
    uint32_t minus[W][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // words; 4 / kGroups of them to a group
      constexpr int kEach = 4 / kGroups;
      const int group = c * kGroups + i / kEach;
      if (group >= g.groups) break;  // (the same for the whole warp)
      if (i % kEach == 0) {
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            scale[w][r] = g.w[w].scale(row[r], group);
            minus[w][r] = int4_minus(g.w[w].zero(row[r], group));
            part[w][r] = part[w][r + 2] = 0.f;
          }
      }
      Columns<T> b;
      b.load(x, (int64_t)c * kChunk + word_column<G>(t, i), g.K, token < g.M, g.vec);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        uint32_t a[2][4];
        int4_pairs(now[w][0][i], minus[w][0], a[0]);
        int4_pairs(now[w][1][i], minus[w][1], a[1]);
#pragma unroll
        for (int p = 0; p < Columns<T>::kParts; ++p) {
          mma_16x8x16(part[w], a[0][0], a[1][0], a[0][1], a[1][1], b.b[p][0], b.b[p][1]);
          mma_16x8x16(part[w], a[0][2], a[1][2], a[0][3], a[1][3], b.b[p][2], b.b[p][3]);
        }
        if (i % kEach == kEach - 1) {
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[w][j] = fmaf(scale[w][j / 2], part[w][j], acc[w][j]);
        }
      }
    }
  }
#pragma unroll
  for (int w = 0; w < W; ++w)
#pragma unroll
    for (int j = 0; j < 4; ++j) s_sum[warp][w][(lane & 3) * 2 * 16 + (j & 1) * 16 + (lane >> 2) + (j >> 1) * 8] = acc[w][j];  // [token][row]
  __syncthreads();
  if (threadIdx.x >= 128) return;
  const int m = threadIdx.x / 16, n = n0 + threadIdx.x % 16;
  if (m >= g.M || n >= g.N) return;
  float v[W];
#pragma unroll
  for (int w = 0; w < W; ++w) {
    v[w] = 0.f;
#pragma unroll
    for (int k = 0; k < kFewWarps; ++k) v[w] += s_sum[k][w][threadIdx.x];
  }
  static_cast<T*>(g.out)[m * g.ld_out + n] = from_f32<T>(W == 2 ? gate_of<T>(v[0], v[W - 1]) : v[0]);
}

// ---- many rows --------------------------------------------------------------------------------------------------------------------------
// 128 weight rows x NT tokens a CTA.  Warps: 0 loads a chunk of 128 columns of both operands (TMA), 2 to 5 unpack the weights, a row a
// thread, into TMEM, 1 issues a group's products, whose left operand is that part of TMEM, and the warps from 6 on fetch a group's sums,
// scale them and add them up in registers.  The CTAs are resident and take their tiles one after the other; few tiles: the chunks are
// split over the CTAs of a cluster, whose sums meet through distributed shared memory in a fixed order.
template <int NT, int W, int PARTS>
struct Many {
  static constexpr int kWBytes = 128 * 64, kXBytes = NT * 256;  // of a chunk: 128 rows x 64 bytes; two halves of NT rows x 128 bytes
  static constexpr int kStageBytes = PARTS * kXBytes + W * kWBytes;
  static constexpr bool kTwo = NT <= 32;  // two CTAs share a multiprocessor
  static constexpr int kBudget = (kTwo ? 100 : 208) * 1024;
  static constexpr int kStages = kBudget / kStageBytes < 8 ? kBudget / kStageBytes : 8;
  static constexpr int kSums = NT == 128 ? 2 : 4, kTmemA = kSums * NT;  // columns: groups' sums; two chunks of one weight
  static constexpr int kTmemCols = kTmemA + 128 > 256 ? 512 : 256;
  static constexpr int kAdders = NT >= 64 ? 8 : 4, kColumns = NT / (kAdders / 4);
  static constexpr int kThreads = (6 + kAdders) * 32;
  static constexpr size_t kSmem = 1024 + kStages * kStageBytes;
  static_assert(kStages >= 2 && W * NT * 128 * 4 <= kStages * kStageBytes, "the sums of a split wait in the stages' memory");
};

struct Int4Maps {
  CUtensorMap x, w[2];
};

enum : int { kGiveUpEmpty = 91, kGiveUpFull = 92, kGiveUpAEmpty = 93, kGiveUpAFull = 94, kGiveUpSumEmpty = 95, kGiveUpSumFull = 96, kGiveUpDrain = 97 };

__device__ __forceinline__ float peer_load(uint32_t at, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(ptx::cluster_map(at, rank)) : "memory");
  return v;
}

template <int NT, typename T, int W, bool SPLIT>
__global__ void __launch_bounds__((Many<NT, W, sizeof(T) == 4 ? 3 : 1>::kThreads), (NT <= 32 ? 2 : 1))
int4_many_kernel(const __grid_constant__ Int4Maps maps, const Int4Args g) {
  constexpr int PARTS = sizeof(T) == 4 ? 3 : 1;
  using C = Many<NT, W, PARTS>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t s_full[C::kStages], s_empty[C::kStages], s_afull[2], s_aempty[2], s_sfull[C::kSums], s_sempty[C::kSums];
  __shared__ uint32_t s_tmem;
  __shared__ int s_dead;  // a wait ran out: nothing waits any more, and the results are NaN
  const uint32_t stages = (ptx::smem_u32(smem_raw) + 1023) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t tiles = g.tiles_m * g.tiles_n;
  const int c0 = SPLIT ? (int)blockIdx.z * g.per : 0, nc = SPLIT ? min(g.chunks - c0, g.per) : g.chunks;
  const int each = kChunk / g.group;  // groups of a chunk
  if (warp == 0) {
    ptx::prefetch_tensormap(&maps.x);
    ptx::prefetch_tensormap(&maps.w[0]);
  } else if (warp == 1) {
    if (lane == 0) {
      for (int i = 0; i < C::kStages; ++i) {
        ptx::mbar_init(&s_full[i], 1);
        ptx::mbar_init(&s_empty[i], 1 + 4);  // the products that read x, and the four warps that read the weights
      }
      for (int i = 0; i < 2; ++i) {
        ptx::mbar_init(&s_afull[i], 4);
        ptx::mbar_init(&s_aempty[i], 1);
      }
      for (int i = 0; i < C::kSums; ++i) {
        ptx::mbar_init(&s_sfull[i], 1);
        ptx::mbar_init(&s_sempty[i], C::kAdders);
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

  if (warp == 0) {
    if (lane == 0) {
      Ring<C::kStages> st;
      uint32_t loads = 0;
      bool on = true;
      for (uint32_t t = blockIdx.x; t < tiles && on; t += gridDim.x) {
        const int m0 = (int)(t % g.tiles_m) * NT, n0 = (int)(t / g.tiles_m) * 128;
        for (int c = c0; c < c0 + nc; ++c, ++loads, st.step()) {
          if (!wait(s_empty[st.at], st.parity ^ 1, kGiveUpEmpty)) {
            on = false;
            break;
          }
          uint8_t* to = smem_raw + (stages - ptx::smem_u32(smem_raw)) + st.at * C::kStageBytes;
          ptx::mbar_arrive_expect_tx(&s_full[st.at], C::kStageBytes);
#pragma unroll
          for (int p = 0; p < PARTS; ++p)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              ptx::tma_load_3d(to + p * C::kXBytes + h * NT * 128, &maps.x, &s_full[st.at], c * kChunk + h * 64, m0, p);
#pragma unroll
          for (int w = 0; w < W; ++w) ptx::tma_load_2d(to + PARTS * C::kXBytes + w * C::kWBytes, &maps.w[w], &s_full[st.at], c * (kChunk / 2), n0);
        }
      }
      const uint32_t n = min(loads, (uint32_t)C::kStages);
      for (uint32_t k = loads - n; k != loads; ++k)  // no copy is in flight when the CTA ends
        if (!ptx::mbar_wait(&s_full[k % C::kStages], (k / C::kStages) & 1, g.status, kGiveUpDrain)) break;
    }
  } else if (warp == 1) {
    const uint32_t el = ptx::elect_one();
    constexpr uint32_t idesc = ptx::make_idesc_bf16(128, NT, 0);
    Ring<C::kStages> st;
    Ring<2> a;
    Ring<C::kSums> sum;
    uint32_t last = 0, last_parity = 0;
    bool on = true, any = false;
    for (uint32_t t = blockIdx.x; t < tiles && on; t += gridDim.x) {
      for (int c = c0; c < c0 + nc && on; ++c, st.step()) {
        if (!wait(s_full[st.at], st.parity, kGiveUpFull)) {
          on = false;
          break;
        }
        const ptx::DescHalves x = ptx::make_desc_halves_sw128(stages + st.at * C::kStageBytes, 16, 1024);
        const int here = min(each, g.groups - c * each);
        for (int w = 0; w < W && on; ++w, a.step()) {
          if (!wait(s_afull[a.at], a.parity, kGiveUpAFull)) {
            on = false;
            break;
          }
          for (int k = 0; k < here; ++k, sum.step()) {
            if (!wait(s_sempty[sum.at], sum.parity ^ 1, kGiveUpSumEmpty)) {
              on = false;
              break;
            }
            ptx::tc_fence_after();
            for (int s = k * (g.group / 16); s < (k + 1) * (g.group / 16); ++s) {  // steps of 16 columns
#pragma unroll
              for (int p = 0; p < PARTS; ++p)
                ptx::mma_ts_w(el, tmem + sum.at * NT, tmem + C::kTmemA + a.at * 64 + s * 8, x, p * C::kXBytes + (s >> 2) * NT * 128 + (s & 3) * 32,
                              idesc, s > k * (g.group / 16) || p > 0);
            }
            ptx::mma_commit_w(el, ptx::smem_u32(&s_sfull[sum.at]));
          }
          ptx::mma_commit_w(el, ptx::smem_u32(&s_aempty[a.at]));
        }
        if (!on) break;
        ptx::mma_commit_w(el, ptx::smem_u32(&s_empty[st.at]));
        last = st.at;
        last_parity = st.parity;
        any = true;
      }
    }
    if (any) ptx::mbar_wait(&s_empty[last], last_parity, g.status, kGiveUpDrain);
  } else if (warp < 6) {
    const int quad = warp & 3, row = quad * 32 + lane;  // a warp reaches the TMEM lanes of its place among four
    const uint32_t at_tmem = tmem + C::kTmemA + ((uint32_t)quad << 21);
    Ring<C::kStages> st;
    Ring<2> a;
    for (uint32_t t = blockIdx.x; t < tiles; t += gridDim.x) {
      const int n = min((int)(t / g.tiles_m) * 128 + row, g.N - 1);
      const auto zeros_of = [&](int c, uint32_t (&z)[W]) {  // a chunk's, a byte each
#pragma unroll
        for (int w = 0; w < W; ++w) {
          z[w] = 0x08080808u;
          if (g.w[w].zeros == nullptr) continue;
          z[w] = 0;
          for (int k = 0; k < each; ++k)
            if (c < c0 + nc && c * each + k < g.groups) z[w] |= (uint32_t)g.w[w].zeros[n * g.w[w].ld_z + c * each + k] << (8 * k);
        }
      };
      uint32_t next[W];
      zeros_of(c0, next);
      for (int c = c0; c < c0 + nc; ++c, st.step()) {
        uint32_t zeros[W];
#pragma unroll
        for (int w = 0; w < W; ++w) zeros[w] = next[w];
        zeros_of(c + 1, next);
        wait(s_full[st.at], st.parity, kGiveUpFull);
        const uint32_t tile = stages + st.at * C::kStageBytes + PARTS * C::kXBytes;
#pragma unroll
        for (int w = 0; w < W; ++w, a.step()) {
          wait(s_aempty[a.at], a.parity ^ 1, kGiveUpAEmpty);
          __syncwarp();
          ptx::tc_fence_after();
          uint32_t r[32];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int piece = 0; piece < 2; ++piece) {
              const int i = half * 2 + piece;
              uint32_t v[4];
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                           : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                           : "r"(tile + w * C::kWBytes + row * 64 + ((i ^ ((row >> 1) & 3)) << 4)));
              const uint32_t minus = int4_minus((zeros[w] >> (8 * (i * 32 / g.group))) & 255u);
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                uint32_t p[4];
                int4_pairs(v[j], minus, p);
                uint32_t* o = r + piece * 16 + j * 4;
                o[0] = __byte_perm(p[0], p[1], 0x5410);
                o[1] = __byte_perm(p[2], p[3], 0x5410);
                o[2] = __byte_perm(p[0], p[1], 0x7632);
                o[3] = __byte_perm(p[2], p[3], 0x7632);
              }
            }
            ptx::tmem_st32(at_tmem + a.at * 64 + half * 32, r);
          }
          ptx::tmem_st_wait();
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            ptx::mbar_arrive(&s_afull[a.at]);
            if (w == W - 1) ptx::mbar_arrive(&s_empty[st.at]);
          }
        }
      }
    }
  } else {
    const int quad = warp & 3, first = ((warp - 6) >> 2) * C::kColumns, row = quad * 32 + lane;
    const uint32_t at_tmem = tmem + ((uint32_t)quad << 21) + first;
    Ring<C::kSums> sum;
    for (uint32_t t = blockIdx.x; t < tiles; t += gridDim.x) {
      const int m0 = (int)(t % g.tiles_m) * NT, n0 = (int)(t / g.tiles_m) * 128, n = min(n0 + row, g.N - 1);
      float acc[W][C::kColumns];
#pragma unroll
      for (int w = 0; w < W; ++w)
#pragma unroll
        for (int j = 0; j < C::kColumns; ++j) acc[w][j] = 0.f;
      float next[W][4];
      const auto scales_of = [&](int c) {
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
          for (int k = 0; k < 4; ++k) next[w][k] = k < each && c < c0 + nc && c * each + k < g.groups ? g.w[w].scale(n, c * each + k) : 0.f;
      };
      scales_of(c0);
      for (int c = c0; c < c0 + nc; ++c) {
        float scale[W][4];
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
          for (int k = 0; k < 4; ++k) scale[w][k] = next[w][k];
        scales_of(c + 1);
        const int here = min(each, g.groups - c * each);
#pragma unroll
        for (int w = 0; w < W; ++w) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (k >= here) break;
            wait(s_sfull[sum.at], sum.parity, kGiveUpSumFull);
            __syncwarp();
            ptx::tc_fence_after();
            constexpr int P = C::kColumns < 32 ? 16 : 32;
#pragma unroll
            for (int j0 = 0; j0 < C::kColumns; j0 += P) {
              uint32_t r[P];
              if constexpr (P == 32) ptx::tmem_ld32(at_tmem + sum.at * NT + j0, r);
              else ptx::tmem_ld16(at_tmem + sum.at * NT + j0, r);
              ptx::tmem_ld_wait();
              if (j0 + P == C::kColumns) {
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&s_sempty[sum.at]);
              }
#pragma unroll
              for (int j = 0; j < P; ++j) acc[w][j0 + j] = fmaf(__uint_as_float(r[j]), scale[w][k], acc[w][j0 + j]);
            }
            sum.step();
          }
        }
      }
      const float poison = *dead ? __uint_as_float(0x7fffffffu) : 0.f;
      if constexpr (SPLIT) {  // (every product that read the stages is finished)
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
          for (int j = 0; j < C::kColumns; ++j)
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(stages + ((w * NT + first + j) * 128 + row) * 4), "f"(acc[w][j] + poison) : "memory");
      } else if (n0 + row < g.N) {
        T* out = static_cast<T*>(g.out) + (int64_t)(m0 + first) * g.ld_out + n0 + row;
#pragma unroll
        for (int j = 0; j < C::kColumns; ++j)
          if (m0 + first + j < g.M) out[j * g.ld_out] = from_f32<T>((W == 2 ? gate_of<T>(acc[0][j], acc[W - 1][j]) : acc[0][j]) + poison);
      }
    }
  }
  if constexpr (SPLIT) {
    __syncwarp();
    ptx::cluster_sync();
    const int m0 = (int)(blockIdx.x % g.tiles_m) * NT, n0 = (int)(blockIdx.x / g.tiles_m) * 128, splits = g.splits;
    for (int i = threadIdx.x; i < NT * 128; i += C::kThreads) {
      const int j = i >> 7, row = i & 127;
      if (j % splits != (int)blockIdx.z || m0 + j >= g.M || n0 + row >= g.N) continue;
      float v[W] = {};
      for (int z = 0; z < splits; ++z)
#pragma unroll
        for (int w = 0; w < W; ++w) v[w] += peer_load(stages + ((w * NT + j) * 128 + row) * 4, z);
      static_cast<T*>(g.out)[(int64_t)(m0 + j) * g.ld_out + n0 + row] = from_f32<T>(W == 2 ? gate_of<T>(v[0], v[W - 1]) : v[0]);
    }
    __syncwarp();
    ptx::cluster_sync();  // nobody's memory goes while it is read
  }
  __syncwarp();
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  if (warp == 1) ptx::tmem_dealloc(tmem, C::kTmemCols);
}

// x as the TMA can read it: bf16 with rows on 16-byte boundaries, an fp32 one in its three parts, a matrix each.
template <typename T>
__global__ void __launch_bounds__(256) int4_lay_out_kernel(const T* __restrict__ x, int64_t ld_x, uint16_t* __restrict__ to, int64_t ld, int64_t M, int K) {
  ptx::griddep_launch();
  ptx::griddep_wait();
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < M * ld; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i / ld, col = i - row * ld;
    if constexpr (sizeof(T) == 4) {
      const Thirds v(col < K ? x[row * ld_x + col] : 0.f);
      to[i] = (uint16_t)(v.hi >> 16);
      to[i + M * ld] = (uint16_t)(v.mid >> 16);
      to[i + 2 * M * ld] = (uint16_t)(v.lo >> 16);
    } else {
      to[i] = col < K ? reinterpret_cast<const uint16_t*>(x)[row * ld_x + col] : (uint16_t)0;
    }
  }
}

constexpr int kFewTokens = 8;

bool in_place(const void* x, int64_t ld_x, int32_t dtype) {
  return dtype == MVPA_BF16 && (reinterpret_cast<uintptr_t>(x) & 15) == 0 && ld_x % 8 == 0;
}

template <int NT, typename T, int W>
int run_many(const void* x, int64_t ld_x, int64_t plane, Int4Args g, cudaStream_t s) {
  constexpr int PARTS = sizeof(T) == 4 ? 3 : 1;
  using C = Many<NT, W, PARTS>;
  Int4Maps maps;
  {
    const uint64_t dims[3] = {(uint64_t)g.K, (uint64_t)g.M, (uint64_t)PARTS}, strides[2] = {(uint64_t)ld_x * 2, (uint64_t)plane * 2};
    const uint32_t box[3] = {64, NT, 1};
    const int rc = encode_bf16_sw128(&maps.x, x, 3, dims, strides, box);
    if (rc != MVPA_OK) return rc;
  }
  for (int w = 0; w < W; ++w) {
    const uint64_t dims[2] = {(uint64_t)(g.K + 1) / 2, (uint64_t)g.N}, strides[1] = {(uint64_t)g.w[w].ld_q};
    const uint32_t box[2] = {64, 128};
    const int rc = encode_sw128(&maps.w[w], CU_TENSOR_MAP_DATA_TYPE_UINT8, g.w[w].q, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_64B);
    if (rc != MVPA_OK) return rc;
  }
  const int64_t tm = (g.M + NT - 1) / NT, tn = (g.N + 127) / 128, tiles = tm * tn, room = (int64_t)device_sm_count() * (C::kTwo ? 2 : 1);
  if (tiles * g.chunks > 0x7fffffff) {
    set_error("mvpa_matmul_int4: more than 2^31 blocks of 128 x %d x 128", NT);
    return MVPA_ERR_UNSUPPORTED;
  }
  g.tiles_m = (uint32_t)tm;
  g.tiles_n = (uint32_t)tn;
  int splits = 1;
  while (splits < 8 && tiles * splits * 2 <= room && g.chunks >= 4 * splits) splits *= 2;
  g.per = (g.chunks + splits - 1) / splits;
  g.splits = (g.chunks + g.per - 1) / g.per;
  if (g.splits > 1) {
    constexpr auto kernel = int4_many_kernel<NT, T, W, true>;
    MVPA_CUDA_CHECK(grant_smem<kernel>(C::kSmem));
    MVPA_CUDA_CHECK(launch_dependent(g.splits, kernel, dim3((unsigned)tiles, 1, g.splits), C::kThreads, C::kSmem, s, maps, g));
  } else {
    constexpr auto kernel = int4_many_kernel<NT, T, W, false>;
    MVPA_CUDA_CHECK(grant_smem<kernel>(C::kSmem));
    MVPA_CUDA_CHECK(launch_dependent(1, kernel, (unsigned)(tiles < room ? tiles : room), C::kThreads, C::kSmem, s, maps, g));
  }
  count_launch();
  MVPA_CUDA_CHECK(cudaGetLastError());
  return MVPA_OK;
}

template <typename T, int W>
int run_few(const Int4Args& g, cudaStream_t s) {
  const unsigned grid = (unsigned)((g.N + 15) / 16);
  const auto kernel = g.group == 128 ? int4_few_kernel<T, 128, W> : g.group == 64 ? int4_few_kernel<T, 64, W> : int4_few_kernel<T, 32, W>;
  MVPA_CUDA_CHECK(launch_dependent(1, kernel, grid, kFewWarps * 32, 0, s, g));
  count_launch();
  MVPA_CUDA_CHECK(cudaGetLastError());
  return MVPA_OK;
}

template <typename T, int W>
int run_int4(Int4Args g, int32_t dtype, void* workspace, cudaStream_t s) {
  if (g.M <= kFewTokens) return run_few<T, W>(g, s);
  const void* x = g.x;
  int64_t ld = g.ld_x, plane = g.ld_x * 8;  // (one part: the stride between parts is never used)
  if (!in_place(g.x, g.ld_x, dtype)) {
    ld = (g.K + 7) / 8 * 8;
    plane = g.M * ld;
    const int64_t ctas = (plane + 255) / 256, most = (int64_t)device_sm_count() * 16;
    MVPA_CUDA_CHECK(launch_dependent(1, int4_lay_out_kernel<T>, (unsigned)(ctas < most ? ctas : most), 256, 0, s, (const T*)g.x, g.ld_x,
                                     (uint16_t*)workspace, ld, g.M, g.K));
    count_launch();
    MVPA_CUDA_CHECK(cudaGetLastError());
    x = workspace;
  }
  if (g.M <= 16) return run_many<16, T, W>(x, ld, plane, g, s);
  if (g.M <= 32) return run_many<32, T, W>(x, ld, plane, g, s);
  if constexpr (sizeof(T) == 2 && W == 1)
    if (g.M > 64) return run_many<128, T, W>(x, ld, plane, g, s);
  return run_many<64, T, W>(x, ld, plane, g, s);
}

}  // namespace
}  // namespace mvpa

using namespace mvpa;

extern "C" size_t mvpa_matmul_int4_workspace_bytes(const void* x, int64_t ld_x, int64_t M, int32_t K, int32_t dtype) {
  if (M <= kFewTokens || K <= 0 || in_place(x, ld_x, dtype)) return 0;
  return (size_t)M * (((size_t)K + 7) / 8 * 8) * 2 * (dtype == MVPA_F32 ? 3 : 1);
}

extern "C" int mvpa_matmul_int4(const void* x, int64_t ld_x, const mvpa_int4* w, const mvpa_int4* up, int32_t scale_dtype, void* out,
                                int64_t ld_out, int64_t M, int32_t N, int32_t K, int32_t group, int32_t dtype, void* workspace,
                                size_t workspace_bytes, int32_t* status, void* cuda_stream) {
  const char* what = "mvpa_matmul_int4";
  int rc = check_int4(what, N, K, group, scale_dtype, w);
  if (rc == MVPA_OK && up != nullptr) rc = check_int4(what, N, K, group, scale_dtype, up);
  if (rc != MVPA_OK) return rc;
  if (M < 0 || M > 0x7fffffff - 1024) {
    set_error("%s: M must not be negative, and at most 2^31 - 1025 (got %lld)", what, (long long)M);
    return MVPA_ERR_SHAPE;
  }
  if (dtype != MVPA_F32 && dtype != MVPA_BF16) {
    set_error("%s: x and out are MVPA_F32 or MVPA_BF16", what);
    return MVPA_ERR_DTYPE;
  }
  if (M == 0 || N == 0) return MVPA_OK;
  const int es = dtype == MVPA_F32 ? 4 : 2;
  if (out == nullptr || ld_out < N || (reinterpret_cast<uintptr_t>(out) & (es - 1)) != 0) {
    set_error("%s: out is NULL, not aligned to its elements, or its leading dimension is below N", what);
    return MVPA_ERR_ALIGNMENT;
  }
  cudaStream_t s = (cudaStream_t)cuda_stream;
  if (K == 0) {  // sums of nothing
    MVPA_CUDA_CHECK(cudaMemset2DAsync(out, (size_t)ld_out * es, 0, (size_t)N * es, (size_t)M, s));
    return MVPA_OK;
  }
  if (x == nullptr || ld_x < K || (reinterpret_cast<uintptr_t>(x) & (es - 1)) != 0) {
    set_error("%s: x is NULL, not aligned to its elements, or its leading dimension is below K", what);
    return MVPA_ERR_ALIGNMENT;
  }
  const size_t need = mvpa_matmul_int4_workspace_bytes(x, ld_x, M, K, dtype);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0)) {
    set_error("%s: needs a workspace of %zu bytes on a 16-byte boundary", what, need);
    return MVPA_ERR_WORKSPACE;
  }
  Int4Args g = {};
  const mvpa_int4* given[2] = {w, up};
  for (int i = 0; i < 2; ++i)
    if (given[i] != nullptr)
      g.w[i] = {(const uint8_t*)given[i]->q, given[i]->scales, (const uint8_t*)given[i]->zeros, given[i]->ld_q, given[i]->ld_s, given[i]->ld_z,
                scale_dtype == MVPA_F32};
  g.x = x;
  g.ld_x = ld_x;
  g.out = out;
  g.ld_out = ld_out;
  g.M = M;
  g.N = N;
  g.K = K;
  g.group = group;
  g.groups = (K + group - 1) / group;
  g.chunks = (K + kChunk - 1) / kChunk;
  g.vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && ld_x * es % 16 == 0;
  g.status = status;
  if (dtype == MVPA_F32) return up != nullptr ? run_int4<float, 2>(g, dtype, workspace, s) : run_int4<float, 1>(g, dtype, workspace, s);
  return up != nullptr ? run_int4<__nv_bfloat16, 2>(g, dtype, workspace, s) : run_int4<__nv_bfloat16, 1>(g, dtype, workspace, s);
}
