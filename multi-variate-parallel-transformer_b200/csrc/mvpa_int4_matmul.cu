// out = x W^T, and silu(x Wg^T) * (x Wu^T), for weights in 4 bits (int4.cuh):
//
//   x W^T [m, n] = sum over groups k of scale[n, k] * sum_{j in k} x[m, j] (q[n, j] - zero[n, k])
//
// The whole numbers q - zero are exact in bf16, so the inner sums are products of bf16 on the tensor cores with fp32 sums, and a group's
// sum is scaled in fp32: no weight is rounded.  (2^-11 of them, that is, up to the last step: see int4_pairs.)  An fp32 x goes in as the three bf16 that it is the sum of.  Two kernels:
//   few     up to 16 tokens: a warp forms 2 x 16 weight rows x 8 or 16 tokens from registers
//   many    128 weight rows x up to 256 tokens a CTA: the weights are the product's M side, unpacked into TMEM on their way
#include <algorithm>
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
  int per, splits;                  // chunks of a split
  uint32_t tiles_m, tiles_n;
  int64_t plane;                    // few: elements between the parts of x
  int* status;
};

constexpr int kChunk = 128;

// A result of its sums (a gate's two), 2^-11 of them up to here.
template <typename T, int W>
__device__ __forceinline__ T result_of(const float (&v)[W]) {
  const float g = v[0] * kInt4Unit;
  if constexpr (W == 1) return from_f32<T>(g);
  else if constexpr (sizeof(T) == 4) return from_f32<T>(silu_mul_f32(g, v[1] * kInt4Unit));
  else return from_f32<T>(Sigmoid(g).times(g, v[1] * kInt4Unit));
}

__device__ __forceinline__ float peer_load(uint32_t at, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(ptx::cluster_map(at, rank)) : "memory");
  return v;
}

// ---- few rows ---------------------------------------------------------------------------------------------------------------------------
// Bound by the weights' bytes, and next to that by the instructions that unpack them.  A warp forms 16 weight rows x all tokens over a
// chunk of 128 columns at a time, with mma.sync (m16n8k16: with these few tokens its rate is far above what the weights' arrival asks
// for, and the unpacked weights never leave the registers).  Which columns stand at which place along K of a product is free as long as
// both operands agree: lane t of a row's four takes 16, 8 or 4 neighbouring bytes, so that all columns of one product lie in one group.
//
// A CTA's eight warps are WR stretches of 16 rows x WK chunks side by side.  Weights and tokens come by cp.async, kDepth - 1 turns ahead:
// what hides the memory's latency is bytes on their way, and those that wait in registers cost warps.  The scales of a CTA's rows are
// loaded once.  A long K is split over the CTAs of a cluster, whose sums meet through distributed shared memory in a fixed order.
constexpr int kFewWarps = 8;

// 16 bytes to shared memory, of which the first `bytes` come from memory and the others are zeros.
__device__ __forceinline__ void copy16(uint32_t to, const void* from, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
template <int N>
__device__ __forceinline__ void load_shared(uint32_t at, uint32_t* v) {
  if constexpr (N == 4) asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at) : "memory");
  else if constexpr (N == 2) asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(at) : "memory");
  else asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v[0]) : "r"(at) : "memory");
}

__device__ __forceinline__ void mma_16x8x16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Each warp has two sets of 16 weight rows: a gate's two weights (W = 2), or two stretches of one.
template <int W, int NT, int PARTS>
struct Few {
  static constexpr int WR = 2, WK = kFewWarps / WR, kTokens = NT * 8, kRows = WR * 16;  // (of a set)
  static constexpr int kDepth = 3;
  static constexpr int kXBytes = WK * PARTS * kTokens * 256, kWBytes = kFewWarps * 2 * 1024;  // [wk][part][token]; [warp][set][row]
  static constexpr int kStageBytes = kXBytes + kWBytes;
  static constexpr int kSums = 2 * kTokens * kRows, kSumBytes = WK * kSums * 4;               // wait in the stages' memory
  static constexpr int kBytes = kDepth * kStageBytes > kSumBytes ? kDepth * kStageBytes : kSumBytes;
  static constexpr int kLeft = 220 * 1024 - kBytes, kMostScales = (kLeft < 48 * 1024 ? kLeft : 48 * 1024) / 8;  // of a CTA's rows, eight bytes each
};

// Where piece `p` (16 bytes) of token `m`'s row of a chunk lies: pieces change places so that the lanes of a load of 16 bytes, two tokens
// and the four words of a row that they read together, meet no bank twice.
template <int G>
__device__ __forceinline__ int token_piece(int m, int p) {
  return G == 128 ? p ^ ((p >> 3) & 1) ^ ((m & 1) << 1) : G == 64 ? p ^ (m & 1) : p ^ ((m & 1) << 2);
}

template <typename T, int G, int W, int NT, int PARTS>
__global__ void __launch_bounds__(kFewWarps * 32) int4_few_kernel(const Int4Args g) {
  using C = Few<W, NT, PARTS>;
  constexpr int kThreads = kFewWarps * 32;
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t base = ptx::smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, t = lane & 3, line = lane >> 2;
  const int wr = warp % C::WR, wk = warp / C::WR;
  const int n0 = blockIdx.x * C::kRows * (W == 1 ? 2 : 1), bytes = (g.K + 1) / 2;
  const auto row_of = [&](int s, int row) { return (int64_t)min(n0 + (W == 1 ? s * C::kRows : 0) + row, g.N - 1); };  // (past the last: not written)
  const int c0 = (int)blockIdx.z * g.per, nc = min(g.chunks - c0, g.per), turns = (nc + C::WK - 1) / C::WK;
  ptx::griddep_launch();
  ptx::griddep_wait();

  // What a thread brings each turn (WK chunks): two pieces of 16 bytes of each set of its warp's weight rows, and pieces of the tokens' rows.
  const int whole = min((g.K >> 7) - c0, nc) / C::WK;  // turns whose columns all exist
  const uint8_t* w_from[2][2];
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const Int4Weight& w = g.w[W == 2 ? s : 0];
      w_from[s][r] = w.q + row_of(s, wr * 16 + r * 8 + line) * w.ld_q + (c0 + wk) * (int64_t)(kChunk / 2) + t * 16;
    }
  const uint32_t w_to = base + C::kXBytes + warp * 2048 + line * 64 + ((t ^ ((line >> 1) & 3)) << 4);  // (in the order of a 64-byte swizzle)
  const auto fetch_w = [&](int turn, uint32_t to) {
    if (turn >= turns) return;
    const int left = turn < whole ? 16 : max(0, min(16, min(bytes, (c0 + nc) * (kChunk / 2)) - (c0 + turn * C::WK + wk) * (kChunk / 2) - t * 16));
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        copy16(w_to + s * 1024 + r * 512 + to, left > 0 ? w_from[s][r] : g.w[0].q, left);
        w_from[s][r] += C::WK * (kChunk / 2);
      }
  };
  // (Rows of tokens that do not exist stay as they are: a token's sums are its own.)
  constexpr int kMine = C::kXBytes / 16 / kThreads;
  static_assert(C::kXBytes / 16 % kThreads == 0, "");
  const int p = threadIdx.x & 15;
  const uint8_t* x_from[kMine];
  uint32_t x_to[kMine];
  const auto fetch_x = [&](int turn, uint32_t to) {
    if (turn >= turns) return;
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      if (x_from[j] == nullptr) continue;
      const int k = c0 + turn * C::WK + ((threadIdx.x >> 4) + j * (kThreads / 16)) / C::kTokens / PARTS;
      const int left = turn < whole ? 8 : max(0, min(8, min(g.K, (c0 + nc) * kChunk) - k * kChunk - p * 8));
      copy16(x_to[j] + to, left > 0 ? x_from[j] : static_cast<const uint8_t*>(g.x), left * 2);
      x_from[j] += C::WK * kChunk * 2;
    }
  };
#pragma unroll 1
  for (int i = 0; i < C::kDepth - 1; ++i) fetch_w(i, i * C::kStageBytes);  // (the weights first: everything else can hide behind them)
#pragma unroll
  for (int j = 0; j < kMine; ++j) {
    const int row = (threadIdx.x >> 4) + j * (kThreads / 16), m = row % C::kTokens, part = row / C::kTokens % PARTS, k = row / C::kTokens / PARTS;
    x_from[j] = m < g.M ? static_cast<const uint8_t*>(g.x) + (part * g.plane + m * g.ld_x + (int64_t)(c0 + k) * kChunk + p * 8) * 2 : nullptr;
    x_to[j] = base + row * 256 + token_piece<G>(m, p) * 16;
  }
#pragma unroll 1
  for (int i = 0; i < C::kDepth - 1; ++i) {
    fetch_x(i, i * C::kStageBytes);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }

  // The scales of the CTA's rows over its chunks, and what their zeros ask to be taken from a nibble: [set][row][group].  Four loads of a
  // thread at once: one after the other they take longer than everything else.
  constexpr int kGroups = kChunk / G, kEach = 4 / kGroups;  // groups of a chunk, words of a group
  const int g0 = c0 * kGroups, ng = min(g.groups - g0, nc * kGroups);
  const uint32_t s_scale = base + C::kBytes;
  {
    constexpr int kAtOnce = 4, kSide = kThreads > 2 * C::kRows ? kThreads / (2 * C::kRows) : 1;  // threads of a row
#pragma unroll 1
    for (int row = threadIdx.x / kSide; row < 2 * C::kRows; row += kThreads / kSide) {
      const Int4Weight& w = g.w[W == 2 ? row / C::kRows : 0];
      const int64_t n = row_of(row / C::kRows, row % C::kRows);
#pragma unroll 1
      for (int k0 = threadIdx.x % kSide; k0 < ng; k0 += kAtOnce * kSide) {
        float scale[kAtOnce];
        uint32_t zero[kAtOnce];
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
          const int k = g0 + min(k0 + j * kSide, ng - 1);
          scale[j] = w.scale(n, k);
          zero[j] = w.zero(n, k);
        }
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j)
          if (k0 + j * kSide < ng)
            asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(s_scale + (row * ng + k0 + j * kSide) * 8), "f"(scale[j]), "r"(int4_minus(zero[j])) : "memory");
      }
    }
  }

  // Lane t's word i of a row's chunk is word (i of t's four), (of t's two in half i / 2) or (t of the four in quarter i).
  uint32_t x_at[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int word = G == 128 ? t * 4 + i : G == 64 ? (i >> 1) * 8 + t * 2 + (i & 1) : i * 4 + t;
    x_at[i] = base + (wk * PARTS * C::kTokens + line) * 256 + token_piece<G>(line, word) * 16;
  }
  const uint32_t w_at = base + C::kXBytes + warp * 2048 + line * 64, turned = (line >> 1) & 3;
  uint32_t my_scale[2][2];  // [set][row]
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int r = 0; r < 2; ++r) my_scale[s][r] = s_scale + (s * C::kRows + wr * 16 + r * 8 + line) * ng * 8;
  float acc[2][NT][4] = {};
  uint32_t from = 0;
#pragma unroll 1
  for (int turn = 0; turn < turns; ++turn) {
    asm volatile("cp.async.wait_group %0;" ::"n"(C::kDepth - 2) : "memory");
    __syncthreads();
    {
      const uint32_t to = from == 0 ? (C::kDepth - 1) * C::kStageBytes : from - C::kStageBytes;
      fetch_w(turn + C::kDepth - 1, to);
      fetch_x(turn + C::kDepth - 1, to);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    const int c = turn * C::WK + wk;  // (of the CTA's)
    if (c < nc) {
      uint32_t word[2][2][4];
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t at = w_at + s * 1024 + r * 512 + from;
          if constexpr (G == 128) {
            load_shared<4>(at + ((t ^ turned) << 4), word[s][r]);
          } else if constexpr (G == 64) {
#pragma unroll
            for (int h = 0; h < 2; ++h) load_shared<2>(at + (((h * 2 + (t >> 1)) ^ turned) << 4) + (t & 1) * 8, word[s][r] + 2 * h);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) load_shared<1>(at + ((i ^ turned) << 4) + t * 4, word[s][r] + i);
          }
        }
      float part[2][NT][4];
      uint32_t sm[2][2][2];  // scale, minus
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i % kEach == 0) {
          const int k = (kGroups == 1 ? c : min(c * kGroups + i / kEach, ng - 1)) * 8;  // (past the last group: columns of zeros)
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            load_shared<2>(my_scale[s][0] + k, sm[s][0]);
            load_shared<2>(my_scale[s][1] + k, sm[s][1]);
#pragma unroll
            for (int j = 0; j < NT; ++j) part[s][j][0] = part[s][j][1] = part[s][j][2] = part[s][j][3] = 0.f;
          }
        }
        uint32_t a[2][2][4];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int r = 0; r < 2; ++r) int4_pairs(word[s][r][i], sm[s][r][1], a[s][r]);
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int q = 0; q < PARTS; ++q) {
            uint32_t v[4];
            load_shared<4>(x_at[i] + (q * C::kTokens + j * 8) * 256 + from, v);
            const uint32_t b0 = __byte_perm(v[0], v[2], 0x5410), b1 = __byte_perm(v[0], v[2], 0x7632), b2 = __byte_perm(v[1], v[3], 0x5410),
                           b3 = __byte_perm(v[1], v[3], 0x7632);  // (columns 0 and 4, 1 and 5, as int4_pairs leaves them)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
              mma_16x8x16(part[s][j], a[s][0][0], a[s][1][0], a[s][0][1], a[s][1][1], b0, b1);
              mma_16x8x16(part[s][j], a[s][0][2], a[s][1][2], a[s][0][3], a[s][1][3], b2, b3);
            }
          }
        if (i % kEach == kEach - 1) {
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[s][j][e] = fmaf(__uint_as_float(sm[s][e / 2][0]), part[s][j][e], acc[s][j][e]);
        }
      }
    }
    from = from == (C::kDepth - 1) * C::kStageBytes ? 0 : from + C::kStageBytes;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  float* s_sum = reinterpret_cast<float*>(smem);  // [wk][set][token][row]
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        s_sum[((wk * 2 + s) * C::kTokens + j * 8 + t * 2 + (e & 1)) * C::kRows + wr * 16 + line + (e >> 1) * 8] = acc[s][j][e];
  __syncthreads();
  if (g.splits > 1) {
    if constexpr (C::WK > 1) {
      for (int i = threadIdx.x; i < C::kSums; i += kThreads) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < C::WK; ++k) v += s_sum[k * C::kSums + i];
        s_sum[i] = v;
      }
    }
    __syncwarp();
    ptx::cluster_sync();
  }
  constexpr int kHalf = C::kTokens * C::kRows;
  for (int i = threadIdx.x + blockIdx.z * kThreads; i < (W == 2 ? 1 : 2) * kHalf; i += kThreads * g.splits) {
    const int m = i % kHalf / C::kRows, n = n0 + (i / kHalf) * C::kRows + i % C::kRows;
    if (m >= g.M || n >= g.N) continue;
    float v[W] = {};
    if (g.splits > 1) {
      for (int z = 0; z < g.splits; ++z)
#pragma unroll
        for (int w = 0; w < W; ++w) v[w] += peer_load(base + (w * kHalf + i) * 4, z);
    } else {
#pragma unroll
      for (int k = 0; k < C::WK; ++k)
#pragma unroll
        for (int w = 0; w < W; ++w) v[w] += s_sum[k * C::kSums + w * kHalf + i];
    }
    static_cast<T*>(g.out)[m * g.ld_out + n] = result_of<T>(v);
  }
  if (g.splits > 1) {
    __syncwarp();
    ptx::cluster_sync();  // nobody's memory goes while it is read
  }
}

// ---- many rows --------------------------------------------------------------------------------------------------------------------------
// 128 weight rows x NT tokens a CTA.  Warps: 0 loads a chunk of 128 columns of both operands (TMA), 1 issues a group's products, whose left
// operand is weights unpacked into TMEM, for 128 tokens at a time, 4 to 11 unpack, a row a thread, four warps every other chunk, and 12 to 19
// fetch a group's sums, scale them and add them up in registers.  The CTAs are resident and
// take their tiles one after the other; few tiles: the chunks are split over the CTAs of a cluster, whose sums meet through distributed
// shared memory in a fixed order.
//
// 2200 x 15360 x 2048 takes 175 us, the tensor pipe active 40 % of it.  A chunk of 128 columns and 256 tokens takes some 2400 cycles, 1024
// of them products: the warp that issues looks at four barriers a chunk, 150 cycles and more each, and shares its scheduler with four
// others.  Without the unpacking, or without most of the additions, it takes as long.  (One set of eight unpacking warps, half a row each,
// with two places in TMEM: 185 us; all adding warps on both products in turn: 189; barriers looked at ahead: 180 to 215.)
template <int NT, int W, int PARTS>
struct Many {
  static constexpr int kWBytes = 128 * 64, kXBytes = NT * 256;  // of a chunk: 128 rows x 64 bytes; two halves of NT rows x 128 bytes
  static constexpr int kStageBytes = PARTS * kXBytes + W * kWBytes;
  static constexpr int kBudget = 216 * 1024, kStages = kBudget / kStageBytes < 8 ? kBudget / kStageBytes : 8;
  static constexpr int kSub = NT < 128 ? NT : 128, kSubs = NT / kSub;   // tokens of one product, products of a tile
  static constexpr int kSums = kSub == 128 ? 2 : 4, kTmemA = 256, kA = 4;  // columns: groups' sums; chunks of one weight
  static constexpr int kThreads = 20 * 32;
  // Two products of a tile: each has four of the adding warps and a place for its sums to itself.  One: four warps take half of its columns.
  static constexpr int kColumns = kSubs == 2 ? kSub : kSub / 2;         // a thread's of a product
  // Registers: 640 x 96 at launch.  Up to 32 sums of a thread fit in that.  For more the first four warps keep 24, the unpackers 48, and the
  // adders take 176: 128 x 24 + 256 x 48 + 256 x 176 = 60416 of 61440.
  static constexpr bool kWide = W * kColumns > 32;
  static_assert(kSubs == 1 || (kSubs == 2 && kSums == 2 && W == 1), "");
  static constexpr size_t kSmem = 1024 + kStages * kStageBytes;
  static_assert(kStages >= 2 && W * NT * 128 * 4 <= kStages * kStageBytes, "the sums of a split wait in the stages' memory");
};

struct Int4Maps {
  CUtensorMap x, w[2];
};

enum : int { kGiveUpEmpty = 91, kGiveUpFull = 92, kGiveUpAEmpty = 93, kGiveUpAFull = 94, kGiveUpSumEmpty = 95, kGiveUpSumFull = 96, kGiveUpDrain = 97 };

template <int NT, typename T, int W>
__global__ void __launch_bounds__((Many<NT, W, sizeof(T) == 4 ? 3 : 1>::kThreads), 1)
int4_many_kernel(const __grid_constant__ Int4Maps maps, const Int4Args g) {
  constexpr int PARTS = sizeof(T) == 4 ? 3 : 1;
  using C = Many<NT, W, PARTS>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t s_full[C::kStages], s_empty[C::kStages], s_afull[C::kA], s_aempty[C::kA], s_sfull[C::kSums], s_sempty[C::kSums];
  __shared__ uint32_t s_tmem;
  __shared__ int s_dead;  // a wait ran out: nothing waits any more, and the results are NaN
  const uint32_t stages = (ptx::smem_u32(smem_raw) + 1023) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t tiles = g.tiles_m * g.tiles_n;
  const int c0 = (int)blockIdx.z * g.per, nc = min(g.chunks - c0, g.per);
  const int each = kChunk / g.group;  // groups of a chunk
  if (warp == 0) {
    ptx::prefetch_tensormap(&maps.x);
    ptx::prefetch_tensormap(&maps.w[0]);
  } else if (warp == 1) {
    if (lane == 0) {
      for (int i = 0; i < C::kStages; ++i) {
        ptx::mbar_init(&s_full[i], 1);
        ptx::mbar_init(&s_empty[i], 1 + 8);  // the products that read x, and the unpacking warps: four read the weights, and all look at s_full
      }
      for (int i = 0; i < C::kA; ++i) {
        ptx::mbar_init(&s_afull[i], 4);
        ptx::mbar_init(&s_aempty[i], 1);
      }
      for (int i = 0; i < C::kSums; ++i) {
        ptx::mbar_init(&s_sfull[i], 1);
        ptx::mbar_init(&s_sempty[i], C::kSubs == 2 ? 4 : 8);
      }
      ptx::mbar_fence_init();
      s_dead = 0;
    }
    __syncwarp();
    ptx::tmem_alloc(&s_tmem, 512);
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

  if (warp < 4) {
    if constexpr (C::kWide) asm volatile("setmaxnreg.dec.sync.aligned.u32 24;");
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
            for (int w = 0; w < W; ++w) ptx::tma_load_2d(to + PARTS * C::kXBytes + w * C::kWBytes, &maps.w[w], &s_full[st.at], c * (kChunk / 2), n0);
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
#pragma unroll
              for (int h = 0; h < 2; ++h)
                ptx::tma_load_3d(to + p * C::kXBytes + h * NT * 128, &maps.x, &s_full[st.at], c * kChunk + h * 64, m0, p);
          }
        }
        const uint32_t n = min(loads, (uint32_t)C::kStages);
        for (uint32_t k = loads - n; k != loads; ++k)  // no copy is in flight when the CTA ends
          if (!ptx::mbar_wait(&s_full[k % C::kStages], (k / C::kStages) & 1, g.status, kGiveUpDrain)) break;
      }
    } else if (warp == 1) {
      const uint32_t el = ptx::elect_one();
      constexpr uint32_t idesc = ptx::make_idesc_bf16(128, C::kSub, 0);
      Ring<C::kStages> st;
      Ring<C::kA> a;
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
            for (int k = 0; k < here && on; ++k) {
              for (int sub = 0; sub < C::kSubs; ++sub, sum.step()) {
                if (!wait(s_sempty[sum.at], sum.parity ^ 1, kGiveUpSumEmpty)) {
                  on = false;
                  break;
                }
                ptx::tc_fence_after();
                // (Few instructions: this warp's loop has to be shorter than the products that it issues.)
                const uint32_t d = tmem + sum.at * C::kSub, left = tmem + C::kTmemA + a.at * 64, right = x.lo + sub * (128 * 128 >> 4);
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
                  const uint32_t part = right + p * (C::kXBytes >> 4);
                  if (each == 1) {
                    ptx::mma_ts_x4_w(el, d, left, part, x.hi, 2, idesc, p > 0);
                    ptx::mma_ts_x4_w(el, d, left + 32, part + (NT * 128 >> 4), x.hi, 2, idesc, 1);
                  } else if (each == 2) {
                    ptx::mma_ts_x4_w(el, d, left + k * 32, part + k * (NT * 128 >> 4), x.hi, 2, idesc, p > 0);
                  } else {
                    ptx::mma_ts_x2_w(el, d, left + k * 16, part + (k >> 1) * (NT * 128 >> 4) + (k & 1) * 4, x.hi, 2, idesc, p > 0);
                  }
                }
                ptx::mma_commit_w(el, ptx::smem_u32(&s_sfull[sum.at]));
              }
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
    }
  } else if (warp < 12) {
    if constexpr (C::kWide) asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    const int quad = warp & 3, set = (warp - 4) >> 2, row = quad * 32 + lane;  // a warp reaches the TMEM lanes of its place among four
    const uint32_t at_tmem = tmem + C::kTmemA + ((uint32_t)quad << 21);
    Ring<C::kStages> st;
    Ring<C::kA> a;
    int turn = 0;  // chunks so far, over all tiles
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
      zeros_of(c0 + ((turn ^ set) & 1), next);
      for (int c = c0; c < c0 + nc; ++c, ++turn, st.step()) {
        // Each stage's, the other set's too: a pass over the ring that is not waited for would make the next look done.  And it is not filled
        // again before this set has looked: of two passes, a look at the first would find the second, and wait for good.
        wait(s_full[st.at], st.parity, kGiveUpFull);
        if (((turn ^ set) & 1) != 0) {  // the other set's
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(&s_empty[st.at]);
#pragma unroll
          for (int w = 0; w < W; ++w) a.step();
          continue;
        }
        uint32_t zeros[W];
#pragma unroll
        for (int w = 0; w < W; ++w) zeros[w] = next[w];
        zeros_of(c + 2, next);
        const uint32_t tile = stages + st.at * C::kStageBytes + PARTS * C::kXBytes + row * 64, turned = (row >> 1) & 3;
#pragma unroll
        for (int w = 0; w < W; ++w, a.step()) {
          wait(s_aempty[a.at], a.parity ^ 1, kGiveUpAEmpty);
          __syncwarp();
          ptx::tc_fence_after();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t minus = int4_minus((zeros[w] >> (8 * (i * 32 / g.group))) & 255u);
            uint32_t v[4], r[16];
            load_shared<4>(tile + w * C::kWBytes + ((i ^ turned) << 4), v);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint32_t p[4];
              int4_pairs(v[j], minus, p);
              r[j * 4] = __byte_perm(p[0], p[1], 0x5410);
              r[j * 4 + 1] = __byte_perm(p[2], p[3], 0x5410);
              r[j * 4 + 2] = __byte_perm(p[0], p[1], 0x7632);
              r[j * 4 + 3] = __byte_perm(p[2], p[3], 0x7632);
            }
            ptx::tmem_st16(at_tmem + a.at * 64 + i * 16, r);
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
    if constexpr (C::kWide) asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
    const int quad = warp & 3, set = (warp - 12) >> 2, first = set * C::kColumns, row = quad * 32 + lane;  // (columns of the tile)
    const uint32_t at_tmem = tmem + ((uint32_t)quad << 21) + (C::kSubs == 2 ? 0 : first);
    Ring<C::kSums> sum;
    if (C::kSubs == 2 && set == 1) sum.step();
    for (uint32_t t = blockIdx.x; t < tiles; t += gridDim.x) {
      const int m0 = (int)(t % g.tiles_m) * NT, n0 = (int)(t / g.tiles_m) * 128, n = min(n0 + row, g.N - 1);
      float2 acc[W][C::kColumns / 2];
#pragma unroll
      for (int w = 0; w < W; ++w)
#pragma unroll
        for (int j = 0; j < C::kColumns / 2; ++j) acc[w][j] = make_float2(0.f, 0.f);
      float next = g.w[0].scale(n, c0 * each);  // (one group ahead)
      for (int c = c0; c < c0 + nc; ++c) {
        const int here = min(each, g.groups - c * each);
#pragma unroll
        for (int w = 0; w < W; ++w) {
#pragma unroll 1
          for (int k = 0; k < here; ++k) {
            const float2 scale = make_float2(next, next);
            {
              const bool same = k + 1 < here;  // the next sums' weight and chunk
              const int w1 = same ? w : w + 1 < W ? w + 1 : 0, c1 = same || w + 1 < W ? c : c + 1, k1 = same ? k + 1 : 0;
              if (c1 < c0 + nc) next = g.w[w1].scale(n, c1 * each + k1);
            }
            wait(s_sfull[sum.at], sum.parity, kGiveUpSumFull);
            __syncwarp();
            ptx::tc_fence_after();
            const uint32_t from = at_tmem + sum.at * C::kSub;
            constexpr int P = C::kColumns < 32 ? 16 : 32;
#pragma unroll
            for (int j0 = 0; j0 < C::kColumns; j0 += P) {
              uint32_t r[P];
              if constexpr (P == 32) ptx::tmem_ld32(from + j0, r);
              else ptx::tmem_ld16(from + j0, r);
              ptx::tmem_ld_wait();
              if (j0 + P == C::kColumns) {
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&s_sempty[sum.at]);
              }
#pragma unroll
              for (int j = 0; j < P / 2; ++j)
                acc[w][j0 / 2 + j] = ptx::ffma2(make_float2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])), scale, acc[w][j0 / 2 + j]);
            }
#pragma unroll
            for (int i = 0; i < C::kSubs; ++i) sum.step();
          }
        }
      }
      const float poison = *dead ? __uint_as_float(0x7fffffffu) : 0.f;
      const auto at = [&](int w, int j) { return (j & 1 ? acc[w][j / 2].y : acc[w][j / 2].x) + poison; };
      if (g.splits > 1) {  // (every product that read the stages is finished)
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
          for (int j = 0; j < C::kColumns; ++j)
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(stages + ((w * NT + first + j) * 128 + row) * 4), "f"(at(w, j)) : "memory");
      } else if (n0 + row < g.N) {
        T* out = static_cast<T*>(g.out) + (int64_t)(m0 + first) * g.ld_out + n0 + row;
#pragma unroll
        for (int j = 0; j < C::kColumns; ++j)
          if (m0 + first + j < g.M) {
            float v[W];
#pragma unroll
            for (int w = 0; w < W; ++w) v[w] = at(w, j);
            out[j * g.ld_out] = result_of<T>(v);
          }
      }
    }
  }
  if (g.splits > 1) {
    __syncwarp();
    ptx::cluster_sync();
    const int m0 = (int)(blockIdx.x % g.tiles_m) * NT, n0 = (int)(blockIdx.x / g.tiles_m) * 128, splits = g.splits;
    for (int i = (int)blockIdx.z * C::kThreads + threadIdx.x; i < NT * 128; i += C::kThreads * splits) {
      const int j = i >> 7, row = i & 127;
      if (m0 + j >= g.M || n0 + row >= g.N) continue;
      float v[W] = {}, part[W][8];
#pragma unroll
      for (int z = 0; z < 8; ++z)  // (all on their way before the first is added)
#pragma unroll
        for (int w = 0; w < W; ++w) part[w][z] = z < splits ? peer_load(stages + ((w * NT + j) * 128 + row) * 4, z) : 0.f;
#pragma unroll
      for (int z = 0; z < 8; ++z)
#pragma unroll
        for (int w = 0; w < W; ++w) v[w] += part[w][z];
      static_cast<T*>(g.out)[(int64_t)(m0 + j) * g.ld_out + n0 + row] = result_of<T>(v);
    }
    __syncwarp();
    ptx::cluster_sync();  // nobody's memory goes while it is read
  }
  __syncwarp();
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  if (warp == 1) ptx::tmem_dealloc(tmem, 512);
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

constexpr int kFewTokens = 16;
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
  const int64_t tm = (g.M + NT - 1) / NT, tn = (g.N + 127) / 128, tiles = tm * tn, room = device_sm_count();
  if (tiles * g.chunks > 0x7fffffff) {
    set_error("mvpa_matmul_int4: more than 2^31 blocks of 128 x %d x 128", NT);
    return MVPA_ERR_UNSUPPORTED;
  }
  g.tiles_m = (uint32_t)tm;
  g.tiles_n = (uint32_t)tn;
  // As many CTAs to a tile as are resident for all tiles at once (clusters of eight: 15 on this device), with two chunks each at least.
  constexpr auto kernel = int4_many_kernel<NT, T, W>;
  MVPA_CUDA_CHECK(grant_smem<kernel>(C::kSmem));
  int splits = 1;
  for (int n = 8; n > 1 && splits == 1; n /= 2) {
    int most = 0;
    if (g.chunks < 2 * n || tiles * n > room) continue;
    MVPA_CUDA_CHECK(resident_clusters<kernel>(n, C::kThreads, C::kSmem, &most));
    if (tiles <= most) splits = n;
  }
  g.per = (g.chunks + splits - 1) / splits;
  g.splits = (g.chunks + g.per - 1) / g.per;
  const dim3 grid((unsigned)(g.splits > 1 || tiles < room ? tiles : room), 1, g.splits);
  MVPA_CUDA_CHECK(launch_dependent((unsigned)g.splits, kernel, grid, C::kThreads, C::kSmem, s, maps, g));
  count_launch();
  MVPA_CUDA_CHECK(cudaGetLastError());
  return MVPA_OK;
}

// -> whether this kernel can do it (a CTA's scales have to fit in shared memory).
template <typename T, int W, int NT>
int run_few(const void* x, int64_t ld_x, int64_t plane, Int4Args g, cudaStream_t s, bool* done) {
  constexpr int PARTS = sizeof(T) == 4 ? 3 : 1;
  using C = Few<W, NT, PARTS>;
  constexpr int kRows = C::kRows * (W == 1 ? 2 : 1);
  const int64_t tiles = (g.N + kRows - 1) / kRows, room = (int64_t)device_sm_count() * 2;
  const auto scales = [&](int splits) {
    const int64_t per = (g.chunks + splits - 1) / splits;
    return 2 * C::kRows * std::min<int64_t>(per * (kChunk / g.group), g.groups);
  };
  int splits = 1;
  while (splits < 8 && ((tiles * splits * 2 <= room && g.chunks >= C::WK * 2 * splits) || scales(splits) > C::kMostScales)) splits *= 2;
  *done = scales(splits) <= C::kMostScales;
  if (!*done) return MVPA_OK;
  g.per = (g.chunks + splits - 1) / splits;
  g.splits = (g.chunks + g.per - 1) / g.per;
  g.x = x;
  g.ld_x = ld_x;
  g.plane = plane;
  const auto launch = [&](auto group) {
    constexpr auto kernel = int4_few_kernel<T, decltype(group)::value, W, NT, PARTS>;
    MVPA_CUDA_CHECK(grant_smem<kernel>(C::kBytes + C::kMostScales * 8));
    MVPA_CUDA_CHECK(launch_dependent((unsigned)g.splits, kernel, dim3((unsigned)tiles, 1, g.splits), kFewWarps * 32, C::kBytes + scales(g.splits) * 8, s, g));
    return MVPA_OK;
  };
  const int rc = g.group == 128  ? launch(std::integral_constant<int, 128>())
                 : g.group == 64 ? launch(std::integral_constant<int, 64>())
                                 : launch(std::integral_constant<int, 32>());
  if (rc != MVPA_OK) return rc;
  count_launch();
  MVPA_CUDA_CHECK(cudaGetLastError());
  return MVPA_OK;
}

template <typename T, int W>
int run_int4(Int4Args g, int32_t dtype, void* workspace, cudaStream_t s) {
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
  // (us, few / many at 16 tokens and 17: 15360 x 2048 11.9 / 14.5, 2048 x 7680 8.3 / 13.6, 768 x 2496 5.6 / 6.4; with 32 tokens in four groups the
  // former took 22, 22 and 7.6, the latter 14.7, 15.1 and 6.4.)
  if (g.M <= kFewTokens) {
    bool done = false;
    const int rc = g.M <= 8 ? run_few<T, W, 1>(x, ld, plane, g, s, &done) : run_few<T, W, 2>(x, ld, plane, g, s, &done);
    if (done || rc != MVPA_OK) return rc;
  }
  if (g.M <= 32) return run_many<32, T, W>(x, ld, plane, g, s);
  if (g.M <= 64 || sizeof(T) == 4) return run_many<64, T, W>(x, ld, plane, g, s);
  if constexpr (sizeof(T) == 2) {
    // 256 tokens a tile where that leaves half of the multiprocessors one (us, 128 / 256: 550 x 768 x 2496 10.9 / 20.6, 256 x 5632 x 2048 17.9 /
    // 20.8).  A gate's two weights take a thread's registers for 128.
    const int64_t wide = ((g.M + 255) / 256) * ((g.N + 127) / 128);
    if (g.M <= 128 || W == 2 || 2 * wide < device_sm_count()) return run_many<128, T, W>(x, ld, plane, g, s);
    if constexpr (W == 1) return run_many<256, T, W>(x, ld, plane, g, s);
  }
  return MVPA_OK;
}

}  // namespace
}  // namespace mvpa

using namespace mvpa;

extern "C" size_t mvpa_matmul_int4_workspace_bytes(const void* x, int64_t ld_x, int64_t M, int32_t K, int32_t dtype) {
  if (M <= 0 || K <= 0 || in_place(x, ld_x, dtype)) return 0;
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
  g.status = status;
  if (dtype == MVPA_F32) return up != nullptr ? run_int4<float, 2>(g, dtype, workspace, s) : run_int4<float, 1>(g, dtype, workspace, s);
  return up != nullptr ? run_int4<__nv_bfloat16, 2>(g, dtype, workspace, s) : run_int4<__nv_bfloat16, 1>(g, dtype, workspace, s);
}
