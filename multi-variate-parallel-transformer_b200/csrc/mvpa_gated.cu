// The gated projection of the MLP in one kernel, and its gradients, in bf16:
//
//   h = silu(g) u,  g = x Wg^T,  u = x Wu^T                    x (M, E), Wg and Wu (I, E)
//   dg = dh u s (1 + g (1 - s)),  du = dh g s,  s = 1 / (1 + e^-g)
//   dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x
//
// Three matrix products of one shape of kernel: a pair of CTAs (cta_group::2) forms 256 rows x 256 columns of sums in TMEM, fp32, from
// blocks of 64 along the summed axis that the TMA stages in shared memory.
//   forward        the first CTA brings 128 rows of Wg and the second the same rows of Wu, so that a thread that holds a token's row of
//                  sums finds g and u of one feature 128 columns apart: h leaves from fp32 in one rounding, and g and u go to memory
//                  only where a backward pass will want them: 24 bits of each, the upper half of the fp32 number and the byte after it,
//                  in matrices of their own.  (In bf16 their roundings are half of the gradients' error: 0.0031 of the gradients' size
//                  against 0.0023, of which 0.0017 is the results' own rounding.)
//   input          dg and du are the left operand one after the other, Wg and Wu, whose rows lie along the columns of the result
//                  (MN-major), the right one: the sum of both products is formed in TMEM.
//   weights        both operands have the summed axis, the tokens, outermost (MN-major).
// dg and du are rounded to bf16 between the kernels: the products take 16-bit operands, and each of their sums is over hundreds of
// terms, whose roundings (up to 2^-8 each, of either sign) leave the sum nearly as exact as its own rounding to bf16 does: the gradients are
// 0.0023 of their size from 64 bits, with dg and du in fp32 they would be 0.0017.
#include "block_rows.cuh"
#include <algorithm>

#include "silu.cuh"
#include "tc_pairs.cuh"
#include "tc_tma_host.cuh"

namespace mvpa {
namespace {

enum : int { kForward = 0, kForwardSave = 1, kInput = 2, kWeights = 3 };

struct GatedMaps {
  CUtensorMap a[2], b[2], out[5];
};
struct GatedArgs {
  uint32_t tiles_m, tiles_n;
  uint32_t part;     // tiles along M of one part (kWeights: dWg, then dWu)
  int blocks;        // blocks along the summed axis in a segment (kInput: dg Wg, then du Wu)
  int segments;
  int rows, cols;    // of the results
  int few;           // rows of the left operand where there are up to 128 (a multiple of 8), else 0
  int* status;
  int splits, per;   // the summed axis in `splits` pieces of up to `per` blocks, each a tile of its own, whose sums go to `sums` in fp32
  float* sums;       // [splits][parts][rows][cols]
};

constexpr int kGatedThreads = 384;
// As many stages as there is room for: a block is some 2 us on its way from memory through the products and back to an empty stage
// (16384 x 2048 x 5632: 493 us with five, 476 with six; where the power does not bound it a block still takes 0.4 us, its products 0.27).
template <int MODE, int TN>
struct Gated {
  static constexpr int kHalfN = TN / 2;                // rows (or columns) of the right operand in each CTA
  static constexpr int kBoxes = (kHalfN + 63) / 64;    // of 64 columns, of an operand whose rows lie along them (192: the last one half used)
  static constexpr int kBytes = 128 * 128 + (MODE >= kInput ? kBoxes * 64 : kHalfN) * 128;
  static constexpr int kOutBytes = 8 * 4096;           // a warp's 32 rows x 64 columns on their way out
  static constexpr int kStages = (225 * 1024 - kOutBytes) / kBytes;
  static constexpr size_t kSmem = 1024 + kStages * kBytes + kOutBytes;
};

enum : int { kGiveUpEmpty = 81, kGiveUpFull = 82, kGiveUpTmemEmpty = 83, kGiveUpTmemFull = 84, kGiveUpDrain = 85 };

// TN: columns of sums of a tile (256, 192 or 128; a gate's are half g, half u).
template <int MODE, int TN, bool SPLIT>
__global__ void __launch_bounds__(kGatedThreads, 1) gated_kernel(const __grid_constant__ GatedMaps maps, const GatedArgs g) {
  constexpr bool kGate = MODE <= kForwardSave, kRowsA = MODE == kWeights, kRowsB = MODE >= kInput;  // (rows along M / N: MN-major)
  using C = Gated<MODE, TN>;
  constexpr int kTileN = kGate ? TN / 2 : TN, kHalfN = C::kHalfN;  // (columns of the result)
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t s_full[C::kStages], s_empty[C::kStages], s_tfull[2], s_tempty[2];
  __shared__ uint32_t s_tmem;
  __shared__ int s_dead;  // a wait ran out: nothing waits any more, and the results are NaN
  const uint32_t stages = (ptx::smem_u32(smem_raw) + 1023) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t half = ptx::cluster_rank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1, each = g.tiles_m * g.tiles_n, tiles = SPLIT ? each * g.splits : each;
  const int all = g.blocks * g.segments;
  const auto piece_of = [&](uint32_t t) { return SPLIT ? t / each : 0u; };
  const auto blocks_of = [&](uint32_t piece) { return SPLIT ? min(g.per, all - (int)piece * g.per) : all; };
  if (warp == 0) {
    ptx::prefetch_tensormap(&maps.a[0]);
    ptx::prefetch_tensormap(&maps.b[0]);
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

  if (warp == 0 || warp == 2) {  // left operand, right operand: a warp of each CTA loads its CTA's 128 rows (or columns) a block
    const bool left = warp == 0;
    const uint32_t el = ptx::elect_one(), there = ptx::cluster_map(ptx::smem_u32(s_full), 0);
    Ring<C::kStages> st;
    uint32_t loads = 0;
    bool on = true;
    for (uint32_t t = pair; t < tiles && on; t += pairs) {
      const uint32_t piece = piece_of(t);
      const Tile at = tile_at<kTileN>(t - piece * each, g.tiles_n, g.tiles_m);
      const uint32_t part = (uint32_t)at.m0 / 256 >= g.part ? 1 : 0;
      const int row = left ? at.m0 - (int)(part * g.part * 256) + (int)half * 128 : kGate ? at.n0 : at.n0 + (int)half * kHalfN;
      const int first = (int)piece * g.per, end = first + blocks_of(piece);
      for (int kb = first; kb < end; ++kb, ++loads, st.step()) {
        if (!wait(s_empty[st.at], st.parity ^ 1, kGiveUpEmpty)) {
          on = false;
          break;
        }
        // (Up to 128 rows are the first CTA's alone, in boxes of that many: rows past the matrix take the TMA as long as others, some 1.6
        // cycles of 128 bytes.  Whatever else lies in the stage is other rows' sums, which are not stored.)
        if (left && half == 0 && el)
          ptx::mbar_arrive_expect_tx(&s_full[st.at], g.few > 0 ? 2 * (C::kBytes - 128 * 128) + g.few * 128 : 2 * C::kBytes);
        __syncwarp();
        if (left && half == 1 && g.few > 0) continue;
        const int seg = kb >= g.blocks ? 1 : 0, k = (kb - seg * g.blocks) * 64;
        const uint32_t to = stages + st.at * C::kBytes + (left ? 0 : 128 * 128), bar = there + 8 * st.at;
        const CUtensorMap* map = left ? &maps.a[kRowsA ? part : seg] : &maps.b[kGate ? half : kRowsA ? 0 : seg];
        if (left ? kRowsA : kRowsB) {
          ptx::tma_load_2d_pair_w(el, to, map, bar, row, k);
          if (left || C::kBoxes == 2) ptx::tma_load_2d_pair_w(el, to + 64 * 128, map, bar, row + 64, k);
        } else {
          ptx::tma_load_2d_pair_w(el, to, map, bar, k, row);
        }
      }
    }
    if (left && half == 0) {  // no copy is in flight when the CTAs end (the other one waits for this one at the end)
      const uint32_t n = min(loads, (uint32_t)C::kStages);
      for (uint32_t k = loads - n; k != loads; ++k)
        if (!ptx::mbar_wait(&s_full[k % C::kStages], (k / C::kStages) & 1, g.status, kGiveUpDrain)) break;
    }
  } else if (warp == 1) {
    if (half == 0) {
      const uint32_t el = ptx::elect_one();
      constexpr uint32_t idesc = ptx::make_idesc_bf16_ab(256, TN, kRowsA, kRowsB);
      constexpr uint32_t kStepA = kRowsA ? 128 : 2, kStepB = kRowsB ? 128 : 2;
      const ptx::DescHalves a0 = ptx::make_desc_halves_sw128(stages, kRowsA ? 64 * 128 : 16, 1024),
                            b0 = ptx::make_desc_halves_sw128(stages + 128 * 128, kRowsB ? 64 * 128 : 16, 1024);
      // (The loop has to be shorter than a block's products: its barriers by address, and the next block's looked at while the products of
      // this one are on their way.)
      const uint32_t full = ptx::smem_u32(s_full), empty = ptx::smem_u32(s_empty);
      Ring<C::kStages> st;
      Ring<2> buf;
      uint32_t last = 0, last_parity = 0;
      bool on = true, any = false, there = false;
      for (uint32_t t = pair; t < tiles && on; t += pairs, buf.step()) {
        if (!wait(s_tempty[buf.at], buf.parity ^ 1, kGiveUpTmemEmpty)) break;
        ptx::tc_fence_after();
        const uint32_t d = tmem + buf.at * 256;
        const int blocks = blocks_of(piece_of(t));
#pragma unroll 4
        for (int kb = 0; kb < blocks; ++kb) {
          if (!there && !wait(s_full[st.at], st.parity, kGiveUpFull)) {
            on = false;
            break;
          }
          ptx::tc_fence_after();
          const uint32_t off = st.at * (C::kBytes >> 4);
          ptx::mma_f16_ss_x4_pair_w(el, d, {a0.lo + off, a0.hi}, {b0.lo + off, b0.hi}, kStepA, kStepB, idesc, kb > 0);
          ptx::mma_commit_pair_w(el, 3, empty + 8 * st.at);
          last = st.at;
          last_parity = st.parity;
          any = true;
          st.step();
          there = ptx::mbar_test_wait_a(full + 8 * st.at, st.parity);
        }
        if (on) ptx::mma_commit_pair_w(el, 3, ptx::smem_u32(&s_tfull[buf.at]));
      }
      if (any) ptx::mbar_wait(&s_empty[last], last_parity, g.status, kGiveUpDrain);
    }
  } else if (warp >= 4) {
    // Eight warps take the sums home: a thread one row, every other 64 columns.  A warp puts 32 rows x 64 columns into shared memory in
    // the 128-byte swizzle and leaves them to the TMA, which skips what lies past the matrix.
    const int quad = warp & 3, group = (warp - 4) >> 2;
    const uint32_t out = stages + C::kStages * C::kBytes + (warp - 4) * 4096, at_tmem = tmem + ((uint32_t)quad << 21);
    const auto place = [&]() {  // (once the store before has been read)
      if (lane == 0) ptx::tma_store_wait_read<0>();
      __syncwarp();
      return out;
    };
    const auto put = [&](uint32_t to, int piece, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + lane * 128 + ((piece ^ (lane & 7)) << 4)), "r"(a), "r"(b), "r"(c), "r"(d)
                   : "memory");
    };
    const auto send = [&](uint32_t from, const CUtensorMap* map, int x, int y) {
      ptx::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        ptx::tma_store_2d(map, from, x, y);
        ptx::tma_store_commit();
      }
    };
    Ring<2> buf;
    for (uint32_t t = pair; t < tiles; t += pairs, buf.step()) {
      const uint32_t piece = piece_of(t);
      const Tile at = tile_at<kTileN>(t - piece * each, g.tiles_n, g.tiles_m);
      const uint32_t part = (uint32_t)at.m0 / 256 >= g.part ? 1 : 0;
      const int y = at.m0 - (int)(part * g.part * 256) + (int)half * 128 + quad * 32;
      wait(s_tfull[buf.at], buf.parity, kGiveUpTmemFull);
      __syncwarp();
      ptx::tc_fence_after();
      const uint32_t from = at_tmem + buf.at * 256;
      const uint32_t poison = *dead ? 0x7fffffffu : 0u;
      const auto release = [&]() {
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive_cluster(ptx::cluster_map(ptx::smem_u32(&s_tempty[buf.at]), 0));
      };
      const auto words = [&](const uint32_t (&r)[32], uint32_t to, int piece) {  // 32 sums as they are, rounded
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const auto two = [&](int i) {
            return ptx::pack_bf16(__uint_as_float(r[k * 8 + 2 * i] | poison), __uint_as_float(r[k * 8 + 2 * i + 1] | poison));
          };
          put(to, piece + k, two(0), two(1), two(2), two(3));
        }
      };
      if constexpr (kGate) {
        if (group * 64 >= kTileN) {  // (no columns for these warps)
          release();
          continue;
        }
        const int x = at.n0 + group * 64;
        const bool inside = y < g.rows && x < g.cols;  // (the same for the whole warp: a store does not begin past the matrix)
        if constexpr (MODE == kForwardSave) {
#pragma unroll 1
          for (int sum = 0; sum < 2; ++sum) {  // g, then u: the numbers' upper halves, and the byte after
            uint32_t lower[2][8];
            place();
#pragma unroll
            for (int c = 0; c < 64; c += 32) {
              uint32_t r[32];
              ptx::tmem_ld32(from + sum * kHalfN + group * 64 + c, r);
              ptx::tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 32; ++j) r[j] |= poison;
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const auto two = [&](int i) { return __byte_perm(r[k * 8 + 2 * i], r[k * 8 + 2 * i + 1], 0x7632); };
                put(out, c / 8 + k, two(0), two(1), two(2), two(3));
              }
#pragma unroll
              for (int k = 0; k < 8; ++k)
                lower[c / 32][k] = __byte_perm(__byte_perm(r[4 * k], r[4 * k + 1], 0x0051), __byte_perm(r[4 * k + 2], r[4 * k + 3], 0x0051), 0x5410);
            }
            if (inside) send(out, &maps.out[1 + sum], x, y);
            place();
#pragma unroll
            for (int k = 0; k < 4; ++k) {  // (rows of 64 bytes, in the 64-byte swizzle)
              const uint32_t* b = lower[k / 2] + (k % 2) * 4;
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(out + lane * 64 + ((k ^ ((lane >> 1) & 3)) << 4)), "r"(b[0]), "r"(b[1]),
                           "r"(b[2]), "r"(b[3])
                           : "memory");
            }
            if (inside) send(out, &maps.out[3 + sum], x, y);
          }
        }
        const uint32_t to = place();
#pragma unroll
        for (int c = 0; c < 64; c += 32) {
          uint32_t rg[32], ru[32];
          ptx::tmem_ld32(from + group * 64 + c, rg);
          ptx::tmem_ld32(from + kHalfN + group * 64 + c, ru);
          ptx::tmem_ld_wait();
          if (c == 32) release();
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const float gate = __uint_as_float(rg[j]);
            rg[j] = __float_as_uint(Sigmoid(gate).times(gate, __uint_as_float(ru[j])));
          }
          words(rg, to, c / 8);
        }
        if (inside) send(to, &maps.out[0], x, y);
      } else {
#pragma unroll
        for (int c = group * 64; c < TN; c += 128) {
          const int x = at.n0 + c;
          const uint32_t to = SPLIT ? 0 : place();
          uint32_t r0[32], r1[32];
          ptx::tmem_ld32(from + c, r0);
          ptx::tmem_ld32(from + c + 32, r1);
          ptx::tmem_ld_wait();
          if (c + 128 >= TN) release();
          if constexpr (SPLIT) {
            if (y + lane < g.rows) {
              float* row = g.sums + (((int64_t)piece * (kRowsA ? 2 : 1) + part) * g.rows + y + lane) * g.cols + x;
              const auto store = [&](const uint32_t (&r)[32], int to) {
#pragma unroll
                for (int j = 0; j < 32; j += 4)
                  if (x + to + j < g.cols)
                    *reinterpret_cast<uint4*>(row + to + j) = make_uint4(r[j] | poison, r[j + 1] | poison, r[j + 2] | poison, r[j + 3] | poison);
              };
              store(r0, 0);
              store(r1, 32);
            }
            __syncwarp();
            continue;
          }
          words(r0, to, 0);
          words(r1, to, 4);
          if (y < g.rows && x < g.cols) send(to, &maps.out[part], x, y);
        }
      }
    }
    if (lane == 0) ptx::tma_store_wait_all();
  }
  __syncwarp();
  ptx::tc_fence_before();
  __syncthreads();
  ptx::cluster_sync();  // neither CTA's memory goes while the other's products or barriers use it
  ptx::tc_fence_after();
  if (warp == 1) ptx::tmem_dealloc_pair(tmem, 512);
}

// What the forward keeps, in one piece of memory: the upper halves of g and of u, (M, I) each, then the bytes after, with rows on 16-byte
// boundaries.
struct Saved {
  uint8_t *upper[2], *lower[2];
  int64_t ld;  // of the bytes
  Saved(void* p, int64_t M, int64_t I) : ld((I + 15) / 16 * 16) {
    uint8_t* at = static_cast<uint8_t*>(p);
    for (int i = 0; i < 2; ++i) {
      upper[i] = at + i * M * I * 2;
      lower[i] = at + 2 * M * I * 2 + i * M * ld;
    }
  }
  static size_t bytes(int64_t M, int64_t I) { return (size_t)M * ((size_t)I * 4 + (size_t)(I + 15) / 16 * 16 * 2); }
};

// Eight numbers of 24 bits.
__device__ __forceinline__ void load24(const uint8_t* upper, const uint8_t* lower, float (&f)[8]) {
  const uint4 h = *reinterpret_cast<const uint4*>(upper);
  const uint2 l = *reinterpret_cast<const uint2*>(lower);
  const uint32_t w[4] = {h.x, h.y, h.z, h.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t b = i < 2 ? l.x : l.y;
    f[2 * i] = __uint_as_float(__byte_perm(w[i], b, i & 1 ? 0x1060 : 0x1040) & 0xffffff00u);
    f[2 * i + 1] = __uint_as_float(__byte_perm(w[i], b, i & 1 ? 0x3270 : 0x3250) & 0xffffff00u);
  }
}

// dg and du from dh and the forward's g and u, in fp32, rounded once.  Bound by memory: 12 bytes an element.
__global__ void __launch_bounds__(256) gate_bwd_kernel(const __nv_bfloat16* __restrict__ dh, int64_t ld_dh, const Saved kept,
                                                       __nv_bfloat16* __restrict__ dgate, __nv_bfloat16* __restrict__ dup, int64_t rows, int width) {
  using V = Vec<__nv_bfloat16>;
  ptx::griddep_launch();
  ptx::griddep_wait();
  const int per_row = width / V::N;
  const int64_t total = rows * per_row;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i / per_row, c = (i - row * per_row) * V::N;
    float x[V::N], u[V::N], d[V::N];
    load24(kept.upper[0] + i * 16, kept.lower[0] + row * kept.ld + c, x);
    load24(kept.upper[1] + i * 16, kept.lower[1] + row * kept.ld + c, u);
    V::load(dh + row * ld_dh + c, d);
#pragma unroll
    for (int e = 0; e < V::N; ++e) {
      const Sigmoid s(x[e]);
      const float dg = s.times_slope(d[e], u[e], x[e]);
      u[e] = s.times(d[e], x[e]);
      x[e] = dg;
    }
    V::store(dgate + i * V::N, x);
    V::store(dup + i * V::N, u);
  }
}

// A matrix of bf16, in boxes of 64 columns.
int encode(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t ld, int box_rows) {
  const uint64_t dims[2] = {(uint64_t)cols, (uint64_t)rows}, strides[1] = {(uint64_t)ld * 2};
  const uint32_t box[2] = {64, (uint32_t)box_rows};
  return encode_bf16_sw128(map, base, 2, dims, strides, box);
}

template <int MODE, int TN, bool SPLIT = false>
int launch_gated(const GatedMaps& maps, const GatedArgs& g, cudaStream_t s) {
  const int64_t tiles = (int64_t)g.tiles_m * g.tiles_n * (SPLIT ? g.splits : 1), pairs = device_sm_count() / 2;
  if (tiles * g.blocks * g.segments > 0x7fffffff) {
    set_error("mvpa_gated_linear: more than 2^31 blocks of 256 x %d x 64", TN);
    return MVPA_ERR_UNSUPPORTED;
  }
  constexpr auto kernel = gated_kernel<MODE, TN, SPLIT>;
  MVPA_CUDA_CHECK(grant_smem<kernel>(Gated<MODE, TN>::kSmem));
  MVPA_CUDA_CHECK(launch_dependent(dim3(2), kernel, dim3(2 * (unsigned)(tiles < pairs ? tiles : pairs)), kGatedThreads, Gated<MODE, TN>::kSmem, s, maps, g));
  count_launch();
  MVPA_CUDA_CHECK(cudaGetLastError());
  return MVPA_OK;
}

// The width of the gate's tiles: the one whose rounds over the pairs of multiprocessors take the least.  A block of 64 along the summed axis
// takes a pair the longer of its products (256 columns 270 ns) and its loads (a multiprocessor takes some 150 bytes in a nanosecond): 270 ns
// at 256 columns, 218 at 192, 164 at 128.
int tile_width(int64_t tiles_m, int64_t cols) {
  const int64_t pairs = device_sm_count() / 2;
  const auto time = [&](int width, int each) { return (tiles_m * ((cols + width / 2 - 1) / (width / 2)) + pairs - 1) / pairs * each; };
  return time(128, 164) < time(256, 270) ? 128 : 256;  // (192: 96 features are not a whole number of the 64 that a warp takes)
}

uint32_t tiles_of(int64_t n, int each) { return (uint32_t)((n + each - 1) / each); }

int few_rows(int64_t rows) { return rows <= 128 ? ((int)rows + 7) / 8 * 8 : 0; }

// The gradients' products: how wide their tiles are, and in how many pieces the summed axis, by the longest pair's blocks.  Pieces are for
// few tiles along a long axis, up to one a pair and eight blocks a piece at least; they cost a launch more and their sums' way to memory
// and back.  In pieces and whole, operands in L2: weights' gradient of 65536 x 64 x 64 15 and 176 us, of 9973 x 64 x 72 10 and 39; dx of 22 x 2048 x 5632 13
// and 36, of 22 x 768 x 1728 8 and 13.
struct Plan {
  int width, splits, per;
  size_t bytes;
};
Plan plan_of(int64_t tiles_m, int64_t cols, int64_t blocks, int64_t rows, bool may_split) {
  const int64_t pairs = device_sm_count() / 2;
  constexpr int kWidths[3] = {256, 192, 128}, kTimes[3] = {270, 218, 164};
  constexpr int kJoin = 5000, kSumBytes = 3000;  // ns, bytes a ns
  Plan best = {256, 1, 0, 0};
  int64_t least = INT64_MAX;
  for (int i = 0; i < 3; ++i) {
    const int64_t tiles = tiles_m * ((cols + kWidths[i] - 1) / kWidths[i]);
    for (int n = 1; n == 1 || (may_split && tiles * n <= pairs && blocks >= 8 * n); ++n) {
      const int64_t per = (blocks + n - 1) / n;
      if ((blocks + per - 1) / per != n) continue;
      const int64_t time = (tiles * n + pairs - 1) / pairs * per * kTimes[i] + (n > 1 ? kJoin + n * rows * cols * 8 / kSumBytes : 0);
      if (time < least) {
        least = time;
        best = {kWidths[i], n, (int)per, n > 1 ? (size_t)n * rows * cols * 4 : 0};
      }
    }
  }
  return best;
}
Plan plan_dx(int64_t M, int32_t E, int32_t I, bool may_split) { return plan_of(tiles_of(M, 256), E, 2 * (int64_t)tiles_of(I, 64), M, may_split); }
Plan plan_dw(int64_t M, int32_t E, int32_t I, bool may_split) {
  return plan_of(2 * (int64_t)tiles_of(I, 256), E, tiles_of(M, 64), 2 * (int64_t)I, may_split);
}

// The pieces' sums of one result or two, `each` numbers (a multiple of 8), added in their order and rounded once.
__global__ void __launch_bounds__(256) gated_join_kernel(const float* __restrict__ sums, int splits, int64_t each, int results,
                                                         __nv_bfloat16* __restrict__ out0, __nv_bfloat16* __restrict__ out1) {
  ptx::griddep_launch();
  ptx::griddep_wait();
  const int64_t all = each * results;
  for (int64_t i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * 4; i < all; i += (int64_t)gridDim.x * blockDim.x * 4) {
    float4 v = *reinterpret_cast<const float4*>(sums + i);
#pragma unroll 8
    for (int z = 1; z < splits; ++z) {
      const float4 a = *reinterpret_cast<const float4*>(sums + z * all + i);
      v.x += a.x;
      v.y += a.y;
      v.z += a.z;
      v.w += a.w;
    }
    *reinterpret_cast<uint2*>(i < each ? out0 + i : out1 + (i - each)) = make_uint2(ptx::pack_bf16(v.x, v.y), ptx::pack_bf16(v.z, v.w));
  }
}

// (tiles_n is filled in.)
template <int MODE>
int run_gated(const GatedMaps& maps, GatedArgs g, const Plan& plan, float* sums, void* out0, void* out1, cudaStream_t s) {
  g.tiles_n = tiles_of(g.cols, plan.width);
  if (plan.splits == 1)
    return plan.width == 256   ? launch_gated<MODE, 256>(maps, g, s)
           : plan.width == 192 ? launch_gated<MODE, 192>(maps, g, s)
                               : launch_gated<MODE, 128>(maps, g, s);
  g.splits = plan.splits;
  g.per = plan.per;
  g.sums = sums;
  const int rc = plan.width == 256   ? launch_gated<MODE, 256, true>(maps, g, s)
                 : plan.width == 192 ? launch_gated<MODE, 192, true>(maps, g, s)
                                     : launch_gated<MODE, 128, true>(maps, g, s);
  if (rc != MVPA_OK) return rc;
  const int results = MODE == kWeights ? 2 : 1;
  const int64_t each = (int64_t)g.rows * g.cols, ctas = (each * results / 4 + 255) / 256, most = (int64_t)device_sm_count() * 8;
  MVPA_CUDA_CHECK(launch_dependent(1, gated_join_kernel, (unsigned)(ctas < most ? ctas : most), 256, 0, s, (const float*)sums, plan.splits, each,
                                   results, (__nv_bfloat16*)out0, (__nv_bfloat16*)out1));
  count_launch();
  MVPA_CUDA_CHECK(cudaGetLastError());
  return MVPA_OK;
}

int check_sizes(const char* what, int64_t M, int32_t E, int32_t I) {
  constexpr int kMost = 0x7fffffff - 1024;  // (the first place past the last tile is a 32-bit coordinate)
  if (M < 1 || E < 1 || I < 1 || M > kMost || E > kMost || I > kMost || E % 8 != 0 || I % 8 != 0) {
    set_error("%s: M, E and I must lie between 1 and %d, E and I be multiples of 8 (got %lld, %d, %d)", what, kMost, (long long)M, E, I);
    return MVPA_ERR_SHAPE;
  }
  return MVPA_OK;
}
bool rows_fit(const void* p, int64_t ld, int64_t width) {
  return p != nullptr && (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld >= width && ld % 8 == 0;
}

}  // namespace
}  // namespace mvpa

using namespace mvpa;

extern "C" size_t mvpa_gated_linear_saved_bytes(int64_t M, int32_t I) { return M < 1 || I < 1 ? 0 : Saved::bytes(M, I); }

extern "C" int mvpa_gated_linear(const void* x, int64_t ld_x, const void* w_gate, const void* w_up, void* h, int64_t ld_h, void* saved,
                                 int64_t M, int32_t E, int32_t I, int32_t* status, void* cuda_stream) {
  const int rc0 = check_sizes("mvpa_gated_linear", M, E, I);
  if (rc0 != MVPA_OK) return rc0;
  if (!rows_fit(x, ld_x, E) || !rows_fit(w_gate, E, E) || !rows_fit(w_up, E, E) || !rows_fit(h, ld_h, I) ||
      (reinterpret_cast<uintptr_t>(saved) & 15) != 0) {
    set_error("mvpa_gated_linear: x, the weights, h and saved must be 16-byte aligned with rows of a multiple of 16 bytes, not shorter than "
              "their widths");
    return MVPA_ERR_ALIGNMENT;
  }
  const uint32_t tm = tiles_of(M, 256);
  const int width = tile_width(tm, I);
  GatedMaps maps = {};
  const int few = few_rows(M);
  int rc = encode(&maps.a[0], x, M, E, ld_x, few > 0 ? few : 128);
  if (rc == MVPA_OK) rc = encode(&maps.b[0], w_gate, I, E, E, width / 2);
  if (rc == MVPA_OK) rc = encode(&maps.b[1], w_up, I, E, E, width / 2);
  if (rc == MVPA_OK) rc = encode(&maps.out[0], h, M, I, ld_h, 32);
  if (saved != nullptr) {
    const Saved kept(saved, M, I);
    for (int i = 0; i < 2 && rc == MVPA_OK; ++i) {
      rc = encode(&maps.out[1 + i], kept.upper[i], M, I, I, 32);
      const uint64_t dims[2] = {(uint64_t)I, (uint64_t)M}, strides[1] = {(uint64_t)kept.ld};
      const uint32_t box[2] = {64, 32};
      if (rc == MVPA_OK)
        rc = encode_sw128(&maps.out[3 + i], CU_TENSOR_MAP_DATA_TYPE_UINT8, kept.lower[i], 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_64B);
    }
  }
  if (rc != MVPA_OK) return rc;
  const GatedArgs g = {tm, tiles_of(I, width / 2), tm, (int)tiles_of(E, 64), 1, (int)M, I, few, status, 1, 0, nullptr};
  cudaStream_t s = (cudaStream_t)cuda_stream;
  if (width == 128) return saved != nullptr ? launch_gated<kForwardSave, 128>(maps, g, s) : launch_gated<kForward, 128>(maps, g, s);
  return saved != nullptr ? launch_gated<kForwardSave, 256>(maps, g, s) : launch_gated<kForward, 256>(maps, g, s);
}

extern "C" size_t mvpa_gated_linear_bwd_workspace_bytes(int64_t M, int32_t E, int32_t I) {
  if (M < 1 || E < 1 || I < 1) return 0;
  return std::max(plan_dx(M, E, I, true).bytes, plan_dw(M, E, I, true).bytes);
}

extern "C" int mvpa_gated_linear_bwd(const void* dh, int64_t ld_dh, const void* saved, const void* x, int64_t ld_x, const void* w_gate,
                                     const void* w_up, void* dgate, void* dup, void* dx, void* dw_gate, void* dw_up, int64_t M, int32_t E,
                                     int32_t I, void* workspace, size_t workspace_bytes, int32_t* status, void* cuda_stream) {
  const int rc0 = check_sizes("mvpa_gated_linear_bwd", M, E, I);
  if (rc0 != MVPA_OK) return rc0;
  if (!rows_fit(dh, ld_dh, I) || saved == nullptr || (reinterpret_cast<uintptr_t>(saved) & 15) != 0 || !rows_fit(dgate, I, I) ||
      !rows_fit(dup, I, I) || (dx != nullptr && (!rows_fit(w_gate, E, E) || !rows_fit(w_up, E, E) || !rows_fit(dx, E, E))) ||
      (dw_gate == nullptr) != (dw_up == nullptr) ||
      (dw_gate != nullptr && (!rows_fit(x, ld_x, E) || !rows_fit(dw_gate, E, E) || !rows_fit(dw_up, E, E)))) {
    set_error("mvpa_gated_linear_bwd: every matrix must be 16-byte aligned with rows of a multiple of 16 bytes, not shorter than its width; "
              "dw_gate and dw_up are wanted both or neither");
    return MVPA_ERR_ALIGNMENT;
  }
  const Plan to_x = plan_dx(M, E, I, workspace != nullptr), to_w = plan_dw(M, E, I, workspace != nullptr);
  const size_t need = std::max(dx != nullptr ? to_x.bytes : 0, dw_gate != nullptr ? to_w.bytes : 0);
  if (workspace != nullptr && ((reinterpret_cast<uintptr_t>(workspace) & 15) != 0 || workspace_bytes < need)) {
    set_error("mvpa_gated_linear_bwd: the workspace needs %zu bytes on a 16-byte boundary (got %zu)", need, workspace_bytes);
    return MVPA_ERR_WORKSPACE;
  }
  cudaStream_t s = (cudaStream_t)cuda_stream;
  const int64_t ctas = (M * (I / 8) + 255) / 256, most = (int64_t)device_sm_count() * 16;
  MVPA_CUDA_CHECK(launch_dependent(1, gate_bwd_kernel, (unsigned)(ctas < most ? ctas : most), 256, 0, s, (const __nv_bfloat16*)dh, ld_dh,
                                   Saved(const_cast<void*>(saved), M, I), (__nv_bfloat16*)dgate, (__nv_bfloat16*)dup, M, (int)I));
  count_launch();
  MVPA_CUDA_CHECK(cudaGetLastError());
  int rc = MVPA_OK;
  if (dx != nullptr) {
    GatedMaps maps = {};
    const int few = few_rows(M), box = few > 0 ? few : 128;
    rc = encode(&maps.a[0], dgate, M, I, I, box);
    if (rc == MVPA_OK) rc = encode(&maps.a[1], dup, M, I, I, box);
    if (rc == MVPA_OK) rc = encode(&maps.b[0], w_gate, I, E, E, 64);
    if (rc == MVPA_OK) rc = encode(&maps.b[1], w_up, I, E, E, 64);
    if (rc == MVPA_OK) rc = encode(&maps.out[0], dx, M, E, E, 32);
    const uint32_t tm = tiles_of(M, 256);
    if (rc == MVPA_OK) rc = run_gated<kInput>(maps, {tm, 0, tm, (int)tiles_of(I, 64), 2, (int)M, E, few, status, 1, 0, nullptr}, to_x, (float*)workspace, dx, nullptr, s);
  }
  if (rc == MVPA_OK && dw_gate != nullptr) {
    GatedMaps maps = {};
    rc = encode(&maps.a[0], dgate, M, I, I, 64);
    if (rc == MVPA_OK) rc = encode(&maps.a[1], dup, M, I, I, 64);
    if (rc == MVPA_OK) rc = encode(&maps.b[0], x, M, E, ld_x, 64);
    if (rc == MVPA_OK) rc = encode(&maps.out[0], dw_gate, I, E, E, 32);
    if (rc == MVPA_OK) rc = encode(&maps.out[1], dw_up, I, E, E, 32);
    const uint32_t tm = tiles_of(I, 256);
    if (rc == MVPA_OK) rc = run_gated<kWeights>(maps, {2 * tm, 0, tm, (int)tiles_of(M, 64), 1, I, E, 0, status, 1, 0, nullptr}, to_w, (float*)workspace, dw_gate, dw_up, s);
  }
  return rc;
}
