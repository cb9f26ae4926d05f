// What the matrix products of pairs of CTAs (and their host sides) share: the order of the tiles, rings of stages, and what is
// asked of a device once.
#pragma once
#include <stdint.h>

#include "tc_ptx.cuh"

namespace mvpa {
namespace {

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

}  // namespace
}  // namespace mvpa
