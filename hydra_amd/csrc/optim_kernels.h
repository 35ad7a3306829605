// optim_kernels.h -- launcher declarations shared by the C-ABI (optim.cpp) and the kernels of the
// optimizer step (optim_kernels.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/hydra_optim.h"

namespace hydra {

constexpr int kOptBlock = 256;      // 4 waves of 64 lanes
constexpr int kMomentBlock = 256;   // elements that share one scale of an 8-bit moment
constexpr size_t kOptTile = 1024;   // elements of one tensor that a workgroup takes
constexpr uint32_t kMaxHead = 64;   // a head is one element per lane of one wave at most
constexpr int kNormBlocks = 2048;   // workgroups (and partial sums) of the norm, at most

// One tensor of a plan, in device memory.  `grad` counts from the bucket that a call gives (null:
// an address).  It has a tile for each kOptTile elements; tile k is number tile0 + k.  To the step it
// holds the elements [head + k * kOptTile, head + (k + 1) * kOptTile), the first one those before them
// too, the last one none at times: `head` puts the vectors of as many of its buffers as possible on
// their natural alignment, and their tiles on whole lines.  To the norm: [k * kOptTile, (k + 1) * kOptTile).
struct OptTensor {
  char* param;
  float* master;
  uint64_t grad;
  char* m;
  char* v;
  float* m_scale;
  float* v_scale;
  uint64_t n;
  float lr_scale, weight_decay;
  uint32_t tile0, index;
  uint32_t head, tiles;
};

// What a plan's launches need, on the host.
struct OptTable {
  const OptTensor* tensors;      // device
  const uint32_t* tile_tensor;   // device: the tensor of each tile
  uint32_t tiles;
  uint32_t filled;               // tensors that have elements
};

// A step's scalars: by value, or (ctrl) the device's.
struct OptStep {
  float beta1, omb1, beta2, omb2, eps;  // omb = 1 - beta, rounded once from fp64
  float lr, mult, inv_bc1, inv_sqrt_bc2;
  int64_t step;
  uint32_t seed_key;  // hash of the seed; stochastic: whether there is one
  uint32_t stochastic;
  const hydra_adamw_ctrl_t* ctrl;
};

struct OptNorm {
  double grad_scale, max_norm, beta1, beta2;
};

// murmur3's 32-bit finaliser
__host__ __device__ inline uint32_t fmix32(uint32_t h) {
  h ^= h >> 16;
  h *= 0x85EBCA6Bu;
  h ^= h >> 13;
  h *= 0xC2B2AE35u;
  return h ^ (h >> 16);
}

// beta^t by squaring, in fp64: at most 2 log2(t) roundings, the same on host and device
__host__ __device__ inline double power(double beta, uint64_t t) {
  double r = 1.0;
  for (; t; t >>= 1, beta *= beta)
    if (t & 1) r *= beta;
  return r;
}

hipError_t launch_adamw(const hydra_adamw_config_t& cfg, const OptTable& t, const OptStep& step,
                        const void* bucket, hipStream_t s);
size_t norm_workspace(const OptTable& t);  // bytes of partial sums
hipError_t launch_grad_norm(const hydra_adamw_config_t& cfg, const OptTable& t, const OptNorm& norm,
                            const void* bucket, hydra_adamw_ctrl_t* ctrl, double* partials,
                            hipStream_t s);
hipError_t launch_moments8_encode(int dtype, uint8_t* m8, float* m_scale, uint8_t* v8,
                                  float* v_scale, const void* m, const void* v, size_t n,
                                  hipStream_t s);
hipError_t launch_moments8_decode(int dtype, void* m, void* v, const uint8_t* m8,
                                  const float* m_scale, const uint8_t* v8, const float* v_scale,
                                  size_t n, hipStream_t s);

}  // namespace hydra
