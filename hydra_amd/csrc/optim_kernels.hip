// optim_kernels.hip -- gfx950 kernels of the optimizer step on a reduced gradient bucket
// (include/hydra_optim.h: the formulas and the 8-bit format).
//
// Every kernel here is a stream over HBM: AdamW moves 28 B per element with fp32 moments and 16
// with 8-bit ones, the norm 4 or 2, the moment conversions 10 to 14.  No reuse, no MFMA.
// A plan's tensors are cut into tiles; a workgroup finds its tile's tensor through a table with
// one entry per tile, so one launch serves any number of tensors.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "optim_kernels.h"
#include "reduce_ops.h"

namespace hydra {
namespace {

// ---- element types -----------------------------------------------------------------------------
// IEEE conversions (the reduction's f16_t keeps gloo's store quirk: not wanted here)
__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(bf16_t x) { return bf2f(x.x); }
__device__ __forceinline__ float widen(f16_t x) { return h2f(x.x); }
__device__ __forceinline__ void narrow(float x, float* out) { *out = x; }
__device__ __forceinline__ void narrow(float x, bf16_t* out) { out->x = f2bf(x); }
__device__ __forceinline__ void narrow(float x, f16_t* out) {
  out->x = __builtin_bit_cast(uint16_t, (_Float16)x);
}

// ---- 8-bit moments -------------------------------------------------------------------------------
// The code of t in [0, 1.875] is the top of its fp32 bits once the exponent is rebased to a 4-bit
// one: t * 2^-112 has exponent field 15 for t in [1, 2), and below 2^-14 it is an fp32 subnormal,
// so the gradual underflow costs nothing.  Adding r below the cut before shifting rounds: 16
// random bits stochastically (the neglected rest of the dropped bits shifts the probability by at
// most 2^-16), 0x8000 to nearest.  Largest code: 127 (m) and 254 (sqrt v), both 1.875.
constexpr float kTop = 1.0f / 1.875f;
constexpr float kTiny = 0x1p-100f;  // 1 / scale stays finite, and x / scale exact enough

__device__ __forceinline__ float moment_scale(float amax) { return amax < kTiny ? 0.0f : amax * kTop; }
__device__ __forceinline__ float moment_inv(float scale) { return scale > 0.0f ? 1.0f / scale : 0.0f; }
// a magnitude's part in its block's largest: not finite ones have none
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.0f;
}

__device__ __forceinline__ uint32_t encode_m(float m, float inv, uint32_t r16) {
  const float a = fabsf(m);
  const uint32_t c = min((fbits(a * inv * 0x1p-112f) + (r16 << 4)) >> 20, 127u);
  if (!(a < INFINITY)) return 0x80u;
  return c ? c | (m < 0.0f ? 0x80u : 0u) : 0u;
}
__device__ __forceinline__ uint32_t encode_root(float root, float inv, uint32_t r16) {
  const uint32_t c = min((fbits(root * inv * 0x1p-112f) + (r16 << 3)) >> 19, 254u);
  if (!(root < INFINITY)) return 255u;
  return root > 0.0f ? max(c, 1u) : 0u;
}
__device__ __forceinline__ float decode_m(uint32_t c, float scale) {
  const float a = bitsf((c & 127u) << 20) * 0x1p112f * scale;
  if (c == 0x80u) return __builtin_nanf("");
  return c & 0x80u ? -a : a;
}
__device__ __forceinline__ float decode_v(uint32_t c, float scale) {
  const float root = bitsf(c << 19) * 0x1p112f * scale;
  return c == 255u ? INFINITY : root * root;
}

// the largest of every thread's x (>= 0) over the workgroup
__device__ __forceinline__ float block_max(float x, float* lds) {
  for (int d = 32; d; d >>= 1) x = fmaxf(x, __shfl_xor(x, d));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  x = fmaxf(fmaxf(lds[0], lds[1]), fmaxf(lds[2], lds[3]));
  __syncthreads();
  return x;
}

// ---- AdamW -----------------------------------------------------------------------------------------
struct Scalars {  // one tensor's, in one step
  float mult, b1, omb1, b2, omb2, isb2, eps, decay, size;
  uint32_t key, stochastic;
};

__device__ __forceinline__ bool load_scalars(const OptStep& st, const OptTensor& T, Scalars* k) {
  float lr = st.lr, mult = st.mult, ib1 = st.inv_bc1, isb2 = st.inv_sqrt_bc2;
  int64_t step = st.step;
  if (st.ctrl) {
    if (st.ctrl->skip) return false;
    lr = st.ctrl->lr;
    mult = st.ctrl->mult;
    ib1 = st.ctrl->inv_bc1;
    isb2 = st.ctrl->inv_sqrt_bc2;
    step = st.ctrl->step;
  }
  lr *= T.lr_scale;
  *k = Scalars{mult, st.beta1, st.omb1, st.beta2, st.omb2, isb2, st.eps, 1.0f - lr * T.weight_decay,
               lr * ib1, 0u, st.stochastic};
  uint32_t h = fmix32(st.seed_key ^ (uint32_t)step);
  h = fmix32(h ^ (uint32_t)((uint64_t)step >> 32));
  k->key = fmix32(h ^ T.index);
  return true;
}

__device__ __forceinline__ void adamw(float& p, float grad, float& m, float& v, const Scalars& k) {
  const float g = grad * k.mult;
  m = m * k.b1 + g * k.omb1;
  v = v * k.b2 + (g * k.omb2) * g;
  const float denom = sqrtf(v) * k.isb2 + k.eps;
  p = p * k.decay - (m / denom) * k.size;
}

__device__ __forceinline__ uint32_t random_word(uint64_t i, uint32_t key) {
  return fmix32(((uint32_t)i * 0x9E3779B1u) ^ ((uint32_t)(i >> 32) * 0x85EBCA6Bu) ^ key);
}

template <typename P, typename G, bool MASTER, bool S8>
__global__ __launch_bounds__(kOptBlock) void k_adamw(const OptTensor* tensors,
                                                     const uint32_t* tile_tensor, OptStep st,
                                                     uint64_t bucket) {
  const OptTensor T = tensors[tile_tensor[blockIdx.x]];
  Scalars k;
  if (!load_scalars(st, T, &k)) return;
  __shared__ float lds[4];
  const uint64_t base = (uint64_t)(blockIdx.x - T.tile0) * kOptTile;
  const G* grad = reinterpret_cast<const G*>(bucket + T.grad);
  P* param = reinterpret_cast<P*>(T.param);
  for (uint64_t i0 = base; i0 < min(base + kOptTile, T.n); i0 += kOptBlock) {
    const uint64_t i = i0 + threadIdx.x;
    const bool on = i < T.n;
    float p = 0.0f, m = 0.0f, v = 0.0f;
    if (on) {
      p = MASTER ? T.master[i] : widen(param[i]);
      if constexpr (S8) {
        m = decode_m((uint8_t)T.m[i], T.m_scale[i / kMomentBlock]);
        v = decode_v((uint8_t)T.v[i], T.v_scale[i / kMomentBlock]);
      } else {
        m = reinterpret_cast<const float*>(T.m)[i];
        v = reinterpret_cast<const float*>(T.v)[i];
      }
      adamw(p, widen(grad[i]), m, v, k);
    }
    if constexpr (S8) {
      const float root = sqrtf(v);
      const float ms = moment_scale(block_max(finite_abs(m), lds));
      const float vs = moment_scale(block_max(finite_abs(root), lds));
      if (on) {
        const uint32_t r = k.stochastic ? random_word(i, k.key) : 0x80008000u;
        T.m[i] = (char)encode_m(m, moment_inv(ms), r & 0xffffu);
        T.v[i] = (char)encode_root(root, moment_inv(vs), r >> 16);
      }
      if (threadIdx.x == 0) {
        T.m_scale[i / kMomentBlock] = ms;
        T.v_scale[i / kMomentBlock] = vs;
      }
    } else if (on) {
      reinterpret_cast<float*>(T.m)[i] = m;
      reinterpret_cast<float*>(T.v)[i] = v;
    }
    if (on) {
      if constexpr (MASTER) T.master[i] = p;
      narrow(p, &param[i]);
    }
  }
}

// ---- the norm --------------------------------------------------------------------------------------
// fp64 sums: no gradient's square overflows, and the sum is not finite exactly when some gradient
// is not.  The order is the grid's, which the plan fixes.
__device__ __forceinline__ double block_sum(double x, double* lds) {
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

template <typename G>
__global__ __launch_bounds__(kOptBlock) void k_norm_partial(const OptTensor* tensors,
                                                            const uint32_t* tile_tensor,
                                                            uint32_t tiles, uint64_t bucket,
                                                            double* partials) {
  __shared__ double lds[4];
  double sum = 0.0;
  for (uint32_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const OptTensor& T = tensors[tile_tensor[tile]];
    const uint64_t base = (uint64_t)(tile - T.tile0) * kOptTile;
    const uint64_t end = min(base + kOptTile, T.n);
    const G* grad = reinterpret_cast<const G*>(bucket + T.grad);
    for (uint64_t i = base + threadIdx.x; i < end; i += kOptBlock) {
      const double g = widen(grad[i]);
      sum += g * g;
    }
  }
  sum = block_sum(sum, lds);
  if (threadIdx.x == 0) partials[blockIdx.x] = sum;
}

__device__ __forceinline__ void finish_norm(double sum, const OptNorm& a, hydra_adamw_ctrl_t* c) {
  const double norm = fabs(a.grad_scale) * sqrt(sum);
  const double clip = a.max_norm > 0.0 ? fmin(1.0, a.max_norm / (norm + 1e-6)) : 1.0;
  c->norm = (float)norm;
  c->mult = (float)(a.grad_scale * clip);
  const bool fine = sum < (double)INFINITY;
  c->skip = fine ? 0 : 1;
  if (!fine) {
    c->skipped += 1;
    return;
  }
  const int64_t t = c->step + 1;
  c->step = t;
  c->inv_bc1 = (float)(1.0 / (1.0 - power(a.beta1, (uint64_t)t)));
  c->inv_sqrt_bc2 = (float)(1.0 / sqrt(1.0 - power(a.beta2, (uint64_t)t)));
}

__global__ __launch_bounds__(kOptBlock) void k_norm_finish(const double* partials, uint32_t count,
                                                           OptNorm a, hydra_adamw_ctrl_t* ctrl) {
  __shared__ double lds[4];
  double sum = 0.0;
  for (uint32_t j = threadIdx.x; j < count; j += kOptBlock) sum += partials[j];
  sum = block_sum(sum, lds);
  if (threadIdx.x == 0) finish_norm(sum, a, ctrl);
}

// ---- 8-bit moments from and to values ---------------------------------------------------------------
template <typename E>
__global__ __launch_bounds__(kOptBlock) void k_encode(uint8_t* m8, float* ms, uint8_t* v8,
                                                      float* vs, const E* m, const E* v, size_t n) {
  __shared__ float lds[4];
  const size_t i = (size_t)blockIdx.x * kMomentBlock + threadIdx.x;
  const float x = m && i < n ? widen(m[i]) : 0.0f;
  const float root = v && i < n ? sqrtf(fabsf(widen(v[i]))) : 0.0f;
  const float sm = moment_scale(block_max(finite_abs(x), lds));
  const float sv = moment_scale(block_max(finite_abs(root), lds));
  if (i < n) {
    if (m) m8[i] = (uint8_t)encode_m(x, moment_inv(sm), 0x8000u);
    if (v) v8[i] = (uint8_t)encode_root(root, moment_inv(sv), 0x8000u);
  }
  if (threadIdx.x == 0) {
    if (m) ms[blockIdx.x] = sm;
    if (v) vs[blockIdx.x] = sv;
  }
}

template <typename E>
__global__ __launch_bounds__(kOptBlock) void k_decode(E* m, E* v, const uint8_t* m8,
                                                      const float* ms, const uint8_t* v8,
                                                      const float* vs, size_t n) {
  const size_t i = (size_t)blockIdx.x * kMomentBlock + threadIdx.x;
  if (i >= n) return;
  if (m) narrow(decode_m(m8[i], ms[blockIdx.x]), &m[i]);
  if (v) narrow(decode_v(v8[i], vs[blockIdx.x]), &v[i]);
}

// ---- launch ------------------------------------------------------------------------------------------
template <typename P, typename G, bool MASTER, bool S8>
hipError_t adamw_t(const OptTable& t, const OptStep& st, const void* bucket, hipStream_t s) {
  hipLaunchKernelGGL((k_adamw<P, G, MASTER, S8>), dim3(t.tiles), dim3(kOptBlock), 0, s, t.tensors,
                     t.tile_tensor, st, reinterpret_cast<uint64_t>(bucket));
  return hipGetLastError();
}

template <typename P, bool MASTER, bool S8>
hipError_t adamw_g(int grad, const OptTable& t, const OptStep& st, const void* b, hipStream_t s) {
  switch (grad) {
    case HYDRA_FLOAT32: return adamw_t<P, float, MASTER, S8>(t, st, b, s);
    case HYDRA_BFLOAT16: return adamw_t<P, bf16_t, MASTER, S8>(t, st, b, s);
    case HYDRA_FLOAT16: return adamw_t<P, f16_t, MASTER, S8>(t, st, b, s);
  }
  return hipErrorInvalidValue;
}

template <bool S8>
hipError_t adamw_p(const hydra_adamw_config_t& c, const OptTable& t, const OptStep& st,
                   const void* b, hipStream_t s) {
  const bool master = (c.flags & HYDRA_ADAMW_MASTER) != 0;
  switch (c.param_dtype) {
    case HYDRA_FLOAT32: return adamw_g<float, false, S8>(c.grad_dtype, t, st, b, s);
    case HYDRA_BFLOAT16:
      return master ? adamw_g<bf16_t, true, S8>(c.grad_dtype, t, st, b, s)
                    : adamw_g<bf16_t, false, S8>(c.grad_dtype, t, st, b, s);
    case HYDRA_FLOAT16:
      return master ? adamw_g<f16_t, true, S8>(c.grad_dtype, t, st, b, s)
                    : adamw_g<f16_t, false, S8>(c.grad_dtype, t, st, b, s);
  }
  return hipErrorInvalidValue;
}

template <typename G>
void norm_partial(const OptTable& t, const void* bucket, double* partials, hipStream_t s) {
  hipLaunchKernelGGL((k_norm_partial<G>), dim3(norm_partials(t.tiles)), dim3(kOptBlock), 0, s,
                     t.tensors, t.tile_tensor, t.tiles, reinterpret_cast<uint64_t>(bucket),
                     partials);
}

constexpr size_t kPart = size_t(1) << 30;  // elements of one launch, whole blocks
template <typename T>
T* after(T* p, size_t i) {  // the absent moment's pointers stay null
  return p ? p + i : p;
}

template <typename E>
hipError_t encode_t(uint8_t* m8, float* ms, uint8_t* v8, float* vs, const E* m, const E* v,
                    size_t n, hipStream_t s) {
  for (size_t at = 0; at < n; at += kPart) {
    const size_t part = std::min(n - at, kPart), row = at / kMomentBlock;
    hipLaunchKernelGGL((k_encode<E>), dim3((unsigned)((part + kMomentBlock - 1) / kMomentBlock)),
                       dim3(kOptBlock), 0, s, after(m8, at), after(ms, row), after(v8, at),
                       after(vs, row), after(m, at), after(v, at), part);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <typename E>
hipError_t decode_t(E* m, E* v, const uint8_t* m8, const float* ms, const uint8_t* v8,
                    const float* vs, size_t n, hipStream_t s) {
  for (size_t at = 0; at < n; at += kPart) {
    const size_t part = std::min(n - at, kPart), row = at / kMomentBlock;
    hipLaunchKernelGGL((k_decode<E>), dim3((unsigned)((part + kMomentBlock - 1) / kMomentBlock)),
                       dim3(kOptBlock), 0, s, after(m, at), after(v, at), after(m8, at),
                       after(ms, row), after(v8, at), after(vs, row), part);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace

hipError_t launch_adamw(const hydra_adamw_config_t& cfg, const OptTable& t, const OptStep& st,
                        const void* bucket, hipStream_t s) {
  if (t.tiles == 0) return hipSuccess;
  return cfg.state_dtype == HYDRA_UINT8 ? adamw_p<true>(cfg, t, st, bucket, s)
                                        : adamw_p<false>(cfg, t, st, bucket, s);
}

uint32_t norm_partials(uint32_t tiles) { return std::max(1u, std::min(tiles, (uint32_t)kNormBlocks)); }

hipError_t launch_grad_norm(int grad_dtype, const OptTable& t, const OptNorm& norm,
                            const void* bucket, hydra_adamw_ctrl_t* ctrl, double* partials,
                            hipStream_t s) {
  switch (grad_dtype) {
    case HYDRA_FLOAT32: norm_partial<float>(t, bucket, partials, s); break;
    case HYDRA_BFLOAT16: norm_partial<bf16_t>(t, bucket, partials, s); break;
    case HYDRA_FLOAT16: norm_partial<f16_t>(t, bucket, partials, s); break;
    default: return hipErrorInvalidValue;
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(k_norm_finish, dim3(1), dim3(kOptBlock), 0, s, partials,
                     norm_partials(t.tiles), norm, ctrl);
  return hipGetLastError();
}

hipError_t launch_moments8_encode(int dtype, uint8_t* m8, float* ms, uint8_t* v8, float* vs,
                                  const void* m, const void* v, size_t n, hipStream_t s) {
  if (dtype == HYDRA_FLOAT32)
    return encode_t(m8, ms, v8, vs, static_cast<const float*>(m), static_cast<const float*>(v), n, s);
  return encode_t(m8, ms, v8, vs, static_cast<const bf16_t*>(m), static_cast<const bf16_t*>(v), n, s);
}

hipError_t launch_moments8_decode(int dtype, void* m, void* v, const uint8_t* m8, const float* ms,
                                  const uint8_t* v8, const float* vs, size_t n, hipStream_t s) {
  if (dtype == HYDRA_FLOAT32)
    return decode_t(static_cast<float*>(m), static_cast<float*>(v), m8, ms, v8, vs, n, s);
  return decode_t(static_cast<bf16_t*>(m), static_cast<bf16_t*>(v), m8, ms, v8, vs, n, s);
}

}  // namespace hydra
