// optim_kernels.hip -- gfx950 kernels of the optimizer step on a reduced gradient bucket
// (include/hydra_optim.h: the formulas and the 8-bit format).
//
// Every kernel here is a stream over HBM: AdamW moves 28 B per element with fp32 moments and 16
// with 8-bit ones, the norm 4 or 2, the conversions of both moments 10 (from fp32) and 6 (to bf16).
// No reuse, no MFMA; what bounds them is the rate at which HBM takes mixed reads and writes (a copy
// 6.3 TB/s, reads alone 6.8), and for 8-bit moments nearly the vector units too (62 issue slots per
// element, 106 us for 64 Mi elements if nothing else ran).
// A plan's tensors are cut into tiles of 1024 elements, one workgroup each (64 Mi fp32: 4096 elements
// by a loop took 346 us where one turn took 320).  A workgroup finds its tile's tensor through a table
// with one entry per tile, so one launch serves any number of tensors; a single tensor's descriptor
// passed in the launch itself was no faster.
// Times below are of whole calls in sequence on rotating buffers, us, unless a kernel is named.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "optim_kernels.h"
#include "reduce_ops.h"

namespace hydra {
namespace {

// ---- 8-bit moments -------------------------------------------------------------------------------
// The code of t in [0, 1.875] is the top of its fp32 bits once the exponent is rebased to a 4-bit
// one: t * 2^-112 has exponent field 15 for t in [1, 2), and below 2^-14 it is an fp32 subnormal,
// so the gradual underflow costs nothing: x / s is then a multiple of 2^-37, rounded once from the
// product with fp32's 1 / s.  Adding r below the cut before shifting rounds: 16
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

// a * inv * 2^-112 rounded once, whatever inv is (in fp64 the products are exact)
__device__ __forceinline__ uint32_t rebased(float a, float inv) {
  return fbits((float)((double)a * inv * 0x1p-112));
}

__device__ __forceinline__ uint32_t encode_m(float m, float inv, uint32_t r16) {
  const float a = fabsf(m);
  const uint32_t c = min((rebased(a, inv) + (r16 << 4)) >> 20, 127u);
  if (!(a < INFINITY)) return 0x80u;
  return c ? c | (m < 0.0f ? 0x80u : 0u) : 0u;
}
__device__ __forceinline__ uint32_t encode_root(float root, float inv, uint32_t r16) {
  const uint32_t c = min((rebased(root, inv) + (r16 << 3)) >> 19, 254u);
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

// ---- memory ----------------------------------------------------------------------------------------
// Global memory by a wave-uniform base and a lane's byte offset.  Pointers that come out of a
// plan's table have to be said to be global: the compiler cannot see it, and flat accesses would
// also occupy the LDS counters.
#define GLOBAL __attribute__((address_space(1)))
typedef GLOBAL char* gptr;
__device__ __forceinline__ gptr global(const void* p) { return (gptr)(uint64_t)p; }
// Four consecutive elements of any alignment (that of the element): tensors are views into buckets.
// gfx950 runs in unaligned access mode, so these stay single 16-, 8- and 4-byte accesses.
typedef uint32_t w4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t w4h __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t w2 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t w2b __attribute__((ext_vector_type(2), aligned(1)));
typedef uint32_t w1 __attribute__((aligned(1)));
typedef float f4 __attribute__((ext_vector_type(4)));
// Nontemporal both ways: a step's state is larger than the caches.  64 Mi fp32 322, plain loads 350,
// plain stores 347; with 8-bit moments 235, 257 and 271.
template <typename V>
__device__ __forceinline__ V ldv(gptr p, uint32_t off) {
  return __builtin_nontemporal_load((const GLOBAL V*)(p + off));
}
template <typename V>
__device__ __forceinline__ void stv(gptr p, uint32_t off, V x) {
  __builtin_nontemporal_store(x, (GLOBAL V*)(p + off));
}
// x as fp32 rounded it: joined with the operation before it, the conversion to fp16 would become one
// mixed-precision instruction that rounds once
__device__ __forceinline__ float settled(float x) {
  asm("" : "+v"(x));
  return x;
}

// Element i of a tensor of E, and the four from i on.
template <typename E> struct At;
template <> struct At<float> {
  __device__ __forceinline__ static float load(gptr p, uint32_t i) { return *(const GLOBAL float*)(p + i * 4); }
  __device__ __forceinline__ static void store(gptr p, uint32_t i, float x) { *(GLOBAL float*)(p + i * 4) = x; }
  typedef w4 raw;
  __device__ __forceinline__ static raw load4(gptr p, uint32_t i) { return ldv<w4>(p, i * 4); }
  __device__ __forceinline__ static f4 wide(raw r) {
    return f4{bitsf(r[0]), bitsf(r[1]), bitsf(r[2]), bitsf(r[3])};
  }
  __device__ __forceinline__ static void store4(gptr p, uint32_t i, f4 x) {
    stv<w4>(p, i * 4, w4{fbits(x[0]), fbits(x[1]), fbits(x[2]), fbits(x[3])});
  }
  __device__ __forceinline__ static void store8(gptr p, uint32_t i, f4 x, f4 y) {
    store4(p, i, x);
    store4(p, i + 4, y);
  }
};
template <> struct At<bf16_t> {
  __device__ __forceinline__ static float load(gptr p, uint32_t i) { return bf2f(*(const GLOBAL uint16_t*)(p + i * 2)); }
  __device__ __forceinline__ static void store(gptr p, uint32_t i, float x) {
    *(GLOBAL uint16_t*)(p + i * 2) = __builtin_bit_cast(uint16_t, (__bf16)x);
  }
  typedef w2 raw;
  __device__ __forceinline__ static raw load4(gptr p, uint32_t i) { return ldv<w2>(p, i * 2); }
  __device__ __forceinline__ static f4 wide(raw r) {
    return f4{bitsf(r[0] << 16), bitsf(r[0] & 0xffff0000u), bitsf(r[1] << 16), bitsf(r[1] & 0xffff0000u)};
  }
  __device__ __forceinline__ static uint32_t pair(float x, float y) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, b2{(__bf16)x, (__bf16)y});
  }
  __device__ __forceinline__ static void store4(gptr p, uint32_t i, f4 x) {
    stv<w2>(p, i * 2, w2{pair(x[0], x[1]), pair(x[2], x[3])});
  }
  __device__ __forceinline__ static void store8(gptr p, uint32_t i, f4 x, f4 y) {
    stv<w4h>(p, i * 2, w4h{pair(x[0], x[1]), pair(x[2], x[3]), pair(y[0], y[1]), pair(y[2], y[3])});
  }
};
template <> struct At<f16_t> {
  __device__ __forceinline__ static float load(gptr p, uint32_t i) { return h2f(*(const GLOBAL uint16_t*)(p + i * 2)); }
  __device__ __forceinline__ static void store(gptr p, uint32_t i, float x) {
    *(GLOBAL uint16_t*)(p + i * 2) = __builtin_bit_cast(uint16_t, (_Float16)settled(x));
  }
  typedef w2 raw;
  __device__ __forceinline__ static raw load4(gptr p, uint32_t i) { return ldv<w2>(p, i * 2); }
  __device__ __forceinline__ static f4 wide(raw r) {
    return f4{h2f((uint16_t)r[0]), h2f((uint16_t)(r[0] >> 16)), h2f((uint16_t)r[1]), h2f((uint16_t)(r[1] >> 16))};
  }
  __device__ __forceinline__ static void store4(gptr p, uint32_t i, f4 x) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 lo{(_Float16)settled(x[0]), (_Float16)settled(x[1])};
    const h2 hi{(_Float16)settled(x[2]), (_Float16)settled(x[3])};
    stv<w2>(p, i * 2, w2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)});
  }
};
// bytes
__device__ __forceinline__ uint32_t load_byte(gptr p, uint32_t i) { return *(const GLOBAL uint8_t*)(p + i); }
__device__ __forceinline__ void store_byte(gptr p, uint32_t i, uint32_t x) { *(GLOBAL uint8_t*)(p + i) = (uint8_t)x; }
// elements from i on
__device__ __forceinline__ uint32_t rest(uint32_t left, uint32_t i) { return left > i ? left - i : 0u; }
// the first `count` (0 to 4) of four
template <typename E>
__device__ __forceinline__ f4 load_upto4(gptr p, uint32_t i, uint32_t count) {
  if (count >= 4) return At<E>::wide(At<E>::load4(p, i));
  f4 x = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < 4; j++)
    if ((uint32_t)j < count) x[j] = At<E>::load(p, i + j);
  return x;
}
template <typename E>
__device__ __forceinline__ void store_upto4(gptr p, uint32_t i, f4 x, uint32_t count) {
  if (count >= 4) {
    At<E>::store4(p, i, x);
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; j++)
    if ((uint32_t)j < count) At<E>::store(p, i + j, x[j]);
}
__device__ __forceinline__ uint32_t load_bytes(gptr p, uint32_t i, uint32_t count) {
  if (count >= 4) return ldv<w1>(p, i);
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; j++)
    if ((uint32_t)j < count) w |= load_byte(p, i + j) << (8 * j);
  return w;
}
__device__ __forceinline__ void store_bytes(gptr p, uint32_t i, uint32_t w, uint32_t count) {
  if (count >= 4) {  // not nontemporal: 4 bytes per lane join in the cache (64 Mi both ways 175, else 186)
    *(GLOBAL w1*)(p + i) = w;
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; j++)
    if ((uint32_t)j < count) store_byte(p, i + j, w >> (8 * j));
}

// Workgroups are dealt to the 8 XCDs in turn: tile numbers so that each XCD streams one contiguous
// eighth of the tiles.
__device__ __forceinline__ uint32_t xcd_tile(uint32_t b, uint32_t tiles) {
  const uint32_t x = b & 7, q = tiles >> 3, r = tiles & 7;
  return x * q + min(x, r) + (b >> 3);
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

__device__ __forceinline__ void moments(float g, float& m, float& v, const Scalars& k) {
  m = m * k.b1 + g * k.omb1;
  v = v * k.b2 + (g * k.omb2) * g;
}
__device__ __forceinline__ float weight(float p, float m, float v, const Scalars& k) {
  return p * k.decay - (m / (sqrtf(v) * k.isb2 + k.eps)) * k.size;
}
__device__ __forceinline__ void adamw(float& p, float grad, float& m, float& v, const Scalars& k) {
  moments(grad * k.mult, m, v, k);
  p = weight(p, m, v, k);
}

// fp32 moments: a workgroup takes one tile, 4 elements per lane.  Tiles in launch order: dealing each
// XCD a contiguous eighth took 1287 instead of 1265 (256 Mi, bf16 with master), though 312 instead of
// 322 for one 64 Mi buffer.  The kernel alone: 296 to 305 us for 64 Mi fp32 (6.2 to 6.35 TB/s), 1240 to
// 1253 for the 256 Mi (6.0), 95 to 97 for 291 ragged tensors' 624 MB.
// fp32 square root and quotient are IEEE's: replacing both by the hardware's estimates gained nothing.
template <typename P, typename G, bool MASTER>
__global__ __launch_bounds__(kOptBlock) void k_adamw(const OptTensor* tensors,
                                                     const uint32_t* tile_tensor, OptStep st,
                                                     uint64_t bucket) {
  const uint32_t tile = blockIdx.x;
  const OptTensor T = tensors[tile_tensor[tile]];
  Scalars k;
  if (!load_scalars(st, T, &k)) return;
  const uint64_t base = T.head + (uint64_t)(tile - T.tile0) * kOptTile;
  const uint32_t left = T.n > base ? (uint32_t)min(T.n - base, (uint64_t)kOptTile) : 0u;
  const gptr grad = global((const void*)(bucket + T.grad)) + base * sizeof(G);
  const gptr param = global(T.param) + base * sizeof(P), master = global(T.master) + base * 4;
  const gptr mm = global(T.m) + base * 4, vv = global(T.v) + base * 4;
  const uint32_t i = threadIdx.x * 4;
  if (i + 4 <= left) {
    typename At<P>::raw p;
    w4 w;
    if (MASTER) w = At<float>::load4(master, i);
    else p = At<P>::load4(param, i);
    const f4 y = At<G>::wide(At<G>::load4(grad, i));
    f4 a = At<float>::wide(At<float>::load4(mm, i)), b = At<float>::wide(At<float>::load4(vv, i));
    f4 x = MASTER ? At<float>::wide(w) : At<P>::wide(p);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      float xj = x[j], aj = a[j], bj = b[j];
      adamw(xj, y[j], aj, bj, k);
      x[j] = xj, a[j] = aj, b[j] = bj;
    }
    if (MASTER) At<float>::store4(master, i, x);
    At<P>::store4(param, i, x);
    At<float>::store4(mm, i, a);
    At<float>::store4(vv, i, b);
  }
  // the tensor's ragged ends, one element per lane: those before the first tile's vectors (wave 0) and
  // up to 3 after the last one's (wave 1)
  static_assert(kMaxHead <= 64, "one wave takes the head");
  const uint32_t before = tile == T.tile0 ? T.head : 0u, after = left & 3;
  if (before | after) {
    const uint32_t t = threadIdx.x;
    int64_t e;
    if (t < before) e = (int64_t)t - before;
    else if (t >= 64 && t - 64 < after) e = left - after + (t - 64);
    else return;
    const gptr m1 = mm + e * 4, v1 = vv + e * 4, p1 = param + e * (int64_t)sizeof(P), w1 = master + e * 4;
    float p = MASTER ? At<float>::load(w1, 0) : At<P>::load(p1, 0);
    float m = At<float>::load(m1, 0), v = At<float>::load(v1, 0);
    adamw(p, At<G>::load(grad + e * (int64_t)sizeof(G), 0), m, v, k);
    At<float>::store(m1, 0, m);
    At<float>::store(v1, 0, v);
    if (MASTER) At<float>::store(w1, 0, p);
    At<P>::store(p1, 0, p);
  }
}

// 8-bit moments: a workgroup takes one tile, a wave one block of 256 elements of it, 4 per lane, so a
// block's scales are wave-uniform.  The kernel alone: 164 us for 64 Mi fp32 (1078 MB, 6.6 TB/s: some of
// the bytes of the last call are still in the Infinity Cache), 231 for 397 tensors of 100 M elements in
// bf16 with master.  Each XCD a contiguous eighth of the tiles: 235 with what follows it, in launch
// order 239; the ragged tensors 371 and 386.
static_assert(kOptTile == kOptBlock * 4 && kOptTile == kOptBlock / 64 * kMomentBlock, "one turn");
// lanes 31 and 63: the largest of their half of the wave
__device__ __forceinline__ uint32_t half_wave_umax(uint32_t x) {
#define HYDRA_DPP_MAX(ctrl) x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, 0xf, 0xf, true))
  HYDRA_DPP_MAX(0x111);  // row_shr:1
  HYDRA_DPP_MAX(0x112);
  HYDRA_DPP_MAX(0x114);
  HYDRA_DPP_MAX(0x118);
  HYDRA_DPP_MAX(0x142);  // row_bcast:15
#undef HYDRA_DPP_MAX
  return x;
}
// lane 31: the wave's largest a, lane 63: its largest b (the halves of a meet in lanes 0-31, those of
// b in the others)
__device__ __forceinline__ uint32_t wave_umax_pair(uint32_t a, uint32_t b) {
  const auto s = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  return half_wave_umax(max((uint32_t)s[0], (uint32_t)s[1]));
}
// c + (low / high half of r) * 16 or * 8: the 16 random bits at the top of what the cut drops
__device__ __forceinline__ uint32_t add_low16(uint32_t c, uint32_t r) {
  uint32_t d;
  asm("v_mad_u32_u16 %0, %1, 16, %2" : "=v"(d) : "v"(r), "v"(c));
  return d;
}
__device__ __forceinline__ uint32_t add_high16(uint32_t c, uint32_t r) {
  uint32_t d;
  asm("v_mad_u32_u16 %0, %1, 8, %2 op_sel:[1,0,0,0]" : "=v"(d) : "v"(r), "v"(c));
  return d;
}
// The square root of v in [0, 2^28], rounded as sqrtf rounds it (all of them checked against it), in 10
// issue slots instead of 17: of w = v * 2^96, which is normal and whose w - s^2 is exact, the reciprocal
// root's estimate s, then s + (w - s^2) / (2 s).  What lies above or is not finite becomes something not
// below 2^14, or a NaN.
__device__ __forceinline__ float plain_sqrt(float v) {
  const float w = v * 0x1p96f;
  const float r = __builtin_amdgcn_rsqf(fmaxf(w, 0x1p-126f));
  const float s = w * r;
  return fmaf(fmaf(-s, s, w), 0.5f * r, s) * 0x1p-48f;
}
// What a block's largest magnitude (its bits) has to be for the encoders below: 2^-112 / scale is
// normal, and every value is finite.  sqrt v also 0, or not below 2^-43: under such a one a v of fewer
// than 256 of fp32's smallest steps has the byte 1, and a minimum with its bits leaves every byte.
__device__ __forceinline__ bool plain_m(uint32_t top) { return top < fbits(0x1p14f); }
__device__ __forceinline__ bool plain_root(uint32_t top) {
  return top == 0 || top - fbits(0x1p-43f) < fbits(0x1p14f) - fbits(0x1p-43f);
}
// 2^-112 / scale (0 for an empty block): exact, so a product with it is rounded as in `rebased`
__device__ __forceinline__ float plain_inv(float scale) { return moment_inv(scale) * 0x1p-112f; }
// The bytes of four values of plain blocks; add(c, j) rounds c by the random bits of element j.
template <typename F>
__device__ __forceinline__ uint32_t encode4_m(f4 m, float inv, F add) {
  uint32_t c[4];
#pragma unroll
  for (int j = 0; j < 4; j++) c[j] = min(add(fbits(fabsf(m[j]) * inv), j) >> 20, 127u);
  const uint32_t w = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
  // the four signs, but not of zeros
  const uint32_t signs = __builtin_amdgcn_perm(fbits(m[3]), fbits(m[2]), 0x07030c0cu) |
                         __builtin_amdgcn_perm(fbits(m[1]), fbits(m[0]), 0x0c0c0703u);
  return w | (signs & (w + 0x7f7f7f7fu) & 0x80808080u);
}
template <typename F>
__device__ __forceinline__ uint32_t encode4_root(f4 root, f4 v, float inv, F add) {
  uint32_t c[4];
#pragma unroll
  for (int j = 0; j < 4; j++)  // 0 for v = 0 alone
    c[j] = min(min(max(add(fbits(root[j] * inv), j) >> 19, 1u), 254u), fbits(v[j]));
  return c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
}
__device__ __forceinline__ uint32_t zero_bytes(uint32_t x) {  // not 0 where x has a byte of 0
  return (x - 0x01010101u) & ~x & 0x80808080u;
}
__device__ __forceinline__ float uniform(float x, int lane) {
  return bitsf((uint32_t)__builtin_amdgcn_readlane((int)fbits(x), lane));
}

// A block's four elements per lane: decode, step, encode.  The vector units have 91 issue slots per
// element while HBM delivers its 16 bytes; this takes 62 (counted in the assembly; with an IEEE
// quotient in p's update the kernel took 170 us instead of 164).  The bytes are those of the documented
// operations, each rounded to fp32.  Decoding is short where no byte stands for something not finite
// and both old scales are below 2^15 (2^112 * scale is finite: one product per value).  The rest is
// short where the block is plain (above) and eps lies in [2^-40, 2^60]: the quotient is then a product
// with the hardware's reciprocal (2 ulp), both of them normal.
template <typename P, typename G, bool MASTER>
__device__ __forceinline__ void block8(gptr master, gptr param, gptr grad, gptr m8, gptr v8,
                                       gptr ms, gptr vs, uint32_t left, uint32_t lane,
                                       uint32_t rnd, uint32_t rkey, const Scalars& k) {
  // the pointers are the block's; left: elements from there to the tensor's end
  const bool whole = left >= kMomentBlock;
  const uint32_t count = rest(left, lane * 4);
  const uint32_t i = lane * 4;
  f4 p, g;
  uint32_t cm, cv;
  if (whole) {
    p = MASTER ? At<float>::wide(At<float>::load4(master, i)) : At<P>::wide(At<P>::load4(param, i));
    g = At<G>::wide(At<G>::load4(grad, i));
    cm = ldv<w1>(m8, i);
    cv = ldv<w1>(v8, i);
  } else {
    p = MASTER ? load_upto4<float>(master, i, count) : load_upto4<P>(param, i, count);
    g = load_upto4<G>(grad, i, count);
    cm = load_bytes(m8, i, count);
    cv = load_bytes(v8, i, count);
  }
  const float ms0 = At<float>::load(ms, 0), vs0 = At<float>::load(vs, 0);
  f4 m, v, root;
  const bool odd = !(ms0 < 0x1p15f && vs0 < 0x1p15f) ||
                   __any((zero_bytes(cm ^ 0x80808080u) | zero_bytes(~cv)) != 0);
  if (odd) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      m[j] = decode_m((cm >> (8 * j)) & 255u, ms0);
      v[j] = decode_v((cv >> (8 * j)) & 255u, vs0);
    }
  } else {
    const float sm = ms0 * 0x1p112f, sv = vs0 * 0x1p112f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      m[j] = bitsf((uint32_t)((int)(int8_t)(cm >> (8 * j)) << 20) & 0x87f00000u) * sm;
      const float r0 = bitsf(((cv >> (8 * j)) & 255u) << 19) * sv;
      v[j] = r0 * r0;
    }
  }
  uint32_t ar = 0;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    float mj = m[j], vj = v[j];
    moments(g[j] * k.mult, mj, vj, k);
    m[j] = mj, v[j] = vj;
    root[j] = plain_sqrt(vj);
    ar = max(ar, fbits(root[j]));
  }
  // (a NaN among m, which the maximum passes over, has an infinite or a NaN v beside it, or was odd)
  const uint32_t am = fbits(fmaxf(fmaxf(fabsf(m[0]), fabsf(m[1])), fmaxf(fabsf(m[2]), fabsf(m[3]))));
  const uint32_t top = wave_umax_pair(am, ar);
  const uint32_t tm = (uint32_t)__builtin_amdgcn_readlane((int)top, 31);
  const uint32_t tr = (uint32_t)__builtin_amdgcn_readlane((int)top, 63);
  float scale;
  uint32_t r[4], wm, wv;
#pragma unroll
  for (int j = 0; j < 4; j++) r[j] = 0x80008000u;
  if (k.stochastic) {
#pragma unroll
    for (int j = 0; j < 4; j++) r[j] = fmix32((rnd + j * 0x9E3779B1u) ^ rkey);
  }
  if (!odd && plain_m(tm) && plain_root(tr) && k.eps >= 0x1p-40f && k.eps <= 0x1p60f) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float denom = fmaf(root[j], k.isb2, k.eps);
      p[j] = fmaf(m[j] * __builtin_amdgcn_rcpf(denom), -k.size, p[j] * k.decay);
    }
    scale = moment_scale(bitsf(top));
    const float inv = plain_inv(scale);
    wm = encode4_m(m, uniform(inv, 31), [&](uint32_t c, int j) { return add_low16(c, r[j]); });
    wv = encode4_root(root, v, uniform(inv, 63), [&](uint32_t c, int j) { return add_high16(c, r[j]); });
  } else {
    float fm = 0.0f, fr = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      p[j] = weight(p[j], m[j], v[j], k);
      root[j] = sqrtf(v[j]);
      fm = fmaxf(fm, finite_abs(m[j]));
      fr = fmaxf(fr, finite_abs(root[j]));
    }
    scale = moment_scale(bitsf(wave_umax_pair(fbits(fm), fbits(fr))));
    const float im = moment_inv(uniform(scale, 31)), iv = moment_inv(uniform(scale, 63));
    wm = wv = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      wm |= encode_m(m[j], im, r[j] & 0xffffu) << (8 * j);
      wv |= encode_root(root[j], iv, r[j] >> 16) << (8 * j);
    }
  }
  if ((lane & 31) == 31) At<float>::store(lane & 32 ? vs : ms, 0, scale);
  if (whole) {
    if (MASTER) At<float>::store4(master, i, p);
    At<P>::store4(param, i, p);
    store_bytes(m8, i, wm, 4);
    store_bytes(v8, i, wv, 4);
  } else {
    if (MASTER) store_upto4<float>(master, i, p, count);
    store_upto4<P>(param, i, p, count);
    store_bytes(m8, i, wm, count);
    store_bytes(v8, i, wv, count);
  }
}

template <typename P, typename G, bool MASTER>
__global__ __launch_bounds__(kOptBlock) void k_adamw8(const OptTensor* tensors,
                                                      const uint32_t* tile_tensor, uint32_t tiles,
                                                      OptStep st, uint64_t bucket) {
  const uint32_t tile = xcd_tile(blockIdx.x, tiles);
  const OptTensor T = tensors[tile_tensor[tile]];
  Scalars k;
  if (!load_scalars(st, T, &k)) return;
  const uint32_t lane = threadIdx.x & 63;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint64_t base = (uint64_t)(tile - T.tile0) * kOptTile;
  const uint32_t left = (uint32_t)min(T.n - base, (uint64_t)kOptTile);
  const uint32_t i0 = wave * kMomentBlock;
  if (i0 >= left) return;  // whole waves
  const uint64_t at = base + i0;  // the wave's block
  const uint32_t rnd = ((uint32_t)at + lane * 4) * 0x9E3779B1u;
  const uint32_t rkey = k.key ^ ((uint32_t)(at >> 32) * 0x85EBCA6Bu);
  const gptr master = global(T.master) + at * 4, param = global(T.param) + at * sizeof(P);
  const gptr grad = global((const void*)(bucket + T.grad)) + at * sizeof(G);
  const gptr m8 = global(T.m) + at, v8 = global(T.v) + at;
  const gptr ms = global(T.m_scale) + at / kMomentBlock * 4;
  const gptr vs = global(T.v_scale) + at / kMomentBlock * 4;
  block8<P, G, MASTER>(master, param, grad, m8, v8, ms, vs, left - i0, lane, rnd, rkey, k);
}

// ---- the norm --------------------------------------------------------------------------------------
// fp64 sums: no gradient's square overflows, and the sum is not finite exactly when some gradient
// is not.  The order is that of the elements' numbers, whatever the addresses: a tensor's tiles count
// from its first element, a tile's vectors go to the threads by their number, and workgroup b sums a
// contiguous run of tiles, cut by the tensors' lengths alone.  One workgroup adds the sums in a second
// launch (4.5 us, nearly all of it the launch; the workgroups counting their arrivals in the first one
// instead cost 9 us more for 1024 of them, 36 where the count also writes the caches back).  A small plan
// is one workgroup's, in one launch.  That takes, beside 6.5 to 6.7 us for two launches at every one of
// these sizes: one fp32 tensor of 16 tiles 3.8, 48 5.1, 64 5.9, 80 6.7, 96 7.5 (bf16: 80 5.6, 112 6.7);
// 4 tensors of a tile 4.1, 8 5.8, 9 6.2, 10 6.7, 12 7.5; 7 of 4 tiles 5.4.
constexpr int kNormAloneBlock = 1024;
bool norm_alone(const OptTable& t) { return t.tiles + 8 * (uint64_t)t.filled <= 88; }

template <int BS>
__device__ __forceinline__ double block_sum(double x, double* lds) {
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  x = 0.0;
#pragma unroll
  for (int w = 0; w < BS / 64; w++) x += lds[w];
  return x;
}

// The step's scalars from the sum of squares: three threads of different waves at once.  t: read from
// ctrl by every thread before the barrier of the last sum.
__device__ __forceinline__ void finish_norm(double sum, uint64_t t, const OptNorm& a, hydra_adamw_ctrl_t* c) {
  const bool fine = sum < (double)INFINITY;
  if (threadIdx.x == 0) {
    const double norm = fabs(a.grad_scale) * sqrt(sum);
    const double clip = a.max_norm > 0.0 ? fmin(1.0, a.max_norm / (norm + 1e-6)) : 1.0;
    c->norm = (float)norm;
    c->mult = (float)(a.grad_scale * clip);
    c->skip = fine ? 0 : 1;
    if (fine) c->step = (int64_t)t;
    else c->skipped += 1;
  } else if (threadIdx.x == 64 && fine) {
    c->inv_bc1 = (float)(1.0 / (1.0 - power(a.beta1, t)));
  } else if (threadIdx.x == 128 && fine) {
    c->inv_sqrt_bc2 = (float)(1.0 / sqrt(1.0 - power(a.beta2, t)));
  }
}

// the squares of a dword's gradients
template <typename G>
__device__ __forceinline__ void add_squares(uint32_t w, double& sum) {
  if constexpr (sizeof(G) == 4) {
    const double g = bitsf(w);
    sum = fma(g, g, sum);
  } else {
    constexpr bool half = std::is_same<G, f16_t>::value;
    const double a = half ? h2f((uint16_t)w) : bitsf(w << 16);
    const double b = half ? h2f((uint16_t)(w >> 16)) : bitsf(w & 0xffff0000u);
    sum = fma(a, a, sum);
    sum = fma(b, b, sum);
  }
}

// The thread's vector of `left` ones, at any alignment of its elements.  16-bit elements whose pairs
// lie across memory's dwords (`odd`) are loaded by whole dwords from the second one on, and the first
// one is the last half of the lane before (of its own load in a wave's first lane): 100 M bf16 elements
// 37.4 us so, 44.4 by loads across the dwords, 36.3 at other offsets.
struct Sixteen {
  w4 d;
  uint32_t first;
};
template <typename G, bool KEEP>
__device__ __forceinline__ Sixteen load_sixteen(gptr at, uint64_t left, bool odd) {
  Sixteen x{{0, 0, 0, 0}, 0};
  if (threadIdx.x >= left) return x;
  const uint32_t o = threadIdx.x * 16;
  if (sizeof(G) == 4 || !odd) {
    x.d = KEEP ? *(const GLOBAL w4*)(at + o) : ldv<w4>(at, o);
    return x;
  }
  if (threadIdx.x + 1 < left) {
    x.d = KEEP ? *(const GLOBAL w4*)(at + o + 2) : ldv<w4>(at, o + 2);
  } else {  // nothing behind the last vector is read
    for (int j = 0; j < 3; j++) x.d[j] = *(const GLOBAL uint32_t*)(at + o + 2 + 4 * j);
    x.d[3] = *(const GLOBAL uint16_t*)(at + o + 14);
  }
  if ((threadIdx.x & 63) == 0) x.first = (uint32_t)*(const GLOBAL uint16_t*)(at + o) << 16;
  return x;
}
template <typename G>
__device__ __forceinline__ w4 dwords_of(const Sixteen& x, bool odd) {
  if (sizeof(G) == 4 || !odd) return x.d;
  const uint32_t first =  // wave_shr:1
      (uint32_t)__builtin_amdgcn_update_dpp((int)x.first, (int)x.d[3], 0x138, 0xf, 0xf, false);
  return w4{__builtin_amdgcn_alignbit(x.d[0], first, 16), __builtin_amdgcn_alignbit(x.d[1], x.d[0], 16),
            __builtin_amdgcn_alignbit(x.d[2], x.d[1], 16), __builtin_amdgcn_alignbit(x.d[3], x.d[2], 16)};
}

// 2048 workgroups, 32 waves per CU: 64 Mi fp32 43 us (6.2 TB/s), 397 bf16 tensors of 100 M elements
// 35 (5.7); fp32 sums instead of fp64 were no faster.
// ALONE: the only workgroup, which finishes too.  KEEP: leave the gradients in the caches for the step
// that reads them next: the norm alone takes 10 % longer, the two together 5 to 10 % less (128 MiB of
// fp32 gradients 181 -> 162 us, 512 MiB 724 -> 702).  A plan of gradients alone has no step.
template <typename G, int BS, bool ALONE, bool KEEP>
__global__ __launch_bounds__(BS) void k_norm(const OptTensor* tensors, const uint32_t* tile_tensor,
                                             uint32_t each, uint32_t more, uint64_t bucket,
                                             double* partials, OptNorm a, hydra_adamw_ctrl_t* ctrl) {
  constexpr int N = 16 / sizeof(G);  // elements of a vector
  __shared__ double lds[BS / 64];
  const uint32_t b = blockIdx.x;
  uint32_t tile = b * each + min(b, more);  // the first `more` workgroups take one tile more
  const uint32_t last = tile + each + (b < more ? 1u : 0u);
  const uint64_t t = ALONE ? (uint64_t)ctrl->step + 1 : 0;
  double sum = 0.0;
  while (tile < last) {  // one tensor's share: [from, to)
    const OptTensor T = tensors[tile_tensor[tile]];
    const uint32_t first = tile - T.tile0, end = min(last - T.tile0, T.tiles);
    const uint64_t from = first * (uint64_t)kOptTile, n = min(end * (uint64_t)kOptTile, T.n) - from;
    const uint64_t vecs = n / N;
    const uint32_t tail = (uint32_t)(n - vecs * N);  // of the tensor's last tile
    gptr at = global((const void*)(bucket + T.grad)) + from * sizeof(G);
    if (threadIdx.x >= 64 && threadIdx.x - 64 < tail) {
      const double g = At<G>::load(at + vecs * 16, threadIdx.x - 64);
      sum = fma(g, g, sum);
    }
    // one vector per thread and turn, the next one's load in flight while this one is summed
    auto add_all = [&](auto odd) {
      Sixteen x = load_sixteen<G, KEEP>(at, vecs, odd);
      for (uint64_t left = vecs; left;) {
        const uint64_t next = left > BS ? left - BS : 0;
        at += BS * 16;
        const Sixteen y = load_sixteen<G, KEEP>(at, next, odd);
        const w4 w = dwords_of<G>(x, odd);
#pragma unroll
        for (int j = 0; j < 4; j++) add_squares<G>(w[j], sum);
        x = y;
        left = next;
      }
    };
    if (sizeof(G) == 2 && ((uint64_t)at & 2)) add_all(std::true_type{});
    else add_all(std::false_type{});
    tile = T.tile0 + end;
  }
  sum = block_sum<BS>(sum, lds);
  if constexpr (ALONE) finish_norm(sum, t, a, ctrl);
  else if (threadIdx.x == 0) partials[b] = sum;
}

__global__ __launch_bounds__(kOptBlock) void k_norm_finish(const double* partials, uint32_t count,
                                                           OptNorm a, hydra_adamw_ctrl_t* ctrl) {
  constexpr int U = kNormBlocks / kOptBlock;
  __shared__ double lds[4];
  const uint64_t t = (uint64_t)ctrl->step + 1;
  double x[U];
#pragma unroll
  for (int u = 0; u < U; u++) {  // all loads at once
    const uint32_t j = u * kOptBlock + threadIdx.x;
    x[u] = j < count ? partials[j] : 0.0;
  }
  double sum = 0.0;
#pragma unroll
  for (int u = 0; u < U; u++) sum += x[u];
  finish_norm(block_sum<kOptBlock>(sum, lds), t, a, ctrl);
}

// ---- 8-bit moments from and to values ---------------------------------------------------------------
// Two blocks of 256 per wave.
constexpr size_t kConvTile = kOptBlock / 64 * 2 * kMomentBlock;  // elements of a workgroup

// a wave's first element, and how many (up to 512) it has
__device__ __forceinline__ uint32_t wave_part(size_t n, size_t* at) {
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  *at = (size_t)blockIdx.x * kConvTile + wave * (2 * kMomentBlock);
  return *at < n ? (uint32_t)min(n - *at, (size_t)(2 * kMomentBlock)) : 0u;
}

// encode: 4 elements per lane of each block, all loads first (8 consecutive ones per lane leave every
// fp32 load half of the lines it touches: 127 us for 64 Mi, this 112, 6.0 TB/s)
template <typename E>
__global__ __launch_bounds__(kOptBlock) void k_encode(uint8_t* m8, float* ms, uint8_t* v8,
                                                      float* vs, const E* m, const E* v, size_t n) {
  size_t at;
  const uint32_t left = wave_part(n, &at), lane = threadIdx.x & 63;
  if (!left) return;
  f4 x[2], y[2];
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const uint32_t i = h * kMomentBlock + lane * 4;
    x[h] = y[h] = f4{0, 0, 0, 0};
    if (m) x[h] = load_upto4<E>(global(m + at), i, rest(left, i));
    if (v) y[h] = load_upto4<E>(global(v + at), i, rest(left, i));
  }
#pragma unroll
  for (int h = 0; h < 2; h++) {
    if (h * kMomentBlock >= left) break;
    const uint32_t i = h * kMomentBlock + lane * 4, count = rest(left, i);
    f4 root;
    uint32_t am = 0, ar = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      y[h][j] = fabsf(y[h][j]);
      root[j] = plain_sqrt(y[h][j]);
      am = max(am, fbits(fabsf(x[h][j])));
      ar = max(ar, fbits(root[j]));
    }
    const uint32_t top = wave_umax_pair(am, ar);
    const uint32_t tm = (uint32_t)__builtin_amdgcn_readlane((int)top, 31);
    const uint32_t tr = (uint32_t)__builtin_amdgcn_readlane((int)top, 63);
    // each moment by itself: its bytes do not depend on the other one's being given
    const bool pm = plain_m(tm), pv = plain_root(tr);
    float scale = moment_scale(bitsf(top));
    if (!pm || !pv) {
      float fm = 0.0f, fr = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if (!pv) root[j] = sqrtf(y[h][j]);
        fm = fmaxf(fm, finite_abs(x[h][j]));
        fr = fmaxf(fr, finite_abs(root[j]));
      }
      scale = moment_scale(bitsf(wave_umax_pair(fbits(fm), fbits(fr))));
    }
    const float inv = plain_inv(scale);
    uint32_t wm = 0, wv = 0;
    if (pm) {
      wm = encode4_m(x[h], uniform(inv, 31), [](uint32_t c, int) { return c + (0x8000u << 4); });
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++)
        wm |= encode_m(x[h][j], moment_inv(uniform(scale, 31)), 0x8000u) << (8 * j);
    }
    if (pv) {
      wv = encode4_root(root, y[h], uniform(inv, 63), [](uint32_t c, int) { return c + (0x8000u << 3); });
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++)
        wv |= encode_root(root[j], moment_inv(uniform(scale, 63)), 0x8000u) << (8 * j);
    }
    if (m) store_bytes(global(m8 + at), i, wm, count);
    if (v) store_bytes(global(v8 + at), i, wv, count);
    if (m && lane == 31) ms[at / kMomentBlock + h] = scale;
    if (v && lane == 63) vs[at / kMomentBlock + h] = scale;
  }
}

// decode: 8 consecutive elements per lane, so a bf16 store is 16 bytes (64 Mi: 66 us, 6.1 TB/s; 4 per
// lane 84)
struct Part {
  uint32_t i, count, lo, hi;  // the lane's first element; how many it has, in all and by fours
};
struct Coded {
  w2b w;
  float scale;
};
__device__ __forceinline__ Coded load_codes(gptr codes, gptr scales, const Part& p) {
  Coded c;
  c.scale = At<float>::load(scales, (threadIdx.x >> 5) & 1);
  if (p.count >= 8) c.w = ldv<w2b>(codes, p.i);
  else c.w = w2b{load_bytes(codes, p.i, p.lo), load_bytes(codes, p.i + 4, p.hi)};
  return c;
}
template <typename E, bool ROOT>
__device__ __forceinline__ void decode_part(gptr values, const Coded& c, const Part& p) {
  f4 x[2];
#pragma unroll
  for (int h = 0; h < 2; h++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const uint32_t b = (c.w[h] >> (8 * j)) & 255u;
      x[h][j] = ROOT ? decode_v(b, c.scale) : decode_m(b, c.scale);
    }
  if (p.count >= 8) {
    At<E>::store8(values, p.i, x[0], x[1]);
  } else {
    store_upto4<E>(values, p.i, x[0], p.lo);
    store_upto4<E>(values, p.i + 4, x[1], p.hi);
  }
}

template <typename E>
__global__ __launch_bounds__(kOptBlock) void k_decode(E* m, E* v, const uint8_t* m8,
                                                      const float* ms, const uint8_t* v8,
                                                      const float* vs, size_t n) {
  size_t at;
  const uint32_t left = wave_part(n, &at), i = (threadIdx.x & 63) * 8;
  if (i >= left) return;
  const Part p{i, left - i, left - i, rest(left, i + 4)};
  const size_t row = at / kMomentBlock;
  Coded a, b;
  if (m) a = load_codes(global(m8 + at), global(ms + row), p);
  if (v) b = load_codes(global(v8 + at), global(vs + row), p);
  if (m) decode_part<E, false>(global(m + at), a, p);
  if (v) decode_part<E, true>(global(v + at), b, p);
}

// ---- launch ------------------------------------------------------------------------------------------
template <typename P, typename G, bool MASTER, bool S8>
hipError_t adamw_t(const OptTable& t, const OptStep& st, const void* bucket, hipStream_t s) {
  if constexpr (S8)
    hipLaunchKernelGGL((k_adamw8<P, G, MASTER>), dim3(t.tiles), dim3(kOptBlock), 0, s, t.tensors,
                       t.tile_tensor, t.tiles, st, reinterpret_cast<uint64_t>(bucket));
  else
    hipLaunchKernelGGL((k_adamw<P, G, MASTER>), dim3(t.tiles), dim3(kOptBlock), 0, s, t.tensors,
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

template <typename G, bool KEEP>
hipError_t norm_t(const OptTable& t, const OptNorm& norm, const void* bucket,
                  hydra_adamw_ctrl_t* ctrl, double* partials, hipStream_t s) {
  const uint64_t at = reinterpret_cast<uint64_t>(bucket);
  if (norm_alone(t)) {
    hipLaunchKernelGGL((k_norm<G, kNormAloneBlock, true, KEEP>), dim3(1), dim3(kNormAloneBlock), 0,
                       s, t.tensors, t.tile_tensor, t.tiles, 0u, at, partials, norm, ctrl);
    return hipGetLastError();
  }
  const uint32_t blocks = std::min(t.tiles, (uint32_t)kNormBlocks);
  hipLaunchKernelGGL((k_norm<G, kOptBlock, false, KEEP>), dim3(blocks), dim3(kOptBlock), 0, s,
                     t.tensors, t.tile_tensor, t.tiles / blocks, t.tiles % blocks, at, partials,
                     norm, ctrl);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(k_norm_finish, dim3(1), dim3(kOptBlock), 0, s, partials, blocks, norm, ctrl);
  return hipGetLastError();
}

template <bool KEEP>
hipError_t norm_g(int grad_dtype, const OptTable& t, const OptNorm& norm, const void* bucket,
                  hydra_adamw_ctrl_t* ctrl, double* partials, hipStream_t s) {
  switch (grad_dtype) {
    case HYDRA_FLOAT32: return norm_t<float, KEEP>(t, norm, bucket, ctrl, partials, s);
    case HYDRA_BFLOAT16: return norm_t<bf16_t, KEEP>(t, norm, bucket, ctrl, partials, s);
    case HYDRA_FLOAT16: return norm_t<f16_t, KEEP>(t, norm, bucket, ctrl, partials, s);
  }
  return hipErrorInvalidValue;
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
    hipLaunchKernelGGL((k_encode<E>), dim3((unsigned)((part + kConvTile - 1) / kConvTile)),
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
    hipLaunchKernelGGL((k_decode<E>), dim3((unsigned)((part + kConvTile - 1) / kConvTile)),
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

static_assert(kNormBlocks * sizeof(double) <= HYDRA_ADAMW_WORKSPACE_MAX, "the bound callers may allocate by");
size_t norm_workspace(const OptTable& t) {
  return norm_alone(t) ? 0 : std::min(t.tiles, (uint32_t)kNormBlocks) * sizeof(double);
}

hipError_t launch_grad_norm(const hydra_adamw_config_t& cfg, const OptTable& t, const OptNorm& norm,
                            const void* bucket, hydra_adamw_ctrl_t* ctrl, double* partials,
                            hipStream_t s) {
  return cfg.flags & HYDRA_ADAMW_NORM_ONLY
             ? norm_g<false>(cfg.grad_dtype, t, norm, bucket, ctrl, partials, s)
             : norm_g<true>(cfg.grad_dtype, t, norm, bucket, ctrl, partials, s);
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
