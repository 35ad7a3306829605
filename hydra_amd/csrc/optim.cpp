// optim.cpp -- the extern "C" boundary of the optimizer step (declared in include/hydra_optim.h):
// argument checks, the plan's tables on the device, launches.  Kernels: optim_kernels.hip.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <exception>
#include <string>
#include <vector>

#include "../../include/hydra_optim.h"
#include "errors.h"
#include "optim_kernels.h"
#include "reduce_kernels.h"
#include "resource_cache.h"

using hydra::fail;
using hydra::hip_fail;
using hydra::ok;

static_assert(sizeof(hydra_adamw_ctrl_t) == 64, "the layout callers allocate");

namespace {
struct Range {  // [lo, hi) of device memory
  uintptr_t lo, hi;
  bool operator<(const Range& o) const { return lo < o.lo; }
};
}  // namespace

struct hydra_adamw {
  int device = 0;
  hydra_adamw_config_t cfg{};
  hydra::OptTable table{};
  void* block = nullptr;           // the device tables
  std::vector<Range> written;      // what a step writes, sorted
  uintptr_t bucket_lo = 0, bucket_hi = 0;  // the hull of the gradients' byte offsets
};

namespace {

constexpr size_t kMaxTiles = (size_t(1) << 24) - 1;  // a launch holds fewer than 2^32 threads
constexpr size_t kMaxElements = size_t(1) << 40;

int fail_at(size_t i, const std::string& msg) {
  return fail(HYDRA_ERR_INVALID, "tensor " + std::to_string(i) + ": " + msg);
}

bool float_dtype(int d) {
  return d == HYDRA_FLOAT32 || d == HYDRA_BFLOAT16 || d == HYDRA_FLOAT16;
}

bool aligned(const void* p, size_t es) { return reinterpret_cast<uintptr_t>(p) % es == 0; }

bool byte_on_device(uintptr_t p, int device) {
  hipPointerAttribute_t a{};
  if (hipPointerGetAttributes(&a, reinterpret_cast<const void*>(p)) != hipSuccess) {
    (void)hipGetLastError();
    return false;
  }
  return (a.type == hipMemoryTypeDevice || a.type == hipMemoryTypeManaged) && a.device == device;
}
// The first and the last byte of r are memory of `device`.  `known`: the allocation that the last
// query found, which holds most of the ranges that follow (views of a few buffers).
bool on_device(const Range& r, int device, Range* known) {
  if (known->lo <= r.lo && r.hi <= known->hi) return true;
  if (!byte_on_device(r.lo, device) || !byte_on_device(r.hi - 1, device)) return false;
  hipDeviceptr_t base = nullptr;
  size_t bytes = 0;
  if (hipMemGetAddressRange(&base, &bytes, reinterpret_cast<hipDeviceptr_t>(r.lo)) == hipSuccess)
    *known = {reinterpret_cast<uintptr_t>(base), reinterpret_cast<uintptr_t>(base) + bytes};
  else
    (void)hipGetLastError();  // (memory mapped by its owner: asked for range by range)
  return true;
}

int check_config(const hydra_adamw_config_t& c) {
  if (!float_dtype(c.grad_dtype))
    return fail(HYDRA_ERR_INVALID, "gradients must be fp32, bf16 or fp16");
  if (c.flags & ~(HYDRA_ADAMW_MASTER | HYDRA_ADAMW_BUCKET | HYDRA_ADAMW_NORM_ONLY))
    return fail(HYDRA_ERR_INVALID, "unknown flags");
  if (!(c.beta1 >= 0.0 && c.beta1 < 1.0 && c.beta2 >= 0.0 && c.beta2 < 1.0))
    return fail(HYDRA_ERR_INVALID, "betas must lie in [0, 1)");
  if (!((float)c.beta1 < 1.0f && (float)c.beta2 < 1.0f))
    return fail(HYDRA_ERR_INVALID, "a beta is 1 in fp32");
  if (!(c.eps >= 0.0 && std::isfinite(c.eps)))
    return fail(HYDRA_ERR_INVALID, "eps must be finite and >= 0");
  if (c.flags & HYDRA_ADAMW_NORM_ONLY) return HYDRA_OK;
  if (!float_dtype(c.param_dtype))
    return fail(HYDRA_ERR_INVALID, "params must be fp32, bf16 or fp16");
  if (c.state_dtype != HYDRA_FLOAT32 && c.state_dtype != HYDRA_UINT8)
    return fail(HYDRA_ERR_INVALID, "moments must be fp32 or 8-bit (HYDRA_UINT8)");
  if ((c.flags & HYDRA_ADAMW_MASTER) && c.param_dtype == HYDRA_FLOAT32)
    return fail(HYDRA_ERR_INVALID, "an fp32 master stands beside 16-bit params only");
  return HYDRA_OK;
}

// Checks one tensor and appends the ranges that a step writes and (addresses only) reads.
int check_tensor(size_t i, const hydra_adamw_config_t& c, const hydra_adamw_tensor_t& t,
                 std::vector<Range>* written, std::vector<Range>* grads) {
  if (t.n > kMaxElements) return fail_at(i, "more than 2^40 elements");
  if (!std::isfinite(t.lr_scale) || !std::isfinite(t.weight_decay))
    return fail_at(i, "lr_scale and weight_decay must be finite");
  if (t.n == 0) return HYDRA_OK;
  const size_t ge = hydra::dtype_size(c.grad_dtype);
  const uintptr_t g = reinterpret_cast<uintptr_t>(t.grad);
  if (!(c.flags & HYDRA_ADAMW_BUCKET) && !t.grad) return fail_at(i, "null gradient");
  if (g % ge) return fail_at(i, "gradient not aligned to its element size");
  if (g > (uintptr_t(1) << 57)) return fail_at(i, "gradient offset out of range");
  grads->push_back({g, g + t.n * ge});
  if (c.flags & HYDRA_ADAMW_NORM_ONLY) return HYDRA_OK;
  const bool master = (c.flags & HYDRA_ADAMW_MASTER) != 0, s8 = c.state_dtype == HYDRA_UINT8;
  const size_t pe = hydra::dtype_size(c.param_dtype), se = s8 ? 1 : 4;
  const size_t scales = (t.n + hydra::kMomentBlock - 1) / hydra::kMomentBlock;
  const struct {
    const void* p;
    size_t es, count;
    bool wanted;
    const char* name;
  } all[] = {{t.param, pe, t.n, true, "param"},       {t.master, 4, t.n, master, "master"},
             {t.m, se, t.n, true, "m"},               {t.v, se, t.n, true, "v"},
             {t.m_scale, 4, scales, s8, "m_scale"},   {t.v_scale, 4, scales, s8, "v_scale"}};
  for (const auto& x : all) {
    if (!x.wanted) {
      if (x.p) return fail_at(i, std::string(x.name) + " given where the plan has none");
      continue;
    }
    if (!x.p) return fail_at(i, std::string("null ") + x.name);
    if (!aligned(x.p, x.es)) return fail_at(i, std::string(x.name) + " not aligned to its element size");
    const uintptr_t lo = reinterpret_cast<uintptr_t>(x.p);
    written->push_back({lo, lo + x.count * x.es});
  }
  return HYDRA_OK;
}

// ranges sorted and apart from each other; r anywhere among them?
bool touches(const std::vector<Range>& sorted, const Range& r) {
  auto it = std::lower_bound(sorted.begin(), sorted.end(), r);  // the first that begins at or after r
  if (it != sorted.end() && it->lo < r.hi) return true;
  return it != sorted.begin() && std::prev(it)->hi > r.lo;
}

// Elements before a tensor's first tile's vectors: those that leave the most bytes of its buffers on
// their natural alignment (16 bytes for four fp32, 8 for four 16-bit values), and then the most
// bytes' tiles on whole 128-byte lines.  Tensors that are views of flat buffers of one layout are all
// aligned by the same head (291 ragged tensors with fp16 gradients, clipped: 113 us; vectors aligned
// alone 124: a tile's ends then write parts of lines).  8-bit moments have none: their blocks count from the first element.
uint32_t head_of(const hydra_adamw_config_t& c, const hydra_adamw_tensor_t& t) {
  if (!(c.flags & HYDRA_ADAMW_NORM_ONLY) && c.state_dtype == HYDRA_UINT8) return 0;
  uint32_t best = 0;
  size_t most = 0;
  for (uint32_t h = 0; h < hydra::kMaxHead; h++) {
    size_t score = 0;
    auto add = [&](const void* p, size_t es, size_t passes) {
      const uintptr_t at = reinterpret_cast<uintptr_t>(p) + h * es;
      if (at % (4 * es) == 0) score += 8 * es * passes;
      if (at % 128 == 0) score += es * passes;
    };
    add(t.grad, hydra::dtype_size(c.grad_dtype), 1);  // (a bucket's address: taken as aligned)
    if (!(c.flags & HYDRA_ADAMW_NORM_ONLY)) {
      add(t.param, hydra::dtype_size(c.param_dtype), t.master ? 1 : 2);  // only written, or both
      if (t.master) add(t.master, 4, 2);
      add(t.m, 4, 2);
      add(t.v, 4, 2);
    }
    if (score > most) {
      most = score;
      best = h;
    }
  }
  return (uint32_t)std::min<size_t>(best, t.n);
}

// Tiles of a tensor, whatever its head: the norm's order of sums hangs on them, and on no address.  (The
// step leaves the last one empty where the head takes its elements.)
size_t tiles_of(size_t n) { return (n + hydra::kOptTile - 1) / hydra::kOptTile; }

int create(int device, const hydra_adamw_config_t* config, const hydra_adamw_tensor_t* tensors,
           size_t count, hydra_adamw** made) {
  if (!config) return fail(HYDRA_ERR_INVALID, "null config");
  if (count && !tensors) return fail(HYDRA_ERR_INVALID, "null tensor list");
  if (int rc = check_config(*config)) return rc;
  std::vector<Range> written, grads;
  size_t tiles = 0;
  for (size_t i = 0; i < count; i++) {
    if (int rc = check_tensor(i, *config, tensors[i], &written, &grads)) return rc;
    tiles += tiles_of(tensors[i].n);
  }
  if (tiles > kMaxTiles || count >= (size_t(1) << 31))
    return fail(HYDRA_ERR_INVALID, "too many elements for one plan: split it");
  std::sort(written.begin(), written.end());
  for (size_t i = 1; i < written.size(); i++)
    if (written[i].lo < written[i - 1].hi)
      return fail(HYDRA_ERR_INVALID, "two of the plan's written ranges overlap");
  const bool bucket = (config->flags & HYDRA_ADAMW_BUCKET) != 0;
  if (!bucket)
    for (const Range& g : grads)
      if (touches(written, g))
        return fail(HYDRA_ERR_INVALID, "a gradient overlaps what the step writes");

  int devices = 0;
  HIP_TRY(hipGetDeviceCount(&devices));
  if (device < 0 || device >= devices) return fail(HYDRA_ERR_NO_DEVICE, "no such device");
  hydra::DeviceScope ds(device);
  HIP_TRY(ds.err);
  Range known{0, 0};
  for (const Range& r : written)
    if (!on_device(r, device, &known))
      return fail(HYDRA_ERR_INVALID, "a param, master or moment is not memory of the plan's device");
  if (!bucket)
    for (const Range& r : grads)
      if (!on_device(r, device, &known))
        return fail(HYDRA_ERR_INVALID, "a gradient is not memory of the plan's device");

  hydra_adamw& P = **made;
  P.device = device;
  P.cfg = *config;
  P.written = std::move(written);
  if (bucket && !grads.empty()) {
    P.bucket_lo = UINTPTR_MAX;
    for (const Range& g : grads) {
      P.bucket_lo = std::min(P.bucket_lo, g.lo);
      P.bucket_hi = std::max(P.bucket_hi, g.hi);
    }
  }
  P.table.tiles = (uint32_t)tiles;
  P.table.filled = (uint32_t)grads.size();
  if (tiles == 0) return HYDRA_OK;

  // [descriptors | the tensor of each tile], through a pinned block
  const size_t desc_bytes = count * sizeof(hydra::OptTensor);
  const size_t bytes = desc_bytes + tiles * sizeof(uint32_t);
  HIP_TRY(hydra::cached_malloc(device, bytes, &P.block));
  void* stage = nullptr;
  HIP_TRY(hydra::cached_malloc_host(bytes, &stage));
  auto* desc = static_cast<hydra::OptTensor*>(stage);
  auto* of_tile = reinterpret_cast<uint32_t*>(static_cast<char*>(stage) + desc_bytes);
  uint32_t tile = 0;
  for (size_t i = 0; i < count; i++) {
    const hydra_adamw_tensor_t& t = tensors[i];
    desc[i] = {static_cast<char*>(t.param), t.master, reinterpret_cast<uint64_t>(t.grad),
               static_cast<char*>(t.m), static_cast<char*>(t.v), t.m_scale, t.v_scale, t.n,
               t.lr_scale, t.weight_decay, tile, (uint32_t)i, head_of(*config, t), 0};
    desc[i].tiles = (uint32_t)tiles_of(t.n);
    for (uint32_t k = 0; k < desc[i].tiles; k++) of_tile[tile++] = (uint32_t)i;
  }
  hipStream_t s = nullptr;
  hipError_t e = hydra::cached_stream(device, &s);
  if (e == hipSuccess) e = hipMemcpyAsync(P.block, stage, bytes, hipMemcpyHostToDevice, s);
  if (e == hipSuccess) e = hipStreamSynchronize(s);
  if (s) (void)hydra::release_stream(s);
  (void)hydra::cached_free_host(stage);
  if (e != hipSuccess) return hip_fail(e, "hydra_adamw_create");
  P.table.tensors = static_cast<const hydra::OptTensor*>(P.block);
  P.table.tile_tensor = reinterpret_cast<const uint32_t*>(static_cast<char*>(P.block) + desc_bytes);
  return HYDRA_OK;
}

// The bucket argument of a call.
int check_bucket(const hydra_adamw& P, const void* bucket) {
  if (!(P.cfg.flags & HYDRA_ADAMW_BUCKET)) {
    if (bucket) return fail(HYDRA_ERR_INVALID, "the plan's gradients are addresses: no bucket");
    return HYDRA_OK;
  }
  if (P.table.tiles == 0) return HYDRA_OK;
  if (!bucket) return fail(HYDRA_ERR_INVALID, "null bucket");
  if (!aligned(bucket, hydra::dtype_size(P.cfg.grad_dtype)))
    return fail(HYDRA_ERR_INVALID, "bucket not aligned to its element size");
  const uintptr_t b = reinterpret_cast<uintptr_t>(bucket);
  const Range r{b + P.bucket_lo, b + P.bucket_hi};
  if (touches(P.written, r))
    return fail(HYDRA_ERR_INVALID, "the bucket overlaps what the step writes");
  if (!byte_on_device(r.lo, P.device) || !byte_on_device(r.hi - 1, P.device))
    return fail(HYDRA_ERR_INVALID, "the bucket is not memory of the plan's device");
  return HYDRA_OK;
}

int step(hydra_adamw_t plan, const void* bucket, hydra::OptStep st, uint64_t seed,
         hydra_stream_t stream) {
  if (plan->cfg.flags & HYDRA_ADAMW_NORM_ONLY)
    return fail(HYDRA_ERR_UNSUPPORTED, "the plan holds gradients alone");
  if (int rc = check_bucket(*plan, bucket)) return rc;
  const hydra_adamw_config_t& c = plan->cfg;
  st.beta1 = (float)c.beta1;
  st.omb1 = (float)(1.0 - c.beta1);
  st.beta2 = (float)c.beta2;
  st.omb2 = (float)(1.0 - c.beta2);
  st.eps = (float)c.eps;
  st.stochastic = seed != 0;
  st.seed_key = hydra::fmix32(hydra::fmix32((uint32_t)seed) ^ (uint32_t)(seed >> 32));
  hydra::DeviceScope ds(plan->device);
  HIP_TRY(ds.err);
  const hipError_t e =
      hydra::launch_adamw(c, plan->table, st, bucket, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "adamw kernel launch");
  return ok();
}

// One moment's three pointers of an encode / decode call: all or none.
int check_moment(const char* name, const void* values, size_t es, const void* codes,
                 const void* scales, bool* given) {
  *given = values || codes || scales;
  if (*given && !(values && codes && scales))
    return fail(HYDRA_ERR_INVALID, std::string("null pointer among those of ") + name);
  if (!aligned(values, es) || !aligned(scales, 4))
    return fail(HYDRA_ERR_INVALID, std::string(name) + " not aligned to its element size");
  return HYDRA_OK;
}

// Shared checks of the two conversions.
int check_moments(const void* m, const void* v, int dtype, const void* m8, const void* ms,
                  const void* v8, const void* vs, size_t n, bool encode) {
  if (dtype != HYDRA_FLOAT32 && dtype != HYDRA_BFLOAT16)
    return fail(HYDRA_ERR_INVALID, "moment values are fp32 or bf16");
  if (n > kMaxElements) return fail(HYDRA_ERR_INVALID, "more than 2^40 elements");
  if (n == 0) return HYDRA_OK;
  const size_t es = hydra::dtype_size(dtype);
  bool has_m = false, has_v = false;
  if (int rc = check_moment("m", m, es, m8, ms, &has_m)) return rc;
  if (int rc = check_moment("v", v, es, v8, vs, &has_v)) return rc;
  if (!has_m && !has_v) return fail(HYDRA_ERR_INVALID, "neither moment given");
  const size_t scales = (n + hydra::kMomentBlock - 1) / hydra::kMomentBlock;
  Range out[4], in[4];
  int nout = 0, nin = 0;
  auto add = [&](const void* p, size_t bytes, bool written) {
    if (!p) return;
    const uintptr_t lo = reinterpret_cast<uintptr_t>(p);
    (written ? out[nout++] : in[nin++]) = {lo, lo + bytes};
  };
  add(m, n * es, !encode);
  add(v, n * es, !encode);
  add(m8, n, encode);
  add(v8, n, encode);
  add(ms, scales * 4, encode);
  add(vs, scales * 4, encode);
  for (int i = 0; i < nout; i++) {
    for (int j = 0; j < i; j++)
      if (out[i].lo < out[j].hi && out[j].lo < out[i].hi)
        return fail(HYDRA_ERR_INVALID, "two outputs overlap");
    for (int j = 0; j < nin; j++)
      if (out[i].lo < in[j].hi && in[j].lo < out[i].hi)
        return fail(HYDRA_ERR_INVALID, "an output overlaps an input");
  }
  return HYDRA_OK;
}

}  // namespace

extern "C" {

int hydra_adamw_create(int device, const hydra_adamw_config_t* config,
                       const hydra_adamw_tensor_t* tensors, size_t count, hydra_adamw_t* out) {
  if (!out) return fail(HYDRA_ERR_INVALID, "null out");
  *out = nullptr;
  hydra_adamw* plan = nullptr;
  int rc;
  try {
    plan = new hydra_adamw;
    rc = create(device, config, tensors, count, &plan);
  } catch (const std::exception& e) {  // (of the vectors: out of host memory)
    rc = fail(HYDRA_ERR_HIP, std::string("hydra_adamw_create: ") + e.what());
  }
  if (rc) {
    if (plan && plan->block) (void)hydra::cached_free(plan->block);
    delete plan;
    return rc;
  }
  *out = plan;
  return ok();
}

int hydra_adamw_destroy(hydra_adamw_t plan) {
  if (!plan) return ok();
  hipError_t e = hipSuccess;
  if (plan->block) {
    hydra::DeviceScope ds(plan->device);
    e = ds.err;
    if (e == hipSuccess) e = hydra::cached_free(plan->block);  // drains the device first
  }
  delete plan;
  if (e != hipSuccess) return hip_fail(e, "hydra_adamw_destroy");
  return ok();
}

int hydra_adamw_workspace(hydra_adamw_t plan, size_t* bytes) {
  if (!plan || !bytes) return fail(HYDRA_ERR_INVALID, "null plan or bytes");
  *bytes = hydra::norm_workspace(plan->table);
  return ok();
}

int hydra_adamw_grad_norm(hydra_adamw_t plan, const void* bucket, double grad_scale,
                          double max_norm, hydra_adamw_ctrl_t* ctrl, void* workspace,
                          size_t workspace_bytes, hydra_stream_t stream) {
  if (!plan || !ctrl) return fail(HYDRA_ERR_INVALID, "null plan or ctrl");
  if (!std::isfinite((float)grad_scale))
    return fail(HYDRA_ERR_INVALID, "grad_scale must be finite in fp32");
  if (!(max_norm >= 0.0)) return fail(HYDRA_ERR_INVALID, "max_norm must be >= 0");
  if (!aligned(ctrl, 8) || !aligned(workspace, 8))
    return fail(HYDRA_ERR_INVALID, "ctrl and workspace must be 8-byte aligned");
  const size_t need = hydra::norm_workspace(plan->table);
  if (workspace_bytes < need || (need && !workspace))
    return fail(HYDRA_ERR_INVALID, "workspace smaller than hydra_adamw_workspace says");
  if (int rc = check_bucket(*plan, bucket)) return rc;
  hydra::DeviceScope ds(plan->device);
  HIP_TRY(ds.err);
  const hydra::OptNorm norm{grad_scale, max_norm, plan->cfg.beta1, plan->cfg.beta2};
  const hipError_t e =
      hydra::launch_grad_norm(plan->cfg, plan->table, norm, bucket, ctrl,
                              static_cast<double*>(workspace), static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "gradient norm kernel launch");
  return ok();
}

int hydra_adamw_step(hydra_adamw_t plan, const void* bucket, double lr, int64_t step_number,
                     double grad_scale, uint64_t seed, hydra_stream_t stream) {
  if (!plan) return fail(HYDRA_ERR_INVALID, "null plan");
  if (step_number < 1) return fail(HYDRA_ERR_INVALID, "steps count from 1");
  if (!std::isfinite((float)lr) || !std::isfinite((float)grad_scale))
    return fail(HYDRA_ERR_INVALID, "lr and grad_scale must be finite in fp32");
  hydra::OptStep st{};
  st.lr = (float)lr;
  st.mult = (float)grad_scale;
  st.step = step_number;
  st.inv_bc1 = (float)(1.0 / (1.0 - hydra::power(plan->cfg.beta1, (uint64_t)step_number)));
  st.inv_sqrt_bc2 = (float)(1.0 / std::sqrt(1.0 - hydra::power(plan->cfg.beta2, (uint64_t)step_number)));
  return step(plan, bucket, st, seed, stream);
}

int hydra_adamw_step_ctrl(hydra_adamw_t plan, const void* bucket, const hydra_adamw_ctrl_t* ctrl,
                          uint64_t seed, hydra_stream_t stream) {
  if (!plan || !ctrl) return fail(HYDRA_ERR_INVALID, "null plan or ctrl");
  if (!aligned(ctrl, 8)) return fail(HYDRA_ERR_INVALID, "ctrl must be 8-byte aligned");
  hydra::OptStep st{};
  st.ctrl = ctrl;
  return step(plan, bucket, st, seed, stream);
}

int hydra_moments8_encode(uint8_t* m8, float* m_scale, uint8_t* v8, float* v_scale, const void* m,
                          const void* v, int dtype, size_t n, hydra_stream_t stream) {
  if (int rc = check_moments(m, v, dtype, m8, m_scale, v8, v_scale, n, true)) return rc;
  if (n == 0) return ok();
  const hipError_t e = hydra::launch_moments8_encode(dtype, m8, m_scale, v8, v_scale, m, v, n,
                                                     static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "moments8 encode kernel launch");
  return ok();
}

int hydra_moments8_decode(void* m, void* v, int dtype, const uint8_t* m8, const float* m_scale,
                          const uint8_t* v8, const float* v_scale, size_t n,
                          hydra_stream_t stream) {
  if (int rc = check_moments(m, v, dtype, m8, m_scale, v8, v_scale, n, false)) return rc;
  if (n == 0) return ok();
  const hipError_t e = hydra::launch_moments8_decode(dtype, m, v, m8, m_scale, v8, v_scale, n,
                                                     static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "moments8 decode kernel launch");
  return ok();
}

}  // extern "C"
