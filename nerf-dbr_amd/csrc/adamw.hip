// One AdamW step over many tensors at once (nerf_adamw_step).
//   g = grad * min(1, max_norm / (|grads| + 1e-6))
//   m = m + (1 - b1)(g - m),  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// Bound by bytes: 28 per fp32 value with 32-bit moments, 16 + 16 / 256 with 8-bit ones.  The tensors'
// addresses travel in the kernel arguments (48 tensors a launch), so nothing is uploaded, nothing is
// kept between calls and a captured call replays as it was made.
#include <cmath>
#include <cstring>

#include "nerf_internal.h"

namespace nerf {
namespace {

constexpr int kTensors = 48;   // per launch: 48 x 72 bytes of the 4 KiB of kernel arguments
struct AdamTensor {
  float* p;
  void* model;
  void* g;
  void* m;
  void* v;
  float* ms;
  float* vs;
  long n;
  float decay;      // 1 - lr * weight_decay with the host's lr; with lr_device the kernel forms it
  float wd;
};
struct AdamArgs {
  AdamTensor t[kTensors];
  unsigned first[kTensors];   // the tensor's first chunk in this launch
  int n_tensors, iters, flags;
  unsigned char wide[kTensors];   // every address allows vector access
  const nerf_adamw_control* ctl;
  const float* lr_dev;
  float lr, b1c, b2, b2c, eps;   // b1c = 1 - beta1, b2c = 1 - beta2
};
static_assert(sizeof(AdamArgs) <= 4096, "kernel arguments");
constexpr int kStep = 1024;    // values a workgroup takes per iteration: 256 threads x 4

// The tensor that a chunk belongs to: the last one whose first chunk is not behind it.
__device__ __forceinline__ int find(const AdamArgs& a, unsigned chunk) {
  int lo = 0, hi = a.n_tensors - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.first[mid] <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <typename T>
struct alignas(sizeof(T) * 4) Quad {
  T v[4];
};
template <typename T>
__device__ __forceinline__ void load4(const T* p, long i, long n, bool wide, float out[4]) {
  if (wide && i + 4 <= n) {
    const Quad<T> q = *reinterpret_cast<const Quad<T>*>(p + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) out[k] = float(q.v[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) out[k] = i + k < n ? float(p[i + k]) : 0.0f;
  }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, long i, long n, bool wide, const float in[4]) {
  if (wide && i + 4 <= n) {
    Quad<T> q;
#pragma unroll
    for (int k = 0; k < 4; ++k) q.v[k] = T(in[k]);
    *reinterpret_cast<Quad<T>*>(p + i) = q;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i + k < n) p[i + k] = T(in[k]);
  }
}
// four e4m3 codes (OCP, the hardware's conversion) as one word
__device__ __forceinline__ void load_codes(const unsigned char* p, long i, long n, bool wide, float out[4]) {
  unsigned w = 0;
  if (wide && i + 4 <= n) w = *reinterpret_cast<const unsigned*>(p + i);
  else
    for (int k = 0; k < 4; ++k)
      if (i + k < n) w |= unsigned(p[i + k]) << (8 * k);
  out[0] = __builtin_amdgcn_cvt_f32_fp8(w, 0);
  out[1] = __builtin_amdgcn_cvt_f32_fp8(w, 1);
  out[2] = __builtin_amdgcn_cvt_f32_fp8(w, 2);
  out[3] = __builtin_amdgcn_cvt_f32_fp8(w, 3);
}
__device__ __forceinline__ void store_codes(unsigned char* p, long i, long n, bool wide, unsigned w) {
  if (wide && i + 4 <= n) *reinterpret_cast<unsigned*>(p + i) = w;
  else
    for (int k = 0; k < 4; ++k)
      if (i + k < n) p[i + k] = (unsigned char)(w >> (8 * k));
}
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o, 64));
  return x;
}
__device__ __forceinline__ double pow_steps(double b, int t) {   // b^t, t > 0, by squaring
  double r = 1.0;
  for (; t; t >>= 1, b *= b)
    if (t & 1) r *= b;
  return r;
}

// The gradients' squares summed in fp64, one partial per workgroup at a fixed place.
template <typename G>
__global__ __launch_bounds__(256) void norm_kernel(AdamArgs a, double* part) {
  __shared__ double red[4];
  const int k = find(a, blockIdx.x);
  const AdamTensor& t = a.t[k];
  long i = (long(blockIdx.x - a.first[k]) * a.iters) * kStep + threadIdx.x * 4;
  double s = 0.0;
  for (int it = 0; it < a.iters && i < t.n; ++it, i += kStep) {
    float g[4];
    load4(static_cast<const G*>(t.g), i, t.n, a.wide[k], g);
#pragma unroll
    for (int j = 0; j < 4; ++j) s += double(g[j]) * double(g[j]);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_down(s, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

// One workgroup: the norm from the partials, added in order (it does not depend on timing), the step
// count and the step's scalars for adamw_kernel.  A launch of its own: a count of finished workgroups in
// the kernels before (one atomic each on one address, ~0.1 us apiece) cost 3.5 ms where there were 35,000.
__global__ __launch_bounds__(1024) void prepare_kernel(nerf_adamw_control* c, const double* part, long n, float max_norm, double b1,
                                                       double b2, int skip_nonfinite) {
  __shared__ double red[16];
  double s = 0.0;
#pragma unroll 8
  for (long j = threadIdx.x; j < n; j += 1024) s += part[j];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_down(s, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x) return;
  s = 0.0;
  for (int w = 0; w < 16; ++w) s += red[w];
  const double norm = sqrt(s), f = max_norm > 0.0f ? double(max_norm) / (norm + 1e-6) : 1.0;
  if (n) c->norm = float(norm);
  c->factor = f > 1.0 ? 1.0f : float(f);   // NaN stays NaN
  const bool skip = skip_nonfinite && !__builtin_isfinite(float(norm));
  c->apply = skip ? 0 : 1;
  if (skip) {
    c->skipped += 1;
    return;
  }
  const int step = c->steps + 1;
  c->steps = step;
  c->rate = float(1.0 / (1.0 - pow_steps(b1, step)));
  c->root = float(sqrt(1.0 - pow_steps(b2, step)));
}

template <typename G, typename M, int BITS>
__global__ __launch_bounds__(256) void adamw_kernel(AdamArgs a) {
  const int k = find(a, blockIdx.x);
  const AdamTensor& t = a.t[k];
  const bool wide = a.wide[k];
  if (!a.ctl->apply) return;
  const float factor = a.ctl->factor, root = a.ctl->root;
  float lr = a.lr;
  // (a global load: a plain one would be merged with the argument's into one through a flat address)
  if (a.lr_dev) lr = *(const __attribute__((address_space(1))) float*)a.lr_dev;
  const float decay = a.lr_dev ? 1.0f - lr * t.wd : t.decay, rate = lr * a.ctl->rate;
  long i = (long(blockIdx.x - a.first[k]) * a.iters) * kStep + threadIdx.x * 4;
  for (int it = 0; it < a.iters; ++it, i += kStep) {
    if (BITS == 32 && i >= t.n) break;
    if (BITS == 8 && i - (threadIdx.x & 63) * 4 >= t.n) break;   // uniform in a wave: its block is behind the end
    float g[4], p[4], m[4], v[4], r[4];
    load4(static_cast<const G*>(t.g), i, t.n, wide, g);
    load4(t.p, i, t.n, wide, p);
    const long block = i >> 8;    // the wave's 256 values are one block
    if (BITS == 32) {
      load4(static_cast<const float*>(t.m), i, t.n, wide, m);
      load4(static_cast<const float*>(t.v), i, t.n, wide, v);
    } else {
      load_codes(static_cast<const unsigned char*>(t.m), i, t.n, wide, m);
      load_codes(static_cast<const unsigned char*>(t.v), i, t.n, wide, v);
      const float ms = t.ms[block], vs = t.vs[block];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        m[j] *= ms;
        v[j] *= vs;
        v[j] *= v[j];
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      g[j] *= factor;
      m[j] += (g[j] - m[j]) * a.b1c;
      v[j] = v[j] * a.b2 + g[j] * g[j] * a.b2c;
      r[j] = sqrtf(v[j]);
      p[j] = p[j] * decay - rate * m[j] / (r[j] / root + a.eps);
    }
    if (a.flags & NERF_ADAMW_WRITE_GRADS) store4(static_cast<G*>(t.g), i, t.n, wide, g);
    store4(t.p, i, t.n, wide, p);
    if (sizeof(M) == 2) store4(static_cast<M*>(t.model), i, t.n, wide, p);
    if (BITS == 32) {
      store4(static_cast<float*>(t.m), i, t.n, wide, m);
      store4(static_cast<float*>(t.v), i, t.n, wide, v);
    } else {
      // values behind the tensor's end were loaded as zeros: they do not raise the block's maximum
      const float top = wave_max(fmaxf(fmaxf(fabsf(m[0]), fabsf(m[1])), fmaxf(fabsf(m[2]), fabsf(m[3]))));
      const float rtop = wave_max(fmaxf(fmaxf(r[0], r[1]), fmaxf(r[2], r[3])));
      const float ms = top / 448.0f, vs = rtop / 448.0f;
      unsigned mw = 0, vw = 0;
      if (ms > 0.0f) {
        mw = __builtin_amdgcn_cvt_pk_fp8_f32(m[0] / ms, m[1] / ms, mw, false);
        mw = __builtin_amdgcn_cvt_pk_fp8_f32(m[2] / ms, m[3] / ms, mw, true);
      }
      if (vs > 0.0f) {
        vw = __builtin_amdgcn_cvt_pk_fp8_f32(r[0] / vs, r[1] / vs, vw, false);
        vw = __builtin_amdgcn_cvt_pk_fp8_f32(r[2] / vs, r[3] / vs, vw, true);
        // a root that is not zero keeps the smallest code: m / (0 + eps) of a value whose v was
        // rounded away would be a step of any size
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (r[j] > 0.0f && ((vw >> (8 * j)) & 0xffu) == 0) vw |= 1u << (8 * j);
      }
      store_codes(static_cast<unsigned char*>(t.m), i, t.n, wide, mw);
      store_codes(static_cast<unsigned char*>(t.v), i, t.n, wide, vw);
      if ((threadIdx.x & 63) == 0) t.ms[block] = ms, t.vs[block] = vs;
    }
  }
}

// Chunks of a call: as many as fill the machine with one iteration each, at most 8 iterations (32 KiB
// of fp32 per array) so that a workgroup's fixed cost (tensor search, bias corrections) is spread.
int iterations(int n, const nerf_adamw_tensor* t) {
  long steps = 0;
  for (int i = 0; i < n; ++i) steps += (t[i].numel + kStep - 1) / kStep;
  const long per = steps / (8L * 256);
  return int(per < 1 ? 1 : per > 8 ? 8 : per);
}
long chunks(const nerf_adamw_tensor& t, int iters) { return (t.numel + long(iters) * kStep - 1) / (long(iters) * kStep); }

template <typename G, typename M>
void launch_step(const AdamArgs& a, int bits, unsigned grid, hipStream_t s) {
  if (bits == 32) hipLaunchKernelGGL((adamw_kernel<G, M, 32>), dim3(grid), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((adamw_kernel<G, M, 8>), dim3(grid), dim3(256), 0, s, a);
}
template <typename G>
void launch_step(const AdamArgs& a, int model, int bits, unsigned grid, hipStream_t s) {
  if (model == NERF_BFLOAT16) launch_step<G, __bf16>(a, bits, grid, s);
  else if (model == NERF_FLOAT16) launch_step<G, _Float16>(a, bits, grid, s);
  else launch_step<G, float>(a, bits, grid, s);
}

int check(const nerf_adamw_config* c, int n, const nerf_adamw_tensor* t) {
  if (!c || (n > 0 && !t) || n < 0) return set_error(NERF_E_INVALID, "nerf_adamw_step: null argument");
  if (!(c->lr >= 0.0) || !(c->beta1 >= 0.0 && c->beta1 < 1.0) || !(c->beta2 >= 0.0 && c->beta2 < 1.0) || !(c->eps >= 0.0))
    return set_error(NERF_E_INVALID, "nerf_adamw_step: lr %g, betas %g %g, eps %g", c->lr, c->beta1, c->beta2, c->eps);
  if (c->state_bits != 32 && c->state_bits != 8) return set_error(NERF_E_INVALID, "nerf_adamw_step: state_bits %d (32 or 8)", c->state_bits);
  if (c->flags & ~(NERF_ADAMW_SKIP_NONFINITE | NERF_ADAMW_WRITE_GRADS)) return set_error(NERF_E_INVALID, "nerf_adamw_step: flags %d", c->flags);
  bool any = false;
  for (int i = 0; i < n; ++i) {
    const nerf_adamw_tensor& x = t[i];
    any = any || x.numel > 0;
    if (x.numel < 0 || x.numel > (1L << 40)) return set_error(NERF_E_INVALID, "nerf_adamw_step: tensor %d has %ld values", i, long(x.numel));
    if (x.numel == 0) continue;
    if (!x.param || !x.grad || !x.exp_avg || !x.exp_avg_sq || (c->state_bits == 8 && (!x.exp_avg_scale || !x.exp_avg_sq_scale)))
      return set_error(NERF_E_INVALID, "nerf_adamw_step: tensor %d has a null store", i);
    if (x.grad_dtype != NERF_F32 && x.grad_dtype != NERF_BFLOAT16 && x.grad_dtype != NERF_FLOAT16)
      return set_error(NERF_E_INVALID, "nerf_adamw_step: tensor %d has gradient dtype %d", i, x.grad_dtype);
    if (x.model && x.model_dtype != NERF_BFLOAT16 && x.model_dtype != NERF_FLOAT16)
      return set_error(NERF_E_INVALID, "nerf_adamw_step: tensor %d has model dtype %d", i, x.model_dtype);
    if (!(x.weight_decay >= 0.0)) return set_error(NERF_E_INVALID, "nerf_adamw_step: tensor %d has weight decay %g", i, x.weight_decay);
    uintptr_t four = uintptr_t(x.param) | uintptr_t(x.exp_avg_scale) | uintptr_t(x.exp_avg_sq_scale);
    uintptr_t two = uintptr_t(x.model);
    (x.grad_dtype == NERF_F32 ? four : two) |= uintptr_t(x.grad);
    if (c->state_bits == 32) four |= uintptr_t(x.exp_avg) | uintptr_t(x.exp_avg_sq);
    if ((four & 3) || (two & 1)) return set_error(NERF_E_INVALID, "nerf_adamw_step: tensor %d is not aligned to its type", i);
  }
  if (!any) return set_error(NERF_E_INVALID, "nerf_adamw_step: no values to step");
  return NERF_OK;
}

}  // namespace
}  // namespace nerf

using namespace nerf;

extern "C" {

size_t nerf_adamw_workspace(int n_tensors, const nerf_adamw_tensor* tensors) {
  if (n_tensors <= 0 || !tensors) return 0;
  const int iters = iterations(n_tensors, tensors);
  long n = 0;
  for (int i = 0; i < n_tensors; ++i) n += chunks(tensors[i], iters);
  return sizeof(double) * size_t(n);
}

int nerf_adamw_step(const nerf_adamw_config* config, int n_tensors, const nerf_adamw_tensor* tensors,
                    nerf_adamw_control* control, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check(config, n_tensors, tensors);
  if (rc != NERF_OK) return rc;
  if (!control) return set_error(NERF_E_INVALID, "nerf_adamw_step: null control");
  const bool clip = config->max_norm > 0.0, norm = clip || (config->flags & NERF_ADAMW_SKIP_NONFINITE);
  if (norm && (workspace_bytes < nerf_adamw_workspace(n_tensors, tensors) ||
               (workspace_bytes && (!workspace || (uintptr_t(workspace) & 7)))))
    return set_error(NERF_E_INVALID, "nerf_adamw_step: workspace of %zu bytes, %zu needed (8-byte aligned)", workspace_bytes,
                     nerf_adamw_workspace(n_tensors, tensors));
  const hipStream_t s = (hipStream_t)stream;
  const int iters = iterations(n_tensors, tensors);
  double* part = static_cast<double*>(workspace);
  // launches of up to kTensors tensors of the same types, in order; pass 0 sums squares, pass 1 steps
  for (int pass = norm ? 0 : 1; pass < 2; ++pass) {
    AdamArgs a;
    std::memset(&a, 0, sizeof a);
    int grad = -1, model = -1;
    unsigned grid = 0;
    long done = 0;      // partials of the launches before
    auto launched = [&]() -> int {
      const hipError_t e = hipGetLastError();
      return e == hipSuccess ? NERF_OK : set_error(NERF_E_HIP, "nerf_adamw_step: %s", hipGetErrorString(e));
    };
    auto flush = [&]() -> int {
      if (a.n_tensors == 0) return NERF_OK;
      if (pass == 0) {
        if (grad == NERF_F32) hipLaunchKernelGGL((norm_kernel<float>), dim3(grid), dim3(256), 0, s, a, part + done);
        else if (grad == NERF_BFLOAT16) hipLaunchKernelGGL((norm_kernel<__bf16>), dim3(grid), dim3(256), 0, s, a, part + done);
        else hipLaunchKernelGGL((norm_kernel<_Float16>), dim3(grid), dim3(256), 0, s, a, part + done);
      } else {
        if (grad == NERF_F32) launch_step<float>(a, model, config->state_bits, grid, s);
        else if (grad == NERF_BFLOAT16) launch_step<__bf16>(a, model, config->state_bits, grid, s);
        else launch_step<_Float16>(a, model, config->state_bits, grid, s);
      }
      done += grid;
      a.n_tensors = 0, grid = 0;
      return launched();
    };
    if (pass == 1) {
      long n = 0;
      if (norm)
        for (int i = 0; i < n_tensors; ++i) n += chunks(tensors[i], iters);
      hipLaunchKernelGGL(prepare_kernel, dim3(1), dim3(1024), 0, s, control, (const double*)part, n, float(clip ? config->max_norm : 0.0),
                         config->beta1, config->beta2, config->flags & NERF_ADAMW_SKIP_NONFINITE);
      if ((rc = launched()) != NERF_OK) return rc;
    }
    a.iters = iters, a.flags = config->flags, a.ctl = control, a.lr_dev = config->lr_device;
    a.lr = float(config->lr), a.b1c = float(1.0 - config->beta1), a.b2 = float(config->beta2), a.b2c = float(1.0 - config->beta2);
    a.eps = float(config->eps);
    for (int i = 0; i < n_tensors; ++i) {
      const nerf_adamw_tensor& x = tensors[i];
      if (x.numel == 0) continue;
      const int md = x.model ? x.model_dtype : NERF_F32;
      const long c = chunks(x, iters);
      if (c > 0x40000000L) return set_error(NERF_E_INVALID, "nerf_adamw_step: tensor %d is too large", i);
      if (a.n_tensors == kTensors || x.grad_dtype != grad || md != model || grid + c > 0x7fffffffL)
        if ((rc = flush()) != NERF_OK) return rc;
      grad = x.grad_dtype, model = md;
      const int k = a.n_tensors++;
      a.t[k] = AdamTensor{x.param, x.model, x.grad, x.exp_avg, x.exp_avg_sq, x.exp_avg_scale, x.exp_avg_sq_scale, long(x.numel),
                          float(1.0 - config->lr * x.weight_decay), float(x.weight_decay)};
      a.first[k] = grid;
      const uintptr_t gsize = x.grad_dtype == NERF_F32 ? 15 : 7;
      a.wide[k] = !(uintptr_t(x.param) & 15) && !(uintptr_t(x.grad) & gsize) && !(uintptr_t(x.model) & 7) &&
                  !((uintptr_t(x.exp_avg) | uintptr_t(x.exp_avg_sq)) & (config->state_bits == 32 ? 15 : 3));
      grid += unsigned(c);
    }
    if ((rc = flush()) != NERF_OK) return rc;
  }
  return NERF_OK;
}

}  // extern "C"
