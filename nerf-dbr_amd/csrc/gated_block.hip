// The gated feed-forward block (nerf_gated_block_forward / _backward):
//   g = x Wg^T, u = x Wu^T, h = act(g) u, y = h Wd^T
//   dh = dy Wd, du = dh act(g), dg = dh u act'(g)
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dy^T h
// g and u never reach memory: the forward's first kernel holds both accumulators of a tile and writes
// h; the backward's first kernel recomputes them beside dh and writes h, dg and du.
#include <cmath>

#include "nerf_internal.h"

namespace nerf {
namespace {

// act(g) and act'(g)
__device__ __forceinline__ void activate(int kind, float g, float& a, float& d) {
  if (kind == NERF_RELU) {
    a = g > 0.0f ? g : (g != g ? g : 0.0f);
    d = g > 0.0f ? 1.0f : 0.0f;
  } else if (kind == NERF_SILU) {
    const float e = 1.0f / (1.0f + expf(-g));
    a = g * e;
    d = e * (1.0f + g * (1.0f - e));
  } else {
    const float c = 0.5f * erfcf(-g * 0.70710678118654752440f);
    a = g * c;
    d = c + g * expf(-0.5f * g * g) * 0.39894228040143267794f;
  }
}

// An operand: element (i, k) at p[i * si + k * sk], i the row or column of the product, k summed over.
struct Operand {
  const void* p;
  long si, sk;
};

constexpr int kT = 64, kK = 16;

// One 64 x 64 tile of sum over k of A(i, k) B(j, k) into acc, 4 x 4 values a thread; staged in LDS as fp32.
template <typename T>
__device__ __forceinline__ void tile_product(const Operand& a, const Operand& b, long i0, long j0, long m, long n, long k,
                                             float (*as)[kT + 1], float (*bs)[kT + 1], float acc[4][4]) {
  const int t = threadIdx.x, ti = t >> 4, tj = t & 15;
  const T* ap = static_cast<const T*>(a.p);
  const T* bp = static_cast<const T*>(b.p);
  for (long k0 = 0; k0 < k; k0 += kK) {
    __syncthreads();
    for (int e = t; e < kT * kK; e += 256) {
      // neighbouring threads along the operand's contiguous direction
      const int ai = a.sk == 1 ? e / kK : e % kT, ak = a.sk == 1 ? e % kK : e / kT;
      const int bi = b.sk == 1 ? e / kK : e % kT, bk = b.sk == 1 ? e % kK : e / kT;
      as[ak][ai] = i0 + ai < m && k0 + ak < k ? float(ap[(i0 + ai) * a.si + (k0 + ak) * a.sk]) : 0.0f;
      bs[bk][bi] = j0 + bi < n && k0 + bk < k ? float(bp[(j0 + bi) * b.si + (k0 + bk) * b.sk]) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kK; ++q)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[r][c] = fmaf(as[q][ti + 16 * r], bs[q][tj + 16 * c], acc[r][c]);
  }
}

// C (m x n, row stride ldc) = A1 B1 (+ A2 B2)
template <typename T>
__global__ __launch_bounds__(256) void product_kernel(Operand a1, Operand b1, Operand a2, Operand b2, long m, long n, long k, T* c,
                                                      long ldc) {
  __shared__ float as[kK][kT + 1], bs[kK][kT + 1];
  const long across = (n + kT - 1) / kT, i0 = blockIdx.x / across * kT, j0 = blockIdx.x % across * kT;
  float acc[4][4] = {};
  tile_product<T>(a1, b1, i0, j0, m, n, k, as, bs, acc);
  if (a2.p) tile_product<T>(a2, b2, i0, j0, m, n, k, as, bs, acc);
  for (int r = 0; r < 4; ++r)
    for (int q = 0; q < 4; ++q) {
      const long i = i0 + (threadIdx.x >> 4) + 16 * r, j = j0 + (threadIdx.x & 15) + 16 * q;
      if (i < m && j < n) c[i * ldc + j] = T(acc[r][q]);
    }
}

// h = act(x Wg^T) (x Wu^T); with dy also dg and du
template <typename T, bool BACK>
__global__ __launch_bounds__(256) void gate_kernel(Operand x, Operand wg, Operand wu, Operand dy, Operand wd, long rows, long hidden,
                                                   long width, long out, int kind, T* h, T* dg, T* du) {
  __shared__ float as[kK][kT + 1], bs[kK][kT + 1];
  const long across = (hidden + kT - 1) / kT, i0 = blockIdx.x / across * kT, j0 = blockIdx.x % across * kT;
  float g[4][4] = {}, u[4][4] = {}, d[4][4] = {};
  tile_product<T>(x, wg, i0, j0, rows, hidden, width, as, bs, g);
  tile_product<T>(x, wu, i0, j0, rows, hidden, width, as, bs, u);
  if (BACK) tile_product<T>(dy, wd, i0, j0, rows, hidden, out, as, bs, d);
  for (int r = 0; r < 4; ++r)
    for (int q = 0; q < 4; ++q) {
      const long i = i0 + (threadIdx.x >> 4) + 16 * r, j = j0 + (threadIdx.x & 15) + 16 * q;
      if (i >= rows || j >= hidden) continue;
      float a, s;
      activate(kind, g[r][q], a, s);
      h[i * hidden + j] = T(a * u[r][q]);
      if (BACK) {
        dg[i * hidden + j] = T(d[r][q] * u[r][q] * s);
        du[i * hidden + j] = T(d[r][q] * a);
      }
    }
}

dim3 tiles(long m, long n) { return dim3(unsigned(((n + kT - 1) / kT) * ((m + kT - 1) / kT))); }

template <typename T>
hipError_t forward(const nerf_block_desc& d, T* y, long ld_y, void* ws, hipStream_t s) {
  T* h = static_cast<T*>(ws);
  const Operand x{d.x, d.ld_x, 1}, wg{d.w_gate, d.ld_gate, 1}, wu{d.w_up, d.ld_up, 1}, wd{d.w_down, d.ld_down, 1}, no{};
  hipLaunchKernelGGL((gate_kernel<T, false>), tiles(d.rows, d.hidden), dim3(256), 0, s, x, wg, wu, no, no, long(d.rows), long(d.hidden),
                     long(d.width), 0L, d.activation, h, (T*)nullptr, (T*)nullptr);
  hipLaunchKernelGGL((product_kernel<T>), tiles(d.rows, d.out), dim3(256), 0, s, Operand{h, d.hidden, 1}, wd, no, no, long(d.rows),
                     long(d.out), long(d.hidden), y, ld_y);
  return hipGetLastError();
}

template <typename T>
hipError_t backward(const nerf_block_desc& d, const void* dy, long ld_dy, T* dx, long ld_dx, T* dwg, T* dwu, T* dwd, void* ws,
                    hipStream_t s) {
  const long n = long(d.rows) * d.hidden;
  T *h = static_cast<T*>(ws), *dg = h + n, *du = dg + n;
  const long rows = d.rows, width = d.width, hidden = d.hidden, out = d.out;
  const Operand x{d.x, d.ld_x, 1}, wg{d.w_gate, d.ld_gate, 1}, wu{d.w_up, d.ld_up, 1}, no{};
  if (rows) hipLaunchKernelGGL((gate_kernel<T, true>), tiles(rows, hidden), dim3(256), 0, s, x, wg, wu, Operand{dy, ld_dy, 1},
                     Operand{d.w_down, 1, d.ld_down}, rows, hidden, width, out, d.activation, h, dg, du);
  auto product = [&](Operand a1, Operand b1, Operand a2, Operand b2, long m, long nn, long k, T* c, long ldc) {
    if (c && m) hipLaunchKernelGGL((product_kernel<T>), tiles(m, nn), dim3(256), 0, s, a1, b1, a2, b2, m, nn, k, c, ldc);
  };
  product({dg, hidden, 1}, {d.w_gate, 1, d.ld_gate}, {du, hidden, 1}, {d.w_up, 1, d.ld_up}, rows, width, hidden, dx, ld_dx);
  const Operand xt{d.x, 1, d.ld_x};
  product({dg, 1, hidden}, xt, no, no, hidden, width, rows, dwg, width);
  product({du, 1, hidden}, xt, no, no, hidden, width, rows, dwu, width);
  product({dy, 1, ld_dy}, {h, 1, hidden}, no, no, out, hidden, rows, dwd, hidden);
  return hipGetLastError();
}

int check(const nerf_block_desc* d, const char* who) {
  if (!d) return set_error(NERF_E_INVALID, "%s: null descriptor", who);
  if (d->dtype != NERF_F32 && d->dtype != NERF_BFLOAT16 && d->dtype != NERF_FLOAT16) return set_error(NERF_E_INVALID, "%s: dtype %d", who, d->dtype);
  if (d->activation < NERF_SILU || d->activation > NERF_RELU) return set_error(NERF_E_INVALID, "%s: activation %d", who, d->activation);
  if (d->rows < 0 || d->rows > (1L << 31) || d->width < 1 || d->hidden < 1 || d->out < 1 || d->width > (1 << 20) || d->hidden > (1 << 20) ||
      d->out > (1 << 20))
    return set_error(NERF_E_INVALID, "%s: rows %ld, width %d, hidden %d, out %d", who, long(d->rows), d->width, d->hidden, d->out);
  const long widest = d->width > d->hidden ? (d->width > d->out ? d->width : d->out) : d->hidden > d->out ? d->hidden : d->out;
  if (((d->rows + kT - 1) / kT) * ((widest + kT - 1) / kT) > 0x7fffffffL) return set_error(NERF_E_INVALID, "%s: too many tiles", who);
  if (d->ld_x < d->width || d->ld_gate < d->width || d->ld_up < d->width || d->ld_down < d->hidden)
    return set_error(NERF_E_INVALID, "%s: a row stride is shorter than its row", who);
  if ((d->rows && !d->x) || !d->w_gate || !d->w_up || !d->w_down) return set_error(NERF_E_INVALID, "%s: null operand", who);
  const uintptr_t low = d->dtype == NERF_F32 ? 3 : 1;
  if ((uintptr_t(d->x) | uintptr_t(d->w_gate) | uintptr_t(d->w_up) | uintptr_t(d->w_down)) & low)
    return set_error(NERF_E_INVALID, "%s: an operand is not aligned to its type", who);
  return NERF_OK;
}

int check_workspace(const nerf_block_desc* d, int back, const void* ws, size_t bytes, const char* who) {
  const size_t need = nerf_gated_block_workspace(d, back);
  if (bytes < need || (need && (!ws || (uintptr_t(ws) & 255))))
    return set_error(NERF_E_INVALID, "%s: workspace of %zu bytes, %zu needed (256-byte aligned)", who, bytes, need);
  return NERF_OK;
}

}  // namespace
}  // namespace nerf

using namespace nerf;

extern "C" {

size_t nerf_gated_block_workspace(const nerf_block_desc* d, int backward) {
  if (check(d, "nerf_gated_block_workspace") != NERF_OK) return 0;
  return size_t(d->rows) * d->hidden * (d->dtype == NERF_F32 ? 4 : 2) * (backward ? 3 : 1);
}

int nerf_gated_block_forward(const nerf_block_desc* d, void* y, int64_t ld_y, void* workspace, size_t workspace_bytes,
                             void* stream) {
  static const char* who = "nerf_gated_block_forward";
  int rc = check(d, who);
  if (rc != NERF_OK) return rc;
  if (d->rows == 0) return NERF_OK;
  if (!y || ld_y < d->out || (uintptr_t(y) & (d->dtype == NERF_F32 ? 3 : 1))) return set_error(NERF_E_INVALID, "%s: y or its row stride %ld", who, long(ld_y));
  if ((rc = check_workspace(d, 0, workspace, workspace_bytes, who)) != NERF_OK) return rc;
  const hipStream_t s = (hipStream_t)stream;
  const hipError_t e = d->dtype == NERF_F32        ? forward<float>(*d, (float*)y, ld_y, workspace, s)
                       : d->dtype == NERF_BFLOAT16 ? forward<__bf16>(*d, (__bf16*)y, ld_y, workspace, s)
                                                   : forward<_Float16>(*d, (_Float16*)y, ld_y, workspace, s);
  if (e != hipSuccess) return set_error(NERF_E_HIP, "%s: %s", who, hipGetErrorString(e));
  return NERF_OK;
}

int nerf_gated_block_backward(const nerf_block_desc* d, const void* dy, int64_t ld_dy, void* dx, int64_t ld_dx, void* dw_gate,
                              void* dw_up, void* dw_down, void* workspace, size_t workspace_bytes, void* stream) {
  static const char* who = "nerf_gated_block_backward";
  int rc = check(d, who);
  if (rc != NERF_OK) return rc;
  const uintptr_t low = d->dtype == NERF_F32 ? 3 : 1;
  if ((d->rows && !dy) || ld_dy < d->out) return set_error(NERF_E_INVALID, "%s: dy or its row stride %ld", who, long(ld_dy));
  if (dx && ld_dx < d->width) return set_error(NERF_E_INVALID, "%s: row stride %ld of dx", who, long(ld_dx));
  if ((uintptr_t(dy) | uintptr_t(dx) | uintptr_t(dw_gate) | uintptr_t(dw_up) | uintptr_t(dw_down)) & low)
    return set_error(NERF_E_INVALID, "%s: a gradient is not aligned to its type", who);
  if (!dx && !dw_gate && !dw_up && !dw_down) return NERF_OK;
  if ((rc = check_workspace(d, 1, workspace, workspace_bytes, who)) != NERF_OK) return rc;
  const hipStream_t s = (hipStream_t)stream;
  const hipError_t e =
      d->dtype == NERF_F32 ? backward<float>(*d, dy, ld_dy, (float*)dx, ld_dx, (float*)dw_gate, (float*)dw_up, (float*)dw_down, workspace, s)
      : d->dtype == NERF_BFLOAT16
          ? backward<__bf16>(*d, dy, ld_dy, (__bf16*)dx, ld_dx, (__bf16*)dw_gate, (__bf16*)dw_up, (__bf16*)dw_down, workspace, s)
          : backward<_Float16>(*d, dy, ld_dy, (_Float16*)dx, ld_dx, (_Float16*)dw_gate, (_Float16*)dw_up, (_Float16*)dw_down, workspace, s);
  if (e != hipSuccess) return set_error(NERF_E_HIP, "%s: %s", who, hipGetErrorString(e));
  return NERF_OK;
}

}  // extern "C"
