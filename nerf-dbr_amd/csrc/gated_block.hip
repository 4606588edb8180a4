// The gated feed-forward block (nerf_gated_block_forward / _backward):
//   g = x Wg^T, u = x Wu^T, h = act(g) u, y = h Wd^T
//   dh = dy Wd, du = dh act(g), dg = dh u act'(g)
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dy^T h
// g and u never reach memory: the forward's first kernel holds both accumulators of a tile and writes
// h; the backward's first kernel recomputes them beside dh and writes h, dg and du.
#include <cmath>

#include "block_mma.h"
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

// ------------------------------------------------------------------ 16-bit types on the matrix cores --
// The 256 x 256 tile of 8 waves carries long products; the 128 x 128 tile of 4 waves (two workgroups a CU)
// fills the machine where there are few tiles.
typedef Tile<2, 4, 8, 4> Large;
typedef Tile<2, 2, 4, 4> Small;

// h = act(x Wg^T) (x Wu^T): the J tile holds TJ / 2 rows of Wg and the same rows of Wu, so a lane owns the
// same (row, column) of both and the activation runs on accumulators.  h's columns behind `hidden` up to
// its row stride are zeros: they are summed over by the next product.
template <typename T, typename C>
__global__ __launch_bounds__(C::NT, 2) void gate_mma_kernel(Side x, Side w, int steps, int kind, T* h, long ld_h, long rows,
                                                                      long hidden, unsigned tiles_i, unsigned tiles_j) {
  __shared__ __attribute__((aligned(1024))) char lds[2 * (C::TI + C::TJ) * 128];
  unsigned ti, tj;
  tile_of(blockIdx.x, gridDim.x, tiles_i, tiles_j, ti, tj);
  const long i0 = long(ti) * C::TI, j0 = long(tj) * (C::TJ / 2);
  f32x4_t acc[C::NJ][C::NI] = {};
  accumulate<T, C, true, true, 2>(acc, x, w, i0, j0, steps, 0, steps, lds_addr(lds));
  const int wave = threadIdx.x >> 6, l = threadIdx.x & 63;
  const long ib = i0 + (wave / C::WJ) * C::NI * 16 + (l & 15), jb = j0 + (wave % C::WJ) * (C::NJ / 2) * 16 + (l >> 4) * 4;
#pragma unroll
  for (int i = 0; i < C::NI; ++i)
#pragma unroll
    for (int j = 0; j < C::NJ / 2; ++j) {
      const long row = ib + i * 16, col = jb + j * 16;
      if (row >= rows || col >= ld_h) continue;
      f32x4_t o;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float a, d;
        activate(kind, acc[j][i][r], a, d);
        o[r] = col + r < hidden ? a * acc[j + C::NJ / 2][i][r] : 0.0f;
      }
      store_row4(h + row * ld_h, col, ld_h, true, o);
    }
}

// The backward's first kernel: g and u as above, then dh = dy Wd of the same tile in a third accumulator,
// and h, dg and du of the tile from the three.
template <typename T, typename C>
__global__ __launch_bounds__(C::NT, 2) void gate_back_mma_kernel(Side x, Side w, Side dy, Side wd, int steps, int steps_dy,
                                                                           int kind, T* h, T* dg, T* du, long ld_h, long rows,
                                                                           long hidden, unsigned tiles_i, unsigned tiles_j) {
  typedef Tile<C::WI, C::WJ, C::NI, C::NJ / 2> Half;
  __shared__ __attribute__((aligned(1024))) char lds[2 * (C::TI + C::TJ) * 128];
  unsigned ti, tj;
  tile_of(blockIdx.x, gridDim.x, tiles_i, tiles_j, ti, tj);
  const long i0 = long(ti) * C::TI, j0 = long(tj) * Half::TJ;
  f32x4_t acc[C::NJ][C::NI] = {}, dh[Half::NJ][C::NI] = {};
  accumulate<T, C, true, true, 2>(acc, x, w, i0, j0, steps, 0, steps, lds_addr(lds));
  accumulate<T, Half, true, false, 1>(dh, dy, wd, i0, j0, steps_dy, 0, steps_dy, lds_addr(lds));
  const int wave = threadIdx.x >> 6, l = threadIdx.x & 63;
  const long ib = i0 + (wave / C::WJ) * C::NI * 16 + (l & 15), jb = j0 + (wave % C::WJ) * Half::NJ * 16 + (l >> 4) * 4;
#pragma unroll
  for (int i = 0; i < C::NI; ++i)
#pragma unroll
    for (int j = 0; j < Half::NJ; ++j) {
      const long row = ib + i * 16, col = jb + j * 16;
      if (row >= rows || col >= ld_h) continue;
      f32x4_t oh, og, ou;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float a, s;
        activate(kind, acc[j][i][r], a, s);
        const float u = acc[j + Half::NJ][i][r], d = dh[j][i][r];
        const bool in = col + r < hidden;
        oh[r] = in ? a * u : 0.0f;
        og[r] = in ? d * u * s : 0.0f;
        ou[r] = in ? d * a : 0.0f;
      }
      store_row4(h + row * ld_h, col, ld_h, true, oh);
      store_row4(dg + row * ld_h, col, ld_h, true, og);
      store_row4(du + row * ld_h, col, ld_h, true, ou);
    }
}

// C(i, j) of up to three problems in one launch, the sum over k cut into `splits` where tiles are few: then
// each piece leaves fp32 partials (fragment order: neighbouring threads, neighbouring 16 bytes) that
// join_kernel adds in order.
struct Problem {
  Side i, j;
  void* out;
  long ld;           // elements
  long m, n;         // C is m x n; a side whose rows were padded to 8 has a larger extent
  int steps;         // steps of 64 k of one segment
  int segs;
  int per;           // steps of a piece
  unsigned splits, tiles_i, tiles_j, first;   // first workgroup
  long part;         // first partial tile of this problem
  int wide;
};
struct Problems {
  Problem p[3];
  int n;
  float* part;
};
template <typename C, typename O>
__device__ __forceinline__ void store_tile(const Problem& p, unsigned ti, unsigned tj, int i, int j, f32x4_t v) {
  const int wave = threadIdx.x >> 6, l = threadIdx.x & 63;
  const long row = long(ti) * C::TI + ((wave / C::WJ) * C::NI + i) * 16 + (l & 15);
  const long col = long(tj) * C::TJ + ((wave % C::WJ) * C::NJ + j) * 16 + (l >> 4) * 4;
  if (row < p.m && col < p.n) store_row4(static_cast<O*>(p.out) + row * p.ld, col, p.n, p.wide, v);
}
template <typename T, typename C, bool IK, bool JK, typename O>
__global__ __launch_bounds__(C::NT, 2) void product_mma_kernel(Problems all) {
  __shared__ __attribute__((aligned(1024))) char lds[2 * (C::TI + C::TJ) * 128];
  int k = 0;
  while (k + 1 < all.n && blockIdx.x >= all.p[k + 1].first) ++k;
  const Problem& p = all.p[k];
  const unsigned tiles = p.tiles_i * p.tiles_j, b = blockIdx.x - p.first;
  const unsigned split = b / tiles;
  unsigned ti, tj;
  tile_of(b - split * tiles, tiles, p.tiles_i, p.tiles_j, ti, tj);
  f32x4_t acc[C::NJ][C::NI] = {};
  const int total = p.steps * p.segs, first = int(split) * p.per, last = first + p.per < total ? first + p.per : total;
  accumulate<T, C, IK, JK, 1>(acc, p.i, p.j, long(ti) * C::TI, long(tj) * C::TJ, p.steps, first, last, lds_addr(lds));
  if (p.splits == 1) {
#pragma unroll
    for (int i = 0; i < C::NI; ++i)
#pragma unroll
      for (int j = 0; j < C::NJ; ++j) store_tile<C, O>(p, ti, tj, i, j, acc[j][i]);
  } else {
    f32x4_t* part = reinterpret_cast<f32x4_t*>(all.part) + (p.part + long(split) * tiles + long(ti) * p.tiles_j + tj) * (C::NI * C::NJ * C::NT);
#pragma unroll
    for (int i = 0; i < C::NI; ++i)
#pragma unroll
      for (int j = 0; j < C::NJ; ++j) part[(i * C::NJ + j) * C::NT + threadIdx.x] = acc[j][i];
  }
}
// workgroup: one fragment of every wave of one tile
template <typename C, typename O>
__global__ __launch_bounds__(C::NT) void join_kernel(Problem p, const float* parts) {
  const unsigned tile = blockIdx.x / (C::NI * C::NJ);
  const int f = int(blockIdx.x % (C::NI * C::NJ));
  const long tiles = long(p.tiles_i) * p.tiles_j, step = tiles * (C::NI * C::NJ * C::NT);
  const f32x4_t* part = reinterpret_cast<const f32x4_t*>(parts) + (p.part + tile) * (C::NI * C::NJ * C::NT) + f * C::NT + threadIdx.x;
  f32x4_t v = part[0];
#pragma unroll 4
  for (unsigned s = 1; s < p.splits; ++s) v += part[s * step];
  store_tile<C, O>(p, tile / p.tiles_j, tile % p.tiles_j, f / C::NJ, f % C::NJ, v);
}

// Rows of `n` values copied to rows of a multiple of 8, zeros behind: operands whose rows are not whole
// aligned 16-byte pieces.
template <typename T>
__global__ __launch_bounds__(256) void pad_kernel(const T* src, long ld, long rows, long n, T* dst, long ld_dst) {
  const long per = ld_dst / 8, e = long(blockIdx.x) * 256 + threadIdx.x;
  if (e >= rows * per) return;
  const long r = e / per, c = (e - r * per) * 8;
  Out4<T> o[2];
#pragma unroll
  for (int k = 0; k < 8; ++k) o[k / 4].v[k % 4] = c + k < n ? src[r * ld + c + k] : T(0.0f);
  Out4<T>* to = reinterpret_cast<Out4<T>*>(dst + r * ld_dst + c);
  to[0] = o[0];
  to[1] = o[1];
}

// --------------------------------------------------------------------------------------------- host --
constexpr long align_up(long n, long a) { return (n + a - 1) / a * a; }

// Takes memory from the workspace; with no base it only counts.
struct Arena {
  char* base;
  size_t used = 0;
  void* take(size_t bytes) {
    void* p = base ? base + used : nullptr;
    used += size_t(align_up(long(bytes), 256));
    return p;
  }
};

// A 16-bit matrix [rows][n] as a product reads it: where it lies, or a padded copy.
struct Matrix {
  const void* p;
  long ld;      // elements
  long rows, n, n8;
};
bool whole(const void* p, long ld, long n) { return !(uintptr_t(p) & 15) && ld % 8 == 0 && n % 8 == 0; }

Side rows_side(const Matrix& m) {      // i = row, k = column
  Side s{};
  s.p[0] = static_cast<const char*>(m.p), s.ld = m.ld * 2, s.n = m.rows, s.k_n = m.n8;
  return s;
}
Side columns_side(const Matrix& m) {   // i = column, k = row
  Side s{};
  s.p[0] = static_cast<const char*>(m.p), s.ld = m.ld * 2, s.n = m.n8, s.k_n = m.rows;
  return s;
}

// Large tiles where they fill the machine nearly as well as small ones do: a small tile runs its products
// at about 3/4 of the large one's rate.
bool use_large(long m, long n) {
  const long l = ((m + 255) / 256) * ((n + 255) / 256), s = ((m + 127) / 128) * ((n + 127) / 128);
  const double fl = double(l) / (256.0 * ((l + 255) / 256)), fs = double(s) / (512.0 * ((s + 511) / 512));
  return fl >= 0.75 * fs;
}

struct Run {
  hipStream_t s;
  Arena a;
  bool go;      // false: only count the workspace

  template <typename T>
  Matrix matrix(const void* p, long ld, long rows, long n) {
    const long n8 = align_up(n, 8);
    if (whole(p, ld, n)) return Matrix{p, ld, rows, n, n8};
    return padded<T>(p, ld, rows, n);
  }
  template <typename T>
  Matrix padded(const void* p, long ld, long rows, long n) {
    const long n8 = align_up(n, 8);
    T* q = static_cast<T*>(a.take(size_t(rows) * n8 * sizeof(T)));
    if (go && rows) hipLaunchKernelGGL((pad_kernel<T>), dim3(unsigned((rows * (n8 / 8) + 255) / 256)), dim3(256), 0, s, static_cast<const T*>(p), ld, rows, n, q, n8);
    return Matrix{q, n8, rows, n, n8};
  }

  // C = the segments' products for up to three problems of one kind; partials come from the arena.
  template <typename T, bool IK, bool JK, typename O, typename C>
  void products_of(Problems& all) {
    unsigned grid = 0;
    long tiles = 0, parts = 0;
    for (int k = 0; k < all.n; ++k) {
      Problem& p = all.p[k];
      p.tiles_i = unsigned((p.m + C::TI - 1) / C::TI), p.tiles_j = unsigned((p.n + C::TJ - 1) / C::TJ);
      tiles += long(p.tiles_i) * p.tiles_j;
    }
    if (tiles == 0) return;      // no rows
    const long slots = 256L * (512 / C::NT);
    for (int k = 0; k < all.n; ++k) {
      Problem& p = all.p[k];
      const int total = p.steps * p.segs;
      // pieces of at least 8 steps, as many as make one full wave of workgroups
      long splits = tiles < slots ? slots / tiles : 1;
      splits = splits > total / 8 ? total / 8 : splits;
      splits = splits < 1 ? 1 : splits;
      p.per = int((total + splits - 1) / splits);
      p.splits = total ? unsigned((total + p.per - 1) / p.per) : 1;
      p.first = grid;
      p.part = parts;
      grid += p.tiles_i * p.tiles_j * p.splits;
      if (p.splits > 1) parts += long(p.tiles_i) * p.tiles_j * p.splits;
    }
    all.part = static_cast<float*>(a.take(size_t(parts) * C::TI * C::TJ * 4));
    if (!go || !grid) return;
    hipLaunchKernelGGL((product_mma_kernel<T, C, IK, JK, O>), dim3(grid), dim3(C::NT), 0, s, all);
    for (int k = 0; k < all.n; ++k)
      if (all.p[k].splits > 1)
        hipLaunchKernelGGL((join_kernel<C, O>), dim3(all.p[k].tiles_i * all.p[k].tiles_j * C::NI * C::NJ), dim3(C::NT), 0, s, all.p[k],
                           (const float*)all.part);
  }
  template <typename T, bool IK, bool JK, typename O>
  void products(Problems& all) {
    bool large = false;
    for (int k = 0; k < all.n; ++k) large = large || use_large(all.p[k].m, all.p[k].n);
    if (large) products_of<T, IK, JK, O, Large>(all);
    else products_of<T, IK, JK, O, Small>(all);
  }
};

template <typename O>
Problem problem(const Side& i, const Side& j, long m, long n, long k, int segs, void* out, long ld) {
  Problem p{};
  p.i = i, p.j = j, p.m = m, p.n = n, p.out = out, p.ld = ld, p.steps = int((k + 63) / 64), p.segs = segs;
  p.wide = !(uintptr_t(out) & (4 * sizeof(O) - 1)) && ld % 4 == 0;
  return p;
}

// Wg and Wu with one row stride, as one side of two halves or one segment list reads them.
struct Pair {
  Matrix g, u;
};
template <typename T>
Pair weights(Run& r, const nerf_block_desc& d) {
  const long n8 = align_up(d.width, 8);
  if (d.ld_gate == d.ld_up && whole(d.w_gate, d.ld_gate, d.width) && whole(d.w_up, d.ld_up, d.width))
    return {{d.w_gate, d.ld_gate, d.hidden, d.width, n8}, {d.w_up, d.ld_up, d.hidden, d.width, n8}};
  return {r.padded<T>(d.w_gate, d.ld_gate, d.hidden, d.width), r.padded<T>(d.w_up, d.ld_up, d.hidden, d.width)};
}
Side halves(const Pair& w) {
  Side s = rows_side(w.g);
  s.split = static_cast<const char*>(w.u.p) - static_cast<const char*>(w.g.p);
  return s;
}

template <typename C>
dim3 gate_grid(long rows, long hidden, unsigned& ti, unsigned& tj) {
  ti = unsigned((rows + C::TI - 1) / C::TI), tj = unsigned((hidden + C::TJ / 2 - 1) / (C::TJ / 2));
  return dim3(ti * tj);
}
int steps_of(long k) { return int((k + 63) / 64); }

template <typename T>
hipError_t forward_mma(const nerf_block_desc& d, T* y, long ld_y, Run& r) {
  const long rows = d.rows, hidden = d.hidden, hp = align_up(hidden, 8);
  const Matrix x = r.matrix<T>(d.x, d.ld_x, rows, d.width);
  const Pair w = weights<T>(r, d);
  const Matrix wd = r.matrix<T>(d.w_down, d.ld_down, d.out, hidden);
  T* h = static_cast<T*>(r.a.take(size_t(rows) * hp * sizeof(T)));
  unsigned ti, tj;
  if (r.go) {
    if (use_large(rows, 2 * hidden))
      hipLaunchKernelGGL((gate_mma_kernel<T, Large>), gate_grid<Large>(rows, hp, ti, tj), dim3(Large::NT), 0, r.s, rows_side(x), halves(w),
                         steps_of(d.width), d.activation, h, hp, rows, hidden, ti, tj);
    else
      hipLaunchKernelGGL((gate_mma_kernel<T, Small>), gate_grid<Small>(rows, hp, ti, tj), dim3(Small::NT), 0, r.s, rows_side(x), halves(w),
                         steps_of(d.width), d.activation, h, hp, rows, hidden, ti, tj);
  }
  Problems all{};
  all.n = 1;
  all.p[0] = problem<T>(rows_side(Matrix{h, hp, rows, hidden, hp}), rows_side(wd), rows, d.out, hidden, 1, y, ld_y);
  r.products<T, true, true, T>(all);
  return hipGetLastError();
}

template <typename T>
hipError_t backward_mma(const nerf_block_desc& d, const void* dy_p, long ld_dy, T* dx, long ld_dx, T* dwg, T* dwu, T* dwd, Run& r) {
  const long rows = d.rows, width = d.width, hidden = d.hidden, out = d.out, hp = align_up(hidden, 8);
  const Matrix x = r.matrix<T>(d.x, d.ld_x, rows, width);
  const Pair w = weights<T>(r, d);
  const Matrix wd = r.matrix<T>(d.w_down, d.ld_down, out, hidden);
  // the workspace is asked for before dy is known: count its copy
  const Matrix dy = r.go ? r.matrix<T>(dy_p, ld_dy, rows, out) : r.padded<T>(nullptr, out, rows, out);
  T* h = static_cast<T*>(r.a.take(size_t(rows) * hp * sizeof(T)));
  T* dg = static_cast<T*>(r.a.take(size_t(rows) * hp * sizeof(T)));
  T* du = static_cast<T*>(r.a.take(size_t(rows) * hp * sizeof(T)));
  unsigned ti, tj;
  if (r.go && rows) {
    if (use_large(rows, 2 * hidden))
      hipLaunchKernelGGL((gate_back_mma_kernel<T, Large>), gate_grid<Large>(rows, hp, ti, tj), dim3(Large::NT), 0, r.s, rows_side(x),
                         halves(w), rows_side(dy), columns_side(wd), steps_of(width), steps_of(out), d.activation, h, dg, du, hp, rows,
                         hidden, ti, tj);
    else
      hipLaunchKernelGGL((gate_back_mma_kernel<T, Small>), gate_grid<Small>(rows, hp, ti, tj), dim3(Small::NT), 0, r.s, rows_side(x),
                         halves(w), rows_side(dy), columns_side(wd), steps_of(width), steps_of(out), d.activation, h, dg, du, hp, rows,
                         hidden, ti, tj);
  }
  const Matrix mh{h, hp, rows, hidden, hp}, mg{dg, hp, rows, hidden, hp}, mu{du, hp, rows, hidden, hp};
  if ((dx || !r.go) && rows) {
    Side i = rows_side(mg), j = columns_side(w.g);
    i.p[1] = reinterpret_cast<const char*>(du);
    j.p[1] = static_cast<const char*>(w.u.p);
    Problems all{};
    all.n = 1;
    all.p[0] = problem<T>(i, j, rows, width, hidden, 2, dx, ld_dx);
    r.products<T, true, false, T>(all);
  }
  Problems all{};
  if (dwg || !r.go) all.p[all.n++] = problem<T>(columns_side(mg), columns_side(x), hidden, width, rows, 1, dwg, width);
  if (dwu || !r.go) all.p[all.n++] = problem<T>(columns_side(mu), columns_side(x), hidden, width, rows, 1, dwu, width);
  if (dwd || !r.go) all.p[all.n++] = problem<T>(columns_side(dy), columns_side(mh), out, hidden, rows, 1, dwd, hidden);
  if (all.n) r.products<T, false, false, T>(all);
  return hipGetLastError();
}

// ------------------------------------------------------------------------------- 32-bit, plain tiles --
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
  if (d->dtype == NERF_F32) return size_t(d->rows) * d->hidden * 4 * (backward ? 3 : 1);
  Run r{nullptr, Arena{nullptr}, false};
  if (backward) (void)backward_mma<__bf16>(*d, nullptr, 0, nullptr, 0, nullptr, nullptr, nullptr, r);
  else (void)forward_mma<__bf16>(*d, nullptr, 0, r);
  return r.a.used;
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
  Run r{s, Arena{static_cast<char*>(workspace)}, true};
  const hipError_t e = d->dtype == NERF_F32        ? forward<float>(*d, (float*)y, ld_y, workspace, s)
                       : d->dtype == NERF_BFLOAT16 ? forward_mma<__bf16>(*d, (__bf16*)y, ld_y, r)
                                                   : forward_mma<_Float16>(*d, (_Float16*)y, ld_y, r);
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
  Run r{s, Arena{static_cast<char*>(workspace)}, true};
  const hipError_t e =
      d->dtype == NERF_F32 ? backward<float>(*d, dy, ld_dy, (float*)dx, ld_dx, (float*)dw_gate, (float*)dw_up, (float*)dw_down, workspace, s)
      : d->dtype == NERF_BFLOAT16
          ? backward_mma<__bf16>(*d, dy, ld_dy, (__bf16*)dx, ld_dx, (__bf16*)dw_gate, (__bf16*)dw_up, (__bf16*)dw_down, r)
          : backward_mma<_Float16>(*d, dy, ld_dy, (_Float16*)dx, ld_dx, (_Float16*)dw_gate, (_Float16*)dw_up, (_Float16*)dw_down, r);
  if (e != hipSuccess) return set_error(NERF_E_HIP, "%s: %s", who, hipGetErrorString(e));
  return NERF_OK;
}

}  // extern "C"
