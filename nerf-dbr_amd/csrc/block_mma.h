// The tiled 16-bit matrix product under the gated block: C(i, j) = sum over k of I(i, k) J(j, k), fp32
// accumulators, on v_mfma_f32_16x16x32.
//
// A side (I or J) is read as it lies: k contiguous (rows of x, of a weight) or its own index contiguous
// (the same rows when the sum runs over them); no operand is transposed in memory.  64 values of k of
// both sides are staged in LDS per step by 16-byte LDS-DMA, two stages deep: the next step's pieces fly
// while this one's fragments are read.
//   k contiguous:   LDS [row][64 k], 128 bytes a row, 16-byte chunk c of row r at chunk c ^ (r & 7): a
//                   fragment is one 16-byte read, and eight neighbouring rows meet all banks once;
//   own contiguous: LDS [64 k][E], 32-byte granule p of row k at granule p ^ f(k); a fragment is two
//                   transposing reads (ds_read_b64_tr_b16: 16 lanes read 4 rows of 16 values and each gets
//                   one column), and the 4 rows a group reads meet different banks.
// The DMA writes lane-linearly, so the swizzle is applied to the global address each lane fetches.
#pragma once
#include <hip/hip_runtime.h>

#include "nerf_asm.h"

namespace nerf {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 frag_bf16 __attribute__((ext_vector_type(8)));
typedef _Float16 frag_f16 __attribute__((ext_vector_type(8)));
typedef short short4_t __attribute__((ext_vector_type(4)));

template <typename T>
struct Frag;
template <>
struct Frag<__bf16> {
  typedef frag_bf16 type;
  static __device__ __forceinline__ f32x4_t mma(type a, type b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Frag<_Float16> {
  typedef frag_f16 type;
  static __device__ __forceinline__ f32x4_t mma(type a, type b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

// 16 bytes per lane from its own address to LDS byte lds_base + lane * 16 (wave-uniform base in M0);
// completion counts in vmcnt.  nerf_asm.h says why this is asm and who checks M0.
__device__ __forceinline__ void lds_dma_16(const void* p, unsigned lds_base) {
  const unsigned base = __builtin_amdgcn_readfirstlane(lds_base);
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  asm volatile(
      "s_mov_b32 m0, %1\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %0, off"
      :
      : "v"(p), "s"(base)
      : "memory", "m0");
#pragma clang diagnostic pop
}

__device__ __attribute__((aligned(16))) const unsigned kZeros[4] = {0, 0, 0, 0};   // what stands behind the end of k

constexpr int kMaxSegs = 6;
// One operand: `segs` matrices of the same shape whose products are added up (the launch's segs).
// k contiguous: element (i, k) at p + i * ld + 2 k; own contiguous: at p + k * ld + 2 i.  Every p and ld is
// a multiple of 16 bytes; the contiguous extent (k_n, or n) is a multiple of 8.  split > 0: rows of a tile
// behind the first half come from p + split (a second matrix of the same shape).
struct Side {
  const char* p[kMaxSegs];
  long ld;
  long split;
  long n;     // extent of i
  long k_n;   // extent of k: zeros behind it
};

// E: the tile's extent of the side; NT: threads; KC: k contiguous; PARTS: 2 = halves from two matrices
template <int E, int NT, bool KC, int PARTS>
struct Stage {
  static constexpr int kBytes = E * 64 * 2;
  static constexpr int kChunks = E * 8 / NT;   // 16-byte pieces a thread fetches per step
  long off[kChunks];                           // from p, without k

  static __device__ __forceinline__ int gran(int k) { return ((k & 3) | (((k >> 3) & 3) << 2)) & (E / 16 - 1); }

  __device__ __forceinline__ void init(const Side& s, long i0) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int q = c * NT + threadIdx.x;
      if (KC) {
        const int r = q >> 3, chunk = (q & 7) ^ (r & 7);
        const int rr = PARTS == 2 ? r & (E / 2 - 1) : r;
        long row = i0 + rr;
        row = row < s.n ? row : s.n - 1;      // behind the edge: any row, its results are not stored
        off[c] = row * s.ld + chunk * 16 + (PARTS == 2 && r >= E / 2 ? s.split : 0);
      } else {
        const int k = q / (E / 8), slot = q & (E / 8 - 1);
        long col = i0 + ((slot >> 1) ^ gran(k)) * 16 + (slot & 1) * 8;
        col = col < s.n ? col : s.n - 8;
        off[c] = k * s.ld + col * 2;
      }
    }
  }
  // fetch the 64 values of k from k0 of one segment into the stage at LDS byte `lds`
  __device__ __forceinline__ void fetch(const char* p, const Side& s, long k0, unsigned lds) const {
    const char* base = p + (KC ? k0 * 2 : k0 * s.ld);
    const unsigned wave = threadIdx.x & ~63u;
    if (k0 + 64 <= s.k_n) {
#pragma unroll
      for (int c = 0; c < kChunks; ++c) lds_dma_16(base + off[c], lds + (c * NT + wave) * 16);
    } else {
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const int q = c * NT + threadIdx.x;
        const long k = k0 + (KC ? ((q & 7) ^ ((q >> 3) & 7)) * 8 : q / (E / 8));
        const char* at = base + off[c];
        lds_dma_16(k < s.k_n ? at : reinterpret_cast<const char*>(kZeros), lds + (c * NT + wave) * 16);
      }
    }
  }
};

// The fragment of 16 rows from `row` (a multiple of 16) and 32 values of k from 32 * ks.
template <typename T, int E, bool KC>
__device__ __forceinline__ typename Frag<T>::type fragment(unsigned lds, int row, int ks) {
  const int l = threadIdx.x & 63, g = l >> 4, e = l & 15;
  if (KC) {
    const unsigned at = lds + (row + e) * 128 + (((4 * ks + g) ^ (e & 7)) << 4);
    return *lds_ptr<typename Frag<T>::type>(at, 0);
  }
  typedef __attribute__((address_space(3))) short4_t lds_short4;
  const int k = 32 * ks + 8 * g + (e >> 2);
  const int f = Stage<E, 64, false, 1>::gran(8 * g + (e >> 2));
  const unsigned at = lds + k * (E * 2) + (((row >> 4) ^ f) << 5) + ((e & 3) << 3);
  const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(uintptr_t)at);
  const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(uintptr_t)(at + 4 * E * 2));
  struct {
    short4_t a, b;
  } both{lo, hi};
  return __builtin_bit_cast(typename Frag<T>::type, both);
}

// A workgroup of WI x WJ waves; a wave owns NI x NJ fragments of 16 x 16.
template <int WI_, int WJ_, int NI_, int NJ_>
struct Tile {
  static constexpr int WI = WI_, WJ = WJ_, NI = NI_, NJ = NJ_;
  static constexpr int NT = WI * WJ * 64, TI = WI * NI * 16, TJ = WJ * NJ * 16;
};

// acc[j][i] += the products of steps [first, last) of the segments' steps (steps_per = ceil(k / 64) each).
// J fragments are the MFMA's first operand: a lane holds 4 neighbouring j of one i.
template <typename T, typename C, bool IK, bool JK, int PARTS>
__device__ __forceinline__ void accumulate(f32x4_t (&acc)[C::NJ][C::NI], const Side& si, const Side& sj, long i0, long j0,
                                           int steps_per, int first, int last, unsigned lds) {
  typedef Stage<C::TI, C::NT, IK, 1> SI;
  typedef Stage<C::TJ, C::NT, JK, PARTS> SJ;
  constexpr unsigned kStage = SI::kBytes + SJ::kBytes;
  if (first >= last) return;
  SI a;
  SJ b;
  a.init(si, i0);
  b.init(sj, j0);
  const int wave = threadIdx.x >> 6, wi = wave / C::WJ, wj = wave % C::WJ;
  int seg = first / steps_per, step = first - seg * steps_per;
  auto fetch = [&](unsigned at) {
    a.fetch(si.p[seg], si, long(step) * 64, at);
    b.fetch(sj.p[seg], sj, long(step) * 64, at + SI::kBytes);
    if (++step == steps_per) step = 0, ++seg;
  };
  fetch(lds);
  wait_vmcnt(0);
  __syncthreads();
  for (int t = first; t < last; ++t) {
    const unsigned now = lds + ((t - first) & 1) * kStage;
    if (t + 1 < last) fetch(lds + ((t - first + 1) & 1) * kStage);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      typename Frag<T>::type fj[C::NJ];
#pragma unroll
      for (int j = 0; j < C::NJ; ++j) {
        constexpr int per = C::NJ / PARTS;
        const int row = (j / per) * (C::TJ / PARTS) + wj * per * 16 + (j % per) * 16;
        fj[j] = fragment<T, C::TJ, JK>(now + SI::kBytes, row, ks);
      }
#pragma unroll
      for (int i = 0; i < C::NI; ++i) {
        const typename Frag<T>::type fi = fragment<T, C::TI, IK>(now, (wi * C::NI + i) * 16, ks);
#pragma unroll
        for (int j = 0; j < C::NJ; ++j) acc[j][i] = Frag<T>::mma(fj[j], fi, acc[j][i]);
      }
    }
    wait_vmcnt(0);      // the next step's pieces of this wave; the barrier makes it every wave's
    __syncthreads();
  }
}

// Four neighbouring values of a row; `wide`: the row's address allows one store.
template <typename O>
struct alignas(sizeof(O) * 4) Out4 {
  O v[4];
};
template <typename O>
__device__ __forceinline__ void store_row4(O* row, long j, long n, bool wide, f32x4_t v) {
  if (wide && j + 4 <= n) {
    Out4<O> o;
#pragma unroll
    for (int r = 0; r < 4; ++r) o.v[r] = O(v[r]);
    *reinterpret_cast<Out4<O>*>(row + j) = o;
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (j + r < n) row[j + r] = O(v[r]);
  }
}

// Workgroup b of n as a tile number: workgroups go round the 8 XCDs, so every XCD gets a contiguous run of
// tiles and its L2 holds the operand rows they share; runs go down `group` rows of tiles before the next
// column.
__device__ __forceinline__ void tile_of(unsigned b, unsigned n, unsigned tiles_i, unsigned tiles_j, unsigned& ti, unsigned& tj) {
  const unsigned q = n / 8, r = n % 8, x = b % 8, y = b / 8;
  const unsigned at = (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + y;
  constexpr unsigned kGroup = 8;
  const unsigned full = kGroup * tiles_j, gi = at / full, left = at - gi * full;
  const unsigned rows = tiles_i - gi * kGroup < kGroup ? tiles_i - gi * kGroup : kGroup;
  tj = left / rows;
  ti = gi * kGroup + left - tj * rows;
}

}  // namespace nerf
