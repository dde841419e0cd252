// Root-mean-square norm with the residual's addition, its 8-bit output, and its adjoint.
//   h = x + r,  y = h * rstd * w,  rstd = 1 / sqrt(mean(h^2) + eps)
//   adjoint: with the row sums  S = sum h^2  and  P = sum dy w h  taken in one pass,
//     dx = rstd * dy w - h * rstd^3 * P / cols (+ dh),   dw = sum over rows of dy h rstd
// Bound by HBM: every element is read once, kept in registers between the sum and the store, and written once.
//
// A group of `tpr` threads (8, 16 .. 128, or any multiple of 32 up to 1024) holds one row as 16-byte vectors, PACKS per thread.  Rows whose start is not
// on a 16-byte boundary (odd pitches) are covered by the aligned vectors that contain them: vectors inside the row move as a
// whole, the two that hang over its ends element by element.  Sums are f32.
#include <algorithm>

#include "internal.h"
#include "rounding.cuh"

namespace zyxb {

namespace {

constexpr uint64_t RMS_MAX_COLS = 16384;

struct RmsParams {
  const void *x, *residual, *weight, *dy, *dh;
  void *h, *y, *dweight;
  float *scales, *partial;
  uint64_t rows, ld, end;      // end: elements up to the last row's last
  uint32_t cols, group, n_groups;
  float eps, inv_cols;
  int log_tpr, tpr, groups;    // threads per row; rows per CTA.  One row: any multiple of 32 threads, log_tpr is 10
  int rn, residual_on, weight_on, dh_on;
};

// Sum over a row's threads of up to two values.  `parity` alternates between calls, so one barrier per call is enough.
template <int N>
__device__ __forceinline__ void row_sum(float (&v)[N], int log_tpr, int wpr, float (*buf)[32][N], int parity) {
  if (log_tpr >= 5) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    }
  } else {
    for (int o = (1 << log_tpr) >> 1; o > 0; o >>= 1) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    }
  }
  if (log_tpr > 5) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) buf[parity][warp][i] = v[i];
    }
    __syncthreads();
    const int first = warp & ~((1 << (log_tpr - 5)) - 1);
    float s[N];
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = 0.0f;
#pragma unroll 4
    for (int w = 0; w < wpr; ++w) {
#pragma unroll
      for (int i = 0; i < N; ++i) s[i] += buf[parity][first + w][i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = s[i];
  }
}

// One row seen through aligned vectors: element 0 of vector 0 is `off` elements before the row.
template <typename T, bool ALIGNED>
struct RowView {
  using S = typename Elem<T>::store_t;
  static constexpr int VEC = 16 / (int)sizeof(S);
  uint64_t start;      // element index of vector 0 (a multiple of VEC)
  int off, cols;
  __device__ __forceinline__ RowView(uint64_t row, uint64_t ld, uint32_t cols_) : cols((int)cols_) {
    const uint64_t at = row * ld;
    off = ALIGNED ? 0 : (int)(at % VEC);
    start = at - off;
  }
  __device__ __forceinline__ bool has(int pack) const { return pack * VEC < off + cols; }
  __device__ __forceinline__ int col(int pack) const { return pack * VEC - off; }                 // may be negative
  __device__ __forceinline__ bool whole(int pack) const { return ALIGNED || (col(pack) >= 0 && col(pack) + VEC <= cols); }
  __device__ __forceinline__ bool inside(int c) const { return ALIGNED || ((unsigned)c < (unsigned)cols); }
  // Whole vectors wherever the buffer (of `end` elements) has them: what lies outside the row is dropped by mask(), which the caller
  // applies when it needs the values and not when it starts the load.
  __device__ __forceinline__ void load(RawVec<T, VEC>& r, const void* base, int pack, uint64_t end) const {
    const S* p = reinterpret_cast<const S*>(base) + start + (uint64_t)pack * VEC;
    if (ALIGNED || start + (uint64_t)pack * VEC + VEC <= end) { r.load_stream(p); return; }
    float v[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[k] = inside(col(pack) + k) ? Elem<T>::load(p[k]) : 0.0f;
    round_encode<T, VEC>(r, v, true);          // exact: the values are of the storage type
  }
  __device__ __forceinline__ void mask(RawVec<T, VEC>& r, int pack) const {
    if (ALIGNED || whole(pack)) return;
#pragma unroll
    for (int k = 0; k < VEC; ++k)
      if (!inside(col(pack) + k)) {
        if constexpr (sizeof(S) == 2) r.w[k / 2] &= k & 1 ? 0x0000ffffu : 0xffff0000u;
        else r.w[k] = 0u;
      }
  }
  __device__ __forceinline__ void store(const typename Nums<VEC>::V (&n)[Nums<VEC>::N], void* base, int pack, bool rn) const {
    S* p = reinterpret_cast<S*>(base) + start + (uint64_t)pack * VEC;
    if (whole(pack)) {
      RawVec<T, VEC> r;
      Nums<VEC>::encode(r, n, rn);
      r.store_stream(p);
      return;
    }
    float v[VEC];
    Nums<VEC>::floats(v, n);
#pragma unroll
    for (int k = 0; k < VEC; ++k)
      if (inside(col(pack) + k)) p[k] = round_store<T>(v[k], rn);
  }
  // the weight's entries under a vector (the weight itself starts on a boundary, the row need not)
  __device__ __forceinline__ void weight(typename Nums<VEC>::V (&n)[Nums<VEC>::N], const void* w, int pack) const {
    const S* p = reinterpret_cast<const S*>(w);
    RawVec<T, VEC> r;
    if constexpr (ALIGNED) r.load(p + pack * VEC);
    else load_shifted<T, VEC>(r, p, col(pack), (uint64_t)cols);
    Nums<VEC>::decode(n, r);
  }
};

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

constexpr float E4M3_MAX = 448.0f, AMAX_FLOOR = 1e-30f;

// 448 / largest: what y is multiplied by.  The reciprocal is the approximate one (1 ulp): a value next to the border between two 8-bit
// floats may go to either, as it may by the f32 rounding of y itself.  At 8192 x 4096 with groups of 128, 975 of 33.6 million values are on
// the other side than in 64 bits, and 949 with a division rounded once, which costs 4 us of 41.
__device__ __forceinline__ float e4m3_factor(float amax) {
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(amax));
  return r * E4M3_MAX;
}

// a vector of y as 8-bit floats; scale_of(column): the reciprocal of its scale
template <typename T, bool ALIGNED, class F>
__device__ __forceinline__ void put_e4m3(const RowView<T, ALIGNED>& view, const float (&y)[RowView<T, ALIGNED>::VEC], const RmsParams& p, uint64_t row, int pack, F scale_of) {
  constexpr int VEC = RowView<T, ALIGNED>::VEC;
  uint8_t* out = reinterpret_cast<uint8_t*>(p.y) + row * p.cols;
  const int c0 = view.col(pack);
  float q[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) q[k] = y[k] * scale_of(c0 + k);
  uint32_t w[VEC / 4];
#pragma unroll
  for (int k = 0; k < VEC / 4; ++k) w[k] = e4m3x2(q[4 * k], q[4 * k + 1]) | (e4m3x2(q[4 * k + 2], q[4 * k + 3]) << 16);
  if (ALIGNED || (view.whole(pack) && (row * p.cols + c0) % VEC == 0)) {       // a dense x and the dense y have the same vector boundaries
    if constexpr (VEC == 8) __stcs(reinterpret_cast<uint2*>(out + c0), make_uint2(w[0], w[1]));
    else __stcs(reinterpret_cast<uint32_t*>(out + c0), w[0]);
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k)
      if (view.inside(c0 + k)) out[c0 + k] = (uint8_t)(w[k / 4] >> (8 * (k % 4)));
  }
}

// How the largest |y| of a column group is found: LANES where a group is a power of two of whole vectors, which lie in neighbouring
// lanes of one warp (shuffles; 1 scale per 128 columns of bf16 is 16 lanes); SHARED for every other group (integer maxima in shared
// memory, one per warp where a row is one group).
enum { QUANT_NONE = 0, QUANT_LANES = 1, QUANT_SHARED = 2 };

// largest of m and |v|; a NaN stays, and becomes its group's scale
__device__ __forceinline__ float max_abs(float m, float a, float b) {
  float r;
  asm("{\n\t.reg .f32 x, y;\n\tabs.f32 x, %1;\n\tabs.f32 y, %2;\n\tmax.NaN.f32 %0, x, y, %3;\n\t}" : "=f"(r) : "f"(a), "f"(b), "f"(m));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
// the bits of |y| order like the values, and a NaN's above all of them
__device__ __forceinline__ uint32_t amax_bits_of(float v) { return __float_as_uint(v) & 0x7fffffffu; }

template <typename T, int PACKS, bool ALIGNED, int QUANT, int THREADS>
__global__ void __launch_bounds__(THREADS) rmsnorm_kernel(const RmsParams p) {
  using View = RowView<T, ALIGNED>;
  constexpr int VEC = View::VEC;
  using Num = Nums<VEC>;
  __shared__ float red[1][32][1];
  extern __shared__ uint32_t amax_bits[];            // QUANT_SHARED: largest |y| of each column group, per row of the CTA, as its bits
  const int tpr = p.tpr, in_cta = threadIdx.x >> p.log_tpr, t = threadIdx.x & ((1 << p.log_tpr) - 1);
  const uint64_t row = (uint64_t)blockIdx.x * p.groups + in_cta;
  const bool live = row < p.rows;
  const View view(live ? row : 0, p.ld, p.cols);
  pdl_trigger();
  pdl_wait();
  typename Num::V v[PACKS][Num::N], sq = Num::splat(0.0f);
  {
    RawVec<T, VEC> rx[PACKS], rr[PACKS];
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
      const int pack = t + i * tpr;
      rx[i].zero(); rr[i].zero();
      if (live && view.has(pack)) {
        view.load(rx[i], p.x, pack, p.end);
        if (p.residual_on) view.load(rr[i], p.residual, pack, p.end);
      }
    }
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
      const int pack = t + i * tpr;
      view.mask(rx[i], pack);
      Num::decode(v[i], rx[i]);
      if (p.residual_on) {
        view.mask(rr[i], pack);
        typename Num::V r[Num::N];
        Num::decode(r, rr[i]);
#pragma unroll
        for (int k = 0; k < Num::N; ++k) v[i][k] = Num::add(v[i][k], r[k]);
        if (live && view.has(pack)) view.store(v[i], p.h, pack, p.rn != 0);
      }
#pragma unroll
      for (int k = 0; k < Num::N; ++k) sq = Num::fma(v[i][k], v[i][k], sq);
    }
  }
  if constexpr (QUANT == QUANT_SHARED) {
    for (uint32_t g = threadIdx.x; g < (uint32_t)p.groups * p.n_groups; g += blockDim.x) amax_bits[g] = __float_as_uint(AMAX_FLOOR);
    if (p.log_tpr <= 5) __syncthreads();             // wider rows pass a barrier in row_sum
  }
  float sum[1] = {Num::sum(sq)};
  row_sum(sum, p.log_tpr, p.tpr >> 5, red, 0);
  const float rstd = rsqrtf(sum[0] * p.inv_cols + p.eps);
  float h[PACKS][VEC];
#pragma unroll
  for (int i = 0; i < PACKS; ++i) {
    const int pack = t + i * tpr;
    const bool in = live && view.has(pack);
    if (in && p.weight_on) {
      typename Num::V w[Num::N];
      view.weight(w, p.weight, pack);
#pragma unroll
      for (int k = 0; k < Num::N; ++k) v[i][k] = Num::mul(Num::mul(v[i][k], Num::splat(rstd)), w[k]);
    } else {
#pragma unroll
      for (int k = 0; k < Num::N; ++k) v[i][k] = Num::mul(v[i][k], Num::splat(rstd));
    }
    if constexpr (QUANT == QUANT_NONE) { if (in) view.store(v[i], p.y, pack, p.rn != 0); }
    else Num::floats(h[i], v[i]);
  }
  if constexpr (QUANT == QUANT_LANES) {
    const int width = (int)p.group / VEC;              // lanes per column group
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
      const int pack = t + i * tpr;
      const bool in = live && view.has(pack);
      float m = AMAX_FLOOR;
      if (in) {
#pragma unroll
        for (int k = 0; k < VEC; k += 2) m = max_abs(m, h[i][k], h[i][k + 1]);
      }
      for (int o = width >> 1; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
      if (!in) continue;
      const float scale = m * (1.0f / E4M3_MAX), inv = e4m3_factor(m);
      put_e4m3<T, ALIGNED>(view, h[i], p, row, pack, [&](int) { return inv; });
      if (pack % width == 0) p.scales[row * p.n_groups + pack / width] = scale;
    }
  }
  if constexpr (QUANT == QUANT_SHARED) {
    uint32_t* mine = amax_bits + in_cta * p.n_groups;
    if (p.n_groups == 1) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < PACKS; ++i)
        if (live && view.has(t + i * tpr)) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) m = max(m, view.inside(view.col(t + i * tpr) + k) ? amax_bits_of(h[i][k]) : 0u);
        }
      for (int o = min(32, tpr) >> 1; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      if ((t & 31) == 0) atomicMax(&mine[0], m);
    } else {
#pragma unroll
      for (int i = 0; i < PACKS; ++i) {
        const int pack = t + i * tpr;
        if (!live || !view.has(pack)) continue;
        const int c0 = max(0, view.col(pack)), c1 = min((int)p.cols, view.col(pack) + VEC) - 1;
        const uint32_t g0 = (uint32_t)c0 / p.group, g1 = (uint32_t)c1 / p.group;
        uint32_t m0 = 0, m1 = 0;                       // a vector meets at most two groups
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const int c = view.col(pack) + k;
          if (!view.inside(c)) continue;
          const uint32_t b = amax_bits_of(h[i][k]);
          if ((uint32_t)c < (g0 + 1) * p.group) m0 = max(m0, b); else m1 = max(m1, b);
        }
        atomicMax(&mine[g0], m0);
        if (g1 != g0) atomicMax(&mine[g1], m1);
      }
    }
    __syncthreads();
    if (live)
      for (uint32_t g = t; g < p.n_groups; g += tpr) p.scales[row * p.n_groups + g] = __uint_as_float(mine[g]) * (1.0f / E4M3_MAX);
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
      const int pack = t + i * tpr;
      if (!live || !view.has(pack)) continue;
      uint32_t g0 = 0, border = p.cols;
      if (p.n_groups > 1) { g0 = (uint32_t)max(0, view.col(pack)) / p.group; border = (g0 + 1) * p.group; }
      const float s0 = e4m3_factor(__uint_as_float(mine[g0])), s1 = border < min(p.cols, (uint32_t)(view.col(pack) + VEC)) ? e4m3_factor(__uint_as_float(mine[g0 + 1])) : s0;
      put_e4m3<T, ALIGNED>(view, h[i], p, row, pack, [&](int c) { return c < (int)border ? s0 : s1; });
    }
  }
}

// Rows are dealt to the groups of a persistent grid, so that a thread keeps its columns' weights and their gradient in registers
// from the first of its rows to the last.  Where rows do not start on vector boundaries, the number of groups is a multiple of the
// vector's length: all of a group's rows then start at the same place in a vector, and a column stays with its thread.
template <typename T, int PACKS, bool ALIGNED, int THREADS>
__global__ void __launch_bounds__(THREADS) rmsnorm_bwd_kernel(const RmsParams p) {
  using View = RowView<T, ALIGNED>;
  constexpr int VEC = View::VEC;
  using Num = Nums<VEC>;
  using V = typename Num::V;
  constexpr int N = Num::N;
  __shared__ float red[2][32][2];
  extern __shared__ float dw_shared[];               // [group of the CTA][cols]
  const int tpr = p.tpr, in_cta = threadIdx.x >> p.log_tpr, t = threadIdx.x & ((1 << p.log_tpr) - 1), groups = p.groups;
  const uint64_t step = (uint64_t)gridDim.x * groups;
  const View first((uint64_t)blockIdx.x * groups + in_cta, p.ld, p.cols);        // stands for all rows where only the place in a vector counts
  // 1024 threads have 64 registers each: no room for the weights and a second row
  constexpr bool LEAN = THREADS > 512;
  V w[LEAN ? 1 : PACKS][N], dw[PACKS][N];
  auto weight = [&](V (&to)[N], int pack) {
#pragma unroll
    for (int k = 0; k < N; ++k) to[k] = Num::splat(1.0f);
    if (p.weight_on && first.has(pack)) first.weight(to, p.weight, pack);
  };
  pdl_trigger();
  pdl_wait();
#pragma unroll
  for (int i = 0; i < PACKS; ++i) {
    if constexpr (!LEAN) weight(w[i], t + i * tpr);
#pragma unroll
    for (int k = 0; k < N; ++k) dw[i][k] = Num::splat(0.0f);
  }
  struct Row { RawVec<T, VEC> h[PACKS], g[PACKS], d[PACKS]; };
  auto fetch = [&](Row& r, uint64_t row) {
    const View view(row, p.ld, p.cols);
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
      const int pack = t + i * tpr;
      r.h[i].zero(); r.g[i].zero(); r.d[i].zero();
      if (row < p.rows && view.has(pack)) {
        view.load(r.h[i], p.h, pack, p.end);
        view.load(r.g[i], p.dy, pack, p.end);
        if (p.dh_on) view.load(r.d[i], p.dh, pack, p.end);
      }
    }
  };
  int parity = 0;
  Row now;
  fetch(now, (uint64_t)blockIdx.x * groups + in_cta);
  for (uint64_t row0 = (uint64_t)blockIdx.x * groups; row0 < p.rows; row0 += step, parity ^= 1) {
    const uint64_t row = row0 + in_cta;
    V hh = Num::splat(0.0f), gh = Num::splat(0.0f);
    Row cur;
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
      first.mask(now.h[i], t + i * tpr); first.mask(now.g[i], t + i * tpr);
      cur.h[i] = now.h[i]; cur.g[i] = now.g[i]; cur.d[i] = now.d[i];
    }
    if constexpr (!LEAN) fetch(now, row + step);     // in flight during this row's sums
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
      V h[N], g[N];
      Num::decode(h, cur.h[i]);
      Num::decode(g, cur.g[i]);
      if constexpr (LEAN) weight(w[0], t + i * tpr);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        hh = Num::fma(h[k], h[k], hh);
        gh = Num::fma(Num::mul(g[k], w[LEAN ? 0 : i][k]), h[k], gh);
      }
    }
    float s[2] = {Num::sum(hh), Num::sum(gh)};
    row_sum(s, p.log_tpr, p.tpr >> 5, red, parity);
    if (row < p.rows) {
      const View view(row, p.ld, p.cols);
      const float rstd = rsqrtf(s[0] * p.inv_cols + p.eps);
      // dx = rstd * (dy w) - h * (rstd^3 * mean(dy w h)) + dh;  dw += dy * h * rstd
      const V up = Num::splat(rstd), down = Num::splat(-(rstd * rstd * rstd) * (s[1] * p.inv_cols));
#pragma unroll
      for (int i = 0; i < PACKS; ++i) {
        const int pack = t + i * tpr;
        if (!view.has(pack)) continue;
        V h[N], g[N], d[N], o[N];
        Num::decode(h, cur.h[i]);
        Num::decode(g, cur.g[i]);
        Num::decode(d, cur.d[i]);
        if constexpr (LEAN) weight(w[0], pack);
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const V gu = Num::mul(g[k], up);
          dw[i][k] = Num::fma(gu, h[k], dw[i][k]);
          o[k] = Num::add(Num::fma(gu, w[LEAN ? 0 : i][k], Num::mul(h[k], down)), d[k]);
        }
        view.store(o, p.y, pack, p.rn != 0);
      }
    }
    if constexpr (LEAN) fetch(now, row + step);
  }
  if (!p.weight_on) return;
  // the CTA's groups are added in order, then one row of partials per CTA
#pragma unroll
  for (int i = 0; i < PACKS; ++i) {
    const int pack = t + i * tpr;
    if (!first.has(pack)) continue;
    float f[VEC];
    Num::floats(f, dw[i]);
#pragma unroll
    for (int k = 0; k < VEC; ++k)
      if (first.inside(first.col(pack) + k)) dw_shared[(size_t)in_cta * p.cols + first.col(pack) + k] = f[k];
  }
  __syncthreads();
  for (uint32_t c = threadIdx.x; c < p.cols; c += blockDim.x) {
    float sum = 0.0f;
    for (int g = 0; g < groups; ++g) sum += dw_shared[(size_t)g * p.cols + c];
    p.partial[(uint64_t)blockIdx.x * p.cols + c] = sum;
  }
}

// dweight[c] = sum over the CTAs' partials, in order: 32 columns per CTA, 32 warps share the list
template <typename T>
__global__ void __launch_bounds__(1024) rmsnorm_dweight_kernel(const float* partial, uint32_t n, uint32_t cols, typename Elem<T>::store_t* dweight, int rn) {
  __shared__ float part[32][33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t c = blockIdx.x * 32 + lane;
  pdl_wait();
  float sum = 0.0f;
  if (c < cols) {
    constexpr int U = 12;                          // loads in flight: 384 CTAs' partials in one go
    for (uint32_t i0 = warp; i0 < n; i0 += 32 * U) {
      float v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = i0 + 32 * u < n ? partial[(uint64_t)(i0 + 32 * u) * cols + c] : 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u) sum += v[u];
    }
  }
  part[warp][lane] = sum;
  __syncthreads();
  const float v = warp_reduce(part[lane][warp], OpSum());        // warp w: column w
  const uint32_t cw = blockIdx.x * 32 + warp;
  if (lane == 0 && cw < cols) dweight[cw] = round_store<T>(v, rn != 0);
}

int log2_up(uint64_t v) {
  int l = 0;
  while ((1ull << l) < v) ++l;
  return l;
}

struct RmsShape { int log_tpr, tpr, packs, threads, groups; };

// Threads per row and vectors per thread.  A thread's fixed work (addresses, the row's sum) is worth about a vector's, so rows are
// held by few threads with several vectors each (four loads in flight per thread: 8192 x 4096 bf16 with residual and 8-bit output takes
// 66 us with one vector per thread, 41 with two, 43 with four) - unless there are too few rows to fill the SMs that way, where a row
// is spread as wide as it goes.
RmsShape rms_shape(uint64_t rows, uint64_t vectors, int packs_wanted, int sm_count) {
  RmsShape s{};
  const int packs = rows * vectors < (uint64_t)sm_count * 2048 ? 1 : packs_wanted;
  const uint64_t want = std::min<uint64_t>(1024, (vectors + packs - 1) / packs);
  if (want <= 128) {
    s.log_tpr = std::max(3, log2_up(want));
    s.tpr = 1 << s.log_tpr;
    s.threads = 256;
    s.groups = 256 >> s.log_tpr;
  } else {
    s.log_tpr = 10;
    s.tpr = (int)((want + 31) / 32 * 32);
    s.threads = s.tpr;
    s.groups = 1;
  }
  s.packs = (int)((vectors + s.tpr - 1) / s.tpr);
  return s;
}

void rms_apply(RmsParams& p, const RmsShape& s) { p.log_tpr = s.log_tpr; p.tpr = s.tpr; p.groups = s.groups; }

// A kernel of PACKS vectors per thread and THREADS threads covers a row of this shape: what it would leave out, it would leave out
// silently, so both directions ask before they launch.
template <int PACKS, int THREADS> bool rms_covers(const RmsShape& s) { return s.packs <= PACKS && s.threads <= THREADS; }

template <typename T, int PACKS, bool ALIGNED, int THREADS>
cudaError_t run_rms(const RmsParams& p, const RmsShape& s, bool quant, const LaunchCtx& lc) {
  if (!rms_covers<PACKS, THREADS>(s)) return cudaErrorInvalidConfiguration;
  const uint64_t per_cta = (uint64_t)s.groups;
  const unsigned grid = (unsigned)((p.rows + per_cta - 1) / per_cta);
  constexpr uint32_t VEC = 16 / sizeof(typename Elem<T>::store_t);
  const uint32_t width = p.group / VEC;
  if (!quant) {
    return launch_pdl(rmsnorm_kernel<T, PACKS, ALIGNED, QUANT_NONE, THREADS>, dim3(grid), s.threads, 0, lc.stream, p);
  }
  if constexpr (ALIGNED) {
    if (p.group % VEC == 0 && (width & (width - 1)) == 0 && width <= 32 && (int)width <= s.tpr) {
      return launch_pdl(rmsnorm_kernel<T, PACKS, ALIGNED, QUANT_LANES, THREADS>, dim3(grid), s.threads, 0, lc.stream, p);
    }
  }
  return launch_pdl(rmsnorm_kernel<T, PACKS, ALIGNED, QUANT_SHARED, THREADS>, dim3(grid), s.threads, per_cta * p.n_groups * 4, lc.stream, p);
}

template <typename T, bool ALIGNED>
cudaError_t run_rms_packs(const RmsParams& p, const RmsShape& s, bool quant, const LaunchCtx& lc) {
  if (s.threads <= 256) {
    if (s.packs == 1) return run_rms<T, 1, ALIGNED, 256>(p, s, quant, lc);
    if (s.packs == 2) return run_rms<T, 2, ALIGNED, 256>(p, s, quant, lc);
    return run_rms<T, 4, ALIGNED, 256>(p, s, quant, lc);
  }
  if (s.packs == 1) return run_rms<T, 1, ALIGNED, 1024>(p, s, quant, lc);
  if (s.packs == 2) return run_rms<T, 2, ALIGNED, 1024>(p, s, quant, lc);
  if constexpr (sizeof(T) == 4 && !ALIGNED) { if (s.packs > 4) return run_rms<T, 8, ALIGNED, 1024>(p, s, quant, lc); }     // 4097 vectors, spread wide
  return run_rms<T, 4, ALIGNED, 1024>(p, s, quant, lc);
}

template <typename T>
cudaError_t rms_forward(const RmsParams& p, bool quant, const LaunchCtx& lc) {
  constexpr uint32_t VEC = 16 / sizeof(typename Elem<T>::store_t);
  RmsParams q = p;
  const bool aligned = p.cols % VEC == 0 && p.ld % VEC == 0;
  const RmsShape s = rms_shape(p.rows, aligned ? p.cols / VEC : (p.cols + 2 * VEC - 2) / VEC, p.residual_on ? 2 : 4, lc.sm_count);
  rms_apply(q, s);
  return aligned ? run_rms_packs<T, true>(q, s, quant, lc) : run_rms_packs<T, false>(q, s, quant, lc);
}

template <typename T, int PACKS, bool ALIGNED, int THREADS>
cudaError_t run_rms_bwd(const RmsParams& p, const RmsShape& s, unsigned* grid_out, const LaunchCtx& lc) {
  if (!rms_covers<PACKS, THREADS>(s)) return cudaErrorInvalidConfiguration;
  constexpr int VEC = 16 / (int)sizeof(typename Elem<T>::store_t);
  const int groups = s.groups;
  const size_t smem = p.weight_on ? (size_t)groups * p.cols * 4 : 0;
  auto kern = rmsnorm_bwd_kernel<T, PACKS, ALIGNED, THREADS>;
  static uint64_t configured = 0;
  cudaError_t e = ensure_dynamic_smem(kern, 80 << 10, &configured);
  if (e != cudaSuccess) return e;
  int per_sm = 1;
  if ((e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, s.threads, smem)) != cudaSuccess) return e;
  const uint64_t work = (p.rows + groups - 1) / groups;
  uint64_t grid = std::min<uint64_t>(work, (uint64_t)lc.sm_count * std::max(1, per_sm));
  if (!ALIGNED && grid < work) grid = std::max<uint64_t>(VEC, grid / VEC * VEC);      // a group's rows: the same place in a vector
  *grid_out = (unsigned)grid;
  return launch_pdl(kern, dim3(*grid_out), s.threads, smem, lc.stream, p);
}

// The adjoint's groups: a column's weight, its gradient, this row's h, dy, dh and the next row's all stay in registers, so a thread
// takes two vectors and the group grows, to 1024 threads - which have 64 registers each, and load the weights anew for every row and
// the next row after this one.
template <typename T, bool ALIGNED>
cudaError_t run_rms_bwd_packs(const RmsParams& p, const RmsShape& s, unsigned* grid, const LaunchCtx& lc) {
  if (s.threads <= 256) return s.packs == 1 ? run_rms_bwd<T, 1, ALIGNED, 256>(p, s, grid, lc) : run_rms_bwd<T, 2, ALIGNED, 256>(p, s, grid, lc);
  if constexpr (sizeof(T) == 4) { if (s.threads <= 512 && s.packs == 3) return run_rms_bwd<T, 3, ALIGNED, 512>(p, s, grid, lc); }
  if (s.threads <= 512) return run_rms_bwd<T, 2, ALIGNED, 512>(p, s, grid, lc);
  if (s.packs <= 2) return run_rms_bwd<T, 2, ALIGNED, 1024>(p, s, grid, lc);
  if constexpr (sizeof(T) == 4 && !ALIGNED) { if (s.packs > 4) return run_rms_bwd<T, 8, ALIGNED, 1024>(p, s, grid, lc); }      // 4097 vectors
  if constexpr (sizeof(T) == 4 || !ALIGNED) return run_rms_bwd<T, 4, ALIGNED, 1024>(p, s, grid, lc);                           // 16-bit: 2049 vectors
  else return run_rms_bwd<T, 2, ALIGNED, 1024>(p, s, grid, lc);
}

template <typename T>
cudaError_t rms_backward(const RmsParams& p, const LaunchCtx& lc) {
  using S = typename Elem<T>::store_t;
  constexpr uint32_t VEC = 16 / sizeof(S);
  RmsParams q = p;
  const bool aligned = p.cols % VEC == 0 && p.ld % VEC == 0;
  const uint64_t vectors = aligned ? p.cols / VEC : (p.cols + 2 * VEC - 2) / VEC;
  // Three vectors of f32 still fit the registers of 512 threads, which hold 6144 columns that way; rows of at most 3 * 256 vectors,
  // which few rows spread over more than 512 threads too, would come back with 256 threads and stay as they are: no form of 256 threads has three
  RmsShape s = rms_shape(p.rows, vectors, 2, lc.sm_count);
  if (sizeof(T) == 4 && s.threads > 512 && vectors > 3 * 256 && vectors <= 3 * 512) s = rms_shape(UINT32_MAX, vectors, 3, lc.sm_count);
  rms_apply(q, s);
  unsigned grid = 0;
  cudaError_t e = aligned ? run_rms_bwd_packs<T, true>(q, s, &grid, lc) : run_rms_bwd_packs<T, false>(q, s, &grid, lc);
  if (e == cudaSuccess && p.weight_on)
    e = launch_pdl(rmsnorm_dweight_kernel<T>, dim3((p.cols + 31) / 32), 1024, 0, lc.stream, (const float*)q.partial, grid, p.cols, (S*)q.dweight, q.rn);
  return e;
}

bool rows_fit(const zyxb_rmsnorm_desc& d, uint64_t ld, uint64_t bytes) {
  return (unsigned __int128)dtype_size(d.dtype) * ((unsigned __int128)(d.rows - 1) * ld + d.cols) <= bytes;
}

}  // namespace

int validate_rmsnorm(const zyxb_rmsnorm_desc& d, bool backward, std::string& err) {
  auto bad = [&](const char* m) { err = m; return (int)ZYXB_ERR_KERNEL_COMPILATION; };
  if (d.dtype != ZYXB_F32 && d.dtype != ZYXB_BF16 && d.dtype != ZYXB_F16) return bad("rmsnorm: dtype must be f32, bf16 or f16");
  if (d.rows == 0 || d.cols == 0) return bad("rmsnorm: rows and cols must be positive");
  if (d.cols > RMS_MAX_COLS) return bad("rmsnorm: cols must be at most 16384");
  if (d.rows > 0x7fffffffull) return bad("rmsnorm: rows must be below 2^31");
  if ((d.ld && d.ld < d.cols) || d.ld > (1ull << 40)) return bad("rmsnorm: row pitch smaller than the row, or too large");
  if (!(d.eps >= 0.0f)) return bad("rmsnorm: eps must not be negative");
  if (d.quant != 0 && d.quant != 1) return bad("rmsnorm: quant must be 0 or 1");
  if (backward && (d.quant || d.has_residual)) return bad("rmsnorm backward: takes h, the stored sum; quant and has_residual are options of the forward");
  if (!backward && d.has_dh) return bad("rmsnorm: has_dh is an option of the backward");
  if (d.group && (!d.quant || d.group < 16)) return bad("rmsnorm: group needs quant and must be at least 16");
  return ZYXB_OK;
}

int launch_rmsnorm(const zyxb_rmsnorm_desc& d, void* const* args, const uint64_t* arg_bytes, int n_args, const LaunchCtx& lc, std::string& err) {
  const int want = 1 + (d.has_residual ? 2 : 0) + (d.has_weight ? 1 : 0) + 1 + (d.quant ? 1 : 0);
  ZYXB_CHECK_ARG(n_args == want, "rmsnorm: expected args x [,residual] [,weight] -> [h,] y [,scales]");
  const uint64_t es = dtype_size(d.dtype);
  RmsParams p{};
  p.rows = d.rows; p.cols = (uint32_t)d.cols; p.ld = d.ld ? d.ld : d.cols; p.end = (d.rows - 1) * p.ld + d.cols; p.eps = d.eps; p.inv_cols = 1.0f / (float)d.cols; p.rn = lc.round_nearest ? 1 : 0;
  p.residual_on = d.has_residual ? 1 : 0; p.weight_on = d.has_weight ? 1 : 0;
  p.group = d.group ? std::min<uint32_t>(d.group, p.cols) : p.cols;
  p.n_groups = (p.cols + p.group - 1) / p.group;
  int i = 0;
  ZYXB_CHECK_ARG(rows_fit(d, p.ld, arg_bytes[i]), "rmsnorm: x too small"); p.x = args[i++];
  if (d.has_residual) { ZYXB_CHECK_ARG(rows_fit(d, p.ld, arg_bytes[i]), "rmsnorm: residual too small"); p.residual = args[i++]; }
  if (d.has_weight) { ZYXB_CHECK_ARG(arg_bytes[i] >= d.cols * es, "rmsnorm: weight too small"); p.weight = args[i++]; }
  if (d.has_residual) { ZYXB_CHECK_ARG(rows_fit(d, p.ld, arg_bytes[i]), "rmsnorm: h too small"); p.h = args[i++]; }
  if (d.quant) {
    ZYXB_CHECK_ARG(arg_bytes[i] >= d.rows * d.cols, "rmsnorm: y too small"); p.y = args[i++];
    ZYXB_CHECK_ARG(arg_bytes[i] >= d.rows * p.n_groups * 4, "rmsnorm: scales too small"); p.scales = (float*)args[i++];
    ZYXB_CHECK_ARG(p.y != p.x && p.y != p.residual && p.y != p.h && (void*)p.scales != p.y && (const void*)p.scales != p.x &&
                   (const void*)p.scales != p.residual && (void*)p.scales != p.h, "rmsnorm: 8-bit y and scales must be buffers of their own");
  } else {
    ZYXB_CHECK_ARG(rows_fit(d, p.ld, arg_bytes[i]), "rmsnorm: y too small"); p.y = args[i++];
    ZYXB_CHECK_ARG(!d.has_residual || p.y != p.h, "rmsnorm: h and y must be different buffers");
  }
  ZYXB_CHECK_ARG(!d.has_weight || (p.weight != p.y && p.weight != p.h && p.weight != (const void*)p.scales), "rmsnorm: an output must not be the weight's buffer");
  cudaError_t e;
  switch (d.dtype) {
    case ZYXB_F32: e = rms_forward<float>(p, d.quant != 0, lc); break;
    case ZYXB_BF16: e = rms_forward<bf16_t>(p, d.quant != 0, lc); break;
    default: e = rms_forward<f16_t>(p, d.quant != 0, lc); break;
  }
  if (e != cudaSuccess) { err = std::string("rmsnorm: ") + cudaGetErrorString(e); return ZYXB_ERR_KERNEL_LAUNCH; }
  return check_launch(lc, err, "rmsnorm");
}

int launch_rmsnorm_bwd(const zyxb_rmsnorm_desc& d, void* const* args, const uint64_t* arg_bytes, int n_args, const LaunchCtx& lc, std::string& err) {
  const int want = 2 + (d.has_weight ? 2 : 0) + (d.has_dh ? 1 : 0) + 1;
  ZYXB_CHECK_ARG(n_args == want, "rmsnorm backward: expected args h, dy [,weight] [,dh] -> dx [,dweight]");
  const uint64_t es = dtype_size(d.dtype);
  RmsParams p{};
  p.rows = d.rows; p.cols = (uint32_t)d.cols; p.ld = d.ld ? d.ld : d.cols; p.end = (d.rows - 1) * p.ld + d.cols; p.eps = d.eps; p.inv_cols = 1.0f / (float)d.cols; p.rn = lc.round_nearest ? 1 : 0;
  p.weight_on = d.has_weight ? 1 : 0; p.dh_on = d.has_dh ? 1 : 0;
  int i = 0;
  ZYXB_CHECK_ARG(rows_fit(d, p.ld, arg_bytes[i]), "rmsnorm backward: h too small"); p.h = args[i++];
  ZYXB_CHECK_ARG(rows_fit(d, p.ld, arg_bytes[i]), "rmsnorm backward: dy too small"); p.dy = args[i++];
  if (d.has_weight) { ZYXB_CHECK_ARG(arg_bytes[i] >= d.cols * es, "rmsnorm backward: weight too small"); p.weight = args[i++]; }
  if (d.has_dh) { ZYXB_CHECK_ARG(rows_fit(d, p.ld, arg_bytes[i]), "rmsnorm backward: dh too small"); p.dh = args[i++]; }
  ZYXB_CHECK_ARG(rows_fit(d, p.ld, arg_bytes[i]), "rmsnorm backward: dx too small"); p.y = args[i++];
  if (d.has_weight) {
    ZYXB_CHECK_ARG(arg_bytes[i] >= d.cols * es, "rmsnorm backward: dweight too small"); p.dweight = args[i++];
    ZYXB_CHECK_ARG(p.y != p.weight && p.dweight != p.y && p.dweight != p.h && p.dweight != p.dy && p.dweight != p.dh,
                   "rmsnorm backward: dx must not be the weight's buffer, dweight no other argument's but the weight's");
  }
  p.partial = (float*)lc.scratch;      // a row of cols per CTA: 2048 threads per SM hold at most 32768 columns, 20 MB in all
  cudaError_t e;
  switch (d.dtype) {
    case ZYXB_F32: e = rms_backward<float>(p, lc); break;
    case ZYXB_BF16: e = rms_backward<bf16_t>(p, lc); break;
    default: e = rms_backward<f16_t>(p, lc); break;
  }
  if (e != cudaSuccess) { err = std::string("rmsnorm backward: ") + cudaGetErrorString(e); return ZYXB_ERR_KERNEL_LAUNCH; }
  return check_launch(lc, err, "rmsnorm backward", d.has_weight ? 2 : 1);
}

}  // namespace zyxb
