// The whole update of a matrix with at most 128 rows (or columns) in one launch: momentum, norm, every Newton-Schulz step and the
// weight's step, by one thread-block cluster per matrix.
//
// X [128, hi] is cut along hi over the cluster's CTAs and stays in their shared memory as f16 parts from the first step to the last.
// Per step and CTA:
//   gram   the partial Gram matrix of its columns (tcgen05, both operands the same tiles), added over the cluster through
//          distributed shared memory: each CTA adds 128 / C of the rows, in CTA order, and hands them to all
//   poly   B = a I + b A + c A^2, by every CTA for itself; B takes A's place
//   apply  X <- B X, its own columns
// A tile of 64 columns holds 128 rows of 128 bytes, 16-byte units swizzled by row: as an operand of the Gram product it is K-major (the
// contraction runs along the 128 bytes), as the right operand of B X it is MN-major (the contraction runs down the rows).  The same
// bytes serve both, so nothing is transposed.
// What a step costs is latency: three dependent groups of products of some 1500 clocks each, and two cluster barriers around the
// exchange (which moves the triangle: distributed shared memory carried some 14 bytes a clock per SM).
#pragma once
#include "muon_gemm.cuh"
#include "rounding.cuh"

namespace zyxb {
namespace muon {

constexpr int SMALL_ROWS = 128, SMALL_THREADS = 256, SMALL_CTAS = 8;
enum { ERR_SMALL = 0x100000u };

template <int PARTS> struct Small {
  static constexpr int COLS = 512 / PARTS;                       // of X per CTA, at most: 128 KB
  static constexpr int TILE_BYTES = SMALL_ROWS * 128;            // 64 columns of one part
  static constexpr int X = 0;                                    // [tile][part]
  static constexpr int A = SMALL_ROWS * COLS * 2 * PARTS;        // [part][tile of 64 columns]
  static constexpr int STAGE = A + PARTS * 2 * TILE_BYTES;       // f32, the lower triangle of [128][128], for the exchange
  static constexpr int TAIL = STAGE + 4 * (32 * 33 / 2) * 16;
  static constexpr int TOTAL = TAIL + 256 + 1024;
};

struct SmallMatrix { void* p; const void* g; void* buf; uint32_t tall; };
constexpr int SMALL_TABLE = 32;
struct SmallArgs {
  SmallMatrix m[SMALL_TABLE];
  uint32_t lo, hi, cols;            // cols of X per CTA, a multiple of 64
  float momentum, grad_scale, eps, a, b, c, decay, step_flat, step_tall;
  int steps, nesterov, rn;
  uint32_t* status;
};

__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ double ld_cluster_f64(uint32_t addr) { double v; asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(addr) : "memory"); return v; }
__device__ __forceinline__ void st_cluster2(uint32_t addr, uint32_t x, uint32_t y) { asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(addr), "r"(x), "r"(y) : "memory"); }
__device__ __forceinline__ void fence_proxy_async_all() { asm volatile("fence.proxy.async;" ::: "memory"); }

// the exchanged lower triangle: units of four columns
constexpr uint32_t STAGE_UNITS = 4 * 32 * 33 / 2;
__device__ __forceinline__ uint32_t unit_at(uint32_t row, uint32_t unit) {
  const uint32_t q = row / 4;
  return (2 * q * (q + 1) + (row % 4) * (q + 1) + unit) * 16;
}
// four 8 x 8 matrices of 16-bit entries; each lane names one row of one of them
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void stmatrix4(uint32_t addr, const uint32_t (&r)[4]) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
__device__ __forceinline__ void stmatrix4_trans(uint32_t addr, const uint32_t (&r)[4]) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}

// byte of element (row, column below 64) inside a tile
__device__ __forceinline__ uint32_t tile_at(uint32_t row, uint32_t col) { return row * 128 + ((((col >> 3) ^ row) & 7) << 4) + ((col & 7) << 1); }

template <typename T, int PARTS>
__global__ void __launch_bounds__(SMALL_THREADS, 1) small_kernel(const __grid_constant__ SmallArgs p) {
  using SM = Small<PARTS>;
  using S = typename Elem<T>::store_t;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw);
  const uint32_t bar = base + SM::TAIL;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + SM::TAIL + 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  double* sums = reinterpret_cast<double*>(smem + SM::TAIL + 16);      // [0] this CTA's, [1..8] the warps'
  const uint32_t rank = cluster_rank(), ctas = cluster_size(), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(smem_u32(tmem_slot), 512);
  // all of X and A, so that rows and columns the matrix does not have are zeros
  for (uint32_t i = threadIdx.x; i < SM::STAGE / 16; i += SMALL_THREADS) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_trigger();
  pdl_wait();

  const SmallMatrix& m = p.m[blockIdx.x / ctas];
  const uint32_t j0 = rank * p.cols, nj = p.hi > j0 ? min(p.cols, p.hi - j0) : 0;        // this CTA's columns of X
  const S* g = (const S*)m.g;
  S* b = (S*)m.buf;
  // Eight neighbours in memory per item.  Lying: eight columns of a row of X.  Standing (the stored matrix is X transposed): this CTA's
  // columns are whole stored rows, one stretch of memory that starts on a 128-byte boundary, whatever the rows' length.
  const uint32_t eights = (nj + 7) / 8, stretch = nj * p.lo, items = m.tall ? (stretch + 7) / 8 : eights * p.lo;
  const bool vector = m.tall || p.hi % 8 == 0;
  auto load = [&](float (&v)[8], const S* from, uint64_t at, uint32_t n) {
    if (vector && n == 8) {
      constexpr int VEC = 16 / (int)sizeof(S);
#pragma unroll
      for (int h = 0; h < 8 / VEC; ++h) {
        RawVec<T, VEC> r;
        r.load(from + at + h * VEC);
        float f[VEC];
        r.decode(f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[h * VEC + j] = f[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = j < (int)n ? Elem<T>::load(from[at + j]) : 0.0f;
    }
  };
  auto save = [&](const float (&v)[8], S* to, uint64_t at, uint32_t n, bool rn) {
    if (vector && n == 8) {
      constexpr int VEC = 16 / (int)sizeof(S);
#pragma unroll
      for (int h = 0; h < 8 / VEC; ++h) {
        RawVec<T, VEC> r;
        float o[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) o[j] = v[h * VEC + j];
        round_encode<T, VEC>(r, o, rn);
        r.store(to + at + h * VEC);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < (int)n) to[at + j] = round_store<T>(v[j], rn);
    }
  };

  // U items at a time, so that their loads are in flight together (four: 63 us at 128 x 784 f32, two: 61)
  constexpr uint32_t U = 2;
  // at: the first element; r, c: its place in X; n: how many of the eight are this item's
  struct Item { uint64_t at; uint32_t r, c, n; };
  auto item_at = [&](uint32_t i) {
    Item t{0, 0, 0, 0};
    if (i < items) {
      if (m.tall) {
        t.at = (uint64_t)j0 * p.lo + i * 8;
        t.c = i * 8 / p.lo; t.r = i * 8 % p.lo;
        t.n = min(8u, stretch - i * 8);
      } else {
        t.r = i / eights; t.c = i % eights * 8;
        t.at = (uint64_t)t.r * p.hi + j0 + t.c;
        t.n = min(8u, nj - t.c);
      }
    }
    return t;
  };

  // an item's eight entries of X, packed in pairs per part, to and from shared memory
  auto x_at = [&](uint32_t s, uint32_t r, uint32_t c) { return smem + SM::X + ((c >> 6) * PARTS + s) * SM::TILE_BYTES + tile_at(r, c & 63); };
  auto put = [&](const Item& t, const uint32_t (&w)[2][4]) {
    if (!m.tall) {
#pragma unroll
      for (int s = 0; s < PARTS; ++s) *reinterpret_cast<uint4*>(x_at(s, t.r, t.c)) = make_uint4(w[s][0], w[s][1], w[s][2], w[s][3]);
      return;
    }
    uint32_t r = t.r, c = t.c;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j < (int)t.n) {
#pragma unroll
        for (int s = 0; s < PARTS; ++s) *reinterpret_cast<uint16_t*>(x_at(s, r, c)) = (uint16_t)(w[s][j / 2] >> (16 * (j & 1)));
      }
      if (++r == p.lo) { r = 0; ++c; }
    }
  };
  auto take = [&](const Item& t, uint32_t (&w)[2][4]) {
    if (!m.tall) {
#pragma unroll
      for (int s = 0; s < PARTS; ++s) {
        const uint4 q = *reinterpret_cast<const uint4*>(x_at(s, t.r, t.c));
        w[s][0] = q.x; w[s][1] = q.y; w[s][2] = q.z; w[s][3] = q.w;
      }
      return;
    }
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j) w[s][j] = 0u;
    uint32_t r = t.r, c = t.c;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j < (int)t.n) {
#pragma unroll
        for (int s = 0; s < PARTS; ++s) w[s][j / 2] |= (uint32_t)*reinterpret_cast<const uint16_t*>(x_at(s, r, c)) << (16 * (j & 1));
      }
      if (++r == p.lo) { r = 0; ++c; }
    }
  };

  // Two parts, lying: between the passes the direction waits in X's place (standing, its entries lie apart: it is read again).
  const bool stash = PARTS == 2 && !m.tall;
  // momentum, and the sum of squares of the direction (64 bits: see muon.cu)
  double sum = 0.0;
  for (uint32_t i0 = threadIdx.x; i0 < items; i0 += U * SMALL_THREADS) {
    Item t[U];
    float u[U][8], f[U][8];
#pragma unroll
    for (uint32_t e = 0; e < U; ++e) {
      t[e] = item_at(i0 + e * SMALL_THREADS);
      load(u[e], g, t[e].at, t[e].n);
      if (b) load(f[e], b, t[e].at, t[e].n);
    }
#pragma unroll
    for (uint32_t e = 0; e < U; ++e) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        u[e][j] *= p.grad_scale;
        if (b) {
          f[e][j] = Elem<T>::load(round_store<T>(p.momentum * f[e][j] + u[e][j], p.rn != 0));
          u[e][j] = p.nesterov ? u[e][j] + p.momentum * f[e][j] : f[e][j];
        }
        sum += (double)u[e][j] * (double)u[e][j];
      }
      if (b) save(f[e], b, t[e].at, t[e].n, true);          // exact: rounded above
      if (stash && t[e].n) {
        // The direction waits for its norm in X's own place: the upper half of its bits where the high part will be, the lower half in
        // the low part's.
        uint32_t w[2][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          w[0][j] = __byte_perm(__float_as_uint(u[e][2 * j]), __float_as_uint(u[e][2 * j + 1]), 0x7632);
          w[1][j] = __byte_perm(__float_as_uint(u[e][2 * j]), __float_as_uint(u[e][2 * j + 1]), 0x5410);
        }
        put(t[e], w);
      }
    }
  }
  sum = warp_reduce(sum, OpSum());
  if (lane == 0) sums[1 + warp] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = 0.0;
    for (int w = 0; w < SMALL_THREADS / 32; ++w) s += sums[1 + w];
    sums[0] = s;
  }
  cluster_sync();
  double total = 0.0;
  for (uint32_t q = 0; q < ctas; ++q) total += ld_cluster_f64(map_to(smem_u32(sums), q));
  const float inv = (float)(SCALE / (sqrt(total) + (double)p.eps));      // the norm itself may lie outside f32
  for (uint32_t i0 = threadIdx.x; i0 < items; i0 += U * SMALL_THREADS) {
    Item t[U];
    float u[U][8], f[U][8];
#pragma unroll
    for (uint32_t e = 0; e < U; ++e) {
      t[e] = item_at(i0 + e * SMALL_THREADS);
      if (!stash) {
        load(u[e], g, t[e].at, t[e].n);
        if (b) load(f[e], b, t[e].at, t[e].n);              // what this thread stored
      }
    }
#pragma unroll
    for (uint32_t e = 0; e < U; ++e) {
      if (t[e].n == 0) continue;
      uint32_t w[2][4];
      if (stash) {
        take(t[e], w);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          u[e][2 * j] = __uint_as_float(__byte_perm(w[1][j], w[0][j], 0x5410)) * inv;
          u[e][2 * j + 1] = __uint_as_float(__byte_perm(w[1][j], w[0][j], 0x7632)) * inv;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          u[e][j] *= p.grad_scale;
          if (b) u[e][j] = p.nesterov ? u[e][j] + p.momentum * f[e][j] : f[e][j];
          u[e][j] *= inv;
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) split2(u[e][2 * j], u[e][2 * j + 1], w[0][j], w[1][j]);
      put(t[e], w);
    }
  }
  fence_proxy_async_all();
  tc_fence_before();
  __syncthreads();

  constexpr uint32_t gram_idesc = make_idesc(false, false, false, 128, 128), poly_idesc = make_idesc(false, false, true, 128, 128);
  const uint32_t tiles = p.cols / 64, x_base = base + SM::X, a_base = base + SM::A, stage = base + SM::STAGE;
  const uint32_t quarter = warp & 3, half = warp >> 2, row = quarter * 32 + lane, lane_addr = (quarter * 32u) << 16;
  uint32_t phase = 0;
  // one product with its parts; the small ones first
  auto multiply = [&](uint32_t d, uint32_t a, uint32_t a_part, uint32_t bb, uint32_t b_part, uint32_t lbo, uint32_t idesc, bool more) {
    auto ad = [&](int q) { return make_smem_desc(a + q * a_part, 16, 1024); };
    auto bd = [&](int q) { return make_smem_desc(bb + q * b_part, lbo, 1024); };
    if constexpr (PARTS == 2) {
      umma_f16(d, ad(1), bd(0), idesc, more ? 1u : 0u);
      umma_f16(d, ad(0), bd(1), idesc, 1u);
      umma_f16(d, ad(0), bd(0), idesc, 1u);
    } else {
      umma_f16(d, ad(0), bd(0), idesc, more ? 1u : 0u);
    }
  };
  auto wait = [&] {
    mbar_wait(bar, phase, abort_flag, p.status, ERR_SMALL);      // given up: the status word tells, every barrier below is still reached
    phase ^= 1;
    tc_fence_after();
  };
  auto a_byte = [&](uint32_t s, uint32_t r, uint32_t c) { return (s * 2 + (c >> 6)) * SM::TILE_BYTES + tile_at(r, c & 63); };     // of A

  // where this warp's blocks of the mirror image lie: the same in every step
  constexpr uint32_t WARPS = SMALL_THREADS / 32, MIRRORS = (30 * PARTS + WARPS - 1) / WARPS;
  uint32_t mirror_from[MIRRORS], mirror_to[MIRRORS];
#pragma unroll
  for (uint32_t e = 0; e < MIRRORS; ++e) {
    const uint32_t op = min(warp + e * WARPS, 30u * PARTS - 1), part = op / 30, t = op % 30 * 4 + (lane >> 3);
    uint32_t bi = (uint32_t)((1.0f + sqrtf(1.0f + 8.0f * (float)t)) * 0.5f);        // bi (bi - 1) / 2 <= t
    while (bi * (bi + 1) / 2 <= t) ++bi;
    while (bi * (bi - 1) / 2 > t) --bi;
    const uint32_t bj = t - bi * (bi - 1) / 2, in = lane & 7;
    mirror_from[e] = a_base + a_byte(part, bi * 8 + in, bj * 8);
    mirror_to[e] = a_base + a_byte(part, bj * 8 + in, bi * 8);
  }
  const uint32_t diagonal_block = (warp & 3) * 4 + (lane >> 3), on_diagonal = a_base + a_byte(warp < 4 ? 0 : 1, diagonal_block * 8 + (lane & 7), diagonal_block * 8);

  for (int it = 0; it < p.steps; ++it) {
    // ---- gram: two parts: an accumulator per 128 of k (24 additions), as in muon_gemm.cuh
    if (threadIdx.x == 0) {
      tc_fence_after();
      for (uint32_t t = 0; t < tiles; ++t)
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          const uint32_t at = x_base + t * PARTS * SM::TILE_BYTES + kk * 32, d = tmem + (PARTS == 2 ? (t >> 1) * 128 : 0);
          multiply(d, at, SM::TILE_BYTES, at, SM::TILE_BYTES, 16, gram_idesc, (PARTS == 2 ? (t & 1) : t) != 0 || kk != 0);
        }
      umma_commit(bar);
    }
    wait();
    // The lower triangle, in units of four columns: row r has r / 4 + 1 of them, behind 2 q (q + 1) + (r % 4)(q + 1) others (q = r / 4).
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      const uint32_t c0 = half * 64 + h * 32;
      if (c0 > quarter * 32) continue;                 // above the diagonal for the whole warp
      float v[32];
      uint32_t r[32];
      tmem_ld32(tmem + lane_addr + c0, r);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
      if (PARTS == 2 && tiles > 2) {
        tmem_ld32(tmem + lane_addr + 128 + c0, r);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] += __uint_as_float(r[j]);
      }
#pragma unroll
      for (uint32_t q = 0; q < 8; ++q)
        if (c0 / 4 + q <= row / 4) *reinterpret_cast<float4*>(smem + SM::STAGE + unit_at(row, c0 / 4 + q)) = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
    }
    cluster_sync();
    // the C-th part of the units each
    const uint32_t share = (STAGE_UNITS + ctas - 1) / ctas;
    const uint32_t last = min(STAGE_UNITS, (rank + 1) * share);
    for (uint32_t i0 = rank * share + threadIdx.x; i0 < last; i0 += 2 * SMALL_THREADS) {      // two at a time: 264 units on 256 threads
      float4 f[2][SMALL_CTAS];
#pragma unroll
      for (uint32_t e = 0; e < 2; ++e)
#pragma unroll
        for (uint32_t k = 0; k < SMALL_CTAS; ++k)
          if (k < ctas && i0 + e * SMALL_THREADS < last) f[e][k] = ld_cluster4(map_to(stage + (i0 + e * SMALL_THREADS) * 16, k));
#pragma unroll
      for (uint32_t e = 0; e < 2; ++e) {
        const uint32_t i = i0 + e * SMALL_THREADS;
        if (i >= last) break;
        uint32_t q4 = (uint32_t)((sqrtf(1.0f + 2.0f * (float)i) - 1.0f) * 0.5f);       // 2 q (q + 1) <= i
        while (2 * (q4 + 1) * (q4 + 2) <= i) ++q4;
        while (2 * q4 * (q4 + 1) > i) --q4;
        const uint32_t in = i - 2 * q4 * (q4 + 1), rr = q4 * 4 + in / (q4 + 1), q = in % (q4 + 1);
        float4 s = f[e][0];
#pragma unroll
        for (uint32_t k = 1; k < SMALL_CTAS; ++k)
          if (k < ctas) { s.x += f[e][k].x; s.y += f[e][k].y; s.z += f[e][k].z; s.w += f[e][k].w; }
        uint32_t w[2][2];
        split2(s.x * UNSCALE, s.y * UNSCALE, w[0][0], w[1][0]);
        split2(s.z * UNSCALE, s.w * UNSCALE, w[0][1], w[1][1]);
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
          const uint32_t to = a_base + a_byte(part, rr, q * 4);
          for (uint32_t k = 0; k < ctas; ++k) st_cluster2(map_to(to, k), w[part][0], w[part][1]);
        }
      }
    }
    cluster_sync();
    // the upper triangle: the 120 blocks of 8 x 8 below the diagonal, four per instruction, loaded and stored transposed ...
#pragma unroll
    for (uint32_t e = 0; e < MIRRORS; ++e) {
      if (warp + e * WARPS >= 30 * PARTS) break;
      uint32_t r[4];
      ldmatrix4(r, mirror_from[e]);
      stmatrix4_trans(mirror_to[e], r);
    }
    // ... and the 16 on it, each put together from itself and its transpose
    if (warp < 4 * PARTS) {
      uint32_t r[4], t[4];
      ldmatrix4(r, on_diagonal);
      ldmatrix4_trans(t, on_diagonal);
      const uint32_t row8 = lane >> 2, col8 = (lane & 3) * 2;          // this lane's two entries of each block
#pragma unroll
      for (int j = 0; j < 4; ++j) r[j] = col8 + 1 <= row8 ? r[j] : col8 <= row8 ? __byte_perm(r[j], t[j], 0x7610) : t[j];
      __syncwarp();
      stmatrix4(on_diagonal, r);
    }
    fence_proxy_async_all();
    tc_fence_before();
    __syncthreads();
    // ---- poly
    if (threadIdx.x == 0) {
      fence_proxy_async_all();
      tc_fence_after();
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        // A is symmetric: as the right operand it is read down its rows (66 clocks a product against 93 of the other reading)
        multiply(tmem, a_base + (kk >> 2) * SM::TILE_BYTES + (kk & 3) * 32, 2 * SM::TILE_BYTES, a_base + kk * 2048, 2 * SM::TILE_BYTES, SM::TILE_BYTES, poly_idesc, kk != 0);
      }
      umma_commit(bar);
    }
    wait();
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      const uint32_t c0 = half * 64 + h * 32;
      uint32_t r[32];
      tmem_ld32(tmem + lane_addr + c0, r);
      tmem_ld_wait();
#pragma unroll
      for (uint32_t q = 0; q < 4; ++q) {
        uint4* at[PARTS];
        float a8[8];
#pragma unroll
        for (int s = 0; s < PARTS; ++s) {
          at[s] = reinterpret_cast<uint4*>(smem + SM::A + a_byte(s, row, c0 + q * 8));
          const uint4 w = *at[s];
          const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&ws[j]));
            a8[2 * j] = s ? a8[2 * j] + f.x : f.x;
            a8[2 * j + 1] = s ? a8[2 * j + 1] + f.y : f.y;
          }
        }
        uint32_t w[2][4];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float v = p.c * (__uint_as_float(r[q * 8 + j]) * UNSCALE) + p.b * a8[j];
          if (c0 + q * 8 + j == row) v += p.a * SCALE;
          a8[j] = v;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) split2(a8[2 * j], a8[2 * j + 1], w[0][j], w[1][j]);
#pragma unroll
        for (int s = 0; s < PARTS; ++s) *at[s] = make_uint4(w[s][0], w[s][1], w[s][2], w[s][3]);
      }
    }
    fence_proxy_async_all();
    tc_fence_before();
    __syncthreads();
    // ---- apply: 256 columns per product at most
    const uint32_t d0 = PARTS == 2 ? 256 : 0;
    if (threadIdx.x == 0) {
      tc_fence_after();
      for (uint32_t c0 = 0; c0 < p.cols; c0 += 256) {
        const uint32_t idesc = make_idesc(false, false, true, 128, (int)min(256u, p.cols - c0));
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          multiply(tmem + d0 + c0, a_base + (kk >> 2) * SM::TILE_BYTES + (kk & 3) * 32, 2 * SM::TILE_BYTES, x_base + (c0 >> 6) * PARTS * SM::TILE_BYTES + kk * 2048,
                   SM::TILE_BYTES, PARTS * SM::TILE_BYTES, idesc, kk != 0);
      }
      umma_commit(bar);
    }
    wait();
#pragma unroll 1
    for (uint32_t c0 = half * 32; c0 < p.cols; c0 += 64) {
      uint32_t r[32];
      tmem_ld32(tmem + lane_addr + d0 + c0, r);
      tmem_ld_wait();
#pragma unroll
      for (uint32_t q = 0; q < 4; ++q) {
        uint32_t w[2][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) split2(__uint_as_float(r[q * 8 + 2 * j]) * UNSCALE, __uint_as_float(r[q * 8 + 2 * j + 1]) * UNSCALE, w[0][j], w[1][j]);
#pragma unroll
        for (int s = 0; s < PARTS; ++s)
          *reinterpret_cast<uint4*>(smem + SM::X + ((c0 >> 6) * PARTS + s) * SM::TILE_BYTES + tile_at(row, (c0 & 63) + q * 8)) = make_uint4(w[s][0], w[s][1], w[s][2], w[s][3]);
      }
    }
    fence_proxy_async_all();
    tc_fence_before();
    __syncthreads();
  }

  // ---- the weight's step
  S* pw = (S*)m.p;
  const float step = (m.tall ? p.step_tall : p.step_flat) * UNSCALE;
  for (uint32_t i0 = threadIdx.x; i0 < items; i0 += U * SMALL_THREADS) {
    Item t[U];
    float f[U][8];
#pragma unroll
    for (uint32_t e = 0; e < U; ++e) {
      t[e] = item_at(i0 + e * SMALL_THREADS);
      load(f[e], pw, t[e].at, t[e].n);
    }
#pragma unroll
    for (uint32_t e = 0; e < U; ++e) {
      if (t[e].n == 0) continue;
      uint32_t w[2][4];
      take(t[e], w);
      float x[8];
#pragma unroll
      for (int s = 0; s < PARTS; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[s][j]));
          x[2 * j] = s ? x[2 * j] + v.x : v.x;
          x[2 * j + 1] = s ? x[2 * j + 1] + v.y : v.y;
        }
#pragma unroll
      for (int j = 0; j < 8; ++j) f[e][j] = f[e][j] * p.decay - step * x[j];
      save(f[e], pw, t[e].at, t[e].n, p.rn != 0);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace muon
}  // namespace zyxb
