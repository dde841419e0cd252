// The three products of a Newton-Schulz step on the 5th-generation tensor cores.
//   gram   A  = X X^T                      [m, m], symmetric
//   poly   B  = a I + b A + c A A^T        [m, m], symmetric (A A^T = A^2)
//   apply  X' = B X                        [m, n]
// Operands and results are f16 in the program's workspace, carried as `PARTS` numbers whose sum is the value: one (11 bits) or two
// (hi + lo, 22 bits).  All are multiplied by 2^10, which keeps the entries of a normed matrix (down to 2^-15 on average at the
// largest extent) and their low halves inside f16's normal range, and the largest possible entry (5, by the bound that the
// program puts on the coefficients) below its end.  Two parts take three products (the product of the low halves, 2^-22, is dropped).
//
// The pipeline is the 16-bit matmul's: one persistent CTA per SM, warp 0 loads tiles by TMA, warp 1 issues tcgen05.mma, warps 2..9
// read the accumulators from TMEM while the next tile is multiplied.  What differs:
//   pairs     CTAS = 2: two CTAs of a cluster share a tile of 256 rows (cta_group::2).  Each loads its 128 rows of the left operand
//             and half of the right one's columns, the first issues the instructions for both, each keeps its own rows' accumulator.
//             A tile's operands then cross L2 and shared memory once per pair: 4 x [2048 x 2048 x 2048] takes 55.5 us against 61.9 of
//             single CTAs with 128 x 256 tiles.
//   symmetry  only tiles that touch the lower triangle are computed, and stored twice: half of the work of gram and poly.
//   split     a gram product with few tiles and a long contraction is cut along it: every CTA leaves its f32 sums, and a second
//             launch adds them in order (129 x 4096 f32: 3 tiles, 64 k-blocks of 0.5 us each).
//   rounding  the tensor core adds with truncation, which over 1536 additions costs 1.5e-4 of the result: below the 2^-11 of one
//             part, far above the 2^-22 of two.  With two parts an accumulator takes 24 additions (128 of k), and the epilogue warps add
//             the accumulators in f32 registers.
// Every wait is bounded, like the matmul's.
#pragma once
#include <algorithm>

#include "common.cuh"
#include "internal.h"
#include "tc_ptx.cuh"

namespace zyxb {
namespace muon {

constexpr int BM = 128, BK = 64, UMMA_K = 16, THREADS = 320, EPI_THREADS = 256;
constexpr int CHUNK_BLOCKS = 2;        // two parts: k-blocks per accumulator
constexpr float SCALE = 1024.0f, UNSCALE = 1.0f / 1024.0f;
enum { ERR_PRODUCER = 0x20000u, ERR_MMA = 0x40000u, ERR_EPILOGUE = 0x80000u };

// [batch][part][rows][ld] f16
struct Operand {
  uint16_t* ptr;
  uint32_t rows, cols, ld;
  __host__ __device__ uint64_t part() const { return (uint64_t)rows * ld; }
};

struct GemmArgs {
  uint16_t* out;
  const uint16_t* gram;     // poly: A, shaped like out
  uint32_t m, n, k, batch, tiles_m, tiles_n, tiles, ld;
  uint64_t part, stride;    // elements from hi to lo, from matrix to matrix, of out
  float a, b, c;            // poly; c is 1 otherwise
  float* partial;           // split gram: [matrix][tile][split][128][BN]
  uint32_t splits;          // 1: none
  uint32_t* status;
};

template <int PARTS, int BN, int CTAS> struct Smem {
  static constexpr int B_ROWS = BN / CTAS;                       // of the right operand, per CTA
  static constexpr int A_PART = BM * BK * 2, B_PART = B_ROWS * BK * 2;
  static constexpr int STAGE = PARTS * (A_PART + B_PART);
  static constexpr int STAGES = 196608 / STAGE;
  static constexpr int BAR = STAGES * STAGE;
  static constexpr int TOTAL = BAR + 256 + 1024;
};

__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = pack2_t<false>(x, y);
  const float hx = __half2float(__ushort_as_half((uint16_t)hi)), hy = __half2float(__ushort_as_half((uint16_t)(hi >> 16)));
  lo = pack2_t<false>(x - hx, y - hy);
}

// ---- clusters --------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t cluster_size() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t map_to(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// a load into this CTA's shared memory that reports to a barrier of either CTA of the pair
__device__ __forceinline__ void tma_load_4d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int zi, int zo) {
  asm volatile(
      "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(zi), "r"(zo) : "memory");
}
template <int CTAS> __device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t more) {
  if constexpr (CTAS == 1) umma_f16(d, a, b, idesc, more);
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(more) : "memory");
}
// the barrier at this place in every CTA of the pair
template <int CTAS> __device__ __forceinline__ void commit(uint32_t bar) {
  if constexpr (CTAS == 1) umma_commit(bar);
  else
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
}
template <int CTAS> __device__ __forceinline__ void alloc(uint32_t dst_smem, uint32_t cols) {
  if constexpr (CTAS == 1) tmem_alloc(dst_smem, cols);
  else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int CTAS> __device__ __forceinline__ void dealloc(uint32_t taddr, uint32_t cols) {
  if constexpr (CTAS == 1) tmem_dealloc(taddr, cols);
  else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}

template <int PARTS, int BN, int CTAS, bool SYM, bool POLY, bool B_MN, bool SPLIT>
__global__ void __launch_bounds__(THREADS, 1)
gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, GemmArgs p) {
  using SM = Smem<PARTS, BN, CTAS>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t* base_ptr = smem_raw + (base - raw);
  const uint32_t bars = base + SM::BAR;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (SM::STAGES + s); };
  auto tfull_bar = [&](int a) { return bars + 8u * (2 * SM::STAGES + a); };
  auto tempty_bar = [&](int a) { return bars + 8u * (2 * SM::STAGES + 2 + a); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(base_ptr + SM::BAR + 8 * (2 * SM::STAGES + 4));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr uint32_t TMEM_COLS = 2 * BN;
  const uint32_t rank = CTAS == 2 ? cluster_rank() : 0;
  if (threadIdx.x == 0) {
    // of a pair, the first CTA's full and tempty barriers count for both; empty and tfull are signalled in both
    for (int s = 0; s < SM::STAGES; ++s) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(tfull_bar(a), 1); mbar_init(tempty_bar(a), CTAS * (EPI_THREADS / 32)); }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) alloc<CTAS>(smem_u32(tmem_slot), TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  if constexpr (CTAS == 2) cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_trigger();
  pdl_wait();

  const uint32_t splits = SPLIT ? p.splits : 1, total = p.tiles * p.batch * splits, all_blocks = (p.k + BK - 1) / BK;
  // the k-blocks of one of the splits (the last of a tile's work items may have fewer, never none)
  const uint32_t per_split = (all_blocks + splits - 1) / splits;
  auto k_range = [&](uint32_t t, uint32_t& k0, uint32_t& k1) {
    k0 = SPLIT ? t % splits * per_split : 0;
    k1 = SPLIT ? min(all_blocks, k0 + per_split) : all_blocks;
  };
  auto tile_coords = [&](uint32_t t, uint32_t& z, uint32_t& tm, uint32_t& tn) {
    if (SPLIT) t /= splits;
    z = t / p.tiles;
    const uint32_t r = t - z * p.tiles;
    if constexpr (SYM) {
      // square tiles (128 or 256): row tm has tm + 1 of them, tm (tm + 1) / 2 lie before it
      tm = (uint32_t)((sqrtf(1.0f + 8.0f * (float)r) - 1.0f) * 0.5f);
      while (tm * (tm + 1) / 2 > r) --tm;
      while ((tm + 1) * (tm + 2) / 2 <= r) ++tm;
      tn = r - tm * (tm + 1) / 2;
    } else {
      constexpr uint32_t GROUP_M = 16;   // tiles that run together share panels in L2
      const uint32_t group_size = GROUP_M * p.tiles_n, g = r / group_size, first_m = g * GROUP_M;
      const uint32_t rows_in_group = min(GROUP_M, p.tiles_m - first_m), in_group = r % group_size;
      tm = first_m + in_group % rows_in_group;
      tn = in_group / rows_in_group;
    }
  };

  if (warp == 0) {
    if (lane == 0) {
      uint32_t stage = 0, phase = 0, issued = 0;
      bool ok = true;
      for (uint32_t t = blockIdx.x / CTAS; t < total && ok; t += gridDim.x / CTAS) {
        uint32_t z, tm, tn;
        tile_coords(t, z, tm, tn);
        uint32_t kb0, kb1;
        k_range(t, kb0, kb1);
        for (uint32_t kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1, abort_flag, p.status, ERR_PRODUCER)) { ok = false; break; }
          const uint32_t a_dst = base + stage * SM::STAGE, b_dst = a_dst + PARTS * SM::A_PART;
          if (rank == 0) mbar_expect_tx(full_bar(stage), CTAS * SM::STAGE);
          const uint32_t full = CTAS == 2 ? map_to(full_bar(stage), 0) : full_bar(stage);
          auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int y, int part) {
            if constexpr (CTAS == 2) tma_load_4d_pair(dst, map, full, x, y, part, (int)z);
            else tma_load_4d(dst, map, full, x, y, part, (int)z);
          };
          const int k0 = (int)(kb * BK), row_a = (int)((tm * CTAS + rank) * BM), row_b = (int)(tn * BN + rank * SM::B_ROWS);
#pragma unroll
          for (int q = 0; q < PARTS; ++q) {
            load(a_dst + q * SM::A_PART, &map_a, k0, row_a, q);
            if constexpr (B_MN) {
#pragma unroll
              for (int j = 0; j < SM::B_ROWS / 64; ++j) load(b_dst + q * SM::B_PART + j * (64 * BK * 2), &map_b, row_b + j * 64, k0, q);
            } else {
              load(b_dst + q * SM::B_PART, &map_b, k0, row_b, q);
            }
          }
          ++issued;
          if (++stage == SM::STAGES) { stage = 0; phase ^= 1; }
        }
      }
      // Every stage's last release is waited for before the CTA goes: the issuer's commits arrive in both CTAs of a pair, tfull's says
      // nothing of the ones before it, and the shared memory has to be there when they come.
      for (uint32_t i = 0, s = stage, ph = phase; i < (uint32_t)SM::STAGES && ok; ++i) {
        ok = mbar_wait(empty_bar(s), ph ^ 1, abort_flag, p.status, ERR_PRODUCER);
        if (++s == SM::STAGES) { s = 0; ph ^= 1; }
      }
      if (!ok && rank == 0) {     // copies in flight land before the CTA goes (a pair's: both wait for each other at the end)
        uint32_t s = stage, ph = phase;
        const uint32_t n_back = issued < (uint32_t)SM::STAGES ? issued : (uint32_t)SM::STAGES;
        for (uint32_t i = 0; i < n_back; ++i) {
          if (s == 0) { s = SM::STAGES - 1; ph ^= 1; } else --s;
          const uint64_t t0 = global_timer_ns();
          while (!mbar_try_wait(full_bar(s), ph) && global_timer_ns() - t0 < TC_WAIT_NS) {}
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = make_idesc(false, false, B_MN, BM * CTAS, BN);
      uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
      bool ok = true;
      for (uint32_t t = blockIdx.x / CTAS; t < total && ok; t += gridDim.x / CTAS) {
        uint32_t kb0, kb1;
        k_range(t, kb0, kb1);
        for (uint32_t kb = kb0; kb < kb1 && ok; ++kb) {
          const uint32_t in_chunk = PARTS == 2 ? (kb - kb0) % CHUNK_BLOCKS : kb - kb0;
          if (in_chunk == 0) {
            if (!mbar_wait(tempty_bar(acc), acc_phase ^ 1, abort_flag, p.status, ERR_MMA)) { ok = false; break; }
            tc_fence_after();
          }
          const uint32_t d_tmem = tmem_base + acc * BN;
          if (!mbar_wait(full_bar(stage), phase, abort_flag, p.status, ERR_MMA)) { ok = false; break; }
          tc_fence_after();
          const uint32_t a_addr = base + stage * SM::STAGE, b_addr = a_addr + PARTS * SM::A_PART;
#pragma unroll
          for (int kk = 0; kk < BK / UMMA_K; ++kk) {
            auto adesc = [&](int q) { return make_smem_desc(a_addr + q * SM::A_PART + kk * (UMMA_K * 2), 16, 1024); };
            auto bdesc = [&](int q) {
              return B_MN ? make_smem_desc(b_addr + q * SM::B_PART + kk * (UMMA_K * 128), 64 * BK * 2, 1024)
                          : make_smem_desc(b_addr + q * SM::B_PART + kk * (UMMA_K * 2), 16, 1024);
            };
            const uint32_t more = (in_chunk | (uint32_t)kk) != 0 ? 1u : 0u;
            if constexpr (PARTS == 2) {     // the small products first
              mma<CTAS>(d_tmem, adesc(1), bdesc(0), idesc, more);
              mma<CTAS>(d_tmem, adesc(0), bdesc(1), idesc, 1u);
              mma<CTAS>(d_tmem, adesc(0), bdesc(0), idesc, 1u);
            } else {
              mma<CTAS>(d_tmem, adesc(0), bdesc(0), idesc, more);
            }
          }
          commit<CTAS>(empty_bar(stage));
          if (++stage == SM::STAGES) { stage = 0; phase ^= 1; }
          if (kb + 1 == kb1 || (PARTS == 2 && in_chunk == CHUNK_BLOCKS - 1)) {
            commit<CTAS>(tfull_bar(acc));
            if (++acc == 2) { acc = 0; acc_phase ^= 1; }
          }
        }
      }
    }
  } else {
    // lane = row; two warps per TMEM lane quarter, each with half of the columns
    const int col_half = (warp - 2) >> 2;
    const uint32_t quarter = (uint32_t)(warp & 3);
    constexpr int HALF = BN / 2, CH = HALF / 32;
    auto release = [&](uint32_t a) {                       // the accumulator goes back to the issuer
      if constexpr (CTAS == 2) mbar_arrive_cluster(map_to(tempty_bar(a), 0));
      else mbar_arrive(tempty_bar(a));
    };
    uint32_t acc = 0, acc_phase = 0;
    bool ok = true;
    for (uint32_t t = blockIdx.x / CTAS; t < total && ok; t += gridDim.x / CTAS) {
      uint32_t z, tm, tn;
      tile_coords(t, z, tm, tn);
      uint32_t kb0, kb1;
      k_range(t, kb0, kb1);
      const uint32_t n_chunks = PARTS == 2 ? (kb1 - kb0 + CHUNK_BLOCKS - 1) / CHUNK_BLOCKS : 1;
      const uint32_t col0 = tn * BN;
      uint16_t* out = p.out + z * p.stride;
      const uint16_t* gram = POLY ? p.gram + z * p.stride : nullptr;
      const uint32_t row0 = (tm * CTAS + rank) * BM + quarter * 32, row = row0 + lane;
      // A's entries under them.  One part: asked for a block of 32 columns ahead, the first while the tile is still being multiplied
      // (some 1.6 us less a launch at 4 x 2048^2); two parts hold their sums in those registers.
      auto load_gram = [&](uint4 (&w)[4], uint32_t c, int s) {
        const uint16_t* from = gram + s * p.part + (uint64_t)row * p.ld + c;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (row < p.m && c <= row0 && c + q * 8 < p.n) w[q] = *reinterpret_cast<const uint4*>(from + q * 8);
      };
      // 32 columns from c on of this lane's row
      auto finish = [&](float (&v)[32], uint32_t c, const uint4 (&ahead)[4]) {
        if (c >= p.n || row0 >= p.m) return;
        if constexpr (SPLIT) {
          float4* to = reinterpret_cast<float4*>(p.partial + ((uint64_t)t * BM + quarter * 32 + lane) * BN + (c - col0));
#pragma unroll
          for (int q = 0; q < 8; ++q) to[q] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
          return;
        }
        if (SYM && c > row0) return;                           // above the diagonal: another warp's mirrored block
        const uint64_t at = (uint64_t)row * p.ld + c;
        const bool mine = row < p.m;
        if constexpr (POLY) {
          if (mine) {
            uint4 wide[PARTS][4];
            if constexpr (PARTS == 2) { load_gram(wide[0], c, 0); load_gram(wide[PARTS - 1], c, 1); }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              if (c + q * 8 >= p.n) break;
              float g[8];
#pragma unroll
              for (int s = 0; s < PARTS; ++s) {
                const uint4 w = PARTS == 2 ? wide[s][q] : ahead[q];
                const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const float lo = __half2float(__ushort_as_half((uint16_t)ws[j])), hi = __half2float(__ushort_as_half((uint16_t)(ws[j] >> 16)));
                  g[2 * j] = s ? g[2 * j] + lo : lo;
                  g[2 * j + 1] = s ? g[2 * j + 1] + hi : hi;
                }
              }
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                v[q * 8 + j] = p.c * (v[q * 8 + j] * UNSCALE) + p.b * g[j];
                if (c + q * 8 + j == row) v[q * 8 + j] += p.a * SCALE;
              }
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] *= UNSCALE;
        }
        uint32_t w[PARTS][16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          if constexpr (PARTS == 2) split2(v[2 * j], v[2 * j + 1], w[0][j], w[PARTS - 1][j]);
          else w[0][j] = pack2_t<false>(v[2 * j], v[2 * j + 1]);
        }
        if (mine) {
#pragma unroll
          for (int s = 0; s < PARTS; ++s)
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (c + q * 8 < p.n)                             // ld is a multiple of 8: what lies behind n is spare
                *reinterpret_cast<uint4*>(out + s * p.part + at + q * 8) = make_uint4(w[s][4 * q], w[s][4 * q + 1], w[s][4 * q + 2], w[s][4 * q + 3]);
        }
        if constexpr (SYM) {
          // Mirrored, unless the warp's 32 x 32 block lies on the diagonal (there the whole block has been computed and stored): two
          // neighbouring lanes trade halves, so that each stores two rows' entries of one column side by side.
          if (c < row0) {
            const bool odd = lane & 1;
#pragma unroll
            for (int s = 0; s < PARTS; ++s)
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                const uint32_t other = __shfl_xor_sync(0xffffffffu, w[s][j], 1);
                const uint32_t pair = odd ? __byte_perm(other, w[s][j], 0x7632) : __byte_perm(w[s][j], other, 0x5410);
                if ((row | 1u) < p.ld)
                  *reinterpret_cast<uint32_t*>(out + s * p.part + (uint64_t)(c + 2 * j + (odd ? 1 : 0)) * p.ld + (row & ~1u)) = pair;
              }
          }
        }
      };
      if constexpr (PARTS == 2) {
        float sum[HALF];
#pragma unroll
        for (int i = 0; i < HALF; ++i) sum[i] = 0.0f;
        for (uint32_t ck = 0; ck < n_chunks && ok; ++ck) {
          if (!mbar_wait(tfull_bar(acc), acc_phase, abort_flag, p.status, ERR_EPILOGUE)) { ok = false; break; }
          tc_fence_after();
#pragma unroll
          for (int ch = 0; ch < CH; ++ch) {
            uint32_t r[32];
            tmem_ld32(tmem_base + ((quarter * 32u) << 16) + acc * BN + (col_half * CH + ch) * 32, r);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) sum[ch * 32 + i] += __uint_as_float(r[i]);
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) release(acc);
          if (++acc == 2) { acc = 0; acc_phase ^= 1; }
        }
        if (!ok) break;
#pragma unroll
        for (int ch = 0; ch < CH; ++ch) {
          float v[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = sum[ch * 32 + i];
          finish(v, col0 + (col_half * CH + ch) * 32, {});
        }
      } else {
        uint4 ahead[4];
        if constexpr (POLY) load_gram(ahead, col0 + col_half * CH * 32, 0);
        if (!mbar_wait(tfull_bar(acc), acc_phase, abort_flag, p.status, ERR_EPILOGUE)) { ok = false; break; }
        tc_fence_after();
#pragma unroll 1
        for (int ch = 0; ch < CH; ++ch) {
          uint32_t r[32];
          tmem_ld32(tmem_base + ((quarter * 32u) << 16) + acc * BN + (col_half * CH + ch) * 32, r);
          tmem_ld_wait();
          float v[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
          uint4 now[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) now[q] = ahead[q];
          if constexpr (POLY) { if (ch + 1 < CH) load_gram(ahead, col0 + (col_half * CH + ch + 1) * 32, 0); }
          finish(v, col0 + (col_half * CH + ch) * 32, now);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) release(acc);
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (CTAS == 2) cluster_sync();                 // the pair's instructions read both CTAs' shared memory
  if (warp == 1) {
    tc_fence_after();
    dealloc<CTAS>(tmem_base, TMEM_COLS);
  }
}

// ---- split gram ----------------------------------------------------------------------------------------------------------------
// A = 2^-10 times the sum of the splits' tiles, as parts, with its mirror image: a 64 x 64 block of the lower triangle per CTA.
template <int PARTS>
__global__ void __launch_bounds__(256) gram_finish_kernel(const float* __restrict__ partial, uint32_t splits, uint32_t tiles, GemmArgs p) {
  __shared__ float block[64][65];
  const uint32_t bi = blockIdx.x, bj = blockIdx.y, z = blockIdx.z;
  pdl_trigger();
  pdl_wait();
  if (bj > bi) return;
  const uint32_t tm = bi / 2, tn = bj / 2, tile = tm * (tm + 1) / 2 + tn;
  const float* from = partial + (((uint64_t)z * tiles + tile) * splits * BM + (bi & 1) * 64) * 128 + (bj & 1) * 64;
  // past m there are rows no split has written; they are not read
  const uint32_t rows = min(64u, p.m - bi * 64);
  for (uint32_t i = threadIdx.x; i < rows * 16; i += 256) {
    const uint32_t r = i / 16, c = i % 16 * 4;
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (bj * 64 + (c & 32) < p.m) {
#pragma unroll 8
      for (uint32_t k = 0; k < splits; ++k) {
        const float4 v = *reinterpret_cast<const float4*>(from + ((uint64_t)k * BM + r) * 128 + c);
        s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
      }
    }
    block[r][c] = s.x; block[r][c + 1] = s.y; block[r][c + 2] = s.z; block[r][c + 3] = s.w;
  }
  __syncthreads();
  uint16_t* out = p.out + z * p.stride;
  auto put = [&](uint32_t row, uint32_t col, const float (&v)[8]) {
    uint32_t w[2][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) split2(v[2 * j] * UNSCALE, v[2 * j + 1] * UNSCALE, w[0][j], w[1][j]);
#pragma unroll
    for (int s = 0; s < PARTS; ++s)
      *reinterpret_cast<uint4*>(out + s * p.part + (uint64_t)row * p.ld + col) = make_uint4(w[s][0], w[s][1], w[s][2], w[s][3]);
  };
  for (uint32_t i = threadIdx.x; i < 512; i += 256) {
    const uint32_t r = i / 8, c = i % 8 * 8;
    if (bi * 64 + r >= p.m || bj * 64 + c >= p.m) continue;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = block[r][c + j];
    put(bi * 64 + r, bj * 64 + c, v);                      // columns behind m: spare
  }
  if (bi == bj) return;
  for (uint32_t i = threadIdx.x; i < 512; i += 256) {
    const uint32_t r = i % 64, c = i / 64 * 8;             // row r of the image: column r of the block
    if (bj * 64 + r >= p.m || bi * 64 + c >= p.m) continue;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < rows ? block[c + j][r] : 0.0f;
    put(bj * 64 + r, bi * 64 + c, v);
  }
}

// CTAs that a split gram product may use: their partial sums are 64 KB each
constexpr uint32_t SPLIT_CTAS = 144;
// Splits of a gram product with 128 x 128 tiles: as many as give every CTA work, of four k-blocks at least.  The second launch costs
// some 5 us a step, a k-block 0.5 us with two parts and 0.15 us with one, so 16 and 40 blocks have to be saved.  Measured, whole
// updates: 129 x 4096 f32 344 -> 204 us, bf16 186 -> 144; 512 x 2048 f32 297 -> 249; below the rule 1024 x 1024 f32 299 -> 308,
// bf16 165 -> 198, 512 x 2048 bf16 162 -> 165.
template <int PARTS> uint32_t split_count(uint32_t m, uint32_t k, uint32_t batch) {
  const uint32_t tiles_m = (m + BM - 1) / BM;
  const uint64_t work = (uint64_t)tiles_m * (tiles_m + 1) / 2 * batch;
  const uint32_t blocks = (k + BK - 1) / BK;
  const uint32_t s = (uint32_t)std::min<uint64_t>(SPLIT_CTAS / std::max<uint64_t>(1, work), blocks / 4);
  if (s < 2) return 1;
  const uint32_t per = (blocks + s - 1) / s;
  if (blocks - per < (PARTS == 2 ? 16 : 40)) return 1;
  return (blocks + per - 1) / per;                          // no split without a block
}

// {contiguous, rows, parts, matrices} with a box of 64 x `box_rows`
inline bool encode(void* fn, CUtensorMap* map, const Operand& o, int parts, uint32_t batch, uint32_t box_rows) {
  return encode_map(fn, map, false, o.ptr, o.cols, o.rows, o.ld, (uint64_t)parts, parts > 1 ? o.part() : 0, batch, batch > 1 ? o.part() * parts : 0, box_rows);
}

// square tiles that cover a result (of a symmetric one: its lower triangle)
template <bool SYM> uint32_t tile_count(uint32_t m, uint32_t n, uint32_t size) {
  const uint32_t tiles_m = (m + size - 1) / size;
  return SYM ? tiles_m * (tiles_m + 1) / 2 : tiles_m * ((n + size - 1) / size);
}
// 1: tiles of 128 x 128, a CTA each; 2: 256 x 256, a pair.  A round of single CTAs' tiles takes 0.92 of a round of the pairs' with one
// part, 0.59 with two, where the tensor core works longest on what it reads (k = 2048: 12.7 against 13.9 us, 25.3 against 42.5).
// (Pairs' tiles of 256 x 128 lose to single CTAs' either way; the last round's tiles in halves changed no whole update: they run
// under the power limit.)
template <int PARTS, bool SYM> int tile_ctas(uint32_t m, uint32_t n, uint32_t batch, int sm_count) {
  const uint32_t pairs = (uint32_t)sm_count / 2, single = tile_count<SYM>(m, n, 128) * batch, wide = tile_count<SYM>(m, n, 256) * batch;
  if (single <= (uint32_t)sm_count) return 1;            // one round either way; a pair's start costs a microsecond more
  return (uint64_t)((single + sm_count - 1) / sm_count) * (PARTS == 1 ? 92 : 59) <= (uint64_t)((wide + pairs - 1) / pairs) * 100 ? 1 : 2;
}

template <int PARTS, int BN, int CTAS, bool SYM, bool POLY, bool B_MN, bool SPLIT = false>
cudaError_t launch(const CUtensorMap& ma, const CUtensorMap& mb, GemmArgs p, const LaunchCtx& lc) {
  using SM = Smem<PARTS, BN, CTAS>;
  static uint64_t configured = 0;
  auto kern = gemm_kernel<PARTS, BN, CTAS, SYM, POLY, B_MN, SPLIT>;
  cudaError_t e = ensure_dynamic_smem(kern, SM::TOTAL, &configured);
  if (e != cudaSuccess) return e;
  p.tiles_m = (p.m + BM * CTAS - 1) / (BM * CTAS);
  p.tiles_n = (p.n + BN - 1) / BN;
  static_assert(BN == BM * CTAS, "square tiles");
  p.tiles = tile_count<SYM>(p.m, p.n, BN);
  p.status = lc.status_word;
  const uint64_t items = (uint64_t)p.tiles * p.batch * (SPLIT ? p.splits : 1);
  const unsigned grid = CTAS * (unsigned)std::min<uint64_t>(items, (uint64_t)lc.sm_count / CTAS);
  if constexpr (CTAS == 2) {
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = CTAS; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = SM::TOTAL; cfg.stream = lc.stream;
    cfg.attrs = attr; cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kern, ma, mb, p);
  }
  return launch_pdl(kern, dim3(grid), THREADS, SM::TOTAL, lc.stream, ma, mb, p);
}

template <int PARTS, bool SYM, bool POLY, bool B_MN>
cudaError_t launch(int ctas, const CUtensorMap& ma, const CUtensorMap& mb, const GemmArgs& p, const LaunchCtx& lc) {
  return ctas == 1 ? launch<PARTS, 128, 1, SYM, POLY, B_MN>(ma, mb, p, lc) : launch<PARTS, 256, 2, SYM, POLY, B_MN>(ma, mb, p, lc);
}

}  // namespace muon
}  // namespace zyxb
