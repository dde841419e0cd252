// Embedding lookup and the gradient of its table.
//   out[i,:]    = scale * table[ids[i],:]                      (zeros for an id outside [0, vocab))
//   dtable[v,:] = scale * sum_{i : ids[i] = v} dout[i,:]       (+ dtable[v,:])
//
// Lookup: a copy, bound by HBM.  A group of threads spans one row's 16-byte vectors and moves four tokens at a time.  Where rows do
// not start on vector boundaries (an odd width or pitch), vectors are aligned to the row that is written and shifted out of the
// two they lie in where they are read.
//
// Gradient, three launches and no floating-point atomic:
//   index    The vocabulary is cut into ranges, one CTA each.  Every CTA scans all token numbers (from L2; 64 KB at 16384 tokens),
//            counts those below its range - which is where its part of the sorted order begins, so no CTA waits for another - and
//            counting-sorts those inside it.
//   sum      The sorted order is cut into chunks of equal length, whatever the token frequencies.  A group of threads adds the rows
//            of the runs that begin in its chunk in f32 registers; a run of more than two chunks is shared by the chunks it
//            crosses, each leaving f32 partials.  The same launch writes the rows of zeros.
//   combine  Adds the partials of each shared run, in chunk order.
// The order of every sum is fixed by ids and by where the chunks end, which the launch chooses by extents, type, SMs and scratch memory.
// The index launch reads all token numbers in every CTA: 0.04 ms at 2^16 tokens and rows, 0.12 at 2^18, 1.0 at 2^20, and as tokens x
// rows from there.
#include <algorithm>

#include "internal.h"
#include "rounding.cuh"

namespace zyxb {

namespace {

constexpr int EMB_THREADS = 256;
constexpr int EMB_TOKENS = 4;          // rows in flight per thread
constexpr int IDX_THREADS = 1024, IDX_WARPS = IDX_THREADS / 32;
constexpr int IDX_MAX_ROWS = 1024;     // rows of a vocabulary range, one per thread (histograms: 32 warps x 1024 x 4 B of shared memory)
constexpr int IDX_BATCH = 4;           // loads of four token numbers in flight per lane
constexpr int CMB_WARPS = 8, CMB_COLS = 128;
constexpr uint32_t CHUNK = 32, CHUNK_LEAST = 8;      // places of the sorted order per group; runs of more than two chunks are shared
constexpr int FILL_ROWS = 64;          // table rows that a CTA of the sum launch looks through for absent ones

template <typename ID> __device__ __forceinline__ int64_t id_at(const ID* ids, uint64_t i) { return (int64_t)ids[i]; }

template <typename T> constexpr int emb_vec() { return 16 / (int)sizeof(typename Elem<T>::store_t); }

// entries [from, to) of a vector, one by one
template <typename T>
__device__ __forceinline__ void emb_store_some(typename Elem<T>::store_t* at, const RawVec<T, emb_vec<T>()>& r, int from, int to) {
#pragma unroll
  for (int k = 0; k < emb_vec<T>(); ++k)
    if (k >= from && k < to) {
      if constexpr (sizeof(typename Elem<T>::store_t) == 2) at[k] = (uint16_t)(r.w[k / 2] >> (16 * (k & 1)));
      else at[k] = __uint_as_float(r.w[k]);
    }
}

// VEC values of a row from column c on (may be negative) to memory: as a vector where all of them are the row's, which then starts on
// a boundary, and one by one at its ends
template <typename T, bool ALIGNED>
__device__ __forceinline__ void emb_store(typename Elem<T>::store_t* row, int64_t c, uint32_t dim, const RawVec<T, emb_vec<T>()>& r) {
  constexpr int VEC = emb_vec<T>();
  if constexpr (ALIGNED) r.store_stream(row + c);
  else if (c >= 0 && c + VEC <= (int64_t)dim) r.store_stream(row + c);
  else emb_store_some<T>(row + c, r, (int)max((int64_t)0, -c), (int)min((int64_t)VEC, (int64_t)dim - c));
}

// A row that starts `off` elements behind a vector boundary (-1: take no notice of boundaries), from the vectors at multiples of VEC columns that neighbouring lanes hold:
// each lane stores the aligned vector that ends in its own, the first and the last lane their ends one by one.  `active`: lanes of
// the warp that hold a vector (all of its lanes take part where off is not 0).  Not inlined: five copies of it in the sum kernel's loop
// did not fit the instruction cache.
template <typename T>
__device__ __noinline__ void emb_store_row(typename Elem<T>::store_t* row, uint32_t col, uint32_t dim, int off, uint4 v, int active) {
  constexpr int VEC = emb_vec<T>();
  RawVec<T, VEC> r;
  r.w[0] = v.x; r.w[1] = v.y; r.w[2] = v.z; r.w[3] = v.w;
  const int mine = min(VEC, (int)(dim - col));
  if (off <= 0) {
    if (off == 0 && mine == VEC) r.store_stream(row + col);
    else emb_store_some<T>(row + col, r, 0, mine);
    return;
  }
  const uint32_t mask = active == 32 ? 0xffffffffu : (1u << active) - 1u;
  const int lane = threadIdx.x & 31;
  uint32_t w[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) { w[j] = __shfl_up_sync(mask, r.w[j], 1); w[4 + j] = r.w[j]; }
  if (lane > 0 && mine >= VEC - off) {
    RawVec<T, VEC> out;
    shift_vector<T, VEC>(out, w, VEC - off);
    out.store_stream(row + col - off);
  } else {
    if (lane > 0) {                       // the row ends inside this vector: the neighbour's end, then this lane's
      RawVec<T, VEC> before;
#pragma unroll
      for (int j = 0; j < 4; ++j) before.w[j] = w[j];
      emb_store_some<T>(row + col - VEC, before, VEC - off, VEC);
    }
    emb_store_some<T>(row + col, r, 0, min(mine, VEC - off));
  }
  if (lane == active - 1) emb_store_some<T>(row + col, r, VEC - off, mine);
}

template <typename T, typename ID, bool ALIGNED>
__global__ void __launch_bounds__(EMB_THREADS)
embedding_kernel(const ID* __restrict__ ids, const typename Elem<T>::store_t* __restrict__ table, typename Elem<T>::store_t* __restrict__ out,
                 uint32_t tokens, uint64_t vocab, uint32_t dim, uint32_t packs, int log_tpt, uint64_t ld_table, uint64_t ld_out, float scale, int rn) {
  constexpr int VEC = emb_vec<T>();
  const uint32_t tpt = 1u << log_tpt, group = threadIdx.x >> log_tpt, groups = EMB_THREADS >> log_tpt;
  const uint32_t pack = blockIdx.y * tpt + (threadIdx.x & (tpt - 1));
  pdl_trigger();
  pdl_wait();
  if (pack >= packs) return;
  const uint64_t first = (uint64_t)blockIdx.x * groups * EMB_TOKENS + group;
  // the first column of this thread's vector: vectors are aligned to the row written
  auto col = [&](uint64_t i) { return (int64_t)pack * VEC - (ALIGNED ? 0 : (int64_t)(i * ld_out % VEC)); };
  int64_t id[EMB_TOKENS];
#pragma unroll
  for (int u = 0; u < EMB_TOKENS; ++u) {
    const uint64_t i = first + (uint64_t)u * groups;
    id[u] = i < tokens ? id_at(ids, i) : -1;
  }
  std::conditional_t<ALIGNED, RawVec<T, VEC>, Shifted<T, VEC>> from[EMB_TOKENS];
#pragma unroll
  for (int u = 0; u < EMB_TOKENS; ++u) {
    from[u].zero();
    if (id[u] >= 0 && (uint64_t)id[u] < vocab) {
      if constexpr (ALIGNED) from[u].load(table + (uint64_t)id[u] * ld_table + (uint64_t)pack * VEC);
      else from[u].load(table, id[u] * (int64_t)ld_table + col(first + (uint64_t)u * groups), (vocab - 1) * ld_table + dim);
    }
  }
#pragma unroll
  for (int u = 0; u < EMB_TOKENS; ++u) {
    const uint64_t i = first + (uint64_t)u * groups;
    if (i >= tokens || col(i) >= (int64_t)dim) continue;
    RawVec<T, VEC> r;
    if constexpr (ALIGNED) r = from[u];
    else from[u].get(r);
    if (scale != 1.0f) {
      float v[VEC];
      r.decode(v);
#pragma unroll
      for (int k = 0; k < VEC; ++k) v[k] *= scale;
      round_encode<T, VEC>(r, v, rn != 0);
    }
    emb_store<T, ALIGNED>(out + i * ld_out, col(i), dim, r);
  }
}

// ---- the sorted order ---------------------------------------------------------------------------------------------------------
// token: its number below 2^24, FIRST on the first of a run (a table row's tokens), SHARED on all of a run longer than two chunks
struct SortedToken { uint32_t row, token; };
constexpr uint32_t FIRST = 1u << 31, SHARED = 1u << 30, TOKEN = (1u << 24) - 1;

// four token numbers from position i on; -1 behind the last and for those that 32 bits do not hold; i is a multiple of 4
template <typename ID> __device__ __forceinline__ void load4(const ID* ids, uint32_t i, uint32_t n, int (&v)[4]) {
  if (i + 4 <= n) {
    if constexpr (sizeof(ID) == 4) {
      const int4 q = *reinterpret_cast<const int4*>(ids + i);
      v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
      const longlong2 a = *reinterpret_cast<const longlong2*>(ids + i), b = *reinterpret_cast<const longlong2*>(ids + i + 2);
      const long long w[4] = {a.x, a.y, b.x, b.y};
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = (uint64_t)w[j] <= 0x7fffffffull ? (int)w[j] : -1;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = i + j < n && (sizeof(ID) == 4 || (uint64_t)ids[i + j] <= 0x7fffffffull) ? (int)ids[i + j] : -1;
  }
}

template <typename ID>
__global__ void __launch_bounds__(IDX_THREADS)
embedding_index_kernel(const ID* __restrict__ ids, uint32_t n, uint32_t vocab, uint32_t range, uint32_t long_run, SortedToken* __restrict__ sorted, uint32_t* __restrict__ starts) {
  extern __shared__ uint32_t hist[];              // [warp][row of the range]: counts, then the next free place
  __shared__ uint32_t first[IDX_MAX_ROWS], shared_run[IDX_MAX_ROWS / 32], warp_sum[IDX_WARPS], below_sum[IDX_WARPS];
  pdl_trigger();
  const uint32_t lo = blockIdx.x * range, rows = min(range, vocab - lo);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t* mine = hist + warp * range;
  for (uint32_t i = threadIdx.x; i < IDX_WARPS * range; i += IDX_THREADS) hist[i] = 0;
  pdl_wait();
  __syncthreads();
  // each warp owns one slice of the tokens, in both passes
  constexpr uint32_t STEP = 128 * IDX_BATCH;
  const uint32_t slice = ((n + IDX_WARPS - 1) / IDX_WARPS + 127) / 128 * 128;
  const uint32_t begin = min(n, warp * slice), end = min(n, begin + slice);
  int v[IDX_BATCH][4];
  uint32_t held = 0xffffffffu;                    // where v begins
  auto fetch = [&](uint32_t i0) {
    if (held == i0) return;                       // up to 16384 tokens: the second pass finds the first one's still there
    held = i0;
#pragma unroll
    for (int q = 0; q < IDX_BATCH; ++q) load4(ids, i0 + q * 128 + lane * 4, end, v[q]);
  };
  uint32_t below = 0;
  for (uint32_t i0 = begin; i0 < end; i0 += STEP) {
    fetch(i0);
#pragma unroll
    for (int q = 0; q < IDX_BATCH; ++q)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t r = (uint32_t)v[q][j] - lo;             // a negative number is far above any range
        if (r < rows) atomicAdd(&mine[r], 1u);
        else below += (uint32_t)v[q][j] < lo;
      }
  }
  below = warp_reduce(below, OpSum());
  if (lane == 0) below_sum[warp] = below;
  __syncthreads();
  // exclusive scan over (row, warp), a row per thread
  uint32_t total = 0, at = 0;
  if (threadIdx.x < rows) {
#pragma unroll 8
    for (int w = 0; w < IDX_WARPS; ++w) total += hist[w * range + threadIdx.x];
  }
  uint32_t s = total;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += up;
  }
  if (lane == 31) warp_sum[warp] = s;
  const uint32_t longs = __ballot_sync(0xffffffffu, total > long_run);
  if (lane == 0) shared_run[warp] = longs;
  __syncthreads();
  at = warp_reduce(below_sum[lane] + (lane < warp ? warp_sum[lane] : 0u), OpSum()) + s - total;
  if (threadIdx.x < rows) {
    starts[lo + threadIdx.x] = at;
    first[threadIdx.x] = at;
    uint32_t run = at;
#pragma unroll 8
    for (int w = 0; w < IDX_WARPS; ++w) { const uint32_t c = hist[w * range + threadIdx.x]; hist[w * range + threadIdx.x] = run; run += c; }
    if (lo + threadIdx.x == vocab - 1) starts[vocab] = run;
  }
  __syncthreads();
  // second pass: equal rows of a warp's 32 lanes take consecutive places
  for (uint32_t i0 = begin; i0 < end; i0 += STEP) {
    fetch(i0);
#pragma unroll
    for (int q = 0; q < IDX_BATCH; ++q)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t r = (uint32_t)v[q][j] - lo;
        const bool in = r < rows;
        const uint32_t active = __ballot_sync(0xffffffffu, in);
        if (active == 0) continue;
        if (in) {
          const uint32_t same = __match_any_sync(active, r), rank = __popc(same & ((1u << lane) - 1u));
          const uint32_t place = mine[r];
          uint32_t token = i0 + q * 128 + lane * 4 + j;
          if (place + rank == first[r]) token |= FIRST;
          if (shared_run[r >> 5] >> (r & 31) & 1u) token |= SHARED;
          sorted[place + rank] = SortedToken{lo + r, token};
          __syncwarp(active);
          if (rank == 0) mine[r] = place + __popc(same);
        }
        __syncwarp();
      }
  }
}

// ---- sums over the sorted order -------------------------------------------------------------------------------------------------
struct EmbGradParams {
  const SortedToken* sorted;
  const uint32_t* starts;      // [vocab + 1]
  float* partial;              // [chunk][2][dim]: 0 the shared run that came in from the chunk before, 1 the one that begins here
  uint32_t tokens, vocab, dim, packs, chunk, chunks, sum_ctas;
  uint64_t ld_table, ld_out;
  float scale;
  int accumulate, rn;
};

// scale * acc (+ what the row held), rounded
template <typename T, int VEC>
__device__ __forceinline__ void emb_finish(RawVec<T, VEC>& r, float (&acc)[VEC], const RawVec<T, VEC>& held, const EmbGradParams& p) {
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] *= p.scale;
  if (p.accumulate) {
    float old[VEC];
    held.decode(old);
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] += old[k];
  }
  round_encode<T, VEC>(r, acc, p.rn != 0);
}

template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(EMB_THREADS, ALIGNED ? 4 : 3)
embedding_sum_kernel(const typename Elem<T>::store_t* __restrict__ dout, typename Elem<T>::store_t* dtable, const EmbGradParams p, int log_tpt) {
  constexpr int VEC = emb_vec<T>(), U = 4;                    // rows in flight per thread; four CTAs per SM (three where a row is two vectors)
  const uint32_t tpt = 1u << log_tpt, groups = EMB_THREADS >> log_tpt, group = threadIdx.x >> log_tpt;
  const uint32_t pack = blockIdx.y * tpt + (threadIdx.x & (tpt - 1));
  const uint32_t col = pack * VEC;
  pdl_trigger();
  pdl_wait();
  if (pack >= p.packs) return;
  if (blockIdx.x >= p.sum_ctas) {         // rows that no token names
    const uint32_t r0 = (blockIdx.x - p.sum_ctas) * FILL_ROWS;
    RawVec<T, VEC> z;
    z.zero();
#pragma unroll 4
    for (uint32_t r = r0 + group; r < min(p.vocab, r0 + FILL_ROWS); r += groups)
      if (p.starts[r] == p.starts[r + 1]) {
        auto* row = dtable + (uint64_t)r * p.ld_table;
        const int off = ALIGNED ? 0 : (int)((uint64_t)r * p.ld_table % VEC);
        if (ALIGNED || (int64_t)col - off < (int64_t)p.dim) emb_store<T, ALIGNED>(row, (int64_t)col - off, p.dim, z);
        if (!ALIGNED && pack + 1 == p.packs && (int64_t)col + VEC - off < (int64_t)p.dim) emb_store<T, false>(row, (int64_t)col + VEC - off, p.dim, z);
      }
    return;
  }
  const uint32_t c = blockIdx.x * groups + group;
  const uint32_t n = p.starts[p.vocab];
  const uint64_t begin64 = (uint64_t)c * p.chunk;
  if (begin64 >= n) return;
  const uint32_t begin = (uint32_t)begin64, end = (uint32_t)min((uint64_t)n, begin64 + p.chunk);
  // runs that begin here are taken whole, unless they are shared; one that came in is taken only if it is shared
  const SortedToken head = p.sorted[begin], tail = p.sorted[end - 1];
  const uint32_t lo = head.token & (FIRST | SHARED) ? begin : p.starts[head.row + 1];
  const uint32_t hi = tail.token & SHARED ? end : p.starts[tail.row + 1];
  if (lo >= hi) return;
  // entries behind the row (the last vector of an odd width) are summed with the others and not stored
  const uint64_t dout_end = ((uint64_t)p.tokens - 1) * p.ld_out + p.dim, table_end = ((uint64_t)p.vocab - 1) * p.ld_table + p.dim;
  using Loaded = std::conditional_t<ALIGNED, RawVec<T, VEC>, Shifted<T, VEC>>;
  auto fetch = [&](Loaded& r, const typename Elem<T>::store_t* from, uint64_t at, uint64_t last) {
    if constexpr (ALIGNED) r.load_stream(from + at);
    else r.load(from, (int64_t)at, last);
  };
  auto vector = [&](const Loaded& l) {
    RawVec<T, VEC> r;
    if constexpr (ALIGNED) r = l;
    else l.get(r);
    return r;
  };
  const int active = (int)min(32u, p.packs - (pack & ~31u));      // lanes of this warp that hold a vector (one group per warp)
  float acc[VEC];
  uint32_t row = 0, slot = (head.token & FIRST) || lo != begin ? 1 : 0;
  bool shared = false;
  Loaded held;                            // accumulate: the row as it was, loaded when its run begins
  held.zero();
  auto flush = [&] {
    if (shared) {
      float* part = p.partial + ((uint64_t)c * 2 + slot) * p.dim + col;
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        if (ALIGNED || col + k < p.dim) part[k] = acc[k];
    } else {
      RawVec<T, VEC> r;
      emb_finish<T, VEC>(r, acc, vector(held), p);
      auto* to = dtable + (uint64_t)row * p.ld_table;
      if (ALIGNED) r.store_stream(to + col);
      else if (log_tpt >= 5) emb_store_row<T>(to, col, p.dim, (int)((uint64_t)row * p.ld_table % VEC), make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]), active);
      else emb_store_row<T>(to, col, p.dim, -1, make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]), 0);       // several runs in a warp
    }
    slot = 1;
  };
  SortedToken s[U];
#pragma unroll
  for (int u = 0; u < U; ++u) s[u] = p.sorted[min(lo + u, hi - 1)];
  for (uint32_t i = lo; i < hi; i += U) {
    Loaded r[U];
    SortedToken next[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u < hi) fetch(r[u], dout, (uint64_t)(s[u].token & TOKEN) * p.ld_out + col, dout_end);
#pragma unroll
    for (int u = 0; u < U; ++u) next[u] = p.sorted[min(i + U + u, hi - 1)];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u < hi) {
        float v[VEC];
        vector(r[u]).decode(v);
        const bool starts_run = (s[u].token & FIRST) || i + u == lo;
        if (starts_run) {
          if (i + u != lo) flush();
          row = s[u].row;
          shared = s[u].token & SHARED;
          if (p.accumulate && !shared) fetch(held, dtable, (uint64_t)row * p.ld_table + col, table_end);
        }
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] = starts_run ? v[k] : acc[k] + v[k];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) s[u] = next[u];
  }
  flush();
}

// CTA: eight chunks x 128 columns.  Each warp looks whether a shared run begins in one of them; each run found is added by all warps,
// which take consecutive shares of its partials.
template <typename T>
__global__ void __launch_bounds__(CMB_WARPS * 32)
embedding_combine_kernel(typename Elem<T>::store_t* dtable, const EmbGradParams p) {
  __shared__ uint32_t found[CMB_WARPS][3];           // row, first chunk, last chunk
  __shared__ float part[CMB_WARPS][CMB_COLS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  const uint32_t c = blockIdx.x * CMB_WARPS + warp;
  const uint64_t begin = (uint64_t)c * p.chunk, end = begin + p.chunk;
  if (lane == 0) {
    found[warp][2] = 0;
    if (end < p.tokens) {
      const SortedToken s = p.sorted[end - 1];       // behind the n named ones (not every token names a row) it holds nothing
      const uint32_t n = p.starts[p.vocab];
      if (end < n && (s.token & SHARED)) {
        const uint32_t r0 = p.starts[s.row], r1 = p.starts[s.row + 1];
        if (r0 >= begin) { found[warp][0] = s.row; found[warp][1] = c; found[warp][2] = (r1 - 1) / p.chunk; }
      }
    }
  }
  __syncthreads();
  for (int q = 0; q < CMB_WARPS; ++q) {
    if (found[q][2] == 0) continue;                  // a shared run ends behind its first chunk
    const uint32_t row = found[q][0], c0 = found[q][1], count = found[q][2] - c0 + 1, per = (count + CMB_WARPS - 1) / CMB_WARPS;
    const uint32_t k0 = min(count, warp * per), k1 = min(count, k0 + per);
    const uint32_t col0 = blockIdx.y * CMB_COLS + lane;
    float sum[CMB_COLS / 32] = {};
#pragma unroll 4
    for (uint32_t k = k0; k < k1; ++k) {
      const float* from = p.partial + ((uint64_t)(c0 + k) * 2 + (k == 0 ? 1 : 0)) * p.dim + col0;
#pragma unroll
      for (int h = 0; h < CMB_COLS / 32; ++h)
        if (col0 + h * 32 < p.dim) sum[h] += from[h * 32];
    }
#pragma unroll
    for (int h = 0; h < CMB_COLS / 32; ++h) part[warp][h * 32 + lane] = sum[h];
    __syncthreads();
    const uint32_t col = blockIdx.y * CMB_COLS + threadIdx.x;
    if (threadIdx.x < CMB_COLS && col < p.dim) {
      float acc[1] = {0.0f};
#pragma unroll
      for (int w = 0; w < CMB_WARPS; ++w) acc[0] += part[w][threadIdx.x];
      auto* dst = dtable + (uint64_t)row * p.ld_table + col;
      RawVec<T, 1> held, r;
      held.zero();
      if (p.accumulate) held.load(dst);
      emb_finish<T, 1>(r, acc, held, p);
      r.store(dst);
    }
    __syncthreads();
  }
}

// whether every row of both matrices starts on a vector boundary and ends on one
bool emb_aligned(const zyxb_embedding_desc& d, uint64_t ld_table, uint64_t ld_out) {
  return ((d.dim | ld_table | ld_out) * dtype_size(d.dtype)) % 16 == 0;
}
uint32_t emb_packs(const zyxb_embedding_desc& d) {
  const uint64_t vec = 16 / dtype_size(d.dtype);
  return (uint32_t)((d.dim + vec - 1) / vec);
}

int log2_ceil(uint64_t v, int most) {
  int l = 0;
  while (l < most && (1ull << l) < v) ++l;
  return l;
}

// rows of `ld` elements, the last one `dim` long, inside `bytes`
bool matrix_fits(uint64_t rows, uint64_t ld, uint64_t dim, uint64_t es, uint64_t bytes) {
  return (unsigned __int128)es * ((unsigned __int128)(rows - 1) * ld + dim) <= bytes;
}

template <typename T, typename ID, bool ALIGNED>
cudaError_t run_embedding(const zyxb_embedding_desc& d, uint64_t ldt, uint64_t ldo, float scale, void* const* args, const LaunchCtx& lc) {
  using S = typename Elem<T>::store_t;
  const uint32_t packs = emb_packs(d) + (ALIGNED ? 0 : 1);          // a row of odd start touches one more
  const int log_tpt = log2_ceil(packs, 8);
  const uint64_t per_cta = (uint64_t)(EMB_THREADS >> log_tpt) * EMB_TOKENS;
  const dim3 grid((unsigned)((d.tokens + per_cta - 1) / per_cta), (unsigned)((packs + (1u << log_tpt) - 1) >> log_tpt));
  return launch_pdl(embedding_kernel<T, ID, ALIGNED>, grid, EMB_THREADS, 0, lc.stream, (const ID*)args[0], (const S*)args[1], (S*)args[2], (uint32_t)d.tokens,
                    d.vocab, (uint32_t)d.dim, packs, log_tpt, ldt, ldo, scale, lc.round_nearest ? 1 : 0);
}

struct EmbPlan { uint32_t range, ranges, chunk, chunks; uint64_t starts_off, partial_off; };

template <typename T, typename ID, bool ALIGNED>
cudaError_t run_embedding_bwd(const zyxb_embedding_desc& d, uint64_t ldt, uint64_t ldo, float scale, const EmbPlan& pl, void* const* args, const LaunchCtx& lc) {
  using S = typename Elem<T>::store_t;
  char* scratch = (char*)lc.scratch;
  EmbGradParams p{};
  p.sorted = (const SortedToken*)scratch; p.starts = (const uint32_t*)(scratch + pl.starts_off); p.partial = (float*)(scratch + pl.partial_off);
  p.tokens = (uint32_t)d.tokens; p.vocab = (uint32_t)d.vocab; p.dim = (uint32_t)d.dim; p.packs = emb_packs(d); p.chunk = pl.chunk;
  p.ld_table = ldt; p.ld_out = ldo; p.scale = scale; p.accumulate = d.accumulate ? 1 : 0; p.rn = lc.round_nearest ? 1 : 0;
  p.chunks = pl.chunks;
  static uint64_t configured = 0;
  cudaError_t e = ensure_dynamic_smem(embedding_index_kernel<ID>, IDX_WARPS * IDX_MAX_ROWS * 4, &configured);
  if (e != cudaSuccess) return e;
  e = launch_pdl(embedding_index_kernel<ID>, dim3(pl.ranges), IDX_THREADS, IDX_WARPS * pl.range * 4, lc.stream, (const ID*)args[0], (uint32_t)d.tokens,
                 (uint32_t)d.vocab, pl.range, 2 * pl.chunk, (SortedToken*)scratch, (uint32_t*)(scratch + pl.starts_off));
  if (e != cudaSuccess) return e;
  const int log_tpt = log2_ceil(p.packs, 8);
  const uint32_t groups = EMB_THREADS >> log_tpt;
  p.sum_ctas = (pl.chunks + groups - 1) / groups;
  const unsigned fill = p.accumulate ? 0 : (p.vocab + FILL_ROWS - 1) / FILL_ROWS;
  const dim3 grid(p.sum_ctas + fill, (unsigned)((p.packs + (1u << log_tpt) - 1) >> log_tpt));
  e = launch_pdl(embedding_sum_kernel<T, ALIGNED>, grid, EMB_THREADS, 0, lc.stream, (const S*)args[1], (S*)args[2], p, log_tpt);
  if (e != cudaSuccess || d.tokens <= 2 * pl.chunk) return e;
  return launch_pdl(embedding_combine_kernel<T>, dim3((pl.chunks + CMB_WARPS - 1) / CMB_WARPS, (unsigned)((d.dim + CMB_COLS - 1) / CMB_COLS)), CMB_WARPS * 32, 0,
                    lc.stream, (S*)args[2], p);
}

}  // namespace

int validate_embedding(const zyxb_embedding_desc& d, bool backward, std::string& err) {
  auto bad = [&](const char* m) { err = m; return (int)ZYXB_ERR_KERNEL_COMPILATION; };
  if (d.dtype != ZYXB_F32 && d.dtype != ZYXB_BF16 && d.dtype != ZYXB_F16) return bad("embedding: dtype must be f32, bf16 or f16");
  if (d.id_dtype != ZYXB_I32 && d.id_dtype != ZYXB_I64) return bad("embedding: id_dtype must be i32 or i64");
  if (d.tokens == 0 || d.vocab == 0 || d.dim == 0) return bad("embedding: tokens, vocab and dim must be positive");
  if (d.tokens > 0x7fffffffull || d.vocab > 0x7fffffffull) return bad("embedding: tokens and vocab must be below 2^31");
  if (d.dim > (1ull << 20)) return bad("embedding: dim must be at most 2^20");
  if ((d.ld_table && d.ld_table < d.dim) || (d.ld_out && d.ld_out < d.dim)) return bad("embedding: row pitch smaller than the row");
  if (d.ld_table > (1ull << 40) || d.ld_out > (1ull << 40)) return bad("embedding: row pitch too large");
  if (!backward && d.accumulate) return bad("embedding: accumulate is an option of the gradient");
  if (backward && (d.tokens > (1ull << 24) || d.vocab > (1ull << 24))) return bad("embedding gradient: tokens and vocab must be at most 2^24");
  return ZYXB_OK;
}

#define ZYXB_EMB_ID(T, F)                                                                    \
  if (d.id_dtype == ZYXB_I32) { if (aligned) { F(T, int32_t, true); } else { F(T, int32_t, false); } } \
  else { if (aligned) { F(T, int64_t, true); } else { F(T, int64_t, false); } }
#define ZYXB_EMB_DISPATCH(F)                                                      \
  switch (d.dtype) {                                                              \
    case ZYXB_F32: ZYXB_EMB_ID(float, F) break;                                   \
    case ZYXB_BF16: ZYXB_EMB_ID(bf16_t, F) break;                                 \
    default: ZYXB_EMB_ID(f16_t, F) break;                                         \
  }

int launch_embedding(const zyxb_embedding_desc& d, void* const* args, const uint64_t* arg_bytes, int n_args, const LaunchCtx& lc, std::string& err) {
  ZYXB_CHECK_ARG(n_args == 3, "embedding: expected args ids, table -> out");
  const uint64_t es = dtype_size(d.dtype), ldt = d.ld_table ? d.ld_table : d.dim, ldo = d.ld_out ? d.ld_out : d.dim;
  ZYXB_CHECK_ARG(arg_bytes[0] >= d.tokens * dtype_size(d.id_dtype), "embedding: ids too small");
  ZYXB_CHECK_ARG(matrix_fits(d.vocab, ldt, d.dim, es, arg_bytes[1]), "embedding: table too small");
  ZYXB_CHECK_ARG(matrix_fits(d.tokens, ldo, d.dim, es, arg_bytes[2]), "embedding: out too small");
  ZYXB_CHECK_ARG(args[2] != args[1] && args[2] != args[0], "embedding: out must be a buffer of its own");
  const float scale = d.scale == 0.0f ? 1.0f : d.scale;
  const bool aligned = emb_aligned(d, ldt, ldo);
  cudaError_t e = cudaSuccess;
#define ZYXB_EMB_FWD(T, ID, V) e = run_embedding<T, ID, V>(d, ldt, ldo, scale, args, lc)
  ZYXB_EMB_DISPATCH(ZYXB_EMB_FWD)
#undef ZYXB_EMB_FWD
  if (e != cudaSuccess) { err = std::string("embedding: ") + cudaGetErrorString(e); return ZYXB_ERR_KERNEL_LAUNCH; }
  return check_launch(lc, err, "embedding");
}

int launch_embedding_bwd(const zyxb_embedding_desc& d, void* const* args, const uint64_t* arg_bytes, int n_args, const LaunchCtx& lc, std::string& err) {
  ZYXB_CHECK_ARG(n_args == 3, "embedding gradient: expected args ids, dout -> dtable");
  const uint64_t es = dtype_size(d.dtype), ldt = d.ld_table ? d.ld_table : d.dim, ldo = d.ld_out ? d.ld_out : d.dim;
  ZYXB_CHECK_ARG(arg_bytes[0] >= d.tokens * dtype_size(d.id_dtype), "embedding gradient: ids too small");
  ZYXB_CHECK_ARG(matrix_fits(d.tokens, ldo, d.dim, es, arg_bytes[1]), "embedding gradient: dout too small");
  ZYXB_CHECK_ARG(matrix_fits(d.vocab, ldt, d.dim, es, arg_bytes[2]), "embedding gradient: dtable too small");
  ZYXB_CHECK_ARG(args[2] != args[1] && args[2] != args[0], "embedding gradient: dtable must be a buffer of its own");
  EmbPlan pl{};
  // one range per SM, within what the histograms hold; fewer rows than 32 are not worth another scan of the tokens
  pl.range = (uint32_t)std::min<uint64_t>(IDX_MAX_ROWS, std::max<uint64_t>(32, (d.vocab + lc.sm_count - 1) / lc.sm_count));
  pl.ranges = (uint32_t)((d.vocab + pl.range - 1) / pl.range);
  pl.starts_off = (d.tokens * sizeof(SortedToken) + 255) / 256 * 256;
  pl.partial_off = pl.starts_off + ((d.vocab + 1) * 4 + 255) / 256 * 256;
  // few tokens: shorter chunks, so that every SM has three CTAs' worth of them (4099 tokens of 777 f32: 24 -> 22 us; at 16384 of 2048
  // bf16, which 32 places fill, chunks of 8 cost more partials than they save: 61 -> 68 us)
  const bool aligned = emb_aligned(d, ldt, ldo);
  const uint64_t threads_wide = (emb_packs(d) + 31) / 32 * 32;
  pl.chunk = CHUNK;
  auto chunks = [&] { return (d.tokens + pl.chunk - 1) / pl.chunk; };
  while (pl.chunk > CHUNK_LEAST && chunks() * threads_wide < (uint64_t)lc.sm_count * 3 * EMB_THREADS) pl.chunk /= 2;
  while (chunks() > 1 && pl.partial_off + chunks() * 2 * d.dim * 4 > lc.scratch_bytes) pl.chunk *= 2;     // partials have to fit the scratch
  pl.chunks = (uint32_t)chunks();
  ZYXB_CHECK_ARG(pl.partial_off + (uint64_t)pl.chunks * 2 * d.dim * 4 <= lc.scratch_bytes, "embedding gradient: too large for the scratch memory");
  const float scale = d.scale == 0.0f ? 1.0f : d.scale;
  cudaError_t e = cudaSuccess;
#define ZYXB_EMB_BWD(T, ID, V) e = run_embedding_bwd<T, ID, V>(d, ldt, ldo, scale, pl, args, lc)
  ZYXB_EMB_DISPATCH(ZYXB_EMB_BWD)
#undef ZYXB_EMB_BWD
  if (e != cudaSuccess) { err = std::string("embedding gradient: ") + cudaGetErrorString(e); return ZYXB_ERR_KERNEL_LAUNCH; }
  return check_launch(lc, err, "embedding gradient", d.tokens > 2 * pl.chunk ? 3 : 2);
}

}  // namespace zyxb
