// Embedding lookup and the gradient of its table.
//   out[i,:]    = scale * table[ids[i],:]                      (zeros for an id outside [0, vocab))
//   dtable[v,:] = scale * sum_{i : ids[i] = v} dout[i,:]       (+ dtable[v,:])
//
// Lookup: a copy, bound by HBM.  A group of threads spans one row's 16-byte vectors and moves four tokens at a time.
//
// Gradient, three launches and no floating-point atomic:
//   index    The vocabulary is cut into ranges, one CTA each.  Every CTA scans all token numbers (from L2; 64 KB at 16384 tokens),
//            counts those below its range - which is where its part of the sorted order begins, so no CTA waits for another - and
//            counting-sorts those inside it.  Rows that no token names are written as zeros here.
//   sum      The sorted order is cut into chunks of equal length, whatever the token frequencies: a group of threads adds a chunk's
//            rows in f32 registers, run by run.  A run inside one chunk is stored; a run that crosses a border leaves f32 partials.
//   combine  Adds the partials of each crossing run, in chunk order.
// The order of every sum depends on ids alone.
#include <algorithm>

#include "internal.h"
#include "rounding.cuh"

namespace zyxb {

namespace {

constexpr int EMB_THREADS = 256;
constexpr int EMB_TOKENS = 4;          // rows in flight per thread
constexpr int IDX_THREADS = 512, IDX_WARPS = IDX_THREADS / 32;
constexpr int IDX_MAX_ROWS = 1024;     // rows of a vocabulary range (histograms: 16 warps x 1024 x 4 B of shared memory)
constexpr int CMB_WARPS = 16;

template <typename ID> __device__ __forceinline__ int64_t id_at(const ID* ids, uint64_t i) { return (int64_t)ids[i]; }

template <typename T, typename ID, int VEC>
__global__ void __launch_bounds__(EMB_THREADS)
embedding_kernel(const ID* __restrict__ ids, const typename Elem<T>::store_t* __restrict__ table, typename Elem<T>::store_t* __restrict__ out,
                 uint32_t tokens, uint64_t vocab, uint32_t packs, int log_tpt, uint64_t ld_table, uint64_t ld_out, float scale, int rn) {
  const uint32_t tpt = 1u << log_tpt, group = threadIdx.x >> log_tpt, groups = EMB_THREADS >> log_tpt;
  const uint32_t pack = blockIdx.y * tpt + (threadIdx.x & (tpt - 1));
  if (pack >= packs) return;
  const uint64_t first = (uint64_t)blockIdx.x * groups * EMB_TOKENS + group;
  int64_t id[EMB_TOKENS];
#pragma unroll
  for (int u = 0; u < EMB_TOKENS; ++u) {
    const uint64_t i = first + (uint64_t)u * groups;
    id[u] = i < tokens ? id_at(ids, i) : -1;
  }
  RawVec<T, VEC> r[EMB_TOKENS];
#pragma unroll
  for (int u = 0; u < EMB_TOKENS; ++u) {
    r[u].zero();
    if (id[u] >= 0 && (uint64_t)id[u] < vocab) r[u].load(table + (uint64_t)id[u] * ld_table + (uint64_t)pack * VEC);
  }
#pragma unroll
  for (int u = 0; u < EMB_TOKENS; ++u) {
    const uint64_t i = first + (uint64_t)u * groups;
    if (i >= tokens) continue;
    if (scale != 1.0f) {
      float v[VEC];
      r[u].decode(v);
#pragma unroll
      for (int k = 0; k < VEC; ++k) v[k] *= scale;
      round_encode<T, VEC>(r[u], v, rn != 0);
    }
    r[u].store_stream(out + i * ld_out + (uint64_t)pack * VEC);
  }
}

// ---- the sorted order ---------------------------------------------------------------------------------------------------------
struct SortedToken { uint32_t row, token; };

// four token numbers from position i on, -1 behind the last; i is a multiple of 4
template <typename ID> __device__ __forceinline__ void load4(const ID* ids, uint32_t i, uint32_t n, int64_t (&v)[4]) {
  if (i + 4 <= n) {
    if constexpr (sizeof(ID) == 4) {
      const int4 q = *reinterpret_cast<const int4*>(ids + i);
      v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
      const longlong2 a = *reinterpret_cast<const longlong2*>(ids + i), b = *reinterpret_cast<const longlong2*>(ids + i + 2);
      v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = i + j < n ? (int64_t)ids[i + j] : -1;
  }
}

template <typename T, typename ID, int VEC>
__global__ void __launch_bounds__(IDX_THREADS)
embedding_index_kernel(const ID* __restrict__ ids, uint32_t n, uint32_t vocab, uint32_t range, SortedToken* __restrict__ sorted,
                       uint32_t* __restrict__ starts, typename Elem<T>::store_t* __restrict__ dtable, uint64_t ld, uint32_t packs, int zero_rows) {
  extern __shared__ uint32_t hist[];              // [warp][row of the range]
  __shared__ uint32_t total[IDX_MAX_ROWS], warp_sum[IDX_WARPS], below_sum[IDX_WARPS];
  const uint32_t lo = blockIdx.x * range, rows = min(range, vocab - lo);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t* mine = hist + warp * range;
  for (uint32_t i = threadIdx.x; i < IDX_WARPS * range; i += IDX_THREADS) hist[i] = 0;
  __syncthreads();
  // each warp owns one slice of the tokens, in both passes
  const uint32_t slice = ((n + IDX_WARPS - 1) / IDX_WARPS + 127) / 128 * 128;
  const uint32_t begin = min(n, warp * slice), end = min(n, begin + slice);
  uint32_t below = 0;
#pragma unroll 4
  for (uint32_t i = begin + lane * 4; i < end; i += 128) {
    int64_t v[4];
    load4(ids, i, end, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint64_t r = (uint64_t)v[j] - lo;             // a negative number is far above any range
      if (r < rows) atomicAdd(&mine[r], 1u);
      else below += v[j] >= 0 && v[j] < (int64_t)lo;
    }
  }
  below = warp_reduce(below, OpSum());
  if (lane == 0) below_sum[warp] = below;
  __syncthreads();
  uint32_t base = 0;
#pragma unroll
  for (int w = 0; w < IDX_WARPS; ++w) base += below_sum[w];
  // exclusive scan over (row, warp): two consecutive rows per thread
  uint32_t t[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint32_t r = threadIdx.x * 2 + k;
    t[k] = 0;
    if (r < rows)
      for (int w = 0; w < IDX_WARPS; ++w) t[k] += hist[w * range + r];
    if (r < rows) total[r] = t[k];
  }
  uint32_t s = t[0] + t[1];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += up;
  }
  if (lane == 31) warp_sum[warp] = s;
  __syncthreads();
  uint32_t at = base + s - (t[0] + t[1]);
  for (int w = 0; w < warp; ++w) at += warp_sum[w];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint32_t r = threadIdx.x * 2 + k;
    if (r < rows) {
      starts[lo + r] = at;
      uint32_t run = at;
      for (int w = 0; w < IDX_WARPS; ++w) { const uint32_t c = hist[w * range + r]; hist[w * range + r] = run; run += c; }
      at = run;
      if (lo + r == vocab - 1) starts[vocab] = at;
    }
  }
  __syncthreads();
  // second pass: equal rows of a warp's 32 lanes take consecutive places
#pragma unroll 4
  for (uint32_t i0 = begin; i0 < end; i0 += 128) {
    int64_t v[4];
    const uint32_t i = i0 + lane * 4;
    if (i < end) load4(ids, i, end, v);
    else { v[0] = v[1] = v[2] = v[3] = -1; }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint64_t r = (uint64_t)v[j] - lo;             // a negative number is far above any range
      const bool in = r < rows;
      const uint32_t active = __ballot_sync(0xffffffffu, in);
      if (active == 0) continue;
      if (in) {
        const uint32_t same = __match_any_sync(active, (uint32_t)r);
        const uint32_t rank = __popc(same & ((1u << lane) - 1u));
        const uint32_t place = mine[r];
        sorted[place + rank] = SortedToken{lo + (uint32_t)r, i + j};
        __syncwarp(active);
        if (rank == 0) mine[r] = place + __popc(same);
      }
      __syncwarp();
    }
  }
  if (zero_rows) {
    RawVec<T, VEC> z;
    z.zero();
    for (uint32_t r = warp; r < rows; r += IDX_WARPS) {
      if (total[r] != 0) continue;
      auto* row = dtable + (uint64_t)(lo + r) * ld;
      for (uint32_t k = lane; k < packs; k += 32) z.store_stream(row + (uint64_t)k * VEC);
    }
  }
}

// ---- sums over the sorted order -------------------------------------------------------------------------------------------------
struct EmbGradParams {
  const SortedToken* sorted;
  const uint32_t* starts;      // [vocab + 1]
  float* partial;              // [chunk][2][dim]: 0 the run that came in from the chunk before, 1 the one that begins here and goes on
  uint32_t vocab, dim, packs, chunk;
  uint64_t ld_table, ld_out;
  float scale;
  int accumulate, rn;
};

template <typename T, int VEC>
__device__ __forceinline__ void emb_store_row(typename Elem<T>::store_t* dst, float (&acc)[VEC], const EmbGradParams& p) {
  RawVec<T, VEC> r;
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] *= p.scale;
  if (p.accumulate) {
    float old[VEC];
    r.load(dst);
    r.decode(old);
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] += old[k];
  }
  round_encode<T, VEC>(r, acc, p.rn != 0);
  r.store_stream(dst);
}

template <typename T, int VEC>
__global__ void __launch_bounds__(EMB_THREADS)
embedding_sum_kernel(const typename Elem<T>::store_t* __restrict__ dout, typename Elem<T>::store_t* dtable, EmbGradParams p, int log_tpt) {
  constexpr int U = 8;
  const uint32_t tpt = 1u << log_tpt, groups = EMB_THREADS >> log_tpt;
  const uint32_t c = blockIdx.x * groups + (threadIdx.x >> log_tpt);
  const uint32_t pack = blockIdx.y * tpt + (threadIdx.x & (tpt - 1));
  const uint32_t n = p.starts[p.vocab];
  const uint64_t begin64 = (uint64_t)c * p.chunk;
  if (begin64 >= n || pack >= p.packs) return;
  const uint32_t begin = (uint32_t)begin64, end = (uint32_t)min((uint64_t)n, begin64 + p.chunk);
  const uint64_t col = (uint64_t)pack * VEC;
  float acc[VEC];
  uint32_t row = 0xffffffffu;
  auto flush = [&](uint32_t stop) {       // the run of `row` ends at `stop` (its end, or the chunk's)
    float* part = p.partial + (uint64_t)c * 2 * p.dim + col;
    const bool came_in = p.starts[row] < begin, goes_on = stop == end && p.starts[row + 1] > end;
    if (came_in) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) part[k] = acc[k];
    } else if (goes_on) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) part[p.dim + k] = acc[k];
    } else {
      emb_store_row<T, VEC>(dtable + (uint64_t)row * p.ld_table + col, acc, p);
    }
  };
  for (uint32_t i = begin; i < end; i += U) {
    SortedToken s[U];
    RawVec<T, VEC> r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) s[u] = i + u < end ? p.sorted[i + u] : SortedToken{0xffffffffu, 0};
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u < end) r[u].load_stream(dout + (uint64_t)s[u].token * p.ld_out + col);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u >= end) break;
      float v[VEC];
      r[u].decode(v);
      if (s[u].row != row) {
        if (row != 0xffffffffu) flush(i + u);
        row = s[u].row;
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] = v[k];
      } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] += v[k];
      }
    }
  }
  flush(end);
}

// One warp per 32 columns and share of the partials; the CTA's warps split each crossing run's list.
template <typename T>
__global__ void __launch_bounds__(CMB_WARPS * 32)
embedding_combine_kernel(typename Elem<T>::store_t* dtable, EmbGradParams p, uint32_t chunks) {
  __shared__ uint32_t list[CMB_WARPS * 32];
  __shared__ uint32_t found;
  __shared__ float part[CMB_WARPS][32];
  const uint32_t n = p.starts[p.vocab];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t col = blockIdx.x * 32 + lane;
  // the chunks this CTA looks at: y, y + Y, ...; those whose last run begins in them and goes on are listed, in order
  for (uint32_t t0 = blockIdx.y; t0 < chunks; t0 += gridDim.y * (CMB_WARPS * 32)) {
    const uint64_t c = t0 + (uint64_t)threadIdx.x * gridDim.y, begin = c * p.chunk, end = begin + p.chunk;
    bool crosses = false;
    if (c < chunks && end < n) {
      const uint32_t row = p.sorted[end - 1].row;
      crosses = p.starts[row] >= begin && p.starts[row + 1] > end;
    }
    const uint32_t ballot = __ballot_sync(0xffffffffu, crosses);
    __shared__ uint32_t warp_count[CMB_WARPS];
    if (lane == 0) warp_count[warp] = __popc(ballot);
    __syncthreads();
    uint32_t at = __popc(ballot & ((1u << lane) - 1u));
    for (int w = 0; w < warp; ++w) at += warp_count[w];
    if (crosses) list[at] = (uint32_t)c;
    if (threadIdx.x == CMB_WARPS * 32 - 1) found = at + (crosses ? 1 : 0);
    __syncthreads();
    const uint32_t m = found;
    for (uint32_t q = 0; q < m; ++q) {
      const uint32_t c0 = list[q];
      const uint32_t row = p.sorted[(uint64_t)c0 * p.chunk + p.chunk - 1].row;
      const uint32_t last = (p.starts[row + 1] - 1) / p.chunk, count = last - c0;       // partials behind the first chunk's
      const uint32_t per = (count + CMB_WARPS - 1) / CMB_WARPS;
      float sum = 0.0f;
      if (col < p.dim) {
        if (warp == 0) sum = p.partial[((uint64_t)c0 * 2 + 1) * p.dim + col];
        const uint32_t k0 = min(count, warp * per), k1 = min(count, k0 + per);
#pragma unroll 8
        for (uint32_t k = k0; k < k1; ++k) sum += p.partial[(uint64_t)(c0 + 1 + k) * 2 * p.dim + col];
      }
      part[warp][lane] = sum;
      __syncthreads();
      if (warp == 0 && col < p.dim) {
        float acc[1] = {0.0f};
#pragma unroll
        for (int w = 0; w < CMB_WARPS; ++w) acc[0] += part[w][lane];
        emb_store_row<T, 1>(dtable + (uint64_t)row * p.ld_table + col, acc, p);
      }
      __syncthreads();
    }
    __syncthreads();
  }
}

// the widest vector (in elements) that every row of both matrices can be cut into
uint32_t emb_vec(const zyxb_embedding_desc& d, uint64_t ld_table, uint64_t ld_out) {
  const uint64_t all = d.dim | ld_table | ld_out;
  uint32_t v = (uint32_t)(16 / dtype_size(d.dtype));
  while (v > 1 && all % v) v >>= 1;
  return v;
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

template <typename T, typename ID, int VEC>
void run_embedding(const zyxb_embedding_desc& d, uint64_t ldt, uint64_t ldo, float scale, void* const* args, const LaunchCtx& lc) {
  using S = typename Elem<T>::store_t;
  const uint32_t packs = (uint32_t)(d.dim / VEC);
  const int log_tpt = log2_ceil(packs, 8);
  const uint64_t per_cta = (uint64_t)(EMB_THREADS >> log_tpt) * EMB_TOKENS;
  const dim3 grid((unsigned)((d.tokens + per_cta - 1) / per_cta), (unsigned)((packs + (1u << log_tpt) - 1) >> log_tpt));
  embedding_kernel<T, ID, VEC><<<grid, EMB_THREADS, 0, lc.stream>>>((const ID*)args[0], (const S*)args[1], (S*)args[2], (uint32_t)d.tokens,
                                                                   d.vocab, packs, log_tpt, ldt, ldo, scale, lc.round_nearest ? 1 : 0);
}

struct EmbPlan { uint32_t range, ranges, chunk, chunks; uint64_t starts_off, partial_off; };

template <typename T, typename ID, int VEC>
cudaError_t run_embedding_bwd(const zyxb_embedding_desc& d, uint64_t ldt, uint64_t ldo, float scale, const EmbPlan& pl, void* const* args, const LaunchCtx& lc) {
  using S = typename Elem<T>::store_t;
  char* scratch = (char*)lc.scratch;
  EmbGradParams p{};
  p.sorted = (const SortedToken*)scratch; p.starts = (const uint32_t*)(scratch + pl.starts_off); p.partial = (float*)(scratch + pl.partial_off);
  p.vocab = (uint32_t)d.vocab; p.dim = (uint32_t)d.dim; p.packs = (uint32_t)(d.dim / VEC); p.chunk = pl.chunk;
  p.ld_table = ldt; p.ld_out = ldo; p.scale = scale; p.accumulate = d.accumulate ? 1 : 0; p.rn = lc.round_nearest ? 1 : 0;
  const int smem = (int)(IDX_WARPS * pl.range * 4);
  static uint64_t configured = 0;
  cudaError_t e = ensure_dynamic_smem(embedding_index_kernel<T, ID, VEC>, IDX_WARPS * IDX_MAX_ROWS * 4, &configured);
  if (e != cudaSuccess) return e;
  embedding_index_kernel<T, ID, VEC><<<pl.ranges, IDX_THREADS, smem, lc.stream>>>((const ID*)args[0], (uint32_t)d.tokens, (uint32_t)d.vocab, pl.range,
                                                                                (SortedToken*)scratch, (uint32_t*)(scratch + pl.starts_off), (S*)args[2],
                                                                                ldt, p.packs, p.accumulate ? 0 : 1);
  const int log_tpt = log2_ceil(p.packs, 8);
  const uint32_t groups = EMB_THREADS >> log_tpt;
  const dim3 grid((pl.chunks + groups - 1) / groups, (unsigned)((p.packs + (1u << log_tpt) - 1) >> log_tpt));
  embedding_sum_kernel<T, VEC><<<grid, EMB_THREADS, 0, lc.stream>>>((const S*)args[1], (S*)args[2], p, log_tpt);
  if (pl.chunks > 1) {
    const unsigned slabs = (unsigned)((d.dim + 31) / 32);
    const unsigned ys = std::max(1u, std::min(pl.chunks, 592u / slabs));
    embedding_combine_kernel<T><<<dim3(slabs, ys), CMB_WARPS * 32, 0, lc.stream>>>((S*)args[2], p, pl.chunks);
  }
  return cudaSuccess;
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

#define ZYXB_EMB_VEC(T, ID, F)                                                    \
  switch (vec) {                                                                  \
    case 8: if constexpr (sizeof(typename Elem<T>::store_t) == 2) { F(T, ID, 8); } break; \
    case 4: F(T, ID, 4); break;                                                   \
    case 2: F(T, ID, 2); break;                                                   \
    default: F(T, ID, 1); break;                                                  \
  }
#define ZYXB_EMB_ID(T, F)                                                         \
  if (d.id_dtype == ZYXB_I32) { ZYXB_EMB_VEC(T, int32_t, F) } else { ZYXB_EMB_VEC(T, int64_t, F) }
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
  const uint32_t vec = emb_vec(d, ldt, ldo);
#define ZYXB_EMB_FWD(T, ID, V) run_embedding<T, ID, V>(d, ldt, ldo, scale, args, lc)
  ZYXB_EMB_DISPATCH(ZYXB_EMB_FWD)
#undef ZYXB_EMB_FWD
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
  pl.chunk = 32;
  auto chunks = [&] { return (d.tokens + pl.chunk - 1) / pl.chunk; };
  while (chunks() > 1 && pl.partial_off + chunks() * 2 * d.dim * 4 > lc.scratch_bytes) pl.chunk *= 2;     // partials have to fit the scratch
  pl.chunks = (uint32_t)chunks();
  ZYXB_CHECK_ARG(pl.partial_off + (uint64_t)pl.chunks * 2 * d.dim * 4 <= lc.scratch_bytes, "embedding gradient: too large for the scratch memory");
  const float scale = d.scale == 0.0f ? 1.0f : d.scale;
  const uint32_t vec = emb_vec(d, ldt, ldo);
  cudaError_t e = cudaSuccess;
#define ZYXB_EMB_BWD(T, ID, V) e = run_embedding_bwd<T, ID, V>(d, ldt, ldo, scale, pl, args, lc)
  ZYXB_EMB_DISPATCH(ZYXB_EMB_BWD)
#undef ZYXB_EMB_BWD
  if (e != cudaSuccess) { err = std::string("embedding gradient: ") + cudaGetErrorString(e); return ZYXB_ERR_KERNEL_LAUNCH; }
  return check_launch(lc, err, "embedding gradient", pl.chunks > 1 ? 3 : 2);
}

}  // namespace zyxb
