// Muon: momentum, then the update made nearly orthogonal by Newton-Schulz products, then the weight's step.
//   momentum   buf = momentum * buf + g, and the sum of squares of the direction (f64)
//   normalize  X = direction / (norm + eps) as f16 parts, transposed where rows > cols: the products see rows <= cols
//   products   three per step (muon_gemm.cuh)
//   step       p = p (1 - lr wd) - lr adjust X
// Matrices of equal extents (or transposes of each other) go through every launch together.
#include <algorithm>
#include <cmath>
#include <vector>

#include "muon_gemm.cuh"
#include "muon_small.cuh"
#include "rounding.cuh"

namespace zyxb {

namespace {

constexpr uint64_t MUON_MAX_EXTENT = 32768;
constexpr int MUON_THREADS = 256, MUON_PARTIALS = 512, MUON_TABLE = 32, TILE = 64, NORM_CTAS = 8;      // NORM_CTAS: per SM
constexpr uint64_t MUON_GROUP_BYTES = 1ull << 30;      // matrices that go together: their operands stay below this, or go alone

struct MuonMatrix { void* p; const void* g; void* buf; uint32_t tall; };
struct MuonGroup {
  MuonMatrix m[MUON_TABLE];
  uint32_t lo, hi;                // extents of the products' X: lo <= hi
  float momentum, grad_scale;
  int nesterov, rn;
};

// the direction that is made orthogonal, from the stored momentum
__device__ __forceinline__ float muon_direction(float g, float buf, const MuonGroup& k) { return k.nesterov ? g + k.momentum * buf : buf; }

// Sum of squares in 64 bits: a gradient's square leaves f32 at 1e19 and 1e-23.
template <typename T>
__global__ void __launch_bounds__(MUON_THREADS) muon_momentum_kernel(const __grid_constant__ MuonGroup k, double* __restrict__ partial) {
  using S = typename Elem<T>::store_t;
  constexpr int VEC = 16 / (int)sizeof(S);
  __shared__ double part[MUON_THREADS / 32];
  pdl_trigger();
  pdl_wait();
  const MuonMatrix& m = k.m[blockIdx.y];
  const uint64_t n = (uint64_t)k.lo * k.hi, vectors = n / VEC;
  const S* g = (const S*)m.g;
  S* b = (S*)m.buf;
  double sum = 0.0;
  auto one = [&](float gv, float bv, float& stored) {     // -> the momentum to store; adds the direction's square
    gv *= k.grad_scale;
    float u = gv;
    if (b) {
      const S s = round_store<T>(k.momentum * bv + gv, k.rn != 0);
      stored = Elem<T>::load(s);
      u = muon_direction(gv, stored, k);
    }
    sum += (double)u * (double)u;
  };
  for (uint64_t i = (uint64_t)blockIdx.x * MUON_THREADS + threadIdx.x; i < vectors; i += (uint64_t)gridDim.x * MUON_THREADS) {
    RawVec<T, VEC> rg, rb;
    rg.load(g + i * VEC);
    if (b) rb.load(b + i * VEC); else rb.zero();
    float fg[VEC], fb[VEC];
    rg.decode(fg);
    rb.decode(fb);
#pragma unroll
    for (int j = 0; j < VEC; ++j) one(fg[j], fb[j], fb[j]);
    if (b) { round_encode<T, VEC>(rb, fb, true); rb.store(b + i * VEC); }      // exact: the values are rounded already
  }
  if (blockIdx.x == 0 && threadIdx.x < n - vectors * VEC) {
    const uint64_t i = vectors * VEC + threadIdx.x;
    float s = 0.0f;
    one(Elem<T>::load(g[i]), b ? Elem<T>::load(b[i]) : 0.0f, s);
    if (b) b[i] = round_store<T>(s, true);
  }
  sum = warp_reduce(sum, OpSum());
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = 0.0;
    for (int w = 0; w < MUON_THREADS / 32; ++w) s += part[w];
    partial[blockIdx.y * MUON_PARTIALS + blockIdx.x] = s;
  }
}

// A 64 x 64 tile of a stored matrix [rows, cols], a step at a time: f(row in tile, column in tile, element's index, step), a vector each
// where rows are whole vectors, else an element
template <int VEC, class F>
__device__ __forceinline__ void muon_tile(uint32_t r0, uint32_t c0, uint32_t rows, uint32_t cols, F f) {
#pragma unroll
  for (int e = 0; e < TILE * (TILE / VEC) / MUON_THREADS; ++e) {
    const uint32_t i = threadIdx.x + e * MUON_THREADS, r = i / (TILE / VEC), c = i % (TILE / VEC) * VEC;
    if (r0 + r < rows && c0 + c < cols) f(r, c, (uint64_t)(r0 + r) * cols + c0 + c, e);
  }
}

// Eight neighbouring entries of X and where they lie in a stored matrix that is not transposed
constexpr int EIGHTS = TILE * TILE / 8 / MUON_THREADS;       // per thread and tile
template <int VEC> constexpr int TILE_VECTORS = TILE * TILE / VEC / MUON_THREADS;

// Eight neighbouring elements of a row of `cols`, from element i (column c) on; zeros behind the row.  Loading and decoding are two
// steps: a thread starts all of its loads before it waits for the first.
template <typename T> struct Eight {
  using S = typename Elem<T>::store_t;
  static constexpr int VEC = 16 / (int)sizeof(S);
  RawVec<T, VEC> r[8 / VEC];
  __device__ __forceinline__ void load(const S* p, uint64_t i, uint32_t c, uint32_t cols, bool vector) {
#pragma unroll
    for (int h = 0; h < 8 / VEC; ++h) {
      if (vector) { r[h].load(p + i + h * VEC); continue; }
      float f[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[j] = c + h * VEC + j < cols ? Elem<T>::load(p[i + h * VEC + j]) : 0.0f;
      round_encode<T, VEC>(r[h], f, true);          // exact: the values are of the storage type
    }
  }
  __device__ __forceinline__ void decode(float (&v)[8]) const {
#pragma unroll
    for (int h = 0; h < 8 / VEC; ++h) {
      float f[VEC];
      r[h].decode(f);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[h * VEC + j] = f[j];
    }
  }
};

// A grid of the CTAs that fit at a time, each with every gridDim.x-th tile: the norm is put together once per CTA, behind its first
// tile's loads.  4 x 2048^2 bf16 17 us, 6.1 TB/s (27 with a CTA per tile and each load used as it came).
template <typename T, int PARTS>
__global__ void __launch_bounds__(MUON_THREADS) muon_normalize_kernel(const __grid_constant__ MuonGroup k, const double* __restrict__ partial, int n_partial, float eps,
                                                                      muon::Operand x) {
  using S = typename Elem<T>::store_t;
  constexpr int VEC = 16 / (int)sizeof(S);
  __shared__ double part[MUON_THREADS / 32];
  __shared__ float tile[TILE][TILE + 1];
  const MuonMatrix& m = k.m[blockIdx.y];
  const uint32_t tiles_x = (k.hi + TILE - 1) / TILE, tiles = tiles_x * ((k.lo + TILE - 1) / TILE);
  const S* g = (const S*)m.g;
  const S* b = (const S*)m.buf;
  uint16_t* out = x.ptr + blockIdx.y * x.part() * PARTS;
  pdl_trigger();
  pdl_wait();
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < MUON_PARTIALS; i += MUON_THREADS)
    if ((int)threadIdx.x + i < n_partial) sum += partial[blockIdx.y * MUON_PARTIALS + threadIdx.x + i];
  sum = warp_reduce(sum, OpSum());
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
  auto scale = [&] {                 // behind a barrier
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < MUON_THREADS / 32; ++w) s += part[w];
    return (float)(muon::SCALE / (sqrt(s) + (double)eps));       // the norm itself may lie outside f32
  };
  auto put = [&](const float (&v)[8], uint32_t y, uint32_t q, float inv) {
    uint32_t w[2][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) muon::split2(v[2 * j] * inv, v[2 * j + 1] * inv, w[0][j], w[1][j]);
#pragma unroll
    for (int s = 0; s < PARTS; ++s)
      *reinterpret_cast<uint4*>(out + s * x.part() + (uint64_t)y * x.ld + q) = make_uint4(w[s][0], w[s][1], w[s][2], w[s][3]);
  };
  float inv = 0.0f;
  if (!m.tall) {
    const bool vector = k.hi % 8 == 0;
    for (uint32_t at_tile = blockIdx.x; at_tile < tiles; at_tile += gridDim.x) {
      const uint32_t x0 = at_tile % tiles_x * TILE, y0 = at_tile / tiles_x * TILE;       // of X
      Eight<T> rg[EIGHTS], rb[EIGHTS];
#pragma unroll
      for (int e = 0; e < EIGHTS; ++e) {
        const uint32_t i = threadIdx.x + e * MUON_THREADS, y = y0 + i / (TILE / 8), q = x0 + i % (TILE / 8) * 8;
        if (y >= k.lo || q >= k.hi) continue;
        rg[e].load(g, (uint64_t)y * k.hi + q, q, k.hi, vector);
        if (b) rb[e].load(b, (uint64_t)y * k.hi + q, q, k.hi, vector);
      }
      if (at_tile == blockIdx.x) {         // the first tile's loads are on their way
        __syncthreads();
        inv = scale();
      }
#pragma unroll
      for (int e = 0; e < EIGHTS; ++e) {
        const uint32_t i = threadIdx.x + e * MUON_THREADS, y = y0 + i / (TILE / 8), q = x0 + i % (TILE / 8) * 8;
        if (y >= k.lo || q >= k.hi) continue;
        float v[8], f[8];
        rg[e].decode(v);
        if (b) rb[e].decode(f);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[j] *= k.grad_scale;
          if (b) v[j] = muon_direction(v[j], f[j], k);
        }
        put(v, y, q, inv);
      }
    }
    return;
  }
  for (uint32_t at_tile = blockIdx.x; at_tile < tiles; at_tile += gridDim.x) {
    const uint32_t x0 = at_tile % tiles_x * TILE, y0 = at_tile / tiles_x * TILE;
    auto before = [&] { if (at_tile != blockIdx.x) __syncthreads(); };          // the tile before has been read
    if (k.lo % VEC == 0) {
      RawVec<T, VEC> rg[TILE_VECTORS<VEC>], rb[TILE_VECTORS<VEC>];
      muon_tile<VEC>(x0, y0, k.hi, k.lo, [&](uint32_t, uint32_t, uint64_t i, int e) {
        rg[e].load(g + i);
        if (b) rb[e].load(b + i); else rb[e].zero();
      });
      before();
      muon_tile<VEC>(x0, y0, k.hi, k.lo, [&](uint32_t r, uint32_t c, uint64_t, int e) {
        float fg[VEC], fb[VEC];
        rg[e].decode(fg);
        rb[e].decode(fb);
#pragma unroll
        for (int j = 0; j < VEC; ++j) tile[r][c + j] = b ? muon_direction(fg[j] * k.grad_scale, fb[j], k) : fg[j] * k.grad_scale;
      });
    } else {
      before();
      muon_tile<1>(x0, y0, k.hi, k.lo, [&](uint32_t r, uint32_t c, uint64_t i, int) {
        const float gv = Elem<T>::load(g[i]) * k.grad_scale;
        tile[r][c] = b ? muon_direction(gv, Elem<T>::load(b[i]), k) : gv;
      });
    }
    __syncthreads();
    if (at_tile == blockIdx.x) inv = scale();
#pragma unroll
    for (int e = 0; e < EIGHTS; ++e) {
      const uint32_t i = threadIdx.x + e * MUON_THREADS, y = i % TILE, q = i / TILE * 8;       // lanes down a column of the tile: no bank twice
      if (y0 + y >= k.lo || x0 + q >= k.hi) continue;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = x0 + q + j < k.hi ? tile[q + j][y] : 0.0f;
      put(v, y0 + y, x0 + q, inv);
    }
  }
}

template <typename T, int PARTS>
__global__ void __launch_bounds__(MUON_THREADS) muon_step_kernel(const __grid_constant__ MuonGroup k, muon::Operand x, float decay, float step_flat, float step_tall) {
  using S = typename Elem<T>::store_t;
  constexpr int VEC = 16 / (int)sizeof(S);
  __shared__ float tile[TILE][TILE + 1];
  const MuonMatrix& m = k.m[blockIdx.z];
  const uint32_t x0 = blockIdx.x * TILE, y0 = blockIdx.y * TILE;
  const uint16_t* in = x.ptr + blockIdx.z * x.part() * PARTS;
  const float step = (m.tall ? step_tall : step_flat) * muon::UNSCALE;
  S* p = (S*)m.p;
  pdl_trigger();
  pdl_wait();
  auto fetch = [&](RawVec<f16_t, 8> (&r)[PARTS], uint32_t y, uint32_t q) {
#pragma unroll
    for (int s = 0; s < PARTS; ++s) r[s].load_stream(in + s * x.part() + (uint64_t)y * x.ld + q);
  };
  auto sum = [&](float (&v)[8], const RawVec<f16_t, 8> (&r)[PARTS]) {
#pragma unroll
    for (int s = 0; s < PARTS; ++s) {
      float f[8];
      r[s].decode(f);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = s ? v[j] + f[j] : f[j];
    }
  };
  if (!m.tall) {
    RawVec<f16_t, 8> rx[EIGHTS][PARTS];
    Eight<T> rp[EIGHTS];
    const bool vector = k.hi % 8 == 0;
#pragma unroll
    for (int e = 0; e < EIGHTS; ++e) {
      const uint32_t i = threadIdx.x + e * MUON_THREADS, y = y0 + i / (TILE / 8), q = x0 + i % (TILE / 8) * 8;
      if (y >= k.lo || q >= k.hi) continue;
      fetch(rx[e], y, q);
      rp[e].load(p, (uint64_t)y * k.hi + q, q, k.hi, vector);
    }
#pragma unroll
    for (int e = 0; e < EIGHTS; ++e) {
      const uint32_t i = threadIdx.x + e * MUON_THREADS, y = y0 + i / (TILE / 8), q = x0 + i % (TILE / 8) * 8;
      if (y >= k.lo || q >= k.hi) continue;
      S* to = p + (uint64_t)y * k.hi + q;
      float v[8], f[8];
      sum(v, rx[e]);
      rp[e].decode(f);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = f[j] * decay - step * v[j];
      if (vector) {
#pragma unroll
        for (int h = 0; h < 8 / VEC; ++h) {
          RawVec<T, VEC> r;
          float o[VEC];
#pragma unroll
          for (int j = 0; j < VEC; ++j) o[j] = f[h * VEC + j];
          round_encode<T, VEC>(r, o, k.rn != 0);
          r.store(to + h * VEC);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (q + j < k.hi) to[j] = round_store<T>(f[j], k.rn != 0);
      }
    }
    return;
  }
  const bool vector = k.lo % VEC == 0;
  RawVec<f16_t, 8> rx[EIGHTS][PARTS];
  RawVec<T, VEC> rp[TILE_VECTORS<VEC>];
#pragma unroll
  for (int e = 0; e < EIGHTS; ++e) {
    const uint32_t i = threadIdx.x + e * MUON_THREADS, y = i / (TILE / 8), q = i % (TILE / 8) * 8;
    if (y0 + y < k.lo && x0 + q < k.hi) fetch(rx[e], y0 + y, x0 + q);
  }
  if (vector) muon_tile<VEC>(x0, y0, k.hi, k.lo, [&](uint32_t, uint32_t, uint64_t i, int e) { rp[e].load(p + i); });
#pragma unroll
  for (int e = 0; e < EIGHTS; ++e) {
    const uint32_t i = threadIdx.x + e * MUON_THREADS, y = i / (TILE / 8), q = i % (TILE / 8) * 8;
    if (y0 + y >= k.lo || x0 + q >= k.hi) continue;
    float v[8];
    sum(v, rx[e]);
#pragma unroll
    for (int j = 0; j < 8; ++j) tile[q + j][y] = v[j];
  }
  __syncthreads();
  if (vector) {
    muon_tile<VEC>(x0, y0, k.hi, k.lo, [&](uint32_t r, uint32_t c, uint64_t i, int e) {
      float f[VEC];
      rp[e].decode(f);
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[j] = f[j] * decay - step * tile[r][c + j];
      round_encode<T, VEC>(rp[e], f, k.rn != 0);
      rp[e].store(p + i);
    });
  } else {
    muon_tile<1>(x0, y0, k.hi, k.lo, [&](uint32_t r, uint32_t c, uint64_t i, int) {
      p[i] = round_store<T>(Elem<T>::load(p[i]) * decay - step * tile[r][c], k.rn != 0);
    });
  }
}

float muon_adjust(int kind, uint64_t rows, uint64_t cols) {
  if (kind == ZYXB_MUON_ADJUST_RMS) return 0.2f * std::sqrt((float)std::max(rows, cols));
  return std::sqrt(std::max(1.0f, (float)((double)rows / (double)cols)));
}

void muon_coefficients(const zyxb_muon_desc& d, float& a, float& b, float& c) {
  a = d.a; b = d.b; c = d.c;
  if (a == 0.0f && b == 0.0f && c == 0.0f) { a = 3.4445f; b = -4.7750f; c = 2.0315f; }
}

// 16-bit matrices come with at most 11 bits and are stored with them again; f32 ones take two parts
int muon_parts(int dtype) { return dtype == ZYXB_F32 ? 2 : 1; }

uint64_t up(uint64_t v, uint64_t a) { return (v + a - 1) / a * a; }

struct MuonPlan { uint64_t lo, hi; std::vector<int> members; };

uint64_t muon_bytes(uint64_t lo, uint64_t hi, uint64_t batch, int parts) {
  const uint32_t splits = parts == 2 ? muon::split_count<2>((uint32_t)lo, (uint32_t)hi, (uint32_t)batch) : muon::split_count<1>((uint32_t)lo, (uint32_t)hi, (uint32_t)batch);
  const uint64_t split = splits > 1 ? muon::SPLIT_CTAS * 65536ull : 0;
  return split + up(batch * MUON_PARTIALS * sizeof(double), 256) + 2 * up(batch * parts * lo * up(hi, 8) * 2, 256) + 2 * up(batch * parts * lo * up(lo, 8) * 2, 256);
}

// matrices that are updated together, in the order of their first members
std::vector<MuonPlan> muon_plan(const zyxb_muon_desc& d, const uint64_t* rows, const uint64_t* cols) {
  std::vector<MuonPlan> plans;
  for (int i = 0; i < d.n_tensors; ++i) {
    const uint64_t lo = std::min(rows[i], cols[i]), hi = std::max(rows[i], cols[i]);
    MuonPlan* to = nullptr;
    for (auto& g : plans)
      if (g.lo == lo && g.hi == hi && g.members.size() < MUON_TABLE && muon_bytes(lo, hi, g.members.size() + 1, muon_parts(d.dtype)) <= MUON_GROUP_BYTES) to = &g;
    if (!to) { plans.push_back(MuonPlan{lo, hi, {}}); to = &plans.back(); }
    to->members.push_back(i);
  }
  return plans;
}

// CTAs per matrix of the one-launch update, 0 where it does not take it: X has to fit the cluster's shared memory, 128 rows of 512 columns
// (256 with two parts) per CTA.  At 128 x 784 f32 it takes 61 us where a launch per product takes 174.
template <int PARTS> uint32_t small_ctas(uint64_t lo, uint64_t hi) {
  if (lo > muon::SMALL_ROWS || hi > (uint64_t)muon::SMALL_CTAS * muon::Small<PARTS>::COLS) return 0;
  uint32_t c = 1;
  while (c < muon::SMALL_CTAS && c * 64 < hi) c *= 2;
  return c;
}

template <typename T, int PARTS>
int muon_run_small(const zyxb_muon_desc& d, const MuonGroup& k, uint32_t batch, uint32_t ctas, const LaunchCtx& lc, std::string& err) {
  static_assert(MUON_TABLE <= muon::SMALL_TABLE, "");
  muon::SmallArgs a{};
  for (uint32_t j = 0; j < batch; ++j) a.m[j] = muon::SmallMatrix{k.m[j].p, k.m[j].g, k.m[j].buf, k.m[j].tall};
  a.lo = k.lo; a.hi = k.hi; a.cols = (uint32_t)up((k.hi + ctas - 1) / ctas, 64);
  a.momentum = k.momentum; a.grad_scale = k.grad_scale; a.eps = d.eps == 0.0f ? 1e-7f : d.eps;
  muon_coefficients(d, a.a, a.b, a.c);
  a.decay = 1.0f - d.lr * d.weight_decay;
  a.step_flat = d.lr * muon_adjust(d.adjust, k.lo, k.hi); a.step_tall = d.lr * muon_adjust(d.adjust, k.hi, k.lo);
  a.steps = d.steps ? d.steps : 5; a.nesterov = k.nesterov; a.rn = k.rn; a.status = lc.status_word;
  using SM = muon::Small<PARTS>;
  auto kern = muon::small_kernel<T, PARTS>;
  static uint64_t configured = 0;
  cudaError_t e = ensure_dynamic_smem(kern, SM::TOTAL, &configured);
  if (e == cudaSuccess) {
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas * batch); cfg.blockDim = dim3(muon::SMALL_THREADS); cfg.dynamicSmemBytes = SM::TOTAL; cfg.stream = lc.stream;
    cfg.attrs = attr; cfg.numAttrs = 2;
    e = cudaLaunchKernelEx(&cfg, kern, a);
  }
  if (e != cudaSuccess) { err = std::string("muon: ") + cudaGetErrorString(e); return ZYXB_ERR_KERNEL_LAUNCH; }
  return check_launch(lc, err, "muon");
}

template <typename T, int PARTS>
int muon_run(const zyxb_muon_desc& d, const uint64_t* rows, const uint64_t* cols, const MuonPlan& pl, void* const* args, void* workspace, const LaunchCtx& lc, std::string& err) {
  const uint32_t lo = (uint32_t)pl.lo, hi = (uint32_t)pl.hi, batch = (uint32_t)pl.members.size();
  MuonGroup k{};
  k.lo = lo; k.hi = hi; k.momentum = d.momentum; k.grad_scale = d.grad_scale == 0.0f ? 1.0f : d.grad_scale;
  k.nesterov = d.nesterov ? 1 : 0; k.rn = lc.round_nearest ? 1 : 0;
  const int n = d.n_tensors;
  for (uint32_t j = 0; j < batch; ++j) {
    const int i = pl.members[j];
    k.m[j] = MuonMatrix{args[i], args[n + i], d.momentum != 0.0f ? args[2 * n + i] : nullptr, rows[i] > cols[i] ? 1u : 0u};
  }
  if (const uint32_t ctas = small_ctas<PARTS>(lo, hi)) return muon_run_small<T, PARTS>(d, k, batch, ctas, lc, err);
  char* at = (char*)workspace;
  double* partial = (double*)at;
  at += up(batch * MUON_PARTIALS * sizeof(double), 256);
  auto operand = [&](uint32_t rows, uint32_t cols) {
    muon::Operand o{(uint16_t*)at, rows, cols, (uint32_t)up(cols, 8)};
    at += up(batch * PARTS * o.part() * 2, 256);
    return o;
  };
  muon::Operand x[2], gram, poly;
  x[0] = operand(lo, hi); x[1] = operand(lo, hi); gram = operand(lo, lo); poly = operand(lo, lo);
  const uint32_t splits = muon::split_count<PARTS>(lo, hi, batch);
  float* split_sums = (float*)at;

  const unsigned sums = (unsigned)std::min<uint64_t>(MUON_PARTIALS, ((uint64_t)lo * hi + MUON_THREADS * 16 - 1) / (MUON_THREADS * 16));
  const dim3 tiles((hi + TILE - 1) / TILE, (lo + TILE - 1) / TILE, batch);
  cudaError_t e = launch_pdl(muon_momentum_kernel<T>, dim3(sums, batch), MUON_THREADS, 0, lc.stream, k, partial);
  const unsigned walkers = std::min(tiles.x * tiles.y, std::max(1u, (unsigned)lc.sm_count * NORM_CTAS / batch));
  if (e == cudaSuccess) e = launch_pdl(muon_normalize_kernel<T, PARTS>, dim3(walkers, batch), MUON_THREADS, 0, lc.stream, k, partial, (int)sums, d.eps == 0.0f ? 1e-7f : d.eps, x[0]);

  // CTAs per tile of the three products; each CTA's share of either operand is 128 rows (or 128 columns, as two boxes of 64) either way
  const int square = muon::tile_ctas<PARTS, true>(lo, lo, batch, lc.sm_count), apply = muon::tile_ctas<PARTS, false>(lo, hi, batch, lc.sm_count);
  CUtensorMap x_rows[2], x_k[2], gram_rows, poly_rows;
  bool ok = true;
  for (int j = 0; j < 2; ++j)
    ok = ok && muon::encode(lc.tma_encode, &x_rows[j], x[j], PARTS, batch, 128) && muon::encode(lc.tma_encode, &x_k[j], x[j], PARTS, batch, 64);
  ok = ok && muon::encode(lc.tma_encode, &gram_rows, gram, PARTS, batch, 128) && muon::encode(lc.tma_encode, &poly_rows, poly, PARTS, batch, 128);
  if (!ok) { err = "muon: cuTensorMapEncodeTiled rejected an operand"; return ZYXB_ERR_KERNEL_LAUNCH; }
  float a, b, c;
  muon_coefficients(d, a, b, c);
  auto gemm_args = [&](const muon::Operand& out, uint32_t contraction) {
    muon::GemmArgs g{};
    g.out = out.ptr; g.m = out.rows; g.n = out.cols; g.k = contraction; g.batch = batch; g.ld = out.ld; g.part = out.part(); g.stride = out.part() * PARTS;
    return g;
  };
  const int steps = d.steps ? d.steps : 5;
  for (int i = 0; i < steps && e == cudaSuccess; ++i) {
    const int from = i & 1;
    if (splits > 1) {
      muon::GemmArgs s = gemm_args(gram, hi);
      s.partial = split_sums; s.splits = splits;
      e = muon::launch<PARTS, 128, 1, true, false, false, true>(x_rows[from], x_rows[from], s, lc);
      const unsigned blocks = (lo + 63) / 64;
      if (e == cudaSuccess)
        e = launch_pdl(muon::gram_finish_kernel<PARTS>, dim3(blocks, blocks, batch), 256, 0, lc.stream, (const float*)split_sums, splits,
                       muon::tile_count<true>(lo, lo, 128), s);
    } else {
      e = muon::launch<PARTS, true, false, false>(square, x_rows[from], x_rows[from], gemm_args(gram, hi), lc);
    }
    if (e != cudaSuccess) break;
    muon::GemmArgs g = gemm_args(poly, lo);
    g.gram = gram.ptr; g.a = a; g.b = b; g.c = c;
    e = muon::launch<PARTS, true, true, false>(square, gram_rows, gram_rows, g, lc);
    if (e != cudaSuccess) break;
    e = muon::launch<PARTS, false, false, true>(apply, poly_rows, x_k[from], gemm_args(x[from ^ 1], lo), lc);
  }
  if (e != cudaSuccess) { err = std::string("muon: ") + cudaGetErrorString(e); return ZYXB_ERR_KERNEL_LAUNCH; }
  e = launch_pdl(muon_step_kernel<T, PARTS>, tiles, MUON_THREADS, 0, lc.stream, k, x[steps & 1], 1.0f - d.lr * d.weight_decay,
                 d.lr * muon_adjust(d.adjust, lo, hi), d.lr * muon_adjust(d.adjust, hi, lo));
  if (e != cudaSuccess) { err = std::string("muon: ") + cudaGetErrorString(e); return ZYXB_ERR_KERNEL_LAUNCH; }
  return check_launch(lc, err, "muon", 3 + (splits > 1 ? 4 : 3) * steps);
}

}  // namespace

int validate_muon(const zyxb_muon_desc& d, std::string& err) {
  auto bad = [&](const char* m) { err = m; return (int)ZYXB_ERR_KERNEL_COMPILATION; };
  if (d.dtype != ZYXB_F32 && d.dtype != ZYXB_BF16 && d.dtype != ZYXB_F16) return bad("muon: dtype must be f32, bf16 or f16");
  if (d.n_tensors <= 0 || d.n_tensors > 1024 || !d.rows || !d.cols) return bad("muon: needs 1 to 1024 matrices and their extents");
  for (int i = 0; i < d.n_tensors; ++i)
    if (d.rows[i] == 0 || d.cols[i] == 0 || d.rows[i] > MUON_MAX_EXTENT || d.cols[i] > MUON_MAX_EXTENT) return bad("muon: extents must be between 1 and 32768");
  if (d.steps < 0 || d.steps > 32) return bad("muon: at most 32 steps");
  if (!(d.eps == 0.0f || d.eps >= 1e-30f)) return bad("muon: eps must be at least 1e-30 (0 means 1e-7)");
  if (d.adjust != ZYXB_MUON_ADJUST_RATIO && d.adjust != ZYXB_MUON_ADJUST_RMS) return bad("muon: unknown adjust");
  // The products keep X in 16-bit floats: a polynomial that lets singular values grow from step to step would leave their range.
  float a, b, c;
  muon_coefficients(d, a, b, c);
  for (int i = 0; i <= 1280; ++i) {
    const double x = i / 1024.0, y = x * (a + x * x * (b + (double)c * x * x));
    if (!(std::fabs(y) <= 1.25)) return bad("muon: a x + b x^3 + c x^5 must map [0, 1.25] into [-1.25, 1.25]");
  }
  return ZYXB_OK;
}

uint64_t muon_workspace_bytes(const zyxb_muon_desc& d, const uint64_t* rows, const uint64_t* cols) {
  uint64_t most = 0;
  for (const MuonPlan& pl : muon_plan(d, rows, cols)) {
    const bool one_launch = muon_parts(d.dtype) == 2 ? small_ctas<2>(pl.lo, pl.hi) != 0 : small_ctas<1>(pl.lo, pl.hi) != 0;
    if (!one_launch) most = std::max(most, muon_bytes(pl.lo, pl.hi, pl.members.size(), muon_parts(d.dtype)));
  }
  return most;
}

int launch_muon(const zyxb_muon_desc& d, const uint64_t* rows, const uint64_t* cols, void* workspace, void* const* args,
                const uint64_t* arg_bytes, int n_args, const LaunchCtx& lc, std::string& err) {
  const int n = d.n_tensors, groups = d.momentum != 0.0f ? 3 : 2;
  ZYXB_CHECK_ARG(n_args == groups * n, "muon: expected args p[0..n), g[0..n) [, buf[0..n)]");
  const uint64_t es = dtype_size(d.dtype);
  std::vector<const void*> written;
  for (int k = 0; k < groups; ++k)
    for (int i = 0; i < n; ++i) {
      ZYXB_CHECK_ARG(arg_bytes[k * n + i] >= rows[i] * cols[i] * es, "muon: buffer smaller than its matrix");
      if (k != 1) written.push_back(args[k * n + i]);
    }
  std::sort(written.begin(), written.end());
  ZYXB_CHECK_ARG(std::adjacent_find(written.begin(), written.end()) == written.end(), "muon: the same buffer is given twice to be updated");
  for (int i = 0; i < n; ++i)
    ZYXB_CHECK_ARG(!std::binary_search(written.begin(), written.end(), (const void*)args[n + i]), "muon: a gradient is given as a buffer to be updated");
  if (!lc.tma_encode) { err = "muon: the driver offers no cuTensorMapEncodeTiled"; return ZYXB_ERR_KERNEL_LAUNCH; }
  for (const MuonPlan& pl : muon_plan(d, rows, cols)) {
    int st;
    switch (d.dtype) {
      case ZYXB_F32: st = muon_run<float, 2>(d, rows, cols, pl, args, workspace, lc, err); break;
      case ZYXB_BF16: st = muon_run<bf16_t, 1>(d, rows, cols, pl, args, workspace, lc, err); break;
      default: st = muon_run<f16_t, 1>(d, rows, cols, pl, args, workspace, lc, err); break;
    }
    if (st) return st;
  }
  return ZYXB_OK;
}

}  // namespace zyxb
