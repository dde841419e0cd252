// Muon: momentum, then the update made nearly orthogonal by Newton-Schulz products, then the weight's step.
#include <algorithm>
#include <cmath>
#include <vector>

#include "gemm.h"
#include "rounding.cuh"

namespace zyxb {

namespace {

constexpr uint64_t MUON_MAX_EXTENT = 32768;
constexpr int MUON_THREADS = 256, MUON_PARTIALS = 512;

struct MuonMatrix {
  void* p;
  const void* g;
  void* buf;
  uint32_t rows, cols;
  float momentum, grad_scale;
  int nesterov, rn;
};

// the step before it is made orthogonal, from the stored momentum
__device__ __forceinline__ float muon_direction(float g, float buf, const MuonMatrix& m) {
  if (!m.buf) return g;
  return m.nesterov ? g + m.momentum * buf : buf;
}

// buf = momentum * buf + g and the sum of squares of the direction, in 64 bits: a gradient's square leaves f32 at 1e19 and 1e-23
template <typename T>
__global__ void __launch_bounds__(MUON_THREADS) muon_momentum_kernel(MuonMatrix m, double* __restrict__ partial) {
  using S = typename Elem<T>::store_t;
  __shared__ double part[MUON_THREADS / 32];
  const uint64_t n = (uint64_t)m.rows * m.cols;
  const S* g = (const S*)m.g;
  S* b = (S*)m.buf;
  double sum = 0.0;
  for (uint64_t i = (uint64_t)blockIdx.x * MUON_THREADS + threadIdx.x; i < n; i += (uint64_t)gridDim.x * MUON_THREADS) {
    const float gv = Elem<T>::load(g[i]) * m.grad_scale;
    float bv = 0.0f;
    if (b) {
      const S s = round_store<T>(m.momentum * Elem<T>::load(b[i]) + gv, m.rn != 0);
      b[i] = s;
      bv = Elem<T>::load(s);
    }
    const double u = muon_direction(gv, bv, m);
    sum += u * u;
  }
  sum = warp_reduce(sum, OpSum());
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = 0.0;
    for (int w = 0; w < MUON_THREADS / 32; ++w) s += part[w];
    partial[blockIdx.x] = s;
  }
}

// X = direction / (norm + eps), lying down: rows <= cols after a transposition where needed
template <typename T>
__global__ void __launch_bounds__(MUON_THREADS) muon_normalize_kernel(MuonMatrix m, const double* __restrict__ partial, int n_partial, float eps, float* __restrict__ x) {
  using S = typename Elem<T>::store_t;
  __shared__ double total;
  __shared__ float tile[32][33];
  if (threadIdx.x < 32) {
    double s = 0.0;
    for (int i = threadIdx.x; i < n_partial; i += 32) s += partial[i];
    s = warp_reduce(s, OpSum());
    if (threadIdx.x == 0) total = s;
  }
  __syncthreads();
  const float inv = 1.0f / ((float)sqrt(total) + eps);
  const bool tall = m.rows > m.cols;
  const uint32_t c0 = blockIdx.x * 32, r0 = blockIdx.y * 32;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const S* g = (const S*)m.g;
  const S* b = (const S*)m.buf;
  for (int j = ty; j < 32; j += 8) {
    const uint32_t r = r0 + j, c = c0 + tx;
    if (r >= m.rows || c >= m.cols) continue;
    const uint64_t i = (uint64_t)r * m.cols + c;
    const float v = muon_direction(Elem<T>::load(g[i]) * m.grad_scale, b ? Elem<T>::load(b[i]) : 0.0f, m) * inv;
    if (tall) tile[j][tx] = v; else x[i] = v;
  }
  if (!tall) return;
  __syncthreads();
  for (int j = ty; j < 32; j += 8) {
    const uint32_t r = r0 + tx, c = c0 + j;
    if (r < m.rows && c < m.cols) x[(uint64_t)c * m.rows + r] = tile[tx][j];
  }
}

// B = a I + b A + c A^2 (A^2 given)
__global__ void muon_polynomial_kernel(const float* __restrict__ a1, float* __restrict__ a2, uint32_t m, float a, float b, float c) {
  for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < (uint64_t)m * m; i += (uint64_t)gridDim.x * blockDim.x)
    a2[i] = (i % (m + 1) == 0 ? a : 0.0f) + b * a1[i] + c * a2[i];
}

template <typename T>
__global__ void muon_step_kernel(MuonMatrix m, const float* __restrict__ x, float decay, float step) {
  using S = typename Elem<T>::store_t;
  S* p = (S*)m.p;
  const bool tall = m.rows > m.cols;
  for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < (uint64_t)m.rows * m.cols; i += (uint64_t)gridDim.x * blockDim.x) {
    const float o = tall ? x[(i % m.cols) * m.rows + i / m.cols] : x[i];
    p[i] = round_store<T>(Elem<T>::load(p[i]) * decay - step * o, m.rn != 0);
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

int muon_gemm(const float* a, const float* b, float* c, uint64_t m, uint64_t n, uint64_t k, bool trans_b, const LaunchCtx& lc, std::string& err) {
  zyxb_gemm_desc g{};
  g.dtype = ZYXB_F32; g.m = m; g.n = n; g.k = k; g.batch = 1; g.trans_b = trans_b ? 1 : 0;
  void* args[3] = {(void*)a, (void*)b, (void*)c};
  const uint64_t bytes[3] = {m * k * 4, n * k * 4, m * n * 4};
  return launch_gemm(g, args, bytes, 3, lc, err);
}

template <typename T>
int muon_update(const zyxb_muon_desc& d, const MuonMatrix& m, void* workspace, const LaunchCtx& lc, std::string& err) {
  const uint64_t lo = std::min(m.rows, m.cols), hi = std::max(m.rows, m.cols), n = lo * hi;
  double* partial = (double*)workspace;
  float* x = (float*)(partial + MUON_PARTIALS);
  float *y = x + n, *a1 = y + n, *a2 = a1 + lo * lo;
  const unsigned sums = (unsigned)std::min<uint64_t>(MUON_PARTIALS, (n + MUON_THREADS * 8 - 1) / (MUON_THREADS * 8));
  muon_momentum_kernel<T><<<sums, MUON_THREADS, 0, lc.stream>>>(m, partial);
  muon_normalize_kernel<T><<<dim3((m.cols + 31) / 32, (m.rows + 31) / 32), MUON_THREADS, 0, lc.stream>>>(m, partial, (int)sums, d.eps == 0.0f ? 1e-7f : d.eps, x);
  float a, b, c;
  muon_coefficients(d, a, b, c);
  int launches = 3, st;
  for (int i = 0; i < (d.steps ? d.steps : 5); ++i) {
    if ((st = muon_gemm(x, x, a1, lo, lo, hi, true, lc, err))) return st;
    if ((st = muon_gemm(a1, a1, a2, lo, lo, lo, true, lc, err))) return st;
    muon_polynomial_kernel<<<(unsigned)std::min<uint64_t>(2048, (lo * lo + 255) / 256), 256, 0, lc.stream>>>(a1, a2, (uint32_t)lo, a, b, c);
    ++launches;
    if ((st = muon_gemm(a2, x, y, lo, hi, lo, false, lc, err))) return st;
    std::swap(x, y);
  }
  muon_step_kernel<T><<<(unsigned)std::min<uint64_t>(4096, (n + 255) / 256), 256, 0, lc.stream>>>(m, x, 1.0f - d.lr * d.weight_decay, d.lr * muon_adjust(d.adjust, m.rows, m.cols));
  return check_launch(lc, err, "muon", launches);
}

}  // namespace

int validate_muon(const zyxb_muon_desc& d, std::string& err) {
  auto bad = [&](const char* m) { err = m; return (int)ZYXB_ERR_KERNEL_COMPILATION; };
  if (d.dtype != ZYXB_F32 && d.dtype != ZYXB_BF16 && d.dtype != ZYXB_F16) return bad("muon: dtype must be f32, bf16 or f16");
  if (d.n_tensors <= 0 || d.n_tensors > 1024 || !d.rows || !d.cols) return bad("muon: needs 1 to 1024 matrices and their extents");
  for (int i = 0; i < d.n_tensors; ++i)
    if (d.rows[i] == 0 || d.cols[i] == 0 || d.rows[i] > MUON_MAX_EXTENT || d.cols[i] > MUON_MAX_EXTENT) return bad("muon: extents must be between 1 and 32768");
  if (d.steps < 0 || d.steps > 32) return bad("muon: at most 32 steps");
  if (!(d.eps >= 0.0f)) return bad("muon: eps must not be negative");
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
  for (int i = 0; i < d.n_tensors; ++i) {
    const uint64_t lo = std::min(rows[i], cols[i]);
    most = std::max(most, 4 * (2 * rows[i] * cols[i] + 2 * lo * lo));
  }
  return MUON_PARTIALS * sizeof(double) + most;
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
  for (int i = 0; i < n; ++i) {
    MuonMatrix m{};
    m.p = args[i]; m.g = args[n + i]; m.buf = groups > 2 ? args[2 * n + i] : nullptr;
    m.rows = (uint32_t)rows[i]; m.cols = (uint32_t)cols[i]; m.momentum = d.momentum;
    m.grad_scale = d.grad_scale == 0.0f ? 1.0f : d.grad_scale; m.nesterov = d.nesterov ? 1 : 0; m.rn = lc.round_nearest ? 1 : 0;
    int st;
    switch (d.dtype) {
      case ZYXB_F32: st = muon_update<float>(d, m, workspace, lc, err); break;
      case ZYXB_BF16: st = muon_update<bf16_t>(d, m, workspace, lc, err); break;
      default: st = muon_update<f16_t>(d, m, workspace, lc, err); break;
    }
    if (st) return st;
  }
  return ZYXB_OK;
}

}  // namespace zyxb
