// Stores of the kernels whose 16-bit rounding follows the context: round_nearest uses the conversion instructions (nearest even,
// subnormals kept, NaN stays NaN); the default truncates like every other kernel of the library (common.cuh).
#pragma once
#include "common.cuh"
#include "tc_ptx.cuh"

namespace zyxb {

template <typename T>
__device__ __forceinline__ typename Elem<T>::store_t round_store(float v, bool rn) {
  if constexpr (std::is_same_v<T, float>) return v;
  else if (rn) return (uint16_t)pack2_t<std::is_same_v<T, bf16_t>>(v, 0.0f);
  else return Elem<T>::store(v, false);
}

// VEC values into the register image of a vector store
template <typename T, int VEC>
__device__ __forceinline__ void round_encode(RawVec<T, VEC>& raw, const float (&v)[VEC], bool rn) {
  if constexpr (sizeof(typename Elem<T>::store_t) == 2 && VEC % 2 == 0) {
    if (rn) {
#pragma unroll
      for (int j = 0; j < VEC / 2; ++j) raw.w[j] = pack2_t<std::is_same_v<T, bf16_t>>(v[2 * j], v[2 * j + 1]);
      return;
    }
    raw.encode(v, false);
  } else if constexpr (sizeof(typename Elem<T>::store_t) == 2) {
    raw.w[0] = round_store<T>(v[0], rn);
  } else {
    raw.encode(v, false);
  }
}

// The numbers of a vector as the arithmetic units take them: pairs (sm_100's packed f32 instructions: two per issue slot), or a
// single float where a vector is one element.
template <int VEC> struct Nums {
  static constexpr int N = VEC > 1 ? VEC / 2 : 1;
  using V = std::conditional_t<(VEC > 1), uint64_t, float>;
  static __device__ __forceinline__ V splat(float x) { if constexpr (VEC > 1) return f2_pack(x, x); else return x; }
  static __device__ __forceinline__ V mul(V a, V b) { if constexpr (VEC > 1) return f2_mul(a, b); else return a * b; }
  static __device__ __forceinline__ V add(V a, V b) { if constexpr (VEC > 1) return f2_add(a, b); else return a + b; }
  static __device__ __forceinline__ V fma(V a, V b, V c) { if constexpr (VEC > 1) return f2_fma(a, b, c); else return fmaf(a, b, c); }
  static __device__ __forceinline__ float sum(V a) {
    if constexpr (VEC > 1) { float x, y; f2_unpack(a, x, y); return x + y; } else return a;
  }
  template <typename T> static __device__ __forceinline__ void decode(V (&v)[N], const RawVec<T, VEC>& r) {
    if constexpr (VEC == 1) {
      float f[1];
      r.decode(f);
      v[0] = f[0];
    } else if constexpr (std::is_same_v<T, bf16_t>) {
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = f2_pack_bits(r.w[j] << 16, r.w[j] & 0xffff0000u);
    } else {
      float f[VEC];
      r.decode(f);
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = f2_pack(f[2 * j], f[2 * j + 1]);
    }
  }
  static __device__ __forceinline__ void floats(float (&f)[VEC], const V (&v)[N]) {
    if constexpr (VEC == 1) f[0] = v[0];
    else {
#pragma unroll
      for (int j = 0; j < N; ++j) f2_unpack(v[j], f[2 * j], f[2 * j + 1]);
    }
  }
  template <typename T> static __device__ __forceinline__ void encode(RawVec<T, VEC>& r, const V (&v)[N], bool rn) {
    float f[VEC];
    floats(f, v);
    round_encode<T, VEC>(r, f, rn);
  }
};

// elements d .. d + VEC of the two vectors in w
template <typename T, int VEC>
__device__ __forceinline__ void shift_vector(RawVec<T, VEC>& r, uint32_t (&w)[2 * RawVec<T, VEC>::NW], int d) {
  constexpr int W = RawVec<T, VEC>::NW, PER = VEC / W;
  const int s = d / PER;
  if (s & 2) {
#pragma unroll
    for (int j = 0; j < 2 * W - 2; ++j) w[j] = w[j + 2];
  }
  if (s & 1) {
#pragma unroll
    for (int j = 0; j < 2 * W - 3; ++j) w[j] = w[j + 1];
  }
#pragma unroll
  for (int j = 0; j < W; ++j) r.w[j] = PER == 2 && (d & 1) ? __funnelshift_r(w[j], w[j + 1], 16) : w[j];
}

// A vector from any element on, of a buffer that starts on a vector boundary and has `end` elements: the two aligned vectors that hold
// it (elements before the buffer or behind its end come as zeros), and how far it lies inside them.  Every lane of a row shifts
// alike, and the second vector is the next lane's first, so the extra read is an L1 hit.  Loading and shifting are two steps: a
// thread starts all of its loads before it waits for the first.
// (its elements at the buffer's ends: rare, and kept out of the way of the loops that inline the rest)
template <typename T, int VEC>
__device__ __noinline__ uint4 vector_at_end(const typename Elem<T>::store_t* base, int64_t first, uint64_t end) {
  constexpr int PER = VEC / 4;
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int k = 0; k < VEC; ++k)
    if (first + k >= 0 && (uint64_t)(first + k) < end) {
      if constexpr (PER == 2) w[k / 2] |= (uint32_t)base[first + k] << (16 * (k & 1));
      else w[k] = __float_as_uint(base[first + k]);
    }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T, int VEC> struct Shifted {
  using S = typename Elem<T>::store_t;
  static constexpr int W = RawVec<T, VEC>::NW, PER = VEC / W;          // words, elements per word
  static_assert(W == 4, "16-byte vectors");
  RawVec<T, VEC> half[2];
  int d;
  __device__ __forceinline__ void zero() { half[0].zero(); half[1].zero(); d = 0; }
  __device__ __forceinline__ void load(const S* base, int64_t e, uint64_t end) {
    const int64_t v = e >= 0 ? e / VEC : -((-e + VEC - 1) / VEC), first = v * VEC;
    d = (int)(e - first);
    if (first >= 0 && (uint64_t)first + 2 * VEC <= end) {
      half[0].load(base + first);
      half[1].load(base + first + VEC);
      return;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 q = vector_at_end<T, VEC>(base, first + h * VEC, end);
      half[h].w[0] = q.x; half[h].w[1] = q.y; half[h].w[2] = q.z; half[h].w[3] = q.w;
    }
  }
  __device__ __forceinline__ void get(RawVec<T, VEC>& r) const {
    uint32_t w[2 * W];
#pragma unroll
    for (int j = 0; j < W; ++j) { w[j] = half[0].w[j]; w[W + j] = half[1].w[j]; }
    shift_vector<T, VEC>(r, w, d);
  }
};
template <typename T, int VEC>
__device__ __forceinline__ void load_shifted(RawVec<T, VEC>& r, const typename Elem<T>::store_t* base, int64_t e, uint64_t end) {
  Shifted<T, VEC> s;
  s.load(base, e, end);
  s.get(r);
}

}  // namespace zyxb
