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

}  // namespace zyxb
