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

}  // namespace zyxb
