// Shared device helpers of the language-model kernels (layer_norm.hip,
// token_loss.hip): element types, row loads that need no alignment beyond the
// element's own, and reductions over a wave (64 lanes) and a block.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dear_lm {

// Codes of the element types at the C entries.
enum Type : int { kF32 = 0, kBF16 = 1, kF16 = 2 };

using bf16 = __bf16;
using f16 = _Float16;

template <typename T>
__device__ __forceinline__ float to_f(T v) {
  return static_cast<float>(v);
}
// bf16 is the upper half of an fp32: exact, and one shift
template <>
__device__ __forceinline__ float to_f<bf16>(bf16 v) {
  return __uint_as_float((uint32_t)__builtin_bit_cast(uint16_t, v) << 16);
}

__device__ __forceinline__ float load_as_float(const void* p, int type,
                                               int64_t i) {
  if (type == kF32) return static_cast<const float*>(p)[i];
  if (type == kBF16) return to_f(static_cast<const bf16*>(p)[i]);
  return to_f(static_cast<const f16*>(p)[i]);
}

__device__ __forceinline__ void store_as(void* p, int type, int64_t i,
                                         float v) {
  if (type == kF32) static_cast<float*>(p)[i] = v;
  else if (type == kBF16) static_cast<bf16*>(p)[i] = static_cast<bf16>(v);
  else static_cast<f16*>(p)[i] = static_cast<f16>(v);
}

struct Add {
  template <typename A>
  __device__ __forceinline__ A operator()(A a, A b) const { return a + b; }
};
// NaN wins: a row that holds one has to say so
struct MaxNan {
  __device__ __forceinline__ float operator()(float a, float b) const {
    return (a > b || a != a) ? a : b;
  }
};

template <typename A, typename Op>
__device__ __forceinline__ A wave_reduce(A v, Op op) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = op(v, __shfl_xor(v, o));
  return v;
}

// Result in every thread. `scratch`: one A per wave; free again on return.
template <typename A, typename Op>
__device__ __forceinline__ A block_reduce(A v, Op op, A* scratch) {
  v = wave_reduce(v, op);
  const int waves = blockDim.x >> 6;
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  v = scratch[0];
  for (int i = 1; i < waves; ++i) v = op(v, scratch[i]);
  __syncthreads();
  return v;
}

}  // namespace dear_lm
