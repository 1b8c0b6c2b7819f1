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

// ------------------------------------------------- 16 bytes of a row at once
using u32x4 = uint32_t __attribute__((ext_vector_type(4)));

template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

// Aligned to the element only: gfx950 loads and stores 16 bytes at any
// address, so that odd widths and strides need no kernel of their own.
template <typename T>
__device__ __forceinline__ u32x4 load16(const T* p) {
  u32x4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
template <typename T>
__device__ __forceinline__ void store16(T* p, u32x4 v) {
  __builtin_memcpy(p, &v, 16);
}

// Past the caches: for what is too large to be found there again.
template <typename T>
__device__ __forceinline__ void stream16(T* p, u32x4 v) {
  typedef u32x4 __attribute__((aligned(2))) any;
  __builtin_nontemporal_store(v, reinterpret_cast<any*>(p));
}

// Element j (known when compiled) of 16 bytes, as fp32.
template <typename T>
__device__ __forceinline__ float elem(u32x4 v, int j) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(v[j]);
  } else if constexpr (__is_same(T, bf16)) {
    return __uint_as_float(j & 1 ? v[j >> 1] & 0xffff0000u : v[j >> 1] << 16);
  } else {
    return to_f(__builtin_bit_cast(f16, (uint16_t)(v[j >> 1] >> (j & 1) * 16)));
  }
}

template <typename T>
__device__ __forceinline__ void put(u32x4& v, int j, T x) {
  if constexpr (sizeof(T) == 4) {
    v[j] = __float_as_uint(x);
  } else {
    const uint32_t u = __builtin_bit_cast(uint16_t, x);
    v[j >> 1] = j & 1 ? (v[j >> 1] & 0xffffu) | u << 16
                      : (v[j >> 1] & 0xffff0000u) | u;
  }
}

template <typename T>
__device__ __forceinline__ u32x4 pack(const float* r) {
  T t[kVec<T>];
#pragma unroll
  for (int j = 0; j < kVec<T>; ++j) t[j] = static_cast<T>(r[j]);
  u32x4 v;
  __builtin_memcpy(&v, t, 16);
  return v;
}

template <typename T>
__device__ __forceinline__ u32x4 minus_inf() {
  const uint32_t u = sizeof(T) == 4         ? 0xff800000u
                     : __is_same(T, bf16) ? 0xff80ff80u
                                          : 0xfc00fc00u;
  return u32x4{u, u, u, u};
}

// A number that is part of a type, to choose a kernel's sizes with.
template <int N>
struct Int {
  static constexpr int value = N;
};

struct Add {
  template <typename A>
  __device__ __forceinline__ A operator()(A a, A b) const { return a + b; }
};
struct Max {
  __device__ __forceinline__ float operator()(float a, float b) const {
    return fmaxf(a, b);
  }
};
struct Larger {
  template <typename A>
  __device__ __forceinline__ A operator()(A a, A b) const {
    return a > b ? a : b;
  }
};
// NaN wins: a row that holds one has to say so
struct MaxNan {
  __device__ __forceinline__ float operator()(float a, float b) const {
    return __builtin_elementwise_maximum(a, b);
  }
};

// The value of a lane and of the one O lanes away (lane ^ O), in either order,
// without a trip through LDS: quad_perm, row_half_mirror and row_ror of the
// data-parallel primitives within rows of 16, swaps of rows beyond.
struct Pair {
  float x, y;
};
template <int Ctrl>
__device__ __forceinline__ float dpp(float v) {
  const int i = __float_as_int(v);
  return __int_as_float(
      __builtin_amdgcn_update_dpp(i, i, Ctrl, 0xf, 0xf, false));
}
template <int O>
__device__ __forceinline__ Pair lanes(float v) {
  if constexpr (O == 1) return {v, dpp<0xb1>(v)};            // quad [1,0,3,2]
  else if constexpr (O == 2) return {v, dpp<0x4e>(v)};       // quad [2,3,0,1]
  else if constexpr (O == 4) return {v, dpp<0x141>(dpp<0x1b>(v))};  // 3, then 7
  else if constexpr (O == 8) return {v, dpp<0x128>(v)};      // rotate by 8
  else {
    const uint32_t u = __float_as_uint(v);
    const auto r = O == 16
                       ? __builtin_amdgcn_permlane16_swap(u, u, false, false)
                       : __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return {__uint_as_float(r[0]), __uint_as_float(r[1])};
  }
}

// What the lanes of a wave have written to LDS is seen by all of them.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ float sum_of(Pair p) { return p.x + p.y; }

// How many lanes below this one have their bit in a ballot.
__device__ __forceinline__ int lanes_before(uint64_t ballot) {
  return __builtin_amdgcn_mbcnt_hi(
      (uint32_t)(ballot >> 32),
      __builtin_amdgcn_mbcnt_lo((uint32_t)ballot, 0));
}

// Reductions over the wave, in every lane.
template <typename Op>
__device__ __forceinline__ float wave_reduce(float v, Op op) {
  Pair p = lanes<1>(v);
  v = op(p.x, p.y);
  p = lanes<2>(v);
  v = op(p.x, p.y);
  p = lanes<4>(v);
  v = op(p.x, p.y);
  p = lanes<8>(v);
  v = op(p.x, p.y);
  p = lanes<16>(v);
  v = op(p.x, p.y);
  p = lanes<32>(v);
  return op(p.x, p.y);
}
// The same exchange of both halves of a double, and the wave's sum of two.
template <int O>
__device__ __forceinline__ double sum_pair(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const Pair lo = lanes<O>(__uint_as_float((uint32_t)u));
  const Pair hi = lanes<O>(__uint_as_float((uint32_t)(u >> 32)));
  auto join = [](float h, float l) {
    return __builtin_bit_cast(double, (uint64_t)__float_as_uint(h) << 32 |
                                          __float_as_uint(l));
  };
  return join(hi.x, lo.x) + join(hi.y, lo.y);
}
__device__ __forceinline__ void wave_sum(double& a, double& b) {
  a = sum_pair<1>(a);
  b = sum_pair<1>(b);
  a = sum_pair<2>(a);
  b = sum_pair<2>(b);
  a = sum_pair<4>(a);
  b = sum_pair<4>(b);
  a = sum_pair<8>(a);
  b = sum_pair<8>(b);
  a = sum_pair<16>(a);
  b = sum_pair<16>(b);
  a = sum_pair<32>(a);
  b = sum_pair<32>(b);
}

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

// The block's maximum in every thread, NaN if there is one. One barrier:
// `scratch` must not be written again before the next.
template <int NT>
__device__ __forceinline__ float block_max(float v, float* scratch) {
  v = wave_reduce(v, MaxNan{});
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  v = scratch[0];
#pragma unroll
  for (int i = 1; i < NT / 64; ++i) v = MaxNan{}(v, scratch[i]);
  return v;
}

}  // namespace dear_lm
