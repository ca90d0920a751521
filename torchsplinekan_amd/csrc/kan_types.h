// The 16-bit types of the operators beside the KAN layers (norms, 8-bit
// activations, grouped and gated products, losses): storage types, conversions, vectors
// and wave sums.
#pragma once

#include "kan_common.h"

namespace kan {

typedef __bf16 bf16;
typedef _Float16 f16;

inline size_t dtype_bytes(int code) {
  return code == KAN_DTYPE_F64 ? 8 : code == KAN_DTYPE_F32 ? 4 : 2;
}
inline bool dtype_is_operator(int code) {
  return code == KAN_DTYPE_F32 || code == KAN_DTYPE_BF16 || code == KAN_DTYPE_F16;
}

template <typename T, int V>
struct VecOf {
  typedef T type __attribute__((ext_vector_type(V)));
};

// A vector at an address that is aligned to one value only (the hardware
// takes it; the compiler must not assume more).
template <typename T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) LooseVec {
  typename VecOf<T, V>::type v;
};

// V consecutive values as floats.  WHOLE: p is aligned to 16 bytes, or to the
// vector if that is shorter.
template <typename T, int V, bool WHOLE = true>
__device__ __forceinline__ void load_f32(const T* __restrict__ p, float (&v)[V]) {
  typename VecOf<T, V>::type u;
  if constexpr (WHOLE) u = *reinterpret_cast<const typename VecOf<T, V>::type*>(p);
  else u = reinterpret_cast<const LooseVec<T, V>*>(p)->v;
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = (float)u[j];
}

// The same rounded to T (to nearest, ties to even).
template <typename T, int V, bool WHOLE = true>
__device__ __forceinline__ void store_f32(T* __restrict__ p, const float (&v)[V]) {
  typename VecOf<T, V>::type u;
#pragma unroll
  for (int j = 0; j < V; ++j) u[j] = (T)v[j];
  if constexpr (WHOLE) *reinterpret_cast<typename VecOf<T, V>::type*>(p) = u;
  else reinterpret_cast<LooseVec<T, V>*>(p)->v = u;
}

// 16 bytes from an address that is even only.  The hardware takes such a load,
// several times slower than one of whole words: 5 words and a shift.  (Nothing
// past the word of the last byte is read.)
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
struct __attribute__((packed, aligned(4))) Words4 {
  u32x4 v;
};
__device__ __forceinline__ u32x4 load16_even(const void* p) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p);
  const uint32_t* words = reinterpret_cast<const uint32_t*>(at & ~(uintptr_t)3);
  const uint32_t shift = (uint32_t)(at & 2) * 8;
  const u32x4 w = reinterpret_cast<const Words4*>(words)->v;
  const uint32_t last = words[3 + (shift >> 4)];
  u32x4 v;
  v[0] = __builtin_amdgcn_alignbit(w[1], w[0], shift);
  v[1] = __builtin_amdgcn_alignbit(w[2], w[1], shift);
  v[2] = __builtin_amdgcn_alignbit(w[3], w[2], shift);
  v[3] = __builtin_amdgcn_alignbit(last, w[3], shift);
  return v;
}

// One value of an array whose type is known at run time (the short vectors of
// weights, read once a row or less).
__device__ __forceinline__ float load_any(const void* __restrict__ p, int64_t i, int dtype) {
  if (dtype == KAN_DTYPE_F32) return static_cast<const float*>(p)[i];
  if (dtype == KAN_DTYPE_BF16) return (float)static_cast<const bf16*>(p)[i];
  return (float)static_cast<const f16*>(p)[i];
}
__device__ __forceinline__ void store_any(void* __restrict__ p, int64_t i, int dtype, float v) {
  if (dtype == KAN_DTYPE_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == KAN_DTYPE_BF16) static_cast<bf16*>(p)[i] = (bf16)v;
  else static_cast<f16*>(p)[i] = (f16)v;
}

template <int CTRL, int ROW_MASK = 0xf>
__device__ __forceinline__ float dpp_or_zero(float v) {
  return __int_as_float(
      __builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROW_MASK, 0xf, false));
}

// Sum over the wave, in every lane (a fixed tree: the same bits every time).
__device__ __forceinline__ float wave_sum(float v) {
  v += dpp_or_zero<0xB1>(v);         // lane ^ 1
  v += dpp_or_zero<0x4E>(v);         // lane ^ 2
  v += dpp_or_zero<0x141>(v);        // mirrored half rows: the other 4 of 8
  v += dpp_or_zero<0x140>(v);        // mirrored rows: the other 8 of 16
  v += dpp_or_zero<0x142, 0xa>(v);   // row 0 into 1, row 2 into 3
  v += dpp_or_zero<0x143, 0xc>(v);   // rows 0 and 1 into 2 and 3
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int m = 1; m < 64; m *= 2) v = fmaxf(v, __shfl_xor(v, m));
  return v;
}

// Sum over aligned groups of 8, 16 or 32 lanes, in each of them.
template <int LANES>
__device__ __forceinline__ float lane_sum(float v) {
  static_assert(LANES == 8 || LANES == 16 || LANES == 32, "groups of lanes in a wave");
  v += dpp_or_zero<0xB1>(v);
  v += dpp_or_zero<0x4E>(v);
  v += dpp_or_zero<0x141>(v);
  if constexpr (LANES >= 16) v += dpp_or_zero<0x140>(v);
  if constexpr (LANES == 32) v += __shfl_xor(v, 16);
  return v;
}

}  // namespace kan
