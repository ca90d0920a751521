// Activations kept in 8 bits between the forward and the backward pass.
// Every row is cut into groups of G = 32, 64, 128 or 256 values along its
// last axis (the last group of a row may be short).  With m = max |x| of the
// group:
//   scale = m * (1 / qmax)  (qmax 127 for int8, 448 for e4m3), float32
//   q     = round(x * (1 / scale))  to nearest, ties to even
//   x     ~ q * scale
// A group whose scale would lie below the smallest normal float32 (m below
// qmax 1.2e-38) keeps scale 0 and comes back as zeros; a group that holds an
// infinity or a NaN keeps scale NaN and comes back as NaN throughout, so that
// a step that went wrong stays visible.
//
// A lane has 8 values, G / 8 lanes a group, their largest magnitude found by
// exchanges between them: one pass, bound by HBM.  65536 x 1024 bf16 to int8 44 us
// (203 MB, 4.6 TB/s), back 32 us (6.3 TB/s, the 8-bit values partly from the
// last-level cache); 10007 x 1001 f16 to e4m3 11 us, back 8 us.
#include "kan_types.h"

namespace kan {

namespace {

constexpr int kActThreads = 256;
constexpr int kActVals = 8;  // values of a lane

struct Act8Params {
  const void* x;
  int64_t ldx;      // x's row stride
  uint8_t* q;       // [rows, C]
  float* scale;     // [rows, parts]
  void* out;        // [rows, C]
  int64_t rows, C, parts;
  int group, vec;   // vec: rows are whole vectors, on their alignment
  int flat;         // groups are whole and follow each other in memory
};

template <int FORMAT>
struct Act8;
template <>
struct Act8<KAN_ACT8_INT8> {
  static constexpr float kMax = 127.0f;
  __device__ static __forceinline__ uint32_t pack4(const float* u) {
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w |= ((uint32_t)(int)rintf(u[j]) & 0xffu) << (8 * j);
    return w;
  }
  __device__ static __forceinline__ void unpack4(uint32_t w, float* u) {
#pragma unroll
    for (int j = 0; j < 4; ++j) u[j] = (float)(int8_t)(w >> (8 * j));
  }
};
template <>
struct Act8<KAN_ACT8_E4M3> {
  static constexpr float kMax = 448.0f;
  __device__ static __forceinline__ uint32_t pack4(const float* u) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(u[0], u[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(u[2], u[3], w, true);
  }
  __device__ static __forceinline__ void unpack4(uint32_t w, float* u) {
    u[0] = __builtin_amdgcn_cvt_f32_fp8((int)w, 0);
    u[1] = __builtin_amdgcn_cvt_f32_fp8((int)w, 1);
    u[2] = __builtin_amdgcn_cvt_f32_fp8((int)w, 2);
    u[3] = __builtin_amdgcn_cvt_f32_fp8((int)w, 3);
  }
};

struct __attribute__((packed, aligned(1))) LooseBytes {
  uint2 v;
};

// This lane's place (false past the last group).
struct Lane {
  int64_t x, q, scale;  // offsets of its values and of its group's scale
  int n;                // its values, 0..8
};
__device__ __forceinline__ bool lane_place(const Act8Params& p, Lane* l) {
  const int lpg = p.group / kActVals;
  const int64_t t = (int64_t)blockIdx.x * (kActThreads / lpg) + threadIdx.x / lpg;
  if (t >= p.rows * p.parts) return false;
  const int in = (threadIdx.x % lpg) * kActVals;
  l->scale = t;
  if (p.flat) {
    l->x = l->q = t * p.group + in;
    l->n = kActVals;
    return true;
  }
  const int64_t row = t < 0x80000000ll ? (int64_t)((uint32_t)t / (uint32_t)p.parts) : t / p.parts;
  const int64_t c = (t - row * p.parts) * p.group + in;
  l->x = row * p.ldx + c;
  l->q = row * p.C + c;
  l->n = (int)max((int64_t)0, min((int64_t)kActVals, p.C - c));
  return true;
}

template <typename T, int FORMAT>
__global__ __launch_bounds__(kActThreads) void quantize_kernel(Act8Params p) {
  typedef Act8<FORMAT> F;
  Lane l;
  const bool in = lane_place(p, &l);
  float v[kActVals] = {};
  if (in) {
    const T* src = static_cast<const T*>(p.x) + l.x;
    if (l.n == kActVals) {
      if (p.vec) load_f32<T, kActVals>(src, v);
      else load_f32<T, kActVals, false>(src, v);
    } else {
#pragma unroll
      for (int j = 0; j < kActVals; ++j)
        if (j < l.n) v[j] = (float)src[j];
    }
  }
  // the largest magnitude as an integer: a NaN is above infinity
  int m = 0;
#pragma unroll
  for (int j = 0; j < kActVals; ++j) m = max(m, __float_as_int(v[j]) & 0x7fffffff);
  for (int d = p.group / kActVals / 2; d > 0; d >>= 1) m = max(m, __shfl_xor(m, d));
  if (!in) return;
  float scale = __int_as_float(m) * (1.0f / F::kMax), inv = 0.0f;
  if (m >= 0x7f800000) scale = __int_as_float(0x7fc00000);
  else if (scale < 1.17549435e-38f) scale = 0.0f;
  else inv = 1.0f / scale;
  float u[kActVals];
#pragma unroll
  for (int j = 0; j < kActVals; ++j) u[j] = inv == 0.0f ? 0.0f : v[j] * inv;
  const uint32_t lo = F::pack4(u), hi = F::pack4(u + 4);
  uint8_t* dst = p.q + l.q;
  if (l.n == kActVals) {
    if (p.vec) *reinterpret_cast<uint2*>(dst) = make_uint2(lo, hi);
    else reinterpret_cast<LooseBytes*>(dst)->v = make_uint2(lo, hi);
  } else {
#pragma unroll
    for (int j = 0; j < kActVals; ++j)
      if (j < l.n) dst[j] = (uint8_t)((j < 4 ? lo : hi) >> (8 * (j & 3)));
  }
  if (threadIdx.x % (p.group / kActVals) == 0) p.scale[l.scale] = scale;
}

template <typename T, int FORMAT>
__global__ __launch_bounds__(kActThreads) void dequantize_kernel(Act8Params p) {
  typedef Act8<FORMAT> F;
  Lane l;
  if (!lane_place(p, &l)) return;
  const uint8_t* src = p.q + l.q;
  uint32_t lo = 0, hi = 0;
  if (l.n == kActVals) {
    const uint2 w = p.vec ? *reinterpret_cast<const uint2*>(src)
                          : reinterpret_cast<const LooseBytes*>(src)->v;
    lo = w.x;
    hi = w.y;
  } else {
#pragma unroll
    for (int j = 0; j < kActVals; ++j)
      if (j < l.n) (j < 4 ? lo : hi) |= (uint32_t)src[j] << (8 * (j & 3));
  }
  const float scale = p.scale[l.scale];
  float u[kActVals];
  F::unpack4(lo, u);
  F::unpack4(hi, u + 4);
#pragma unroll
  for (int j = 0; j < kActVals; ++j) u[j] *= scale;
  T* dst = static_cast<T*>(p.out) + l.q;
  if (l.n == kActVals) {
    if (p.vec) store_f32<T, kActVals>(dst, u);
    else store_f32<T, kActVals, false>(dst, u);
  } else {
#pragma unroll
    for (int j = 0; j < kActVals; ++j)
      if (j < l.n) dst[j] = (T)u[j];
  }
}

template <typename T>
int launch_act8(const Act8Params& p, int format, bool quantize, hipStream_t st) {
  const int64_t per = kActThreads / (p.group / kActVals);
  const dim3 grid((unsigned)ceil_div(p.rows * p.parts, per));
  if (quantize) {
    if (format == KAN_ACT8_INT8) quantize_kernel<T, KAN_ACT8_INT8><<<grid, kActThreads, 0, st>>>(p);
    else quantize_kernel<T, KAN_ACT8_E4M3><<<grid, kActThreads, 0, st>>>(p);
    return check_launch("quantize_activation");
  }
  if (format == KAN_ACT8_INT8) dequantize_kernel<T, KAN_ACT8_INT8><<<grid, kActThreads, 0, st>>>(p);
  else dequantize_kernel<T, KAN_ACT8_E4M3><<<grid, kActThreads, 0, st>>>(p);
  return check_launch("dequantize_activation");
}

int run_act8(const char* who, int dtype, int format, Act8Params p, bool quantize, void* stream) {
  if (!dtype_is_operator(dtype))
    return set_error(KAN_ERR_INVALID, "%s: dtype must be FP32, BF16 or FP16 (code %d)", who, dtype);
  if (format != KAN_ACT8_INT8 && format != KAN_ACT8_E4M3)
    return set_error(KAN_ERR_INVALID, "%s: unknown 8-bit format %d", who, format);
  if (p.group != 32 && p.group != 64 && p.group != 128 && p.group != 256)
    return set_error(KAN_ERR_INVALID, "%s: group must be 32, 64, 128 or 256, got %d", who, p.group);
  if (p.rows < 0 || p.C < 0) return set_error(KAN_ERR_INVALID, "%s: negative size", who);
  if (quantize && p.rows > 1 && p.ldx < p.C)
    return set_error(KAN_ERR_INVALID, "%s: row stride smaller than the row", who);
  if (p.rows == 0 || p.C == 0) return KAN_OK;
  if ((quantize ? p.x == nullptr : p.out == nullptr) || p.q == nullptr || p.scale == nullptr)
    return set_error(KAN_ERR_INVALID, "%s: buffers must not be NULL", who);
  p.parts = ceil_div(p.C, p.group);
  if (ceil_div(p.rows * p.parts, kActThreads / (p.group / kActVals)) > 0x7fffffff)
    return set_error(KAN_ERR_LIMIT, "%s: too many groups", who);
  const uintptr_t value = dtype_bytes(dtype) * (uintptr_t)kActVals;
  const uintptr_t at = reinterpret_cast<uintptr_t>(quantize ? p.x : p.out);
  p.vec = p.C % kActVals == 0 && (!quantize || p.ldx % kActVals == 0) &&
          at % (value < 16 ? value : 16) == 0 && reinterpret_cast<uintptr_t>(p.q) % 8 == 0;
  p.flat = p.C % p.group == 0 && (!quantize || p.ldx == p.C || p.rows == 1);
  hipStream_t st = static_cast<hipStream_t>(stream);
  TimedLaunch timed(kClassOther, st,
                    (double)p.rows * (p.C * (1.0 + dtype_bytes(dtype)) + 4.0 * p.parts));
  if (dtype == KAN_DTYPE_F32) return launch_act8<float>(p, format, quantize, st);
  if (dtype == KAN_DTYPE_BF16) return launch_act8<bf16>(p, format, quantize, st);
  return launch_act8<f16>(p, format, quantize, st);
}

}  // namespace
}  // namespace kan

using namespace kan;

extern "C" {

int kan_hip_act8_quantize(int dtype, int format, const void* x, int64_t row_stride, int64_t rows,
                          int64_t C, int64_t group, void* q, float* scale, void* stream) {
  Act8Params p{};
  p.x = x;
  p.ldx = row_stride;
  p.q = static_cast<uint8_t*>(q);
  p.scale = scale;
  p.rows = rows;
  p.C = C;
  p.group = group > 0 && group <= 256 ? (int)group : 0;
  return run_act8("quantize_activation", dtype, format, p, true, stream);
}

int kan_hip_act8_dequantize(int dtype, int format, const void* q, const float* scale, int64_t rows,
                            int64_t C, int64_t group, void* out, void* stream) {
  Act8Params p{};
  p.q = static_cast<uint8_t*>(const_cast<void*>(q));
  p.scale = const_cast<float*>(scale);
  p.out = out;
  p.rows = rows;
  p.C = C;
  p.group = group > 0 && group <= 256 ? (int)group : 0;
  return run_act8("dequantize_activation", dtype, format, p, false, stream);
}

}  // extern "C"
