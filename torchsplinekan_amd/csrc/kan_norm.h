// The norm after a block, its gate and residual scale, and the norm before
// the next block, in one pass over the rows of a residual stream:
//   u  = post * y r1,           r1 = (mean(y^2) + eps)^(-1/2)    (u = y without post)
//   x' = x + s a(g) u,          a = identity, sigmoid, tanh or silu
//   h  = pre * x' r2,           r2 = (mean(x'^2) + eps)^(-1/2)
// and its backward pass: with t = dh pre, xh = x' r2 and yh = y r1,
//   D  = dx' + r2 (t - xh mean(t xh)),   dx = D,   dpre = sum_rows dh xh
//   v  = D s a(g),  w = v post
//   dy = r1 (w - yh mean(w yh)),         dpost = sum_rows v yh     (dy = v without post)
//   dg = D s u a'(g), summed over what g is broadcast over;  ds = sum_rows D a(g) u.
//
// All arithmetic is in float32, rounded once where a result is stored: x' is
// recomputed from x and y in the backward (the same bytes as reading x'), so
// both passes see the unrounded stream.  Sums over rows go through one partial
// row per block and are added in block order: no atomics, the same bits every
// time.
//
// This header holds what the forward (kan_norm.hip) and the backward
// (kan_norm_grad.hip) share.
#pragma once

#include "kan_types.h"

namespace kan {

enum GateKind {
  kGateNone = 0,
  kGateElement = 1,   // [n, C]
  kGateToken = 2,     // [n]
  kGateRows = 3,      // [n / L, C]: one row of the gate for L rows, L > 1
  kGateScalars = 4    // [n / L]: one value for L rows, L > 1
};

struct NormParams {
  const void *x, *y, *gate, *post, *pre, *scale;
  void *x_out, *h_out;
  float* rstd;             // [2, n]: r1, r2 (optional in the forward)
  const void *dxo, *dh;    // backward: gradients of x' and h, either may be null
  void *dx, *dy, *dgate;
  float *part_pre, *part_branch;  // [blocks, C]: sums of dh xh and of D a(g) yh
  float* part_gate;        // kGateRows: [n / L * nchunk, C]; kGateScalars: [n]
  int64_t n, C, L;
  int64_t chunk, nchunk, seg_rows;  // rows of a block; see row_range
  float scale_const, eps;
  int gate_kind, act, wdtype;
};

// The rows of block b.  A gate row's rows are either cut into nchunk blocks
// (seg_rows = L) or handled whole, several gate rows to a block (nchunk = 1,
// chunk a multiple of L); any other gate has one segment of n rows.
struct RowRange {
  int64_t lo, hi;
};
__device__ __forceinline__ RowRange row_range(const NormParams& p, int64_t b) {
  RowRange r;
  const int64_t seg = b / p.nchunk;
  r.lo = seg * p.seg_rows + (b - seg * p.nchunk) * p.chunk;
  const int64_t end = p.nchunk > 1 ? min(p.n, (seg + 1) * p.seg_rows) : p.n;
  r.hi = min(end, r.lo + p.chunk);
  return r;
}

__device__ __forceinline__ float sigmoid_of(float v) { return 1.0f / (1.0f + expf(-v)); }

__device__ __forceinline__ float act_of(float g, int act) {
  switch (act) {
    case KAN_GATE_SIGMOID: return sigmoid_of(g);
    case KAN_GATE_TANH: return tanhf(g);
    case KAN_GATE_SILU: return g * sigmoid_of(g);
    default: return g;
  }
}
// a(g) and a'(g) from one evaluation.
__device__ __forceinline__ void act_both(float g, int act, float* a, float* slope) {
  switch (act) {
    case KAN_GATE_SIGMOID:
      *a = sigmoid_of(g);
      *slope = *a * (1.0f - *a);
      break;
    case KAN_GATE_TANH:
      *a = tanhf(g);
      *slope = 1.0f - *a * *a;
      break;
    case KAN_GATE_SILU: {
      const float s = sigmoid_of(g);
      *a = g * s;
      *slope = s * (1.0f + g * (1.0f - s));
      break;
    }
    default:
      *a = g;
      *slope = 1.0f;
  }
}
__device__ __forceinline__ float act_slope(float g, int act) {
  float a, slope;
  act_both(g, act, &a, &slope);
  return slope;
}

// ---- rows of any width ------------------------------------------------------
// One block per row at a time, its values read again in every pass.
constexpr int kRowThreads = 256;

__device__ __forceinline__ float block_sum(float v, float* red) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.0f;
#pragma unroll
  for (int w = 0; w < kRowThreads / 64; ++w) s += red[w];
  return s;
}

template <typename TX, typename TY>
struct RowView {
  const NormParams& p;
  const TX* x;
  const TY *y, *gate;
  int64_t gstep;  // 0: one value for the row
  float r1;
  __device__ RowView(const NormParams& p_, int64_t row) : p(p_), r1(1.0f) {
    x = static_cast<const TX*>(p.x) + row * p.C;
    y = p.y == nullptr ? nullptr : static_cast<const TY*>(p.y) + row * p.C;
    gate = nullptr;
    gstep = 0;
    if (p.gate_kind != kGateNone) {
      gstep = p.gate_kind == kGateElement || p.gate_kind == kGateRows;
      gate = static_cast<const TY*>(p.gate) + (row / p.L) * (gstep ? p.C : 1);
    }
  }
  __device__ __forceinline__ float scale(int64_t c) const {
    return p.scale == nullptr ? p.scale_const : load_any(p.scale, c, p.wdtype);
  }
  __device__ __forceinline__ float post(int64_t c) const { return load_any(p.post, c, p.wdtype); }
  __device__ __forceinline__ float g(int64_t c) const { return (float)gate[c * gstep]; }
  __device__ __forceinline__ float a(int64_t c) const {
    return gate == nullptr ? 1.0f : act_of(g(c), p.act);
  }
  __device__ __forceinline__ float u(int64_t c) const {
    return p.post == nullptr ? (float)y[c] : (float)y[c] * r1 * post(c);
  }
  __device__ __forceinline__ float stream(int64_t c) const {
    const float v = (float)x[c];
    return y == nullptr ? v : v + scale(c) * a(c) * u(c);
  }
};

// ---- rows held in registers ---------------------------------------------------
// TPR lanes share a row, each with 8 of its values (16 in rows of more than 8192)
// in NV pieces of VEC; a block is one row's lanes, or four waves with a row (8 or 4
// narrow ones) each, and runs through its rows, the weights staying in registers.
// Every value is read once: the passes above happen on registers, a row's sums
// cross its waves through LDS.
template <int TPR>
struct RowShape {
  static constexpr int kThreads = TPR <= 64 ? 256 : TPR;
  static constexpr int kRows = kThreads / TPR;          // rows at once
  static constexpr int kWaves = TPR <= 64 ? 1 : TPR / 64;  // of a row
  static_assert(kRows == 1 || kWaves == 1, "rows side by side share no barrier");
};

// Sums of M values over a row's lanes.  Rows of several waves take two buffers
// in turn, so that one barrier a sum is enough: a wave that writes a buffer
// again has passed the barrier after which all had read it.
template <int TPR, int M>
__device__ __forceinline__ void row_sums(float (&v)[M], float* red, int& turn) {
#pragma unroll
  for (int m = 0; m < M; ++m) {
    if constexpr (TPR >= 64) v[m] = wave_sum(v[m]);
    else v[m] = lane_sum<TPR>(v[m]);
  }
  constexpr int W = RowShape<TPR>::kWaves;
  if constexpr (W > 1) {
    float* buf = red + turn * (2 * W) + 0;
    turn ^= 1;
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int m = 0; m < M; ++m) buf[m * W + w] = v[m];
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < M; ++m) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < W; ++i) s += buf[m * W + i];
      v[m] = s;
    }
  }
}

#define KAN_EACH                     \
  _Pragma("unroll") for (int i = 0; i < NV; ++i) _Pragma("unroll") for (int j = 0; j < VEC; ++j)

// The lane's pieces of a row of C values: piece i starts at (i TPR + lane) VEC.
// Values past the row's end are zero and not stored.  WHOLE: rows are whole
// vectors, on 16 bytes; otherwise vectors lie anywhere, and a row's last piece
// goes value by value.
template <typename T, int TPR, int VEC, int NV, bool WHOLE>
struct Pieces {
  __device__ __forceinline__ static int64_t at(int i) {
    return (int64_t)(i * TPR + (int)threadIdx.x % TPR) * VEC;
  }
  typedef typename VecOf<T, VEC>::type vec;
  __device__ __forceinline__ static void fetch(vec (&v)[NV], const T* __restrict__ row, int64_t C) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (at(i) + VEC <= C) {
        if constexpr (WHOLE) v[i] = *reinterpret_cast<const vec*>(row + at(i));
        else v[i] = reinterpret_cast<const LooseVec<T, VEC>*>(row + at(i))->v;
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] = !WHOLE && at(i) + j < C ? row[at(i) + j] : (T)0.0f;
      }
    }
  }
  __device__ __forceinline__ static void unpack(float (&v)[NV][VEC], const vec (&raw)[NV]) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] = (float)raw[i][j];
  }
  __device__ __forceinline__ static void load(float (&v)[NV][VEC], const T* __restrict__ row,
                                              int64_t C) {
    vec raw[NV];
    fetch(raw, row, C);
    unpack(v, raw);
  }
  __device__ __forceinline__ static void store(const float (&v)[NV][VEC], T* __restrict__ row,
                                               int64_t C) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (at(i) + VEC <= C) {
        store_f32<T, VEC, WHOLE>(row + at(i), v[i]);
      } else if constexpr (!WHOLE) {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (at(i) + j < C) row[at(i) + j] = (T)v[i][j];
      }
    }
  }
};

// The lane's pieces of a weight vector (of `none` where there is no vector).
template <int TPR, bool WHOLE, int VEC, int NV>
__device__ __forceinline__ void load_weight(float (&v)[NV][VEC], const void* __restrict__ w,
                                            int dtype, int64_t C, float none) {
  if (w == nullptr) {
    KAN_EACH v[i][j] = none;
  } else if (dtype == KAN_DTYPE_F32) {
    Pieces<float, TPR, VEC, NV, WHOLE>::load(v, static_cast<const float*>(w), C);
  } else if (dtype == KAN_DTYPE_BF16) {
    Pieces<bf16, TPR, VEC, NV, WHOLE>::load(v, static_cast<const bf16*>(w), C);
  } else {
    Pieces<f16, TPR, VEC, NV, WHOLE>::load(v, static_cast<const f16*>(w), C);
  }
}

// Lanes that share a row of C values, 8 each (16 past 8192; rows past kMaxHeld
// stay in memory, on blocks of 256).
constexpr int64_t kMaxHeld = 16384;
inline int held_tpr(int64_t C) {
  if (C > kMaxHeld) return 256;
  if (C <= 128) return C <= 64 ? 8 : 16;
  int tpr = 64;
  while (tpr < 1024 && tpr * 8 < C) tpr *= 2;
  return tpr;
}

// How rows are dealt to blocks, and the backward's partial sums.
struct RowPlan {
  int64_t blocks, chunk, nchunk, seg_rows, gate_rows;  // gate_rows of part_gate
  size_t bytes;
};
constexpr int kGradWaves = 16;  // waves a CU (one block of the widest shape)
inline RowPlan row_plan(int64_t n, int64_t C, int kind, int64_t L, int waves_per_cu) {
  const int tpr = held_tpr(C);
  const int threads = tpr <= 64 ? 256 : tpr, at_once = threads / tpr;
  const int64_t target = device_cu_count() * (int64_t)std::max(1, 64 * waves_per_cu / threads);
  RowPlan g{};
  const int64_t want = std::max<int64_t>(1, ceil_div(n, target));
  if (kind == kGateRows && L > want) {
    g.nchunk = ceil_div(L, want);
    g.chunk = ceil_div(L, g.nchunk);
    g.nchunk = ceil_div(L, g.chunk);
    g.seg_rows = L;
    g.blocks = n / L * g.nchunk;
    g.gate_rows = g.blocks;
  } else {
    g.nchunk = 1;
    g.chunk = kind == kGateRows ? want / L * L : round_up(want, at_once);
    g.seg_rows = g.chunk;
    g.blocks = ceil_div(n, g.chunk);
    g.gate_rows = kind == kGateRows ? n / L : 0;
  }
  size_t floats = (size_t)(2 * g.blocks + g.gate_rows) * (size_t)C;
  if (kind == kGateScalars) floats += (size_t)n;
  g.bytes = 4 * floats;
  return g;
}

// Whether rows are whole vectors (16 bytes of the branch's type) and every
// operand lies on 16 bytes.
inline bool whole_vectors(const NormParams& p, int vec, size_t xb, size_t yb) {
  if (p.C % vec != 0) return false;
  auto ok = [](const void* q, size_t bytes) {
    return reinterpret_cast<uintptr_t>(q) % (bytes < 16 ? bytes : 16) == 0;
  };
  return ok(p.x, vec * xb) && ok(p.x_out, vec * xb) && ok(p.dxo, vec * xb) && ok(p.dx, vec * xb) &&
         ok(p.y, vec * yb) && ok(p.gate, p.gate_kind == kGateToken || p.gate_kind == kGateScalars
                                             ? 1 : vec * yb) &&
         ok(p.h_out, vec * yb) && ok(p.dh, vec * yb) && ok(p.dy, vec * yb) &&
         ok(p.dgate, p.gate_kind == kGateElement ? vec * yb : 1) && ok(p.post, 16) &&
         ok(p.pre, 16) && ok(p.scale, 16);
}

// Calls Launch::run<TX, TY, TPR, VALS, GATE, WHOLE>() for a row held in registers:
// TPR lanes with VALS values each.
template <class Launch, typename TX, typename TY, int GATE, bool WHOLE>
int launch_shape(const Launch& l, int64_t C) {
  switch (held_tpr(C)) {
    case 8: return l.template run<TX, TY, 8, 8, GATE, WHOLE>();
    case 16: return l.template run<TX, TY, 16, 8, GATE, WHOLE>();
    case 64: return l.template run<TX, TY, 64, 8, GATE, WHOLE>();
    case 128: return l.template run<TX, TY, 128, 8, GATE, WHOLE>();
    case 256: return l.template run<TX, TY, 256, 8, GATE, WHOLE>();
    case 512: return l.template run<TX, TY, 512, 8, GATE, WHOLE>();
    default:
      return C <= 8192 ? l.template run<TX, TY, 1024, 8, GATE, WHOLE>()
                       : l.template run<TX, TY, 1024, 16, GATE, WHOLE>();
  }
}
template <class Launch, typename TX, typename TY, bool WHOLE>
int launch_gate(const Launch& l, const NormParams& p) {
  if (p.gate_kind == kGateElement) return launch_shape<Launch, TX, TY, 1, WHOLE>(l, p.C);
  if (p.gate_kind == kGateRows) return launch_shape<Launch, TX, TY, 2, WHOLE>(l, p.C);
  return launch_shape<Launch, TX, TY, 0, WHOLE>(l, p.C);
}
// The same for the call's types; Launch::rows<TX, TY>() for rows of any width.
template <class Launch, typename TX, typename TY>
int launch_typed(const Launch& l, const NormParams& p) {
  if (p.C > kMaxHeld) return l.template rows<TX, TY>();
  return whole_vectors(p, sizeof(TY) == 2 ? 8 : 4, sizeof(TX), sizeof(TY))
             ? launch_gate<Launch, TX, TY, true>(l, p)
             : launch_gate<Launch, TX, TY, false>(l, p);
}
template <class Launch>
int launch_norm(const Launch& l, const NormParams& p, int xdtype, int ydtype) {
  if (xdtype == KAN_DTYPE_BF16) return launch_typed<Launch, bf16, bf16>(l, p);
  if (xdtype == KAN_DTYPE_F16) return launch_typed<Launch, f16, f16>(l, p);
  if (ydtype == KAN_DTYPE_BF16) return launch_typed<Launch, float, bf16>(l, p);
  if (ydtype == KAN_DTYPE_F16) return launch_typed<Launch, float, f16>(l, p);
  return launch_typed<Launch, float, float>(l, p);
}

// The backward's launches (kan_norm_grad.hip); p.dx .. p.part_gate as given.
int launch_norm_grad(const NormParams& p, const RowPlan& g, int xdtype, int ydtype, void* dpre,
                     void* dpost, void* dscale, hipStream_t st);

}  // namespace kan
