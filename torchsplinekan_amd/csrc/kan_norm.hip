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
#include "kan_types.h"

namespace kan {

namespace {

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

template <typename TX, typename TY>
__global__ __launch_bounds__(kRowThreads) void norm_rows_kernel(NormParams p) {
  __shared__ float red[kRowThreads / 64];
  const float inv_c = 1.0f / (float)p.C;
  for (int64_t row = blockIdx.x; row < p.n; row += gridDim.x) {
    RowView<TX, TY> v(p, row);
    if (v.y != nullptr && p.post != nullptr) {
      float s = 0.0f;
      for (int64_t c = threadIdx.x; c < p.C; c += kRowThreads) {
        const float t = (float)v.y[c];
        s += t * t;
      }
      v.r1 = 1.0f / sqrtf(block_sum(s, red) * inv_c + p.eps);
      if (p.rstd != nullptr && threadIdx.x == 0) p.rstd[row] = v.r1;
    }
    float s = 0.0f;
    for (int64_t c = threadIdx.x; c < p.C; c += kRowThreads) {
      const float t = v.stream(c);
      s += t * t;
      if (p.x_out != nullptr) static_cast<TX*>(p.x_out)[row * p.C + c] = (TX)t;
    }
    if (p.h_out == nullptr) continue;
    const float r2 = 1.0f / sqrtf(block_sum(s, red) * inv_c + p.eps);
    if (p.rstd != nullptr && threadIdx.x == 0) p.rstd[p.n + row] = r2;
    for (int64_t c = threadIdx.x; c < p.C; c += kRowThreads)
      static_cast<TY*>(p.h_out)[row * p.C + c] =
          (TY)(v.stream(c) * r2 * load_any(p.pre, c, p.wdtype));
  }
}

// A thread owns the columns c = threadIdx.x + i kRowThreads of every row of
// its block, so a block's partial sums are plain reads and writes of its own.
__device__ __forceinline__ void add_part(float* part, int64_t at, bool first, float v) {
  if (part != nullptr) part[at] = first ? v : part[at] + v;
}

template <typename TX, typename TY>
__global__ __launch_bounds__(kRowThreads) void norm_rows_grad_kernel(NormParams p) {
  __shared__ float red[kRowThreads / 64];
  const float inv_c = 1.0f / (float)p.C;
  const RowRange rr = row_range(p, blockIdx.x);
  const int64_t b = blockIdx.x;
  for (int64_t row = rr.lo; row < rr.hi; ++row) {
    RowView<TX, TY> v(p, row);
    const bool first = row == rr.lo;
    const bool gate_rows = p.gate_kind == kGateRows;
    const bool gate_first = gate_rows && (first || row % p.L == 0);
    const int64_t gate_at =
        (p.nchunk > 1 ? b : row / p.L) * p.C;  // (kGateRows: its partial row)
    const TX* dxo = p.dxo == nullptr ? nullptr : static_cast<const TX*>(p.dxo) + row * p.C;
    const TY* dh = p.dh == nullptr ? nullptr : static_cast<const TY*>(p.dh) + row * p.C;
    if (v.y != nullptr && p.post != nullptr) v.r1 = p.rstd[row];
    float r2 = 0.0f, m2 = 0.0f;
    if (dh != nullptr) {
      r2 = p.rstd[p.n + row];
      float s = 0.0f;
      for (int64_t c = threadIdx.x; c < p.C; c += kRowThreads)
        s += (float)dh[c] * load_any(p.pre, c, p.wdtype) * (v.stream(c) * r2);
      m2 = block_sum(s, red) * inv_c;
    }
    auto total = [&](int64_t c) {  // D
      float d = dxo == nullptr ? 0.0f : (float)dxo[c];
      if (dh != nullptr)
        d += r2 * ((float)dh[c] * load_any(p.pre, c, p.wdtype) - v.stream(c) * r2 * m2);
      return d;
    };
    float s1 = 0.0f, sg = 0.0f;
    for (int64_t c = threadIdx.x; c < p.C; c += kRowThreads) {
      const float d = total(c);
      if (p.dx != nullptr) static_cast<TX*>(p.dx)[row * p.C + c] = (TX)d;
      if (dh != nullptr) add_part(p.part_pre, b * p.C + c, first, (float)dh[c] * v.stream(c) * r2);
      if (v.y == nullptr) continue;
      const float a = v.a(c), u = v.u(c), sc = v.scale(c), vv = d * sc * a;
      const float yh = (float)v.y[c] * v.r1;
      add_part(p.part_branch, b * p.C + c, first, d * a * yh);
      if (p.post != nullptr) {
        s1 += vv * v.post(c) * yh;
      } else if (p.dy != nullptr) {
        static_cast<TY*>(p.dy)[row * p.C + c] = (TY)vv;
      }
      if (p.dgate != nullptr) {
        const float dg = d * sc * u * act_slope(v.g(c), p.act);
        if (p.gate_kind == kGateElement) static_cast<TY*>(p.dgate)[row * p.C + c] = (TY)dg;
        else if (gate_rows) add_part(p.part_gate, gate_at + c, gate_first, dg);
        else sg += dg;
      }
    }
    if (v.y == nullptr) continue;
    if (p.dgate != nullptr && (p.gate_kind == kGateToken || p.gate_kind == kGateScalars)) {
      sg = block_sum(sg, red);
      if (threadIdx.x == 0) {
        if (p.gate_kind == kGateToken) static_cast<TY*>(p.dgate)[row] = (TY)sg;
        else p.part_gate[row] = sg;
      }
    }
    if (p.post == nullptr || p.dy == nullptr) continue;
    const float m1 = block_sum(s1, red) * inv_c;
    for (int64_t c = threadIdx.x; c < p.C; c += kRowThreads) {
      const float yh = (float)v.y[c] * v.r1;
      const float w = total(c) * v.scale(c) * v.a(c) * v.post(c);
      static_cast<TY*>(p.dy)[row * p.C + c] = (TY)(v.r1 * (w - yh * m1));
    }
  }
}

// ---- rows held in registers ---------------------------------------------------
// TPR lanes share a row, each with 8 of its values in NV pieces of VEC; a block
// is one row's lanes, or four waves with a row (8 or 4 narrow ones) each, and
// runs through its rows, the weights staying in registers.  Every value is read once: the
// passes above happen on registers, a row's sums cross its waves through LDS.
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

// GATE: 0 none or one value a row, 1 a value for every element, 2 a row of
// values for L rows, evaluated once for all of them that a block has.
template <typename TX, typename TY, int TPR, int VEC, int NV, int GATE, bool WHOLE>
__global__ __launch_bounds__(RowShape<TPR>::kThreads) void norm_kernel(NormParams p) {
  typedef RowShape<TPR> S;
  typedef Pieces<TX, TPR, VEC, NV, WHOLE> PX;
  typedef Pieces<TY, TPR, VEC, NV, WHOLE> PY;
  __shared__ float red[4 * S::kWaves];
  int turn = 0;
  const float inv_c = 1.0f / (float)p.C;
  const bool branch = p.y != nullptr, normed = p.post != nullptr;
  float sp[NV][VEC], pre[NV][VEC], gate[NV][VEC];  // scale * post; pre; scale * post * a(g)
  if (branch) {
    load_weight<TPR, WHOLE>(sp, p.post, p.wdtype, p.C, 1.0f);
    load_weight<TPR, WHOLE>(pre, p.scale, p.wdtype, p.C, p.scale_const);
    KAN_EACH sp[i][j] *= pre[i][j];
  }
  if (p.h_out != nullptr) load_weight<TPR, WHOLE>(pre, p.pre, p.wdtype, p.C, 1.0f);
  const RowRange rr = row_range(p, blockIdx.x);
  for (int64_t seg = rr.lo; seg < rr.hi;) {  // (one turn but for gate rows)
    const int64_t end = GATE == 2 ? min(rr.hi, (seg / p.L + 1) * p.L) : rr.hi;
    if constexpr (GATE == 2) {
      PY::load(gate, static_cast<const TY*>(p.gate) + seg / p.L * p.C, p.C);
      KAN_EACH gate[i][j] = act_of(gate[i][j], p.act) * sp[i][j];
    }
    // (every wave of a row takes the same number of turns)
    for (int64_t r0 = seg; r0 < end; r0 += S::kRows) {
      const int64_t row = r0 + threadIdx.x / TPR;
      if (S::kRows > 1 && row >= end) break;
      float x[NV][VEC];
      PX::load(x, static_cast<const TX*>(p.x) + row * p.C, p.C);
      if (branch) {
        float y[NV][VEC];
        PY::load(y, static_cast<const TY*>(p.y) + row * p.C, p.C);
        float r1 = 1.0f;
        if constexpr (GATE == 1) PY::load(gate, static_cast<const TY*>(p.gate) + row * p.C, p.C);
        if (normed) {
          float s[1] = {0.0f};
          KAN_EACH s[0] += y[i][j] * y[i][j];
          row_sums<TPR>(s, red, turn);
          r1 = 1.0f / sqrtf(s[0] * inv_c + p.eps);
          if (p.rstd != nullptr && threadIdx.x % TPR == 0) p.rstd[row] = r1;
        }
        if (GATE == 0 && p.gate_kind != kGateNone)
          r1 *= act_of((float)static_cast<const TY*>(p.gate)[row / p.L], p.act);
        KAN_EACH {
          if constexpr (GATE == 0) x[i][j] += y[i][j] * r1 * sp[i][j];
          else if constexpr (GATE == 1)
            x[i][j] += y[i][j] * r1 * sp[i][j] * act_of(gate[i][j], p.act);
          else x[i][j] += y[i][j] * r1 * gate[i][j];
        }
        if (p.x_out != nullptr) PX::store(x, static_cast<TX*>(p.x_out) + row * p.C, p.C);
      }
      if (p.h_out == nullptr) continue;
      float s[1] = {0.0f};
      KAN_EACH s[0] += x[i][j] * x[i][j];
      row_sums<TPR>(s, red, turn);
      const float r2 = 1.0f / sqrtf(s[0] * inv_c + p.eps);
      if (p.rstd != nullptr && threadIdx.x % TPR == 0) p.rstd[p.n + row] = r2;
      KAN_EACH x[i][j] *= r2 * pre[i][j];
      PY::store(x, static_cast<TY*>(p.h_out) + row * p.C, p.C);
    }
    seg = end;
  }
}

// This block's column sums into one partial row: rows that were handled side
// by side are added through LDS in order.
template <int TPR, bool WHOLE, int VEC, int NV>
__device__ __forceinline__ void flush_columns(float (&v)[NV][VEC], float* __restrict__ out,
                                              int64_t C, float* lds) {
  typedef RowShape<TPR> S;
  const int r = threadIdx.x / TPR, t = threadIdx.x % TPR;
  if constexpr (S::kRows > 1) {
    __syncthreads();
    KAN_EACH lds[(i * VEC + j) * S::kThreads + threadIdx.x] = v[i][j];
    __syncthreads();
    if (r != 0) return;
    KAN_EACH {
#pragma unroll
      for (int q = 1; q < S::kRows; ++q)
        v[i][j] += lds[(i * VEC + j) * S::kThreads + q * TPR + t];
    }
  }
  Pieces<float, TPR, VEC, NV, WHOLE>::store(v, out, C);
}

// Four waves a SIMD (128 registers; a float32 row of 512 lanes with a gate would
// spill there and takes two).  dpost = scale * (sum of D a yh) and dscale = post *
// (the same sum): one column sum serves both, a weight's factor applied after
// it.  A gate row's gradient comes from the sum of D yh, times scale, post and
// a'(g), and what its rows add to the first sum is a(g) times the same: two sums
// a row.  In 16 bits the next row's
// loads are in flight while a row is worked on (but beside a gate's values).
template <typename TX, typename TY, int TPR, int VEC, int NV, int GATE, bool WHOLE>
__global__ __launch_bounds__(RowShape<TPR>::kThreads) __attribute__((
    amdgpu_waves_per_eu(sizeof(TY) == 4 && TPR == 512 && GATE != 0 ? 2 : 4))) void
norm_grad_kernel(NormParams p) {
  typedef RowShape<TPR> S;
  typedef Pieces<TX, TPR, VEC, NV, WHOLE> PX;
  typedef Pieces<TY, TPR, VEC, NV, WHOLE> PY;
  constexpr bool kAhead = sizeof(TX) == 2 && GATE != 1;
  constexpr int kCols = S::kRows > 1 ? NV * VEC * S::kThreads : 1;
  __shared__ float red[4 * S::kWaves];
  __shared__ float cols[kCols];
  int turn = 0;
  const float inv_c = 1.0f / (float)p.C;
  const bool branch = p.y != nullptr, normed = p.post != nullptr, with_h = p.dh != nullptr;
  const bool one = GATE == 0 && p.gate_kind != kGateNone;
  float sp[NV][VEC], pre[NV][VEC];  // scale * post (a gate row: times a(g)); pre
  float s_pre[NV][VEC] = {}, s_branch[NV][VEC] = {}, s_gate[NV][VEC] = {};
  auto load_sp = [&](float (&v)[NV][VEC]) __attribute__((always_inline)) {
    float t[NV][VEC];
    load_weight<TPR, WHOLE>(v, p.post, p.wdtype, p.C, 1.0f);
    load_weight<TPR, WHOLE>(t, p.scale, p.wdtype, p.C, p.scale_const);
    KAN_EACH v[i][j] *= t[i][j];
  };
  if (branch && GATE != 2) load_sp(sp);
  if (with_h) load_weight<TPR, WHOLE>(pre, p.pre, p.wdtype, p.C, 1.0f);

  const TX *xs = static_cast<const TX*>(p.x), *dxs = static_cast<const TX*>(p.dxo);
  const TY *ys = static_cast<const TY*>(p.y), *dhs = static_cast<const TY*>(p.dh);
  const TY* gs = static_cast<const TY*>(p.gate);
  struct Row {  // as loaded
    typename PX::vec d[NV], x[NV];
    typename PY::vec y[NV], dh[NV];
  };
  auto fetch = [&](Row& r, int64_t row) __attribute__((always_inline)) {
    if (p.dxo != nullptr) PX::fetch(r.d, dxs + row * p.C, p.C);
    if (with_h) {
      PX::fetch(r.x, xs + row * p.C, p.C);
      PY::fetch(r.dh, dhs + row * p.C, p.C);
    }
    if (branch) PY::fetch(r.y, ys + row * p.C, p.C);
  };

  const RowRange rr = row_range(p, blockIdx.x);
  const int mine = threadIdx.x / TPR;
  Row in;
  for (int64_t seg = rr.lo; seg < rr.hi;) {  // (one turn but for gate rows)
    const int64_t end = GATE == 2 ? min(rr.hi, (seg / p.L + 1) * p.L) : rr.hi;
    if constexpr (GATE == 2) {
      float a[NV][VEC];
      load_sp(sp);
      PY::load(a, static_cast<const TY*>(p.gate) + seg / p.L * p.C, p.C);
      KAN_EACH sp[i][j] *= act_of(a[i][j], p.act);
    }
    if (kAhead && seg + mine < end) fetch(in, seg + mine);
    for (int64_t r0 = seg; r0 < end; r0 += S::kRows) {
      const int64_t row = r0 + mine;
      if (S::kRows > 1 && row >= end) break;
      float d[NV][VEC], x[NV][VEC], y[NV][VEC], dh[NV][VEC], a[NV][VEC], slope[NV][VEC];
      float a1 = 1.0f, slope1 = 0.0f, r1 = 1.0f, r2 = 0.0f;
      if constexpr (kAhead) {
        PX::unpack(d, in.d);
        PX::unpack(x, in.x);
        PY::unpack(y, in.y);
        PY::unpack(dh, in.dh);
      } else {
        if (p.dxo != nullptr) PX::load(d, dxs + row * p.C, p.C);
        if (with_h) {
          PX::load(x, xs + row * p.C, p.C);
          PY::load(dh, dhs + row * p.C, p.C);
        }
        if (branch) PY::load(y, ys + row * p.C, p.C);
      }
      if (p.dxo == nullptr) KAN_EACH d[i][j] = 0.0f;
      if (with_h) r2 = p.rstd[p.n + row];
      if (branch) {
        if (normed) r1 = p.rstd[row];
        if constexpr (GATE == 1) {
          PY::load(a, gs + row * p.C, p.C);
          KAN_EACH act_both(a[i][j], p.act, &a[i][j], &slope[i][j]);
        }
        if (one) act_both((float)gs[row / p.L], p.act, &a1, &slope1);
        KAN_EACH y[i][j] *= r1;  // yh (y itself without post)
      }
      if (kAhead && row + S::kRows < end) fetch(in, row + S::kRows);
      // a(g), and scale * post * a(g)
      auto gate_of = [&](int i, int j) __attribute__((always_inline)) {
        if constexpr (GATE == 1) return a[i][j];
        else return a1;
      };
      auto factor = [&](int i, int j) __attribute__((always_inline)) {
        if constexpr (GATE == 2) return sp[i][j];
        else return sp[i][j] * gate_of(i, j);
      };
      if (with_h) {
        float s[1] = {0.0f};
        KAN_EACH {
          if (branch) x[i][j] += y[i][j] * factor(i, j);
          x[i][j] *= r2;  // xh
          s_pre[i][j] += dh[i][j] * x[i][j];
          dh[i][j] *= pre[i][j];  // t
          s[0] += dh[i][j] * x[i][j];
        }
        row_sums<TPR>(s, red, turn);
        const float m2 = s[0] * inv_c;
        KAN_EACH d[i][j] += r2 * (dh[i][j] - x[i][j] * m2);
      }
      if (p.dx != nullptr) PX::store(d, static_cast<TX*>(p.dx) + row * p.C, p.C);
      if (!branch) continue;
      float s[2] = {0.0f, 0.0f};  // of w yh; of the gate's gradient
      KAN_EACH {
        const float dy = d[i][j] * y[i][j];
        if constexpr (GATE == 2) s_gate[i][j] += dy;
        else s_branch[i][j] += dy * gate_of(i, j);
        if constexpr (GATE == 0) s[1] += dy * sp[i][j];
        if constexpr (GATE == 1) slope[i][j] *= dy * sp[i][j];
        d[i][j] *= factor(i, j);  // w
        s[0] += d[i][j] * y[i][j];
      }
      if constexpr (GATE == 1) {
        if (p.dgate != nullptr) PY::store(slope, static_cast<TY*>(p.dgate) + row * p.C, p.C);
      }
      if (normed || one) row_sums<TPR>(s, red, turn);
      if (one && p.dgate != nullptr && threadIdx.x % TPR == 0) {
        if (p.gate_kind == kGateToken) static_cast<TY*>(p.dgate)[row] = (TY)(s[1] * slope1);
        else p.part_gate[row] = s[1] * slope1;
      }
      if (p.dy == nullptr) continue;
      const float m1 = normed ? s[0] * inv_c : 0.0f;
      KAN_EACH d[i][j] = r1 * (d[i][j] - y[i][j] * m1);
      PY::store(d, static_cast<TY*>(p.dy) + row * p.C, p.C);
    }
    if constexpr (GATE == 2) {
      float a[NV][VEC], slope[NV][VEC];
      load_sp(sp);
      PY::load(a, static_cast<const TY*>(p.gate) + seg / p.L * p.C, p.C);
      KAN_EACH {
        act_both(a[i][j], p.act, &a[i][j], &slope[i][j]);
        s_branch[i][j] += a[i][j] * s_gate[i][j];
        s_gate[i][j] *= sp[i][j] * slope[i][j];
      }
      if (p.dgate != nullptr) {
        const int64_t at = p.nchunk > 1 ? (int64_t)blockIdx.x : seg / p.L;
        flush_columns<TPR, WHOLE>(s_gate, p.part_gate + at * p.C, p.C, cols);
      }
      KAN_EACH s_gate[i][j] = 0.0f;
    }
    seg = end;
  }
  const int64_t at = (int64_t)blockIdx.x * p.C;
  if (p.part_pre != nullptr) flush_columns<TPR, WHOLE>(s_pre, p.part_pre + at, p.C, cols);
  if (p.part_branch != nullptr) flush_columns<TPR, WHOLE>(s_branch, p.part_branch + at, p.C, cols);
}

// Column sums of partial rows in a fixed order: 16 lanes of rows a column,
// their sums added in order.
constexpr int kSumRowLanes = 16;
__device__ __forceinline__ bool column_sum(const float* __restrict__ part, int64_t rows, int64_t C,
                                           int64_t* col, float* sum) {
  __shared__ float red[kSumRowLanes][64];
  const int lane = threadIdx.x & 63, rl = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane;
  float s = 0.0f;
  if (c < C) {
#pragma unroll 4
    for (int64_t r = rl; r < rows; r += kSumRowLanes) s += part[r * C + c];
  }
  red[rl][lane] = s;
  __syncthreads();
  if (rl != 0 || c >= C) return false;
#pragma unroll
  for (int w = 1; w < kSumRowLanes; ++w) s += red[w][lane];
  *col = c;
  *sum = s;
  return true;
}

// grid y 0: dpre; 1: dpost and dscale from their common sum.
__global__ __launch_bounds__(64 * kSumRowLanes) void norm_weights_kernel(
    NormParams p, int64_t rows, void* __restrict__ dpre, void* __restrict__ dpost,
    void* __restrict__ dscale) {
  int64_t c;
  float s;
  if (blockIdx.y == 0) {
    if (p.part_pre != nullptr && column_sum(p.part_pre, rows, p.C, &c, &s))
      store_any(dpre, c, p.wdtype, s);
  } else if (p.part_branch != nullptr && column_sum(p.part_branch, rows, p.C, &c, &s)) {
    if (dpost != nullptr)
      store_any(dpost, c, p.wdtype,
                s * (p.scale == nullptr ? p.scale_const : load_any(p.scale, c, p.wdtype)));
    if (dscale != nullptr)
      store_any(dscale, c, p.wdtype, p.post == nullptr ? s : s * load_any(p.post, c, p.wdtype));
  }
}

// dgate[g, c] = sum of the gate row's `rows` partial rows.
__global__ __launch_bounds__(64 * kSumRowLanes) void norm_gate_kernel(
    const float* __restrict__ part, int64_t rows, int64_t C, int64_t g0, void* __restrict__ dgate,
    int dtype) {
  const int64_t g = g0 + blockIdx.y;
  int64_t c;
  float s;
  if (column_sum(part + g * rows * C, rows, C, &c, &s)) store_any(dgate, g * C + c, dtype, s);
}

// out[g] = sum of part[g rows .. (g + 1) rows), one wave a sum.
__global__ __launch_bounds__(64) void sum_runs_kernel(const float* __restrict__ part, int64_t rows,
                                                      void* __restrict__ out, int dtype) {
  const int64_t g = blockIdx.x;
  float s = 0.0f;
  for (int64_t r = threadIdx.x; r < rows; r += 64) s += part[g * rows + r];
  s = wave_sum(s);
  if (threadIdx.x == 0) store_any(out, g, dtype, s);
}

constexpr int64_t kMaxGridY = 65535;

// Lanes that share a row of C values, 8 each (rows past kMaxHeld stay in memory,
// on blocks of 256).
constexpr int64_t kMaxHeld = 8192;
int held_tpr(int64_t C) {
  if (C > kMaxHeld) return 256;
  if (C <= 128) return C <= 64 ? 8 : 16;
  int tpr = 64;
  while (tpr * 8 < C) tpr *= 2;
  return tpr;
}

// How rows are dealt to blocks, and the backward's partial sums.
struct RowPlan {
  int64_t blocks, chunk, nchunk, seg_rows, gate_rows;  // gate_rows of part_gate
  size_t bytes;
};
constexpr int kGradWaves = 16;  // waves a CU (one block of the widest shape)
RowPlan row_plan(int64_t n, int64_t C, int kind, int64_t L, int waves_per_cu) {
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
bool whole_vectors(const NormParams& p, int vec, size_t xb, size_t yb) {
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

template <typename TX, typename TY, int TPR, int GATE, bool WHOLE>
int launch_held(NormParams p, int64_t grad_blocks, hipStream_t st) {
  typedef RowShape<TPR> S;
  constexpr int VEC = sizeof(TY) == 2 ? 8 : 4;
  if (grad_blocks > 0) {
    norm_grad_kernel<TX, TY, TPR, VEC, 8 / VEC, GATE, WHOLE>
        <<<dim3((unsigned)grad_blocks), S::kThreads, 0, st>>>(p);
    return check_launch("residual_norm_backward");
  }
  const RowPlan g = row_plan(p.n, p.C, p.gate_kind, p.L, 32);
  p.chunk = g.chunk;
  p.nchunk = g.nchunk;
  p.seg_rows = g.seg_rows;
  norm_kernel<TX, TY, TPR, VEC, 8 / VEC, GATE, WHOLE>
      <<<dim3((unsigned)g.blocks), S::kThreads, 0, st>>>(p);
  return check_launch("residual_norm");
}

template <typename TX, typename TY, int GATE, bool WHOLE>
int launch_tpr(const NormParams& p, int64_t grad_blocks, hipStream_t st) {
  switch (held_tpr(p.C)) {
    case 8: return launch_held<TX, TY, 8, GATE, WHOLE>(p, grad_blocks, st);
    case 16: return launch_held<TX, TY, 16, GATE, WHOLE>(p, grad_blocks, st);
    case 64: return launch_held<TX, TY, 64, GATE, WHOLE>(p, grad_blocks, st);
    case 128: return launch_held<TX, TY, 128, GATE, WHOLE>(p, grad_blocks, st);
    case 256: return launch_held<TX, TY, 256, GATE, WHOLE>(p, grad_blocks, st);
    case 512: return launch_held<TX, TY, 512, GATE, WHOLE>(p, grad_blocks, st);
    default: return launch_held<TX, TY, 1024, GATE, WHOLE>(p, grad_blocks, st);
  }
}

template <typename TX, typename TY, bool WHOLE>
int launch_gate(const NormParams& p, int64_t grad_blocks, hipStream_t st) {
  if (p.gate_kind == kGateElement) return launch_tpr<TX, TY, 1, WHOLE>(p, grad_blocks, st);
  if (p.gate_kind == kGateRows) return launch_tpr<TX, TY, 2, WHOLE>(p, grad_blocks, st);
  return launch_tpr<TX, TY, 0, WHOLE>(p, grad_blocks, st);
}

// grad_blocks > 0: the backward, on that many blocks.
template <typename TX, typename TY>
int launch_norm(const NormParams& p, int64_t grad_blocks, hipStream_t st) {
  if (p.C <= kMaxHeld)
    return whole_vectors(p, sizeof(TY) == 2 ? 8 : 4, sizeof(TX), sizeof(TY))
               ? launch_gate<TX, TY, true>(p, grad_blocks, st)
               : launch_gate<TX, TY, false>(p, grad_blocks, st);
  if (grad_blocks > 0) {
    norm_rows_grad_kernel<TX, TY><<<dim3((unsigned)grad_blocks), kRowThreads, 0, st>>>(p);
    return check_launch("residual_norm_backward");
  }
  const int64_t blocks = std::min<int64_t>(p.n, 16 * (int64_t)device_cu_count());
  norm_rows_kernel<TX, TY><<<dim3((unsigned)blocks), kRowThreads, 0, st>>>(p);
  return check_launch("residual_norm");
}

int check_norm(const char* who, int xdtype, int ydtype, int wdtype, const void* x, const void* y,
               const void* gate, const void* post, const void* scale, int gate_act,
               int64_t gate_rows, int64_t gate_cols, int64_t n, int64_t C, NormParams* p) {
  if (!dtype_is_operator(xdtype) || !dtype_is_operator(ydtype) || !dtype_is_operator(wdtype))
    return set_error(KAN_ERR_INVALID, "%s: dtype codes must be FP32, BF16 or FP16", who);
  if (xdtype != ydtype && xdtype != KAN_DTYPE_F32)
    return set_error(KAN_ERR_INVALID, "%s: the stream is in the branch's type or in FP32", who);
  if (n < 0 || C < 0) return set_error(KAN_ERR_INVALID, "%s: negative size", who);
  if (gate_act < KAN_GATE_IDENTITY || gate_act > KAN_GATE_SILU)
    return set_error(KAN_ERR_INVALID, "%s: unknown gate activation %d", who, gate_act);
  if (y == nullptr && (gate != nullptr || post != nullptr || scale != nullptr))
    return set_error(KAN_ERR_INVALID, "%s: gate, post_weight and scale need a branch", who);
  p->gate_kind = kGateNone;
  p->L = 1;
  if (gate != nullptr) {
    if (gate_rows < 1 || n % gate_rows != 0 || (gate_cols != 1 && gate_cols != C))
      return set_error(KAN_ERR_INVALID,
                       "%s: a gate has rows that divide n and 1 or C columns, got [%lld, %lld]", who,
                       (long long)gate_rows, (long long)gate_cols);
    p->L = n / gate_rows;
    if (gate_cols == C && C > 1) p->gate_kind = p->L == 1 ? kGateElement : kGateRows;
    else p->gate_kind = p->L == 1 ? kGateToken : kGateScalars;
  }
  p->x = x;
  p->y = y;
  p->gate = gate;
  p->post = post;
  p->scale = scale;
  p->act = gate_act;
  p->wdtype = wdtype;
  p->n = n;
  p->C = C;
  return KAN_OK;
}

#define KAN_NORM_TYPES(xd, yd, CALL)                                          \
  (xd == KAN_DTYPE_F32 ? (yd == KAN_DTYPE_F32    ? CALL(float, float)         \
                          : yd == KAN_DTYPE_BF16 ? CALL(float, bf16)          \
                                                 : CALL(float, f16))          \
   : xd == KAN_DTYPE_BF16 ? CALL(bf16, bf16)                                  \
                          : CALL(f16, f16))

}  // namespace
}  // namespace kan

using namespace kan;

extern "C" {

int kan_hip_residual_norm(int xdtype, int ydtype, int wdtype, const void* x, const void* y,
                          const void* gate, const void* post_weight, const void* pre_weight,
                          const void* scale, double scale_const, int gate_act, int64_t gate_rows,
                          int64_t gate_cols, int64_t n, int64_t C, double eps, void* x_out,
                          void* h_out, float* rstd, void* stream) {
  NormParams p{};
  const int rc = check_norm("residual_norm", xdtype, ydtype, wdtype, x, y, gate, post_weight, scale,
                            gate_act, gate_rows, gate_cols, n, C, &p);
  if (rc != KAN_OK) return rc;
  if (n == 0 || C == 0) return KAN_OK;
  if (x == nullptr) return set_error(KAN_ERR_INVALID, "residual_norm: x must not be NULL");
  if ((h_out == nullptr) != (pre_weight == nullptr))
    return set_error(KAN_ERR_INVALID, "residual_norm: h_out and pre_weight go together");
  if (x_out == nullptr && h_out == nullptr) return KAN_OK;
  p.pre = pre_weight;
  p.x_out = x_out;
  p.h_out = h_out;
  p.rstd = rstd;
  p.scale_const = (float)scale_const;
  p.eps = (float)eps;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const double moved = (double)n * C *
                       (dtype_bytes(xdtype) * (x_out != nullptr ? 2 : 1) +
                        dtype_bytes(ydtype) * ((y != nullptr) + (h_out != nullptr)));
  TimedLaunch timed(kClassOther, st, moved);
#define KAN_CALL(TX, TY) launch_norm<TX, TY>(p, 0, st)
  return KAN_NORM_TYPES(xdtype, ydtype, KAN_CALL);
#undef KAN_CALL
}

int kan_hip_residual_norm_backward_workspace(int64_t gate_rows, int64_t gate_cols, int64_t n,
                                             int64_t C, size_t* bytes) {
  if (bytes == nullptr)
    return set_error(KAN_ERR_INVALID, "residual_norm_backward_workspace: bytes must not be NULL");
  NormParams p{};
  const int rc = check_norm("residual_norm_backward", KAN_DTYPE_F32, KAN_DTYPE_F32, KAN_DTYPE_F32,
                            &p, &p, gate_rows > 0 ? &p : nullptr, nullptr, nullptr, 0, gate_rows,
                            gate_cols, n, C, &p);
  if (rc != KAN_OK) return rc;
  *bytes = n == 0 || C == 0 ? 0 : row_plan(n, C, p.gate_kind, p.L, kGradWaves).bytes;
  return KAN_OK;
}

int kan_hip_residual_norm_backward(int xdtype, int ydtype, int wdtype, const void* grad_x_out,
                                   const void* grad_h, const void* x, const void* y,
                                   const void* gate, const void* post_weight,
                                   const void* pre_weight, const void* scale, double scale_const,
                                   int gate_act, int64_t gate_rows, int64_t gate_cols, int64_t n,
                                   int64_t C, const float* rstd, void* grad_x, void* grad_y,
                                   void* grad_gate, void* grad_post, void* grad_pre,
                                   void* grad_scale, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  const char* who = "residual_norm_backward";
  NormParams p{};
  const int rc = check_norm(who, xdtype, ydtype, wdtype, x, y, gate, post_weight, scale, gate_act,
                            gate_rows, gate_cols, n, C, &p);
  if (rc != KAN_OK) return rc;
  if ((grad_y != nullptr && y == nullptr) || (grad_gate != nullptr && gate == nullptr) ||
      (grad_post != nullptr && post_weight == nullptr) ||
      (grad_scale != nullptr && scale == nullptr) || (grad_pre != nullptr && grad_h == nullptr) ||
      (grad_h != nullptr && pre_weight == nullptr))
    return set_error(KAN_ERR_INVALID, "%s: a gradient of an absent operand", who);
  if (n == 0 || C == 0) return KAN_OK;
  if (x == nullptr || rstd == nullptr)
    return set_error(KAN_ERR_INVALID, "%s: x and rstd must not be NULL", who);
  const RowPlan g = row_plan(n, C, p.gate_kind, p.L, kGradWaves);
  if (workspace == nullptr || workspace_bytes < g.bytes)
    return set_error(KAN_ERR_WORKSPACE, "%s: needs %zu bytes of workspace, got %zu", who, g.bytes,
                     workspace == nullptr ? (size_t)0 : workspace_bytes);
  float* ws = static_cast<float*>(workspace);
  const int64_t row_part = g.blocks * C;
  p.pre = grad_h == nullptr ? nullptr : pre_weight;
  p.part_pre = grad_pre == nullptr ? nullptr : ws;
  p.part_branch = grad_post == nullptr && grad_scale == nullptr ? nullptr : ws + row_part;
  p.part_gate = grad_gate == nullptr ? nullptr : ws + 2 * row_part;
  p.dxo = grad_x_out;
  p.dh = grad_h;
  p.dx = grad_x;
  p.dy = grad_y;
  p.dgate = grad_gate;
  p.rstd = const_cast<float*>(rstd);
  p.chunk = g.chunk;
  p.nchunk = g.nchunk;
  p.seg_rows = g.seg_rows;
  p.scale_const = (float)scale_const;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const double moved =
      (double)n * C *
      (dtype_bytes(xdtype) * (1 + (grad_x_out != nullptr) + (grad_x != nullptr)) +
       dtype_bytes(ydtype) * ((y != nullptr) + (grad_h != nullptr) + (grad_y != nullptr)));
  {
    TimedLaunch timed(kClassOther, st, moved);
#define KAN_CALL(TX, TY) launch_norm<TX, TY>(p, g.blocks, st)
    const int e = KAN_NORM_TYPES(xdtype, ydtype, KAN_CALL);
#undef KAN_CALL
    if (e != KAN_OK) return e;
  }
  const unsigned cols = (unsigned)ceil_div(C, 64);
  TimedLaunch timed(kClassOther, st, (double)g.bytes);
  if (p.part_pre != nullptr || p.part_branch != nullptr)
    norm_weights_kernel<<<dim3(cols, 2), 64 * kSumRowLanes, 0, st>>>(p, g.blocks, grad_pre,
                                                                    grad_post, grad_scale);
  if (grad_gate != nullptr && p.gate_kind == kGateRows) {
    for (int64_t g0 = 0; g0 < n / p.L; g0 += kMaxGridY)
      norm_gate_kernel<<<dim3(cols, (unsigned)std::min(kMaxGridY, n / p.L - g0)),
                         64 * kSumRowLanes, 0, st>>>(p.part_gate, g.nchunk, C, g0, grad_gate,
                                                     ydtype);
  }
  if (grad_gate != nullptr && p.gate_kind == kGateScalars)
    sum_runs_kernel<<<dim3((unsigned)(n / p.L)), 64, 0, st>>>(p.part_gate, p.L, grad_gate, ydtype);
  return check_launch(who);
}

}  // extern "C"
