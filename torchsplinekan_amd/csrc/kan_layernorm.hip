// Layer norm over n rows of C values,
//   m = mean(x),  r = (mean((x - m)^2) + eps)^(-1/2),  xh = (x - m) r,
//   y = weight * xh + bias,
// and its backward pass: with t = dy weight
//   dx = r (t - mean(t) - xh mean(t xh)),  dweight = sum_rows dy xh,  dbias = sum_rows dy.
//
// A row lies in the registers of 8 to 1024 lanes (kan_norm.h), so that the
// variance is taken of the values less their mean without a second read.  The mean of
// what is left of the values goes into the mean: a constant row becomes zero, and rows far
// from zero are off by the mean's own rounding.  All arithmetic is in float32, rounded once where a result is stored.  The column
// sums go through one partial row a block, added in block order: no atomics, the
// same bits every time.  Bound by HBM: 16384 rows of 4096 in bf16, forward 47 us (5.7
// TB/s, part of it from the last-level cache), forward and backward 138 us for 671 MB (135
// without the mean's second part); 32768 x 1024 in float32 42 and 140 us.
#include "kan_norm.h"

namespace kan {

namespace {

struct LayerNormParams {
  const void *x, *w, *b, *dy;
  void *y, *dx;
  float* stats;            // [2, n]: m, r (optional in the forward)
  float *part_w, *part_b;  // [blocks, C]
  int64_t n, C, chunk;     // rows of a block
  float eps;
  int wdtype;
};

// Lanes of a row: 8 values each, or 16 in rows of more than 8192.  (129 .. 256 columns
// in 32 lanes: the other norms' row shapes have none between 16 and 64.)
inline int row_lanes(int64_t C) {
  if (C > 128 && C <= 256) return 32;
  return held_tpr(C);
}
struct Rows {
  int64_t blocks, chunk;
};
inline Rows plan_rows(int64_t n, int64_t C, int waves_per_cu) {
  const int tpr = row_lanes(C), threads = tpr <= 64 ? 256 : tpr;
  const int64_t target = device_cu_count() * (int64_t)std::max(1, 64 * waves_per_cu / threads);
  const int64_t chunk = round_up(std::max<int64_t>(1, ceil_div(n, target)), threads / tpr);
  return {ceil_div(n, chunk), chunk};
}

// The squares of values less m + d are those less m, less d^2: taken so where d^2 is
// below this part of the variance, and its rounding with it.
constexpr float kShift = 1.0f / 1024;
template <typename TX, typename TY, int TPR, int VEC, int NV, bool WHOLE>
__global__ __launch_bounds__(RowShape<TPR>::kThreads) void layer_norm_kernel(LayerNormParams p) {
  typedef RowShape<TPR> S;
  typedef Pieces<TX, TPR, VEC, NV, WHOLE> PX;
  typedef Pieces<TY, TPR, VEC, NV, WHOLE> PY;
  __shared__ float red[4 * S::kWaves];
  int turn = 0;
  const float inv_c = 1.0f / (float)p.C;
  float w[NV][VEC], b[NV][VEC];
  load_weight<TPR, WHOLE>(w, p.w, p.wdtype, p.C, 1.0f);
  load_weight<TPR, WHOLE>(b, p.b, p.wdtype, p.C, 0.0f);
  const int64_t lo = (int64_t)blockIdx.x * p.chunk, end = min(p.n, lo + p.chunk);
  // (every wave of a row takes the same number of turns)
  for (int64_t r0 = lo; r0 < end; r0 += S::kRows) {
    const int64_t row = r0 + threadIdx.x / TPR;
    if (S::kRows > 1 && row >= end) break;
    float x[NV][VEC];
    PX::load(x, static_cast<const TX*>(p.x) + row * p.C, p.C);
    float s[1] = {0.0f};
    KAN_EACH s[0] += x[i][j];
    row_sums<TPR>(s, red, turn);
    float m = s[0] / (float)p.C;
    float t[2] = {0.0f, 0.0f};
    KAN_EACH {
      const float d = PX::at(i) + j < p.C ? x[i][j] - m : 0.0f;
      t[0] += d;
      t[1] += d * d;
    }
    row_sums<TPR>(t, red, turn);
    // (the sum over C values was off by a few units in m's last place, and so is d)
    const float d = t[0] * inv_c;
    m += d;
    float var = t[1] * inv_c - d * d;
    if (!(d * d <= kShift * var)) {  // (all of a row alike; its squares may be beyond a float)
      s[0] = 0.0f;
      KAN_EACH {
        const float v = PX::at(i) + j < p.C ? x[i][j] - m : 0.0f;
        s[0] += v * v;
      }
      row_sums<TPR>(s, red, turn);
      var = s[0] * inv_c;
    }
    const float r = 1.0f / sqrtf(var + p.eps);
    if (p.stats != nullptr && threadIdx.x % TPR == 0) {
      p.stats[row] = m;
      p.stats[p.n + row] = r;
    }
    KAN_EACH x[i][j] = (x[i][j] - m) * r * w[i][j] + b[i][j];
    PY::store(x, static_cast<TY*>(p.y) + row * p.C, p.C);
  }
}

template <typename TX, typename TY, int TPR, int VEC, int NV, bool WHOLE>
__global__ __launch_bounds__(RowShape<TPR>::kThreads) void layer_norm_grad_kernel(
    LayerNormParams p) {
  typedef RowShape<TPR> S;
  typedef Pieces<TX, TPR, VEC, NV, WHOLE> PX;
  typedef Pieces<TY, TPR, VEC, NV, WHOLE> PY;
  constexpr int kCols = S::kRows > 1 ? NV * VEC * S::kThreads : 1;
  __shared__ float red[4 * S::kWaves];
  __shared__ float cols[kCols];
  int turn = 0;
  const float inv_c = 1.0f / (float)p.C;
  float w[NV][VEC], sw[NV][VEC] = {}, sb[NV][VEC] = {};
  load_weight<TPR, WHOLE>(w, p.w, p.wdtype, p.C, 1.0f);
  const int64_t lo = (int64_t)blockIdx.x * p.chunk, end = min(p.n, lo + p.chunk);
  for (int64_t r0 = lo; r0 < end; r0 += S::kRows) {
    const int64_t row = r0 + threadIdx.x / TPR;
    if (S::kRows > 1 && row >= end) break;
    float x[NV][VEC], dy[NV][VEC];
    PX::load(x, static_cast<const TX*>(p.x) + row * p.C, p.C);
    PY::load(dy, static_cast<const TY*>(p.dy) + row * p.C, p.C);
    const float m = p.stats[row], r = p.stats[p.n + row];
    float s[2] = {0.0f, 0.0f};
    KAN_EACH {  // (past the row's end dy is zero, and so is what it adds)
      x[i][j] = (x[i][j] - m) * r;
      sw[i][j] += dy[i][j] * x[i][j];
      sb[i][j] += dy[i][j];
      dy[i][j] *= w[i][j];
      s[0] += dy[i][j];
      s[1] += dy[i][j] * x[i][j];
    }
    if (p.dx == nullptr) continue;
    row_sums<TPR>(s, red, turn);
    const float m1 = s[0] * inv_c, m2 = s[1] * inv_c;
    KAN_EACH dy[i][j] = r * (dy[i][j] - m1 - x[i][j] * m2);
    PX::store(dy, static_cast<TX*>(p.dx) + row * p.C, p.C);
  }
  const int64_t at = (int64_t)blockIdx.x * p.C;
  if (p.part_w != nullptr) flush_columns<TPR, WHOLE>(sw, p.part_w + at, p.C, cols);
  if (p.part_b != nullptr) flush_columns<TPR, WHOLE>(sb, p.part_b + at, p.C, cols);
}

// Rows wider than registers hold, one at a time, read again in every pass (4096 x 16392
// in bf16: forward 217 us, 16384 columns 52).
template <typename TX, typename TY>
__global__ __launch_bounds__(kRowThreads) void layer_norm_rows_kernel(LayerNormParams p) {
  __shared__ float red[kRowThreads / 64];
  const float inv_c = 1.0f / (float)p.C;
  for (int64_t row = blockIdx.x; row < p.n; row += gridDim.x) {
    const TX* x = static_cast<const TX*>(p.x) + row * p.C;
    float s = 0.0f;
    for (int64_t c = threadIdx.x; c < p.C; c += kRowThreads) s += (float)x[c];
    float m = block_sum(s, red) / (float)p.C, t = 0.0f;
    s = 0.0f;
    for (int64_t c = threadIdx.x; c < p.C; c += kRowThreads) {
      const float v = (float)x[c] - m;
      t += v;
      s += v * v;
    }
    const float d = block_sum(t, red) * inv_c;
    m += d;
    float var = block_sum(s, red) * inv_c - d * d;
    if (!(d * d <= kShift * var)) {  // (as above)
      s = 0.0f;
      for (int64_t c = threadIdx.x; c < p.C; c += kRowThreads) {
        const float v = (float)x[c] - m;
        s += v * v;
      }
      var = block_sum(s, red) * inv_c;
    }
    const float r = 1.0f / sqrtf(var + p.eps);
    if (p.stats != nullptr && threadIdx.x == 0) {
      p.stats[row] = m;
      p.stats[p.n + row] = r;
    }
    for (int64_t c = threadIdx.x; c < p.C; c += kRowThreads) {
      const float w = p.w == nullptr ? 1.0f : load_any(p.w, c, p.wdtype);
      const float b = p.b == nullptr ? 0.0f : load_any(p.b, c, p.wdtype);
      static_cast<TY*>(p.y)[row * p.C + c] = (TY)(((float)x[c] - m) * r * w + b);
    }
  }
}

// (A thread has the columns threadIdx.x + i kRowThreads of every row of its
// block, so the partial sums are plain reads and writes of its own.)
template <typename TX, typename TY>
__global__ __launch_bounds__(kRowThreads) void layer_norm_rows_grad_kernel(LayerNormParams p) {
  __shared__ float red[kRowThreads / 64];
  const float inv_c = 1.0f / (float)p.C;
  const int64_t lo = (int64_t)blockIdx.x * p.chunk, end = min(p.n, lo + p.chunk);
  const int64_t part = (int64_t)blockIdx.x * p.C;
  for (int64_t row = lo; row < end; ++row) {
    const TX* x = static_cast<const TX*>(p.x) + row * p.C;
    const TY* dy = static_cast<const TY*>(p.dy) + row * p.C;
    const float m = p.stats[row], r = p.stats[p.n + row];
    float s1 = 0.0f, s2 = 0.0f;
    for (int64_t c = threadIdx.x; c < p.C; c += kRowThreads) {
      const float d = (float)dy[c], xh = ((float)x[c] - m) * r;
      const float t = p.w == nullptr ? d : d * load_any(p.w, c, p.wdtype);
      s1 += t;
      s2 += t * xh;
      if (p.part_w != nullptr) p.part_w[part + c] = (row == lo ? 0.0f : p.part_w[part + c]) + d * xh;
      if (p.part_b != nullptr) p.part_b[part + c] = (row == lo ? 0.0f : p.part_b[part + c]) + d;
    }
    if (p.dx == nullptr) continue;
    const float m1 = block_sum(s1, red) * inv_c;
    const float m2 = block_sum(s2, red) * inv_c;
    for (int64_t c = threadIdx.x; c < p.C; c += kRowThreads) {
      const float d = (float)dy[c], xh = ((float)x[c] - m) * r;
      const float t = p.w == nullptr ? d : d * load_any(p.w, c, p.wdtype);
      static_cast<TX*>(p.dx)[row * p.C + c] = (TX)(r * (t - m1 - xh * m2));
    }
  }
}

// grid y 0: dweight; 1: dbias.
__global__ __launch_bounds__(64 * kSumRowLanes) void layer_norm_weights_kernel(
    LayerNormParams p, int64_t rows, void* __restrict__ dw, void* __restrict__ db) {
  int64_t c;
  float s;
  const float* part = blockIdx.y == 0 ? p.part_w : p.part_b;
  if (part != nullptr && column_sum(part, rows, p.C, &c, &s))
    store_any(blockIdx.y == 0 ? dw : db, c, p.wdtype, s);
}

template <bool GRAD>
struct LayerNormLaunch {
  LayerNormParams p;
  int64_t blocks;
  hipStream_t st;
  template <typename TX, typename TY, int TPR, int VALS, bool WHOLE>
  void shape() const {
    constexpr int VEC = sizeof(TY) == 2 ? 8 : 4;
    if constexpr (GRAD)
      layer_norm_grad_kernel<TX, TY, TPR, VEC, VALS / VEC, WHOLE>
          <<<dim3((unsigned)blocks), RowShape<TPR>::kThreads, 0, st>>>(p);
    else
      layer_norm_kernel<TX, TY, TPR, VEC, VALS / VEC, WHOLE>
          <<<dim3((unsigned)blocks), RowShape<TPR>::kThreads, 0, st>>>(p);
  }
  template <typename TX, typename TY, bool WHOLE>
  void held() const {
    switch (row_lanes(p.C)) {
      case 8: return shape<TX, TY, 8, 8, WHOLE>();
      case 16: return shape<TX, TY, 16, 8, WHOLE>();
      case 32: return shape<TX, TY, 32, 8, WHOLE>();
      case 64: return shape<TX, TY, 64, 8, WHOLE>();
      case 128: return shape<TX, TY, 128, 8, WHOLE>();
      case 256: return shape<TX, TY, 256, 8, WHOLE>();
      case 512: return shape<TX, TY, 512, 8, WHOLE>();
      default:
        return p.C <= 8192 ? shape<TX, TY, 1024, 8, WHOLE>() : shape<TX, TY, 1024, 16, WHOLE>();
    }
  }
  template <typename TX, typename TY>
  int typed() const {
    constexpr int64_t VEC = sizeof(TY) == 2 ? 8 : 4;
    auto ok = [](const void* q, size_t bytes) {
      return reinterpret_cast<uintptr_t>(q) % std::min<size_t>(bytes, 16) == 0;
    };
    if (p.C > kMaxHeld) {
      if constexpr (GRAD)
        layer_norm_rows_grad_kernel<TX, TY><<<dim3((unsigned)blocks), kRowThreads, 0, st>>>(p);
      else
        layer_norm_rows_kernel<TX, TY><<<dim3((unsigned)blocks), kRowThreads, 0, st>>>(p);
    } else if (p.C % VEC == 0 && ok(p.x, VEC * sizeof(TX)) && ok(p.dx, VEC * sizeof(TX)) &&
               ok(p.y, VEC * sizeof(TY)) && ok(p.dy, VEC * sizeof(TY)) && ok(p.w, 16) &&
               ok(p.b, 16)) {
      held<TX, TY, true>();
    } else {
      held<TX, TY, false>();
    }
    return check_launch(GRAD ? "layer_norm_backward" : "layer_norm");
  }
  int run(int xdtype, int ydtype) const {
    if (xdtype == KAN_DTYPE_BF16) return typed<bf16, bf16>();
    if (xdtype == KAN_DTYPE_F16) return typed<f16, f16>();
    if (ydtype == KAN_DTYPE_BF16) return typed<float, bf16>();
    if (ydtype == KAN_DTYPE_F16) return typed<float, f16>();
    return typed<float, float>();
  }
};

int check_layer_norm(const char* who, int xdtype, int ydtype, int wdtype, int64_t n, int64_t C) {
  if (!dtype_is_operator(xdtype) || !dtype_is_operator(ydtype) || !dtype_is_operator(wdtype))
    return set_error(KAN_ERR_INVALID, "%s: dtype codes must be FP32, BF16 or FP16", who);
  if (xdtype != ydtype && xdtype != KAN_DTYPE_F32)
    return set_error(KAN_ERR_INVALID, "%s: x is in y's type or in FP32", who);
  if (n < 0 || C < 0) return set_error(KAN_ERR_INVALID, "%s: negative size", who);
  return KAN_OK;
}

constexpr int kForwardWaves = 32;  // waves a CU
size_t grad_bytes(int64_t n, int64_t C) {
  return n == 0 || C == 0 ? 0 : 2 * 4 * (size_t)(plan_rows(n, C, kGradWaves).blocks * C);
}

}  // namespace
}  // namespace kan

using namespace kan;

extern "C" {

int kan_hip_layer_norm(int xdtype, int ydtype, int wdtype, const void* x, const void* weight,
                       const void* bias, int64_t n, int64_t C, double eps, void* y, float* stats,
                       void* stream) {
  const int rc = check_layer_norm("layer_norm", xdtype, ydtype, wdtype, n, C);
  if (rc != KAN_OK) return rc;
  if (n == 0 || C == 0) return KAN_OK;
  if (x == nullptr || y == nullptr)
    return set_error(KAN_ERR_INVALID, "layer_norm: x and y must not be NULL");
  LayerNormParams p{};
  p.x = x;
  p.w = weight;
  p.b = bias;
  p.y = y;
  p.stats = stats;
  p.n = n;
  p.C = C;
  p.eps = (float)eps;
  p.wdtype = wdtype;
  const Rows rows = plan_rows(n, C, kForwardWaves);
  p.chunk = rows.chunk;
  const int64_t blocks =
      C > kMaxHeld ? std::min<int64_t>(n, 16 * (int64_t)device_cu_count()) : rows.blocks;
  hipStream_t st = static_cast<hipStream_t>(stream);
  TimedLaunch timed(kClassOther, st, (double)n * C * (dtype_bytes(xdtype) + dtype_bytes(ydtype)));
  return LayerNormLaunch<false>{p, blocks, st}.run(xdtype, ydtype);
}

int kan_hip_layer_norm_backward_workspace(int64_t n, int64_t C, size_t* bytes) {
  if (bytes == nullptr)
    return set_error(KAN_ERR_INVALID, "layer_norm_backward_workspace: bytes must not be NULL");
  if (n < 0 || C < 0)
    return set_error(KAN_ERR_INVALID, "layer_norm_backward_workspace: negative size");
  *bytes = grad_bytes(n, C);
  return KAN_OK;
}

int kan_hip_layer_norm_backward(int xdtype, int ydtype, int wdtype, const void* grad_y,
                                const void* x, const void* weight, const float* stats, int64_t n,
                                int64_t C, void* grad_x, void* grad_weight, void* grad_bias,
                                void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "layer_norm_backward";
  const int rc = check_layer_norm(who, xdtype, ydtype, wdtype, n, C);
  if (rc != KAN_OK) return rc;
  if (n == 0 || C == 0) return KAN_OK;
  if (x == nullptr || grad_y == nullptr || stats == nullptr)
    return set_error(KAN_ERR_INVALID, "%s: grad_y, x and stats must not be NULL", who);
  const size_t need = grad_weight != nullptr || grad_bias != nullptr ? grad_bytes(n, C) : 0;
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return set_error(KAN_ERR_WORKSPACE, "%s: needs %zu bytes of workspace, got %zu", who, need,
                     workspace == nullptr ? (size_t)0 : workspace_bytes);
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
    return set_error(KAN_ERR_INVALID, "%s: the workspace lies on 16 bytes", who);
  const Rows rows = plan_rows(n, C, kGradWaves);
  LayerNormParams p{};
  p.x = x;
  p.w = weight;
  p.dy = grad_y;
  p.dx = grad_x;
  p.stats = const_cast<float*>(stats);
  p.n = n;
  p.C = C;
  p.chunk = rows.chunk;
  p.wdtype = wdtype;
  float* ws = static_cast<float*>(workspace);
  if (grad_weight != nullptr) p.part_w = ws;
  if (grad_bias != nullptr) p.part_b = ws + rows.blocks * C;
  hipStream_t st = static_cast<hipStream_t>(stream);
  TimedLaunch timed(kClassOther, st,
                    (double)n * C * (2 * dtype_bytes(xdtype) + dtype_bytes(ydtype)));
  const int e = LayerNormLaunch<true>{p, rows.blocks, st}.run(xdtype, ydtype);
  if (e != KAN_OK || need == 0) return e;
  layer_norm_weights_kernel<<<dim3((unsigned)ceil_div(C, 64), 2), 64 * kSumRowLanes, 0, st>>>(
      p, rows.blocks, grad_weight, grad_bias);
  return check_launch(who);
}

}  // extern "C"
