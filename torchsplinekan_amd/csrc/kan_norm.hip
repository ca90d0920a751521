// Residual norm (kan_norm.h): the forward's kernels and the C entries.
#include "kan_norm.h"

namespace kan {

namespace {

// A row read again in every pass, from its XCD's L2: 0.8 TB/s at 4096 x 16384
// bf16 (107 us in registers, 659 so), which is why only wider rows come here.
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

// GATE: 0 none or one value a row, 1 a value for every element, 2 a row of
// values for L rows, evaluated once for all of them that a block has (row by row
// tanhf alone took the VALU as long as the loads: 146 us against 122 at 16384 x
// 4096 bf16).  Bound by HBM: there 4.4 TB/s of 537 MB; 65536 x 512 bf16 without
// a gate 49 us, 5.4 TB/s; 262144 x 64 23 us, 5.8 TB/s.
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

struct ForwardLaunch {
  NormParams p;
  hipStream_t st;
  template <typename TX, typename TY, int TPR, int VALS, int GATE, bool WHOLE>
  int run() const {
    constexpr int VEC = sizeof(TY) == 2 ? 8 : 4;
    const RowPlan g = row_plan(p.n, p.C, p.gate_kind, p.L, 32);
    NormParams q = p;
    q.chunk = g.chunk;
    q.nchunk = g.nchunk;
    q.seg_rows = g.seg_rows;
    norm_kernel<TX, TY, TPR, VEC, VALS / VEC, GATE, WHOLE>
        <<<dim3((unsigned)g.blocks), RowShape<TPR>::kThreads, 0, st>>>(q);
    return check_launch("residual_norm");
  }
  template <typename TX, typename TY>
  int rows() const {
    const int64_t blocks = std::min<int64_t>(p.n, 16 * (int64_t)device_cu_count());
    norm_rows_kernel<TX, TY><<<dim3((unsigned)blocks), kRowThreads, 0, st>>>(p);
    return check_launch("residual_norm");
  }
};

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
  return launch_norm(ForwardLaunch{p, st}, p, xdtype, ydtype);
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
  TimedLaunch timed(kClassOther, st, moved);
  return launch_norm_grad(p, g, xdtype, ydtype, grad_pre, grad_post, grad_scale, st);
}

}  // extern "C"
