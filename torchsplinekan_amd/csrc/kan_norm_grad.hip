// Residual norm (kan_norm.h): the backward's kernels.
#include "kan_norm.h"

namespace kan {

namespace {

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

// Bound by HBM: 16384 x 4096 bf16 with a gate row for 2048 rows 178 us (805 MB
// and 25 of partial sums, 4.6 TB/s); 32768 x 1024 float32 150 us, 5.4 TB/s.
// Four waves a SIMD, two for a float32 row of 512 lanes with a gate.  In the 128
// registers that four leave not every row fits; the compiler keeps in scratch, a
// lane: 52 to 92 bytes of 16-bit rows with a gate row (76 at the size above), up to
// 28 without; 44 to 120 of a float32 stream with a 16-bit gate for every element;
// 92 to 388 of float32 rows of 8 or 16 lanes, up to 28 of longer ones; and 196 to 584 of
// all rows of more than 8192 columns (4096 x 16384 bf16 0.58 ms, their bytes 0.17).
// dpost = scale * (sum of D a yh) and dscale = post * (the same sum): one column
// sum serves both, a weight's factor applied after it.  A gate row's gradient
// comes from the sum of D yh, times scale, post and a'(g), and what its rows add to
// the first sum is a(g) times the same: two sums a row.  In 16 bits the next row's
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

struct GradLaunch {
  NormParams p;
  int64_t blocks;
  hipStream_t st;
  template <typename TX, typename TY, int TPR, int VALS, int GATE, bool WHOLE>
  int run() const {
    constexpr int VEC = sizeof(TY) == 2 ? 8 : 4;
    norm_grad_kernel<TX, TY, TPR, VEC, VALS / VEC, GATE, WHOLE>
        <<<dim3((unsigned)blocks), RowShape<TPR>::kThreads, 0, st>>>(p);
    return check_launch("residual_norm_backward");
  }
  template <typename TX, typename TY>
  int rows() const {
    norm_rows_grad_kernel<TX, TY><<<dim3((unsigned)blocks), kRowThreads, 0, st>>>(p);
    return check_launch("residual_norm_backward");
  }
};

}  // namespace

int launch_norm_grad(const NormParams& p, const RowPlan& g, int xdtype, int ydtype, void* dpre,
                     void* dpost, void* dscale, hipStream_t st) {
  const int rc = launch_norm(GradLaunch{p, g.blocks, st}, p, xdtype, ydtype);
  if (rc != KAN_OK) return rc;
  const unsigned cols = (unsigned)ceil_div(p.C, 64);
  if (p.part_pre != nullptr || p.part_branch != nullptr)
    norm_weights_kernel<<<dim3(cols, 2), 64 * kSumRowLanes, 0, st>>>(p, g.blocks, dpre, dpost,
                                                                    dscale);
  if (p.dgate != nullptr && p.gate_kind == kGateRows) {
    constexpr int64_t kMaxGridY = 65535;
    for (int64_t g0 = 0; g0 < p.n / p.L; g0 += kMaxGridY)
      norm_gate_kernel<<<dim3(cols, (unsigned)std::min(kMaxGridY, p.n / p.L - g0)),
                         64 * kSumRowLanes, 0, st>>>(p.part_gate, g.nchunk, p.C, g0, p.dgate,
                                                     ydtype);
  }
  if (p.dgate != nullptr && p.gate_kind == kGateScalars)
    sum_runs_kernel<<<dim3((unsigned)(p.n / p.L)), 64, 0, st>>>(p.part_gate, p.L, p.dgate, ydtype);
  return check_launch("residual_norm_backward");
}

}  // namespace kan
