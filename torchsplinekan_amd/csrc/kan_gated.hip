// Gated products: rows x [T, K], sorted by expert as those of the grouped products
// (kan_grouped.h) or all of one, and two weights of [N, K] an expert, gate and up:
//   g = x gate^T,  u = x up^T,  h = act(g) u                         [T, N]
// and the part of the backward pass that is no product:
//   dg = dh u act'(g),  du = dh act(g),                              [T, 2 N]
// from which dx = [dg du] [gate; up] and d[gate; up] = [dg du]^T x are grouped
// products.
//
// Both projections, the activation and the product are one kernel: a tile's 256
// columns are 32 of the gate and the same 32 of up in turn, so that a wave holds
// g and u of the same outputs.  Sums and everything behind them are in float32,
// and h is rounded once.
//
// What the backward pass needs of g and u is kept as words with their sign,
// exponent and leading 7 bits of mantissa, and 4 (bf16) or 8 (f16) bits more of
// each in a second array: 20 or 24 bits.  Gradients are then off by what the
// operands of their products and their own rounding make (normwise 0.0023 in bf16,
// 0.00030 in f16, where [dg du] is stored times a power of 2 if its largest value asks for
// it); with g and u in the type itself they would be off by 0.0029 and
// 0.00037, and in float32 the kept values and the bytes both passes move for them
// would be 1.6 (1.3) times as many.
#include "kan_grouped.h"
#include "kan_norm.h"
#include "kan_tile.h"

namespace kan {

namespace {

struct GatedParams : GroupedParams {  // N: outputs; B [E, 2 N, K]; C: h
  void* pre;  // null: not kept.  fp32: [T, 2 N]; 16 bits: words [T, 2 N]
  void* low;  // 16 bits: [T, N], the low bits of g before those of u
  int act;
  float* factor;  // null, or [kScaleValues]: the gradients' factor, then largest values
  int parts;      // how many of those
};

// bytes of the words, on 16
inline size_t word_bytes(int64_t T, int64_t N) { return (size_t)round_up(4 * T * N, 16); }

// ---- activations --------------------------------------------------------------
// For 16-bit results: exponentials and reciprocals of the hardware, off by a few units of
// 2^-24 and by |v| more, for the rounding of the exponential's argument.
__device__ __forceinline__ float quick_sigmoid(float v) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * v));
}
__device__ __forceinline__ float normal_cdf(float v) {  // (exact far below 0 too)
  return 0.5f * erfcf(-0.70710678f * v);
}
// act(v) and act'(v)
template <bool QUICK>
__device__ __forceinline__ void gated_act(float v, int act, float* a, float* slope) {
  auto sigmoid = [](float t) { return QUICK ? quick_sigmoid(t) : sigmoid_of(t); };
  switch (act) {
    case KAN_GATE_SIGMOID: {
      const float s = sigmoid(v);
      *a = s;
      *slope = s * (1.0f - s);
      break;
    }
    case KAN_GATE_TANH: {
      const float t = tanhf(v);
      *a = t;
      *slope = 1.0f - t * t;
      break;
    }
    case KAN_GATE_SILU: {
      const float s = sigmoid(v);
      *a = v * s;
      *slope = s * (1.0f + v * (1.0f - s));
      break;
    }
    case KAN_GATE_GELU: {
      const float c = normal_cdf(v);
      *a = v * c;
      *slope = c + v * 0.39894228f * expf(-0.5f * v * v);
      break;
    }
    case KAN_GATE_RELU:
      *a = v < 0.0f ? 0.0f : v;  // (NaN stays)
      *slope = v > 0.0f ? 1.0f : 0.0f;
      break;
    default:
      *a = v;
      *slope = 1.0f;
  }
}
template <bool QUICK>
__device__ __forceinline__ float gated_value(float g, float u, int act) {
  float a, slope;
  gated_act<QUICK>(g, act, &a, &slope);
  return a * u;
}

// ---- kept values ----------------------------------------------------------------
template <typename T>
struct Kept {  // bf16
  static constexpr int kLow = 4;
  typedef uint8_t low;
};
template <>
struct Kept<f16> {
  static constexpr int kLow = 8;
  typedef uint16_t low;
};
inline size_t low_bytes(int dtype, int64_t T, int64_t N) {
  return (size_t)(T * N) * (dtype == KAN_DTYPE_F16 ? 2 : 1);
}
// The leading 16 + LOW bits, to nearest, ties to even.
template <int LOW>
__device__ __forceinline__ uint32_t to_kept(float v) {
  constexpr int kCut = 16 - LOW;
  const uint32_t b = __float_as_uint(v);
  if (v != v) return 0x7fc00000 >> kCut;
  return (b + (1 << (kCut - 1)) - 1 + ((b >> kCut) & 1)) >> kCut;
}
template <int LOW>
__device__ __forceinline__ float from_kept(uint32_t high, uint32_t low) {
  return __uint_as_float(high << 16 | low << (16 - LOW));
}

// The first `count` of 8 values to dst; whole: all, and dst lies on their size.
template <typename T>
__device__ __forceinline__ void store_whole(T* dst, typename VecOf<T, 8>::type t, int count,
                                            bool whole) {
  if (whole) {
    *reinterpret_cast<decltype(t)*>(dst) = t;
  } else if (count >= 8) {
    reinterpret_cast<LooseVec<T, 8>*>(dst)->v = t;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < count) dst[j] = t[j];
  }
}
// h and what is kept of g and u, from column n of a row on; count columns exist.
template <typename T>
__device__ __forceinline__ void finish_8(const GatedParams& p, int64_t row, int64_t n, int count,
                                         bool whole, const float (&g)[8], const float (&u)[8]) {
  typename VecOf<T, 8>::type h;
#pragma unroll
  for (int j = 0; j < 8; ++j) h[j] = (T)gated_value<true>(g[j], u[j], p.act);
  store_whole(static_cast<T*>(p.C) + row * p.N + n, h, count, whole);
  if (p.pre == nullptr) return;
  constexpr int kLow = Kept<T>::kLow;
  typedef typename Kept<T>::low Low;
  typename VecOf<uint16_t, 8>::type words[2];
  typename VecOf<Low, 8>::type low;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t a = to_kept<kLow>(g[j]), b = to_kept<kLow>(u[j]), mask = (1 << kLow) - 1;
    words[0][j] = (uint16_t)(a >> kLow);
    words[1][j] = (uint16_t)(b >> kLow);
    low[j] = (Low)((a & mask) << kLow | (b & mask));
  }
  uint16_t* at = static_cast<uint16_t*>(p.pre) + row * 2 * p.N + n;
  store_whole(at, words[0], count, whole);
  store_whole(at + p.N, words[1], count, whole);
  store_whole(static_cast<Low*>(p.low) + row * p.N + n, low, count, whole);
}

// ---- tiles in 16 bits -------------------------------------------------------------
// Bound by MFMA at the power cap, and where K is short by the stores: 16384 rows of
// 4096 -> 4096 in bf16 844 us (1.30 PFLOP/s); of 1024 -> 4096 275 us (1.0), and 358 with
// the kept values, 3.5 times h's bytes behind 16 slabs of product.
template <typename T, class G, int MODE>
__global__ __launch_bounds__(G::NT) void gated_tile_kernel(GatedParams p, int tiles_n, int whole) {
  constexpr int BM = G::BM, BN = G::BN, FM = G::FM;
  static_assert(G::FN == 2, "a wave has 32 columns of each weight");
  __shared__ __align__(16) char lds[2 * G::kBuf];
  RowTile t;
  int tn;
  if (!row_tile(p, BM, tiles_n, &t, &tn)) return;
  const int64_t n0 = (int64_t)tn * (BN / 2), kend = t.e == p.E ? 0 : p.K;
  Operand<T, BM, true, MODE, G::NT> a;
  Operand<T, BN, true, MODE, G::NT, true> b;
  a.init(p.A, p.lda, t.m0, t.m1 - t.m0);
  b.init(static_cast<const T*>(p.B) + (int64_t)t.e * 2 * p.N * p.ldb, p.ldb, n0, p.N - n0);
  b.up = p.N * p.ldb * (int64_t)sizeof(T);
  f32x16 acc[FM][2];
  tile_loop<T, G, true, true>(a, b, 0, kend, lds, acc);

  // 32 rows at a time, a wave's g and u go through LDS to become 8 consecutive
  // outputs a lane (chunks of 4 values, exchanged by row against bank conflicts).
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / G::WN, wn = wave % G::WN;
  typedef float f4 __attribute__((ext_vector_type(4)));
  f4* stage = reinterpret_cast<f4*>(lds) + wave * 32 * 16;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int r = lane & 31;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        f4 v;
#pragma unroll
        for (int s = 0; s < 4; ++s) v[s] = acc[i][j][4 * q + s];
        stage[r * 16 + ((8 * j + 2 * q + (lane >> 5)) ^ (r & 15))] = v;
      }
#pragma unroll 1
    for (int it = 0; it < 2; ++it) {
      const int rr = it * 16 + (lane >> 2), c = 2 * (lane & 3);
      float g[8], u[8];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const f4 vg = stage[rr * 16 + ((c + k) ^ (rr & 15))];
        const f4 vu = stage[rr * 16 + ((8 + c + k) ^ (rr & 15))];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          g[4 * k + s] = vg[s];
          u[4 * k + s] = vu[s];
        }
      }
      const int64_t row = t.m0 + (wm * FM + i) * 32 + rr, n = n0 + wn * 32 + 4 * c;
      if (row < t.m1 && n < p.N)
        finish_8<T>(p, row, n, (int)min(p.N - n, (int64_t)8), whole != 0, g, u);
    }
  }
}

// ---- few rows ---------------------------------------------------------------------
// As the grouped products' kernel for groups of a few rows: 16 rows and 16 NP
// outputs a block, bound by the weights' bytes: 8 rows of 1024 -> 4096 in bf16, 16.8 MB,
// in 6 us (from the last-level cache); one row of 4096 -> 4096, 67 MB, in 13.
template <typename T, int NP, bool WHOLE>
__global__ __launch_bounds__(256) void gated_few_kernel(GatedParams p, int tiles_n) {
  typedef RowsMma<T> M;
  constexpr int kCols = 16 * NP;
  __shared__ float red[4][kFewRows][2 * kCols + 1];
  RowTile t;
  int tn;
  if (!row_tile(p, kFewRows, tiles_n, &t, &tn)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n0 = tn * kCols;
  typename M::acc_t acc[2 * NP];
#pragma unroll
  for (int c = 0; c < 2 * NP; ++c) acc[c] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (t.e < p.E) {
    const int m = min(t.m0 + (lane & 15), t.m1 - 1);
    const T* x = static_cast<const T*>(p.A) + (int64_t)m * p.K;
    const T* w[2 * NP];
#pragma unroll
    for (int c = 0; c < 2 * NP; ++c) {
      const int64_t n = min((int64_t)(n0 + 16 * (c >> 1) + (lane & 15)), p.N - 1);
      w[c] = static_cast<const T*>(p.B) + ((int64_t)t.e * 2 * p.N + (c & 1) * p.N + n) * p.K;
    }
    few_rows<T, 2 * NP, WHOLE>(x, w, p.K, acc);
  }
#pragma unroll
  for (int c = 0; c < 2 * NP; ++c)
#pragma unroll
    for (int v = 0; v < 4; ++v)
      red[wave][lane & 15][(c & 1) * kCols + 16 * (c >> 1) + 4 * (lane >> 4) + v] = acc[c][v];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int at = i * 256 + threadIdx.x, m = at / kCols, c = at % kCols;
    auto sum = [&](int col) __attribute__((always_inline)) {
      return red[0][m][col] + red[1][m][col] + red[2][m][col] + red[3][m][col];
    };
    const float g = sum(c), u = sum(kCols + c);
    const int64_t row = t.m0 + m, n = n0 + c;
    if (row >= t.m1 || n >= p.N) continue;
    static_cast<T*>(p.C)[row * p.N + n] = (T)gated_value<sizeof(T) == 2>(g, u, p.act);
    if (p.pre == nullptr) continue;
    if constexpr (sizeof(T) == 4) {
      float* at_pre = static_cast<float*>(p.pre) + row * 2 * p.N + n;
      at_pre[0] = g;
      at_pre[p.N] = u;
    } else {
      constexpr int kLow = Kept<T>::kLow;
      const uint32_t a = to_kept<kLow>(g), b = to_kept<kLow>(u), mask = (1 << kLow) - 1;
      uint16_t* at_pre = static_cast<uint16_t*>(p.pre) + row * 2 * p.N + n;
      at_pre[0] = (uint16_t)(a >> kLow);
      at_pre[p.N] = (uint16_t)(b >> kLow);
      static_cast<typename Kept<T>::low*>(p.low)[row * p.N + n] =
          (typename Kept<T>::low)((a & mask) << kLow | (b & mask));
    }
  }
}

// ---- elementwise ------------------------------------------------------------------
// V outputs a thread, in the order of memory; V divides N where V > 1.
template <int V, class F>
__device__ __forceinline__ void each_output(int64_t T, int64_t N, const F& f) {
  const int64_t per = N / V, total = T * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * 256) {
    const int64_t row = total >> 32 == 0 ? (uint32_t)i / (uint32_t)per : i / per;
    f(row, (i - row * per) * V);
  }
}
unsigned flat_blocks(int64_t threads) {
  return (unsigned)std::min<int64_t>(std::max<int64_t>(1, ceil_div(threads, 256)), 1 << 16);
}

// fp32: h from the product [T, 2 N].
template <int V>
__global__ __launch_bounds__(256) void gated_value_kernel(GatedParams p) {
  each_output<V>(p.T, p.N, [&](int64_t row, int64_t n) {
    const float* at = static_cast<const float*>(p.pre) + row * 2 * p.N + n;
    float g[V], u[V];
    load_f32<float, V>(at, g);
    load_f32<float, V>(at + p.N, u);
#pragma unroll
    for (int j = 0; j < V; ++j) g[j] = gated_value<false>(g[j], u[j], p.act);
    store_f32<float, V>(static_cast<float*>(p.C) + row * p.N + n, g);
  });
}

// 16 bits: h and what is kept from the partial sums [cuts, T, 2 N] of a product on few
// tiles, 8 outputs a thread.
template <typename T>
__global__ __launch_bounds__(256) void gated_join_kernel(GatedParams p, int whole) {
  const int64_t per = (p.N + 7) / 8, total = p.T * per, slice = p.T * 2 * p.N;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / per, n = (i - row * per) * 8;
    const int count = (int)min(p.N - n, (int64_t)8);
    const float* at = p.part + row * 2 * p.N + n;
    float g[8] = {}, u[8] = {};
    if (whole) {
#pragma unroll 4
      for (int q = 0; q < p.cuts; ++q) {
        float a[8], b[8];
        load_f32<float, 4>(at + q * slice, reinterpret_cast<float(&)[4]>(a[0]));
        load_f32<float, 4>(at + q * slice + 4, reinterpret_cast<float(&)[4]>(a[4]));
        load_f32<float, 4>(at + q * slice + p.N, reinterpret_cast<float(&)[4]>(b[0]));
        load_f32<float, 4>(at + q * slice + p.N + 4, reinterpret_cast<float(&)[4]>(b[4]));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          g[j] += a[j];
          u[j] += b[j];
        }
      }
    } else {
      for (int q = 0; q < p.cuts; ++q)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < count) {
            g[j] += at[q * slice + j];
            u[j] += at[q * slice + p.N + j];
          }
    }
    finish_8<T>(p, row, n, count, whole != 0, g, u);
  }
}

// V values of dg and du from dh (A) and what was kept.
template <typename T, int V>
__device__ __forceinline__ void gated_grads(const GatedParams& p, int64_t row, int64_t n,
                                            float (&g)[V], float (&u)[V]) {
  float dh[V];
  if constexpr (sizeof(T) == 4) {
    const float* at = static_cast<const float*>(p.pre) + row * 2 * p.N + n;
    load_f32<float, V>(at, g);
    load_f32<float, V>(at + p.N, u);
  } else {
    const uint16_t* at = static_cast<const uint16_t*>(p.pre) + row * 2 * p.N + n;
    typedef uint16_t words __attribute__((ext_vector_type(V)));
    constexpr int kLow = Kept<T>::kLow;
    typedef typename Kept<T>::low Low;
    typedef typename VecOf<Low, V>::type lows;
    const words hg = *reinterpret_cast<const words*>(at);
    const words hu = *reinterpret_cast<const words*>(at + p.N);
    const lows low = *reinterpret_cast<const lows*>(static_cast<const Low*>(p.low) + row * p.N + n);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      g[j] = from_kept<kLow>(hg[j], low[j] >> kLow);
      u[j] = from_kept<kLow>(hu[j], low[j] & ((1 << kLow) - 1));
    }
  }
  load_f32<T, V>(static_cast<const T*>(p.A) + row * p.N + n, dh);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    float a, slope;
    gated_act<sizeof(T) == 2>(g[j], p.act, &a, &slope);
    g[j] = dh[j] * u[j] * slope;
    u[j] = dh[j] * a;
  }
}

// [dg du]; C: [T, 2 N].  Bound by HBM: 16384 x 4096 in bf16, 738 MB, 148 us (5.0 TB/s).
// MOST: the block's largest finite value too.
__device__ __forceinline__ float block_most(float v) {
  __shared__ float red[4];
  v = wave_max(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}
template <typename T, int V, bool MOST>
__global__ __launch_bounds__(256) void gated_grad_kernel(GatedParams p) {
  float most = 0.0f;
  each_output<V>(p.T, p.N, [&](int64_t row, int64_t n) {
    float g[V], u[V];
    gated_grads<T, V>(p, row, n, g, u);
    T* out = static_cast<T*>(p.C) + row * 2 * p.N + n;
    store_f32<T, V>(out, g);
    store_f32<T, V>(out + p.N, u);
    if constexpr (MOST) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float a = fabsf(g[j]), b = fabsf(u[j]);
        most = fmaxf(most, fmaxf(a < INFINITY ? a : 0.0f, b < INFINITY ? b : 0.0f));
      }
    }
  });
  if constexpr (MOST) {
    most = block_most(most);
    if (threadIdx.x == 0) p.factor[1 + blockIdx.x] = most;
  }
}

// f16 has 30 binades of normal values.  Gradients of a mean over many rows lie below
// them, and over small weights products lie above them whose sums do not: where the
// largest of dg and du is not within 1 .. 2^15 they are written again, times the power of 2
// that takes it to 2^14 .. 2^15, and the products behind them undo that on their
// float32 sums.  (Within that range a value is off by 2^-25 at most, 2^-25 of the largest.)
// 8192 x 1024: 4.2 us where nothing is written again, 18 where it is (19 for the kernel
// before); 16384 x 4096: 6.7 and 155.  Scaled in every call, from a pass that only
// looked for the largest: 13 and 155.
constexpr int kScaleValues = KAN_GATED_SCALE_VALUES;
template <typename T, int V>
__global__ __launch_bounds__(256) void gated_rescale_kernel(GatedParams p) {
  float most = 0.0f;
#pragma unroll 8
  for (int i = threadIdx.x; i < p.parts; i += 256) most = fmaxf(most, p.factor[1 + i]);
  most = block_most(most);
  float unit = 1.0f;
  if (most != 0.0f && (most < 1.0f || most >= 32768.0f)) {
    int e;
    frexpf(most, &e);  // (most < 2^e; one over the unit is a normal number)
    unit = ldexpf(1.0f, min(max(15 - e, -126), 126));
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.factor = 1.0f / unit;
  if (unit == 1.0f) return;
  each_output<V>(p.T, p.N, [&](int64_t row, int64_t n) {
    float g[V], u[V];
    gated_grads<T, V>(p, row, n, g, u);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      g[j] *= unit;
      u[j] *= unit;
    }
    T* out = static_cast<T*>(p.C) + row * 2 * p.N + n;
    store_f32<T, V>(out, g);
    store_f32<T, V>(out + p.N, u);
  });
}

// ---- host ---------------------------------------------------------------------------
template <typename T, class G>
int launch_gated_tile(const GatedParams& p, hipStream_t st) {
  const int64_t tiles_n = ceil_div(p.N, G::BN / 2), blocks = row_grid(p, G::BM, tiles_n);
  if (!grid_fits(blocks, G::NT)) return set_error(KAN_ERR_LIMIT, "gated: too many tiles");
  const int whole = p.N % 8 == 0 && aligned16(p.C) && aligned16(p.pre);
  if (whole_rows(p.A, p.lda) && whole_rows(p.B, p.ldb))
    gated_tile_kernel<T, G, kDirect><<<dim3((unsigned)blocks), G::NT, 0, st>>>(p, (int)tiles_n,
                                                                             whole);
  else
    gated_tile_kernel<T, G, kGuarded><<<dim3((unsigned)blocks), G::NT, 0, st>>>(p, (int)tiles_n,
                                                                              whole);
  return check_launch("gated");
}
template <typename T>
int launch_gated_half(const GatedParams& p, HalfCfg cfg, hipStream_t st) {
  return cfg == kBig   ? launch_gated_tile<T, TileBig>(p, st)
         : cfg == kMid ? launch_gated_tile<T, TileMid>(p, st)
                       : launch_gated_tile<T, TileSmall>(p, st);
}

template <typename T, int NP, bool WHOLE>
int launch_gated_few_cols(const GatedParams& p, hipStream_t st) {
  const int64_t tiles_n = ceil_div(p.N, 16 * NP), blocks = row_grid(p, kFewRows, tiles_n);
  if (!grid_fits(blocks, 256)) return set_error(KAN_ERR_LIMIT, "gated: too many tiles");
  gated_few_kernel<T, NP, WHOLE><<<dim3((unsigned)blocks), 256, 0, st>>>(p, (int)tiles_n);
  return check_launch("gated");
}
template <typename T>
int launch_gated_few(const GatedParams& p, hipStream_t st) {
  // (32 outputs a block where such blocks number two a CU, as grouped products)
  const bool wide = std::min<int64_t>(p.E, p.T) * ceil_div(p.N, 32) >= 2 * device_cu_count();
  if (sizeof(T) == 2 && !(whole_rows(p.A, p.K) && whole_rows(p.B, p.K)))
    return wide ? launch_gated_few_cols<T, 2, false>(p, st)
                : launch_gated_few_cols<T, 1, false>(p, st);
  return wide ? launch_gated_few_cols<T, 2, true>(p, st) : launch_gated_few_cols<T, 1, true>(p, st);
}

template <typename T, int V>
int launch_gated_grad(GatedParams p, hipStream_t st) {
  const unsigned blocks = flat_blocks(p.T * p.N / V);
  if (p.factor == nullptr) {
    gated_grad_kernel<T, V, false><<<blocks, 256, 0, st>>>(p);
  } else if constexpr (std::is_same<T, f16>::value) {
    p.parts = (int)std::min<unsigned>(blocks, kScaleValues - 1);
    gated_grad_kernel<T, V, true><<<p.parts, 256, 0, st>>>(p);
    gated_rescale_kernel<T, V><<<std::min<unsigned>(blocks, 8 * device_cu_count()), 256, 0, st>>>(p);
  }
  return check_launch("gated_backward");
}

int check_gated(const char* who, int dtype, int act, int64_t T, int64_t E, int64_t N, int64_t K) {
  if (!dtype_is_operator(dtype))
    return set_error(KAN_ERR_INVALID, "%s: dtype must be FP32, BF16 or FP16 (code %d)", who, dtype);
  if (act < KAN_GATE_IDENTITY || act > KAN_GATE_RELU)
    return set_error(KAN_ERR_INVALID, "%s: unknown activation %d", who, act);
  if (T < 0 || E < 0 || N < 0 || K < 0) return set_error(KAN_ERR_INVALID, "%s: negative size", who);
  if (T > 0x3fffffff || N > (1 << 21) || K > (1 << 22) || E > 65535)
    return set_error(KAN_ERR_LIMIT,
                     "%s: at most 2^30 - 1 rows, 2^21 outputs, 2^22 inputs and 65535 experts", who);
  return KAN_OK;
}

// A forward call's workspace: 16 bits: operands brought onto 16 bytes, then the partial
// sums of a product whose tiles would leave places idle.  fp32: g and u where they are
// not kept, then the product's partial sums.
struct GatedPlan {
  HalfPlan plan;
  AlignPlan align;
  size_t pre_bytes, bytes;  // before the partial sums; all
};
// Cuts of long sums on tiles of 128 x 128 that leave places idle: a slab takes 0.63 us, the
// weights are read at 4.7 TB/s, and the cuts' sums written, read and joined at 4 TB/s by
// one more launch, 7 us in all.  4096 -> 4096 in bf16, without cuts and in them: 64 rows
// 41.3 and 23.2 us, 256 rows 43.0 and 34.7; 300 rows of 2048 -> 1000 19.2 and 17.7 (23.5 in
// 8 cuts, as the grouped products' rule has it).
int gated_cuts(int64_t T, int64_t E, int64_t N, int64_t K) {
  const double tiles = row_tiles(T, E, 128) * (double)ceil_div(N, 64);
  const double read = 4.0 * (double)std::min(E, T) * (double)N * (double)K / 4.7e6;
  const int64_t slabs = ceil_div(K, kDepth);
  int best = 1;
  double least = 0.0;
  for (int cuts = 1; cuts <= 32 && (cuts == 1 || slabs / cuts >= 4); ++cuts) {
    const double turns = std::max(1.0, rounds(tiles * cuts, 2.0 * device_cu_count()));
    double t = std::max(0.63 * turns * (double)ceil_div(slabs, cuts), read);
    if (cuts > 1) t += 7.0 + (double)cuts * (double)(2 * T * N) * 8.0 / 4.0e6;
    if (cuts == 1 || t < least) {
      least = t;
      best = cuts;
    }
  }
  return best;
}
GatedPlan plan_gated(int dtype, const void* x, const void* w, int64_t T, int64_t E, int64_t N,
                     int64_t K, bool keep) {
  GatedPlan g{};
  if (T == 0 || N == 0) return g;
  g.plan = product_plan(dtype, KAN_GROUPED_FORWARD, T, E, 2 * N, K);
  if (g.plan.cfg == kFew) return g;
  if (dtype == KAN_DTYPE_F32) {
    if (!keep) g.pre_bytes = (size_t)round_up(8 * T * N, 16);
    g.bytes = g.pre_bytes + product_part_bytes(KAN_GROUPED_FORWARD, g.plan, T, E, 2 * N, K);
  } else if (E > 0 && K > 0) {  // (without experts or inputs nothing is read)
    g.align = align_plan(KAN_GROUPED_FORWARD, KAN_ACT8_NONE, x, w, T, E, 2 * N, K);
    g.plan.cuts = g.plan.cfg == kSmall ? gated_cuts(T, E, N, K) : 1;
    g.pre_bytes = (size_t)round_up((int64_t)(g.align.a_bytes + g.align.b_bytes), 16);
    g.bytes = g.pre_bytes + product_part_bytes(KAN_GROUPED_FORWARD, g.plan, T, E, 2 * N, K);
  }
  return g;
}

}  // namespace
}  // namespace kan

using namespace kan;

extern "C" {

int kan_hip_gated_kept(int dtype, int64_t T, int64_t N, size_t* bytes) {
  if (bytes == nullptr) return set_error(KAN_ERR_INVALID, "gated_kept: bytes must not be NULL");
  const int rc = check_gated("gated_kept", dtype, 0, T, 0, N, 0);
  if (rc != KAN_OK) return rc;
  *bytes = dtype == KAN_DTYPE_F32 ? (size_t)(8 * T * N) : word_bytes(T, N) + low_bytes(dtype, T, N);
  return KAN_OK;
}

int kan_hip_gated_workspace(int dtype, const void* x, const void* w, int64_t T, int64_t E, int64_t N,
                            int64_t K, int keep, size_t* bytes) {
  if (bytes == nullptr)
    return set_error(KAN_ERR_INVALID, "gated_workspace: bytes must not be NULL");
  const int rc = check_gated("gated_workspace", dtype, 0, T, E, N, K);
  if (rc != KAN_OK) return rc;
  *bytes = plan_gated(dtype, x, w, T, E, N, K, keep != 0).bytes;
  return KAN_OK;
}

int kan_hip_gated(int dtype, int act, const void* x, const void* w, const void* offsets,
                  int offsets64, int64_t T, int64_t E, int64_t N, int64_t K, void* h, void* kept,
                  void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = check_gated("gated", dtype, act, T, E, N, K);
  if (rc != KAN_OK) return rc;
  if (T == 0 || N == 0) return KAN_OK;
  if (h == nullptr || (K > 0 && E > 0 && (x == nullptr || w == nullptr)) ||
      (E > 1 && offsets == nullptr))
    return set_error(KAN_ERR_INVALID, "gated: operands must not be NULL");
  if (!aligned16(kept) || !aligned16(workspace))
    return set_error(KAN_ERR_INVALID, "gated: kept values and the workspace lie on 16 bytes");
  const GatedPlan g = plan_gated(dtype, x, w, T, E, N, K, kept != nullptr);
  if (g.bytes > 0 && (workspace == nullptr || workspace_bytes < g.bytes))
    return set_error(KAN_ERR_WORKSPACE, "gated: needs %zu bytes of workspace, got %zu", g.bytes,
                     workspace == nullptr ? (size_t)0 : workspace_bytes);
  char* ws = static_cast<char*>(workspace);
  GatedParams p{};
  p.A = x;
  p.B = w;
  p.C = h;
  p.offsets = offsets;
  p.offsets64 = offsets64;
  p.E = (int)E;
  p.T = T;
  p.N = N;
  p.K = p.lda = p.ldb = K;
  p.act = act;
  p.pre = kept;
  if (kept != nullptr && dtype != KAN_DTYPE_F32)
    p.low = static_cast<char*>(kept) + word_bytes(T, N);
  hipStream_t st = static_cast<hipStream_t>(stream);
  TimedLaunch timed(kClassContraction, st, 4.0 * (double)T * N * K);
  if (g.plan.cfg == kFew)
    return dtype == KAN_DTYPE_F32    ? launch_gated_few<float>(p, st)
           : dtype == KAN_DTYPE_BF16 ? launch_gated_few<bf16>(p, st)
                                     : launch_gated_few<f16>(p, st);
  if (dtype != KAN_DTYPE_F32) {
    int e = launch_aligned(g.align, &p, ws, st);
    if (e != KAN_OK) return e;
    if (g.plan.cuts > 1) {
      p.part = reinterpret_cast<float*>(ws + g.pre_bytes);
      p.cuts = g.plan.cuts;
      GroupedParams q = p;
      q.C = nullptr;
      q.N = 2 * N;
      e = launch_product(dtype, KAN_GROUPED_FORWARD, q, g.plan, st);
      if (e != KAN_OK) return e;
      const int whole = N % 8 == 0 && aligned16(h);
      const unsigned blocks = flat_blocks(T * ceil_div(N, 8));
      if (dtype == KAN_DTYPE_BF16) gated_join_kernel<bf16><<<blocks, 256, 0, st>>>(p, whole);
      else gated_join_kernel<f16><<<blocks, 256, 0, st>>>(p, whole);
      return check_launch("gated");
    }
    return dtype == KAN_DTYPE_BF16 ? launch_gated_half<bf16>(p, g.plan.cfg, st)
                                   : launch_gated_half<f16>(p, g.plan.cfg, st);
  }
  if (p.pre == nullptr) p.pre = ws;
  GroupedParams q = p;
  q.C = p.pre;
  q.N = 2 * N;
  if (g.bytes > g.pre_bytes) q.part = reinterpret_cast<float*>(ws + g.pre_bytes);
  const int e = launch_product(dtype, KAN_GROUPED_FORWARD, q, g.plan, st);
  if (e != KAN_OK) return e;
  if (N % 4 == 0 && aligned16(h)) gated_value_kernel<4><<<flat_blocks(T * N / 4), 256, 0, st>>>(p);
  else gated_value_kernel<1><<<flat_blocks(T * N), 256, 0, st>>>(p);
  return check_launch("gated");
}

static int gated_backward(int dtype, int act, const void* grad_h, const void* kept, int64_t T,
                          int64_t N, void* grad_pre, float* scale, void* stream) {
  const int rc = check_gated("gated_backward", dtype, act, T, 0, N, 0);
  if (rc != KAN_OK) return rc;
  if (T == 0 || N == 0) return KAN_OK;
  if (grad_h == nullptr || kept == nullptr || grad_pre == nullptr)
    return set_error(KAN_ERR_INVALID, "gated_backward: operands must not be NULL");
  if (!aligned16(kept))
    return set_error(KAN_ERR_INVALID, "gated_backward: kept values lie on 16 bytes");
  GatedParams p{};
  p.A = grad_h;
  p.C = grad_pre;
  p.pre = const_cast<void*>(kept);
  if (dtype != KAN_DTYPE_F32) p.low = static_cast<char*>(p.pre) + word_bytes(T, N);
  p.T = T;
  p.N = N;
  p.act = act;
  p.factor = scale;
  hipStream_t st = static_cast<hipStream_t>(stream);
  TimedLaunch timed(kClassOther, st, (double)T * N * (dtype == KAN_DTYPE_F32 ? 20 : 11));
  const bool whole = aligned16(grad_h) && aligned16(grad_pre);
  if (dtype == KAN_DTYPE_F32)
    return whole && N % 4 == 0 ? launch_gated_grad<float, 4>(p, st)
                               : launch_gated_grad<float, 1>(p, st);
  if (dtype == KAN_DTYPE_BF16)
    return whole && N % 8 == 0 ? launch_gated_grad<bf16, 8>(p, st)
                               : launch_gated_grad<bf16, 1>(p, st);
  return whole && N % 8 == 0 ? launch_gated_grad<f16, 8>(p, st) : launch_gated_grad<f16, 1>(p, st);
}

int kan_hip_gated_backward(int dtype, int act, const void* grad_h, const void* kept, int64_t T,
                           int64_t N, void* grad_pre, void* stream) {
  return gated_backward(dtype, act, grad_h, kept, T, N, grad_pre, nullptr, stream);
}

int kan_hip_gated_backward_scaled(int dtype, int act, const void* grad_h, const void* kept,
                                  int64_t T, int64_t N, void* grad_pre, float* scale,
                                  void* stream) {
  if (dtype != KAN_DTYPE_F16 || scale == nullptr)
    return set_error(KAN_ERR_INVALID, "gated_backward_scaled: FP16 and a place for the factor");
  return gated_backward(dtype, act, grad_h, kept, T, N, grad_pre, scale, stream);
}

}  // extern "C"
