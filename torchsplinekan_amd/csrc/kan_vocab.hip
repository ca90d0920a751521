// Losses of logits z = x W^T, x [T, D], W [V, D], that are never kept whole.  Row t
// has a target distribution p on a few ids (one with p = 1 for the cross entropy, a
// teacher's top ids for distillation) and a temperature tau; with q = softmax(z / tau)
// over all V
//   loss_t = tau^2 sum_j p_j (log p_j - log q_{id_j})
//   dz_t   = g_t tau (q - sum_j p_j e_{id_j}),   dx = dz W,   dW = dz^T x.
// (tau = 1 and one id: lse(z) - z_id and g_t (q - e_id).)
//
// Forward: the product's tiles end in each row's maximum, rest and sum of p z over the
// tile's columns (see below); a second kernel joins a row's tiles.  Backward:
// piece by piece of the vocabulary the product again, whose tiles end in dz in the
// operands' type, and dx += dz W, dW = dz^T x from that piece.  4/3 of the
// operations that kept logits would take, and 2 bytes a logit of one piece.
//
// A row keeps its largest z, top, and rest = the sum of exp((z - top) / tau) over the
// others (1 for each that equals top but one): lse = top / tau + log1p(rest), and
//   q_j - p_j = ((e_j - p_j) - p_j rest) / (1 + rest),   e_j = exp((z_j - top) / tau),
// so the small loss and gradient of a row that is nearly certain keep their accuracy,
// which 1 + rest alone rounds away.
// dz is rounded to 16 bits as (q - p) w with w = 1 in rows that all count alike (in
// f16 2^15, so that probabilities of 1e-8 still are normal numbers); the common
// factor g tau is applied to the float32 sums of dx and dW.
//
// Everything is added in a fixed order; no atomics.
#include "kan_grouped.h"
#include "kan_tile.h"

namespace kan {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kNoId = 0x7fffffff;  // past every column

struct VocabParams {
  const void *x, *w;
  int64_t T, V, D, k;
  int64_t ldx, ldw;
  float tau;
  // cross entropy (k = 1); null: distillation
  const void* target;  // [T]
  int target64;
  int64_t ignore;
  // kept for the backward pass
  float *top, *rest;   // [T]
  float* flag;         // [T]: 1; 0: the row does not count; NaN: an id that is no column
  float* count;        // rows that count
  float* logits;       // [T, V] of few classes
  int* ids;            // [T, k] of distillation: ascending (kNoId: absent)
  float* prob;         // [T, k]: p
  // of a call
  float* entropy;      // [T]: sum_j p_j log p_j
  float* stats;        // [3, tiles, T]
  int tiles;           // of all pieces
  float* weight;       // [T]: w
  float* z;            // fp32: [T, cols] logits, then dz of a piece
  void* G;             // 16 bits: [T, ldg] dz of a piece, zeros behind its columns as far
                       // as 16 bytes go; then, or null,
  void* G2;            // [T, ldg]: what the rounding of G's values has left, rounded
  int64_t ldg;
  int64_t v0, cols;    // the piece
};

// ---- targets ----------------------------------------------------------------------
// Cross entropy: the row's column (kNoId: none) and its flag.
__device__ __forceinline__ int target_of(const VocabParams& p, int64_t row, float* flag) {
  const int64_t id = p.target64 ? static_cast<const int64_t*>(p.target)[row]
                                : (int64_t)static_cast<const int*>(p.target)[row];
  const bool in = id >= 0 && id < p.V && id != p.ignore;
  *flag = in ? 1.0f : id == p.ignore ? 0.0f : NAN;
  return in ? (int)id : kNoId;
}

// Blocks of a kernel that takes rows in turns: a grid has fewer than 2^32 threads, which
// T rows of a wave each pass from 2^26 on.
constexpr int64_t kMaxBlocks = 1 << 20;
unsigned row_blocks(int64_t rows, int64_t each) {
  return (unsigned)std::min<int64_t>(ceil_div(rows, each), kMaxBlocks);
}

// One wave a row: p = softmax(teacher / tau) over its ids, sorted by id (a place is the
// number of smaller ones, so equal ids keep their order).
constexpr int64_t kMaxTop = 1024;
__global__ __launch_bounds__(64) void vocab_teacher_kernel(VocabParams p, const void* ids, int is64,
                                                           const float* __restrict__ teacher) {
  __shared__ int id_of[kMaxTop];
  __shared__ float value_of[kMaxTop];
  const int k = (int)p.k, lane = threadIdx.x;
  for (int64_t t = blockIdx.x; t < p.T; t += gridDim.x) {
    const int64_t base = t * p.k;
    float top = -INFINITY;
    bool bad = false;
    for (int j = lane; j < k; j += 64) {
      const int64_t id = is64 ? static_cast<const int64_t*>(ids)[base + j]
                              : (int64_t)static_cast<const int*>(ids)[base + j];
      const bool in = id >= 0 && id < p.V;
      const float v = in ? teacher[base + j] / p.tau : -INFINITY;
      bad |= id >= p.V;
      id_of[j] = in ? (int)id : kNoId;
      value_of[j] = v;
      top = fmaxf(top, v);
    }
    top = wave_max(top);
    if (top == -INFINITY) top = 0.0f;
    float sum = 0.0f;
    for (int j = lane; j < k; j += 64) {
      const float e = expf(value_of[j] - top);
      sum += e;
    }
    sum = wave_sum(sum);
    const float log_sum = logf(sum);
    __syncthreads();
    float entropy = 0.0f;
    for (int j = lane; j < k; j += 64) {
      const int id = id_of[j];
      const float v = value_of[j], e = expf(v - top);
      const float prob = sum == 0.0f ? 0.0f : e / sum;
      if (!(prob == 0.0f)) entropy += prob * (v - top - log_sum);
      int place = 0;
      for (int i = 0; i < k; ++i) place += id_of[i] < id || (id_of[i] == id && i < j);
      p.ids[base + place] = id;
      p.prob[base + place] = prob;
    }
    entropy = wave_sum(entropy);
    bad = __any(bad);
    if (lane == 0) {
      p.entropy[t] = entropy;
      p.flag[t] = bad ? NAN : sum == 0.0f ? 0.0f : 1.0f;
    }
    __syncthreads();  // (its ids may be the next row's)
  }
}

// The first of a row's k ascending ids that is `from` or more.
__device__ __forceinline__ int first_id(const int* __restrict__ ids, int k, int from) {
  int lo = 0, hi = k;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (ids[mid] < from) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

// The part of `rest` of a value z, `from` the largest (or 0 for none), which is itself
// counted in `most`.
__device__ __forceinline__ float below(float z, float from, float c) {
  return z == from ? 0.0f : __builtin_amdgcn_exp2f((z - from) * c);
}
// top and rest of two sets of logits as those of both (top -INFINITY: an empty set, whose
// rest is 0).
__device__ __forceinline__ void join(float* top, float* rest, float m, float s, float c) {
  const bool more = m > *top;
  const float most = more ? m : *top, least = more ? *top : m;
  const float mine = more ? s : *rest, other = more ? *rest : s;
  const float f = least == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((least - most) * c);
  *rest = mine + (other + 1.0f) * f;
  *top = most;
}

// ---- tiles in 16 bits -------------------------------------------------------------
// Bound by MFMA at the power cap, and with few inputs by what follows the product (an
// exponential of every logit): 8192 rows of 2048 -> 65536 in bf16 1.80 ms forward (1.22
// PFLOP/s) and 2.0 for dz; 4096 of 1024 -> 65536 with 64 ids a row 0.59 and
// 0.66 (without a teacher 0.50 forward); 33 of 1024 -> 32768 by W's bytes, 16 us.
// A lane holds rows 32 i + (lane & 31) of its wave's and 32 columns: 32 j + 8 q +
// 4 (lane >> 5) + s at acc[i][j][4 q + s].
// PARTS (0: the forward pass): of dz.  Only the smallest tile takes two: on the
// largest the second time over its sums would not stay in registers.
template <typename T, class G, int MODE, int PARTS>
__global__ __launch_bounds__(G::NT) void vocab_tile_kernel(VocabParams p, int tiles_n) {
  constexpr int BM = G::BM, BN = G::BN, FM = G::FM, WN = G::WN;
  constexpr bool GRAD = PARTS > 0;
  static_assert(G::FN == 2, "a wave has 64 columns");
  __shared__ __align__(16) char lds[2 * G::kBuf];
  __shared__ int first[BM], last[BM];  // the row's ids in the tile's columns; its target
  __shared__ float row_top[GRAD ? BM : 1], row_rest[GRAD ? BM : 1], row_weight[GRAD ? BM : 1];
  RowTile t;
  int tn;
  dense_tile(p.T, BM, tiles_n, &t, &tn);
  const int64_t n0 = (int64_t)tn * BN;
  const int col0 = (int)(p.v0 + n0);
  const float c = kLog2e / p.tau;
  auto look_up = [&]() __attribute__((always_inline)) {
    for (int r = threadIdx.x; r < BM; r += G::NT) {
      const int64_t row = t.m0 + r;
      int lo = 0, hi = 0;
      if (row < t.m1) {
        if (p.target != nullptr) {
          float flag;
          lo = target_of(p, row, &flag);
        } else {
          const int* ids = p.ids + row * p.k;
          hi = lo = first_id(ids, (int)p.k, col0);
          while (hi < p.k && ids[hi] < col0 + BN) ++hi;
        }
        if constexpr (GRAD) {
          row_top[r] = p.top[row];
          row_weight[r] = p.weight[row];
          row_rest[r] = p.rest[row];
        }
      }
      first[r] = lo;
      last[r] = hi;
    }
  };
  Operand<T, BM, true, MODE, G::NT> a;
  Operand<T, BN, true, MODE, G::NT> b;
  a.init(p.x, p.ldx, t.m0, t.m1 - t.m0);
  b.init(p.w, p.ldw, col0, p.cols - n0);
  f32x16 acc[FM][2];
  tile_loop<T, G, true, true>(a, b, 0, p.D, lds, acc, look_up);
  __syncthreads();

  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int left = (int)min(p.cols - n0 - wn * 64, (int64_t)64);  // the wave's columns that exist
  auto col_of = [&](int j, int v) { return 32 * j + 8 * (v >> 2) + 4 * half + (v & 3); };
  // f(column of the wave's, p) for the row's ids, the same number of turns in all lanes
  auto entries = [&](int r, int64_t row, auto f) __attribute__((always_inline)) {
    const int lo = first[r], hi = last[r];
    if (p.target != nullptr) {
      const int at = lo - col0 - wn * 64;
      if (__any(at >= 0 && at < 64)) f(at, 1.0f);
      return;
    }
    for (int e = lo; __any(e < hi); ++e) {
      int at = -1;
      float prob = 0.0f;
      if (e < hi) {
        at = p.ids[row * p.k + e] - col0 - wn * 64;
        prob = p.prob[row * p.k + e];
      }
      f(at, prob);
    }
  };
  if constexpr (!GRAD) {
    float* red = reinterpret_cast<float*>(lds);  // [3][WN][BM]
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int r = (wm * FM + i) * 32 + (lane & 31);
      if (left < 64) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int v = 0; v < 16; ++v)
            if (col_of(j, v) >= left) acc[i][j][v] = -INFINITY;
      }
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v) top = fmaxf(top, acc[i][j][v]);
      top = fmaxf(top, __shfl_xor(top, 32));
      const float from = top == -INFINITY ? 0.0f : top;
      float rest = 0.0f;
      int most = 0;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          rest += below(acc[i][j][v], from, c);
          most += acc[i][j][v] == from ? 1 : 0;
        }
      rest += __shfl_xor(rest, 32);
      most += __shfl_xor(most, 32);
      if (top > -INFINITY) rest += (float)(most - 1);
      float dot = 0.0f;
      entries(r, t.m0 + r, [&](int at, float prob) __attribute__((always_inline)) {
        if (at < 0 || at >= 64 || ((at >> 2) & 1) != half || prob == 0.0f) return;
        float z = 0.0f;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (__any(at >> 3 == 4 * j + q)) {
#pragma unroll
              for (int s = 0; s < 4; ++s)
                if (col_of(j, 4 * q + s) == at) z = acc[i][j][4 * q + s];
            }
        dot += prob * z;
      });
      dot += __shfl_xor(dot, 32);
      if (half == 0) {
        red[wn * BM + r] = top;
        red[(WN + wn) * BM + r] = rest;
        red[(2 * WN + wn) * BM + r] = dot;
      }
    }
    __syncthreads();
    for (int r = threadIdx.x; r < BM; r += G::NT) {
      if (t.m0 + r >= t.m1) break;
      float top = red[r], rest = red[WN * BM + r], dot = red[2 * WN * BM + r];
#pragma unroll
      for (int q = 1; q < WN; ++q) {
        join(&top, &rest, red[q * BM + r], red[(WN + q) * BM + r], c);
        dot += red[(2 * WN + q) * BM + r];
      }
      float* out = p.stats + (int64_t)tn * p.T + t.m0 + r;
      out[0] = top;
      out[p.tiles * p.T] = rest;
      out[2 * p.tiles * p.T] = dot;
    }
  } else {
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int r = (wm * FM + i) * 32 + (lane & 31);
      const float top = row_top[r], rest = row_rest[r], weight = row_weight[r];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v)
          acc[i][j][v] = __builtin_amdgcn_exp2f((acc[i][j][v] - top) * c);
      entries(r, t.m0 + r, [&](int at, float prob) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (__any(at >> 3 == 4 * j + q)) {  // (of 8 such columns few waves need a second)
#pragma unroll
              for (int s = 0; s < 4; ++s) {
                const float here = col_of(j, 4 * q + s) == at ? prob : 0.0f;
                acc[i][j][4 * q + s] = __builtin_fmaf(-here, rest, acc[i][j][4 * q + s] - here);
              }
            }
      });
      const float part = weight / (1.0f + rest);
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[i][j][v] *= part;
      if (left < 64 || __any(weight == 0.0f)) {  // (a row that does not count may hold NaN)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int v = 0; v < 16; ++v)
            if (weight == 0.0f || col_of(j, v) >= left) acc[i][j][v] = 0.0f;
      }
    }
    // through LDS, to become whole 16-byte pieces of rows
    constexpr int kWaveRows = FM * 32, kRowBytes = 128, kChunks = 8;
    char* stage = lds + wave * kWaveRows * kRowBytes;
    typedef T t4 __attribute__((ext_vector_type(4)));
    const int64_t row0 = t.m0 + wm * kWaveRows, col0 = n0 + wn * 64;
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
      T* to = static_cast<T*>(part == 0 ? p.G : p.G2);
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int r = i * 32 + (lane & 31);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            t4 v;
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = (T)acc[i][j][4 * q + u];
            const int ch = (4 * j + q) ^ (r & (kChunks - 1));
            *reinterpret_cast<t4*>(stage + r * kRowBytes + ch * 16 + half * 8) = v;
          }
      }
#pragma unroll 4
      for (int it = 0; it < kWaveRows / 8; ++it) {
        const int r = it * 8 + lane / kChunks, ch = lane % kChunks;
        const u32x4 v = *reinterpret_cast<const u32x4*>(stage + r * kRowBytes +
                                                        ((ch ^ (r & (kChunks - 1))) * 16));
        const int64_t row = row0 + r, col = col0 + 8 * ch;
        if (row < t.m1 && col < p.ldg) *reinterpret_cast<u32x4*>(to + row * p.ldg + col) = v;
      }
      if (part + 1 == PARTS) break;
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int v = 0; v < 16; ++v) acc[i][j][v] -= (float)(T)acc[i][j][v];
    }
  }
}

// ---- fp32: logits of a piece in memory ----------------------------------------------
// A wave has kSpan columns of a row, column lane + 64 i at v[i].
constexpr int kSpan = 1024, kSpanValues = kSpan / 64;
template <bool GRAD>
__global__ __launch_bounds__(256) void vocab_span_kernel(VocabParams p) {
  const int lane = threadIdx.x & 63;
  const float c = kLog2e / p.tau;
  for (int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); row < p.T;
       row += (int64_t)gridDim.x * 4) {
    for (int64_t n0 = (int64_t)blockIdx.y * kSpan; n0 < p.cols; n0 += (int64_t)gridDim.y * kSpan) {
      float* z = p.z + row * p.cols + n0;
      const int64_t left = p.cols - n0;
      float v[kSpanValues];
#pragma unroll
      for (int i = 0; i < kSpanValues; ++i) v[i] = lane + 64 * i < left ? z[lane + 64 * i] : -INFINITY;
      const int from = (int)(p.v0 + n0);
      // f(column of the span's, p) for the row's ids
      auto entries = [&](auto f) __attribute__((always_inline)) {
        if (p.target != nullptr) {
          float flag;
          const int at = target_of(p, row, &flag) - from;
          if (at >= 0 && at < kSpan) f(at, 1.0f);
          return;
        }
        const int* ids = p.ids + row * p.k;
        for (int e = first_id(ids, (int)p.k, from); e < p.k && ids[e] < from + kSpan; ++e)
          f(ids[e] - from, p.prob[row * p.k + e]);
      };
      if constexpr (!GRAD) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < kSpanValues; ++i) top = fmaxf(top, v[i]);
        top = wave_max(top);
        const float base = top == -INFINITY ? 0.0f : top;
        float rest = 0.0f, most = 0.0f;
#pragma unroll
        for (int i = 0; i < kSpanValues; ++i) {
          rest += below(v[i], base, c);
          most += v[i] == base ? 1.0f : 0.0f;
        }
        rest = wave_sum(rest);
        most = wave_sum(most);
        if (top > -INFINITY) rest += most - 1.0f;
        float dot = 0.0f;
        entries([&](int at, float prob) {
          if (prob != 0.0f) dot += prob * z[at];
        });
        if (lane == 0) {
          float* out = p.stats + ((p.v0 + n0) / kSpan) * p.T + row;
          out[0] = top;
          out[p.tiles * p.T] = rest;
          out[2 * p.tiles * p.T] = dot;
        }
      } else {
        const float top = p.top[row], rest = p.rest[row], weight = p.weight[row];
        const float part = weight / (1.0f + rest);
#pragma unroll
        for (int i = 0; i < kSpanValues; ++i) v[i] = exp2f((v[i] - top) * c);
        entries([&](int at, float prob) __attribute__((always_inline)) {
#pragma unroll
          for (int i = 0; i < kSpanValues; ++i) {
            const float here = lane + 64 * i == at ? prob : 0.0f;
            v[i] = __builtin_fmaf(-here, rest, v[i] - here);
          }
        });
#pragma unroll
        for (int i = 0; i < kSpanValues; ++i)
          if (lane + 64 * i < left) z[lane + 64 * i] = weight == 0.0f ? 0.0f : v[i] * part;
      }
    }
  }
}

// ---- rows ---------------------------------------------------------------------------
// The row's loss from its top, rest and dot = sum_j p_j z_j, and what is kept of it.
__device__ __forceinline__ void finish_row(const VocabParams& p, int64_t row, float top, float rest,
                                           float dot, float* __restrict__ loss) {
  float flag, entropy = 0.0f;
  if (p.target != nullptr) {
    target_of(p, row, &flag);
    p.flag[row] = flag;
  } else {
    flag = p.flag[row];
    entropy = p.entropy[row];
  }
  p.top[row] = top;
  if (top == INFINITY) rest = NAN;  // (inf - inf, as everywhere else in the row)
  p.rest[row] = rest;
  loss[row] = flag == 0.0f ? 0.0f
              : flag != flag ? flag
                             : p.tau * p.tau * (entropy + (top - dot) / p.tau + log1pf(rest));
}
// A row's tiles joined: 16 rows a block, 64 lanes of tiles a row, joined by fours in
// a wave and then in the waves' order.  8192 rows of 256 tiles: 12 us; 33 rows 4.4, latency.
constexpr int kBlockRows = 16, kRowWaves = 16;
__global__ __launch_bounds__(64 * kRowWaves) void vocab_rows_kernel(VocabParams p,
                                                                    float* __restrict__ loss) {
  __shared__ float red[3][kRowWaves][kBlockRows];
  const int r = threadIdx.x % kBlockRows, tl = threadIdx.x / kBlockRows, wave = threadIdx.x >> 6;
  const float c = kLog2e / p.tau;
  for (int64_t row0 = (int64_t)blockIdx.x * kBlockRows; row0 < p.T;
       row0 += (int64_t)gridDim.x * kBlockRows) {
    const int64_t row = row0 + r;
    float top = -INFINITY, rest = 0.0f, dot = 0.0f;
    if (row < p.T) {
      for (int i = tl; i < p.tiles; i += 64 * kRowWaves / kBlockRows) {
        const float* at = p.stats + (int64_t)i * p.T + row;
        join(&top, &rest, at[0], at[p.tiles * p.T], c);
        dot += at[2 * p.tiles * p.T];
      }
    }
#pragma unroll
    for (int m = kBlockRows; m < 64; m *= 2) {
      const float other = __shfl_xor(top, m), s = __shfl_xor(rest, m);
      join(&top, &rest, other, s, c);
      dot += __shfl_xor(dot, m);
    }
    if ((threadIdx.x & 63) < kBlockRows) {
      red[0][wave][r] = top;
      red[1][wave][r] = rest;
      red[2][wave][r] = dot;
    }
    __syncthreads();
    if (threadIdx.x < kBlockRows && row < p.T) {
#pragma unroll
      for (int i = 1; i < kRowWaves; ++i) {
        join(&top, &rest, red[0][i][r], red[1][i][r], c);
        dot += red[2][i][r];
      }
      finish_row(p, row, top, rest, dot, loss);
    }
    __syncthreads();
  }
}

// ---- few classes ----------------------------------------------------------------------
// Up to kFewClasses columns: 16 rows and all columns a block, x and W straight from
// memory into matrix instructions (few_rows), whose sums are a row's logits, its loss
// and what is kept of it.  The logits are kept, being fewer than x's values.
// 4096 rows of 256 -> 10 in fp32: 4.6 us and one launch; the product on a tile, the
// span kernel and the rows' kernel took 32.  65536 rows of 1024 -> 64 in bf16: 95 us
// forward this way, 53 on tiles; forward and backward 249 and 252.
constexpr int64_t kFewClasses = 32;
template <typename T, int NC, bool WHOLE>
__global__ __launch_bounds__(256) void vocab_few_kernel(VocabParams p, float* __restrict__ loss) {
  typedef RowsMma<T> M;
  __shared__ float red[4][kFewRows][16 * NC + 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int64_t m0 = (int64_t)blockIdx.x * kFewRows; m0 < p.T;
       m0 += (int64_t)gridDim.x * kFewRows) {
    typename M::acc_t acc[NC];
    const T* w[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      acc[c] = {0.0f, 0.0f, 0.0f, 0.0f};
      w[c] = static_cast<const T*>(p.w) + min((int64_t)(16 * c + (lane & 15)), p.V - 1) * p.D;
    }
    const T* x = static_cast<const T*>(p.x) + min(m0 + (lane & 15), p.T - 1) * p.D;
    few_rows<T, NC, WHOLE>(x, w, p.D, acc);
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int v = 0; v < 4; ++v) red[wave][lane & 15][16 * c + 4 * (lane >> 4) + v] = acc[c][v];
    __syncthreads();
    // 16 lanes a row, column 16 c + lane at z[c]
    const int r = threadIdx.x >> 4, l = threadIdx.x & 15;
    const int64_t row = m0 + r;
    if (row < p.T) {
      const float c2 = kLog2e / p.tau;
      float z[NC], top = -INFINITY, rest = 0.0f, most = 0.0f, dot = 0.0f;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int v = 16 * c + l;
        z[c] = -INFINITY;
        if (v < p.V) {
          z[c] = red[0][r][v] + red[1][r][v] + red[2][r][v] + red[3][r][v];
          p.logits[row * p.V + v] = z[c];
        }
        top = fmaxf(top, z[c]);
      }
#pragma unroll
      for (int m = 1; m < 16; m *= 2) top = fmaxf(top, __shfl_xor(top, m));
      const float from = top == -INFINITY ? 0.0f : top;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        rest += below(z[c], from, c2);
        most += z[c] == from ? 1.0f : 0.0f;
      }
      auto add = [&](int id, float prob) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < NC; ++c)
          if (16 * c + l == id && prob != 0.0f) dot += prob * z[c];
      };
      if (p.target != nullptr) {
        float flag;
        add(target_of(p, row, &flag), 1.0f);
      } else {
        for (int e = 0; e < p.k; ++e) add(p.ids[row * p.k + e], p.prob[row * p.k + e]);
      }
      rest = lane_sum<16>(rest);
      most = lane_sum<16>(most);
      if (top > -INFINITY) rest += most - 1.0f;
      dot = lane_sum<16>(dot);
      if (l == 0) finish_row(p, row, top, rest, dot, loss);
    }
    __syncthreads();
  }
}

// ---- sums of the rows -------------------------------------------------------------------
constexpr int kOneBlock = 1024;
template <typename V>
__device__ __forceinline__ V block_total(V v, V* red) {
  __syncthreads();
  red[threadIdx.x] = v;
  __syncthreads();
  for (int m = kOneBlock / 2; m > 0; m /= 2) {
    if (threadIdx.x < m) red[threadIdx.x] += red[threadIdx.x + m];
    __syncthreads();
  }
  return red[0];
}
// The sum or mean of the rows that count.
__global__ __launch_bounds__(kOneBlock) void vocab_sum_kernel(VocabParams p,
                                                              const float* __restrict__ rows,
                                                              int mean, float* __restrict__ loss) {
  __shared__ double red[kOneBlock];
  double sum = 0.0, count = 0.0;
#pragma unroll 8
  for (int64_t t = threadIdx.x; t < p.T; t += kOneBlock) {
    sum += rows[t];
    count += p.flag[t] == 0.0f ? 0.0 : 1.0;
  }
  sum = block_total(sum, red);
  count = block_total(count, red);
  if (threadIdx.x != 0) return;
  *p.count = (float)count;
  *loss = (float)(mean ? sum / (count > 0.0 ? count : 1.0) : sum);
}

// w and the common factor from the gradient of the loss: of a scalar loss g is one
// value (over the count for a mean) and w = flag; of the rows' losses w = g_t /
// max|g|, or in fp32 g_t; w times `unit`, a power of 2.  fp32: w is the whole factor.
struct Upstream {
  const float* g;
  int reduction, fp32;
  float unit;
  const float* most;  // the largest finite |g| of the rows' losses in 16 bits
  float* scale;
};
__device__ __forceinline__ float common_of(const VocabParams& p, const Upstream& u) {
  if (u.reduction == KAN_REDUCE_NONE) return u.fp32 ? p.tau : p.tau * *u.most;
  const float c = p.tau * *u.g;
  return u.reduction == KAN_REDUCE_MEAN ? c / fmaxf(*p.count, 1.0f) : c;
}
__device__ __forceinline__ float weight_of(const VocabParams& p, const Upstream& u, int64_t row,
                                           float common) {
  const float flag = p.flag[row];
  float w = flag;
  if (u.reduction == KAN_REDUCE_NONE) w = u.fp32 ? flag * u.g[row] : flag * u.g[row] / *u.most;
  return flag == 0.0f ? 0.0f : w * (u.fp32 ? common : u.unit);
}
__global__ __launch_bounds__(kOneBlock) void vocab_most_kernel(VocabParams p,
                                                               const float* __restrict__ g,
                                                               float* __restrict__ out) {
  __shared__ float red[kOneBlock];
  float most = 0.0f;
#pragma unroll 8
  for (int64_t t = threadIdx.x; t < p.T; t += kOneBlock)
    most = fmaxf(most, p.flag[t] != 0.0f && fabsf(g[t]) < INFINITY ? fabsf(g[t]) : 0.0f);
  red[threadIdx.x] = most;
  __syncthreads();
  for (int m = kOneBlock / 2; m > 0; m /= 2) {
    if (threadIdx.x < m) red[threadIdx.x] = fmaxf(red[threadIdx.x], red[threadIdx.x + m]);
    __syncthreads();
  }
  if (threadIdx.x == 0) *out = red[0] == 0.0f ? 1.0f : red[0];
}

// The rows' weights and, for the weight's gradient, x's rows, those that do not count
// as zeros: what they hold may be anything, and 0 times NaN is NaN.  [T, D] -> [T, ld],
// zeros behind D (8192 x 2048 in bf16: 13 us); ld 0: none; a second time behind them with
// a second part of dz.  FEW: also dz of few classes from their kept logits, in 16 bits with
// zeros as far as 16 bytes go.
template <typename T, bool FEW>
__global__ __launch_bounds__(256) void vocab_prepare_kernel(VocabParams p, Upstream u,
                                                            T* __restrict__ out, int64_t ld,
                                                            int whole) {
  constexpr int V = 16 / sizeof(T);
  typedef typename VecOf<T, V>::type vec;
  const int64_t first = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
  const float common = common_of(p, u);
  if (first == 0) *u.scale = common / u.unit;
  for (int64_t row = first; row < p.T; row += step) p.weight[row] = weight_of(p, u, row, common);
  if constexpr (FEW) {
    const float c = kLog2e / p.tau;
    const int64_t cols = sizeof(T) == 2 ? round_up(p.V, 8) : p.V;
    for (int64_t i = first; i < p.T * cols; i += step) {
      const int64_t row = i / cols, v = i - row * cols;
      const float weight = weight_of(p, u, row, common);
      float d = 0.0f;
      if (v < p.V && weight != 0.0f) {
        const float rest = p.rest[row];
        auto take = [&](float prob) { d = __builtin_fmaf(-prob, rest, d - prob); };
        d = exp2f((p.logits[row * p.V + v] - p.top[row]) * c);
        if (p.target != nullptr) {
          float flag;
          if (target_of(p, row, &flag) == v) take(1.0f);
        } else {
          for (int e = 0; e < p.k; ++e)
            if (p.ids[row * p.k + e] == v) take(p.prob[row * p.k + e]);
        }
        d *= weight / (1.0f + rest);
      }
      const T whole = (T)d;
      static_cast<T*>(p.G)[row * p.ldg + v] = whole;
      if (p.G2 != nullptr) static_cast<T*>(p.G2)[row * p.ldg + v] = (T)(d - (float)whole);
    }
  }
  const int64_t per = ceil_div(ld, V), total = p.T * per;
  for (int64_t i = first; i < total; i += step) {
    const int64_t row = i / per, c = (i - row * per) * V;
    const T* src = static_cast<const T*>(p.x) + row * p.D + c;
    const bool on = p.flag[row] != 0.0f;
    vec v;
    if (on && c + V <= p.D) {
      v = reinterpret_cast<const LooseVec<T, V>*>(src)->v;
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = on && c + j < p.D ? src[j] : (T)0.0f;
    }
    for (int64_t to = row; to < p.T * (p.G2 != nullptr ? 2 : 1); to += p.T) {
      if (whole) {
        *reinterpret_cast<vec*>(out + to * ld + c) = v;
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (c + j < ld) out[to * ld + c + j] = v[j];
      }
    }
  }
}

// acc (+)= the sum of `cuts` slices; the last piece's call gives out = acc * scale.
template <typename T>
__global__ __launch_bounds__(256) void vocab_add_kernel(const float* __restrict__ part, int cuts,
                                                        int64_t count, float* __restrict__ acc,
                                                        int start, const float* __restrict__ scale,
                                                        T* __restrict__ out) {
  const float factor = scale == nullptr ? 1.0f : *scale;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count;
       i += (int64_t)gridDim.x * 256) {
    float v = part[i];
#pragma unroll 8
    for (int q = 1; q < cuts; ++q) v += part[q * count + i];
    if (!start) v += acc[i];
    if (out == nullptr) acc[i] = v;
    else out[i] = (T)(v * factor);
  }
}

// ---- host -----------------------------------------------------------------------------
// Places in a workspace, each on 16 bytes.
struct Places {
  char* base;
  size_t bytes;
  template <typename T = char>
  T* take(size_t count) {
    T* at = reinterpret_cast<T*>(base + bytes);
    bytes = (size_t)round_up((int64_t)(bytes + count * sizeof(T)), 16);
    return at;
  }
};

// 512 MiB of a piece's logits or dz: 8192 rows of 32768 columns in 16 bits, products
// that are as long as the tiles can use; past 262144 rows (131072 in fp32) 1024 columns,
// whatever they take.
constexpr int64_t kPieceBytes = (int64_t)1 << 29;
int64_t piece_columns(int dtype, int64_t T, int64_t V) {
  const int64_t most =
      std::max<int64_t>(kSpan, kPieceBytes / (T * (int64_t)dtype_bytes(dtype)) / kSpan * kSpan);
  if (most >= V) return V;
  return round_up(ceil_div(V, ceil_div(V, most)), kSpan);
}
// Values between rows of dz in 16 bits: an odd number of 128 bytes, so that a tile's
// rows spread over the memory's channels.
int64_t padded(int64_t cols) { return round_up(cols, 128) + 64; }
// (k 0: cross entropy)
size_t kept_floats(int64_t T, int64_t V, int64_t k) {
  return (size_t)(3 * T + 4 + 2 * T * k) + (V <= kFewClasses ? (size_t)(T * V) : 0);
}
void set_kept(VocabParams* p, void* kept) {
  p->top = static_cast<float*>(kept);
  p->rest = p->top + p->T;
  p->flag = p->rest + p->T;
  p->count = p->flag + p->T;
  p->prob = p->count + 4;
  p->ids = reinterpret_cast<int*>(p->prob + p->T * p->k);
  p->logits = p->prob + 2 * p->T * p->k;
}
GroupedParams product_of(int64_t T, int64_t N, int64_t K) {
  GroupedParams g{};
  g.E = 1;
  g.T = T;
  g.N = N;
  g.K = K;
  g.lda = g.ldb = K;
  return g;
}
// (the products' own rule for few rows does not hold here: those tiles end in sums)
HalfCfg tile_of(int64_t T, int64_t cols, int64_t D) {
  return half_plan(KAN_GROUPED_FORWARD, T, 1, cols, D).cfg;
}
int64_t tile_columns(HalfCfg cfg) { return cfg == kSmall ? 128 : 256; }

// Whether dz is taken in two parts of 16 bits, one behind the other as 2 T rows of the
// second products.  The error of a single rounding is spread over all values that a sum
// takes in, and vanishes in the gradient's own; with few rows or columns there is little to
// spread it over, and it made the gradients' error 1.5 to 3 times that of their own
// rounding.  The second part costs little there (bf16, forward and backward; one row more
// is one part): 64 rows of 4096 -> 131072 1.21 ms, 65 1.13; 512 of 512 -> 8192 150 us, 513
// 145; 2000 of 1024 -> 1024 153 us.  131072 rows of 1024 -> 16 took 0.95 ms so and take 0.36.
bool in_parts(int64_t T, int64_t V, int64_t D) {
  return T <= 64 || (T <= 4096 && T * V <= ((int64_t)1 << 31) / D);
}
HalfPlan plan_product(int dtype, int op, int64_t T, int64_t cols, int64_t D) {
  if (dtype != KAN_DTYPE_F32 && op == KAN_GROUPED_INPUT) return long_plan(T, cols, D);
  return product_plan(dtype, op, T, 1, cols, D, true);
}

template <typename T, class G, int PARTS>
int launch_vocab_tile(const VocabParams& p, hipStream_t st) {
  const int64_t tiles_n = ceil_div(p.cols, G::BN), blocks = dense_grid(p.T, G::BM, tiles_n);
  if (!grid_fits(blocks, G::NT)) return set_error(KAN_ERR_LIMIT, "vocab_loss: too many tiles");
  if (whole_rows(p.x, p.ldx) && whole_rows(p.w, p.ldw))
    vocab_tile_kernel<T, G, kDirect, PARTS><<<dim3((unsigned)blocks), G::NT, 0, st>>>(p, (int)tiles_n);
  else
    vocab_tile_kernel<T, G, kGuarded, PARTS><<<dim3((unsigned)blocks), G::NT, 0, st>>>(p, (int)tiles_n);
  return check_launch("vocab_loss");
}
template <typename T, int PARTS>
int launch_vocab_half(const VocabParams& p, HalfCfg cfg, hipStream_t st) {
  if constexpr (PARTS == 2) return launch_vocab_tile<T, TileSmall, 2>(p, st);
  else
    return cfg == kBig   ? launch_vocab_tile<T, TileBig, PARTS>(p, st)
           : cfg == kMid ? launch_vocab_tile<T, TileMid, PARTS>(p, st)
                         : launch_vocab_tile<T, TileSmall, PARTS>(p, st);
}
template <int PARTS>
int launch_vocab_tiles(int dtype, const VocabParams& p, HalfCfg cfg, hipStream_t st) {
  return dtype == KAN_DTYPE_BF16 ? launch_vocab_half<bf16, PARTS>(p, cfg, st)
                                 : launch_vocab_half<f16, PARTS>(p, cfg, st);
}
template <bool GRAD>
int launch_vocab_span(const VocabParams& p, hipStream_t st) {
  const int64_t spans = std::min<int64_t>(ceil_div(p.cols, kSpan), 65535);
  vocab_span_kernel<GRAD><<<dim3(row_blocks(p.T, 4), (unsigned)spans), 256, 0, st>>>(p);
  return check_launch("vocab_loss");
}

int check_vocab(const char* who, int dtype, int64_t T, int64_t V, int64_t D, int64_t k, double tau,
                int reduction) {
  if (!dtype_is_operator(dtype))
    return set_error(KAN_ERR_INVALID, "%s: dtype must be FP32, BF16 or FP16 (code %d)", who, dtype);
  if (T < 0 || V < 1 || D < 1 || k < 1)
    return set_error(KAN_ERR_INVALID, "%s: sizes must be positive", who);
  if (!(tau > 0.0) || tau > 1e30 || tau < 1e-30)
    return set_error(KAN_ERR_INVALID, "%s: the temperature must be positive and finite", who);
  if (reduction < KAN_REDUCE_NONE || reduction > KAN_REDUCE_MEAN)
    return set_error(KAN_ERR_INVALID, "%s: unknown reduction %d", who, reduction);
  if (T > 0x3fffffff || V > (1 << 22) || D > (1 << 22) || k > kMaxTop)
    return set_error(KAN_ERR_LIMIT,
                     "%s: at most 2^30 - 1 rows, 2^22 columns and inputs and %d ids a row", who,
                     (int)kMaxTop);
  return KAN_OK;
}

// ---- a call's workspace ------------------------------------------------------------------
struct ForwardPlan {
  HalfCfg cfg;
  AlignPlan align;
  int64_t piece;
  HalfPlan product;  // fp32
  char* aligned;
  float *stats, *entropy, *rows, *z, *part;
  int tiles;
  size_t bytes;
};
ForwardPlan plan_forward(int dtype, const void* x, const void* w, int64_t T, int64_t V, int64_t D,
                         char* ws) {
  ForwardPlan f{};
  Places at{ws, 0};
  f.piece = V;
  if (V <= kFewClasses) {
  } else if (dtype == KAN_DTYPE_F32) {
    f.piece = piece_columns(dtype, T, V);
    f.tiles = (int)ceil_div(V, kSpan);
    f.product = product_plan(dtype, KAN_GROUPED_FORWARD, T, 1, f.piece, D);
    f.z = at.take<float>((size_t)(T * f.piece));
    // (a shorter last piece may be cut more often, but never into more values)
    size_t part = product_part_bytes(KAN_GROUPED_FORWARD, f.product, T, 1, f.piece, D);
    const int64_t rest = V % f.piece;
    if (rest != 0)
      part = std::max(part, product_part_bytes(KAN_GROUPED_FORWARD,
                                               product_plan(dtype, KAN_GROUPED_FORWARD, T, 1, rest, D),
                                               T, 1, rest, D));
    f.part = part == 0 ? nullptr : at.take<float>(part / 4);
  } else {
    f.cfg = tile_of(T, V, D);
    f.tiles = (int)ceil_div(V, tile_columns(f.cfg));
    f.align = align_operands(x, T, D, w, V, D, 2, align_saves_us(KAN_GROUPED_FORWARD, T, V, D));
    f.aligned = at.take(f.align.a_bytes + f.align.b_bytes);
  }
  f.stats = at.take<float>((size_t)(3 * T) * (size_t)f.tiles);
  f.entropy = at.take<float>((size_t)T);
  f.rows = at.take<float>((size_t)T);
  f.bytes = at.bytes;
  return f;
}

struct BackwardPlan {
  HalfCfg cfg;
  AlignPlan align;
  int64_t piece, ldg, ldx;
  int parts;        // of dz
  bool sliced;      // dx is added from slices
  char *rows, *aligned, *G;  // rows: x's for the weight's gradient
  float *weight, *scale, *most, *part, *slices, *acc;
  size_t bytes;
};
BackwardPlan plan_backward(int dtype, const void* x, const void* w, int64_t T, int64_t V, int64_t D,
                           bool dx, bool dw, char* ws) {
  BackwardPlan b{};
  Places at{ws, 0};
  const bool half = dtype != KAN_DTYPE_F32;
  b.piece = piece_columns(dtype, T, V);
  b.parts = half && in_parts(T, V, D) ? 2 : 1;
  b.sliced = b.piece < V || b.parts == 2;
  b.ldg = half ? padded(b.piece) : b.piece;
  if (half) {
    b.cfg = tile_of(T, b.piece, D);
    double saved = align_saves_us(KAN_GROUPED_FORWARD, T, V, D);
    if (dx) saved += align_saves_us(KAN_GROUPED_INPUT, T, V, D);
    if (dw) saved += align_saves_us(KAN_GROUPED_WEIGHT, T, V, D);
    // (rows copied for dw lie on 16 bytes)
    b.align = align_operands(dw ? nullptr : x, T, dw ? round_up(D, 8) : D, w, V, D, 2, saved);
    b.aligned = at.take(b.align.a_bytes + b.align.b_bytes);
  }
  b.ldx = half ? round_up(D, 8) : D;
  if (dw) b.rows = at.take((size_t)(b.parts * T * b.ldx) * dtype_bytes(dtype));
  b.weight = at.take<float>((size_t)T);
  b.scale = at.take<float>(1);
  b.most = at.take<float>(1);
  b.G = at.take((size_t)(b.parts * T * b.ldg) * dtype_bytes(dtype));
  size_t part = 0, slices = 0;
  const int64_t rest = V % b.piece;
  for (const int64_t cols : {b.piece, rest}) {
    if (cols == 0) continue;
    auto need = [&](int op) {
      const int64_t rows = op == KAN_GROUPED_FORWARD ? T : b.parts * T;
      return product_part_bytes(op, plan_product(dtype, op, rows, cols, D), rows, 1, cols, D);
    };
    if (!half && V > kFewClasses) part = std::max(part, need(KAN_GROUPED_FORWARD));
    if (dw) part = std::max(part, need(KAN_GROUPED_WEIGHT));
    if (dx && (!half || !b.sliced)) part = std::max(part, need(KAN_GROUPED_INPUT));
    else if (dx) slices = std::max(slices, need(KAN_GROUPED_INPUT));
  }
  if (dx && b.sliced) {
    slices = std::max(slices, 4 * (size_t)(b.parts * T * D));
    b.slices = at.take<float>(slices / 4);
    if (b.piece < V) b.acc = at.take<float>((size_t)(T * D));
  }
  b.part = part == 0 ? nullptr : at.take<float>(part / 4);
  b.bytes = at.bytes;
  return b;
}

template <typename T>
void launch_prepare(const VocabParams& p, const Upstream& u, char* out, int64_t ld,
                    hipStream_t st) {
  constexpr int64_t V = 16 / sizeof(T);
  const bool few = p.V <= kFewClasses;
  const int64_t most = p.T * std::max<int64_t>(ceil_div(ld, V), few ? p.V : 1);
  const dim3 blocks((unsigned)std::min<int64_t>(ceil_div(most, 256), 1 << 16));
  T* to = reinterpret_cast<T*>(out);
  if (few) vocab_prepare_kernel<T, true><<<blocks, 256, 0, st>>>(p, u, to, ld, ld % V == 0);
  else vocab_prepare_kernel<T, false><<<blocks, 256, 0, st>>>(p, u, to, ld, ld % V == 0);
}
template <typename T, bool WHOLE>
int launch_few_classes(const VocabParams& p, float* loss, hipStream_t st) {
  const unsigned blocks = row_blocks(p.T, kFewRows);
  if (p.V <= 16) vocab_few_kernel<T, 1, WHOLE><<<blocks, 256, 0, st>>>(p, loss);
  else vocab_few_kernel<T, 2, WHOLE><<<blocks, 256, 0, st>>>(p, loss);
  return check_launch("vocab_loss");
}
template <typename T>
int launch_few_forward(const VocabParams& p, float* loss, hipStream_t st) {
  if (sizeof(T) == 2 && !(whole_rows(p.x, p.D) && whole_rows(p.w, p.D)))
    return launch_few_classes<T, false>(p, loss, st);
  return launch_few_classes<T, true>(p, loss, st);
}
template <typename T>
void launch_add(const float* part, int cuts, int64_t count, float* acc, bool start,
                const float* scale, void* out, hipStream_t st) {
  vocab_add_kernel<T><<<dim3((unsigned)std::min<int64_t>(ceil_div(count, 256), 8192)), 256, 0, st>>>(
      part, cuts, count, acc, start ? 1 : 0, scale, static_cast<T*>(out));
}

}  // namespace
}  // namespace kan

using namespace kan;

extern "C" {

int kan_hip_vocab_loss_kept(int64_t T, int64_t V, int64_t k, size_t* bytes) {
  if (bytes == nullptr) return set_error(KAN_ERR_INVALID, "vocab_loss_kept: bytes must not be NULL");
  const int rc = check_vocab("vocab_loss_kept", KAN_DTYPE_F32, T, V, 1, k + (k == 0), 1.0, 0);
  if (rc != KAN_OK) return rc;
  *bytes = 4 * kept_floats(T, V, k);
  return KAN_OK;
}

int kan_hip_vocab_loss_workspace(int dtype, const void* x, const void* w, int64_t T, int64_t V,
                                 int64_t D, size_t* bytes) {
  if (bytes == nullptr)
    return set_error(KAN_ERR_INVALID, "vocab_loss_workspace: bytes must not be NULL");
  const int rc = check_vocab("vocab_loss_workspace", dtype, T, V, D, 1, 1.0, 0);
  if (rc != KAN_OK) return rc;
  *bytes = T == 0 ? 0 : plan_forward(dtype, x, w, T, V, D, nullptr).bytes;
  return KAN_OK;
}

int kan_hip_vocab_loss(int dtype, const void* x, const void* w, const void* ids, int ids64,
                       const float* teacher, int64_t T, int64_t V, int64_t D, int64_t k,
                       int64_t ignore_index, double temperature, int reduction, float* loss,
                       void* kept, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "vocab_loss";
  const int rc = check_vocab(who, dtype, T, V, D, k + (k == 0), temperature, reduction);
  if (rc != KAN_OK) return rc;
  if ((teacher == nullptr) != (k == 0))
    return set_error(KAN_ERR_INVALID, "%s: k is 0 without a teacher and positive with one", who);
  if (T == 0) return KAN_OK;
  if (x == nullptr || w == nullptr || ids == nullptr || loss == nullptr || kept == nullptr)
    return set_error(KAN_ERR_INVALID, "%s: operands must not be NULL", who);
  if (!aligned16(kept) || !aligned16(workspace))
    return set_error(KAN_ERR_INVALID, "%s: kept values and the workspace lie on 16 bytes", who);
  const ForwardPlan f = plan_forward(dtype, x, w, T, V, D, static_cast<char*>(workspace));
  if (workspace == nullptr || workspace_bytes < f.bytes)
    return set_error(KAN_ERR_WORKSPACE, "%s: needs %zu bytes of workspace, got %zu", who, f.bytes,
                     workspace == nullptr ? (size_t)0 : workspace_bytes);
  VocabParams p{};
  p.x = x;
  p.w = w;
  p.T = T;
  p.V = V;
  p.D = p.ldx = p.ldw = D;
  p.k = k;
  p.tau = (float)temperature;
  set_kept(&p, kept);
  p.entropy = f.entropy;
  p.stats = f.stats;
  p.tiles = f.tiles;
  p.cols = V;
  hipStream_t st = static_cast<hipStream_t>(stream);
  TimedLaunch timed(kClassContraction, st, 2.0 * (double)T * (double)V * (double)D);
  int e = KAN_OK;
  if (teacher == nullptr) {
    p.target = ids;
    p.target64 = ids64;
    p.ignore = ignore_index;
  } else {
    vocab_teacher_kernel<<<row_blocks(T, 1), 64, 0, st>>>(p, ids, ids64, teacher);
    e = check_launch(who);
  }
  float* rows = reduction == KAN_REDUCE_NONE ? loss : f.rows;
  const bool few = V <= kFewClasses;
  if (few && e == KAN_OK)
    e = dtype == KAN_DTYPE_F32    ? launch_few_forward<float>(p, rows, st)
        : dtype == KAN_DTYPE_BF16 ? launch_few_forward<bf16>(p, rows, st)
                                  : launch_few_forward<f16>(p, rows, st);
  if (e != KAN_OK) return e;
  if (!few && dtype != KAN_DTYPE_F32) {
    GroupedParams g = product_of(T, V, D);
    g.A = x;
    g.B = w;
    e = launch_aligned(f.align, &g, f.aligned, st);
    if (e != KAN_OK) return e;
    p.x = g.A;
    p.w = g.B;
    p.ldx = g.lda;
    p.ldw = g.ldb;
    e = launch_vocab_tiles<0>(dtype, p, f.cfg, st);
    if (e != KAN_OK) return e;
  }
  for (p.v0 = 0; !few && dtype == KAN_DTYPE_F32 && p.v0 < V; p.v0 += f.piece) {
    p.cols = std::min(f.piece, V - p.v0);
    p.z = f.z;
    GroupedParams g = product_of(T, p.cols, D);
    g.A = x;
    g.B = static_cast<const float*>(w) + p.v0 * D;
    g.C = f.z;
    const HalfPlan pl = product_plan(dtype, KAN_GROUPED_FORWARD, T, 1, p.cols, D);
    g.part = pl.cuts > 1 ? f.part : nullptr;
    e = launch_product(dtype, KAN_GROUPED_FORWARD, g, pl, st);
    if (e == KAN_OK) e = launch_vocab_span<false>(p, st);
    if (e != KAN_OK) return e;
  }
  if (!few)
    vocab_rows_kernel<<<row_blocks(T, kBlockRows), 64 * kRowWaves, 0, st>>>(p, rows);
  if (reduction != KAN_REDUCE_NONE)
    vocab_sum_kernel<<<1, kOneBlock, 0, st>>>(p, rows, reduction == KAN_REDUCE_MEAN, loss);
  return check_launch(who);
}

int kan_hip_vocab_loss_backward_workspace(int dtype, const void* x, const void* w, int64_t T,
                                          int64_t V, int64_t D, int with_dx, int with_dw,
                                          size_t* bytes) {
  if (bytes == nullptr)
    return set_error(KAN_ERR_INVALID, "vocab_loss_backward_workspace: bytes must not be NULL");
  const int rc = check_vocab("vocab_loss_backward_workspace", dtype, T, V, D, 1, 1.0, 0);
  if (rc != KAN_OK) return rc;
  *bytes = T == 0 ? 0 : plan_backward(dtype, x, w, T, V, D, with_dx != 0, with_dw != 0, nullptr).bytes;
  return KAN_OK;
}

int kan_hip_vocab_loss_backward(int dtype, const float* grad_loss, const void* x, const void* w,
                                const void* ids, int ids64, const void* kept, int64_t T, int64_t V,
                                int64_t D, int64_t k, int64_t ignore_index, double temperature,
                                int reduction, void* grad_x, void* grad_w, void* workspace,
                                size_t workspace_bytes, void* stream) {
  const char* who = "vocab_loss_backward";
  const int rc = check_vocab(who, dtype, T, V, D, k + (k == 0), temperature, reduction);
  if (rc != KAN_OK) return rc;
  if (T == 0 || (grad_x == nullptr && grad_w == nullptr)) return KAN_OK;
  if (grad_loss == nullptr || x == nullptr || w == nullptr || kept == nullptr ||
      (k == 0 && ids == nullptr))
    return set_error(KAN_ERR_INVALID, "%s: operands must not be NULL", who);
  if (!aligned16(kept) || !aligned16(workspace))
    return set_error(KAN_ERR_INVALID, "%s: kept values and the workspace lie on 16 bytes", who);
  const BackwardPlan b = plan_backward(dtype, x, w, T, V, D, grad_x != nullptr, grad_w != nullptr,
                                       static_cast<char*>(workspace));
  if (workspace == nullptr || workspace_bytes < b.bytes)
    return set_error(KAN_ERR_WORKSPACE, "%s: needs %zu bytes of workspace, got %zu", who, b.bytes,
                     workspace == nullptr ? (size_t)0 : workspace_bytes);
  const bool half = dtype != KAN_DTYPE_F32;
  const int64_t value = (int64_t)dtype_bytes(dtype);
  hipStream_t st = static_cast<hipStream_t>(stream);
  TimedLaunch timed(kClassContraction, st, 6.0 * (double)T * (double)V * (double)D);
  VocabParams p{};
  p.T = T;
  p.V = V;
  p.D = D;
  p.k = k;
  p.tau = (float)temperature;
  if (k == 0) {
    p.target = ids;
    p.target64 = ids64;
    p.ignore = ignore_index;
  }
  set_kept(&p, const_cast<void*>(kept));
  p.weight = b.weight;
  p.x = x;
  p.G = b.G;
  if (b.parts == 2) p.G2 = b.G + T * b.ldg * value;
  p.z = reinterpret_cast<float*>(b.G);
  p.ldg = b.ldg;
  GroupedParams in = product_of(T, V, D);
  in.A = x;
  in.B = w;
  const Upstream up{grad_loss, reduction, half ? 0 : 1, dtype == KAN_DTYPE_F16 ? 32768.0f : 1.0f,
                    b.most, b.scale};
  if (half && reduction == KAN_REDUCE_NONE)
    vocab_most_kernel<<<1, kOneBlock, 0, st>>>(p, grad_loss, b.most);
  const int64_t ld = grad_w == nullptr ? 0 : b.ldx;
  if (dtype == KAN_DTYPE_F32) launch_prepare<float>(p, up, b.rows, ld, st);
  else if (dtype == KAN_DTYPE_BF16) launch_prepare<bf16>(p, up, b.rows, ld, st);
  else launch_prepare<f16>(p, up, b.rows, ld, st);
  if (ld > 0) {
    in.A = b.rows;
    in.lda = ld;
  }
  int e = launch_aligned(b.align, &in, b.aligned, st);
  if (e != KAN_OK) return e;
  p.x = in.A;
  p.w = in.B;
  p.ldx = in.lda;
  p.ldw = in.ldb;
  if (e == KAN_OK) e = check_launch(who);
  const bool few = V <= kFewClasses;
  for (p.v0 = 0; e == KAN_OK && p.v0 < V; p.v0 += b.piece) {
    p.cols = std::min(b.piece, V - p.v0);
    const char* wp = static_cast<const char*>(p.w) + p.v0 * p.ldw * value;
    auto product = [&](int op, const void* A, int64_t lda, const void* B, int64_t ldb, void* C,
                       float* part) {
      const int64_t rows = op == KAN_GROUPED_FORWARD ? T : b.parts * T;
      GroupedParams g = product_of(rows, p.cols, D);
      g.A = A;
      g.B = B;
      g.lda = lda;
      g.ldb = ldb;
      g.C = C;
      g.scale = half ? b.scale : nullptr;
      const HalfPlan pl = plan_product(dtype, op, rows, p.cols, D);
      g.part = C == nullptr || product_part_bytes(op, pl, rows, 1, p.cols, D) > 0 ? part : nullptr;
      return launch_product(dtype, op, g, pl, st);
    };
    // dz of the piece
    p.ldg = half ? padded(p.cols) : p.cols;
    if (b.parts == 2) p.G2 = b.G + T * p.ldg * value;
    if (few) {  // (the first kernel's)
    } else if (half) {
      e = b.parts == 2 ? launch_vocab_tiles<2>(dtype, p, b.cfg, st)
                       : launch_vocab_tiles<1>(dtype, p, b.cfg, st);
    } else {
      e = product(KAN_GROUPED_FORWARD, p.x, D, wp, D, p.z, b.part);
      if (e == KAN_OK) e = launch_vocab_span<true>(p, st);
    }
    if (e == KAN_OK && grad_w != nullptr)
      e = product(KAN_GROUPED_WEIGHT, p.G, p.ldg, p.x, p.ldx,
                  static_cast<char*>(grad_w) + p.v0 * D * value, b.part);
    if (e != KAN_OK || grad_x == nullptr) continue;
    if (!b.sliced) {
      e = product(KAN_GROUPED_INPUT, p.G, p.ldg, wp, p.ldw, grad_x, b.part);
      continue;
    }
    int cuts = 1;
    if (half) {
      e = product(KAN_GROUPED_INPUT, p.G, p.ldg, wp, p.ldw, nullptr, b.slices);
      // (a cut's slice has the parts' rows one behind the other)
      cuts = b.parts * plan_product(dtype, KAN_GROUPED_INPUT, b.parts * T, p.cols, D).cuts;
    } else {
      e = product(KAN_GROUPED_INPUT, p.G, p.ldg, wp, p.ldw, b.slices, b.part);
    }
    if (e != KAN_OK) return e;
    void* out = p.v0 + b.piece >= V ? grad_x : nullptr;
    const float* scale = half ? b.scale : nullptr;
    if (dtype == KAN_DTYPE_F32) launch_add<float>(b.slices, cuts, T * D, b.acc, p.v0 == 0, scale, out, st);
    else if (dtype == KAN_DTYPE_BF16) launch_add<bf16>(b.slices, cuts, T * D, b.acc, p.v0 == 0, scale, out, st);
    else launch_add<f16>(b.slices, cuts, T * D, b.acc, p.v0 == 0, scale, out, st);
    e = check_launch(who);
  }
  return e;
}

}  // extern "C"
