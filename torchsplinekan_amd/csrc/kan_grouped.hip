// Matrix products grouped by expert with ragged sizes.  The rows t of x [T, K]
// are sorted by expert: expert e has the rows offsets[e] .. offsets[e + 1] - 1,
// offsets [E + 1] lying on the device, so that the host never waits for the
// router.  With w [E, N, K]:
//   y[t]  = w[e(t)] x[t]                    [T, N]
//   dx[t] = w[e(t)]^T dy[t]                 [T, K]
//   dw[e] = sum over t in e of dy[t] x[t]^T [E, N, K]
// Rows from offsets[E] on belong to no expert: their y and dx are zero.
//
// Sums are in float32, rounded once.  A grid covers the largest number of
// row tiles T rows can make of E groups (T / BM + E + 1); a block finds its
// group from the offsets (kan_grouped.h), and blocks past the last tile end at
// once.  float32 products run on the contraction engine's tiles (kan_gemm.hip).
#include "kan_grouped.h"
#include "kan_tile.h"

namespace kan {

namespace {

// ---- 16-bit products on MFMA (tiles: kan_tile.h) ----------------------------
// What bounds it: MFMA at the power cap.  16384 rows over 8 equal groups of 4096 x
// 4096 in bf16: forward 1.23 PFLOP/s, input 1.25, weight gradient 1.16, where
// torch.mm reaches 1.28, 1.15 and 1.02 at 8192^3; the MFMA pipes are busy for 0.55
// of the cycles at 2.0 GHz, LDS for 0.2 of them, and neither bank conflicts (5.5e7
// to 1.1e6 cycles) nor the waves' priority changed its time.  Uneven groups (0.3 to
// 2.4 times the mean) lose the empty half of their last tiles and part of the last
// round: 1.06 PFLOP/s.  Two waves a SIMD, as 4 waves of 128 x 128 were 10 % slower.
template <typename T, class G, int OP, int MA, int MB>
__global__ __launch_bounds__(G::NT) void grouped_tile_kernel(GroupedParams p, int tiles_m,
                                                             int tiles_n, int store_vec) {
  constexpr bool KA = OP != 2, KB = OP == 0;
  constexpr int BM = G::BM, BN = G::BN, FM = G::FM, FN = G::FN;
  __shared__ __align__(16) char lds[2 * G::kBuf];

  // the tile: rows [m0, m_end) and columns [n0, n_end) of the output, k range
  int e, tn, slot = -1, cut = 0;
  int64_t m0, m_end, kbeg = 0, kend;
  if constexpr (OP == 2) {
    WeightTile t;
    if (!weight_tile(p, tiles_m, tiles_n, &t)) return;
    e = t.e;
    tn = t.tn;
    slot = t.slot;
    kbeg = t.lo;
    kend = t.hi;
    m0 = (int64_t)t.tm * BM;
    m_end = p.N;
  } else {
    RowTile t;
    if (!row_tile(p, BM, tiles_n, &t, &tn, &cut)) return;
    e = t.e;
    m0 = t.m0;
    m_end = t.m1;
    kend = e == p.E ? 0 : OP == 0 ? p.K : p.N;
    cut_range(p, cut, &kbeg, &kend);
  }
  const int64_t n_end = OP == 0 ? p.N : p.K, n0 = (int64_t)tn * BN;
  const int64_t weight = (int64_t)e * p.N * (OP == 2 ? p.K : p.ldb);

  Operand<T, BM, KA, MA, G::NT> a;
  Operand<T, BN, KB, MB, G::NT> b;
  a.init(p.A, p.lda, m0, m_end - m0);
  b.init(OP == 2 ? p.B : static_cast<const T*>(p.B) + weight, p.ldb, n0, n_end - n0);
  if constexpr (MB >= kInt8)
    b.init_scale(p.b_scale, (p.K + p.group - 1) / p.group, p.group, n0);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / G::WN, wn = wave % G::WN, lane = threadIdx.x & 63;
  f32x16 acc[FM][FN];
  tile_loop<T, G, KA, KB>(a, b, kbeg, kend, lds, acc);

  if (OP == 2 ? slot >= 0 : p.part != nullptr) {  // an item of several, a cut's part
    float* part =
        p.part + (OP == 2 ? (int64_t)slot * p.N * p.K : (int64_t)cut * p.T * n_end);
    // (4 columns of a row lie side by side in a lane; value by value the stores of a
    // whole tile took 100 us and more)
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int64_t row = m0 + (wm * FM + i) * 32 + (lane & 31);
          const int64_t col = n0 + (wn * FN + j) * 32 + 8 * q + 4 * (lane >> 5);
          if (row >= m_end || col >= n_end) continue;
          float* at = part + row * n_end + col;
          if (col + 4 <= n_end) {
            reinterpret_cast<LooseVec<float, 4>*>(at)->v = {
                acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
          } else {
#pragma unroll
            for (int s = 0; s < 4; ++s)
              if (col + s < n_end) at[s] = acc[i][j][4 * q + s];
          }
        }
    return;
  }
  // The wave's outputs go through LDS to become whole 16-byte pieces of rows.
  const float factor = p.scale == nullptr ? 1.0f : *p.scale;
  __syncthreads();
  T* out = static_cast<T*>(p.C) + (OP == 2 ? weight : 0);
  constexpr int kWaveRows = FM * 32, kRowBytes = FN * 64, kChunks = kRowBytes / 16;
  char* stage = lds + wave * kWaveRows * kRowBytes;
  typedef T t4 __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int r = i * 32 + (lane & 31);
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        t4 v;
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = (T)(acc[i][j][4 * q + u] * factor);
        const int c = (4 * j + q) ^ (r & (kChunks - 1));
        *reinterpret_cast<t4*>(stage + r * kRowBytes + c * 16 + (lane >> 5) * 8) = v;
      }
  }
  const int64_t row0 = m0 + wm * kWaveRows, col0 = n0 + wn * FN * 32;
  constexpr int kStep = 64 / kChunks;  // rows a wave stores at once
#pragma unroll 4
  for (int it = 0; it < kWaveRows / kStep; ++it) {
    const int r = it * kStep + lane / kChunks, c = lane % kChunks;
    const u32x4 v =
        *reinterpret_cast<const u32x4*>(stage + r * kRowBytes + ((c ^ (r & (kChunks - 1))) * 16));
    const int64_t row = row0 + r, col = col0 + 8 * c;
    if (row >= m_end || col >= n_end) continue;
    T* dst = out + row * n_end + col;
    if (store_vec) {
      *reinterpret_cast<u32x4*>(dst) = v;
    } else if (col + 8 <= n_end) {
      reinterpret_cast<Loose16*>(dst)->v = v;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (col + j < n_end)
          reinterpret_cast<uint16_t*>(dst)[j] = (uint16_t)(v[j >> 1] >> (16 * (j & 1)));
    }
  }
}

template <typename T, class G, int OP, int MA, int MB>
int launch_tile(const GroupedParams& p, hipStream_t st) {
  const int64_t cols = OP == 0 ? p.N : p.K;
  const int64_t tiles_n = ceil_div(cols, G::BN), tiles_m = ceil_div(p.N, G::BM);
  const int64_t blocks = OP == 2 ? weight_grid(p, tiles_m * tiles_n) : row_grid(p, G::BM, tiles_n);
  if (!grid_fits(blocks, G::NT)) return set_error(KAN_ERR_LIMIT, "grouped_matmul: too many tiles");
  grouped_tile_kernel<T, G, OP, MA, MB><<<dim3((unsigned)blocks, OP == 2 ? 1 : p.cuts), G::NT, 0,
                                         st>>>(
      p, (int)tiles_m, (int)tiles_n, cols % 8 == 0 && aligned16(p.C) ? 1 : 0);
  const int rc = check_launch("grouped_matmul");
  if (rc != KAN_OK) return rc;
  return OP == 2 ? launch_grouped_sum<T>(p, st) : launch_grouped_cuts<T>(p, cols, st);
}

// ---- few rows ---------------------------------------------------------------
// The forward of groups of a few rows (single tokens): bound by the weights'
// bytes, which a 128-row tile would hold up behind MFMAs on rows that do not
// exist.  A block has 16 rows and 16 columns; its four waves take the k in
// turns, each lane 64 consecutive bytes of one weight row (and of one x row),
// straight from memory into v_mfma_f32_16x16 operands: which k a lane's values
// are does not matter as long as both operands agree.  The waves' sums are added
// through LDS in order.
// (8 rows at 16 experts of 1024 -> 4096: fp32 66 us on tiles, bf16 rows of 1023
// 33 us.)
template <typename T, int NC, bool WHOLE>
__global__ __launch_bounds__(256) void grouped_few_kernel(GroupedParams p, int tiles_n) {
  typedef RowsMma<T> M;
  constexpr int kCols = 16 * NC;
  __shared__ float red[4][kFewRows][kCols + 1];
  RowTile t;
  int tn;
  if (!row_tile(p, kFewRows, tiles_n, &t, &tn)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n0 = tn * kCols;
  typename M::acc_t acc[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) acc[c] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (t.e < p.E) {
    const int m = min(t.m0 + (lane & 15), t.m1 - 1);
    const T* x = static_cast<const T*>(p.A) + (int64_t)m * p.K;
    const T* w[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c)
      w[c] = static_cast<const T*>(p.B) +
             ((int64_t)t.e * p.N + min((int64_t)(n0 + 16 * c + (lane & 15)), p.N - 1)) * p.K;
    few_rows<T, NC, WHOLE>(x, w, p.K, acc);
  }
  // lane l has row l & 15 and columns 4 (l >> 4) .. + 3 of each 16
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int v = 0; v < 4; ++v) red[wave][lane & 15][16 * c + 4 * (lane >> 4) + v] = acc[c][v];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int at = i * 256 + threadIdx.x, m = at / kCols, n = at % kCols;
    const float s = red[0][m][n] + red[1][m][n] + red[2][m][n] + red[3][m][n];
    if (t.m0 + m < t.m1 && n0 + n < p.N)
      static_cast<T*>(p.C)[(int64_t)(t.m0 + m) * p.N + n0 + n] = (T)s;
  }
}

template <typename T, int NC, bool WHOLE>
int launch_few_cols(const GroupedParams& p, hipStream_t st) {
  const int64_t tiles_n = ceil_div(p.N, 16 * NC), blocks = row_grid(p, kFewRows, tiles_n);
  if (!grid_fits(blocks, 256)) return set_error(KAN_ERR_LIMIT, "grouped_matmul: too many tiles");
  grouped_few_kernel<T, NC, WHOLE><<<dim3((unsigned)blocks), 256, 0, st>>>(p, (int)tiles_n);
  return check_launch("grouped_matmul");
}

}  // namespace

// Groups of up to 8 rows on average in 16 bits, 32 in fp32 (whose tiles multiply
// six times): 128 rows, 16 experts of 1024 x 1024, 8.4 us against 11.9 on tiles
// in bf16, 14.8 against 32 in fp32; at 16 rows a group (64 rows, 4 experts of
// 4096 x 4096, bf16) 42 against 33, at 32 in fp32 (512 rows, 16 experts of 1024 x
// 1024) 30.6 against 35.5.  The mean decides, so one expert may get all rows and its
// weights are read once for every 16 of them, from the caches: never slower than
// equal groups of the same rows, up to twice the tiles' time for that expert alone
// (512 rows, 64 experts of 1024 x 1024, bf16: equal 25.0 us, all at one 15.5, tiles
// 12.5; 2048 rows, 64 experts, fp32: 102, 96 and 50).
bool takes_few(int dtype, int op, int64_t T, int64_t E) {
  return op == KAN_GROUPED_FORWARD && T <= (dtype == KAN_DTYPE_F32 ? 32 : 8) * E;
}
namespace {

// 32 columns a block (the x rows are read once for both halves) where such
// blocks number two a CU: 16 experts of 1024 x 1024 and 128 rows 9.9 -> 8.4 us;
// one expert of 4096 x 4096 and one row 7.9 us on 16 columns, 11.3 on 32.
template <typename T>
int launch_few(const GroupedParams& p, hipStream_t st) {
  const bool wide = std::min<int64_t>(p.E, p.T) * ceil_div(p.N, 32) >= 2 * device_cu_count();
  if (sizeof(T) == 2 && !(aligned16(p.A) && aligned16(p.B) && p.K % 8 == 0))
    return wide ? launch_few_cols<T, 2, false>(p, st) : launch_few_cols<T, 1, false>(p, st);
  return wide ? launch_few_cols<T, 2, true>(p, st) : launch_few_cols<T, 1, true>(p, st);
}

template <typename T, class G, int OP>
int launch_half_op(const GroupedParams& p, hipStream_t st) {
  const bool a16 = whole_rows(p.A, p.lda), b16 = whole_rows(p.B, p.ldb);
  if constexpr (OP == 2) {
    if (p.format == KAN_ACT8_INT8)
      return a16 ? launch_tile<T, G, 2, kDirect, kInt8>(p, st)
                 : launch_tile<T, G, 2, kGuarded, kInt8>(p, st);
    if (p.format == KAN_ACT8_E4M3)
      return a16 ? launch_tile<T, G, 2, kDirect, kE4m3>(p, st)
                 : launch_tile<T, G, 2, kGuarded, kE4m3>(p, st);
  }
  return a16 && b16 ? launch_tile<T, G, OP, kDirect, kDirect>(p, st)
                    : launch_tile<T, G, OP, kGuarded, kGuarded>(p, st);
}

}  // namespace

// What a product in 16 bits runs on.  Time of a round of each tile, 16384 rows
// over 8 equal groups, 4096 x 4096 in bf16: 111 us on 256 x 256, 88 on 192 x
// 256, 73 on two 128 x 128 a CU.  (32768 rows over 16 groups, 4096 -> 1024: 314
// us on 256 rows, 285 on 192; 16384 over 8, 4096 -> 4096: 510 and 528.)
HalfPlan half_plan(int op, int64_t T, int64_t E, int64_t N, int64_t K) {
  const int cus = device_cu_count();
  HalfPlan pl{kSmall, 1, kNoRuns};
  if (op == 2) {
    const int64_t big = ceil_div(N, 256) * ceil_div(K, 256);
    // (64 rows of the large tile take 1.0 us, of the small one 0.65)
    if (big * E >= cus) {
      pl.cfg = kBig;
      pl.run = weight_run(T, E, N, K, big, {cus, 0.016, 5.0});
    } else {
      pl.run = weight_run(T, E, N, K, ceil_div(N, 128) * ceil_div(K, 128), {2 * cus, 0.010, 4.0});
    }
    return pl;
  }
  const int64_t cols = op == 0 ? N : K, depth = op == 0 ? K : N;
  const double wide = (double)ceil_div(cols, 256);
  const double small = row_tiles(T, E, 128) * (double)ceil_div(cols, 128);
  const double t[3] = {1.0 * rounds(row_tiles(T, E, 256) * wide, cus),
                       0.8 * rounds(row_tiles(T, E, 192) * wide, cus),
                       0.65 * rounds(small, 2.0 * cus)};
  for (int c = 0; c < 2; ++c)
    if (t[c] < t[pl.cfg]) pl.cfg = (HalfCfg)c;
  if (pl.cfg == kSmall) pl.cuts = sum_cuts(small, 2 * cus, ceil_div(depth, kDepth), 0.7);
  return pl;
}

// The same of one group's long sums over few outputs (dx of a piece of a vocabulary),
// where cuts pay on every tile: 4096 x 1024 outputs of 65536 terms in bf16 took 738
// us on 128 x 128 in 2 cuts, 560 on 256 x 256 in 4.  A slab takes 1.7 us on the
// largest tile; a cut's results are written and read again at 4 TB/s.
HalfPlan long_plan(int64_t T, int64_t N, int64_t K) {
  const int cus = device_cu_count();
  const double slab_us[3] = {1.73, 1.4, 2.0};
  const int64_t rows[3] = {256, 192, 128}, columns[3] = {256, 256, 128}, slabs = ceil_div(N, kDepth);
  HalfPlan best{kSmall, 1, kNoRuns};
  double least = 1e30;
  for (int c = 0; c < 3; ++c) {
    const double tiles = (double)ceil_div(T, rows[c]) * (double)ceil_div(K, columns[c]);
    for (int cuts = 1; cuts <= 32 && (cuts == 1 || slabs / cuts >= 8); ++cuts) {
      double t = slab_us[c] * rounds(tiles * cuts, c == 2 ? 2.0 * cus : cus) *
                 (double)ceil_div(slabs, cuts);
      if (cuts > 1) t += 5.0 + (double)cuts * (double)(T * K) * 8.0 / 4.0e6;
      if (t < least) {
        least = t;
        best = {(HalfCfg)c, cuts, kNoRuns};
      }
    }
  }
  return best;
}

namespace {

// Rows of [rows, C] at any address onto whole chunks of 8 values: out [rows, ld],
// ld a multiple of 8, the rest of a row zero.  (U: an integer of a value's size.)
template <typename U>
__global__ __launch_bounds__(256) void align_rows_kernel(const U* __restrict__ x, int64_t rows,
                                                         int64_t C, int64_t ld,
                                                         U* __restrict__ out) {
  typedef typename std::conditional<sizeof(U) == 2, Loose16, Loose8>::type Loose;
  typedef decltype(Loose::v) Chunk;
  const int64_t chunks = ld / 8, total = rows * chunks;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / chunks, c = 8 * (i - r * chunks);
    const U* src = x + r * C + c;
    U v[8] = {};
    if (c + 8 <= C) {
      *reinterpret_cast<Chunk*>(v) = reinterpret_cast<const Loose*>(src)->v;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < C) v[j] = src[j];
    }
    *reinterpret_cast<Chunk*>(out + i * 8) = *reinterpret_cast<const Chunk*>(v);
  }
}
template <typename U>
int launch_align(const void* x, int64_t rows, int64_t C, int64_t ld, void* out, hipStream_t st) {
  const int64_t blocks = std::min<int64_t>(ceil_div(rows * (ld / 8), 256), 1 << 16);
  align_rows_kernel<U><<<dim3((unsigned)blocks), 256, 0, st>>>(static_cast<const U*>(x), rows, C,
                                                               ld, static_cast<U*>(out));
  return check_launch("grouped_matmul rows");
}

}  // namespace

// Operands with rows off 16 bytes are brought onto them first where the
// products then save more than the copies take: at 32768 rows, 16 groups of
// 1023 -> 4095 the products took 636 (forward), 937 (input) and 1015 us
// (weight) on rows as they were, against 293, 323 and 262 on aligned ones; a
// copy moves its rows twice at about 4 TB/s, and takes 5 us at least.
AlignPlan align_operands(const void* A, int64_t a_rows, int64_t a_cols, const void* B,
                         int64_t b_rows, int64_t b_cols, int b_value, double saved_us) {
  AlignPlan pl{};
  pl.a_rows = a_rows;
  pl.a_cols = a_cols;
  pl.b_rows = b_rows;
  pl.b_cols = b_cols;
  pl.b_value = b_value;
  pl.a = !whole_rows(A, a_cols);
  pl.b = b_value == 2 ? !whole_rows(B, b_cols)
                      : b_cols % 8 != 0 || reinterpret_cast<uintptr_t>(B) % 8 != 0;
  double copies_us = 0.0;
  if (pl.a) copies_us += 5.0 + 4.0 * (double)(a_rows * a_cols) / 4.0e6;
  if (pl.b) copies_us += 5.0 + 2.0 * b_value * (double)(b_rows * b_cols) / 4.0e6;
  if (saved_us <= copies_us) pl.a = pl.b = false;
  if (pl.a) pl.a_bytes = (size_t)(2 * a_rows * round_up(a_cols, 8));
  if (pl.b) pl.b_bytes = (size_t)(b_value * b_rows * round_up(b_cols, 8));
  return pl;
}
double align_saves_us(int op, int64_t T, int64_t N, int64_t K) {
  const double extra[3] = {1.2, 1.9, 2.9};  // of the aligned product's time
  return extra[op] * 2.0 * (double)T * (double)N * (double)K / 1.0e9;
}
AlignPlan align_plan(int op, int format, const void* A, const void* B, int64_t T, int64_t E,
                     int64_t N, int64_t K) {
  return align_operands(A, T, op == 0 ? K : N, B, op == 2 ? T : E * N, K,
                        format == KAN_ACT8_NONE ? 2 : 1, align_saves_us(op, T, N, K));
}

int launch_aligned(const AlignPlan& al, GroupedParams* p, char* ws, hipStream_t st) {
  if (al.a) {
    const int64_t ld = round_up(al.a_cols, 8);
    const int rc = launch_align<uint16_t>(p->A, al.a_rows, al.a_cols, ld, ws, st);
    if (rc != KAN_OK) return rc;
    p->A = ws;
    p->lda = ld;
    ws += al.a_bytes;
  }
  if (al.b) {
    const int64_t ld = round_up(al.b_cols, 8);
    const int rc = al.b_value == 2
                       ? launch_align<uint16_t>(p->B, al.b_rows, al.b_cols, ld, ws, st)
                       : launch_align<uint8_t>(p->B, al.b_rows, al.b_cols, ld, ws, st);
    if (rc != KAN_OK) return rc;
    p->B = ws;
    p->ldb = ld;
  }
  return KAN_OK;
}

// The weight gradient of one group that has all rows, of fewer large tiles than CUs: runs
// of rows on either tile.  16384 rows, 8192 x 1024 in bf16: 272 us on 128 x 128, 237 on
// 256 x 256 in two runs; 65536 rows, 512 x 256: 55 us in the runs of groups, 48 in these.
// (64 rows of two small tiles a CU take 1.14 us.)
HalfPlan long_weight_plan(int64_t T, int64_t N, int64_t K) {
  const int cus = device_cu_count();
  const double slab_us[2] = {1.73, 1.14};
  const int64_t side[2] = {256, 128};
  HalfPlan best{kSmall, 1, kNoRuns};
  double least = 1e30;
  for (int c = 0; c < 2; ++c) {
    const double tiles = (double)ceil_div(N, side[c]) * (double)ceil_div(K, side[c]);
    for (int64_t runs = 1; runs <= 32 && (runs == 1 || T / runs >= 512); ++runs) {
      const int64_t run = round_up(ceil_div(T, runs), kDepth);
      double t = slab_us[c] * rounds(tiles * (double)ceil_div(T, run), (c + 1.0) * cus) *
                 (double)(run / kDepth);
      if (runs > 1) t += 5.0 + (double)runs * (double)(N * K) * 8.0 / 4.0e6;
      if (t < least) {
        least = t;
        best = {c == 0 ? kBig : kSmall, 1, runs == 1 ? kNoRuns : (int)run};
      }
    }
  }
  return best;
}

namespace {

template <typename T>
int launch_half(int op, const GroupedParams& p, const HalfPlan& plan, hipStream_t st) {
  if (op == 2)
    return plan.cfg == kBig ? launch_half_op<T, TileBig, 2>(p, st)
                            : launch_half_op<T, TileSmall, 2>(p, st);
  if (op == 0)
    return plan.cfg == kBig   ? launch_half_op<T, TileBig, 0>(p, st)
           : plan.cfg == kMid ? launch_half_op<T, TileMid, 0>(p, st)
                              : launch_half_op<T, TileSmall, 0>(p, st);
  return plan.cfg == kBig   ? launch_half_op<T, TileBig, 1>(p, st)
         : plan.cfg == kMid ? launch_half_op<T, TileMid, 1>(p, st)
                            : launch_half_op<T, TileSmall, 1>(p, st);
}

}  // namespace

HalfPlan product_plan(int dtype, int op, int64_t T, int64_t E, int64_t N, int64_t K, bool dense) {
  HalfPlan pl{kSmall, 1, kNoRuns};
  if (T == 0 || E == 0 || N == 0 || K == 0) return pl;  // (their product can pass 64 bits)
  if (takes_few(dtype, op, T, E)) {
    pl.cfg = kFew;
  } else if (dtype != KAN_DTYPE_F32) {
    pl = half_plan(op, T, E, N, K);
    if (dense && op == KAN_GROUPED_WEIGHT && pl.cfg == kSmall) pl = long_weight_plan(T, N, K);
  } else if (op == KAN_GROUPED_WEIGHT) {
    pl.run = grouped_f32_run(T, E, N, K);
  } else {
    pl.cuts = grouped_f32_cuts(op, T, E, N, K);
  }
  return pl;
}
size_t product_part_bytes(int op, const HalfPlan& pl, int64_t T, int64_t E, int64_t N, int64_t K) {
  if (op == KAN_GROUPED_WEIGHT) return 4 * (size_t)weight_part_elems(T, E, N, K, pl.run);
  return pl.cuts > 1 ? 4 * (size_t)pl.cuts * (size_t)(T * (op == KAN_GROUPED_FORWARD ? N : K)) : 0;
}
int launch_product(int dtype, int op, GroupedParams p, const HalfPlan& pl, hipStream_t st) {
  p.run = pl.run;
  p.cuts = pl.cuts;
  if (pl.cfg == kFew)
    return dtype == KAN_DTYPE_F32    ? launch_few<float>(p, st)
           : dtype == KAN_DTYPE_BF16 ? launch_few<bf16>(p, st)
                                     : launch_few<f16>(p, st);
  if (dtype == KAN_DTYPE_F32) return launch_grouped_f32(op, p, st);
  return dtype == KAN_DTYPE_BF16 ? launch_half<bf16>(op, p, pl, st)
                                 : launch_half<f16>(op, p, pl, st);
}

namespace {

int check_grouped(int dtype, int op, int64_t T, int64_t E, int64_t N, int64_t K) {
  if (!dtype_is_operator(dtype))
    return set_error(KAN_ERR_INVALID, "grouped_matmul: dtype must be FP32, BF16 or FP16 (code %d)",
                     dtype);
  if (op < KAN_GROUPED_FORWARD || op > KAN_GROUPED_WEIGHT)
    return set_error(KAN_ERR_INVALID, "grouped_matmul: unknown product %d", op);
  if (T < 0 || E < 0 || N < 0 || K < 0)
    return set_error(KAN_ERR_INVALID, "grouped_matmul: negative size");
  // (tile ends are held in 32 bits, as are the bytes from a tile's first row)
  if (T > 0x3fffffff || N > (1 << 22) || K > (1 << 22) || E > 65535)
    return set_error(KAN_ERR_LIMIT,
                     "grouped_matmul: at most 2^30 - 1 rows, 2^22 columns and 65535 experts");
  return KAN_OK;
}

// Whether a weight gradient in 16 bits restores its 8-bit rows once, in a pass of
// their own, rather than in every tile that reads them: the tiles then run as on
// 16-bit rows, about a fifth faster (16384 rows, 8 experts of 4096 x 4096: 605 us
// from int8, 501 from bf16 and 32 for the pass), which pays from some 1800
// outputs on.  The rows' 16-bit copy lives for the call only.
bool restores_first(int64_t T, int64_t N, int64_t K) {
  const double saved_us = 0.2 * 2.0 * (double)T * (double)N * (double)K / 1.05e9;
  return K % 8 == 0 && saved_us > 5.0 + 3.0 * (double)(T * K) / 4.5e6;
}

// A call's workspace: rows brought onto 16 bytes (16-bit types) or restored from
// 8 bits (always in fp32, whose engine takes floats), then the partial sums.
struct Workspace {
  HalfPlan plan;
  AlignPlan align;
  bool restore;
  size_t rows_bytes, part_bytes;  // (part from a multiple of 16 bytes on)
};
Workspace plan_call(int dtype, int op, int format, const void* A, const void* B, int64_t T,
                    int64_t E, int64_t N, int64_t K, bool dense = false) {
  Workspace w{};
  w.plan = product_plan(dtype, op, T, E, N, K, dense && E == 1 && format == KAN_ACT8_NONE);
  if (T == 0 || E == 0 || N == 0 || K == 0 || w.plan.cfg == kFew) return w;
  if (dtype == KAN_DTYPE_F32) {
    w.restore = format != KAN_ACT8_NONE;
    if (w.restore) w.rows_bytes = 4 * (size_t)(T * K);
  } else {
    w.restore = format != KAN_ACT8_NONE && restores_first(T, N, K);
    // (restored rows lie on 16 bytes; those of A come behind them)
    if (w.restore) w.rows_bytes = (size_t)round_up(2 * T * K, 16);
    w.align = align_plan(op, w.restore ? KAN_ACT8_NONE : format, A, w.restore ? nullptr : B, T, E, N,
                         K);
    w.rows_bytes += w.align.a_bytes + w.align.b_bytes;
  }
  w.rows_bytes = (size_t)round_up((int64_t)w.rows_bytes, 16);
  w.part_bytes = product_part_bytes(op, w.plan, T, E, N, K);
  return w;
}

}  // namespace
}  // namespace kan

using namespace kan;

extern "C" {

int kan_hip_grouped_matmul_workspace(int dtype, int op, const void* a, const void* b, int b_format,
                                     int64_t T, int64_t E, int64_t N, int64_t K, size_t* bytes) {
  if (bytes == nullptr)
    return set_error(KAN_ERR_INVALID, "grouped_matmul_workspace: bytes must not be NULL");
  const int rc = check_grouped(dtype, op, T, E, N, K);
  if (rc != KAN_OK) return rc;
  const Workspace w = plan_call(dtype, op, b_format, a, b, T, E, N, K);
  *bytes = w.rows_bytes + w.part_bytes;
  // (a call without offsets may be planned otherwise)
  const Workspace d = plan_call(dtype, op, b_format, a, b, T, E, N, K, true);
  *bytes = std::max(*bytes, d.rows_bytes + d.part_bytes);
  return KAN_OK;
}

static int report_plan(int dtype, int op, const void* a, const void* b, int b_format, int64_t T,
                       int64_t E, int64_t N, int64_t K, bool dense, int64_t* plan) {
  if (plan == nullptr)
    return set_error(KAN_ERR_INVALID, "grouped_matmul_plan: plan must not be NULL");
  const int rc = check_grouped(dtype, op, T, E, N, K);
  if (rc != KAN_OK) return rc;
  const Workspace w = plan_call(dtype, op, b_format, a, b, T, E, N, K, dense);
  const bool f32 = dtype == KAN_DTYPE_F32, few = w.plan.cfg == kFew;
  const int rows[] = {256, 192, 128, kFewRows};  // by HalfCfg
  plan[0] = f32 && !few ? grouped_f32_rows(op, T, E, N, K) : rows[w.plan.cfg];
  plan[1] = w.plan.cuts;
  plan[2] = w.plan.run == kNoRuns ? 0 : w.plan.run;
  plan[3] = w.restore;
  plan[4] = (w.align.a ? 1 : 0) + (w.align.b ? 2 : 0);
  plan[5] = 0;
  if (!f32 && !few) {
    const bool whole_a = w.align.a || whole_rows(a, op == KAN_GROUPED_FORWARD ? K : N);
    const bool bytes = b_format != KAN_ACT8_NONE && !w.restore;
    const bool whole_b = w.restore || w.align.b || whole_rows(b, K);
    plan[5] = bytes ? (whole_a ? 1 : 0) : whole_a && whole_b ? 3 : 0;
  }
  return KAN_OK;
}

int kan_hip_grouped_matmul_plan(int dtype, int op, const void* a, const void* b, int b_format,
                                int64_t T, int64_t E, int64_t N, int64_t K, int64_t* plan) {
  return report_plan(dtype, op, a, b, b_format, T, E, N, K, false, plan);
}

int kan_hip_grouped_matmul_dense_plan(int dtype, int op, const void* a, const void* b, int64_t T,
                                      int64_t N, int64_t K, int64_t* plan) {
  return report_plan(dtype, op, a, b, KAN_ACT8_NONE, T, 1, N, K, true, plan);
}

static int grouped_matmul(int dtype, int op, const void* a, const void* b, int b_format,
                          const float* b_scale, int64_t b_group, const void* offsets,
                          int offsets64, int64_t T, int64_t E, int64_t N, int64_t K,
                          const float* scale, void* out, void* workspace, size_t workspace_bytes,
                          void* stream) {
  const int rc = check_grouped(dtype, op, T, E, N, K);
  if (rc != KAN_OK) return rc;
  if (b_format != KAN_ACT8_NONE) {
    if (b_format != KAN_ACT8_INT8 && b_format != KAN_ACT8_E4M3)
      return set_error(KAN_ERR_INVALID, "grouped_matmul: unknown 8-bit format %d", b_format);
    if (op != KAN_GROUPED_WEIGHT)
      return set_error(KAN_ERR_INVALID, "grouped_matmul: 8-bit rows go into the weight product only");
    if (b_group != 32 && b_group != 64 && b_group != 128 && b_group != 256)
      return set_error(KAN_ERR_INVALID, "grouped_matmul: group must be 32, 64, 128 or 256");
    if (b_scale == nullptr && T > 0 && K > 0)
      return set_error(KAN_ERR_INVALID, "grouped_matmul: 8-bit rows need their scales");
  }
  const int64_t outputs = op == KAN_GROUPED_WEIGHT    ? E * N * K
                          : op == KAN_GROUPED_FORWARD ? T * N
                                                      : T * K;
  if (outputs == 0) return KAN_OK;
  const bool some = op == KAN_GROUPED_WEIGHT ? T > 0 : E * N * K > 0;  // any term to add up
  if (out == nullptr || (some && (a == nullptr || b == nullptr)) || (E > 1 && offsets == nullptr))
    return set_error(KAN_ERR_INVALID, "grouped_matmul: operands must not be NULL");
  const Workspace w = plan_call(dtype, op, b_format, a, b, T, E, N, K, offsets == nullptr);
  const size_t need = w.rows_bytes + w.part_bytes;
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return set_error(KAN_ERR_WORKSPACE, "grouped_matmul: needs %zu bytes of workspace, got %zu",
                     need, workspace == nullptr ? (size_t)0 : workspace_bytes);
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
    return set_error(KAN_ERR_INVALID, "grouped_matmul: the workspace lies on 16 bytes");
  char* ws = static_cast<char*>(workspace);
  GroupedParams p{};
  p.A = a;
  p.B = b;
  p.b_scale = b_scale;
  p.C = out;
  p.offsets = offsets;
  p.offsets64 = offsets64;
  p.E = (int)E;
  p.T = T;
  p.N = N;
  p.K = K;
  p.group = (int)b_group;
  p.format = b_format;
  p.scale = scale;
  hipStream_t st = static_cast<hipStream_t>(stream);
  TimedLaunch timed(kClassContraction, st, 2.0 * (double)T * N * K);
  p.lda = op == KAN_GROUPED_FORWARD ? K : N;
  p.ldb = K;
  if (w.part_bytes > 0) p.part = reinterpret_cast<float*>(ws + w.rows_bytes);
  if (w.restore) {
    const int e = kan_hip_act8_dequantize(dtype, b_format, b, b_scale, T, K, b_group, ws, stream);
    if (e != KAN_OK) return e;
    p.B = ws;
    p.format = KAN_ACT8_NONE;
    ws += round_up((int64_t)dtype_bytes(dtype) * T * K, 16);
  }
  const int e = launch_aligned(w.align, &p, ws, st);
  return e != KAN_OK ? e : launch_product(dtype, op, p, w.plan, st);
}

int kan_hip_grouped_matmul(int dtype, int op, const void* a, const void* b, int b_format,
                           const float* b_scale, int64_t b_group, const void* offsets,
                           int offsets64, int64_t T, int64_t E, int64_t N, int64_t K, void* out,
                           void* workspace, size_t workspace_bytes, void* stream) {
  return grouped_matmul(dtype, op, a, b, b_format, b_scale, b_group, offsets, offsets64, T, E, N, K,
                        nullptr, out, workspace, workspace_bytes, stream);
}

int kan_hip_grouped_matmul_scaled(int dtype, int op, const void* a, const void* b,
                                  const void* offsets, int offsets64, int64_t T, int64_t E,
                                  int64_t N, int64_t K, const float* scale, void* out,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  if (dtype == KAN_DTYPE_F32 || op == KAN_GROUPED_FORWARD || scale == nullptr)
    return set_error(KAN_ERR_INVALID,
                     "grouped_matmul_scaled: gradients' products in 16 bits and a factor");
  return grouped_matmul(dtype, op, a, b, KAN_ACT8_NONE, nullptr, 0, offsets, offsets64, T, E, N, K,
                        scale, out, workspace, workspace_bytes, stream);
}

}  // extern "C"
