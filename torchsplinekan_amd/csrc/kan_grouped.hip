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
#include <type_traits>

#include "kan_grouped.h"

namespace kan {

namespace {

// ---- 16-bit products on MFMA ------------------------------------------------
// Block tiles of BM x BN outputs, 64 deep, WM x WN waves; v_mfma_f32_32x32x16
// on bf16 or f16 operands.
//
// An operand's slab lies in LDS in 16-byte chunks of 8 values, in the layout of
// its rows in memory: K-contiguous operands as [row][8 chunks of k], the others
// as [64 k][chunks of rows].  A thread's chunks are the same in every slab, so
// their offsets are set once and a slab costs one scalar addition.  Whole slabs
// go from memory to LDS without passing registers (a wave's 64 chunks of 16
// bytes lie in a row there, so the chunks are exchanged on the memory side:
// chunk c of row r at position c ^ (r / 2 % 8), of k row k at c ^ 4 (k % 4),
// which spreads 16 lanes' reads over all 64 banks).  K-contiguous fragments are
// one 16-byte read a lane, the others two 8-byte reads that transpose 4 x 16
// values across the lanes of a row.  Last slabs, rows off 16 bytes and 8-bit
// rows pass registers.
//
// What bounds it: MFMA at the power cap.  16384 rows over 8 equal groups of 4096 x
// 4096 in bf16: forward 1.23 PFLOP/s, input 1.25, weight gradient 1.16, where
// torch.mm reaches 1.28, 1.15 and 1.02 at 8192^3; the MFMA pipes are busy for 0.55
// of the cycles at 2.0 GHz, LDS for 0.2 of them, and neither bank conflicts (5.5e7
// to 1.1e6 cycles) nor the waves' priority changed its time.  Uneven groups (0.3 to
// 2.4 times the mean) lose the empty half of their last tiles and part of the last
// round: 1.06 PFLOP/s.  Two waves a SIMD, as 4 waves of 128 x 128 were 10 % slower.
//
// Rows and columns past a tile's last repeat an earlier one: their products
// are not stored.  k past the last is zero in both operands, as what lies there
// (another expert's rows) may be anything.
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <typename T>
struct Half;
template <>
struct Half<bf16> {
  typedef bf16 frag __attribute__((ext_vector_type(8)));
  __device__ static __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Half<f16> {
  typedef f16 frag __attribute__((ext_vector_type(8)));
  __device__ static __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};

constexpr int kDepth = 64;  // k of a slab

template <int BM_, int BN_, int WM_, int WN_>
struct TileCfg {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, NT = 64 * WM * WN;
  static constexpr int FM = BM / WM / 32, FN = BN / WN / 32;
  static constexpr int kBuf = (BM + BN) * kDepth * 2;  // bytes of one slab pair
};
using TileBig = TileCfg<256, 256, 2, 4>;
using TileMid = TileCfg<192, 256, 2, 4>;  // (rows of K-contiguous operands only)
using TileSmall = TileCfg<128, 128, 2, 2>;

// How an operand reaches LDS.
enum OperandMode { kDirect = 0, kGuarded = 1, kInt8 = 2, kE4m3 = 3 };

// Values of 16 bytes (of 2 where rows are not aligned): memcpy keeps the
// load's alignment honest.
struct __attribute__((packed, aligned(2))) Loose16 {
  u32x4 v;
};
struct __attribute__((packed, aligned(1))) Loose8 {
  uint2 v;
};

template <typename T, int ROWS, bool KCONT, int MODE, int NT>
struct Operand {
  static constexpr int kPer = ROWS * (kDepth / 8) / NT;  // chunks of a thread
  static constexpr int kRowChunks = KCONT ? kDepth / 8 : ROWS / 8;
  static constexpr int kValue = MODE >= kInt8 ? 1 : 2;   // bytes of a value in memory
  static constexpr int kMode = MODE;
  static_assert(ROWS * (kDepth / 8) % NT == 0, "whole rounds of chunks");
  static_assert(MODE < kInt8 || !KCONT, "8-bit rows are the weight product's");

  const char* base;  // of the tile's first row (KCONT) or column, at k = 0
  int64_t ld;        // bytes between rows
  int rows;          // valid rows (KCONT) or columns from the tile's first on
  uint32_t off[kPer];
  u32x4 reg[kPer];
  // 8-bit rows
  const float* scale;               // of row 0
  int64_t parts;                    // scales of a row
  uint32_t part[MODE >= kInt8 ? kPer : 1];  // the chunk's, from the slab's first row on
  float step[MODE >= kInt8 ? kPer : 1];

  __device__ __forceinline__ void init_scale(const float* src, int64_t parts_, int group,
                                             int64_t col0) {
    scale = src;
    parts = parts_;
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
      const int c = 8 * chunk_col(p);
      part[p] = (uint32_t)(chunk_row(p) * parts) + ((uint32_t)col0 + (c < rows ? c : 0)) / group;
    }
  }

  // Row of the thread's chunk p in the slab's layout, and the chunk of that
  // row which belongs at the thread's position.
  __device__ __forceinline__ static int chunk_row(int p) {
    return (p * NT + (int)threadIdx.x) / kRowChunks;
  }
  __device__ __forceinline__ static int chunk_col(int p) {
    const int r = chunk_row(p), pos = (p * NT + (int)threadIdx.x) % kRowChunks;
    return KCONT ? pos ^ ((r >> 1) & 7) : pos ^ ((r & 3) << 2);
  }

  __device__ __forceinline__ void init(const void* src, int64_t ld_values, int64_t first,
                                       int64_t valid) {
    ld = ld_values * kValue;
    rows = (int)min(valid, (int64_t)ROWS);
    base = static_cast<const char*>(src) + (KCONT ? first * ld : first * kValue);
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
      const int r = chunk_row(p), c = 8 * chunk_col(p);
      off[p] = KCONT ? (uint32_t)(min(r, rows - 1) * ld) + (uint32_t)(c * kValue)
                     : (uint32_t)(r * ld) + (uint32_t)((c < rows ? c : 0) * kValue);
    }
  }
  __device__ __forceinline__ const char* slab(int64_t k0) const {
    return base + (KCONT ? k0 * kValue : k0 * ld);
  }

  // A whole slab straight into LDS.  (In assembly: the compiler would wait for
  // these loads before any transposing LDS read, taking it for a read of the
  // same bytes; slab_barrier waits for them.  They write no register.)
  __device__ __forceinline__ void issue(int64_t k0, char* lds) const {
    const char* src = slab(k0);
    const uint32_t to = __builtin_amdgcn_readfirstlane(
        (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds + (threadIdx.x >> 6) * 1024);
#pragma unroll
    for (int p = 0; p < kPer; ++p)
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(
                       to + p * NT * 16),
                   "v"(off[p]), "s"(src)
                   : "m0");
  }

  // A slab into registers.  GUARD: k from kend on is zero, and chunks that lie
  // partly outside the operand go value by value; otherwise every chunk of the
  // slab exists.
  template <bool GUARD>
  __device__ __forceinline__ void load(int64_t k0, int64_t kend) {
    const char* src = slab(k0);
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
      int n = 8;  // how many of the chunk's values exist: k for KCONT, columns otherwise
      if constexpr (GUARD) {
        const int r = chunk_row(p), c = 8 * chunk_col(p);
        const int64_t left = KCONT ? kend - k0 - c : (int64_t)(rows - c);
        n = (!KCONT && k0 + r >= kend) || left <= 0 ? 0 : (int)min(left, (int64_t)8);
        // (aligned rows end with whole chunks: their own, or zeros up to ld)
        if (MODE == kDirect && n > 0) n = 8;
      }
      u32x4 v = {0, 0, 0, 0};
      if constexpr (MODE >= kInt8) {
        if (n == 8) {
          const uint2 u = reinterpret_cast<const Loose8*>(src + off[p])->v;
          v[0] = u.x;
          v[1] = u.y;
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (j < n) v[j >> 2] |= (uint32_t)(uint8_t)src[off[p] + j] << (8 * (j & 3));
        }
        step[p] = n > 0 ? (scale + k0 * parts)[part[p]] : 0.0f;
      } else if (n == 8) {
        if constexpr (MODE == kGuarded) v = reinterpret_cast<const Loose16*>(src + off[p])->v;
        else v = *reinterpret_cast<const u32x4*>(src + off[p]);
      } else if constexpr (MODE == kGuarded) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < n)
            v[j >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(src + off[p])[j]
                         << (16 * (j & 1));
      }
      reg[p] = v;
    }
  }
  // Whether a slab whose k all exist needs no guard: chunks past the last column
  // repeat the first, and rows of whole chunks have no part of one.
  __device__ __forceinline__ bool interior() const {
    return MODE == kDirect || KCONT || rows == ROWS || (MODE >= kInt8 && ld % 8 == 0);
  }

  __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
      u32x4 v = reg[p];
      if constexpr (MODE >= kInt8) v = restore(v, step[p]);
      *reinterpret_cast<u32x4*>(lds + (p * NT + threadIdx.x) * 16) = v;
    }
  }
  // 8 values q * scale rounded to T: MFMA takes 16-bit operands, and what the rounding
  // leaves out would be a product of its own, twice the time.  In bf16 a result is
  // off by 0.0023 normwise where its own rounding alone makes 0.0017 (1 to 256 rows
  // an expert alike), and the 8 bits themselves have cost 0.006 (int8) or 0.026 (e4m3).
  // (int8: no detour over q + 128, whose product with a scale above FLT_MAX / 128
  // is infinite.)
  __device__ __forceinline__ static u32x4 restore(u32x4 q, float s) {
    typename Half<T>::frag f;
    if constexpr (MODE == kInt8) {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = (T)((float)(int8_t)(q[j >> 2] >> (8 * (j & 3))) * s);
    } else {
      typedef float f32x2 __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[j], false);
        const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[j], true);
        f[4 * j] = (T)(lo[0] * s);
        f[4 * j + 1] = (T)(lo[1] * s);
        f[4 * j + 2] = (T)(hi[0] * s);
        f[4 * j + 3] = (T)(hi[1] * s);
      }
    }
    return __builtin_bit_cast(u32x4, f);
  }
};

// Fragments of 32 rows x 16 k of a slab in LDS (ROWS rows in all, the wave's
// FR x 32 from `first` on): lane l has row l & 31 and k 8 (l >> 5) .. + 7.
template <typename T, int ROWS, int FR, bool KCONT>
struct Fragments {
  typedef typename Half<T>::frag frag;
  uint32_t at[KCONT ? 4 : FR];  // by k step, or by group of 32 rows
  __device__ __forceinline__ void init(int first) {
    const int lane = threadIdx.x & 63;
    if constexpr (KCONT) {
      const int r = first + (lane & 31);
#pragma unroll
      for (int s = 0; s < 4; ++s)
        at[s] = (uint32_t)(r * 128 + (((2 * s + (lane >> 5)) ^ ((r >> 1) & 7)) << 4));
    } else {
      // 16 lanes read 4 k rows of 16 columns, 4 columns each, and lane l then
      // holds column l & 15 of the 4 k rows
      const int k = 8 * (lane >> 5) + ((lane & 15) >> 2);
#pragma unroll
      for (int i = 0; i < FR; ++i) {
        const int col = first + 32 * i + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
        at[i] = (uint32_t)(k * ROWS * 2 + (((col >> 3) ^ ((k & 3) << 2)) << 4) +
                           ((col >> 2) & 1) * 8);
      }
    }
  }
  __device__ __forceinline__ frag read(const char* lds, int i, int s) const {
    if constexpr (KCONT) {
      return *reinterpret_cast<const frag*>(lds + at[s] + i * 32 * 128);
    } else {
      typedef __attribute__((address_space(3))) s16x4* lds4;
      const char* p = lds + at[i] + 16 * s * ROWS * 2;
      struct {
        s16x4 lo, hi;
      } v;
      v.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p));
      v.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + 4 * ROWS * 2));
      return __builtin_bit_cast(frag, v);
    }
  }
};

// Every wave's slab loads and LDS accesses are done, then every wave goes on.
__device__ __forceinline__ void slab_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <typename T, class G, int OP, int MA, int MB>
__global__ __launch_bounds__(G::NT) void grouped_tile_kernel(GroupedParams p, int tiles_m,
                                                             int tiles_n, int store_vec) {
  constexpr bool KA = OP != 2, KB = OP == 0;
  constexpr int BM = G::BM, BN = G::BN, FM = G::FM, FN = G::FN;
  __shared__ __align__(16) char lds[2 * G::kBuf];

  // the tile: rows [m0, m_end) and columns [n0, n_end) of the output, k range
  int e, tn, slot = -1;
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
    if (!row_tile(p, BM, tiles_n, &t, &tn)) return;
    e = t.e;
    m0 = t.m0;
    m_end = t.m1;
    kend = e == p.E ? 0 : OP == 0 ? p.K : p.N;
    cut_range(p, &kbeg, &kend);
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
  Fragments<T, BM, FM, KA> fa;
  Fragments<T, BN, FN, KB> fb;
  fa.init(wm * FM * 32);
  fb.init(wn * FN * 32);

  f32x16 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.0f;

  constexpr int kB = BM * kDepth * 2;  // B's slab lies behind A's
  constexpr int kSteps = kDepth / 16;
  typename Half<T>::frag av[2][FM], bv[2][FN];  // by the parity of the k step
  auto read_step = [&](const char* buf, int st) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < FN; ++j) bv[st & 1][j] = fb.read(buf + kB, j, st);
#pragma unroll
    for (int i = 0; i < FM; ++i) av[st & 1][i] = fa.read(buf, i, st);
  };
  auto mma_step = [&](int st) __attribute__((always_inline)) {
    // (B first: a lane then holds 4 columns of one row of the output)
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
        acc[i][j] = Half<T>::mma(bv[st & 1][j], av[st & 1][i], acc[i][j]);
    // the step's reads one by one between its MFMAs (left alone they sink below
    // them; all of them first: 1 to 5 % slower)
#pragma unroll
    for (int q = 0; q < FM + FN; ++q) {
      __builtin_amdgcn_sched_group_barrier(0x100, KA && KB ? 1 : 2, 0);  // LDS reads
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                 // MFMA
    }
    __builtin_amdgcn_sched_group_barrier(0x008, FM * FN, 0);
    __builtin_amdgcn_sched_barrier(0);
  };

  const int slabs = (int)((kend - kbeg + kDepth - 1) / kDepth);
  // slabs whose chunks all exist
  const int whole = a.interior() && b.interior() ? (int)((kend - kbeg) / kDepth) : 0;
  // start: sends slab kt on its way into buf; one of the others (rest) of an
  // operand that goes straight to LDS is there when it returns.  finish: stores
  // what passes registers.
  auto start_one = [&](auto& x, int64_t k0, char* buf, auto rest) __attribute__((always_inline)) {
    typedef typename std::remove_reference<decltype(x)>::type X;
    constexpr bool kRest = decltype(rest)::value;
    if constexpr (X::kMode != kDirect) {
      x.template load<kRest>(k0, kend);
    } else if constexpr (!kRest) {
      x.issue(k0, buf);
    } else if (k0 + kDepth <= kend) {
      x.issue(k0, buf);
    } else {
      x.template load<true>(k0, kend);
      x.store(buf);
    }
  };
  auto start = [&](int kt, char* buf, auto rest) __attribute__((always_inline)) {
    const int64_t k0 = kbeg + (int64_t)kt * kDepth;
    start_one(a, k0, buf, rest);
    start_one(b, k0, buf + kB, rest);
  };
  auto finish = [&](char* buf) __attribute__((always_inline)) {
    if constexpr (MA != kDirect) a.store(buf);
    if constexpr (MB != kDirect) b.store(buf + kB);
  };
  // One slab.  The fragments of a k step are read under the step before it;
  // the last step's MFMAs cover the barrier that publishes the next slab, its
  // first reads, and the start of the slab after it, which takes the buffer
  // that every wave has just read for the last time.
  auto slab = [&](int kt, bool next, bool third, auto rest) __attribute__((always_inline)) {
    char* cur = lds + (kt & 1) * G::kBuf;
    char* nxt = lds + ((kt + 1) & 1) * G::kBuf;
#pragma unroll
    for (int st = 0; st + 1 < kSteps; ++st) {
      read_step(cur, st + 1);
      mma_step(st);
    }
    if (next) {
      finish(nxt);
      slab_barrier();
      if (third) start(kt + 2, cur, rest);
      read_step(nxt, 0);
    }
    mma_step(kSteps - 1);
  };
  if (slabs > 0) {
    constexpr std::true_type rest{};
    constexpr std::false_type full{};
    if (whole > 0) start(0, lds, full);
    else start(0, lds, rest);
    finish(lds);
    slab_barrier();
    if (whole > 1) start(1, lds + G::kBuf, full);
    else if (slabs > 1) start(1, lds + G::kBuf, rest);
    read_step(lds, 0);
    int kt = 0;
#pragma unroll 1
    for (; kt + 2 < whole; ++kt) slab(kt, true, true, full);
#pragma unroll 1
    for (; kt < slabs; ++kt) slab(kt, kt + 1 < slabs, kt + 2 < slabs, rest);
  }

  if (OP == 2 ? slot >= 0 : p.cuts > 1) {  // an item of several, a cut of several
    float* part =
        p.part + (OP == 2 ? (int64_t)slot * p.N * p.K : (int64_t)blockIdx.y * p.T * n_end);
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int64_t row = m0 + (wm * FM + i) * 32 + (lane & 31);
          const int64_t col = n0 + (wn * FN + j) * 32 + 8 * (v >> 2) + 4 * (lane >> 5) + (v & 3);
          if (row < m_end && col < n_end) part[row * n_end + col] = acc[i][j][v];
        }
    return;
  }
  // The wave's outputs go through LDS to become whole 16-byte pieces of rows.
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
        for (int u = 0; u < 4; ++u) v[u] = (T)acc[i][j][4 * q + u];
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

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T, class G, int OP, int MA, int MB>
int launch_tile(const GroupedParams& p, hipStream_t st) {
  const int64_t cols = OP == 0 ? p.N : p.K;
  const int64_t tiles_n = ceil_div(cols, G::BN), tiles_m = ceil_div(p.N, G::BM);
  const int64_t blocks = OP == 2 ? weight_grid(p, tiles_m * tiles_n) : row_grid(p, G::BM, tiles_n);
  if (blocks > 0x7fffffff) return set_error(KAN_ERR_LIMIT, "grouped_matmul: too many tiles");
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
template <typename T>
struct RowsMma;
template <>
struct RowsMma<float> {
  typedef float vec __attribute__((ext_vector_type(4)));
  typedef float acc_t __attribute__((ext_vector_type(4)));
  __device__ static __forceinline__ acc_t mma(vec a, vec b, acc_t c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
};
template <>
struct RowsMma<bf16> {
  typedef bf16 vec __attribute__((ext_vector_type(8)));
  typedef float acc_t __attribute__((ext_vector_type(4)));
  __device__ static __forceinline__ acc_t mma(vec a, vec b, acc_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct RowsMma<f16> {
  typedef f16 vec __attribute__((ext_vector_type(8)));
  typedef float acc_t __attribute__((ext_vector_type(4)));
  __device__ static __forceinline__ acc_t mma(vec a, vec b, acc_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

constexpr int kFewRows = 16;
template <typename T, int NC, bool WHOLE>
__global__ __launch_bounds__(256) void grouped_few_kernel(GroupedParams p, int tiles_n) {
  typedef RowsMma<T> M;
  constexpr int V = 16 / sizeof(T), U = 4;  // values of a load, loads of a lane's turn
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
    auto load = [](const T* q) __attribute__((always_inline)) {
      if constexpr (sizeof(T) == 2 && !WHOLE)
        return __builtin_bit_cast(typename M::vec, load16_even(q));
      else
        return reinterpret_cast<const LooseVec<T, V>*>(q)->v;
    };
    constexpr int kTurn = 4 * U * V;
    for (int64_t k0 = wave * kTurn; k0 < p.K; k0 += 4 * kTurn) {
      typename M::vec a[NC][U], b[U];
      const int64_t k = k0 + (lane >> 4) * V;
      if (k0 + kTurn <= p.K) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
          for (int c = 0; c < NC; ++c)
            a[c][u] = load(w[c] + k + u * 4 * V);
          b[u] = load(x + k + u * 4 * V);
        }
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const int64_t at = k + u * 4 * V + j;
#pragma unroll
            for (int c = 0; c < NC; ++c) a[c][u][j] = at < p.K ? w[c][at] : (T)0.0f;
            b[u][j] = at < p.K ? x[at] : (T)0.0f;
          }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int c = 0; c < NC; ++c) acc[c] = M::mma(a[c][u], b[u], acc[c]);
    }
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
  if (blocks > 0x7fffffff) return set_error(KAN_ERR_LIMIT, "grouped_matmul: too many tiles");
  grouped_few_kernel<T, NC, WHOLE><<<dim3((unsigned)blocks), 256, 0, st>>>(p, (int)tiles_n);
  return check_launch("grouped_matmul");
}

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

// Operands are read straight into LDS where their rows are whole 16 bytes.
bool whole_rows(const void* p, int64_t ld) { return aligned16(p) && ld % 8 == 0; }

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

enum HalfCfg { kBig, kMid, kSmall, kFew };

// What a product in 16 bits runs on.  Time of a round of each tile, 16384 rows
// over 8 equal groups, 4096 x 4096 in bf16: 111 us on 256 x 256, 88 on 192 x
// 256, 73 on two 128 x 128 a CU.  (32768 rows over 16 groups, 4096 -> 1024: 314
// us on 256 rows, 285 on 192; 16384 over 8, 4096 -> 4096: 510 and 528.)
struct HalfPlan {
  HalfCfg cfg;
  int cuts, run;
};
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

// Operands with rows off 16 bytes are brought onto them first where the
// products then save more than the copies take: at 32768 rows, 16 groups of
// 1023 -> 4095 the products took 636 (forward), 937 (input) and 1015 us
// (weight) on rows as they were, against 293, 323 and 262 on aligned ones; a
// copy moves its rows twice at about 4 TB/s, and takes 5 us at least.
struct AlignPlan {
  bool a, b;
  int64_t a_rows, a_cols, b_rows, b_cols;
  size_t a_bytes, b_bytes;
};
AlignPlan align_plan(int op, int format, const void* A, const void* B, int64_t T, int64_t E,
                     int64_t N, int64_t K) {
  AlignPlan pl{};
  pl.a_rows = T;
  pl.a_cols = op == 0 ? K : N;
  pl.b_rows = op == 2 ? T : E * N;
  pl.b_cols = K;
  const int64_t b_value = format == KAN_ACT8_NONE ? 2 : 1;
  pl.a = !whole_rows(A, pl.a_cols);
  pl.b = format == KAN_ACT8_NONE ? !whole_rows(B, pl.b_cols)
                                 : pl.b_cols % 8 != 0 || reinterpret_cast<uintptr_t>(B) % 8 != 0;
  const double extra[3] = {1.2, 1.9, 2.9};  // of the aligned product's time
  const double saved_us = extra[op] * 2.0 * (double)T * (double)N * (double)K / 1.0e9;
  double copies_us = 0.0;
  if (pl.a) copies_us += 5.0 + 4.0 * (double)(pl.a_rows * pl.a_cols) / 4.0e6;
  if (pl.b) copies_us += 5.0 + 2.0 * b_value * (double)(pl.b_rows * pl.b_cols) / 4.0e6;
  if (saved_us <= copies_us) pl.a = pl.b = false;
  if (pl.a) pl.a_bytes = (size_t)(2 * pl.a_rows * round_up(pl.a_cols, 8));
  if (pl.b) pl.b_bytes = (size_t)(b_value * pl.b_rows * round_up(pl.b_cols, 8));
  return pl;
}

template <typename T>
int launch_half(int op, GroupedParams p, const HalfPlan& plan, const AlignPlan& al, char* ws,
                hipStream_t st) {
  if (al.a) {
    const int64_t ld = round_up(al.a_cols, 8);
    const int rc = launch_align<uint16_t>(p.A, al.a_rows, al.a_cols, ld, ws, st);
    if (rc != KAN_OK) return rc;
    p.A = ws;
    p.lda = ld;
    ws += al.a_bytes;
  }
  if (al.b) {
    const int64_t ld = round_up(al.b_cols, 8);
    const int rc = p.format == KAN_ACT8_NONE
                       ? launch_align<uint16_t>(p.B, al.b_rows, al.b_cols, ld, ws, st)
                       : launch_align<uint8_t>(p.B, al.b_rows, al.b_cols, ld, ws, st);
    if (rc != KAN_OK) return rc;
    p.B = ws;
    p.ldb = ld;
  }
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
                    int64_t E, int64_t N, int64_t K) {
  Workspace w{};
  w.plan = {kSmall, 1, kNoRuns};
  if (T == 0 || E == 0 || N == 0 || K == 0) return w;  // (their product can pass 64 bits)
  if (takes_few(dtype, op, T, E)) {
    w.plan.cfg = kFew;
    return w;
  }
  if (dtype == KAN_DTYPE_F32) {
    if (op == KAN_GROUPED_WEIGHT) w.plan.run = grouped_f32_run(T, E, N, K);
    else w.plan.cuts = grouped_f32_cuts(op, T, E, N, K);
    w.restore = format != KAN_ACT8_NONE;
    if (w.restore) w.rows_bytes = 4 * (size_t)(T * K);
  } else {
    w.plan = half_plan(op, T, E, N, K);
    w.restore = format != KAN_ACT8_NONE && restores_first(T, N, K);
    // (restored rows lie on 16 bytes; those of A come behind them)
    if (w.restore) w.rows_bytes = (size_t)round_up(2 * T * K, 16);
    w.align = align_plan(op, format, A, w.restore ? nullptr : B, T, E, N, K);
    w.rows_bytes += w.align.a_bytes + w.align.b_bytes;
  }
  w.rows_bytes = (size_t)round_up((int64_t)w.rows_bytes, 16);
  if (op == KAN_GROUPED_WEIGHT) w.part_bytes = 4 * (size_t)weight_part_elems(T, E, N, K, w.plan.run);
  else if (w.plan.cuts > 1)
    w.part_bytes = 4 * (size_t)w.plan.cuts * (size_t)(T * (op == KAN_GROUPED_FORWARD ? N : K));
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
  return KAN_OK;
}

int kan_hip_grouped_matmul_plan(int dtype, int op, const void* a, const void* b, int b_format,
                                int64_t T, int64_t E, int64_t N, int64_t K, int64_t* plan) {
  if (plan == nullptr)
    return set_error(KAN_ERR_INVALID, "grouped_matmul_plan: plan must not be NULL");
  const int rc = check_grouped(dtype, op, T, E, N, K);
  if (rc != KAN_OK) return rc;
  const Workspace w = plan_call(dtype, op, b_format, a, b, T, E, N, K);
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

int kan_hip_grouped_matmul(int dtype, int op, const void* a, const void* b, int b_format,
                           const float* b_scale, int64_t b_group, const void* offsets,
                           int offsets64, int64_t T, int64_t E, int64_t N, int64_t K, void* out,
                           void* workspace, size_t workspace_bytes, void* stream) {
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
  if (out == nullptr || (some && (a == nullptr || b == nullptr)) || (E > 0 && offsets == nullptr))
    return set_error(KAN_ERR_INVALID, "grouped_matmul: operands must not be NULL");
  const Workspace w = plan_call(dtype, op, b_format, a, b, T, E, N, K);
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
  hipStream_t st = static_cast<hipStream_t>(stream);
  TimedLaunch timed(kClassContraction, st, 2.0 * (double)T * N * K);
  p.lda = op == KAN_GROUPED_FORWARD ? K : N;
  p.ldb = K;
  p.run = w.plan.run;
  p.cuts = w.plan.cuts;
  if (w.part_bytes > 0) p.part = reinterpret_cast<float*>(ws + w.rows_bytes);
  if (w.plan.cfg == kFew)
    return dtype == KAN_DTYPE_F32    ? launch_few<float>(p, st)
           : dtype == KAN_DTYPE_BF16 ? launch_few<bf16>(p, st)
                                     : launch_few<f16>(p, st);
  if (w.restore) {
    const int e = kan_hip_act8_dequantize(dtype, b_format, b, b_scale, T, K, b_group, ws, stream);
    if (e != KAN_OK) return e;
    p.B = ws;
    p.format = KAN_ACT8_NONE;
    ws += round_up((int64_t)dtype_bytes(dtype) * T * K, 16);
  }
  if (dtype == KAN_DTYPE_F32) return launch_grouped_f32(op, p, st);
  return dtype == KAN_DTYPE_BF16 ? launch_half<bf16>(op, p, w.plan, w.align, ws, st)
                                 : launch_half<f16>(op, p, w.plan, w.align, ws, st);
}

}  // extern "C"
