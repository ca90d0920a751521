// Matrix products in 16 bits: an operand's way into LDS, fragments, and the loop
// over a tile's k, which the grouped products, the gated products and the losses
// over a vocabulary share.
#pragma once

#include <type_traits>

#include "kan_types.h"

namespace kan {

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

// PAIRS: the rows of two weights in turn, 32 of each (K-contiguous): rows 64 i ..
// 64 i + 31 of the tile are rows 32 i .. of the first, the 32 behind them the same
// rows of the second, `up` bytes further on.
template <typename T, int ROWS, bool KCONT, int MODE, int NT, bool PAIRS = false>
struct Operand {
  static constexpr int kPer = ROWS * (kDepth / 8) / NT;  // chunks of a thread
  static constexpr int kRowChunks = KCONT ? kDepth / 8 : ROWS / 8;
  static constexpr int kValue = MODE >= kInt8 ? 1 : 2;   // bytes of a value in memory
  static constexpr int kMode = MODE;
  static_assert(ROWS * (kDepth / 8) % NT == 0, "whole rounds of chunks");
  static_assert(MODE < kInt8 || !KCONT, "8-bit rows are the weight product's");
  static_assert(!PAIRS || (KCONT && MODE < kInt8), "pairs of K-contiguous rows");

  const char* base;  // of the tile's first row (KCONT) or column, at k = 0
  int64_t ld;        // bytes between rows
  int rows;          // valid rows (KCONT) or columns from the tile's first on (PAIRS: of each)
  int64_t up;        // PAIRS
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
      const int c = 8 * chunk_col(p);
      int r = chunk_row(p);
      if constexpr (PAIRS) r = (r >> 6) * 32 + (r & 31);
      off[p] = KCONT ? (uint32_t)(min(r, rows - 1) * ld) + (uint32_t)(c * kValue)
                     : (uint32_t)(r * ld) + (uint32_t)((c < rows ? c : 0) * kValue);
    }
  }
  // The slab that the wave's chunk p comes from (its 8 rows are of one weight).
  __device__ __forceinline__ const char* slab(int64_t k0, int p) const {
    const char* src = base + (KCONT ? k0 * kValue : k0 * ld);
    if constexpr (PAIRS) {
      const int row = p * (NT / 8) + (__builtin_amdgcn_readfirstlane(threadIdx.x) >> 6) * 8;
      src += (row & 32) != 0 ? up : 0;
    }
    return src;
  }

  // A whole slab straight into LDS.  (In assembly: the compiler would wait for
  // these loads before any transposing LDS read, taking it for a read of the
  // same bytes; slab_barrier waits for them.  They write no register.)
  __device__ __forceinline__ void issue_part(int64_t k0, char* lds, int p) const {
    const uint32_t to = __builtin_amdgcn_readfirstlane(
        (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds + (threadIdx.x >> 6) * 1024);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(
                     to + p * NT * 16),
                 "v"(off[p]), "s"(slab(k0, p))
                 : "m0");
  }
  __device__ __forceinline__ void issue(int64_t k0, char* lds) const {
#pragma unroll
    for (int p = 0; p < kPer; ++p) issue_part(k0, lds, p);
  }

  // A slab into registers.  GUARD: k from kend on is zero, and chunks that lie
  // partly outside the operand go value by value; otherwise every chunk of the
  // slab exists.
  template <bool GUARD>
  __device__ __forceinline__ void load(int64_t k0, int64_t kend) {
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
      const char* src = slab(k0, p);
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

struct Nothing {
  __device__ __forceinline__ void operator()() const {}
};
// acc = the tile's product over k in kbeg .. kend - 1 (KA, KB: K-contiguous
// operands).  lds: 2 G::kBuf bytes on 16; waves are done with their reads of it
// only after a barrier.  meanwhile(): what else a block has to look up, called
// while its first slab is on its way and before a barrier.
template <typename T, class G, bool KA, bool KB, class A, class B, class F = Nothing>
__device__ __forceinline__ void tile_loop(A& a, B& b, int64_t kbeg, int64_t kend, char* lds,
                                          f32x16 (&acc)[G::FM][G::FN], const F& meanwhile = F()) {
  constexpr int BM = G::BM, BN = G::BN, FM = G::FM, FN = G::FN;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / G::WN, wn = wave % G::WN;
  Fragments<T, BM, FM, KA> fa;
  Fragments<T, BN, FN, KB> fb;
  fa.init(wm * FM * 32);
  fb.init(wn * FN * 32);

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
    if constexpr (A::kMode != kDirect) a.store(buf);
    if constexpr (B::kMode != kDirect) b.store(buf + kB);
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
    constexpr bool kStraight = A::kMode == kDirect && B::kMode == kDirect;
    if constexpr (kStraight && !decltype(rest)::value) {
      // (a whole slab in the midst of others: its loads and reads one by one under the
      // step's MFMAs; the loads before them all, as the barrier leaves both of a
      // SIMD's waves, kept its matrix unit waiting)
      slab_barrier();
      const int64_t k0 = kbeg + (int64_t)(kt + 2) * kDepth;
      constexpr int kLoads = A::kPer + B::kPer, kSteps1 = (kSteps - 1) & 1;
#pragma unroll
      for (int q = 0; q < FM * FN || q < kLoads; ++q) {
        if (q < FM * FN) {
          const int i = q / FN, j = q % FN;
          acc[i][j] = Half<T>::mma(bv[kSteps1][j], av[kSteps1][i], acc[i][j]);
        }
        if (q < FN) bv[0][q] = fb.read(nxt + kB, q, 0);
        else if (q < FN + FM) av[0][q - FN] = fa.read(nxt, q - FN, 0);
        if (q < A::kPer) a.issue_part(k0, cur, q);
        else if (q < kLoads) b.issue_part(k0, cur + kB, q - A::kPer);
        __builtin_amdgcn_sched_barrier(0);
      }
      return;
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
    meanwhile();
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
}

// ---- products of a few rows ---------------------------------------------------
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

// acc[c] += the products of 16 rows (a lane's row at x) with 16 weight rows each
// (a lane's at w[c]) over the k of the block's wave: four waves take the k in
// turns, each lane 64 consecutive bytes of its rows, straight from memory into
// v_mfma_f32_16x16 operands: which k a lane's values are does not matter as long
// as both operands agree.  WHOLE: rows lie on 16 bytes.
template <typename T, int NC, bool WHOLE>
__device__ __forceinline__ void few_rows(const T* x, const T* (&w)[NC], int64_t K,
                                         typename RowsMma<T>::acc_t (&acc)[NC]) {
  typedef RowsMma<T> M;
  constexpr int V = 16 / sizeof(T), U = 4;  // values of a load, loads of a lane's turn
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  auto load = [](const T* q) __attribute__((always_inline)) {
    if constexpr (sizeof(T) == 2 && !WHOLE)
      return __builtin_bit_cast(typename M::vec, load16_even(q));
    else
      return reinterpret_cast<const LooseVec<T, V>*>(q)->v;
  };
  constexpr int kTurn = 4 * U * V;
  for (int64_t k0 = wave * kTurn; k0 < K; k0 += 4 * kTurn) {
    typename M::vec a[NC][U], b[U];
    const int64_t k = k0 + (lane >> 4) * V;
    if (k0 + kTurn <= K) {
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
          for (int c = 0; c < NC; ++c) a[c][u][j] = at < K ? w[c][at] : (T)0.0f;
          b[u][j] = at < K ? x[at] : (T)0.0f;
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int c = 0; c < NC; ++c) acc[c] = M::mma(a[c][u], b[u], acc[c]);
  }
}

// ---- host ---------------------------------------------------------------------
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// Operands are read straight into LDS where their rows are whole 16 bytes.
inline bool whole_rows(const void* p, int64_t ld) { return aligned16(p) && ld % 8 == 0; }

}  // namespace kan
