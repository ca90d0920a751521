// Products grouped by expert with ragged sizes: their parameters, and how a
// block finds the rows its tile has from offsets that lie on the device.
#pragma once

#include <cmath>

#include "kan_types.h"

namespace kan {

struct GroupedParams {
  const void *A, *B;      // op 0: x, w; 1: dy, w; 2: dy, x
  const float* b_scale;   // op 2 with 8-bit rows: [T, ceil(K / group)]
  void* C;
  const void* offsets;
  int offsets64;
  int E;
  int64_t T, N, K;
  int64_t lda, ldb;       // values between rows of A and B
  int group, format;      // of 8-bit rows (KAN_ACT8_NONE: B is in the products' type)
  int run;                // op 2: rows of an item of work; the sums of a group of
  float* part;            // several items go to part [T / run + E, N, K]
  int cuts;               // op 0, 1: the sums are cut into this many (grid y), whose
                          // results go to part [cuts, T, columns] if there are several
};

// ---- which rows a tile has --------------------------------------------------

template <int CTRL, int ROW_MASK = 0xf>
__device__ __forceinline__ int dpp_int(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROW_MASK, 0xf, false);
}
// inclusive scans over the wave, of values that are not negative
__device__ __forceinline__ int scan_add(int v) {
  v += dpp_int<0x111>(v);
  v += dpp_int<0x112>(v);
  v += dpp_int<0x114>(v);
  v += dpp_int<0x118>(v);
  v += dpp_int<0x142, 0xa>(v);
  v += dpp_int<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ int scan_max(int v) {
  v = max(v, dpp_int<0x111>(v));
  v = max(v, dpp_int<0x112>(v));
  v = max(v, dpp_int<0x114>(v));
  v = max(v, dpp_int<0x118>(v));
  v = max(v, dpp_int<0x142, 0xa>(v));
  v = max(v, dpp_int<0x143, 0xc>(v));
  return v;
}

// End of group e's rows as stored, within 0 .. T; the rows past the last
// group's are a group E of their own that ends at T.
__device__ __forceinline__ int group_end(const GroupedParams& p, int e) {
  if (e >= p.E) return (int)p.T;
  const int64_t v = p.offsets64 ? static_cast<const int64_t*>(p.offsets)[e + 1]
                                : (int64_t)static_cast<const int*>(p.offsets)[e + 1];
  return (int)max((int64_t)0, min(p.T, v));
}

// Offsets that do not ascend are taken as their running maximum, so that
// every row belongs to one group whatever the offsets hold.
struct GroupScan {
  int begin, end, tiles, last;  // of this lane's group; last: tiles up to and with it
  int carry_end = 0, carry_tiles = 0;
  __device__ __forceinline__ void step(const GroupedParams& p, int base, int bm) {
    const int lane = threadIdx.x & 63, e = base + lane;
    end = max(carry_end, scan_max(e <= p.E ? group_end(p, e) : 0));
    begin = __shfl_up(end, 1);
    if (lane == 0) begin = carry_end;
    tiles = (end - begin + bm - 1) / bm;
    last = carry_tiles + scan_add(tiles);
    carry_end = __builtin_amdgcn_readlane(end, 63);
    carry_tiles = __builtin_amdgcn_readlane(last, 63);
  }
};

// Group (E: none) and rows [m0, m1) of a row tile.
struct RowTile {
  int e, m0, m1;
};
// The tile from the scan of its 64 groups from `base` on (false: not one of them).
__device__ __forceinline__ bool take_tile(const GroupScan& s, int base, int tile, int bm,
                                          RowTile* r) {
  if (tile >= s.carry_tiles) return false;
  const int l = __builtin_ctzll(__ballot(tile < s.last));
  const int before = __builtin_amdgcn_readlane(s.last - s.tiles, l);
  r->e = base + l;
  r->m0 = __builtin_amdgcn_readlane(s.begin, l) + (tile - before) * bm;
  r->m1 = min(__builtin_amdgcn_readlane(s.end, l), r->m0 + bm);
  return true;
}

// ---- tiles of the weight gradient -------------------------------------------
// A group's rows are cut into items of `run` rows and a rest; every item has
// all tiles of [N, K].  Items cost what their rows are many: whole runs come
// first, then the rests (and groups without rows, which get zeros), the largest
// first (past 64 groups, one a lane, in the groups' order).  Each item's tiles
// are dealt to all XCDs, in stretches for their L2 (which XCD has the first
// turns with the item, as the last may be short).  At 16384 rows over 8
// experts of 4096 x 4096 in bf16, sizes 0.3 to 2.4 times the mean, this order
// took 0.51 ms, expert after expert 0.65.
struct WeightTile {
  int e, tm, tn;
  int lo, hi;   // rows
  int slot;     // of part, or -1: the group's only item
};
inline int64_t weight_items(const GroupedParams& p) { return p.T / p.run + p.E; }
inline int64_t weight_grid(const GroupedParams& p, int64_t tiles) {
  return ceil_div(tiles, kNumXcd) * kNumXcd * weight_items(p);
}
__device__ __forceinline__ bool weight_tile(const GroupedParams& p, int tiles_m, int tiles_n,
                                            WeightTile* t) {
  const int per = tiles_m * tiles_n, stretch = (per + kNumXcd - 1) / kNumXcd;
  const int xcd = blockIdx.x % kNumXcd, idx = blockIdx.x / kNumXcd;
  int item = __builtin_amdgcn_readfirstlane(idx / stretch);
  const int id = __builtin_amdgcn_readfirstlane(((xcd + item) % kNumXcd) * stretch + idx % stretch);
  if (id >= per) return false;
  t->tm = __builtin_amdgcn_readfirstlane(id / tiles_n);
  t->tn = id - t->tm * tiles_n;
  const int lane = threadIdx.x & 63;
  int found = -1, at = 0, slot = 0, begin = 0, end = 0;
  // lane l's group is the one asked for (l < 0: none of these 64)
  auto take = [&](const GroupScan& s, int base, int l, int row) __attribute__((always_inline)) {
    if (l < 0) return;
    found = base + l;
    begin = __builtin_amdgcn_readlane(s.begin, l);
    end = __builtin_amdgcn_readlane(s.end, l);
    at = row;
    slot = __builtin_amdgcn_readlane(s.last - s.tiles, l) + row / p.run;
    if (__builtin_amdgcn_readlane(s.tiles, l) <= 1) slot = -1;
  };
  auto lane_of = [&](bool is) __attribute__((always_inline)) {
    const uint64_t m = __ballot(is);
    return m == 0 ? -1 : (int)__builtin_ctzll(m);
  };
  // whole runs
  GroupScan s;
  int before = 0;
  for (int base = 0; base < p.E && found < 0; base += 64) {
    s.step(p, base, p.run);
    const int full = base + lane < p.E ? (s.end - s.begin) / p.run : 0;
    const int last = before + scan_add(full);
    const int l = lane_of(item < last && full > 0 && item >= last - full);
    if (l >= 0) take(s, base, l, (item - __builtin_amdgcn_readlane(last - full, l)) * p.run);
    before = __builtin_amdgcn_readlane(last, 63);
  }
  if (found >= 0) {
    t->hi = begin + at + p.run;
  } else {
    // rests
    item -= before;
    GroupScan r;
    before = 0;
    for (int base = 0; base < p.E && found < 0; base += 64) {
      r.step(p, base, p.run);
      const int size = r.end - r.begin, rest = size % p.run;
      const bool is = base + lane < p.E && (rest > 0 || size == 0);
      int rank;
      if (p.E <= 64) {
        rank = 0;
        for (int j = 0; j < p.E; ++j) {
          const int other = __builtin_amdgcn_readlane(is ? rest : -1, j);
          rank += other > rest || (other == rest && j < lane);
        }
      } else {
        rank = before + scan_add(is ? 1 : 0) - 1;
        before = __builtin_amdgcn_readlane(rank, 63) + 1;
      }
      const int l = lane_of(is && rank == item);
      if (l >= 0) take(r, base, l, __builtin_amdgcn_readlane(size - rest, l));
    }
    if (found < 0) return false;
    t->hi = end;
  }
  t->e = found;
  t->lo = begin + at;
  t->slot = slot;
  return true;
}

// Rows of an item: the run whose estimated time is least, or no runs.  A tile
// takes fixed_us and row_us for each row; the longest group is taken for three
// times the mean; partial sums are written and read once at 3.5 TB/s, and their
// sum is one more launch.
constexpr int kNoRuns = 0x40000000;
struct WeightCost {
  int places;  // blocks that run at once
  double row_us, fixed_us;
};
inline int weight_run(int64_t T, int64_t E, int64_t N, int64_t K, int64_t tiles,
                      const WeightCost& c) {
  if (T <= 0 || E <= 0 || tiles <= 0) return kNoRuns;
  const double mean = (double)T / (double)E, work = (double)tiles * (double)T * c.row_us;
  auto est = [&](double items, double longest) {
    const double busy = (work + items * (double)tiles * c.fixed_us) / c.places;
    return std::max(busy, longest * c.row_us + c.fixed_us);
  };
  int best = kNoRuns;
  double least = est((double)E, std::min((double)T, 3.0 * mean));
  for (int64_t run = 256; run < T; run *= 2) {
    const double items = (double)(T / run + E);
    const double part_us = items * (double)(N * K) * 8.0 / 3.5e6;
    const double t = est(items, (double)run) + part_us + 5.0;
    if (t < least) {
      least = t;
      best = (int)run;
    }
  }
  return best;
}
// Elements of part: none where no group can have several items.
inline int64_t weight_part_elems(int64_t T, int64_t E, int64_t N, int64_t K, int64_t run) {
  return T > run ? (T / run + E) * N * K : 0;
}

// dw of the groups of several items: the sum of their slots, in order.
template <typename T>
__global__ __launch_bounds__(256) void grouped_sum_kernel(GroupedParams p) {
  const int e = blockIdx.y;
  GroupScan s;
  int slots = 0, first = 0;
  for (int base = 0; base <= e; base += 64) {
    s.step(p, base, p.run);
    if (e < base + 64) {
      slots = __builtin_amdgcn_readlane(s.tiles, e - base);
      first = __builtin_amdgcn_readlane(s.last - s.tiles, e - base);
    }
  }
  if (slots <= 1) return;
  const int64_t count = p.N * p.K;
  const float* part = p.part + first * count;
  T* out = static_cast<T*>(p.C) + e * count;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count;
       i += (int64_t)gridDim.x * 256) {
    float v = part[i];
#pragma unroll 8
    for (int q = 1; q < slots; ++q) v += part[q * count + i];
    out[i] = (T)v;
  }
}
template <typename T>
int launch_grouped_sum(const GroupedParams& p, hipStream_t st) {
  if (p.part == nullptr) return KAN_OK;
  const int64_t blocks = std::min<int64_t>(ceil_div(p.N * p.K, 256), 4096);
  grouped_sum_kernel<T><<<dim3((unsigned)blocks, (unsigned)p.E), 256, 0, st>>>(p);
  return check_launch("grouped_matmul sum");
}

// ---- tiles of the other two products ------------------------------------------
// The row tiles of all groups in a row, kGroupedM of them at a time over all
// columns; false past the last.
constexpr int kGroupedM = 8;
__device__ __forceinline__ bool row_tile(const GroupedParams& p, int bm, int tiles_n, RowTile* t,
                                         int* tn) {
  GroupScan s;  // the number of row tiles first
  for (int base = 0; base <= p.E; base += 64) s.step(p, base, bm);
  const int tiles_m = s.carry_tiles, total = tiles_m * tiles_n;
  if ((int)blockIdx.x >= total) return false;
  const int id = xcd_remap(blockIdx.x, total), group = kGroupedM * tiles_n;
  const int first = id / group * kGroupedM, in = id % group;
  const int gm = min(tiles_m - first, kGroupedM);
  *tn = __builtin_amdgcn_readfirstlane(in / gm);
  const int tile = __builtin_amdgcn_readfirstlane(first + in % gm);
  if (p.E < 64) return take_tile(s, 0, tile, bm, t);  // (one scan has them all)
  GroupScan again;
  for (int base = 0; base <= p.E; base += 64) {
    again.step(p, base, bm);
    if (take_tile(again, base, tile, bm, t)) break;
  }
  return true;
}
inline int64_t row_grid(const GroupedParams& p, int64_t bm, int64_t tiles_n) {
  return (p.T / bm + p.E + 1) * tiles_n;
}
// About how many row tiles T rows of E groups make: half of a group's last one
// is empty, and no more groups have rows than there are rows.
inline double row_tiles(int64_t T, int64_t E, int64_t bm) {
  return (double)(T / bm) + std::max(0.5, 0.5 * (double)std::min(E, T));
}
// Rounds of `places` blocks at once that `blocks` equal ones take.  (The last
// round, where it is not full, runs at a higher clock: half way to whole rounds.)
inline double rounds(double blocks, double places) {
  const double x = blocks / places;
  return 0.5 * (x + std::max(1.0, std::ceil(x)));
}
// Cuts of the sums (`slabs` of them) of `tiles` tiles that would leave places
// idle: to fill them once, a cut of 4 slabs at least.  The cuts' results are
// written, read and added by one more launch of about 5 us, so they have to save
// more than that: slab_us is the time of a slab.
inline int sum_cuts(double tiles, int places, int64_t slabs, double slab_us) {
  const int64_t cuts = std::min<int64_t>((int64_t)(places / std::max(tiles, 1.0)), slabs / 4);
  if (cuts < 2 || (double)(slabs - slabs / cuts) * slab_us < 10.0) return 1;
  return (int)std::min<int64_t>(cuts, 32);
}
// The k range of this block's cut, whole slabs of 64.
__device__ __forceinline__ void cut_range(const GroupedParams& p, int64_t* kbeg, int64_t* kend) {
  if (p.cuts <= 1) return;
  const int k = (int)*kend, each = ((k + p.cuts - 1) / p.cuts + 63) / 64 * 64;
  // (uniform values: the division runs in vector registers)
  *kbeg = __builtin_amdgcn_readfirstlane(min(k, (int)blockIdx.y * each));
  *kend = __builtin_amdgcn_readfirstlane(min(k, (int)*kbeg + each));
}

// out = the sum of `cuts` slices of `count` values, in order.
template <typename T>
__global__ __launch_bounds__(256) void grouped_cuts_kernel(const float* __restrict__ part, int cuts,
                                                           int64_t count, T* __restrict__ out) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count;
       i += (int64_t)gridDim.x * 256) {
    float v = part[i];
#pragma unroll 8
    for (int q = 1; q < cuts; ++q) v += part[q * count + i];
    out[i] = (T)v;
  }
}
template <typename T>
int launch_grouped_cuts(const GroupedParams& p, int64_t cols, hipStream_t st) {
  if (p.cuts <= 1) return KAN_OK;
  const int64_t count = p.T * cols;
  grouped_cuts_kernel<T><<<dim3((unsigned)std::min<int64_t>(ceil_div(count, 256), 8192)), 256, 0,
                           st>>>(p.part, p.cuts, count, static_cast<T*>(p.C));
  return check_launch("grouped_matmul sum");
}

// fp32 products on the split contraction engine's tiles (kan_gemm.hip); the rows
// of a tile and of an item and the cuts of a sum there.
int grouped_f32_rows(int op, int64_t T, int64_t E, int64_t N, int64_t K);
int grouped_f32_run(int64_t T, int64_t E, int64_t N, int64_t K);
int grouped_f32_cuts(int op, int64_t T, int64_t E, int64_t N, int64_t K);
int launch_grouped_f32(int op, const GroupedParams& p, hipStream_t st);

}  // namespace kan
