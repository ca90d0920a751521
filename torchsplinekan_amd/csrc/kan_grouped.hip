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
// group from the offsets, and blocks past the last tile end at once.
#include "kan_types.h"

namespace kan {

namespace {

struct GroupedParams {
  const void *A, *B;      // op 0: x, w; 1: dy, w; 2: dy, x
  const float* b_scale;   // op 2 with 8-bit rows: [T, ceil(K / group)]
  void* C;
  const void* offsets;
  int offsets64;
  int E;
  int64_t T, N, K;
  int group, format;      // of 8-bit rows (KAN_ACT8_NONE: B is in the products' type)
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

// Number of row tiles of all groups.
__device__ __forceinline__ int count_tiles(const GroupedParams& p, int bm) {
  GroupScan s;
  for (int base = 0; base <= p.E; base += 64) s.step(p, base, bm);
  return s.carry_tiles;
}

// Group (E: none) and rows [m0, m1) of a row tile.
struct RowTile {
  int e, m0, m1;
};
__device__ __forceinline__ RowTile find_tile(const GroupedParams& p, int tile, int bm) {
  GroupScan s;
  RowTile r{p.E, 0, 0};
  for (int base = 0; base <= p.E; base += 64) {
    s.step(p, base, bm);
    if (tile >= s.carry_tiles) continue;
    const int l = __builtin_ctzll(__ballot(tile < s.last));
    r.e = base + l;
    const int before = __builtin_amdgcn_readlane(s.last - s.tiles, l);
    r.m0 = __builtin_amdgcn_readlane(s.begin, l) + (tile - before) * bm;
    r.m1 = min(__builtin_amdgcn_readlane(s.end, l), r.m0 + bm);
    break;
  }
  return r;
}

// Rows [begin, end) of group e.
__device__ __forceinline__ void group_rows(const GroupedParams& p, int e, int* begin, int* end) {
  GroupScan s;
  for (int base = 0; base <= e; base += 64) {
    s.step(p, base, 1);
    if (e < base + 64) {
      *begin = __builtin_amdgcn_readlane(s.begin, e - base);
      *end = __builtin_amdgcn_readlane(s.end, e - base);
    }
  }
}

// ---- plain tiles ------------------------------------------------------------

__device__ __forceinline__ float kept_value(const GroupedParams& p, int64_t t, int64_t k) {
  const uint8_t b = static_cast<const uint8_t*>(p.B)[t * p.K + k];
  const float s = p.b_scale[t * ((p.K + p.group - 1) / p.group) + k / p.group];
  const float q = p.format == KAN_ACT8_INT8 ? (float)(int8_t)b
                                            : __builtin_amdgcn_cvt_f32_fp8((int)b, 0);
  return q * s;
}

// 64 x 64 outputs a block, 4 x 4 a thread, 16 deep.
constexpr int kPlainTile = 64, kPlainDepth = 16;
template <typename T, int OP>
__global__ __launch_bounds__(256) void grouped_plain_kernel(GroupedParams p, int tiles_m,
                                                            int tiles_n) {
  __shared__ float la[kPlainDepth][kPlainTile + 4], lb[kPlainDepth][kPlainTile + 4];
  const int tile = blockIdx.x / tiles_n, n0 = (blockIdx.x % tiles_n) * kPlainTile;
  RowTile rt;
  int64_t kbeg = 0, kend, m_end, n_end, ldc;
  const T *A = static_cast<const T*>(p.A), *B = static_cast<const T*>(p.B);
  T* C = static_cast<T*>(p.C);
  if constexpr (OP == 2) {
    rt.e = tile / tiles_m;
    rt.m0 = (tile % tiles_m) * kPlainTile;
    int lo = 0, hi = 0;
    group_rows(p, rt.e, &lo, &hi);
    kbeg = lo;
    kend = hi;
    m_end = p.N;
    n_end = ldc = p.K;
    C += (int64_t)rt.e * p.N * p.K;
  } else {
    if (tile >= count_tiles(p, kPlainTile)) return;
    rt = find_tile(p, tile, kPlainTile);
    kend = rt.e == p.E ? 0 : OP == 0 ? p.K : p.N;
    m_end = rt.m1;
    n_end = ldc = OP == 0 ? p.N : p.K;
    B += (int64_t)rt.e * p.N * p.K;
  }
  float acc[4][4] = {};
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  for (int64_t k0 = kbeg; k0 < kend; k0 += kPlainDepth) {
    __syncthreads();
    for (int i = threadIdx.x; i < kPlainTile * kPlainDepth; i += 256) {
      const int r = OP == 2 ? i % kPlainTile : i / kPlainDepth;
      const int d = OP == 2 ? i / kPlainTile : i % kPlainDepth;
      const int64_t m = rt.m0 + r, k = k0 + d;
      float v = 0.0f;
      if (m < m_end && k < kend)
        v = (float)(OP == 0 ? A[m * p.K + k] : OP == 1 ? A[m * p.N + k] : A[k * p.N + m]);
      la[d][r] = v;
    }
    for (int i = threadIdx.x; i < kPlainTile * kPlainDepth; i += 256) {
      const int r = OP == 0 ? i / kPlainDepth : i % kPlainTile;
      const int d = OP == 0 ? i % kPlainDepth : i / kPlainTile;
      const int64_t n = n0 + r, k = k0 + d;
      float v = 0.0f;
      if (n < n_end && k < kend) {
        if (OP == 2 && p.format != KAN_ACT8_NONE) v = kept_value(p, k, n);
        else v = (float)(OP == 0 ? B[n * p.K + k] : B[k * p.K + n]);
      }
      lb[d][r] = v;
    }
    __syncthreads();
#pragma unroll
    for (int d = 0; d < kPlainDepth; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[i][j] = __builtin_fmaf(la[d][ty * 4 + i], lb[d][tx * 4 + j], acc[i][j]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t m = rt.m0 + ty * 4 + i, n = n0 + tx * 4 + j;
      if (m < m_end && n < n_end) C[m * ldc + n] = (T)acc[i][j];
    }
}

template <typename T>
int launch_plain(int op, const GroupedParams& p, hipStream_t st) {
  const int64_t cols = op == 0 ? p.N : p.K;
  const int64_t tiles_n = ceil_div(cols, kPlainTile);
  const int64_t tiles_m = op == 2 ? ceil_div(p.N, kPlainTile) : p.T / kPlainTile + p.E + 1;
  const int64_t blocks = tiles_n * tiles_m * (op == 2 ? p.E : 1);
  if (blocks > 0x7fffffff) return set_error(KAN_ERR_LIMIT, "grouped_matmul: too many tiles");
  const dim3 g((unsigned)blocks);
  if (op == 0) grouped_plain_kernel<T, 0><<<g, 256, 0, st>>>(p, (int)tiles_m, (int)tiles_n);
  else if (op == 1) grouped_plain_kernel<T, 1><<<g, 256, 0, st>>>(p, (int)tiles_m, (int)tiles_n);
  else grouped_plain_kernel<T, 2><<<g, 256, 0, st>>>(p, (int)tiles_m, (int)tiles_n);
  return check_launch("grouped_matmul");
}

int check_grouped(int dtype, int op, int64_t T, int64_t E, int64_t N, int64_t K) {
  if (!dtype_is_operator(dtype))
    return set_error(KAN_ERR_INVALID, "grouped_matmul: dtype must be FP32, BF16 or FP16 (code %d)",
                     dtype);
  if (op < KAN_GROUPED_FORWARD || op > KAN_GROUPED_WEIGHT)
    return set_error(KAN_ERR_INVALID, "grouped_matmul: unknown product %d", op);
  if (T < 0 || E < 0 || N < 0 || K < 0)
    return set_error(KAN_ERR_INVALID, "grouped_matmul: negative size");
  constexpr int64_t kMost = 0x7fffffff - 4096;  // (tile ends are held in 32 bits)
  if (T > kMost || N > kMost || K > kMost || E > (1 << 20))
    return set_error(KAN_ERR_LIMIT, "grouped_matmul: at most 2^31 - 4097 rows and columns and 2^20 experts");
  return KAN_OK;
}

}  // namespace
}  // namespace kan

using namespace kan;

extern "C" {

int kan_hip_grouped_matmul_workspace(int dtype, int op, int64_t T, int64_t E, int64_t N, int64_t K,
                                     size_t* bytes) {
  if (bytes == nullptr)
    return set_error(KAN_ERR_INVALID, "grouped_matmul_workspace: bytes must not be NULL");
  const int rc = check_grouped(dtype, op, T, E, N, K);
  if (rc != KAN_OK) return rc;
  *bytes = 0;
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
  (void)workspace;
  (void)workspace_bytes;
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
  if (dtype == KAN_DTYPE_F32) return launch_plain<float>(op, p, st);
  if (dtype == KAN_DTYPE_BF16) return launch_plain<bf16>(op, p, st);
  return launch_plain<f16>(op, p, st);
}

}  // extern "C"
