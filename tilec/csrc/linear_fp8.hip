// tilec_linear_fp8: the choice of a kernel of linear_fp8.h, operands whose rows do
// not begin at multiples of 16 bytes, and the sums of split groups.
#include <algorithm>

#include "abi.h"
#include "linear_fp8.h"
#include "zeros.h"

namespace tilec {

namespace {

constexpr int64_t kMaxScaleRow = int64_t(1) << 21, kMaxScaleGroup = int64_t(1) << 40;
constexpr int64_t kMaxTiles = (int64_t(1) << 23) - 1;  // of up to 512 threads: a grid has less than 2^32

struct Plan {
  int tile;            // -1: the streaming kernel
  int splits, steps;   // groups of K a split
  bool copy_x, copy_w;
  int64_t padded;      // row stride of a copied operand
  size_t x_bytes, w_bytes, partial_bytes, counter_bytes;
  size_t bytes() const { return x_bytes + w_bytes + partial_bytes; }
};

size_t round16(int64_t n) { return (size_t)(n + 15) / 16 * 16; }

struct Scales {
  int block;
  int64_t row, group;  // strides
};

Plan plan_of(const void* x, const void* w, int64_t M, int64_t N, int64_t K, int64_t ldx, int64_t ldw, bool f8) {
  Plan p{};
  auto aligned = [](const void* q, int64_t rows, int64_t ld) {
    return reinterpret_cast<uintptr_t>(q) % 16 == 0 && (rows <= 1 || (ld % 16 == 0 && ld <= (int64_t(1) << 22)));
  };
  p.copy_x = !aligned(x, M, ldx), p.copy_w = !aligned(w, N, ldw);
  p.padded = (int64_t)round16(K);
  p.x_bytes = p.copy_x ? (size_t)(M * p.padded) : 0;
  p.w_bytes = p.copy_w ? (size_t)(N * p.padded) : 0;
  const int64_t G = cdiv(K, kGroup), cus = device_cus();
  p.splits = 1, p.steps = (int)G;
  if (M <= kFp8StreamRows) {
    p.tile = -1;
    return p;
  }
  // The tile and the splits of K that are estimated to be done first: whole turns
  // over the chip, and with splits the partial sums, added up by the last of a tile's
  // workgroups `batch` splits at a time (measured 1.5 to 2.2 us for one batch, 3.5 and
  // 5.3 for two and three; a kernel of its own took 4 to 13: 38 x 3584 x 4800 bf16 13.0
  // us so, 8.3 now, 70 x 192 x 9088 17.5 and 9.1).
  p.tile = kFp8TileCount;
  double best = 1e30;
  for (int t = 0; t < kFp8TileCount; ++t) {
    const Fp8Tile& g = kFp8Tiles[t];
    const int64_t n = cdiv(M, g.bm) * cdiv(N, g.bn[f8]);
    if (n > kMaxTiles) continue;
    const int64_t most = t == 0 ? 1 : std::min<int64_t>(G, 64);
    for (int64_t s = 1; s <= most; ++s) {
      const int64_t steps = cdiv(G, s), splits = cdiv(G, steps);
      if (splits != s) continue;
      const int64_t groups = n * splits;
      if (s > 1 && (groups > 2 * cus || groups * g.bm * g.bn[f8] >= (int64_t(1) << 29))) break;
      const bool two = g.step2[f8] > 0.f && groups > cus;
      double time = (double)cdiv(groups, two ? 2 * cus : cus) * (g.fixed[f8] + (double)steps * (two ? g.step2 : g.step)[f8]);
      if (s > 1) time += 0.2 + 1.6 * (double)cdiv(s, g.batch) + (double)M * (double)N * 8. * (double)s / 12e6;
      if (time < best) best = time, p.tile = t, p.splits = (int)splits, p.steps = (int)steps;
    }
  }
  if (p.splits > 1) {
    const Fp8Tile& g = kFp8Tiles[p.tile];
    const int64_t n = cdiv(M, g.bm) * cdiv(N, g.bn[f8]);
    p.partial_bytes = (size_t)(p.splits * n * g.bm * g.bn[f8] * 4);
    p.counter_bytes = (size_t)n * kSplitCounterStride * sizeof(unsigned);
  }
  return p;
}

int check_linear(int64_t M, int64_t N, int64_t K, int64_t ldx, int64_t ldw, int32_t x_dtype, int32_t w_dtype,
                 int32_t out_dtype, Scales sx, Scales sw) {
  if (!is_fp8(x_dtype) || !is_fp8(w_dtype))
    return fail(TILEC_ERR_TYPE, "tilec: linear_fp8: unsupported dtype codes %d, %d of x and weight (use an 8-bit type)",
                x_dtype, w_dtype);
  if (out_dtype != TILEC_F32 && out_dtype != TILEC_BF16)
    return fail(TILEC_ERR_TYPE, "tilec: linear_fp8: unsupported dtype code %d of out (use float32 or bfloat16)", out_dtype);
  if (M < 0 || N < 0 || K < 0 || M > kMaxDim || N > kMaxDim || K > (int64_t(1) << 22))
    return fail(TILEC_ERR_VALUE, "tilec: linear_fp8: bad shape M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  if ((M > 1 && (ldx < K || ldx > (int64_t(1) << 40))) || (N > 1 && (ldw < K || ldw > (int64_t(1) << 40))))
    return fail(TILEC_ERR_VALUE, "tilec: linear_fp8: bad row strides ldx=%lld ldw=%lld for K=%lld", (long long)ldx,
                (long long)ldw, (long long)K);
  if ((sx.block != 1 && sx.block != kGroup) || (sw.block != 1 && sw.block != kGroup))
    return fail(TILEC_ERR_VALUE, "tilec: linear_fp8: blocks have 1 or 128 rows (got %d and %d)", sx.block, sw.block);
  // (256 rows' scales lie within 2^31 bytes.)
  for (const Scales& s : {sx, sw})
    if (s.row < 0 || s.group < 0 || s.row > kMaxScaleRow || s.group > kMaxScaleGroup)
      return fail(TILEC_ERR_VALUE, "tilec: linear_fp8: bad strides %lld, %lld of scales", (long long)s.row, (long long)s.group);
  return TILEC_OK;
}

}  // namespace

}  // namespace tilec

using namespace tilec;

extern "C" {

int tilec_linear_fp8_scratch_bytes(const void* x, const void* weight, int64_t M, int64_t N, int64_t K, int64_t ldx,
                                   int64_t ldw, int32_t x_dtype, int32_t w_dtype, int32_t out_dtype,
                                   size_t* workspace_bytes, size_t* counter_bytes) {
  clear_error();
  const Scales sx{1, 0, 0}, sw{1, 0, 0};
  const int rc = check_linear(M, N, K, ldx, ldw, x_dtype, w_dtype, out_dtype, sx, sw);
  if (rc != TILEC_OK) return rc;
  const Plan p = M > 0 && N > 0 && K > 0 ? plan_of(x, weight, M, N, K, ldx, ldw, out_dtype == TILEC_BF16) : Plan{};
  if (workspace_bytes != nullptr) *workspace_bytes = p.bytes();
  if (counter_bytes != nullptr) *counter_bytes = p.counter_bytes;
  return TILEC_OK;
}

int tilec_linear_fp8(const void* x, const float* x_scale, const void* weight, const float* w_scale, void* out,
                     int64_t M, int64_t N, int64_t K, int64_t ldx, int64_t ldw, int64_t ldo, int64_t x_scale_row,
                     int64_t x_scale_group, int64_t w_scale_row, int64_t w_scale_group, int32_t x_dtype, int32_t w_dtype,
                     int32_t out_dtype, int32_t x_block, int32_t w_block, void* workspace, size_t workspace_bytes,
                     void* counters, size_t counter_bytes, void* stream) {
  clear_error();
  const Scales sx{x_block, x_scale_row, x_scale_group}, sw{w_block, w_scale_row, w_scale_group};
  const int rc = check_linear(M, N, K, ldx, ldw, x_dtype, w_dtype, out_dtype, sx, sw);
  if (rc != TILEC_OK) return rc;
  if (M == 0 || N == 0) return TILEC_OK;
  if (M > 1 && (ldo < N || ldo > (int64_t(1) << 40)))
    return fail(TILEC_ERR_VALUE, "tilec: linear_fp8: bad row stride ldo=%lld for N=%lld", (long long)ldo, (long long)N);
  if (out == nullptr || (K > 0 && (x == nullptr || weight == nullptr || x_scale == nullptr || w_scale == nullptr)))
    return fail(TILEC_ERR_VALUE, "tilec: linear_fp8: a pointer is NULL");
  const bool f8 = out_dtype == TILEC_BF16;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (K == 0) {
    const int64_t row = M > 1 ? ldo : N;
    const hipError_t e = f8 ? enqueue_zeros(static_cast<uint16_t*>(out), M, N, row, st)
                            : enqueue_zeros(static_cast<float*>(out), M, N, row, st);
    if (e != hipSuccess) return fail(TILEC_ERR_HIP, "tilec: launching linear_fp8 failed: %s", hipGetErrorString(e));
    return TILEC_OK;
  }
  const Plan p = plan_of(x, weight, M, N, K, ldx, ldw, f8);
  if (p.tile == kFp8TileCount)
    return fail(TILEC_ERR_VALUE, "tilec: linear_fp8: %lld x %lld outputs are too many for one launch", (long long)M,
                (long long)N);
  if (p.bytes() > 0 && (workspace == nullptr || workspace_bytes < p.bytes()))
    return fail(TILEC_ERR_WORKSPACE, "tilec: linear_fp8 needs %zu workspace bytes (got %zu)", p.bytes(),
                workspace == nullptr ? (size_t)0 : workspace_bytes);
  if (p.counter_bytes > 0 && (counters == nullptr || counter_bytes < p.counter_bytes))
    return fail(TILEC_ERR_WORKSPACE, "tilec: linear_fp8 needs %zu counter bytes (got %zu)", p.counter_bytes,
                counters == nullptr ? (size_t)0 : counter_bytes);
  char* const ws = static_cast<char*>(workspace);
  hipError_t e = hipSuccess;
  if (p.copy_x || p.copy_w) {
    e = pad_copy<1>(x, ws, M, K, ldx, p.copy_x ? M : 0, p.padded, weight, ws + p.x_bytes, N, K, ldw,
                    p.copy_w ? N : 0, p.padded, st);
    if (e != hipSuccess) return fail(TILEC_ERR_HIP, "tilec: linear_fp8: copying an operand failed: %s", hipGetErrorString(e));
  }
  Fp8Args a{};
  a.x = p.copy_x ? reinterpret_cast<unsigned char*>(ws) : static_cast<const unsigned char*>(x);
  a.w = p.copy_w ? reinterpret_cast<unsigned char*>(ws + p.x_bytes) : static_cast<const unsigned char*>(weight);
  a.sx = x_scale, a.sw = w_scale, a.out = out;
  a.sx_row = sx.row, a.sx_group = sx.group, a.sw_row = sw.row, a.sw_group = sw.group;
  a.partial = reinterpret_cast<float*>(ws + p.x_bytes + p.w_bytes);
  a.counters = static_cast<unsigned*>(counters);
  // (One row has no stride; its length stands in.)
  a.ldx = p.copy_x || M == 1 ? p.padded : ldx, a.ldw = p.copy_w || N == 1 ? p.padded : ldw, a.ldo = M > 1 ? ldo : N;
  a.M = (int)M, a.N = (int)N, a.K = (int)K, a.G = (int)cdiv(K, kGroup);
  a.xshift = x_block == 1 ? 0 : 7, a.wshift = w_block == 1 ? 0 : 7;
  a.group_m = 8, a.xcds = device_xcds(), a.split_steps = p.steps;
  const int fx = x_dtype == TILEC_F8E5M2, fw = w_dtype == TILEC_F8E5M2;
  e = fx ? (fw ? launch_fp8<1, 1>(a, f8, p.tile, p.splits, st) : launch_fp8<1, 0>(a, f8, p.tile, p.splits, st))
         : (fw ? launch_fp8<0, 1>(a, f8, p.tile, p.splits, st) : launch_fp8<0, 0>(a, f8, p.tile, p.splits, st));
  if (e != hipSuccess) return fail(TILEC_ERR_HIP, "tilec: launching linear_fp8 failed: %s", hipGetErrorString(e));
  return TILEC_OK;
}

}  // extern "C"
