// Quantisation to 8-bit floating point in blocks of 128 values of a row or 128 x
// 128 tiles (fp8.h says what a block's scale and codes are), and back.
//
// Bound by HBM: values are read once, 16 bytes or more a load, and stay in
// registers from the block's maximum to its codes.
//   Blocks of a row, row-major: 16 threads hold a block, 8 values each (16384 x 4096
//   bf16: 39-41 us, 4.9-5.2 TB/s).
//   Tiles, and matrices whose memory runs along their columns: a workgroup of 256
//   holds 128 x 128 values, 8 x 8 a thread where it transposes: a thread's 8
//   values of one output row leave as 8 bytes into LDS, and from there in
//   16-byte pieces of whole 128-byte runs.
#include <algorithm>

#include "abi.h"
#include "common.h"
#include "enqueue.h"
#include "fp8.h"
#include "rows.h"
#include "../../include/tilec.h"

namespace tilec {

namespace {

struct QuantArgs {
  const void* x;
  unsigned char* codes;
  float* scales;
  int64_t R, C, ldx, ldq;  // of the result; ldx: row stride of x, or of its transpose
  int64_t G;               // scales of a row
  int64_t s_row, s_group;  // strides of the scales
  int e5m2, lg;            // rows kernel: 2^lg blocks of a row side by side
  int xcds, group_m;       // tile kernel: its tiles' order
};

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// The 8 of 128 neighbouring values that one of 16 threads holds: in 16-byte pieces,
// so that a load or store of the 16 threads is one run of 256 bytes (8 fp32 values
// side by side instead: 35.8 us for 4099 x 3001, transposed and back; 32.1 so,
// and 27.8 in the tiles' present order).
template <typename T>
struct Eight {
  static constexpr int V = 16 / (int)sizeof(T), PIECES = 8 / V;
  Group<T, V> g[PIECES];
  __device__ __forceinline__ static int at(int sub, int e) { return V * sub + 128 / PIECES * (e / V) + e % V; }
  __device__ __forceinline__ float get(int e) const { return g[e / V].get(e % V); }
  __device__ __forceinline__ void load(const T* row, int c, int sub, int D) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) g[i].load(row, c + at(sub, V * i), D);
  }
  __device__ __forceinline__ uint32_t top() const {
    uint32_t t = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) t = max(t, __float_as_uint(get(e)) & 0x7fffffffu);
    return t;
  }
  // The codes at columns c + .. of a row, up to column `end` (a multiple of 16); `bits`
  // of them, zeros elsewhere (past a row, where zero times the inverse may be a NaN).
  __device__ __forceinline__ void store(unsigned char* row, int c, int sub, int end, float inverse, bool e5m2,
                                        const uint32_t (&bits)[2]) const {
    uint32_t q[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      q[i] = bits[i] &
             to_fp8(get(4 * i) * inverse, get(4 * i + 1) * inverse, get(4 * i + 2) * inverse, get(4 * i + 3) * inverse, e5m2);
    if constexpr (PIECES == 1) {
      if (c + at(sub, 0) < end) *reinterpret_cast<u32x2*>(row + c + at(sub, 0)) = u32x2{q[0], q[1]};
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (c + at(sub, 4 * i) < end) *reinterpret_cast<uint32_t*>(row + c + at(sub, 4 * i)) = q[i];
    }
  }
};

// Where a row of codes ends: with the bytes that fill its last 16.
__device__ __forceinline__ int row_end(int C) { return (C + 15) / 16 * 16; }

// A workgroup takes 2^lg blocks of 16 >> lg rows at a time, U of those in flight.
template <typename T>
__global__ __launch_bounds__(256) void quant_rows_kernel(QuantArgs a) {
  constexpr int U = 4;
  const int slot = threadIdx.x >> 4, sub = threadIdx.x & 15;
  const int64_t g = ((int64_t)blockIdx.x << a.lg) + (slot & ((1 << a.lg) - 1));
  if (g >= a.G) return;
  const int rpb = 16 >> a.lg;
  const int c = (int)(g * kGroup), C = (int)a.C;
  const bool e5m2 = a.e5m2;
  const int64_t step = (int64_t)gridDim.y * rpb;
  const uint32_t bits[2] = {code_bits(C - c - Eight<T>::at(sub, 0)), code_bits(C - c - Eight<T>::at(sub, 4))};
  for (int64_t r0 = (int64_t)blockIdx.y * rpb + (slot >> a.lg); r0 < a.R; r0 += U * step) {
    Eight<T> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = min(r0 + u * step, a.R - 1);
      v[u].load(static_cast<const T*>(a.x) + r * a.ldx, c, sub, C);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = r0 + u * step;
      if (r >= a.R) break;
      uint32_t top = v[u].top();
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
      float scale, inverse;
      block_scale(top, fp8_largest(e5m2), scale, inverse);
      if (sub == 0) a.scales[r * a.s_row + g * a.s_group] = scale;
      v[u].store(a.codes + r * a.ldq, c, sub, row_end(C), inverse, e5m2, bits);
    }
  }
}

// One 128 x 128 tile of the result a workgroup.  TRANS: x holds its transpose.
// TILE: one scale; otherwise one a row (with TRANS only).
template <typename T, bool TRANS, bool TILE>
__global__ __launch_bounds__(256) void quant_tile_kernel(QuantArgs a, int tiles_c) {
  static_assert(TRANS || TILE, "blocks of row-major rows have a kernel of their own");
  __shared__ uint32_t red[4][TILE ? 1 : 128];
  __shared__ __align__(16) char out[TRANS ? 128 * 128 : 16];
  const int tid = threadIdx.x, lo = tid & 15, hi = tid >> 4, wave = tid >> 6;
  int tr, tc;
  tile_of(blockIdx.x, a.xcds, (int)((a.R + 127) / 128), tiles_c, a.group_m, tr, tc);
  const int64_t r0 = (int64_t)tr * 128;
  const int c0 = tc * 128, C = (int)a.C;
  const bool e5m2 = a.e5m2;
  // TRANS: v[p] is of memory row c0 + 8 hi + p (a column of the result), its values
  // those of eight of the result's rows from r0 on; otherwise of row r0 + 16 p + hi,
  // eight columns from c0 on.
  auto mine = [&](int e) { return Eight<T>::at(lo, e); };
  Eight<T> v[8];
  uint32_t top[8];
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    const int64_t m = TRANS ? c0 + 8 * hi + p : r0 + 16 * p + hi;
    const bool live = m < (TRANS ? a.C : a.R);
    const T* row = static_cast<const T*>(a.x) + (live ? m : 0) * a.ldx;
    v[p].load(row, TRANS ? (int)r0 : c0, lo, live ? (int)(TRANS ? a.R : a.C) : 0);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    top[e] = 0;
#pragma unroll
    for (int p = 0; p < 8; ++p) top[e] = max(top[e], __float_as_uint(v[p].get(e)) & 0x7fffffffu);
  }
  float inverse[8], scale;
  if constexpr (TILE) {
    uint32_t t = top[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) t = max(t, top[e]);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) t = max(t, (uint32_t)__shfl_xor((int)t, o));
    if ((tid & 63) == 0) red[wave][0] = t;
    __syncthreads();
    t = max(max(red[0][0], red[1][0]), max(red[2][0], red[3][0]));
    block_scale(t, fp8_largest(e5m2), scale, inverse[0]);
#pragma unroll
    for (int e = 1; e < 8; ++e) inverse[e] = inverse[0];
    if (tid == 0) a.scales[tr * a.s_row + tc * a.s_group] = scale;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      top[e] = max(top[e], (uint32_t)__shfl_xor((int)top[e], 16));
      top[e] = max(top[e], (uint32_t)__shfl_xor((int)top[e], 32));
    }
    if ((hi & 3) == 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) red[wave][mine(e)] = top[e];
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int r = mine(e);
      const uint32_t t = max(max(red[0][r], red[1][r]), max(red[2][r], red[3][r]));
      block_scale(t, fp8_largest(e5m2), scale, inverse[e]);
      if (hi == 0 && r0 + r < a.R) a.scales[(r0 + r) * a.s_row + tc * a.s_group] = scale;
    }
  }
  const int end = row_end(C);
  if constexpr (!TRANS) {
    const uint32_t bits[2] = {code_bits(C - c0 - mine(0)), code_bits(C - c0 - mine(4))};
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      const int64_t r = r0 + 16 * p + hi;
      if (r < a.R) v[p].store(a.codes + r * a.ldq, c0, lo, end, inverse[0], e5m2, bits);
    }
  } else {
    // Row mine(e) of the tile, columns 8 hi ..: 8-byte piece hi of its 16, exchanged
    // by rows (by lo).
    constexpr int ROWS = Eight<T>::V;  // side by side in one thread
    const uint32_t bits[2] = {code_bits(C - c0 - 8 * hi), code_bits(C - c0 - 8 * hi - 4)};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      u32x2 q;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        q[i] = bits[i] & to_fp8(v[4 * i].get(e) * inverse[e], v[4 * i + 1].get(e) * inverse[e],
                                v[4 * i + 2].get(e) * inverse[e], v[4 * i + 3].get(e) * inverse[e], e5m2);
      *reinterpret_cast<u32x2*>(out + 128 * mine(e) + 8 * (hi ^ lo)) = q;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int row = 32 * k + (tid >> 3), piece = tid & 7, swap = row / ROWS & 15;
      const u32x2 a0 = *reinterpret_cast<const u32x2*>(out + 128 * row + 8 * ((2 * piece) ^ swap));
      const u32x2 a1 = *reinterpret_cast<const u32x2*>(out + 128 * row + 8 * ((2 * piece + 1) ^ swap));
      if (r0 + row < a.R && c0 + 16 * piece < end)
        *reinterpret_cast<u32x4*>(a.codes + (r0 + row) * a.ldq + c0 + 16 * piece) = u32x4{a0.x, a0.y, a1.x, a1.y};
    }
  }
}

struct ValuesArgs {
  const unsigned char* codes;
  const float* scales;
  void* out;
  int64_t R, C, ldq, ldo, G, s_row, s_group;
  int shift, e5m2, lg;
};

// The values that codes stand for, mapped as in quant_rows_kernel.
template <typename T>
__global__ __launch_bounds__(256) void values_kernel(ValuesArgs a) {
  constexpr int U = 4, V = Eight<T>::V, PIECES = Eight<T>::PIECES;
  const int slot = threadIdx.x >> 4, sub = threadIdx.x & 15;
  const int64_t g = ((int64_t)blockIdx.x << a.lg) + (slot & ((1 << a.lg) - 1));
  if (g >= a.G) return;
  const int c = (int)(g * kGroup), C = (int)a.C, rpb = 16 >> a.lg;
  const int64_t step = (int64_t)gridDim.y * rpb;
  for (int64_t r0 = (int64_t)blockIdx.y * rpb + (slot >> a.lg); r0 < a.R; r0 += U * step) {
    uint32_t q[U][2];
    float s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = min(r0 + u * step, a.R - 1);
      s[u] = a.scales[(r >> a.shift) * a.s_row + g * a.s_group];
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int k = c + Eight<T>::at(sub, V * i);
        const unsigned char* p = a.codes + r * a.ldq + k;
        uint32_t* const to = q[u] + i;  // V codes
        if (k + V <= C) {
          typedef u32x2 __attribute__((aligned(1))) u32x2_any;
          typedef uint32_t __attribute__((aligned(1))) u32_any;
          if constexpr (V == 8) {
            const u32x2 w = *reinterpret_cast<const u32x2_any*>(p);
            to[0] = w.x, to[1] = w.y;
          } else {
            to[0] = *reinterpret_cast<const u32_any*>(p);
          }
        } else {
#pragma unroll
          for (int w = 0; w < V / 4; ++w) {
            to[w] = 0u;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (k + 4 * w + e < C) to[w] |= (uint32_t)p[4 * w + e] << (8 * e);
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = r0 + u * step;
      if (r >= a.R) break;
      float v[PIECES][V];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        const int w = (int)q[u][i];
        f32x2 x, y;
        if (a.e5m2) x = __builtin_amdgcn_cvt_pk_f32_bf8(w, false), y = __builtin_amdgcn_cvt_pk_f32_bf8(w, true);
        else x = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), y = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
        float* const to = v[4 * i / V] + 4 * i % V;
        to[0] = x.x * s[u], to[1] = x.y * s[u], to[2] = y.x * s[u], to[3] = y.y * s[u];
      }
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int k = c + Eight<T>::at(sub, V * i);
        if (k < C) store_group<T, V>(static_cast<T*>(a.out) + r * a.ldo, k, C, v[i]);
      }
    }
  }
}

// The grid over a matrix of G blocks a row, 2^lg of them side by side in a
// workgroup of 16.
dim3 rows_grid(int64_t R, int64_t G, int& lg) {
  lg = 0;
  while (lg < 4 && (int64_t(1) << lg) < G) ++lg;
  const int64_t gx = cdiv(G, int64_t(1) << lg);
  const int64_t full = cdiv(R, 4 * (16 >> lg));  // 4 rows a thread
  return dim3((unsigned)gx, (unsigned)std::max<int64_t>(1, std::min<int64_t>(full, 65535)));
}

int check_matrix(const char* what, int64_t R, int64_t C, int32_t wide, int32_t fp8, int32_t block) {
  if ((wide != TILEC_F32 && wide != TILEC_BF16) || !is_fp8(fp8))
    return fail(TILEC_ERR_TYPE, "tilec: %s: unsupported dtype codes %d, %d (use float32 or bfloat16, and an 8-bit type)",
                what, wide, fp8);
  if (R < 0 || C < 0 || R > kMaxDim || C > kMaxDim)
    return fail(TILEC_ERR_VALUE, "tilec: %s: bad shape %lld x %lld", what, (long long)R, (long long)C);
  if (block != 1 && block != kGroup)
    return fail(TILEC_ERR_VALUE, "tilec: %s: blocks have 1 or 128 rows (got %d)", what, block);
  return TILEC_OK;
}

constexpr int64_t kMaxStride = int64_t(1) << 40;

}  // namespace

}  // namespace tilec

using namespace tilec;

extern "C" {

int tilec_quantize_fp8(const void* x, void* codes, float* scales, int64_t R, int64_t C, int64_t ldx, int64_t ldq,
                       int64_t scale_row, int64_t scale_group, int32_t layout, int32_t x_dtype, int32_t q_dtype,
                       int32_t block, void* stream) {
  clear_error();
  const int rc = check_matrix("quantize_fp8", R, C, x_dtype, q_dtype, block);
  if (rc != TILEC_OK) return rc;
  if (layout != 0 && layout != TILEC_X1_COL_MAJOR)
    return fail(TILEC_ERR_VALUE, "tilec: quantize_fp8: bad layout %d", layout);
  if (R == 0 || C == 0) return TILEC_OK;
  const bool trans = layout != 0;
  const int64_t rows = trans ? C : R, cols = trans ? R : C, room = cdiv(C, 16) * 16;
  if ((rows > 1 && ldx < cols) || ldx > kMaxStride)
    return fail(TILEC_ERR_VALUE, "tilec: quantize_fp8: bad stride %lld of x", (long long)ldx);
  if (x == nullptr || codes == nullptr || scales == nullptr)
    return fail(TILEC_ERR_VALUE, "tilec: quantize_fp8: a pointer is NULL");
  if (scale_row < 0 || scale_group < 0 || scale_row > kMaxStride || scale_group > kMaxStride)
    return fail(TILEC_ERR_VALUE, "tilec: quantize_fp8: bad strides %lld, %lld of scales",
                (long long)scale_row, (long long)scale_group);
  if (reinterpret_cast<uintptr_t>(codes) % 16 != 0 || (R > 1 && (ldq % 16 != 0 || ldq < room || ldq > kMaxStride)))
    return fail(TILEC_ERR_VALUE, "tilec: quantize_fp8: rows of codes begin at multiples of 16 bytes (row stride %lld)",
                (long long)ldq);
  QuantArgs a{};
  a.x = x, a.codes = static_cast<unsigned char*>(codes), a.scales = scales;
  a.R = R, a.C = C, a.ldx = rows > 1 ? ldx : cols, a.ldq = R > 1 ? ldq : room, a.G = cdiv(C, kGroup);
  a.s_row = scale_row, a.s_group = scale_group, a.e5m2 = q_dtype == TILEC_F8E5M2;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  auto by_type = [&](auto t) {
    using T = decltype(t);
    if (!trans && block == 1) {
      const dim3 grid = rows_grid(R, a.G, a.lg);
      return enqueue(quant_rows_kernel<T>, grid, dim3(256), st, a);
    }
    const int64_t tiles = cdiv(R, 128) * a.G;
    if (tiles > INT32_MAX) return hipErrorInvalidValue;
    // Neighbours on one XCD, so that lines that two tiles share meet in its L2 (bf16
    // 8192 x 8192 transposed, 47.4 us in the order of their numbers and 37.0; 4099 x
    // 3001 fp32 tiles 16.8 and 15.1); tiles of whole lines side by side go by numbers
    // (8192 x 4096 bf16 18.9 us, 20.9 the other way).
    const bool shared = trans || ldx * (int64_t)sizeof(T) % 128 != 0;
    a.xcds = shared ? device_xcds() : 1, a.group_m = shared ? 8 : 1;
    const dim3 grid((unsigned)tiles);
    const int tiles_c = (int)a.G;
    const auto kernel = !trans       ? quant_tile_kernel<T, false, true>
                        : block == 1 ? quant_tile_kernel<T, true, false>
                                     : quant_tile_kernel<T, true, true>;
    return enqueue(kernel, grid, dim3(256), st, a, tiles_c);
  };
  const hipError_t e = x_dtype == TILEC_F32 ? by_type(float{}) : by_type(u16{});
  if (e != hipSuccess) return fail(TILEC_ERR_HIP, "tilec: launching quantize_fp8 failed: %s", hipGetErrorString(e));
  return TILEC_OK;
}

int tilec_dequantize_fp8(const void* codes, const float* scales, void* out, int64_t R, int64_t C, int64_t ldq,
                         int64_t ldo, int64_t scale_row, int64_t scale_group, int32_t q_dtype, int32_t out_dtype,
                         int32_t block, void* stream) {
  clear_error();
  const int rc = check_matrix("dequantize_fp8", R, C, out_dtype, q_dtype, block);
  if (rc != TILEC_OK) return rc;
  if (R == 0 || C == 0) return TILEC_OK;
  if (R > 1 && (ldq < C || ldo < C || ldq > kMaxStride || ldo > kMaxStride))
    return fail(TILEC_ERR_VALUE, "tilec: dequantize_fp8: bad row strides %lld, %lld", (long long)ldq, (long long)ldo);
  if (codes == nullptr || scales == nullptr || out == nullptr)
    return fail(TILEC_ERR_VALUE, "tilec: dequantize_fp8: a pointer is NULL");
  if (scale_row < 0 || scale_group < 0 || scale_row > kMaxStride || scale_group > kMaxStride)
    return fail(TILEC_ERR_VALUE, "tilec: dequantize_fp8: bad strides %lld, %lld of scales",
                (long long)scale_row, (long long)scale_group);
  ValuesArgs a{};
  a.codes = static_cast<const unsigned char*>(codes), a.scales = scales, a.out = out;
  a.R = R, a.C = C, a.ldq = ldq, a.ldo = ldo, a.G = cdiv(C, kGroup);
  a.s_row = scale_row, a.s_group = scale_group, a.shift = block == 1 ? 0 : 7, a.e5m2 = q_dtype == TILEC_F8E5M2;
  const dim3 grid = rows_grid(R, a.G, a.lg);
  const auto kernel = out_dtype == TILEC_F32 ? values_kernel<float> : values_kernel<u16>;
  const hipError_t e = enqueue(kernel, grid, dim3(256), static_cast<hipStream_t>(stream), a);
  if (e != hipSuccess) return fail(TILEC_ERR_HIP, "tilec: launching dequantize_fp8 failed: %s", hipGetErrorString(e));
  return TILEC_OK;
}

}  // extern "C"
