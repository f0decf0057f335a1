// Cross entropy of a linear layer's outputs, without giving them out:
//   l = x W^T  (x [N, H], W [V, H])        lse_r = log sum_v exp(l_rv)
//   loss_r = lse_r - l[r, t_r]             (0 where t_r is ignored)
//   d_rv = g_r (exp(l_rv - lse_r) - [v = t_r])   (0 in ignored rows)
//   dx = d W       dW = d^T x
// with g_r the gradient of row r's loss (1 / count times the scalar's for the
// mean).
//
// Three products of 2 N H V operations bound it: the logits are formed once,
// and what the gradients need of them is one 16-bit value each.  Rows are
// taken in chunks, so that those values fit the workspace.
//
// bf16 inputs.  The logits' product ends in an epilogue that never stores
// them.  It runs with W as its row operand, so a lane holds consecutive
// vocabulary entries of one token: a wave takes the maximum m and the sum of
// exp(l - m) over 64 entries of a token in its own registers and two shuffles,
// writes those two, and (for gradients) exp(l - m) 2^15 in fp16, whose 11 bits
// leave the one rounding to bf16 that d itself gets as the only one that
// counts; values below 2^-29 of the largest in their group lose bits, below
// 2^-39 they are lost.  (The matrix cores take d in bf16 or not at all: with it,
// dx and dW are 1.90e-3 off in the 2-norm at 7 x 1024 x 32768, 1.68e-3 with their
// own rounding alone; 1.72e-3 and 1.66e-3 at 1000 x 1000 x 50021, 1.68e-3 and
// 1.66e-3 at 4096 x 4096 x 131072.)  One pass over them (ce_rows_kernel) then
// joins the groups to lse and turns each, in place, into d in bf16.  The target's
// own entry, where exp(l - lse) - 1 cancels, is taken from the fp32 logit.  The
// scalar factor of d (1 / count) is kept out of it and applied to the fp32 sums
// of dx and dW, so that it costs no rounding of its own.
//
// fp32 inputs.  The library's own products (tilec_matmul) form the logits
// chunk and the gradients; l becomes d in place, in fp32.
#include <algorithm>
#include <cfloat>

#include "abi.h"
#include "gemm_bf16_lds.h"
#include "../../include/tilec.h"

namespace tilec {

namespace {

typedef _Float16 f16;
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef int i32x2 __attribute__((ext_vector_type(2)));

constexpr float kScale16 = 32768.f;  // exp(l - m) <= 1 uses fp16's range up to 2^15

__device__ __forceinline__ u16 bf16_bits(float f) { return __builtin_bit_cast(u16, (__bf16)f); }

// ---------------------------------------------------------------------------
// Epilogues of the bf16 products
// ---------------------------------------------------------------------------

constexpr int kGroup = 64;  // vocabulary entries of one (m, sum) pair

// The logits: rows are vocabulary entries (from v0 on), columns tokens.
struct CeLogits {
  static constexpr bool kStaged = true, kOwnSplits = false;
  u16* e;      // exp(l - m) 2^15 in fp16, [token][lde]; NULL: losses only
  int64_t lde;
  f32x2* stat;  // (m, sum of exp(l - m)), [token][groups]
  int groups;   // even
  int v0;
  const int64_t* target;
  float* tlogit;  // the target's logit, [token]

  template <class P, int MF>
  __device__ __forceinline__ void run(const TileOut<P, MF>& t, typename P::Acc (&acc)[P::TM][P::TN], int V,
                                      int N) const {
    if (t.interior) tile<P, MF, true>(t, acc, V, N);
    else tile<P, MF, false>(t, acc, V, N);
  }

  template <class P, int MF, bool FULL>
  __device__ __forceinline__ void tile(const TileOut<P, MF>& t, typename P::Acc (&acc)[P::TM][P::TN], int V,
                                       int N) const {
    static_assert(MF == 16 && P::WTM % kGroup == 0, "a wave's rows are whole groups");
    constexpr float kLog2e = 1.44269504088896f;
    constexpr int G = P::WTM / kGroup, BPG = P::TM / G;  // groups of a wave, row blocks of a group
    const int first = t.m0 + t.wm * P::WTM;
    int64_t want[P::TN];  // read ahead of their use
#pragma unroll
    for (int j = 0; j < P::TN; ++j) want[j] = FULL || t.col(j) < N ? target[t.col(j)] : -1;
#pragma unroll
    for (int j = 0; j < P::TN; ++j) {
      const int tok = t.col(j);
      float m[G], s[G];
#pragma unroll
      for (int g = 0; g < G; ++g) {
        m[g] = -FLT_MAX;
#pragma unroll
        for (int i = g * BPG; i < (g + 1) * BPG; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (FULL || t.row(i, r) < V) m[g] = fmaxf(m[g], acc[i][j][r]);
        m[g] = fmaxf(m[g], __shfl_xor(m[g], 16));
        m[g] = fmaxf(m[g], __shfl_xor(m[g], 32));
      }
      // exp(l - m) 2^15 = 2^((l - m) log2 e + 15): the difference first, so that
      // it is exact where it matters.
#pragma unroll
      for (int g = 0; g < G; ++g) {
        s[g] = 0.f;
#pragma unroll
        for (int i = g * BPG; i < (g + 1) * BPG; ++i) {
          f32x4 x;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            x[c] = __builtin_amdgcn_exp2f(fmaf(acc[i][j][c] - m[g], kLog2e, 15.f));
            if (!FULL && t.row(i, c) >= V) x[c] = 0.f;
          }
          s[g] += (x[0] + x[1]) + (x[2] + x[3]);
          if (e != nullptr) {
            const i32x2 h = __builtin_bit_cast(i32x2, __builtin_convertvector(x, f16x4));
            t.put(i, 0, j, h.x, h.y);
          }
        }
        s[g] += __shfl_xor(s[g], 16);
        s[g] += __shfl_xor(s[g], 32);
      }
      if (t.lane < 16 && (FULL || tok < N)) {
        f32x2* to = stat + (int64_t)tok * groups + (v0 + first) / kGroup;
        if constexpr (G == 2) {
          *reinterpret_cast<f32x4*>(to) = f32x4{m[0], s[0] * (1.f / kScale16), m[1], s[1] * (1.f / kScale16)};
        } else {
#pragma unroll
          for (int g = 0; g < G; ++g) to[g] = f32x2{m[g], s[g] * (1.f / kScale16)};
        }
      }
    }
    if (e != nullptr)
      t.store_all([&](int n, int v, i32x4 x) {
        if (FULL || (n < N && v0 + v < lde)) *reinterpret_cast<i32x4*>(e + (int64_t)n * lde + v0 + v) = x;
      });
#pragma unroll
    for (int j = 0; j < P::TN; ++j) {
      // The target's logit: one wave in V / WTM holds it.
      const int64_t at = want[j] - v0 - first;
      if (want[j] >= 0 && at >= 0 && at < P::WTM && first + at < V) {
#pragma unroll
        for (int i = 0; i < P::TM; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (t.row(i, r) - first == (int)at) tlogit[t.col(j)] = acc[i][j][r];
      }
    }
  }
};

// A gradient, stored transposed: rows are the hidden dimension, columns
// tokens (dx) or vocabulary entries (dW).  Over several chunks of rows dW is
// added up in fp32 and rounded once, by the last; each K split of a product
// stores its own fp32 sums, which ce_finish_kernel adds in order (the tile
// kernel's own combine, in which a tile's last workgroup reads every split,
// took 16 of the 31 us of a 7 x 32768 x 1024 dx in 32 splits).
struct CeGrad {
  static constexpr bool kStaged = true, kOwnSplits = true;
  u16* out;  // bf16, [column][ldo]; NULL: fp32 sums only
  int64_t ldo;
  float* acc32;         // fp32 sums, [split][column][ld32]
  int64_t ld32, split;  // split: elements of one
  bool add;             // to what acc32 holds
  const float* scale;   // applied when out is written
  // dx: the rows' targets.  Ignored rows get zeros by choice, not by a product:
  // their sums are zeros, but the scalar factor may be infinite or a NaN.
  const int64_t* target;  // NULL: dW
  int64_t ignore;

  template <class P, int MF>
  __device__ __forceinline__ void run(const TileOut<P, MF>& t, typename P::Acc (&acc)[P::TM][P::TN], int H,
                                      int N) const {
    const float f = out != nullptr ? *scale : 1.f;
    bool skip[P::TN] = {};
    if (out != nullptr && target != nullptr) {
#pragma unroll
      for (int j = 0; j < P::TN; ++j) skip[j] = target[min(t.col(j), N - 1)] == ignore;
    }
#pragma unroll
    for (int j = 0; j < P::TN; ++j)
#pragma unroll
      for (int i = 0; i < P::TM; ++i)
#pragma unroll
        for (int q = 0; q < P::ACC / 4; ++q) {
          f32x4 v = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
          if (acc32 != nullptr && t.col(j) < N && t.row(i, 4 * q) < H) {  // ld32 is a multiple of 16
            f32x4* p = reinterpret_cast<f32x4*>(acc32 + t.split * split + (int64_t)t.col(j) * ld32 + t.row(i, 4 * q));
            if (add) v += *p;
            if (out == nullptr) *p = v;
          }
          if (out != nullptr) {
            const int lo = (int)(bf16_bits(v[0] * f) | (uint32_t)bf16_bits(v[1] * f) << 16);
            const int hi = (int)(bf16_bits(v[2] * f) | (uint32_t)bf16_bits(v[3] * f) << 16);
            t.put(i, q, j, skip[j] ? 0 : lo, skip[j] ? 0 : hi);
          }
        }
    if (out == nullptr) return;
    t.store_all([&](int n, int h, i32x4 x) {
      typedef i32x4 __attribute__((aligned(2))) i32x4_any;
      u16* o = out + (int64_t)n * ldo + h;
      if (t.interior || (n < N && h + 8 <= H)) {
        *reinterpret_cast<i32x4_any*>(o) = x;
      } else if (n < N) {
#pragma unroll
        for (int c = 0; c < 8; ++c)
          if (h + c < H) o[c] = (u16)((uint32_t)x[c / 2] >> (16 * (c & 1)));
      }
    });
  }
};

// ---------------------------------------------------------------------------
// Kernels around the products
// ---------------------------------------------------------------------------

enum Reduction { kNone, kSum, kMean };

constexpr int kFewRows = 32;  // of ce_few_rows_kernel

// xs = x with the ignored rows cleared (whatever they hold must not reach dW,
// where 0 times a NaN would be one) and rows padded with zeros to Hp; where xt
// is set, also its transpose [H][kFewRows], padded with zeros; and, by the last
// workgroup where `scale` is set, the scalar factor of the gradients.
template <typename T>
struct CePrepare {
  const T* x;
  int64_t ldx;
  T *xs, *xt;
  int64_t Hp, N, H;
  const int64_t* target;
  int64_t ignore;
  float* scale;
  int64_t all;  // rows of all chunks, and their targets
  const int64_t* all_targets;
  int reduction;
  const float* grad_loss;

  // Workgroup `block` of `blocks` (two at least where scale is set), 256 threads.
  __device__ void run(int64_t block, int64_t blocks, int* count) const {
    constexpr int E = 16 / (int)sizeof(T);
    typedef i32x4 __attribute__((aligned(2))) i32x4_any;
    if (scale != nullptr && block == --blocks) {
      int n = 0;
#pragma unroll 8
      for (int64_t i = threadIdx.x; i < all; i += 256) n += all_targets[i] != ignore;
      count[threadIdx.x] = n;
      for (int o = 128; o > 0; o >>= 1) {
        __syncthreads();
        if ((int)threadIdx.x < o) count[threadIdx.x] += count[threadIdx.x + o];
      }
      if (threadIdx.x == 0) {
        float f = 1.f;
        if (reduction != kNone && grad_loss != nullptr) f = *grad_loss;
        if (reduction == kMean) f /= (float)max(count[0], 1);
        if (count[0] == 0) f = 0.f;  // zeros, whatever grad_loss is
        *scale = f;
      }
      return;
    }
    const int64_t per_row = Hp / E;
    for (int64_t i = block * 256 + threadIdx.x; i < N * per_row; i += blocks * 256) {
      const int64_t r = i / per_row, c = (i - r * per_row) * E;
      i32x4 v = {0, 0, 0, 0};
      if (target[r] != ignore) {
        const T* p = x + r * ldx + c;
        if (c + E <= H) {
          v = *reinterpret_cast<const i32x4_any*>(p);
        } else {
#pragma unroll
          for (int k = 0; k < E; ++k)
            if (c + k < H) {
              if constexpr (sizeof(T) == 4) v[k] = reinterpret_cast<const int*>(p)[k];
              else v[k / 2] |= (int)((uint32_t)p[k] << (16 * (k & 1)));
            }
        }
      }
      *reinterpret_cast<i32x4*>(xs + r * Hp + c) = v;
    }
    if (xt == nullptr) return;
    for (int64_t i = block * 256 + threadIdx.x; i < kFewRows * H; i += blocks * 256) {
      const int64_t r = i / H, h = i - r * H;
      xt[h * kFewRows + r] = r < N && target[r] != ignore ? x[r * ldx + h] : T{0};
    }
  }
};

template <typename T>
__global__ __launch_bounds__(256) void ce_prepare_kernel(CePrepare<T> a) {
  __shared__ int count[256];
  a.run(blockIdx.x, gridDim.x, count);
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// fp32 logits: (m, sum of exp(l - m)) of each group of kGroup32 columns (grid
// y < groups) of each row (grid x), and the target's logit; the workgroups from
// grid y = groups on prepare the gradients' operands.
constexpr int kGroup32 = 4096;

__global__ __launch_bounds__(256) void ce_stats_kernel(const float* __restrict__ l, int64_t ldl, int64_t V,
                                                       const int64_t* __restrict__ target, f32x2* __restrict__ stat,
                                                       int groups, float* __restrict__ tlogit,
                                                       CePrepare<float> prepare) {
  __shared__ float red[2][4];
  if ((int)blockIdx.y >= groups) {
    __shared__ int count[256];
    prepare.run((int64_t)((int)blockIdx.y - groups) * gridDim.x + blockIdx.x,
                (int64_t)((int)gridDim.y - groups) * gridDim.x, count);
    return;
  }
  const int64_t r = blockIdx.x;
  const int64_t v0 = (int64_t)blockIdx.y * kGroup32;
  const float* row = l + r * ldl;
  const int64_t want = target[r];
  f32x4 w[4];
  float m = -FLT_MAX;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int64_t v = v0 + 4 * (threadIdx.x + 256 * q);
    w[q] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    if (v < V) w[q] = *reinterpret_cast<const f32x4*>(row + v);  // ldl is a multiple of 4
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (v + c >= V) w[q][c] = -INFINITY;  // adds exp(-inf) = 0
      if (v + c < V && v + c == want) tlogit[r] = w[q][c];
      m = fmaxf(m, w[q][c]);
    }
  }
  m = wave_max(m);
  if ((threadIdx.x & 63) == 0) red[0][threadIdx.x >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  float s = 0.f;
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int c = 0; c < 4; ++c) s += __expf(w[q][c] - m);
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) red[1][threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0)
    stat[r * groups + blockIdx.y] = f32x2{m, (red[1][0] + red[1][1]) + (red[1][2] + red[1][3])};
}

// One row (grid x) of a chunk: lse from its groups, the loss, and, where p is
// set, d in place of what the row holds (grid y workgroups share a row).
//   T = u16: exp(l - m) 2^15 in fp16 -> d in bf16, without the scalar factor.
//   T = float: l -> d, with it.
struct CeRows {
  void* p;
  int64_t ldp, V, R;
  const f32x2* stat;
  int groups, stride, group_shift;  // groups of a row, from one row's to the next, columns of one: 2^group_shift
  const int64_t* target;
  int64_t ignore;
  const float* tlogit;
  float* loss;             // [row]
  const float* row_grad;   // per-row gradients of the losses, or NULL
  const float* scale;      // (T = float)
};

// ROWS = 4: a wave a row, no barriers, for short rows.  The workgroups from grid
// y = `share` on prepare the operands of the gradients instead (bf16), where the
// logits' product did not need them (one launch less, 3 us).
template <typename T, int ROWS>
__global__ __launch_bounds__(256) void ce_rows_kernel(CeRows a, int share, CePrepare<T> prepare) {
  constexpr int NT = 256 / ROWS;  // threads of a row
  static_assert(ROWS == 1 || NT == 64, "a row is a workgroup's or a wave's");
  __shared__ float red[2][4];
  if ((int)blockIdx.y >= share) {
    __shared__ int count[256];
    prepare.run((int64_t)((int)blockIdx.y - share) * gridDim.x + blockIdx.x, (int64_t)((int)gridDim.y - share) * gridDim.x,
                count);
    return;
  }
  const int64_t r = ROWS == 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * ROWS + (threadIdx.x >> 6);
  if (ROWS > 1 && r >= a.R) return;
  const int tid = threadIdx.x % NT;
  const int64_t want = a.target[r];
  const bool ignored = want == a.ignore, bad = !ignored && (want < 0 || want >= a.V);
  constexpr int E = sizeof(T) == 2 ? 8 : 4;
  T* row = static_cast<T*>(a.p) + r * a.ldp;
  if (ignored) {
    if (a.loss != nullptr && blockIdx.y == 0 && tid == 0) a.loss[r] = 0.f;
    if (a.p == nullptr) return;
    for (int64_t v = E * ((int64_t)blockIdx.y * NT + tid); v < a.ldp; v += E * NT * (int64_t)share)
      *reinterpret_cast<i32x4*>(row + v) = i32x4{0, 0, 0, 0};
    return;
  }
  const f32x2* stat = a.stat + r * a.stride;
  float m = -FLT_MAX;
  for (int g = tid; g < a.groups; g += NT) m = fmaxf(m, stat[g].x);
  m = wave_max(m);
  if constexpr (ROWS == 1) {
    if ((tid & 63) == 0) red[0][tid >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  }
  float s = 0.f;
  for (int g = tid; g < a.groups; g += NT) s += stat[g].y * __expf(stat[g].x - m);
  s = wave_sum(s);
  if constexpr (ROWS == 1) {
    if ((tid & 63) == 0) red[1][tid >> 6] = s;
    __syncthreads();
    s = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  }
  const float lse = m + logf(s);
  const float tl = bad ? NAN : a.tlogit[r];  // a target that is no class: NaN, in loss and gradients
  if (a.loss != nullptr && blockIdx.y == 0 && tid == 0) a.loss[r] = lse - tl;
  if (a.p == nullptr) return;
  float g = a.row_grad != nullptr ? a.row_grad[r] : 1.f;
  if (sizeof(T) == 4) g *= *a.scale;
  if (bad) g = NAN;
  const float at_target = expm1f(tl - lse) * g;
  for (int64_t v = E * ((int64_t)blockIdx.y * NT + tid); v < a.ldp; v += E * NT * (int64_t)share) {
    float d[E];
    if constexpr (sizeof(T) == 2) {
      const f16x8 e = *reinterpret_cast<const f16x8*>(row + v);
      const float f = __expf(stat[min(v, a.V - 1) >> a.group_shift].x - lse) * (1.f / kScale16);
#pragma unroll
      for (int c = 0; c < E; ++c) d[c] = (float)e[c] * f * g;  // zeros from V on
    } else {
      const f32x4 l = *reinterpret_cast<const f32x4*>(row + v);
#pragma unroll
      for (int c = 0; c < E; ++c) d[c] = v + c < a.V ? __expf(l[c] - lse) * g : 0.f;
    }
    if ((uint64_t)(want - v) < (uint64_t)E) {
#pragma unroll
      for (int c = 0; c < E; ++c) d[c] = v + c == want ? at_target : d[c];
    }
    i32x4 o;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int c = 0; c < 4; ++c) o[c] = (int)(bf16_bits(d[2 * c]) | (uint32_t)bf16_bits(d[2 * c + 1]) << 16);
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) o[c] = __float_as_int(d[c]);
    }
    *reinterpret_cast<i32x4*>(row + v) = o;
  }
}

// The K splits of a gradient, added in order: out = bf16(scale sum), or acc =
// sum, in both cases onto acc where `add` is set.
struct CeJoin {
  const float* part;  // [splits][rows][ld]
  int splits, lanes;  // lanes: threads that share the splits of a result; splits 0: nothing to join
  int64_t rows, cols, ld;
  u16* out;  // [rows][cols]
  float* acc;
  bool add;
  const float* scale;
  const int64_t* target;  // as CeGrad's
  int64_t ignore;

  // Workgroup `block` of `blocks`: each thread every lanes-th split, then those
  // sums in order.
  __device__ void run(int64_t block, int64_t blocks, f32x4* share) const {
    const int64_t per_row = ld / 4, stride = rows * ld;
    const int per = 256 / lanes, mine = (int)threadIdx.x % per, lane = (int)threadIdx.x / per;
    const float f = out != nullptr ? *scale : 1.f;
    for (int64_t i0 = block * per; i0 < rows * per_row; i0 += blocks * per) {
      const int64_t i = i0 + mine;
      const bool live = i < rows * per_row;
      const int64_t r = live ? i / per_row : 0, c = 4 * (i - r * per_row);
      const bool skip = target != nullptr && target[r] == ignore;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
      if (live) {
        const float* p = part + 4 * i;
#pragma unroll 4
        for (int k = lane; k < splits; k += lanes) v += *reinterpret_cast<const f32x4*>(p + k * stride);
      }
      if (lanes > 1) {
        __syncthreads();
        share[threadIdx.x] = v;
        __syncthreads();
        for (int k = 1; k < lanes && lane == 0; ++k) v += share[k * per + mine];
      }
      if (!live || lane != 0) continue;
      f32x4* to = reinterpret_cast<f32x4*>(acc + 4 * i);
      if (add) v += *to;
      if (out == nullptr) {
        *to = v;
        continue;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (c + k < cols) out[r * cols + c + k] = skip ? (u16)0 : bf16_bits(v[k] * f);
    }
  }
};

// The sum or mean of the rows' losses by one workgroup, in 64 bits and a fixed
// order.
struct CeLoss {
  float* loss;  // NULL: not wanted, or not yet
  const float* row_loss;
  const int64_t* target;
  int64_t N, ignore;
  int reduction;

  __device__ void run(double* sum, int* count) const {
    double s = 0;
    int n = 0;
#pragma unroll 8
    for (int64_t i = threadIdx.x; i < N; i += 256) {
      s += (double)row_loss[i];
      n += target[i] != ignore;
    }
    sum[threadIdx.x] = s;
    count[threadIdx.x] = n;
    for (int o = 128; o > 0; o >>= 1) {
      __syncthreads();
      if ((int)threadIdx.x < o) {
        sum[threadIdx.x] += sum[threadIdx.x + o];
        count[threadIdx.x] += count[threadIdx.x + o];
      }
    }
    if (threadIdx.x == 0) *loss = (float)(reduction == kMean ? sum[0] / (double)max(count[0], 1) : sum[0]);
  }
};

// What is left after a gradient's product: its join by the first `join_blocks`
// workgroups, and the loss by one more.
struct CeFinish {
  CeJoin join;
  CeLoss loss;
  int join_blocks;

  int blocks() const { return join_blocks + (loss.loss != nullptr ? 1 : 0); }
  __device__ void run(int64_t block) const {
    __shared__ f32x4 share[256];  // (also the losses' sums, 12 bytes a thread)
    if (block < join_blocks) join.run(block, join_blocks, share);
    else if (block == join_blocks && loss.loss != nullptr)
      loss.run(reinterpret_cast<double*>(share), reinterpret_cast<int*>(share) + 512);
  }
};

__global__ __launch_bounds__(256) void ce_finish_kernel(CeFinish a) { a.run(blockIdx.x); }

// dW [V, H] of up to 32 rows: one k-slice of a 16x16x32 MFMA, so no tile is
// worth staging; the kernel is bound by writing dW.  A wave keeps the x
// operand of its 128 columns of h (grid x) in registers, 16 bytes a lane from
// the transposed x, and walks over tiles of 16 vocabulary entries.  Row i of
// the MFMA's output is column 8 (i / 4) + 4 t + i % 4 of a block of 32, for the
// two MFMAs t = 0, 1 of the block: a lane's 4 + 4 results are then 8
// consecutive h, one 16-byte store, and the four lanes of an entry write 64
// bytes.  The workgroups from grid y = `ys` on join dx and the loss.
__global__ __launch_bounds__(256) void ce_few_rows_kernel(const u16* __restrict__ d, int64_t ldd,
                                                          const u16* __restrict__ xt, u16* __restrict__ dw, int R,
                                                          int H, int V, const float* __restrict__ scale, int ys,
                                                          CeFinish finish) {
  if ((int)blockIdx.y >= ys) {
    finish.run((int64_t)((int)blockIdx.y - ys) * gridDim.x + blockIdx.x);
    return;
  }
  typedef u16 u16x8 __attribute__((ext_vector_type(8)));
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int i = lane & 15, g = lane >> 4;  // MFMA row or column; k group, and group of output rows
  const int h0 = blockIdx.x * 128;
  const float f = *scale;
  bf16x8 a[4][2];
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int h = min(h0 + 32 * b + 8 * (i >> 2) + 4 * t + (i & 3), H - 1);  // past H: not stored
      a[b][t] = *reinterpret_cast<const bf16x8*>(xt + (int64_t)h * kFewRows + 8 * g);
    }
  auto load = [&](int v0) {  // rows of d are padded past V
    u16x8 v;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const u16 t = d[(int64_t)min(8 * g + k, R - 1) * ldd + v0 + i];
      v[k] = 8 * g + k < R ? t : (u16)0;
    }
    return __builtin_bit_cast(bf16x8, v);
  };
  const int step = 64 * ys;
  int v0 = 16 * (4 * (int)blockIdx.y + wave);
  if (v0 >= V) return;
  bf16x8 next = load(v0);
  for (; v0 < V; v0 += step) {
    const bf16x8 b8 = next;
    if (v0 + step < V) next = load(v0 + step);
    const int v = v0 + i;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const f32x4 lo = mfma16x16x32bf16(a[b][0], b8, f32x4{0.f, 0.f, 0.f, 0.f});
      const f32x4 hi = mfma16x16x32bf16(a[b][1], b8, f32x4{0.f, 0.f, 0.f, 0.f});
      const int h = h0 + 32 * b + 8 * g;
      u16* o = dw + (int64_t)v * H + h;
      u16 w[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = bf16_bits(lo[k] * f), w[4 + k] = bf16_bits(hi[k] * f);
      if (v < V && h + 8 <= H) {
        typedef i32x4 __attribute__((aligned(2))) i32x4_any;
        *reinterpret_cast<i32x4_any*>(o) =
            i32x4{(int)(w[0] | (uint32_t)w[1] << 16), (int)(w[2] | (uint32_t)w[3] << 16),
                  (int)(w[4] | (uint32_t)w[5] << 16), (int)(w[6] | (uint32_t)w[7] << 16)};
      } else if (v < V) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (h + k < H) o[k] = w[k];
      }
    }
  }
}

// acc += part, or acc = part.
__global__ __launch_bounds__(256) void ce_add_kernel(float* __restrict__ acc, const float* __restrict__ part,
                                                     int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) acc[i] += part[i];
}

// A gradient of no rows.
__global__ __launch_bounds__(256) void ce_zero_kernel(unsigned char* __restrict__ p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = 0;
}

// ---------------------------------------------------------------------------
// The bf16 products
// ---------------------------------------------------------------------------

// Output tiles: 256 x 256 and 128 x 128 (8 waves, one workgroup a CU), 128 x
// 64 (4 waves, two a CU).
enum CeTile { kT256, kT128, kT64 };

// How a product runs: K in `splits`, its long extent (the vocabulary) up to
// `main` in tiles of one kind and the rest, unsplit, in smaller ones: at 3.06
// turns of tiles over the chip the last 16 of 784 took a turn of their own.
struct CeProduct {
  CeTile tile;
  int splits;
  int64_t main;
  CeTile tail;
};

struct TileCost {
  int bm, bn, per_cu;
  double step, fixed;  // us of a 64-deep K step, and of a tile beside them
};
constexpr TileCost kTiles[] = {{256, 256, 1, 1.5, 9.0}, {128, 128, 1, 0.5, 6.0}, {128, 64, 2, 0.75, 5.0}};

int64_t tiles_of(CeTile t, int64_t M, int64_t N) { return cdiv(M, kTiles[t].bm) * cdiv(N, kTiles[t].bn); }

// Estimated us, from what the tiles measured: turns over the chip, and for a
// split K the fp32 sums written by the tiles (20 KB/us a CU) and joined.
double product_cost(CeTile t, int64_t splits, int64_t M, int64_t N, int64_t K) {
  const TileCost& c = kTiles[t];
  const int64_t cus = device_cus();
  const double steps = (double)cdiv(cdiv(K, 64), splits);
  double one = steps * c.step + c.fixed, join = 0;
  if (splits > 1) {
    one += c.bm * c.bn * 4 * c.per_cu / 20e3;
    join = 5 + (double)splits * M * N * 4 / 4e6;
  }
  return (double)cdiv(tiles_of(t, M, N) * splits, c.per_cu * cus) * one + join;
}

// The cheapest way for an M x N output; `long_m`, `long_n`: which extent may be
// cut in two (then K is not split).
CeProduct choose(int64_t M, int64_t N, int64_t K, bool can_split, bool long_m, bool long_n) {
  const int64_t cus = device_cus(), extent = long_m ? M : N;
  CeProduct best{kT256, 1, extent, kT128};
  double least = 1e30;
  auto offer = [&](const CeProduct& p, double cost) {
    if (cost < least) least = cost, best = p;
  };
  for (const CeTile t : {kT256, kT128, kT64}) {
    const int64_t most = can_split ? std::min<int64_t>(64, std::max<int64_t>(1, cdiv(K, 64) / 4)) : 1;
    for (int64_t s = 1; s <= most; ++s) {
      if (s > 1 && tiles_of(t, M, N) * s > 2 * kTiles[t].per_cu * cus) break;
      offer(CeProduct{t, (int)s, extent, t}, product_cost(t, s, M, N, K));
    }
    if (t == kT64 || !(long_m || long_n)) continue;
    // Whole turns of these tiles, the rest in the next smaller ones.
    const int64_t across = long_m ? cdiv(N, kTiles[t].bn) : cdiv(M, kTiles[t].bm);
    const int64_t turns = tiles_of(t, M, N) / cus, b = long_m ? kTiles[t].bm : kTiles[t].bn;
    const int64_t main = turns * cus / across * b;
    if (main <= 0 || main >= extent) continue;
    const CeTile small = t == kT256 ? kT128 : kT64;
    const double cost = long_m ? product_cost(t, 1, main, N, K) + product_cost(small, 1, M - main, N, K)
                               : product_cost(t, 1, M, main, K) + product_cost(small, 1, M, N - main, K);
    offer(CeProduct{t, 1, main, small}, cost + 2);
  }
  return best;
}

// Row length of fp32 sums of M: the lanes' 64-byte pieces are whole sectors.
int64_t sum_ld(int64_t M) { return cdiv(M, 16) * 16; }

// The splits' fp32 sums of an N x M gradient.
size_t split_workspace(const CeProduct& c, int64_t M, int64_t N) {
  return c.splits > 1 ? (size_t)(c.splits * N * sum_ld(M)) * sizeof(float) : 0;
}

struct Operands {
  const u16 *a, *b;
  int64_t lda, ldb;
  int64_t M, N, K;
};

template <int BM, int BN, int NBUF, int WM, int WN, KMask KM, bool CA, bool CB, int MF, class Epi>
hipError_t run_tile(const Operands& o, const Epi& epi, int splits, hipStream_t stream) {
  using P = LdsGemm<BM, BN, 64, NBUF, WM, WN, CA, CB, MF>;
  const int64_t tiles = cdiv(o.M, BM) * cdiv(o.N, BN);
  const SplitGeom g = gemm_split_geom(o.K, 64, splits);
  auto kern = gemm_bf16_lds_kernel<BM, BN, 64, NBUF, WM, WN, KM, CA, CB, MF, Epi>;
  hipLaunchKernelGGL(kern, dim3((unsigned)tiles, (unsigned)g.splits), dim3(P::NT), 0, stream, o.a, o.b, epi, (int)o.M,
                     (int)o.N, (int)o.K, o.lda, o.ldb, 4, device_xcds(), (int)g.steps, nullptr, nullptr);
  return hipGetLastError();
}

template <KMask KM, bool CA, bool CB, class Epi>
hipError_t run_product(const Operands& o, const Epi& epi, CeTile tile, int splits, hipStream_t stream) {
  if (tile == kT256) return run_tile<256, 256, 2, 2, 4, KM, CA, CB, 16>(o, epi, splits, stream);
  if (tile == kT128) return run_tile<128, 128, 4, 2, 4, KM, CA, CB, 16>(o, epi, splits, stream);
  return run_tile<128, 64, 3, 2, 2, KM, CA, CB, 16>(o, epi, splits, stream);
}

// ---------------------------------------------------------------------------
// Plan: chunking and where everything lies in the workspace
// ---------------------------------------------------------------------------

constexpr int64_t kChunkBytes = int64_t(2) << 30;  // of the values kept for the gradients
constexpr int64_t kMaxChunkRows = int64_t(1) << 22;  // a workgroup a row: within the grid's 2^32 threads
constexpr int64_t kMaxVocab = (int64_t(1) << 22) - 64;

struct CeArgs {
  const void *x, *w;
  const int64_t* target;
  float* loss;
  const float* grad_loss;
  void *dx, *dw;
  int64_t N, H, V, ldx, ldw;
  int dtype, reduction;
  int64_t ignore;
  bool grad;
  int64_t chunk_rows;
  const int32_t* configs;  // fp32: variant and split of each product, or NULL
};

struct CePlan {
  int64_t R, chunks;     // rows of a chunk
  int64_t Vp, Hp;        // padded row lengths of the kept values, of xs and wp
  bool pad;              // bf16: operands copied with padded rows
  bool copy_first;       // the logits' product needs xs too
  bool few;              // bf16: dW by ce_few_rows_kernel
  int groups, shift;
  CeProduct p1, p2, p3;  // bf16
  size_t stat, tlogit, rows, scale, xs, xt, wp, keep, acc, split;  // offsets
  size_t split_bytes, bytes, counter_bytes;
};

// The variant and K split of a product (0: logits, 1: dx, 2: dW) of a chunk of
// R rows: the caller's for whole chunks, the library's rule for a shorter last.
struct Config {
  int32_t variant, split;
};
Config config_of(const CeArgs& a, const CePlan& p, int which, int64_t R) {
  if (a.configs == nullptr || R != p.R) return {TILEC_VARIANT_AUTO, 0};
  return {a.configs[2 * which], a.configs[2 * which + 1]};
}

// Where a configuration is refused, the product's own call says so.
size_t matmul_scratch(const CeArgs& a, Config c, int64_t M, int64_t N, int64_t K, int64_t ld1, int64_t ld2, int layout,
                      size_t* counters) {
  size_t ws = 0, cnt = 0;
  if (tilec_matmul_scratch_bytes(M, N, K, ld1, ld2, layout, a.dtype, c.variant, c.split, &ws, &cnt) != TILEC_OK)
    return 0;
  *counters = std::max(*counters, cnt);
  return ws;
}

CePlan make_plan(const CeArgs& a) {
  CePlan p{};
  const bool bf16 = a.dtype == TILEC_BF16;
  const int64_t esz = bf16 ? 2 : 4;
  p.Vp = bf16 ? cdiv(a.V, 64) * 64 : cdiv(a.V, 4) * 4;
  // bf16 losses keep nothing but their groups' sums; fp32 losses go through
  // the chunk's logits.
  const int64_t row_bytes = p.Vp * (a.grad || !bf16 ? esz : 1);
  p.R = std::max<int64_t>(256, kChunkBytes / row_bytes / 256 * 256);
  if (a.chunk_rows > 0) p.R = a.chunk_rows;
  p.R = std::min({a.N, p.R, kMaxChunkRows});
  p.chunks = cdiv(a.N, p.R);
  p.Hp = cdiv(a.H, bf16 ? 64 : 4) * (bf16 ? 64 : 4);
  if (bf16) {
    auto fits = [&](const void* q, int64_t ld) {
      return reinterpret_cast<uintptr_t>(q) % 16 == 0 && ld % 8 == 0 && ld < (int64_t(1) << 22);
    };
    p.pad = a.H % 8 != 0 || !fits(a.w, a.ldw) || !fits(a.x, a.ldx);
    p.p1 = choose(a.V, p.R, a.H, false, true, false);
    p.p2 = choose(a.H, p.R, a.V, true, false, false);
    p.p3 = choose(a.H, a.V, p.R, true, false, true);
    p.shift = 6;
    // The largest tiles write groups past the vocabulary's end too.
    p.groups = (int)(cdiv(a.V, 256) * 4);
  } else {
    p.shift = 12;
    p.groups = (int)cdiv(a.V, kGroup32);
  }
  // Widths of no whole K steps: the largest tiles have no registers left to mask
  // both operands by (1000 x 1000 x 50021: 398 us with x copied, 404 in place);
  // the smaller ones save the copy's launch (640 x 928 x 978: 42.7, 40.3).
  p.copy_first = bf16 && (p.pad || (p.Hp != a.H && p.p1.tile == kT256));
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  p.stat = take((size_t)(p.R * p.groups) * sizeof(f32x2));
  p.tlogit = take((size_t)p.R * sizeof(float));
  p.rows = take(a.reduction == kNone ? 0 : (size_t)a.N * sizeof(float));
  p.scale = take(sizeof(float));
  p.xs = take(a.grad || p.copy_first ? (size_t)(p.R * p.Hp * esz) : 0);
  p.few = bf16 && a.grad && p.chunks == 1 && p.R <= kFewRows;
  p.xt = take(p.few ? (size_t)(a.H * kFewRows * 2) : 0);
  p.wp = take(p.pad ? (size_t)(a.V * p.Hp * esz) : 0);
  p.keep = take(a.grad || !bf16 ? (size_t)(p.R * p.Vp * esz) : 0);
  p.acc = take(a.grad && p.chunks > 1 ? (size_t)(a.V * sum_ld(a.H)) * sizeof(float) : 0);
  if (bf16) {
    if (a.grad) {
      p.split_bytes = std::max(split_workspace(p.p2, a.H, p.R), p.few ? 0 : split_workspace(p.p3, a.H, a.V));
    }
  } else {
    for (const int64_t R : {p.R, a.N - (p.chunks - 1) * p.R}) {
      auto more = [&](int which, int64_t M, int64_t N, int64_t K, int64_t ld1, int64_t ld2, int layout) {
        p.split_bytes = std::max(p.split_bytes, matmul_scratch(a, config_of(a, p, which, R), M, N, K, ld1, ld2, layout,
                                                               &p.counter_bytes));
      };
      more(0, R, a.V, a.H, a.ldx, a.ldw, TILEC_X2_COL_MAJOR);
      if (!a.grad) continue;
      more(1, R, a.H, a.V, p.Vp, a.ldw, 0);
      more(2, a.V, a.H, R, p.Vp, p.Hp, TILEC_X1_COL_MAJOR);
    }
  }
  p.split = take(p.split_bytes);
  p.bytes = at;
  return p;
}

unsigned grid_for(int64_t n) { return (unsigned)std::min<int64_t>(std::max<int64_t>(cdiv(n, 256), 1), 1 << 16); }

#define CE_TRY(call)                  \
  do {                                \
    const hipError_t e_ = (call);     \
    if (e_ != hipSuccess) return e_;  \
  } while (0)

// The kernels around the products of one chunk.
template <typename T>
CePrepare<T> prepare_of(const CeArgs& a, const CePlan& p, char* ws, int64_t r0, int64_t R) {
  CePrepare<T> q{};
  q.x = static_cast<const T*>(a.x) + r0 * a.ldx, q.ldx = a.ldx;
  q.xs = reinterpret_cast<T*>(ws + p.xs), q.xt = p.few ? reinterpret_cast<T*>(ws + p.xt) : nullptr;
  q.Hp = p.Hp, q.N = R, q.H = a.H, q.target = a.target + r0, q.ignore = a.ignore;
  q.scale = a.grad && r0 == 0 ? reinterpret_cast<float*>(ws + p.scale) : nullptr;
  q.all = a.N, q.all_targets = a.target, q.reduction = a.reduction, q.grad_loss = a.grad_loss;
  return q;
}
template <typename T>
unsigned prepare_blocks(const CeArgs& a, const CePlan& p, int64_t R) {
  return grid_for(std::max(R * p.Hp / (16 / (int64_t)sizeof(T)), p.few ? kFewRows * a.H : 0)) + 1;
}

// The same as rows of a grid `width` wide, where they run beside another kernel's: not
// more than fit into grid y with that kernel's own (each takes what is left over
// in steps).
constexpr unsigned kMoreBlocks = 1024;
constexpr int64_t kMaxGroups = 65535 - kMoreBlocks;
template <typename T>
unsigned more_blocks(const CeArgs& a, const CePlan& p, int64_t R, int64_t width) {
  if (!a.grad || p.copy_first) return 0;
  return (unsigned)std::min<int64_t>(std::max<int64_t>(cdiv(prepare_blocks<T>(a, p, R), width), width == 1 ? 2 : 1), kMoreBlocks);
}

template <typename T>
hipError_t run_prepare(const CeArgs& a, const CePlan& p, char* ws, int64_t r0, int64_t R, hipStream_t stream) {
  if (!p.copy_first) return hipSuccess;
  hipLaunchKernelGGL((ce_prepare_kernel<T>), dim3(prepare_blocks<T>(a, p, R)), dim3(256), 0, stream,
                     prepare_of<T>(a, p, ws, r0, R));
  return hipGetLastError();
}

template <typename T>
hipError_t run_rows(const CeArgs& a, const CePlan& p, char* ws, int64_t r0, int64_t R, hipStream_t stream) {
  CeRows q{};
  q.p = a.grad ? ws + p.keep : nullptr;
  q.ldp = p.Vp, q.V = a.V, q.R = R;
  q.stat = reinterpret_cast<const f32x2*>(ws + p.stat);
  q.groups = (int)cdiv(a.V, int64_t(1) << p.shift), q.stride = p.groups, q.group_shift = p.shift;
  q.target = a.target + r0, q.ignore = a.ignore;
  q.tlogit = reinterpret_cast<const float*>(ws + p.tlogit);
  q.loss = (a.reduction == kNone ? a.loss : reinterpret_cast<float*>(ws + p.rows)) + r0;
  q.row_grad = a.reduction == kNone && a.grad_loss != nullptr ? a.grad_loss + r0 : nullptr;
  q.scale = reinterpret_cast<const float*>(ws + p.scale);
  // Workgroups that share a row each join its groups again: only as many as
  // it takes to fill the chip.
  const int64_t want = cdiv(4 * (int64_t)device_cus(), R), most = cdiv(p.Vp, 256 * 16 / (int64_t)sizeof(T));
  const unsigned share = a.grad ? (unsigned)std::max<int64_t>(1, std::min(want, most)) : 1;
  // A wave a row where rows are short and many: 20000 rows x 128 x 1000 in 98 us
  // for all, 114 with a workgroup each; 1024 x 128 x 3000 would go from 40.1 to
  // 41.5.  (16-byte pieces of a row; groups are read twice.)
  const int64_t pieces = a.grad ? p.Vp * (int64_t)sizeof(T) / 16 : 2 * q.groups;
  const bool waves = pieces <= 512 && R >= 8 * (int64_t)device_cus();
  const int64_t width = waves ? cdiv(R, 4) : R;
  const unsigned more = sizeof(T) == 2 ? more_blocks<T>(a, p, R, width) : 0;  // (fp32: beside the statistics)
  const auto kern = waves ? ce_rows_kernel<T, 4> : ce_rows_kernel<T, 1>;
  hipLaunchKernelGGL(kern, dim3((unsigned)width, share + more), dim3(256), 0, stream, q, (int)share,
                     prepare_of<T>(a, p, ws, r0, R));
  return hipGetLastError();
}

// `last`: all rows are through.
CeFinish finish_of(const CeArgs& a, const CePlan& p, char* ws, const CeJoin& join, bool last) {
  CeFinish f{join, {}, 0};
  if (join.splits > 0) {
    f.join.lanes = join.splits >= 32 ? 8 : join.splits >= 8 ? 2 : 1;
    f.join_blocks = (int)grid_for(join.rows * join.ld / 4 * f.join.lanes);
  }
  if (last && a.reduction != kNone)
    f.loss = {a.loss, reinterpret_cast<const float*>(ws + p.rows), a.target, a.N, a.ignore, a.reduction};
  return f;
}

hipError_t run_finish(const CeFinish& f, hipStream_t stream) {
  if (f.blocks() == 0) return hipSuccess;
  hipLaunchKernelGGL(ce_finish_kernel, dim3((unsigned)f.blocks()), dim3(256), 0, stream, f);
  return hipGetLastError();
}

// One gradient: its product, in splits or not, and in `join` what joins them.
// `acc`: fp32 sums over the chunks (NULL: one chunk), written to `out` by the
// last.
template <bool CB>
hipError_t run_grad(const CeArgs& a, const CePlan& p, char* ws, const Operands& o, const CeProduct& c, u16* out,
                    float* acc, bool add, const int64_t* target, CeJoin* join, hipStream_t stream) {
  const float* scale = reinterpret_cast<const float*>(ws + p.scale);
  float* part = reinterpret_cast<float*>(ws + p.split);
  const int64_t ld = sum_ld(a.H);
  const int64_t splits = gemm_split_geom(o.K, 64, c.splits).splits;
  CeGrad g{out, a.H, acc, ld, 0, add, scale, target, a.ignore};
  if (splits > 1) g = CeGrad{nullptr, 0, part, ld, o.N * ld, false, nullptr, nullptr, 0};
  Operands main = o;
  if (c.main < o.N) {  // CB false: d's rows, N the vocabulary
    Operands rest = o;
    rest.N = o.N - c.main;
    rest.b += c.main;
    CeGrad gr = g;
    if (gr.out != nullptr) gr.out += c.main * a.H;
    if (gr.acc32 != nullptr) gr.acc32 += c.main * ld;
    CE_TRY((run_product<kKRows, true, CB>(rest, gr, c.tail, 1, stream)));
    main.N = c.main;
  }
  CE_TRY((run_product<kKRows, true, CB>(main, g, c.tile, c.splits, stream)));
  if (splits > 1) *join = CeJoin{part, (int)splits, 1, o.N, a.H, ld, out, acc, add, scale, target, a.ignore};
  return hipSuccess;
}

hipError_t run_bf16(const CeArgs& a, const CePlan& p, char* ws, hipStream_t stream) {
  const u16 *x = static_cast<const u16*>(a.x), *w = static_cast<const u16*>(a.w);
  u16* xs = reinterpret_cast<u16*>(ws + p.xs);
  u16* keep = reinterpret_cast<u16*>(ws + p.keep);
  int64_t ldw = a.ldw;
  if (p.pad) {
    u16* wp = reinterpret_cast<u16*>(ws + p.wp);
    CE_TRY(pad_copy<2>(w, wp, a.V, a.H, a.ldw, a.V, p.Hp, w, wp, 0, 0, a.ldw, 0, 0, stream));
    w = wp, ldw = p.Hp;
  }
  for (int64_t c = 0; c < p.chunks; ++c) {
    const int64_t r0 = c * p.R, R = std::min(p.R, a.N - r0);
    const bool last = c + 1 == p.chunks;
    CE_TRY(run_prepare<u16>(a, p, ws, r0, R, stream));
    const u16* xc = p.copy_first ? xs : x + r0 * a.ldx;
    const int64_t ldx = p.copy_first ? p.Hp : a.ldx;
    CeLogits le{a.grad ? keep : nullptr,
                p.Vp,
                reinterpret_cast<f32x2*>(ws + p.stat),
                p.groups,
                0,
                a.target + r0,
                reinterpret_cast<float*>(ws + p.tlogit)};
    for (int64_t v0 = 0; v0 < a.V; v0 += p.p1.main) {
      const bool rest = v0 > 0;
      const int64_t V = rest ? a.V - v0 : p.p1.main;
      const CeTile tile = rest ? p.p1.tail : p.p1.tile;
      const Operands o{w + v0 * ldw, xc, ldw, ldx, V, R, p.pad ? p.Hp : a.H};
      le.v0 = (int)v0;
      if (o.K % 64 == 0) CE_TRY((run_product<kKFull, false, true>(o, le, tile, 1, stream)));
      else if (tile == kT256) CE_TRY((run_tile<256, 256, 2, 2, 4, kKColsA, false, true, 16>(o, le, 1, stream)));
      else if (tile == kT128) CE_TRY((run_tile<128, 128, 4, 2, 4, kKMasked, false, true, 16>(o, le, 1, stream)));
      else CE_TRY((run_tile<128, 64, 3, 2, 2, kKMasked, false, true, 16>(o, le, 1, stream)));
      if (rest) break;
    }
    CE_TRY(run_rows<u16>(a, p, ws, r0, R, stream));
    if (!a.grad) {
      if (last) CE_TRY(run_finish(finish_of(a, p, ws, {}, true), stream));
      continue;
    }
    // dx^T [H, R] = W^T d^T over the vocabulary, first, while d is in the caches
    // (1000 rows x 50021: 110 us, 130 after dW); d is padded with zeros to
    // whole K steps, W ends with its rows.
    CeJoin jx{}, jw{};
    CE_TRY(run_grad<true>(a, p, ws, Operands{w, keep, ldw, p.Vp, a.H, R, a.V}, p.p2,
                          static_cast<u16*>(a.dx) + r0 * a.H, nullptr, false, a.target + r0, &jx, stream));
    const CeFinish f = finish_of(a, p, ws, jx, last);
    // dW^T [H, V] = x^T d over the chunk's rows.  Its kernel of few rows joins
    // dx and the losses beside it (7 x 1024 x 32768: 52.5 -> 48.9 us for all);
    // a tile kernel's dW would evict the split sums (1000 x 1000 x 50021: 407
    // and 408 us).  (Calls in a row.)
    u16* dw = static_cast<u16*>(a.dw);
    if (p.few) {
      const unsigned gx = (unsigned)cdiv(a.H, 128);
      const unsigned gy = (unsigned)std::min<int64_t>(cdiv(a.V, 64), std::max<int64_t>(1, 4 * device_cus() / gx));
      hipLaunchKernelGGL(ce_few_rows_kernel, dim3(gx, gy + (unsigned)cdiv(f.blocks(), gx)), dim3(256), 0, stream, keep,
                         p.Vp, reinterpret_cast<const u16*>(ws + p.xt), dw, (int)R, (int)a.H, (int)a.V,
                         reinterpret_cast<const float*>(ws + p.scale), (int)gy, f);
      CE_TRY(hipGetLastError());
      continue;
    }
    CE_TRY(run_finish(f, stream));
    CE_TRY(run_grad<false>(a, p, ws, Operands{xs, keep, p.Hp, p.Vp, a.H, a.V, R}, p.p3, last ? dw : nullptr,
                           p.chunks > 1 ? reinterpret_cast<float*>(ws + p.acc) : nullptr, c > 0, nullptr, &jw, stream));
    CE_TRY(run_finish(finish_of(a, p, ws, jw, false), stream));
  }
  return hipSuccess;
}

int run_f32(const CeArgs& a, const CePlan& p, char* ws, unsigned* counters, size_t counter_bytes, hipStream_t stream,
            hipError_t* err) {
  const float *x = static_cast<const float*>(a.x), *w = static_cast<const float*>(a.w);
  float* xs = reinterpret_cast<float*>(ws + p.xs);
  float* keep = reinterpret_cast<float*>(ws + p.keep);
  float* part = reinterpret_cast<float*>(ws + p.acc);
  auto product = [&](int which, int64_t R, const float* x1, const float* x2, float* out, int64_t M, int64_t N,
                     int64_t K, int64_t ld1, int64_t ld2, int64_t ldo, int layout) {
    const Config c = config_of(a, p, which, R);
    return tilec_matmul(x1, x2, out, M, N, K, ld1, ld2, ldo, layout, TILEC_F32, c.variant, c.split, ws + p.split,
                        p.split_bytes, counters, counter_bytes, stream);
  };
  for (int64_t c = 0; c < p.chunks; ++c) {
    const int64_t r0 = c * p.R, R = std::min(p.R, a.N - r0);
    int rc = product(0, R, x + r0 * a.ldx, w, keep, R, a.V, a.H, a.ldx, a.ldw, p.Vp, TILEC_X2_COL_MAJOR);
    if (rc != TILEC_OK) return rc;
    hipLaunchKernelGGL(ce_stats_kernel, dim3((unsigned)R, (unsigned)p.groups + more_blocks<float>(a, p, R, R)), dim3(256), 0,
                       stream, keep, p.Vp, a.V, a.target + r0, reinterpret_cast<f32x2*>(ws + p.stat), p.groups,
                       reinterpret_cast<float*>(ws + p.tlogit), prepare_of<float>(a, p, ws, r0, R));
    if ((*err = hipGetLastError()) != hipSuccess) return TILEC_ERR_HIP;
    if ((*err = run_rows<float>(a, p, ws, r0, R, stream)) != hipSuccess) return TILEC_ERR_HIP;
    if (!a.grad) continue;
    rc = product(1, R, keep, w, static_cast<float*>(a.dx) + r0 * a.H, R, a.H, a.V, p.Vp, a.ldw, a.H, 0);
    if (rc != TILEC_OK) return rc;
    float* dw = static_cast<float*>(a.dw);
    rc = product(2, R, keep, xs, c == 0 ? dw : part, a.V, a.H, R, p.Vp, p.Hp, a.H, TILEC_X1_COL_MAJOR);
    if (rc != TILEC_OK) return rc;
    if (c == 0) continue;
    hipLaunchKernelGGL(ce_add_kernel, dim3(grid_for(a.V * a.H)), dim3(256), 0, stream, dw, part, a.V * a.H);
    if ((*err = hipGetLastError()) != hipSuccess) return TILEC_ERR_HIP;
  }
  if ((*err = run_finish(finish_of(a, p, ws, {}, true), stream)) != hipSuccess) return TILEC_ERR_HIP;
  return TILEC_OK;
}

int check(const CeArgs& a) {
  if (a.dtype != TILEC_F32 && a.dtype != TILEC_BF16)
    return fail(TILEC_ERR_TYPE, "tilec: linear cross entropy: unsupported dtype code %d (use float32 or bfloat16)",
                a.dtype);
  if (a.N < 0 || a.H < 1 || a.V < 1 || a.N > kMaxDim || a.H > kMaxDim || a.V > kMaxDim)
    return fail(TILEC_ERR_VALUE, "tilec: linear cross entropy: bad shape N=%lld H=%lld V=%lld", (long long)a.N,
                (long long)a.H, (long long)a.V);
  if (a.reduction < kNone || a.reduction > kMean)
    return fail(TILEC_ERR_VALUE, "tilec: linear cross entropy: unknown reduction %d", a.reduction);
  if (a.ldw < a.H || (a.N > 1 && a.ldx < a.H) || a.ldw > (int64_t(1) << 40) || a.ldx > (int64_t(1) << 40))
    return fail(TILEC_ERR_VALUE, "tilec: linear cross entropy: bad row strides ldx=%lld ldw=%lld for H=%lld",
                (long long)a.ldx, (long long)a.ldw, (long long)a.H);
  if (a.chunk_rows < 0)
    return fail(TILEC_ERR_VALUE, "tilec: linear cross entropy: chunk_rows=%lld < 0", (long long)a.chunk_rows);
  if (a.dtype == TILEC_BF16 && (a.V > kMaxVocab || a.H > kMaxVocab))
    return fail(TILEC_ERR_UNSUPPORTED, "tilec: linear cross entropy: bf16 takes V and H up to %lld (got %lld, %lld)",
                (long long)kMaxVocab, (long long)a.V, (long long)a.H);
  if (cdiv(a.V, kGroup32) > kMaxGroups)
    return fail(TILEC_ERR_UNSUPPORTED, "tilec: linear cross entropy: V=%lld is too large", (long long)a.V);
  return TILEC_OK;
}

}  // namespace

}  // namespace tilec

using namespace tilec;

extern "C" {

int tilec_linear_ce_scratch_bytes(const void* x, const void* weight, int64_t N, int64_t H, int64_t V, int64_t ldx,
                                  int64_t ldw, int32_t dtype, int32_t reduction, int32_t grad, int64_t chunk_rows,
                                  const int32_t* configs, size_t* workspace_bytes, size_t* counter_bytes,
                                  int64_t* rows_per_chunk) {
  clear_error();
  if (workspace_bytes) *workspace_bytes = 0;
  if (counter_bytes) *counter_bytes = 0;
  if (rows_per_chunk) *rows_per_chunk = 0;
  CeArgs a{};
  a.x = x, a.w = weight, a.N = N, a.H = H, a.V = V, a.ldx = ldx, a.ldw = ldw, a.dtype = dtype;
  a.reduction = reduction, a.grad = grad != 0, a.chunk_rows = chunk_rows, a.configs = configs;
  const int rc = check(a);
  if (rc != TILEC_OK || N == 0) return rc;
  const CePlan p = make_plan(a);
  clear_error();
  if (workspace_bytes) *workspace_bytes = p.bytes;
  if (counter_bytes) *counter_bytes = p.counter_bytes;
  if (rows_per_chunk) *rows_per_chunk = p.R;
  return TILEC_OK;
}

int tilec_linear_ce(const void* x, const void* weight, const int64_t* target, float* loss, const float* grad_loss,
                    void* dx, void* dweight, int64_t N, int64_t H, int64_t V, int64_t ldx, int64_t ldw, int32_t dtype,
                    int32_t reduction, int64_t ignore_index, int32_t grad, int64_t chunk_rows, const int32_t* configs,
                    void* workspace, size_t workspace_bytes, void* counters, size_t counter_bytes, void* stream_ptr) {
  clear_error();
  CeArgs a{};
  a.x = x, a.w = weight, a.target = target, a.loss = loss, a.grad_loss = grad_loss, a.dx = dx, a.dw = dweight;
  a.N = N, a.H = H, a.V = V, a.ldx = ldx, a.ldw = ldw, a.dtype = dtype, a.reduction = reduction;
  a.ignore = ignore_index, a.grad = grad != 0, a.chunk_rows = chunk_rows, a.configs = configs;
  int rc = check(a);
  if (rc != TILEC_OK) return rc;
  if (a.grad && dweight == nullptr) return fail(TILEC_ERR_VALUE, "tilec: linear cross entropy: dweight is NULL");
  if (loss == nullptr && (N > 0 || reduction != kNone))
    return fail(TILEC_ERR_VALUE, "tilec: linear cross entropy: loss is NULL");
  hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
  hipError_t e = hipSuccess;
  auto launched = [&](hipError_t err) {
    return err == hipSuccess ? (int)TILEC_OK
                             : fail(TILEC_ERR_HIP, "tilec: launching the linear cross entropy failed: %s",
                                    hipGetErrorString(err));
  };
  if (N > 0) {
    if (x == nullptr || weight == nullptr || target == nullptr || (a.grad && dx == nullptr))
      return fail(TILEC_ERR_VALUE, "tilec: linear cross entropy: x/weight/target/dx is NULL");
    const CePlan p = make_plan(a);
    clear_error();
    if (workspace == nullptr || workspace_bytes < p.bytes || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
      return fail(TILEC_ERR_WORKSPACE, "tilec: linear cross entropy needs %zu workspace bytes, 16-byte aligned (got %zu)",
                  p.bytes, workspace == nullptr ? (size_t)0 : workspace_bytes);
    if (p.counter_bytes > 0 && (counters == nullptr || counter_bytes < p.counter_bytes))
      return fail(TILEC_ERR_WORKSPACE, "tilec: linear cross entropy needs %zu bytes of counters (got %zu)",
                  p.counter_bytes, counters == nullptr ? (size_t)0 : counter_bytes);
    char* ws = static_cast<char*>(workspace);
    if (dtype == TILEC_BF16) {
      e = run_bf16(a, p, ws, stream);
    } else {
      rc = run_f32(a, p, ws, static_cast<unsigned*>(counters), counter_bytes, stream, &e);
      if (rc != TILEC_OK && e == hipSuccess) return rc;
    }
    return launched(e);
  }
  // No rows: a loss of 0 and a gradient of zeros.
  if (reduction != kNone) {
    hipLaunchKernelGGL(ce_zero_kernel, dim3(1), dim3(256), 0, stream, reinterpret_cast<unsigned char*>(loss),
                       (int64_t)sizeof(float));
    e = hipGetLastError();
  }
  if (e == hipSuccess && a.grad) {
    const int64_t n = V * H * (dtype == TILEC_BF16 ? 2 : 4);
    hipLaunchKernelGGL(ce_zero_kernel, dim3(grid_for(n)), dim3(256), 0, stream, static_cast<unsigned char*>(dweight), n);
    e = hipGetLastError();
  }
  return launched(e);
}

}  // extern "C"
