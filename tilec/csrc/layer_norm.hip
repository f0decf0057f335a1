// Layer norm over the rows of x [R, D], forward and backward:
//   mean = sum(x) / D          rstd = 1 / sqrt(sum((x - mean)^2) / D + eps)
//   xhat = (x - mean) rstd     y = xhat w + b
//   dx   = rstd (dy w - c1 - xhat c2),  c1 = sum(dy w) / D,  c2 = sum(dy w xhat) / D
//   dw   = sum over rows of dy xhat     db = sum over rows of dy
// x, y / dy and w / b are each fp32 or bf16; every sum, the statistics and dw
// and db are fp32, outputs are rounded once, at the store.
//
// Both passes are bound by HBM: forward reads x and writes y, backward reads
// x and dy and writes dx.  So each value is read once: a row is held in
// registers by the TPR threads that serve it (16-byte loads; a power of two
// of threads up to a wave, whole waves up to a 1024-thread workgroup) and both statistics are
// taken from there, the variance from the deviations themselves, not from a
// difference of sums; the deviations' own sum, what the rounded mean left
// out, corrects both (a row of equal values comes out as zeros).  Rows of any length, stride and element alignment take
// the same 16-byte loads at the element's own alignment; only a row's last,
// partial group is read by elements.
//
// The backward pass keeps each thread's columns fixed while its workgroup
// walks over rows, so the column sums dw and db stay in registers and leave
// once, as one partial per workgroup; a second kernel adds the partials in
// order (no atomics: the same bits every time).
#include <algorithm>

#include "abi.h"
#include "common.h"
#include "rows.h"
#include "zeros.h"
#include "../../include/tilec.h"

namespace tilec {

namespace {

// The row's statistics from its rounded mean and the sums of the deviations
// from that and of their squares; inv_d = 1 / D, whose rounding the deviations'
// sum makes up for in the mean.  (Divisions and a correctly rounded root instead, by
// every lane of every row: 35.5 us for 8192 x 4096 bf16, 34.9 so.)
__device__ __forceinline__ void finish_stats(float& mean, float& rstd, const float (&q)[2], float inv_d, float eps) {
  const float off = q[0] * inv_d;
  mean += off;
  const float var = fmaf(-off, off, q[1] * inv_d), v = (var < 0.f ? 0.f : var) + eps;  // a NaN stays one
  rstd = inv_root(v);
}

struct NormArgs {
  const void *x, *w, *b, *dy;
  void *y, *dx;
  float *mean, *rstd;  // forward: written where not NULL
  const float *mean_in, *rstd_in;
  float *dw, *db, *partial;  // backward: dw / db NULL where not wanted
  int64_t ldx, ldy, lddx;    // ldy: of y, or of dy
  int64_t R;
  int D, Dp;  // Dp: columns of a partial row
  int w_bf16, tpr;
  float eps, inv_d;
};

// NV groups of E values a thread: rows of up to tpr * NV * E values.
template <typename TX, typename TY, int NV, int NT>
__global__ __launch_bounds__(NT) void norm_kernel(NormArgs a) {
  constexpr int E = 16 / (int)sizeof(TX);
  __shared__ float red1[2][16][1], red2[2][16][2];
  int slot1 = 0, slot2 = 0;
  const int tpr = a.tpr, D = a.D;
  const int rpb = blockDim.x / tpr;
  const int sub = rpb == 1 ? threadIdx.x : threadIdx.x & (tpr - 1);
  float w[NV][E], b[NV][E];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    load_params<E>(a.w, a.w_bf16, E * (sub + i * tpr), D, 1.f, w[i]);
    load_params<E>(a.b, a.w_bf16, E * (sub + i * tpr), D, 0.f, b[i]);
  }
  for (int64_t r0 = (int64_t)blockIdx.x * rpb; r0 < a.R; r0 += (int64_t)gridDim.x * rpb) {
    const int64_t r = r0 + (rpb == 1 ? 0 : threadIdx.x / tpr);
    const bool live = r < a.R;  // rows past the end: read as the last one, not stored
    const TX* row = static_cast<const TX*>(a.x) + (live ? r : a.R - 1) * a.ldx;
    Group<TX, E> g[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) g[i].load(row, E * (sub + i * tpr), D);
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e) s[0] += g[i].get(e);
    row_sums(s, tpr, red1, slot1);
    float mean = s[0] * a.inv_d, rstd;
    float q[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float d = E * (sub + i * tpr) + e < D ? g[i].get(e) - mean : 0.f;
        q[0] += d;
        q[1] = fmaf(d, d, q[1]);
      }
    row_sums(q, tpr, red2, slot2);
    finish_stats(mean, rstd, q, a.inv_d, a.eps);
    if (!live) continue;
    if (sub == 0) {
      if (a.mean) a.mean[r] = mean;
      if (a.rstd) a.rstd[r] = rstd;
    }
    TY* out = static_cast<TY*>(a.y) + r * a.ldy;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = E * (sub + i * tpr);
      if (c >= D) continue;
      float y[E];
#pragma unroll
      for (int e = 0; e < E; ++e) y[e] = fmaf((g[i].get(e) - mean) * rstd, w[i][e], b[i][e]);
      store_group<TY, E>(out, c, D, y);
    }
  }
}

// Rows too long for the registers of one workgroup: read three times (the
// second and third from the caches where they fit).
template <typename TX, typename TY>
__global__ __launch_bounds__(1024) void norm_long_kernel(NormArgs a) {
  constexpr int E = 16 / (int)sizeof(TX);
  __shared__ float red1[2][16][1], red2[2][16][2];
  int slot1 = 0, slot2 = 0;
  const int D = a.D;
  for (int64_t r = blockIdx.x; r < a.R; r += gridDim.x) {
    const TX* row = static_cast<const TX*>(a.x) + r * a.ldx;
    float s[1] = {0.f};
    for (int64_t c = E * threadIdx.x; c < D; c += E * 1024) {
      Group<TX, E> g;
      g.load(row, (int)c, D);
#pragma unroll
      for (int e = 0; e < E; ++e) s[0] += g.get(e);
    }
    row_sums(s, 1024, red1, slot1);
    float mean = s[0] * a.inv_d, rstd;
    float q[2] = {0.f, 0.f};
    for (int64_t c = E * threadIdx.x; c < D; c += E * 1024) {
      Group<TX, E> g;
      g.load(row, (int)c, D);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float d = c + e < D ? g.get(e) - mean : 0.f;
        q[0] += d;
        q[1] = fmaf(d, d, q[1]);
      }
    }
    row_sums(q, 1024, red2, slot2);
    finish_stats(mean, rstd, q, a.inv_d, a.eps);
    if (threadIdx.x == 0) {
      if (a.mean) a.mean[r] = mean;
      if (a.rstd) a.rstd[r] = rstd;
    }
    TY* out = static_cast<TY*>(a.y) + r * a.ldy;
    for (int64_t c = E * threadIdx.x; c < D; c += E * 1024) {
      Group<TX, E> g;
      g.load(row, (int)c, D);
      float w[E], b[E], y[E];
      load_params<E>(a.w, a.w_bf16, (int)c, D, 1.f, w);
      load_params<E>(a.b, a.w_bf16, (int)c, D, 0.f, b);
#pragma unroll
      for (int e = 0; e < E; ++e) y[e] = fmaf((g.get(e) - mean) * rstd, w[e], b[e]);
      store_group<TY, E>(out, (int)c, D, y);
    }
  }
}

// Where a workgroup's column sums go: its row of the partials, or, when it is
// the only one, the outputs themselves.
template <int E>
__device__ __forceinline__ void store_sums(const NormArgs& a, int part, int parts, int c, const float (&dw)[E],
                                           const float (&db)[E]) {
  if (parts == 1) {
    if (a.dw) store_group<float, E>(a.dw, c, a.D, dw);
    if (a.db) store_group<float, E>(a.db, c, a.D, db);
  } else {
    if (a.dw) store_group<float, E>(a.partial + (int64_t)(2 * part) * a.Dp, c, a.Dp, dw);
    if (a.db) store_group<float, E>(a.partial + (int64_t)(2 * part + 1) * a.Dp, c, a.Dp, db);
  }
}

template <typename TX, typename TY, int NV, int NT>
__global__ __launch_bounds__(NT) void norm_grad_kernel(NormArgs a) {
  constexpr int E = 16 / (int)sizeof(TX);
  __shared__ float red[2][16][2];
  __shared__ float sums[NT == 256 ? 256 * E : 1];
  int slot = 0;
  const int tpr = a.tpr, D = a.D;
  const int rpb = blockDim.x / tpr;
  const int sub = rpb == 1 ? threadIdx.x : threadIdx.x & (tpr - 1);
  float w[NV][E], dw[NV][E], db[NV][E];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    load_params<E>(a.w, a.w_bf16, E * (sub + i * tpr), D, 1.f, w[i]);
#pragma unroll
    for (int e = 0; e < E; ++e) dw[i][e] = db[i][e] = 0.f;
  }
  for (int64_t r0 = (int64_t)blockIdx.x * rpb; r0 < a.R; r0 += (int64_t)gridDim.x * rpb) {
    const int64_t r = r0 + (rpb == 1 ? 0 : threadIdx.x / tpr);
    const bool live = r < a.R;
    const int64_t rr = live ? r : a.R - 1;
    const TX* row = static_cast<const TX*>(a.x) + rr * a.ldx;
    const TY* drow = static_cast<const TY*>(a.dy) + rr * a.ldy;
    Group<TX, E> x[NV];
    Group<TY, E> dy[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      x[i].load(row, E * (sub + i * tpr), D);
      dy[i].load(drow, E * (sub + i * tpr), D);
    }
    const float mean = a.mean_in[rr], rstd = a.rstd_in[rr];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e) {  // columns past D: dy = 0
        const float t = dy[i].get(e), h = (x[i].get(e) - mean) * rstd, u = t * w[i][e];
        s[0] += u;
        s[1] = fmaf(u, h, s[1]);
        if (live) {
          dw[i][e] = fmaf(t, h, dw[i][e]);
          db[i][e] += t;
        }
      }
    row_sums(s, tpr, red, slot);
    if (!live) continue;
    const float c1 = s[0] * a.inv_d, c2 = s[1] * a.inv_d;
    TY* out = static_cast<TY*>(a.dx) + r * a.lddx;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = E * (sub + i * tpr);
      if (c >= D) continue;
      float v[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float h = (x[i].get(e) - mean) * rstd;
        v[e] = rstd * (fmaf(dy[i].get(e), w[i][e], -c1) - h * c2);
      }
      store_group<TY, E>(out, c, D, v);
    }
  }
  if (!a.dw && !a.db) return;
  // The rows that ran side by side: within a wave by shuffles, then the waves
  // in order through LDS.  (Through LDS alone, by a row's 8 threads, it took 25
  // of the 28 us of a 20000 x 79 pass.)
  if constexpr (NT == 256) {
    if (rpb > 1) {
      for (int o = tpr; o < 64; o <<= 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int e = 0; e < E; ++e) {
            dw[i][e] += __shfl_xor(dw[i][e], o);
            db[i][e] += __shfl_xor(db[i][e], o);
          }
      }
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          __syncthreads();
#pragma unroll
          for (int e = 0; e < E; ++e) sums[e * 256 + threadIdx.x] = k ? db[i][e] : dw[i][e];
          __syncthreads();
          if ((int)threadIdx.x < tpr) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
              float t = sums[e * 256 + threadIdx.x];
              for (int at = 64; at < 256; at += 64) t += sums[e * 256 + at + threadIdx.x];
              (k ? db[i][e] : dw[i][e]) = t;
            }
          }
        }
    }
  }
  if ((int)threadIdx.x >= tpr) return;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = E * (sub + i * tpr);
    if (c < D) store_sums<E>(a, blockIdx.x, gridDim.x, c, dw[i], db[i]);
  }
}

// Long rows, first pass: c1 and c2 of every row.
template <typename TX, typename TY>
__global__ __launch_bounds__(1024) void norm_grad_rows_kernel(NormArgs a, float* __restrict__ c12) {
  constexpr int E = 16 / (int)sizeof(TX);
  __shared__ float red[2][16][2];
  int slot = 0;
  const int D = a.D;
  for (int64_t r = blockIdx.x; r < a.R; r += gridDim.x) {
    const TX* row = static_cast<const TX*>(a.x) + r * a.ldx;
    const TY* drow = static_cast<const TY*>(a.dy) + r * a.ldy;
    const float mean = a.mean_in[r], rstd = a.rstd_in[r];
    float s[2] = {0.f, 0.f};
    for (int64_t c = E * threadIdx.x; c < D; c += E * 1024) {
      Group<TX, E> x;
      Group<TY, E> dy;
      x.load(row, (int)c, D);
      dy.load(drow, (int)c, D);
      float w[E];
      load_params<E>(a.w, a.w_bf16, (int)c, D, 1.f, w);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float u = dy.get(e) * w[e];
        s[0] += u;
        s[1] = fmaf(u, (x.get(e) - mean) * rstd, s[1]);
      }
    }
    row_sums(s, 1024, red, slot);
    if (threadIdx.x == 0) {
      c12[2 * r] = s[0] * a.inv_d;
      c12[2 * r + 1] = s[1] * a.inv_d;
    }
  }
}

// Long rows, second pass: one group of columns a thread (grid x), every
// gridDim.y-th row: dx, and the workgroup's share of dw and db.
template <typename TX, typename TY>
__global__ __launch_bounds__(256) void norm_grad_cols_kernel(NormArgs a, const float* __restrict__ c12) {
  constexpr int E = 16 / (int)sizeof(TX);
  const int D = a.D;
  const int64_t c64 = E * ((int64_t)blockIdx.x * 256 + threadIdx.x);
  if (c64 >= D) return;
  const int c = (int)c64;
  float w[E], dw[E], db[E];
  load_params<E>(a.w, a.w_bf16, c, D, 1.f, w);
#pragma unroll
  for (int e = 0; e < E; ++e) dw[e] = db[e] = 0.f;
  for (int64_t r = blockIdx.y; r < a.R; r += gridDim.y) {
    Group<TX, E> x;
    Group<TY, E> dy;
    x.load(static_cast<const TX*>(a.x) + r * a.ldx, c, D);
    dy.load(static_cast<const TY*>(a.dy) + r * a.ldy, c, D);
    const float mean = a.mean_in[r], rstd = a.rstd_in[r], c1 = c12[2 * r], c2 = c12[2 * r + 1];
    float v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float t = dy.get(e), h = (x.get(e) - mean) * rstd;
      dw[e] = fmaf(t, h, dw[e]);
      db[e] += t;
      v[e] = rstd * (fmaf(t, w[e], -c1) - h * c2);
    }
    store_group<TY, E>(static_cast<TY*>(a.dx) + r * a.lddx, c, D, v);
  }
  if (a.dw || a.db) store_sums<E>(a, blockIdx.y, gridDim.y, c, dw, db);
}

// dw[c] and db[c]: the sums of `parts` partial rows, 16 columns a workgroup,
// 64 threads a column (every 64th row each, then those in order).
__global__ __launch_bounds__(1024) void norm_grad_sum_kernel(NormArgs a, int parts) {
  __shared__ float red[64][17];
  const int col = threadIdx.x & 15, g = threadIdx.x >> 4;
  const int blocks = (a.D + 15) / 16;
  const int which = (int)blockIdx.x >= blocks;  // 0: dw, 1: db
  float* out = which ? a.db : a.dw;
  if (out == nullptr) return;
  const int c = 16 * ((int)blockIdx.x - which * blocks) + col;
  float s = 0.f;
  if (c < a.D) {
    const float* p = a.partial + (int64_t)which * a.Dp + c;
#pragma unroll 8
    for (int k = g; k < parts; k += 64) s += p[(int64_t)(2 * k) * a.Dp];
  }
  red[g][col] = s;
  __syncthreads();
  // Each wave's first 16 threads take 4 rows of `red`, then one wave those 16.
  if (g < 16) {
    s = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) s += red[4 * g + k][col];
  }
  __syncthreads();
  if (g < 16) red[g][col] = s;
  __syncthreads();
  if (g == 0 && c < a.D) {
    s = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) s += red[k][col];
    out[c] = s;
  }
}

constexpr int kMaxGrid = 1 << 20;  // workgroups of the passes over long rows; their loops stride over the rest

// Waves a CU of the forward pass, whose workgroups walk over rows with their
// parameters in registers: read again for every row, from the caches, they made
// 8192 x 4096 bf16 35 us instead of 28, 4099 x 3001 fp32 22 instead of 20 (16,
// 24 and 32 waves: 28, 30 and 31 us).  As many whole workgroups as fit into
// them: rows of 576 to 960 threads (of many rows, fp32 from 8193 values on, bf16
// from 16385) have one a CU, 9 to 15 waves.
constexpr int kWaves = 16;

template <typename TX, typename TY>
hipError_t launch_norm(NormArgs a, hipStream_t stream) {
  constexpr int E = 16 / (int)sizeof(TX);
  const NormGeom g = norm_geom(a.R, a.D, E, 4);
  if (g.nv == 0) {
    const unsigned grid = (unsigned)std::min<int64_t>(a.R, kMaxGrid);
    hipLaunchKernelGGL((norm_long_kernel<TX, TY>), dim3(grid), dim3(1024), 0, stream, a);
    return hipGetLastError();
  }
  a.tpr = g.tpr;
  const int threads = g.nt;
  const dim3 grid((unsigned)std::min<int64_t>(cdiv(a.R, threads / g.tpr), kWaves * 64 / threads * (int64_t)device_cus())), block(threads);
  auto go = [&](auto nv, auto nt) {
    hipLaunchKernelGGL((norm_kernel<TX, TY, decltype(nv)::value, decltype(nt)::value>), grid, block, 0, stream, a);
    return hipGetLastError();
  };
  using std::integral_constant;
  auto by_nv = [&](auto nt) {
    return g.nv == 1   ? go(integral_constant<int, 1>{}, nt)
           : g.nv == 2 ? go(integral_constant<int, 2>{}, nt)
                       : go(integral_constant<int, 4>{}, nt);
  };
  return g.nt <= 256   ? by_nv(integral_constant<int, 256>{})
         : g.nt <= 512 ? by_nv(integral_constant<int, 512>{})
                       : by_nv(integral_constant<int, 1024>{});
}

// The backward pass holds 16 columns a thread: their two sums, w, x and dy.
struct GradGeom {
  NormGeom g;
  int64_t parts;  // partial rows of dw and db
  int64_t Dp;
  size_t partial_bytes, c12_bytes;
};

GradGeom grad_geom(int64_t R, int64_t D, int xsz) {
  const int e = 16 / xsz;
  GradGeom q{};
  q.g = norm_geom(R, D, e, 16 / e);
  q.Dp = cdiv(D, 8) * 8;
  if (q.g.nv > 0) {
    const int rpb = q.g.nt / q.g.tpr;
    // 8 waves a CU, and 12 for bf16, which has twice the arithmetic a byte:
    // fewer leave the memory idle, more write more partials (8192 x 4096, 1, 2,
    // 3 and 4 workgroups of 4 waves a CU: fp32 98, 83, 89, 92 us, bf16 74, 52,
    // 49, 53; 4096 x 8192, 1 and 2 of 8 waves: fp32 88 and 95, bf16 60 and 53).
    q.parts = std::min<int64_t>(cdiv(R, rpb), cdiv(xsz == 4 ? 8 : 12, q.g.nt / 64) * device_cus());
  } else {
    q.parts = std::min<int64_t>(R, std::max<int64_t>(1, cdiv(4 * (int64_t)device_cus(), cdiv(D, 256 * e))));
    q.c12_bytes = (size_t)(R * 2 * sizeof(float) + 15) / 16 * 16;
  }
  q.partial_bytes = q.parts > 1 ? (size_t)(q.parts * 2 * q.Dp) * sizeof(float) : 0;
  return q;
}

template <typename TX, typename TY>
hipError_t launch_norm_grad(NormArgs a, const GradGeom& q, float* c12, hipStream_t stream) {
  constexpr int E = 16 / (int)sizeof(TX);
  hipError_t e;
  if (a.R == 0) {
    e = a.dw ? enqueue_zeros(a.dw, 1, a.D, a.D, stream) : hipSuccess;
    return e == hipSuccess && a.db ? enqueue_zeros(a.db, 1, a.D, a.D, stream) : e;
  }
  if (q.g.nv == 0) {
    const unsigned grid = (unsigned)std::min<int64_t>(a.R, kMaxGrid);
    hipLaunchKernelGGL((norm_grad_rows_kernel<TX, TY>), dim3(grid), dim3(1024), 0, stream, a, c12);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((norm_grad_cols_kernel<TX, TY>),
                       dim3((unsigned)cdiv(a.D, 256 * E), (unsigned)q.parts), dim3(256), 0, stream, a, c12);
    e = hipGetLastError();
  } else {
    a.tpr = q.g.tpr;
    const dim3 grid((unsigned)q.parts), block(q.g.nt);
    auto go = [&](auto nv, auto nt) {
      hipLaunchKernelGGL((norm_grad_kernel<TX, TY, decltype(nv)::value, decltype(nt)::value>), grid, block, 0, stream,
                         a);
      return hipGetLastError();
    };
    using std::integral_constant;
    auto by_nv = [&](auto nt) {
      if constexpr (E == 4) {
        if (q.g.nv == 4) return go(integral_constant<int, 4>{}, nt);
      }
      return q.g.nv == 1 ? go(integral_constant<int, 1>{}, nt) : go(integral_constant<int, 2>{}, nt);
    };
    e = q.g.nt <= 256   ? by_nv(integral_constant<int, 256>{})
        : q.g.nt <= 512 ? by_nv(integral_constant<int, 512>{})
                        : by_nv(integral_constant<int, 1024>{});
  }
  if (e != hipSuccess || (!a.dw && !a.db) || q.parts == 1) return e;
  hipLaunchKernelGGL(norm_grad_sum_kernel, dim3((unsigned)(2 * cdiv(a.D, 16))), dim3(1024), 0, stream, a,
                     (int)q.parts);
  return hipGetLastError();
}

int check_norm(int64_t R, int64_t D, int32_t x_dtype, int32_t y_dtype, int32_t w_dtype) {
  for (int32_t t : {x_dtype, y_dtype, w_dtype})
    if (t != TILEC_F32 && t != TILEC_BF16)
      return fail(TILEC_ERR_TYPE, "tilec: layer norm: unsupported dtype code %d (use float32 or bfloat16)", t);
  if (R < 0 || D < 1 || R > kMaxDim || D > kMaxDim)
    return fail(TILEC_ERR_VALUE, "tilec: layer norm: bad shape R=%lld D=%lld", (long long)R, (long long)D);
  return TILEC_OK;
}

int check_rows(const char* what, const void* p, int64_t ld, int64_t R, int64_t D) {
  if (R == 0) return TILEC_OK;
  if (p == nullptr) return fail(TILEC_ERR_VALUE, "tilec: layer norm: %s is NULL", what);
  if (R > 1 && ld < D)
    return fail(TILEC_ERR_VALUE, "tilec: layer norm: the row stride of %s, %lld, is less than D=%lld", what,
                (long long)ld, (long long)D);
  if (ld > (int64_t(1) << 40))
    return fail(TILEC_ERR_VALUE, "tilec: layer norm: the row stride of %s, %lld, is too large", what, (long long)ld);
  return TILEC_OK;
}

// f of the element types of x and of y (or dy and dx).
template <typename F>
hipError_t by_types(int32_t x_dtype, int32_t y_dtype, F f) {
  if (x_dtype == TILEC_F32) return y_dtype == TILEC_F32 ? f(float{}, float{}) : f(float{}, u16{});
  return y_dtype == TILEC_F32 ? f(u16{}, float{}) : f(u16{}, u16{});
}

}  // namespace

}  // namespace tilec

using namespace tilec;

extern "C" {

int tilec_layer_norm(const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd, int64_t R,
                     int64_t D, int64_t ldx, int64_t ldy, int32_t x_dtype, int32_t y_dtype, int32_t w_dtype, float eps,
                     void* stream) {
  clear_error();
  int rc = check_norm(R, D, x_dtype, y_dtype, w_dtype);
  if (rc == TILEC_OK) rc = check_rows("x", x, ldx, R, D);
  if (rc == TILEC_OK) rc = check_rows("y", y, ldy, R, D);
  if (rc != TILEC_OK || R == 0) return rc;
  NormArgs a{};
  a.x = x, a.w = weight, a.b = bias, a.y = y, a.mean = mean, a.rstd = rstd;
  a.ldx = ldx, a.ldy = ldy, a.R = R, a.D = (int)D, a.w_bf16 = w_dtype == TILEC_BF16, a.eps = eps, a.inv_d = 1.f / (float)D;
  const hipError_t e = by_types(x_dtype, y_dtype, [&](auto tx, auto ty) {
    return launch_norm<decltype(tx), decltype(ty)>(a, static_cast<hipStream_t>(stream));
  });
  if (e != hipSuccess) return fail(TILEC_ERR_HIP, "tilec: launching the layer norm failed: %s", hipGetErrorString(e));
  return TILEC_OK;
}

size_t tilec_layer_norm_backward_workspace_bytes(int64_t R, int64_t D, int32_t x_dtype) {
  if (check_norm(R, D, x_dtype, x_dtype, x_dtype) != TILEC_OK) return 0;
  const GradGeom q = grad_geom(R, D, x_dtype == TILEC_F32 ? 4 : 2);
  return q.c12_bytes + q.partial_bytes;
}

int tilec_layer_norm_backward(const void* dy, const void* x, const float* mean, const float* rstd, const void* weight,
                              void* dx, float* dweight, float* dbias, int64_t R, int64_t D, int64_t lddy, int64_t ldx,
                              int64_t lddx, int32_t x_dtype, int32_t y_dtype, int32_t w_dtype, void* workspace,
                              size_t workspace_bytes, void* stream) {
  clear_error();
  int rc = check_norm(R, D, x_dtype, y_dtype, w_dtype);
  if (rc == TILEC_OK) rc = check_rows("dy", dy, lddy, R, D);
  if (rc == TILEC_OK) rc = check_rows("x", x, ldx, R, D);
  if (rc == TILEC_OK) rc = check_rows("dx", dx, lddx, R, D);
  if (rc != TILEC_OK) return rc;
  if (R > 0 && (mean == nullptr || rstd == nullptr))
    return fail(TILEC_ERR_VALUE, "tilec: layer norm: mean/rstd is NULL");
  const GradGeom q = grad_geom(R, D, x_dtype == TILEC_F32 ? 4 : 2);
  const size_t need = q.c12_bytes + q.partial_bytes;
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(TILEC_ERR_WORKSPACE, "tilec: layer norm's backward pass needs %zu workspace bytes (got %zu)", need,
                workspace == nullptr ? (size_t)0 : workspace_bytes);
  NormArgs a{};
  a.x = x, a.dy = dy, a.w = weight, a.dx = dx, a.mean_in = mean, a.rstd_in = rstd, a.dw = dweight, a.db = dbias;
  a.ldx = ldx, a.ldy = lddy, a.lddx = lddx, a.R = R, a.D = (int)D, a.Dp = (int)q.Dp;
  a.w_bf16 = w_dtype == TILEC_BF16, a.inv_d = 1.f / (float)D;
  a.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + q.c12_bytes);
  float* c12 = static_cast<float*>(workspace);
  const hipError_t e = by_types(x_dtype, y_dtype, [&](auto tx, auto ty) {
    return launch_norm_grad<decltype(tx), decltype(ty)>(a, q, c12, static_cast<hipStream_t>(stream));
  });
  if (e != hipSuccess)
    return fail(TILEC_ERR_HIP, "tilec: launching the layer norm's backward pass failed: %s", hipGetErrorString(e));
  return TILEC_OK;
}

}  // extern "C"
