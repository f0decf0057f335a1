// Root mean square norm over the rows of h = x + residual, forward and backward:
//   rstd = 1 / sqrt(sum(h^2) / D + eps)    hhat = h rstd     y = hhat w
//   dx   = rstd (dy w - hhat c) + dh,   c = sum(dy w hhat) / D
//   dw   = sum over rows of dy hhat
// with dh what h's other reader (the residual stream) gives back.  h is rounded to
// the residual's type before anything is computed from it, so that what the
// backward pass reads is what the forward pass normalised.  Every sum, rstd and dw
// are fp32; y and dx are rounded once, at the store.
//
// y may leave in 8 bits with a scale for every 128 values (fp8.h): a block's
// largest magnitude is a maximum over the 16 or 32 neighbouring threads that hold
// it, so the next product's operand costs no pass of its own.
//
// Both passes are bound by HBM: every value is read once, a row held in the
// registers of the threads that serve it, and the backward pass keeps each
// thread's columns fixed while its workgroup walks over rows, so that dw leaves
// once, a partial row per workgroup, added in order by a second kernel (no
// atomics: the same bits every time).  Where launches cost more than reading, some
// workgroups take dx's rows and others dw's columns, in one launch.
#include <algorithm>
#include <type_traits>

#include "abi.h"
#include "common.h"
#include "enqueue.h"
#include "fp8.h"
#include "rows.h"
#include "zeros.h"
#include "../../include/tilec.h"

namespace tilec {

namespace {

struct None {};  // the type of an absent operand

struct RmsArgs {
  const void *x, *res, *w, *dy, *dh;
  void *y, *h, *dx;
  float *y_scale, *rstd;  // forward; rstd written where not NULL
  const float* rstd_in;
  float *dw, *partial;    // backward: dw NULL where not wanted
  int64_t ldx, ldr, ldy, ldh, lddh, lddx;  // ldy: of y, or of dy; ldh: of h written; ldx: of h read
  int64_t s_row, s_group;  // strides of y's scales
  int64_t R;
  int D, Dp;  // Dp: columns of a partial row
  int y_type, w_bf16, tpr, groups;  // groups: scales of a row of y
  float eps, inv_d;
};

// A thread's values of a row: x, plus the residual, rounded to its type.
template <typename TX, typename TR, int E>
struct Sum {
  Group<TX, E> x;
  Group<std::conditional_t<std::is_same_v<TR, None>, float, TR>, E> r;
  __device__ __forceinline__ void load(const RmsArgs& a, int64_t row, int c) {
    x.load(static_cast<const TX*>(a.x) + row * a.ldx, c, a.D);
    if constexpr (!std::is_same_v<TR, None>) r.load(static_cast<const TR*>(a.res) + row * a.ldr, c, a.D);
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (std::is_same_v<TR, None>) return x.get(e);
    else if constexpr (sizeof(TR) == 4) return x.get(e) + r.get(e);
    else return __uint_as_float(to_bf16(x.get(e) + r.get(e)) << 16);
  }
};

// E values of y at columns c .. of a row, those below D; in 8 bits with the scale
// of the block, which 128 / E neighbouring threads hold.
template <int E>
__device__ __forceinline__ void store_y(const RmsArgs& a, int64_t r, int c, const float (&y)[E]) {
  if (a.y_type == TILEC_F32 || a.y_type == TILEC_BF16) {
    if (c >= a.D) return;
    if (a.y_type == TILEC_F32) store_group<float, E>(static_cast<float*>(a.y) + r * a.ldy, c, a.D, y);
    else store_group<u16, E>(static_cast<u16*>(a.y) + r * a.ldy, c, a.D, y);
    return;
  }
  const bool e5m2 = a.y_type == TILEC_F8E5M2;
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) top = max(top, c + e < a.D ? __float_as_uint(y[e]) & 0x7fffffffu : 0u);
#pragma unroll
  for (int o = 1; o < kGroup / E; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
  float scale, inverse;
  block_scale(top, fp8_largest(e5m2), scale, inverse);
  if (c >= a.ldy) return;
  uint32_t q[E / 4];
#pragma unroll
  for (int i = 0; i < E / 4; ++i) {
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = c + 4 * i + e < a.D ? y[4 * i + e] * inverse : 0.f;
    q[i] = to_fp8(v[0], v[1], v[2], v[3], e5m2);
  }
  if (c >= a.D && c / 16 != (a.D - 1) / 16) return;  // past the 16 bytes that the row ends in
  uint32_t* const out = reinterpret_cast<uint32_t*>(static_cast<unsigned char*>(a.y) + r * a.ldy + c);
#pragma unroll
  for (int i = 0; i < E / 4; ++i) out[i] = q[i];
  if (c % kGroup == 0) a.y_scale[r * a.s_row + c / kGroup * a.s_group] = scale;
}

template <typename TX, typename TR, int NV, int NT>
__global__ __launch_bounds__(NT) void rms_kernel(RmsArgs a) {
  constexpr int E = 16 / (int)sizeof(TX);
  __shared__ float red[2][16][1];
  int slot = 0;
  const int tpr = a.tpr, D = a.D;
  const int rpb = blockDim.x / tpr;
  const int sub = rpb == 1 ? threadIdx.x : threadIdx.x & (tpr - 1);
  float w[NV][E];
#pragma unroll
  for (int i = 0; i < NV; ++i) load_params<E>(a.w, a.w_bf16, E * (sub + i * tpr), D, 1.f, w[i]);
  for (int64_t r0 = (int64_t)blockIdx.x * rpb; r0 < a.R; r0 += (int64_t)gridDim.x * rpb) {
    const int64_t r = r0 + (rpb == 1 ? 0 : threadIdx.x / tpr);
    const bool live = r < a.R;  // rows past the end: read as the last one, not stored
    Sum<TX, TR, E> g[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) g[i].load(a, live ? r : a.R - 1, E * (sub + i * tpr));
    float h[NV][E], s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e) {  // zeros past D
        h[i][e] = g[i].get(e);
        s[0] = fmaf(h[i][e], h[i][e], s[0]);
      }
    row_sums(s, tpr, red, slot);
    const float rstd = inv_root(fmaf(s[0], a.inv_d, a.eps));
    if (!live) continue;
    if (sub == 0 && a.rstd) a.rstd[r] = rstd;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = E * (sub + i * tpr);
      if constexpr (!std::is_same_v<TR, None>) {
        if (c < D) store_group<TR, E>(static_cast<TR*>(a.h) + r * a.ldh, c, D, h[i]);
      }
      float y[E];
#pragma unroll
      for (int e = 0; e < E; ++e) y[e] = h[i][e] * rstd * w[i][e];
      store_y<E>(a, r, c, y);
    }
  }
}

// Rows too long for the registers of one workgroup: read twice (the second time
// from the caches where they fit).
template <typename TX, typename TR>
__global__ __launch_bounds__(1024) void rms_long_kernel(RmsArgs a) {
  constexpr int E = 16 / (int)sizeof(TX);
  __shared__ float red[2][16][1];
  int slot = 0;
  const int64_t end = (int64_t)a.groups * kGroup;  // whole blocks of 128
  for (int64_t r = blockIdx.x; r < a.R; r += gridDim.x) {
    float s[1] = {0.f};
    for (int64_t c = E * threadIdx.x; c < a.D; c += E * 1024) {
      Sum<TX, TR, E> g;
      g.load(a, r, (int)c);
#pragma unroll
      for (int e = 0; e < E; ++e) s[0] = fmaf(g.get(e), g.get(e), s[0]);
    }
    row_sums(s, 1024, red, slot);
    const float rstd = inv_root(fmaf(s[0], a.inv_d, a.eps));
    if (threadIdx.x == 0 && a.rstd) a.rstd[r] = rstd;
    for (int64_t c = E * threadIdx.x; c < end; c += E * 1024) {
      Sum<TX, TR, E> g;
      g.load(a, r, (int)c);
      float w[E], h[E], y[E];
      load_params<E>(a.w, a.w_bf16, (int)c, a.D, 1.f, w);
#pragma unroll
      for (int e = 0; e < E; ++e) h[e] = g.get(e), y[e] = h[e] * rstd * w[e];
      if constexpr (!std::is_same_v<TR, None>) {
        if (c < a.D) store_group<TR, E>(static_cast<TR*>(a.h) + r * a.ldh, (int)c, a.D, h);
      }
      store_y<E>(a, r, (int)c, y);
    }
  }
}

// E values of dh at column c of a row; zeros where there is none.
template <typename TD, int E>
struct Other {
  Group<std::conditional_t<std::is_same_v<TD, None>, float, TD>, E> g;
  __device__ __forceinline__ void load(const RmsArgs& a, int64_t row, int c) {
    if constexpr (!std::is_same_v<TD, None>) g.load(static_cast<const TD*>(a.dh) + row * a.lddh, c, a.D);
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (std::is_same_v<TD, None>) return 0.f;
    else return g.get(e);
  }
};
template <typename TY, typename TD>
using Dx = std::conditional_t<std::is_same_v<TD, None>, TY, TD>;

template <int E>
__device__ __forceinline__ void store_dw(const RmsArgs& a, int part, int parts, int c, const float (&dw)[E]) {
  if (parts == 1) store_group<float, E>(a.dw, c, a.D, dw);
  else store_group<float, E>(a.partial + (int64_t)part * a.Dp, c, a.Dp, dw);
}

// dx of the rows that workgroup `block` of `blocks` takes, and its share of dw where
// DW says so.
template <typename TX, typename TY, typename TD, bool DW, int NV, int E>
__device__ __forceinline__ void grad_rows(const RmsArgs& a, int block, int blocks, float (&dw)[NV][E]) {
  __shared__ float red[2][16][1];
  int slot = 0;
  const int tpr = a.tpr, D = a.D;
  const int rpb = blockDim.x / tpr;
  const int sub = rpb == 1 ? threadIdx.x : threadIdx.x % tpr;
  float w[NV][E];
#pragma unroll
  for (int i = 0; i < NV; ++i) load_params<E>(a.w, a.w_bf16, E * (sub + i * tpr), D, 1.f, w[i]);
  for (int64_t r0 = (int64_t)block * rpb; r0 < a.R; r0 += (int64_t)blocks * rpb) {
    const int64_t r = r0 + (rpb == 1 ? 0 : threadIdx.x / tpr);
    const bool live = r < a.R;
    const int64_t rr = live ? r : a.R - 1;
    Group<TX, E> x[NV];
    Group<TY, E> dy[NV];
    Other<TD, E> dh[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = E * (sub + i * tpr);
      x[i].load(static_cast<const TX*>(a.x) + rr * a.ldx, c, D);
      dy[i].load(static_cast<const TY*>(a.dy) + rr * a.ldy, c, D);
      dh[i].load(a, rr, c);
    }
    const float rstd = a.rstd_in[rr];
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float t = dy[i].get(e), h = x[i].get(e) * rstd;
        s[0] = fmaf(t * w[i][e], h, s[0]);
        if constexpr (DW) {
          if (live) dw[i][e] = fmaf(t, h, dw[i][e]);
        }
      }
    row_sums(s, tpr, red, slot);
    if (!live) continue;
    const float k = s[0] * a.inv_d;
    using TO = Dx<TY, TD>;
    TO* out = static_cast<TO*>(a.dx) + r * a.lddx;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = E * (sub + i * tpr);
      if (c >= D) continue;
      float v[E];
#pragma unroll
      for (int e = 0; e < E; ++e)
        v[e] = fmaf(rstd, dy[i].get(e) * w[i][e] - x[i].get(e) * rstd * k, dh[i].get(e));
      store_group<TO, E>(out, c, D, v);
    }
  }
}

template <typename TX, typename TY, typename TD, int NV, int NT>
__global__ __launch_bounds__(NT) void rms_grad_kernel(RmsArgs a) {
  constexpr int E = 16 / (int)sizeof(TX);
  __shared__ float sums[NT == 256 ? 256 * E : 1];
  const int tpr = a.tpr, D = a.D, rpb = blockDim.x / tpr;
  const int sub = rpb == 1 ? threadIdx.x : threadIdx.x & (tpr - 1);
  float dw[NV][E];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < E; ++e) dw[i][e] = 0.f;
  grad_rows<TX, TY, TD, true>(a, blockIdx.x, gridDim.x, dw);
  if (!a.dw) return;
  // The rows that ran side by side: within a wave by shuffles, then the waves
  // in order through LDS.
  if constexpr (NT == 256) {
    if (rpb > 1) {
      for (int o = tpr; o < 64; o <<= 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int e = 0; e < E; ++e) dw[i][e] += __shfl_xor(dw[i][e], o);
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; ++e) sums[e * 256 + threadIdx.x] = dw[i][e];
        __syncthreads();
        if ((int)threadIdx.x < tpr) {
#pragma unroll
          for (int e = 0; e < E; ++e) {
            float t = sums[e * 256 + threadIdx.x];
            for (int at = 64; at < 256; at += 64) t += sums[e * 256 + at + threadIdx.x];
            dw[i][e] = t;
          }
        }
      }
    }
  }
  if ((int)threadIdx.x >= tpr) return;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = E * (sub + i * tpr);
    if (c < D) store_dw<E>(a, blockIdx.x, gridDim.x, c, dw[i]);
  }
}

// dw of E ACROSS columns by one workgroup: ACROSS threads across them, the others each a
// share of the rows, which meet by shuffles and then, waves in order, in LDS.
template <typename TX, typename TY, int ACROSS>
__device__ __forceinline__ void grad_columns(const RmsArgs& a, int block) {
  constexpr int E = 16 / (int)sizeof(TX), U = 4;
  __shared__ float sums[16][ACROSS * E];
  const int tid = threadIdx.x, first = E * ACROSS * block, at = tid % ACROSS, c = first + E * at;
  const int R = (int)a.R, rows = blockDim.x / ACROSS;
  float dw[E];
#pragma unroll
  for (int e = 0; e < E; ++e) dw[e] = 0.f;
  for (int r0 = tid / ACROSS; r0 < R; r0 += U * rows) {
    Group<TX, E> x[U];
    Group<TY, E> dy[U];
    float rstd[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = min(r0 + u * rows, R - 1);
      x[u].load(static_cast<const TX*>(a.x) + r * a.ldx, c, a.D);
      dy[u].load(static_cast<const TY*>(a.dy) + r * a.ldy, c, a.D);
      rstd[u] = a.rstd_in[r];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (r0 + u * rows >= R) break;
#pragma unroll
      for (int e = 0; e < E; ++e) dw[e] = fmaf(dy[u].get(e), x[u].get(e) * rstd[u], dw[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
#pragma unroll
    for (int o = ACROSS; o < 64; o <<= 1) dw[e] += __shfl_xor(dw[e], o);
    if ((tid & 63) == at) sums[tid >> 6][E * at + e] = dw[e];
  }
  __syncthreads();
  if (tid < E * ACROSS && first + tid < a.D) {
    float t = sums[0][tid];
    for (int v = 1; v < (int)blockDim.x / 64; ++v) t += sums[v][tid];
    a.dw[first + tid] = t;
  }
}

// Both gradients in one launch: the first workgroups take columns, the others rows.
// dw needs nothing that the rows compute, so no workgroup waits for another; h and dy
// are read twice, the second time from the caches.
template <typename TX, typename TY, typename TD, int NV>
__global__ __launch_bounds__(1024) void rms_grad_small_kernel(RmsArgs a, int column_blocks, bool lines) {
  constexpr int E = 16 / (int)sizeof(TX);
  if ((int)blockIdx.x < column_blocks) {
    if (lines) grad_columns<TX, TY, 8>(a, blockIdx.x);
    else grad_columns<TX, TY, 4>(a, blockIdx.x);
  } else {
    float none[NV][E];
    grad_rows<TX, TY, TD, false>(a, (int)blockIdx.x - column_blocks, (int)gridDim.x - column_blocks, none);
  }
}

// Long rows, first pass: every row's c.
template <typename TX, typename TY>
__global__ __launch_bounds__(1024) void rms_grad_rows_kernel(RmsArgs a, float* __restrict__ cs) {
  constexpr int E = 16 / (int)sizeof(TX);
  __shared__ float red[2][16][1];
  int slot = 0;
  for (int64_t r = blockIdx.x; r < a.R; r += gridDim.x) {
    const float rstd = a.rstd_in[r];
    float s[1] = {0.f};
    for (int64_t c = E * threadIdx.x; c < a.D; c += E * 1024) {
      Group<TX, E> x;
      Group<TY, E> dy;
      x.load(static_cast<const TX*>(a.x) + r * a.ldx, (int)c, a.D);
      dy.load(static_cast<const TY*>(a.dy) + r * a.ldy, (int)c, a.D);
      float w[E];
      load_params<E>(a.w, a.w_bf16, (int)c, a.D, 1.f, w);
#pragma unroll
      for (int e = 0; e < E; ++e) s[0] = fmaf(dy.get(e) * w[e], x.get(e) * rstd, s[0]);
    }
    row_sums(s, 1024, red, slot);
    if (threadIdx.x == 0) cs[r] = s[0] * a.inv_d;
  }
}

// Long rows, second pass: one group of columns a thread (grid x), every
// gridDim.y-th row: dx, and the workgroup's share of dw.
template <typename TX, typename TY, typename TD>
__global__ __launch_bounds__(256) void rms_grad_cols_kernel(RmsArgs a, const float* __restrict__ cs) {
  constexpr int E = 16 / (int)sizeof(TX);
  const int64_t c64 = E * ((int64_t)blockIdx.x * 256 + threadIdx.x);
  if (c64 >= a.D) return;
  const int c = (int)c64;
  float w[E], dw[E];
  load_params<E>(a.w, a.w_bf16, c, a.D, 1.f, w);
#pragma unroll
  for (int e = 0; e < E; ++e) dw[e] = 0.f;
  for (int64_t r = blockIdx.y; r < a.R; r += gridDim.y) {
    Group<TX, E> x;
    Group<TY, E> dy;
    Other<TD, E> dh;
    x.load(static_cast<const TX*>(a.x) + r * a.ldx, c, a.D);
    dy.load(static_cast<const TY*>(a.dy) + r * a.ldy, c, a.D);
    dh.load(a, r, c);
    const float rstd = a.rstd_in[r], k = cs[r];
    float v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float t = dy.get(e), h = x.get(e) * rstd;
      dw[e] = fmaf(t, h, dw[e]);
      v[e] = fmaf(rstd, t * w[e] - h * k, dh.get(e));
    }
    using TO = Dx<TY, TD>;
    store_group<TO, E>(static_cast<TO*>(a.dx) + r * a.lddx, c, a.D, v);
  }
  if (a.dw) store_dw<E>(a, blockIdx.y, gridDim.y, c, dw);
}

// dw[c]: the sum of `parts` partial rows, 16 columns a workgroup, 64 threads a
// column (every 64th row each, then those in order).
__global__ __launch_bounds__(1024) void rms_grad_sum_kernel(RmsArgs a, int parts) {
  __shared__ float red[64][17];
  const int col = threadIdx.x & 15, g = threadIdx.x >> 4;
  const int c = 16 * (int)blockIdx.x + col;
  float s = 0.f;
  if (c < a.D) {
    // Eight loads at a time, whatever is left (a loop over what an unrolled one leaves
    // waits for each: 1000 x 1009 fp32, 512 and 500 parts, 9.9 us and 11.3).
    for (int k0 = g; k0 < parts; k0 += 512) {
      float t[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) t[u] = a.partial[(int64_t)min(k0 + 64 * u, parts - 1) * a.Dp + c];
#pragma unroll
      for (int u = 0; u < 8; ++u) s += k0 + 64 * u < parts ? t[u] : 0.f;
    }
  }
  red[g][col] = s;
  __syncthreads();
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
    a.dw[c] = s;
  }
}

constexpr int kMaxGrid = 1 << 20;  // workgroups of the passes over long rows; their loops stride over the rest
constexpr int kWaves = 16;         // a CU, of the forward pass

// f of the kernel's groups a thread, and (by_geom) threads a workgroup, as constants.
template <int MAX_NV, typename F>
hipError_t by_nv(const NormGeom& g, F f) {
  if constexpr (MAX_NV == 4) {
    if (g.nv == 4) return f(std::integral_constant<int, 4>{});
  }
  return g.nv == 1 ? f(std::integral_constant<int, 1>{}) : f(std::integral_constant<int, 2>{});
}
template <int MAX_NV, typename F>
hipError_t by_geom(const NormGeom& g, F f) {
  using std::integral_constant;
  return by_nv<MAX_NV>(g, [&](auto nv) {
    return g.nt <= 256   ? f(nv, integral_constant<int, 256>{})
           : g.nt <= 512 ? f(nv, integral_constant<int, 512>{})
                         : f(nv, integral_constant<int, 1024>{});
  });
}

template <typename TX, typename TR>
hipError_t launch_rms(RmsArgs a, hipStream_t stream) {
  constexpr int E = 16 / (int)sizeof(TX);
  const NormGeom g = norm_geom(a.R, a.D, E, 4, is_fp8(a.y_type) ? kGroup / E : 1);
  if (g.nv == 0) {
    const unsigned grid = (unsigned)std::min<int64_t>(a.R, kMaxGrid);
    return enqueue(rms_long_kernel<TX, TR>, dim3(grid), dim3(1024), stream, a);
  }
  a.tpr = g.tpr;
  const int64_t most = kWaves * 64 / g.nt * (int64_t)device_cus();
  const dim3 grid((unsigned)std::min<int64_t>(cdiv(a.R, g.nt / g.tpr), most)), block(g.nt);
  return by_geom<4>(g, [&](auto nv, auto nt) {
    return enqueue(rms_kernel<TX, TR, decltype(nv)::value, decltype(nt)::value>, grid, block, stream, a);
  });
}

// The backward pass holds 16 columns a thread: their sum, w, h, dy and dh.
struct GradGeom {
  NormGeom g;
  bool small;     // both gradients in one launch
  int64_t parts;  // partial rows of dw, or workgroups that take rows
  int64_t Dp;
  size_t partial_bytes, c_bytes;
};

GradGeom grad_geom(int64_t R, int64_t D, int hsz, bool dw) {
  const int e = 16 / hsz;
  GradGeom q{};
  q.g = norm_geom(R, D, e, 16 / e);
  q.Dp = cdiv(D, 8) * 8;
  if (q.g.nv > 0) {
    // 8 waves a CU, and 12 for bf16, as many rows allow; where those would have one
    // turn each, half as many with two leave half the partial sums (1000 x 1009 bf16
    // 11.6 us and 9.4, 512 x 4096 14.7 and 11.8).
    const int64_t cus = device_cus(), turns = cdiv(R, q.g.nt / q.g.tpr);
    q.parts = std::min({turns, cdiv(hsz == 4 ? 8 : 12, q.g.nt / 64) * cus, std::max(cus, cdiv(turns, 2))});
  } else {
    q.parts = std::min<int64_t>(R, std::max<int64_t>(1, cdiv(4 * (int64_t)device_cus(), cdiv(D, 256 * e))));
    q.c_bytes = (size_t)(R * sizeof(float) + 15) / 16 * 16;
  }
  // Up to 1024 rows of 16 MiB in all, 8 where rows are not whole lines: one launch
  // instead of two, though h and dy are read twice (fp32, 64 x 4096 7.4 us and 4.7, 512
  // x 4096 12.0 and 9.1, 1024 x 4096 16.2 and 14.7, 1000 x 1009 9.7 and 8.5, but 1000 x
  // 4001 17.9 and 25.1, 2048 x 512 7.9 and 11.1, 1024 x 8192 24.4 and 26.1; bf16, 512 x
  // 2048 8.3 and 4.8, 1024 x 8192 19.7 and 15.3, 1000 x 4001 16.6 and 12.8, 2048 x 1024
  // 9.2 and 12.0).
  const int64_t most = int64_t(D * hsz % 128 == 0 ? 16 : 8) << 20;
  q.small = dw && q.g.nv > 0 && q.parts > 1 && R <= 1024 && R * D * hsz <= most;
  if (q.small) {
    q.g.nt = 1024 / q.g.tpr * q.g.tpr;
    q.parts = cdiv(R, q.g.nt / q.g.tpr);
  }
  q.partial_bytes = dw && !q.small && q.parts > 1 ? (size_t)(q.parts * q.Dp) * sizeof(float) : 0;
  return q;
}

template <typename TX, typename TY, typename TD>
hipError_t launch_rms_grad(RmsArgs a, const GradGeom& q, float* cs, hipStream_t stream) {
  constexpr int E = 16 / (int)sizeof(TX);
  if (a.R == 0) return a.dw ? enqueue_zeros(a.dw, 1, a.D, a.D, stream) : hipSuccess;
  hipError_t e;
  if (q.g.nv == 0) {
    const unsigned grid = (unsigned)std::min<int64_t>(a.R, kMaxGrid);
    e = enqueue(rms_grad_rows_kernel<TX, TY>, dim3(grid), dim3(1024), stream, a, cs);
    if (e != hipSuccess) return e;
    e = enqueue(rms_grad_cols_kernel<TX, TY, TD>, dim3((unsigned)cdiv(a.D, 256 * E), (unsigned)q.parts), dim3(256), stream,
                a, cs);
  } else {
    a.tpr = q.g.tpr;
    if (q.small) {
      // Lines of 128 bytes where rows begin at them (512 x 4096 fp32 12.1 us and 9.2),
      // elsewhere half as much and twice the workgroups (1000 x 1009 fp32 10.2 and 8.5).
      const bool lines = a.ldx * sizeof(TX) % 128 == 0 && a.ldy * sizeof(TY) % 128 == 0;
      const int columns = (int)cdiv(a.D, lines ? 8 * E : 4 * E);
      return by_nv<16 / E>(q.g, [&](auto nv) {
        return enqueue(rms_grad_small_kernel<TX, TY, TD, decltype(nv)::value>, dim3((unsigned)(columns + q.parts)),
                       dim3(q.g.nt), stream, a, columns, lines);
      });
    }
    e = by_geom<16 / E>(q.g, [&](auto nv, auto nt) {
      return enqueue(rms_grad_kernel<TX, TY, TD, decltype(nv)::value, decltype(nt)::value>, dim3((unsigned)q.parts),
                     dim3(q.g.nt), stream, a);
    });
  }
  if (e != hipSuccess || !a.dw || q.parts == 1) return e;
  return enqueue(rms_grad_sum_kernel, dim3((unsigned)cdiv(a.D, 16)), dim3(1024), stream, a, (int)q.parts);
}

bool is_wide(int32_t t) { return t == TILEC_F32 || t == TILEC_BF16; }

int check_shape(int64_t R, int64_t D) {
  if (R < 0 || D < 1 || R > kMaxDim || D > kMaxDim)
    return fail(TILEC_ERR_VALUE, "tilec: RMS norm: bad shape R=%lld D=%lld", (long long)R, (long long)D);
  return TILEC_OK;
}

int check_rows(const char* what, const void* p, int64_t ld, int64_t R, int64_t D) {
  if (R == 0) return TILEC_OK;
  if (p == nullptr) return fail(TILEC_ERR_VALUE, "tilec: RMS norm: %s is NULL", what);
  if (R > 1 && ld < D)
    return fail(TILEC_ERR_VALUE, "tilec: RMS norm: the row stride of %s, %lld, is less than D=%lld", what,
                (long long)ld, (long long)D);
  if (ld > (int64_t(1) << 40))
    return fail(TILEC_ERR_VALUE, "tilec: RMS norm: the row stride of %s, %lld, is too large", what, (long long)ld);
  return TILEC_OK;
}

// f of the element type of a code, or of None for an absent operand.
template <typename F>
hipError_t by_type(bool present, int32_t dtype, F f) {
  return !present ? f(None{}) : dtype == TILEC_F32 ? f(float{}) : f(u16{});
}

}  // namespace

}  // namespace tilec

using namespace tilec;

extern "C" {

int tilec_rms_norm(const void* x, const void* residual, const void* weight, void* y, float* y_scale, void* h,
                   float* rstd, int64_t R, int64_t D, int64_t ldx, int64_t ldr, int64_t ldy, int64_t ldh,
                   int64_t scale_row, int64_t scale_group, int32_t x_dtype, int32_t r_dtype, int32_t y_dtype,
                   int32_t w_dtype, float eps, void* stream) {
  clear_error();
  if (!is_wide(x_dtype) || (residual != nullptr && !is_wide(r_dtype)) || !is_wide(w_dtype) ||
      (!is_wide(y_dtype) && !is_fp8(y_dtype)))
    return fail(TILEC_ERR_TYPE, "tilec: RMS norm: unsupported dtype codes %d, %d, %d, %d of x, residual, y and weight",
                x_dtype, r_dtype, y_dtype, w_dtype);
  int rc = check_shape(R, D);
  if (rc == TILEC_OK) rc = check_rows("x", x, ldx, R, D);
  if (rc == TILEC_OK && residual != nullptr) rc = check_rows("residual", residual, ldr, R, D);
  if (rc == TILEC_OK && residual != nullptr) rc = check_rows("h", h, ldh, R, D);
  if (rc == TILEC_OK) rc = check_rows("y", y, ldy, R, D);
  if (rc != TILEC_OK || R == 0) return rc;
  if (R > 1 && residual != nullptr && h == residual && ldh != ldr)
    return fail(TILEC_ERR_VALUE, "tilec: RMS norm: h is the residual, with rows %lld apart instead of %lld", (long long)ldh,
                (long long)ldr);
  const int64_t room = cdiv(D, 16) * 16;
  if (is_fp8(y_dtype) && (y_scale == nullptr || reinterpret_cast<uintptr_t>(y) % 16 != 0 ||
                          (R > 1 && (ldy % 16 != 0 || ldy < room))))
    return fail(TILEC_ERR_VALUE, "tilec: RMS norm: 8-bit codes need scales and rows at multiples of 16 bytes");
  constexpr int64_t most = int64_t(1) << 40;
  if (is_fp8(y_dtype) && (scale_row < 0 || scale_group < 0 || scale_row > most || scale_group > most))
    return fail(TILEC_ERR_VALUE, "tilec: RMS norm: bad strides %lld, %lld of scales", (long long)scale_row,
                (long long)scale_group);
  RmsArgs a{};
  a.x = x, a.res = residual, a.w = weight, a.y = y, a.y_scale = y_scale, a.h = h, a.rstd = rstd;
  a.s_row = scale_row, a.s_group = scale_group;
  a.ldx = ldx, a.ldr = ldr, a.ldy = is_fp8(y_dtype) && R == 1 ? room : ldy, a.ldh = ldh;
  a.R = R, a.D = (int)D, a.y_type = y_dtype, a.w_bf16 = w_dtype == TILEC_BF16, a.groups = (int)cdiv(D, kGroup);
  a.eps = eps, a.inv_d = 1.f / (float)D;
  const hipError_t e = by_type(residual != nullptr, r_dtype, [&](auto tr) {
    using TR = decltype(tr);
    return x_dtype == TILEC_F32 ? launch_rms<float, TR>(a, static_cast<hipStream_t>(stream))
                                : launch_rms<u16, TR>(a, static_cast<hipStream_t>(stream));
  });
  if (e != hipSuccess) return fail(TILEC_ERR_HIP, "tilec: launching the RMS norm failed: %s", hipGetErrorString(e));
  return TILEC_OK;
}

size_t tilec_rms_norm_backward_workspace_bytes(int64_t R, int64_t D, int32_t h_dtype) {
  if (!is_wide(h_dtype) || check_shape(R, D) != TILEC_OK) return 0;
  const GradGeom q = grad_geom(R, D, h_dtype == TILEC_F32 ? 4 : 2, true);
  return q.c_bytes + q.partial_bytes;
}

int tilec_rms_norm_backward(const void* dy, const void* h, const float* rstd, const void* weight, const void* dh,
                            void* dx, float* dweight, int64_t R, int64_t D, int64_t lddy, int64_t ldh, int64_t lddh,
                            int64_t lddx, int32_t dy_dtype, int32_t h_dtype, int32_t dh_dtype, int32_t w_dtype,
                            void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  if (!is_wide(dy_dtype) || !is_wide(h_dtype) || !is_wide(w_dtype) || (dh != nullptr && !is_wide(dh_dtype)))
    return fail(TILEC_ERR_TYPE, "tilec: RMS norm: unsupported dtype codes %d, %d, %d, %d of dy, h, dh and weight",
                dy_dtype, h_dtype, dh_dtype, w_dtype);
  int rc = check_shape(R, D);
  if (rc == TILEC_OK) rc = check_rows("dy", dy, lddy, R, D);
  if (rc == TILEC_OK) rc = check_rows("h", h, ldh, R, D);
  if (rc == TILEC_OK && dh != nullptr) rc = check_rows("dh", dh, lddh, R, D);
  if (rc == TILEC_OK) rc = check_rows("dx", dx, lddx, R, D);
  if (rc != TILEC_OK) return rc;
  if (R > 0 && (dx == dy || dx == h))  // (both are read again after rows of dx are written)
    return fail(TILEC_ERR_VALUE, "tilec: RMS norm: dx is %s", dx == dy ? "dy" : "h");
  if (R > 1 && dx == dh && lddx != lddh)  // (a row of dx would be another's dh)
    return fail(TILEC_ERR_VALUE, "tilec: RMS norm: dx is dh, with rows %lld apart instead of %lld", (long long)lddx,
                (long long)lddh);
  if (R > 0 && rstd == nullptr) return fail(TILEC_ERR_VALUE, "tilec: RMS norm: rstd is NULL");
  const GradGeom q = grad_geom(R, D, h_dtype == TILEC_F32 ? 4 : 2, dweight != nullptr);
  const size_t need = q.c_bytes + q.partial_bytes;
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(TILEC_ERR_WORKSPACE, "tilec: RMS norm's backward pass needs %zu workspace bytes (got %zu)", need,
                workspace == nullptr ? (size_t)0 : workspace_bytes);
  RmsArgs a{};
  a.x = h, a.dy = dy, a.w = weight, a.dh = dh, a.dx = dx, a.rstd_in = rstd, a.dw = dweight;
  a.ldx = ldh, a.ldy = lddy, a.lddh = lddh, a.lddx = lddx, a.R = R, a.D = (int)D, a.Dp = (int)q.Dp;
  a.w_bf16 = w_dtype == TILEC_BF16, a.inv_d = 1.f / (float)D;
  a.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + q.c_bytes);
  float* cs = static_cast<float*>(workspace);
  const hipError_t e = by_type(dh != nullptr, dh_dtype, [&](auto td) {
    using TD = decltype(td);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (h_dtype == TILEC_F32)
      return dy_dtype == TILEC_F32 ? launch_rms_grad<float, float, TD>(a, q, cs, st)
                                   : launch_rms_grad<float, u16, TD>(a, q, cs, st);
    return dy_dtype == TILEC_F32 ? launch_rms_grad<u16, float, TD>(a, q, cs, st)
                                 : launch_rms_grad<u16, u16, TD>(a, q, cs, st);
  });
  if (e != hipSuccess)
    return fail(TILEC_ERR_HIP, "tilec: launching the RMS norm's backward pass failed: %s", hipGetErrorString(e));
  return TILEC_OK;
}

}  // extern "C"
