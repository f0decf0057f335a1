// What the passes over the rows of a matrix share: groups of a row's values in
// 16-byte loads at any element alignment, sums over the threads that serve a row,
// and how many of them do.
#pragma once

#include <algorithm>

#include "common.h"

namespace tilec {

namespace {

typedef unsigned short u16;

// N values of type T (16 or 8 bytes a load) at the element's own alignment.
template <typename T, int N>
struct Group {
  static constexpr int WORDS = N * (int)sizeof(T) / 4;
  int w[WORDS];

  __device__ __forceinline__ float get(int e) const {
    if constexpr (sizeof(T) == 4) return __int_as_float(w[e]);
    else return __int_as_float((e & 1) ? w[e >> 1] & (int)0xffff0000u : w[e >> 1] << 16);
  }
  // Elements c .. c + N - 1 of the row; zeros past D.
  __device__ __forceinline__ void load(const T* __restrict__ row, int c, int D) {
    if (c + N <= D) {
      if constexpr (WORDS == 2) {
        typedef int i32x2 __attribute__((ext_vector_type(2)));
        typedef i32x2 __attribute__((aligned(2))) i32x2_any;
        const i32x2 v = *reinterpret_cast<const i32x2_any*>(row + c);
        w[0] = v.x, w[1] = v.y;
      } else {
        typedef i32x4 __attribute__((aligned(2))) i32x4_any;
#pragma unroll
        for (int q = 0; q < WORDS / 4; ++q) {
          const i32x4 v = reinterpret_cast<const i32x4_any*>(row + c)[q];
          w[4 * q] = v.x, w[4 * q + 1] = v.y, w[4 * q + 2] = v.z, w[4 * q + 3] = v.w;
        }
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = 0;
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (c + e < D) {
        if constexpr (sizeof(T) == 4) w[e] = reinterpret_cast<const int*>(row)[c + e];
        else w[e >> 1] |= (int)((uint32_t)row[c + e] << (16 * (e & 1)));
      }
  }
};

__device__ __forceinline__ uint32_t to_bf16(float f) {
  return (uint32_t)__builtin_bit_cast(u16, (__bf16)f);  // to nearest, ties to even
}

// Round N values to T and store them at elements c .. of the row, those below D.
template <typename T, int N>
__device__ __forceinline__ void store_group(T* __restrict__ row, int c, int D, const float (&v)[N]) {
  constexpr int WORDS = N * (int)sizeof(T) / 4;
  int w[WORDS];
#pragma unroll
  for (int i = 0; i < WORDS; ++i) {
    if constexpr (sizeof(T) == 4) w[i] = __float_as_int(v[i]);
    else w[i] = (int)(to_bf16(v[2 * i]) | to_bf16(v[2 * i + 1]) << 16);
  }
  if (c + N <= D) {
    if constexpr (WORDS == 2) {
      typedef int i32x2 __attribute__((ext_vector_type(2)));
      typedef i32x2 __attribute__((aligned(2))) i32x2_any;
      *reinterpret_cast<i32x2_any*>(row + c) = i32x2{w[0], w[1]};
    } else {
      typedef i32x4 __attribute__((aligned(2))) i32x4_any;
#pragma unroll
      for (int q = 0; q < WORDS / 4; ++q)
        reinterpret_cast<i32x4_any*>(row + c)[q] = i32x4{w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]};
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (c + e < D) {
      if constexpr (sizeof(T) == 4) reinterpret_cast<int*>(row)[c + e] = w[e];
      else row[c + e] = (T)((uint32_t)w[e >> 1] >> (16 * (e & 1)));
    }
}

// N parameters (fp32 or bf16, decided at run time: every thread alike) from
// element c on; `none` where there are none.
template <int N>
__device__ __forceinline__ void load_params(const void* p, bool bf16, int c, int D, float none, float (&v)[N]) {
  if (p == nullptr) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = none;
  } else if (bf16) {
    Group<u16, N> g;
    g.load(static_cast<const u16*>(p), c, D);
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = g.get(e);
  } else {
    Group<float, N> g;
    g.load(static_cast<const float*>(p), c, D);
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = g.get(e);
  }
}

// Sums of NS values over the tpr consecutive threads that serve a row, in
// every one of them.  Past a wave they meet in LDS, in wave order; `slot`
// alternates between calls, so that one barrier a call is enough.
template <int NS>
__device__ __forceinline__ void row_sums(float (&s)[NS], int tpr, float (*red)[16][NS], int& slot) {
  for (int o = min(tpr, 64) >> 1; o > 0; o >>= 1) {
#pragma unroll
    for (int i = 0; i < NS; ++i) s[i] += __shfl_xor(s[i], o);
  }
  if (tpr <= 64) return;
  const int wave = threadIdx.x >> 6, waves = tpr >> 6;
  const int first = tpr == (int)blockDim.x ? 0 : wave / waves * waves;  // of the row
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int i = 0; i < NS; ++i) red[slot][wave][i] = s[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NS; ++i) s[i] = red[slot][first][i];
  for (int w = first + 1; w < first + waves; ++w) {
#pragma unroll
    for (int i = 0; i < NS; ++i) s[i] += red[slot][w][i];
  }
  slot ^= 1;
}

// 1 / sqrt(v): one Newton step on the hardware's root, which is 1 ulp off.
__device__ __forceinline__ float inv_root(float v) {
  const float y = rsqrtf(v), r = fmaf(-v * y, y, 1.f);
  return v > 0.f && v < INFINITY ? fmaf(0.5f * y, r, y) : y;
}

// How a row is spread: tpr threads of nv groups each (nv 0: too long).
struct NormGeom {
  int tpr, nv, nt;  // nt: threads of a workgroup
};

// Among the spreads that leave few lanes idle (within a third of the fewest):
// with enough rows to fill the chip anyway, the fewest threads a row (fewer
// steps of the sums, more loads in flight each) up to 4 groups a thread (4099 x
// 3001 fp32, 1, 2, 4 and 8 groups: 42, 28, 23 and 28 us; 8192 x 1600, 1 group
// in 448 threads 40 us, 4 in 128 24), and with few rows the most.  min_tpr: the
// fewest threads a row, a power of two up to a wave.
NormGeom norm_geom(int64_t R, int64_t D, int e, int max_nv, int min_tpr = 1) {
  const int64_t groups = cdiv(D, e);
  NormGeom best{0, 0, 0};
  auto threads = [&](int nv) {  // of a row: a power of two up to a wave, then whole waves
    const int64_t n = cdiv(groups, nv);
    if (n > 64) return cdiv(n, 64) * 64;
    int64_t t = min_tpr;
    while (t < n) t *= 2;
    return t;
  };
  int64_t least = INT64_MAX;
  for (int nv = 1; nv <= max_nv; nv *= 2)
    if (threads(nv) <= 1024) least = std::min(least, threads(nv) * nv);
  const bool many = R >= 8 * (int64_t)device_cus();
  for (int nv = 1; nv <= max_nv; nv *= 2) {
    const int64_t tpr = threads(nv);
    if (tpr > 1024 || 3 * tpr * nv > 4 * least || (best.nv != 0 && !many)) continue;
    best = {(int)tpr, nv, tpr <= 64 ? 256 : (int)tpr};
  }
  return best;
}

}  // namespace

}  // namespace tilec
