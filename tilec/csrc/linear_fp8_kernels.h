// The kernels of linear_fp8.h, for one pair of formats a file.
#pragma once

#include <type_traits>

#include "linear_fp8.h"

namespace tilec {

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void* lds_ptr_t;

// Two 8-bit values as bf16, exactly.
template <int FMT, bool HIGH>
__device__ __forceinline__ bf16x2 widen2(int v) {
  if constexpr (FMT == 0) return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)v, 1.0f, HIGH);
  else return __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8((unsigned)v, 1.0f, HIGH);
}

// A lane's share of an operand of one block: 32 of a row's 128 codes.  Which 32
// does not matter as long as both operands' lanes hold the same.
template <bool F8, int FMT>
struct Frag;
template <int FMT>
struct Frag<true, FMT> {
  i32x8 v;
  __device__ __forceinline__ void set(i32x4 lo, i32x4 hi) { v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7); }
};
template <int FMT>
struct Frag<false, FMT> {
  bf16x8 v[4];
  __device__ __forceinline__ void set(i32x4 lo, i32x4 hi) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int a = q < 2 ? lo[2 * q] : hi[2 * q - 4], b = q < 2 ? lo[2 * q + 1] : hi[2 * q - 3];
      const bf16x2 e[4] = {widen2<FMT, false>(a), widen2<FMT, true>(a), widen2<FMT, false>(b), widen2<FMT, true>(b)};
      v[q] = bf16x8{e[0].x, e[0].y, e[1].x, e[1].y, e[2].x, e[2].y, e[3].x, e[3].y};
    }
  }
};

// P_g of a block: rows 4 (lane / 16) + r of w, row lane % 16 of x.
template <int FX, int FW>
__device__ __forceinline__ f32x4 block(const Frag<true, FW>& w, const Frag<true, FX>& x) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v, x.v, f32x4{0.f, 0.f, 0.f, 0.f}, FW, FX, 0, 0, 0, 0);
}
template <int FX, int FW>
__device__ __forceinline__ f32x4 block(const Frag<false, FW>& w, const Frag<false, FX>& x) {
  f32x4 p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int q = 0; q < 4; ++q) p = mfma16x16x32bf16(w.v[q], x.v[q], p);
  return p;
}

// Four consecutive outputs of row m, those below N.
template <typename TO>
__device__ __forceinline__ void store4(TO* __restrict__ row, int n, int N, f32x4 v) {
  if constexpr (sizeof(TO) == 4) {
    if (n + 4 <= N) {
      typedef f32x4 __attribute__((aligned(4))) f32x4_any;
      *reinterpret_cast<f32x4_any*>(row + n) = v;
      return;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (n + r < N) row[n + r] = v[r];
  } else {
    typedef __bf16 bf16x4v __attribute__((ext_vector_type(4)));
    const bf16x4v b = __builtin_convertvector(v, bf16x4v);
    if (n + 4 <= N) {
      typedef bf16x4v __attribute__((aligned(2))) bf16x4_any;
      *reinterpret_cast<bf16x4_any*>(row + n) = b;
      return;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (n + r < N) reinterpret_cast<__bf16*>(row)[n + r] = b[r];
  }
}
template <bool F8>
using Out = std::conditional_t<F8, unsigned short, float>;  // bf16, or float32

template <int BM_, int BN_, int WM_, int WN_>
struct TileGeom {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr int NW = WM * WN, NT = 64 * NW;
  static constexpr int MT = BM / WM / 16, NB = BN / WN / 16;  // blocks of a wave
  static constexpr int XI = BM * 8 / NT, WI = BN * 8 / NT;    // 16-byte copies a thread and step
  static constexpr int SI = (BM + BN + NT - 1) / NT;          // scales a thread and step
  static constexpr int W_AT = BM * 128, S_AT = W_AT + BN * 128, STAGE = S_AT + SI * NT * 4;
  static_assert(BM * 8 % NT == 0 && BN * 8 % NT == 0 && BM % 64 == 0 && BN % 64 == 0, "whole copies");
  static_assert(BN / WN <= 128 && 128 % (BN / WN) == 0, "a wave's columns lie in one tile of w");
  static_assert(2 * STAGE <= 160 * 1024, "LDS is 160 KiB");
};

// BM x BN outputs a workgroup, a group of 128 k a step.  Two stages: a step's
// codes and scales are copied into one (global to LDS, 16 bytes a lane) while
// the other is multiplied.  A stage holds rows of 128 bytes whose 16-byte chunks
// are exchanged by (row / 2) % 8, so that 16 rows' reads spread over the banks.
// What lies past M, N or K is never read: those copies have an address out of
// range and leave zeros; where K ends inside a chunk the rest of it is cleared
// in LDS before the last step.
template <class P, bool F8, int FX, int FW, bool WROWS>
__global__ __launch_bounds__(P::NT, 1) void fp8_tile_kernel(Fp8Args a) {
  __shared__ __align__(16) char lds0[P::STAGE];
  __shared__ __align__(16) char lds1[P::STAGE];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / P::WN, wn = wave % P::WN;
  const int tiles_m = (a.M + P::BM - 1) / P::BM, tiles_n = (a.N + P::BN - 1) / P::BN;
  int tm, tn;
  tile_of(blockIdx.x, a.xcds, tiles_m, tiles_n, a.group_m, tm, tn);
  const int m0 = tm * P::BM, n0 = tn * P::BN;
  const int split = blockIdx.y, g0 = split * a.split_steps, nk = min(a.G, g0 + a.split_steps) - g0;

  // Copies: physical chunk p = 64 (wave * I + i) + lane of an operand is chunk
  // (p % 8) ^ (p / 16 % 8) of row p / 8, which is c0 or, for odd 64s, c0 ^ 4.
  const int c0 = (lane & 7) ^ (lane >> 4);
  uint32_t off_x[P::XI], off_w[P::WI], off_s[P::SI];
#pragma unroll
  for (int i = 0; i < P::XI; ++i) {
    const int q = wave * P::XI + i, r = 8 * q + (lane >> 3);
    off_x[i] = ((uint32_t)r * (uint32_t)a.ldx + 16u * (c0 ^ 4 * (q & 1))) | oob_unless(m0 + r < a.M);
  }
#pragma unroll
  for (int i = 0; i < P::WI; ++i) {
    const int q = wave * P::WI + i, r = 8 * q + (lane >> 3);
    off_w[i] = ((uint32_t)r * (uint32_t)a.ldw + 16u * (c0 ^ 4 * (q & 1))) | oob_unless(n0 + r < a.N);
  }
  // Scales: entry e is that of row m0 + e of x, and from BM on of row n0 + e - BM of w.
#pragma unroll
  for (int i = 0; i < P::SI; ++i) {
    const int first = 64 * (wave * P::SI + i);  // wave-uniform
    const bool is_x = first < P::BM;
    const int e = first + lane - (is_x ? 0 : P::BM), shift = is_x ? a.xshift : a.wshift, r0 = is_x ? m0 : n0;
    off_s[i] = 4u * (uint32_t)(((r0 + e) >> shift) - (r0 >> shift)) * (uint32_t)a.G |
               oob_unless(r0 + e < (is_x ? a.M : a.N) && (is_x || e < P::BN));
  }
  const unsigned char* const xb = a.x + (int64_t)m0 * a.ldx + (int64_t)g0 * kGroup;
  const unsigned char* const wb = a.w + (int64_t)n0 * a.ldw + (int64_t)g0 * kGroup;
  const float* const sxb = a.sx + (int64_t)(m0 >> a.xshift) * a.G + g0;
  const float* const swb = a.sw + (int64_t)(n0 >> a.wshift) * a.G + g0;
  // A step past the last has resources without records: nothing is read.
  auto copy = [&](int kt, char* st) __attribute__((always_inline)) {
    const uint32_t records = kt < nk ? 0x7FFFFFFFu : 0u;
    const int left = a.K - (g0 + kt) * kGroup;  // bytes of a row from here on
    const uint32_t past[2] = {oob_unless(16 * c0 < left), oob_unless(16 * (c0 ^ 4) < left)};
    const BufRsrc rx = make_rsrc_uniform(xb + (int64_t)kt * kGroup, records);
    const BufRsrc rw = make_rsrc_uniform(wb + (int64_t)kt * kGroup, records);
#pragma unroll
    for (int i = 0; i < P::XI; ++i) {
      const int q = wave * P::XI + i;
      const uint32_t off = off_x[i] | past[P::XI % 2 == 0 ? i & 1 : q & 1];
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (lds_ptr_t)(st + 1024 * q), 16, off, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < P::WI; ++i) {
      const int q = wave * P::WI + i;
      const uint32_t off = off_w[i] | past[P::WI % 2 == 0 ? i & 1 : q & 1];
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (lds_ptr_t)(st + P::W_AT + 1024 * q), 16, off, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < P::SI; ++i) {
      const int first = 64 * (wave * P::SI + i);
      const uint32_t off = off_s[i];
      const BufRsrc rs = make_rsrc_uniform((first < P::BM ? sxb : swb) + kt, records);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)(st + P::S_AT + 4 * first), 4, off, 0, 0, 0);
    }
  };

  f32x4 acc[P::MT][P::NB];
#pragma unroll
  for (int i = 0; i < P::MT; ++i)
#pragma unroll
    for (int j = 0; j < P::NB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  // A lane's 32 codes of row lane % 16: chunks lane / 16 and 4 + lane / 16.
  const int row = lane & 15, quad = lane >> 4;
  const int at = 128 * row + 16 * (quad ^ ((row >> 1) & 7));
  auto frag = [&](auto& f, const char* rows) __attribute__((always_inline)) {
    f.set(*reinterpret_cast<const i32x4*>(rows + at), *reinterpret_cast<const i32x4*>(rows + (at ^ 64)));
  };
  auto multiply = [&](const char* st) __attribute__((always_inline)) {
    const char* const xs = st + 128 * (wm * (P::BM / P::WM));
    const char* const ws = st + P::W_AT + 128 * (wn * (P::BN / P::WN));
    const float* const ssx = reinterpret_cast<const float*>(st + P::S_AT) + wm * (P::BM / P::WM) + row;
    const float* const ssw = reinterpret_cast<const float*>(st + P::S_AT) + P::BM + wn * (P::BN / P::WN);
    Frag<F8, FW> fw[P::NB];
    Frag<F8, FX> fx[2];
    f32x4 s4[P::NB], p[2][P::NB];
    float s[2], s1 = 1.f;
    frag(fx[0], xs);
#pragma unroll
    for (int j = 0; j < P::NB; ++j) {
      frag(fw[j], ws + 2048 * j);
      if constexpr (WROWS) s4[j] = *reinterpret_cast<const f32x4*>(ssw + 16 * j + 4 * quad);
    }
    if constexpr (!WROWS) s1 = *ssw;
    s[0] = ssx[0] * s1;
    __builtin_amdgcn_sched_barrier(0);
    // Row i's blocks on the matrix core, beside them the multiply-adds of row i - 1.
#pragma unroll
    for (int i = 0; i <= P::MT; ++i) {
      if (i + 1 < P::MT) frag(fx[(i + 1) & 1], xs + 2048 * (i + 1));
#pragma unroll
      for (int j = 0; j < P::NB; ++j) {
        if (i < P::MT) p[i & 1][j] = block<FX, FW>(fw[j], fx[i & 1]);
        if (i > 0) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            acc[i - 1][j][r] = fmaf(p[(i - 1) & 1][j][r], WROWS ? s[(i - 1) & 1] * s4[j][r] : s[(i - 1) & 1], acc[i - 1][j][r]);
        }
      }
      if (i + 1 < P::MT) s[(i + 1) & 1] = ssx[16 * (i + 1)] * s1;
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Clears what the last chunk of every row holds past K.
  auto clear_tail = [&](char* st) {
    const int in = a.K & 127;
    for (int r = tid; r < P::BM + P::BN; r += P::NT) {
      uint32_t* const c = reinterpret_cast<uint32_t*>(st + 128 * r + 16 * ((in >> 4) ^ ((r >> 1) & 7)));
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const int keep = (in & 15) - 4 * d;
        c[d] &= keep >= 4 ? ~0u : keep <= 0 ? 0u : (1u << (8 * keep)) - 1u;
      }
    }
  };
  auto arrive = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(0);  // this wave's copies of the step, and its reads of the other stage
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  auto step = [&](int kt, char* cur, char* next) __attribute__((always_inline)) {
    arrive();
    copy(kt + 1, next);
    multiply(cur);
  };
  if (nk > 0) {
    copy(0, lds0);
    int kt = 0;
#pragma unroll 1
    for (; kt + 2 < nk; kt += 2) {
      step(kt, lds0, lds1);
      step(kt + 1, lds1, lds0);
    }
    char* last = lds0;
    if (kt + 2 == nk) {
      step(kt, lds0, lds1);
      last = lds1;
    }
    arrive();
    if ((a.K & 15) != 0 && g0 + nk == a.G) {
      clear_tail(last);
      __syncthreads();
    }
    multiply(last);
  }

  const bool inside = m0 + P::BM <= a.M && n0 + P::BN <= a.N;
  auto store = [&](auto* out, int64_t ld) __attribute__((always_inline)) {
    using T = std::remove_pointer_t<decltype(out)>;
    const int mw = m0 + wm * (P::BM / P::WM) + row, nw = n0 + wn * (P::BN / P::WN) + 4 * quad;
    T* const first = out + (int64_t)mw * ld;
#pragma unroll
    for (int i = 0; i < P::MT; ++i) {
      T* const line = first + (int64_t)(16 * i) * ld;
#pragma unroll
      for (int j = 0; j < P::NB; ++j)
        if (inside || mw + 16 * i < a.M) store4<T>(line, nw + 16 * j, inside ? INT32_MAX : a.N, acc[i][j]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  if (gridDim.y > 1) store(a.partial + (int64_t)split * a.M * a.N, a.N);
  else store(static_cast<Out<F8>*>(a.out), a.ldo);
}

// Few rows of x (16 MT of them): bound by reading w, which goes from memory into
// the matrix core's registers.  A workgroup takes 16 rows of w, its waves every
// NW-th group each, U of them in flight; the waves' sums meet in LDS, in order.
template <int MT, int NW, int U, bool F8, int FX, int FW, bool WROWS>
__global__ __launch_bounds__(64 * NW) void fp8_stream_kernel(Fp8Args a) {
  __shared__ f32x4 red[NW][MT][64];
  const int tid = threadIdx.x, lane = tid & 63, row = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = blockIdx.x * 16;
  const BufRsrc rw = make_rsrc(a.w + (int64_t)n0 * a.ldw), rx = make_rsrc(a.x);
  const BufRsrc rsx = make_rsrc(a.sx), rsw = make_rsrc(a.sw + (int64_t)(n0 >> a.wshift) * a.G);
  const uint32_t w_row = (uint32_t)row * (uint32_t)a.ldw | oob_unless(n0 + row < a.N);
  uint32_t x_row[MT], sx_row[MT], sw_row[4];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = 16 * i + row;
    x_row[i] = (uint32_t)m * (uint32_t)a.ldx | oob_unless(m < a.M);
    sx_row[i] = 4u * (uint32_t)(m >> a.xshift) * (uint32_t)a.G | oob_unless(m < a.M);
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) sw_row[r] = 4u * (4 * quad + r) * (uint32_t)a.G | oob_unless(n0 + 4 * quad + r < a.N);
  auto load = [&](BufRsrc r, uint32_t off) {
    return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, 0));
  };
  auto load_once = [&](BufRsrc r, uint32_t off) {
    return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, 2));
  };
  auto cut = [&](i32x4 v, int left) {  // the first `left` bytes
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      const int keep = left - 4 * d;
      v[d] &= keep >= 4 ? ~0 : keep <= 0 ? 0 : (1 << (8 * keep)) - 1;
    }
    return v;
  };
  f32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int first = wave; first < a.G; first += NW * U) {
    i32x4 w[U][2], x[U][MT][2];
    float sx[U][MT], sw[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int g = first + NW * u, k = kGroup * g + 16 * quad;
      const uint32_t lo = (uint32_t)k | oob_unless(k < a.K), hi = (uint32_t)(k + 64) | oob_unless(k + 64 < a.K);
      const uint32_t live = oob_unless(g < a.G);
      w[u][0] = load_once(rw, (w_row + lo) | ((w_row | lo) & kOob));
      w[u][1] = load_once(rw, (w_row + hi) | ((w_row | hi) & kOob));
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        x[u][i][0] = load(rx, (x_row[i] + lo) | ((x_row[i] | lo) & kOob));
        x[u][i][1] = load(rx, (x_row[i] + hi) | ((x_row[i] | hi) & kOob));
        sx[u][i] = load_f32(rsx, (sx_row[i] + 4u * g) | ((sx_row[i] | live) & kOob));
      }
      if constexpr (WROWS) {
#pragma unroll
        for (int r = 0; r < 4; ++r) sw[u][r] = load_f32(rsw, (sw_row[r] + 4u * g) | ((sw_row[r] | live) & kOob));
      } else {
        sw[u][0] = load_f32(rsw, 4u * g | live);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int g = first + NW * u;
      if (g >= a.G) break;  // wave-uniform
      if (g == a.G - 1 && (a.K & 15) != 0) {
        const int left = a.K - kGroup * g - 16 * quad;
        w[u][0] = cut(w[u][0], left), w[u][1] = cut(w[u][1], left - 64);
#pragma unroll
        for (int i = 0; i < MT; ++i) x[u][i][0] = cut(x[u][i][0], left), x[u][i][1] = cut(x[u][i][1], left - 64);
      }
      Frag<F8, FW> fw;
      fw.set(w[u][0], w[u][1]);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        Frag<F8, FX> fx;
        fx.set(x[u][i][0], x[u][i][1]);
        const f32x4 p = block<FX, FW>(fw, fx);
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][r] = fmaf(p[r], sx[u][i] * sw[u][WROWS ? r : 0], acc[i][r]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) red[wave][i][lane] = acc[i];
  __syncthreads();
  for (int t = tid; t < MT * 64; t += 64 * NW) {
    const int i = t >> 6, l = t & 63, m = 16 * i + (l & 15);
    f32x4 s = red[0][i][l];
#pragma unroll
    for (int v = 1; v < NW; ++v) s += red[v][i][l];
    if (m < a.M) store4<Out<F8>>(static_cast<Out<F8>*>(a.out) + (int64_t)m * a.ldo, n0 + 4 * (l >> 4), a.N, s);
  }
}

template <class P, bool F8, int FX, int FW>
hipError_t launch_tile(const Fp8Args& a, int splits, hipStream_t stream) {
  const dim3 grid((unsigned)(cdiv(a.M, P::BM) * cdiv(a.N, P::BN)), (unsigned)splits);
  if (a.wshift == 0) hipLaunchKernelGGL((fp8_tile_kernel<P, F8, FX, FW, true>), grid, dim3(P::NT), 0, stream, a);
  else hipLaunchKernelGGL((fp8_tile_kernel<P, F8, FX, FW, false>), grid, dim3(P::NT), 0, stream, a);
  return hipGetLastError();
}

template <int MT, int U, bool F8, int FX, int FW>
hipError_t launch_stream(const Fp8Args& a, hipStream_t stream) {
  constexpr int NW = 8;
  const dim3 grid((unsigned)cdiv(a.N, 16));
  if (a.wshift == 0)
    hipLaunchKernelGGL((fp8_stream_kernel<MT, NW, U, F8, FX, FW, true>), grid, dim3(64 * NW), 0, stream, a);
  else hipLaunchKernelGGL((fp8_stream_kernel<MT, NW, U, F8, FX, FW, false>), grid, dim3(64 * NW), 0, stream, a);
  return hipGetLastError();
}

template <bool F8, int FX, int FW>
hipError_t launch_kind(const Fp8Args& a, int tile, int splits, hipStream_t stream) {
  if (tile < 0) {
    if (a.M <= 16) return launch_stream<1, 4, F8, FX, FW>(a, stream);
    if (a.M <= 32) return launch_stream<2, 2, F8, FX, FW>(a, stream);
    return launch_stream<4, 2, F8, FX, FW>(a, stream);
  }
  if (tile == 0) return launch_tile<TileGeom<256, F8 ? 256 : 128, F8 ? 2 : 4, F8 ? 4 : 2>, F8, FX, FW>(a, splits, stream);
  if (tile == 1) return launch_tile<TileGeom<128, 128, 2, 2>, F8, FX, FW>(a, splits, stream);
  return launch_tile<TileGeom<64, 128, 1, 4>, F8, FX, FW>(a, splits, stream);
}

}  // namespace

template <int FX, int FW>
hipError_t launch_fp8(const Fp8Args& a, bool f8, int tile, int splits, hipStream_t stream) {
  return f8 ? launch_kind<true, FX, FW>(a, tile, splits, stream) : launch_kind<false, FX, FW>(a, tile, splits, stream);
}

}  // namespace tilec
