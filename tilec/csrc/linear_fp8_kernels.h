// The kernels of linear_fp8.h, for one pair of formats a file.
#pragma once

#include <type_traits>

#include "enqueue.h"
#include "linear_fp8.h"

namespace tilec {

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void* lds_ptr_t;

constexpr int kReadOnce = 2;  // cache policy: non-temporal

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

template <int BM_, int BN_, int WM_, int WN_, int NBUF_>
struct TileGeom {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, NBUF = NBUF_;
  static constexpr int NW = WM * WN, NT = 64 * NW;
  static constexpr int MT = BM / WM / 16, NB = BN / WN / 16;  // blocks of a wave
  static constexpr int XI = BM * 8 / NT, WI = BN * 8 / NT;    // 16-byte copies a thread and step
  static constexpr int SI = (BM + BN + NT - 1) / NT;          // scales a thread and step
  static constexpr int W_AT = BM * 128, S_AT = W_AT + BN * 128, STAGE = S_AT + SI * NT * 4;  // of a stage
  static_assert(BM * 8 % NT == 0 && BN * 8 % NT == 0 && BM % 64 == 0 && BN % 64 == 0, "whole copies");
  static_assert(BN / WN <= 128 && 128 % (BN / WN) == 0, "a wave's columns lie in one tile of w");
  static_assert(NBUF * STAGE <= 160 * 1024 && (NBUF == 2 || NBUF == 4), "LDS is 160 KiB");
};

// BM x BN outputs a workgroup, a group of 128 k a step, NBUF stages: the codes and
// scales of up to NBUF steps are on their way (global to LDS, 16 bytes a lane) while
// one is multiplied, and a wave reads its operands from LDS a step before it
// multiplies them.  A stage holds rows of 128 bytes whose 16-byte chunks are
// exchanged by (row / 2) % 8, so that 16 rows' reads spread over the banks.  What
// lies past M, N or K is never read: those copies have an address out of range and
// leave zeros; where K ends inside a chunk the rest of it is cleared in LDS before
// the last step's operands are read.
//
// A step of 128 x 128 takes 0.5 us: 8 waves read 96 KiB and the copies write 36 KiB,
// which LDS passes on at 128 bytes a clock; without any copies it takes as long, and
// the copies alone take as long too where rows begin at multiples of 128 bytes (1.45
// times where they do not, two lines a row).
template <class P, bool F8, int FX, int FW, bool WROWS>
__global__ __launch_bounds__(P::NT, 1) void fp8_tile_kernel(Fp8Args a) {
  // Objects of their own, so that the compiler knows which copies a read waits for.
  __shared__ __align__(16) char lds0[P::STAGE];
  __shared__ __align__(16) char lds1[P::STAGE];
  __shared__ __align__(16) char lds2[P::NBUF > 2 ? P::STAGE : 16];
  __shared__ __align__(16) char lds3[P::NBUF > 3 ? P::STAGE : 16];
  auto slot = [&](auto i) -> char* {
    constexpr int k = decltype(i)::value % P::NBUF;
    if constexpr (k == 0) return lds0;
    else if constexpr (k == 1) return lds1;
    else if constexpr (k == 2) return lds2;
    else return lds3;
  };
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
    off_s[i] = 4u * (uint32_t)(((r0 + e) >> shift) - (r0 >> shift)) * (uint32_t)(is_x ? a.sx_row : a.sw_row) |
               oob_unless(r0 + e < (is_x ? a.M : a.N) && (is_x || e < P::BN));
  }
  const unsigned char* const xb = a.x + (int64_t)m0 * a.ldx + (int64_t)g0 * kGroup;
  const unsigned char* const wb = a.w + (int64_t)n0 * a.ldw + (int64_t)g0 * kGroup;
  const float* const sxb = a.sx + (int64_t)(m0 >> a.xshift) * a.sx_row + (int64_t)g0 * a.sx_group;
  const float* const swb = a.sw + (int64_t)(n0 >> a.wshift) * a.sw_row + (int64_t)g0 * a.sw_group;
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
      const BufRsrc rs = make_rsrc_uniform(first < P::BM ? sxb + kt * a.sx_group : swb + kt * a.sw_group, records);
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
  // What a wave multiplies in a step, read from LDS a step ahead.
  struct Operands {
    i32x4 w[P::NB][2], x[P::MT][2];
    f32x4 s4[P::NB];
    float sx[P::MT], sw;
  };
  Operands ops[2];
  auto read = [&](const char* st, Operands& o) __attribute__((always_inline)) {
    const char* const xs = st + 128 * (wm * (P::BM / P::WM)) + at;
    const char* const ws = st + P::W_AT + 128 * (wn * (P::BN / P::WN)) + at;
    const char* const xs2 = st + 128 * (wm * (P::BM / P::WM)) + (at ^ 64);
    const char* const ws2 = st + P::W_AT + 128 * (wn * (P::BN / P::WN)) + (at ^ 64);
    const float* const ssx = reinterpret_cast<const float*>(st + P::S_AT) + wm * (P::BM / P::WM) + row;
    const float* const ssw = reinterpret_cast<const float*>(st + P::S_AT) + P::BM + wn * (P::BN / P::WN);
#pragma unroll
    for (int j = 0; j < P::NB; ++j) {
      o.w[j][0] = *reinterpret_cast<const i32x4*>(ws + 2048 * j);
      o.w[j][1] = *reinterpret_cast<const i32x4*>(ws2 + 2048 * j);
      if constexpr (WROWS) o.s4[j] = *reinterpret_cast<const f32x4*>(ssw + 16 * j + 4 * quad);
    }
    if constexpr (!WROWS) o.sw = *ssw;
#pragma unroll
    for (int i = 0; i < P::MT; ++i) {
      o.x[i][0] = *reinterpret_cast<const i32x4*>(xs + 2048 * i);
      o.x[i][1] = *reinterpret_cast<const i32x4*>(xs2 + 2048 * i);
      o.sx[i] = ssx[16 * i];
    }
  };
  // A block's P_g on the matrix core, beside it the multiply-adds of the one before last.
  auto multiply = [&](const Operands& o) __attribute__((always_inline)) {
    constexpr int LAG = 2, BLOCKS = P::MT * P::NB;
    Frag<F8, FW> fw[P::NB];
    Frag<F8, FX> fx;
    f32x4 p[LAG + 1];
#pragma unroll
    for (int b = 0; b < BLOCKS + LAG; ++b) {
      if (b < BLOCKS) {
        const int i = b / P::NB, j = b % P::NB;
        if (i == 0) fw[j].set(o.w[j][0], o.w[j][1]);
        if (j == 0) fx.set(o.x[i][0], o.x[i][1]);
        p[b % (LAG + 1)] = block<FX, FW>(fw[j], fx);
      }
      if (b >= LAG) {
        const int i = (b - LAG) / P::NB, j = (b - LAG) % P::NB;
        const float s = WROWS ? o.sx[i] : o.sx[i] * o.sw;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          acc[i][j][r] = fmaf(p[(b - LAG) % (LAG + 1)][r], WROWS ? s * o.s4[j][r] : s, acc[i][j][r]);
      }
      __builtin_amdgcn_sched_barrier(0);  // (else the multiply-adds move up to their block and wait for it)
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
  // This wave's copies are there but for the last `later` steps', and its reads are
  // done: then everybody's.
  auto arrive = [&](auto later) __attribute__((always_inline)) {
    constexpr int n = decltype(later)::value * (P::XI + P::WI + P::SI);
    static_assert(n < 64, "vmcnt has 6 bits");
    __builtin_amdgcn_s_waitcnt(0x0070 | (n & 15) | (n >> 4) << 14);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  using std::integral_constant;
  // Step kt, whose operands are in registers; its stage takes the copies of step
  // kt + NBUF.
  auto step = [&](auto i, int kt) __attribute__((always_inline)) {
    constexpr int k = decltype(i)::value;
    arrive(integral_constant<int, P::NBUF - 2>{});
    read(slot(integral_constant<int, k + 1>{}), ops[(k + 1) & 1]);
    copy(kt + P::NBUF, slot(i));
    __builtin_amdgcn_sched_barrier(0);
    multiply(ops[k & 1]);
    __builtin_amdgcn_sched_barrier(0);
  };
  if (nk > 0) {
    copy(0, lds0);
    copy(1, lds1);
    if constexpr (P::NBUF > 2) copy(2, lds2);
    if constexpr (P::NBUF > 3) copy(3, lds3);
    arrive(integral_constant<int, P::NBUF - 1>{});
    const bool tail = (a.K & 15) != 0 && g0 + nk == a.G;
    if (tail && nk == 1) {
      clear_tail(lds0);
      __syncthreads();
    }
    read(lds0, ops[0]);
    // All steps but the last two, whose operands may need clearing.
    int kt = 0;
#pragma unroll 1
    for (; kt + P::NBUF + 1 < nk; kt += P::NBUF) {
      step(integral_constant<int, 0>{}, kt);
      step(integral_constant<int, 1>{}, kt + 1);
      if constexpr (P::NBUF > 2) step(integral_constant<int, 2>{}, kt + 2);
      if constexpr (P::NBUF > 3) step(integral_constant<int, 3>{}, kt + 3);
    }
    // Up to NBUF + 1 steps are left, of which all copies but one's are on their way.
    auto rest = [&](auto i) __attribute__((always_inline)) {
      constexpr int k = decltype(i)::value;
      if (kt >= nk) return;
      if (kt + 1 < nk) {
        arrive(integral_constant<int, k == 0 ? P::NBUF - 2 : 0>{});
        char* const next = slot(integral_constant<int, k + 1>{});
        if (tail && kt + 2 == nk) {
          clear_tail(next);
          __syncthreads();
        }
        read(next, ops[(k + 1) & 1]);
        if constexpr (k == 0) copy(kt + P::NBUF, slot(i));
      }
      multiply(ops[k & 1]);
      ++kt;
    };
    rest(integral_constant<int, 0>{});
    rest(integral_constant<int, 1>{});
    rest(integral_constant<int, 2>{});
    if constexpr (P::NBUF > 2) rest(integral_constant<int, 3>{});
    if constexpr (P::NBUF > 3) rest(integral_constant<int, 4>{});
  }

  const int mw = m0 + wm * (P::BM / P::WM) + row, nw = n0 + wn * (P::BN / P::WN) + 4 * quad;
  if (gridDim.y > 1) {  // the split that comes last adds them all up, in order
    __shared__ int last;
    constexpr int NV = P::MT * P::NB;
    f32x4 v[NV];
    bool live[NV];
#pragma unroll
    for (int b = 0; b < NV; ++b) {
      v[b] = acc[b / P::NB][b % P::NB];
      live[b] = (mw + 16 * (b / P::NB) < a.M) & (nw + 16 * (b % P::NB) < a.N);
    }
    if (!splitk_combine<P::NT, NV>(v, live, split, gridDim.y, blockIdx.x, gridDim.x, a.partial, a.counters, &last)) return;
#pragma unroll
    for (int b = 0; b < NV; ++b) acc[b / P::NB][b % P::NB] = v[b];
  }
  const bool inside = m0 + P::BM <= a.M && n0 + P::BN <= a.N;
  Out<F8>* const first = static_cast<Out<F8>*>(a.out) + (int64_t)mw * a.ldo;
#pragma unroll
  for (int i = 0; i < P::MT; ++i) {
    Out<F8>* const line = first + (int64_t)(16 * i) * a.ldo;
#pragma unroll
    for (int j = 0; j < P::NB; ++j)
      if (inside || mw + 16 * i < a.M) store4<Out<F8>>(line, nw + 16 * j, inside ? INT32_MAX : a.N, acc[i][j]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// The same product for large outputs: 256 rows, and the eight waves in two groups
// of four, one wave of each on every SIMD.  While one group multiplies, the other
// reads its next operands from LDS; they change places at a barrier, so the matrix
// cores are never without a wave whose operands are in registers.  In half step 2 k
// the first group reads step k and the second multiplies step k - 1, in half step
// 2 k + 1 the first multiplies step k and the second reads it.
//
// Two stages.  A group's own rows of x are read until it has multiplied the step, w
// and the scales until the second group has read it.  So in half step 2 k the first
// group may copy w, the scales and its rows of x of step k + 1, in half step 2 k + 1
// the second group its own rows of x; each wave waits for its copies before the
// barrier that ends its multiplying, two half steps later.  (Each group has a loop
// of its own: one loop with a branch around the copies left the compiler without
// registers.)
//
// 8192^3 with tiles of w: 465-494 us, 2226-2365 TFLOP/s, from run to run; a
// library's plain 8-bit product with one scale takes 399.  In runs that gave 460-470:
// fp8_tile_kernel with this tile, whose waves all read and then all multiply, 540-550;
// copies after the reads of a half step instead of before 486; w copied by the second
// group between its multiplications 500.  The clock is at 1.9 GHz (2.4 without load):
// what bounds it is power, with the matrix cores busy in 60 % of the cycles.
// With scales of w's rows a lane holds four of every block column: for bf16 outputs 6
// registers more than there are (28 bytes of scratch), and a reload waits for all
// vector memory, the next step's copies among it: 640 us at 8192^3.  (fp32 outputs
// have half the sums and spill nothing: 901 us with tiles of w, 1050 with rows.)
template <class P, bool F8, int FX, int FW, bool WROWS>
__global__ __launch_bounds__(512, 1) void fp8_pair_kernel(Fp8Args a) {
  static_assert(P::NW == 8, "two groups of four waves");
  // Copies of a thread: the second group's of its own rows of x, the first's of all else.
  constexpr int XI = P::BM * 4 / 256, WI = P::BN * 8 / 256, SI = (P::BM + P::BN + 255) / 256;
  // Rows of x in registers, refilled while multiplying, and blocks whose sums are
  // under way.
  constexpr int RING = F8 && WROWS ? 2 : 3, LAG = 2;
  // Objects of their own, so that the compiler knows which copies a read waits for.
  __shared__ __align__(16) char x0[P::BM * 128];
  __shared__ __align__(16) char x1[P::BM * 128];
  __shared__ __align__(16) char w0[P::BN * 128];
  __shared__ __align__(16) char w1[P::BN * 128];
  __shared__ __align__(16) float s0[SI * 256];
  __shared__ __align__(16) float s1[SI * 256];
  struct Stage {
    char *x, *w;
    float* s;
  };
  const Stage st0 = {x0, w0, s0}, st1 = {x1, w1, s1};
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), group = wave >> 2, w4 = wave & 3;
  const int wm = wave / P::WN, wn = wave % P::WN;
  const int tiles_m = (a.M + P::BM - 1) / P::BM, tiles_n = (a.N + P::BN - 1) / P::BN;
  int tm, tn;
  tile_of(blockIdx.x, a.xcds, tiles_m, tiles_n, a.group_m, tm, tn);
  const int m0 = tm * P::BM, n0 = tn * P::BN;
  const int nk = a.G;

  const int c0 = (lane & 7) ^ (lane >> 4);
  const uint32_t row8 = lane >> 3;
  const uint32_t rx8 = (P::BM / 2 * group + 8u * XI * w4 + row8) * (uint32_t)a.ldx, rw8 = (8u * WI * w4 + row8) * (uint32_t)a.ldw;
  const uint32_t vx[2] = {rx8 + 16u * c0, rx8 + 16u * (c0 ^ 4)}, vw[2] = {rw8 + 16u * c0, rw8 + 16u * (c0 ^ 4)};
  const uint32_t sx8 = 8u * (uint32_t)a.ldx, sw8 = 8u * (uint32_t)a.ldw;
  uint32_t off_s[SI];
#pragma unroll
  for (int i = 0; i < SI; ++i) {
    const int first = 64 * (w4 * SI + i);
    const bool is_x = first < P::BM;
    const int e = first + lane - (is_x ? 0 : P::BM), shift = is_x ? a.xshift : a.wshift, r0 = is_x ? m0 : n0;
    off_s[i] = 4u * (uint32_t)(((r0 + e) >> shift) - (r0 >> shift)) * (uint32_t)(is_x ? a.sx_row : a.sw_row) |
               oob_unless(r0 + e < (is_x ? a.M : a.N) && (is_x || e < P::BN));
  }
  const unsigned char* const xb = a.x + (int64_t)m0 * a.ldx;
  const unsigned char* const wb = a.w + (int64_t)n0 * a.ldw;
  const float* const sxb = a.sx + (int64_t)(m0 >> a.xshift) * a.sx_row;
  const float* const swb = a.sw + (int64_t)(n0 >> a.wshift) * a.sw_row;
  // Bytes of the tile's rows: what lies past the last row is past the end.
  const uint32_t x_bytes = a.M - m0 >= P::BM ? 0x7FFFFFFFu : (uint32_t)(a.M - m0) * (uint32_t)a.ldx;
  const uint32_t w_bytes = a.N - n0 >= P::BN ? 0x7FFFFFFFu : (uint32_t)(a.N - n0) * (uint32_t)a.ldw;
  auto past_of = [&](int kt, uint32_t (&past)[2]) __attribute__((always_inline)) {
    const int left = a.K - kt * kGroup;
    past[0] = oob_unless(16 * c0 < left), past[1] = oob_unless(16 * (c0 ^ 4) < left);
  };
  auto rsrc_of = [&](const unsigned char* base, uint32_t n, int kt) __attribute__((always_inline)) {
    const uint32_t r = n == 0x7FFFFFFFu ? n : n - (uint32_t)(kt * kGroup);
    return make_rsrc_uniform(base + kt * kGroup, kt < nk ? r : 0u);
  };
  // A group's own half of x's rows.
  auto copy_x = [&](int kt, const Stage& st) __attribute__((always_inline)) {
    uint32_t past[2];
    past_of(kt, past);
    const BufRsrc rx = rsrc_of(xb, x_bytes, kt);
#pragma unroll
    for (int i = 0; i < XI; ++i) {
      const uint32_t off = (vx[i & 1] + i * sx8) | past[i & 1];
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (lds_ptr_t)(st.x + P::BM * 64 * group + 1024 * (w4 * XI + i)), 16, off, 0, 0, 0);
    }
  };
  auto copy_w = [&](const Stage& st, int i, BufRsrc rw, const uint32_t (&past)[2]) __attribute__((always_inline)) {
    const uint32_t off = (vw[i & 1] + i * sw8) | past[i & 1];
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (lds_ptr_t)(st.w + 1024 * (w4 * WI + i)), 16, off, 0, 0, 0);
  };
  auto copy_s = [&](int kt, const Stage& st) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < SI; ++i) {
      const int first = 64 * (w4 * SI + i);
      const uint32_t off = off_s[i];
      const BufRsrc rs = make_rsrc_uniform(first < P::BM ? sxb + kt * a.sx_group : swb + kt * a.sw_group, kt < nk ? 0x7FFFFFFFu : 0u);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)(st.s + first), 4, off, 0, 0, 0);
    }
  };

  auto copy = [&](auto first_t, int kt, const Stage& st) __attribute__((always_inline)) {
    copy_x(kt, st);
    if constexpr (decltype(first_t)::value) {
      uint32_t past[2];
      past_of(kt, past);
      const BufRsrc rw = rsrc_of(wb, w_bytes, kt);
#pragma unroll
      for (int i = 0; i < WI; ++i) copy_w(st, i, rw, past);
      copy_s(kt, st);
    }
  };
  f32x4 acc[P::MT][P::NB];
#pragma unroll
  for (int i = 0; i < P::MT; ++i)
#pragma unroll
    for (int j = 0; j < P::NB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int row = lane & 15, quad = lane >> 4;
  const int at = 128 * row + 16 * (quad ^ ((row >> 1) & 7));
  Frag<F8, FW> fw[P::NB];
  Frag<F8, FX> fx[RING];
  f32x4 p[LAG + 1], s4[P::NB];
  float s[P::MT];
#pragma unroll
  for (int j = 0; j <= LAG; ++j) p[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < P::NB; ++j) s4[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < P::MT; ++i) s[i] = 0.f;
  constexpr int BLOCKS = P::MT * P::NB;
  auto add = [&](int b) __attribute__((always_inline)) {  // block b's P_g to its sums
    const int i = b / P::NB, j = b % P::NB;
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[i][j][r] = fmaf(p[b % (LAG + 1)][r], WROWS ? s[i] * s4[j][r] : s[i], acc[i][j][r]);
  };
  auto change = [&]() __attribute__((always_inline)) {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  auto step = [&](auto first_t, auto last_t, int kt, const Stage& st, const Stage& next) __attribute__((always_inline)) {
    constexpr bool LAST = decltype(last_t)::value;
    const int left = a.K - kt * kGroup - 16 * quad;  // LAST: codes of the lane's first 16
    auto cut = [&](i32x4 v, int n) {
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const int keep = n - 4 * d;
        v[d] &= keep >= 4 ? ~0 : keep <= 0 ? 0 : (1 << (8 * keep)) - 1;
      }
      return v;
    };
    auto frag = [&](auto& f, const char* rows) __attribute__((always_inline)) {
      i32x4 lo = *reinterpret_cast<const i32x4*>(rows + at), hi = *reinterpret_cast<const i32x4*>(rows + (at ^ 64));
      if constexpr (LAST) lo = cut(lo, left), hi = cut(hi, left - 64);
      f.set(lo, hi);
    };
    const char* const xs = st.x + 128 * (wm * (P::BM / P::WM));
    const char* const ws = st.w + 128 * (wn * (P::BN / P::WN));
    const float* const ssx = st.s + wm * (P::BM / P::WM) + row;
    const float* const ssw = st.s + P::BM + wn * (P::BN / P::WN);
    // Reading, beside the other group's multiplying.
    if constexpr (!LAST) copy(first_t, kt + 1, next);
#pragma unroll
    for (int b = BLOCKS - LAG; b < BLOCKS; ++b) add(b);
#pragma unroll
    for (int j = 0; j < P::NB; ++j) frag(fw[j], ws + 2048 * j);
#pragma unroll
    for (int i = 0; i < RING; ++i) frag(fx[i], xs + 2048 * i);
    float sw1 = 1.f;
    if constexpr (WROWS) {
#pragma unroll
      for (int j = 0; j < P::NB; ++j) s4[j] = *reinterpret_cast<const f32x4*>(ssw + 16 * j + 4 * quad);
    } else {
      sw1 = *ssw;
    }
#pragma unroll
    for (int i = 0; i < P::MT; ++i) s[i] = ssx[16 * i] * sw1;
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    change();
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
      const int i = b / P::NB, j = b % P::NB;
      p[b % (LAG + 1)] = block<FX, FW>(fw[j], fx[i % RING]);
      if (b >= LAG) add(b - LAG);
      if (j == P::NB - 1 && i + RING < P::MT) frag(fx[i % RING], xs + 2048 * (i + RING));
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_s_waitcnt(0);
    change();
    __builtin_amdgcn_sched_barrier(0);
  };
  using std::integral_constant;
  if (nk > 0) {
    if (group == 0) copy(integral_constant<bool, true>{}, 0, st0);
    else copy(integral_constant<bool, false>{}, 0, st0);
    __builtin_amdgcn_s_waitcnt(0);
    change();
    if (group == 1) change();
    auto loop = [&](auto first_t) __attribute__((always_inline)) {
      int kt = 0;
#pragma unroll 1
      for (; kt + 2 < nk; kt += 2) {
        step(first_t, integral_constant<bool, false>{}, kt, st0, st1);
        step(first_t, integral_constant<bool, false>{}, kt + 1, st1, st0);
      }
      Stage last = st0;
      if (kt + 2 == nk) {
        step(first_t, integral_constant<bool, false>{}, kt, st0, st1);
        last = st1;
      }
      step(first_t, integral_constant<bool, true>{}, nk - 1, last, last);
    };
    if (group == 0) loop(integral_constant<bool, true>{});
    else loop(integral_constant<bool, false>{});
    if (group == 0) change();
#pragma unroll
    for (int b = BLOCKS - LAG; b < BLOCKS; ++b) add(b);
  }

  const bool inside = m0 + P::BM <= a.M && n0 + P::BN <= a.N;
  const int mw = m0 + wm * (P::BM / P::WM) + row, nw = n0 + wn * (P::BN / P::WN) + 4 * quad;
  Out<F8>* const first = static_cast<Out<F8>*>(a.out) + (int64_t)mw * a.ldo;
#pragma unroll
  for (int i = 0; i < P::MT; ++i) {
    Out<F8>* const line = first + (int64_t)(16 * i) * a.ldo;
#pragma unroll
    for (int j = 0; j < P::NB; ++j)
      if (inside || mw + 16 * i < a.M) store4<Out<F8>>(line, nw + 16 * j, inside ? INT32_MAX : a.N, acc[i][j]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Few rows of x, up to 8 XR: bound by reading w, once.  Tiles of 16 rows of w,
// workgroups that walk over tiles; a workgroup's NW waves take every NW-th group of a
// tile, and their sums meet in LDS, in order.  Every wave copies its own codes and
// scales through its own LDS, D groups at a time and across the ends of tiles,
// without a barrier: memory is then read in runs of 128 bytes, where operands loaded
// straight into registers, a row a lane, come in pieces of 16 (16 rows against 4096 x
// 4096 and 16384 x 4096, w from memory: 7.8 and 22.3 us so, 6.6 and 16.2 by way of
// LDS; one row: 6.2 and 15.5, 6.0 and 14.2).
template <int XR, int NW, int D, bool F8, int FX, int FW, bool WROWS>
__global__ __launch_bounds__(64 * NW, 1) void fp8_stream_kernel(Fp8Args a) {
  static_assert(XR == 1 || XR == 2, "one block of the matrix core");
  // A group's codes of w and x, then 64 scales of each.
  constexpr int X_AT = 2048, S_AT = X_AT + XR * 1024, SLOT = S_AT + 512, COPIES = 2 + XR + 2;
  static_assert((D - 1) * COPIES < 64, "vmcnt has 6 bits");
  __shared__ __align__(16) char ring[NW][D][SLOT];
  __shared__ f32x4 red[2][NW][64];
  const int tid = threadIdx.x, lane = tid & 63, row = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tiles = (a.N + 15) / 16, mine = (tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;
  const int turns = (a.G + NW - 1) / NW, items = mine * turns;  // groups of a wave: a tile's, and all (some past the last)

  const int c0 = (lane & 7) ^ (lane >> 4);
  uint32_t off_w[2], off_x[XR];
#pragma unroll
  for (int i = 0; i < 2; ++i) off_w[i] = (8 * i + (lane >> 3)) * (uint32_t)a.ldw + 16u * (c0 ^ 4 * i);
#pragma unroll
  for (int i = 0; i < XR; ++i) off_x[i] = (8 * i + (lane >> 3)) * (uint32_t)a.ldx + 16u * (c0 ^ 4 * i);
  const uint32_t off_sx = 4u * (uint32_t)(lane >> a.xshift) * (uint32_t)a.sx_row | oob_unless(lane < a.M);
  const uint32_t sw_step = 4u * (uint32_t)(lane >> a.wshift) * (uint32_t)a.sw_row;

  int tile = blockIdx.x, g = wave, left = items, to = 0;  // of the next copies
  auto copy = [&]() __attribute__((always_inline)) {
    const bool live = left > 0 && g < a.G;
    const int n0 = 16 * tile, skip = g * kGroup, rest = a.K - skip;
    const uint32_t past[2] = {oob_unless(16 * c0 < rest), oob_unless(16 * (c0 ^ 4) < rest)};
    const int64_t w_rows = a.N - n0 < 16 ? a.N - n0 : 16;
    const BufRsrc rw = make_rsrc_uniform(a.w + (int64_t)n0 * a.ldw + skip, live ? (uint32_t)(w_rows * a.ldw - skip) : 0u);
    const BufRsrc rx = make_rsrc_uniform(a.x + skip, live ? (uint32_t)(a.M * a.ldx - skip) : 0u);
    const BufRsrc rsx = make_rsrc_uniform(a.sx + g * a.sx_group, live ? 0x7FFFFFFFu : 0u);
    const BufRsrc rsw = make_rsrc_uniform(a.sw + (int64_t)(n0 >> a.wshift) * a.sw_row + g * a.sw_group, live ? 0x7FFFFFFFu : 0u);
    const uint32_t off_sw = sw_step | oob_unless(lane < w_rows);
    char* const at = ring[wave][to];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t off = off_w[j] | past[j];
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (lds_ptr_t)(at + 1024 * j), 16, off, 0, 0, kReadOnce);
    }
#pragma unroll
    for (int j = 0; j < XR; ++j) {
      const uint32_t off = off_x[j] | past[j];
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (lds_ptr_t)(at + X_AT + 1024 * j), 16, off, 0, 0, 0);
    }
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsx, (lds_ptr_t)(at + S_AT), 4, off_sx, 0, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsw, (lds_ptr_t)(at + S_AT + 256), 4, off_sw, 0, 0, 0);
    --left;
    to = to + 1 == D ? 0 : to + 1;
    g += NW;
    if (g >= turns * NW) g = wave, tile += gridDim.x;
  };
  auto cut = [&](i32x4 v, int n) {  // the first n bytes
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      const int keep = n - 4 * d;
      v[d] &= keep >= 4 ? ~0 : keep <= 0 ? 0 : (1 << (8 * keep)) - 1;
    }
    return v;
  };
  auto lds_of = [](const void* q) __attribute__((always_inline)) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)q;
  };
  // Where a lane reads in a slot.
  const uint32_t w_at = 128 * row + 16 * (quad ^ ((row >> 1) & 7));
  const int xr = XR == 2 ? row : row & 7;  // eight rows stand for themselves twice
  const uint32_t x_at = X_AT + 128 * xr + 16 * (quad ^ ((xr >> 1) & 7));
  const uint32_t sx_at = S_AT + 4 * xr, sw_at = S_AT + 256 + (WROWS ? 16 * quad : 0);

  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  int at_tile = blockIdx.x, at_g = wave, from = 0, half = 0;  // of the next group to multiply
#pragma unroll
  for (int i = 0; i < D; ++i) copy();
  // `items` is the same for every wave of the workgroup: so are its barriers.
#pragma unroll 1
  for (int i = 0; i < items; ++i) {
    // The group's copies are there, those of the D - 1 after it may be under way.
    // (LDS is read in assembly, wait included: before reads of its own the compiler
    // waits for every copy.)
    constexpr int n = (D - 1) * COPIES;
    __builtin_amdgcn_s_waitcnt(0x0f70 | (n & 15) | (n >> 4) << 14);
    const uint32_t base = lds_of(ring[wave][from]);
    i32x4 w0, w1, x0, x1;
    float sx;
    f32x4 sw;
    asm volatile(
        "ds_read_b128 %0, %6\n\tds_read_b128 %1, %7\n\tds_read_b128 %2, %8\n\tds_read_b128 %3, %9\n\t"
        "ds_read_b32 %4, %10\n\tds_read_b128 %5, %11\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(w0), "=&v"(w1), "=&v"(x0), "=&v"(x1), "=&v"(sx), "=&v"(sw)
        : "v"(base + w_at), "v"(base + (w_at ^ 64)), "v"(base + x_at), "v"(base + (x_at ^ 64)), "v"(base + sx_at),
          "v"(base + sw_at)
        : "memory");
    copy();
    from = from + 1 == D ? 0 : from + 1;
    if ((a.K & 15) != 0 && at_g == a.G - 1) {
      const int m = a.K - kGroup * at_g - 16 * quad;
      w0 = cut(w0, m), w1 = cut(w1, m - 64), x0 = cut(x0, m), x1 = cut(x1, m - 64);
    }
    Frag<F8, FW> fw;
    Frag<F8, FX> fx;
    fw.set(w0, w1);
    fx.set(x0, x1);
    const f32x4 p = block<FX, FW>(fw, fx);
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[r] = fmaf(p[r], sx * sw[WROWS ? r : 0], acc[r]);
    at_g += NW;
    if (at_g < turns * NW) continue;
    // The tile's last group.
    red[half][wave][lane] = acc;
    acc = f32x4{0.f, 0.f, 0.f, 0.f};
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): copies go on
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (wave == at_tile % NW) {
      f32x4 part[NW];
#pragma unroll
      for (int v = 0; v < NW; ++v) {
        const uint32_t q = lds_of(&red[half][v][lane]);
        asm volatile("ds_read_b128 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=&v"(part[v]) : "v"(q) : "memory");
      }
      f32x4 s = part[0];
#pragma unroll
      for (int v = 1; v < NW; ++v) s += part[v];
      if (row < a.M)
        store4<Out<F8>>(static_cast<Out<F8>*>(a.out) + (int64_t)row * a.ldo, 16 * at_tile + 4 * quad, a.N, s);
    }
    half ^= 1;
    at_g = wave, at_tile += gridDim.x;
  }
  __builtin_amdgcn_s_waitcnt(0);  // copies past the end leave zeros: not after the workgroup's LDS is another's
}

template <class P, bool F8, int FX, int FW>
hipError_t launch_tile(const Fp8Args& a, int splits, hipStream_t stream) {
  const dim3 grid((unsigned)(cdiv(a.M, P::BM) * cdiv(a.N, P::BN)), (unsigned)splits);
  const auto kernel = a.wshift == 0 ? fp8_tile_kernel<P, F8, FX, FW, true> : fp8_tile_kernel<P, F8, FX, FW, false>;
  return enqueue(kernel, grid, dim3(P::NT), stream, a);
}

template <class P, bool F8, int FX, int FW>
hipError_t launch_pair(const Fp8Args& a, hipStream_t stream) {
  const dim3 grid((unsigned)(cdiv(a.M, P::BM) * cdiv(a.N, P::BN)));
  const auto kernel = a.wshift == 0 ? fp8_pair_kernel<P, F8, FX, FW, true> : fp8_pair_kernel<P, F8, FX, FW, false>;
  return enqueue(kernel, grid, dim3(P::NT), stream, a);
}

template <int XR, int NW, bool F8, int FX, int FW>
hipError_t launch_stream(const Fp8Args& a, int64_t most, hipStream_t stream) {
  const dim3 grid((unsigned)std::min<int64_t>(cdiv(a.N, 16), most));
  const auto kernel = a.wshift == 0 ? fp8_stream_kernel<XR, NW, 2, F8, FX, FW, true> : fp8_stream_kernel<XR, NW, 2, F8, FX, FW, false>;
  return enqueue(kernel, grid, dim3(64 * NW), stream, a);
}

// Eight waves a tile while every workgroup has one tile (4096 x 4096, one row: 5.3
// us, 5.8 with four), four and three workgroups a CU where they have several (16384 x
// 4096: 13.5 us, 14.2 with eight; 16 rows: 15.8 and 18.6).
template <int XR, bool F8, int FX, int FW>
hipError_t launch_stream(const Fp8Args& a, hipStream_t stream) {
  const int64_t cus = device_cus();
  return cdiv(a.N, 16) <= 2 * cus ? launch_stream<XR, 8, F8, FX, FW>(a, 2 * cus, stream)
                                  : launch_stream<XR, 4, F8, FX, FW>(a, 3 * cus, stream);
}

template <bool F8, int FX, int FW>
hipError_t launch_kind(const Fp8Args& a, int tile, int splits, hipStream_t stream) {
  if (tile < 0) return a.M <= 8 ? launch_stream<1, F8, FX, FW>(a, stream) : launch_stream<2, F8, FX, FW>(a, stream);
  if (tile == 0) return launch_pair<TileGeom<256, F8 ? 256 : 128, F8 ? 2 : 4, F8 ? 4 : 2, 2>, F8, FX, FW>(a, stream);
  if (tile == 1) return launch_tile<TileGeom<128, 128, 2, 4, 4>, F8, FX, FW>(a, splits, stream);
  if (tile == 2) return launch_tile<TileGeom<64, 128, 2, 4, 4>, F8, FX, FW>(a, splits, stream);
  return launch_tile<TileGeom<64, 64, 2, 2, 4>, F8, FX, FW>(a, splits, stream);
}

}  // namespace

template <int FX, int FW>
hipError_t launch_fp8(const Fp8Args& a, bool f8, int tile, int splits, hipStream_t stream) {
  return f8 ? launch_kind<true, FX, FW>(a, tile, splits, stream) : launch_kind<false, FX, FW>(a, tile, splits, stream);
}

}  // namespace tilec
