// One AdamW step over many tensors:
//   g = grad * grad_scale                      (a clipping coefficient, or 1)
//   p = p (1 - lr wd)
//   m = b1 m + (1 - b1) g        v = b2 v + (1 - b2) g g
//   p = p - (lr / (1 - b1^t)) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// p fp32 or bf16, grad fp32 or bf16, all arithmetic fp32; where asked for, a
// bf16 copy of the new p is written too (the weights of the next forward pass).
//
// The states m and v are fp32, or 8-bit codes with one fp32 scale per block
// of 256 values (of a tensor read flat; the last block may be shorter).  A
// block's scale is its largest magnitude, held exactly, and
//   m = sign(c) (c / 127)^2 scale,   c = -127 .. 127
//   v = (c / 255)^4 scale,           c = 0 .. 255
// so steps shrink towards zero: m's smallest is 6e-5 of the block's largest,
// v's 2e-10.  Codes are rounded to nearest, and a v that is not 0 never gets
// the code 0: a vanished v would turn whatever is left of m into a step of
// m / eps.  The update itself uses the m and v of this step before they are
// coded.
//
// Bound by HBM: p, grad, m and v are read once, p, m and v written once.  One
// launch serves up to kMaxTensors tensors, whose descriptions travel as
// kernel arguments; a workgroup takes 4096 consecutive values of one tensor,
// 16 a thread, with all its loads issued before the first result is needed.
// A wave's 64 threads hold 4 consecutive values each, 256 in all: one block,
// so a block's largest value is a reduction within the wave.
//
// No operation is contracted (a product and a sum round separately), so that
// the codes can be reproduced exactly outside.
#include <algorithm>
#include <cmath>

#include "abi.h"
#include "common.h"
#include "../../include/tilec.h"

namespace tilec {

namespace {

typedef unsigned short u16;
typedef int i32x2 __attribute__((ext_vector_type(2)));

constexpr int kBlock = 256;       // values per scale
constexpr int kChunk = 4096;      // values per workgroup
constexpr int kMaxTensors = 48;   // per launch: 3.4 KiB of arguments

struct Tensor {
  void* p;
  const void* g;
  void *m, *v;         // fp32, or codes
  float *ms, *vs;      // scales of the codes
  u16* copy;           // or NULL
  int64_t n;
  int first;           // the tensor's first workgroup
  int types;           // bit 0: p is bf16, bit 1: g is bf16
};

struct AdamwArgs {
  int count;
  float decay, b1, c1, b2, c2, inv_root, eps, rate;  // c1 = 1 - b1, c2 = 1 - b2
  const float* grad_scale;
  Tensor t[kMaxTensors];
};
static_assert(sizeof(AdamwArgs) <= 4096, "kernel arguments");

// 4 values from element i on, at the element's own alignment; `n` of them.
__device__ __forceinline__ f32x4 load4(const float* p, int n) {
  if (n >= 4) {
    typedef f32x4 __attribute__((aligned(4))) any;
    return *reinterpret_cast<const any*>(p);
  }
  return f32x4{n > 0 ? p[0] : 0.f, n > 1 ? p[1] : 0.f, n > 2 ? p[2] : 0.f, 0.f};
}
__device__ __forceinline__ f32x4 load4(const u16* p, int n) {
  uint32_t a = 0, b = 0;
  if (n >= 4) {
    typedef i32x2 __attribute__((aligned(2))) any;
    const i32x2 w = *reinterpret_cast<const any*>(p);
    a = (uint32_t)w.x, b = (uint32_t)w.y;
  } else {
    if (n > 0) a = p[0];
    if (n > 1) a |= (uint32_t)p[1] << 16;
    if (n > 2) b = p[2];
  }
  return f32x4{__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u), __uint_as_float(b << 16),
               __uint_as_float(b & 0xffff0000u)};
}
__device__ __forceinline__ uint32_t load4(const unsigned char* p, int n) {
  if (n >= 4) {
    typedef uint32_t __attribute__((aligned(1))) any;
    return *reinterpret_cast<const any*>(p);
  }
  return (n > 0 ? p[0] : 0u) | (n > 1 ? (uint32_t)p[1] << 8 : 0u) | (n > 2 ? (uint32_t)p[2] << 16 : 0u);
}
__device__ __forceinline__ void store4(float* p, int n, f32x4 v) {
  if (n >= 4) {
    typedef f32x4 __attribute__((aligned(4))) any;
    *reinterpret_cast<any*>(p) = v;
    return;
  }
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (i < n) p[i] = v[i];
}
__device__ __forceinline__ void store4(u16* p, int n, f32x4 v) {
  u16 b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) b[i] = __builtin_bit_cast(u16, (__bf16)v[i]);  // to nearest, ties to even
  if (n >= 4) {
    typedef i32x2 __attribute__((aligned(2))) any;
    *reinterpret_cast<any*>(p) = i32x2{(int)(b[0] | (uint32_t)b[1] << 16), (int)(b[2] | (uint32_t)b[3] << 16)};
    return;
  }
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (i < n) p[i] = b[i];
}
__device__ __forceinline__ void store4(unsigned char* p, int n, uint32_t v) {
  if (n >= 4) {
    typedef uint32_t __attribute__((aligned(1))) any;
    *reinterpret_cast<any*>(p) = v;
    return;
  }
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (i < n) p[i] = (unsigned char)(v >> (8 * i));
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float u = __shfl_xor(v, o);
    v = u > v || u != u ? u : v;  // a NaN stays: it must spoil the block's scale
  }
  return v;
}

__device__ __forceinline__ float m_value(int code, float scale) {
#pragma clang fp contract(off)
  const float t = (float)code * (1.f / 127.f);
  return t * fabsf(t) * scale;
}
__device__ __forceinline__ float v_value(uint32_t code, float scale) {
#pragma clang fp contract(off)
  float t = (float)code * (1.f / 255.f);
  t = t * t;
  return t * t * scale;
}
__device__ __forceinline__ f32x4 m_values(uint32_t codes, float scale) {
  f32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = m_value((int)(codes << (24 - 8 * i)) >> 24, scale);
  return r;
}
__device__ __forceinline__ f32x4 v_values(uint32_t codes, float scale) {
  f32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = v_value(codes >> (8 * i) & 255u, scale);
  return r;
}

// The codes of 4 values; scale > 0, or 1 for a block of zeros.  The code is by
// definition that of correctly rounded quotients and roots, which are long
// sequences; an approximation (a product with 1 / scale and the hardware's
// root, together under 2^-21 of the result, so 2e-5 and 5e-5 of a code) settles
// all values but those within 1e-4 of a code from halfway between two, two in
// ten thousand.  Scales outside 2^-60 .. 2^100, where the approximation could
// leave the range of normal numbers, go the long way.  (151 M values: 496 us,
// 627 with the long way for all.)
__device__ __forceinline__ bool plain_scale(float s) { return s >= 0x1p-60f && s <= 0x1p100f; }
__device__ __forceinline__ bool near_half(float t) { return fabsf(fabsf(t - rintf(t)) - 0.5f) < 1e-4f; }

__device__ __forceinline__ uint32_t m_codes(f32x4 m, float scale) {
#pragma clang fp contract(off)
  float t[4];
  const float inv = 1.f / scale;
  bool exact = !plain_scale(scale);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    t[i] = __builtin_amdgcn_sqrtf(fabsf(m[i]) * inv) * 127.f;
    exact |= near_half(t[i]);
  }
  if (exact) {
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = sqrtf(fabsf(m[i]) / scale) * 127.f;
  }
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = (int)rintf(t[i]);
    w |= ((uint32_t)(m[i] < 0.f ? -c : c) & 255u) << (8 * i);
  }
  return w;
}
__device__ __forceinline__ uint32_t v_codes(f32x4 v, float scale) {
#pragma clang fp contract(off)
  float t[4];
  const float inv = 1.f / scale;
  bool exact = !plain_scale(scale);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    t[i] = __builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf(v[i] * inv)) * 255.f;
    exact |= near_half(t[i]);
  }
  if (exact) {
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = sqrtf(sqrtf(v[i] / scale)) * 255.f;
  }
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    int c = (int)rintf(t[i]);
    c = v[i] > 0.f && c < 1 ? 1 : c;
    w |= ((uint32_t)c & 255u) << (8 * i);
  }
  return w;
}

__device__ __forceinline__ int find(const AdamwArgs& a, int block) {
  int lo = 0, hi = a.count;  // t[lo].first <= block < t[hi].first
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.t[mid].first <= block) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <bool BITS8>
__global__ __launch_bounds__(256) void adamw_kernel(AdamwArgs a) {
#pragma clang fp contract(off)
  const Tensor& t = a.t[find(a, blockIdx.x)];
  const int64_t base = (int64_t)((int)blockIdx.x - t.first) * kChunk + 4 * threadIdx.x;
  constexpr int IT = kChunk / 1024;
  const float gs = a.grad_scale != nullptr ? *a.grad_scale : 1.f;
  f32x4 p[IT], g[IT], m[IT], v[IT];
  uint32_t mc[IT], vc[IT];
  float ms[IT], vs[IT];
  int n[IT];
#pragma unroll
  for (int k = 0; k < IT; ++k) {
    const int64_t i = base + 1024 * k;
    n[k] = (int)max((int64_t)0, min((int64_t)4, t.n - i));
    const int64_t at = n[k] > 0 ? i : 0;
    p[k] = (t.types & 1) ? load4(static_cast<const u16*>(t.p) + at, n[k]) : load4(static_cast<const float*>(t.p) + at, n[k]);
    g[k] = (t.types & 2) ? load4(static_cast<const u16*>(t.g) + at, n[k]) : load4(static_cast<const float*>(t.g) + at, n[k]);
    if constexpr (BITS8) {
      mc[k] = load4(static_cast<const unsigned char*>(t.m) + at, n[k]);
      vc[k] = load4(static_cast<const unsigned char*>(t.v) + at, n[k]);
      ms[k] = t.ms[at / kBlock];
      vs[k] = t.vs[at / kBlock];
    } else {
      m[k] = load4(static_cast<const float*>(t.m) + at, n[k]);
      v[k] = load4(static_cast<const float*>(t.v) + at, n[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < IT; ++k) {
    const int64_t i = base + 1024 * k;
    if constexpr (BITS8) {
      m[k] = m_values(mc[k], ms[k]);
      v[k] = v_values(vc[k], vs[k]);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float gr = a.grad_scale != nullptr ? g[k][c] * gs : g[k][c];
      const float q = p[k][c] * a.decay;
      m[k][c] = m[k][c] * a.b1 + gr * a.c1;
      v[k][c] = v[k][c] * a.b2 + gr * a.c2 * gr;
      const float denom = sqrtf(v[k][c]) * a.inv_root + a.eps;
      p[k][c] = q - m[k][c] / denom * a.rate;
    }
    if constexpr (BITS8) {
      // Values past the tensor's end (all of them zeros before) stay out.
      float tm = 0.f, tv = 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float am = c < n[k] ? fabsf(m[k][c]) : 0.f, av = c < n[k] ? v[k][c] : 0.f;
        tm = am > tm || am != am ? am : tm;
        tv = av > tv || av != av ? av : tv;
      }
      tm = wave_max(tm);
      tv = wave_max(tv);
      if (n[k] > 0) {
        store4(static_cast<unsigned char*>(t.m) + i, n[k], m_codes(m[k], tm > 0.f ? tm : 1.f));
        store4(static_cast<unsigned char*>(t.v) + i, n[k], v_codes(v[k], tv > 0.f ? tv : 1.f));
        if ((threadIdx.x & 63) == 0) {
          t.ms[i / kBlock] = tm;
          t.vs[i / kBlock] = tv;
        }
      }
    } else if (n[k] > 0) {
      store4(static_cast<float*>(t.m) + i, n[k], m[k]);
      store4(static_cast<float*>(t.v) + i, n[k], v[k]);
    }
    if (n[k] <= 0) continue;
    if (t.types & 1) store4(static_cast<u16*>(t.p) + i, n[k], p[k]);
    else store4(static_cast<float*>(t.p) + i, n[k], p[k]);
    if (t.copy != nullptr) store4(t.copy + i, n[k], p[k]);
  }
}

// The values that 8-bit states stand for.  types bit 0: v's codes (else m's).
__global__ __launch_bounds__(256) void adamw_values_kernel(AdamwArgs a) {
  const Tensor& t = a.t[find(a, blockIdx.x)];
  const int64_t base = (int64_t)((int)blockIdx.x - t.first) * kChunk + 4 * threadIdx.x;
#pragma unroll
  for (int k = 0; k < kChunk / 1024; ++k) {
    const int64_t i = base + 1024 * k;
    const int n = (int)max((int64_t)0, min((int64_t)4, t.n - i));
    if (n <= 0) continue;
    const uint32_t c = load4(static_cast<const unsigned char*>(t.g) + i, n);
    const float s = t.ms[i / kBlock];
    store4(static_cast<float*>(t.p) + i, n, (t.types & 1) ? v_values(c, s) : m_values(c, s));
  }
}

// Launch `f` for the tensors in groups of up to kMaxTensors, with at most
// 2^22 workgroups each.
template <typename F>
hipError_t in_groups(AdamwArgs& a, const tilec_adamw_tensor* tensors, int count, F f) {
  constexpr int64_t kMaxBlocks = int64_t(1) << 22;
  int64_t blocks = 0;
  a.count = 0;
  auto flush = [&]() -> hipError_t {
    if (a.count == 0) return hipSuccess;
    f((unsigned)blocks);
    a.count = 0;
    blocks = 0;
    return hipGetLastError();
  };
  for (int i = 0; i < count; ++i) {
    const tilec_adamw_tensor& s = tensors[i];
    // A tensor of more than kMaxBlocks chunks goes in pieces.
    for (int64_t at = 0; at < s.n; at += kMaxBlocks * kChunk) {
      const int64_t n = std::min(s.n - at, kMaxBlocks * kChunk), need = cdiv(n, kChunk);
      if (a.count == kMaxTensors || blocks + need > kMaxBlocks) {
        const hipError_t e = flush();
        if (e != hipSuccess) return e;
      }
      a.t[a.count] = f(s, at, n);
      a.t[a.count].first = (int)blocks;
      ++a.count;
      blocks += need;
    }
  }
  return flush();
}

char* offset(void* p, int64_t bytes) { return static_cast<char*>(p) + bytes; }

struct Step {
  AdamwArgs& a;
  bool bits8;
  hipStream_t stream;
  void operator()(unsigned blocks) const {
    if (bits8) hipLaunchKernelGGL(adamw_kernel<true>, dim3(blocks), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL(adamw_kernel<false>, dim3(blocks), dim3(256), 0, stream, a);
  }
  Tensor operator()(const tilec_adamw_tensor& s, int64_t at, int64_t n) const {
    const int64_t psz = s.param_dtype == TILEC_BF16 ? 2 : 4, gsz = s.grad_dtype == TILEC_BF16 ? 2 : 4;
    const int64_t ssz = bits8 ? 1 : 4;
    Tensor t{};
    t.p = offset(s.param, at * psz);
    t.g = offset(const_cast<void*>(s.grad), at * gsz);
    t.m = offset(s.exp_avg, at * ssz);
    t.v = offset(s.exp_avg_sq, at * ssz);
    t.ms = bits8 ? s.exp_avg_scale + at / kBlock : nullptr;
    t.vs = bits8 ? s.exp_avg_sq_scale + at / kBlock : nullptr;
    t.copy = s.copy ? static_cast<u16*>(s.copy) + at : nullptr;
    t.n = n;
    t.types = (s.param_dtype == TILEC_BF16 ? 1 : 0) | (s.grad_dtype == TILEC_BF16 ? 2 : 0);
    return t;
  }
};

struct Values {
  AdamwArgs& a;
  hipStream_t stream;
  void operator()(unsigned blocks) const {
    hipLaunchKernelGGL(adamw_values_kernel, dim3(blocks), dim3(256), 0, stream, a);
  }
  Tensor operator()(const tilec_adamw_tensor& s, int64_t at, int64_t n) const {
    Tensor t{};
    const bool sq = s.exp_avg == nullptr;
    t.p = offset(s.param, at * 4);
    t.g = offset(sq ? s.exp_avg_sq : s.exp_avg, at);
    t.ms = (sq ? s.exp_avg_sq_scale : s.exp_avg_scale) + at / kBlock;
    t.n = n;
    t.types = sq;
    return t;
  }
};

}  // namespace

}  // namespace tilec

using namespace tilec;

extern "C" {

int tilec_adamw(const tilec_adamw_tensor* tensors, int32_t count, int32_t state_bits, int64_t step, double lr,
                double beta1, double beta2, double eps, double weight_decay, const float* grad_scale, void* stream) {
  clear_error();
  if (count < 0 || (count > 0 && tensors == nullptr))
    return fail(TILEC_ERR_VALUE, "tilec: AdamW: no tensors (count %d)", count);
  if (state_bits != 32 && state_bits != 8)
    return fail(TILEC_ERR_VALUE, "tilec: AdamW: states have 32 or 8 bits (got %d)", state_bits);
  if (step < 1) return fail(TILEC_ERR_VALUE, "tilec: AdamW: steps count from 1 (got %lld)", (long long)step);
  if (!(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && eps >= 0 && lr >= 0 && weight_decay >= 0))
    return fail(TILEC_ERR_VALUE, "tilec: AdamW: lr=%g betas=(%g, %g) eps=%g weight_decay=%g out of range", lr, beta1,
                beta2, eps, weight_decay);
  for (int i = 0; i < count; ++i) {
    const tilec_adamw_tensor& s = tensors[i];
    if (s.n < 0) return fail(TILEC_ERR_VALUE, "tilec: AdamW: tensor %d has %lld elements", i, (long long)s.n);
    if ((s.param_dtype != TILEC_F32 && s.param_dtype != TILEC_BF16) ||
        (s.grad_dtype != TILEC_F32 && s.grad_dtype != TILEC_BF16))
      return fail(TILEC_ERR_TYPE, "tilec: AdamW: tensor %d: unsupported dtype codes %d, %d (use float32 or bfloat16)",
                  i, s.param_dtype, s.grad_dtype);
    if (s.n > 0 && (!s.param || !s.grad || !s.exp_avg || !s.exp_avg_sq ||
                    (state_bits == 8 && (!s.exp_avg_scale || !s.exp_avg_sq_scale))))
      return fail(TILEC_ERR_VALUE, "tilec: AdamW: tensor %d has a NULL pointer", i);
  }
  AdamwArgs a{};
  a.decay = (float)(1 - lr * weight_decay);
  a.b1 = (float)beta1, a.c1 = (float)(1 - beta1), a.b2 = (float)beta2, a.c2 = (float)(1 - beta2);
  a.inv_root = (float)(1 / std::sqrt(1 - std::pow(beta2, (double)step)));
  a.eps = (float)eps;
  a.rate = (float)(lr / (1 - std::pow(beta1, (double)step)));
  a.grad_scale = grad_scale;
  const hipError_t e = in_groups(a, tensors, count, Step{a, state_bits == 8, static_cast<hipStream_t>(stream)});
  if (e != hipSuccess) return fail(TILEC_ERR_HIP, "tilec: launching the AdamW step failed: %s", hipGetErrorString(e));
  return TILEC_OK;
}

int tilec_adamw_values(const tilec_adamw_tensor* tensors, int32_t count, void* stream) {
  clear_error();
  if (count < 0 || (count > 0 && tensors == nullptr))
    return fail(TILEC_ERR_VALUE, "tilec: AdamW values: no tensors (count %d)", count);
  for (int i = 0; i < count; ++i) {
    const tilec_adamw_tensor& s = tensors[i];
    if (s.n < 0 || (s.n > 0 && (!s.param || !((s.exp_avg && s.exp_avg_scale) || (s.exp_avg_sq && s.exp_avg_sq_scale)))))
      return fail(TILEC_ERR_VALUE, "tilec: AdamW values: tensor %d has a NULL pointer or %lld elements", i,
                  (long long)s.n);
  }
  AdamwArgs a{};
  const hipError_t e = in_groups(a, tensors, count, Values{a, static_cast<hipStream_t>(stream)});
  if (e != hipSuccess) return fail(TILEC_ERR_HIP, "tilec: launching the AdamW values failed: %s", hipGetErrorString(e));
  return TILEC_OK;
}

}  // extern "C"
