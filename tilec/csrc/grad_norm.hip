// The norm of a list of gradients and the factor that clips it:
//   norm = |grad_scale| sqrt(sum over all values of g^2)
//   scale = grad_scale min(1, max_norm / (norm + 1e-6))
// and the gradients multiplied by that factor in place.
//
// Bound by HBM: every value is read once (clipping: once more, and written).  One
// launch serves up to kMaxTensors tensors, whose descriptions travel as kernel
// arguments; a workgroup adds up one chunk of one tensor.  Squares and sums are
// float64: nothing overflows, whatever the gradients, and nothing is lost; at two
// float64 operations a value the memory still sets the pace.  Every chunk's sum is
// a value of its own; the last workgroup of the call to finish (a counter, left
// zero) adds them in order, so the same bits come out every time, and writes both
// results: a second launch for that would cost a small model's norm half again.
#include <algorithm>
#include <cmath>

#include "abi.h"
#include "common.h"
#include "enqueue.h"
#include "../../include/tilec.h"

namespace tilec {

namespace {

typedef unsigned short u16;
typedef u32x4 __attribute__((aligned(2))) u32x4_any;

constexpr int kMaxTensors = 224;  // per launch: 3.6 KiB of arguments, of at most 4
constexpr int kUnit = 4096;       // chunks are a multiple of this

constexpr int64_t kMaxBlocks = int64_t(1) << 22;  // workgroups of a launch
constexpr int64_t kMaxPiece = int64_t(1) << 38;   // values of a piece of a tensor: at most kMaxBlocks chunks

// A tensor, or a piece of one: 16 bytes, since a launch takes the longer the more
// its arguments are.
struct Tensor {
  void* data;
  uint64_t packed;  // n (39 bits), the first workgroup (23), bf16 (1)
  __host__ __device__ int64_t n() const { return (int64_t)(packed & ((uint64_t(1) << 39) - 1)); }
  __host__ __device__ int first() const { return (int)(packed >> 39 & ((1 << 23) - 1)); }
  __host__ __device__ bool bf16() const { return packed >> 62 != 0; }
  static Tensor of(void* data, int64_t n, int64_t first, bool bf16) {
    return {data, (uint64_t)n | (uint64_t)first << 39 | (uint64_t)bf16 << 62};
  }
};

template <int MAX>
struct GradArgs {
  int count, chunk;
  int64_t base, total;  // this launch's first chunk among `total`; the last launch has base + grid == total
  double* partial;
  unsigned* counter;
  const float *grad_scale, *scale_in;
  float *norm, *scale;
  double max_norm;  // negative: none
  Tensor t[MAX];
};
using Args = GradArgs<kMaxTensors>;

// The tensor of workgroup b: the last whose first is not past it.  Every lane looks
// at one in 64: arguments lie in the host's memory, and this is one trip there where
// a search is one a step.
template <int MAX>
__device__ __forceinline__ Tensor tensor_of(const GradArgs<MAX>& a, int b) {
  const int lane = threadIdx.x & 63;
  constexpr int N = (MAX + 63) / 64;
  uint64_t data[N], packed[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const Tensor& t = a.t[min(lane + 64 * i, a.count - 1)];
    data[i] = reinterpret_cast<uint64_t>(t.data), packed[i] = t.packed;
  }
  int at = -1;
#pragma unroll
  for (int i = 0; i < N; ++i)
    at += __popcll(__ballot(lane + 64 * i < a.count && Tensor{nullptr, packed[i]}.first() <= b));
#pragma unroll
  for (int i = 1; i < N; ++i)
    if (at >= 64 * i) data[0] = data[i], packed[0] = packed[i];
  auto from = [&](uint64_t v) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)v, at & 63), hi = __builtin_amdgcn_readlane((int)(v >> 32), at & 63);
    return (uint64_t)hi << 32 | lo;
  };
  return {reinterpret_cast<void*>(from(data[0])), from(packed[0])};
}

// Sum over a workgroup of 256, in thread order within a wave and wave order.
__device__ __forceinline__ double block_sum(double s, double* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  s = ((red[0] + red[1]) + red[2]) + red[3];
  __syncthreads();
  return s;
}

template <bool BF16>
__device__ __forceinline__ void add_squares(u32x4 v, double (&s)[4]) {
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    if constexpr (BF16) {
      const double a = (double)__uint_as_float(v[d] << 16), b = (double)__uint_as_float(v[d] & 0xffff0000u);
      s[d] = fma(a, a, s[d]);
      s[d] = fma(b, b, s[d]);
    } else {
      const double a = (double)__uint_as_float(v[d]);
      s[d] = fma(a, a, s[d]);
    }
  }
}

// Squares of n values at p (at most a chunk), the thread's share.
template <bool BF16>
__device__ __forceinline__ double squares(const void* p, int n) {
  constexpr int E = BF16 ? 8 : 4, U = 4;
  typedef std::conditional_t<BF16, u16, float> T;
  const T* const x = static_cast<const T*>(p);
  double s[4] = {0., 0., 0., 0.};
  int i = E * (int)threadIdx.x;
  for (; i + (U - 1) * 256 * E + E <= n; i += U * 256 * E) {
    u32x4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = *reinterpret_cast<const u32x4_any*>(x + i + u * 256 * E);
#pragma unroll
    for (int u = 0; u < U; ++u) add_squares<BF16>(v[u], s);
  }
  for (; i < n; i += 256 * E) {
    u32x4 v = {0u, 0u, 0u, 0u};
    if (i + E <= n) {
      v = *reinterpret_cast<const u32x4_any*>(x + i);
    } else {
      for (int e = 0; i + e < n; ++e) {
        if constexpr (BF16) v[e >> 1] |= (uint32_t)x[i + e] << (16 * (e & 1));
        else v[e] = __float_as_uint(x[i + e]);
      }
    }
    add_squares<BF16>(v, s);
  }
  return (s[0] + s[1]) + (s[2] + s[3]);
}

template <int MAX>
__global__ __launch_bounds__(256) void grad_norm_kernel(GradArgs<MAX> a) {
  __shared__ double red[4];
  __shared__ int last;
  if (a.count > 0) {
    const Tensor t = tensor_of(a, blockIdx.x);
    const int64_t at = (int64_t)((int)blockIdx.x - t.first()) * a.chunk;
    const int n = (int)min((int64_t)a.chunk, t.n() - at);
    double s = t.bf16() ? squares<true>(static_cast<const u16*>(t.data) + at, n)
                      : squares<false>(static_cast<const float*>(t.data) + at, n);
    s = block_sum(s, red);
    if (threadIdx.x == 0)
      __hip_atomic_store(&a.partial[a.base + blockIdx.x], s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (a.base + gridDim.x < a.total) return;
    // The sum is at the device's coherence point before the arrival is counted.
    __builtin_amdgcn_s_waitcnt(0);
    if (threadIdx.x == 0)
      last = __hip_atomic_fetch_add(a.counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
    __syncthreads();
    if (!last) return;
    if (threadIdx.x == 0) __hip_atomic_store(a.counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  double s = 0.;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < a.total; i += 256)
    s += __hip_atomic_load(&a.partial[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  s = block_sum(s, red);
  if (threadIdx.x != 0) return;
  const double gs = a.grad_scale != nullptr ? (double)*a.grad_scale : 1.;
  const double norm = fabs(gs) * sqrt(s);
  double clip = 1.;
  if (a.max_norm >= 0.) {
    clip = a.max_norm / (norm + 1e-6);
    clip = clip > 1. ? 1. : clip;  // a NaN stays one
  }
  *a.norm = (float)norm;
  if (a.scale != nullptr) *a.scale = (float)(gs * clip);
}

// Values multiplied by a factor in place; none is touched where it is 1.
template <int MAX>
__global__ __launch_bounds__(256) void grad_scale_kernel(GradArgs<MAX> a) {
  const float f = *a.scale_in;
  if (f == 1.f) return;
  const Tensor t = tensor_of(a, blockIdx.x);
  const int64_t at = (int64_t)((int)blockIdx.x - t.first()) * a.chunk;
  const int n = (int)min((int64_t)a.chunk, t.n() - at);
  auto go = [&](auto* x, auto bf16) {
    constexpr bool BF16 = decltype(bf16)::value;
    constexpr int E = BF16 ? 8 : 4, U = 4;
    auto times = [&](u32x4 v) {
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        if constexpr (BF16) {
          const __bf16 lo = (__bf16)(__uint_as_float(v[d] << 16) * f), hi = (__bf16)(__uint_as_float(v[d] & 0xffff0000u) * f);
          v[d] = (uint32_t)__builtin_bit_cast(u16, lo) | (uint32_t)__builtin_bit_cast(u16, hi) << 16;
        } else {
          v[d] = __float_as_uint(__uint_as_float(v[d]) * f);
        }
      }
      return v;
    };
    int i = E * (int)threadIdx.x;
    for (; i + (U - 1) * 256 * E + E <= n; i += U * 256 * E) {
      u32x4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = *reinterpret_cast<const u32x4_any*>(x + i + u * 256 * E);
#pragma unroll
      for (int u = 0; u < U; ++u) *reinterpret_cast<u32x4_any*>(x + i + u * 256 * E) = times(v[u]);
    }
    for (; i < n; i += 256 * E) {
      if (i + E <= n) {
        *reinterpret_cast<u32x4_any*>(x + i) = times(*reinterpret_cast<const u32x4_any*>(x + i));
        continue;
      }
      for (int e = 0; i + e < n; ++e) {
        if constexpr (BF16) x[i + e] = __builtin_bit_cast(u16, (__bf16)(__uint_as_float((uint32_t)x[i + e] << 16) * f));
        else x[i + e] *= f;
      }
    }
  };
  if (t.bf16()) go(static_cast<u16*>(t.data) + at, std::true_type{});
  else go(static_cast<float*>(t.data) + at, std::false_type{});
}

// Values a workgroup takes: enough workgroups to fill the chip, then up to 64 Ki
// values each, so that few sums are left to add.
int chunk_of(const tilec_grad* grads, int32_t count) {
  int64_t n = 0;
  for (int i = 0; i < count; ++i) n += grads[i].n;
  const int64_t each = n / (8 * (int64_t)device_cus());
  return kUnit * (int)std::max<int64_t>(1, std::min<int64_t>(16, each / kUnit));
}

int64_t chunks_of(const tilec_grad* grads, int32_t count, int chunk) {
  int64_t n = 0;
  for (int i = 0; i < count; ++i) n += cdiv(grads[i].n, chunk);
  return n;
}

// f(workgroups) for the tensors in groups of up to kMaxTensors, with at most 2^22
// workgroups each; a.base counts them.
template <typename F>
hipError_t in_groups(Args& a, const tilec_grad* grads, int32_t count, F f) {
  int64_t blocks = 0;
  a.count = 0, a.base = 0;
  auto flush = [&]() -> hipError_t {
    if (a.count == 0) return hipSuccess;
    const hipError_t e = f((unsigned)blocks);
    a.base += blocks;
    a.count = 0, blocks = 0;
    return e;
  };
  for (int i = 0; i < count; ++i) {
    const int64_t esz = grads[i].dtype == TILEC_BF16 ? 2 : 4;
    static_assert(kMaxBlocks * 16 * kUnit <= kMaxPiece, "a piece's size fits its bits");
    for (int64_t at = 0; at < grads[i].n; at += kMaxBlocks * a.chunk) {
      const int64_t n = std::min(grads[i].n - at, kMaxBlocks * a.chunk), need = cdiv(n, a.chunk);
      if (a.count == kMaxTensors || blocks + need > kMaxBlocks) {
        const hipError_t e = flush();
        if (e != hipSuccess) return e;
      }
      a.t[a.count++] = Tensor::of(static_cast<char*>(grads[i].data) + at * esz, n, blocks, esz == 2);
      blocks += need;
    }
  }
  return flush();
}

// Launches the kernel that takes no more arguments than it has to: a launch copies
// them to memory that the GPU reads over the bus.  Theirs are the beginning of `a`.
template <template <int> class KERNEL, int MAX = 32>
hipError_t launch(const Args& a, unsigned blocks, hipStream_t stream) {
  if constexpr (MAX < kMaxTensors) {
    if (a.count > MAX) return launch<KERNEL, MAX + 32>(a, blocks, stream);
  }
  return enqueue(KERNEL<MAX>::get(), dim3(blocks), dim3(256), stream, reinterpret_cast<const GradArgs<MAX>&>(a));
}
template <int MAX>
struct NormKernel {
  static auto get() { return grad_norm_kernel<MAX>; }
};
template <int MAX>
struct ScaleKernel {
  static auto get() { return grad_scale_kernel<MAX>; }
};

int check_grads(const char* what, const tilec_grad* grads, int32_t count) {
  if (count < 0 || (count > 0 && grads == nullptr))
    return fail(TILEC_ERR_VALUE, "tilec: %s: no tensors (count %d)", what, count);
  for (int i = 0; i < count; ++i) {
    if (grads[i].dtype != TILEC_F32 && grads[i].dtype != TILEC_BF16)
      return fail(TILEC_ERR_TYPE, "tilec: %s: tensor %d: unsupported dtype code %d (use float32 or bfloat16)", what, i,
                  grads[i].dtype);
    if (grads[i].n < 0 || (grads[i].n > 0 && grads[i].data == nullptr))
      return fail(TILEC_ERR_VALUE, "tilec: %s: tensor %d has a NULL pointer or %lld elements", what, i,
                  (long long)grads[i].n);
  }
  return TILEC_OK;
}

}  // namespace

}  // namespace tilec

using namespace tilec;

extern "C" {

size_t tilec_grad_norm_workspace_bytes(const tilec_grad* grads, int32_t count) {
  if (check_grads("grad_norm", grads, count) != TILEC_OK) return 0;
  return (size_t)chunks_of(grads, count, chunk_of(grads, count)) * sizeof(double);
}

int tilec_grad_norm(const tilec_grad* grads, int32_t count, const float* grad_scale, double max_norm, float* norm,
                    float* scale, void* workspace, size_t workspace_bytes, void* counter, size_t counter_bytes,
                    void* stream) {
  clear_error();
  const int rc = check_grads("grad_norm", grads, count);
  if (rc != TILEC_OK) return rc;
  if (norm == nullptr) return fail(TILEC_ERR_VALUE, "tilec: grad_norm: norm is NULL");
  if (max_norm != max_norm) return fail(TILEC_ERR_VALUE, "tilec: grad_norm: max_norm is not a number");
  Args a{};
  a.chunk = chunk_of(grads, count);
  a.total = chunks_of(grads, count, a.chunk);
  const size_t need = (size_t)a.total * sizeof(double);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || counter == nullptr || counter_bytes < sizeof(unsigned)))
    return fail(TILEC_ERR_WORKSPACE, "tilec: grad_norm needs %zu workspace bytes and 4 bytes of counter (got %zu and %zu)",
                need, workspace == nullptr ? (size_t)0 : workspace_bytes, counter == nullptr ? (size_t)0 : counter_bytes);
  a.partial = static_cast<double*>(workspace), a.counter = static_cast<unsigned*>(counter);
  a.grad_scale = grad_scale, a.norm = norm, a.scale = scale;
  a.max_norm = max_norm < 0 || std::isinf(max_norm) ? -1. : max_norm;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  hipError_t e;
  if (a.total == 0) {  // the norm of nothing
    e = launch<NormKernel>(a, 1, st);
  } else {
    e = in_groups(a, grads, count, [&](unsigned blocks) { return launch<NormKernel>(a, blocks, st); });
  }
  if (e != hipSuccess) return fail(TILEC_ERR_HIP, "tilec: launching grad_norm failed: %s", hipGetErrorString(e));
  return TILEC_OK;
}

int tilec_scale_grads(const tilec_grad* grads, int32_t count, const float* scale, void* stream) {
  clear_error();
  const int rc = check_grads("scale_grads", grads, count);
  if (rc != TILEC_OK) return rc;
  if (scale == nullptr) return fail(TILEC_ERR_VALUE, "tilec: scale_grads: scale is NULL");
  Args a{};
  a.chunk = chunk_of(grads, count);
  a.scale_in = scale;
  const hipError_t e = in_groups(a, grads, count, [&](unsigned blocks) {
    return launch<ScaleKernel>(a, blocks, static_cast<hipStream_t>(stream));
  });
  if (e != hipSuccess) return fail(TILEC_ERR_HIP, "tilec: launching scale_grads failed: %s", hipGetErrorString(e));
  return TILEC_OK;
}

}  // extern "C"
