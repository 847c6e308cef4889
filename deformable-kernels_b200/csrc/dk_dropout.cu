// Dropout whose mask is never stored: the draws come from a counter-based generator, so the backward call (the same map,
// applied to the gradient) makes them again.
//
//   y[i] = draw(i / run) >= round(p * 2^32) ? x[i] / (1 - p) : 0
//
// `run` consecutive elements share a draw: 1 (every element for itself), a feature plane, a sample.  draw(j) has 32 bits.
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011) with the seed as key
// and (j / 8, offset) as counter gives the upper 16 bits of eight draws at once; their lower 16 bits come from the counter
// with the highest bit of j / 8 set, and only a draw whose upper half equals the threshold's (one of 65536) looks at them.
// With 32 bits of one word per element the generator, not memory, is the bound: 142 us against 102 for 154 M fp16 values
// (308 MB in, 308 MB out, 6.0 TB/s; a copy kernel of the same shape without any generator takes 101).
//
// A dropped element is zero whatever x holds there (infinities and NaN included).  x / (1 - p) is a product with the fp32
// (fp64) reciprocal, rounded once to the tensor's type.
#include <cuda_bf16.h>

#include "dk_common.cuh"

namespace dk {
namespace {

struct DropArgs {
  unsigned long long count, run;   // elements; elements per draw
  unsigned long long seed, offset;
  const unsigned long long* state; // device: seed and offset (the argument `offset` is added); NULL: the two above
  unsigned long long* used;        // device or NULL: where the seed and offset of this call are kept for its backward
  unsigned hi, lo;                 // threshold: upper 16 bits (65536: nothing is kept), lower 16 bits
  double scale;
};

struct Key {
  unsigned k0, k1, o0, o1;
};

__device__ __forceinline__ uint4 philox(unsigned long long group, unsigned second, const Key& k) {
  unsigned c0 = (unsigned)group, c1 = (unsigned)(group >> 32) | second, c2 = k.o0, c3 = k.o1;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
    c0 = (unsigned)(b >> 32) ^ c1 ^ (k.k0 + r * 0x9E3779B9u);
    c2 = (unsigned)(a >> 32) ^ c3 ^ (k.k1 + r * 0xBB67AE85u);
    c1 = (unsigned)b, c3 = (unsigned)a;
  }
  return make_uint4(c0, c1, c2, c3);
}
__device__ __forceinline__ unsigned half_word(const uint4& w, int i) {
  const unsigned v = (i & 4) ? ((i & 2) ? w.w : w.z) : ((i & 2) ? w.y : w.x);
  return (i & 1) ? v >> 16 : v & 0xffffu;
}
// u: the upper half of draw 8 group + i
__device__ __forceinline__ bool kept(unsigned u, unsigned long long group, int i, const Key& k, unsigned hi, unsigned lo) {
  if (u != hi) return u > hi;
  return lo == 0 || half_word(philox(group, 0x80000000u, k), i) >= lo;
}

template <typename T> struct Value {
  using A = typename Compute<T>::type;
  static __device__ __forceinline__ T times(T v, A s) { return (T)((A)v * s); }
};
template <> struct Value<__half> {
  using A = float;
  static __device__ __forceinline__ __half times(__half v, float s) { return __float2half_rn(__half2float(v) * s); }
};
template <> struct Value<__nv_bfloat16> {
  using A = float;
  static __device__ __forceinline__ __nv_bfloat16 times(__nv_bfloat16 v, float s) { return __float2bfloat16_rn(__bfloat162float(v) * s); }
};

// A thread takes eight consecutive elements at a time: one counter's worth of draws when every element has its own.
// VECTOR: both tensors begin on 16 bytes.  SHARED: run > 1; at most two counters for eight elements, and elements whose
// run is dropped are not read.
template <typename T, bool VECTOR, bool SHARED>
__global__ void __launch_bounds__(256) dropout_kernel(const T* __restrict__ x, T* __restrict__ y, const DropArgs a) {
  constexpr int kPieces = 8 * sizeof(T) / 16;
  using A = typename Value<T>::A;
  unsigned long long seed = a.seed, offset = a.offset;
  if (a.state) seed = a.state[0], offset += a.state[1];
  if (a.used && blockIdx.x == 0 && threadIdx.x == 0) a.used[0] = seed, a.used[1] = offset;
  const Key key = {(unsigned)seed, (unsigned)(seed >> 32), (unsigned)offset, (unsigned)(offset >> 32)};
  const A scale = (A)a.scale;
  const T zero = (T)0.0f;
  const unsigned long long groups = (a.count + 7) >> 3, step = (unsigned long long)gridDim.x * blockDim.x;
  for (unsigned long long g = (unsigned long long)blockIdx.x * blockDim.x + threadIdx.x; g < groups; g += step) {
    const unsigned long long first = g << 3;
    const int n = a.count - first < 8 ? (int)(a.count - first) : 8;
    unsigned keep = 0;
    if (!SHARED) {
      const uint4 w = philox(g, 0, key);
#pragma unroll
      for (int i = 0; i < 8; ++i) keep |= (unsigned)kept(half_word(w, i), g, i, key, a.hi, a.lo) << i;
    } else {
      unsigned long long j = first / a.run;
      unsigned long long left = a.run - (first - j * a.run);  // elements of run j from here on
      unsigned long long have = ~0ull;
      uint4 w = make_uint4(0, 0, 0, 0);
      bool k = false;
      bool fresh = true;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (left == 0) ++j, left = a.run, fresh = true;
        if (fresh && i < n) {
          if (j >> 3 != have) have = j >> 3, w = philox(have, 0, key);
          k = kept(half_word(w, (int)(j & 7)), have, (int)(j & 7), key, a.hi, a.lo);
          fresh = false;
        }
        --left;
        keep |= (unsigned)k << i;
      }
    }
    if (VECTOR && n == 8) {
      alignas(16) T v[8];
      if (!SHARED || keep) {
#pragma unroll
        for (int q = 0; q < kPieces; ++q) reinterpret_cast<uint4*>(v)[q] = __ldg(reinterpret_cast<const uint4*>(x + first) + q);
      } else {
#pragma unroll
        for (int q = 0; q < kPieces; ++q) reinterpret_cast<uint4*>(v)[q] = make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = (keep >> i & 1) ? Value<T>::times(v[i], scale) : zero;
#pragma unroll
      for (int q = 0; q < kPieces; ++q) reinterpret_cast<uint4*>(y + first)[q] = reinterpret_cast<const uint4*>(v)[q];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) y[first + i] = (keep >> i & 1) ? Value<T>::times(x[first + i], scale) : zero;
    }
  }
}

template <typename T>
int launch_dropout(const void* input, void* output, const DropArgs& a, cudaStream_t s) {
  const T* x = (const T*)input;
  T* y = (T*)output;
  const bool vector = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & 15) == 0;
  const unsigned long long blocks = (((a.count + 7) >> 3) + 255) >> 8;
  // 16 blocks per SM and a loop: 102 us where a block per 2048 elements takes 111 (154 M fp16 values)
  const unsigned long long most = (unsigned long long)device_sm_count() * 16;
  const unsigned grid = (unsigned)(blocks < most ? blocks : most);
  if (a.run == 1) {
    if (vector) dropout_kernel<T, true, false><<<grid, 256, 0, s>>>(x, y, a);
    else dropout_kernel<T, false, false><<<grid, 256, 0, s>>>(x, y, a);
  } else {
    if (vector) dropout_kernel<T, true, true><<<grid, 256, 0, s>>>(x, y, a);
    else dropout_kernel<T, false, true><<<grid, 256, 0, s>>>(x, y, a);
  }
  return check_launch();
}

}  // namespace
}  // namespace dk

using namespace dk;

extern "C" int dk_dropout(const void* input, void* output, long long count, long long run, double p, unsigned long long seed,
                          unsigned long long offset, const void* state, void* used, int dtype, void* stream) {
  if (!input || !output || count <= 0 || run <= 0 || !(p >= 0.0 && p <= 1.0)) return DK_ERR_BAD_ARGUMENT;
  if ((reinterpret_cast<uintptr_t>(state) | reinterpret_cast<uintptr_t>(used)) & 7) return DK_ERR_BAD_ARGUMENT;
  DropArgs a;
  a.count = (unsigned long long)count, a.run = (unsigned long long)run;
  a.seed = seed, a.offset = offset;
  a.state = (const unsigned long long*)state, a.used = (unsigned long long*)used;
  const unsigned long long threshold = (unsigned long long)(p * 4294967296.0 + 0.5);
  a.hi = (unsigned)(threshold >> 16), a.lo = (unsigned)(threshold & 0xffff);
  a.scale = p < 1.0 ? 1.0 / (1.0 - p) : 0.0;
  cudaStream_t s = (cudaStream_t)stream;
  switch (dtype) {
    case DK_F32: return launch_dropout<float>(input, output, a, s);
    case DK_F16: return launch_dropout<__half>(input, output, a, s);
    case DK_BF16: return launch_dropout<__nv_bfloat16>(input, output, a, s);
    case DK_F64: return launch_dropout<double>(input, output, a, s);
    default: return DK_ERR_BAD_ARGUMENT;
  }
}
