// Dropout whose mask is never stored: the draws come from a counter-based generator, so the backward call (the same map,
// applied to the gradient) makes them again.
//
//   y[i] = draw(i / run) >= round(p * 2^32) ? x[i] / (1 - p) : 0
//
// `run` consecutive elements share a draw: 1 (every element for itself), a feature plane, a sample.  draw(j) has 32 bits.
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011) with the seed as key
// and (j / 8, offset) as counter gives the upper 16 bits of eight draws at once; their lower 16 bits come from the counter
// with the highest bit of j / 8 set, and only a draw whose upper half equals the threshold's (one of 65536) looks at them.
// With 32 bits of one word per element the generator, not memory, is the bound: 142 us against 109 for 154 M fp16 values
// (308 MB in, 308 MB out, 5.7 TB/s; a copy of them takes 96).
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
  unsigned long long first_group;  // of this launch: groups of eight elements, all with the same upper 32 bits
  unsigned groups;
  int small;  // the index of a warp's part fits 32 bits
};

struct Key {
  unsigned k0, k1, o0, o1;
};

// The generator's key, kept for the backward where that is wanted.  As 32-bit words that are loaded without a condition it stays in
// uniform registers, its ten round keys with it: 18 % less time (154 M fp16 values).
template <bool STATE>
__device__ __forceinline__ Key key_of(const DropArgs& a) {
  const unsigned add0 = (unsigned)a.offset, add1 = (unsigned)(a.offset >> 32);
  Key k = {(unsigned)a.seed, (unsigned)(a.seed >> 32), add0, add1};
  if (STATE) {
    const unsigned* s = reinterpret_cast<const unsigned*>(a.state);
    const unsigned o0 = s[2], o1 = s[3], sum = o0 + add0;
    k = {s[0], s[1], sum, o1 + add1 + (sum < o0 ? 1u : 0u)};
    if (a.used && blockIdx.x == 0 && threadIdx.x == 0) {
      unsigned* u = reinterpret_cast<unsigned*>(a.used);
      u[0] = k.k0, u[1] = k.k1, u[2] = k.o0, u[3] = k.o1;
    }
  }
  return k;
}

__device__ __forceinline__ uint4 philox(unsigned c0, unsigned c1, const Key& k) {
  unsigned c2 = k.o0, c3 = k.o1;
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
// bit i: draw 8 group + i is kept; any threshold
__device__ __forceinline__ unsigned kept8(unsigned long long group, const Key& k, unsigned hi, unsigned lo) {
  const unsigned c0 = (unsigned)group, c1 = (unsigned)(group >> 32);
  const uint4 w = philox(c0, c1, k);
  unsigned keep = 0, even = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const unsigned u = half_word(w, i);
    keep |= (unsigned)(u > hi) << i;
    even |= (unsigned)(u == hi) << i;
  }
  if (even) {
    const uint4 l = philox(c0, c1 | 0x80000000u, k);
#pragma unroll
    for (int i = 0; i < 8; ++i) keep |= (even >> i & 1 & (unsigned)(half_word(l, i) >= lo)) << i;
  }
  return keep;
}

__device__ __forceinline__ unsigned settled(unsigned w, unsigned low, unsigned both, unsigned lo) {
  const unsigned d = w ^ both;
  if ((d & 0xffffu) == 0) w = (w & 0xffff0000u) | ((low & 0xffffu) >= lo ? 0xffffu : 0u);
  if ((d >> 16) == 0) w = (w & 0xffffu) | ((low >> 16) >= lo ? 0xffff0000u : 0u);
  return w;
}
// The upper halves of draws 8 group ... + 7, moved off the threshold: one that equals it becomes the lowest or the highest, as
// the draw's lower half says.  `both`: the threshold's upper half twice, below 0xffff.
__device__ __forceinline__ uint4 draws8(unsigned c0, unsigned c1, const Key& k, unsigned both, unsigned lo) {
  uint4 w = philox(c0, c1, k);
  // a half word that is zero sets its highest bit (so may the one above it: `settled` looks again)
  const unsigned a = w.x ^ both, b = w.y ^ both, c = w.z ^ both, d = w.w ^ both;
  const unsigned even = ((a - 0x00010001u) & ~a) | ((b - 0x00010001u) & ~b) | ((c - 0x00010001u) & ~c) | ((d - 0x00010001u) & ~d);
  if (even & 0x80008000u) {
    const uint4 l = philox(c0, c1 | 0x80000000u, k);
    w.x = settled(w.x, l.x, both, lo), w.y = settled(w.y, l.y, both, lo), w.z = settled(w.z, l.z, both, lo);
    w.w = settled(w.w, l.w, both, lo);
  }
  return w;
}

// Sixteen bytes of values: what is kept times the scale, zeros elsewhere.  16-bit values are converted and rounded in pairs, which the
// conversion units do at twice the rate.
template <typename T> struct Piece {
  static __device__ __forceinline__ void apply(uint4& v, float s, const bool* k);
};
template <> struct Piece<float> {
  static __device__ __forceinline__ void apply(uint4& v, float s, const bool* k) {
    v.x = k[0] ? __float_as_uint(__uint_as_float(v.x) * s) : 0u, v.y = k[1] ? __float_as_uint(__uint_as_float(v.y) * s) : 0u;
    v.z = k[2] ? __float_as_uint(__uint_as_float(v.z) * s) : 0u, v.w = k[3] ? __float_as_uint(__uint_as_float(v.w) * s) : 0u;
  }
};
template <> struct Piece<double> {
  static __device__ __forceinline__ void apply(uint4& v, double s, const bool* k) {
    double a = __hiloint2double((int)v.y, (int)v.x), b = __hiloint2double((int)v.w, (int)v.z);
    a = k[0] ? a * s : 0.0, b = k[1] ? b * s : 0.0;
    v = make_uint4((unsigned)__double2loint(a), (unsigned)__double2hiint(a), (unsigned)__double2loint(b), (unsigned)__double2hiint(b));
  }
};
__device__ __forceinline__ unsigned pair_of(unsigned v, float s, bool k0, bool k1, __half) {
  float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
  f.x = k0 ? f.x * s : 0.0f, f.y = k1 ? f.y * s : 0.0f;
  const __half2 h = __float22half2_rn(f);
  return *reinterpret_cast<const unsigned*>(&h);
}
__device__ __forceinline__ unsigned pair_of(unsigned v, float s, bool k0, bool k1, __nv_bfloat16) {
  float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
  f.x = k0 ? f.x * s : 0.0f, f.y = k1 ? f.y * s : 0.0f;
  const __nv_bfloat162 h = __float22bfloat162_rn(f);
  return *reinterpret_cast<const unsigned*>(&h);
}
template <typename T>
__device__ __forceinline__ void Piece<T>::apply(uint4& v, float s, const bool* k) {
  v.x = pair_of(v.x, s, k[0], k[1], T()), v.y = pair_of(v.y, s, k[2], k[3], T());
  v.z = pair_of(v.z, s, k[4], k[5], T()), v.w = pair_of(v.w, s, k[6], k[7], T());
}
template <typename T, typename A> __device__ __forceinline__ T times(T v, A s) { return (T)((A)v * s); }
template <> __device__ __forceinline__ __half times<__half, float>(__half v, float s) { return __float2half_rn(__half2float(v) * s); }
template <> __device__ __forceinline__ __nv_bfloat16 times<__nv_bfloat16, float>(__nv_bfloat16 v, float s) {
  return __float2bfloat16_rn(__bfloat162float(v) * s);
}

// Every element has its own draw; both tensors begin on 16 bytes, hold whole groups of eight (the elements of this launch), and the
// threshold's upper half is below 0xffff.  A thread takes eight elements at a time, one counter's worth of draws.  All the warps an SM can hold, with registers to
// match, hide the generator's latency: 17 % less time than with the registers that ptxas takes by itself.
template <typename T, bool STATE>
__global__ void __launch_bounds__(256, 8) dropout_kernel(const T* __restrict__ x, T* __restrict__ y, const DropArgs a) {
  constexpr int kPieces = 8 * sizeof(T) / 16;
  using A = typename Compute<T>::type;
  const Key key = key_of<STATE>(a);
  const A scale = (A)a.scale;
  // as upper half of a word a draw is above these whatever the lower half holds, as lower half after a shift
  const unsigned above_hi = a.hi << 16 | 0xffffu, above_lo = a.hi << 16, both = a.hi * 0x00010001u;
  for (unsigned i = blockIdx.x * 256 + threadIdx.x; i < a.groups; i += gridDim.x * 256) {
    uint4 v[kPieces];
#pragma unroll
    for (int q = 0; q < kPieces; ++q) v[q] = __ldg(reinterpret_cast<const uint4*>(x) + (size_t)i * kPieces + q);
    const uint4 w = draws8((unsigned)a.first_group + i, (unsigned)(a.first_group >> 32), key, both, a.lo);
    const bool k[8] = {w.x << 16 > above_lo, w.x > above_hi, w.y << 16 > above_lo, w.y > above_hi,
                       w.z << 16 > above_lo, w.z > above_hi, w.w << 16 > above_lo, w.w > above_hi};
#pragma unroll
    for (int q = 0; q < kPieces; ++q) {
      Piece<T>::apply(v[q], scale, k + q * (8 / kPieces));
      reinterpret_cast<uint4*>(y)[(size_t)i * kPieces + q] = v[q];
    }
  }
}

// The same for tensors that begin elsewhere (VECTOR = false), for runs of elements that share a draw (those that are dropped are
// not read), and for any threshold.
template <typename T, bool VECTOR, bool STATE>
__global__ void __launch_bounds__(256) dropout_runs_kernel(const T* __restrict__ x, T* __restrict__ y, const DropArgs a) {
  constexpr int kPieces = 8 * sizeof(T) / 16;
  using A = typename Compute<T>::type;
  const Key key = key_of<STATE>(a);
  const A scale = (A)a.scale;
  for (unsigned i = blockIdx.x * 256 + threadIdx.x; i < a.groups; i += gridDim.x * 256) {
    const unsigned long long g = a.first_group + i, first = g << 3;
    const int n = a.count - first < 8 ? (int)(a.count - first) : 8;
    unsigned long long j = a.run == 1 ? first : first / a.run;
    unsigned long long left = a.run - (first - j * a.run);  // elements of run j from here on
    unsigned keep = 0, eight = kept8(j >> 3, key, a.hi, a.lo);
    if (a.run == 1) {
      keep = eight;
    } else if (left >= 8) {
      keep = (eight >> (j & 7) & 1) ? 0xffu : 0u;
    } else {
      for (int e = 0; e < n; ++e, --left) {
        if (left == 0) {
          ++j, left = a.run;
          if ((j & 7) == 0) eight = kept8(j >> 3, key, a.hi, a.lo);
        }
        keep |= (eight >> (j & 7) & 1) << e;
      }
    }
    if (VECTOR && n == 8) {
      bool k[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) k[e] = keep >> e & 1;
#pragma unroll
      for (int q = 0; q < kPieces; ++q) {
        uint4 v = keep ? __ldg(reinterpret_cast<const uint4*>(x + first) + q) : make_uint4(0, 0, 0, 0);
        Piece<T>::apply(v, scale, k + q * (8 / kPieces));
        reinterpret_cast<uint4*>(y + first)[q] = v;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < n) y[first + e] = (keep >> e & 1) ? times<T, A>(x[first + e], scale) : (T)0.0f;
    }
  }
}

// Long runs (planes, samples) of a multiple of eight elements, both tensors on 16 bytes: a warp has up to kPart elements of one run, so that the division and the
// counter are its own and not those of every eight elements (28.9 M fp32 values in planes of 3136, p = 0.2: 37 us against 41).
constexpr int kPart = 1024;
// Runs from here on go that way; below, a warp has too little to do for its counter (67 M values, p = 0.2, us here / in dropout_runs_kernel: fp16 runs of 64
// 383 / 81, 192 133 / 81, 256 101 / 81, 384 72 / 81, 1024 41 / 81; fp32 64 314 / 88, 192 112 / 88, 256 87 / 86, 384 78 / 86, 1024 76 / 86).
constexpr unsigned long long kLongRun = 320;
template <typename T, bool STATE>
__global__ void __launch_bounds__(256) dropout_long_runs_kernel(const T* __restrict__ x, T* __restrict__ y, const DropArgs a, unsigned parts,
                                                                unsigned long long units) {
  constexpr int kEach = 16 / sizeof(T), kSteps = 4;  // values of a 16-byte piece; pieces in flight
  using A = typename Compute<T>::type;
  const Key key = key_of<STATE>(a);
  const A scale = (A)a.scale;
  const int lane = threadIdx.x & 31;
  for (unsigned long long u = (unsigned long long)blockIdx.x * 8 + (threadIdx.x >> 5); u < units; u += (unsigned long long)gridDim.x * 8) {
    const unsigned long long j = a.small ? (unsigned long long)((unsigned)u / parts) : u / parts;
    const unsigned long long in_run = (u - j * parts) * kPart, left = a.run - in_run;
    const int n = left < kPart ? (int)left : kPart;
    const T* from = x + j * a.run + in_run;
    T* to = y + j * a.run + in_run;
    const bool keep = kept8(j >> 3, key, a.hi, a.lo) >> (j & 7) & 1;
    const bool all[8] = {keep, keep, keep, keep, keep, keep, keep, keep};
    for (int e0 = lane * kEach; e0 < n; e0 += 32 * kEach * kSteps) {
      uint4 v[kSteps];
#pragma unroll
      for (int q = 0; q < kSteps; ++q) {
        const int e = e0 + q * 32 * kEach;
        v[q] = keep && e < n ? __ldg(reinterpret_cast<const uint4*>(from + e)) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int q = 0; q < kSteps; ++q) {
        const int e = e0 + q * 32 * kEach;
        Piece<T>::apply(v[q], scale, all);
        if (e < n) *reinterpret_cast<uint4*>(to + e) = v[q];
      }
    }
  }
}

template <typename T, bool STATE>
int launch_dropout(const void* input, void* output, DropArgs a, cudaStream_t s) {
  const T* x = (const T*)input;
  T* y = (T*)output;
  const bool vector = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & 15) == 0;
  const unsigned most = (unsigned)device_sm_count() * 32;
  if (vector && a.run >= kLongRun && a.run % 8 == 0) {
    const unsigned long long parts = (a.run + kPart - 1) / kPart, units = a.count / a.run * parts;
    if (a.count % a.run == 0 && parts <= 0xffffffffull) {
      a.small = units <= 0xffffffffull;
      const unsigned long long blocks = (units + 7) / 8;
      dropout_long_runs_kernel<T, STATE><<<(unsigned)(blocks < most ? blocks : most), 256, 0, s>>>(x, y, a, (unsigned)parts, units);
      return check_launch();
    }
  }
  unsigned long long at = 0, total = (a.count + 7) >> 3;
  while (at < total) {
    unsigned long long n = total - at < 1ull << 30 ? total - at : 1ull << 30;
    // whole groups first, an incomplete one by itself: looking for it in the kernel costs every group a tenth of its time
    const bool whole = a.run == 1 && vector && a.hi < 0xffffu && (a.count >> 3) > at;
    if (whole && n > (a.count >> 3) - at) n = (a.count >> 3) - at;
    a.first_group = at, a.groups = (unsigned)n;
    const unsigned blocks = (a.groups + 255) >> 8, grid = blocks < most ? blocks : most;
    if (whole) dropout_kernel<T, STATE><<<grid, 256, 0, s>>>(x + (at << 3), y + (at << 3), a);
    else if (vector) dropout_runs_kernel<T, true, STATE><<<grid, 256, 0, s>>>(x, y, a);
    else dropout_runs_kernel<T, false, STATE><<<grid, 256, 0, s>>>(x, y, a);
    const int rc = check_launch();
    if (rc != DK_OK) return rc;
    at += n;
  }
  return DK_OK;
}

}  // namespace
}  // namespace dk

using namespace dk;

extern "C" int dk_dropout(const void* input, void* output, long long count, long long run, double p, unsigned long long seed,
                          unsigned long long offset, const void* state, void* used, int dtype, void* stream) {
  if (!input || !output || count <= 0 || run <= 0 || !(p >= 0.0 && p <= 1.0) || (used && !state)) return DK_ERR_BAD_ARGUMENT;
  if ((reinterpret_cast<uintptr_t>(state) | reinterpret_cast<uintptr_t>(used)) & 7) return DK_ERR_BAD_ARGUMENT;
  // every block reads `state`, one of them writes `used`
  const uintptr_t from = reinterpret_cast<uintptr_t>(state), to = reinterpret_cast<uintptr_t>(used);
  if (used && from < to + 16 && to < from + 16) return DK_ERR_BAD_ARGUMENT;
  DropArgs a = {};
  a.count = (unsigned long long)count, a.run = (unsigned long long)run;
  a.seed = seed, a.offset = offset;
  a.state = (const unsigned long long*)state, a.used = (unsigned long long*)used;
  const unsigned long long threshold = (unsigned long long)(p * 4294967296.0 + 0.5);
  a.hi = (unsigned)(threshold >> 16), a.lo = (unsigned)(threshold & 0xffff);
  a.scale = p < 1.0 ? 1.0 / (1.0 - p) : 0.0;
  cudaStream_t s = (cudaStream_t)stream;
  switch (dtype) {
    case DK_F32: return state ? launch_dropout<float, true>(input, output, a, s) : launch_dropout<float, false>(input, output, a, s);
    case DK_F16: return state ? launch_dropout<__half, true>(input, output, a, s) : launch_dropout<__half, false>(input, output, a, s);
    case DK_BF16: return state ? launch_dropout<__nv_bfloat16, true>(input, output, a, s) : launch_dropout<__nv_bfloat16, false>(input, output, a, s);
    case DK_F64: return state ? launch_dropout<double, true>(input, output, a, s) : launch_dropout<double, false>(input, output, a, s);
    default: return DK_ERR_BAD_ARGUMENT;
  }
}
