// The last linear layer of a classifier with its softmax cross entropy: what dk_head.cu (entry points, small kernels, the
// general kernels) and dk_head_tc.cu (the tensor-core kernels) share.
#pragma once

#include <cuda_bf16.h>

#include "dk_common.cuh"

namespace dk {
namespace head {

constexpr double kLog2e = 1.4426950408889634074, kLn2 = 0.69314718055994530942;

struct Shape {
  int T, D, V;  // rows, features, classes
  long long ignore;
  int reduction;
  double smoothing;
};

// What a tile of logits leaves of its rows; a slot is a run of classes.
template <typename A>
struct Partials {
  A* top;     // [slots][T] maximum of z
  A* sum;     // [slots][T] sum of exp(z - top): the largest logit's term is exactly one
  A* all;     // [slots][T] sum of z (label smoothing only)
  A* picked;  // [T] z of the row's own class
};

inline size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }
inline int div_up(long long a, long long b) { return (int)((a + b - 1) / b); }

// offsets of the parts of a workspace
struct Layout {
  size_t bytes = 0;
  size_t take(size_t n) {
    const size_t at = bytes;
    bytes += up256(n);
    return at;
  }
};

// What arrives from behind the loss, g_t.  dz_t = g_t (p - (1 - s) [v = y_t] - s / V) is an operand of two products, so the factor that all
// its rows have in common is left to their results: what is rounded to 16 bits is dz `unit` / g, with `unit` 1 / (1 - s) so that a class that the
// network gives no chance has exactly one (a power of two): the rounding of g (1 - s) would be the same in every row and add up.  fp16: `unit`
// has a factor 2^14 besides, which keeps small probabilities out of the subnormal numbers.  DK_REDUCE_NONE: every row has its own g; `unit`
// brings the largest to [2^14, 2^15) (fp16) or is 1.
template <typename A>
struct Upstream {
  const A* up;       // one value, or one a row (DK_REDUCE_NONE)
  const A* count;    // rows that count
  const A* largest;  // DK_REDUCE_NONE, fp16: the largest |up| of those
  int reduction;
  A unit;
};
template <typename A>
__device__ __forceinline__ A upstream_unit(const Upstream<A>& u) {
  if (!u.largest) return u.unit;
  const A largest = *u.largest;
  if (!(largest > (A)0) || !isfinite(largest)) return (A)1;
  const int e = 14 - ilogb(largest);
  return (A)ldexp((A)1, e < -100 ? -100 : e > 100 ? 100 : e);
}
// dz's factor of row r, whose class is y: nothing for an ignored row, NaN for a class that does not exist
template <typename A>
__device__ __forceinline__ A upstream_row(const Upstream<A>& u, int r, long long y, long long ignore, int classes) {
  if (y == ignore) return (A)0;
  if (y < 0 || y >= classes) return (A)(0.0 / 0.0);
  return u.reduction == DK_REDUCE_NONE ? u.up[r] * upstream_unit(u) : u.unit;
}
// the factor of the products
template <typename A>
__device__ __forceinline__ A upstream_back(const Upstream<A>& u) {
  if (u.reduction == DK_REDUCE_NONE) return (A)1 / upstream_unit(u);
  if (*u.count == (A)0) return (A)0;  // no row counts: their dz are zeros, and the mean's g is not finite
  return (u.reduction == DK_REDUCE_MEAN ? u.up[0] / *u.count : u.up[0]) / u.unit;
}

// ---- the slots of a row joined (dk_head.cu)
constexpr int kCombineRows = 32;  // rows of a block, or a multiple
// sums of the blocks, and the count of those that are done, which the kernel before sets to zero
inline size_t combine_bytes(int T) { return (size_t)div_up(T, kCombineRows) * 3 * sizeof(double) + sizeof(double); }
// losses, log-sum-exps and counts; `partial`: combine_bytes(), the count last
template <typename A>
int launch_combine(const Partials<A>& p, const long long* y, int slots, void* loss, void* saved, double* partial, const Shape& h,
                   cudaStream_t s);
inline unsigned* combine_count(double* partial, int T) { return (unsigned*)(partial + 3ll * div_up(T, kCombineRows)); }

// ---- the loss of a few rows without a backward (dk_head.cu): memory is the bound, the products are taken on the CUDA cores
bool few_rows(int T, int dtype);
int few_slots(int V);
template <typename T>
int launch_few_rows(const void* x, const void* w, const void* b, const long long* y, const Partials<float>& p, unsigned* count,
                    const Shape& h, cudaStream_t s);

// ---- launches that may begin while the kernel before still runs: before_all() waits for what it wrote
__device__ __forceinline__ void before_all() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }
__device__ __forceinline__ void let_next() { asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory"); }
template <typename K, typename... Args>
int launch_after(K kernel, unsigned grid, unsigned block, size_t smem, int cluster, cudaStream_t s, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid), cfg.blockDim = dim3(block), cfg.dynamicSmemBytes = smem, cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization, attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr, cfg.numAttrs = cluster > 1 ? 2 : 1;
  cudaLaunchKernelEx(&cfg, kernel, args...);
  return check_launch();
}

// ---- fp16, bf16 and fp32 on the tensor cores (dk_head_tc.cu)
size_t tc_forward_bytes(int T, int D, int V, int dtype);
int tc_forward(const void* x, const void* w, const void* b, const long long* y, void* loss, void* saved, const Shape& h, int dtype,
               void* ws, size_t ws_bytes, cudaStream_t s);
long long set_wait_limit(long long nanoseconds);  // of the launches from now on; the one before
size_t tc_backward_bytes(int T, int D, int V, int dtype);
int tc_backward(const void* up, const void* x, const void* w, const void* b, const long long* y, const void* saved, void* dx, void* dw,
                void* db, const Shape& h, int dtype, void* ws, size_t ws_bytes, cudaStream_t s);

}  // namespace head
}  // namespace dk
