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
  A* top;     // [slots][T] maximum of z log2(e)
  A* sum;     // [slots][T] sum of 2^(z log2(e) - top)
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

// ---- small kernels (dk_head.cu)
constexpr int kCombineRows = 32;  // rows of a block of the kernel that joins the slots
inline size_t combine_bytes(int T) { return (size_t)div_up(T, kCombineRows) * 3 * sizeof(double); }
// losses, log-sum-exps and counts from the slots; `partial`: combine_bytes()
template <typename A>
int launch_combine(const Partials<A>& p, const long long* y, int slots, void* loss, void* saved, double* partial, const Shape& h,
                   cudaStream_t s);
// g_t of every row.  `back` (NULL: nothing is scaled): two floats, g comes out multiplied with a power of two that brings the
// largest to about 2^14, back[0] is the reciprocal of that
template <typename A>
int launch_rows(const void* up, const long long* y, const void* saved, A* g, A* back, const Shape& h, cudaStream_t s);

// ---- fp16, bf16 and fp32 on the tensor cores (dk_head_tc.cu)
size_t tc_forward_bytes(int T, int D, int V, int dtype);
int tc_forward(const void* x, const void* w, const void* b, const long long* y, void* loss, void* saved, const Shape& h, int dtype,
               void* ws, size_t ws_bytes, cudaStream_t s);
size_t tc_backward_bytes(int T, int D, int V, int dtype);
int tc_backward(const void* up, const void* x, const void* w, const void* b, const long long* y, const void* saved, void* dx, void* dw,
                void* db, const Shape& h, int dtype, void* ws, size_t ws_bytes, cudaStream_t s);

}  // namespace head
}  // namespace dk
