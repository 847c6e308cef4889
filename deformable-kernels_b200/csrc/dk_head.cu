// The last linear layer of a classifier with its softmax cross entropy, without keeping the logits.
//
//   z = x W^T + b                        x [T, D], W [V, D], b [V] or none
//   lse_t = log sum_v exp z_tv
//   loss_t = lse_t - (1 - s) z_t[y_t] - s / V sum_v z_tv            s: label smoothing; 0 for a row that is ignored
//   dz_tv = g_t (exp(z_tv - lse_t) - (1 - s) [v = y_t] - s / V)     g_t: what arrives from behind the loss
//   dx = dz W,   dW = dz^T x,   db = sum_t dz_t
//
// Forward: tiles of logits live in registers only; each leaves (maximum, sum of exponentials) of its rows, kept to the
// base 2, and a second kernel joins the tiles of a row in fixed order.  Backward: a piece of the vocabulary at a time, the
// logits of the piece once more, dz of the piece into the workspace, then the two products.
//
// Here: the C entry points, the small kernels, and kernels on the CUDA cores for every type.
#include <math_constants.h>

#include "dk_head.cuh"

namespace dk {
namespace head {

template <typename A, typename T> __device__ __forceinline__ A get(const T* p) { return (A)*p; }
template <> __device__ __forceinline__ float get<float, __half>(const __half* p) { return __half2float(*p); }
template <> __device__ __forceinline__ float get<float, __nv_bfloat16>(const __nv_bfloat16* p) { return __bfloat162float(*p); }
template <typename T, typename A> __device__ __forceinline__ void put(T* p, A v) { *p = (T)v; }
template <> __device__ __forceinline__ void put<__half, float>(__half* p, float v) { *p = __float2half_rn(v); }
template <> __device__ __forceinline__ void put<__nv_bfloat16, float>(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

template <typename A> __device__ __forceinline__ A minus_inf() { return (A)-CUDART_INF_F; }

struct Shape {
  int T, D, V;
  long long ignore;
  int reduction;
  double smoothing;
};

// ------------------------------------------------------------------ logits, a 64 x 64 tile of them a block

constexpr int kTile = 64, kDepth = 16, kPitch = kTile + 4;

// acc[i][j] = sum_k x[r0 + 4 ty + i][k] W[c0 + 4 tx + j][k]; rows and classes outside count as zeros
template <typename T, typename A>
__device__ __forceinline__ void logits_tile(A (&acc)[4][4], A* sx, A* sw, const T* __restrict__ x, const T* __restrict__ w, int r0,
                                            int c0, const Shape& h) {
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = (A)0;
  for (int k0 = 0; k0 < h.D; k0 += kDepth) {
    for (int e = threadIdx.x; e < kTile * kDepth; e += 256) {
      const int r = e / kDepth, k = e % kDepth;
      const bool in = k0 + k < h.D;
      sx[k * kPitch + r] = in && r0 + r < h.T ? get<A>(x + (long long)(r0 + r) * h.D + k0 + k) : (A)0;
      sw[k * kPitch + r] = in && c0 + r < h.V ? get<A>(w + (long long)(c0 + r) * h.D + k0 + k) : (A)0;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kDepth; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += sx[k * kPitch + 4 * ty + i] * sw[k * kPitch + 4 * tx + j];
    __syncthreads();
  }
}

// a warp's sixteen threads of one row
template <typename A>
__device__ __forceinline__ A max16(A v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <typename A>
__device__ __forceinline__ A sum16(A v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// What a tile leaves of its rows: slot = tile of classes
template <typename A>
struct Partials {
  A* top;     // [slots][T] maximum of z log2(e)
  A* sum;     // [slots][T] sum of 2^(z log2(e) - top)
  A* all;     // [slots][T] sum of z (label smoothing only)
  A* picked;  // [T] z of the row's own class
};

template <typename T, typename A>
__global__ void __launch_bounds__(256) logits_stats_kernel(const T* __restrict__ x, const T* __restrict__ w, const T* __restrict__ b,
                                                           const long long* __restrict__ y, Partials<A> p, Shape h) {
  __shared__ A sx[kDepth * kPitch], sw[kDepth * kPitch];
  const int r0 = blockIdx.y * kTile, c0 = blockIdx.x * kTile;
  A z[4][4];
  logits_tile<T, A>(z, sx, sw, x, w, r0, c0, h);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + 4 * ty + i;
    const long long yr = r < h.T ? y[r] : -1;
    A top = minus_inf<A>(), all = (A)0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = c0 + 4 * tx + j;
      if (c < h.V) {
        if (b) z[i][j] += get<A>(b + c);
        if (yr == c) p.picked[r] = z[i][j];
        all += z[i][j];
        z[i][j] *= (A)kLog2e;
      } else {
        z[i][j] = minus_inf<A>();
      }
      top = fmax(top, z[i][j]);
    }
    top = max16(top);
    const A ref = top == minus_inf<A>() ? (A)0 : top;
    A sum = (A)0;
#pragma unroll
    for (int j = 0; j < 4; ++j) sum += exp2(z[i][j] - ref);
    sum = sum16(sum);
    all = sum16(all);
    if (tx == 0 && r < h.T) {
      const long long at = (long long)blockIdx.x * h.T + r;
      p.top[at] = top, p.sum[at] = sum;
      if (h.smoothing != 0.0) p.all[at] = all;
    }
  }
}

// dz of the classes [v0, v0 + vc), in A
template <typename T, typename A>
__global__ void __launch_bounds__(256) logits_dz_kernel(const T* __restrict__ x, const T* __restrict__ w, const T* __restrict__ b,
                                                        const long long* __restrict__ y, const A* __restrict__ lse2,
                                                        const A* __restrict__ g, A* __restrict__ dz, int v0, int vc, Shape h) {
  __shared__ A sx[kDepth * kPitch], sw[kDepth * kPitch];
  const int r0 = blockIdx.y * kTile, c0 = v0 + blockIdx.x * kTile;
  A z[4][4];
  logits_tile<T, A>(z, sx, sw, x, w, r0, c0, h);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + 4 * ty + i;
    if (r >= h.T) continue;
    const long long yr = y[r];
    const A l2 = lse2[r], gr = g[r];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = c0 + 4 * tx + j;
      if (c >= v0 + vc) continue;
      if (b) z[i][j] += get<A>(b + c);
      A d = exp2(z[i][j] * (A)kLog2e - l2) - (A)(h.smoothing / h.V);
      if (yr == c) d -= (A)(1.0 - h.smoothing);
      // an ignored row has no gradient, whatever its logits are
      dz[(long long)r * vc + c - v0] = yr == h.ignore ? (A)0 : d * gr;
    }
  }
}

// ------------------------------------------------------------------ the tiles of a row joined

// A block has 32 rows; its 32 warps share the slots.  partial: per block the sum of the losses, the rows that count, and
// whether an ignored row's logits are not finite.
template <typename A>
__global__ void __launch_bounds__(1024) combine_kernel(Partials<A> p, const long long* __restrict__ y, int slots, void* loss,
                                                       A* saved, double* partial, Shape h) {
  __shared__ A s_top[32][33], s_sum[32][33], s_all[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = blockIdx.x * 32 + lane;
  A top = minus_inf<A>(), sum = (A)0, all = (A)0;
  if (r < h.T)
    for (int s = warp; s < slots; s += 32) {
      const long long at = (long long)s * h.T + r;
      const A t = p.top[at], n = fmax(top, t), ref = n == minus_inf<A>() ? (A)0 : n;
      sum = sum * exp2(top - ref) + p.sum[at] * exp2(t - ref);
      top = n;
      if (h.smoothing != 0.0) all += p.all[at];
    }
  s_top[lane][warp] = top, s_sum[lane][warp] = sum, s_all[lane][warp] = all;
  __syncthreads();
  if (warp) return;
  A most = minus_inf<A>();
  for (int i = 0; i < 32; ++i) most = fmax(most, s_top[lane][i]);
  const A ref = most == minus_inf<A>() ? (A)0 : most;
  sum = all = (A)0;
  for (int i = 0; i < 32; ++i) sum += s_sum[lane][i] * exp2(s_top[lane][i] - ref), all += s_all[lane][i];
  const A lse2 = ref + log2(sum);
  double counted = 0, lost = 0, strange = 0;
  if (r < h.T) {
    const long long yr = y[r];
    A v = (A)0;
    if (yr != h.ignore) {
      v = (A)kLn2 * lse2;
      // a class that does not exist: the loss is NaN (and so are the gradients it reaches)
      if (yr < 0 || yr >= h.V) v = (A)CUDART_NAN_F;
      else if (h.smoothing != 1.0) v -= (A)(1.0 - h.smoothing) * p.picked[r];
      if (h.smoothing != 0.0) v -= (A)(h.smoothing / h.V) * all;
      counted = 1, lost = (double)v;
    } else {
      strange = isfinite(lse2) ? 0 : 1;
    }
    if (h.reduction == DK_REDUCE_NONE) ((A*)loss)[r] = v;
    if (saved) saved[r] = lse2;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    counted += __shfl_xor_sync(0xffffffffu, counted, o);
    lost += __shfl_xor_sync(0xffffffffu, lost, o);
    strange += __shfl_xor_sync(0xffffffffu, strange, o);
  }
  if (lane) return;
  if (gridDim.x > 1) {
    partial[3 * blockIdx.x] = lost, partial[3 * blockIdx.x + 1] = counted, partial[3 * blockIdx.x + 2] = strange;
  } else {
    if (h.reduction != DK_REDUCE_NONE) *(A*)loss = (A)(h.reduction == DK_REDUCE_MEAN ? lost / counted : lost);
    if (saved) saved[h.T] = (A)counted, saved[h.T + 1] = (A)strange;
  }
}

// the blocks of combine_kernel joined, in fixed order
template <typename A>
__global__ void __launch_bounds__(1024) finish_kernel(const double* __restrict__ partial, int blocks, void* loss, A* saved, Shape h) {
  __shared__ double s[3][32];
  double v[3] = {0, 0, 0};
  for (int i = threadIdx.x; i < blocks; i += 1024)
    for (int k = 0; k < 3; ++k) v[k] += partial[3 * i + k];
  for (int k = 0; k < 3; ++k) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    if ((threadIdx.x & 31) == 0) s[k][threadIdx.x >> 5] = v[k];
  }
  __syncthreads();
  if (threadIdx.x >= 32) return;
  for (int k = 0; k < 3; ++k) {
    v[k] = s[k][threadIdx.x];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  }
  if (threadIdx.x) return;
  if (h.reduction != DK_REDUCE_NONE) *(A*)loss = (A)(h.reduction == DK_REDUCE_MEAN ? v[0] / v[1] : v[0]);
  if (saved) saved[h.T] = (A)v[1], saved[h.T + 1] = (A)v[2];
}

// ------------------------------------------------------------------ gradients

// g_t: what arrives for row t; nothing for an ignored one, NaN for a class that does not exist
template <typename A>
__global__ void rows_kernel(const A* __restrict__ up, const long long* __restrict__ y, const A* __restrict__ saved, A* __restrict__ g,
                            Shape h) {
  const int r = blockIdx.x * blockDim.x + threadIdx.x;
  if (r >= h.T) return;
  const long long yr = y[r];
  A v = h.reduction == DK_REDUCE_NONE ? up[r] : h.reduction == DK_REDUCE_MEAN ? up[0] / saved[h.T] : up[0];
  if (yr == h.ignore) v = (A)0;
  else if (yr < 0 || yr >= h.V) v = (A)CUDART_NAN_F;
  g[r] = v;
}

// out[m][n] (+)= sum_k a[m sm + k sk] b[k][n]; `keep`: rows of b that count (the class of a row of x; NULL: all of them)
template <typename T, typename A>
__global__ void __launch_bounds__(256) product_kernel(const A* __restrict__ a, long long sm, long long sk, const T* __restrict__ b,
                                                      const long long* __restrict__ keep, long long ignore, A* acc, T* out, int M,
                                                      int N, int K, int first, int last) {
  __shared__ A sa[kDepth * kPitch], sb[kDepth * kPitch];
  const int m0 = blockIdx.y * kTile, n0 = blockIdx.x * kTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  A v[4][4] = {};
  for (int k0 = 0; k0 < K; k0 += kDepth) {
    for (int e = threadIdx.x; e < kTile * kDepth; e += 256) {
      const int k = e / kTile, i = e % kTile;
      const bool in = k0 + k < K;
      sa[k * kPitch + i] = in && m0 + i < M ? a[(m0 + i) * sm + (k0 + k) * sk] : (A)0;
      sb[k * kPitch + i] = in && n0 + i < N && !(keep && keep[k0 + k] == ignore) ? get<A>(b + (long long)(k0 + k) * N + n0 + i) : (A)0;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kDepth; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[i][j] += sa[k * kPitch + 4 * ty + i] * sb[k * kPitch + 4 * tx + j];
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + 4 * ty + i, n = n0 + 4 * tx + j;
      if (m >= M || n >= N) continue;
      const long long at = (long long)m * N + n;
      A s = v[i][j];
      if (!first) s += acc[at];
      if (last) put<T, A>(out + at, s);
      else acc[at] = s;
    }
}

// out[v] = sum_t dz[t][v], 32 classes a block
template <typename T, typename A>
__global__ void __launch_bounds__(1024) column_sum_kernel(const A* __restrict__ dz, T* __restrict__ out, int rows, int classes) {
  __shared__ A s[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  A v = (A)0;
  if (c < classes)
    for (int r = warp; r < rows; r += 32) v += dz[(long long)r * classes + c];
  s[warp][lane] = v;
  __syncthreads();
  if (warp || c >= classes) return;
  v = (A)0;
  for (int i = 0; i < 32; ++i) v += s[i][lane];
  put<T, A>(out + c, v);
}

// ------------------------------------------------------------------ plans and launches

inline size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }

struct Layout {
  size_t bytes = 0;
  size_t take(size_t n) {
    const size_t at = bytes;
    bytes += up256(n);
    return at;
  }
};

struct ForwardPlan {
  int slots, blocks;
  size_t top, sum, all, picked, partial, bytes;
};
ForwardPlan forward_plan(int T, int V, size_t elem) {
  ForwardPlan p;
  Layout l;
  p.slots = (V + kTile - 1) / kTile, p.blocks = (T + 31) / 32;
  const size_t each = (size_t)p.slots * T * elem;
  p.top = l.take(each), p.sum = l.take(each), p.all = l.take(each);
  p.picked = l.take((size_t)T * elem), p.partial = l.take((size_t)p.blocks * 3 * sizeof(double));
  p.bytes = l.bytes;
  return p;
}

struct BackwardPlan {
  int vc;  // classes of a piece
  size_t g, dz, acc, bytes;
};
BackwardPlan backward_plan(int T, int D, int V, size_t elem, bool own_acc) {
  BackwardPlan p;
  Layout l;
  const long long budget = 64ll << 20;
  long long vc = budget / ((long long)T * (long long)elem) / kTile * kTile;
  if (vc < kTile) vc = kTile;
  p.vc = vc < V ? (int)vc : V;
  p.g = l.take((size_t)T * elem), p.dz = l.take((size_t)T * p.vc * elem);
  p.acc = p.vc < V && !own_acc ? l.take((size_t)T * D * elem) : 0;
  p.bytes = l.bytes;
  return p;
}

template <typename T, typename A>
int forward(const void* x, const void* w, const void* b, const long long* y, void* loss, void* saved, const Shape& h, void* ws,
            size_t ws_bytes, cudaStream_t s) {
  const ForwardPlan p = forward_plan(h.T, h.V, sizeof(A));
  if (!ws || ws_bytes < p.bytes) return DK_ERR_WORKSPACE;
  if ((h.T + kTile - 1) / kTile > 65535) return DK_ERR_UNSUPPORTED;
  char* m = (char*)ws;
  const Partials<A> part = {(A*)(m + p.top), (A*)(m + p.sum), (A*)(m + p.all), (A*)(m + p.picked)};
  double* partial = (double*)(m + p.partial);
  logits_stats_kernel<T, A><<<dim3(p.slots, (h.T + kTile - 1) / kTile), 256, 0, s>>>((const T*)x, (const T*)w, (const T*)b, y, part, h);
  int rc = check_launch();
  if (rc != DK_OK) return rc;
  combine_kernel<A><<<p.blocks, 1024, 0, s>>>(part, y, p.slots, loss, (A*)saved, partial, h);
  rc = check_launch();
  if (rc != DK_OK || p.blocks == 1) return rc;
  finish_kernel<A><<<1, 1024, 0, s>>>(partial, p.blocks, loss, (A*)saved, h);
  return check_launch();
}

template <typename T, typename A>
int backward(const void* up, const void* x, const void* w, const void* b, const long long* y, const void* saved, void* dx, void* dw,
             void* db, const Shape& h, void* ws, size_t ws_bytes, cudaStream_t s) {
  constexpr bool kOwn = sizeof(T) == sizeof(A);  // the gradient itself can hold the running sum
  const BackwardPlan p = backward_plan(h.T, h.D, h.V, sizeof(A), kOwn);
  if (!ws || ws_bytes < p.bytes) return DK_ERR_WORKSPACE;
  if ((h.T + kTile - 1) / kTile > 65535 || (h.V + kTile - 1) / kTile > 65535) return DK_ERR_UNSUPPORTED;
  char* m = (char*)ws;
  A *g = (A*)(m + p.g), *dz = (A*)(m + p.dz), *acc = kOwn ? (A*)dx : (A*)(m + p.acc);
  rows_kernel<A><<<(h.T + 255) / 256, 256, 0, s>>>((const A*)up, y, (const A*)saved, g, h);
  int rc = check_launch();
  const int row_tiles = (h.T + kTile - 1) / kTile, feature_tiles = (h.D + kTile - 1) / kTile;
  for (int v0 = 0; v0 < h.V && rc == DK_OK; v0 += p.vc) {
    const int vc = h.V - v0 < p.vc ? h.V - v0 : p.vc, class_tiles = (vc + kTile - 1) / kTile;
    logits_dz_kernel<T, A><<<dim3(class_tiles, row_tiles), 256, 0, s>>>((const T*)x, (const T*)w, (const T*)b, y, (const A*)saved, g,
                                                                       dz, v0, vc, h);
    rc = check_launch();
    if (rc == DK_OK && dx) {
      product_kernel<T, A><<<dim3(feature_tiles, row_tiles), 256, 0, s>>>(dz, vc, 1, (const T*)w + (long long)v0 * h.D, nullptr, 0, acc,
                                                                          (T*)dx, h.T, h.D, vc, v0 == 0, v0 + vc == h.V);
      rc = check_launch();
    }
    if (rc == DK_OK && dw) {
      product_kernel<T, A><<<dim3(feature_tiles, class_tiles), 256, 0, s>>>(dz, 1, vc, (const T*)x, y, h.ignore, nullptr,
                                                                            (T*)dw + (long long)v0 * h.D, vc, h.D, h.T, 1, 1);
      rc = check_launch();
    }
    if (rc == DK_OK && db) {
      column_sum_kernel<T, A><<<(vc + 31) / 32, 1024, 0, s>>>(dz, (T*)db + v0, h.T, vc);
      rc = check_launch();
    }
  }
  return rc;
}

bool shape_ok(int rows, int features, int classes) { return rows > 0 && features > 0 && classes > 0; }
bool dtype_ok(int d) { return d == DK_F32 || d == DK_F16 || d == DK_BF16 || d == DK_F64; }
size_t acc_size(int d) { return d == DK_F64 ? 8 : 4; }

}  // namespace head
}  // namespace dk

using namespace dk;

#define DK_HEAD_DISPATCH(dtype, EXPR)                                       \
  switch (dtype) {                                                          \
    case DK_F32: { using T = float; using A = float; return EXPR; }         \
    case DK_F16: { using T = __half; using A = float; return EXPR; }        \
    case DK_BF16: { using T = __nv_bfloat16; using A = float; return EXPR; } \
    case DK_F64: { using T = double; using A = double; return EXPR; }       \
    default: return DK_ERR_BAD_ARGUMENT;                                    \
  }

extern "C" {

size_t dk_linear_cross_entropy_forward_workspace_bytes(int rows, int features, int classes, int dtype) {
  if (!head::shape_ok(rows, features, classes) || !head::dtype_ok(dtype)) return 0;
  return head::forward_plan(rows, classes, head::acc_size(dtype)).bytes;
}

int dk_linear_cross_entropy_forward(const void* input, const void* weight, const void* bias, const long long* target, void* loss,
                                    void* saved, int rows, int features, int classes, long long ignore_index, int reduction,
                                    double label_smoothing, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (!input || !weight || !target || !loss || !head::shape_ok(rows, features, classes) || reduction < DK_REDUCE_NONE ||
      reduction > DK_REDUCE_SUM || !(label_smoothing >= 0.0 && label_smoothing <= 1.0))
    return DK_ERR_BAD_ARGUMENT;
  const head::Shape h = {rows, features, classes, ignore_index, reduction, label_smoothing};
  DK_HEAD_DISPATCH(dtype, (head::forward<T, A>(input, weight, bias, target, loss, saved, h, workspace, workspace_bytes,
                                               (cudaStream_t)stream)))
}

size_t dk_linear_cross_entropy_backward_workspace_bytes(int rows, int features, int classes, int dtype) {
  if (!head::shape_ok(rows, features, classes) || !head::dtype_ok(dtype)) return 0;
  return head::backward_plan(rows, features, classes, head::acc_size(dtype), dtype == DK_F32 || dtype == DK_F64).bytes;
}

int dk_linear_cross_entropy_backward(const void* grad_loss, const void* input, const void* weight, const void* bias,
                                     const long long* target, const void* saved, void* grad_input, void* grad_weight,
                                     void* grad_bias, int rows, int features, int classes, long long ignore_index, int reduction,
                                     double label_smoothing, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (!grad_loss || !input || !weight || !target || !saved || !head::shape_ok(rows, features, classes) ||
      reduction < DK_REDUCE_NONE || reduction > DK_REDUCE_SUM || !(label_smoothing >= 0.0 && label_smoothing <= 1.0))
    return DK_ERR_BAD_ARGUMENT;
  const head::Shape h = {rows, features, classes, ignore_index, reduction, label_smoothing};
  DK_HEAD_DISPATCH(dtype, (head::backward<T, A>(grad_loss, input, weight, bias, target, saved, grad_input, grad_weight, grad_bias, h,
                                                workspace, workspace_bytes, (cudaStream_t)stream)))
}

}  // extern "C"
