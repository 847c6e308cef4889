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

template <typename A> __device__ __forceinline__ A minus_inf() { return (A)-CUDART_INF_F; }

// ------------------------------------------------------------------ fp64 on the CUDA cores (what gradients are checked with)

constexpr int kTile = 64, kDepth = 16, kPitch = kTile + 4;

// acc[i][j] = sum_k x[r0 + 4 ty + i][k] W[c0 + 4 tx + j][k]; rows and classes outside count as zeros
__device__ __forceinline__ void logits_tile(double (&acc)[4][4], double* sx, double* sw, const double* __restrict__ x,
                                            const double* __restrict__ w, int r0, int c0, const Shape& h) {
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0;
  for (int k0 = 0; k0 < h.D; k0 += kDepth) {
    for (int e = threadIdx.x; e < kTile * kDepth; e += 256) {
      const int r = e / kDepth, k = e % kDepth;
      const bool in = k0 + k < h.D;
      sx[k * kPitch + r] = in && r0 + r < h.T ? x[(long long)(r0 + r) * h.D + k0 + k] : 0;
      sw[k * kPitch + r] = in && c0 + r < h.V ? w[(long long)(c0 + r) * h.D + k0 + k] : 0;
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
__device__ __forceinline__ double max16(double v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ double sum16(double v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__global__ void __launch_bounds__(256) logits_stats_kernel(const double* __restrict__ x, const double* __restrict__ w,
                                                           const double* __restrict__ b, const long long* __restrict__ y,
                                                           Partials<double> p, Shape h) {
  __shared__ double sx[kDepth * kPitch], sw[kDepth * kPitch];
  const int r0 = blockIdx.y * kTile, c0 = blockIdx.x * kTile;
  double z[4][4];
  logits_tile(z, sx, sw, x, w, r0, c0, h);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + 4 * ty + i;
    const long long yr = r < h.T ? y[r] : -1;
    double top = minus_inf<double>(), all = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = c0 + 4 * tx + j;
      if (c < h.V) {
        if (b) z[i][j] += b[c];
        if (yr == c) p.picked[r] = z[i][j];
        all += z[i][j];
        z[i][j] *= kLog2e;
      } else {
        z[i][j] = minus_inf<double>();
      }
      top = fmax(top, z[i][j]);
    }
    top = max16(top);
    const double ref = top == minus_inf<double>() ? 0 : top;
    double sum = 0;
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

// dz of the classes [v0, v0 + vc)
__global__ void __launch_bounds__(256) logits_dz_kernel(const double* __restrict__ x, const double* __restrict__ w,
                                                        const double* __restrict__ b, const long long* __restrict__ y,
                                                        const double* __restrict__ lse2, const double* __restrict__ g,
                                                        double* __restrict__ dz, int v0, int vc, Shape h) {
  __shared__ double sx[kDepth * kPitch], sw[kDepth * kPitch];
  const int r0 = blockIdx.y * kTile, c0 = v0 + blockIdx.x * kTile;
  double z[4][4];
  logits_tile(z, sx, sw, x, w, r0, c0, h);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + 4 * ty + i;
    if (r >= h.T) continue;
    const long long yr = y[r];
    const double l2 = lse2[r], gr = g[r];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = c0 + 4 * tx + j;
      if (c >= v0 + vc) continue;
      if (b) z[i][j] += b[c];
      double d = exp2(z[i][j] * kLog2e - l2) - h.smoothing / h.V;
      if (yr == c) d -= 1.0 - h.smoothing;
      // an ignored row has no gradient, whatever its logits are
      dz[(long long)r * vc + c - v0] = yr == h.ignore ? 0 : d * gr;
    }
  }
}

// out[m][n] (+)= sum_k a[m sm + k sk] b[k][n]; target (NULL: all rows count): the class of row k of b, which an ignored row's is not
__global__ void __launch_bounds__(256) product_kernel(const double* __restrict__ a, long long sm, long long sk,
                                                      const double* __restrict__ b, const long long* __restrict__ target,
                                                      long long ignore, double* out, int M, int N, int K, int first) {
  __shared__ double sa[kDepth * kPitch], sb[kDepth * kPitch];
  const int m0 = blockIdx.y * kTile, n0 = blockIdx.x * kTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  double v[4][4] = {};
  for (int k0 = 0; k0 < K; k0 += kDepth) {
    for (int e = threadIdx.x; e < kTile * kDepth; e += 256) {
      const int k = e / kTile, i = e % kTile;
      const bool in = k0 + k < K;
      sa[k * kPitch + i] = in && m0 + i < M ? a[(m0 + i) * sm + (k0 + k) * sk] : 0;
      sb[k * kPitch + i] = in && n0 + i < N && !(target && target[k0 + k] == ignore) ? b[(long long)(k0 + k) * N + n0 + i] : 0;
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
      out[at] = first ? v[i][j] : out[at] + v[i][j];
    }
}

// out[v] = sum_t dz[t][v], 32 classes a block
__global__ void __launch_bounds__(1024) column_sum_kernel(const double* __restrict__ dz, double* __restrict__ out, int rows, int classes) {
  __shared__ double s[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  double v = 0;
  if (c < classes)
    for (int r = warp; r < rows; r += 32) v += dz[(long long)r * classes + c];
  s[warp][lane] = v;
  __syncthreads();
  if (warp || c >= classes) return;
  v = 0;
  for (int i = 0; i < 32; ++i) v += s[i][lane];
  out[c] = v;
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

// ------------------------------------------------------------------ what arrives for each row

// for a whole call, g of a row that counts (not DK_REDUCE_NONE)
template <typename A>
__device__ __forceinline__ A common_g(const A* up, const A* saved, const Shape& h) {
  return h.reduction == DK_REDUCE_MEAN ? up[0] / saved[h.T] : up[0];
}
// the power of two that brings `largest` to [2^14, 2^15)
template <typename A>
__device__ __forceinline__ A scale_for(A largest) {
  if (!(largest > (A)0) || !isfinite(largest)) return (A)1;
  const int e = 14 - ilogb(largest);
  return (A)ldexp(1.0, e < -100 ? -100 : e > 100 ? 100 : e);
}

// the largest |g| of the rows, one block
template <typename A>
__global__ void __launch_bounds__(1024) largest_kernel(const A* __restrict__ up, const long long* __restrict__ y, A* back, Shape h) {
  __shared__ A s[32];
  A v = (A)0;
  for (int r = threadIdx.x; r < h.T; r += 1024)
    if (y[r] != h.ignore) v = fmax(v, fabs(up[r]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x >= 32) return;
  v = s[threadIdx.x];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (threadIdx.x == 0) back[1] = v;
}

// g_t: what arrives for row t; nothing for an ignored one, NaN for a class that does not exist
template <typename A>
__global__ void rows_kernel(const A* __restrict__ up, const long long* __restrict__ y, const A* __restrict__ saved, A* __restrict__ g,
                            A* back, Shape h) {
  const int r = blockIdx.x * blockDim.x + threadIdx.x;
  if (r >= h.T) return;
  const long long yr = y[r];
  const bool each = h.reduction == DK_REDUCE_NONE;
  A v = each ? up[r] : common_g(up, saved, h);
  if (back) {
    const A f = scale_for(each ? back[1] : (A)fabs(v));
    if (r == 0) back[0] = (A)1 / f;
    v *= f;
  }
  if (yr == h.ignore) v = (A)0;
  else if (yr < 0 || yr >= h.V) v = (A)CUDART_NAN_F;
  g[r] = v;
}

template <typename A>
int launch_combine(const Partials<A>& p, const long long* y, int slots, void* loss, void* saved, double* partial, const Shape& h,
                   cudaStream_t s) {
  const int blocks = div_up(h.T, kCombineRows);
  combine_kernel<A><<<blocks, 1024, 0, s>>>(p, y, slots, loss, (A*)saved, partial, h);
  const int rc = check_launch();
  if (rc != DK_OK || blocks == 1) return rc;
  finish_kernel<A><<<1, 1024, 0, s>>>(partial, blocks, loss, (A*)saved, h);
  return check_launch();
}
template int launch_combine<float>(const Partials<float>&, const long long*, int, void*, void*, double*, const Shape&, cudaStream_t);

template <typename A>
int launch_rows(const void* up, const long long* y, const void* saved, A* g, A* back, const Shape& h, cudaStream_t s) {
  if (back && h.reduction == DK_REDUCE_NONE) {
    largest_kernel<A><<<1, 1024, 0, s>>>((const A*)up, y, back, h);
    const int rc = check_launch();
    if (rc != DK_OK) return rc;
  }
  rows_kernel<A><<<div_up(h.T, 256), 256, 0, s>>>((const A*)up, y, (const A*)saved, g, back, h);
  return check_launch();
}
template int launch_rows<float>(const void*, const long long*, const void*, float*, float*, const Shape&, cudaStream_t);

// ------------------------------------------------------------------ fp64 calls

namespace {

struct ForwardPlan {
  int slots;
  size_t top, sum, all, picked, partial, bytes;
};
ForwardPlan forward_plan(int T, int V) {
  ForwardPlan p;
  Layout l;
  p.slots = div_up(V, kTile);
  const size_t each = (size_t)p.slots * T * sizeof(double);
  p.top = l.take(each), p.sum = l.take(each), p.all = l.take(each);
  p.picked = l.take((size_t)T * sizeof(double)), p.partial = l.take(combine_bytes(T));
  p.bytes = l.bytes;
  return p;
}

struct BackwardPlan {
  int vc;  // classes of a piece
  size_t g, dz, bytes;
};
BackwardPlan backward_plan(int T, int V) {
  BackwardPlan p;
  Layout l;
  long long vc = (64ll << 20) / ((long long)T * 8) / kTile * kTile;
  if (vc < kTile) vc = kTile;
  p.vc = vc < V ? (int)vc : V;
  p.g = l.take((size_t)T * 8), p.dz = l.take((size_t)T * p.vc * 8);
  p.bytes = l.bytes;
  return p;
}

int forward64(const double* x, const double* w, const double* b, const long long* y, void* loss, void* saved, const Shape& h, void* ws,
              size_t ws_bytes, cudaStream_t s) {
  const ForwardPlan p = forward_plan(h.T, h.V);
  if (!ws || ws_bytes < p.bytes) return DK_ERR_WORKSPACE;
  const int row_tiles = div_up(h.T, kTile);
  if (row_tiles > 65535) return DK_ERR_UNSUPPORTED;
  char* m = (char*)ws;
  const Partials<double> part = {(double*)(m + p.top), (double*)(m + p.sum), (double*)(m + p.all), (double*)(m + p.picked)};
  logits_stats_kernel<<<dim3(p.slots, row_tiles), 256, 0, s>>>(x, w, b, y, part, h);
  const int rc = check_launch();
  return rc != DK_OK ? rc : launch_combine<double>(part, y, p.slots, loss, saved, (double*)(m + p.partial), h, s);
}

int backward64(const void* up, const double* x, const double* w, const double* b, const long long* y, const double* saved, double* dx,
               double* dw, double* db, const Shape& h, void* ws, size_t ws_bytes, cudaStream_t s) {
  const BackwardPlan p = backward_plan(h.T, h.V);
  if (!ws || ws_bytes < p.bytes) return DK_ERR_WORKSPACE;
  const int row_tiles = div_up(h.T, kTile), feature_tiles = div_up(h.D, kTile);
  if (row_tiles > 65535 || div_up(p.vc, kTile) > 65535) return DK_ERR_UNSUPPORTED;
  double *g = (double*)((char*)ws + p.g), *dz = (double*)((char*)ws + p.dz);
  int rc = launch_rows<double>(up, y, saved, g, nullptr, h, s);
  for (int v0 = 0; v0 < h.V && rc == DK_OK; v0 += p.vc) {
    const int vc = h.V - v0 < p.vc ? h.V - v0 : p.vc, class_tiles = div_up(vc, kTile);
    logits_dz_kernel<<<dim3(class_tiles, row_tiles), 256, 0, s>>>(x, w, b, y, saved, g, dz, v0, vc, h);
    rc = check_launch();
    if (rc == DK_OK && dx) {
      product_kernel<<<dim3(feature_tiles, row_tiles), 256, 0, s>>>(dz, vc, 1, w + (long long)v0 * h.D, nullptr, 0, dx, h.T, h.D, vc, v0 == 0);
      rc = check_launch();
    }
    if (rc == DK_OK && dw) {
      product_kernel<<<dim3(feature_tiles, class_tiles), 256, 0, s>>>(dz, 1, vc, x, y, h.ignore, dw + (long long)v0 * h.D, vc, h.D, h.T, 1);
      rc = check_launch();
    }
    if (rc == DK_OK && db) {
      column_sum_kernel<<<div_up(vc, 32), 1024, 0, s>>>(dz, db + v0, h.T, vc);
      rc = check_launch();
    }
  }
  return rc;
}

bool shape_ok(int rows, int features, int classes) { return rows > 0 && features > 0 && classes > 0; }
bool dtype_ok(int d) { return d == DK_F32 || d == DK_F16 || d == DK_BF16 || d == DK_F64; }
bool options_ok(int reduction, double smoothing) {
  return reduction >= DK_REDUCE_NONE && reduction <= DK_REDUCE_SUM && smoothing >= 0.0 && smoothing <= 1.0;
}
bool aligned16(const void* a, const void* b) { return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) == 0; }

}  // namespace
}  // namespace head
}  // namespace dk

using namespace dk;

extern "C" {

size_t dk_linear_cross_entropy_forward_workspace_bytes(int rows, int features, int classes, int dtype) {
  if (!head::shape_ok(rows, features, classes) || !head::dtype_ok(dtype)) return 0;
  return dtype == DK_F64 ? head::forward_plan(rows, classes).bytes : head::tc_forward_bytes(rows, features, classes, dtype);
}

int dk_linear_cross_entropy_forward(const void* input, const void* weight, const void* bias, const long long* target, void* loss,
                                    void* saved, int rows, int features, int classes, long long ignore_index, int reduction,
                                    double label_smoothing, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (!input || !weight || !target || !loss || !head::shape_ok(rows, features, classes) || !head::dtype_ok(dtype) ||
      !head::options_ok(reduction, label_smoothing) || !head::aligned16(input, weight))
    return DK_ERR_BAD_ARGUMENT;
  const head::Shape h = {rows, features, classes, ignore_index, reduction, label_smoothing};
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == DK_F64)
    return head::forward64((const double*)input, (const double*)weight, (const double*)bias, target, loss, saved, h, workspace,
                           workspace_bytes, s);
  return head::tc_forward(input, weight, bias, target, loss, saved, h, dtype, workspace, workspace_bytes, s);
}

size_t dk_linear_cross_entropy_backward_workspace_bytes(int rows, int features, int classes, int dtype) {
  if (!head::shape_ok(rows, features, classes) || !head::dtype_ok(dtype)) return 0;
  return dtype == DK_F64 ? head::backward_plan(rows, classes).bytes : head::tc_backward_bytes(rows, features, classes, dtype);
}

int dk_linear_cross_entropy_backward(const void* grad_loss, const void* input, const void* weight, const void* bias,
                                     const long long* target, const void* saved, void* grad_input, void* grad_weight,
                                     void* grad_bias, int rows, int features, int classes, long long ignore_index, int reduction,
                                     double label_smoothing, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (!grad_loss || !input || !weight || !target || !saved || !head::shape_ok(rows, features, classes) || !head::dtype_ok(dtype) ||
      !head::options_ok(reduction, label_smoothing) || !head::aligned16(input, weight) || !head::aligned16(grad_input, grad_weight))
    return DK_ERR_BAD_ARGUMENT;
  if (!grad_input && !grad_weight && !grad_bias) return DK_OK;
  const head::Shape h = {rows, features, classes, ignore_index, reduction, label_smoothing};
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == DK_F64)
    return head::backward64(grad_loss, (const double*)input, (const double*)weight, (const double*)bias, target, (const double*)saved,
                            (double*)grad_input, (double*)grad_weight, (double*)grad_bias, h, workspace, workspace_bytes, s);
  return head::tc_backward(grad_loss, input, weight, bias, target, saved, grad_input, grad_weight, grad_bias, h, dtype, workspace,
                           workspace_bytes, s);
}

}  // extern "C"
