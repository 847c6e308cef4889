// The last linear layer of a classifier with its softmax cross entropy, without keeping the logits.
//
//   z = x W^T + b                        x [T, D], W [V, D], b [V] or none
//   lse_t = log sum_v exp z_tv
//   loss_t = lse_t - (1 - s) z_t[y_t] - s / V sum_v z_tv            s: label smoothing; 0 for a row that is ignored
//   dz_tv = g_t (exp(z_tv - lse_t) - (1 - s) [v = y_t] - s / V)     g_t: what arrives from behind the loss
//   dx = dz W,   dW = dz^T x,   db = sum_t dz_t
//
// Forward: tiles of logits live in registers only; each leaves (maximum, sum of exponentials) of its rows, and a second
// kernel joins the tiles of a row in fixed order.  Backward: a piece of the rows or of the classes at a time (all of
// them, where dz is no larger than a piece), its logits once more, its dz into the workspace, then the two products.
//
// Here: the C entry points, the kernel that joins a row's tiles, and fp64 on the CUDA cores.  The other types: dk_head_tc.cu.
#include <limits.h>
#include <math_constants.h>

#include "dk_head.cuh"

namespace dk {
namespace head {

// e^v of differences that are not above zero
__device__ __forceinline__ double power(double v) { return exp(v); }
__device__ __forceinline__ float power(float v) { return exp2f(v * (float)kLog2e); }

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
                                                           Partials<double> p, unsigned* count, Shape h) {
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *count = 0;
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
      } else {
        z[i][j] = minus_inf<double>();
      }
      top = fmax(top, z[i][j]);
    }
    top = max16(top);
    const double ref = top == minus_inf<double>() ? 0 : top;
    double sum = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) sum += exp(z[i][j] - ref);
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
                                                        const double* __restrict__ saved, Upstream<double> up, double* __restrict__ dz, int v0, int vc, Shape h) {
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
    const double ref = saved[r], inv = saved[h.T + r], gr = upstream_row(up, r, yr, h.ignore, h.V) * upstream_back(up);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = c0 + 4 * tx + j;
      if (c >= v0 + vc) continue;
      if (b) z[i][j] += b[c];
      double d = exp(z[i][j] - ref) * inv - h.smoothing / h.V;
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

// ------------------------------------------------------------------ a few rows

// eight values, beginning on 16 bytes
template <typename T> __device__ __forceinline__ void load8(float (&v)[8], const T* p);
template <> __device__ __forceinline__ void load8<float>(float (&v)[8], const float* p) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
template <> __device__ __forceinline__ void load8<__half>(float (&v)[8], const __half* p) {
  const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
  const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}
template <> __device__ __forceinline__ void load8<__nv_bfloat16>(float (&v)[8], const __nv_bfloat16* p) {
  const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
  const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}

// R rows of x (h.T of them exist), read again and again from L1; a warp takes C classes at a time, its lanes share the features, lane r keeps
// the statistics of row r.  One slot a block.
template <typename T, int R, int C>
__global__ void __launch_bounds__(256, R * C <= 8 ? 4 : 2) few_rows_kernel(const T* __restrict__ x, const T* __restrict__ w,
                                                                          const T* __restrict__ b, const long long* __restrict__ y,
                                                                          Partials<float> p, unsigned* count, Shape h) {
  __shared__ float s_top[8][R], s_sum[8][R], s_all[8][R];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  before_all();
  let_next();
  if (blockIdx.x == 0 && threadIdx.x == 0) *count = 0;
  const long long own = lane < h.T && lane < R ? y[lane] : -1;
  const T* from[R];
#pragma unroll
  for (int r = 0; r < R; ++r) from[r] = x + (long long)(r < h.T ? r : 0) * h.D;
  float top = minus_inf<float>(), sum = 0, all = 0;
  for (int c0 = (blockIdx.x * 8 + warp) * C; c0 < h.V; c0 += gridDim.x * 8 * C) {
    float acc[C][R] = {};
    const T* row[C];
#pragma unroll
    for (int c = 0; c < C; ++c) row[c] = w + (long long)(c0 + c < h.V ? c0 + c : c0) * h.D;
    if (h.D % 8 == 0) {
#pragma unroll(R * C <= 4 ? 4 : 1)
      for (int k = lane * 8; k < h.D; k += 256) {
        float wv[C][8];
#pragma unroll
        for (int c = 0; c < C; ++c) load8<T>(wv[c], row[c] + k);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          float xv[8];
          load8<T>(xv, from[r] + k);
#pragma unroll
          for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[c][r] += wv[c][e] * xv[e];
        }
      }
    } else {
      for (int k = lane; k < h.D; k += 32)
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const float v = (float)row[c][k];
#pragma unroll
          for (int r = 0; r < R; ++r) acc[c][r] += v * (float)from[r][k];
        }
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float z = 0;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float v = acc[c][r];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane == r) z = v;
      }
      if (c0 + c < h.V) {
        if (b) z += (float)b[c0 + c];
        if (own == c0 + c) p.picked[lane] = z;
        all += z;
        const float n = fmaxf(top, z), ref = n == minus_inf<float>() ? 0.0f : n;
        sum = sum * power(top - ref) + power(z - ref);
        top = n;
      }
    }
  }
  if (lane < R) s_top[warp][lane] = top, s_sum[warp][lane] = sum, s_all[warp][lane] = all;
  __syncthreads();
  if (threadIdx.x >= R || threadIdx.x >= h.T) return;
  top = minus_inf<float>(), sum = 0, all = 0;
  for (int i = 0; i < 8; ++i) top = fmaxf(top, s_top[i][lane]);
  const float ref = top == minus_inf<float>() ? 0.0f : top;
  for (int i = 0; i < 8; ++i) sum += s_sum[i][lane] * power(s_top[i][lane] - ref), all += s_all[i][lane];
  const long long at = (long long)blockIdx.x * h.T + lane;
  p.top[at] = top, p.sum[at] = sum;
  if (h.smoothing != 0.0) p.all[at] = all;
}

// 16-bit weights: four rows take 10.2 / 25.6 / 77.8 us here and 12.5 / 28.7 / 77.8 on the tensor cores (1000 and 21841 classes of 1280 features, 65536 of
// 2048), eight 10.4 / 34.8 / 114.  fp32 weights, which the tensor cores want laid out in pieces first: eight rows 12.3 / 53.6 / 162 and 30.7 / 127 / 567.
bool few_rows(int T, int dtype) { return T <= (dtype == DK_F32 ? 8 : 4); }
// one class a warp, four where there are enough of them
static bool four_classes(int V) { return V >= device_sm_count() * 8 * 4; }
int few_slots(int V) {
  const int blocks = div_up(V, 8 * (four_classes(V) ? 4 : 1)), most = device_sm_count() * 4;
  return blocks < most ? blocks : most;
}
template <typename T, int R>
static int launch_few(const void* x, const void* w, const void* b, const long long* y, const Partials<float>& p, unsigned* count,
                      const Shape& h, cudaStream_t s) {
  return launch_after(four_classes(h.V) ? few_rows_kernel<T, R, 4> : few_rows_kernel<T, R, 1>, few_slots(h.V), 256, 0, 1, s, (const T*)x,
                      (const T*)w, (const T*)b, y, p, count, h);
}
template <typename T>
int launch_few_rows(const void* x, const void* w, const void* b, const long long* y, const Partials<float>& p, unsigned* count,
                    const Shape& h, cudaStream_t s) {
  if (h.T == 1) return launch_few<T, 1>(x, w, b, y, p, count, h, s);
  if (h.T == 2) return launch_few<T, 2>(x, w, b, y, p, count, h, s);
  if (sizeof(T) == 2 || h.T <= 4) return launch_few<T, 4>(x, w, b, y, p, count, h, s);
  return launch_few<T, sizeof(T) == 2 ? 4 : 8>(x, w, b, y, p, count, h, s);
}
template int launch_few_rows<__half>(const void*, const void*, const void*, const long long*, const Partials<float>&, unsigned*, const Shape&, cudaStream_t);
template int launch_few_rows<__nv_bfloat16>(const void*, const void*, const void*, const long long*, const Partials<float>&, unsigned*, const Shape&, cudaStream_t);
template int launch_few_rows<float>(const void*, const void*, const void*, const long long*, const Partials<float>&, unsigned*, const Shape&, cudaStream_t);

// ------------------------------------------------------------------ the tiles of a row joined

// A block has `groups` times 32 rows; its other warps share the slots of those.  partial: per block the sum of the losses, the rows that
// count, and whether an ignored row's logits are not finite; the last block to finish joins those, in fixed order.
template <typename A>
__global__ void __launch_bounds__(1024) combine_kernel(Partials<A> p, const long long* __restrict__ y, int slots, int groups, void* loss,
                                                       A* saved, double* partial, unsigned* count, Shape h) {
  __shared__ A s_top[32][33], s_sum[32][33], s_all[32][33];  // [warp][lane]
  __shared__ double s_v[32][3];
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5, share = warps / groups;
  const int group = (threadIdx.x >> 5) / share, warp = (threadIdx.x >> 5) - group * share;
  const int r = (blockIdx.x * groups + group) * 32 + lane;
  before_all();
  A top = minus_inf<A>(), sum = (A)0, all = (A)0;
  if (r < h.T) {
#pragma unroll 4
    for (int s = warp; s < slots; s += share) {
      const long long at = (long long)s * h.T + r;
      const A t = p.top[at], n = fmax(top, t), ref = n == minus_inf<A>() ? (A)0 : n;
      sum = sum * power(top - ref) + p.sum[at] * power(t - ref);
      top = n;
      if (h.smoothing != 0.0) all += p.all[at];
    }
  }
  if (share > 1) {
    s_top[threadIdx.x >> 5][lane] = top, s_sum[threadIdx.x >> 5][lane] = sum, s_all[threadIdx.x >> 5][lane] = all;
    __syncthreads();
  }
  A ref = top == minus_inf<A>() ? (A)0 : top;
  if (warp == 0 && share > 1) {
    const int first = group * share;
#pragma unroll 8
    for (int i = 1; i < share; ++i) top = fmax(top, s_top[first + i][lane]);
    ref = top == minus_inf<A>() ? (A)0 : top;
    sum = all = (A)0;
#pragma unroll 8
    for (int i = 0; i < share; ++i) sum += s_sum[first + i][lane] * power(s_top[first + i][lane] - ref), all += s_all[first + i][lane];
  }
  const A ls = log(sum);
  double v[3] = {0, 0, 0};  // loss, rows that count, ignored rows that are not finite
  if (warp == 0 && r < h.T) {
    const long long yr = y[r];
    A one = (A)0;
    if (yr != h.ignore) {
      // from differences to the largest logit: a loss near zero is not that of two large numbers
      one = ls;
      if (yr < 0 || yr >= h.V) one = (A)CUDART_NAN_F;  // a class that does not exist: so are the gradients it reaches
      else if (h.smoothing != 1.0) one += (A)(1.0 - h.smoothing) * (ref - p.picked[r]);
      if (h.smoothing != 0.0) one += (A)h.smoothing * (ref - all / (A)h.V);
      v[0] = (double)one, v[1] = 1;
    } else {
      v[2] = isfinite(ref + ls) ? 0 : 1;
    }
    if (h.reduction == DK_REDUCE_NONE) ((A*)loss)[r] = one;
    if (saved) saved[r] = ref, saved[h.T + r] = (A)1 / sum;
  }
  if (!saved && h.reduction == DK_REDUCE_NONE) return;
  if (warp == 0) {
    for (int k = 0; k < 3; ++k)
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    if (lane == 0 && groups > 1)
      for (int k = 0; k < 3; ++k) s_v[group][k] = v[k];
  }
  if (groups > 1) __syncthreads();
  if (threadIdx.x >= 32) return;
  if (groups > 1) {
    v[0] = v[1] = v[2] = 0;
    for (int g = 0; g < groups; ++g)
      for (int k = 0; k < 3; ++k) v[k] += s_v[g][k];
  }
  if (gridDim.x > 1) {
    unsigned turn = 0;
    if (lane == 0) {
      for (int k = 0; k < 3; ++k) partial[3ll * blockIdx.x + k] = v[k];
      __threadfence();
      turn = atomicAdd(count, 1u);
    }
    if (__shfl_sync(0xffffffffu, turn, 0) != gridDim.x - 1) return;
    __threadfence();
    v[0] = v[1] = v[2] = 0;
#pragma unroll 4
    for (unsigned i = lane; i < gridDim.x; i += 32)
      for (int k = 0; k < 3; ++k) v[k] += __ldcg(partial + 3ll * i + k);
    for (int k = 0; k < 3; ++k)
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  }
  if (lane) return;
  if (h.reduction != DK_REDUCE_NONE) *(A*)loss = (A)(h.reduction == DK_REDUCE_MEAN ? v[0] / v[1] : v[0]);
  if (saved) saved[2ll * h.T] = (A)v[1], saved[2ll * h.T + 1] = (A)v[2];
}

template <typename A>
int launch_combine(const Partials<A>& p, const long long* y, int slots, void* loss, void* saved, double* partial, const Shape& h,
                   cudaStream_t s) {
  int share = 1;  // four slots a warp
  while (share < 32 && share * 4 < slots) share *= 2;
  // as many rows a block as leave every SM one: fewer blocks to join
  int groups = 1;
  while (groups * 2 * share <= 32 && div_up(h.T, 64 * groups) >= device_sm_count()) groups *= 2;
  return launch_after(combine_kernel<A>, div_up(h.T, kCombineRows * groups), 32 * share * groups, 0, 1, s, p, y, slots, groups, loss, (A*)saved,
                      partial, combine_count(partial, h.T), h);
}
template int launch_combine<float>(const Partials<float>&, const long long*, int, void*, void*, double*, const Shape&, cudaStream_t);

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
  size_t dz, bytes;
};
BackwardPlan backward_plan(int T, int V) {
  BackwardPlan p;
  Layout l;
  long long vc = (64ll << 20) / ((long long)T * 8) / kTile * kTile;
  if (vc < kTile) vc = kTile;
  p.vc = vc < V ? (int)vc : V;
  p.dz = l.take((size_t)T * p.vc * 8);
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
  double* partial = (double*)(m + p.partial);
  logits_stats_kernel<<<dim3(p.slots, row_tiles), 256, 0, s>>>(x, w, b, y, part, combine_count(partial, h.T), h);
  const int rc = check_launch();
  return rc != DK_OK ? rc : launch_combine<double>(part, y, p.slots, loss, saved, partial, h, s);
}

int backward64(const void* up, const double* x, const double* w, const double* b, const long long* y, const double* saved, double* dx,
               double* dw, double* db, const Shape& h, void* ws, size_t ws_bytes, cudaStream_t s) {
  const BackwardPlan p = backward_plan(h.T, h.V);
  if (!ws || ws_bytes < p.bytes) return DK_ERR_WORKSPACE;
  const int row_tiles = div_up(h.T, kTile), feature_tiles = div_up(h.D, kTile);
  if (row_tiles > 65535 || div_up(p.vc, kTile) > 65535) return DK_ERR_UNSUPPORTED;
  double* dz = (double*)((char*)ws + p.dz);
  const Upstream<double> u = {(const double*)up, saved + 2ll * h.T, nullptr, h.reduction, 1.0};
  int rc = DK_OK;
  for (int v0 = 0; v0 < h.V && rc == DK_OK; v0 += p.vc) {
    const int vc = h.V - v0 < p.vc ? h.V - v0 : p.vc, class_tiles = div_up(vc, kTile);
    logits_dz_kernel<<<dim3(class_tiles, row_tiles), 256, 0, s>>>(x, w, b, y, saved, u, dz, v0, vc, h);
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
// Loops and tiles step past a size by up to 19 thousand (few_rows_kernel: 4 blocks an SM, 32 classes a block); their indices are 32-bit.
// The bytes of dz as a whole, from which its pieces are planned, are a 64-bit number.
constexpr int kLargest = INT_MAX - 0xffff;
bool sizes_fit(int rows, int features, int classes) {
  return rows <= kLargest && features <= kLargest && classes <= kLargest && (long long)rows * classes <= 1ll << 56;
}
bool dtype_ok(int d) { return d == DK_F32 || d == DK_F16 || d == DK_BF16 || d == DK_F64; }
bool options_ok(int reduction, double smoothing) {
  return reduction >= DK_REDUCE_NONE && reduction <= DK_REDUCE_SUM && smoothing >= 0.0 && smoothing <= 1.0;
}
// the kernels store 16 bytes at a time into the workspace as well
bool aligned16(const void* a, const void* b) { return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) == 0; }

}  // namespace
}  // namespace head
}  // namespace dk

using namespace dk;

extern "C" {

long long dk_linear_cross_entropy_wait_limit(long long nanoseconds) { return head::set_wait_limit(nanoseconds); }

size_t dk_linear_cross_entropy_forward_workspace_bytes(int rows, int features, int classes, int dtype) {
  if (!head::shape_ok(rows, features, classes) || !head::dtype_ok(dtype) || !head::sizes_fit(rows, features, classes)) return 0;
  return dtype == DK_F64 ? head::forward_plan(rows, classes).bytes : head::tc_forward_bytes(rows, features, classes, dtype);
}

int dk_linear_cross_entropy_forward(const void* input, const void* weight, const void* bias, const long long* target, void* loss,
                                    void* saved, int rows, int features, int classes, long long ignore_index, int reduction,
                                    double label_smoothing, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (!input || !weight || !target || !loss || !head::shape_ok(rows, features, classes) || !head::dtype_ok(dtype) ||
      !head::options_ok(reduction, label_smoothing) || !head::aligned16(input, weight) || !head::aligned16(workspace, nullptr))
    return DK_ERR_BAD_ARGUMENT;
  if (!head::sizes_fit(rows, features, classes)) return DK_ERR_UNSUPPORTED;
  const head::Shape h = {rows, features, classes, ignore_index, reduction, label_smoothing};
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == DK_F64)
    return head::forward64((const double*)input, (const double*)weight, (const double*)bias, target, loss, saved, h, workspace,
                           workspace_bytes, s);
  return head::tc_forward(input, weight, bias, target, loss, saved, h, dtype, workspace, workspace_bytes, s);
}

size_t dk_linear_cross_entropy_backward_workspace_bytes(int rows, int features, int classes, int dtype) {
  if (!head::shape_ok(rows, features, classes) || !head::dtype_ok(dtype) || !head::sizes_fit(rows, features, classes)) return 0;
  return dtype == DK_F64 ? head::backward_plan(rows, classes).bytes : head::tc_backward_bytes(rows, features, classes, dtype);
}

int dk_linear_cross_entropy_backward(const void* grad_loss, const void* input, const void* weight, const void* bias,
                                     const long long* target, const void* saved, void* grad_input, void* grad_weight,
                                     void* grad_bias, int rows, int features, int classes, long long ignore_index, int reduction,
                                     double label_smoothing, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (!grad_loss || !input || !weight || !target || !saved || !head::shape_ok(rows, features, classes) || !head::dtype_ok(dtype) ||
      !head::options_ok(reduction, label_smoothing) || !head::aligned16(input, weight) || !head::aligned16(grad_input, grad_weight) ||
      !head::aligned16(workspace, nullptr))
    return DK_ERR_BAD_ARGUMENT;
  if (!head::sizes_fit(rows, features, classes)) return DK_ERR_UNSUPPORTED;
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
