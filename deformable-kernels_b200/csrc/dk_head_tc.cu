// The three products of the classifier head on the fifth-generation tensor cores: logits with the statistics of their rows
// (forward), logits with dz (backward), and both gradient products in one launch.
//
// One persistent kernel with one block per SM; where there are enough tiles two SMs share one of 256 x 256
// (cta_group::2: each holds 128 rows of either operand in shared memory and 128 rows of the accumulator in TMEM), else
// each has its own of 128 x BN.  Warp 0 fills a ring of shared-memory stages by TMA, warp 1 of the leading block issues
// the mma, the last eight warps take the finished accumulator out of TMEM while the other half of TMEM receives the next
// tile.  An operand is K-major (rows of the tensor are rows of the product) or MN-major (columns are); both
// come as boxes of 64 x 64 values, 128 swizzled bytes a row.
//
// 16-bit sums stay in TMEM, those of the logits up to 4096 features (kLongDepth).
// fp32 operands are three bf16 pieces each (8 bits a piece, 24 in all).  A stage holds one piece of both; the six products of
// pieces that reach 2^-24 are taken from three stages, that of the leading pieces into one accumulator, the five
// small ones into another: the additions of the tensor cores cut, and a cut of the small sum costs nothing.  After every four steps
// the epilogue adds both to sums in registers, which round, so that no more than 16 cuts meet in one value.
//
// Measured, one B200: logits with statistics 1.29 ms at 8192 x 2048 x 65536 (2.20 Tflop: 1.71 Pflop/s, tensor pipe 96 % of the
// cycles), 0.146 at 4096 x 1280 x 21841 (1.57 Pflop/s, 87 %: 19 rounds of tiles, the last a half); with dz 0.174 (70 %: its 179 MB
// contend with the loads in L2, 10 TB/s of them; without the stores 88 % of the cycles); the two products 0.313
// (1.46 Pflop/s, 83 %).  The clock is at 1.5 GHz under this load: power is the bound of large calls.
// Small calls are launches and the latency of one tile: 10 us for a tile of 1280 features.

#include <float.h>
#include <math_constants.h>

#include <atomic>
#include <type_traits>

#include "dk_head.cuh"
#include "dk_tc.cuh"

namespace dk {
namespace head {

using ring::smem_u32;

namespace {

__device__ int g_head_error;  // set when a bounded wait ran out
// Nanoseconds.  The longest wait is the epilogue's for one sum in TMEM: 1024 steps of a gradient (split_products), 64 of the logits (kLongDepth), 4 of
// fp32 with six products each.  A step takes 0.235 us where nothing hides the loads' latency: a quarter of a millisecond.
constexpr unsigned long long kWaitLimit = 2000000000;
std::atomic<unsigned long long> g_wait_limit{kWaitLimit};

constexpr int kBox = 64;                    // values per side of a TMA box
constexpr int kBoxBytes = kBox * kBox * 2;  // 8192
constexpr int kStages = 6;
constexpr int kThreads = 384;
constexpr int kStageWarp = 4096;            // staging of an epilogue warp: 32 rows of 128 bytes

struct SharedTail {
  float bias[2][256];
  unsigned long long full[kStages], empty[kStages], acc_full[2], acc_empty[2];
  unsigned tmem;
  int abort_flag;
};

template <int CG, int BN>
__host__ __device__ constexpr int stage_bytes() { return 128 * 128 + BN / CG * 128; }
template <int CG, int BN>
constexpr int smem_bytes() { return kStages * stage_bytes<CG, BN>() + 8 * kStageWarp + (int)sizeof(SharedTail); }

// ---- PTX

__device__ __forceinline__ unsigned cluster_rank() {
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// the address of the same variable in block `rank` of the cluster
__device__ __forceinline__ unsigned map_rank(unsigned addr, unsigned rank) {
  unsigned r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void arrive_cluster(unsigned bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(bar) : "memory");
}
template <int CG>
__device__ __forceinline__ void tmem_alloc(unsigned slot) {
  if (CG == 1) {
    tc::tmem_alloc_all(slot);
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(slot) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
  }
}
template <int CG>
__device__ __forceinline__ void tmem_free(unsigned addr) {
  if (CG == 1) tc::tmem_free_all(addr);
  else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;\n" ::"r"(addr) : "memory");
}
// all mma of this thread so far -> one arrival on `bar`, in both blocks of a pair
template <int CG>
__device__ __forceinline__ void commit(unsigned bar) {
  if (CG == 1) {
    tc::commit(bar);
  } else {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(bar),
                 "h"((unsigned short)3)
                 : "memory");
  }
}
template <int CG>
__device__ __forceinline__ void mma_ss(unsigned d, uint64_t a, uint64_t b, unsigned idesc, bool acc) {
  if (CG == 1)
    asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"((unsigned)acc)
                 : "memory");
  else
    asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"((unsigned)acc)
                 : "memory");
}
// One box into this block's shared memory; a pair counts the bytes of both blocks on the leader's barrier.
template <int CG>
__device__ __forceinline__ void load_box(unsigned dst, const CUtensorMap* tm, int x, int y, int z, unsigned bar) {
  if (CG == 1)
    ring::tma_load_3d(dst, tm, x, y, z, bar);
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(
            dst),
        "l"(tm), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void store_box(const CUtensorMap* tm, unsigned src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];\n" ::"l"(tm), "r"(x), "r"(y), "r"(z),
               "r"(src)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;\n" ::: "memory");
}
__device__ __forceinline__ void stores_have_read() { asm volatile("cp.async.bulk.wait_group.read 0;\n" ::: "memory"); }
__device__ __forceinline__ void stores_done() { asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory"); }

__device__ __forceinline__ void ld32(float (&r)[32], unsigned a) {
  unsigned* u = reinterpret_cast<unsigned*>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
      "%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]),
        "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]), "=r"(u[18]),
        "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]), "=r"(u[25]), "=r"(u[26]), "=r"(u[27]),
        "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(a));
}
__device__ __forceinline__ void wait_ld(float (&r)[32]) {
  unsigned* u = reinterpret_cast<unsigned*>(r);
  asm volatile("tcgen05.wait::ld.sync.aligned;\n"
               : "+r"(u[0]), "+r"(u[1]), "+r"(u[2]), "+r"(u[3]), "+r"(u[4]), "+r"(u[5]), "+r"(u[6]), "+r"(u[7]), "+r"(u[8]), "+r"(u[9]),
                 "+r"(u[10]), "+r"(u[11]), "+r"(u[12]), "+r"(u[13]), "+r"(u[14]), "+r"(u[15]), "+r"(u[16]), "+r"(u[17]), "+r"(u[18]),
                 "+r"(u[19]), "+r"(u[20]), "+r"(u[21]), "+r"(u[22]), "+r"(u[23]), "+r"(u[24]), "+r"(u[25]), "+r"(u[26]), "+r"(u[27]),
                 "+r"(u[28]), "+r"(u[29]), "+r"(u[30]), "+r"(u[31])
               :
               : "memory");
}
__device__ __forceinline__ void ld16(float (&r)[16], unsigned a) {
  unsigned* u = reinterpret_cast<unsigned*>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]),
        "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
      : "r"(a));
}
__device__ __forceinline__ void wait_ld(float (&r)[16]) {
  unsigned* u = reinterpret_cast<unsigned*>(r);
  asm volatile("tcgen05.wait::ld.sync.aligned;\n"
               : "+r"(u[0]), "+r"(u[1]), "+r"(u[2]), "+r"(u[3]), "+r"(u[4]), "+r"(u[5]), "+r"(u[6]), "+r"(u[7]), "+r"(u[8]), "+r"(u[9]),
                 "+r"(u[10]), "+r"(u[11]), "+r"(u[12]), "+r"(u[13]), "+r"(u[14]), "+r"(u[15])
               :
               : "memory");
}
__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(v));
  return r;
}

// ---- descriptors
template <typename E>
__host__ __device__ constexpr unsigned type_bits() { return sizeof(E) == 2 && std::is_same<E, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u; }
// operand of 128-byte rows, swizzled in groups of eight rows.  K-major: `lead` is not looked at, `stride` = bytes between groups of eight
// rows; MN-major: `lead` = bytes between blocks of 64 columns, `stride` = between groups of eight rows (of K)
__device__ __forceinline__ uint64_t swizzled(unsigned addr, unsigned lead, unsigned stride) {
  return tc::sdesc(addr, lead, stride) | (2ull << 61);
}

// ---- a wait of a whole warp that ends: true once any thread of the block gave up
__device__ __forceinline__ bool try_wait(unsigned bar, unsigned parity) {
  unsigned ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ unsigned long long nanoseconds() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;\n" : "=l"(t));
  return t;
}
// True once any thread of the block gave up: `limit` nanoseconds without the phase.  Of the time between two polls ten milliseconds count at
// most: a process that is suspended for longer has not waited.
constexpr unsigned long long kMostBetweenPolls = 10000000;
__device__ __forceinline__ bool wait(unsigned bar, unsigned parity, volatile int* abort_flag, unsigned long long limit) {
  bool gone = *abort_flag != 0;
  if (!gone && !try_wait(bar, parity)) {
    unsigned long long last = nanoseconds(), spent = 0;
    gone = true;
    for (unsigned i = 0; i < 1u << 30; ++i) {
      if (try_wait(bar, parity)) {
        gone = false;
        break;
      }
      const unsigned long long now = nanoseconds(), step = now - last;
      spent += step < kMostBetweenPolls ? step : kMostBetweenPolls, last = now;
      if (*abort_flag || spent > limit) break;
    }
    if (gone) *abort_flag = 1;
  }
  return __any_sync(0xffffffffu, gone);
}

// 16-byte piece q of row r in a staging buffer of 128-byte rows
__device__ __forceinline__ unsigned staged(unsigned base, int r, int q) { return base + r * 128 + ((q ^ (r & 7)) << 4); }
__device__ __forceinline__ void sts16(unsigned a, unsigned x, unsigned y, unsigned z, unsigned w) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};\n" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ uint4 lds16(unsigned a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ unsigned lds4(unsigned a) {
  unsigned v;
  asm volatile("ld.shared.b32 %0, [%1];\n" : "=r"(v) : "r"(a) : "memory");
  return v;
}
template <typename E> __device__ __forceinline__ unsigned pack(float a, float b);
template <> __device__ __forceinline__ unsigned pack<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const unsigned*>(&h);
}
template <> __device__ __forceinline__ unsigned pack<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const unsigned*>(&h);
}
template <typename E> __device__ __forceinline__ float2 unpack(unsigned v);
template <> __device__ __forceinline__ float2 unpack<__half>(unsigned v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
template <> __device__ __forceinline__ float2 unpack<__nv_bfloat16>(unsigned v) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}

// ---- arguments

__device__ __forceinline__ int div_up_device(int a, int b) { return (a + b - 1) / b; }

enum Role { kStats, kDz, kGrad };

// one of the gradient products, out[M][N] = sum over K; tiles [splits][m][n]
struct Product {
  int M, N, blocks;           // blocks: 64-deep steps of K
  int tiles_m, tiles_n, splits, per;  // per: steps of a split
  float* acc;                 // running sum over the pieces, or [splits][M][N]
  void* out;                  // NULL: the sums stay in acc
  int first;                  // 0: add what acc holds
};

// which items a cluster takes (item_of); short_less <= short_more
struct Schedule {
  int long_product, n_long, n_short, short_less, short_more;
};

struct Args {
  CUtensorMap x, x_clean, w, dz, dz_out;
  // logits
  int rows, classes;          // of this piece
  int row0, class0;           // where the piece begins
  int depth;                  // 64-deep steps over the features
  int tiles_m, tiles_n, group;
  const void* bias;           // of the parameters' type, or NULL
  const long long* target;    // of the piece's first row
  long long ignore;
  float* top;                 // [slots][rows]
  float* sum;
  float* all;                 // NULL without label smoothing
  float* picked;
  unsigned* done;             // forward: set to zero for the kernel that follows
  const float *ref, *inv;     // of the piece's rows: p = exp(z - ref) inv
  Upstream<float> up;
  int all_classes;            // of the call
  float* column_sums;         // [rows / 32][classes], NULL: no bias gradient
  float smooth_each, smooth_own;  // s / V, 1 - s
  const float* strange;       // != 0: some ignored row's features are not finite, x_clean has them zeroed; NULL: they are zero anyway
  const void* dirty;          // backward, first piece: x, of which `clean` becomes a copy without ignored rows where `strange` says so
  void* clean;
  int width;                  // of x
  int up_rows;                // of the call
  const long long* target_all;
  unsigned long long wait_limit;  // nanoseconds
  // gradients
  Product dw, dx;
  Schedule schedule;
  float* acc_b;               // bias gradient of the pieces before
  void* out_b;                // NULL: it goes to acc_b
  int first_b;
};

struct Item {
  int product;  // gradients: 0 dw, 1 dx
  int m, n;     // tile
  int split, first, count;  // steps of K
};

// The i-th item of a cluster.  The tiles of the logits are alike and go round.  Those of the two gradient products are not: the product with
// the longer sums goes round first, and of the shorter ones the clusters that got one less of the long get `short_more` rounds, the
// others `short_less` (Schedule below), so that all end together.
template <int ROLE>
__device__ __forceinline__ bool item_of(const Args& a, int cluster, int clusters, int i, Item& t) {
  t.product = 0, t.split = 0, t.first = 0, t.count = a.depth;
  if (ROLE != kGrad) {
    i = i * clusters + cluster;
    if (i >= a.tiles_m * a.tiles_n) return false;
    // columns of tiles, `group` tiles of rows high: their part of x stays in L2 while the weights stream past once a group
    const int per = a.group * a.tiles_n, gi = i / per, left = a.tiles_m - gi * a.group, high = left < a.group ? left : a.group;
    const int r = i - gi * per;
    t.n = r / high, t.m = gi * a.group + r - t.n * high;
    return true;
  }
  const Schedule& c = a.schedule;
  const int rest = c.n_long % clusters;
  const bool more_long = cluster < rest;
  const int own_long = c.n_long / clusters + (more_long ? 1 : 0);
  bool is_long = i < own_long;
  if (is_long) {
    i = i * clusters + cluster;
  } else {
    i -= own_long;
    const int own_short = more_long ? c.short_less : c.short_more;
    if (i >= own_short) return false;
    // rounds of all clusters, then those of the clusters with more of them
    i = i < c.short_less ? i * clusters + cluster : c.short_less * clusters + (i - c.short_less) * (clusters - rest) + cluster - rest;
    if (i >= c.n_short) return false;
  }
  t.product = is_long ? c.long_product : 1 - c.long_product;
  const Product& p = t.product ? a.dx : a.dw;
  t.n = i % p.tiles_n, i /= p.tiles_n;
  t.m = i % p.tiles_m, t.split = i / p.tiles_m;
  t.first = t.split * p.per;
  t.count = p.blocks - t.first < p.per ? p.blocks - t.first : p.per;
  return true;
}

// ---- on the side, a warp of every block

// the 16-bit x with its ignored rows zeroed
__device__ __forceinline__ void clean_rows(const Args& a, int lane) {
  const int pieces = a.width / 8;
  const uint4* src = (const uint4*)a.dirty;
  uint4* dst = (uint4*)a.clean;
  for (int r = blockIdx.x; r < a.up_rows; r += gridDim.x) {
    const bool in = a.target_all[r] != a.ignore;
    for (int q = lane; q < pieces; q += 32) dst[(long long)r * pieces + q] = in ? src[(long long)r * pieces + q] : make_uint4(0, 0, 0, 0);
  }
}

// db from the sums over 32 rows each, in fixed order: a warp has 32 classes, or fewer (and several lanes for each) where that keeps
// more warps busy
template <typename O>
__device__ __forceinline__ void join_columns(const Args& a, int lane) {
  int wide = 32;
  while (wide > 4 && div_up_device(a.classes, wide) * 2 <= (int)gridDim.x) wide >>= 1;
  const int slabs = div_up_device(a.rows, 32), c_lane = lane & (wide - 1), s_lane = lane / wide, step = 32 / wide;
  const float back = upstream_back(a.up);
  for (int c0 = blockIdx.x * wide; c0 < a.classes; c0 += gridDim.x * wide) {
    const int c = c0 + c_lane;
    float v = 0;
    if (c < a.classes) {
#pragma unroll 8
      for (int r = s_lane; r < slabs; r += step) v += a.column_sums[(long long)r * a.classes + c];
    }
    for (int o = wide; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (s_lane == 0 && c < a.classes) {
      v *= back;
      if (!a.first_b) v += a.acc_b[c];
      if (a.out_b) ((O*)a.out_b)[c] = (O)v;
      else a.acc_b[c] = v;
    }
  }
}

// one 64-deep step of a product: four mma; `fresh`: what the accumulator held is dropped
template <int CG>
__device__ __forceinline__ void product(unsigned d, uint64_t a, uint64_t b, unsigned at, unsigned idesc, unsigned step_a, unsigned step_b,
                                        bool fresh) {
#pragma unroll
  for (int q = 0; q < 4; ++q) mma_ss<CG>(d + at, a + (uint64_t)(q * step_a >> 4), b + (uint64_t)(q * step_b >> 4), idesc, !fresh || q > 0);
}

// lane j: the sum over the warp's lanes of v[j], in fixed order; every step halves the columns that a lane still has
__device__ __forceinline__ float column_sum(const float (&v)[32], int lane) {
  float r[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float mine = lane & 16 ? v[i + 16] : v[i], other = lane & 16 ? v[i] : v[i + 16];
    r[i] = mine + __shfl_xor_sync(0xffffffffu, other, 16);
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float mine = lane & o ? r[i + o] : r[i], other = lane & o ? r[i] : r[i + o];
      r[i] = mine + __shfl_xor_sync(0xffffffffu, other, o);
    }
  return r[0];
}

// 16 columns of both sums of an fp32 accumulator, added to v (set: stored)
template <int BN>
__device__ __forceinline__ void take_both(float* v, unsigned a, bool set) {
  float lead[16], small[16];
  ld16(lead, a);
  ld16(small, a + BN);
  wait_ld(lead);
  wait_ld(small);
#pragma unroll
  for (int j = 0; j < 16; ++j) v[j] = set ? lead[j] + small[j] : v[j] + (lead[j] + small[j]);
}

// the same where there is one sum
__device__ __forceinline__ void take_one(float* v, unsigned a, bool set) {
  float sum[16];
  ld16(sum, a);
  wait_ld(sum);
#pragma unroll
  for (int j = 0; j < 16; ++j) v[j] = set ? sum[j] : v[j] + sum[j];
}

// ---- the kernel

// 16-bit logits: an addition of the tensor cores cuts, so the error of a sum in TMEM grows with its length (losses of 1024 rows, 1000 classes, bf16
// features: 4.7e-7 of themselves at 1024 features, 1.1e-6 at 2560, 1.8e-6 at 4096, 7.8e-6 at 16384, 1.2e-4 at 262144).  Above 4096 features the sum is added up in
// registers every 2048 (9e-7 at 16384); that costs up to a fifth of the time of many tiles (4096 rows, 4096 features, 21841 classes: loss 458 -> 540 us, step
// 2.34 -> 2.49 ms; at 2560 features it would be 300 -> 355 and 1.43 -> 1.64), and 1 to 3 % of few (1024 x 16384 x 1000).
constexpr int kLongDepth = 64, kLongChunk = 32;  // steps of 64 features
// fp32: errors of dx and dw against fp64 as 32-bit products have them or smaller (256 x 1280 x 1000: 3.5e-7 and 3.4e-7, theirs 7.1e-7 and 5.1e-7; features of
// one sign 4.7e-7 and 7.5e-7, theirs 4.7e-7 and 3.0e-7).  Every eight steps: 6.6e-7 and 3.7e-7, 6.6e-7 and 8.2e-7, losses near zero (4 x 2225 x 2) 1.6e-6 in
// place of 4.8e-7, for 1 % less time; every two halves them again for 5 % more.
constexpr int kPiecesChunk = 4;
static_assert(kLongDepth >= kLongChunk, "the last sum is taken by itself: there is one before it");

// LONG: many features, whose sums are added up in registers every kLongChunk steps
template <int CG, int BN, int ROLE, typename E, int PIECES, bool LONG>
__global__ void __launch_bounds__(kThreads, 1) head_kernel(const __grid_constant__ Args a) {
  extern __shared__ __align__(1024) unsigned char smem[];
  constexpr int kStage = stage_bytes<CG, BN>();
  constexpr int kBoxesB = BN / CG / kBox;          // boxes of B a block loads
  constexpr int kGroups = BN >= 128 ? 2 : 1;       // epilogue warps side by side
  constexpr int kWide = BN / kGroups;              // columns of an epilogue warp
  constexpr int kAcc = PIECES == 1 ? BN : 2 * BN;  // columns of an accumulator
  constexpr bool kTaken = PIECES > 1 || LONG;      // sums in registers
  constexpr int kChunk = PIECES > 1 ? kPiecesChunk : LONG ? kLongChunk : 1 << 30;  // steps between two takings of the accumulator
  static_assert(PIECES == 1 || kWide == 64, "the sums of a row are 64 registers");
  static_assert(2 * kAcc <= 512, "two accumulators in TMEM");
  SharedTail& t = *reinterpret_cast<SharedTail*>(smem + kStages * kStage + 8 * kStageWarp);
  const unsigned base = smem_u32(smem);
  if (base & 1023) {  // the swizzled boxes need it; the same in every block
    if (threadIdx.x == 0) g_head_error = 2;
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned rank = CG == 1 ? 0u : cluster_rank();
  const int cluster = blockIdx.x / CG, clusters = gridDim.x / CG;
  volatile int* abort_flag = &t.abort_flag;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) ring::mbar_init(smem_u32(&t.full[s]), 1), ring::mbar_init(smem_u32(&t.empty[s]), 1);
    for (int b = 0; b < 2; ++b) ring::mbar_init(smem_u32(&t.acc_full[b]), 1), ring::mbar_init(smem_u32(&t.acc_empty[b]), CG * 4 * kGroups);
    t.abort_flag = 0;
    ring::fence_barrier_init();
  }
  if (warp == 2) tmem_alloc<CG>(smem_u32(&t.tmem));
  tc::fence_before();
  if (CG == 1) __syncthreads();
  else cluster_sync();
  tc::fence_after();
  const unsigned tmem = t.tmem;

  let_next();
  if (warp == 0) {
    // ---------------- producer
    const bool one = tc::elect_one();
    const CUtensorMap* mx = &a.x;
    before_all();
    if (ROLE == kGrad && a.strange && *a.strange != 0.0f) mx = &a.x_clean;
    int fill = 0;
    Item it;
    for (int i = 0; item_of<ROLE>(a, cluster, clusters, i, it); ++i) {
      const int m0 = (it.m * CG + (int)rank) * 128, n0 = it.n * BN + (int)rank * (BN / CG);
      for (int kb = it.first; kb < it.first + it.count; ++kb) {
        for (int piece = 0; piece < PIECES; ++piece, ++fill) {
          const int s = fill % kStages;
          if (wait(smem_u32(&t.empty[s]), ((fill / kStages) & 1) ^ 1, abort_flag, a.wait_limit)) continue;
          const unsigned sa = base + s * kStage, sb = sa + 128 * 128;
          unsigned bar = smem_u32(&t.full[s]);
          if (CG == 2) bar = map_rank(bar, 0);
          if (one) {
            if (rank == 0) ring::mbar_arrive_expect_tx(smem_u32(&t.full[s]), CG * kStage);
            const int k0 = kb * kBox;
            if (ROLE != kGrad) {
              for (int q = 0; q < 2; ++q) load_box<CG>(sa + q * kBoxBytes, &a.x, k0, a.row0 + m0 + q * kBox, piece, bar);
              for (int q = 0; q < kBoxesB; ++q) load_box<CG>(sb + q * kBoxBytes, &a.w, k0, a.class0 + n0 + q * kBox, piece, bar);
            } else if (it.product == 0) {
              for (int q = 0; q < 2; ++q) load_box<CG>(sa + q * kBoxBytes, &a.dz, m0 + q * kBox, k0, piece, bar);
              for (int q = 0; q < kBoxesB; ++q) load_box<CG>(sb + q * kBoxBytes, mx, n0 + q * kBox, a.row0 + k0, piece, bar);
            } else {
              for (int q = 0; q < 2; ++q) load_box<CG>(sa + q * kBoxBytes, &a.dz, k0, m0 + q * kBox, piece, bar);
              for (int q = 0; q < kBoxesB; ++q) load_box<CG>(sb + q * kBoxBytes, &a.w, n0 + q * kBox, a.class0 + k0, piece, bar);
            }
          }
          __syncwarp();
        }
      }
    }
    // every stage handed back: nothing of this block is in flight any more
    for (int s = 0; s < kStages && s < fill; ++s) {
      const int last = (fill - 1 - s) / kStages * kStages + s;
      (void)wait(smem_u32(&t.empty[s]), (last / kStages) & 1, abort_flag, a.wait_limit);
    }
  } else if (warp == 1) {
    // ---------------- mma, the leading block only
    before_all();  // it reads nothing, but its waits are not to run while the kernel before does
    if (rank == 0) {
      const bool one = tc::elect_one();
      constexpr unsigned kDesc = (1u << 4) | type_bits<E>() | ((unsigned)(BN >> 3) << 17) | ((unsigned)(128 * CG >> 4) << 24);
      int fill = 0, round = 0;
      Item it;
      for (int tile = 0; item_of<ROLE>(a, cluster, clusters, tile, it); ++tile) {
        // both operands of the logits are K-major; W and x of the gradients are MN-major, dz is either
        const bool ta = ROLE == kGrad && it.product == 0, tb = ROLE == kGrad;
        const unsigned idesc = kDesc | ((unsigned)ta << 15) | ((unsigned)tb << 16);
        const unsigned lead = kBoxBytes, step_a = ta ? 2048 : 32, step_b = tb ? 2048 : 32;
        for (int k0 = 0; k0 < it.count; k0 += kChunk, ++round) {
          const int b = round & 1, end = it.count - k0 < kChunk ? it.count : k0 + kChunk;
          bool gone = wait(smem_u32(&t.acc_empty[b]), ((round >> 1) & 1) ^ 1, abort_flag, a.wait_limit);
          tc::fence_after();
          const unsigned d = tmem + b * kAcc;
          for (int k = k0; k < end; ++k, fill += PIECES) {
            uint64_t da[PIECES], db[PIECES];
#pragma unroll
            for (int p = 0; p < PIECES; ++p) {
              const int s = (fill + p) % kStages;
              gone = wait(smem_u32(&t.full[s]), ((fill + p) / kStages) & 1, abort_flag, a.wait_limit);
              if (gone) break;
              tc::fence_after();
              const unsigned sa = base + s * kStage;
              da[p] = swizzled(sa, lead, 1024), db[p] = swizzled(sa + 128 * 128, lead, 1024);
              if (one) {
                // product (i, j) of pieces i + j <= 2 as soon as the later of the two has landed
#pragma unroll
                for (int i = 0; i <= p; ++i) {
                  if (PIECES == 1 || i + p <= 2) product<CG>(d, da[p], db[i], p == 0 ? 0 : BN, idesc, step_a, step_b,
                                                            k == k0 && (p == 0 || (p == 1 && i == 0)));
                  if (i != p && i + p <= 2) product<CG>(d, da[i], db[p], BN, idesc, step_a, step_b, false);
                }
              }
              __syncwarp();
            }
            if (gone) continue;
            if (one) {
#pragma unroll
              for (int p = 0; p < PIECES; ++p) commit<CG>(smem_u32(&t.empty[(fill + p) % kStages]));
            }
            __syncwarp();
          }
          if (one && !gone) commit<CG>(smem_u32(&t.acc_full[b]));
          __syncwarp();
        }
      }
    }
  } else if (warp == 3) {
    // ---------------- what else there is to do
    before_all();
    if (ROLE == kStats && blockIdx.x == 0 && lane == 0) *a.done = 0;
    if (ROLE == kDz && a.clean && *a.strange != 0.0f) clean_rows(a, lane);
    if (ROLE == kGrad && a.column_sums) join_columns<typename std::conditional<PIECES == 1, E, float>::type>(a, lane);
  } else if (warp >= 4 && (warp - 4) >> 2 < kGroups) {
    // ---------------- epilogue
    before_all();
    const int sub = warp & 3, grp = (warp - 4) >> 2;
    const unsigned stage = base + kStages * kStage + (warp - 4) * kStageWarp;
    const unsigned lanes = (unsigned)(32 * sub) << 16;
    constexpr float kL2 = (float)kLog2e;
    // the accumulator `b` is taken: the mma may write it again
    auto release = [&](int b) {
      tc::fence_before();
      __syncwarp();
      if (lane == 0) {
        const unsigned bar = smem_u32(&t.acc_empty[b]);
        if (CG == 1) ring::mbar_arrive(bar);
        else arrive_cluster(map_rank(bar, 0));
      }
    };
    // What a tile needs from global memory is asked for a tile ahead: the row's class and statistics, and the thread's share of what is added to
    // the logits (-inf outside, where the product is zero).
    constexpr int kShare = (BN + 128 * kGroups - 1) / (128 * kGroups);
    struct Ahead {
      long long y;
      float ref, inv, up, bias[kShare];
    };
    auto ask = [&](Ahead& n, const Item& it) {
      if (ROLE == kGrad) return;
#pragma unroll
      for (int i = 0; i < kShare; ++i) {
        const int v = it.n * BN + (int)threadIdx.x - 128 + i * 128 * kGroups;
        n.bias[i] = v < a.classes ? (a.bias ? (PIECES == 1 ? (float)((const E*)a.bias)[a.class0 + v] : ((const float*)a.bias)[a.class0 + v]) : 0.0f)
                                  : -CUDART_INF_F;
      }
      const int row = (it.m * CG + (int)rank) * 128 + 32 * sub + lane;
      n.y = a.ignore;
      if (row < a.rows) {
        n.y = a.target[row];
        if (ROLE == kDz) n.ref = a.ref[row], n.inv = a.inv[row], n.up = a.up.reduction == DK_REDUCE_NONE ? a.up.up[row] : 1.0f;
      }
    };
    const float unit = ROLE == kDz ? upstream_unit(a.up) : 0.0f, back = ROLE == kGrad ? upstream_back(a.up) : 0.0f;
    int round = 0;
    Item it, next;
    Ahead now = {}, ahead = {};
    bool more = item_of<ROLE>(a, cluster, clusters, 0, next);
    if (more) ask(ahead, next);
    for (int tile = 0; more; ++tile) {
      it = next, now = ahead;
      const int row_base = (it.m * CG + (int)rank) * 128 + 32 * sub, row = row_base + lane;
      const int col_base = it.n * BN + grp * kWide;
      float* bias = t.bias[tile & 1];
      if (ROLE != kGrad) {
        // the other half is read until the next tile's barrier
#pragma unroll
        for (int i = 0; i < kShare; ++i)
          if ((int)threadIdx.x - 128 + i * 128 * kGroups < BN) bias[(int)threadIdx.x - 128 + i * 128 * kGroups] = now.bias[i];
        __syncwarp();
        asm volatile("bar.sync 1, %0;\n" ::"n"(128 * kGroups) : "memory");
      }
      more = item_of<ROLE>(a, cluster, clusters, tile + 1, next);
      if (more) ask(ahead, next);
      const long long y = row < a.rows ? now.y : -1;
      const bool live = ROLE == kDz && row < a.rows && y != a.ignore;
      const float ref = now.ref, inv = now.inv;
      // the row's own class as a column of this warp, -1: elsewhere
      const long long far = y - a.class0 - col_base;
      const int own = far >= 0 && far < kWide ? (int)far : -1;
      float got[kTaken ? kWide / 32 : 1][32];  // the sums that have left TMEM
      bool gone = false;  // the products never came: what the tile leaves is NaN
      if (kTaken) {
        // fp32: all of them; else all but the last
        for (int k = 0; PIECES > 1 ? k < it.count : k + kChunk < it.count; k += kChunk, ++round) {
          const int bk = round & 1;
          gone |= wait(smem_u32(&t.acc_full[bk]), (round >> 1) & 1, abort_flag, a.wait_limit);
          tc::fence_after();
#pragma unroll
          for (int h = 0; h < (kTaken ? kWide / 16 : 0); ++h) {
            __syncwarp();
            float* sums = &got[h >> 1][(h & 1) * 16];
            const unsigned from = tmem + lanes + bk * kAcc + grp * kWide + 16 * h;
            if (PIECES == 1) take_one(sums, from, k == 0);
            else take_both<BN>(sums, from, k == 0);
          }
          release(bk);
        }
      }
      const int b = round & 1;
      const unsigned d = tmem + lanes + b * kAcc + grp * kWide;
      if (PIECES == 1) {
        gone |= wait(smem_u32(&t.acc_full[b]), (round >> 1) & 1, abort_flag, a.wait_limit);
        tc::fence_after();
        ++round;
      }
      const float g = !gone && y >= 0 && y < a.all_classes ? now.up * unit : CUDART_NAN_F;  // of a live row
      const float factor = gone ? CUDART_NAN_F : back;
      // 32 columns from c on
      auto columns = [&](float (&v)[32], int c) {
        if (PIECES == 1) {
          __syncwarp();
          ld32(v, d + c);
          wait_ld(v);
        }
        if (kTaken) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = PIECES == 1 ? v[j] + got[kTaken ? c >> 5 : 0][j] : got[kTaken ? c >> 5 : 0][j];
        }
      };
      if (ROLE == kStats) {
        float top = -CUDART_INF_F, sum = 0, all = 0, picked = 0;
#pragma unroll(kTaken ? kWide / 32 : 1)
        for (int c0 = 0; c0 < kWide; c0 += 32) {
          float z[32];
          columns(z, c0);
          const float4* bp = reinterpret_cast<const float4*>(bias + grp * kWide + c0);
          float most[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const float4 v = bp[q];
            z[4 * q] += v.x, z[4 * q + 1] += v.y, z[4 * q + 2] += v.z, z[4 * q + 3] += v.w;
          }
          if (own >= c0 && own < c0 + 32) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (own == c0 + j) picked = z[j];
          }
          if (a.all) {
            const int in = a.classes - col_base - c0;
            float some[4] = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 32; ++j) some[j & 3] += j < in ? z[j] : 0.0f;
            all += (some[0] + some[1]) + (some[2] + some[3]);
          }
          // chains of eight: four at a time
#pragma unroll
          for (int j = 0; j < 32; ++j) most[j & 3] = fmaxf(most[j & 3], z[j]);
          const float n = fmaxf(top, fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]))), ref = n == -CUDART_INF_F ? 0.0f : n;
          float part[4] = {0, 0, 0, 0};
#pragma unroll
          for (int j = 0; j < 32; ++j) part[j & 3] += ex2((z[j] - ref) * kL2);
          sum = sum * ex2((top - ref) * kL2) + ((part[0] + part[1]) + (part[2] + part[3]));
          top = n;
        }
        if (row < a.rows) {
          const long long at = (long long)(it.n * kGroups + grp) * a.rows + row;
          a.top[at] = top, a.sum[at] = gone ? CUDART_NAN_F : sum;
          if (a.all) a.all[at] = all;
          if (own >= 0 && own + col_base < a.classes) a.picked[row] = picked;
        }
      } else if (ROLE == kDz) {
#pragma unroll(kTaken ? kWide / kBox : 1)
        for (int c0 = 0; c0 < kWide; c0 += kBox) {
          const bool inside = row_base < a.rows && col_base + c0 < a.classes;
          if (!inside) break;  // of the whole warp
          float v[2][32];
          columns(v[0], c0);
          columns(v[1], c0 + 32);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float4* bp = reinterpret_cast<const float4*>(bias + grp * kWide + c0 + 32 * h);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const float4 bb = bp[q];
              v[h][4 * q] += bb.x, v[h][4 * q + 1] += bb.y, v[h][4 * q + 2] += bb.z, v[h][4 * q + 3] += bb.w;
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              float p = fmaf(ex2((v[h][j] - ref) * kL2), inv, -a.smooth_each);
              if (own == c0 + 32 * h + j) p -= a.smooth_own;
              v[h][j] = live ? p * g : 0.0f;
            }
          }
          // of dz as it is, not as the products take it; 16-bit types: while the copy of the tile is under way
          auto sum_columns = [&] {
            float* to = a.column_sums + (long long)(row_base >> 5) * a.classes;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int c = col_base + c0 + 32 * h + lane;
              const float all = column_sum(v[h], lane);
              if (c < a.classes) to[c] = all;
            }
          };
          if (PIECES > 1 && a.column_sums) sum_columns();  // the pieces take v apart
#pragma unroll
          for (int pc = 0; pc < PIECES; ++pc) {
            if (lane == 0) stores_have_read();
            __syncwarp();
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              unsigned w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float& v0 = v[q >> 2][(q & 3) * 8 + 2 * e];
                float& v1 = v[q >> 2][(q & 3) * 8 + 2 * e + 1];
                w[e] = pack<E>(v0, v1);
                if (PIECES > 1) {
                  const float2 f = unpack<E>(w[e]);
                  v0 -= f.x, v1 -= f.y;
                }
              }
              sts16(staged(stage, lane, q), w[0], w[1], w[2], w[3]);
            }
            ring::fence_proxy_async();
            __syncwarp();
            if (lane == 0) store_box(&a.dz_out, stage, col_base + c0, row_base, pc);
          }
          if (PIECES == 1 && a.column_sums) sum_columns();
        }
      } else {
        const Product& p = it.product ? a.dx : a.dw;
        float* acc = p.acc ? p.acc + (p.splits > 1 ? (long long)it.split * p.M * p.N : 0) : nullptr;
        const bool out16 = PIECES == 1 && p.out;  // 16-bit results; else fp32, to the gradient or to the sums
        float* to32 = p.out ? (float*)p.out : acc;
        const bool vec = (p.N & (out16 ? 7 : 3)) == 0;
        if (PIECES == 1 && out16 && vec && p.first) {
          // the result at once: packed before the staging, 16 bytes a lane and eight lanes a row behind it
#pragma unroll 1
          for (int c0 = 0; c0 < kWide; c0 += kBox) {
            if (row_base >= p.M || col_base + c0 >= p.N) break;  // of the whole warp
            float v[2][32];
            __syncwarp();
            ld32(v[0], d + c0);
            ld32(v[1], d + c0 + 32);
            wait_ld(v[0]);
            wait_ld(v[1]);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const float* f = &v[q >> 2][(q & 3) * 8];
              sts16(staged(stage, lane, q), pack<E>(f[0] * factor, f[1] * factor), pack<E>(f[2] * factor, f[3] * factor),
                    pack<E>(f[4] * factor, f[5] * factor), pack<E>(f[6] * factor, f[7] * factor));
            }
            __syncwarp();
            const int c = col_base + c0 + 8 * (lane & 7);
            E* to = (E*)p.out + (long long)(row_base + (lane >> 3)) * p.N + c;
#pragma unroll
            for (int r = 0; r < 32; r += 4, to += 4ll * p.N)
              if (row_base + r + (lane >> 3) < p.M && c < p.N) *reinterpret_cast<uint4*>(to) = lds16(staged(stage, r + (lane >> 3), lane & 7));
          }
          release(b);
          continue;
        }
#pragma unroll(PIECES == 1 ? 1 : 2)
        for (int c0 = 0; c0 < kWide; c0 += 32) {
          if (row_base >= p.M || col_base + c0 >= p.N) break;  // of the whole warp
          float v[32];
          columns(v, c0);
          __syncwarp();  // the lanes have read what the 32 columns before left in the staging buffer
#pragma unroll
          for (int q = 0; q < 8; ++q)
            sts16(staged(stage, lane, q), __float_as_uint(v[4 * q] * factor), __float_as_uint(v[4 * q + 1] * factor),
                  __float_as_uint(v[4 * q + 2] * factor), __float_as_uint(v[4 * q + 3] * factor));
          __syncwarp();
          if (vec) {
            // eight lanes a row: four values each
#pragma unroll
            for (int r4 = 0; r4 < 32; r4 += 4) {
              const int r = r4 + (lane >> 3), q = lane & 7, c = col_base + c0 + 4 * q;
              if (row_base + r < p.M && c < p.N) {
                const uint4 u = lds16(staged(stage, r, q));
                float4 f = make_float4(__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w));
                const long long at = (long long)(row_base + r) * p.N + c;
                if (!p.first) {
                  const float4 o = *reinterpret_cast<const float4*>(acc + at);
                  f.x += o.x, f.y += o.y, f.z += o.z, f.w += o.w;
                }
                if (out16) *reinterpret_cast<uint2*>((E*)p.out + at) = make_uint2(pack<E>(f.x, f.y), pack<E>(f.z, f.w));
                else *reinterpret_cast<float4*>(to32 + at) = f;
              }
            }
          } else {
            const int c = col_base + c0 + lane;
#pragma unroll 8
            for (int r = 0; r < 32; ++r)
              if (row_base + r < p.M && c < p.N) {
                float f = __uint_as_float(lds4(staged(stage, r, lane >> 2) + (lane & 3) * 4));
                const long long at = (long long)(row_base + r) * p.N + c;
                if (!p.first) f += acc[at];
                if (out16) ((E*)p.out)[at] = (E)f;
                else to32[at] = f;
              }
          }
        }
      }
      if (PIECES == 1) release(b);
    }
    if (ROLE == kDz && lane == 0) stores_done();
  }
  __syncwarp();
  tc::fence_before();
  if (CG == 1) __syncthreads();
  else cluster_sync();
  tc::fence_after();
  if (*abort_flag) {
    // copies and products that were under way end within microseconds: give them a millisecond before the memory goes
    if (threadIdx.x == 0) g_head_error = 1;
    for (int i = 0; i < 50; ++i) __nanosleep(20000);
    if (CG == 1) __syncthreads();
  }
  if (CG == 2) cluster_sync();  // neither block ends while the other may still reach its barriers
  if (warp == 2) tmem_free<CG>(tmem);
}

// ------------------------------------------------------------------ operands as the tensor cores take them

template <typename T> __device__ __forceinline__ float as_float(T v) { return (float)v; }

struct LayOut {
  const void* src;
  void* dst;
  long long rows;
  int width, per_row;        // per_row: groups of eight values of a row
  const long long* target;   // rows whose target is `ignore` become zeros; NULL: all rows count
};
// `at`: the first of eight values of a row that begins anywhere, c: its column.  The aligned 16-byte pieces around them, moved into place; the last values of the
// tensor, behind which there is no whole piece, go one by one.
template <typename T>
__device__ __forceinline__ void load_odd(T (&v)[8], const LayOut& l, long long at, int c) {
  constexpr int kVec = 8 * sizeof(T) / 16;
  const T* src = (const T*)l.src + at;
  if (at + 8 + 16 / (int)sizeof(T) > l.rows * l.width) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e < l.width ? src[e] : (T)0.0f;
    return;
  }
  const int off = (int)(reinterpret_cast<uintptr_t>(src) & 15);
  const uint4* from = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(src) - off);
  unsigned w[4 * (kVec + 1)];
#pragma unroll
  for (int q = 0; q <= kVec; ++q) {
    const uint4 u = __ldg(from + q);
    w[4 * q] = u.x, w[4 * q + 1] = u.y, w[4 * q + 2] = u.z, w[4 * q + 3] = u.w;
  }
#pragma unroll
  for (int i = 0; i + 2 < 4 * (kVec + 1); ++i) w[i] = (off & 8) ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i + 1 < 4 * (kVec + 1); ++i) w[i] = (off & 4) ? w[i + 1] : w[i];
  if (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 4 * kVec; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], (off & 2) * 8);
  }
#pragma unroll
  for (int i = 0; i < 4 * kVec; ++i) reinterpret_cast<unsigned*>(v)[i] = w[i];
  if (c + 8 > l.width) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e >= l.width) v[e] = (T)0.0f;
  }
}
constexpr float kLargestBf16 = 3.3895314e38f;  // (2 - 2^-7) 2^127
// [rows][width] -> PIECES planes [rows][8 per_row] of E: fp32 in three bf16 pieces, 16-bit rows on 16 bytes; eight values a lane, `lanes` lanes a row
template <typename T, typename E, int PIECES>
__device__ __forceinline__ void lay_out_row(const LayOut& l, long long r, int first, int stride, long long ignore) {
  const bool in = !(l.target && l.target[r] == ignore);
  for (int g = first; g < l.per_row; g += stride) {
    const long long at = r * l.width + g * 8;
    alignas(16) T v[8];
    if (!in) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (T)0.0f;
    } else if (l.width % 8 == 0) {
      constexpr int kVec = 8 * sizeof(T) / 16;
#pragma unroll
      for (int q = 0; q < kVec; ++q) reinterpret_cast<uint4*>(v)[q] = __ldg(reinterpret_cast<const uint4*>((const T*)l.src + at) + q);
    } else {
      load_odd<T>(v, l, at, g * 8);
    }
    alignas(16) E out[PIECES][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (PIECES == 1) {
        out[0][e] = (E)v[e];
      } else {
        float left = as_float(v[e]);
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
          // the last 2^-9 of fp32's range would round to infinity
          out[p][e] = (E)(p == 0 && fabsf(left) <= FLT_MAX ? fminf(fmaxf(left, -kLargestBf16), kLargestBf16) : left);
          left -= as_float(out[p][e]);
        }
      }
    }
    const long long pitch = 8ll * l.per_row;
#pragma unroll
    for (int p = 0; p < PIECES; ++p)
      *reinterpret_cast<uint4*>((E*)l.dst + (p * l.rows + r) * pitch + 8 * g) = *reinterpret_cast<const uint4*>(out[p]);
  }
}
// Rows of x, then of w; a warp has one at a time, or several short ones, or where there are few rows one of `parts` parts of one.
template <typename T, typename E, int PIECES>
__global__ void __launch_bounds__(256) lay_out_kernel(const LayOut x, const LayOut w, int lanes, int parts, long long ignore) {
  before_all();
  let_next();
  const int lane = threadIdx.x & 31, at_once = 32 / lanes, part = blockIdx.x % parts, block = blockIdx.x / parts;
  const int first = part * lanes + (lane & (lanes - 1)), stride = parts * lanes;
  const long long n = x.rows + w.rows, step = (long long)(gridDim.x / parts) * 8 * at_once;
  for (long long r = ((long long)block * 8 + (threadIdx.x >> 5)) * at_once + lane / lanes; r < n; r += step) {
    if (r < x.rows) lay_out_row<T, E, PIECES>(x, r, first, stride, ignore);
    else lay_out_row<T, E, PIECES>(w, r - x.rows, first, stride, ignore);
  }
}

// the largest |up| of the rows that count, one block
__global__ void __launch_bounds__(1024) largest_kernel(const float* __restrict__ up, const long long* __restrict__ y, long long ignore,
                                                       int rows, float* largest) {
  __shared__ float s[32];
  before_all();
  float v = 0;
  for (int r = threadIdx.x; r < rows; r += 1024)
    if (y[r] != ignore) v = fmaxf(v, fabsf(up[r]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x >= 32) return;
  v = s[threadIdx.x];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (threadIdx.x == 0) *largest = v;
}

// ---- sums over splits, in fixed order

struct Join {
  const float* parts;  // [splits][count]
  float* acc;
  void* out;           // NULL: the sum goes to acc
  long long count;     // 0: nothing to do
  int splits, first;
};
template <typename O>
__device__ __forceinline__ void join_one(const Join& j, long long i) {
  float v = j.first ? 0.0f : j.acc[i];
  for (int s = 0; s < j.splits; ++s) v += j.parts[s * j.count + i];
  if (j.out) ((O*)j.out)[i] = (O)v;
  else j.acc[i] = v;
}
template <typename O>
__global__ void __launch_bounds__(256) join_kernel(const Join a, const Join b) {
  before_all();
  let_next();
  const long long n = a.count + b.count;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    if (i < a.count) join_one<O>(a, i);
    else join_one<O>(b, i - a.count);
  }
}

// ------------------------------------------------------------------ plans

struct Config {
  int cg, bn;
};
// Tiles of the logits (us of the loss as a CUDA graph, 1280 features; pairs / 128 wide / 64 wide).  Pairs where one round of 128 x 128 tiles is not enough
// (4096 rows, 1000 classes 19.4 / 22.3 / 32.0; 2048 rows 18.2 / 16.0 / 21.1), unless half of their rows would be empty (64 rows, 16384 classes 18.6 / 16.5 /
// 22.2); narrow tiles while one round of them is (1024 rows, 1000 classes 17.5 / 15.0 / 14.5).  fp32: pairs also for fewer tiles when there are 16 steps or more,
// whose loads they halve (256 rows, 1000 classes 30.3 / 34.4 / 32.0; of 256 features 16.0 / 15.5 / 14.9; 64 rows, 16384 classes 101 / 75 / 93).
Config pick(long long rows, long long cols, int D, int pieces) {
  const int sms = device_sm_count();
  const long long tiles = (long long)div_up(rows, 128) * div_up(cols, 128);
  if (rows > 128 && pieces == 1 && tiles > sms) return {2, 256};
  if (rows > 128 && pieces == 3 && (tiles * 2 >= sms || div_up(D, kBox) >= 16)) return {2, 128};
  return tiles * 2 >= sms ? Config{1, 128} : Config{1, 64};
}
// Tiles of the gradients (us of loss and gradients, as above).  Pairs where there is work for 27 steps of each (4096 rows, 16384 classes 465 / 600 / 867), or where
// both sums are 16 steps long and a quarter of the SMs get a tile (1024 rows, 1000 classes 34.8 / 37.5 / 39.7); thin sums end sooner in tiles of one
// SM (64 rows, 4096 classes 40.1 / 36.9 / 39.0; 512 rows 46.7 / 45.1 / 48.9), narrow ones while they are few (512 rows, 1000 classes of 256 features
// 25.2 / 22.5 / 21.7).  fp32: pairs unless half of their rows would be empty (256 rows, 4096 classes 103 / 107 / 122; 64 rows 95 / 89 / 96).
Config pick_gradients(long long rows, long long classes, int D, int pieces) {
  const int sms = device_sm_count();
  if (pieces == 3) return rows > 128 ? Config{2, 128} : Config{1, 128};
  const long long row_tiles = div_up(rows, 256), class_tiles = div_up(classes, 256), n = div_up(D, 256);
  const long long row_steps = div_up(rows, kBox), class_steps = div_up(classes, kBox);
  if ((row_tiles * class_steps + class_tiles * row_steps) * n >= 27ll * (sms / 2)) return {2, 256};
  if (row_steps >= 16 && class_steps >= 16 && (row_tiles + class_tiles) * n * 4 >= sms) return {2, 256};
  return (long long)(div_up(rows, 128) + div_up(classes, 128)) * div_up(D, 128) * 2 >= sms ? Config{1, 128} : Config{1, 64};
}
int groups_of(const Config& c) { return c.bn >= 128 ? 2 : 1; }
int clusters_of(const Config& c) { return device_sm_count() / c.cg; }

template <int CG, int BN, int ROLE, typename E, int PIECES>
int launch_one(const Args& a, int items, cudaStream_t s) {
  auto kernel = head_kernel<CG, BN, ROLE, E, PIECES, false>;
  if constexpr (PIECES == 1 && ROLE != kGrad)
    if (a.depth > kLongDepth) kernel = head_kernel<CG, BN, ROLE, E, PIECES, true>;
  const int rc = enable_smem(kernel, smem_bytes<CG, BN>());
  if (rc != DK_OK) return rc;
  const int clusters = device_sm_count() / CG;
  // the gradients' schedule is one of all clusters
  return launch_after(kernel, (ROLE == kGrad || items > clusters ? clusters : items) * CG, kThreads, smem_bytes<CG, BN>(), CG, s, a);
}
template <int ROLE, typename E, int PIECES>
int launch(const Config& c, const Args& a, int items, cudaStream_t s) {
  if (c.cg == 2) return launch_one<2, PIECES == 1 ? 256 : 128, ROLE, E, PIECES>(a, items, s);
  if constexpr (!(ROLE == kGrad && PIECES == 3))
    if (c.bn == 64) return launch_one<1, 64, ROLE, E, PIECES>(a, items, s);
  return launch_one<1, 128, ROLE, E, PIECES>(a, items, s);
}

int pieces_of(int dtype) { return dtype == DK_F32 ? 3 : 1; }
// whether the operands are laid out anew: fp32 always, 16-bit rows that TMA cannot fetch
bool laid_out(int D, int dtype) { return dtype == DK_F32 || D % 8 != 0; }
int pitch_of(int n) { return (n + 7) & ~7; }

struct ForwardPlan {
  Config c;
  int tiles_m, tiles_n, slots;
  bool few;
  size_t x, w, top, sum, all, picked, partial, bytes;
};
// few: the CUDA cores' form, for a few rows without a backward
ForwardPlan forward_plan(int T, int D, int V, int dtype, bool few) {
  ForwardPlan p;
  Layout l;
  p.c = pick(T, V, D, pieces_of(dtype));
  p.tiles_m = div_up(T, 128 * p.c.cg), p.tiles_n = div_up(V, p.c.bn), p.slots = p.tiles_n * groups_of(p.c);
  p.few = few;
  if (p.few) p.slots = few_slots(V);
  const bool lay = !p.few && laid_out(D, dtype);
  const size_t row = (size_t)pitch_of(D) * 2 * pieces_of(dtype);
  p.x = lay ? l.take(T * row) : 0, p.w = lay ? l.take(V * row) : 0;
  const size_t each = (size_t)p.slots * T * sizeof(float);
  p.top = l.take(each), p.sum = l.take(each), p.all = l.take(each);
  p.picked = l.take((size_t)T * sizeof(float)), p.partial = l.take(combine_bytes(T));
  p.bytes = l.bytes;
  return p;
}

// dz of one piece; the whole call is one piece where it fits.  Fewer, larger pieces fill their last rounds of tiles better than smaller ones gain
// from L2: 4096 rows, 21841 classes (179 MB) 758 us as one piece, 813 as two; 8192 rows, 65536 classes 6.68 ms with 256 MB,
// 6.77 with 128, 7.10 with 64, 6.65 with 512.
constexpr long long kPieceBytes = 256ll << 20;

struct BackwardPlan {
  Config dz, grad;
  int tc, vc;                    // rows and classes of a piece: one of them is all there are
  int splits_w, per_w, splits_x, per_x;
  size_t x, w, largest, buffer, acc, acc_b, sums, parts_w, parts_x, bytes;
};

// splits of the two products so that a launch fills the SMs once where their tiles alone do not
void split_products(BackwardPlan& p, int D, int pieces) {
  const int clusters = clusters_of(p.grad), bm = 128 * p.grad.cg, tn = div_up(D, p.grad.bn);
  const long long tiles_w = (long long)div_up(p.vc, bm) * tn, tiles_x = (long long)div_up(p.tc, bm) * tn;
  const int blocks_w = div_up(p.tc, kBox), blocks_x = div_up(p.vc, kBox);
  const long long total = tiles_w * blocks_w + tiles_x * blocks_x;
  // at least 32 steps a split (of fp32, six products each, 8): the launch that joins the sums takes as long as some 20 steps.  Steps of training as
  // graphs, bf16, with at least 16 / 32 / 64, us: 1024 rows of 1280 features, 1000 classes 38 / 38 / 38 (8: 51), 2048 x 256 x 4096 57 / 51 / 54, 25088 x 256 x 150
  // 53 / 51 / 55, 100 x 264 x 11000 37 / 41 / 49, 4096 x 256 x 150 29 / 33 / 37, 9000 x 64 x 40 27 / 31 / 35; fp32 with 4 / 8 / 16: 64 x 520 x 4099
  // 63 / 64 / 70, 100 x 264 x 11000 70 / 69 / 75, 4096 x 256 x 150 45 / 47 / 55
  const int least = pieces == 1 ? 32 : 8;
  // and of 16-bit types at most 1024, 4096 additions that cut: 2^-12 of a sum of one sign, half of what fp16 rounds.  Parts of sums are rounded additions; they
  // take 8 KB of scratch a feature at most (a piece has 2^27 values of dz).
  constexpr long long kMostSteps = 1024;
  long long per = total / clusters + 1;
  if (per < least) per = least;
  if (pieces == 1 && per > kMostSteps) per = kMostSteps;
  p.per_w = (int)(per < blocks_w ? per : blocks_w), p.per_x = (int)(per < blocks_x ? per : blocks_x);
  p.splits_w = div_up(blocks_w, p.per_w), p.splits_x = div_up(blocks_x, p.per_x);
  p.per_w = div_up(blocks_w, p.splits_w), p.per_x = div_up(blocks_x, p.splits_x);
  p.splits_w = div_up(blocks_w, p.per_w), p.splits_x = div_up(blocks_x, p.per_x);
}

// the rounds of the two products' items that let all clusters end at about the same time
Schedule schedule_of(const Product& dw, const Product& dx, int clusters, int pieces) {
  // a tile takes the epilogue as long as it takes the tensor cores ten steps (six products a step: two).  Steps of training as graphs, bf16, counted as at
  // least 1 / 5 / 10 / 20 steps, us: 64 rows of 1280 features, 32768 classes, whose dw tiles are one step, 176 / 103 / 103 / 106, 25088 x 256 x 150 51 / 51 / 51 / 53,
  // 65536 x 256 x 21 69 / 69 / 70 / 72; fp32, 1 / 2 / 4: the first 443 / 414 / 421, the last 245 / 204 / 194
  const int least = pieces == 1 ? 10 : 2;
  const int n_w = dw.tiles_m * dw.tiles_n * dw.splits, n_x = dx.tiles_m * dx.tiles_n * dx.splits;
  Schedule c = {};
  c.long_product = n_w == 0 || (n_x != 0 && dx.per > dw.per);
  c.n_long = c.long_product ? n_x : n_w, c.n_short = c.long_product ? n_w : n_x;
  long long per_long = c.long_product ? dx.per : dw.per, per_short = c.long_product ? dw.per : dx.per;
  per_long = per_long < least ? least : per_long, per_short = per_short < least ? least : per_short;
  const int rest = c.n_long % clusters;
  long long dealt = 0;
  while (dealt < c.n_short) {
    // the clusters with one long item less go on until they would pass the others
    if (rest == 0 || (c.short_more - c.short_less + 1) * per_short <= per_long) c.short_more += 1, dealt += clusters - rest;
    else c.short_less += 1, dealt += rest;
    if (rest == 0) c.short_less = c.short_more;
  }
  return c;
}

BackwardPlan backward_plan(int T, int D, int V, int dtype) {
  BackwardPlan p;
  Layout l;
  const int pieces = pieces_of(dtype);
  p.tc = T, p.vc = V;
  const long long each = 2ll * pieces;
  if ((long long)T * pitch_of(V) * each > kPieceBytes) {
    // the longer side is cut: the sums that run over the pieces are those of the shorter one
    int& side = V >= T ? p.vc : p.tc;
    const int all = side, other = V >= T ? T : pitch_of(V);
    long long most = kPieceBytes / (other * each) / 256 * 256;
    if (most < 256) most = 256;
    const int n = div_up(all, most);
    const long long even = (long long)div_up(div_up(all, n), 256) * 256;
    side = even < all ? (int)even : all;
  }
  p.dz = pick(T, V, D, pieces);  // the forward's: p - 1 of a class that is nearly certain takes the same logits, bit by bit
  p.grad = pick_gradients(p.tc, p.vc, D, pieces);
  split_products(p, D, pieces);
  const bool lay = laid_out(D, dtype);
  const size_t row = (size_t)pitch_of(D) * 2 * pieces;
  p.x = l.take(T * row);  // laid out, or the copy without ignored rows
  p.w = lay ? l.take(V * row) : 0;
  p.largest = l.take(sizeof(float));
  p.buffer = l.take((size_t)p.tc * pitch_of(p.vc) * each);
  const bool cut_v = p.vc < V, cut_t = p.tc < T;
  p.acc = (cut_v || cut_t) && dtype != DK_F32 ? l.take((size_t)(cut_v ? T : V) * D * sizeof(float)) : 0;
  p.acc_b = cut_t ? l.take((size_t)V * sizeof(float)) : 0;
  p.sums = l.take((size_t)div_up(p.tc, 32) * p.vc * sizeof(float));
  p.parts_w = p.splits_w > 1 ? l.take((size_t)p.splits_w * p.vc * D * sizeof(float)) : 0;
  p.parts_x = p.splits_x > 1 ? l.take((size_t)p.splits_x * p.tc * D * sizeof(float)) : 0;
  p.bytes = l.bytes;
  return p;
}

// ------------------------------------------------------------------ calls

unsigned blocks_for(long long n) {
  const long long b = (n + 255) / 256, most = (long long)device_sm_count() * 8;
  return (unsigned)(b < most ? b : most);
}

// tiles of rows whose part of x stays in L2 (126 MB) beside the weights that stream past
int row_group(const Config& c, int D, int pieces, int tiles_m) {
  const long long g = (40ll << 20) / ((long long)128 * c.cg * D * 2 * pieces);
  return g < 1 ? 1 : (int)(g > tiles_m ? tiles_m : g);
}

// x and w as planes of 16-bit values that TMA can fetch
template <typename T, typename E, int PIECES>
int operands(const void*& x, const void*& w, char* to_x, char* to_w, const long long* y, const Shape& h, int dtype, cudaStream_t s) {
  if (!laid_out(h.D, dtype)) return DK_OK;
  const int per_row = pitch_of(h.D) / 8;
  const LayOut lx = {x, to_x, h.T, h.D, per_row, y}, lw = {w, to_w, h.V, h.D, per_row, nullptr};
  x = to_x, w = to_w;
  int lanes = 1;
  while (lanes < 32 && lanes < per_row) lanes *= 2;
  // eight blocks an SM: as many parts of a row as it takes (1256 rows of 160 groups: 5 us in five parts, 8.6 in one)
  const long long blocks = ((long long)h.T + h.V) * lanes / 256 + 1, most = (long long)device_sm_count() * 8;
  int parts = 1;
  while (blocks * (parts + 1) <= most && parts * lanes < per_row) ++parts;
  return launch_after(lay_out_kernel<T, E, PIECES>, (unsigned)(blocks * parts < most ? blocks * parts : most / parts * parts), 256, 0, 1, s, lx,
                      lw, lanes, parts, h.ignore);
}
template <typename E, int PIECES>
bool operand_map(CUtensorMap* tm, const void* p, int rows, int width, int pitch, int box_rows = kBox) {
  return ring::make_swizzled_map(tm, p, std::is_same<E, __nv_bfloat16>::value, width, rows, PIECES, pitch * 2ll, (long long)rows * pitch * 2,
                                 box_rows);
}

template <typename T, typename E, int PIECES>
int forward(const void* x, const void* w, const void* b, const long long* y, void* loss, void* saved, const Shape& h, int dtype, void* ws,
            size_t ws_bytes, cudaStream_t s) {
  // With a backward to come the logits have to be the ones that it will compute: where p is nearly one, p - 1 is the difference of the two.
  const ForwardPlan p = forward_plan(h.T, h.D, h.V, dtype, few_rows(h.T, dtype) && !saved);
  if (!ws || ws_bytes < tc_forward_bytes(h.T, h.D, h.V, dtype)) return DK_ERR_WORKSPACE;
  char* m = (char*)ws;
  if (p.few) {
    const Partials<float> part = {(float*)(m + p.top), (float*)(m + p.sum), (float*)(m + p.all), (float*)(m + p.picked)};
    double* partial = (double*)(m + p.partial);
    const int rc = launch_few_rows<T>(x, w, b, y, part, combine_count(partial, h.T), h, s);
    return rc != DK_OK ? rc : launch_combine<float>(part, y, p.slots, loss, saved, partial, h, s);
  }
  int rc = operands<T, E, PIECES>(x, w, m + p.x, m + p.w, y, h, dtype, s);
  if (rc != DK_OK) return rc;
  Args a = {};
  if (!operand_map<E, PIECES>(&a.x, x, h.T, h.D, pitch_of(h.D)) || !operand_map<E, PIECES>(&a.w, w, h.V, h.D, pitch_of(h.D)))
    return DK_ERR_CUDA;
  a.rows = h.T, a.classes = h.V, a.depth = div_up(h.D, kBox);
  a.tiles_m = p.tiles_m, a.tiles_n = p.tiles_n, a.group = row_group(p.c, h.D, PIECES, p.tiles_m);
  a.bias = b, a.target = y, a.ignore = h.ignore;
  a.wait_limit = g_wait_limit.load(std::memory_order_relaxed);
  a.top = (float*)(m + p.top), a.sum = (float*)(m + p.sum), a.all = h.smoothing != 0.0 ? (float*)(m + p.all) : nullptr;
  a.picked = (float*)(m + p.picked), a.done = combine_count((double*)(m + p.partial), h.T);
  if ((long long)p.tiles_m * p.tiles_n > 0x3fffffff) return DK_ERR_UNSUPPORTED;
  rc = launch<kStats, E, PIECES>(p.c, a, p.tiles_m * p.tiles_n, s);
  if (rc != DK_OK) return rc;
  const Partials<float> part = {a.top, a.sum, a.all, a.picked};
  return launch_combine<float>(part, y, p.slots, loss, saved, (double*)(m + p.partial), h, s);
}

template <typename T, typename E, int PIECES>
int backward(const void* up, const void* x, const void* w, const void* b, const long long* y, const void* saved, void* dx, void* dw,
             void* db, const Shape& h, int dtype, void* ws, size_t ws_bytes, cudaStream_t s) {
  const BackwardPlan p = backward_plan(h.T, h.D, h.V, dtype);
  if (!ws || ws_bytes < p.bytes) return DK_ERR_WORKSPACE;
  char* m = (char*)ws;
  const float* stat = (const float*)saved;
  float* largest = dtype == DK_F16 && h.reduction == DK_REDUCE_NONE ? (float*)(m + p.largest) : nullptr;
  int rc = DK_OK;
  if (largest) rc = launch_after(largest_kernel, 1, 1024, 0, 1, s, (const float*)up, y, h.ignore, h.T, largest);
  if (rc != DK_OK) return rc;
  Args a = {};
  const int pitch = pitch_of(h.D);
  if (laid_out(h.D, dtype)) {
    rc = operands<T, E, PIECES>(x, w, m + p.x, m + p.w, y, h, dtype, s);
    if (rc != DK_OK) return rc;
  } else if (dw) {
    a.strange = stat + 2ll * h.T + 1;
  }
  if (!operand_map<E, PIECES>(&a.x, x, h.T, h.D, pitch) || !operand_map<E, PIECES>(&a.w, w, h.V, h.D, pitch) ||
      !operand_map<E, PIECES>(&a.x_clean, m + p.x, h.T, h.D, pitch))
    return DK_ERR_CUDA;
  a.depth = div_up(h.D, kBox), a.bias = b, a.ignore = h.ignore, a.all_classes = h.V;
  a.wait_limit = g_wait_limit.load(std::memory_order_relaxed);
  a.up = {(const float*)up, stat + 2ll * h.T, largest, h.reduction, 1.0f};
  // up to one half: beyond, p unit would leave fp16's range
  if (h.reduction != DK_REDUCE_NONE)
    a.up.unit = (float)((dtype == DK_F16 ? 16384.0 : 1.0) / (h.smoothing <= 0.5 ? 1.0 - h.smoothing : 1.0));
  a.smooth_each = (float)(h.smoothing / h.V), a.smooth_own = (float)(1.0 - h.smoothing);
  a.column_sums = db ? (float*)(m + p.sums) : nullptr;
  const bool cut_v = p.vc < h.V;
  const int bm = 128 * p.grad.cg, tn = div_up(h.D, p.grad.bn);
  for (int t0 = 0; t0 < h.T; t0 += p.tc)
    for (int v0 = 0; v0 < h.V; v0 += p.vc) {
      const int rows = h.T - t0 < p.tc ? h.T - t0 : p.tc, classes = h.V - v0 < p.vc ? h.V - v0 : p.vc;
      const bool first_t = t0 == 0, last_t = t0 + rows == h.T, first_v = v0 == 0, last_v = v0 + classes == h.V;
      const int dz_pitch = pitch_of(classes);
      if (!operand_map<E, PIECES>(&a.dz, m + p.buffer, rows, classes, dz_pitch) ||
          !operand_map<E, PIECES>(&a.dz_out, m + p.buffer, rows, classes, dz_pitch, 32))
        return DK_ERR_CUDA;
      a.rows = rows, a.classes = classes, a.row0 = t0, a.class0 = v0;
      a.tiles_m = div_up(rows, 128 * p.dz.cg), a.tiles_n = div_up(classes, p.dz.bn), a.group = row_group(p.dz, h.D, PIECES, a.tiles_m);
      a.target = y + t0, a.ref = stat + t0, a.inv = stat + h.T + t0;
      if (h.reduction == DK_REDUCE_NONE) a.up.up = (const float*)up + t0;
      if (a.strange && first_t && first_v) a.dirty = x, a.clean = m + p.x, a.width = h.D, a.up_rows = h.T, a.target_all = y;
      else a.clean = nullptr;
      if ((long long)a.tiles_m * a.tiles_n > 0x3fffffff) return DK_ERR_UNSUPPORTED;
      rc = launch<kDz, E, PIECES>(p.dz, a, a.tiles_m * a.tiles_n, s);
      if (rc != DK_OK) return rc;
      // dw [classes][D] sums over rows, dx [rows][D] over classes; the running sums of fp32 gradients are the gradients
      Product pw = {}, px = {};
      Join jw = {}, jx = {};
      if (dw) {
        T* out = (T*)dw + (long long)v0 * h.D;
        float* acc = PIECES == 3 ? (float*)out : (float*)(m + p.acc);
        pw.M = classes, pw.N = h.D, pw.blocks = div_up(rows, kBox), pw.tiles_m = div_up(classes, bm), pw.tiles_n = tn;
        pw.per = p.per_w, pw.splits = div_up(pw.blocks, pw.per);
        pw.acc = acc, pw.out = last_t ? out : nullptr, pw.first = first_t;
        if (pw.splits > 1) {
          jw.parts = (float*)(m + p.parts_w), jw.acc = acc, jw.out = pw.out, jw.count = (long long)classes * h.D;
          jw.splits = pw.splits, jw.first = first_t;
          pw.acc = (float*)(m + p.parts_w), pw.out = nullptr, pw.first = 1;
        }
      }
      if (dx) {
        T* out = (T*)dx + (long long)t0 * h.D;
        float* acc = PIECES == 3 ? (float*)out : (float*)(m + p.acc);
        px.M = rows, px.N = h.D, px.blocks = div_up(classes, kBox), px.tiles_m = div_up(rows, bm), px.tiles_n = tn;
        px.per = p.per_x, px.splits = div_up(px.blocks, px.per);
        px.acc = acc, px.out = last_v ? out : nullptr, px.first = first_v;
        if (px.splits > 1) {
          jx.parts = (float*)(m + p.parts_x), jx.acc = acc, jx.out = px.out, jx.count = (long long)rows * h.D;
          jx.splits = px.splits, jx.first = first_v;
          px.acc = (float*)(m + p.parts_x), px.out = nullptr, px.first = 1;
        }
      }
      if (db) a.acc_b = cut_v ? nullptr : (float*)(m + p.acc_b), a.out_b = last_t ? (T*)db + v0 : nullptr, a.first_b = first_t;
      const long long items = (long long)pw.tiles_m * tn * pw.splits + (long long)px.tiles_m * tn * px.splits;
      if (items > 0x3fffffff) return DK_ERR_UNSUPPORTED;
      a.dw = pw, a.dx = px, a.schedule = schedule_of(pw, px, clusters_of(p.grad), PIECES);
      rc = launch<kGrad, E, PIECES>(p.grad, a, (int)items, s);
      if (rc == DK_OK && jw.count + jx.count > 0) rc = launch_after(join_kernel<T>, blocks_for(jw.count + jx.count), 256, 0, 1, s, jw, jx);
      if (rc != DK_OK) return rc;
    }
  return DK_OK;
}

}  // namespace

size_t tc_forward_bytes(int T, int D, int V, int dtype) {
  const size_t n = forward_plan(T, D, V, dtype, false).bytes, few = few_rows(T, dtype) ? forward_plan(T, D, V, dtype, true).bytes : 0;
  return n > few ? n : few;
}
size_t tc_backward_bytes(int T, int D, int V, int dtype) { return backward_plan(T, D, V, dtype).bytes; }

int tc_forward(const void* x, const void* w, const void* b, const long long* y, void* loss, void* saved, const Shape& h, int dtype,
               void* ws, size_t ws_bytes, cudaStream_t s) {
  switch (dtype) {
    case DK_F16: return forward<__half, __half, 1>(x, w, b, y, loss, saved, h, dtype, ws, ws_bytes, s);
    case DK_BF16: return forward<__nv_bfloat16, __nv_bfloat16, 1>(x, w, b, y, loss, saved, h, dtype, ws, ws_bytes, s);
    default: return forward<float, __nv_bfloat16, 3>(x, w, b, y, loss, saved, h, dtype, ws, ws_bytes, s);
  }
}

int tc_backward(const void* up, const void* x, const void* w, const void* b, const long long* y, const void* saved, void* dx, void* dw,
                void* db, const Shape& h, int dtype, void* ws, size_t ws_bytes, cudaStream_t s) {
  switch (dtype) {
    case DK_F16: return backward<__half, __half, 1>(up, x, w, b, y, saved, dx, dw, db, h, dtype, ws, ws_bytes, s);
    case DK_BF16: return backward<__nv_bfloat16, __nv_bfloat16, 1>(up, x, w, b, y, saved, dx, dw, db, h, dtype, ws, ws_bytes, s);
    default: return backward<float, __nv_bfloat16, 3>(up, x, w, b, y, saved, dx, dw, db, h, dtype, ws, ws_bytes, s);
  }
}

long long set_wait_limit(long long nanoseconds) {
  return (long long)g_wait_limit.exchange(nanoseconds > 0 ? (unsigned long long)nanoseconds : kWaitLimit);
}

// Code of the last bounded wait that ran out on the current device (0 = none); synchronises with the device.
int head_error_status() {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_head_error, sizeof(int)) != cudaSuccess) return -1;
  return v;
}

}  // namespace head
}  // namespace dk
