// fastmax_decode_step: one new token per (batch, head) against the carried moment state.
//
//     S   <-  S + Phi(k)^T [v | 1]                (un-weighted sums, the exchange format of the forward call)
//     o'  =   sum_r  w_r Phi(q)_r S[r, :]          (w_r = a2/T^2 (x2 off the block diagonal), a1/T, a0)
//     o   =   o'[:D] / o'[D],   g = o'[D]
//
// The state of a head (D=64, order 2: 2369 rows x 68 floats = 644 KB) is read once and written once; nothing
// else moves, so the kernel is bound by HBM: 2 x state bytes per step.  A cluster of 1, 2, 4 or 8 thread blocks
// shares one head (the host picks the smallest cluster that still gives the GPU about a thousand blocks: few, long
// blocks stream best, but there must be enough of them to fill 148 SMs several times over), each block streams its
// share of the rows with 128-bit accesses (thread = one float4 column of a row, four rows in flight), the partial
// outputs meet in the first block's shared memory over the cluster's distributed shared memory, and that block
// divides and stores the token's output.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <atomic>

#include "../../include/fastmax_b200.h"
#include "common.cuh"
#include "launchers.cuh"
#include "pages.cuh"

namespace cg = cooperative_groups;

namespace fm {

int report_cuda_error(cudaError_t e);
int sm_count();

namespace dec {

constexpr int MAX_CL = 8;   // largest cluster: thread blocks that share one head
constexpr int UNROLL = 4;   // rows a thread has in flight
// RG: rows a block works on at a time.  Sixteen, or 48 where a thread's rows are then fewer memory latencies behind one another (more
// than 16 UNROLL rows a block) and all blocks run at once, one to an SM: 816 threads leave room for no more, and a cluster of eight
// needs eight SMs of one GPC (fifteen such clusters fit).  us a step with 16 / 48 rows, order 2: d = 64, 8 heads 6.4 / 5.8, 15 heads
// 6.5 / 5.9, 16 heads 7.7 / 10.7, 18 heads 7.7 / 10.9; d = 32, 8 heads 3.80 / 3.52, 18 heads 4.05 / 3.97, 32 heads 4.24 / 5.03; few
// rows a block: d = 16, 8 heads 3.13 / 3.11, order 1, d = 64, 8 heads 3.25 / 3.84, 16 heads 3.3 / 6.3.  The partial sums of either are
// added in an order of their own: float32 outputs may differ in their last bits between a call that takes 48 and one that takes 16.
// Launched behind the step before (grid_wait), 8 heads take 8.2 -> 6.2 us a step, where the host's call ends up; 512 heads 117.8 -> 116.0.

struct DecodeParams {
  View q, k, v, o, g;
  float* state;
  const int* table;         // page of each sequence, or NULL: heads follow one another without gaps
  long long page_stride;    // floats
  int pages;
  int heads, rows;
  float c0, c1, c2;
};

template <typename T>
__device__ __forceinline__ float to_f(T x);
template <>
__device__ __forceinline__ float to_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename T, int D, int ORDER, int RG>
__global__ void __launch_bounds__(((D + 4) / 4) * RG)
decode_step_kernel(const DecodeParams P) {
  using G = Geo<D>;
  constexpr int C4 = (D + 4) / 4;          // float4 columns of a state row
  constexpr int NT = C4 * RG;
  constexpr int PAIR_ROWS = ORDER == 2 ? 64 * G::NPAIRS : 0;

  __shared__ float sq[D], sk[D];
  __shared__ float4 sv[C4];
  __shared__ float4 red[RG][C4];
  __shared__ float4 part[MAX_CL][C4];      // block 0 of the cluster: one row per block
  __shared__ unsigned char tab_a[G::NPAIRS], tab_b[G::NPAIRS];

  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x;
  const int rank = (int)cluster.block_rank();
  const int CL = (int)gridDim.x;            // the cluster spans the grid's x extent
  const int head = blockIdx.y;
  const int bi = head / P.heads, hi = head - bi * P.heads;

  if (ORDER == 2 && tid < G::NPAIRS) {
    int a, b;
    pair_decode(tid, G::NB, a, b);
    tab_a[tid] = (unsigned char)a;
    tab_b[tid] = (unsigned char)b;
  }
  grid_wait();   // the step before this one wrote the state
  grid_trigger();
  long long first = (long long)bi * P.page_stride + (long long)hi * (P.rows * (D + 4));
  if (P.table != nullptr) {
    const int page = P.table[bi];
    if (page < 0 || page >= P.pages) return;   // the whole cluster: an absent sequence
    first += (long long)(page - bi) * P.page_stride;
  }
  if (tid < D) {
    const long long off_q = (long long)bi * P.q.sb + (long long)hi * P.q.sh;
    const long long off_k = (long long)bi * P.k.sb + (long long)hi * P.k.sh;
    sq[tid] = to_f<T>(reinterpret_cast<const T*>(P.q.ptr)[off_q + tid]);
    sk[tid] = to_f<T>(reinterpret_cast<const T*>(P.k.ptr)[off_k + tid]);
  }
  if (tid < C4) {
    const T* vp = reinterpret_cast<const T*>(P.v.ptr) + (long long)bi * P.v.sb + (long long)hi * P.v.sh;
    float4 x = make_float4(1.f, 0.f, 0.f, 0.f);   // the ones column of [v | 1] and the padding
    if (tid < D / 4) x = make_float4(to_f<T>(vp[4 * tid]), to_f<T>(vp[4 * tid + 1]), to_f<T>(vp[4 * tid + 2]), to_f<T>(vp[4 * tid + 3]));
    sv[tid] = x;
  }
  __syncthreads();

  const int c4 = tid % C4, rg = tid / C4;
  const int rows_per = (P.rows + CL - 1) / CL;
  const int r0 = rank * rows_per;
  const int r1 = min(P.rows, r0 + rows_per);
  const float4 v4 = sv[c4];
  float4* base = reinterpret_cast<float4*>(P.state + first) + c4;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);

  // feature r of k (un-weighted) and of q (weighted)
  auto feature = [&](int r, float& pk, float& pq) {
    if (ORDER == 2 && r < PAIR_ROWS) {
      const int u = r >> 6, i = r & 63;
      const int a = tab_a[u], b = tab_b[u];
      const int m = 8 * a + (i >> 3), n = 8 * b + (i & 7);
      pk = sk[m] * sk[n];
      pq = sq[m] * sq[n] * (a == b ? P.c2 : 2.f * P.c2);
    } else {
      const int m = r - PAIR_ROWS;
      if (m < D) {
        pk = sk[m];
        pq = sq[m] * P.c1;
      } else {
        pk = 1.f;
        pq = P.c0;
      }
    }
  };

  for (int r = r0 + rg; r < r1; r += RG * UNROLL) {
    float4 s[UNROLL];
    float pk[UNROLL], pq[UNROLL];
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
      const int rr = r + j * RG;
      if (rr < r1) {
        s[j] = __ldcs(base + (long long)rr * C4);
        feature(rr, pk[j], pq[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
      const int rr = r + j * RG;
      if (rr < r1) {
        s[j].x = fmaf(pk[j], v4.x, s[j].x);
        s[j].y = fmaf(pk[j], v4.y, s[j].y);
        s[j].z = fmaf(pk[j], v4.z, s[j].z);
        s[j].w = fmaf(pk[j], v4.w, s[j].w);
        __stcs(base + (long long)rr * C4, s[j]);
        acc.x = fmaf(pq[j], s[j].x, acc.x);
        acc.y = fmaf(pq[j], s[j].y, acc.y);
        acc.z = fmaf(pq[j], s[j].z, acc.z);
        acc.w = fmaf(pq[j], s[j].w, acc.w);
      }
    }
  }

  red[rg][c4] = acc;
  // Every block of the cluster must be known to have started before another block writes into its shared memory;
  // this barrier also orders the `red` rows for the reduction below (it is a superset of __syncthreads).
  cluster.sync();
  if (tid < C4) {
    float4 t = red[0][tid];
#pragma unroll
    for (int j = 1; j < RG; ++j) {
      const float4 x = red[j][tid];
      t.x += x.x, t.y += x.y, t.z += x.z, t.w += x.w;
    }
    float4* dst = cluster.map_shared_rank(&part[rank][tid], 0);
    *dst = t;
  }
  cluster.sync();
  if (rank != 0) return;

  float* fin = reinterpret_cast<float*>(&red[0][0]);   // [C4 * 4]: o'[0..D-1], g, padding
  if (tid < C4) {
    float4 t = part[0][tid];
    for (int j = 1; j < CL; ++j) {
      const float4 x = part[j][tid];
      t.x += x.x, t.y += x.y, t.z += x.z, t.w += x.w;
    }
    reinterpret_cast<float4*>(fin)[tid] = t;
  }
  __syncthreads();
  const float gsum = fin[D];
  if (tid < D) {
    T* op = reinterpret_cast<T*>(const_cast<void*>(P.o.ptr)) + (long long)bi * P.o.sb + (long long)hi * P.o.sh;
    op[tid] = from_f<T>(fin[tid] / gsum);
  }
  if (tid == 0 && P.g.ptr != nullptr) {
    float* gp = reinterpret_cast<float*>(const_cast<void*>(P.g.ptr)) + (long long)bi * P.g.sb + (long long)hi * P.g.sh;
    *gp = gsum;
  }
}

// ---- many heads, on pages ----------------------------------------------------------------------------------------------------
// The same step as short blocks without clusters: a block has four units of one head (a unit: the 64 products of a pair of blocks, or the linear
// rows), a thread one float4 column of four rows (m .. m + 3, n) of a unit and the next unit's four in flight; the parts of the outputs go through
// the workspace and a second, small launch adds them in the units' order and divides.  Bound by HBM: 512 heads of 64 dims 104.7 us, 96 % of the copy
// rate (clusters 115.7), of which the second launch is some 3.
template <int D>
struct RowsGeo {
  static constexpr int C4 = (D + 4) / 4;
  static constexpr int THREADS = 16 * C4;
  static constexpr int EACH = 4;   // units
};
__host__ __device__ inline int row_groups(int d, int order) { return ((order == 2 ? (d / 8) * (d / 8 + 1) / 2 : 0) + 1 + 3) / 4; }

template <typename T, int D>
__global__ void __launch_bounds__(RowsGeo<D>::THREADS)
step_rows_kernel(const DecodeParams P, float4* parts) {
  using G = RowsGeo<D>;
  constexpr int C4 = G::C4, NB = D / 8;
  __shared__ __align__(16) float sq[D], sk[D];
  __shared__ float4 red[16][C4];
  const int tid = threadIdx.x, head = blockIdx.y, bi = head / P.heads, hi = head - bi * P.heads;
  const int npairs = (P.rows - D - 1) / 64;
  const int u0 = blockIdx.x * G::EACH, u1 = min(u0 + G::EACH, npairs + 1);
  grid_wait();
  grid_trigger();
  long long first = (long long)bi * P.page_stride + (long long)hi * (P.rows * (D + 4));
  if (P.table != nullptr) {
    const int page = P.table[bi];
    if (page < 0 || page >= P.pages) return;
    first += (long long)(page - bi) * P.page_stride;
  }
  const int c4 = tid % C4, rg = tid / C4;
  const int n8 = rg & 7, m8 = 4 * (rg >> 3);
  float4* base = reinterpret_cast<float4*>(P.state + first) + c4;
  auto row_of = [&](int u, int j) { return u < npairs ? 64 * u + 8 * (m8 + j) + n8 : 64 * npairs + rg + 16 * j; };
  auto there = [&](int u, int j) { return u < npairs || rg + 16 * j < D; };
  float4 next[4], ones = make_float4(0.f, 0.f, 0.f, 0.f);
  auto fetch = [&](int u) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (there(u, j)) next[j] = __ldcs(base + (long long)row_of(u, j) * C4);
    if (u == npairs && rg == 0) ones = __ldcs(base + (long long)(64 * npairs + D) * C4);   // the constant's row
  };
  fetch(u0);
  if (tid < D) {
    sq[tid] = to_f<T>(reinterpret_cast<const T*>(P.q.ptr)[(long long)bi * P.q.sb + (long long)hi * P.q.sh + tid]);
    sk[tid] = to_f<T>(reinterpret_cast<const T*>(P.k.ptr)[(long long)bi * P.k.sb + (long long)hi * P.k.sh + tid]);
  }
  float4 v4 = make_float4(1.f, 0.f, 0.f, 0.f);
  if (c4 < D / 4) {
    const T* vp = reinterpret_cast<const T*>(P.v.ptr) + (long long)bi * P.v.sb + (long long)hi * P.v.sh + 4 * c4;
    v4 = make_float4(to_f<T>(vp[0]), to_f<T>(vp[1]), to_f<T>(vp[2]), to_f<T>(vp[3]));
  }
  __syncthreads();
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  auto update = [&](float4& s, float pk, float pq) {
    s.x = fmaf(pk, v4.x, s.x), s.y = fmaf(pk, v4.y, s.y), s.z = fmaf(pk, v4.z, s.z), s.w = fmaf(pk, v4.w, s.w);
    acc.x = fmaf(pq, s.x, acc.x), acc.y = fmaf(pq, s.y, acc.y), acc.z = fmaf(pq, s.z, acc.z), acc.w = fmaf(pq, s.w, acc.w);
  };
  int ua = 0, ub = 0;
  if (u0 < npairs) pair_decode(u0, NB, ua, ub);
  for (int u = u0; u < u1; ++u) {
    float4 s[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] = next[j];
    if (u + 1 < u1) fetch(u + 1);
    if (u < npairs) {
      const float4 km = *reinterpret_cast<const float4*>(sk + 8 * ua + m8), qm = *reinterpret_cast<const float4*>(sq + 8 * ua + m8);
      const float kn = sk[8 * ub + n8], qn = sq[8 * ub + n8], weight = ua == ub ? P.c2 : 2.f * P.c2;
      update(s[0], km.x * kn, qm.x * qn * weight);
      update(s[1], km.y * kn, qm.y * qn * weight);
      update(s[2], km.z * kn, qm.z * qn * weight);
      update(s[3], km.w * kn, qm.w * qn * weight);
      if (++ub == NB) ub = ++ua;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (there(u, j)) update(s[j], sk[rg + 16 * j], sq[rg + 16 * j] * P.c1);
      if (rg == 0) {
        update(ones, 1.f, P.c0);
        __stcs(base + (long long)(64 * npairs + D) * C4, ones);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (there(u, j)) __stcs(base + (long long)row_of(u, j) * C4, s[j]);
  }
  red[rg][c4] = acc;
  __syncthreads();
  if (tid < C4) {
    float4 t = red[0][tid];
#pragma unroll
    for (int j = 1; j < 16; ++j) {
      const float4 x = red[j][tid];
      t.x += x.x, t.y += x.y, t.z += x.z, t.w += x.w;
    }
    parts[((long long)head * gridDim.x + blockIdx.x) * C4 + tid] = t;
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(256)
step_divide_kernel(const DecodeParams P, const float* parts, int groups, int total) {
  constexpr int LD = D + 4, MOST = (Geo<D>::NPAIRS + 1 + RowsGeo<D>::EACH - 1) / RowsGeo<D>::EACH;
  grid_wait();
  grid_trigger();
  const int head = blockIdx.x * blockDim.y + threadIdx.y, c = threadIdx.x;   // a column of the state
  if (head >= total) return;
  const int bi = head / P.heads, hi = head - bi * P.heads;
  const int page = P.table != nullptr ? P.table[bi] : 0;
  const float* at = parts + (long long)head * groups * LD;
  float xs[MOST], gs[MOST];   // all on their way at once; an absent sequence's are not used
#pragma unroll
  for (int i = 0; i < MOST; ++i) xs[i] = i < groups ? at[i * LD + c] : 0.f, gs[i] = i < groups ? at[i * LD + D] : 0.f;
  if (page < 0 || page >= P.pages) return;
  float x = xs[0], g = gs[0];
#pragma unroll
  for (int i = 1; i < MOST; ++i) x += xs[i], g += gs[i];
  T* op = reinterpret_cast<T*>(const_cast<void*>(P.o.ptr)) + (long long)bi * P.o.sb + (long long)hi * P.o.sh;
  op[c] = from_f<T>(x / g);
  if (c == 0 && P.g.ptr != nullptr)
    *(reinterpret_cast<float*>(const_cast<void*>(P.g.ptr)) + (long long)bi * P.g.sb + (long long)hi * P.g.sh) = g;
}

template <typename T, int D>
static cudaError_t launch_rows(int order, const DecodeParams& P, int bh, float* parts, cudaStream_t st) {
  const int groups = row_groups(D, order);
  {
    LaunchScope ls(KK_DECODE, st);
    const cudaError_t e = launch_after(step_rows_kernel<T, D>, dim3((unsigned)groups, (unsigned)bh), RowsGeo<D>::THREADS, 0, st, P, reinterpret_cast<float4*>(parts));
    if (e != cudaSuccess) return e;
  }
  LaunchScope ls(KK_DECODE, st);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((bh + 256 / D - 1) / (256 / D)));
  cfg.blockDim = dim3(D, 256 / D);
  cfg.stream = st;
  cudaLaunchAttribute attr = launch_attribute_after();
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return launched(cudaLaunchKernelEx(&cfg, step_divide_kernel<T, D>, P, (const float*)parts, groups, bh));
}

template <int D, int RG>
static void configure(cudaLaunchConfig_t& cfg, cudaLaunchAttribute (&attr)[2], int bh, int cl, cudaStream_t st) {
  cfg.gridDim = dim3(cl, bh);
  cfg.blockDim = dim3(((D + 4) / 4) * RG);
  cfg.dynamicSmemBytes = 0;
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cl;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1] = launch_attribute_after();
  cfg.attrs = attr;
  cfg.numAttrs = 2;
}
template <typename T, int D, int ORDER, int RG>
static cudaError_t launch(const DecodeParams& P, int bh, int cl, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  configure<D, RG>(cfg, attr, bh, cl, st);
  return launched(cudaLaunchKernelEx(&cfg, decode_step_kernel<T, D, ORDER, RG>, P));
}
// clusters of MAX_CL blocks of the 48-row kernel that the current device runs at once with a block to an SM
template <typename T, int D>
static int clusters_at_once() {
  static std::atomic<int> cached[64];   // + 1
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  int n = cached[dev].load(std::memory_order_relaxed) - 1;
  if (n < 0) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    configure<D, 48>(cfg, attr, 1, MAX_CL, nullptr);
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, decode_step_kernel<T, D, 2, 48>, &cfg) != cudaSuccess) {
      cudaGetLastError();
      n = 0;
    }
    if (n > sm_count() / MAX_CL) n = sm_count() / MAX_CL;
    cached[dev].store(n + 1, std::memory_order_relaxed);
  }
  return n;
}
template <typename T, int D>
static cudaError_t launch(int order, const DecodeParams& P, int bh, cudaStream_t st) {
  int cl = 1;
  while (cl < MAX_CL && (long long)cl * bh < 1024) cl *= 2;
  // (order 1 and D = 16 have at most 9 and 27 rows a block where the cluster is that large)
  if constexpr (D > 16)
    if (order == 2 && cl == MAX_CL && (P.rows + cl - 1) / cl > 16 * UNROLL && bh <= clusters_at_once<T, D>()) return launch<T, D, 2, 48>(P, bh, cl, st);
  return order == 2 ? launch<T, D, 2, 16>(P, bh, cl, st) : launch<T, D, 1, 16>(P, bh, cl, st);
}

template <typename T>
static cudaError_t launch_d(int d, int order, const DecodeParams& P, int bh, float* parts, cudaStream_t st) {
  if (parts != nullptr) {
    switch (d) {
      case 16: return launch_rows<T, 16>(order, P, bh, parts, st);
      case 32: return launch_rows<T, 32>(order, P, bh, parts, st);
      default: return launch_rows<T, 64>(order, P, bh, parts, st);
    }
  }
  LaunchScope ls(KK_DECODE, st);
  switch (d) {
    case 16: return launch<T, 16>(order, P, bh, st);
    case 32: return launch<T, 32>(order, P, bh, st);
    default: return launch<T, 64>(order, P, bh, st);
  }
}

}  // namespace dec
}  // namespace fm

// parts: NULL, or the workspace of the form for many heads
static int32_t decode_step(const fastmax_problem* pb, const fastmax_paged_decode_args* a, float* parts, void* cuda_stream) {
  using namespace fm;
  if (!pb || !a) return FASTMAX_ERR_INVALID_ARGUMENT;
  if (pb->batch <= 0 || pb->heads <= 0) return FASTMAX_ERR_INVALID_ARGUMENT;
  if (pb->dtype != FASTMAX_F32 && pb->dtype != FASTMAX_BF16) return FASTMAX_ERR_INVALID_ARGUMENT;
  if (pb->d != 16 && pb->d != 32 && pb->d != 64) return FASTMAX_ERR_UNSUPPORTED;
  if (pb->order != 1 && pb->order != 2) return FASTMAX_ERR_UNSUPPORTED;
  if (pb->nq != 1 || pb->nk != 1) return FASTMAX_ERR_UNSUPPORTED;
  if ((long long)pb->batch * pb->heads > 65535) return FASTMAX_ERR_UNSUPPORTED;
  if (!a->q.ptr || !a->k.ptr || !a->v.ptr || !a->o.ptr) return FASTMAX_ERR_INVALID_ARGUMENT;
  if (const int rc = check_pages(pb, a->cache)) return rc;
  dec::DecodeParams P;
  P.q = View{a->q.ptr, a->q.stride_b, a->q.stride_h, a->q.stride_n};
  P.k = View{a->k.ptr, a->k.stride_b, a->k.stride_h, a->k.stride_n};
  P.v = View{a->v.ptr, a->v.stride_b, a->v.stride_h, a->v.stride_n};
  P.o = View{a->o.ptr, a->o.stride_b, a->o.stride_h, a->o.stride_n};
  P.g = View{a->g.ptr, a->g.stride_b, a->g.stride_h, a->g.stride_n};
  P.state = a->cache.state;
  P.table = a->cache.table;
  P.page_stride = a->cache.page_stride;
  P.pages = a->cache.pages;
  P.heads = pb->heads;
  P.rows = state_rows(pb->d, pb->order);
  P.c0 = pb->a0;
  P.c1 = pb->a1 * pb->inv_temperature;
  P.c2 = pb->order == 2 ? pb->a2 * pb->inv_temperature * pb->inv_temperature : 0.f;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  const int bh = pb->batch * pb->heads;
  const cudaError_t e = pb->dtype == FASTMAX_BF16 ? dec::launch_d<__nv_bfloat16>(pb->d, pb->order, P, bh, parts, st)
                                                  : dec::launch_d<float>(pb->d, pb->order, P, bh, parts, st);
  return e == cudaSuccess ? FASTMAX_OK : report_cuda_error(e);
}

extern "C" size_t fastmax_decode_step_workspace(const fastmax_problem* pb) {
  using namespace fm;
  if (!pb || pb->batch <= 0 || pb->heads <= 0 || (pb->d != 16 && pb->d != 32 && pb->d != 64) || (pb->order != 1 && pb->order != 2)) return 0;
  const long long bh = (long long)pb->batch * pb->heads;
  // us by clusters / by short blocks: d = 64, 32 heads 12.4 / 11.1, 64 19.1 / 18.2, 96 29.7 / 24.1, 512 115.7 / 104.7; d = 32, 64 heads 6.9 / 7.3, 128
  // 12.4 / 9.0, 512 27.9 / 21.2; d = 16, 512 heads 7.2 / 7.8, 1024 10.9 / 10.5; order 1, d = 64, 128 heads 8.1 / 3.9, 512 9.6 / 8.2.
  if (pb->order == 2 ? bh * pb->d * pb->d < 1 << 17 : bh < 128) return 0;
  return (size_t)(bh * dec::row_groups(pb->d, pb->order) * state_ld(pb->d) * 4);
}

extern "C" int32_t fastmax_decode_step_paged(const fastmax_problem* pb, const fastmax_paged_decode_args* a, void* workspace, size_t workspace_bytes,
                                             void* cuda_stream) {
  const size_t need = fastmax_decode_step_workspace(pb);
  if (need > 0 && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 || workspace_bytes < need)) return FASTMAX_ERR_WORKSPACE;
  return decode_step(pb, a, need > 0 ? reinterpret_cast<float*>(workspace) : nullptr, cuda_stream);
}

extern "C" int32_t fastmax_decode_step(const fastmax_problem* pb, const fastmax_decode_args* a, void* cuda_stream) {
  if (!pb || !a) return FASTMAX_ERR_INVALID_ARGUMENT;
  fastmax_paged_decode_args paged{};
  paged.q = a->q, paged.k = a->k, paged.v = a->v, paged.o = a->o, paged.g = a->g;
  paged.cache.state = a->state;
  paged.cache.page_stride = (int64_t)pb->heads * fm::state_rows(pb->d, pb->order) * fm::state_ld(pb->d);
  paged.cache.pages = pb->batch;
  return decode_step(pb, &paged, nullptr, cuda_stream);
}
