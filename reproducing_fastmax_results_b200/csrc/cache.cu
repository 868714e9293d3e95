// Pages of moment states change hands: fastmax_cache_arrange (fork, end and begin sequences), fastmax_cache_compact and
// fastmax_pages_copy.
//
// A page is a few hundred kilobytes to many megabytes (one layer of eight heads, d = 64, order 2: 5.2 MB), the table a few hundred entries:
// the bytes that are copied are all that costs.  So a page moves only where two places go on from it: a single block decides which (the
// lists go into the workspace), then the whole GPU copies.  The pages that are written are free ones and those that are read are kept, so no
// copy waits for another.  A call that copies nothing takes 3.5 us (1000 places 3.8, 30 000 places 34), 31 writes of 31 MB 152.5 us (96 % of
// the copy rate), 37 moves of 21 MB 238 us (98 %).
#include <cuda_runtime.h>
#include <limits.h>

#include <atomic>

#include "../../include/fastmax_b200.h"
#include "common.cuh"
#include "launchers.cuh"
#include "pages.cuh"

namespace fm {

int report_cuda_error(cudaError_t e);
int sm_count();

namespace cache {

constexpr int PLAN_THREADS = 1024;

// What a plan leaves in the workspace: moves (count), their sources (-1: the page is cleared), their destinations; `held` is the plan's own.
struct PlanLists {
  int* count;
  int* src;
  int* dst;
  int* held;
};
static PlanLists plan_lists(void* workspace, int places) {
  int* w = reinterpret_cast<int*>(workspace);
  return PlanLists{w, w + 4, w + 4 + places, w + 4 + 2 * (long long)places};
}

// Rank of this thread among the threads of the block for which `mine` holds, behind `before`, which grows by their number.
// Two barriers; every thread of the block calls it.
__device__ __forceinline__ int block_rank(bool mine, int& before, int* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned ball = __ballot_sync(0xffffffffu, mine);
  if (lane == 0) warp_sums[warp] = __popc(ball);
  __syncthreads();
  int total = warp_sums[lane];   // as many warps as lanes
  int scan = total;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int x = __shfl_up_sync(0xffffffffu, scan, o);
    if (lane >= o) scan += x;
  }
  const int mine_before = __shfl_sync(0xffffffffu, scan - total, warp);
  total = __shfl_sync(0xffffffffu, scan, 31);
  __syncthreads();
  const int rank = before + mine_before + __popc(ball & ((1u << lane) - 1u));
  before += total;
  return rank;
}

// One block.  first[p]: the lowest place that goes on from page p.
__global__ void __launch_bounds__(PLAN_THREADS)
arrange_plan_kernel(int* table, const int* sources, int places, int pages, int* unserved, const PlanLists L) {
  extern __shared__ int smem[];
  int* first = smem;                                                     // [pages]
  unsigned short* freed = reinterpret_cast<unsigned short*>(smem + pages);   // [pages]: the free ones, ascending
  __shared__ int sums[32];
  __shared__ int wrong;
  const int tid = threadIdx.x;
  if (tid == 0) wrong = 0;
  for (int p = tid; p < pages; p += PLAN_THREADS) first[p] = INT_MAX;
  __syncthreads();
  grid_wait();
  grid_trigger();
  constexpr int BATCH = 4;   // places of a thread whose loads are under way together
  for (int i0 = tid; i0 < places; i0 += BATCH * PLAN_THREADS) {
    int j[BATCH], held[BATCH];
#pragma unroll
    for (int t = 0; t < BATCH; ++t) j[t] = i0 + t * PLAN_THREADS < places ? sources[i0 + t * PLAN_THREADS] : -1;
#pragma unroll
    for (int t = 0; t < BATCH; ++t) held[t] = j[t] >= 0 && j[t] < places ? table[j[t]] : -1;
#pragma unroll
    for (int t = 0; t < BATCH; ++t) {
      const int i = i0 + t * PLAN_THREADS;
      if (held[t] < 0 || held[t] >= pages) held[t] = j[t] == -2 ? -2 : -1;
      if (j[t] < -2 || j[t] >= places) atomicAdd(&wrong, 1);
      if (held[t] >= 0) atomicMin(&first[held[t]], i);
      if (i < places) L.held[i] = held[t];   // read again by this thread alone
    }
  }
  __syncthreads();   // from here on nobody reads the table any more
  int nfree = 0;
  for (int p0 = 0; p0 < pages; p0 += PLAN_THREADS) {
    const int p = p0 + tid;
    const bool is_free = p < pages && first[p] == INT_MAX;
    const int r = block_rank(is_free, nfree, sums);
    if (is_free) freed[r] = (unsigned short)p;
  }
  __syncthreads();
  int nwant = 0;
  int ahead = tid < places ? L.held[tid] : -1;
  for (int i0 = 0; i0 < places; i0 += PLAN_THREADS) {
    const int i = i0 + tid;
    const int held = ahead;
    ahead = i + PLAN_THREADS < places ? L.held[i + PLAN_THREADS] : -1;
    const bool keeps = held >= 0 && first[held] == i;
    const bool wants = held == -2 || (held >= 0 && !keeps);
    const int r = block_rank(wants, nwant, sums);
    if (i < places) {
      int page = keeps ? held : -1;
      if (wants && r < nfree) {
        page = freed[r];
        L.src[r] = held == -2 ? -1 : held;
        L.dst[r] = page;
      }
      table[i] = page;
    }
  }
  if (tid == 0) {
    *L.count = min(nwant, nfree);
    *unserved = wrong + max(0, nwant - nfree);
  }
}

// One block.  where[p]: 0 a free page, 1 a live one; then the position of page p afterwards.
__global__ void __launch_bounds__(PLAN_THREADS)
compact_plan_kernel(int* table, int places, int pages, int* live, const PlanLists L) {
  extern __shared__ int smem[];
  int* where = smem;
  unsigned short* holes = reinterpret_cast<unsigned short*>(smem + pages);
  __shared__ int sums[32];
  const int tid = threadIdx.x;
  for (int p = tid; p < pages; p += PLAN_THREADS) where[p] = 0;
  __syncthreads();
  grid_wait();
  grid_trigger();
  for (int i = tid; i < places; i += PLAN_THREADS) {
    const int p = table[i];
    if (p >= 0 && p < pages) where[p] = 1;
  }
  __syncthreads();
  int n = 0;
  for (int p0 = 0; p0 < pages; p0 += PLAN_THREADS) {
    const int p = p0 + tid;
    block_rank(p < pages && where[p] == 1, n, sums);
  }
  int nholes = 0;
  for (int p0 = 0; p0 < n; p0 += PLAN_THREADS) {
    const int p = p0 + tid;
    const bool hole = p < n && where[p] == 0;
    const int r = block_rank(hole, nholes, sums);
    if (hole) holes[r] = (unsigned short)p;
  }
  __syncthreads();
  int nmove = 0;   // as many as there are holes
  for (int p0 = 0; p0 < pages; p0 += PLAN_THREADS) {
    const int p = p0 + tid;
    const bool is_live = p < pages && where[p] == 1;
    const bool moves = is_live && p >= n;
    const int r = block_rank(moves, nmove, sums);
    if (moves) {
      L.src[r] = p;
      L.dst[r] = holes[r];
      where[p] = holes[r];
    } else if (is_live) {
      where[p] = p;
    }
  }
  __syncthreads();
  for (int i = tid; i < places; i += PLAN_THREADS) {
    const int p = table[i];
    table[i] = p >= 0 && p < pages ? where[p] : -1;
  }
  if (tid == 0) {
    *L.count = nmove;
    *live = n;
  }
}

struct CopyParams {
  const float4* src;
  float4* dst;
  long long src_stride, dst_stride, page;   // float4
  int src_pages, dst_pages;
  const int *src_index, *dst_index;         // NULL: i itself
  const int* count_at;                      // NULL: `count`
  int count;
  bool clear;                               // a source of -1 clears the destination
};

constexpr int COPY_THREADS = 256;
constexpr int COPY_UNROLL = 2;
constexpr int COPY_CHUNK = COPY_THREADS * COPY_UNROLL;   // float4 of a step: 8 KB
constexpr int COPY_BLOCKS = 4;                           // to an SM
// 64 KB in flight an SM.  GB/s at 760 MB read and written (a copy of one tensor by PyTorch: 6440), steps of KB x blocks to an SM: 8 x 4
// 6390, 8 x 3 5850, 8 x 5 5850, 16 x 2 6220, 16 x 4 5870, 32 x 1 5990, 32 x 2 5910, 4 x 8 6050; streaming loads too 6290, ordinary stores 6160.

// A block's steps are gridDim.x chunks apart; the next step's loads are in flight while one is stored.
__global__ void __launch_bounds__(COPY_THREADS, COPY_BLOCKS)
pages_copy_kernel(const CopyParams P) {
  grid_wait();
  grid_trigger();
  const int count = P.count_at != nullptr ? *P.count_at : P.count;
  const long long chunks = (P.page + COPY_CHUNK - 1) / COPY_CHUNK;
  struct Step {
    float4 x[COPY_UNROLL];
    float4* to;     // NULL: nothing to store
    int quads;      // of this thread's: the first of them lies at the thread's number
  };
  int i = (int)(blockIdx.x / chunks);
  long long c = blockIdx.x - i * chunks;
  auto fetch = [&](Step& s) {
    s.to = nullptr;
    if (i >= count) return;
    const int from = P.src_index != nullptr ? P.src_index[i] : i;
    const int to = P.dst_index != nullptr ? P.dst_index[i] : i;
    const bool known = from >= 0 && from < P.src_pages;
    const long long at = c * COPY_CHUNK;
    s.quads = (int)(P.page - at < COPY_CHUNK ? P.page - at : COPY_CHUNK);
    if (to >= 0 && to < P.dst_pages && (known || P.clear)) s.to = P.dst + to * P.dst_stride + at + threadIdx.x;
    const float4* src = P.src + from * P.src_stride + at + threadIdx.x;
#pragma unroll
    for (int j = 0; j < COPY_UNROLL; ++j) {
      s.x[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (known && s.to != nullptr && (int)threadIdx.x + j * COPY_THREADS < s.quads) s.x[j] = src[j * COPY_THREADS];
    }
    c += gridDim.x;
    while (c >= chunks) c -= chunks, ++i;
  };
  auto put = [&](const Step& s) {
    if (s.to == nullptr) return;
#pragma unroll
    for (int j = 0; j < COPY_UNROLL; ++j)
      if ((int)threadIdx.x + j * COPY_THREADS < s.quads) __stcs(s.to + j * COPY_THREADS, s.x[j]);
  };
  Step a, b;
  fetch(a);
  while (i < count) {
    fetch(b);
    put(a);
    a = b;
  }
  put(a);
}

static cudaError_t launch_copy(const CopyParams& P, int most, cudaStream_t st) {
  const long long chunks = (P.page + COPY_CHUNK - 1) / COPY_CHUNK;
  const long long room = (long long)COPY_BLOCKS * sm_count();
  const long long blocks = most * chunks < room ? most * chunks : room;
  LaunchScope ls(KK_CACHE_COPY, st);
  return launch_after(pages_copy_kernel, dim3((unsigned)blocks), COPY_THREADS, 0, st, P);
}

// The plan kernels keep six bytes per page in shared memory; above 48 KB that has to be allowed once per device and kernel.
static int plan_bytes(int pages) { return 6 * pages + 2; }
template <typename K>
static cudaError_t allow_plan_bytes(K kernel, int which) {
  static std::atomic<bool> done[2][64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !done[which][dev].load(std::memory_order_relaxed)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, plan_bytes(FASTMAX_CACHE_PAGES));
    if (e != cudaSuccess) return launched(e);
    if (dev < 64) done[which][dev].store(true, std::memory_order_relaxed);
  }
  return cudaSuccess;
}

static int check_cache(const float* state, int64_t page_floats, int32_t pages, const int32_t* table, int32_t places, const int32_t* result,
                       const void* workspace, size_t workspace_bytes) {
  if (!state || !table || !result || page_floats <= 0 || pages <= 0 || places <= 0) return FASTMAX_ERR_INVALID_ARGUMENT;
  if (pages > FASTMAX_CACHE_PAGES || places > FASTMAX_CACHE_PAGES) return FASTMAX_ERR_UNSUPPORTED;
  if (reinterpret_cast<uintptr_t>(state) % 16 != 0 || page_floats % 4 != 0) return FASTMAX_ERR_MISALIGNED;
  if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 || workspace_bytes < fastmax_cache_workspace(places)) return FASTMAX_ERR_WORKSPACE;
  return FASTMAX_OK;
}

static CopyParams moves(float* state, int64_t page_floats, int pages, const PlanLists& L) {
  CopyParams P{};
  P.src = reinterpret_cast<const float4*>(state);
  P.dst = reinterpret_cast<float4*>(state);
  P.src_stride = P.dst_stride = P.page = page_floats / 4;
  P.src_pages = P.dst_pages = pages;
  P.src_index = L.src;
  P.dst_index = L.dst;
  P.count_at = L.count;
  P.clear = true;
  return P;
}

}  // namespace cache
}  // namespace fm

extern "C" size_t fastmax_cache_workspace(int32_t places) { return places <= 0 ? 0 : 16 + 12 * (size_t)places; }

extern "C" int32_t fastmax_cache_arrange(float* state, int64_t page_floats, int32_t pages, int32_t* table, int32_t places, const int32_t* sources,
                                         int32_t* unserved, void* workspace, size_t workspace_bytes, void* cuda_stream) {
  using namespace fm;
  using namespace fm::cache;
  if (!sources) return FASTMAX_ERR_INVALID_ARGUMENT;
  if (const int rc = check_cache(state, page_floats, pages, table, places, unserved, workspace, workspace_bytes)) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  const PlanLists L = plan_lists(workspace, places);
  cudaError_t e = allow_plan_bytes(arrange_plan_kernel, 0);
  if (e == cudaSuccess) {
    LaunchScope ls(KK_CACHE_PLAN, st);
    e = launch_after(arrange_plan_kernel, dim3(1), PLAN_THREADS, plan_bytes(pages), st, table, sources, places, pages, unserved, L);
  }
  if (e == cudaSuccess) e = launch_copy(moves(state, page_floats, pages, L), places < pages ? places : pages, st);
  return e == cudaSuccess ? FASTMAX_OK : report_cuda_error(e);
}

extern "C" int32_t fastmax_cache_compact(float* state, int64_t page_floats, int32_t pages, int32_t* table, int32_t places, int32_t* live,
                                         void* workspace, size_t workspace_bytes, void* cuda_stream) {
  using namespace fm;
  using namespace fm::cache;
  if (const int rc = check_cache(state, page_floats, pages, table, places, live, workspace, workspace_bytes)) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  const PlanLists L = plan_lists(workspace, places);
  cudaError_t e = allow_plan_bytes(compact_plan_kernel, 1);
  if (e == cudaSuccess) {
    LaunchScope ls(KK_CACHE_PLAN, st);
    e = launch_after(compact_plan_kernel, dim3(1), PLAN_THREADS, plan_bytes(pages), st, table, places, pages, live, L);
  }
  if (e == cudaSuccess) e = launch_copy(moves(state, page_floats, pages, L), places < pages ? places : pages, st);
  return e == cudaSuccess ? FASTMAX_OK : report_cuda_error(e);
}

extern "C" int32_t fastmax_pages_copy(const fastmax_pages_copy_args* a, void* cuda_stream) {
  using namespace fm;
  using namespace fm::cache;
  if (!a || !a->src || !a->dst || a->page_floats <= 0 || a->src_pages <= 0 || a->dst_pages <= 0 || a->count < 0) return FASTMAX_ERR_INVALID_ARGUMENT;
  if ((a->src_pages > 1 && a->src_stride < a->page_floats) || (a->dst_pages > 1 && a->dst_stride < a->page_floats)) return FASTMAX_ERR_INVALID_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(a->src) % 16 != 0 || reinterpret_cast<uintptr_t>(a->dst) % 16 != 0 || a->page_floats % 4 != 0 ||
      a->src_stride % 4 != 0 || a->dst_stride % 4 != 0)
    return FASTMAX_ERR_MISALIGNED;
  if (a->count == 0) return FASTMAX_OK;
  CopyParams P{};
  P.src = reinterpret_cast<const float4*>(a->src);
  P.dst = reinterpret_cast<float4*>(a->dst);
  P.src_stride = a->src_stride / 4;
  P.dst_stride = a->dst_stride / 4;
  P.page = a->page_floats / 4;
  P.src_pages = a->src_pages;
  P.dst_pages = a->dst_pages;
  P.src_index = a->src_index;
  P.dst_index = a->dst_index;
  P.count = a->count;
  const cudaError_t e = launch_copy(P, a->count, reinterpret_cast<cudaStream_t>(cuda_stream));
  return e == cudaSuccess ? FASTMAX_OK : report_cuda_error(e);
}
