// Trees of drafted tokens over cached moment states: fastmax_tree_attention and fastmax_tree_accept.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "../../include/fastmax_b200.h"
#include "common.cuh"
#include "launchers.cuh"
#include "pages.cuh"

namespace fm {

int report_cuda_error(cudaError_t e);
int sm_count();

namespace tree {

struct TreeParams {
  View q, k, v, o, g;
  float* state;
  const int* table;
  long long page_stride;
  int pages;
  int heads, rows, nodes;
  const int* parents;
  long long parents_stride;
  const int* ends;          // attention: lengths; accepting: last
  float a0, a1, a2, inv_t;
};

__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store1(float* p, float x) { *p = x; }
__device__ __forceinline__ void store1(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

__device__ __forceinline__ int parent_of(const TreeParams& P, int b, int i) {
  if (P.parents == nullptr) return i - 1;
  const int p = P.parents[b * P.parents_stride + i];
  return p >= 0 && p < i ? p : -1;
}
// first float of the sequence's head, or NULL for an absent sequence
__device__ __forceinline__ float* head_state(const TreeParams& P, int b, int h, int d) {
  int page = b;
  if (P.table != nullptr) {
    page = P.table[b];
    if (page < 0 || page >= P.pages) return nullptr;
  }
  return P.state + page * P.page_stride + (long long)h * P.rows * (d + 4);
}

template <typename T, int D, int ORDER>
__global__ void attention_kernel(const TreeParams P) {
  using G = Geo<D>;
  grid_wait();
  grid_trigger();
  const int i = blockIdx.x, b = blockIdx.y / P.heads, h = blockIdx.y - b * P.heads, c = threadIdx.x;
  const float* S = head_state(P, b, h, D);
  if (S == nullptr || (P.ends != nullptr && i >= P.ends[b])) return;
  __shared__ float sq[D], out[D + 1];
  const T* q = head_base<T>(P.q, blockIdx.y, P.heads) + i * P.q.sn;
  if (c < D) sq[c] = load1(q + c);
  __syncthreads();
  float sum = 0.f;
  if (c <= D) {
    const float c1 = P.a1 * P.inv_t, c2 = P.a2 * P.inv_t * P.inv_t;
    int r = 0;
    if (ORDER == 2)
      for (int x = 0; x < D; x += 8)
        for (int y = x; y < D; y += 8)
          for (int m = 0; m < 8; ++m)
            for (int n = 0; n < 8; ++n, ++r) sum = fmaf(sq[x + m] * sq[y + n] * (x == y ? c2 : 2.f * c2), S[(long long)r * (D + 4) + c], sum);
    for (int m = 0; m < D; ++m, ++r) sum = fmaf(sq[m] * c1, S[(long long)r * (D + 4) + c], sum);
    sum = fmaf(P.a0, S[(long long)r * (D + 4) + c], sum);
    for (int j = i; j >= 0; j = parent_of(P, b, j)) {
      const T* k = head_base<T>(P.k, blockIdx.y, P.heads) + j * P.k.sn;
      float s = 0.f;
      for (int m = 0; m < D; ++m) s = fmaf(sq[m], load1(k + m), s);
      s *= P.inv_t;
      const float f = P.a0 + s * (P.a1 + (ORDER == 2 ? P.a2 * s : 0.f));
      sum = fmaf(f, c < D ? load1(head_base<T>(P.v, blockIdx.y, P.heads) + j * P.v.sn + c) : 1.f, sum);
    }
    out[c] = sum;
  }
  __syncthreads();
  if (c < D) store1(const_cast<T*>(head_base<T>(P.o, blockIdx.y, P.heads)) + i * P.o.sn + c, out[c] / out[D]);
  if (c == D && P.g.ptr != nullptr) const_cast<float*>(head_base<float>(P.g, blockIdx.y, P.heads))[i * P.g.sn] = out[D];
}

template <typename T, int D, int ORDER>
__global__ void accept_kernel(const TreeParams P) {
  using G = Geo<D>;
  grid_wait();
  grid_trigger();
  const int b = blockIdx.y / P.heads, h = blockIdx.y - b * P.heads;
  float* S = head_state(P, b, h, D);
  if (S == nullptr || P.ends[b] < 0 || P.ends[b] >= P.nodes) return;
  const long long at = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const int r = (int)(at / (D + 4)), c = (int)(at - (long long)r * (D + 4));
  if (r >= P.rows || c > D) return;
  int path[FASTMAX_TREE_NODES], n = 0;
  for (int j = P.ends[b]; j >= 0; j = parent_of(P, b, j)) path[n++] = j;
  float s = S[at];
  while (n > 0) {
    const int j = path[--n];
    const T* k = head_base<T>(P.k, blockIdx.y, P.heads) + j * P.k.sn;
    const T* v = head_base<T>(P.v, blockIdx.y, P.heads) + j * P.v.sn;
    float f = 1.f;
    if (ORDER == 2 && r < 64 * G::NPAIRS) {
      int x, y;
      pair_decode(r >> 6, G::NB, x, y);
      f = load1(k + 8 * x + ((r & 63) >> 3)) * load1(k + 8 * y + (r & 7));
    } else {
      const int m = r - (ORDER == 2 ? 64 * G::NPAIRS : 0);
      if (m < D) f = load1(k + m);
    }
    s = fmaf(f, c < D ? load1(v + c) : 1.f, s);
  }
  S[at] = s;
}

template <typename T, int D, int ORDER>
static cudaError_t launch(bool attend, const TreeParams& P, int bh, cudaStream_t st) {
  if (attend) return launch_after(attention_kernel<T, D, ORDER>, dim3((unsigned)P.nodes, (unsigned)bh), 96, 0, st, P);
  return launch_after(accept_kernel<T, D, ORDER>, dim3((unsigned)((P.rows * (D + 4) + 255) / 256), (unsigned)bh), 256, 0, st, P);
}
template <typename T, int D>
static cudaError_t launch_order(bool attend, int order, const TreeParams& P, int bh, cudaStream_t st) {
  return order == 2 ? launch<T, D, 2>(attend, P, bh, st) : launch<T, D, 1>(attend, P, bh, st);
}
template <typename T>
static cudaError_t launch_d(bool attend, int d, int order, const TreeParams& P, int bh, cudaStream_t st) {
  switch (d) {
    case 16: return launch_order<T, 16>(attend, order, P, bh, st);
    case 32: return launch_order<T, 32>(attend, order, P, bh, st);
    default: return launch_order<T, 64>(attend, order, P, bh, st);
  }
}

static int check_problem(const fastmax_problem* pb) {
  if (pb->batch <= 0 || pb->heads <= 0 || pb->nq <= 0) return FASTMAX_ERR_INVALID_ARGUMENT;
  if (pb->dtype != FASTMAX_F32 && pb->dtype != FASTMAX_BF16) return FASTMAX_ERR_INVALID_ARGUMENT;
  if (pb->d != 16 && pb->d != 32 && pb->d != 64) return FASTMAX_ERR_UNSUPPORTED;
  if (pb->order != 1 && pb->order != 2) return FASTMAX_ERR_UNSUPPORTED;
  if (pb->nq != pb->nk || pb->nq > FASTMAX_TREE_NODES) return FASTMAX_ERR_UNSUPPORTED;
  if ((long long)pb->batch * pb->heads > 65535) return FASTMAX_ERR_UNSUPPORTED;
  return FASTMAX_OK;
}

static TreeParams params(const fastmax_problem* pb, const fastmax_pages& cache, const int32_t* parents, int64_t parents_stride, const int32_t* ends) {
  TreeParams P{};
  P.state = cache.state;
  P.table = cache.table;
  P.page_stride = cache.page_stride;
  P.pages = cache.pages;
  P.heads = pb->heads;
  P.rows = state_rows(pb->d, pb->order);
  P.nodes = pb->nq;
  P.parents = parents;
  P.parents_stride = parents_stride;
  P.ends = ends;
  P.a0 = pb->a0;
  P.a1 = pb->a1;
  P.a2 = pb->a2;
  P.inv_t = pb->inv_temperature;
  return P;
}
static View view(const fastmax_tensor& t) { return View{t.ptr, t.stride_b, t.stride_h, t.stride_n}; }

}  // namespace tree
}  // namespace fm

extern "C" int32_t fastmax_tree_attention(const fastmax_problem* pb, const fastmax_tree_args* a, void* cuda_stream) {
  using namespace fm;
  if (!pb || !a) return FASTMAX_ERR_INVALID_ARGUMENT;
  if (const int rc = tree::check_problem(pb)) return rc;
  if (!a->q.ptr || !a->k.ptr || !a->v.ptr || !a->o.ptr) return FASTMAX_ERR_INVALID_ARGUMENT;
  if (const int rc = check_pages(pb, a->cache)) return rc;
  tree::TreeParams P = tree::params(pb, a->cache, a->parents, a->parents_stride, a->lengths);
  P.q = tree::view(a->q), P.k = tree::view(a->k), P.v = tree::view(a->v), P.o = tree::view(a->o), P.g = tree::view(a->g);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  cudaError_t e;
  {
    LaunchScope ls(KK_TREE, st);
    e = pb->dtype == FASTMAX_BF16 ? tree::launch_d<__nv_bfloat16>(true, pb->d, pb->order, P, pb->batch * pb->heads, st)
                                  : tree::launch_d<float>(true, pb->d, pb->order, P, pb->batch * pb->heads, st);
  }
  return e == cudaSuccess ? FASTMAX_OK : report_cuda_error(e);
}

extern "C" int32_t fastmax_tree_accept(const fastmax_problem* pb, const fastmax_accept_args* a, void* cuda_stream) {
  using namespace fm;
  if (!pb || !a) return FASTMAX_ERR_INVALID_ARGUMENT;
  if (const int rc = tree::check_problem(pb)) return rc;
  if (!a->k.ptr || !a->v.ptr || !a->last) return FASTMAX_ERR_INVALID_ARGUMENT;
  if (const int rc = check_pages(pb, a->cache)) return rc;
  tree::TreeParams P = tree::params(pb, a->cache, a->parents, a->parents_stride, a->last);
  P.k = tree::view(a->k), P.v = tree::view(a->v);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  cudaError_t e;
  {
    LaunchScope ls(KK_TREE_ACCEPT, st);
    e = pb->dtype == FASTMAX_BF16 ? tree::launch_d<__nv_bfloat16>(false, pb->d, pb->order, P, pb->batch * pb->heads, st)
                                  : tree::launch_d<float>(false, pb->d, pb->order, P, pb->batch * pb->heads, st);
  }
  return e == cudaSuccess ? FASTMAX_OK : report_cuda_error(e);
}
