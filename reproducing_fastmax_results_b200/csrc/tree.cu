// Trees of drafted tokens over cached moment states: fastmax_tree_attention and fastmax_tree_accept.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <type_traits>

#include "../../include/fastmax_b200.h"
#include "common.cuh"
#include "launchers.cuh"
#include "pages.cuh"
#include "tc_launchers.cuh"
#include "tc_ptx.cuh"

namespace cg = cooperative_groups;

namespace fm {

int report_cuda_error(cudaError_t e);
int sm_count();

namespace tree {

using namespace tc;

__device__ int g_status = 0;       // see tc_device_status
__device__ int g_wait_hist[256];

constexpr long long WAIT_CYCLES = 4000000000ll;   // ~2 s at 2 GHz
constexpr int WAIT_SLOT = 210;                    // the site's code: a slot of the state

// Waits for the phase of parity `parity`.  Returns in any case: when the wait runs out (code `code`), the flag is up, no further copy is
// asked for and every later wait of the block falls through at once.  The thread that raises the flag reports, so a block counts once.
template <long long LIMIT = WAIT_CYCLES>
__device__ __noinline__ void wait_slow(uint64_t* bar, uint32_t parity, int code, volatile int* abort_flag) {
  if (*abort_flag == 0 && !mbar_wait_abortable(bar, parity, LIMIT, abort_flag) && atomicExch(const_cast<int*>(abort_flag), 1) == 0) {
    atomicAdd(&g_wait_hist[code & 255], 1);
    atomicExch(&g_status, code);
  }
}
template <long long LIMIT = WAIT_CYCLES>
__device__ __forceinline__ void wait(uint64_t* bar, uint32_t parity, int code, volatile int* abort_flag) {
  // (a test that does not suspend the thread: waking it costs some 250 clocks, and the copy has mostly arrived)
  for (int i = 0; i < 64; ++i)
    if (mbar_test_wait(bar, parity)) return;
  wait_slow<LIMIT>(bar, parity, code, abort_flag);
}
// Behind a block's last wait and a barrier, called by all threads where a wait ran out: nobody writes into the slots or leaves while a copy is
// under way.
__device__ __noinline__ void drain(uint64_t* full, const volatile int* issued, int slots) {
  if (threadIdx.x == 0)
    for (int i = 0; i < slots; ++i)
      if (issued[i] > 0) mbar_wait_bounded(&full[i], (uint32_t)(issued[i] - 1) & 1u, WAIT_CYCLES);
  __syncthreads();
}

// What a block does that gives up, without a state: one slot's copy never comes (nobody asks for it), the other's is under way meanwhile.
// A slot that the drain leaves before its copy is there counts at the site behind.
constexpr int SELFTEST_FLOATS = 64;
__device__ __align__(16) float g_selftest_source[SELFTEST_FLOATS];   // zeros
__global__ void wait_selftest_kernel() {
  __shared__ __align__(128) float slot[SELFTEST_FLOATS];
  __shared__ uint64_t full[2];
  __shared__ int flags[3];
  volatile int* issued = flags;
  volatile int* abort_flag = flags + 2;
  const int tid = threadIdx.x;
  slot[tid] = 1.f;
  if (tid == 0) {
    mbar_init(&full[0], 1), mbar_init(&full[1], 1);
    issued[0] = 0, issued[1] = 1, *abort_flag = 0;
    fence_mbar_init();
  }
  fence_proxy_async_smem();
  __syncthreads();
  if (tid == 0) {
    mbar_arrive_expect_tx(&full[1], sizeof(slot));
    bulk_load(slot, g_selftest_source, sizeof(slot), &full[1]);
  }
  wait<2000000ll>(&full[0], 0u, WAIT_SLOT, abort_flag);   // about a millisecond
  wait(&full[0], 0u, WAIT_SLOT, abort_flag);              // falls through
  __syncthreads();
  if (*abort_flag != 0) drain(full, issued, 2);
  if (slot[tid] != 0.f) atomicAdd(&g_wait_hist[WAIT_SLOT + 1], 1);
}

struct TreeParams {
  View q, k, v, o, g;
  float* state;
  const int* table;
  long long page_stride;
  int pages;
  int heads, rows, nodes, order;
  bool aligned;             // the rows of q, k, v, o can be accessed four dims at a time
  const int* parents;
  long long parents_stride;
  const int* ends;          // attention: lengths; accepting: last
  float a0, a1, a2, inv_t;
};

// four neighbours; `aligned`: all addresses are multiples of their size
__device__ __forceinline__ void load4v(const float* p, bool aligned, float (&x)[4]) {
  if (aligned) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = p[i];
  }
}
// the same in two steps: what is in flight, and its floats
template <typename T>
struct Raw4;
template <>
struct Raw4<float> {
  float4 v;
  __device__ __forceinline__ void load(const float* p, bool aligned) {
    float x[4];
    load4v(p, aligned, x);
    v = make_float4(x[0], x[1], x[2], x[3]);
  }
  __device__ __forceinline__ void get(bool there, float (&x)[4]) const {
    x[0] = there ? v.x : 0.f, x[1] = there ? v.y : 0.f, x[2] = there ? v.z : 0.f, x[3] = there ? v.w : 0.f;
  }
};
template <>
struct Raw4<__nv_bfloat16> {
  uint2 v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p, bool aligned) {
    if (aligned) {
      v = *reinterpret_cast<const uint2*>(p);
    } else {
      const unsigned short* u = reinterpret_cast<const unsigned short*>(p);
      v = make_uint2(u[0] | (uint32_t)u[1] << 16, u[2] | (uint32_t)u[3] << 16);
    }
  }
  __device__ __forceinline__ void get(bool there, float (&x)[4]) const {
    const uint32_t a = there ? v.x : 0u, b = there ? v.y : 0u;
    x[0] = __uint_as_float(a << 16), x[1] = __uint_as_float(a & 0xffff0000u);
    x[2] = __uint_as_float(b << 16), x[3] = __uint_as_float(b & 0xffff0000u);
  }
};
__device__ __forceinline__ void store4v(float* p, bool aligned, float a, float b, float c, float d) {
  if (aligned) {
    *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
  } else {
    p[0] = a, p[1] = b, p[2] = c, p[3] = d;
  }
}
__device__ __forceinline__ void store4v(__nv_bfloat16* p, bool aligned, float a, float b, float c, float d) {
  if (aligned) {
    __nv_bfloat162 x = __floats2bfloat162_rn(a, b), y = __floats2bfloat162_rn(c, d);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<uint32_t*>(&x), *reinterpret_cast<uint32_t*>(&y));
  } else {
    p[0] = __float2bfloat16_rn(a), p[1] = __float2bfloat16_rn(b), p[2] = __float2bfloat16_rn(c), p[3] = __float2bfloat16_rn(d);
  }
}

// Who sees whom, by one warp: of nodes lane and lane + 32 the node itself and its ancestors as bits.  `up`: their parents.  Pointers reach
// twice as far in every round.
__device__ __forceinline__ void load_parents(const TreeParams& P, int b, int lane, int (&up)[2]) {   // as they stand there
#pragma unroll
  for (int k = 0; k < 2; ++k) up[k] = P.parents != nullptr && lane + 32 * k < P.nodes ? P.parents[b * P.parents_stride + lane + 32 * k] : -1;
}
__device__ __forceinline__ void ancestors(const TreeParams& P, int n, int lane, int (&up)[2], unsigned long long (&seen)[2]) {
#pragma unroll
  for (int k = 0; k < 2; ++k) seen[k] = P.parents == nullptr ? (2ull << (lane + 32 * k)) - 1ull : 1ull << (lane + 32 * k);
  if (P.parents == nullptr) return;
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (up[k] >= lane + 32 * k || up[k] < 0) up[k] = -1;   // no node before it
  for (int far = 1; far < n; far *= 2) {
    unsigned long long more[2];
    int next[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const unsigned long long m0 = __shfl_sync(0xffffffffu, seen[0], up[k] & 31), m1 = __shfl_sync(0xffffffffu, seen[1], up[k] & 31);
      const int n0 = __shfl_sync(0xffffffffu, up[0], up[k] & 31), n1 = __shfl_sync(0xffffffffu, up[1], up[k] & 31);
      more[k] = up[k] < 0 ? 0ull : up[k] < 32 ? m0 : m1;
      next[k] = up[k] < 0 ? -1 : up[k] < 32 ? n0 : n1;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) seen[k] |= more[k], up[k] = next[k];
  }
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

// ---- attention ---------------------------------------------------------------------------------------------------------
//     o'_i = sum_r w_r Phi(q_i)_r S[r] + sum_{j in A(i)} f(q_i . k_j / T) [v_j | 1],      o_i = o'_i[:D] / o'_i[D]
//
// The sums over the state are matrix products in which the state is read once for all nodes of a tree.  For a row m the products x_m x_n of the
// blocks b >= a lie one after the other, so  sum_n S[(m, n)][c] x_n  are products with x itself, and x_m times them (with the pairs' weight) is
// added in float32: only the state is split into bfloat16 pieces, and x where it is float32.
//
// Layout of a product m16n8k16: 16 rows = columns c of the state, 8 columns = nodes, 16 terms = 8 + 8 rows n of two units (a, b), (a, b + 1).
// A block has one head, or a cluster of blocks shares one; its warps divide the columns by 16 and the rows m of a unit (KG groups).  Units come
// by the copy engine into a ring of slots; whichever warp is done last with a step asks for the units that take its place.
//
// Products by warps and not tcgen05: the operand that streams is the state, which has to be split on its way.  In registers it goes straight from
// one wide load into the product; for tcgen05 its pieces would have to be written to shared memory once more.  Up to 8 nodes that could only
// lose (HBM bounds it); for the largest trees, where the accumulators of this form leave room for 16 warps an SM, it has not been built or measured.
//
// What bounds it (bf16, 512 heads of 64 dims, order 2, 330 MB of states, 50 us at the copy rate): up to 8 nodes HBM, 53.9 us; 25 nodes 70 us and 64
// nodes 116 us, the chain of a step (load, split, product, scale: issue slots 51 and 47 %, tensor pipe active 34 and 41 %) and the rounds of blocks:
// 288 heads of 25 nodes take 38 us, 464 70 us, 592 73 us.  float32 (512 heads, 64 dims; six products where bfloat16 has two): 8 nodes 65 us, 16 81, 25 132,
// 40 211, 64 276.  Built and left (bf16): 25 nodes, 464 heads (70 us): sixteen warps a block and one block to an SM
// 94, two of them 91, four warps 78, three blocks of eight 90; slots 3 / 4 / 5: 85 / 71 / 70; halves of heads in clusters 79.  Copies by the
// threads instead of the copy engine: 91 instead of 71 us for 8 nodes at that stage.  The tree's sums as products, too: chains of 64 nodes 115
// instead of 134 us, but trees as before and small ones 1 to 3 % slower.  The last units of rows of odd length paired up with m and n exchanged (18
// steps instead of 20, the units out of their order): 77.  Groups of products written out in turn, and cutting off instead of rounding the
// pieces (fewer instructions), changed nothing.

template <typename T>
struct Pieces {   // of x and of the state.  bfloat16 x is one piece; two of the state keep 2^-16 of each term, far below the output's 2^-8
  static constexpr int Q = 1, S = 2;
};
template <>
struct Pieces<float> {   // three of both keep 2^-24: six products
  static constexpr int Q = 3, S = 3;
};

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {   // rounded to nearest
  __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&p);
}
// the pieces of two floats, each what the ones before it leave
template <int N>
__device__ __forceinline__ void split2(float x, float y, uint32_t (&out)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    out[i] = pack_bf16(x, y);
    if (i + 1 < N) {
      x -= __uint_as_float(out[i] << 16);
      y -= __uint_as_float(out[i] & 0xffff0000u);
    }
  }
}
__device__ __forceinline__ uint32_t twice(uint32_t x) {   // of two bfloat16, exact
  const __nv_bfloat162 v = *reinterpret_cast<__nv_bfloat162*>(&x);
  const __nv_bfloat162 r = __hadd2(v, v);
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ int count_up(int* counter) {   // in shared memory; orders what the warps did before
  int old;
  asm volatile("atom.add.acq_rel.cta.shared::cta.s32 %0, [%1], 1;" : "=r"(old) : "r"(smem_u32(counter)) : "memory");
  return old;
}
// c += s * p, two at a time
__device__ __forceinline__ void fma2(float& c0, float& c1, float2 s, float p0, float p1) {
  asm("{\n\t.reg .b64 c, s, p;\n\t"
      "mov.b64 c, {%0, %1};\n\tmov.b64 s, {%2, %3};\n\tmov.b64 p, {%4, %5};\n\t"
      "fma.rn.f32x2 c, s, p, c;\n\tmov.b64 {%0, %1}, c;\n\t}"
      : "+f"(c0), "+f"(c1) : "f"(s.x), "f"(s.y), "f"(p0), "f"(p1));
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816_from_zero(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// a product of 16 terms from the pieces of the state and of x, the smallest first
template <int SP, int QP>
__device__ __forceinline__ void products(float (&c)[4], const uint32_t (&a)[SP][4], const uint32_t (&x)[2][QP]) {
#pragma unroll
  for (int p = SP - 1; p >= 0; --p)
#pragma unroll
    for (int i = 0; i <= p; ++i)
      if (p - i < QP) {
        if (p == SP - 1 && i == (p < QP ? 0 : p - QP + 1)) mma16816_from_zero(c, a[i], x[0][p - i], x[1][p - i]);
        else mma16816(c, a[i], x[0][p - i], x[1][p - i]);
      }
}

template <typename T, int D, int NT>
struct TreeGeo {
  static constexpr int N = 8 * NT;                     // nodes, filled up
  static constexpr int NB = D / 8;
  static constexpr int CG = D / 16;                    // groups of 16 columns of the state: one to a warp
  // Blocks to an SM, and warps that share a group of columns and divide the rows m of a unit among them: eight warps for 64 dims, four for fewer (us
  // with eight warps, two blocks / four warps, four blocks, 512 heads: 32 dims, 8 nodes 16.2 / 11.6, 25 nodes 21.6 / 16.9; 16 dims, 16 nodes 11.6 / 7.5).
  // float32 trees of more than 32 nodes: half as many blocks, so that 32 and 16 dims have 255 and 238 registers a thread; 64 dims have one block of
  // sixteen warps with 128 and keep 492 bytes of them in local memory (512 heads of 64 nodes: 276 us).
  static constexpr bool LARGE = NT == 8 && sizeof(T) == 4;
  static constexpr int BLOCKS = (D == 64 ? 2 : 4) / (LARGE ? 2 : 1);
  static constexpr int KG = D == 16 || (D == 64 && LARGE) ? 4 : 2;
  static constexpr int RI = 8 / KG;
  static constexpr int WARPS = CG * KG;
  static constexpr int THREADS = 32 * WARPS;
  static constexpr int LDS = D + 4, C4 = LDS / 4;
  static constexpr int LQ = D + 8;                     // rows of pieces: fragments without bank conflicts
  static constexpr int UNIT = 64 * LDS;                // floats
  static constexpr int QP = Pieces<T>::Q, SP = Pieces<T>::S;
  static constexpr bool HOLD = 2 * NT * QP <= 16;      // a step's fragments of x stay in registers
  // Shared memory in bytes: slots for units of the state, then what stays for the whole head.  The keys, values, weights and sums of the tree lie
  // in the last slots until the accumulators start from them, the warps' sums in the first ones at the end.
  static constexpr int PIECES = QP * N * LQ * 2;
  static constexpr int SCALES = D * N * 4;
  static constexpr int ROWS = N * LDS * 4;
  static constexpr int TREE = PIECES + 2 * ROWS + N * N * 4;
  static constexpr int SUMS = KG * ROWS;
  static constexpr int FIXED = PIECES + SCALES + N * 8 + 144;
  static constexpr int SLOT = (D == 64 ? D + 1 : 64) * LDS * 4;   // a unit, or the linear rows
  static constexpr int ROOM = (BLOCKS == 4 ? 55 : BLOCKS == 2 ? 113 : 227) * 1024 - FIXED;
  static constexpr int SLOTS = ROOM / SLOT > 6 ? 6 : ROOM / SLOT;
  static constexpr int REGION = SLOTS * SLOT > TREE ? (SLOTS * SLOT > SUMS ? SLOTS * SLOT : SUMS) : (TREE > SUMS ? TREE : SUMS);
  static constexpr int EARLY = (REGION - TREE) / SLOT > SLOTS ? SLOTS : (REGION - TREE) / SLOT;   // slots that are free from the start
  static constexpr int BYTES = REGION + FIXED;
  static_assert(BYTES <= 227 * 1024);
  static_assert(SLOTS >= 3);
};

template <typename T, int D, int NT>
__global__ void __launch_bounds__(TreeGeo<T, D, NT>::THREADS, TreeGeo<T, D, NT>::BLOCKS)
attention_kernel(const TreeParams P) {
  using G = TreeGeo<T, D, NT>;
  constexpr int N = G::N, LDS = G::LDS, LQ = G::LQ, QP = G::QP, SP = G::SP, NB = G::NB, KG = G::KG, RI = G::RI, SLOTS = G::SLOTS, THREADS = G::THREADS;
  extern __shared__ __align__(128) unsigned char smem[];
  float* part = reinterpret_cast<float*>(smem);                                     // [KG][N][LDS], at the end in the slots' place
  float* sT = reinterpret_cast<float*>(smem + G::REGION - G::TREE);                 // [N][LDS], in the last slots' place: the tree's own sums
  float* sV = sT + N * LDS;                                                         // [N][LDS]
  float* sW = sV + N * LDS;                                                         // [N][N]: f of the nodes' pairs
  __nv_bfloat16* sK = reinterpret_cast<__nv_bfloat16*>(sW + N * N);                 // [QP][N][LQ]: pieces of the keys
  __nv_bfloat16* sQ = reinterpret_cast<__nv_bfloat16*>(smem + G::REGION);           // [QP][N][LQ]: pieces of x
  float* sX = reinterpret_cast<float*>(smem + G::REGION + G::PIECES);               // [D][N]: x times the weight of the pairs, transposed
  unsigned long long* sA = reinterpret_cast<unsigned long long*>(sX + D * N);       // [N]: ancestors
  uint64_t* full = reinterpret_cast<uint64_t*>(sA + N);                             // [SLOTS]: a slot's copy has arrived
  int* through = reinterpret_cast<int*>(full + 8);                                  // [SLOTS]: warps that are done with it
  volatile int* issued = reinterpret_cast<volatile int*>(through + 8);              // [SLOTS]: copies that were asked for
  volatile int* abort_flag = issued + 8;

  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = (int)cluster.block_rank(), CL = (int)gridDim.x;
  const int head = blockIdx.y, b = head / P.heads;
  const int npairs = P.order == 2 ? Geo<D>::NPAIRS : 0;
  if (tid == 0) {
    for (int i = 0; i < SLOTS; ++i) mbar_init(&full[i], 1), through[i] = 0, issued[i] = 0;
    *abort_flag = 0;
    fence_mbar_init();
  }
  const float c1 = P.a1 * P.inv_t, c2 = P.a2 * P.inv_t * P.inv_t;
  auto meet = [&]() {
    if (CL > 1) cluster.sync();
    else __syncthreads();
  };
  grid_wait();
  grid_trigger();
  // Queries, keys and values of all rows that the tensors have (the caller sees to it that they are readable) are asked for at once, before it
  // is known which of them count: what comes behind the copies of the state waits for those.
  constexpr int ITEMS = (N * (D / 4) + THREADS - 1) / THREADS;
  Raw4<T> rq[ITEMS], rk[ITEMS], rv[ITEMS];
  {
    const T* q = head_base<T>(P.q, head, P.heads);
    const T* k = head_base<T>(P.k, head, P.heads);
    const T* v = head_base<T>(P.v, head, P.heads);
#pragma unroll
    for (int t = 0; t < ITEMS; ++t) {
      const int idx = tid + t * THREADS, i = idx / (D / 4), c = 4 * (idx - i * (D / 4));
      if (i < P.nodes) {
        rq[t].load(q + i * P.q.sn + c, P.aligned);
        rk[t].load(k + i * P.k.sn + c, P.aligned);
        rv[t].load(v + i * P.v.sn + c, P.aligned);
      }
    }
  }
  const float* S = head_state(P, b, head - b * P.heads, D);
  const int n = P.ends == nullptr ? P.nodes : min(max(P.ends[b], 0), P.nodes);
  if (S == nullptr || n == 0) return;   // the whole cluster

  // This block's units of the state: pairs of blocks (a, b), at the end the linear rows as one.
  const int u_first = rank * (npairs + 1) / CL, u_end = (rank + 1) * (npairs + 1) / CL;
  auto load = [&](int i) {
    const int slot = i % SLOTS, u = u_first + i;
    const uint32_t bytes = (u < npairs ? 64 : D + 1) * LDS * 4;
    issued[slot] = i / SLOTS + 1;
    mbar_arrive_expect_tx(&full[slot], bytes);
    bulk_load(smem + slot * G::SLOT, S + (long long)u * G::UNIT, bytes, &full[slot]);
  };
  if (tid == 0)
    for (int i = 0; i < G::EARLY && u_first + i < u_end; ++i) load(i);
  int up[2];   // warp 0 finds out who sees whom
  if (warp == 0) load_parents(P, b, lane, up);

  // ---- x, keys, values ----------------------------------------------------------------------------------------------------------
  {
#pragma unroll
    for (int t = 0; t < ITEMS; ++t) {
      const int idx = tid + t * THREADS, i = idx / (D / 4), c = 4 * (idx - i * (D / 4));
      if (i >= N) continue;
      float x[4], y[4], z[4];
      rq[t].get(i < n, x);
      rk[t].get(i < n, y);
      rv[t].get(i < n, z);
      *reinterpret_cast<float4*>(sV + i * LDS + c) = make_float4(z[0], z[1], z[2], z[3]);
#pragma unroll
      for (int j = 0; j < 4; ++j) sX[(c + j) * N + i] = c2 * x[j];
      uint32_t p0[QP], p1[QP];
      split2(x[0], x[1], p0);
      split2(x[2], x[3], p1);
#pragma unroll
      for (int p = 0; p < QP; ++p) *reinterpret_cast<uint2*>(sQ + (p * N + i) * LQ + c) = make_uint2(p0[p], p1[p]);
      split2(y[0], y[1], p0);
      split2(y[2], y[3], p1);
#pragma unroll
      for (int p = 0; p < QP; ++p) *reinterpret_cast<uint2*>(sK + (p * N + i) * LQ + c) = make_uint2(p0[p], p1[p]);
    }
  }
  if (warp == 0) {
    unsigned long long seen[2];
    ancestors(P, n, lane, up, seen);
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (lane + 32 * k < N) sA[lane + 32 * k] = seen[k];
  }
  const int g = lane >> 2, t2 = 2 * (lane & 3);
  auto x_pieces = [&](uint32_t (&out)[QP], int nt, int m, bool doubled) {
#pragma unroll
    for (int p = 0; p < QP; ++p) {
      out[p] = *reinterpret_cast<const uint32_t*>(sQ + (p * N + 8 * nt + g) * LQ + m + t2);
      if (doubled) out[p] = twice(out[p]);   // a block off the diagonal stands for two
    }
  };
  __syncthreads();
  // ---- the tree: this block's share of the nodes ----------------------------------------------------------------------------------
  // Scores are products of keys (rows) and x (columns); each depends on its own pair alone.  The sums over the ancestors touch only what a
  // node sees, by CUDA cores: an infinity or NaN in another branch stays there.
  const int per = (n + CL - 1) / CL, i0 = min(n, rank * per), mine = min(n, i0 + per) - i0;
  {
    const int nt0 = i0 / 8, nt1 = (i0 + mine + 7) / 8, jts = (n + 15) / 16;
    for (int w = warp; w < (nt1 - nt0) * jts; w += G::WARPS) {
      const int jt = w % jts, nt = nt0 + w / jts;
      if (16 * jt > 8 * nt + 7) continue;   // nobody of them is an ancestor
      float c[4] = {};
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t a[QP][4], x[2][QP];
#pragma unroll
        for (int p = 0; p < QP; ++p)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int j = 16 * jt + g + 8 * (r & 1);   // (with one tile of eight nodes the lower rows do not exist)
            a[p][r] = j < N ? *reinterpret_cast<const uint32_t*>(sK + (p * N + j) * LQ + 16 * ks + 8 * (r >> 1) + t2) : 0u;
          }
        x_pieces(x[0], nt, 16 * ks, false);
        x_pieces(x[1], nt, 16 * ks + 8, false);
        float d[4];
        products(d, a, x);
#pragma unroll
        for (int r = 0; r < 4; ++r) c[r] += d[r];
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = 16 * jt + g + 8 * (r >> 1), i = 8 * nt + t2 + (r & 1);
        const float s = c[r] * P.inv_t;
        if (j < N) sW[i * N + j] = P.a0 + s * (P.a1 + (P.order == 2 ? P.a2 * s : 0.f));
      }
    }
  }
  __syncthreads();
  for (int idx = tid; idx < mine * (D / 4); idx += THREADS) {
    const int i = idx / (D / 4), c = 4 * (idx - i * (D / 4));
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    float total = 0.f;
    for (unsigned long long left = sA[i0 + i]; left != 0;) {
      float w[4];
      float4 y[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {   // four nodes' loads at a time
        w[t] = 0.f, y[t] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (left != 0) {
          const int j = __ffsll((long long)left) - 1;
          left &= left - 1;
          w[t] = sW[(i0 + i) * N + j];
          y[t] = *reinterpret_cast<const float4*>(sV + j * LDS + c);
        }
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        sum.x = fmaf(w[t], y[t].x, sum.x), sum.y = fmaf(w[t], y[t].y, sum.y), sum.z = fmaf(w[t], y[t].z, sum.z), sum.w = fmaf(w[t], y[t].w, sum.w);
        total += w[t];
      }
    }
    *reinterpret_cast<float4*>(sT + i * LDS + c) = sum;
    if (c == 0) sT[i * LDS + D] = total;
  }

  // ---- the state --------------------------------------------------------------------------------------------------------------
  const int kg = warp / G::CG, column = 16 * (warp % G::CG) + 2 * g;   // this warp's rows m, this thread's two columns
  float acc[NT][4] = {}, den[NT][2] = {};
  __syncthreads();
  if (kg == 0) {   // this block's nodes start from the tree's sums
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = 8 * nt + t2 + e - i0;
        if (i < 0 || i >= mine) continue;
        const float2 x = *reinterpret_cast<const float2*>(sT + i * LDS + column);
        acc[nt][e] = x.x, acc[nt][2 + e] = x.y;
        if (warp == 0 && g == 0) den[nt][e] = sT[i * LDS + D];
      }
  }
  __syncthreads();   // nobody reads what the tree needed any more
  if (tid == 0) {
    fence_proxy_async_smem();
    for (int i = G::EARLY; i < SLOTS && u_first + i < u_end; ++i) load(i);
  }
  // pieces of two rows of two columns (of the product: rows g and g + 8)
  auto s_pieces = [&](uint32_t (&a)[SP][4], int half, const float* at) {
    const float2 x = *reinterpret_cast<const float2*>(at), y = *reinterpret_cast<const float2*>(at + LDS);
    uint32_t p[SP];
    split2(x.x, y.x, p);
#pragma unroll
    for (int k = 0; k < SP; ++k) a[k][2 * half] = p[k];
    split2(x.y, y.y, p);
#pragma unroll
    for (int k = 0; k < SP; ++k) a[k][2 * half + 1] = p[k];
  };
  auto last_pieces = [&](uint32_t (&a)[SP][4], int half, const float* at) {
    uint32_t p[SP];
    split2(at[0], at[LDS], p);
#pragma unroll
    for (int k = 0; k < SP; ++k) a[k][2 * half] = p[k];
  };
  int ua = NB, ub = NB, step = 0;
  if (u_first < npairs) pair_decode(u_first, NB, ua, ub);
  // one or two units of a block row for the tiles of eight nodes that there are: straight code for each number of them
  auto pair_step = [&](auto tiles, const float* U0, const float* U1) {
    constexpr int TILES = decltype(tiles)::value;
    const int second = 8 * (U1 != nullptr ? ub + 1 : ub);
    uint32_t held[G::HOLD ? TILES : 1][2][QP];
    auto fragments = [&](uint32_t (&x)[2][QP], int nt) {
      x_pieces(x[0], nt, 8 * ub, ub != ua);
      x_pieces(x[1], nt, second, true);
    };
    if (G::HOLD) {
#pragma unroll
      for (int nt = 0; nt < TILES; ++nt) fragments(held[G::HOLD ? nt : 0], nt);
    }
#pragma unroll
    for (int r = 0; r < RI; ++r) {
      const int at = (8 * (kg * RI + r) + t2) * LDS + column;
      uint32_t a[SP][4];
      s_pieces(a, 0, U0 + at);
      if (U1 != nullptr) {
        s_pieces(a, 1, U1 + at);
      } else {   // without a second unit its terms are zeros
#pragma unroll
        for (int k = 0; k < SP; ++k) a[k][2] = a[k][3] = 0u;
      }
      const float* scale = sX + (8 * ua + kg * RI + r) * N + t2;
#pragma unroll
      for (int nt = 0; nt < TILES; ++nt) {
        if (!G::HOLD) fragments(held[0], nt);
        const float2 xm = *reinterpret_cast<const float2*>(scale + 8 * nt);
        float c[4];
        products(c, a, held[G::HOLD ? nt : 0]);
        fma2(acc[nt][0], acc[nt][1], xm, c[0], c[1]);
        fma2(acc[nt][2], acc[nt][3], xm, c[2], c[3]);
      }
    }
    if (step % G::WARPS == warp) {   // the last column: the rows of its product are the eight m instead
      const int at = (8 * g + t2) * LDS + D;
      uint32_t a[SP][4] = {};
      last_pieces(a, 0, U0 + at);
      if (U1 != nullptr) last_pieces(a, 1, U1 + at);
      const float* scale = sX + (8 * ua + g) * N + t2;
#pragma unroll
      for (int nt = 0; nt < TILES; ++nt) {
        if (!G::HOLD) fragments(held[0], nt);
        const float2 xm = *reinterpret_cast<const float2*>(scale + 8 * nt);
        float c[4];
        products(c, a, held[G::HOLD ? nt : 0]);
        den[nt][0] = fmaf(xm.x, c[0], den[nt][0]);
        den[nt][1] = fmaf(xm.y, c[1], den[nt][1]);
      }
    }
  };
  int done = 0;   // units
  auto unit = [&](int i) -> const float* {
    wait(&full[i % SLOTS], (uint32_t)(i / SLOTS) & 1u, WAIT_SLOT, abort_flag);
    return reinterpret_cast<const float*>(smem + (i % SLOTS) * G::SLOT);
  };
  // the last warp that is done with a step asks for the units that take its slots
  auto release = [&](int i, int units) {
    if (u_first + i + SLOTS >= u_end) return;
    if (count_up(&through[i % SLOTS]) == G::WARPS - 1 && *abort_flag == 0) {
      through[i % SLOTS] = 0;   // seen by whoever finds the next copy arrived
      load(i + SLOTS);
      if (units == 2 && u_first + i + 1 + SLOTS < u_end) load(i + 1 + SLOTS);
    }
  };
  while (u_first + done < min(u_end, npairs)) {
    const bool pair = ub + 1 < NB && u_first + done + 1 < u_end;
    const float* U0 = unit(done);
    const float* U1 = pair ? unit(done + 1) : nullptr;
    const int tiles = (n + 7) / 8;
    if (NT <= 2 || tiles > 3 * NT / 4) pair_step(std::integral_constant<int, NT>{}, U0, U1);
    else if (tiles > NT / 2) pair_step(std::integral_constant<int, NT <= 2 ? NT : 3 * NT / 4>{}, U0, U1);
    else pair_step(std::integral_constant<int, NT <= 2 ? NT : NT / 2>{}, U0, U1);
    __syncwarp();
    if (lane == 0) release(done, pair ? 2 : 1);
    done += pair ? 2 : 1, ub += pair ? 2 : 1, ++step;
    if (ub >= NB) ++ua, ub = ua;
  }
  if (u_end > npairs) {
    // the linear rows, x_m S[m], 16 of them a warp, and the constant's row
    const float* U = unit(done);
    for (int ks = kg; ks < D / 16; ks += KG) {
      uint32_t a[SP][4], al[SP][4] = {};
      const float* rows = U + (16 * ks + t2) * LDS;
      s_pieces(a, 0, rows + column);
      s_pieces(a, 1, rows + 8 * LDS + column);
      if (g == 0 && warp % G::CG == 0) {   // the last column, as a product of one row
        last_pieces(al, 0, rows + D);
        last_pieces(al, 1, rows + 8 * LDS + D);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        if (8 * nt < n) {
          uint32_t x[2][QP];
          x_pieces(x[0], nt, 16 * ks, false);
          x_pieces(x[1], nt, 16 * ks + 8, false);
          float c[4];
          products(c, a, x);
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[nt][j] = fmaf(c1, c[j], acc[nt][j]);
          products(c, al, x);
          den[nt][0] = fmaf(c1, c[0], den[nt][0]);
          den[nt][1] = fmaf(c1, c[1], den[nt][1]);
        }
    }
    if (kg == KG - 1) {
      const float2 ones = *reinterpret_cast<const float2*>(U + D * LDS + column);
      const float last = g == 0 && warp % G::CG == 0 ? P.a0 * U[D * LDS + D] : 0.f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        acc[nt][0] = fmaf(P.a0, ones.x, acc[nt][0]), acc[nt][1] = fmaf(P.a0, ones.x, acc[nt][1]);
        acc[nt][2] = fmaf(P.a0, ones.y, acc[nt][2]), acc[nt][3] = fmaf(P.a0, ones.y, acc[nt][3]);
        den[nt][0] += last, den[nt][1] += last;
      }
    }
  }
  __syncthreads();   // nobody reads the state any more
  if (*abort_flag != 0) drain(full, issued, SLOTS);
  // ---- partial sums meet, the warps' and the cluster's blocks', in a fixed order ------------------------------------------------
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
    if (8 * nt < n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float* at = part + (kg * N + 8 * nt + t2 + e) * LDS;
        *reinterpret_cast<float2*>(at + column) = make_float2(acc[nt][e], acc[nt][2 + e]);
        float d = den[nt][e];
        d += __shfl_xor_sync(0xffffffffu, d, 4);
        d += __shfl_xor_sync(0xffffffffu, d, 8);
        d += __shfl_xor_sync(0xffffffffu, d, 16);
        if (g < (G::CG == 4 ? 1 : 4 / G::CG)) at[D + warp % G::CG + G::CG * g] = g == 0 ? d : 0.f;   // four parts, added up at the end
      }
    }
  meet();
  T* o = const_cast<T*>(head_base<T>(P.o, head, P.heads));
  for (int idx = tid; idx < mine * (D / 4); idx += THREADS) {
    const int i = i0 + idx / (D / 4), c = 4 * (idx % (D / 4));
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f), last = x;
    for (int r = 0; r < CL; ++r) {
      const float* sums = (CL > 1 ? cluster.map_shared_rank(part, r) : part) + i * LDS;
#pragma unroll
      for (int w = 0; w < KG; ++w) {
        const float4 y = *reinterpret_cast<const float4*>(sums + w * N * LDS + c), z = *reinterpret_cast<const float4*>(sums + w * N * LDS + D);
        x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
        last.x += z.x, last.y += z.y, last.z += z.z, last.w += z.w;
      }
    }
    const float total = (last.x + last.y) + (last.z + last.w);
    store4v(o + i * P.o.sn + c, P.aligned, x.x / total, x.y / total, x.z / total, x.w / total);
    if (c == 0 && P.g.ptr != nullptr) const_cast<float*>(head_base<float>(P.g, head, P.heads))[i * P.g.sn] = total;
  }
  if (CL > 1) cluster.sync();   // nobody's sums are read any more
}

// ---- taking a path ---------------------------------------------------------------------------------------------------------
// S[(m, n)][:] += sum over the path of k_m (k_n [v | 1]): every float of the state is read and written once.  A thread has one float4 column of four
// rows of a unit, (m .. m + 3, n), and the next unit's four in flight meanwhile; k_n v is made once for the four.  bfloat16 k and v: exact products,
// one rounding a token.  Short blocks of four units stream best: 512 heads of 64 dims, a path of 5: 101.7 us, the copy rate (6490 GB/s); from
// some ten tokens on shared-memory loads bound it: 16 tokens 127 us, 64 372 us (keys kept twice to save moves: 476).
template <int D>
struct AcceptGeo {
  static constexpr int C4 = (D + 4) / 4;
  static constexpr int THREADS = 16 * C4;              // 64 rows of a unit, four to a thread
  static constexpr int BLOCKS = D == 64 ? 3 : D == 32 ? 5 : 9;   // to an SM: two of 64 dims take 117 us for 512 heads where three take 101
  static constexpr int LV = D + 4;
  static int bytes(int nodes) { return nodes * (D + LV) * 4; }
};

template <typename T, int D>
__global__ void __launch_bounds__(AcceptGeo<D>::THREADS, AcceptGeo<D>::BLOCKS)
accept_kernel(const TreeParams P, int units_each) {
  using G = AcceptGeo<D>;
  constexpr int C4 = G::C4, LV = G::LV, NB = D / 8;
  extern __shared__ __align__(128) unsigned char smem[];
  float* sK = reinterpret_cast<float*>(smem);              // [nodes][D]: keys of the path, from the root down
  float* sV = sK + P.nodes * D;                            // [nodes][LV]: [v | 1 0 0 0]
  const int tid = threadIdx.x, head = blockIdx.y, b = head / P.heads;
  const int npairs = P.order == 2 ? Geo<D>::NPAIRS : 0;
  const int u0 = blockIdx.x * units_each, u1 = min(u0 + units_each, npairs + 1);
  grid_wait();
  grid_trigger();
  int up[2];
  if (tid < 32) load_parents(P, b, tid, up);
  const int last = P.ends[b];   // (in flight beside the parents and the table's entry)
  float* S = head_state(P, b, head - b * P.heads, D);
  if (S == nullptr || last < 0 || last >= P.nodes) return;

  const int c4 = tid % C4, rg = tid / C4;
  const int n8 = rg & 7, m8 = 4 * (rg >> 3);               // of a pair of blocks: rows (m8 .. m8 + 3, n8)
  auto row_of = [&](int u, int j) { return u < npairs ? 64 * u + 8 * (m8 + j) + n8 : 64 * npairs + rg + 16 * j; };
  auto there = [&](int u, int j) { return u < npairs || rg + 16 * j < D; };
  float4* base = reinterpret_cast<float4*>(S) + c4;
  float4 next[4];
  auto fetch = [&](int u) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (there(u, j)) next[j] = __ldcs(base + (long long)row_of(u, j) * C4);
  };
  fetch(u0);
  // the path from the root down: parents come before their children, so it is the ancestors' bits in their order
  __shared__ int nodes[FASTMAX_TREE_NODES], length;
  int n = last + 1;
  if (P.parents != nullptr) {
    if (tid < 32) {
      unsigned long long seen[2];
      ancestors(P, n, tid, up, seen);
      const unsigned long long path = __shfl_sync(0xffffffffu, last < 32 ? seen[0] : seen[1], last & 31);
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if ((path >> (tid + 32 * k)) & 1ull) nodes[__popcll(path & ((1ull << (tid + 32 * k)) - 1ull))] = tid + 32 * k;
      if (tid == 0) length = __popcll(path);
    }
    __syncthreads();
    n = length;
  }
  {
    const T* k = head_base<T>(P.k, head, P.heads);
    const T* v = head_base<T>(P.v, head, P.heads);
    for (int i = rg; i < n; i += 16) {
      const int node = P.parents != nullptr ? nodes[i] : i;
      float x[4], y[4] = {1.f, 0.f, 0.f, 0.f};
      if (c4 < D / 4) {
        Raw4<T> rk, rv;
        rk.load(k + node * P.k.sn + 4 * c4, P.aligned);
        rv.load(v + node * P.v.sn + 4 * c4, P.aligned);
        rk.get(true, x);
        rv.get(true, y);
        *reinterpret_cast<float4*>(sK + i * D + 4 * c4) = make_float4(x[0], x[1], x[2], x[3]);
      }
      *reinterpret_cast<float4*>(sV + i * LV + 4 * c4) = make_float4(y[0], y[1], y[2], y[3]);
    }
  }
  __syncthreads();
  int ua = 0, ub = 0;
  if (u0 < npairs) pair_decode(u0, NB, ua, ub);
  for (int u = u0; u < u1; ++u) {
    float4 s[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] = next[j];
    if (u + 1 < u1) fetch(u + 1);
    if (u < npairs) {
      const float* km = sK + 8 * ua + m8;
      const float* kn = sK + 8 * ub + n8;
#pragma unroll 2
      for (int i = 0; i < n; ++i) {
        const float4 m = *reinterpret_cast<const float4*>(km + i * D);
        const float4 y = *reinterpret_cast<const float4*>(sV + i * LV + 4 * c4);
        const float x = kn[i * D];
        const float4 w = make_float4(x * y.x, x * y.y, x * y.z, x * y.w);
        fma2(s[0].x, s[0].y, make_float2(m.x, m.x), w.x, w.y), fma2(s[0].z, s[0].w, make_float2(m.x, m.x), w.z, w.w);
        fma2(s[1].x, s[1].y, make_float2(m.y, m.y), w.x, w.y), fma2(s[1].z, s[1].w, make_float2(m.y, m.y), w.z, w.w);
        fma2(s[2].x, s[2].y, make_float2(m.z, m.z), w.x, w.y), fma2(s[2].z, s[2].w, make_float2(m.z, m.z), w.z, w.w);
        fma2(s[3].x, s[3].y, make_float2(m.w, m.w), w.x, w.y), fma2(s[3].z, s[3].w, make_float2(m.w, m.w), w.z, w.w);
      }
      if (++ub == NB) ub = ++ua;
    } else {
      float4 ones = make_float4(0.f, 0.f, 0.f, 0.f);   // the constant's row
      if (rg == 0) ones = __ldcs(base + (long long)(64 * npairs + D) * C4);
      for (int i = 0; i < n; ++i) {
        const float4 y = *reinterpret_cast<const float4*>(sV + i * LV + 4 * c4);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (there(u, j)) {
            const float x = sK[i * D + rg + 16 * j];
            s[j].x = fmaf(x, y.x, s[j].x), s[j].y = fmaf(x, y.y, s[j].y), s[j].z = fmaf(x, y.z, s[j].z), s[j].w = fmaf(x, y.w, s[j].w);
          }
        ones.x += y.x, ones.y += y.y, ones.z += y.z, ones.w += y.w;
      }
      if (rg == 0) __stcs(base + (long long)(64 * npairs + D) * C4, ones);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (there(u, j)) __stcs(base + (long long)row_of(u, j) * C4, s[j]);
  }
}

// Dynamic shared memory beyond 48 KB has to be allowed once per device and kernel.
template <auto Kernel>
static cudaError_t allow_bytes(int bytes) {
  static std::atomic<bool> done[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return launched(e);
  if (dev < 64 && done[dev].load(std::memory_order_relaxed)) return cudaSuccess;
  e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) done[dev].store(true, std::memory_order_relaxed);
  return launched(e);
}

template <typename T, int D, int NT>
static cudaError_t launch_attention(const TreeParams& P, int bh, cudaStream_t st) {
  using G = TreeGeo<T, D, NT>;
  cudaError_t e = allow_bytes<attention_kernel<T, D, NT>>(G::BYTES);
  if (e != cudaSuccess) return e;
  // A head is divided among blocks of a cluster as far as there are then no more than two of them for every SM, each with two units or more.  us
  // with 1 / 2 / 4 blocks a head, order 2, float32 heads of 32 dims, 5 nodes: 37 heads 9.5 / 7.8 / 6.8, 74 heads 9.4 / 8.0 / 7.9, 148 heads 9.9 / 9.3 /
  // 14.3, 288 heads 10.9 / 10.7 / 20.5, 400 heads 13.9 / 19.0 / 23.3; bf16, 25 nodes: 37 heads 10.7 / 8.9 / 8.4, 148 heads 11.2 / 10.6 / 17.9, 288
  // heads 13.1 / 13.7 / 26.5, so a third or fourth block to an SM gains nothing although there is room for them.  16 dims, 1 / 2 blocks (of two
  // units): 8 nodes, 8 heads 4.9 / 5.6, 148 heads 5.0 / 5.7; float32, 25 nodes, 8 heads 7.5 / 7.6, 148 heads 7.8 / 8.7.
  const int units = (P.order == 2 ? Geo<D>::NPAIRS : 0) + 1;
  int cl = 1;
  while (cl < 8 && 2LL * cl * bh <= (G::BLOCKS < 2 ? 1LL : 2LL) * sm_count() && 4 * cl <= units + 1) cl *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(cl, bh);
  cfg.blockDim = dim3(G::THREADS);
  cfg.dynamicSmemBytes = G::BYTES;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cl;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1] = launch_attribute_after();
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return launched(cudaLaunchKernelEx(&cfg, attention_kernel<T, D, NT>, P));
}
template <typename T, int D>
static cudaError_t launch_accept(const TreeParams& P, int bh, cudaStream_t st) {
  const int units = (P.order == 2 ? Geo<D>::NPAIRS : 0) + 1;
  // Four units a block where the launch still has some blocks for every SM, so that a unit's loads cover the one before it; fewer where
  // it would not.  us with 1 / 2 / 4 / 8 units, paths of 4 or 5: d = 64, 8 heads 4.4 / 4.4 / 5.6 / 8.3, 512 heads 126 / 106 / 101 / 106; d = 16,
  // 512 heads 5.7 / 5.4 / 6.2 / 6.2.
  int each = 4;
  while (each > 1 && (long long)((units + each - 1) / each) * bh < 4LL * sm_count()) each /= 2;
  return launch_after(accept_kernel<T, D>, dim3((unsigned)((units + each - 1) / each), (unsigned)bh), AcceptGeo<D>::THREADS, AcceptGeo<D>::bytes(P.nodes), st, P, each);
}
template <typename T, int D>
static cudaError_t launch(bool attend, const TreeParams& P, int bh, cudaStream_t st) {
  if (!attend) return launch_accept<T, D>(P, bh, st);
  return P.nodes <= 8    ? launch_attention<T, D, 1>(P, bh, st)
         : P.nodes <= 16 ? launch_attention<T, D, 2>(P, bh, st)
         : P.nodes <= 32 ? launch_attention<T, D, 4>(P, bh, st)
                         : launch_attention<T, D, 8>(P, bh, st);
}
template <typename T>
static cudaError_t launch_d(bool attend, int d, const TreeParams& P, int bh, cudaStream_t st) {
  switch (d) {
    case 16: return launch<T, 16>(attend, P, bh, st);
    case 32: return launch<T, 32>(attend, P, bh, st);
    default: return launch<T, 64>(attend, P, bh, st);
  }
}
// whether every row of a tensor can be accessed four elements at a time
static bool rows_aligned(const fastmax_tensor& t, int dtype) {
  const int size = dtype == FASTMAX_BF16 ? 2 : 4;
  return reinterpret_cast<uintptr_t>(t.ptr) % (4 * size) == 0 && t.stride_b % 4 == 0 && t.stride_h % 4 == 0 && t.stride_n % 4 == 0;
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
  P.order = pb->order;
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

int tree_status(int* out) {
  cudaError_t e = cudaMemcpyFromSymbol(out, tree::g_status, sizeof(int), 0, cudaMemcpyDeviceToHost);
  if (e != cudaSuccess) return report_cuda_error(e);
  if (*out != 0) {
    const int zero = 0;
    cudaMemcpyToSymbol(tree::g_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice);
  }
  return FASTMAX_OK;
}
int tree_wait_histogram(int* out, int n) {
  int h[256];
  cudaError_t e = cudaMemcpyFromSymbol(h, tree::g_wait_hist, sizeof(h), 0, cudaMemcpyDeviceToHost);
  if (e != cudaSuccess) return report_cuda_error(e);
  for (int i = 0; i < n && i < 256; ++i) out[i] += h[i];
  static const int zeros[256] = {0};
  cudaMemcpyToSymbol(tree::g_wait_hist, zeros, sizeof(zeros), 0, cudaMemcpyHostToDevice);
  return FASTMAX_OK;
}

}  // namespace fm

extern "C" int32_t fastmax_debug_tree_wait_selftest(void* cuda_stream) {
  using namespace fm;
  tree::wait_selftest_kernel<<<1, tree::SELFTEST_FLOATS, 0, reinterpret_cast<cudaStream_t>(cuda_stream)>>>();
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? FASTMAX_OK : report_cuda_error(e);
}

extern "C" int32_t fastmax_tree_attention(const fastmax_problem* pb, const fastmax_tree_args* a, void* cuda_stream) {
  using namespace fm;
  if (!pb || !a) return FASTMAX_ERR_INVALID_ARGUMENT;
  if (const int rc = tree::check_problem(pb)) return rc;
  if (!a->q.ptr || !a->k.ptr || !a->v.ptr || !a->o.ptr) return FASTMAX_ERR_INVALID_ARGUMENT;
  if (const int rc = check_pages(pb, a->cache)) return rc;
  tree::TreeParams P = tree::params(pb, a->cache, a->parents, a->parents_stride, a->lengths);
  P.q = tree::view(a->q), P.k = tree::view(a->k), P.v = tree::view(a->v), P.o = tree::view(a->o), P.g = tree::view(a->g);
  P.aligned = tree::rows_aligned(a->q, pb->dtype) && tree::rows_aligned(a->k, pb->dtype) && tree::rows_aligned(a->v, pb->dtype) &&
              tree::rows_aligned(a->o, pb->dtype);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  cudaError_t e;
  {
    LaunchScope ls(KK_TREE, st);
    e = pb->dtype == FASTMAX_BF16 ? tree::launch_d<__nv_bfloat16>(true, pb->d, P, pb->batch * pb->heads, st)
                                  : tree::launch_d<float>(true, pb->d, P, pb->batch * pb->heads, st);
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
  P.aligned = tree::rows_aligned(a->k, pb->dtype) && tree::rows_aligned(a->v, pb->dtype);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  cudaError_t e;
  {
    LaunchScope ls(KK_TREE_ACCEPT, st);
    e = pb->dtype == FASTMAX_BF16 ? tree::launch_d<__nv_bfloat16>(false, pb->d, P, pb->batch * pb->heads, st)
                                  : tree::launch_d<float>(false, pb->d, P, pb->batch * pb->heads, st);
  }
  return e == cudaSuccess ? FASTMAX_OK : report_cuda_error(e);
}
