// Trees of drafted tokens over cached moment states: fastmax_tree_attention and fastmax_tree_accept.
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

namespace tree {

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

__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __nv_bfloat16* p) { return __bfloat162float(*p); }

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
__device__ __forceinline__ void load4v(const __nv_bfloat16* p, bool aligned, float (&x)[4]) {
  if (aligned) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    x[0] = __uint_as_float(v.x << 16), x[1] = __uint_as_float(v.x & 0xffff0000u);
    x[2] = __uint_as_float(v.y << 16), x[3] = __uint_as_float(v.y & 0xffff0000u);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __bfloat162float(p[i]);
  }
}
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

// ---- attention ---------------------------------------------------------------------------------------------------------
// The sums over the state are matrix products in which the state is read once for all nodes of a tree.  For one feature row-group m (the
// rows x_m x_n, n in the blocks b >= a) the inner sums  sum_n S[(m, n)][c] x_n  are products with x itself, and  x_m  times them is added
// in float32: nothing but the state is split into bfloat16 pieces (and x, where it is float32).
//
// Layout of a product m16n8k16: 16 rows = columns c of the state, 8 columns = nodes, 16 terms = 8 + 8 rows n of two units (a, b), (a, b + 1).

template <typename T>
struct Pieces {   // of x and of the state; with two pieces of the state 2^-16 of each term is lost, with three of both 2^-24
  static constexpr int Q = 1, S = 2;
};
template <>
struct Pieces<float> {
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
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void copy16_async(void* smem, const void* global) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(smem)), "l"(global) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <typename T, int D, int NT>
struct TreeGeo {
  static constexpr int WARPS = NT == 8 && D > 16 ? 16 : 8;
  static constexpr int THREADS = 32 * WARPS;
  static constexpr int BLOCKS = NT == 8 ? 1 : 2;       // to an SM
  static constexpr int N = 8 * NT;                     // nodes, filled up
  static constexpr int NB = D / 8;
  static constexpr int MT = D / 16;                    // tiles of 16 state columns
  static constexpr int KG = WARPS / MT;                // groups of warps that share a tile and take turns with the rows m
  static constexpr int RI = 8 / KG;
  static constexpr int LDS = D + 4, C4 = LDS / 4;
  static constexpr int LQ = D + 8;                     // rows of x pieces: fragments without bank conflicts
  static constexpr int UNIT = 64 * LDS;                // floats
  static constexpr int QP = Pieces<T>::Q, SP = Pieces<T>::S;
  // shared memory in bytes; the slots also hold the partial sums at the end
  static constexpr int PIECES = QP * N * LQ * 2;
  static constexpr int SCALES = D * N * 4;
  static constexpr int ROWS = N * LDS * 4;
  static constexpr int WEIGHTS = N * N * 4;
  static constexpr int FIXED = PIECES + SCALES + 3 * ROWS + WEIGHTS + N * 16;
  static constexpr int SLOT = 2 * UNIT * 4;
  static constexpr int RED = KG * ROWS + WARPS * N * 4;
  static constexpr int ROOM = (BLOCKS == 2 ? 113 : 227) * 1024 - FIXED;
  static constexpr int SLOTS = ROOM / SLOT < 2 ? 2 : ROOM / SLOT > 5 ? 5 : ROOM / SLOT;
  static constexpr int BYTES = FIXED + (SLOTS * SLOT > RED ? SLOTS * SLOT : RED);
  static_assert(KG * MT == WARPS && RI * KG == 8);
};

template <typename T, int D, int NT>
__global__ void __launch_bounds__(TreeGeo<T, D, NT>::THREADS, TreeGeo<T, D, NT>::BLOCKS)
attention_kernel(const TreeParams P) {
  using G = TreeGeo<T, D, NT>;
  constexpr int N = G::N, LDS = G::LDS, C4 = G::C4, QP = G::QP, SP = G::SP, THREADS = G::THREADS, NB = G::NB;
  extern __shared__ __align__(16) unsigned char smem[];
  __nv_bfloat16* sQ = reinterpret_cast<__nv_bfloat16*>(smem);                       // [QP][N][LQ]
  float* sX = reinterpret_cast<float*>(smem + G::PIECES);                           // [D][N]: x, transposed
  float* sK = sX + D * N;                                                           // [N][LDS]
  float* sV = sK + N * LDS;                                                         // [N][LDS]: [v | 1 0 0 0]
  float* sT = sV + N * LDS;                                                         // [N][LDS]: the tree's own sums, then the results
  float* sW = sT + N * LDS;                                                         // [N][N]: f of the nodes' pairs
  unsigned long long* sA = reinterpret_cast<unsigned long long*>(sW + N * N);       // [N]: ancestors
  int* sP = reinterpret_cast<int*>(sA + N);                                         // [N]
  float* slots = reinterpret_cast<float*>(smem + G::FIXED);                         // [SLOTS][2 UNIT]

  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = (int)cluster.block_rank(), CL = (int)gridDim.x;
  const int head = blockIdx.y, b = head / P.heads, h = head - b * P.heads;
  grid_wait();
  grid_trigger();
  const float* S = head_state(P, b, h, D);
  const int n = P.ends == nullptr ? P.nodes : min(max(P.ends[b], 0), P.nodes);
  if (S == nullptr || n == 0) return;   // the whole cluster

  // ---- this block's steps: one or two units (a, b), (a, b + 1), then the linear rows -------------------------------------------
  const int npairs = P.order == 2 ? Geo<D>::NPAIRS : 0;
  const int u_first = rank * (npairs + 1) / CL, u_end = (rank + 1) * (npairs + 1) / CL;   // the linear rows are the last unit
  auto row_of = [&](int u, int& a, int& bb) {
    if (u < npairs) pair_decode(u, NB, a, bb);
    else a = bb = NB;
  };
  auto units_of = [&](int u, int bb) { return u < npairs ? min(min(2, NB - bb), min(u_end, npairs) - u) : 1; };
  int lu = u_first, la, lb;   // next step to load
  row_of(lu, la, lb);
  auto load_step = [&](int slot) {
    if (lu < u_end) {
      const int count = units_of(lu, lb);
      const int quads = (lu < npairs ? count * 64 : D + 1) * C4;
      const float4* src = reinterpret_cast<const float4*>(S) + (long long)lu * 64 * C4;
      float4* dst = reinterpret_cast<float4*>(slots + slot * 2 * G::UNIT);
      for (int i = tid; i < quads; i += THREADS) copy16_async(dst + i, src + i);
      lu += count, lb += count;
      if (lb >= NB) ++la, lb = la;
    }
    copies_commit();
  };
#pragma unroll
  for (int i = 0; i + 1 < G::SLOTS; ++i) load_step(i);

  // ---- x, keys, values --------------------------------------------------------------------------------------------------------
  {
    const T* q = head_base<T>(P.q, head, P.heads);
    const T* k = head_base<T>(P.k, head, P.heads);
    const T* v = head_base<T>(P.v, head, P.heads);
    for (int idx = tid; idx < N * (D / 4); idx += THREADS) {
      const int i = idx / (D / 4), c = 4 * (idx - i * (D / 4));
      float x[4] = {}, y[4] = {}, z[4] = {};
      if (i < n) {
        load4v(q + i * P.q.sn + c, P.aligned, x);
        load4v(k + i * P.k.sn + c, P.aligned, y);
        load4v(v + i * P.v.sn + c, P.aligned, z);
      }
      *reinterpret_cast<float4*>(sK + i * LDS + c) = make_float4(y[0], y[1], y[2], y[3]);
      *reinterpret_cast<float4*>(sV + i * LDS + c) = make_float4(z[0], z[1], z[2], z[3]);
#pragma unroll
      for (int j = 0; j < 4; ++j) sX[(c + j) * N + i] = x[j];
      uint32_t p0[QP], p1[QP];
      split2(x[0], x[1], p0);
      split2(x[2], x[3], p1);
#pragma unroll
      for (int p = 0; p < QP; ++p) *reinterpret_cast<uint2*>(sQ + (p * N + i) * G::LQ + c) = make_uint2(p0[p], p1[p]);
    }
    for (int i = tid; i < N; i += THREADS) {
      *reinterpret_cast<float4*>(sV + i * LDS + D) = make_float4(1.f, 0.f, 0.f, 0.f);
      sA[i] = P.parents == nullptr ? (2ull << i) - 1ull : 1ull << i;
      sP[i] = P.parents == nullptr || i >= n ? -1 : parent_of(P, b, i);
    }
  }
  __syncthreads();
  if (P.parents != nullptr) {   // pointers twice as far up in every round
    for (int far = 1; far < n; far *= 2) {
      unsigned long long seen = 0;
      int up = -1;
      if (tid < N && sP[tid] >= 0) seen = sA[sP[tid]], up = sP[sP[tid]];
      __syncthreads();
      if (tid < N) sA[tid] |= seen, sP[tid] = up;
      __syncthreads();
    }
  }
  // ---- the tree: this block's share of the nodes, by CUDA cores: only what a node sees is touched -----------------------------
  const int per = (n + CL - 1) / CL, i0 = min(n, rank * per), mine = min(n, i0 + per) - i0;
  const int jgroups = (n + 3) / 4;
  for (int idx = tid; idx < mine * jgroups; idx += THREADS) {
    const int j = 4 * (idx / mine), i = i0 + idx % mine;
    if (((sA[i] >> j) & 15ull) == 0) continue;
    float dot[4] = {};
#pragma unroll 4
    for (int m = 0; m < D; m += 4) {
      float x[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) x[t] = sX[(m + t) * N + i];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const float4 y = *reinterpret_cast<const float4*>(sK + (j + t) * LDS + m);
        dot[t] = fmaf(x[0], y.x, fmaf(x[1], y.y, fmaf(x[2], y.z, fmaf(x[3], y.w, dot[t]))));
      }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const float s = dot[t] * P.inv_t;
      sW[(i - i0) * N + j + t] = P.a0 + s * (P.a1 + (P.order == 2 ? P.a2 * s : 0.f));
    }
  }
  __syncthreads();
  for (int idx = tid; idx < mine * C4; idx += THREADS) {
    const int i = idx / C4, c = 4 * (idx - i * C4);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (unsigned long long left = sA[i0 + i]; left != 0; left &= left - 1) {
      const int j = __ffsll((long long)left) - 1;
      const float w = sW[i * N + j];
      const float4 y = *reinterpret_cast<const float4*>(sV + j * LDS + c);
      acc.x = fmaf(w, y.x, acc.x), acc.y = fmaf(w, y.y, acc.y), acc.z = fmaf(w, y.z, acc.z), acc.w = fmaf(w, y.w, acc.w);
    }
    *reinterpret_cast<float4*>(sT + i * LDS + c) = acc;   // read by this thread alone
  }

  // ---- the state --------------------------------------------------------------------------------------------------------------
  const int mt = warp % G::MT, kg = warp / G::MT;
  const int g = lane >> 2, t2 = 2 * (lane & 3);
  float acc[NT][4] = {}, den[NT][2] = {};
  // products of 16 terms: `a` the pieces of the state, b0 / b1 those of x
  auto products = [&](float (&c)[4], const uint32_t (&a)[SP][4], const uint32_t (&b0)[QP], const uint32_t (&b1)[QP]) {
#pragma unroll
    for (int p = QP + SP - 2; p >= 0; --p)   // the smallest first
#pragma unroll
      for (int i = 0; i < SP; ++i)
        if (p - i >= 0 && p - i < QP && p < SP) mma16816(c, a[i], b0[p - i], b1[p - i]);
  };
  auto x_pieces = [&](uint32_t (&out)[QP], int node, int m) {
#pragma unroll
    for (int p = 0; p < QP; ++p) out[p] = *reinterpret_cast<const uint32_t*>(sQ + (p * N + node) * G::LQ + m);
  };
  // pieces of rows r, r + 1 (terms 0..7 of two threads' rows) of one column
  auto s_pieces = [&](uint32_t (&a)[SP][4], int reg, const float* at, int ld) {
    uint32_t p[SP];
    split2(at[0], at[ld], p);
#pragma unroll
    for (int i = 0; i < SP; ++i) a[i][reg] = p[i];
  };

  int u = u_first, ua, ub, slot = 0, step = 0;
  row_of(u, ua, ub);
  while (u < u_end) {
    copies_wait<G::SLOTS - 2>();
    __syncthreads();   // the step has arrived; everybody is done with the slot before it
    load_step(slot == 0 ? G::SLOTS - 1 : slot - 1);
    const float* U = slots + slot * 2 * G::UNIT;
    if (u < npairs) {
      const int count = units_of(u, ub);
      // (the second unit of a step without one: zeros)
#pragma unroll
      for (int r = 0; r < G::RI; ++r) {
        const int mi = kg * G::RI + r;
        const float* row = U + (8 * mi + t2) * LDS + 16 * mt + g;
        uint32_t a[SP][4];
        s_pieces(a, 0, row, LDS);
        s_pieces(a, 1, row + 8, LDS);
        if (count == 2) {
          s_pieces(a, 2, row + G::UNIT, LDS);
          s_pieces(a, 3, row + G::UNIT + 8, LDS);
        } else {
#pragma unroll
          for (int i = 0; i < SP; ++i) a[i][2] = a[i][3] = 0u;
        }
        const float* scale = sX + (8 * ua + mi) * N + t2;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          if (8 * nt < n) {
            uint32_t b0[QP], b1[QP];
            x_pieces(b0, 8 * nt + g, 8 * ub + t2);
            x_pieces(b1, 8 * nt + g, 8 * (count == 2 ? ub + 1 : ub) + t2);
#pragma unroll
            for (int p = 0; p < QP; ++p) {
              if (ub != ua) b0[p] = twice(b0[p]);
              b1[p] = twice(b1[p]);
            }
            float c[4] = {};
            products(c, a, b0, b1);
            const float2 x = *reinterpret_cast<const float2*>(scale + 8 * nt);
            acc[nt][0] = fmaf(x.x, c[0], acc[nt][0]);
            acc[nt][1] = fmaf(x.y, c[1], acc[nt][1]);
            acc[nt][2] = fmaf(x.x, c[2], acc[nt][2]);
            acc[nt][3] = fmaf(x.y, c[3], acc[nt][3]);
          }
      }
      if (step % G::WARPS == warp) {
        // the last column: rows of the product are the eight m instead
        uint32_t a[SP][4];
        s_pieces(a, 0, U + (8 * g + t2) * LDS + D, LDS);
        if (count == 2) s_pieces(a, 2, U + G::UNIT + (8 * g + t2) * LDS + D, LDS);
#pragma unroll
        for (int i = 0; i < SP; ++i) {
          a[i][1] = a[i][3] = 0u;
          if (count != 2) a[i][2] = 0u;
        }
        const float* scale = sX + (8 * ua + g) * N + t2;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          if (8 * nt < n) {
            uint32_t b0[QP], b1[QP];
            x_pieces(b0, 8 * nt + g, 8 * ub + t2);
            x_pieces(b1, 8 * nt + g, 8 * (count == 2 ? ub + 1 : ub) + t2);
#pragma unroll
            for (int p = 0; p < QP; ++p) {
              if (ub != ua) b0[p] = twice(b0[p]);
              b1[p] = twice(b1[p]);
            }
            float c[4] = {};
            products(c, a, b0, b1);
            const float2 x = *reinterpret_cast<const float2*>(scale + 8 * nt);
            den[nt][0] = fmaf(x.x, c[0], den[nt][0]);
            den[nt][1] = fmaf(x.y, c[1], den[nt][1]);
          }
      }
      u += count, ub += count;
      if (ub >= NB) ++ua, ub = ua;
    } else {
      // the linear rows: x_m S[m] and the constant's row.  What was summed so far takes its weight.
      const float c1 = P.a1 * P.inv_t, c2 = P.a2 * P.inv_t * P.inv_t;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[nt][i] *= c2;
        den[nt][0] *= c2, den[nt][1] *= c2;
      }
      for (int ks = kg; ks < D / 16; ks += G::KG) {
        const float* row = U + (16 * ks + t2) * LDS + 16 * mt + g;
        uint32_t a[SP][4], ad[SP][4];
        s_pieces(a, 0, row, LDS);
        s_pieces(a, 1, row + 8, LDS);
        s_pieces(a, 2, row + 8 * LDS, LDS);
        s_pieces(a, 3, row + 8 * LDS + 8, LDS);
        if (mt == 0) {   // and the last column, as a product of one row
          const float* last = U + (16 * ks + t2) * LDS + D;
          s_pieces(ad, 0, last, LDS);
          s_pieces(ad, 2, last + 8 * LDS, LDS);
#pragma unroll
          for (int i = 0; i < SP; ++i) {
            ad[i][1] = ad[i][3] = 0u;
            if (g != 0) ad[i][0] = ad[i][2] = 0u;
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          if (8 * nt < n) {
            uint32_t b0[QP], b1[QP];
            x_pieces(b0, 8 * nt + g, 16 * ks + t2);
            x_pieces(b1, 8 * nt + g, 16 * ks + 8 + t2);
            float c[4] = {};
            products(c, a, b0, b1);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[nt][i] = fmaf(c1, c[i], acc[nt][i]);
            if (mt == 0) {
              float cd[4] = {};
              products(cd, ad, b0, b1);
              den[nt][0] = fmaf(c1, cd[0], den[nt][0]);
              den[nt][1] = fmaf(c1, cd[1], den[nt][1]);
            }
          }
      }
      if (kg == G::KG - 1) {
        const float* ones = U + D * LDS;
        const float s0 = P.a0 * ones[16 * mt + g], s1 = P.a0 * ones[16 * mt + g + 8], sd = mt == 0 && g == 0 ? P.a0 * ones[D] : 0.f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          acc[nt][0] += s0, acc[nt][1] += s0, acc[nt][2] += s1, acc[nt][3] += s1;
          den[nt][0] += sd, den[nt][1] += sd;
        }
      }
      u += 1;
    }
    slot = slot + 1 == G::SLOTS ? 0 : slot + 1;
    ++step;
  }
  if (u_end <= npairs) {   // the linear rows are another block's: the weight here
    const float c2 = P.a2 * P.inv_t * P.inv_t;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[nt][i] *= c2;
      den[nt][0] *= c2, den[nt][1] *= c2;
    }
  }
  copies_wait<0>();
  __syncthreads();
  // ---- partial sums meet: warps of a block, then blocks of the cluster, both in a fixed order ----------------------------------
  float* red = slots;                          // [KG][N][LDS]
  float* last = slots + G::KG * N * LDS;       // [WARPS][N]
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float* at = red + (kg * N + 8 * nt + t2) * LDS + 16 * mt + g;
    at[0] = acc[nt][0], at[LDS] = acc[nt][1], at[8] = acc[nt][2], at[LDS + 8] = acc[nt][3];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float d = den[nt][i];
      d += __shfl_xor_sync(0xffffffffu, d, 4);
      d += __shfl_xor_sync(0xffffffffu, d, 8);
      d += __shfl_xor_sync(0xffffffffu, d, 16);
      if (g == 0) last[warp * N + 8 * nt + t2 + i] = d;
    }
  }
  __syncthreads();
  for (int idx = tid; idx < n * C4; idx += THREADS) {
    const int i = idx / C4, c = 4 * (idx - i * C4);
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (c < D) {
#pragma unroll
      for (int w = 0; w < G::KG; ++w) {
        const float4 y = *reinterpret_cast<const float4*>(red + (w * N + i) * LDS + c);
        x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
      }
    } else {
#pragma unroll
      for (int w = 0; w < G::WARPS; ++w) x.x += last[w * N + i];
    }
    *reinterpret_cast<float4*>(red + i * LDS + c) = x;   // nobody else reads or writes these
  }
  cluster.sync();
  for (int idx = tid; idx < mine * C4; idx += THREADS) {
    const int i = idx / C4, c = 4 * (idx - i * C4);
    float4 x = *reinterpret_cast<const float4*>(sT + i * LDS + c);
    for (int r = 0; r < CL; ++r) {
      const float4 y = *reinterpret_cast<const float4*>(cluster.map_shared_rank(red, r) + (i0 + i) * LDS + c);
      x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
    }
    *reinterpret_cast<float4*>(sT + i * LDS + c) = x;
  }
  cluster.sync();   // (also: nobody's shared memory is read any more)
  T* o = const_cast<T*>(head_base<T>(P.o, head, P.heads));
  for (int idx = tid; idx < mine * (D / 4); idx += THREADS) {
    const int i = idx / (D / 4), c = 4 * (idx - i * (D / 4));
    const float sum = sT[i * LDS + D];
    const float4 x = *reinterpret_cast<const float4*>(sT + i * LDS + c);
    store4v(o + (i0 + i) * P.o.sn + c, P.aligned, x.x / sum, x.y / sum, x.z / sum, x.w / sum);
    if (c == 0 && P.g.ptr != nullptr) const_cast<float*>(head_base<float>(P.g, head, P.heads))[(i0 + i) * P.g.sn] = sum;
  }
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
  int cl = 1;
  while (cl < 8 && (long long)cl * bh < 4 * sm_count()) cl *= 2;
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
static cudaError_t launch(bool attend, const TreeParams& P, int bh, cudaStream_t st) {
  if (!attend) {
    const dim3 grid((unsigned)((P.rows * (D + 4) + 255) / 256), (unsigned)bh);
    return P.order == 2 ? launch_after(accept_kernel<T, D, 2>, grid, 256, 0, st, P) : launch_after(accept_kernel<T, D, 1>, grid, 256, 0, st, P);
  }
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
}  // namespace fm

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
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  cudaError_t e;
  {
    LaunchScope ls(KK_TREE_ACCEPT, st);
    e = pb->dtype == FASTMAX_BF16 ? tree::launch_d<__nv_bfloat16>(false, pb->d, P, pb->batch * pb->heads, st)
                                  : tree::launch_d<float>(false, pb->d, P, pb->batch * pb->heads, st);
  }
  return e == cudaSuccess ? FASTMAX_OK : report_cuda_error(e);
}
