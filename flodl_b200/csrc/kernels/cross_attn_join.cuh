// Join of the pieces of a split key axis inside a thread-block cluster.
//
// The CTAs of a cluster hold one piece each of the same query rows:
//   o_p = sum_j 2^(s_j - lse_p) v_j,   lse_p = log2 sum_j 2^(s_j)
// over the piece's keys j, and the rows' result is
//   o = sum_p w_p o_p / sum_p w_p,   w_p = 2^(lse_p - max lse).
// Each CTA leaves its rows in its own shared memory and joins a share of them
// from all, so the pieces never pass through global memory and no second kernel
// waits for the first to drain (4 to 5 us): 42 heads of 128 x 1500 x 64 take 12.1 us
// forward, and 20.8 joined by a kernel of its own. The backward's pieces are summed
// likewise: dQ and dK, dV of 3 x 6 heads, 131 x 777 x 96, 13.0 and 16.1 us, 15.4 and 19.1
// by a second kernel.
#pragma once
#include "cross_attn.h"
#include "sm100_ptx.cuh"

namespace flodl {

constexpr int kAhead = 8;  // pieces in flight

// Offset (in floats) of columns 4c..4c+3 of row r: 16-byte chunks rotated by the row, so
// that rows written by a lane each do not meet in the same banks.
template <int kDP>
__device__ __forceinline__ int piece_at(int r, int c) {
  return r * kDP + ((c ^ (r & 7)) << 2);
}

// All threads of all CTAs of the cluster call it, converged, with their rows' o
// (piece_at) and lse (-inf: no visible key) written. store(r, c, value) takes
// four columns; store_lse(r, lse) +inf for a row without a visible key.
template <int kDP, typename Store, typename StoreLse>
__device__ __forceinline__ void cluster_join(const float* o, const float* lse, int rows, int D,
                                             int pieces, Store store, StoreLse store_lse) {
  __syncwarp();  // an aligned barrier
  cluster_sync_all();
  const int chunks = D / 4;
  const uint32_t o0 = smem_u32(o), lse0 = smem_u32(lse);
  for (int i = cluster_ctarank() * blockDim.x + threadIdx.x; i < rows * chunks;
       i += pieces * blockDim.x) {
    const int r = i / chunks, c = i - r * chunks;
    float top = -INFINITY, w = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int p0 = 0; p0 < pieces; p0 += kAhead) {
      float ls[kAhead];
      float4 v[kAhead];
#pragma unroll
      for (int p = 0; p < kAhead; ++p) {
        ls[p] = -INFINITY;
        v[p] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (p0 + p < pieces) {
          ls[p] = ld_cluster(lse0 + 4 * r, p0 + p);
          v[p] = ld_cluster4(o0 + 4 * piece_at<kDP>(r, c), p0 + p);
        }
      }
      const float before = top;
#pragma unroll
      for (int p = 0; p < kAhead; ++p) top = fmaxf(top, ls[p]);
      const float base = top == -INFINITY ? 0.f : top;
      const float f0 = exp2f(before - base);
      w *= f0;
      a = make_float4(a.x * f0, a.y * f0, a.z * f0, a.w * f0);
#pragma unroll
      for (int p = 0; p < kAhead; ++p) {
        const float f = exp2f(ls[p] - base);
        w += f;
        a.x = fmaf(v[p].x, f, a.x);
        a.y = fmaf(v[p].y, f, a.y);
        a.z = fmaf(v[p].z, f, a.z);
        a.w = fmaf(v[p].w, f, a.w);
      }
    }
    // no visible key: zeros. A NaN sum (NaN scores) passes through.
    const bool none = w == 0.f;
    const float inv = none ? 0.f : 1.f / w;
    store(r, c, make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv));
    if (c == 0) store_lse(r, none ? INFINITY : top + log2f(w));
  }
  __syncwarp();
  cluster_sync_all();  // no CTA leaves while others read its rows
}

// The backward's form: the plain sum of the pieces, in their order.
template <int kDP, typename Store>
__device__ __forceinline__ void cluster_sum(const float* o, int rows, int D, int pieces, Store store) {
  const int chunks = D / 4;
  const uint32_t o0 = smem_u32(o);
  for (int i = cluster_ctarank() * blockDim.x + threadIdx.x; i < rows * chunks;
       i += pieces * blockDim.x) {
    const int r = i / chunks, c = i - r * chunks;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int p0 = 0; p0 < pieces; p0 += kAhead) {
      float4 v[kAhead];
#pragma unroll
      for (int p = 0; p < kAhead; ++p)
        v[p] = p0 + p < pieces ? ld_cluster4(o0 + 4 * piece_at<kDP>(r, c), p0 + p)
                               : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int p = 0; p < kAhead; ++p)
        a = make_float4(a.x + v[p].x, a.y + v[p].y, a.z + v[p].z, a.w + v[p].w);
    }
    store(r, c, a);
  }
}

}  // namespace flodl
