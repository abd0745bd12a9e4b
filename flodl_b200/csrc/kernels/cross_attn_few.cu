// Attention of a few query rows over a memory, forward: the single-token form
// of serving (one decoder token per sequence against the projected encoder
// states), and the join of partial results that all forms share.
//
// All rows that read one memory head - Sq queries of H / Hk heads, at most 16 -
// form one tile, so a memory head's keys and values are read once:
//   s = c q . k (base 2),  m = running max,  p = 2^(s - m),
//   l = sum p,  o = sum p v,  out = o / l,  lse2 = m + log2 l.
//
// What bounds it: the bytes of K and V (1 multiply-add per byte and row), so
// the kernel is built around loads in flight. Tiles of 64 keys come by TMA from
// the strided tensors into a ring of shared-memory stages (64 KB per CTA, three
// CTAs per SM: loads in flight need no registers), four consumer warps take 16
// keys of every tile each, with a running maximum, sum and output of their own,
// and read the fragments of mma.m16n8k16 with ldmatrix: the 16 rows of that
// shape are what a serving batch's token has (tcgen05 would compute 128), and
// the tensor pipe is not the limit. (A first version loaded the fragments
// straight from global memory: 680 instructions per 16 keys, 2.5 TB/s.)
// The key axis is split over CTAs until the SMs are covered; the pieces are
// joined by their lse, in a fixed order, by a cluster of up to sixteen CTAs through
// distributed shared memory or by a second kernel. Measured (one query per head, bf16): 512
// heads x 4096 x 64 in 86.7 us, 6.2 TB/s (0.96 of a copy's rate); 384 padded heads x
// 512 x 64 in 8.4; 16 memory heads x 32768 x 128 (64 query heads) in 45.6, 5.9 TB/s; one sequence's 8 heads x 100 in 2.8, a launch. (17 to 64 rows as two to
// four groups of 16, a warp to each: 21 us at 37 rows x 4001 keys of 16 heads, where
// the 128-row tiles of tcgen05 take 13.)
#include "sm100_ptx.cuh"
#include "cross_attn.h"
#include "cross_attn_join.cuh"

#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

namespace flodl {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kKeys = 64;               // keys of a tile: two mask words
constexpr int kWarps = 4;               // consumer warps, 16 keys of a tile each
constexpr int kThreads = 32 * (kWarps + 1);
constexpr int kStageBytes = 64 * 1024;  // of all stages
constexpr int kMaxWords = 2048;         // mask words a CTA holds: 65536 keys of a split
constexpr uint64_t kWaitNs = 2000000000ull;

struct FewParams {
  const void* q;
  void *out, *out_res;
  float *lse2, *part_o, *part_lse;
  const uint8_t* key_pad;
  int64_t qb, qs, qh;
  int B, Sq, Sk, H, Hk, D, G, rows, splits;
  int causal;
  float sl2;
  uint32_t* err;
};

template <int kDP>
struct FewSmem {
  static constexpr int kTile = kKeys * kDP * 2;
  static constexpr int kStages = kStageBytes / (2 * kTile);
  uint8_t k[kStages][kTile], v[kStages][kTile];  // the warps' outputs once all are read
  float m[kWarps][16], l[kWarps][16];
  float lse[16];  // of this CTA's piece
  uint64_t full[kStages], empty[kStages];
  uint32_t abort;
  int vis_end;  // of this CTA's words
  // uint32_t words[] behind it, only with a mask
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4],
                                                        uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                                 uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T>
__device__ __forceinline__ uint32_t pack(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float lo, float hi) {
  return pack_bf16x2(lo, hi);
}
template <>
__device__ __forceinline__ uint32_t pack<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// What the rounding of a pair to 16 bits leaves off, rounded.
template <typename T>
__device__ __forceinline__ uint32_t remainder2(uint32_t packed, float a, float b);
template <>
__device__ __forceinline__ uint32_t remainder2<__nv_bfloat16>(uint32_t packed, float a, float b) {
  const float2 f = unpack_bf16x2(packed);
  return pack<__nv_bfloat16>(a - f.x, b - f.y);
}
template <>
__device__ __forceinline__ uint32_t remainder2<__half>(uint32_t packed, float a, float b) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&packed));
  return pack<__half>(a - f.x, b - f.y);
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// Byte offset of 16-byte chunk `c` of row r in a tile of kN rows: 64-column
// blocks of kN rows x 128 bytes in the TMA's 128-byte swizzle.
template <int kN>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  return (uint32_t)((c >> 3) * (kN * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

template <typename T, int kDP>
__global__ void __launch_bounds__(kThreads, 3)
    few_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
               const __grid_constant__ FewParams p) {
  using Smem = FewSmem<kDP>;
  constexpr int kStages = Smem::kStages, kSteps = kDP / 16, kBlocks = kDP / 64;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                      ~uintptr_t(1023));
  uint32_t* words = reinterpret_cast<uint32_t*>(&sm + 1);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int unit = blockIdx.x / p.splits, split = blockIdx.x - unit * p.splits;
  const int b = unit / p.Hk, kh = unit - b * p.Hk;
  const int n_tiles = (p.Sk + kKeys - 1) / kKeys;
  const int t0 = (int)((int64_t)n_tiles * split / p.splits);
  const int t1 = (int)((int64_t)n_tiles * (split + 1) / p.splits);
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], kWarps);
    }
    sm.abort = 0;
    sm.vis_end = 0;
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait();
  pdl_trigger();

  // the first tiles are on their way while the queries and the mask are read;
  // with a mask only one: the keys behind may all be hidden
  const int ahead = std::min(t1 - t0, p.key_pad ? 1 : kStages);
  auto load = [&](int i) {
    const int st = i % kStages;
    mbar_arrive_expect_tx(&sm.full[st], 2 * Smem::kTile);
#pragma unroll
    for (int c = 0; c < kBlocks; ++c) {
      tma_load_4d(sm.k[st] + c * kKeys * 128, &tm_k, &sm.full[st], c * 64, (t0 + i) * kKeys, kh, b);
      tma_load_4d(sm.v[st] + c * kKeys * 128, &tm_v, &sm.full[st], c * 64, (t0 + i) * kKeys, kh, b);
    }
  };
  if (warp == kWarps && lane == 0)
    for (int i = 0; i < ahead; ++i) load(i);

  // visible keys, a bit each (keys past Sk count as hidden), and their end
  int n_load = t1 - t0;
  if (p.key_pad) {
    const uint8_t* kp = p.key_pad + (int64_t)b * p.Sk;
    int end = 0;
#pragma unroll 4
    for (int w = warp; w < 2 * (t1 - t0); w += kWarps + 1) {
      const int key = t0 * kKeys + w * 32 + lane;
      const uint32_t bits = __ballot_sync(0xffffffffu, key < p.Sk && __ldg(kp + key) == 0);
      if (lane == 0) words[w] = bits;
      if (bits) end = w + 1;
    }
    if (lane == 0 && end) atomicMax(&sm.vis_end, end);
    __syncthreads();
    n_load = std::max(ahead, (sm.vis_end + 1) / 2);
  }

  float o[kDP / 8][4];
#pragma unroll
  for (int n = 0; n < kDP / 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[n][i] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  const int g = lane >> 2, t = lane & 3;

  if (warp == kWarps) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      int i = ahead;
      bool ok = true;
      for (; i < n_load; ++i) {
        ok = mbar_wait_bounded(&sm.empty[i % kStages], ((i / kStages) & 1) ^ 1, &sm.abort, p.err,
                               kWaitNs);
        if (!ok) break;
        load(i);
      }
      if (!ok) {  // copies in flight land (bounded) before the CTA leaves
        const uint64_t from = global_timer_ns();
        for (int j = std::max(0, i - kStages); j < i; ++j)
          while (!mbar_try_wait(&sm.full[j % kStages], (j / kStages) & 1) &&
                 global_timer_ns() - from < 100000000ull) {
          }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ consumers
    // the queries as A fragments, rows (head, position) of the group; rows past the
    // end are zero
    uint32_t qa[kSteps][4];
    int row_q[2];
#pragma unroll
    for (int r2 = 0; r2 < 2; ++r2) {
      const int r = g + 8 * r2, h = r / p.Sq;
      row_q[r2] = r - h * p.Sq;
      const uint32_t* src = reinterpret_cast<const uint32_t*>(
          (const T*)p.q + b * p.qb + (int64_t)row_q[r2] * p.qs + (int64_t)(kh * p.G + h) * p.qh);
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int half = 0; half < 2; ++half)
          qa[s][r2 + 2 * half] =
              r < p.rows && 16 * s + 8 * half < p.D ? __ldg(src + 8 * s + 4 * half + t) : 0u;
    }
    const int key0 = warp * 16;  // this warp's keys in a tile
    for (int i = 0; i < n_load; ++i) {
      const int st = i % kStages;
      const int first = (t0 + i) * kKeys + key0;  // its first key
      uint32_t bits = 0xffffu;                    // visible keys among the 16
      if (p.key_pad)
        bits = (words[2 * i + (warp >> 1)] >> ((warp & 1) * 16)) & 0xffffu;
      else if (first + 16 > p.Sk)
        bits = first < p.Sk ? (1u << (p.Sk - first)) - 1u : 0u;
      bool ok = mbar_wait_bounded(&sm.full[st], (i / kStages) & 1, &sm.abort, p.err, kWaitNs);
      if (!__all_sync(0xffffffffu, ok)) break;
      if (bits != 0) {
        const uint32_t kt = smem_u32(sm.k[st]), vt = smem_u32(sm.v[st]);
        // S = Q K^T: 8 keys per column tile
        float s[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
        for (int c = 0; c < kSteps; ++c) {
          uint32_t kf[4];
          ldsm4(kf, kt + chunk_at<kKeys>(key0 + (lane & 7) + (lane >> 4) * 8, 2 * c + ((lane >> 3) & 1)));
          mma16816<T>(s[0], qa[c], kf[0], kf[1]);
          mma16816<T>(s[1], qa[c], kf[2], kf[3]);
        }
        // s[n][2 * r2 + j]: row g + 8 r2, key 8 n + 2 t + j
        const bool all = bits == 0xffffu && !p.causal;
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[n][e] *= p.sl2;
            if (!all) {
              const int kk = n * 8 + 2 * t + (e & 1);
              if (!((bits >> kk) & 1u) || (p.causal && first + kk > row_q[e >> 1])) s[n][e] = -INFINITY;
            }
            mx[e >> 1] = fmaxf(mx[e >> 1], s[n][e]);
          }
        float corr[2], base[2];
#pragma unroll
        for (int r2 = 0; r2 < 2; ++r2) {
          mx[r2] = fmaxf(mx[r2], __shfl_xor_sync(0xffffffffu, mx[r2], 1));
          mx[r2] = fmaxf(mx[r2], __shfl_xor_sync(0xffffffffu, mx[r2], 2));
          const float mn = fmaxf(m[r2], mx[r2]);
          base[r2] = mn == -INFINITY ? 0.f : mn;
          corr[r2] = ex2(m[r2] - base[r2]);
          m[r2] = mn;
        }
        if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
          l[0] *= corr[0];
          l[1] *= corr[1];
#pragma unroll
          for (int n = 0; n < kDP / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][e] *= corr[e >> 1];
        }
        uint32_t pa[4];  // P as the A fragment, rounded to 16 bits for the product
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float p0 = ex2(s[n][0] - base[0]), p1 = ex2(s[n][1] - base[0]);
          const float p2 = ex2(s[n][2] - base[1]), p3 = ex2(s[n][3] - base[1]);
          l[0] += p0 + p1;
          l[1] += p2 + p3;
          pa[2 * n] = pack<T>(p0, p1);
          pa[2 * n + 1] = pack<T>(p2, p3);
        }
        // hidden keys' values may hold anything: zero them (0 * NaN is NaN)
        if (bits != 0xffffu && p.key_pad) {
          const int r = lane & 15;
          if (!((bits >> r) & 1u))
#pragma unroll
            for (int c = 0; c < kDP / 16; ++c)
              *reinterpret_cast<uint4*>(sm.v[st] + chunk_at<kKeys>(key0 + r, 2 * c + (lane >> 4))) =
                  make_uint4(0, 0, 0, 0);
          fence_proxy_async_shared();  // before the stage's next copy
          __syncwarp();
        }
#pragma unroll
        for (int c = 0; c < kSteps; ++c) {
          uint32_t vf[4];
          ldsm4_t(vf, vt + chunk_at<kKeys>(key0 + (lane & 7) + ((lane >> 3) & 1) * 8, 2 * c + (lane >> 4)));
          mma16816<T>(o[2 * c], pa, vf[0], vf[1]);
          mma16816<T>(o[2 * c + 1], pa, vf[2], vf[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.empty[st]);
    }
  }
  __syncthreads();  // every tile has been read: its memory takes the warps' outputs

  // join the warps: o[n][2 r2 + j] is row g + 8 r2, column 8 n + 2 t + j
  float* s_o = reinterpret_cast<float*>(sm.k);
  float* s_piece = s_o + kWarps * 16 * kDP;
  static_assert((kWarps + 1) * 16 * kDP * 4 <= kStageBytes, "outputs in the stages");
  if (warp < kWarps) {
#pragma unroll
    for (int r2 = 0; r2 < 2; ++r2) {
      l[r2] += __shfl_xor_sync(0xffffffffu, l[r2], 1);
      l[r2] += __shfl_xor_sync(0xffffffffu, l[r2], 2);
      const int r = g + 8 * r2;
      if (r < p.rows) {
        if (t == 0) {
          sm.m[warp][r] = m[r2];
          sm.l[warp][r] = l[r2];
        }
#pragma unroll
        for (int n = 0; n < kDP / 8; ++n)
          *reinterpret_cast<float2*>(s_o + (warp * 16 + r) * kDP + n * 8 + 2 * t) =
              make_float2(o[n][2 * r2], o[n][2 * r2 + 1]);
      }
    }
  }
  __syncthreads();
  const int64_t rows_all = (int64_t)p.B * p.Sq * p.H;
  auto orow_of = [&](int r) {
    return ((int64_t)b * p.Sq + r % p.Sq) * p.H + kh * p.G + r / p.Sq;
  };
  auto lrow_of = [&](int r) {
    return ((int64_t)b * p.H + kh * p.G + r / p.Sq) * p.Sq + r % p.Sq;
  };
  const int pairs = p.D / 2;
  for (int i = threadIdx.x; i < p.rows * pairs; i += kThreads) {
    const int r = i / pairs, d = 2 * (i - r * pairs);
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, sm.m[w][r]);
    const float top = mm == -INFINITY ? 0.f : mm;
    float ll = 0.f, a0 = 0.f, a1 = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = ex2(sm.m[w][r] - top);
      ll = fmaf(sm.l[w][r], f, ll);
      const float2 v = *reinterpret_cast<const float2*>(s_o + (w * 16 + r) * kDP + d);
      a0 = fmaf(v.x, f, a0);
      a1 = fmaf(v.y, f, a1);
    }
    // no visible key: zeros. A NaN sum (NaN scores) passes through.
    const bool none = ll == 0.f;
    const float inv = none ? 0.f : 1.f / ll;
    const int64_t orow = orow_of(r);
    if (p.splits == 1) {
      const uint32_t w = pack<T>(a0 * inv, a1 * inv);
      *reinterpret_cast<uint32_t*>((T*)p.out + orow * p.D + d) = w;
      if (p.out_res)
        *reinterpret_cast<uint32_t*>((T*)p.out_res + orow * p.D + d) =
            remainder2<T>(w, a0 * inv, a1 * inv);
      if (d == 0 && p.lse2) p.lse2[lrow_of(r)] = none ? INFINITY : top + log2f(ll);
    } else if (p.part_o == nullptr) {  // a cluster's piece, behind the warps' outputs
      *reinterpret_cast<float2*>(s_piece + piece_at<kDP>(r, d / 4) + d % 4) =
          make_float2(a0 * inv, a1 * inv);
      if (d == 0) sm.lse[r] = none ? -INFINITY : top + log2f(ll);
    } else {
      *reinterpret_cast<float2*>(p.part_o + (split * rows_all + orow) * p.D + d) =
          make_float2(a0 * inv, a1 * inv);
      if (d == 0) p.part_lse[split * rows_all + lrow_of(r)] = none ? -INFINITY : top + log2f(ll);
    }
  }
  if (p.splits > 1 && p.part_o == nullptr)
    cluster_join<kDP>(
        s_piece, sm.lse, p.rows, p.D, p.splits,
        [&](int r, int c, float4 v) {
          const int64_t at = orow_of(r) * p.D + 4 * c;
          const uint2 w = make_uint2(pack<T>(v.x, v.y), pack<T>(v.z, v.w));
          *reinterpret_cast<uint2*>((T*)p.out + at) = w;
          if (p.out_res)
            *reinterpret_cast<uint2*>((T*)p.out_res + at) =
                make_uint2(remainder2<T>(w.x, v.x, v.y), remainder2<T>(w.y, v.z, v.w));
        },
        [&](int r, float lse) {
          if (p.lse2) p.lse2[lrow_of(r)] = lse;
        });
}

// Joins the pieces of `splits` key ranges: a warp per query row, four columns
// per lane, kLanes lanes for the row (16 for D <= 64: the warp's halves take every
// other piece). Weight of a piece: 2^(lse - max lse); pieces in a fixed order.
// Bound by latency: eight pieces' values and weights are in flight at once.
template <typename T, int kLanes>
__global__ void __launch_bounds__(256) join_kernel(const float* __restrict__ part_o,
                                                   const float* __restrict__ part_lse,
                                                   T* __restrict__ out, T* __restrict__ out_res,
                                                   float* __restrict__ lse2, int splits,
                                                   uint32_t rows, uint32_t Sq, uint32_t H, int D) {
  constexpr int kHalves = 32 / kLanes, kAhead = 8;
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, half = lane / kLanes, col = lane % kLanes * 4;
  const bool mine = col < D;
  for (uint32_t row = blockIdx.x * 8 + (threadIdx.x >> 5); row < rows; row += gridDim.x * 8) {
    const uint32_t bi = row / H, b = bi / Sq;  // bi = b * Sq + i
    const uint32_t lrow = (b * H + (row - bi * H)) * Sq + (bi - b * Sq);
    float mm = -INFINITY, w = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    auto scale = [&](float f) {
      w *= f;
      a.x *= f;
      a.y *= f;
      a.z *= f;
      a.w *= f;
    };
    auto add = [&](const float4& v, float vw, float f) {
      w = fmaf(vw, f, w);
      a.x = fmaf(v.x, f, a.x);
      a.y = fmaf(v.y, f, a.y);
      a.z = fmaf(v.z, f, a.z);
      a.w = fmaf(v.w, f, a.w);
    };
    for (int s0 = half; s0 < splits; s0 += kAhead * kHalves) {
      float ls[kAhead];
      float4 v[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int s = s0 + i * kHalves;
        ls[i] = s < splits ? part_lse[(int64_t)s * rows + lrow] : -INFINITY;
        v[i] = s < splits && mine
                   ? *reinterpret_cast<const float4*>(part_o + ((int64_t)s * rows + row) * D + col)
                   : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      float top = mm;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) top = fmaxf(top, ls[i]);
      const float base = top == -INFINITY ? 0.f : top;
      scale(ex2(mm - base));
#pragma unroll
      for (int i = 0; i < kAhead; ++i) add(v[i], 1.f, ex2(ls[i] - base));
      mm = top;
    }
    if (kHalves == 2) {
      const float om = __shfl_xor_sync(0xffffffffu, mm, 16), ow = __shfl_xor_sync(0xffffffffu, w, 16);
      const float4 oa = make_float4(
          __shfl_xor_sync(0xffffffffu, a.x, 16), __shfl_xor_sync(0xffffffffu, a.y, 16),
          __shfl_xor_sync(0xffffffffu, a.z, 16), __shfl_xor_sync(0xffffffffu, a.w, 16));
      const float top = fmaxf(mm, om), base = top == -INFINITY ? 0.f : top;
      scale(ex2(mm - base));
      add(oa, ow, ex2(om - base));
      mm = top;
    }
    const bool none = w == 0.f;
    const float inv = none ? 0.f : 1.f / w;
    if (half != 0) continue;
    if (mine) {
      const int64_t at = (int64_t)row * D + col;
      const uint2 o = make_uint2(pack<T>(a.x * inv, a.y * inv), pack<T>(a.z * inv, a.w * inv));
      *reinterpret_cast<uint2*>(out + at) = o;
      if (out_res)
        *reinterpret_cast<uint2*>(out_res + at) =
            make_uint2(remainder2<T>(o.x, a.x * inv, a.y * inv), remainder2<T>(o.y, a.z * inv, a.w * inv));
    }
    if (lane == 0 && lse2) lse2[lrow] = none ? INFINITY : mm + log2f(w);
  }
}

template <typename T, int kDP>
cudaError_t run_few(const CrossAttnArgs& a, const FewParams& p, cudaStream_t st) {
  CUtensorMap mk, mv;
  if (!cross_attn_map(&mk, a.k, a.half, a.D, a.Sk, a.Hk, a.B, a.k_st, kKeys) ||
      !cross_attn_map(&mv, a.v, a.half, a.D, a.Sk, a.Hk, a.B, a.v_st, kKeys))
    return cudaErrorInvalidValue;
  const int64_t ctas = (int64_t)a.B * a.Hk * p.splits;
  if (ctas > 0x7fffffff) return cudaErrorInvalidValue;
  const int tiles = (a.Sk + kKeys - 1) / kKeys;
  const size_t words = a.key_pad ? 2 * (size_t)((tiles + p.splits - 1) / p.splits) : 0;
  static std::atomic<uint64_t> done{0};
  constexpr size_t base = sizeof(FewSmem<kDP>) + 1024;
  cudaError_t e = cross_attn_opt_in((const void*)few_kernel<T, kDP>, base + 4 * kMaxWords, done);
  if (e != cudaSuccess) return e;
  e = launch_pdl_cluster(few_kernel<T, kDP>, dim3((unsigned)ctas), dim3(kThreads),
                         p.splits > 1 && p.part_o == nullptr ? p.splits : 1, base + 4 * words, st, mk,
                         mv, p);
  if (e != cudaSuccess) return e;
  note_launch();
  return cudaSuccess;
}

template <int kDP>
int64_t few_clusters(int size) {
  static CrossFits fits{};
  return cross_attn_clusters((const void*)few_kernel<__nv_bfloat16, kDP>, kThreads,
                             sizeof(FewSmem<kDP>) + 1024 + 4 * kMaxWords, size, fits);
}

}  // namespace

bool cross_attn_is_few(const CrossAttnArgs& a) {
  return (int64_t)a.Sq * (a.H / a.Hk) <= kCrossFewRows;
}

// Key ranges per memory head: as many CTAs as fit the SMs at once (three each),
// with four tiles or more in a range (a shorter one costs more in its join than
// it saves), and no more mask words than a CTA's shared memory holds.
CrossSplits cross_attn_few_splits(const CrossAttnArgs& a) {
  const int64_t units = (int64_t)a.B * a.Hk;
  const int64_t tiles = ((int64_t)a.Sk + kKeys - 1) / kKeys;
  const int64_t want = std::min(3ll * num_sms() / units, (long long)(tiles / 4));
  const int64_t need = (2 * tiles + kMaxWords - 1) / kMaxWords;
  const int64_t least = a.key_pad ? std::max<int64_t>(1, need) : 1;
  // Between one and one and a half times the CTAs that fit, a second wave would leave
  // most SMs idle: three shorter waves instead (512 heads x 4096 x 64: 104 -> 89 us;
  // 448 x 1500 x 128: 66.5 -> 65; 512 x 1024 x 64 would go from 30 to 36).
  const int64_t places = 3ll * num_sms();
  if (units > places && 2 * units < 3 * places && tiles >= 24 && least <= 3) return {3, true};
  // as many as a cluster joins and the GPU holds at once (63 heads x 8192 x 64: 24 us
  // with five or six pieces each, 34 with seven that wait for one another, 28 joined
  // by a second kernel)
  int64_t s = std::min<int64_t>(want, kCrossCluster);
  while (s > 1 && units > (a.D > 64 ? few_clusters<128>((int)s) : few_clusters<64>((int)s))) --s;
  if (s < least || cross_attn_joins_more(units, s, kCrossCluster, want, tiles, num_sms()))
    return {(int)std::max<int64_t>(least, want), false};
  return {(int)std::max<int64_t>(1, s), s > 1};
}

cudaError_t launch_cross_attn_few(const CrossAttnArgs& a, cudaStream_t st) {
  FewParams p{};
  p.q = a.q; p.out = a.out; p.out_res = a.out_res; p.lse2 = a.lse2; p.key_pad = a.key_pad;
  p.qb = a.q_st[0]; p.qs = a.q_st[1]; p.qh = a.q_st[2];
  p.B = a.B; p.Sq = a.Sq; p.Sk = a.Sk; p.H = a.H; p.Hk = a.Hk; p.D = a.D;
  p.G = a.H / a.Hk;
  p.rows = p.G * a.Sq;
  const CrossSplits splits = cross_attn_few_splits(a);
  p.splits = splits.n;
  p.causal = a.causal;
  p.sl2 = a.scale * kLog2e;
  p.err = default_err_word();
  if (splits.joined()) {
    if (!a.partials) return cudaErrorInvalidValue;
    p.part_o = a.partials;
    p.part_lse = a.partials + (int64_t)p.splits * a.B * a.Sq * a.H * a.D;
  }
  const bool wide = a.D > 64;
  const cudaError_t e =
      a.half ? (wide ? run_few<__half, 128>(a, p, st) : run_few<__half, 64>(a, p, st))
             : (wide ? run_few<__nv_bfloat16, 128>(a, p, st) : run_few<__nv_bfloat16, 64>(a, p, st));
  if (e != cudaSuccess) return e;
  return splits.joined() ? launch_cross_attn_join(a, p.splits, st) : cudaGetLastError();
}

cudaError_t launch_cross_attn_join(const CrossAttnArgs& a, int splits, cudaStream_t st) {
  const int64_t rows = (int64_t)a.B * a.Sq * a.H;
  if (rows > 0x7fffffff) return cudaErrorInvalidValue;
  const float* po = a.partials;
  const float* pl = a.partials + (int64_t)splits * rows * a.D;
  const int grid = (int)std::min<int64_t>((rows + 7) / 8, (int64_t)num_sms() * 8);
  auto launch = [&](auto t, auto kernel) {
    using T = decltype(t);
    return launch_pdl(kernel, dim3(grid), dim3(256), 0, st, po, pl, (T*)a.out, (T*)a.out_res, a.lse2,
                      splits, (uint32_t)rows, (uint32_t)a.Sq, (uint32_t)a.H, a.D);
  };
  const bool wide = a.D > 64;
  const cudaError_t e =
      a.half ? launch(__half(), wide ? join_kernel<__half, 32> : join_kernel<__half, 16>)
             : launch(__nv_bfloat16(),
                      wide ? join_kernel<__nv_bfloat16, 32> : join_kernel<__nv_bfloat16, 16>);
  if (e != cudaSuccess) return e;
  note_launch();
  return cudaGetLastError();
}

}  // namespace flodl
