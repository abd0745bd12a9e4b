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
// the kernel is built around loads in flight, not around the tensor pipe. A
// warp takes 32 keys at a time and loads K and V straight into the registers
// of mma.m16n8k16 fragments with 16-byte loads, without shared memory:
//  * S = Q K^T: the contraction index may be permuted as long as Q and K agree,
//    so lane t of a quad takes 8 consecutive values of a key (one 16-byte load
//    is two k-steps' B fragments).
//  * O += P V: the output column index may be permuted, so lane group g takes
//    D / 8 consecutive columns of the four keys its fragment needs and pairs
//    them with byte permutes. P's accumulator layout is the A fragment's.
// (tcgen05 would need 128 rows and a shared-memory stage for the same bytes.)
// K is reloaded for the warp's next keys as soon as its fragments are used,
// V likewise, so one of the two is always in flight. The key axis is split
// over CTAs until the SMs are covered; the pieces are joined by their lse in
// a second kernel, in a fixed order.
#include "sm100_ptx.cuh"
#include "cross_attn.h"

#include <cuda_fp16.h>

#include <algorithm>

namespace flodl {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kKeys = 32;               // keys per warp step and per mask word
constexpr int kMaxWords = 4096;         // mask words a CTA holds: 131072 keys of a split

struct FewParams {
  const void *q, *k, *v;
  void* out;
  float *lse2, *part_o, *part_lse;
  const uint8_t* key_pad;
  int64_t qb, qs, qh, kb, ks, kh, vb, vs, vh;
  int B, Sq, Sk, H, Hk, D, G, rows, splits;
  int causal;
  float sl2;
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

__device__ __forceinline__ uint4 ldg_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// kDP: the head size rounded up to 64 or 128; kSub: 16-key groups per step (a
// step's K and V take 64 registers either way).
template <typename T, int kDP, int kSub, int kWarps>
__global__ void __launch_bounds__(kWarps * 32) few_kernel(const __grid_constant__ FewParams p) {
  constexpr int kB32 = kDP / 32;        // 32-column blocks of a key
  constexpr int kNT = kDP / 8;          // output column tiles, and columns per lane group
  constexpr int kVL = kNT / 8;          // 16-byte loads of a value row per lane
  constexpr int kStep = 16 * kSub;
  extern __shared__ __align__(16) float smem[];  // [kWarps][16][kDP] o, [kWarps][16] m, l; words
  float* s_o = smem;
  float* s_m = s_o + kWarps * 16 * kDP;
  float* s_l = s_m + kWarps * 16;
  uint32_t* s_words = reinterpret_cast<uint32_t*>(s_l + kWarps * 16);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int unit = blockIdx.x / p.splits, split = blockIdx.x - unit * p.splits;
  const int b = unit / p.Hk, kh = unit - b * p.Hk;
  // this CTA's words (32 keys each)
  const int n_words = (p.Sk + kKeys - 1) / kKeys;
  const int w0 = (int)((int64_t)n_words * split / p.splits);
  const int w1 = (int)((int64_t)n_words * (split + 1) / p.splits);
  pdl_wait();
  pdl_trigger();

  // visible keys, a bit each (only with a mask; keys past Sk count as hidden)
  if (p.key_pad) {
    const uint8_t* kp = p.key_pad + (int64_t)b * p.Sk;
#pragma unroll 4
    for (int w = w0 + warp; w < w1; w += kWarps) {
      const int key = w * kKeys + lane;
      const uint32_t bits = __ballot_sync(0xffffffffu, key < p.Sk && __ldg(kp + key) == 0);
      if (lane == 0) s_words[w - w0] = bits;
    }
    __syncthreads();
  }
  auto bits_of = [&](int step) -> uint32_t {  // visible keys of a step, low kStep bits
    const int key = step * kStep, w = key / kKeys;
    uint32_t bits;
    if (p.key_pad)
      bits = s_words[w - w0];
    else {
      const int left = p.Sk - w * kKeys;
      bits = left >= kKeys ? 0xffffffffu : (1u << left) - 1u;
    }
    return kStep == 32 ? bits : (bits >> (key & 31)) & 0xffffu;
  };

  // query fragments: rows g and g + 8 of the tile, 8 columns per 32-column block
  uint32_t qa[kB32][2][4];
  int row_q[2];  // position of the lane's two rows
#pragma unroll
  for (int r2 = 0; r2 < 2; ++r2) {
    const int r = g + 8 * r2;
    row_q[r2] = r % p.Sq;
    const T* qr = (const T*)p.q + b * p.qb + (int64_t)row_q[r2] * p.qs +
                  (int64_t)(kh * p.G + r / p.Sq) * p.qh;
#pragma unroll
    for (int c = 0; c < kB32; ++c) {
      const int col = c * 32 + t * 8;
      const uint4 v = (r < p.rows && col < p.D) ? *reinterpret_cast<const uint4*>(qr + col)
                                                : make_uint4(0, 0, 0, 0);
      qa[c][r2][0] = v.x; qa[c][r2][1] = v.y; qa[c][r2][2] = v.z; qa[c][r2][3] = v.w;
    }
  }

  const T* kbase = (const T*)p.k + b * p.kb + kh * p.kh;
  const T* vbase = (const T*)p.v + b * p.vb + kh * p.vh;
  uint4 kr[kSub][2][kB32];   // key 8 n + g of a group, columns 32 c + 8 t ..
  uint4 vr[kSub][4][kVL];    // keys 2t, 2t+1, 2t+8, 2t+9, columns g * kNT ..
  auto load_k = [&](int step) {
#pragma unroll
    for (int s = 0; s < kSub; ++s)
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int key = step * kStep + s * 16 + n * 8 + g;
        const T* row = kbase + (int64_t)key * p.ks;
#pragma unroll
        for (int c = 0; c < kB32; ++c) {
          const int col = c * 32 + t * 8;
          kr[s][n][c] = (key < p.Sk && col < p.D) ? ldg_stream(row + col) : make_uint4(0, 0, 0, 0);
        }
      }
  };
  auto load_v = [&](int step) {
#pragma unroll
    for (int s = 0; s < kSub; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = step * kStep + s * 16 + 2 * t + (i & 1) + 8 * (i >> 1);
        const T* row = vbase + (int64_t)key * p.vs;
#pragma unroll
        for (int c = 0; c < kVL; ++c) {
          const int col = g * kNT + c * 8;
          vr[s][i][c] = (key < p.Sk && col < p.D) ? ldg_stream(row + col) : make_uint4(0, 0, 0, 0);
        }
      }
  };

  constexpr int kPerWord = kKeys / kStep;
  const int end = std::min(w1 * kPerWord, (p.Sk + kStep - 1) / kStep);
  auto visible_from = [&](int step) {
    while (step < end && bits_of(step) == 0) step += kWarps;
    return step;
  };

  float o[kNT][4];
#pragma unroll
  for (int n = 0; n < kNT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[n][i] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

  int step = visible_from(w0 * kPerWord + warp);
  if (step < end) {
    load_k(step);
    load_v(step);
  }
  while (step < end) {
    const uint32_t bits = bits_of(step);
    const int next = visible_from(step + kWarps);
    float s[kSub][2][4];
#pragma unroll
    for (int u = 0; u < kSub; ++u)
#pragma unroll
      for (int n = 0; n < 2; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) s[u][n][i] = 0.f;
#pragma unroll
        for (int c = 0; c < kB32; ++c) {
          const uint32_t a0[4] = {qa[c][0][0], qa[c][1][0], qa[c][0][1], qa[c][1][1]};
          mma16816<T>(s[u][n], a0, kr[u][n][c].x, kr[u][n][c].y);
          const uint32_t a1[4] = {qa[c][0][2], qa[c][1][2], qa[c][0][3], qa[c][1][3]};
          mma16816<T>(s[u][n], a1, kr[u][n][c].z, kr[u][n][c].w);
        }
      }
    if (next < end) load_k(next);

    // s[u][n][2 * r2 + j]: row g + 8 r2, key 16 u + 8 n + 2 t + j
    const bool all = bits == (kStep == 32 ? 0xffffffffu : 0xffffu) && !p.causal;
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int u = 0; u < kSub; ++u)
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int kk = u * 16 + n * 8 + 2 * t + (i & 1);
          float x = s[u][n][i] * p.sl2;
          if (!all && (!((bits >> kk) & 1u) || (p.causal && step * kStep + kk > row_q[i >> 1])))
            x = -INFINITY;
          s[u][n][i] = x;
          mx[i >> 1] = fmaxf(mx[i >> 1], x);
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
      l[r2] *= corr[r2];
    }
    if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][i] *= corr[i >> 1];
    }
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
      uint32_t pa[4];  // P as the A fragment (rounded to 16 bits for the product, summed in f32)
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float p0 = ex2(s[u][n][0] - base[0]), p1 = ex2(s[u][n][1] - base[0]);
        const float p2 = ex2(s[u][n][2] - base[1]), p3 = ex2(s[u][n][3] - base[1]);
        l[0] += p0 + p1;
        l[1] += p2 + p3;
        pa[2 * n] = pack<T>(p0, p1);
        pa[2 * n + 1] = pack<T>(p2, p3);
      }
      // hidden keys' values may hold anything: zero them (0 * NaN is NaN)
      if (!all) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!((bits >> (u * 16 + 2 * t + (i & 1) + 8 * (i >> 1))) & 1u))
#pragma unroll
            for (int c = 0; c < kVL; ++c) vr[u][i][c] = make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int c = 0; c < kVL; ++c) {
        const uint32_t x0[4] = {vr[u][0][c].x, vr[u][0][c].y, vr[u][0][c].z, vr[u][0][c].w};
        const uint32_t x1[4] = {vr[u][1][c].x, vr[u][1][c].y, vr[u][1][c].z, vr[u][1][c].w};
        const uint32_t x2[4] = {vr[u][2][c].x, vr[u][2][c].y, vr[u][2][c].z, vr[u][2][c].w};
        const uint32_t x3[4] = {vr[u][3][c].x, vr[u][3][c].y, vr[u][3][c].z, vr[u][3][c].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          mma16816<T>(o[c * 8 + 2 * j], pa, __byte_perm(x0[j], x1[j], 0x5410),
                      __byte_perm(x2[j], x3[j], 0x5410));
          mma16816<T>(o[c * 8 + 2 * j + 1], pa, __byte_perm(x0[j], x1[j], 0x7632),
                      __byte_perm(x2[j], x3[j], 0x7632));
        }
      }
    }
    if (next < end) load_v(next);
    step = next;
  }

  // join the warps: o[n][2 r2 + j] is row g + 8 r2, column (2 t + j) * kNT + n
#pragma unroll
  for (int r2 = 0; r2 < 2; ++r2) {
    l[r2] += __shfl_xor_sync(0xffffffffu, l[r2], 1);
    l[r2] += __shfl_xor_sync(0xffffffffu, l[r2], 2);
    const int r = g + 8 * r2;
    if (r < p.rows) {
      if (t == 0) {
        s_m[warp * 16 + r] = m[r2];
        s_l[warp * 16 + r] = l[r2];
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float* dst = s_o + (warp * 16 + r) * kDP + (2 * t + j) * kNT;
#pragma unroll
        for (int n = 0; n < kNT; n += 4)
          *reinterpret_cast<float4*>(dst + n) =
              make_float4(o[n][2 * r2 + j], o[n + 1][2 * r2 + j], o[n + 2][2 * r2 + j],
                          o[n + 3][2 * r2 + j]);
      }
    }
  }
  __syncthreads();
  const int pairs = p.D / 2;
  for (int i = threadIdx.x; i < p.rows * pairs; i += kWarps * 32) {
    const int r = i / pairs, d = 2 * (i - r * pairs);
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, s_m[w * 16 + r]);
    const float top = mm == -INFINITY ? 0.f : mm;
    float ll = 0.f, a0 = 0.f, a1 = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = ex2(s_m[w * 16 + r] - top);
      ll = fmaf(s_l[w * 16 + r], f, ll);
      const float2 v = *reinterpret_cast<const float2*>(s_o + (w * 16 + r) * kDP + d);
      a0 = fmaf(v.x, f, a0);
      a1 = fmaf(v.y, f, a1);
    }
    // no visible key: zeros. A NaN sum (NaN scores) passes through.
    const bool none = ll == 0.f;
    const float inv = none ? 0.f : 1.f / ll;
    const int h = kh * p.G + r / p.Sq, iq = r % p.Sq;
    const int64_t orow = ((int64_t)b * p.Sq + iq) * p.H + h;
    const int64_t lrow = ((int64_t)b * p.H + h) * p.Sq + iq;
    if (p.splits == 1) {
      *reinterpret_cast<uint32_t*>((T*)p.out + orow * p.D + d) = pack<T>(a0 * inv, a1 * inv);
      if (d == 0 && p.lse2) p.lse2[lrow] = none ? INFINITY : top + log2f(ll);
    } else {
      const int64_t rows_all = (int64_t)p.B * p.Sq * p.H;
      *reinterpret_cast<float2*>(p.part_o + (split * rows_all + orow) * p.D + d) =
          make_float2(a0 * inv, a1 * inv);
      if (d == 0) p.part_lse[split * rows_all + lrow] = none ? -INFINITY : top + log2f(ll);
    }
  }
}

// Joins the pieces of `splits` key ranges: a warp per query row, four columns
// per lane (D <= 128), pieces in order. Weight of a piece: 2^(lse - max lse).
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(const float* __restrict__ part_o,
                                                   const float* __restrict__ part_lse,
                                                   T* __restrict__ out, float* __restrict__ lse2,
                                                   int splits, int B, int Sq, int H, int D) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const int64_t rows = (int64_t)B * Sq * H;
  const int64_t nw = (int64_t)gridDim.x * 8;
  for (int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); row < rows; row += nw) {
    const int64_t bi = row / H;  // b * Sq + i
    const int h = (int)(row - bi * H);
    const int64_t b = bi / Sq;
    const int64_t lrow = (b * H + h) * Sq + (bi - b * Sq);
    float mm = -INFINITY;
    for (int s = lane; s < splits; s += 32) mm = fmaxf(mm, part_lse[s * rows + lrow]);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, x));
    const float base = mm == -INFINITY ? 0.f : mm;
    float w = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    const bool mine = lane * 4 < D;
#pragma unroll 8
    for (int s = 0; s < splits; ++s) {
      const float f = ex2(part_lse[s * rows + lrow] - base);
      w += f;
      if (mine) {
        const float4 v = *reinterpret_cast<const float4*>(part_o + (s * rows + row) * D + lane * 4);
        a.x = fmaf(v.x, f, a.x);
        a.y = fmaf(v.y, f, a.y);
        a.z = fmaf(v.z, f, a.z);
        a.w = fmaf(v.w, f, a.w);
      }
    }
    const bool none = w == 0.f;
    const float inv = none ? 0.f : 1.f / w;
    if (mine)
      *reinterpret_cast<uint2*>(out + row * D + lane * 4) =
          make_uint2(pack<T>(a.x * inv, a.y * inv), pack<T>(a.z * inv, a.w * inv));
    if (lane == 0 && lse2) lse2[lrow] = none ? INFINITY : base + log2f(w);
  }
}

constexpr int kWarps64 = 8, kWarps128 = 4;

size_t few_smem(int dp, int warps, int words) {
  return sizeof(float) * ((size_t)warps * 16 * dp + 2 * warps * 16) + 4ull * words;
}

template <typename K>
cudaError_t opt_in(K kernel, size_t smem) {
  return smem > 48 * 1024
             ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)
             : cudaSuccess;
}

}  // namespace

bool cross_attn_is_few(const CrossAttnArgs& a) {
  return (int64_t)a.Sq * (a.H / a.Hk) <= kCrossFewRows;
}

// Key ranges per memory head: enough CTAs for two per SM, each with four steps
// or more of keys per warp (a shorter range costs more in its join than it
// saves), and no more mask words than a CTA's shared memory holds.
int cross_attn_few_splits(const CrossAttnArgs& a) {
  const int warps = a.D <= 64 ? kWarps64 : kWarps128, step = a.D <= 64 ? 32 : 16;
  const int64_t units = (int64_t)a.B * a.Hk;
  const int64_t want = (2ll * num_sms() + units - 1) / units;
  const int64_t fit = std::max<int64_t>(1, a.Sk / (4ll * warps * step));
  const int64_t words = ((int64_t)a.Sk + kKeys - 1) / kKeys;
  const int64_t need = (words + kMaxWords - 1) / kMaxWords;
  return (int)std::max<int64_t>(need, std::min<int64_t>(want, fit));
}

cudaError_t launch_cross_attn_few(const CrossAttnArgs& a, cudaStream_t st) {
  FewParams p{};
  p.q = a.q; p.k = a.k; p.v = a.v; p.out = a.out; p.lse2 = a.lse2; p.key_pad = a.key_pad;
  p.qb = a.q_st[0]; p.qs = a.q_st[1]; p.qh = a.q_st[2];
  p.kb = a.k_st[0]; p.ks = a.k_st[1]; p.kh = a.k_st[2];
  p.vb = a.v_st[0]; p.vs = a.v_st[1]; p.vh = a.v_st[2];
  p.B = a.B; p.Sq = a.Sq; p.Sk = a.Sk; p.H = a.H; p.Hk = a.Hk; p.D = a.D;
  p.G = a.H / a.Hk;
  p.rows = p.G * a.Sq;
  p.splits = cross_attn_few_splits(a);
  p.causal = a.causal;
  p.sl2 = a.scale * kLog2e;
  if (p.splits > 1) {
    if (!a.partials) return cudaErrorInvalidValue;
    p.part_o = a.partials;
    p.part_lse = a.partials + (int64_t)p.splits * a.B * a.Sq * a.H * a.D;
  }
  const int64_t ctas = (int64_t)a.B * a.Hk * p.splits;
  if (ctas > 0x7fffffff) return cudaErrorInvalidValue;
  const int words = a.key_pad ? ((a.Sk + kKeys - 1) / kKeys + p.splits - 1) / p.splits + 1 : 0;
  const bool wide = a.D > 64;
  const int warps = wide ? kWarps128 : kWarps64;
  const size_t smem = few_smem(wide ? 128 : 64, warps, words);
  void (*k)(FewParams) = a.half ? (wide ? few_kernel<__half, 128, 1, kWarps128>
                                        : few_kernel<__half, 64, 2, kWarps64>)
                                : (wide ? few_kernel<__nv_bfloat16, 128, 1, kWarps128>
                                        : few_kernel<__nv_bfloat16, 64, 2, kWarps64>);
  cudaError_t e = opt_in(k, smem);
  if (e != cudaSuccess) return e;
  e = launch_pdl(k, dim3((unsigned)ctas), dim3(warps * 32), smem, st, p);
  if (e != cudaSuccess) return e;
  note_launch();
  return p.splits > 1 ? launch_cross_attn_join(a, p.splits, st) : cudaGetLastError();
}

cudaError_t launch_cross_attn_join(const CrossAttnArgs& a, int splits, cudaStream_t st) {
  const int64_t rows = (int64_t)a.B * a.Sq * a.H;
  const float* po = a.partials;
  const float* pl = a.partials + (int64_t)splits * rows * a.D;
  const int grid = (int)std::min<int64_t>((rows + 7) / 8, (int64_t)num_sms() * 8);
  cudaError_t e =
      a.half ? launch_pdl(join_kernel<__half>, dim3(grid), dim3(256), 0, st, po, pl, (__half*)a.out,
                          a.lse2, splits, a.B, a.Sq, a.H, a.D)
             : launch_pdl(join_kernel<__nv_bfloat16>, dim3(grid), dim3(256), 0, st, po, pl,
                          (__nv_bfloat16*)a.out, a.lse2, splits, a.B, a.Sq, a.H, a.D);
  if (e != cudaSuccess) return e;
  note_launch();
  return cudaGetLastError();
}

}  // namespace flodl
