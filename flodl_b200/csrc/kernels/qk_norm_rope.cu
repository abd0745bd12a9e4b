// RMS norm of every query and key head with the rotary position embedding in
// the same pass, forward and backward (memory-bound, one launch for queries
// and keys together).
//
//   y = Rot(pos) (x * r * w),   r = 1 / sqrt(mean_d x^2 + eps)   per head row
// where Rot turns the pairs (2i, 2i + 1), i < R / 2, by the angles whose cosine
// and sine stand in row pos of two f32 tables; values past R are only normed.
// Backward, with g = Rot(pos)^T dy (the rotation is orthogonal), xh = x r:
//   dx = r (g w - xh mean_d(g w xh)),   dw = sum over rows of g xh
// r is recomputed from x, which the backward reads anyway, so the forward
// stores nothing but y.
//
// What bounds it: HBM bytes (x in, y out; the backward x and dy in, dx out).
// Measured in bf16: 4 x 8192 tokens, 16 + 4 heads of 128, forward 57.8 us, 5.8 TB/s
// (0.90 of a copy's rate); 64 x 256 tokens, 8 + 8 heads of 64, forward 11.8 us, 5.7
// TB/s, backward 18.3 us, 5.5 TB/s; a token of 8 sequences 2.0 us, a launch.
// Split: a lane holds 8 values of a row - two 16-byte loads in f32, one in 16
// bits - so a row of D values takes L = pow2ceil(D / 8) lanes (4 at least) and a
// warp 32 / L rows at a time; a work unit is kSteps such row groups of one token,
// or of two where a token's heads fill no more than half of them. The unit's
// rows are loaded first and kept as loaded (4 registers a row in 16 bits) and
// its cos/sin are read once per token. A block serves either
// queries or keys, so weights, strides and weight-gradient sums are its own.
// All arithmetic is f32; y and dx are rounded once. Weight gradients stay in
// registers over a warp's units, meet in shared memory and leave as one row per
// block; a second small kernel adds the rows in a fixed order, so results do
// not depend on scheduling.
#include "sm100_ptx.cuh"
#include "kernels.h"

#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

namespace flodl {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

struct Strides {
  uint32_t b, s, h;  // elements; a tensor's span stays below 2^31 (see run)
};

struct Side {                // queries or keys
  const void *x, *dy;        // dy: backward only
  void* out;                 // y (forward) or dx (backward)
  const float* w;
  Strides sx, sg, so;        // x, dy, out
  FastDiv per_token;         // units per token
  uint32_t units;
  int heads;
};
struct Params {
  Side side[2];
  int q_blocks;              // blocks before it serve queries, the others keys
  const float *cos, *sin;
  const int64_t* pos;        // [B, S] (rows pos_stride apart) or null: offset + s
  float* partials;           // backward: [grid, D] or null
  int64_t pos_stride;
  uint32_t offset, table_rows;
  FastDiv seq;               // S
  int D, R;
  float eps;
  uint32_t* err;
};

template <typename T>
__device__ __forceinline__ void unpack2(uint32_t v, float& a, float& b);
template <>
__device__ __forceinline__ void unpack2<__nv_bfloat16>(uint32_t v, float& a, float& b) {
  const float2 f = unpack_bf16x2(v);
  a = f.x;
  b = f.y;
}
template <>
__device__ __forceinline__ void unpack2<__half>(uint32_t v, float& a, float& b) {
  const float2 f = __half22float2(*reinterpret_cast<__half2*>(&v));
  a = f.x;
  b = f.y;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  return pack_bf16x2(a, b);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float as_f32(float v) { return v; }
__device__ __forceinline__ float as_f32(__nv_bfloat16 v) { return to_f32(v); }
__device__ __forceinline__ float as_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }

// Index of a lane's value e (0..7) within its row. kVec: 8 consecutive values;
// otherwise four pairs, 64 apart, of a row that takes the whole warp (rows
// whose size, strides or address do not allow 16-byte accesses).
template <bool kVec>
__device__ __forceinline__ int elem(int part, int e) {
  return kVec ? part * 8 + e : 2 * (part + 32 * (e >> 1)) + (e & 1);
}

// A lane's 8 values of a row as they were loaded.
template <typename T, bool kVec>
struct Raw {
  T v[8];
};
template <typename T>
struct Raw<T, true> {
  uint4 v[sizeof(T) / 2];  // 8 * sizeof(T) bytes
};

template <typename T, bool kVec>
__device__ __forceinline__ void load8(const T* row, int part, int D, Raw<T, kVec>& r) {
  if constexpr (kVec) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i)
      r.v[i] = __ldg(reinterpret_cast<const uint4*>(row + part * 8) + i);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = elem<false>(part, e);
      if (d < D) r.v[e] = row[d];
    }
  }
}
// The values as four f32 pairs.
template <typename T, bool kVec>
__device__ __forceinline__ void unpack8(const Raw<T, kVec>& r, float (&v)[8]) {
  if constexpr (!kVec) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = as_f32(r.v[e]);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      v[4 * i] = __uint_as_float(r.v[i].x);
      v[4 * i + 1] = __uint_as_float(r.v[i].y);
      v[4 * i + 2] = __uint_as_float(r.v[i].z);
      v[4 * i + 3] = __uint_as_float(r.v[i].w);
    }
  } else {
    unpack2<T>(r.v[0].x, v[0], v[1]);
    unpack2<T>(r.v[0].y, v[2], v[3]);
    unpack2<T>(r.v[0].z, v[4], v[5]);
    unpack2<T>(r.v[0].w, v[6], v[7]);
  }
}

template <typename T, bool kVec>
__device__ __forceinline__ void store8(T* row, int part, int D, const float (&v)[8]) {
  if constexpr (!kVec) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = elem<false>(part, e);
      if (d < D) put(row + d, v[e]);
    }
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(row + part * 8) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(row + part * 8 + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4*>(row + part * 8) =
        make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]),
                   pack2<T>(v[6], v[7]));
  }
}

// 1 / sqrt(x): the hardware approximation (relative error 2^-22.9) and one
// Newton step, which 0 and infinity (whose product with their root is NaN) skip.
__device__ __forceinline__ float inv_sqrt(float x) {
  const float y = rsqrtf(x);
  return y > 0.f && y < INFINITY ? y * fmaf(-0.5f * x * y, y, 1.5f) : y;
}

// Two row groups per unit; blocks per SM as registers allow without spills.
// Measured on 16384 tokens of 8 + 8 heads of 64 in bf16 (forward, backward in
// us): 2 groups at 5 and 3 blocks 13.5, 23.8; 2 at 4 and 4 (one group backward)
// 13.8, 24.8; 4 groups at 4 and 2 blocks 14.3, 25.9. The forward moves 67 MB
// (0.77 of the copy rate), with 16 + 4 heads of 128 on 32768 tokens 0.90.
constexpr int kFwdSteps = 2, kBwdSteps = 2;
__host__ __device__ constexpr int ctas_per_sm(bool bwd, size_t type) {
  return (bwd ? 3 : 5) - (type == 4 ? 1 : 0);
}
// One block's rows of the queries (kSide 0) or the keys (kSide 1): the side is
// known at compile time so that its strides stay constant operands.
// kLanes: lanes per row of the vector form, 0 for the pair form (a warp per row).
template <int kSide, typename T, int kLanes, bool kBwd, int kSteps>
__device__ __forceinline__ void rows_of(const Params& p, uint32_t block, uint32_t blocks,
                                        uint64_t (&acc)[4]) {
  constexpr bool kVec = kLanes != 0;
  constexpr int L = kVec ? kLanes : 32, kRows = 32 / L;  // rows per step
  const Side& sd = p.side[kSide];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int part = lane & (L - 1), sub = lane / L;
  const int D = p.D, half = p.R / 2;
  const bool active = elem<kVec>(part, 0) < D;
  const float inv_d = 1.0f / (float)D;
  const int heads = sd.heads;

  uint64_t w2[4];  // weights as pairs
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int d = elem<kVec>(part, 2 * j);
    w2[j] = f2_pack((sd.w && d < D) ? __ldg(sd.w + d) : 1.f,
                    (sd.w && d + 1 < D) ? __ldg(sd.w + d + 1) : 1.f);
  }

  const uint32_t nwarps = blocks * kWarps;
  for (uint32_t unit = block * kWarps + warp; unit < sd.units; unit += nwarps) {
    const uint32_t token = sd.per_token.div(unit);
    const int h0 = (int)(unit - token * sd.per_token.d) * (kSteps * kRows) + sub;
    const uint32_t b = p.seq.div(token), s = token - b * p.seq.d;

    // loads of every step first, so that they are in flight together
    Raw<T, kVec> x[kSteps], g[kBwd ? kSteps : 1];
    const uint32_t xo = b * sd.sx.b + s * sd.sx.s + h0 * sd.sx.h;
#pragma unroll
    for (int u = 0; u < kSteps; ++u) {
      x[u] = Raw<T, kVec>{};
      if (active && h0 + u * kRows < heads)
        load8<T, kVec>((const T*)sd.x + (xo + u * kRows * sd.sx.h), part, D, x[u]);
    }
    if constexpr (kBwd) {
      const uint32_t go = b * sd.sg.b + s * sd.sg.s + h0 * sd.sg.h;
#pragma unroll
      for (int u = 0; u < kSteps; ++u) {
        g[u] = Raw<T, kVec>{};
        if (active && h0 + u * kRows < heads)
          load8<T, kVec>((const T*)sd.dy + (go + u * kRows * sd.sg.h), part, D, g[u]);
      }
    }
    // the token's angles: pair j of this lane (elements 2j, 2j + 1)
    float c[4], sn[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c[j] = 1.f;
      sn[j] = 0.f;
    }
    if (half > 0) {
      uint32_t at = p.offset + s;
      bool known = true;  // an offset was checked on the host
      if (p.pos) {
        const int64_t v = __ldg(p.pos + b * p.pos_stride + s);
        known = v >= 0 && v < (int64_t)p.table_rows;
        at = (uint32_t)v;
      }
      if (known) {
        const float* cr = p.cos + at * (uint32_t)half;
        const float* sr = p.sin + at * (uint32_t)half;
        if (kVec && (half & 3) == 0) {
          if (part * 4 < half) {
            const float4 cv = __ldg(reinterpret_cast<const float4*>(cr) + part);
            const float4 sv = __ldg(reinterpret_cast<const float4*>(sr) + part);
            c[0] = cv.x; c[1] = cv.y; c[2] = cv.z; c[3] = cv.w;
            sn[0] = sv.x; sn[1] = sv.y; sn[2] = sv.z; sn[3] = sv.w;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int i = elem<kVec>(part, 2 * j) >> 1;
            if (i < half) {
              c[j] = __ldg(cr + i);
              sn[j] = __ldg(sr + i);
            }
          }
        }
      } else {  // outside the tables: the rotated values become NaN
        if (lane == 0) report_error(p.err, kErrBadPosition);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if ((elem<kVec>(part, 2 * j) >> 1) < half) c[j] = sn[j] = __int_as_float(0x7fffffff);
      }
    }

    const uint32_t oo = b * sd.so.b + s * sd.so.s + h0 * sd.so.h;
#pragma unroll
    for (int u = 0; u < kSteps; ++u) {
      const int h = h0 + u * kRows;
      if (h - sub >= heads) break;  // uniform over the warp
      const bool live = active && h < heads;
      float v[8];
      unpack8<T, kVec>(x[u], v);
      uint64_t xp[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) xp[j] = f2_pack(v[2 * j], v[2 * j + 1]);
      uint64_t ss2 = f2_mul(xp[0], xp[0]);
#pragma unroll
      for (int j = 1; j < 4; ++j) ss2 = f2_fma(xp[j], xp[j], ss2);
      float ss, t;
      f2_unpack(ss2, ss, t);
      ss += t;
      float y[8];
      if constexpr (!kBwd) {
#pragma unroll
        for (int o = L >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const uint64_t r = f2_splat(inv_sqrt(fmaf(ss, inv_d, p.eps)));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float a, d;
          f2_unpack(f2_mul(f2_mul(xp[j], r), w2[j]), a, d);
          y[2 * j] = fmaf(a, c[j], -d * sn[j]);
          y[2 * j + 1] = fmaf(a, sn[j], d * c[j]);
        }
      } else {
        float gv[8];
        unpack8<T, kVec>(g[u], gv);
        uint64_t gp[4], gw[4], dot2 = f2_splat(0.f);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float a = gv[2 * j], d = gv[2 * j + 1];
          gp[j] = f2_pack(fmaf(a, c[j], d * sn[j]), fmaf(d, c[j], -a * sn[j]));
          gw[j] = f2_mul(gp[j], w2[j]);
          dot2 = f2_fma(gw[j], xp[j], dot2);
        }
        float dot;
        f2_unpack(dot2, dot, t);
        dot += t;
#pragma unroll
        for (int o = L >> 1; o > 0; o >>= 1) {
          ss += __shfl_xor_sync(0xffffffffu, ss, o);
          dot += __shfl_xor_sync(0xffffffffu, dot, o);
        }
        // a row that is not there counts nothing in the weight gradient
        const float r = live ? inv_sqrt(fmaf(ss, inv_d, p.eps)) : 0.f;
        const uint64_t r2 = f2_splat(r), m = f2_splat(-dot * r * inv_d);  // -mean of g w xh
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint64_t xh = f2_mul(xp[j], r2);
          f2_unpack(f2_mul(f2_fma(xh, m, gw[j]), r2), y[2 * j], y[2 * j + 1]);
          acc[j] = f2_fma(gp[j], xh, acc[j]);
        }
      }
      if (live) store8<T, kVec>((T*)sd.out + (oo + u * kRows * sd.so.h), part, D, y);
    }
  }
}

template <typename T, int kLanes, bool kBwd, int kSteps>
__global__ void __launch_bounds__(kThreads, kLanes ? ctas_per_sm(kBwd, sizeof(T)) : 1)
    qk_norm_rope_kernel(const __grid_constant__ Params p) {
  constexpr bool kVec = kLanes != 0;
  constexpr int L = kVec ? kLanes : 32;
  extern __shared__ float s_dw[];  // backward with weight gradients: [kWarps][D]
  pdl_wait();
  pdl_trigger();
  uint64_t acc[4];  // the weight gradients' sums, as pairs
#pragma unroll
  for (int j = 0; j < 4; ++j) acc[j] = f2_splat(0.f);
  if ((int)blockIdx.x < p.q_blocks)
    rows_of<0, T, kLanes, kBwd, kSteps>(p, blockIdx.x, p.q_blocks, acc);
  else
    rows_of<1, T, kLanes, kBwd, kSteps>(p, blockIdx.x - p.q_blocks, gridDim.x - p.q_blocks, acc);

  if constexpr (kBwd) {
    if (p.partials == nullptr) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int part = lane & (L - 1), sub = lane / L, D = p.D;
    // lanes of the same part meet by shuffles, warps in shared memory
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float v[2];
      f2_unpack(acc[j], v[0], v[1]);
#pragma unroll
      for (int o = 16; o >= L; o >>= 1) {
        v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
        v[1] += __shfl_xor_sync(0xffffffffu, v[1], o);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int d = elem<kVec>(part, 2 * j + i);
        if (sub == 0 && d < D) s_dw[warp * D + d] = v[i];
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < D; i += kThreads) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) t += s_dw[w * D + i];
      p.partials[(int64_t)blockIdx.x * D + i] = t;
    }
  }
}

// dw (+)= the column sums of the blocks' rows, queries' rows first: 32 columns of
// one weight per block, 32 rows at a time, then the 32 row sums in order.
__global__ void __launch_bounds__(1024) qk_norm_rope_dw_kernel(const float* __restrict__ partials,
                                                               int q_rows, int rows, int D,
                                                               float* __restrict__ dwq,
                                                               float* __restrict__ dwk, int add_q,
                                                               int add_k) {
  __shared__ float s[32][33];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;
  float* out = blockIdx.y == 0 ? dwq : dwk;
  const int r0 = blockIdx.y == 0 ? 0 : q_rows, r1 = blockIdx.y == 0 ? q_rows : rows;
  float t = 0.f;
  if (col < D && out) {
#pragma unroll 8
    for (int r = r0 + warp; r < r1; r += 32) t += partials[(int64_t)r * D + col];
  }
  s[warp][lane] = t;
  __syncthreads();
  // warp c adds the 32 row sums of column c
  t = s[lane][warp];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  const int mine = blockIdx.x * 32 + warp;
  if (lane == 0 && mine < D && out)
    out[mine] = (blockIdx.y == 0 ? add_q : add_k) ? out[mine] + t : t;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }


template <typename T, int kLanes>
void (*kernel_of(bool bwd))(Params) {
  return bwd ? qk_norm_rope_kernel<T, kLanes, true, kLanes ? kBwdSteps : 1>
             : qk_norm_rope_kernel<T, kLanes, false, kLanes ? kFwdSteps : 1>;
}
template <typename T>
void (*kernel_of(int lanes, bool bwd))(Params) {
  switch (lanes) {
    case 0: return kernel_of<T, 0>(bwd);
    case 4: return kernel_of<T, 4>(bwd);
    case 8: return kernel_of<T, 8>(bwd);
    case 16: return kernel_of<T, 16>(bwd);
    default: return kernel_of<T, 32>(bwd);
  }
}

struct Plan {
  int lanes, per_q, per_k, q_blocks, grid;
  int64_t units_q, units_k;
};

bool vec_ok(const QkNormRopeArgs& a, bool bwd);

// The grid is what fits the SMs at once, shared between queries and keys by
// their rows.
Plan plan_of(const QkNormRopeArgs& a, bool bwd) {
  Plan q{};
  if (vec_ok(a, bwd)) {
    q.lanes = 4;
    while (q.lanes * 8 < a.D) q.lanes *= 2;
  }
  const int rows = q.lanes ? 32 / q.lanes : 1;
  const int steps = q.lanes ? (bwd ? kBwdSteps : kFwdSteps) : 1;
  const int per = rows * steps;
  q.per_q = (a.H + per - 1) / per;
  q.per_k = (a.Hk + per - 1) / per;
  q.units_q = (int64_t)a.B * a.S * q.per_q;
  q.units_k = (int64_t)a.B * a.S * q.per_k;
  const int64_t bq = (q.units_q + kWarps - 1) / kWarps, bk = (q.units_k + kWarps - 1) / kWarps;
  const int64_t cap = (int64_t)num_sms() * (q.lanes ? ctas_per_sm(bwd, a.dtype == 0 ? 4 : 2) : 2);
  if (bq + bk <= cap) {
    q.q_blocks = (int)bq;
    q.grid = (int)(bq + bk);
  } else {
    q.q_blocks = (int)std::min(cap - 1, std::max<int64_t>(1, (cap * a.H + (a.H + a.Hk) / 2) / (a.H + a.Hk)));
    q.grid = (int)cap;
  }
  return q;
}

bool vec_ok(const QkNormRopeArgs& a, bool bwd) {
  if (a.D % 8) return false;
  const int64_t unit = a.dtype == 0 ? 4 : 8;  // elements of 16 bytes
  auto ok = [&](const void* p, const int64_t (&s)[3]) {
    return aligned16(p) && s[0] % unit == 0 && s[1] % unit == 0 && s[2] % unit == 0;
  };
  bool v = ok(a.q, a.q_st) && ok(a.k, a.k_st) && ok(a.out_q, a.oq_st) && ok(a.out_k, a.ok_st);
  if (bwd) v = v && ok(a.dyq, a.dyq_st) && ok(a.dyk, a.dyk_st);
  // the tables are read as float4 only where a row of them is a multiple of 16 bytes
  return v && (a.R % 8 != 0 || (aligned16(a.cos) && aligned16(a.sin)));
}

// Whether every tensor's span, counted in elements, fits the kernels' 32-bit
// offsets. Strides are not negative.
bool narrow(const QkNormRopeArgs& a, bool bwd) {
  auto fits = [&](const int64_t (&s)[3], int heads) {
    const int64_t n[3] = {a.B - 1, a.S - 1, heads - 1};
    int64_t span = a.D;
    for (int i = 0; i < 3; ++i) {
      if (n[i] > 0 && s[i] > kMaxFlatIndex / n[i]) return false;
      span += n[i] * s[i];
    }
    return span < kMaxFlatIndex;
  };
  return fits(a.q_st, a.H) && fits(a.k_st, a.Hk) && fits(a.oq_st, a.H) && fits(a.ok_st, a.Hk) &&
         (!bwd || (fits(a.dyq_st, a.H) && fits(a.dyk_st, a.Hk)));
}

// The same arguments for samples (or, of one sample, positions) [lo, lo + n).
QkNormRopeArgs part_of(const QkNormRopeArgs& a, bool samples, int lo, int n) {
  QkNormRopeArgs r = a;
  const int64_t bytes = a.dtype == 0 ? 4 : 2;
  const int dim = samples ? 0 : 1;
  auto move = [&](auto& ptr, const int64_t (&s)[3]) {
    if (ptr) ptr = (std::decay_t<decltype(ptr)>)((uintptr_t)ptr + (uintptr_t)(lo * s[dim] * bytes));
  };
  move(r.q, a.q_st);
  move(r.k, a.k_st);
  move(r.dyq, a.dyq_st);
  move(r.dyk, a.dyk_st);
  move(r.out_q, a.oq_st);
  move(r.out_k, a.ok_st);
  if (a.pos) r.pos = a.pos + (samples ? lo * a.pos_stride : lo);
  if (samples) {
    r.B = n;
  } else {
    r.S = n;
    if (!a.pos) r.offset = a.offset + lo;
  }
  return r;
}

cudaError_t run(const QkNormRopeArgs& a, bool bwd, cudaStream_t st) {
  if (a.B > 0 && a.S > 0 && !narrow(a, bwd) && (a.B > 1 || a.S > 1)) {
    // halves; weight gradients add up launch by launch, in order
    const bool samples = a.B > 1;
    const int n = samples ? a.B : a.S;
    const cudaError_t e = run(part_of(a, samples, 0, n / 2), bwd, st);
    if (e != cudaSuccess) return e;
    QkNormRopeArgs rest = part_of(a, samples, n / 2, n - n / 2);
    rest.dwq_add = rest.dwk_add = true;
    return run(rest, bwd, st);
  }
  if (!narrow(a, bwd) || a.table_rows * (int64_t)(a.R / 2) >= kMaxFlatIndex || a.B <= 0 ||
      a.S <= 0 || a.H <= 0 || a.Hk <= 0 || a.D <= 0 || a.D > kQkNormRopeMaxD || a.R < 0 ||
      a.R > a.D || a.R % 2 || a.dtype < 0 || a.dtype > 2)
    return cudaErrorInvalidValue;
  const Plan plan = plan_of(a, bwd);
  if (plan.units_q >= kMaxFlatIndex || plan.units_k >= kMaxFlatIndex) return cudaErrorInvalidValue;
  auto s3 = [](const int64_t (&v)[3]) {
    return Strides{(uint32_t)v[0], (uint32_t)v[1], (uint32_t)v[2]};
  };
  Params p{};
  p.side[0] = Side{a.q, a.dyq, a.out_q, a.wq, s3(a.q_st), s3(a.dyq_st), s3(a.oq_st),
                   FastDiv((uint32_t)plan.per_q), (uint32_t)plan.units_q, a.H};
  p.side[1] = Side{a.k, a.dyk, a.out_k, a.wk, s3(a.k_st), s3(a.dyk_st), s3(a.ok_st),
                   FastDiv((uint32_t)plan.per_k), (uint32_t)plan.units_k, a.Hk};
  p.q_blocks = plan.q_blocks;
  p.cos = a.cos; p.sin = a.sin; p.pos = a.pos;
  p.pos_stride = a.pos_stride;
  p.offset = (uint32_t)a.offset; p.table_rows = (uint32_t)a.table_rows;
  p.seq = FastDiv((uint32_t)a.S);
  p.D = a.D; p.R = a.R; p.eps = a.eps;
  p.err = default_err_word();
  const int grid = plan.grid;
  const bool dw = bwd && (a.dwq || a.dwk);
  if (dw) {
    if (!a.partials || a.partial_rows < grid) return cudaErrorInvalidValue;
    p.partials = a.partials;
  }
  const size_t smem = dw ? sizeof(float) * kWarps * a.D : 0;
  auto kernel = a.dtype == 0   ? kernel_of<float>(plan.lanes, bwd)
                : a.dtype == 1 ? kernel_of<__nv_bfloat16>(plan.lanes, bwd)
                               : kernel_of<__half>(plan.lanes, bwd);
  cudaError_t e = launch_pdl(kernel, dim3(grid), dim3(kThreads), smem, st, p);
  if (e != cudaSuccess) return e;
  note_launch();
  if (dw) {
    e = launch_pdl(qk_norm_rope_dw_kernel, dim3((a.D + 31) / 32, 2), dim3(1024), 0, st,
                   (const float*)a.partials, plan.q_blocks, grid, a.D, a.dwq, a.dwk,
                   (int)a.dwq_add, (int)a.dwk_add);
    if (e != cudaSuccess) return e;
    note_launch();
  }
  return cudaGetLastError();
}

}  // namespace

int qk_norm_rope_partial_rows(const QkNormRopeArgs& a) {
  return plan_of(a, true).grid;
}
cudaError_t launch_qk_norm_rope_fwd(const QkNormRopeArgs& a, cudaStream_t st) {
  return run(a, false, st);
}
cudaError_t launch_qk_norm_rope_bwd(const QkNormRopeArgs& a, cudaStream_t st) {
  return run(a, true, st);
}

}  // namespace flodl
