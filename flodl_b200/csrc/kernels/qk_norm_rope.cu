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
// Split: a lane holds 8 values of a row - two 16-byte loads in f32, one in 16
// bits - so a row of D values takes L = pow2ceil(D / 8) lanes and a warp 32 / L
// rows at a time; a work unit is one token and up to kSteps such row groups,
// which keeps kSteps loads per lane in flight and reads the token's cos/sin
// once for all of them. All arithmetic is f32; y and dx are rounded once.
// Weight gradients stay in registers over a warp's units, meet in shared
// memory and leave as one row per block; a second small kernel adds the rows
// in a fixed order, so results do not depend on scheduling.
#include "sm100_ptx.cuh"
#include "kernels.h"

#include <cuda_fp16.h>

#include <algorithm>

namespace flodl {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kSteps = 4;

struct Strides {
  int64_t b, s, h;  // elements
};

struct Params {
  const void *q, *k, *dyq, *dyk;  // dy*: backward only
  void *oq, *ok;                  // y (forward) or dx (backward)
  const float *wq, *wk, *cos, *sin;
  const int64_t* pos;  // [B, S] or null: offset + s
  float* partials;     // backward: [grid, 2, D] or null
  Strides sq, sk, gq, gk, uq, uk;  // x, dy, output
  int64_t offset, table_rows;
  FastDiv per_token, seq;  // units per token, S
  uint32_t units;
  int H, Hk, D, R, lanes_log2;
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

template <typename T, bool kVec>
__device__ __forceinline__ void load8(const T* row, int part, int D, float (&v)[8]) {
  if constexpr (!kVec) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = elem<false>(part, e);
      v[e] = d < D ? as_f32(row[d]) : 0.f;
    }
  } else if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(row + part * 8);
    const float4 b = *reinterpret_cast<const float4*>(row + part * 8 + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(row + part * 8);
    unpack2<T>(a.x, v[0], v[1]);
    unpack2<T>(a.y, v[2], v[3]);
    unpack2<T>(a.z, v[4], v[5]);
    unpack2<T>(a.w, v[6], v[7]);
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

template <typename T, bool kVec, bool kBwd>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(const __grid_constant__ Params p) {
  extern __shared__ float s_dw[];  // backward with weight gradients: [kWarps][2][D]
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int L = 1 << p.lanes_log2, rows_per_step = 32 >> p.lanes_log2;
  const int part = lane & (L - 1), sub = lane >> p.lanes_log2;
  const int D = p.D, half = p.R / 2;
  const bool active = elem<kVec>(part, 0) < D;
  const int heads = p.H + p.Hk;
  const float inv_d = 1.0f / (float)D;

  float wq[8], wk[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int d = elem<kVec>(part, e);
    wq[e] = (p.wq && d < D) ? __ldg(p.wq + d) : 1.f;
    wk[e] = (p.wk && d < D) ? __ldg(p.wk + d) : 1.f;
  }
  float aq[8], ak[8];  // weight-gradient sums
#pragma unroll
  for (int e = 0; e < 8; ++e) aq[e] = ak[e] = 0.f;

  const uint32_t nwarps = gridDim.x * kWarps;
  for (uint32_t unit = blockIdx.x * kWarps + warp; unit < p.units; unit += nwarps) {
    const uint32_t token = p.per_token.div(unit);
    const int h0 = (int)(unit - token * p.per_token.d) * (kSteps * rows_per_step) + sub;
    const uint32_t b = p.seq.div(token), s = token - b * p.seq.d;

    // loads of every step first, so that they are in flight together
    float x[kSteps][8], g[kBwd ? kSteps : 1][8];
#pragma unroll
    for (int u = 0; u < kSteps; ++u) {
      const int h = h0 + u * rows_per_step;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[u][e] = 0.f;
      if constexpr (kBwd) {
#pragma unroll
        for (int e = 0; e < 8; ++e) g[u][e] = 0.f;
      }
      if (active && h < heads) {
        const bool isq = h < p.H;
        const int hh = isq ? h : h - p.H;
        const Strides& st = isq ? p.sq : p.sk;
        load8<T, kVec>((const T*)(isq ? p.q : p.k) + b * st.b + s * st.s + hh * st.h, part, D, x[u]);
        if constexpr (kBwd) {
          const Strides& gt = isq ? p.gq : p.gk;
          load8<T, kVec>((const T*)(isq ? p.dyq : p.dyk) + b * gt.b + s * gt.s + hh * gt.h, part, D,
                         g[u]);
        }
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
      const int64_t at = p.pos ? p.pos[token] : p.offset + (int64_t)s;
      const bool known = at >= 0 && at < p.table_rows;
      if (!known && lane == 0) report_error(p.err, kErrBadPosition);
      const float* cr = p.cos + at * half;
      const float* sr = p.sin + at * half;
      if (kVec && (half & 3) == 0) {
        if (part * 4 < half) {
          const float nan = __int_as_float(0x7fffffff);
          const float4 cv = known ? __ldg(reinterpret_cast<const float4*>(cr + part * 4))
                                  : make_float4(nan, nan, nan, nan);
          const float4 sv = known ? __ldg(reinterpret_cast<const float4*>(sr + part * 4))
                                  : make_float4(nan, nan, nan, nan);
          c[0] = cv.x; c[1] = cv.y; c[2] = cv.z; c[3] = cv.w;
          sn[0] = sv.x; sn[1] = sv.y; sn[2] = sv.z; sn[3] = sv.w;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = elem<kVec>(part, 2 * j) >> 1;
          if (i < half) {
            c[j] = known ? __ldg(cr + i) : __int_as_float(0x7fffffff);
            sn[j] = known ? __ldg(sr + i) : __int_as_float(0x7fffffff);
          }
        }
      }
    }

#pragma unroll
    for (int u = 0; u < kSteps; ++u) {
      const int h = h0 + u * rows_per_step;
      // uniform over the warp: the step's first row decides
      if (h - sub >= heads) break;
      const bool isq = h < p.H;
      float ss = 0.f, dot = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(x[u][e], x[u][e], ss);
      if constexpr (kBwd) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float a = g[u][2 * j], d = g[u][2 * j + 1];
          g[u][2 * j] = fmaf(a, c[j], d * sn[j]);
          g[u][2 * j + 1] = fmaf(d, c[j], -a * sn[j]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) dot = fmaf(g[u][e] * (isq ? wq[e] : wk[e]), x[u][e], dot);
      }
      for (int o = L >> 1; o > 0; o >>= 1) {
        ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if constexpr (kBwd) dot += __shfl_xor_sync(0xffffffffu, dot, o);
      }
      const float r = 1.0f / sqrtf(fmaf(ss, inv_d, p.eps));
      const bool live = active && h < heads;
      const int hh = isq ? h : h - p.H;
      float y[8];
      if constexpr (!kBwd) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float a = x[u][2 * j] * r * (isq ? wq[2 * j] : wk[2 * j]);
          const float d = x[u][2 * j + 1] * r * (isq ? wq[2 * j + 1] : wk[2 * j + 1]);
          y[2 * j] = fmaf(a, c[j], -d * sn[j]);
          y[2 * j + 1] = fmaf(a, sn[j], d * c[j]);
        }
      } else {
        const float m = dot * r * inv_d;  // mean of g w xh
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float xh = x[u][e] * r;
          const float t = g[u][e] * xh;
          if (live && isq) aq[e] += t;
          if (live && !isq) ak[e] += t;
          y[e] = r * fmaf(-xh, m, g[u][e] * (isq ? wq[e] : wk[e]));
        }
      }
      if (live) {
        const Strides& ot = isq ? p.uq : p.uk;
        store8<T, kVec>((T*)(isq ? p.oq : p.ok) + b * ot.b + s * ot.s + hh * ot.h, part, D, y);
      }
    }
  }

  if constexpr (kBwd) {
    if (p.partials == nullptr) return;
    // lanes of the same part meet by shuffles, warps in shared memory
#pragma unroll
    for (int e = 0; e < 8; ++e)
      for (int o = 16; o >= L; o >>= 1) {
        aq[e] += __shfl_xor_sync(0xffffffffu, aq[e], o);
        ak[e] += __shfl_xor_sync(0xffffffffu, ak[e], o);
      }
    if (sub == 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = elem<kVec>(part, e);
        if (d < D) {
          s_dw[(warp * 2 + 0) * D + d] = aq[e];
          s_dw[(warp * 2 + 1) * D + d] = ak[e];
        }
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * D; i += kThreads) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) t += s_dw[w * 2 * D + i];
      p.partials[(int64_t)blockIdx.x * 2 * D + i] = t;
    }
  }
}

// dw += the column sums of partials [rows, 2, D]: 32 columns per block, 8 rows
// at a time, then the 8 row sums in order.
__global__ void __launch_bounds__(kThreads) qk_norm_rope_dw_kernel(
    const float* __restrict__ partials, int rows, int D, float* __restrict__ dwq,
    float* __restrict__ dwk) {
  __shared__ float s[kWarps][32];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;
  float t = 0.f;
  if (col < 2 * D) {
#pragma unroll 8
    for (int r = warp; r < rows; r += kWarps) t += partials[(int64_t)r * 2 * D + col];
  }
  s[warp][lane] = t;
  __syncthreads();
  if (warp == 0 && col < 2 * D) {
    float a = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) a += s[w][lane];
    float* out = col < D ? dwq : dwk;
    if (out) out[col < D ? col : col - D] += a;
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T>
cudaError_t launch(const QkNormRopeArgs& a, const Params& p, bool vec, bool bwd, int grid,
                   size_t smem, cudaStream_t st) {
  void (*k)(Params) = bwd ? (vec ? qk_norm_rope_kernel<T, true, true> : qk_norm_rope_kernel<T, false, true>)
                          : (vec ? qk_norm_rope_kernel<T, true, false> : qk_norm_rope_kernel<T, false, false>);
  return launch_pdl(k, dim3(grid), dim3(kThreads), smem, st, p);
}

// Units per block are kept at kWarps or more until the grid holds this many
// blocks per SM; the backward's blocks each leave a row of weight-gradient sums.
int grid_for(int64_t units, bool bwd) {
  const int64_t b = (units + kWarps - 1) / kWarps, cap = (int64_t)num_sms() * (bwd ? 2 : 8);
  return (int)std::max<int64_t>(1, std::min(b, cap));
}

int64_t units_of(const QkNormRopeArgs& a, bool vec, int& lanes_log2, int& per_token) {
  lanes_log2 = 5;
  if (vec) {
    lanes_log2 = 0;
    while ((1 << lanes_log2) * 8 < a.D) ++lanes_log2;
  }
  const int rows = kSteps * (32 >> lanes_log2);
  per_token = (a.H + a.Hk + rows - 1) / rows;
  return (int64_t)a.B * a.S * per_token;
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

cudaError_t run(const QkNormRopeArgs& a, bool bwd, cudaStream_t st) {
  if (a.B <= 0 || a.S <= 0 || a.H <= 0 || a.Hk <= 0 || a.D <= 0 || a.D > kQkNormRopeMaxD ||
      a.R < 0 || a.R > a.D || a.R % 2 || a.dtype < 0 || a.dtype > 2)
    return cudaErrorInvalidValue;
  const bool vec = vec_ok(a, bwd);
  Params p{};
  int per_token = 1;
  const int64_t units = units_of(a, vec, p.lanes_log2, per_token);
  if (units >= kMaxFlatIndex) return cudaErrorInvalidValue;
  p.q = a.q; p.k = a.k; p.dyq = a.dyq; p.dyk = a.dyk; p.oq = a.out_q; p.ok = a.out_k;
  p.wq = a.wq; p.wk = a.wk; p.cos = a.cos; p.sin = a.sin; p.pos = a.pos;
  auto s3 = [](const int64_t (&v)[3]) { return Strides{v[0], v[1], v[2]}; };
  p.sq = s3(a.q_st); p.sk = s3(a.k_st); p.gq = s3(a.dyq_st); p.gk = s3(a.dyk_st);
  p.uq = s3(a.oq_st); p.uk = s3(a.ok_st);
  p.offset = a.offset; p.table_rows = a.table_rows;
  p.per_token = FastDiv((uint32_t)per_token);
  p.seq = FastDiv((uint32_t)a.S);
  p.units = (uint32_t)units;
  p.H = a.H; p.Hk = a.Hk; p.D = a.D; p.R = a.R; p.eps = a.eps;
  p.err = default_err_word();
  const int grid = grid_for(units, bwd);
  const bool dw = bwd && (a.dwq || a.dwk);
  if (dw) {
    if (!a.partials || a.partial_rows < grid) return cudaErrorInvalidValue;
    p.partials = a.partials;
  }
  const size_t smem = dw ? sizeof(float) * kWarps * 2 * a.D : 0;
  cudaError_t e = a.dtype == 0   ? launch<float>(a, p, vec, bwd, grid, smem, st)
                  : a.dtype == 1 ? launch<__nv_bfloat16>(a, p, vec, bwd, grid, smem, st)
                                 : launch<__half>(a, p, vec, bwd, grid, smem, st);
  if (e != cudaSuccess) return e;
  note_launch();
  if (dw) {
    e = launch_pdl(qk_norm_rope_dw_kernel, dim3((2 * a.D + 31) / 32), dim3(kThreads), 0, st,
                   (const float*)a.partials, grid, a.D, a.dwq, a.dwk);
    if (e != cudaSuccess) return e;
    note_launch();
  }
  return cudaGetLastError();
}

}  // namespace

int qk_norm_rope_partial_rows(const QkNormRopeArgs& a) {
  int l, n;
  return grid_for(units_of(a, vec_ok(a, true), l, n), true);
}
cudaError_t launch_qk_norm_rope_fwd(const QkNormRopeArgs& a, cudaStream_t st) {
  return run(a, false, st);
}
cudaError_t launch_qk_norm_rope_bwd(const QkNormRopeArgs& a, cudaStream_t st) {
  return run(a, true, st);
}

}  // namespace flodl
