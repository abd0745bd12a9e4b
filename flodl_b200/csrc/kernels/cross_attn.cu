// Attention with queries, keys and values in tensors of their own, forward and
// backward, on tcgen05 tensor cores: cross attention to an encoder's states of
// another length, memory heads shared by several query heads, any strides.
// The form for a few query rows is in cross_attn_few.cu.
//
//   S = Q K^T,  P = softmax(c S + mask),  O = P V
//   backward, from the base-2 log-sum-exp and delta = rowsum(dO * O):
//   P = 2^(c log2e S - lse2),  dS = P (dO V^T - delta),
//   dQ = c dS K,  dK = c dS^T Q,  dV = P^T dO
// (in f16 dS is formed at a power of two of its value, see range_shift)
//
// Tiles come by 4-D TMA maps {D, position, head, batch} straight from the
// strided tensors: no copy for packed projections, rows past the end and
// columns past D are zero-filled (D is rounded up to 64 or 128).
//
// All three kernels have one shape: 128 rows of the stationary side lie on the
// TMEM lanes (a compute thread owns a row), tiles of the other side stream
// through shared memory, the elementwise result is written back to TMEM as
// 16-bit pairs and is the A operand of the next product, so no score touches
// shared memory. Scores of one tile are computed by the tensor cores while the
// compute warps are on another.
//   forward  rows = queries, stream K, V:  S -> P, O += P V
//   dQ       rows = queries, stream K, V:  S, dP -> dS, dQ += dS K
//   dK/dV    rows = keys, stream Q, dO:    S^T, dP^T -> P^T, dS^T, dV += P^T dO, dK += dS^T Q
// dQ has a kernel of its own, which recomputes S and dP (seven products instead
// of five), so that no gradient is summed by atomics: results do not depend on
// the order of execution. Where the items are fewer than the SMs, the streamed
// axis is split; the CTAs of an item's pieces form a cluster and add them (the
// forward's joined by lse) in order, or a second kernel does.
//
// What bounds it, and what it takes (bf16; us, TFLOP/s of the products named above; the
// library's 16-bit product reaches 1653):
//   heads x queries x keys x D    forward     for training   dQ           dK/dV
//   512 x 256 x 256 x 64          20.6 (416)  24.9 (345)     24.9 (518)   35.0 (490)
//   384 x 256 x 512 x 64          27.1 (476)  31.5 (409)     32.9 (588)   51.5 (500)
//   128 x 1024 x 1024 x 64        57 (603)    65 (531)       62 (830)     89 (771)
//   64 x 2048^2 x 128, causal     79 (873)    92 (751)       113 (914)    150 (915)
//   32 x 2048 x 8192 x 128        226 (1216)  246 (1117)     347 (1189)   560 (982)
// At head size 128 and long axes the tensor pipe is busy two thirds of the time: the
// products of a tile and its elementwise work overlap but for the tile's round trip.
// At head size 64 and a few tiles per item the round trip bounds it (scores, TMEM
// loads, maximum, exponentials, TMEM stores, product: a warp's tile takes about 2100
// cycles with another CTA's warp beside it, of which 512 are exponentials): tensor
// pipe 14 to 21% busy, exponentials 23 to 29%, instruction issue 37 to 47%, DRAM 20 to 29%.
// The seventh product and the statistics' pass are the price of sums in a fixed order.
//
// Hidden keys: a packing kernel turns the padding mask into a bit per key and
// the end of the visible keys of each sample; tiles past it are not visited.
// Scores of hidden keys are replaced, not added to, and in a tile that mixes
// hidden and visible keys the hidden rows of the B operand (V, or K for dQ) are
// zeroed in shared memory, so that whatever a padded position holds (NaN too)
// has no effect.
//
// All waits are bounded (see sm100_ptx.cuh).
#include "sm100_ptx.cuh"
#include "cross_attn.h"
#include "cross_attn_join.cuh"

#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <mutex>
#include <type_traits>

namespace flodl {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kRows = 128;  // stationary rows of a tile: the TMEM lanes
constexpr uint64_t kWaitNs = 2000000000ull;
constexpr float kRescaleThreshold = 8.0f;  // log2 units: P stays below 2^8

template <typename T>
struct Type;
template <>
struct Type<__nv_bfloat16> {
  static constexpr uint32_t kIdesc = 1;  // tcgen05 kind::f16 operand format
  static constexpr float kShift = 0.f;
  static constexpr bool kCubic = true;  // (see f2_exp2_cubic)
  static constexpr bool kRanged = false;
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16x2(a, b); }
  static __device__ __forceinline__ uint64_t unpack(uint32_t v) {
    const float2 f = unpack_bf16x2(v);
    return f2_pack(f.x, f.y);
  }
};
template <>
struct Type<__half> {
  static constexpr uint32_t kIdesc = 0;
  // P of a long row lies below f16's normal range (2^-14): the backward's P^T
  // is formed at 2^7 times its value and dV scaled back
  static constexpr float kShift = 7.f;
  static constexpr bool kCubic = false;
  static constexpr bool kRanged = true;  // dS is formed at a power of two (see range_shift)
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ uint64_t unpack(uint32_t v) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
    return f2_pack(f.x, f.y);
  }
};

__host__ __device__ constexpr uint32_t idesc(uint32_t fmt, uint32_t M, uint32_t N, uint32_t b_mn) {
  return (1u << 4) | (fmt << 7) | (fmt << 10) | (b_mn << 16) | ((N >> 3) << 17) | ((M >> 4) << 24);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^x of a pair on the FMA pipe, for x <= 128 (below -126.5: zero; NaN stays NaN):
// 2^n by the exponent bits times a cubic for 2^f, |f| <= 1/2, fitted by Remez' exchange
// for relative error (7.5e-5). The exponential unit takes 8 cycles for a warp's 32
// values; every fourth pair done this way shortens a tile's round trip (128 heads,
// 1024 x 1024 x 64: forward 61.9 -> 58.1 us, dQ 66.5 -> 62.6; every second pair 66.6 and 72,
// issue then bounds it; dK/dV, which needs an addition more per pair, 90 -> 94).
// Only for P that is rounded to bf16 (half a step: 2e-3): f16 would want a degree more,
// and gains nothing then.
__device__ __forceinline__ uint64_t f2_exp2_cubic(uint64_t x) {
  float a, b;
  f2_unpack(x, a, b);
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(-127.f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(b) : "f"(-127.f));
  x = f2_pack(a, b);
  const uint64_t t = f2_add(x, f2_splat(12582912.f));  // 1.5 * 2^23: n in the low bits
  const uint64_t f = f2_fma(f2_add(t, f2_splat(-12582912.f)), f2_splat(-1.f), x);
  uint64_t p = f2_fma(f, f2_splat(0.0551716685f), f2_splat(0.242611125f));
  p = f2_fma(p, f, f2_splat(0.693260968f));
  p = f2_fma(p, f, f2_splat(0.999928057f));
  f2_unpack(t, a, b);
  return f2_mul(p, f2_pack(__uint_as_float((__float_as_uint(a) << 23) + 0x3f800000u),
                           __uint_as_float((__float_as_uint(b) << 23) + 0x3f800000u)));
}
// 2^x of a pair, the kind by the pair's index.
template <bool kCubic>
__device__ __forceinline__ void exp2_pair(uint64_t x, int pair, float& p0, float& p1) {
  if (kCubic && pair % 4 == 0) {
    f2_unpack(f2_exp2_cubic(x), p0, p1);
  } else {
    f2_unpack(x, p0, p1);
    p0 = ex2(p0);
    p1 = ex2(p1);
  }
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// A tile of kN rows and kDP columns: kDP / 64 blocks of kN rows x 128 bytes in
// 128-byte swizzle.
template <int kN, int kDP>
__device__ __forceinline__ void load_tile(uint8_t* dst, const CUtensorMap* map, uint64_t* bar,
                                          int row, int head, int batch) {
#pragma unroll
  for (int c = 0; c < kDP / 64; ++c)
    tma_load_4d(dst + c * kN * 128, map, bar, c * 64, row, head, batch);
}

// The MMA thread's instructions. Descriptors are a constant upper half and a
// lower half (address / 16) that advances by constants.
constexpr uint32_t desc_hi(uint32_t sbo) {
  return ((sbo >> 4) & 0x3FFFu) | (1u << 14) | (2u << 29);  // version, 128-byte swizzle
}
// (In a cluster the bits above a CTA's own 256 KB of shared addresses hold its
// rank; they would run into the stride's field.)
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) {
  return ((addr & 0x3FFFFu) >> 4) | ((lbo >> 4) << 16);
}
__device__ __forceinline__ void umma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t id,
                                        uint32_t acc) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      ".reg .b64 da, db;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "mov.b64 da, {%1, %5};\n"
      "mov.b64 db, {%2, %5};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n"
      "}\n" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(id), "r"(acc), "n"(desc_hi(1024))
      : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t id,
                                        uint32_t acc) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      ".reg .b64 db;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "mov.b64 db, {%2, %5};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n"
      "}\n" ::"r"(d),
      "r"(a_tmem), "r"(b_lo), "r"(id), "r"(acc), "n"(desc_hi(1024))
      : "memory");
}
// D[128, n] = A[128, kDP] B[n, kDP]^T, both tiles K-major in shared memory.
template <int kNA, int kNB, int kDP>
__device__ __forceinline__ void mma_rows(uint32_t d, uint32_t a, uint32_t b, uint32_t id) {
  const uint32_t al = desc_lo(a, 16), bl = desc_lo(b, 16);
#pragma unroll
  for (int kk = 0; kk < kDP / 16; ++kk)
    umma_ss(d, al + ((kk / 4) * (kNA * 128) + (kk % 4) * 32) / 16,
            bl + ((kk / 4) * (kNB * 128) + (kk % 4) * 32) / 16, id, kk > 0);
}
// D[128, kDP] (+)= A[128, kK] B[kK, kDP], A 16-bit pairs in TMEM, B a streamed
// tile read along its rows (MN-major).
template <int kK, int kDP>
__device__ __forceinline__ void mma_cols(uint32_t d, uint32_t a_tmem, uint32_t b, uint32_t id,
                                         bool acc) {
  const uint32_t bl = desc_lo(b, kK * 128);
#pragma unroll
  for (int kk = 0; kk < kK / 16; ++kk)
    umma_ts(d, a_tmem + kk * 8, bl + kk * 2048 / 16, id, (acc || kk > 0) ? 1u : 0u);
}

// Zero the rows of a streamed tile whose bit in words is clear (thread `tid` of
// `nthreads`), before a product reads them as B.
template <int kN, int kDP>
__device__ __forceinline__ void zero_hidden_rows(uint8_t* tile, uint2 words, int tid, int nthreads) {
  static_assert(kN == 64, "two words");
  for (int i = tid; i < kN * (kDP / 64); i += nthreads) {
    const int row = i % kN;
    if (!(((row < 32 ? words.x : words.y) >> (row % 32)) & 1u)) {
      uint4* r = reinterpret_cast<uint4*>(tile + (i / kN) * kN * 128 + row * 128);
#pragma unroll
      for (int c = 0; c < 8; ++c) r[c] = make_uint4(0, 0, 0, 0);
    }
  }
  fence_proxy_async_shared();
  __syncwarp();  // the caller's next TMEM instruction is aligned
}

// Sixteen columns of a row that lies in TMEM from t on, times f (`use` false:
// zeros; `there`, the same for the warp, says whether TMEM holds them).
__device__ __forceinline__ void row16(uint32_t t, bool there, bool use, float f, float (&v)[16]) {
  uint32_t o[16];
  if (there) {
    tmem_ld_16cols(t, o);
    tmem_ld_wait();
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = there && use ? __uint_as_float(o[i]) * f : 0.f;
}
// An item's output tile leaves through the shared memory of its stationary
// operand, which no product reads any more, by TMA. (Stored from registers, a
// row per lane, an instruction touches 32 lines with 16 bytes each: the 128 rows
// of dK and dV then took 3000 cycles.) `block`: the warp's 32 rows x 64 columns
// in 128-byte swizzle.
// Eight values in 16 bits; kRes: instead what that rounding leaves off.
template <typename T, bool kRes>
__device__ __forceinline__ uint4 pack8(const float* v) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = Type<T>::pack(v[2 * i], v[2 * i + 1]);
    if (kRes) {
      float a, b;
      f2_unpack(Type<T>::unpack(w[i]), a, b);
      w[i] = Type<T>::pack(v[2 * i] - a, v[2 * i + 1] - b);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T, bool kRes>
__device__ __forceinline__ void stage_rows(uint32_t t, int lane, bool use, float f, uint8_t* block) {
#pragma unroll 2
  for (int c = 0; c < 4; ++c) {
    float v[16];
    row16(t + c * 16, true, use, f, v);
#pragma unroll
    for (int h = 0; h < 2; ++h)
      *reinterpret_cast<uint4*>(block + lane * 128 + (((2 * c + h) ^ (lane & 7)) << 4)) =
          pack8<T, kRes>(v + 8 * h);
  }
}
// Values to `block` and their remainders to `res`, 64 columns.
template <typename T>
__device__ __forceinline__ void stage_pair(uint32_t t, int lane, bool use, float f, uint8_t* block,
                                           uint8_t* res) {
#pragma unroll 2
  for (int c = 0; c < 4; ++c) {
    float v[16];
    row16(t + c * 16, true, use, f, v);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = lane * 128 + (((2 * c + h) ^ (lane & 7)) << 4);
      *reinterpret_cast<uint4*>(block + at) = pack8<T, false>(v + 8 * h);
      *reinterpret_cast<uint4*>(res + at) = pack8<T, true>(v + 8 * h);
    }
  }
}
// The plain form: a row's columns below D as 16-bit values to out (and their
// remainders to res), or as f32 to part (pieces of a split axis; rows without a
// visible tile).
template <typename T>
__device__ __forceinline__ void store_row(uint32_t t, int D, bool there, bool use, bool row, float f,
                                          T* out, T* res, float* part) {
#pragma unroll 1
  for (int c = 0; c < D; c += 16) {
    float v[16];
    row16(t + c, there, use, f, v);
    if (row && part == nullptr) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (c + 8 * h < D) {
          *reinterpret_cast<uint4*>(out + c + 8 * h) = pack8<T, false>(v + 8 * h);
          if (res != nullptr) *reinterpret_cast<uint4*>(res + c + 8 * h) = pack8<T, true>(v + 8 * h);
        }
    } else if (row) {
#pragma unroll
      for (int h = 0; h < 4; ++h)
        if (c + 4 * h < D)
          *reinterpret_cast<float4*>(part + c + 4 * h) =
              make_float4(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]);
    }
    __syncwarp();  // a tile may end inside a warp: the next TMEM load is aligned
  }
}

struct Shape {
  int B, Sq, Sk, H, Hk, G, D, causal;
  int splits;
  float scale;
  const uint32_t* words;  // [B, nwords] or null
  const int* vis_end;     // [B]
  int nwords, n_items;
  uint32_t* err;
  // item -> (row tile, batch, head, piece): divisors of an item's index
  FastDiv by_splits, by_outer, by_heads, by_group;
};

// The items of a CTA, one of each round of gridDim.x: every second round is dealt
// backwards, so that a CTA with one of the heaviest items gets one of the lightest
// next (causal 2 x 16 heads, 4096 x 4096 x 64: forward 136 -> 113 us, dQ 137 -> 124, dK/dV
// 195 -> 178).
struct Walk {
  int at = blockIdx.x, step = 2 * (int)(gridDim.x - blockIdx.x) - 1;
  __device__ __forceinline__ int after() const { return at + step; }
  __device__ __forceinline__ void next() {
    at += step;
    step = 2 * (int)gridDim.x - step;
  }
};

// An item's coordinates: the piece fastest, then heads; samples slowest (a sample
// with few visible keys has light items), or under a causal mask row tiles.
struct ItemAt {
  int rt, b, head, split;
};
__device__ __forceinline__ ItemAt item_at(const Shape& s, int item) {
  ItemAt a;
  const uint32_t i = s.by_splits.div(item);
  a.split = item - i * s.by_splits.d;
  const uint32_t outer = s.by_outer.div(i), rest = i - outer * s.by_outer.d;
  const uint32_t inner = s.by_heads.div(rest);
  a.head = rest - inner * s.by_heads.d;
  a.rt = s.causal ? outer : inner;
  a.b = s.causal ? inner : outer;
  return a;
}
// Streamed tiles [lo, hi) of piece `split` of nt.
__device__ __forceinline__ void piece_of(const Shape& s, int split, int nt, int& lo, int& hi) {
  lo = 0;
  hi = nt;
  if (s.splits > 1) {  // (64-bit divisions: not for every item)
    lo = (int)((int64_t)nt * split / s.splits);
    hi = (int)((int64_t)nt * (split + 1) / s.splits);
  }
}

__device__ __forceinline__ int visible_end(const Shape& s, int b) {
  return s.vis_end ? __ldg(s.vis_end + b) : s.Sk;
}

struct Waiter {
  volatile uint32_t* abort;
  uint32_t* err;
  __device__ __forceinline__ bool operator()(uint64_t* bar, uint32_t parity) const {
    return mbar_wait_bounded(bar, parity, abort, err, kWaitNs);
  }
};

// Position and parity in a ring of barriers.
template <uint32_t kSize>
struct Ring {
  uint32_t at = 0, phase = 0;
  __device__ __forceinline__ void next() {
    if (++at == kSize) {
      at = 0;
      phase ^= 1;
    }
  }
};

// After a failed wait: the copies still in flight write this CTA's shared
// memory, so give each issued load (bounded) time to land before leaving.
__device__ __forceinline__ void settle(uint64_t* bar, uint32_t issued) {
  if (issued == 0) return;
  const uint64_t t0 = global_timer_ns();
  while (!mbar_try_wait(bar, (issued - 1) & 1) && global_timer_ns() - t0 < 100000000ull) {
  }
}

// ============================================================== forward
// One item: 128 queries of a head, and a range of its key tiles (64 keys).
// Warps: 0 TMA, 1 MMA, 2..5 softmax (a row per thread: 64 scores in registers).
// Two CTAs per SM (256 TMEM columns, 97 KB of shared memory each) cover each
// other's waits. TMEM: two score buffers at 0 and 64, P over its own scores, O
// at 128. S of a tile is computed while the softmax works on the one before;
// P V of a tile is issued behind S of the next. (Three CTAs with one score buffer
// each, at head size 64, have 96 registers a thread and spill: 87 instead of 62
// us on 8 x 16 heads, 1024 x 1024.)
constexpr int kN = 64;
constexpr int kFwdThreads = 192;
template <int kDP, bool kTrain>
struct FwdGeo {
  static constexpr int kQBufs = kDP == 64 ? 2 : 1;
  static constexpr bool kResBuf = kTrain && kDP == 64;  // the remainders have a buffer
  static constexpr int kStages = kDP == 64 ? (kResBuf ? 3 : 4) : 2;
};
constexpr int kFwdCtas = 2;       // per SM
constexpr uint32_t kTmemO = 128;

template <int kDP, bool kTrain>
struct FwdSmem {
  using G = FwdGeo<kDP, kTrain>;
  uint8_t q[G::kQBufs][kRows * kDP * 2];
  uint8_t k[G::kStages][kN * kDP * 2];
  uint8_t v[G::kStages][kN * kDP * 2];
  uint8_t res[G::kResBuf ? kRows * kDP * 2 : 16];  // (behind what needs 1024-byte alignment)
  uint64_t q_full[G::kQBufs], q_empty[G::kQBufs];
  uint64_t k_full[G::kStages], k_empty[G::kStages], v_full[G::kStages], v_empty[G::kStages];
  uint64_t s_full[2], p_full[2], pv_done[2], drain;  // [2]: by tile parity (a softmax warp
                                                     // may be a tile ahead of another)
  uint32_t tmem_base, abort;
};

// Query tiles run from the last to the first: under a causal mask the heaviest first.
struct FwdItem {
  int qt, h, b, split, lo, hi;  // key tiles [lo, hi)
};
__device__ __forceinline__ FwdItem fwd_item(const Shape& s, int item, int n_qt) {
  FwdItem it{};
  if (item >= s.n_items) return it;  // asked for ahead of time
  const ItemAt at = item_at(s, item);
  it.split = at.split;
  it.qt = n_qt - 1 - at.rt;
  it.h = at.head;
  it.b = at.b;
  int end = visible_end(s, it.b);
  if (s.causal) end = min(end, (it.qt + 1) * kRows);
  piece_of(s, it.split, (end + kN - 1) / kN, it.lo, it.hi);
  return it;
}

// Visible-key words of the 64 keys from k0 (keys past Sk are clear).
__device__ __forceinline__ uint2 tile_words(const Shape& s, int b, int k0) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int at = k0 / 32 + i;
    if (s.words) {
      w[i] = at < s.nwords ? __ldg(s.words + (int64_t)b * s.nwords + at) : 0u;
    } else {
      const int left = s.Sk - at * 32;
      w[i] = left >= 32 ? 0xffffffffu : (left <= 0 ? 0u : (1u << left) - 1u);
    }
  }
  return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ bool is_whole(uint2 w) { return (w.x & w.y) == 0xffffffffu; }

template <typename T, int kDP, bool kTrain>
__global__ void __launch_bounds__(kFwdThreads, kFwdCtas)
    cross_fwd_kernel(const __grid_constant__ CUtensorMap tm_q,
                     const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v,
                     const __grid_constant__ CUtensorMap tm_o,
                     const __grid_constant__ CUtensorMap tm_r, const __grid_constant__ Shape sh,
                     T* __restrict__ out, T* __restrict__ out_res, float* __restrict__ lse2,
                     float* __restrict__ part_o, float* __restrict__ part_lse, int n_items,
                     int n_qt) {
  using Geo = FwdGeo<kDP, kTrain>;
  constexpr uint32_t kStages = Geo::kStages, kQBufs = Geo::kQBufs;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  FwdSmem<kDP, kTrain>& sm = *reinterpret_cast<FwdSmem<kDP, kTrain>*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const Waiter wait{&sm.abort, sh.err};
  // a cluster's piece takes the memory of the keys and values once all are read
  float* s_piece = reinterpret_cast<float*>(sm.k);
  float* s_lse = reinterpret_cast<float*>(sm.q);
  static_assert(sizeof(sm.k) + sizeof(sm.v) >= kRows * kDP * 4, "a piece in the stages");

  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < kQBufs; ++i) {
      mbar_init(&sm.q_full[i], 1);
      mbar_init(&sm.q_empty[i], 4);
    }
    for (uint32_t i = 0; i < kStages; ++i) {
      mbar_init(&sm.k_full[i], 1);
      mbar_init(&sm.k_empty[i], 1);
      mbar_init(&sm.v_full[i], 1);
      mbar_init(&sm.v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.s_full[i], 1);
      mbar_init(&sm.p_full[i], 4);
      mbar_init(&sm.pv_done[i], 1);
    }
    mbar_init(&sm.drain, 1);
    sm.abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc<256>(&sm.tmem_base);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  pdl_wait();
  pdl_trigger();

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (elect_one_sync()) {
      tma_prefetch_desc(&tm_q);
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
      uint32_t n = 0, t = 0;
      bool ok = true;
      for (Walk item; item.at < n_items && ok; item.next()) {
        const FwdItem it = fwd_item(sh, item.at, n_qt);
        if (it.lo >= it.hi) continue;
        const uint32_t qb = n % kQBufs;
        if (!(ok = wait(&sm.q_empty[qb], ((n / kQBufs) & 1) ^ 1))) break;
        mbar_arrive_expect_tx(&sm.q_full[qb], kRows * kDP * 2);
        load_tile<kRows, kDP>(sm.q[qb], &tm_q, &sm.q_full[qb], it.qt * kRows, it.h, it.b);
        ++n;
        const int kh = sh.by_group.div(it.h);
        for (int j = it.lo; j < it.hi; ++j, ++t) {
          const uint32_t st = t % kStages, par = ((t / kStages) & 1) ^ 1;
          if (!(ok = wait(&sm.k_empty[st], par))) break;
          mbar_arrive_expect_tx(&sm.k_full[st], kN * kDP * 2);
          load_tile<kN, kDP>(sm.k[st], &tm_k, &sm.k_full[st], j * kN, kh, it.b);
          if (!(ok = wait(&sm.v_empty[st], par))) break;
          mbar_arrive_expect_tx(&sm.v_full[st], kN * kDP * 2);
          load_tile<kN, kDP>(sm.v[st], &tm_v, &sm.v_full[st], j * kN, kh, it.b);
        }
      }
      if (!ok) {
        for (uint32_t i = 0; i < kQBufs; ++i) settle(&sm.q_full[i], (n + kQBufs - 1 - i) / kQBufs);
        for (uint32_t i = 0; i < kStages; ++i) {
          settle(&sm.k_full[i], (t + kStages - i) / kStages);
          settle(&sm.v_full[i], (t + kStages - 1 - i) / kStages);
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (elect_one_sync()) {
      constexpr uint32_t id_s = idesc(Type<T>::kIdesc, kRows, kN, 0);
      constexpr uint32_t id_o = idesc(Type<T>::kIdesc, kRows, kDP, 1);
      const uint32_t q0 = smem_u32(sm.q[0]), k0 = smem_u32(sm.k[0]), v0 = smem_u32(sm.v[0]);
      Ring<kStages> ks, vs;  // stages of K (tile t) and V (the tile behind)
      Ring<kQBufs> qs;
      Ring<2> ss, ps;   // score buffers of tile t and of the tile behind
      bool ok = true, issued = false;
      // P V of the tile behind
      auto issue_pv = [&](bool acc) -> bool {
        if (!wait(&sm.v_full[vs.at], vs.phase)) return false;
        if (!wait(&sm.p_full[ps.at], ps.phase)) return false;
        tc_fence_after();
        mma_cols<kN, kDP>(tmem + kTmemO, tmem + ps.at * 64u, v0 + vs.at * (kN * kDP * 2), id_o, acc);
        umma_commit(&sm.pv_done[ps.at]);
        umma_commit(&sm.v_empty[vs.at]);
        vs.next();
        ps.next();
        return true;
      };
      // P V of a tile is issued behind S of the next one, over item borders too
      // where the next item's Q has a buffer of its own
      bool behind = false, behind_acc = false;
      FwdItem after = fwd_item(sh, blockIdx.x, n_qt);
      for (Walk item; item.at < n_items && ok; item.next()) {
        const FwdItem it = after;
        if (it.lo >= it.hi) {
          after = fwd_item(sh, item.after(), n_qt);
          continue;
        }
        if (kQBufs == 1 && behind) {
          if (!(ok = issue_pv(behind_acc))) break;
          behind = false;
        }
        if (!(ok = wait(&sm.q_full[qs.at], qs.phase))) break;
        const uint32_t q_addr = q0 + qs.at * (kRows * kDP * 2);
        for (int j = it.lo; j < it.hi; ++j) {
          if (!(ok = wait(&sm.k_full[ks.at], ks.phase))) break;
          tc_fence_after();
          // the products with this buffer's last P were issued before: in order
          mma_rows<kRows, kN, kDP>(tmem + ss.at * 64u, q_addr, k0 + ks.at * (kN * kDP * 2), id_s);
          issued = true;
          umma_commit(&sm.s_full[ss.at]);
          umma_commit(&sm.k_empty[ks.at]);
          ks.next();
          ss.next();
          if (j == it.hi - 1) after = fwd_item(sh, item.after(), n_qt);  // while products run
          if (behind && !(ok = issue_pv(behind_acc))) break;
          behind = true;
          behind_acc = j > it.lo;
        }
        qs.next();
      }
      if (ok && behind) ok = issue_pv(behind_acc);
      if (!ok && issued) {
        umma_commit(&sm.drain);
        settle(&sm.drain, 1);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ softmax
    const int r = (warp & 3) * 32 + lane;  // query row within the tile
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_o = tmem + kTmemO + lanes;
    const float sl2 = sh.scale * kLog2e;
    const uint64_t sl2x2 = f2_splat(sl2);
    Ring<2> ss, last;  // score buffers of this tile and of the one before
    Ring<kStages> vs;
    Ring<kQBufs> qs;
    bool ok = true;
    // The Q buffer whose output store may still be read: given back once the
    // next item is under way, or at once where there is no other buffer.
    uint64_t* owed = nullptr;
    auto give_back = [&]() {
      if (owed != nullptr && lane == 0) {
        bulk_wait_group_read<0>();
        mbar_arrive(owed);
      }
      owed = nullptr;
    };
    FwdItem after = fwd_item(sh, blockIdx.x, n_qt);
    for (Walk item; item.at < n_items && ok; item.next()) {
      const FwdItem it = after;
      const int qi = it.qt * kRows + r;
      // tiles before `plain` hold no hidden score
      int plain = sh.Sk / kN;
      if (sh.causal) plain = min(plain, (it.qt * kRows + 1) / kN);
      if (sh.words) plain = 0;
      // Reference maximum (scaled, log2 units), and the sum of P. For a backward
      // pass lr sums P as rounded for the product as well, and O is divided by
      // it: a mean of the values with weights that add up to 1, or else a row
      // that one key dominates has that weight's rounding in its dO * O.
      float m_ref = -INFINITY, l = 0.f, lr = 0.f;
      uint2 words = sh.words && it.lo < it.hi ? tile_words(sh, it.b, it.lo * kN) : make_uint2(0, 0);
      for (int j = it.lo; j < it.hi; ++j) {
        const uint32_t t_s = tmem + lanes + ss.at * 64u;
        ok = wait(&sm.s_full[ss.at], ss.phase);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        tc_fence_after();
        uint32_t v[64];  // the row's scores
        tmem_ld_64cols(t_s, v);
        tmem_ld_wait();
        if (j >= plain) {  // hidden scores become -inf
          const uint2 w = sh.words ? words : tile_words(sh, it.b, j * kN);
          if (sh.words && j + 1 < it.hi) words = tile_words(sh, it.b, (j + 1) * kN);
          const int lim = sh.causal ? qi - j * kN : kN;  // last visible column
          if (!is_whole(w) || __any_sync(0xffffffffu, lim < kN - 1)) {
#pragma unroll
            for (int i = 0; i < 64; ++i)
              v[i] = (((i < 32 ? w.x : w.y) >> (i % 32)) & 1u) && i <= lim ? v[i] : 0xff800000u;
            if (sh.words && !is_whole(w)) {
              ok = wait(&sm.v_full[vs.at], vs.phase);
              if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
              zero_hidden_rows<kN, kDP>(sm.v[vs.at], w, threadIdx.x - 64, 128);
            }
          }
        }
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 64; i += 2)
          m4[(i >> 1) & 3] = max3(m4[(i >> 1) & 3], __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
        const float mraw = max3(m4[0], m4[1], fmaxf(m4[2], m4[3]));
        const float mx = mraw == -INFINITY ? -INFINITY : mraw * sl2;
        // the reference moves only when the maximum grew by more than the
        // threshold, so O is seldom rescaled
        const bool move = mx > m_ref + kRescaleThreshold;
        if (__any_sync(0xffffffffu, move)) {
          const float c = (move && m_ref != -INFINITY) ? ex2(m_ref - mx) : 1.f;
          if (move) m_ref = mx;
          l *= c;
          if (kTrain) lr *= c;
          if (j > it.lo) {
            // P V of the tile before adds to O no more. (Not waited for at every
            // tile: of this barrier's phases all but that one are complete,
            // since S of this tile is.)
            ok = wait(&sm.pv_done[last.at], last.phase);
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            tc_fence_after();
#pragma unroll 1
            for (int k = 0; k < kDP / 16; ++k) {
              uint32_t o[16];
              tmem_ld_16cols(t_o + k * 16, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * c);
              tmem_st_16cols(t_o + k * 16, o);
            }
          }
        }
        // P = 2^(c s - m) as 16-bit pairs
        const uint64_t neg_m = f2_splat(m_ref == -INFINITY ? 0.f : -m_ref);
        uint64_t a[2] = {f2_splat(0.f), f2_splat(0.f)}, b[2] = {f2_splat(0.f), f2_splat(0.f)};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pw[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float p0, p1;
            exp2_pair<Type<T>::kCubic>(
                f2_fma(f2_pack(__uint_as_float(v[c * 16 + 2 * i]),
                               __uint_as_float(v[c * 16 + 2 * i + 1])), sl2x2, neg_m), i, p0, p1);
            pw[i] = Type<T>::pack(p0, p1);
            a[i & 1] = f2_add(a[i & 1], f2_pack(p0, p1));
            if (kTrain) b[i & 1] = f2_add(b[i & 1], Type<T>::unpack(pw[i]));
          }
          tmem_st_8cols(t_s + c * 8, pw);
        }
        float x0, x1;
        f2_unpack(f2_add(a[0], a[1]), x0, x1);
        l += x0 + x1;
        if (kTrain) {
          f2_unpack(f2_add(b[0], b[1]), x0, x1);
          lr += x0 + x1;
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full[ss.at]);
        last = ss;
        ss.next();
        vs.next();
        give_back();
      }
      if (!ok) break;
      after = fwd_item(sh, item.after(), n_qt);  // while the last product runs
      // ---- output: O / l and lse
      const bool any = it.lo < it.hi;
      if (any) {
        ok = wait(&sm.pv_done[last.at], last.phase);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        tc_fence_after();
      }
      // no visible key: zeros (a NaN sum passes through). Rounded, P is not 0 where
      // l is not: the row's maximum is at least 2^0 of its reference.
      const bool none = l == 0.f;
      const float inv_l = none ? 0.f : 1.f / (kTrain ? lr : l);
      const int64_t rows_all = (int64_t)sh.B * sh.Sq * sh.H;
      const int64_t orow = ((int64_t)it.b * sh.Sq + qi) * sh.H + it.h;
      const int64_t lrow = ((int64_t)it.b * sh.H + it.h) * sh.Sq + qi;
      if (any && sh.splits == 1) {
        uint8_t* block = sm.q[qs.at] + (warp & 3) * 4096;
        if (Geo::kResBuf) {
          if (lane == 0) bulk_wait_group_read<0>();  // the item before, long read
          __syncwarp();
          stage_pair<T>(t_o, lane, !none, inv_l, block, sm.res + (warp & 3) * 4096);
        } else if (kTrain) {  // the remainders first: the same memory
#pragma unroll 1
          for (int c = 0; c < kDP / 64; ++c)
            stage_rows<T, true>(t_o + c * 64, lane, !none, inv_l, block + c * kRows * 128);
          fence_proxy_async_shared();
          __syncwarp();
          if (lane == 0) {
            for (int c = 0; c * 64 < sh.D; ++c)
              tma_store_4d(&tm_r, block + c * kRows * 128, c * 64, qi - lane, it.h, it.b);
            bulk_commit_group();
            bulk_wait_group_read<0>();
          }
          __syncwarp();
        }
        if (!Geo::kResBuf)
#pragma unroll 1
          for (int c = 0; c < kDP / 64; ++c)
            stage_rows<T, false>(t_o + c * 64, lane, !none, inv_l, block + c * kRows * 128);
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) {
          if (Geo::kResBuf) tma_store_4d(&tm_r, sm.res + (warp & 3) * 4096, 0, qi - lane, it.h, it.b);
          for (int c = 0; c * 64 < sh.D; ++c)
            tma_store_4d(&tm_o, block + c * kRows * 128, c * 64, qi - lane, it.h, it.b);
          bulk_commit_group();
        }
      } else if (sh.splits > 1 && part_o == nullptr) {  // a cluster's piece
#pragma unroll 1
        for (int c = 0; c < kDP; c += 16) {
          float v[16];
          row16(t_o + c, any, !none, inv_l, v);
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            *reinterpret_cast<float4*>(s_piece + piece_at<kDP>(r, (c + i) / 4)) =
                make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        }
        s_lse[r] = none ? -INFINITY : m_ref + log2f(l);
      } else {
        store_row<T>(t_o, sh.D, any, !none, qi < sh.Sq, inv_l, out + orow * sh.D,
                     kTrain ? out_res + orow * sh.D : nullptr,
                     sh.splits > 1 ? part_o + (it.split * rows_all + orow) * sh.D : nullptr);
      }
      if (any) {
        owed = &sm.q_empty[qs.at];
        if (kQBufs == 1) give_back();
        qs.next();
      }
      if (qi < sh.Sq) {
        if (sh.splits > 1 && part_o == nullptr)
          ;  // joined below
        else if (sh.splits > 1)
          part_lse[it.split * rows_all + lrow] = none ? -INFINITY : m_ref + log2f(l);
        else if (kTrain)
          lse2[lrow] = none ? INFINITY : m_ref + log2f(l);
      }
      __syncwarp();
      tc_fence_before();
    }
    if (lane == 0) bulk_wait_group<0>();
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<256>(tmem);
  }
  if (sh.splits > 1 && part_o == nullptr) {  // one item per CTA
    const FwdItem it = fwd_item(sh, blockIdx.x, n_qt);
    const int q0 = it.qt * kRows;
    cluster_join<kDP>(
        s_piece, s_lse, min(kRows, sh.Sq - q0), sh.D, sh.splits,
        [&](int r, int c, float4 v) {
          const int64_t at = (((int64_t)it.b * sh.Sq + q0 + r) * sh.H + it.h) * sh.D + 4 * c;
          const uint2 w = make_uint2(Type<T>::pack(v.x, v.y), Type<T>::pack(v.z, v.w));
          *reinterpret_cast<uint2*>(out + at) = w;
          if (kTrain) {
            float4 f;
            f2_unpack(Type<T>::unpack(w.x), f.x, f.y);
            f2_unpack(Type<T>::unpack(w.y), f.z, f.w);
            *reinterpret_cast<uint2*>(out_res + at) =
                make_uint2(Type<T>::pack(v.x - f.x, v.y - f.y), Type<T>::pack(v.z - f.z, v.w - f.w));
          }
        },
        [&](int r, float lse) {
          if (kTrain) lse2[((int64_t)it.b * sh.H + it.h) * sh.Sq + q0 + r] = lse;
        });
  }
}

// ============================================================== mask packing
// A CTA per sample: visible-key words and the end of the visible keys.
__global__ void __launch_bounds__(256) pack_mask_kernel(const uint8_t* __restrict__ pad, int Sk,
                                                        int nwords, uint32_t* __restrict__ words,
                                                        int* __restrict__ vis_end) {
  __shared__ int s_end[8];
  pdl_wait();
  pdl_trigger();
  const int b = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int end = 0;
#pragma unroll 4
  for (int w = warp; w < nwords; w += 8) {
    const int key = w * 32 + lane;
    const uint32_t bits =
        __ballot_sync(0xffffffffu, key < Sk && __ldg(pad + (int64_t)b * Sk + key) == 0);
    if (lane == 0) words[(int64_t)b * nwords + w] = bits;
    if (bits) end = w * 32 + 32 - __clz(bits);
  }
  if (lane == 0) s_end[warp] = end;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) end = max(end, s_end[w]);
    vis_end[b] = end;
  }
}

// ============================================================== backward
// delta = rowsum(dO * O): kLanes lanes per row, 8 values each.
template <typename T>
__device__ __forceinline__ float dot8(uint4 a, uint4 b);
template <>
__device__ __forceinline__ float dot8<__nv_bfloat16>(uint4 a, uint4 b) {
  const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 u = unpack_bf16x2(x[i]), v = unpack_bf16x2(y[i]);
    s = fmaf(u.x, v.x, fmaf(u.y, v.y, s));
  }
  return s;
}
template <>
__device__ __forceinline__ float dot8<__half>(uint4 a, uint4 b) {
  const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&x[i]));
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&y[i]));
    s = fmaf(u.x, v.x, fmaf(u.y, v.y, s));
  }
  return s;
}
struct Stride3 {
  int64_t b, s, h;
};
// f16 has no normal numbers below 2^-14, and dS = P (dP - delta) of a long row or of
// a small dO lies below (8192 keys, D = 64: with dO of 1e-3 the input gradients were off
// by 0.010 of their norm, where rounding them once is off by 0.0009). So f16 dS is formed
// at 2^k of its value and the products scaled back in f32. k comes from
//   |dP - delta| <= 2 |dO_i| max_j |V_j|   (norms; j over the visible keys; O is a mean of V)
// so that 2^k |dS| stays within 2^15: for dQ from its row's dO, for dK, which sums rows, from
// the largest dO of the memory head's queries. The power is folded into exponents
// and factors that are there anyway; what it costs is a pass over V behind the row
// statistics (64 x 8 heads, 256 x 256 x 64: 14.2 us for both, the statistics alone 7.4, and dQ
// 27.3 instead of 25.6; 42 heads of 128 x 1500 x 64: 6.1 instead of 2.5).
struct Range {
  const float* norms;  // |dO_i|^2 [B, H, stat_pitch]
  // [B, Hk, parts] the largest |dO_i|^2 and |V_j|^2 of a part of the rows, as bits (of
  // numbers >= 0 in their order, NaN above all)
  const uint32_t *d_max, *v_max;
  int parts;  // kRangeParts at most: a lane each
};
constexpr int kRangeParts = 32;
__device__ __forceinline__ int range_shift(float d2, float v2) {
  const float p = d2 * v2;
  if (!(p > 0.f && p < INFINITY)) return 0;  // nothing to scale, or no finite result
  const int e = (int)(__float_as_uint(p) >> 23) - 127;  // sqrt(p) < 2^ceil((e + 1) / 2)
  return 14 - ((e + 2) >> 1);
}
// The backward's row statistics: {-lse2, -delta} of every query, [B, H, pitch]
// with the pitch Sq rounded up to 64 so that a streamed tile's 64 pairs are one
// aligned 512-byte copy. Rows past Sq hold {-inf, 0}: their P is 0. (Made by the
// queries' kernel instead, from tiles of O and its remainders, they cost a kernel
// less, but a training step of 64 x 8 heads, 256 x 256 x 64, took 108 us instead of 101.)
__host__ __device__ constexpr int stat_pitch(int Sq) { return (Sq + 63) / 64 * 64; }
// Bound by the bytes of dO, O and its remainders (which the forward leaves in L2 where
// they fit). kLanes lanes take a row; two rows of each are in flight, and indexes are 32
// bits (64-bit divisions for every row took 10.6 instead of 7.3 us on 64 x 8 heads,
// 256 rows of 64; 19.9 instead of 13.4 on 4 x 16 heads, 2048 rows of 128).
constexpr int kRowsAhead = 2;
template <typename T, int kLanes>
__global__ void __launch_bounds__(256) cross_stats_kernel(const T* __restrict__ out,
                                                          const T* __restrict__ out_res,
                                                          const T* __restrict__ dout, Stride3 ds,
                                                          const float* __restrict__ lse2,
                                                          float2* __restrict__ stats,
                                                          float* __restrict__ norms, int B, int Sq,
                                                          FastDiv by_heads, int D) {
  pdl_wait();
  pdl_trigger();
  constexpr int kPer = 256 / kLanes;
  const int part = threadIdx.x % kLanes, sub = threadIdx.x / kLanes;
  const int pitch = stat_pitch(Sq), H = by_heads.d;
  const uint32_t rows = (uint32_t)pitch * H;  // of a sample
  const bool mine = part * 8 < D;
  for (int b = blockIdx.y; b < B; b += gridDim.y)
    for (uint32_t base = blockIdx.x * (kPer * kRowsAhead); base < rows;
         base += gridDim.x * (kPer * kRowsAhead)) {
      uint4 g[kRowsAhead], o[kRowsAhead], r[kRowsAhead];
      uint32_t i[kRowsAhead], h[kRowsAhead];
#pragma unroll
      for (int k = 0; k < kRowsAhead; ++k) {
        const uint32_t row = base + k * kPer + sub;  // i * H + h
        i[k] = by_heads.div(row);
        h[k] = row - i[k] * H;
        g[k] = o[k] = r[k] = make_uint4(0, 0, 0, 0);
        if (i[k] < (uint32_t)Sq && mine) {
          const int64_t at = (((int64_t)b * Sq + i[k]) * H + h[k]) * D + part * 8;
          g[k] = __ldg(reinterpret_cast<const uint4*>(dout + b * ds.b + i[k] * ds.s + h[k] * ds.h +
                                                      part * 8));
          o[k] = __ldg(reinterpret_cast<const uint4*>(out + at));
          r[k] = __ldg(reinterpret_cast<const uint4*>(out_res + at));
        }
      }
#pragma unroll
      for (int k = 0; k < kRowsAhead; ++k) {
        // with what O's rounding left off: in a row that one key dominates, dP and
        // delta nearly cancel, and the rounding of O would be the largest error
        float s = dot8<T>(o[k], g[k]) + dot8<T>(r[k], g[k]);
#pragma unroll
        for (int x = kLanes / 2; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        if (part == 0 && i[k] < (uint32_t)pitch)
          stats[((int64_t)b * H + h[k]) * pitch + i[k]] = make_float2(
              i[k] < (uint32_t)Sq ? -__ldg(lse2 + ((int64_t)b * H + h[k]) * Sq + i[k]) : -INFINITY, -s);
        if constexpr (Type<T>::kRanged) {
          float n = dot8<T>(g[k], g[k]);
#pragma unroll
          for (int x = kLanes / 2; x > 0; x >>= 1) n += __shfl_xor_sync(0xffffffffu, n, x);
          if (part == 0 && i[k] < (uint32_t)pitch) norms[((int64_t)b * H + h[k]) * pitch + i[k]] = n;
        }
      }
    }
}

// The largest |V_j|^2 over the visible keys of a part of each (sample, memory head), by
// kLanes lanes a row, and the largest of a part of its queries' |dO_i|^2. (Raised by atomics
// in the statistics' kernel, the second cost 20 us on 8 x 16 heads, 1024 x 1024 x 64.)
template <typename T, int kLanes>
__global__ void __launch_bounds__(256) cross_range_kernel(const T* __restrict__ v, Stride3 vs,
                                                          const uint32_t* __restrict__ words,
                                                          const int* __restrict__ vis_end, int Sk,
                                                          FastDiv by_heads, uint32_t units, int D,
                                                          const float* __restrict__ norms, int64_t rows,
                                                          uint32_t* __restrict__ d_max,
                                                          uint32_t* __restrict__ v_max) {
  __shared__ uint2 s_top[8];
  pdl_wait();
  pdl_trigger();
  constexpr int kPer = 256 / kLanes;
  const int part = threadIdx.x % kLanes, sub = threadIdx.x / kLanes;
  const bool mine = part * 8 < D;
  const int nwords = (Sk + 31) / 32;
  for (uint32_t unit = blockIdx.y; unit < units; unit += gridDim.y) {
    const uint32_t b = by_heads.div(unit), kh = unit - b * by_heads.d;
    const int end = vis_end ? __ldg(vis_end + b) : Sk;
    const T* base = v + b * vs.b + kh * vs.h + part * 8;
    uint2 top = make_uint2(0, 0);  // of dO, of V
#pragma unroll 4
    for (int64_t i = blockIdx.x * 256 + threadIdx.x; i < rows; i += gridDim.x * 256)
      top.x = max(top.x, __float_as_uint(__ldg(norms + unit * rows + i)));
#pragma unroll 4
    for (int j0 = blockIdx.x * kPer; j0 < end; j0 += gridDim.x * kPer) {
      const int j = j0 + sub;
      const bool seen =
          j < end && (!words || ((__ldg(words + (int64_t)b * nwords + j / 32) >> (j & 31)) & 1u));
      uint4 x = make_uint4(0, 0, 0, 0);
      if (seen && mine) x = __ldg(reinterpret_cast<const uint4*>(base + (int64_t)j * vs.s));
      float n = dot8<T>(x, x);
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
      top.y = max(top.y, __float_as_uint(n));
    }
    top.x = __reduce_max_sync(0xffffffffu, top.x);
    top.y = __reduce_max_sync(0xffffffffu, top.y);
    if (threadIdx.x % 32 == 0) s_top[threadIdx.x / 32] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < 8; ++w) top = make_uint2(max(top.x, s_top[w].x), max(top.y, s_top[w].y));
      d_max[(int64_t)unit * gridDim.x + blockIdx.x] = top.x;
      v_max[(int64_t)unit * gridDim.x + blockIdx.x] = top.y;
    }
    __syncthreads();
  }
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes,
                                          uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

// One kernel for both halves. kKeys false: rows are 128 queries (A1 = Q,
// A2 = dO), the stream is K, V, acc1 = dS K. kKeys true: rows are 128 keys
// (A1 = K, A2 = V), the stream is Q, dO of every query head that reads this
// memory head, acc1 = dS^T Q, acc2 = P^T dO.
// Warps: 0 TMA, 1 the scores' MMA, 2..5 and 6..9 two compute groups that take
// the streamed tiles of 64 in turn, 10 the products' MMA. TMEM: [S, dP] of kBufs
// tiles, 128 columns each, then acc1 and acc2; dS lies over S (kKeys: P over S,
// dS over dP). With three buffers (all but the keys' kernel at head size 128,
// whose accumulators leave room for two) the tensor cores' round trip for a
// tile passes while the groups are on two others, and two warps issue the MMAs,
// because one thread's waits, issues and commits for a tile took about 1000
// cycles. With two buffers a tile's scores follow the products before them in
// the tensor pipe's order, from one thread (two threads: 592 instead of 528 us
// on 16 x 2048 queries, 8192 keys, batch 2).
constexpr int kBN = 64;

// Shared memory: kABufs stationary pairs (two: the next item's loads early) and
// kStages streamed pairs.
template <int kDP, bool kKeys, int kABufs>
struct BwdGeo {
  static constexpr int kBufs = kKeys && kDP == 128 ? 2 : 3;
  static constexpr int kStages = kDP == 64 ? 6 : (kABufs == 2 ? 3 : 5);
  static constexpr int kABytes = kRows * kDP * 2;
  static constexpr int kBBytes = kBN * kDP * 2;
  static constexpr uint32_t kAcc = 128 * kBufs;
  static constexpr bool kSplitMma = kBufs == 3;
  static constexpr int kThreads = kSplitMma ? 352 : 320;
  static_assert(kAcc + (kKeys ? 2 : 1) * kDP <= 512, "TMEM columns");
};
template <int kDP, bool kKeys, int kABufs>
struct BwdSmem {
  using G = BwdGeo<kDP, kKeys, kABufs>;
  uint8_t a1[kABufs][G::kABytes], a2[kABufs][G::kABytes];
  uint8_t b1[G::kStages][G::kBBytes], b2[G::kStages][G::kBBytes];
  float2 stat[kKeys ? G::kStages : 1][kBN];  // kKeys: the streamed queries' statistics
  uint64_t a_full[kABufs], a_empty[kABufs], b_full[G::kStages], b_empty[G::kStages];
  uint64_t s_full[G::kBufs], ds_full[G::kBufs], buf_free[G::kBufs], acc_full, acc_free, drain[2];
  uint32_t tmem_base, abort;
};

struct BwdItem {
  int row0, head, b, split, lo, hi;  // stream tiles [lo, hi); kKeys: tile index = group * n + tile
  int first, n;                      // kKeys: first query tile, query tiles per head
};
template <bool kKeys>
__device__ __forceinline__ BwdItem bwd_item(const Shape& s, int item, int n_rt) {
  BwdItem it{};
  if (item >= s.n_items) return it;  // asked for ahead of time
  const ItemAt at = item_at(s, item);
  it.split = at.split;
  // heaviest first under a causal mask: the last queries, the first keys
  it.row0 = (kKeys ? at.rt : n_rt - 1 - at.rt) * kRows;
  it.head = at.head;
  it.b = at.b;
  const int end = visible_end(s, it.b);
  int nt;
  it.first = 0;
  it.n = 0;
  if (kKeys) {
    const int nq = (s.Sq + kBN - 1) / kBN;
    it.first = s.causal ? min(it.row0 / kBN, nq) : 0;
    it.n = nq - it.first;
    nt = it.row0 < end ? s.G * it.n : 0;
  } else {
    nt = ((s.causal ? min(end, it.row0 + kRows) : end) + kBN - 1) / kBN;
  }
  piece_of(s, it.split, nt, it.lo, it.hi);
  return it;
}

template <typename T>
struct BwdOut {
  T *o1, *o2;          // dQ, or dK and dV
  Stride3 s1, s2;
  float* part;         // [splits][1 or 2][rows][D] when splits > 1
  Range range;
};

// kSplit: pieces of the streamed axis (a template because the code that joins them
// costs the others registers: 28.3 instead of 26.7 us on 64 x 8 heads, 256 x 256 x 64; the
// split queries' kernels, at the 168 registers of a thread, spill 4 to 60 bytes).
template <typename T, int kDP, bool kKeys, int kABufs, bool kSplit>
__global__ void __launch_bounds__(BwdGeo<kDP, kKeys, kABufs>::kThreads, 1)
    cross_bwd_kernel(const __grid_constant__ CUtensorMap tm_a1,
                     const __grid_constant__ CUtensorMap tm_a2,
                     const __grid_constant__ CUtensorMap tm_b1,
                     const __grid_constant__ CUtensorMap tm_b2,
                     const __grid_constant__ CUtensorMap tm_o1,
                     const __grid_constant__ CUtensorMap tm_o2, const __grid_constant__ Shape sh,
                     const float2* __restrict__ stats,
                     const __grid_constant__ BwdOut<T> outs, int n_items, int n_rt) {
  using Geo = BwdGeo<kDP, kKeys, kABufs>;
  using Smem = BwdSmem<kDP, kKeys, kABufs>;
  constexpr uint32_t kStages = Geo::kStages, kBufs = Geo::kBufs;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                      ~uintptr_t(1023));
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const Waiter wait{&sm.abort, sh.err};

  // a cluster's piece takes the stationary tiles' memory once all are read
  static_assert(sizeof(sm.a1) + sizeof(sm.a2) >= (kKeys ? 2 : 1) * kRows * kDP * 4, "a piece there");

  if (threadIdx.x == 0) {
    for (int i = 0; i < kABufs; ++i) {
      mbar_init(&sm.a_full[i], 1);
      mbar_init(&sm.a_empty[i], 8);
    }
    for (uint32_t i = 0; i < kBufs; ++i) {
      mbar_init(&sm.s_full[i], 1);
      mbar_init(&sm.ds_full[i], 4);
      mbar_init(&sm.buf_free[i], 1);
    }
    for (uint32_t i = 0; i < kStages; ++i) {
      mbar_init(&sm.b_full[i], 1);
      mbar_init(&sm.b_empty[i], 1);
    }
    mbar_init(&sm.acc_full, 1);
    mbar_init(&sm.acc_free, 8);
    mbar_init(&sm.drain[0], 1);
    mbar_init(&sm.drain[1], 1);
    sm.abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc<512>(&sm.tmem_base);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  const uint32_t t_acc1 = tmem + Geo::kAcc, t_acc2 = t_acc1 + kDP;
  pdl_wait();
  pdl_trigger();

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (elect_one_sync()) {
      tma_prefetch_desc(&tm_a1);
      tma_prefetch_desc(&tm_a2);
      tma_prefetch_desc(&tm_b1);
      tma_prefetch_desc(&tm_b2);
      uint32_t n = 0, u = 0;
      bool ok = true;
      for (Walk item; item.at < n_items && ok; item.next()) {
        const BwdItem it = bwd_item<kKeys>(sh, item.at, n_rt);
        if (it.lo >= it.hi) continue;
        const uint32_t ab = n % kABufs;
        if (!(ok = wait(&sm.a_empty[ab], ((n / kABufs) & 1) ^ 1))) break;
        mbar_arrive_expect_tx(&sm.a_full[ab], 2 * Geo::kABytes);
        load_tile<kRows, kDP>(sm.a1[ab], &tm_a1, &sm.a_full[ab], it.row0, it.head, it.b);
        load_tile<kRows, kDP>(sm.a2[ab], &tm_a2, &sm.a_full[ab], it.row0, it.head, it.b);
        ++n;
        // keys: tile j is query tile `first + j % n` of head j / n of the group
        int row = (kKeys ? it.first + (it.lo > 0 ? it.lo % it.n : 0) : it.lo) * kBN;
        int head = kKeys ? it.head * sh.G + (it.lo > 0 ? it.lo / it.n : 0)
                         : (int)sh.by_group.div(it.head);
        for (int j = it.lo; j < it.hi; ++j, ++u) {
          const uint32_t st = u % kStages;
          if (!(ok = wait(&sm.b_empty[st], ((u / kStages) & 1) ^ 1))) break;
          mbar_arrive_expect_tx(&sm.b_full[st],
                                2 * Geo::kBBytes + (kKeys ? (uint32_t)sizeof(sm.stat[st]) : 0u));
          if (kKeys)
            bulk_load(sm.stat[st], stats + ((int64_t)it.b * sh.H + head) * stat_pitch(sh.Sq) + row,
                      sizeof(sm.stat[st]), &sm.b_full[st]);
          load_tile<kBN, kDP>(sm.b1[st], &tm_b1, &sm.b_full[st], row, head, it.b);
          load_tile<kBN, kDP>(sm.b2[st], &tm_b2, &sm.b_full[st], row, head, it.b);
          row += kBN;
          if (kKeys && row >= (it.first + it.n) * kBN) {
            row = it.first * kBN;
            ++head;
          }
        }
      }
      if (!ok) {
        for (uint32_t i = 0; i < kABufs; ++i) settle(&sm.a_full[i], (n + kABufs - 1 - i) / kABufs);
        for (uint32_t i = 0; i < kStages; ++i)
          settle(&sm.b_full[i], (u + kStages - 1 - i) / kStages);
      }
    }
    __syncwarp();
  } else if (warp == 1 && !Geo::kSplitMma) {
    // ------------------------------------------------------------ both MMAs
    if (elect_one_sync()) {
      constexpr uint32_t id_s = idesc(Type<T>::kIdesc, kRows, kBN, 0);
      constexpr uint32_t id_acc = idesc(Type<T>::kIdesc, kRows, kDP, 1);
      const uint32_t a10 = smem_u32(sm.a1[0]), a20 = smem_u32(sm.a2[0]);
      const uint32_t b10 = smem_u32(sm.b1[0]), b20 = smem_u32(sm.b2[0]);
      Ring<kStages> ss, as;  // stages of the tile whose scores come next, and of the products
      Ring<kBufs> sb, ab;    // their TMEM buffers
      Ring<kABufs> is;       // stationary pairs
      uint32_t m = 0;        // items whose products began
      bool ok = true, issued = false;
      // tiles whose products are still to come, the oldest's flags in bit 0
      uint32_t pending = 0, firsts = 0, lasts = 0;
      auto issue_acc = [&]() -> bool {
        const bool first = firsts & 1u, last = lasts & 1u;
        firsts >>= 1;
        lasts >>= 1;
        --pending;
        if (first) {  // the item before has been read out
          if (!wait(&sm.acc_free, (m & 1) ^ 1)) return false;
          ++m;
        }
        if (!wait(&sm.ds_full[ab.at], ab.phase)) return false;
        tc_fence_after();
        const uint32_t t_s = tmem + ab.at * 128u;
        const uint32_t b1 = b10 + as.at * Geo::kBBytes, b2 = b20 + as.at * Geo::kBBytes;
        if (kKeys) {
          mma_cols<kBN, kDP>(t_acc2, t_s, b2, id_acc, !first);
          mma_cols<kBN, kDP>(t_acc1, t_s + 64, b1, id_acc, !first);
        } else {
          mma_cols<kBN, kDP>(t_acc1, t_s, b1, id_acc, !first);
        }
        umma_commit(&sm.b_empty[as.at]);
        if (last) umma_commit(&sm.acc_full);
        ab.next();
        as.next();
        return true;
      };
      for (Walk item; item.at < n_items && ok; item.next()) {
        const BwdItem it = bwd_item<kKeys>(sh, item.at, n_rt);
        if (it.lo >= it.hi) continue;
        if (!(ok = wait(&sm.a_full[is.at], is.phase))) break;
        const uint32_t a1 = a10 + is.at * Geo::kABytes, a2 = a20 + is.at * Geo::kABytes;
        for (int j = it.lo; j < it.hi; ++j) {
          if (!(ok = wait(&sm.b_full[ss.at], ss.phase))) break;
          tc_fence_after();
          // this buffer's last product (kBufs tiles ago) was issued before: in order
          const uint32_t t_s = tmem + sb.at * 128u;
          mma_rows<kRows, kBN, kDP>(t_s, a1, b10 + ss.at * Geo::kBBytes, id_s);
          mma_rows<kRows, kBN, kDP>(t_s + 64, a2, b20 + ss.at * Geo::kBBytes, id_s);
          issued = true;
          umma_commit(&sm.s_full[sb.at]);
          ss.next();
          sb.next();
          firsts |= (j == it.lo ? 1u : 0u) << pending;
          lasts |= (j == it.hi - 1 ? 1u : 0u) << pending;
          if (++pending == kBufs && !(ok = issue_acc())) break;
        }
        is.next();
      }
      while (ok && pending) ok = issue_acc();
      if (!ok && issued) {
        umma_commit(&sm.drain[0]);
        settle(&sm.drain[0], 1);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ scores' MMA
    if (elect_one_sync()) {
      constexpr uint32_t id_s = idesc(Type<T>::kIdesc, kRows, kBN, 0);
      const uint32_t a10 = smem_u32(sm.a1[0]), a20 = smem_u32(sm.a2[0]);
      const uint32_t b10 = smem_u32(sm.b1[0]), b20 = smem_u32(sm.b2[0]);
      Ring<kStages> ss;
      Ring<kBufs> sb;
      Ring<kABufs> is;
      bool ok = true, issued = false;
      for (Walk item; item.at < n_items && ok; item.next()) {
        const BwdItem it = bwd_item<kKeys>(sh, item.at, n_rt);
        if (it.lo >= it.hi) continue;
        if (!(ok = wait(&sm.a_full[is.at], is.phase))) break;
        const uint32_t a1 = a10 + is.at * Geo::kABytes, a2 = a20 + is.at * Geo::kABytes;
        for (int j = it.lo; j < it.hi; ++j) {
          if (!(ok = wait(&sm.b_full[ss.at], ss.phase))) break;
          // the products with this buffer's last dS are complete
          if (!(ok = wait(&sm.buf_free[sb.at], sb.phase ^ 1))) break;
          tc_fence_after();
          const uint32_t t_s = tmem + sb.at * 128u;
          mma_rows<kRows, kBN, kDP>(t_s, a1, b10 + ss.at * Geo::kBBytes, id_s);
          mma_rows<kRows, kBN, kDP>(t_s + 64, a2, b20 + ss.at * Geo::kBBytes, id_s);
          issued = true;
          umma_commit(&sm.s_full[sb.at]);
          ss.next();
          sb.next();
        }
        is.next();
      }
      if (!ok && issued) {
        umma_commit(&sm.drain[0]);
        settle(&sm.drain[0], 1);
      }
    }
    __syncwarp();
  } else if (warp == 10) {
    // ------------------------------------------------------------ products' MMA
    if (elect_one_sync()) {
      constexpr uint32_t id_acc = idesc(Type<T>::kIdesc, kRows, kDP, 1);
      const uint32_t b10 = smem_u32(sm.b1[0]), b20 = smem_u32(sm.b2[0]);
      Ring<kStages> ss;
      Ring<kBufs> sb;
      uint32_t n = 0;
      bool ok = true, issued = false;
      for (Walk item; item.at < n_items && ok; item.next()) {
        const BwdItem it = bwd_item<kKeys>(sh, item.at, n_rt);
        if (it.lo >= it.hi) continue;
        // the item before has been read out
        if (!(ok = wait(&sm.acc_free, (n & 1) ^ 1))) break;
        ++n;
        for (int j = it.lo; j < it.hi; ++j) {
          if (!(ok = wait(&sm.b_full[ss.at], ss.phase))) break;
          if (!(ok = wait(&sm.ds_full[sb.at], sb.phase))) break;
          tc_fence_after();
          const uint32_t t_s = tmem + sb.at * 128u;
          const uint32_t b1 = b10 + ss.at * Geo::kBBytes, b2 = b20 + ss.at * Geo::kBBytes;
          if (kKeys) {
            mma_cols<kBN, kDP>(t_acc2, t_s, b2, id_acc, j > it.lo);
            mma_cols<kBN, kDP>(t_acc1, t_s + 64, b1, id_acc, j > it.lo);
          } else {
            mma_cols<kBN, kDP>(t_acc1, t_s, b1, id_acc, j > it.lo);
          }
          issued = true;
          umma_commit(&sm.buf_free[sb.at]);
          umma_commit(&sm.b_empty[ss.at]);
          if (j == it.hi - 1) umma_commit(&sm.acc_full);
          ss.next();
          sb.next();
        }
      }
      if (!ok && issued) {
        umma_commit(&sm.drain[1]);
        settle(&sm.drain[1], 1);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ compute
    const int group = (warp - 2) >> 2;
    const int r = (warp & 3) * 32 + lane;  // row within the tile
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint64_t sl2x2 = f2_splat(sh.scale * kLog2e);
    constexpr float kShift = kKeys ? Type<T>::kShift : 0.f;
    const float unshift = exp2f(-kShift);
    Ring<kStages> ss;
    Ring<kBufs> sb;
    Ring<kABufs> is;
    uint32_t turn = 0, n = 0;
    bool ok = true;
    // The stationary buffer whose output store may still be read (see forward)
    uint64_t* owed = nullptr;
    auto give_back = [&]() {
      if (owed != nullptr && lane == 0) {
        bulk_wait_group_read<0>();
        mbar_arrive(owed);
      }
      owed = nullptr;
    };
    // row statistics (queries; negated) or the row's visibility (keys) of an item
    auto row_of = [&](const BwdItem& x) {
      float2 v = make_float2(-INFINITY, 0.f);
      const int row = x.row0 + r;
      if (!kKeys) {
        if (x.lo < x.hi && row < sh.Sq)
          v = __ldg(stats + ((int64_t)x.b * sh.H + x.head) * stat_pitch(sh.Sq) + row);
      } else {
        bool visible = row < sh.Sk;
        if (visible && sh.words)
          visible = (__ldg(sh.words + (int64_t)x.b * sh.nwords + row / 32) >> (row & 31)) & 1u;
        v.y = visible ? 1.f : 0.f;
      }
      return v;
    };
    // the exponent at which dS of an item (queries: of its row) is formed
    auto shift_of = [&](const BwdItem& x) {
      if constexpr (Type<T>::kRanged) {
        if (x.lo >= x.hi) return 0;
        const int64_t unit = (int64_t)x.b * sh.Hk + (kKeys ? (uint32_t)x.head : sh.by_group.div(x.head));
        auto most = [&](const uint32_t* of) {
          return __uint_as_float(__reduce_max_sync(
              0xffffffffu, lane < outs.range.parts ? __ldg(of + unit * outs.range.parts + lane) : 0u));
        };
        float d2 = 0.f;
        if (kKeys)
          d2 = most(outs.range.d_max);
        else if (x.row0 + r < sh.Sq)
          d2 = __ldg(outs.range.norms + ((int64_t)x.b * sh.H + x.head) * stat_pitch(sh.Sq) + x.row0 + r);
        return range_shift(d2, most(outs.range.v_max));
      }
      return 0;
    };
    BwdItem after = bwd_item<kKeys>(sh, blockIdx.x, n_rt);
    float2 after_row = row_of(after);
    int after_shift = shift_of(after);
    for (Walk item; item.at < n_items && ok; item.next()) {
      const BwdItem it = after;
      const int row = it.row0 + r;
      const bool any = it.lo < it.hi;
      // 2^shift dS: queries by P's exponent, keys (where P is wanted too) by dP's factor
      const int shift = after_shift;
      const uint64_t row_lse = f2_splat(kKeys ? after_row.x : after_row.x + (float)shift);
      const uint64_t row_delta = f2_splat(after_row.y);
      const uint64_t d_factor = f2_splat(kShift != 0.f ? exp2f((float)shift - kShift) : 1.f);
      const bool row_ok = !kKeys || after_row.y != 0.f;
      const bool rows_ok = __all_sync(0xffffffffu, row_ok);
      // the CTA's tiles alternate between the groups: mine is every second one
      int col0 = (kKeys ? it.first + (it.lo > 0 ? it.lo % it.n : 0) : it.lo) * kBN;
      for (int j = it.lo; j < it.hi; ++j) {
        const bool mine = turn == (uint32_t)group;
        const uint32_t stage = ss.at, sphase = ss.phase, buf = sb.at, bphase = sb.phase;
        const int col = col0;
        turn ^= 1;
        ss.next();
        sb.next();
        col0 += kBN;
        if (kKeys && col0 >= (it.first + it.n) * kBN) col0 = it.first * kBN;
        if (!mine) continue;
        const uint32_t t_s = tmem + lanes + buf * 128u;
        // the statistics came with the tile (already complete: S was computed)
        ok = !kKeys || wait(&sm.b_full[stage], sphase);
        ok = ok && wait(&sm.s_full[buf], bphase);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        tc_fence_after();
        uint2 words = make_uint2(0xffffffffu, 0xffffffffu);
        if (!kKeys && (sh.words || col + kBN > sh.Sk)) words = tile_words(sh, it.b, col);
        const bool diag = sh.causal && (kKeys ? col < it.row0 + kRows - 1
                                              : col + kBN - 1 > it.row0);
        // P and dS as 16-bit pairs, 16 columns at a time with the next 16 on
        // their way from TMEM. Hidden pairs are replaced by zero, whatever the
        // products gave.
        auto columns = [&](auto masked) {
          uint32_t rs[2][16], rd[2][16];
          tmem_ld_16cols(t_s, rs[0]);
          tmem_ld_16cols(t_s + 64, rd[0]);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            tmem_ld_wait();
            if (c < 3) {
              tmem_ld_16cols(t_s + (c + 1) * 16, rs[(c + 1) & 1]);
              tmem_ld_16cols(t_s + 64 + (c + 1) * 16, rd[(c + 1) & 1]);
            }
            const uint32_t (&s16)[16] = rs[c & 1];
            const uint32_t (&d16)[16] = rd[c & 1];
            uint32_t pk[8], dk[8];
            const uint32_t wc = (c < 2 ? words.x : words.y) >> (c % 2 * 16);
            const int lim = row - (col + c * 16);  // causal: key <= query
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              uint64_t nl = row_lse, nd = row_delta;
              if (kKeys) {
                const float4 v = *reinterpret_cast<const float4*>(&sm.stat[stage][c * 16 + i]);
                nl = f2_pack(v.x, v.z);
                nd = f2_pack(v.y, v.w);
              }
              uint64_t e =
                  f2_fma(f2_pack(__uint_as_float(s16[i]), __uint_as_float(s16[i + 1])), sl2x2, nl);
              if (kShift != 0.f) e = f2_add(e, f2_splat(kShift));
              float p0, p1, d0, d1;
              exp2_pair<!kKeys && Type<T>::kCubic>(e, i / 2, p0, p1);
              uint64_t d = f2_add(f2_pack(__uint_as_float(d16[i]), __uint_as_float(d16[i + 1])), nd);
              if (kShift != 0.f) d = f2_mul(d, d_factor);
              f2_unpack(f2_mul(f2_pack(p0, p1), d), d0, d1);
              if (decltype(masked)::value) {
                bool v0 = row_ok && ((wc >> i) & 1u), v1 = row_ok && ((wc >> (i + 1)) & 1u);
                if (diag) {
                  v0 = v0 && (kKeys ? i >= lim : i <= lim);
                  v1 = v1 && (kKeys ? i + 1 >= lim : i + 1 <= lim);
                }
                p0 = v0 ? p0 : 0.f;
                p1 = v1 ? p1 : 0.f;
                d0 = v0 ? d0 : 0.f;
                d1 = v1 ? d1 : 0.f;
              }
              if (kKeys) pk[i / 2] = Type<T>::pack(p0, p1);
              dk[i / 2] = Type<T>::pack(d0, d1);
            }
            if (kKeys) tmem_st_8cols(t_s + c * 8, pk);
            tmem_st_8cols(t_s + (kKeys ? 64u : 0u) + c * 8, dk);
          }
        };
        if (diag || !rows_ok || !is_whole(words))
          columns(std::true_type{});
        else
          columns(std::false_type{});
        if (!kKeys && sh.words && !is_whole(words))
          zero_hidden_rows<kBN, kDP>(sm.b1[stage], words, (warp & 3) * 32 + lane, 128);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.ds_full[buf]);
        give_back();
      }
      if (!ok) break;
      // the next item, and its row's load, while the last product runs
      after = bwd_item<kKeys>(sh, item.after(), n_rt);
      after_row = row_of(after);
      after_shift = shift_of(after);
      // A group without a tile in this item gives the buffer back here, before it waits
      // for the products: of items of one tile each, these may come behind scores
      // that need the buffer.
      give_back();
      // ---- read the accumulators out
      if (any) {
        ok = wait(&sm.acc_full, n & 1);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        tc_fence_after();
        ++n;
      }
      // keys: group 0 takes dV, group 1 dK; queries: 64 of dQ's columns each (one
      // group at head size 64)
      const bool second = kKeys && group == 0;
      const uint32_t t_a = (second ? t_acc2 : t_acc1) + lanes;
      const float f = second ? unshift : Type<T>::kRanged ? sh.scale * exp2f((float)-shift) : sh.scale;
      if (any && !kSplit) {
        uint8_t* block = (second ? sm.a2[is.at] : sm.a1[is.at]) + (warp & 3) * 4096;
#pragma unroll 1
        for (int c = kKeys ? 0 : group; c < kDP / 64; c += kKeys ? 1 : 2)
          stage_rows<T, false>(t_a + c * 64, lane, true, f, block + c * kRows * 128);
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) {
          for (int c = kKeys ? 0 : group; c * 64 < sh.D; c += kKeys ? 1 : 2)
            tma_store_4d(second ? &tm_o2 : &tm_o1, block + c * kRows * 128, c * 64, row - lane, it.head,
                         it.b);
          bulk_commit_group();
        }
      } else if (kSplit && outs.part == nullptr) {  // a cluster's piece
        float* to = reinterpret_cast<float*>(sm.a1) + (second ? kRows * kDP : 0);
        const int c1 = kKeys ? kDP : (group + 1) * (kDP / 2);
#pragma unroll 1
        for (int c = kKeys ? 0 : group * (kDP / 2); c < c1; c += 16) {
          float v[16];
          row16(t_a + c, any, true, f, v);
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            *reinterpret_cast<float4*>(to + piece_at<kDP>(r, (c + i) / 4)) =
                make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        }
      } else if (kKeys || group == 0) {
        const int rows_n = kKeys ? sh.Sk : sh.Sq, heads = kKeys ? sh.Hk : sh.H;
        const int64_t flat = ((int64_t)it.b * rows_n + row) * heads + it.head;
        const int64_t rows_all = (int64_t)sh.B * rows_n * heads;
        const Stride3 st3 = second ? outs.s2 : outs.s1;
        T* dst = (second ? outs.o2 : outs.o1) + it.b * st3.b + (int64_t)row * st3.s + it.head * st3.h;
        float* part = !kSplit ? nullptr
                                     : outs.part + ((int64_t)it.split * (kKeys ? 2 : 1) + (second ? 1 : 0)) *
                                                       rows_all * sh.D + flat * sh.D;
        store_row<T>(t_a, sh.D, any, true, row < rows_n, f, dst, (T*)nullptr, part);
      }
      if (any) {
        owed = &sm.a_empty[is.at];
        if (kABufs == 1) give_back();
        is.next();
      }
      if (any) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.acc_free);
      }
    }
    if (lane == 0) bulk_wait_group<0>();
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<512>(tmem);
  }
  if (kSplit && outs.part == nullptr) {  // one item per CTA
    const BwdItem it = bwd_item<kKeys>(sh, blockIdx.x, n_rt);
    const int rows = min(kRows, (kKeys ? sh.Sk : sh.Sq) - it.row0);
    __syncwarp();  // an aligned barrier
    cluster_sync_all();
    for (int which = 0; which < (kKeys ? 2 : 1); ++which) {
      const Stride3& st3 = which ? outs.s2 : outs.s1;
      T* dst = (which ? outs.o2 : outs.o1) + it.b * st3.b + (int64_t)it.row0 * st3.s + it.head * st3.h;
      cluster_sum<kDP>(reinterpret_cast<float*>(sm.a1) + which * kRows * kDP, rows, sh.D, sh.splits,
                       [&](int r, int c, float4 v) {
                         *reinterpret_cast<uint2*>(dst + (int64_t)r * st3.s + 4 * c) =
                             make_uint2(Type<T>::pack(v.x, v.y), Type<T>::pack(v.z, v.w));
                       });
    }
    __syncwarp();
    cluster_sync_all();  // no CTA leaves while others read its rows
  }
}

// out = the sum of the pieces, in order: part [splits][n_out][rows][D], rows
// (b, i, h). Eight columns per thread.
template <typename T>
__global__ void __launch_bounds__(256) cross_sum_kernel(const __grid_constant__ BwdOut<T> outs,
                                                        int splits, int n_out, int B, int S, int H,
                                                        int D) {
  pdl_wait();
  pdl_trigger();
  const int64_t rows = (int64_t)B * S * H, vec = D / 8, total = rows * vec * n_out;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * 256) {
    const int64_t which = i / (rows * vec), rest = i - which * rows * vec;
    const int64_t row = rest / vec;
    const int col = (int)(rest - row * vec) * 8;
    float a[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) a[k] = 0.f;
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
      const float4* p = reinterpret_cast<const float4*>(
          outs.part + (((int64_t)s * n_out + which) * rows + row) * D + col);
      const float4 x = p[0], y = p[1];
      a[0] += x.x; a[1] += x.y; a[2] += x.z; a[3] += x.w;
      a[4] += y.x; a[5] += y.y; a[6] += y.z; a[7] += y.w;
    }
    const int64_t bi = row / H, h = row - bi * H, b = bi / S, s = bi - b * S;
    const Stride3& st = which ? outs.s2 : outs.s1;
    *reinterpret_cast<uint4*>((which ? outs.o2 : outs.o1) + b * st.b + s * st.s + h * st.h + col) =
        make_uint4(Type<T>::pack(a[0], a[1]), Type<T>::pack(a[2], a[3]), Type<T>::pack(a[4], a[5]),
                   Type<T>::pack(a[6], a[7]));
  }
}

// ============================================================== host
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                   const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// cuTensorMapEncodeTiled is a driver call: it needs a context current on the
// calling thread (an autograd thread may not have one before its first launch).
EncodeTiledFn encode_fn() {
  thread_local int bound = -1;
  int dev = 0;
  if (cudaGetDevice(&dev) == cudaSuccess && bound != dev) {
    cudaSetDevice(dev);
    bound = dev;
  }
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

}  // namespace

// Map {D, position, head, batch} of a strided 16-bit tensor; box = 64 columns x
// `rows` positions. The stride of a dimension of one does not matter: any valid
// value goes.
bool cross_attn_map(CUtensorMap* m, const void* base, bool half, int D, int S, int heads, int B,
              const int64_t (&st)[3], int rows) {
  auto enc = encode_fn();
  if (!enc) return false;
  const int n[3] = {S, heads, B};
  const int64_t e[3] = {st[1], st[2], st[0]};
  cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)S, (cuuint64_t)heads, (cuuint64_t)B};
  cuuint64_t strides[3];
  for (int i = 0; i < 3; ++i) {
    const int64_t bytes = n[i] > 1 ? e[i] * 2 : 256;
    if (bytes <= 0 || bytes % 16 || bytes >= ((int64_t)1 << 40)) return false;
    strides[i] = (cuuint64_t)bytes;
  }
  cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1};
  cuuint32_t es[4] = {1, 1, 1, 1};
  return enc(m, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
             const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

cudaError_t cross_attn_opt_in(const void* kernel, size_t smem, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                             cudaSharedmemCarveoutMaxShared);
  if (e == cudaSuccess)  // clusters of more than 8 CTAs
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) done.fetch_or(bit);
  return e;
}

int64_t cross_attn_clusters(const void* kernel, int threads, size_t smem, int size,
                            CrossFits& fits) {
  if (size < 2) return INT64_MAX;
  int n = fits[size].load(std::memory_order_relaxed);
  if (n == 0) {
    cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                         cudaSharedmemCarveoutMaxShared);
    cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(size);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) {
      cudaGetLastError();
      n = -1;  // none
    }
    fits[size].store(n, std::memory_order_relaxed);
  }
  return n;
}

namespace {

// `heads` of the rows that an item's index runs over.
Shape shape_of(const CrossAttnArgs& a, int splits, int heads, int64_t items) {
  Shape s{};
  s.B = a.B; s.Sq = a.Sq; s.Sk = a.Sk; s.H = a.H; s.Hk = a.Hk; s.G = a.H / a.Hk; s.D = a.D;
  s.causal = a.causal;
  s.splits = splits;
  s.n_items = (int)items;
  s.scale = a.scale;
  s.words = a.key_pad ? a.words : nullptr;
  s.vis_end = a.key_pad ? a.vis_end : nullptr;
  s.nwords = (a.Sk + 31) / 32;
  s.err = default_err_word();
  s.by_splits = FastDiv((uint32_t)splits);
  // row tiles of an item's head: items / (pieces * heads * samples)
  const int64_t tiles = items / ((int64_t)splits * heads * a.B);
  s.by_outer = FastDiv((uint32_t)(heads * (a.causal ? a.B : tiles)));
  s.by_heads = FastDiv((uint32_t)heads);
  s.by_group = FastDiv((uint32_t)s.G);
  return s;
}

bool bad_shape(const CrossAttnArgs& a) {
  return a.B <= 0 || a.Sq <= 0 || a.Sk <= 0 || a.H <= 0 || a.Hk <= 0 || a.H % a.Hk || a.D <= 0 ||
         a.D > 128 || a.D % 8 || (a.causal && a.Sq != a.Sk) || !(a.scale > 0.f) ||
         (int64_t)a.H * a.B > 0x3fffffff ||
         (a.key_pad && !cross_attn_is_few(a) && (!a.words || !a.vis_end));
}

// Pieces of the streamed axis: fewer items than places take as many pieces as
// fill them, as long as a piece keeps four tiles (the pieces cost a join).
int pieces(int64_t items, int64_t places, int64_t tiles) {
  if (items >= places) return 1;
  return (int)std::max<int64_t>(1, std::min(places / items, tiles / 4));
}
int64_t row_tiles(int n) { return ((int64_t)n + kRows - 1) / kRows; }

// Clusters of the forward kernel that the GPU holds. The runtime counts one CTA per
// SM (it rounds six warps up to eight); two fit, so twice as many clusters.
template <int kDP>
int64_t fwd_clusters(int size) {
  static CrossFits fits{};
  if (size < 2) return INT64_MAX;
  return kFwdCtas * cross_attn_clusters((const void*)cross_fwd_kernel<__nv_bfloat16, kDP, false>,
                                        kFwdThreads, sizeof(FwdSmem<kDP, false>) + 1024, size, fits);
}
CrossSplits fwd_splits(const CrossAttnArgs& a) {
  const int64_t items = row_tiles(a.Sq) * a.H * a.B;
  const int64_t tiles = ((int64_t)a.Sk + kN - 1) / kN;
  const int want = pieces(items, (int64_t)kFwdCtas * num_sms(), tiles);
  // as many as a cluster joins and the GPU holds at once (98 items of 128 x 1500 x 64:
  // 21 us with two pieces each, 27 with three and a second kernel)
  int s = std::min(want, kCrossTileCluster);
  while (s > 1 && items > (a.D > 64 ? fwd_clusters<128>(s) : fwd_clusters<64>(s))) --s;
  if (cross_attn_joins_more(items, s, kCrossTileCluster, want, tiles, num_sms())) return {want, false};
  return {s, s > 1};
}
// Both halves of the backward have one CTA per SM.
CrossSplits bwd_splits(int64_t items, int64_t tiles) {
  static CrossFits fits{};
  const int want = pieces(items, num_sms(), tiles);
  int s = std::min(want, kCrossTileCluster);
  using G = BwdGeo<64, true, 2>;
  while (s > 1 && items > cross_attn_clusters((const void*)cross_bwd_kernel<__nv_bfloat16, 64, true, 2, true>,
                                              G::kThreads, sizeof(BwdSmem<64, true, 2>) + 1024, s, fits))
    --s;
  if (cross_attn_joins_more(items, s, kCrossTileCluster, want, tiles, num_sms())) return {want, false};
  return {s, s > 1};
}
CrossSplits dq_splits(const CrossAttnArgs& a) {
  return bwd_splits(row_tiles(a.Sq) * a.H * a.B, ((int64_t)a.Sk + kBN - 1) / kBN);
}
CrossSplits dkv_splits(const CrossAttnArgs& a) {
  return bwd_splits(row_tiles(a.Sk) * a.Hk * a.B, ((int64_t)a.Sq + kBN - 1) / kBN * (a.H / a.Hk));
}

// Parts of the keys in cross_range_kernel: as many CTAs as eight to an SM, with four
// rows a lane or more.
int range_parts(const CrossAttnArgs& a) {
  const int64_t units = (int64_t)a.B * a.Hk, rows = (a.D <= 64 ? 32 : 16) * 4;
  return (int)std::max<int64_t>(
      1, std::min<int64_t>({kRangeParts, num_sms() * 8 / units, (a.Sk + rows - 1) / rows}));
}
// The scratch of `stats`: the row statistics, then (f16) the norms of dO's rows, the
// maxima of their parts and those of V's.
Range range_of(const CrossAttnArgs& a) {
  Range r{};
  if (!a.half) return r;
  const int64_t rows = (int64_t)a.B * a.H * stat_pitch(a.Sq);
  r.norms = a.stats + 2 * rows;
  r.d_max = reinterpret_cast<const uint32_t*>(r.norms + rows);
  r.parts = range_parts(a);
  r.v_max = r.d_max + (int64_t)a.B * a.Hk * r.parts;
  return r;
}

template <typename T, int kDP, bool kTrain>
cudaError_t run_fwd(const CrossAttnArgs& a, cudaStream_t st) {
  const CrossSplits plan = fwd_splits(a);
  const int splits = plan.n;
  const int64_t rows = (int64_t)a.B * a.Sq * a.H;
  const bool joined = plan.joined();
  if (joined && !a.partials) return cudaErrorInvalidValue;
  CUtensorMap mq, mk, mv, mo, mr;
  const int64_t o_st[3] = {(int64_t)a.Sq * a.H * a.D, (int64_t)a.H * a.D, a.D};
  if (!cross_attn_map(&mq, a.q, a.half, a.D, a.Sq, a.H, a.B, a.q_st, kRows) ||
      !cross_attn_map(&mo, a.out, a.half, a.D, a.Sq, a.H, a.B, o_st, 32) ||
      (a.out_res && !cross_attn_map(&mr, a.out_res, a.half, a.D, a.Sq, a.H, a.B, o_st, 32)) ||
      !cross_attn_map(&mk, a.k, a.half, a.D, a.Sk, a.Hk, a.B, a.k_st, kN) ||
      !cross_attn_map(&mv, a.v, a.half, a.D, a.Sk, a.Hk, a.B, a.v_st, kN))
    return cudaErrorInvalidValue;
  static std::atomic<uint64_t> done{0};
  const int smem = (int)sizeof(FwdSmem<kDP, kTrain>) + 1024;
  auto kernel = cross_fwd_kernel<T, kDP, kTrain>;
  cudaError_t e = cross_attn_opt_in((const void*)kernel, smem, done);
  if (e != cudaSuccess) return e;
  const int n_qt = (int)row_tiles(a.Sq);
  const int64_t items = (int64_t)n_qt * a.H * a.B * splits;
  if (items > 0x7fffffff - 4096) return cudaErrorInvalidValue;
  const int grid = (int)std::min<int64_t>(items, (int64_t)kFwdCtas * num_sms());
  // (several pieces: one item per CTA, as many items as places at most)
  e = launch_pdl_cluster(kernel, dim3(grid), dim3(kFwdThreads), plan.clustered ? splits : 1, smem, st, mq,
                         mk, mv, mo, a.out_res ? mr : mo, shape_of(a, splits, a.H, items), (T*)a.out,
                         (T*)a.out_res, a.lse2, joined ? a.partials : nullptr,
                         joined ? a.partials + splits * rows * a.D : nullptr, (int)items, n_qt);
  if (e != cudaSuccess) return e;
  note_launch();
  return joined ? launch_cross_attn_join(a, splits, st) : cudaGetLastError();
}

template <typename T, int kDP, bool kKeys, int kABufs, bool kSplit>
cudaError_t run_bwd_half(const CrossAttnArgs& a, const CrossSplits& plan, cudaStream_t st) {
  const int splits = plan.n;
  if (plan.joined() && !a.partials) return cudaErrorInvalidValue;
  const int rb = kRows, cb = kBN;
  CUtensorMap mq, mk, mv, mo;
  if (!cross_attn_map(&mq, a.q, a.half, a.D, a.Sq, a.H, a.B, a.q_st, kKeys ? cb : rb) ||
      !cross_attn_map(&mo, a.dout, a.half, a.D, a.Sq, a.H, a.B, a.do_st, kKeys ? cb : rb) ||
      !cross_attn_map(&mk, a.k, a.half, a.D, a.Sk, a.Hk, a.B, a.k_st, kKeys ? rb : cb) ||
      !cross_attn_map(&mv, a.v, a.half, a.D, a.Sk, a.Hk, a.B, a.v_st, kKeys ? rb : cb))
    return cudaErrorInvalidValue;
  CUtensorMap m1, m2;
  if (!(kKeys ? cross_attn_map(&m1, a.dk, a.half, a.D, a.Sk, a.Hk, a.B, a.dk_st, 32) &&
                    cross_attn_map(&m2, a.dv, a.half, a.D, a.Sk, a.Hk, a.B, a.dv_st, 32)
              : cross_attn_map(&m1, a.dq, a.half, a.D, a.Sq, a.H, a.B, a.dq_st, 32)))
    return cudaErrorInvalidValue;
  static std::atomic<uint64_t> done{0};
  constexpr int smem = (int)sizeof(BwdSmem<kDP, kKeys, kABufs>) + 1024;
  static_assert(smem <= 227 * 1024, "shared memory");
  auto kernel = cross_bwd_kernel<T, kDP, kKeys, kABufs, kSplit>;
  cudaError_t e = cross_attn_opt_in((const void*)kernel, smem, done);
  if (e != cudaSuccess) return e;
  const int S = kKeys ? a.Sk : a.Sq, heads = kKeys ? a.Hk : a.H;
  const int n_rt = (int)row_tiles(S);
  const int64_t items = (int64_t)n_rt * heads * a.B * splits;
  if (items > 0x7fffffff - 4096) return cudaErrorInvalidValue;
  BwdOut<T> o{};
  auto s3 = [](const int64_t (&v)[3]) { return Stride3{v[0], v[1], v[2]}; };
  o.o1 = (T*)(kKeys ? a.dk : a.dq);
  o.s1 = kKeys ? s3(a.dk_st) : s3(a.dq_st);
  o.o2 = kKeys ? (T*)a.dv : o.o1;
  o.s2 = kKeys ? s3(a.dv_st) : o.s1;
  o.part = plan.joined() ? a.partials : nullptr;
  o.range = range_of(a);
  const int grid = (int)std::min<int64_t>(items, num_sms());
  e = launch_pdl_cluster(kernel, dim3(grid), dim3(BwdGeo<kDP, kKeys, kABufs>::kThreads),
                         plan.clustered ? splits : 1, smem, st, kKeys ? mk : mq, kKeys ? mv : mo,
                         kKeys ? mq : mk, kKeys ? mo : mv, m1, kKeys ? m2 : m1,
                         shape_of(a, splits, heads, items), (const float2*)a.stats, o, (int)items, n_rt);
  if (e != cudaSuccess) return e;
  note_launch();
  if (plan.joined()) {
    const int n_out = kKeys ? 2 : 1;
    const int64_t total = (int64_t)a.B * S * heads * (a.D / 8) * n_out;
    e = launch_pdl(cross_sum_kernel<T>,
                   dim3((unsigned)std::min<int64_t>((total + 255) / 256, num_sms() * 8ll)), dim3(256),
                   0, st, o, splits, n_out, a.B, S, heads, a.D);
    if (e != cudaSuccess) return e;
    note_launch();
  }
  return cudaGetLastError();
}

template <typename T>
cudaError_t run_range(const CrossAttnArgs& a, const Range& r, cudaStream_t st) {
  const uint32_t units = (uint32_t)a.B * (uint32_t)a.Hk;
  auto k = a.D <= 64 ? cross_range_kernel<T, 8> : cross_range_kernel<T, 16>;
  cudaError_t e = launch_pdl(k, dim3(r.parts, std::min(units, 65535u)), dim3(256), 0, st, (const T*)a.v,
                             Stride3{a.v_st[0], a.v_st[1], a.v_st[2]},
                             (const uint32_t*)(a.key_pad ? a.words : nullptr),
                             (const int*)(a.key_pad ? a.vis_end : nullptr), a.Sk, FastDiv((uint32_t)a.Hk),
                             units, a.D, r.norms, (int64_t)stat_pitch(a.Sq) * (a.H / a.Hk),
                             const_cast<uint32_t*>(r.d_max), const_cast<uint32_t*>(r.v_max));
  if (e != cudaSuccess) return e;
  note_launch();
  return cudaGetLastError();
}

template <typename T>
cudaError_t run_stats(const CrossAttnArgs& a, cudaStream_t st) {
  const int64_t rows = (int64_t)stat_pitch(a.Sq) * a.H;  // of a sample
  if (rows >= kMaxFlatIndex - (1 << 24)) return cudaErrorInvalidValue;  // (over 170 GB of tensors)
  const int per = (a.D <= 64 ? 32 : 16) * kRowsAhead;
  const int64_t x = std::min<int64_t>((rows + per - 1) / per, num_sms() * 16ll);
  const int64_t y = std::min<int64_t>({a.B, std::max<int64_t>(1, num_sms() * 16ll / x), 65535});
  const Range r = range_of(a);
  const dim3 grid((unsigned)x, (unsigned)y);
  const Stride3 ds{a.do_st[0], a.do_st[1], a.do_st[2]};
  auto k = a.D <= 64 ? cross_stats_kernel<T, 8> : cross_stats_kernel<T, 16>;
  cudaError_t e = launch_pdl(k, grid, dim3(256), 0, st, (const T*)a.out,
                             (const T*)a.out_res, (const T*)a.dout, ds,
                             (const float*)a.lse2, (float2*)a.stats, const_cast<float*>(r.norms), a.B,
                             a.Sq, FastDiv((uint32_t)a.H), a.D);
  if (e != cudaSuccess) return e;
  note_launch();
  if constexpr (Type<T>::kRanged) return run_range<T>(a, r, st);
  return cudaGetLastError();
}

constexpr int kLongItem = 1024;  // keys of a query tile (half of them under a causal mask)
template <typename T, int kDP>
cudaError_t run_dq(const CrossAttnArgs& a, cudaStream_t st) {
  const CrossSplits plan = dq_splits(a);
  // At head size 128 the queries' kernel has room for two stationary pairs and
  // three stages or for one and five: the second where items are long (96 instead of
  // 105 us on 32 x 12 heads, 256 x 1024, but 60.7 instead of 59.5 at 256 x 512; causal 207
  // instead of 219 at 4096, 82 instead of 79 at 1024), or one to a CTA.
  if constexpr (kDP == 128) {
    if (plan.n > 1) return run_bwd_half<T, kDP, false, 1, true>(a, plan, st);
    return (a.causal ? a.Sk / 2 : a.Sk) >= kLongItem
               ? run_bwd_half<T, kDP, false, 1, false>(a, plan, st)
               : run_bwd_half<T, kDP, false, 2, false>(a, plan, st);
  } else {
    return plan.n > 1 ? run_bwd_half<T, kDP, false, 2, true>(a, plan, st)
                      : run_bwd_half<T, kDP, false, 2, false>(a, plan, st);
  }
}
template <typename T, int kDP>
cudaError_t run_dkv(const CrossAttnArgs& a, cudaStream_t st) {
  const CrossSplits plan = dkv_splits(a);
  return plan.n > 1 ? run_bwd_half<T, kDP, true, 2, true>(a, plan, st)
                    : run_bwd_half<T, kDP, true, 2, false>(a, plan, st);
}
template <typename T, int kDP>
cudaError_t run_bwd(const CrossAttnArgs& a, cudaStream_t st) {
  cudaError_t e = run_stats<T>(a, st);
  if (e == cudaSuccess && a.dq) e = run_dq<T, kDP>(a, st);
  if (e == cudaSuccess && a.dk) e = run_dkv<T, kDP>(a, st);
  return e;
}

}  // namespace

int64_t cross_attn_stats_floats(const CrossAttnArgs& a) {
  const int64_t rows = (int64_t)a.B * a.H * stat_pitch(a.Sq);
  if (!a.half) return 2 * rows;
  return 3 * rows + ((int64_t)a.B * a.Hk * 2 * range_parts(a) + 3) / 4 * 4;  // (what follows is 16-byte aligned)
}
int64_t cross_attn_fwd_partials(const CrossAttnArgs& a) {
  const CrossSplits s = cross_attn_is_few(a) ? cross_attn_few_splits(a) : fwd_splits(a);
  return s.joined() ? (int64_t)s.n * a.B * a.Sq * a.H * (a.D + 1) : 0;
}
// The two halves run one after the other and use the same scratch.
int64_t cross_attn_bwd_partials(const CrossAttnArgs& a) {
  const CrossSplits sq = dq_splits(a), sk = dkv_splits(a);
  const int64_t nq = a.dq && sq.joined() ? (int64_t)sq.n * a.B * a.Sq * a.H * a.D : 0;
  const int64_t nk = a.dk && sk.joined() ? (int64_t)sk.n * 2 * a.B * a.Sk * a.Hk * a.D : 0;
  return std::max(nq, nk);
}

cudaError_t launch_cross_attn_pack_mask(const CrossAttnArgs& a, cudaStream_t st) {
  if (!a.key_pad || !a.words || !a.vis_end || a.B <= 0 || a.Sk <= 0) return cudaErrorInvalidValue;
  cudaError_t e = launch_pdl(pack_mask_kernel, dim3(a.B), dim3(256), 0, st, a.key_pad, a.Sk,
                             (a.Sk + 31) / 32, a.words, a.vis_end);
  if (e != cudaSuccess) return e;
  note_launch();
  return cudaGetLastError();
}

cudaError_t launch_cross_attn_fwd(const CrossAttnArgs& a, cudaStream_t st) {
  if (bad_shape(a)) return cudaErrorInvalidValue;
  if (cross_attn_is_few(a)) return launch_cross_attn_few(a, st);
  // a backward pass needs the lse and the remainders of O, both or neither
  if ((a.lse2 != nullptr) != (a.out_res != nullptr)) return cudaErrorInvalidValue;
  if (a.lse2 != nullptr) {
    if (a.D <= 64)
      return a.half ? run_fwd<__half, 64, true>(a, st) : run_fwd<__nv_bfloat16, 64, true>(a, st);
    return a.half ? run_fwd<__half, 128, true>(a, st) : run_fwd<__nv_bfloat16, 128, true>(a, st);
  }
  if (a.D <= 64)
    return a.half ? run_fwd<__half, 64, false>(a, st) : run_fwd<__nv_bfloat16, 64, false>(a, st);
  return a.half ? run_fwd<__half, 128, false>(a, st) : run_fwd<__nv_bfloat16, 128, false>(a, st);
}

cudaError_t launch_cross_attn_bwd(const CrossAttnArgs& a, cudaStream_t st) {
  if (bad_shape(a) || !a.lse2 || !a.out_res || !a.stats || !a.dk != !a.dv ||
      (a.key_pad && (!a.words || !a.vis_end)))
    return cudaErrorInvalidValue;
  if (a.D <= 64) return a.half ? run_bwd<__half, 64>(a, st) : run_bwd<__nv_bfloat16, 64>(a, st);
  return a.half ? run_bwd<__half, 128>(a, st) : run_bwd<__nv_bfloat16, 128>(a, st);
}

}  // namespace flodl
