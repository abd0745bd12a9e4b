// Host interface of attention with queries, keys and values in tensors of
// their own (cross_attn.cu, cross_attn_few.cu).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "gemm_sm100.h"

namespace flodl {

// Queries [B, Sq, H, D], keys and values [B, Sk, Hk, D], output and its
// gradient likewise; strides in elements for (batch, position, head), the last
// dimension contiguous, every stride of a dimension longer than one a multiple
// of 8 and every base address of 16 bytes. D is a multiple of 8 up to 128.
struct CrossAttnArgs {
  const void *q = nullptr, *k = nullptr, *v = nullptr;
  int64_t q_st[3] = {}, k_st[3] = {}, v_st[3] = {};
  void* out = nullptr;                 // [B, Sq, H, D] contiguous (backward: the forward's output)
  void* out_res = nullptr;             // like out: what its rounding left off, rounded (nullable;
                                       // the backward's row sums dO * O need it)
  float* lse2 = nullptr;               // [B, H, Sq] base-2 log-sum-exp, +inf for a row without a key
  const uint8_t* key_pad = nullptr;    // [B, Sk] contiguous, nonzero = hidden (nullable)
  // from cross_attn_pack_mask, only with key_pad and outside the few-row form
  uint32_t* words = nullptr;           // [B, ceil(Sk / 32)] bit per visible key
  int* vis_end = nullptr;              // [B] index past the last visible key
  // backward
  const void* dout = nullptr;
  int64_t do_st[3] = {};
  float* stats = nullptr;              // scratch of cross_attn_stats_floats, 16-byte aligned
  void *dq = nullptr, *dk = nullptr, *dv = nullptr;  // null dq, or null dk and dv: not wanted
  int64_t dq_st[3] = {}, dk_st[3] = {}, dv_st[3] = {};
  int B = 0, Sq = 0, Sk = 0, H = 0, Hk = 0, D = 0;
  bool causal = false;                 // needs Sq == Sk
  bool half = false;                   // f16 instead of bf16
  float scale = 1.f;
  float* partials = nullptr;           // scratch of the sizes below (nullable where 0)
};

constexpr int kCrossFewRows = 16;  // query rows per memory head of the few-row form

// Pieces of a split axis that a cluster joins, at most: of the few-row form (one sample's
// 8 heads x 8192 x 64 8.6 us, 9.4 with 8; 16 memory heads x 32768 x 128 45.6, 49.5 with 8
// or a second kernel), and of the others, whose CTAs are larger (100 x 4000 x 128, 8
// heads: 17 us with 16, 13.2 with 8).
constexpr int kCrossCluster = 16;
constexpr int kCrossTileCluster = 8;

// Whether the forward takes the few-row form: all query rows of a memory head
// (Sq * H / Hk) fit one 16-row tensor-core tile.
bool cross_attn_is_few(const CrossAttnArgs& a);
// Floats of scratch that the forward / backward needs in `partials` (0: none).
int64_t cross_attn_stats_floats(const CrossAttnArgs& a);
int64_t cross_attn_fwd_partials(const CrossAttnArgs& a);
int64_t cross_attn_bwd_partials(const CrossAttnArgs& a);

cudaError_t launch_cross_attn_pack_mask(const CrossAttnArgs& a, cudaStream_t st);
cudaError_t launch_cross_attn_fwd(const CrossAttnArgs& a, cudaStream_t st);
cudaError_t launch_cross_attn_bwd(const CrossAttnArgs& a, cudaStream_t st);

// Pieces shared by the two files.
// Map {D, position, head, batch} of a strided 16-bit tensor; box = 64 columns x
// `rows` positions.
bool cross_attn_map(CUtensorMap* m, const void* base, bool half, int D, int S, int heads, int B,
                    const int64_t (&st)[3], int rows);
// Shared-memory opt-in of a kernel, once per device.
cudaError_t cross_attn_opt_in(const void* kernel, size_t smem, std::atomic<uint64_t>& done);
// Pieces of the key axis, and whether a cluster joins them (else a second kernel).
struct CrossSplits {
  int n;
  bool clustered;
  bool joined() const { return n > 1 && !clustered; }
};
CrossSplits cross_attn_few_splits(const CrossAttnArgs& a);
// Whether `want` pieces of an axis of `tiles`, joined by a second kernel, beat the s that
// a cluster joins (at most `most`). That kernel costs 3 to 4 us, a tile about 0.5 (64
// keys, a CTA to itself): where the s leave SMs idle and more than five tiles a piece
// go. (16 heads x 128 rows x 64 columns, pieces 8 and 15 to 18: 13.6 us joined by
// clusters and 14.3 by a kernel at 4001 keys, 42 and 29 at 20000.)
inline bool cross_attn_joins_more(int64_t items, int64_t s, int64_t most, int64_t want,
                                  int64_t tiles, int sms) {
  return want > most && items * s < sms && tiles / s - tiles / want > 5;
}
// Clusters of `size` CTAs of a kernel that the GPU holds at once (`fits`: a cache of
// the kernel's own; a cluster's CTAs share a part of the GPU, so that fewer CTAs fit
// in clusters than alone).
using CrossFits = std::atomic<int>[kCrossCluster + 1];
int64_t cross_attn_clusters(const void* kernel, int threads, size_t smem, int size, CrossFits& fits);
cudaError_t launch_cross_attn_few(const CrossAttnArgs& a, cudaStream_t st);
// out = the partial results of `splits` key ranges joined by their lse.
cudaError_t launch_cross_attn_join(const CrossAttnArgs& a, int splits, cudaStream_t st);

}  // namespace flodl
