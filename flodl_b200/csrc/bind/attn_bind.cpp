// Torch bindings for the attention kernels.
#include <cmath>
#include <tuple>

#include "common.h"
#include "../kernels/flash_attn.h"
#include "../kernels/cross_attn.h"

namespace {

using at::Tensor;
using c10::optional;

void flash_fwd(const Tensor& qkv, Tensor& out, Tensor& lse2, int64_t B, int64_t S, int64_t H,
               int64_t D, bool causal, double scale, const optional<Tensor>& key_pad) {
  FL_CHECK_CUDA(qkv);
  FL_CHECK_BF16(qkv);
  FL_CHECK_BF16(out);
  FL_CHECK_F32(lse2);
  FL_CHECK(qkv.is_contiguous() && out.is_contiguous() && lse2.is_contiguous(), "layout");
  FL_CHECK(qkv.numel() == B * S * 3 * H * D && out.numel() == B * S * H * D &&
               lse2.numel() == B * H * S, "flash_fwd sizes");
  FL_CHECK(D == 64, "flash attention kernels support head_dim 64");
  flodl::FlashArgs a;
  a.qkv = reinterpret_cast<const __nv_bfloat16*>(qkv.data_ptr());
  a.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  a.lse2 = lse2.data_ptr<float>();
  if (key_pad) {
    FL_CHECK(key_pad->scalar_type() == at::kBool && key_pad->is_contiguous() &&
                 key_pad->numel() == B * S && key_pad->device() == qkv.device(),
             "key_pad must be bool [B, S] on ", qkv.device());
    a.key_pad = reinterpret_cast<const uint8_t*>(key_pad->data_ptr());
  }
  a.B = (int)B; a.S = (int)S; a.H = (int)H; a.D = (int)D;
  a.causal = causal;
  a.scale = (float)scale;
  c10::cuda::CUDAGuard guard(qkv.device());
  FL_CUDA_OK(flodl::launch_flash_fwd(a, cur_stream()));
}

void flash_bwd(const Tensor& dout, const Tensor& qkv, const Tensor& out, const Tensor& lse2,
               Tensor& dqkv, int64_t B, int64_t S, int64_t H, int64_t D, bool causal,
               double scale, const optional<Tensor>& key_pad, const optional<Tensor>& dbias) {
  FL_CHECK_BF16(dout); FL_CHECK_BF16(qkv); FL_CHECK_BF16(out); FL_CHECK_BF16(dqkv);
  FL_CHECK(dout.is_contiguous() && qkv.is_contiguous() && out.is_contiguous() &&
               dqkv.is_contiguous(), "layout");
  FL_CHECK(D == 64, "flash attention kernels support head_dim 64");
  auto opts = qkv.options().dtype(at::kFloat);
  Tensor delta = at::empty({B, H, S}, opts);
  Tensor dq_acc;
  if (flodl::flash_bwd_needs_dq_acc((int)S)) dq_acc = at::empty({B * S, H * D}, opts);
  flodl::FlashArgs a;
  a.qkv = reinterpret_cast<const __nv_bfloat16*>(qkv.data_ptr());
  a.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  a.lse2 = lse2.data_ptr<float>();
  a.dout = reinterpret_cast<const __nv_bfloat16*>(dout.data_ptr());
  a.dqkv = reinterpret_cast<__nv_bfloat16*>(dqkv.data_ptr());
  a.delta = delta.data_ptr<float>();
  a.dq_acc = dq_acc.defined() ? dq_acc.data_ptr<float>() : nullptr;
  if (key_pad) {
    FL_CHECK(key_pad->scalar_type() == at::kBool && key_pad->is_contiguous() &&
                 key_pad->numel() == B * S && key_pad->device() == qkv.device(),
             "key_pad must be bool [B, S] on ", qkv.device());
    a.key_pad = reinterpret_cast<const uint8_t*>(key_pad->data_ptr());
  }
  if (dbias) {
    FL_CHECK_F32(*dbias);
    FL_CHECK(dbias->is_contiguous() && dbias->numel() == 3 * H * D, "dbias must be f32 [3*H*D]");
    a.dbias = dbias->data_ptr<float>();
  }
  a.B = (int)B; a.S = (int)S; a.H = (int)H; a.D = (int)D;
  a.causal = causal;
  a.scale = (float)scale;
  c10::cuda::CUDAGuard guard(qkv.device());
  FL_CUDA_OK(flodl::launch_flash_bwd(a, cur_stream()));
}

// ---- attention with queries, keys and values in tensors of their own
// [B, positions, heads, D], 16-bit, last dimension contiguous, strides of 16
// bytes, 16-byte aligned.
void cross_strides(const Tensor& t, const char* what, int64_t B, int64_t S, int64_t heads,
                   int64_t D, const Tensor& like, int64_t (&st)[3]) {
  FL_CHECK(t.dim() == 4 && t.size(0) == B && t.size(1) == S && t.size(2) == heads && t.size(3) == D,
           "cross_attn: ", what, " must be [", B, ", ", S, ", ", heads, ", ", D, "] (got ", t.sizes(), ")");
  FL_CHECK(t.scalar_type() == like.scalar_type() && t.device() == like.device(), "cross_attn: ", what,
           " must have the queries' dtype and device");
  FL_CHECK(t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, "cross_attn: ",
           what, " needs a contiguous last dimension and 16-byte alignment");
  for (int i = 0; i < 3; ++i) {
    st[i] = t.size(i) > 1 ? t.stride(i) : 0;
    FL_CHECK(t.size(i) == 1 || (st[i] > 0 && st[i] % 8 == 0), "cross_attn: ", what,
             " needs strides of 16 bytes (got ", t.strides(), ")");
  }
}

flodl::CrossAttnArgs cross_args(const Tensor& q, const Tensor& k, const Tensor& v,
                                const optional<Tensor>& key_pad, const optional<Tensor>& mask_bits,
                                bool causal, double scale) {
  FL_CHECK_CUDA(q);
  FL_CHECK(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf,
           "cross_attn: bf16 or f16 inputs");
  FL_CHECK(q.dim() == 4 && k.dim() == 4, "cross_attn: [B, positions, heads, D] inputs");
  const int64_t B = q.size(0), Sq = q.size(1), H = q.size(2), D = q.size(3);
  const int64_t Sk = k.size(1), Hk = k.size(2);
  constexpr int64_t kMax = (int64_t)1 << 30;
  FL_CHECK(B > 0 && Sq > 0 && Sk > 0 && H > 0 && Hk > 0 && H % Hk == 0 && B < kMax && Sq < kMax &&
               Sk < kMax && H < kMax,
           "cross_attn: sizes (positive, query heads a multiple of the memory heads)");
  FL_CHECK(D > 0 && D <= 128 && D % 8 == 0, "cross_attn: head size a multiple of 8 up to 128");
  FL_CHECK(!causal || Sq == Sk, "cross_attn: causal needs equal lengths");
  FL_CHECK(scale > 0 && std::isfinite(scale), "cross_attn: scale must be positive");
  flodl::CrossAttnArgs a;
  cross_strides(q, "q", B, Sq, H, D, q, a.q_st);
  cross_strides(k, "k", B, Sk, Hk, D, q, a.k_st);
  cross_strides(v, "v", B, Sk, Hk, D, q, a.v_st);
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.B = (int)B; a.Sq = (int)Sq; a.Sk = (int)Sk; a.H = (int)H; a.Hk = (int)Hk; a.D = (int)D;
  a.causal = causal;
  a.half = q.scalar_type() == at::kHalf;
  a.scale = (float)scale;
  if (key_pad) {
    FL_CHECK(key_pad->scalar_type() == at::kBool && key_pad->is_contiguous() && key_pad->dim() == 2 &&
                 key_pad->size(0) == B && key_pad->size(1) == Sk && key_pad->device() == q.device(),
             "cross_attn: key_pad must be bool [B, Sk]");
    a.key_pad = reinterpret_cast<const uint8_t*>(key_pad->data_ptr());
    if (mask_bits) {
      FL_CHECK(mask_bits->scalar_type() == at::kInt && mask_bits->is_contiguous() &&
                   mask_bits->numel() == B * ((Sk + 31) / 32 + 1) && mask_bits->device() == q.device(),
               "cross_attn: mask_bits of another mask");
      a.vis_end = mask_bits->data_ptr<int>();
      a.words = reinterpret_cast<uint32_t*>(a.vis_end + B);
    }
  }
  return a;
}

// The mask as [B] ends of the visible keys, then [B, ceil(Sk / 32)] words with
// a bit per visible key.
Tensor cross_attn_mask(const Tensor& key_pad) {
  FL_CHECK_CUDA(key_pad);
  FL_CHECK(key_pad.scalar_type() == at::kBool && key_pad.is_contiguous() && key_pad.dim() == 2 &&
               key_pad.numel() > 0 && key_pad.size(0) < (int64_t)1 << 30 &&
               key_pad.size(1) < (int64_t)1 << 30, "cross_attn: key_pad must be bool [B, Sk]");
  const int64_t B = key_pad.size(0), Sk = key_pad.size(1);
  c10::cuda::CUDAGuard guard(key_pad.device());
  Tensor bits = at::empty({B * ((Sk + 31) / 32 + 1)}, key_pad.options().dtype(at::kInt));
  flodl::CrossAttnArgs a;
  a.key_pad = reinterpret_cast<const uint8_t*>(key_pad.data_ptr());
  a.vis_end = bits.data_ptr<int>();
  a.words = reinterpret_cast<uint32_t*>(a.vis_end + B);
  a.B = (int)B;
  a.Sk = (int)Sk;
  FL_CUDA_OK(flodl::launch_cross_attn_pack_mask(a, cur_stream()));
  return bits;
}

// -> (output [B, Sq, H, D]; for a backward pass the remainders of its rounding
// and lse2 [B, H, Sq] f32; mask bits), undefined where not there
std::tuple<Tensor, Tensor, Tensor, Tensor> cross_attn_fwd(
    const Tensor& q, const Tensor& k, const Tensor& v, const optional<Tensor>& key_pad, bool causal,
    double scale, bool want_lse) {
  auto a = cross_args(q, k, v, key_pad, c10::nullopt, causal, scale);
  c10::cuda::CUDAGuard guard(q.device());
  Tensor out = at::empty({a.B, a.Sq, a.H, a.D}, q.options());
  a.out = out.data_ptr();
  Tensor res, lse, bits;
  if (want_lse) {
    res = at::empty({a.B, a.Sq, a.H, a.D}, q.options());
    a.out_res = res.data_ptr();
    lse = at::empty({a.B, a.H, a.Sq}, q.options().dtype(at::kFloat));
    a.lse2 = lse.data_ptr<float>();
  }
  if (a.key_pad && !flodl::cross_attn_is_few(a)) {
    bits = cross_attn_mask(*key_pad);
    a.vis_end = bits.data_ptr<int>();
    a.words = reinterpret_cast<uint32_t*>(a.vis_end + a.B);
  }
  Tensor part;
  if (const int64_t n = flodl::cross_attn_fwd_partials(a)) {
    part = at::empty({n}, q.options().dtype(at::kFloat));
    a.partials = part.data_ptr<float>();
  }
  FL_CUDA_OK(flodl::launch_cross_attn_fwd(a, cur_stream()));
  return {out, res, lse, bits};
}

optional<Tensor> if_defined(const Tensor& t) { return t.defined() ? optional<Tensor>(t) : c10::nullopt; }

// Gradients into dq, dk, dv (any strides of 16 bytes); without dq, or without dk
// and dv, that half is left out.
void cross_attn_bwd(const Tensor& dout, const Tensor& q, const Tensor& k, const Tensor& v,
                    const Tensor& out, const Tensor& res, const Tensor& lse2,
                    const optional<Tensor>& key_pad,
                    const optional<Tensor>& mask_bits, bool causal, double scale,
                    const optional<Tensor>& dq, const optional<Tensor>& dk,
                    const optional<Tensor>& dv) {
  auto a = cross_args(q, k, v, key_pad, mask_bits, causal, scale);
  cross_strides(dout, "dout", a.B, a.Sq, a.H, a.D, q, a.do_st);
  FL_CHECK(dk.has_value() == dv.has_value(), "cross_attn: dk and dv come together");
  if (dq) cross_strides(*dq, "dq", a.B, a.Sq, a.H, a.D, q, a.dq_st);
  if (dk) cross_strides(*dk, "dk", a.B, a.Sk, a.Hk, a.D, q, a.dk_st);
  if (dv) cross_strides(*dv, "dv", a.B, a.Sk, a.Hk, a.D, q, a.dv_st);
  for (const Tensor* t : {&out, &res})
    FL_CHECK(t->sizes() == q.sizes() && t->is_contiguous() && t->scalar_type() == q.scalar_type() &&
                 t->device() == q.device(), "cross_attn: out and its remainders must be the forward's");
  FL_CHECK(lse2.scalar_type() == at::kFloat && lse2.is_contiguous() &&
               lse2.numel() == (int64_t)a.B * a.H * a.Sq && lse2.device() == q.device(),
           "cross_attn: lse2 must be the forward's");
  c10::cuda::CUDAGuard guard(q.device());
  a.dout = dout.data_ptr();
  a.out = out.data_ptr();
  a.out_res = res.data_ptr();
  a.lse2 = lse2.data_ptr<float>();
  a.dq = dq ? dq->data_ptr() : nullptr;
  a.dk = dk ? dk->data_ptr() : nullptr;
  a.dv = dv ? dv->data_ptr() : nullptr;
  Tensor bits;
  if (a.key_pad && !a.words) {
    bits = cross_attn_mask(*key_pad);
    a.vis_end = bits.data_ptr<int>();
    a.words = reinterpret_cast<uint32_t*>(a.vis_end + a.B);
  }
  // one allocation: the row statistics, then the pieces of split axes
  const int64_t n_stats = flodl::cross_attn_stats_floats(a), n_part = flodl::cross_attn_bwd_partials(a);
  Tensor scratch = at::empty({n_stats + n_part}, q.options().dtype(at::kFloat));
  a.stats = scratch.data_ptr<float>();
  a.partials = n_part ? a.stats + n_stats : nullptr;
  FL_CUDA_OK(flodl::launch_cross_attn_bwd(a, cur_stream()));
}

// A tensor the tile loads can read in place, or a contiguous copy.
Tensor tma_ready(const Tensor& t) {
  bool ok = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int i = 0; i < 3; ++i) ok = ok && (t.size(i) == 1 || (t.stride(i) > 0 && t.stride(i) % 8 == 0));
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

struct CrossAttn : public torch::autograd::Function<CrossAttn> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& q0, const Tensor& k0,
                        const Tensor& v0, const optional<Tensor>& key_pad, bool causal,
                        double scale) {
    const Tensor q = tma_ready(q0), k = tma_ready(k0), v = tma_ready(v0);
    auto [out, res, lse, bits] = cross_attn_fwd(q, k, v, key_pad, causal, scale, true);
    ctx->save_for_backward({q, k, v, out, res, lse, key_pad ? *key_pad : Tensor(), bits});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    return out;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor &q = s[0], &k = s[1], &v = s[2];
    torch::autograd::variable_list out(6);
    if (!grads[0].defined()) return out;
    Tensor dq, dk, dv;
    {
      at::NoGradGuard no_grad;
      const Tensor dout = tma_ready(grads[0].to(q.scalar_type()));
      if (ctx->needs_input_grad(0)) dq = at::empty(q.sizes(), q.options());
      if (ctx->needs_input_grad(1) || ctx->needs_input_grad(2)) {
        dk = at::empty(k.sizes(), k.options());
        dv = at::empty(v.sizes(), v.options());
      }
      cross_attn_bwd(dout, q, k, v, s[3], s[4], s[5], if_defined(s[6]), if_defined(s[7]),
                     ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble(),
                     if_defined(dq), if_defined(dk), if_defined(dv));
    }
    return once_differentiable({dq, dk, dv, Tensor(), Tensor(), Tensor()}, "cross_attention");
  }
};

// Scales that the kernels take: products with powers of two up to 2^61 of the backward's
// stay normal in f32.
constexpr double kLeastScale = 1e-18;

// Attention over a memory: argument errors are ValueErrors. Nothing comes back
// where the kernels do not apply (another dtype or head size, an empty
// dimension, a scale far from 1, a forward-mode tangent); the caller then checks and composes.
optional<Tensor> cross_attention(const Tensor& q, const Tensor& k, const Tensor& v,
                                 const optional<Tensor>& key_pad, bool causal, optional<double> scale) {
  if (q.dim() != 4 || k.dim() != 4 || v.dim() != 4 || !q.is_cuda() ||
      !(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf) ||
      k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type() ||
      k.device() != q.device() || v.device() != q.device() || k.sizes() != v.sizes())
    return c10::nullopt;
  const int64_t B = q.size(0), D = q.size(3);
  if (k.size(0) != B || k.size(3) != D || D % 8 || D > 128 || q.numel() == 0 || k.numel() == 0 ||
      q.size(2) % k.size(2) || has_tangent(q) || has_tangent(k) || has_tangent(v))
    return c10::nullopt;
  TORCH_CHECK_VALUE(!key_pad || (key_pad->scalar_type() == at::kBool && key_pad->dim() == 2 &&
                                 key_pad->size(0) == B && key_pad->size(1) == k.size(1) &&
                                 key_pad->device() == q.device()),
                    "key_padding must be bool [", B, ", ", k.size(1), "] on ", q.device());
  TORCH_CHECK_VALUE(!causal || q.size(1) == k.size(1), "causal attention needs equal lengths (got ",
                    q.size(1), " and ", k.size(1), ")");
  const double c = scale ? *scale : 1.0 / std::sqrt((double)D);
  TORCH_CHECK_VALUE(c > 0 && std::isfinite(c), "scale must be positive and finite (got ", c, ")");
  if (c < kLeastScale || c > 1 / kLeastScale) return c10::nullopt;
  optional<Tensor> pad = key_pad;
  if (pad) pad = pad->contiguous();
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad()))
    return CrossAttn::apply(q, k, v, pad, causal, c);
  return std::get<0>(cross_attn_fwd(tma_ready(q), tma_ready(k), tma_ready(v), pad, causal, c, false));
}

}  // namespace

void register_attention(py::module& m) {
  m.def("set_flash_wait_limit_ns", [](int64_t ns) { flodl::set_flash_wait_limit_ns((uint64_t)ns); });
  m.def("flash_attn_fwd", &flash_fwd, py::arg("qkv"), py::arg("out"), py::arg("lse2"),
        py::arg("B"), py::arg("S"), py::arg("H"), py::arg("D"), py::arg("causal"),
        py::arg("scale"), py::arg("key_pad") = py::none());
  m.def("flash_attn_bwd", &flash_bwd, py::arg("dout"), py::arg("qkv"), py::arg("out"),
        py::arg("lse2"), py::arg("dqkv"), py::arg("B"), py::arg("S"), py::arg("H"), py::arg("D"),
        py::arg("causal"), py::arg("scale"), py::arg("key_pad") = py::none(),
        py::arg("dbias") = py::none());
  m.def("cross_attention", &cross_attention, py::arg("q"), py::arg("k"), py::arg("v"),
        py::arg("key_padding"), py::arg("causal"), py::arg("scale"));
  m.attr("CROSS_ATTN_LEAST_SCALE") = kLeastScale;
  m.def("cross_attn_mask", &cross_attn_mask, py::arg("key_pad"));
  m.def("cross_attn_fwd",
        [](const Tensor& q, const Tensor& k, const Tensor& v, const optional<Tensor>& key_pad,
           bool causal, double scale, bool want_lse) {
          auto [out, res, lse, bits] = cross_attn_fwd(q, k, v, key_pad, causal, scale, want_lse);
          return std::make_tuple(out, if_defined(res), if_defined(lse), if_defined(bits));
        },
        py::arg("q"), py::arg("k"), py::arg("v"), py::arg("key_pad"), py::arg("causal"),
        py::arg("scale"), py::arg("want_lse"));
  m.def("cross_attn_bwd", &cross_attn_bwd, py::arg("dout"), py::arg("q"), py::arg("k"),
        py::arg("v"), py::arg("out"), py::arg("res"), py::arg("lse2"), py::arg("key_pad"),
        py::arg("mask_bits"),
        py::arg("causal"), py::arg("scale"), py::arg("dq"), py::arg("dk"), py::arg("dv"));
}
