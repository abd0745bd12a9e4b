// Torch bindings for LayerNorm, cross-entropy, embedding, optimizer and
// elementwise kernels.
#include "common.h"
#include "../kernels/kernels.h"

namespace {

using at::Tensor;
using c10::optional;

template <typename T>
T* ptr(const Tensor& t) { return reinterpret_cast<T*>(t.data_ptr()); }

void ln_fwd(const Tensor& x, const optional<Tensor>& gamma, const optional<Tensor>& beta,
            const optional<Tensor>& y_bf16, const optional<Tensor>& y_f32, const Tensor& mean,
            const Tensor& rstd, double eps) {
  FL_CHECK_CUDA(x);
  FL_CHECK(x.is_contiguous(), "x must be contiguous");
  const int C = (int)x.size(-1);
  const int rows = (int)(x.numel() / C);
  flodl::LnFwdArgs a;
  a.x = x.data_ptr();
  a.x_bf16 = x.scalar_type() == at::kBFloat16;
  FL_CHECK(a.x_bf16 || x.scalar_type() == at::kFloat, "x must be f32 or bf16");
  a.gamma = opt_ptr<const float>(gamma);
  a.beta = opt_ptr<const float>(beta);
  a.y_bf16 = opt_ptr<__nv_bfloat16>(y_bf16);
  a.y_f32 = opt_ptr<float>(y_f32);
  a.mean = ptr<float>(mean);
  a.rstd = ptr<float>(rstd);
  a.rows = rows;
  a.C = C;
  a.eps = (float)eps;
  c10::cuda::CUDAGuard guard(x.device());
  FL_CUDA_OK(flodl::launch_ln_fwd(a, cur_stream()));
}

// RMSNorm over the last dimension: y = x * rstd * w (x, y f32 or bf16).
void rms_fwd(const Tensor& x, const optional<Tensor>& w, Tensor& y, Tensor& rstd, double eps) {
  FL_CHECK_CUDA(x);
  FL_CHECK(x.is_contiguous() && y.is_contiguous() && y.scalar_type() == x.scalar_type() &&
               y.numel() == x.numel(), "rms_fwd: x, y contiguous, same dtype and size");
  const bool bf16 = x.scalar_type() == at::kBFloat16;
  FL_CHECK(bf16 || x.scalar_type() == at::kFloat, "rms_fwd: x must be f32 or bf16");
  const int C = (int)x.size(-1);
  const int rows = (int)(x.numel() / C);
  FL_CHECK(rstd.scalar_type() == at::kFloat && rstd.numel() >= rows, "rms_fwd: rstd [rows] f32");
  if (w) FL_CHECK(w->scalar_type() == at::kFloat && w->numel() == C, "rms_fwd: w [C] f32");
  c10::cuda::CUDAGuard guard(x.device());
  FL_CUDA_OK(flodl::launch_rms_fwd(x.data_ptr(), bf16, opt_ptr<const float>(w), y.data_ptr(),
                                   ptr<float>(rstd), rows, C, (float)eps, cur_stream()));
}

void rms_bwd(const Tensor& dy, const Tensor& x, const optional<Tensor>& w, const Tensor& rstd,
             Tensor& dx, const optional<Tensor>& dw) {
  FL_CHECK_CUDA(x);
  FL_CHECK(dy.is_contiguous() && x.is_contiguous() && dx.is_contiguous() &&
               dy.scalar_type() == x.scalar_type() && dx.scalar_type() == x.scalar_type() &&
               dy.numel() == x.numel() && dx.numel() == x.numel(),
           "rms_bwd: dy, x, dx contiguous, same dtype and size");
  const int C = (int)x.size(-1);
  const int rows = (int)(x.numel() / C);
  if (dw) FL_CHECK(dw->scalar_type() == at::kFloat && dw->numel() == C, "rms_bwd: dw [C] f32");
  c10::cuda::CUDAGuard guard(x.device());
  FL_CUDA_OK(flodl::launch_rms_bwd(dy.data_ptr(), x.data_ptr(), x.scalar_type() == at::kBFloat16,
                                   opt_ptr<const float>(w), ptr<float>(rstd), dx.data_ptr(),
                                   opt_ptr<float>(dw), rows, C, cur_stream()));
}

// Per-head RMS norm of queries and keys with the rotary embedding. Tensors are
// [B, S, heads, D] with a contiguous last dimension, any other strides.
int dtype_code(const Tensor& t) {
  return t.scalar_type() == at::kFloat      ? 0
         : t.scalar_type() == at::kBFloat16 ? 1
         : t.scalar_type() == at::kHalf     ? 2
                                            : -1;
}

flodl::QkNormRopeArgs qk_args(const Tensor& q, const Tensor& k, const optional<Tensor>& wq,
                              const optional<Tensor>& wk, const optional<Tensor>& cos,
                              const optional<Tensor>& sin, const optional<Tensor>& pos,
                              int64_t offset, const Tensor& out_q, const Tensor& out_k,
                              double eps) {
  FL_CHECK_CUDA(q);
  FL_CHECK(dtype_code(q) >= 0, "qk_norm_rope: f32, bf16 or f16 inputs");
  const int64_t B = q.dim() == 4 ? q.size(0) : 0, S = q.dim() == 4 ? q.size(1) : 0;
  auto heads = [&](const Tensor& t, const Tensor& like, const char* what) {
    FL_CHECK(t.dim() == 4 && t.size(0) == B && t.size(1) == S && t.size(3) == q.size(3) &&
                 t.size(2) == like.size(2) && t.scalar_type() == q.scalar_type() &&
                 t.device() == q.device() && t.stride(3) == 1,
             "qk_norm_rope: ", what, " must be [B, S, heads, D] of the queries' B, S, D, dtype and "
             "device with a contiguous last dimension");
  };
  heads(q, q, "q");
  heads(k, k, "k");
  heads(out_q, q, "q output");
  heads(out_k, k, "k output");
  const int64_t D = q.size(3);
  FL_CHECK(B > 0 && S > 0 && q.size(2) > 0 && k.size(2) > 0 && D > 0, "qk_norm_rope: empty input");
  FL_CHECK(D <= flodl::kQkNormRopeMaxD, "qk_norm_rope: head size above ", flodl::kQkNormRopeMaxD);
  FL_CHECK(B * S < (int64_t)1 << 31 && q.size(2) + k.size(2) < (int64_t)1 << 20,
           "qk_norm_rope: too many rows");
  flodl::QkNormRopeArgs a;
  for (const optional<Tensor>* w : {&wq, &wk})
    if (*w)
      FL_CHECK((*w)->scalar_type() == at::kFloat && (*w)->is_contiguous() && (*w)->numel() == D &&
                   (*w)->device() == q.device(), "qk_norm_rope: weights must be f32 [D]");
  a.wq = opt_ptr<const float>(wq);
  a.wk = opt_ptr<const float>(wk);
  FL_CHECK(cos.has_value() == sin.has_value(), "qk_norm_rope: cos and sin come together");
  if (cos) {
    for (const Tensor* t : {&*cos, &*sin})
      FL_CHECK(t->scalar_type() == at::kFloat && t->dim() == 2 && t->is_contiguous() &&
                   t->device() == q.device() && t->sizes() == cos->sizes(),
               "qk_norm_rope: cos and sin must be f32 [positions, R / 2]");
    FL_CHECK(2 * cos->size(1) <= D, "qk_norm_rope: the tables rotate more than the head size");
    a.cos = cos->data_ptr<float>();
    a.sin = sin->data_ptr<float>();
    a.R = (int)(2 * cos->size(1));
    a.table_rows = cos->size(0);
  }
  if (a.R > 0 && pos) {
    FL_CHECK(pos->scalar_type() == at::kLong && pos->is_contiguous() && pos->dim() == 2 &&
                 pos->size(0) == B && pos->size(1) == S && pos->device() == q.device(),
             "qk_norm_rope: positions must be int64 [B, S]");
    a.pos = pos->data_ptr<int64_t>();
    a.pos_stride = S;
  } else if (a.R > 0) {
    FL_CHECK(offset >= 0 && offset <= a.table_rows - S, "qk_norm_rope: positions ", offset, " to ",
             offset + S - 1, " outside the tables' ", a.table_rows, " rows");
  }
  a.offset = offset;
  auto st = [](const Tensor& t, int64_t (&s)[3]) {
    for (int i = 0; i < 3; ++i) s[i] = t.size(i) > 1 ? t.stride(i) : 0;
  };
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.out_q = out_q.data_ptr();
  a.out_k = out_k.data_ptr();
  st(q, a.q_st);
  st(k, a.k_st);
  st(out_q, a.oq_st);
  st(out_k, a.ok_st);
  a.B = (int)B; a.S = (int)S; a.H = (int)q.size(2); a.Hk = (int)k.size(2); a.D = (int)D;
  a.dtype = dtype_code(q);
  a.eps = (float)eps;
  return a;
}

void qk_norm_rope_fwd(const Tensor& q, const Tensor& k, const optional<Tensor>& wq,
                      const optional<Tensor>& wk, const optional<Tensor>& cos,
                      const optional<Tensor>& sin, const optional<Tensor>& pos, int64_t offset,
                      Tensor& yq, Tensor& yk, double eps) {
  const auto a = qk_args(q, k, wq, wk, cos, sin, pos, offset, yq, yk, eps);
  c10::cuda::CUDAGuard guard(q.device());
  FL_CUDA_OK(flodl::launch_qk_norm_rope_fwd(a, cur_stream()));
}

void qk_norm_rope_bwd(const Tensor& dyq, const Tensor& dyk, const Tensor& q, const Tensor& k,
                      const optional<Tensor>& wq, const optional<Tensor>& wk,
                      const optional<Tensor>& cos, const optional<Tensor>& sin,
                      const optional<Tensor>& pos, int64_t offset, Tensor& dq, Tensor& dk,
                      const optional<Tensor>& dwq, const optional<Tensor>& dwk, double eps,
                      bool dwq_add = true, bool dwk_add = true) {
  auto a = qk_args(q, k, wq, wk, cos, sin, pos, offset, dq, dk, eps);
  for (const Tensor* t : {&dyq, &dyk})
    FL_CHECK(t->scalar_type() == q.scalar_type() && t->device() == q.device() && t->dim() == 4 &&
                 t->stride(3) == 1, "qk_norm_rope: output gradients of the inputs' dtype and device "
             "with a contiguous last dimension");
  FL_CHECK(dyq.sizes() == q.sizes() && dyk.sizes() == k.sizes(),
           "qk_norm_rope: output gradients of the outputs' shapes");
  a.dyq = dyq.data_ptr();
  a.dyk = dyk.data_ptr();
  for (int i = 0; i < 3; ++i) {
    a.dyq_st[i] = dyq.size(i) > 1 ? dyq.stride(i) : 0;
    a.dyk_st[i] = dyk.size(i) > 1 ? dyk.stride(i) : 0;
  }
  for (const optional<Tensor>* w : {&dwq, &dwk})
    if (*w)
      FL_CHECK((*w)->scalar_type() == at::kFloat && (*w)->is_contiguous() &&
                   (*w)->numel() == q.size(3) && (*w)->device() == q.device(),
               "qk_norm_rope: weight gradients must be f32 [D]");
  a.dwq = opt_ptr<float>(dwq);
  a.dwk = opt_ptr<float>(dwk);
  a.dwq_add = dwq_add;
  a.dwk_add = dwk_add;
  FL_CHECK(!a.dwq || a.dwq != a.dwk, "qk_norm_rope: one buffer for both weight gradients");
  c10::cuda::CUDAGuard guard(q.device());
  Tensor partials;
  if (a.dwq || a.dwk) {
    a.partial_rows = flodl::qk_norm_rope_partial_rows(a);
    partials = at::empty({a.partial_rows, q.size(3)}, q.options().dtype(at::kFloat));
    a.partials = partials.data_ptr<float>();
  }
  FL_CUDA_OK(flodl::launch_qk_norm_rope_bwd(a, cur_stream()));
}

// Gradient-ready listeners of a parameter live on its Python object.
void notify_grad_ready(const Tensor& w) {
  py::gil_scoped_acquire gil;
  static py::object& fn =
      *new py::object(py::module_::import("flodl_b200.ops._common").attr("grad_ready"));
  fn(w);
}

Tensor rows_ready(const Tensor& t) {
  return t.stride(-1) == 1 ? t : t.clone(at::MemoryFormat::Contiguous);
}
optional<Tensor> some(const Tensor& t) { return t.defined() ? optional<Tensor>(t) : c10::nullopt; }

// Input gradients into dq / dk, and the weight gradients: a leaf weight's is
// added to its .grad and its listeners are notified, as the other fused norms
// do; a computed weight's is returned for autograd.
std::pair<Tensor, Tensor> qk_norm_rope_backward(const Tensor& dyq, const Tensor& dyk,
                                                const Tensor& q, const Tensor& k, const Tensor& wq,
                                                const Tensor& wk, const Tensor& cos,
                                                const Tensor& sin, const Tensor& pos,
                                                int64_t offset, double eps, Tensor& dq, Tensor& dk) {
  at::NoGradGuard no_grad;
  const Tensor* w[2] = {&wq, &wk};
  Tensor buf[2], ret[2];
  bool add[2] = {false, false};
  const bool shared = wq.defined() && wk.defined() && wq.is_same(wk);
  for (int i = 0; i < 2; ++i) {
    if (!w[i]->defined() || !w[i]->requires_grad()) continue;
    const bool leaf = w[i]->is_leaf() && !shared;
    add[i] = leaf && w[i]->grad().defined();
    buf[i] = add[i] ? w[i]->grad() : at::empty(w[i]->sizes(), q.options().dtype(at::kFloat));
    if (leaf && !add[i]) w[i]->mutable_grad() = buf[i];
    if (!w[i]->is_leaf()) ret[i] = buf[i];
  }
  qk_norm_rope_bwd(dyq, dyk, q, k, some(wq), some(wk), some(cos), some(sin), some(pos), offset, dq,
                   dk, some(buf[0]), some(buf[1]), eps, add[0], add[1]);
  if (shared && wq.requires_grad() && wq.is_leaf()) {
    buf[0].add_(buf[1]);
    if (wq.grad().defined())
      wq.mutable_grad().add_(buf[0]);
    else
      wq.mutable_grad() = buf[0];
  }
  for (int i = 0; i < (shared ? 1 : 2); ++i)
    if (w[i]->defined() && w[i]->requires_grad() && w[i]->is_leaf()) notify_grad_ready(*w[i]);
  return {ret[0], ret[1]};
}

struct QkNormRope : public torch::autograd::Function<QkNormRope> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx,
                                                const Tensor& q0, const Tensor& k0,
                                                const optional<Tensor>& wq,
                                                const optional<Tensor>& wk,
                                                const optional<Tensor>& cos,
                                                const optional<Tensor>& sin,
                                                const optional<Tensor>& pos, int64_t offset,
                                                double eps) {
    const Tensor q = rows_ready(q0), k = rows_ready(k0);
    Tensor yq = at::empty(q.sizes(), q.options()), yk = at::empty(k.sizes(), k.options());
    qk_norm_rope_fwd(q, k, wq, wk, cos, sin, pos, offset, yq, yk, eps);
    auto t = [](const optional<Tensor>& x) { return x ? *x : Tensor(); };
    ctx->save_for_backward({q, k, t(wq), t(wk), t(cos), t(sin), t(pos)});
    ctx->saved_data["offset"] = offset;
    ctx->saved_data["eps"] = eps;
    return {yq, yk};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor &q = s[0], &k = s[1];
    torch::autograd::variable_list out(9);
    {
      at::NoGradGuard no_grad;
      Tensor dy[2];
      for (int i = 0; i < 2; ++i)
        dy[i] = grads[i].defined() ? rows_ready(grads[i].to(q.scalar_type()))
                                   : at::zeros(s[i].sizes(), q.options());
      out[0] = at::empty(q.sizes(), q.options());
      out[1] = at::empty(k.sizes(), k.options());
      std::tie(out[2], out[3]) = qk_norm_rope_backward(
          dy[0], dy[1], q, k, s[2], s[3], s[4], s[5], s[6], ctx->saved_data["offset"].toInt(),
          ctx->saved_data["eps"].toDouble(), out[0], out[1]);
    }
    return once_differentiable(out, "qk_norm_rope");
  }
};

// The operator: argument errors are ValueErrors. Nothing comes back where the
// kernels do not apply (another dtype or head size, an empty input, a forward-mode
// tangent, tables that want gradients); the caller then checks and composes.
optional<std::pair<Tensor, Tensor>> qk_norm_rope(const Tensor& q, const Tensor& k,
                                                 const optional<Tensor>& q_weight,
                                                 const optional<Tensor>& k_weight,
                                                 const optional<Tensor>& cos,
                                                 const optional<Tensor>& sin,
                                                 const optional<Tensor>& positions, int64_t offset,
                                                 double eps) {
  if (!q.is_cuda() || dtype_code(q) < 0 || q.dim() != 4 || k.dim() != 4 || q.size(3) < 2 ||
      q.size(3) > flodl::kQkNormRopeMaxD || q.numel() == 0 || k.numel() == 0)
    return c10::nullopt;
  if (has_tangent(q) || has_tangent(k) || has_tangent(q_weight) || has_tangent(k_weight) ||
      has_tangent(cos) || has_tangent(sin))
    return c10::nullopt;
  const int64_t B = q.size(0), S = q.size(1), D = q.size(3);
  TORCH_CHECK_VALUE(k.size(0) == B && k.size(1) == S && k.size(3) == D, "queries ", q.sizes(),
                    " and keys ", k.sizes(), " differ in batch, positions or head size");
  TORCH_CHECK_VALUE(k.scalar_type() == q.scalar_type() && k.device() == q.device(),
                    "queries and keys must be floating-point tensors of one dtype and device");
  for (const optional<Tensor>* w : {&q_weight, &k_weight}) {
    TORCH_CHECK_VALUE(!*w || ((*w)->dim() == 1 && (*w)->numel() == D &&
                              (*w)->scalar_type() == at::kFloat && (*w)->device() == q.device()),
                      "weights must be f32 [", D, "] on ", q.device());
  }
  TORCH_CHECK_VALUE(cos.has_value() == sin.has_value(), "cos and sin come together");
  TORCH_CHECK_VALUE(cos || !positions, "positions need the cos and sin tables");
  const bool turn = cos && cos->dim() == 2 && cos->size(1) > 0;
  if (cos) {
    TORCH_CHECK_VALUE(cos->dim() == 2 && cos->sizes() == sin->sizes() && 2 * cos->size(1) <= D &&
                          cos->scalar_type() == at::kFloat && sin->scalar_type() == at::kFloat &&
                          cos->device() == q.device() && sin->device() == q.device(),
                      "cos and sin must be f32 [positions, R / 2] with R <= ", D, " on ", q.device());
    if (positions) {
      TORCH_CHECK_VALUE(offset == 0 && positions->scalar_type() == at::kLong &&
                            positions->dim() == 2 && positions->size(0) == B &&
                            positions->size(1) == S && positions->device() == q.device(),
                        "positions must be int64 [", B, ", ", S, "] on ", q.device(),
                        ", without an offset");
    } else {
      TORCH_CHECK_VALUE(offset >= 0 && offset <= cos->size(0) - S, "positions ", offset, " to ",
                        offset + S - 1, " are outside the tables' ", cos->size(0), " rows");
    }
  }
  auto plain = [](const optional<Tensor>& t) {
    return t ? optional<Tensor>(t->contiguous()) : c10::nullopt;
  };
  const auto wq = plain(q_weight), wk = plain(k_weight);
  const auto c = turn ? plain(cos) : c10::nullopt, s = turn ? plain(sin) : c10::nullopt;
  const auto pos = turn ? plain(positions) : c10::nullopt;
  auto grad = [](const optional<Tensor>& t) { return t && t->requires_grad(); };
  if (at::GradMode::is_enabled() && (grad(c) || grad(s))) return c10::nullopt;  // learned tables
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || grad(wq) || grad(wk))) {
    auto y = QkNormRope::apply(q, k, wq, wk, c, s, pos, offset, eps);
    return std::make_pair(y[0], y[1]);
  }
  Tensor yq = at::empty(q.sizes(), q.options()), yk = at::empty(k.sizes(), k.options());
  qk_norm_rope_fwd(rows_ready(q), rows_ready(k), wq, wk, c, s, pos, offset, yq, yk, eps);
  return std::make_pair(yq, yk);
}

// GroupNorm over x [N, C, *] contiguous (f32 or bf16), G groups.
void gn_fwd(const Tensor& x, const optional<Tensor>& gamma, const optional<Tensor>& beta,
            Tensor& y, Tensor& mean, Tensor& rstd, int64_t G, double eps) {
  FL_CHECK_CUDA(x);
  FL_CHECK(x.dim() >= 2 && x.is_contiguous() && y.is_contiguous() &&
               y.scalar_type() == x.scalar_type() && y.numel() == x.numel(),
           "gn_fwd: x, y contiguous [N, C, *], same dtype and size");
  const bool bf16 = x.scalar_type() == at::kBFloat16;
  FL_CHECK(bf16 || x.scalar_type() == at::kFloat, "gn_fwd: x must be f32 or bf16");
  const int N = (int)x.size(0), Cc = (int)x.size(1);
  const int HW = (int)(x.numel() / ((int64_t)N * Cc));
  FL_CHECK(G > 0 && Cc % G == 0, "gn_fwd: C must divide into G groups");
  FL_CHECK(mean.numel() >= N * G && rstd.numel() >= N * G, "gn_fwd: mean/rstd [N*G] f32");
  c10::cuda::CUDAGuard guard(x.device());
  FL_CUDA_OK(flodl::launch_gn_fwd(x.data_ptr(), bf16, opt_ptr<const float>(gamma),
                                  opt_ptr<const float>(beta), y.data_ptr(), ptr<float>(mean),
                                  ptr<float>(rstd), N, Cc, HW, (int)G, (float)eps, cur_stream()));
}

void gn_bwd(const Tensor& dy, const Tensor& x, const optional<Tensor>& gamma, const Tensor& mean,
            const Tensor& rstd, Tensor& dx, const optional<Tensor>& dgamma,
            const optional<Tensor>& dbeta, int64_t G) {
  FL_CHECK_CUDA(x);
  FL_CHECK(dy.is_contiguous() && x.is_contiguous() && dx.is_contiguous() &&
               dy.scalar_type() == x.scalar_type() && dx.scalar_type() == x.scalar_type() &&
               dy.numel() == x.numel() && dx.numel() == x.numel(),
           "gn_bwd: dy, x, dx contiguous, same dtype and size");
  const int N = (int)x.size(0), Cc = (int)x.size(1);
  const int HW = (int)(x.numel() / ((int64_t)N * Cc));
  c10::cuda::CUDAGuard guard(x.device());
  FL_CUDA_OK(flodl::launch_gn_bwd(dy.data_ptr(), x.data_ptr(), x.scalar_type() == at::kBFloat16,
                                  opt_ptr<const float>(gamma), ptr<float>(mean), ptr<float>(rstd),
                                  dx.data_ptr(), opt_ptr<float>(dgamma), opt_ptr<float>(dbeta), N,
                                  Cc, HW, (int)G, cur_stream()));
}

// Max pooling of x [planes, H, W] (f32 or bf16) into y [planes, Ho, Wo] with
// the argmax index per output (int32).
void maxpool_fwd(const Tensor& x, Tensor& y, Tensor& idx, int64_t kh, int64_t kw, int64_t sh,
                 int64_t sw, int64_t ph, int64_t pw, int64_t dh, int64_t dw) {
  FL_CHECK_CUDA(x);
  FL_CHECK(x.is_contiguous() && y.is_contiguous() && idx.is_contiguous() && x.dim() >= 2 &&
               y.scalar_type() == x.scalar_type() && idx.scalar_type() == at::kInt &&
               idx.numel() == y.numel(),
           "maxpool_fwd: contiguous x, y (same dtype) and int32 idx like y");
  const bool bf16 = x.scalar_type() == at::kBFloat16;
  FL_CHECK(bf16 || x.scalar_type() == at::kFloat, "maxpool_fwd: x must be f32 or bf16");
  const int H = (int)x.size(-2), W = (int)x.size(-1);
  const int Ho = (int)y.size(-2), Wo = (int)y.size(-1);
  const int planes = (int)(x.numel() / ((int64_t)H * W));
  FL_CHECK(y.numel() == (int64_t)planes * Ho * Wo, "maxpool_fwd: y shape");
  c10::cuda::CUDAGuard guard(x.device());
  FL_CUDA_OK(flodl::launch_maxpool_fwd(
      x.data_ptr(), bf16, y.data_ptr(), ptr<int32_t>(idx), planes, H, W, Ho, Wo,
      flodl::PoolGeo{(int)kh, (int)kw, (int)sh, (int)sw, (int)ph, (int)pw, (int)dh, (int)dw},
      cur_stream()));
}

void maxpool_bwd(const Tensor& dy, const Tensor& idx, Tensor& dx) {
  FL_CHECK_CUDA(dy);
  FL_CHECK(dy.is_contiguous() && idx.is_contiguous() && dx.is_contiguous() &&
               dy.scalar_type() == dx.scalar_type() && idx.numel() == dy.numel(),
           "maxpool_bwd: contiguous dy, dx (same dtype), idx like dy");
  const int H = (int)dx.size(-2), W = (int)dx.size(-1);
  const int Ho = (int)dy.size(-2), Wo = (int)dy.size(-1);
  const int planes = (int)(dx.numel() / ((int64_t)H * W));
  c10::cuda::CUDAGuard guard(dy.device());
  FL_CUDA_OK(flodl::launch_maxpool_bwd(dy.data_ptr(), dy.scalar_type() == at::kBFloat16,
                                       ptr<int32_t>(idx), dx.data_ptr(), planes, H, W, Ho, Wo,
                                       cur_stream()));
}

// Dropout with a counter-based mask (same seed and offset: same mask).
void dropout(const Tensor& x, Tensor& y, double p, int64_t seed, int64_t offset) {
  FL_CHECK_CUDA(x);
  FL_CHECK(x.is_contiguous() && y.is_contiguous() && y.scalar_type() == x.scalar_type() &&
               y.numel() == x.numel(), "dropout: x, y contiguous, same dtype and size");
  const bool bf16 = x.scalar_type() == at::kBFloat16;
  FL_CHECK(bf16 || x.scalar_type() == at::kFloat, "dropout: x must be f32 or bf16");
  FL_CHECK(p >= 0.0 && p < 1.0, "dropout: 0 <= p < 1");
  c10::cuda::CUDAGuard guard(x.device());
  FL_CUDA_OK(flodl::launch_dropout(x.data_ptr(), y.data_ptr(), bf16, x.numel(), (float)p,
                                   (uint64_t)seed, (uint64_t)offset, cur_stream()));
}

void ln_bwd(const Tensor& dy, const Tensor& x, const Tensor& mean, const Tensor& rstd,
            const optional<Tensor>& gamma, const optional<Tensor>& dres,
            const optional<Tensor>& dx_f32, const optional<Tensor>& dx_bf16,
            const optional<Tensor>& dgamma, const optional<Tensor>& dbeta,
            const optional<Tensor>& colsum, bool pre_add) {
  FL_CHECK_CUDA(dy);
  FL_CHECK_BF16(dy);
  FL_CHECK(dy.is_contiguous() && x.is_contiguous(), "ln_bwd inputs must be contiguous");
  const int C = (int)x.size(-1);
  flodl::LnBwdArgs a;
  a.dy = ptr<__nv_bfloat16>(dy);
  a.x = x.data_ptr();
  a.x_bf16 = x.scalar_type() == at::kBFloat16;
  a.mean = ptr<float>(mean);
  a.rstd = ptr<float>(rstd);
  a.gamma = opt_ptr<const float>(gamma);
  a.dres = opt_ptr<const float>(dres);
  a.dx_f32 = opt_ptr<float>(dx_f32);
  a.dx_bf16 = opt_ptr<__nv_bfloat16>(dx_bf16);
  a.dgamma = opt_ptr<float>(dgamma);
  a.dbeta = opt_ptr<float>(dbeta);
  a.colsum = opt_ptr<float>(colsum);
  a.pre_add = pre_add;
  a.rows = (int)(x.numel() / C);
  a.C = C;
  c10::cuda::CUDAGuard guard(x.device());
  // column reductions (dgamma, dbeta, bias gradient) accumulate with one
  // atomic per column and block: no scratch, no second pass
  FL_CUDA_OK(flodl::launch_ln_bwd(a, cur_stream()));
}

void colsum(const Tensor& m, Tensor& out, const optional<Tensor>& scale) {
  FL_CHECK_CUDA(m);
  FL_CHECK_F32(out);
  const int C = (int)m.size(-1);
  c10::cuda::CUDAGuard guard(m.device());
  if (!m.is_contiguous()) {
    // row-strided 2-D view (e.g. the first V columns of a padded buffer)
    FL_CHECK(m.dim() == 2 && m.stride(1) == 1, "colsum input must be contiguous or a row-strided 2-D view");
    FL_CUDA_OK(flodl::launch_colsum(m.data_ptr(), m.scalar_type() == at::kBFloat16, ptr<float>(out),
                                    (int)m.size(0), C, cur_stream(), opt_ptr<const float>(scale),
                                    (int)m.stride(0)));
    return;
  }
  const int rows = (int)(m.numel() / C);
  const int nb = flodl::colsum_partial_blocks(rows);
  FL_CUDA_OK(flodl::launch_colsum_atomic(m.data_ptr(), m.scalar_type() == at::kBFloat16,
                                         ptr<float>(out), rows, C, nb, cur_stream(),
                                         opt_ptr<const float>(scale)));
}

// Returns nothing; writes loss (scalar, overwritten) and dlogits.
void softmax_ce(const Tensor& logits, const Tensor& targets, Tensor& loss, Tensor& inv_count,
                const optional<Tensor>& dlogits, int64_t ignore_index, double smoothing) {
  FL_CHECK_CUDA(logits);
  FL_CHECK_BF16(logits);
  FL_CHECK(logits.dim() == 2 && logits.stride(1) == 1, "logits must be 2-D row-major");
  FL_CHECK(targets.scalar_type() == at::kLong && targets.is_contiguous(), "targets must be int64");
  const int T = (int)logits.size(0), V = (int)logits.size(1);
  c10::cuda::CUDAGuard guard(logits.device());
  auto st = cur_stream();
  FL_CUDA_OK(flodl::launch_ce_count(ptr<int64_t>(targets), T, V, ignore_index,
                                    ptr<float>(inv_count), ptr<float>(loss), nullptr, st));
  flodl::CeArgs a;
  a.logits = ptr<__nv_bfloat16>(logits);
  a.ld = (int)logits.stride(0);
  a.targets = ptr<int64_t>(targets);
  a.T = T;
  a.V = V;
  a.ignore_index = ignore_index;
  a.smoothing = (float)smoothing;
  a.inv_count = ptr<float>(inv_count);
  a.loss = ptr<float>(loss);
  if (dlogits) {
    FL_CHECK(dlogits->dim() == 2 && dlogits->stride(1) == 1 && dlogits->size(0) == T &&
                 dlogits->size(1) == V,
             "dlogits must be [T, V] row-major (any row pitch)");
    a.dlogits = ptr<__nv_bfloat16>(*dlogits);
    a.ld_d = (int)dlogits->stride(0);
  }
  FL_CUDA_OK(flodl::launch_softmax_ce(a, st));
}

void embed_fwd(const Tensor& ids, const Tensor& tok, const optional<Tensor>& pos,
               const optional<Tensor>& type_ids, const optional<Tensor>& type_tab,
               const optional<Tensor>& out, const optional<Tensor>& out_bf16, int64_t S) {
  FL_CHECK_CUDA(ids);
  FL_CHECK(ids.scalar_type() == at::kLong && ids.is_contiguous(), "ids must be int64");
  FL_CHECK_F32(tok);
  const int C = (int)tok.size(1), V = (int)tok.size(0);
  c10::cuda::CUDAGuard guard(ids.device());
  FL_CUDA_OK(flodl::launch_embed_fwd(ptr<int64_t>(ids), ptr<float>(tok), opt_ptr<float>(pos),
                                     opt_ptr<int64_t>(type_ids), opt_ptr<float>(type_tab),
                                     opt_ptr<float>(out), opt_ptr<__nv_bfloat16>(out_bf16),
                                     (int)ids.numel(), (int)S, C, V, cur_stream()));
}

void embed_bwd_atomic(const Tensor& ids, const Tensor& dy, Tensor& dtok) {
  c10::cuda::CUDAGuard guard(ids.device());
  FL_CHECK_F32(dy);
  FL_CUDA_OK(flodl::launch_embed_bwd_atomic(ptr<int64_t>(ids), ptr<float>(dy), ptr<float>(dtok),
                                            (int)ids.numel(), (int)dtok.size(1), cur_stream()));
}

void pos_grad(const Tensor& dy, Tensor& dpos, int64_t B, int64_t S) {
  c10::cuda::CUDAGuard guard(dy.device());
  FL_CHECK_F32(dy);
  FL_CUDA_OK(flodl::launch_pos_grad(ptr<float>(dy), ptr<float>(dpos), (int)B, (int)S,
                                    (int)dpos.size(1), cur_stream()));
}

void onehot_bf16(const Tensor& ids, Tensor& out) {
  c10::cuda::CUDAGuard guard(ids.device());
  FL_CUDA_OK(flodl::launch_onehot_bf16(ptr<int64_t>(ids), ptr<__nv_bfloat16>(out),
                                       (int)ids.numel(), (int)out.size(1), cur_stream()));
}

void adamw(Tensor& p, Tensor& g, Tensor& m, Tensor& v, const optional<Tensor>& shadow,
           const Tensor& lr, const Tensor& step, const optional<Tensor>& gscale, double beta1,
           double beta2, double eps, double wd, bool decoupled, bool zero_grad) {
  FL_CHECK_F32(p); FL_CHECK_F32(g); FL_CHECK_F32(m); FL_CHECK_F32(v);
  FL_CHECK(p.is_contiguous() && g.is_contiguous() && m.is_contiguous() && v.is_contiguous(),
           "adamw buffers must be contiguous");
  FL_CHECK(g.numel() == p.numel() && m.numel() == p.numel() && v.numel() == p.numel(), "adamw sizes");
  flodl::AdamWArgs a;
  a.p = ptr<float>(p); a.g = ptr<float>(g); a.m = ptr<float>(m); a.v = ptr<float>(v);
  if (shadow) { FL_CHECK_BF16(*shadow); FL_CHECK(shadow->numel() == p.numel(), "shadow size"); }
  a.shadow = opt_ptr<__nv_bfloat16>(shadow);
  a.n = p.numel();
  a.lr = ptr<float>(lr);
  a.step = ptr<float>(step);
  a.gscale = opt_ptr<float>(gscale);
  a.beta1 = (float)beta1; a.beta2 = (float)beta2; a.eps = (float)eps; a.wd = (float)wd;
  a.decoupled = decoupled;
  a.zero_grad = zero_grad;
  c10::cuda::CUDAGuard guard(p.device());
  FL_CUDA_OK(flodl::launch_adamw(a, cur_stream()));
}

void sgd(Tensor& p, Tensor& g, const optional<Tensor>& buf, const optional<Tensor>& shadow,
         const Tensor& lr, const optional<Tensor>& gscale, const optional<Tensor>& first,
         double momentum, double dampening, double wd, bool nesterov, bool zero_grad) {
  FL_CHECK_F32(p); FL_CHECK_F32(g);
  flodl::SgdArgs a;
  a.p = ptr<float>(p); a.g = ptr<float>(g);
  a.buf = opt_ptr<float>(buf);
  a.shadow = opt_ptr<__nv_bfloat16>(shadow);
  a.n = p.numel();
  a.lr = ptr<float>(lr);
  a.gscale = opt_ptr<float>(gscale);
  a.first = opt_ptr<float>(first);
  a.momentum = (float)momentum; a.dampening = (float)dampening; a.wd = (float)wd;
  a.nesterov = nesterov;
  a.zero_grad = zero_grad;
  c10::cuda::CUDAGuard guard(p.device());
  FL_CUDA_OK(flodl::launch_sgd(a, cur_stream()));
}

void sumsq(const Tensor& x, Tensor& out) {
  FL_CHECK_F32(x);
  c10::cuda::CUDAGuard guard(x.device());
  FL_CUDA_OK(flodl::launch_sumsq(ptr<float>(x), x.numel(), ptr<float>(out), cur_stream()));
}

void clip_coef(const Tensor& sumsq_t, double max_norm, Tensor& coef, const optional<Tensor>& norm) {
  c10::cuda::CUDAGuard guard(coef.device());
  FL_CUDA_OK(flodl::launch_clip_coef(ptr<float>(sumsq_t), (float)max_norm, ptr<float>(coef),
                                     opt_ptr<float>(norm), cur_stream()));
}

void add_scalar(Tensor& x, double v) {
  c10::cuda::CUDAGuard guard(x.device());
  FL_CUDA_OK(flodl::launch_add_scalar(ptr<float>(x), (float)v, cur_stream()));
}

void cast_f32_bf16(const Tensor& x, Tensor& y) {
  FL_CHECK_F32(x); FL_CHECK_BF16(y);
  FL_CHECK_CUDA(x);
  FL_CHECK(y.device() == x.device(), "cast devices");
  FL_CHECK(x.numel() == y.numel() && x.is_contiguous() && y.is_contiguous(), "cast sizes");
  c10::cuda::CUDAGuard guard(x.device());
  FL_CUDA_OK(flodl::launch_cast_f32_bf16(ptr<float>(x), ptr<__nv_bfloat16>(y), x.numel(), cur_stream()));
}

void gelu_bwd(const Tensor& dy, const Tensor& h, Tensor& dh) {
  FL_CHECK_BF16(dy); FL_CHECK_BF16(h); FL_CHECK_BF16(dh);
  FL_CHECK(dy.numel() == h.numel() && dh.numel() == h.numel(), "gelu_bwd sizes");
  FL_CHECK(dy.is_contiguous() && h.is_contiguous() && dh.is_contiguous(), "gelu_bwd layout");
  c10::cuda::CUDAGuard guard(h.device());
  FL_CUDA_OK(flodl::launch_gelu_bwd(ptr<__nv_bfloat16>(dy), ptr<__nv_bfloat16>(h),
                                    ptr<__nv_bfloat16>(dh), h.numel(), cur_stream()));
}

void mul_bf16(const Tensor& a, const Tensor& b, Tensor& y) {
  FL_CHECK_CUDA(a);
  FL_CHECK_BF16(a);
  FL_CHECK_BF16(b);
  FL_CHECK_BF16(y);
  FL_CHECK(a.is_contiguous() && b.is_contiguous() && y.is_contiguous() &&
               a.numel() == b.numel() && a.numel() == y.numel(),
           "mul_bf16 layout");
  c10::cuda::CUDAGuard guard(a.device());
  FL_CUDA_OK(flodl::launch_mul_bf16(ptr<__nv_bfloat16>(a), ptr<__nv_bfloat16>(b),
                                    ptr<__nv_bfloat16>(y), a.numel(), cur_stream()));
}

void gelu_eval_f32(const Tensor& x, Tensor& y, Tensor& dydx) {
  FL_CHECK_CUDA(x);
  FL_CHECK_F32(x);
  FL_CHECK_F32(y);
  FL_CHECK_F32(dydx);
  FL_CHECK(x.is_contiguous() && y.is_contiguous() && dydx.is_contiguous() &&
               x.numel() == y.numel() && x.numel() == dydx.numel(),
           "gelu_eval_f32 layout");
  c10::cuda::CUDAGuard guard(x.device());
  FL_CUDA_OK(flodl::launch_gelu_eval_f32(x.data_ptr<float>(), y.data_ptr<float>(),
                                         dydx.data_ptr<float>(), x.numel(), cur_stream()));
}

void gelu_fwd(const Tensor& x, Tensor& y) {
  FL_CHECK_BF16(x); FL_CHECK_BF16(y);
  FL_CHECK(x.is_contiguous() && y.is_contiguous() && x.numel() == y.numel(), "gelu_fwd layout");
  c10::cuda::CUDAGuard guard(x.device());
  FL_CUDA_OK(flodl::launch_gelu_fwd(ptr<__nv_bfloat16>(x), ptr<__nv_bfloat16>(y), x.numel(),
                                    cur_stream()));
}

}  // namespace

void register_norm(py::module& m) {
  m.def("ln_fwd", &ln_fwd, py::arg("x"), py::arg("gamma"), py::arg("beta"), py::arg("y_bf16"),
        py::arg("y_f32"), py::arg("mean"), py::arg("rstd"), py::arg("eps"));
  m.def("ln_bwd", &ln_bwd, py::arg("dy"), py::arg("x"), py::arg("mean"), py::arg("rstd"),
        py::arg("gamma"), py::arg("dres"), py::arg("dx_f32"), py::arg("dx_bf16"),
        py::arg("dgamma"), py::arg("dbeta"), py::arg("colsum"), py::arg("pre_add") = false);
  m.def("colsum", &colsum, py::arg("m"), py::arg("out"), py::arg("scale") = py::none());
}

void register_loss(py::module& m) {
  m.def("softmax_ce", &softmax_ce, py::arg("logits"), py::arg("targets"), py::arg("loss"),
        py::arg("inv_count"), py::arg("dlogits"), py::arg("ignore_index"), py::arg("smoothing"));
}

void register_elementwise(py::module& m) {
  m.def("embed_fwd", &embed_fwd, py::arg("ids"), py::arg("tok"), py::arg("pos"),
        py::arg("type_ids"), py::arg("type_tab"), py::arg("out"), py::arg("out_bf16"), py::arg("S"));
  m.def("embed_bwd_atomic", &embed_bwd_atomic);
  m.def("pos_grad", &pos_grad);
  m.def("onehot_bf16", &onehot_bf16);
  m.def("cast_f32_bf16", &cast_f32_bf16);
  m.def("rms_fwd", &rms_fwd, py::arg("x"), py::arg("w"), py::arg("y"), py::arg("rstd"),
        py::arg("eps"));
  m.def("rms_bwd", &rms_bwd, py::arg("dy"), py::arg("x"), py::arg("w"), py::arg("rstd"),
        py::arg("dx"), py::arg("dw"));
  m.def("qk_norm_rope", &qk_norm_rope, py::arg("q"), py::arg("k"), py::arg("q_weight"),
        py::arg("k_weight"), py::arg("cos"), py::arg("sin"), py::arg("positions"),
        py::arg("offset"), py::arg("eps"));
  m.def("qk_norm_rope_fwd", &qk_norm_rope_fwd, py::arg("q"), py::arg("k"), py::arg("wq"),
        py::arg("wk"), py::arg("cos"), py::arg("sin"), py::arg("pos"), py::arg("offset"),
        py::arg("yq"), py::arg("yk"), py::arg("eps"));
  m.def("qk_norm_rope_backward", [](const Tensor& dyq, const Tensor& dyk, const Tensor& q,
                                    const Tensor& k, const optional<Tensor>& wq,
                                    const optional<Tensor>& wk, const optional<Tensor>& cos,
                                    const optional<Tensor>& sin, const optional<Tensor>& pos,
                                    int64_t offset, double eps, Tensor& dq, Tensor& dk) {
    auto t = [](const optional<Tensor>& x) { return x ? *x : Tensor(); };
    auto [a, b] = qk_norm_rope_backward(dyq, dyk, q, k, t(wq), t(wk), t(cos), t(sin), t(pos), offset,
                                        eps, dq, dk);
    return std::make_pair(some(a), some(b));
  }, py::arg("dyq"), py::arg("dyk"), py::arg("q"), py::arg("k"), py::arg("q_weight"),
        py::arg("k_weight"), py::arg("cos"), py::arg("sin"), py::arg("positions"),
        py::arg("offset"), py::arg("eps"), py::arg("dq"), py::arg("dk"));
  m.def("gn_fwd", &gn_fwd, py::arg("x"), py::arg("gamma"), py::arg("beta"), py::arg("y"),
        py::arg("mean"), py::arg("rstd"), py::arg("groups"), py::arg("eps"));
  m.def("gn_bwd", &gn_bwd, py::arg("dy"), py::arg("x"), py::arg("gamma"), py::arg("mean"),
        py::arg("rstd"), py::arg("dx"), py::arg("dgamma"), py::arg("dbeta"), py::arg("groups"));
  m.def("maxpool_fwd", &maxpool_fwd);
  m.def("maxpool_bwd", &maxpool_bwd);
  m.def("dropout", &dropout, py::arg("x"), py::arg("y"), py::arg("p"), py::arg("seed"),
        py::arg("offset"));
  m.def("gelu_bwd", &gelu_bwd);
  m.def("gelu_fwd", &gelu_fwd);
  m.def("gelu_eval_f32", &gelu_eval_f32);
  m.def("mul_bf16", &mul_bf16);
}

void register_optim(py::module& m) {
  m.def("adamw", &adamw, py::arg("p"), py::arg("g"), py::arg("m"), py::arg("v"),
        py::arg("shadow"), py::arg("lr"), py::arg("step"), py::arg("gscale"), py::arg("beta1"),
        py::arg("beta2"), py::arg("eps"), py::arg("wd"), py::arg("decoupled"),
        py::arg("zero_grad"));
  m.def("sgd", &sgd, py::arg("p"), py::arg("g"), py::arg("buf"), py::arg("shadow"), py::arg("lr"),
        py::arg("gscale"), py::arg("first"), py::arg("momentum"), py::arg("dampening"),
        py::arg("wd"), py::arg("nesterov"), py::arg("zero_grad"));
  m.def("sumsq", &sumsq);
  m.def("clip_coef", &clip_coef, py::arg("sumsq"), py::arg("max_norm"), py::arg("coef"),
        py::arg("norm") = py::none());
  m.def("add_scalar", &add_scalar);
}
