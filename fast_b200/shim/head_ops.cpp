// `head_ops`: the node-ranking head's operators on torch tensors, over the
// libfast_b200 C ABI -- checks of the arguments, outputs and workspaces from
// torch's allocator, torch's current stream of the inputs' device.  Small
// calls of these operators are bound by the host: the same wrapper in Python
// (ctypes) took 19 us for a layer norm whose kernel takes 3.
// Bad operands raise ValueError, library errors fast_b200.capi.FastB200Error.
#include "tensor_args.h"

namespace {

// ---- layer norm --------------------------------------------------------------------------------
int norm_params(const Tensor &x, const Tensor &gamma, const OptTensor &beta, const char *name) {
  const auto bad = [&](const Tensor &t) {
    return (t.scalar_type() != at::kFloat && t.scalar_type() != x.scalar_type()) ||
           t.scalar_type() != gamma.scalar_type() || !t.is_cuda() || t.get_device() != x.get_device() || t.dim() != 1 ||
           t.size(0) != x.size(1) || !t.is_contiguous();
  };
  if (bad(gamma) || (beta && bad(*beta)))
    refuse(std::string(name) + ": gamma and beta must be contiguous CUDA vectors of the row width, fp32 or of the "
                               "rows' type, on the rows' device");
  return gamma.scalar_type() == at::kFloat ? FB_F32 : FB_BF16;
}

py::tuple layer_norm_fwd(const Tensor &x, const Tensor &gamma, const OptTensor &beta, double eps, const OptTensor &res) {
  const int type = head_type(x, "layer_norm_fwd x");
  rows(x, "layer_norm_fwd x", x.scalar_type(), x);
  const int pt = norm_params(x, gamma, beta, "layer_norm_fwd");
  const int64_t n = x.size(0), D = x.size(1);
  if (res) rows(*res, "layer_norm_fwd res", x.scalar_type(), x, n, D);
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor y = empty({n, D}, x, x.scalar_type()), s;
  Tensor mean = empty({n}, x, at::kFloat), rstd = empty({n}, x, at::kFloat);
  if (res) s = empty({n, D}, x, x.scalar_type());
  const Count count;
  check(fb_layer_norm_fwd(type, ptr(x), ld(x), ptr(res), res ? ld(*res) : 0, ptr(gamma), ptr(beta), pt, (float)eps,
                          res ? ptr(s) : nullptr, D, ptr(y), D, (float *)ptr(mean), (float *)ptr(rstd), n, (int)D,
                          stream_of(x)));
  return res ? py::make_tuple(y, s, mean, rstd) : py::make_tuple(y, mean, rstd);
}

py::tuple layer_norm_bwd(const Tensor &dy, const Tensor &x, const Tensor &gamma, const Tensor &mean, const Tensor &rstd,
                         const OptTensor &ds, const OptTensor &dgamma, const OptTensor &dbeta) {
  const int type = head_type(x, "layer_norm_bwd x");
  rows(x, "layer_norm_bwd x", x.scalar_type(), x);
  const int64_t n = x.size(0), D = x.size(1);
  rows(dy, "layer_norm_bwd dy", x.scalar_type(), x, n, D);
  const int pt = norm_params(x, gamma, std::nullopt, "layer_norm_bwd");
  vec(mean, "layer_norm_bwd mean", at::kFloat, x, n);
  vec(rstd, "layer_norm_bwd rstd", at::kFloat, x, n);
  if (ds) rows(*ds, "layer_norm_bwd ds", x.scalar_type(), x, n, D);
  const c10::cuda::CUDAGuard guard(x.device());
  const bool acc = dgamma || dbeta;
  if (acc) {
    if (!dgamma || !dbeta || pt != FB_F32)
      refuse("layer_norm_bwd: dgamma and dbeta to accumulate into must be given together, beside an fp32 gamma");
    vec(*dgamma, "layer_norm_bwd dgamma", at::kFloat, x, D);
    vec(*dbeta, "layer_norm_bwd dbeta", at::kFloat, x, D);
  }
  const Tensor dg = acc ? *dgamma : empty({D}, x, gamma.scalar_type());
  const Tensor db = acc ? *dbeta : empty({D}, x, gamma.scalar_type());
  const Tensor dx = empty({n, D}, x, x.scalar_type());
  const size_t nb = fb_layer_norm_bwd_ws_bytes(n, (int)D);
  const Tensor ws = empty({(int64_t)nb}, x, at::kByte);
  const Count count;
  check(fb_layer_norm_bwd(type, ptr(dy), ld(dy), ptr(x), ld(x), ptr(gamma), pt, (const float *)ptr(mean),
                          (const float *)ptr(rstd), ptr(ds), ds ? ld(*ds) : 0, ptr(dx), D, ptr(dg), ptr(db), acc, n,
                          (int)D, ptr(ws), nb, stream_of(x)));
  return py::make_tuple(dx, dg, db);
}

// A weight gradient: fresh, of the weights' type or (f32) fp32, or the fp32 buffer given.
Tensor grad(const OptTensor &given, const char *name, const Tensor &like, int64_t r, int64_t c, bool f32) {
  if (!given) return empty({r, c}, like, f32 ? at::kFloat : like.scalar_type());
  rows(*given, name, at::kFloat, like, r, c);
  return *given;
}

// ---- gated feed-forward block ------------------------------------------------------------------
fb_gated_ffn ffn_args(const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd, int act) {
  fb_gated_ffn a{};
  a.type = a.grad_type = head_type(x, "gated_ffn x");
  const auto st = x.scalar_type();
  rows(x, "gated_ffn x", st, x);
  a.n = x.size(0);
  const int64_t D = x.size(1);
  rows(wg, "gated_ffn w_gate", st, x, -1, D);
  const int64_t F = wg.size(0);
  rows(wu, "gated_ffn w_up", st, x, F, D);
  rows(wd, "gated_ffn w_down", st, x, D, F);
  a.act = act;
  a.D = (int)D, a.F = (int)F;
  a.x = ptr(x), a.ldx = ld(x);
  a.w_gate = ptr(wg), a.ld_gate = ld(wg);
  a.w_up = ptr(wu), a.ld_up = ld(wu);
  a.w_down = ptr(wd), a.ld_down = ld(wd);
  return a;
}

Tensor gated_ffn_fwd(const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd, int act) {
  fb_gated_ffn a = ffn_args(x, wg, wu, wd, act);
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor y = empty({a.n, a.D}, x, x.scalar_type());
  a.y = ptr(y), a.ldy = a.D;
  const size_t nb = fb_gated_ffn_ws_bytes(&a, 0);
  const Tensor ws = empty({(int64_t)nb}, x, at::kByte);
  const Count count;
  check(fb_gated_ffn_fwd(&a, ptr(ws), nb, stream_of(x)));
  return y;
}

py::tuple gated_ffn_bwd(const Tensor &dy, const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd, int act,
                        const std::optional<std::vector<Tensor>> &grads, bool f32) {
  fb_gated_ffn a = ffn_args(x, wg, wu, wd, act);
  rows(dy, "gated_ffn_bwd dy", x.scalar_type(), x, a.n, a.D);
  if (grads && grads->size() != 3) refuse("gated_ffn_bwd: 3 gradient buffers expected");
  const c10::cuda::CUDAGuard guard(x.device());
  const auto given = [&](int i) { return grads ? OptTensor((*grads)[i]) : std::nullopt; };
  const Tensor dg = grad(given(0), "gated_ffn_bwd gradient buffer", x, a.F, a.D, f32);
  const Tensor du = grad(given(1), "gated_ffn_bwd gradient buffer", x, a.F, a.D, f32);
  const Tensor dd = grad(given(2), "gated_ffn_bwd gradient buffer", x, a.D, a.F, f32);
  const Tensor dx = empty({a.n, a.D}, x, x.scalar_type());
  if (grads || f32) a.grad_type = FB_F32;
  a.accumulate = grads.has_value();
  a.dy = ptr(dy), a.lddy = ld(dy);
  a.dx = ptr(dx), a.lddx = a.D;
  a.dw_gate = ptr(dg), a.ldd_gate = ld(dg);
  a.dw_up = ptr(du), a.ldd_up = ld(du);
  a.dw_down = ptr(dd), a.ldd_down = ld(dd);
  const size_t nb = fb_gated_ffn_ws_bytes(&a, 1);
  const Tensor ws = empty({(int64_t)nb}, x, at::kByte);
  const Count count;
  check(fb_gated_ffn_bwd(&a, ptr(ws), nb, stream_of(x)));
  return py::make_tuple(dx, dg, du, dd);
}

// ---- softmax cross entropy ---------------------------------------------------------------------
fb_softmax_xent xent_args(const Tensor &h, const Tensor &w, const Tensor &target) {
  fb_softmax_xent a{};
  a.type = a.grad_type = head_type(h, "softmax_xent h");
  rows(h, "softmax_xent h", h.scalar_type(), h);
  a.n = h.size(0);
  rows(w, "softmax_xent w", h.scalar_type(), h, -1, h.size(1));
  vec(target, "softmax_xent target", at::kLong, h, a.n);
  a.D = (int)h.size(1), a.V = w.size(0);
  a.h = ptr(h), a.ldh = ld(h);
  a.w = ptr(w), a.ldw = ld(w);
  a.target = (const int64_t *)ptr(target);
  return a;
}

py::tuple softmax_xent_fwd(const Tensor &h, const Tensor &w, const Tensor &target) {
  fb_softmax_xent a = xent_args(h, w, target);
  const c10::cuda::CUDAGuard guard(h.device());
  const Tensor loss = empty({a.n}, h, at::kFloat), lse = empty({a.n}, h, at::kFloat);
  a.loss = (float *)ptr(loss), a.lse = (float *)ptr(lse);
  const size_t nb = fb_softmax_xent_ws_bytes(&a, 0);
  const Tensor ws = empty({(int64_t)nb}, h, at::kByte);
  const Count count;
  check(fb_softmax_xent_fwd(&a, ptr(ws), nb, stream_of(h)));
  return py::make_tuple(loss, lse);
}

py::tuple softmax_xent_bwd(const Tensor &h, const Tensor &w, const Tensor &target, const Tensor &lse,
                           const Tensor &dloss, const OptTensor &dw_in, bool f32) {
  fb_softmax_xent a = xent_args(h, w, target);
  vec(lse, "softmax_xent_bwd lse", at::kFloat, h, a.n);
  vec(dloss, "softmax_xent_bwd dloss", at::kFloat, h, a.n);
  const c10::cuda::CUDAGuard guard(h.device());
  const Tensor dh = empty({a.n, a.D}, h, h.scalar_type());
  const Tensor dw = grad(dw_in, "softmax_xent_bwd dw", h, a.V, a.D, f32);
  if (dw_in || f32) a.grad_type = FB_F32;
  a.accumulate = dw_in.has_value();
  a.lse = (float *)ptr(lse), a.dloss = (const float *)ptr(dloss);
  a.dh = ptr(dh), a.lddh = a.D;
  a.dw = ptr(dw), a.lddw = ld(dw);
  const size_t nb = fb_softmax_xent_ws_bytes(&a, 1);
  const Tensor ws = empty({(int64_t)nb}, h, at::kByte);
  const Count count;
  check(fb_softmax_xent_bwd(&a, ptr(ws), nb, stream_of(h)));
  return py::make_tuple(dh, dw);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "Node-ranking head operators of fast_b200 (wrapped by fast_b200.ops)";
  m.def("count_into", [](py::list counter) { count_list() = counter.release(); },
        "Adds every call's kernel launches to element 0 of a list");
  m.def("layer_norm_fwd", &layer_norm_fwd);
  m.def("layer_norm_bwd", &layer_norm_bwd);
  m.def("gated_ffn_fwd", &gated_ffn_fwd);
  m.def("gated_ffn_bwd", &gated_ffn_bwd);
  m.def("softmax_xent_fwd", &softmax_xent_fwd);
  m.def("softmax_xent_bwd", &softmax_xent_bwd);
}
