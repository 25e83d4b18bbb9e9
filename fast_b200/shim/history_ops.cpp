// `history_ops`: the event-history operators on torch tensors, over the
// libfast_b200 C ABI -- checks of the arguments, outputs and workspaces from
// torch's allocator, torch's current stream of the inputs' device.
// Bad operands raise ValueError, library errors fast_b200.capi.FastB200Error.
#include "tensor_args.h"

#include <cmath>

namespace {

// fp32, contiguous, on the inputs' device, of the given shape.
void params(const Tensor &t, const std::string &name, const Tensor &like, at::IntArrayRef shape) {
  if (t.scalar_type() != at::kFloat || !t.is_cuda() || t.get_device() != like.get_device() || !t.is_contiguous() ||
      t.sizes() != shape) {
    std::string s;
    for (const int64_t n : shape) s += (s.empty() ? "" : ", ") + std::to_string(n);
    refuse(name + " must be a contiguous CUDA fp32 tensor of shape [" + s + "] on the inputs' device");
  }
}
void params(const OptTensor &t, const std::string &name, const Tensor &like, at::IntArrayRef shape) {
  if (t) params(*t, name, like, shape);
}

// Per-sequence states [n, a, b] of `type`, contiguous.
void states(const Tensor &t, const std::string &name, at::ScalarType type, const Tensor &like, int64_t n, int64_t a, int64_t b) {
  if (t.scalar_type() != type || t.dim() != 3 || !t.is_cuda() || t.get_device() != like.get_device() || !t.is_contiguous() ||
      (n >= 0 && t.size(0) != n) || t.size(1) != a || t.size(2) != b)
    refuse(name + " must be a contiguous CUDA " + type_name(type) + " tensor of shape [" +
           (n < 0 ? "states" : std::to_string(n)) + ", " + std::to_string(a) + ", " + std::to_string(b) +
           "] on the inputs' device");
}

// Number of sequences; the type of their starts.
int64_t sequences(const OptTensor &starts, const char *name, const Tensor &like, const void *&p, int &type) {
  p = nullptr, type = FB_I64;
  if (!starts) return 1;
  const Tensor &t = *starts;
  if ((t.scalar_type() != at::kLong && t.scalar_type() != at::kInt) || t.dim() != 1 || t.size(0) < 1 || !t.is_cuda() ||
      t.get_device() != like.get_device() || !t.is_contiguous())
    refuse(std::string(name) + " starts must be a contiguous CUDA int64 or int32 vector of at least one element on the inputs' device");
  p = t.data_ptr();
  type = t.scalar_type() == at::kLong ? FB_I64 : FB_I32;
  return t.size(0) - 1;
}

int width(int64_t n, const char *name) {
  if (n < 1 || n > (1 << 20)) refuse(std::string(name) + ": rows must be 1 to 1,048,576 wide");
  return (int)n;
}

// ---- short convolution ---------------------------------------------------------------------------
fb_short_conv conv_args(const Tensor &x, const Tensor &w, const OptTensor &bias, const OptTensor &starts, const OptTensor &init,
                        int act, const std::string &name) {
  fb_short_conv a{};
  a.type = head_type(x, (name + " x").c_str());
  rows(x, (name + " x").c_str(), x.scalar_type(), x);
  a.act = act;
  a.rows = x.size(0), a.D = width(x.size(1), name.c_str());
  if (w.dim() != 2 || w.size(1) < 1 || w.size(1) > 8) refuse(name + " w must be a matrix [D, K] with 1 to 8 taps");
  a.K = (int)w.size(1);
  params(w, name + " w", x, {a.D, a.K});
  params(bias, name + " bias", x, {a.D});
  a.seqs = sequences(starts, name.c_str(), x, a.starts, a.starts_type);
  if (init) states(*init, name + " init", x.scalar_type(), x, a.seqs, a.K - 1, a.D);
  a.x = ptr(x), a.ldx = ld(x);
  a.w = (const float *)ptr(w), a.bias = (const float *)ptr(bias);
  a.init = ptr(init);
  return a;
}

py::object short_conv_fwd(const Tensor &x, const Tensor &w, const OptTensor &bias, const OptTensor &starts, const OptTensor &init,
                          int act, bool final) {
  fb_short_conv a = conv_args(x, w, bias, starts, init, act, "short_conv_fwd");
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor y = empty({a.rows, a.D}, x, x.scalar_type());
  a.y = ptr(y), a.ldy = a.D;
  Tensor f;
  if (final) f = empty({a.seqs, a.K - 1, a.D}, x, x.scalar_type()), a.final = ptr(f);
  const Count count;
  check(fb_short_conv_fwd(&a, nullptr, 0, stream_of(x)));
  return final ? py::object(py::make_tuple(y, f)) : py::cast(y);
}

py::tuple short_conv_bwd(const Tensor &dy, const Tensor &x, const Tensor &w, const OptTensor &bias, const OptTensor &starts,
                         const OptTensor &init, int act, const OptTensor &dfinal) {
  fb_short_conv a = conv_args(x, w, bias, starts, init, act, "short_conv_bwd");
  rows(dy, "short_conv_bwd dy", x.scalar_type(), x, a.rows, a.D);
  if (dfinal) states(*dfinal, "short_conv_bwd dfinal", x.scalar_type(), x, a.seqs, a.K - 1, a.D);
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor dx = empty({a.rows, a.D}, x, x.scalar_type());
  const Tensor dw = empty({a.D, a.K}, x, at::kFloat), db = empty({a.D}, x, at::kFloat);
  Tensor di;
  if (init) di = empty({a.seqs, a.K - 1, a.D}, x, x.scalar_type()), a.dinit = ptr(di);
  a.dy = ptr(dy), a.lddy = ld(dy), a.dfinal = ptr(dfinal);
  a.dx = ptr(dx), a.lddx = a.D, a.dw = (float *)ptr(dw), a.dbias = (float *)ptr(db);
  const size_t nb = fb_short_conv_ws_bytes(&a, 1);
  const Tensor ws = empty({(int64_t)nb}, x, at::kByte);
  const Count count;
  check(fb_short_conv_bwd(&a, ptr(ws), nb, stream_of(x)));
  return py::make_tuple(dx, dw, bias ? py::cast(db) : py::none(), init ? py::cast(di) : py::none());
}

const int64_t *index_of(const OptTensor &index, const char *name, const Tensor &like, int64_t n, int64_t states) {
  if (!index) {
    if (n > states) refuse(std::string(name) + ": more rows than states and no index");
    return nullptr;
  }
  vec(*index, (std::string(name) + " index").c_str(), at::kLong, like, n);
  return (const int64_t *)ptr(*index);
}

Tensor short_conv_step(const Tensor &x, const Tensor &state, const Tensor &w, const OptTensor &bias, const OptTensor &index,
                       int act) {
  const int type = head_type(x, "short_conv_step x");
  rows(x, "short_conv_step x", x.scalar_type(), x);
  const int64_t n = x.size(0);
  const int D = width(x.size(1), "short_conv_step");
  if (w.dim() != 2 || w.size(1) < 1 || w.size(1) > 8) refuse("short_conv_step w must be a matrix [D, K] with 1 to 8 taps");
  const int K = (int)w.size(1);
  params(w, "short_conv_step w", x, {D, K});
  params(bias, "short_conv_step bias", x, {D});
  states(state, "short_conv_step state", x.scalar_type(), x, -1, K - 1, D);
  const int64_t *at = index_of(index, "short_conv_step", x, n, state.size(0));
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor y = empty({n, D}, x, x.scalar_type());
  const size_t nb = at ? fb_event_step_ws_bytes(n) : 0;
  Tensor ws;
  if (nb) ws = empty({(int64_t)nb}, x, at::kByte);
  const Count count;
  check(fb_short_conv_step(type, act, ptr(x), ld(x), (const float *)ptr(w), (const float *)ptr(bias), ptr(state), state.size(0),
                           at, ptr(y), D, n, D, K, nb ? ptr(ws) : nullptr, nb, stream_of(x)));
  return y;
}

// ---- selective scan --------------------------------------------------------------------------------
// B or C [rows, N] or [rows, G, N]: (groups, row pitch, group pitch).
struct Group {
  int64_t G, N, ld, gs;
};
Group grouped(const Tensor &t, const std::string &name, const Tensor &like, int64_t n) {
  if (t.scalar_type() != like.scalar_type() || (t.dim() != 2 && t.dim() != 3) || !t.is_cuda() || t.get_device() != like.get_device())
    refuse(name + " must be a CUDA " + type_name(like.scalar_type()) + " tensor [rows, N] or [rows, groups, N] on the inputs' device");
  const int64_t G = t.dim() == 3 ? t.size(1) : 1, N = t.size(-1);
  if (t.size(0) != n || G < 1 || N < 1) refuse(name + " must have a row for each of the inputs', and at least one group and state");
  if (N > 1 && t.stride(-1) != 1) refuse(name + " must have unit stride along the states");
  const int64_t gs = t.dim() == 3 && G > 1 ? t.stride(1) : N;
  if (gs < 0 || (n > 1 && t.stride(0) < 0)) refuse(name + " must not have negative strides");
  return {G, N, n > 1 ? t.stride(0) : G * N, gs};
}

template <typename Args>
void scan_args(Args &a, const std::string &name, const Tensor &u, const Tensor &delta, const Tensor &A, const Tensor &B,
               const Tensor &C, const OptTensor &D, const OptTensor &z, const OptTensor &delta_bias, bool softplus) {
  a.type = head_type(u, (name + " u").c_str());
  rows(u, (name + " u").c_str(), u.scalar_type(), u);
  const int64_t n = u.size(0);
  a.D = width(u.size(1), name.c_str());
  a.softplus = softplus;
  rows(delta, (name + " delta").c_str(), u.scalar_type(), u, n, a.D);
  if (z) rows(*z, (name + " z").c_str(), u.scalar_type(), u, n, a.D);
  const Group gb = grouped(B, name + " B", u, n), gc = grouped(C, name + " C", u, n);
  if (gb.G != gc.G || gb.N != gc.N) refuse(name + ": B and C must have the same groups and states");
  if (gb.N > 64) refuse(name + ": at most 64 states");
  if (a.D % gb.G) refuse(name + ": the groups must divide the width");
  a.G = (int)gb.G, a.N = (int)gb.N;
  params(A, name + " A", u, {a.D, a.N});
  params(D, name + " D", u, {a.D});
  params(delta_bias, name + " delta_bias", u, {a.D});
  a.u = ptr(u), a.ldu = ld(u), a.delta = ptr(delta), a.ld_delta = ld(delta);
  a.B = ptr(B), a.ldb = gb.ld, a.ldb_group = gb.gs, a.C = ptr(C), a.ldc = gc.ld, a.ldc_group = gc.gs;
  a.z = ptr(z), a.ldz = z ? ld(*z) : 0;
  a.A = (const float *)ptr(A), a.skip = (const float *)ptr(D), a.delta_bias = (const float *)ptr(delta_bias);
}

void scan_sequences(fb_selective_scan &a, const std::string &name, const Tensor &u, const OptTensor &starts, const OptTensor &init) {
  a.rows = u.size(0);
  a.seqs = sequences(starts, name.c_str(), u, a.starts, a.starts_type);
  if (init) states(*init, name + " init", at::kFloat, u, a.seqs, a.D, a.N);
  a.init = (const float *)ptr(init);
}

py::tuple selective_scan_fwd(const Tensor &u, const Tensor &delta, const Tensor &A, const Tensor &B, const Tensor &C,
                             const OptTensor &D, const OptTensor &z, const OptTensor &delta_bias, const OptTensor &starts,
                             const OptTensor &init, bool softplus, bool final, bool keep) {
  fb_selective_scan a{};
  const std::string name = "selective_scan_fwd";
  scan_args(a, name, u, delta, A, B, C, D, z, delta_bias, softplus);
  scan_sequences(a, name, u, starts, init);
  const c10::cuda::CUDAGuard guard(u.device());
  const Tensor y = empty({a.rows, a.D}, u, u.scalar_type());
  a.y = ptr(y), a.ldy = a.D;
  Tensor f, k;
  if (final) f = empty({a.seqs, a.D, a.N}, u, at::kFloat), a.final = (float *)ptr(f);
  if (keep) k = empty({(a.rows + 7) / 8, a.D, a.N}, u, at::kFloat), a.keep = (float *)ptr(k);
  const size_t nb = fb_selective_scan_ws_bytes(&a, 0);
  Tensor ws;
  if (nb) ws = empty({(int64_t)nb}, u, at::kByte);
  const Count count;
  check(fb_selective_scan_fwd(&a, nb ? ptr(ws) : nullptr, nb, stream_of(u)));
  return py::make_tuple(y, keep ? py::cast(k) : py::none(), final ? py::cast(f) : py::none());
}

py::tuple selective_scan_bwd(const Tensor &dy, const Tensor &u, const Tensor &delta, const Tensor &A, const Tensor &B,
                             const Tensor &C, const Tensor &carry, const OptTensor &D, const OptTensor &z,
                             const OptTensor &delta_bias, const OptTensor &starts, const OptTensor &init, bool softplus,
                             const OptTensor &dfinal) {
  fb_selective_scan a{};
  const std::string name = "selective_scan_bwd";
  scan_args(a, name, u, delta, A, B, C, D, z, delta_bias, softplus);
  scan_sequences(a, name, u, starts, init);
  rows(dy, "selective_scan_bwd dy", u.scalar_type(), u, a.rows, a.D);
  states(carry, name + " carry", at::kFloat, u, (a.rows + 7) / 8, a.D, a.N);
  if (dfinal) states(*dfinal, name + " dfinal", at::kFloat, u, a.seqs, a.D, a.N);
  const c10::cuda::CUDAGuard guard(u.device());
  const auto t = u.scalar_type();
  const Tensor du = empty({a.rows, a.D}, u, t), dd = empty({a.rows, a.D}, u, t);
  const Tensor dB = empty(B.sizes(), u, t), dC = empty(C.sizes(), u, t);
  const Tensor dA = empty({a.D, a.N}, u, at::kFloat), dD = empty({a.D}, u, at::kFloat), db = empty({a.D}, u, at::kFloat);
  Tensor dz, di;
  if (z) dz = empty({a.rows, a.D}, u, t), a.dz = ptr(dz);
  if (init) di = empty({a.seqs, a.D, a.N}, u, at::kFloat), a.dinit = (float *)ptr(di);
  a.keep = (float *)ptr(carry);
  a.dy = ptr(dy), a.lddy = ld(dy), a.dfinal = (const float *)ptr(dfinal);
  a.du = ptr(du), a.ddelta = ptr(dd), a.dB = ptr(dB), a.dC = ptr(dC);
  a.dA = (float *)ptr(dA), a.dD = (float *)ptr(dD), a.ddelta_bias = (float *)ptr(db);
  const size_t nb = fb_selective_scan_ws_bytes(&a, 1);
  Tensor ws;
  if (nb) ws = empty({(int64_t)nb}, u, at::kByte);
  const Count count;
  check(fb_selective_scan_bwd(&a, nb ? ptr(ws) : nullptr, nb, stream_of(u)));
  const py::object none = py::none();
  return py::make_tuple(du, dd, dA, dB, dC, D ? py::cast(dD) : none, z ? py::cast(dz) : none,
                        delta_bias ? py::cast(db) : none, init ? py::cast(di) : none);
}

Tensor selective_scan_step(const Tensor &u, const Tensor &delta, const Tensor &A, const Tensor &B, const Tensor &C,
                           const Tensor &state, const OptTensor &D, const OptTensor &z, const OptTensor &delta_bias,
                           const OptTensor &index, bool softplus) {
  fb_selective_scan_event a{};
  const std::string name = "selective_scan_step";
  scan_args(a, name, u, delta, A, B, C, D, z, delta_bias, softplus);
  a.n = u.size(0);
  states(state, name + " state", at::kFloat, u, -1, a.D, a.N);
  a.states = state.size(0);
  a.index = index_of(index, name.c_str(), u, a.n, a.states);
  a.state = (float *)ptr(state);
  const c10::cuda::CUDAGuard guard(u.device());
  const Tensor y = empty({a.n, a.D}, u, u.scalar_type());
  a.y = ptr(y), a.ldy = a.D;
  const size_t nb = a.index ? fb_event_step_ws_bytes(a.n) : 0;
  Tensor ws;
  if (nb) ws = empty({(int64_t)nb}, u, at::kByte);
  const Count count;
  check(fb_selective_scan_step(&a, nb ? ptr(ws) : nullptr, nb, stream_of(u)));
  return y;
}

// ---- dropout -----------------------------------------------------------------------------------------
Tensor dropout(const Tensor &x, double p, uint64_t seed, uint64_t offset, const OptTensor &res, const OptTensor &offset_dev) {
  const int type = head_type(x, "dropout x");
  rows(x, "dropout x", x.scalar_type(), x);
  const int64_t n = x.size(0);
  const int D = width(x.size(1), "dropout");
  if (!(p >= 0.0 && p < 1.0) || (float)p >= 1.f) refuse("dropout: p must be in [0, 1)");
  if (n >= (int64_t)1 << 32) refuse("dropout: at most 2^32 - 1 rows");
  if (res) rows(*res, "dropout res", x.scalar_type(), x, n, D);
  if (offset_dev) vec(*offset_dev, "dropout offset_dev", at::kLong, x, 1);
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor y = empty({n, D}, x, x.scalar_type());
  const Count count;
  check(fb_dropout(type, ptr(x), ld(x), ptr(res), res ? ld(*res) : 0, ptr(y), D, n, D, (float)p, seed, offset,
                   (const int64_t *)ptr(offset_dev), stream_of(x)));
  return y;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "Event-history operators of fast_b200 (wrapped by fast_b200.ops)";
  m.def("count_into", [](py::list counter) { count_list() = counter.release(); },
        "Adds every call's kernel launches to element 0 of a list");
  m.def("short_conv_fwd", &short_conv_fwd);
  m.def("short_conv_bwd", &short_conv_bwd);
  m.def("short_conv_step", &short_conv_step);
  m.def("selective_scan_fwd", &selective_scan_fwd);
  m.def("selective_scan_bwd", &selective_scan_bwd);
  m.def("selective_scan_step", &selective_scan_step);
  m.def("dropout", &dropout);
}
