// Torch-side of the state-space operators and the slot maps (part of the _cc1d_torch module): the
// argument checks of the package's public functions (ssm.py), outputs and workspaces from torch's
// caching allocator, the device guard, torch's current stream, then the C ABI of
// include/causal_conv1d_b200.h. All of it is C++ because it is all that a small call costs: a decode
// step's kernel runs for 4 us, and the same checks written in Python took 17.
//
// Bad arguments raise AssertionError (shapes, devices) and TypeError (element types), forward-mode tangents
// NotImplementedError, a failing library call the package's CausalConv1dError; inside the autograd Function, which runs on torch's
// own threads, it is a RuntimeError.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/extension.h>

#include <initializer_list>
#include <string>
#include <tuple>
#include <vector>

#include "causal_conv1d_b200.h"

namespace {

namespace py = pybind11;
using Opt = c10::optional<at::Tensor>;

PyObject* g_error = nullptr;  // the package's CausalConv1dError

[[noreturn]] void raise(PyObject* type, const std::string& text) {
  PyErr_SetString(type, text.c_str());
  throw py::error_already_set();
}
inline void need(bool ok, const char* text) {
  if (!ok) raise(PyExc_AssertionError, text);
}
std::string reason(int rc, const char* what) {
  std::string m = std::string(what) + ": " + cc1d_error_string(rc);
  if (rc == CC1D_ERR_CUDA) m += " (cudaError " + std::to_string(cc1d_last_cuda_error()) + ")";
  return m;
}
void check(int rc, const char* what) {
  if (rc != CC1D_OK) raise(g_error != nullptr ? g_error : PyExc_RuntimeError, reason(rc, what));
}

int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return CC1D_F32;
    case at::kHalf: return CC1D_F16;
    case at::kBFloat16: return CC1D_BF16;
    default: return -1;
  }
}
const char* name(const at::Tensor& t) { return c10::toString(t.scalar_type()); }

void* stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
const int32_t* ints(const Opt& t) { return t.has_value() ? t->data_ptr<int32_t>() : nullptr; }
at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt);
}

// One entry per token, (batch, seqlen, channels) or (batch, seqlen, groups, dstate); without the
// seqlen dimension where `one` (a decode step of one token).
cc1d_tokens tokens(const at::Tensor& t, bool one = false) {
  const int64_t g = one ? 1 : 2;
  return {t.data_ptr(), t.stride(0), one ? 0 : t.stride(1), t.dim() == g + 2 ? t.stride(g) : 0};
}
cc1d_param param(const Opt& t) {
  if (!t.has_value()) return {nullptr, CC1D_F32};
  return {t->data_ptr(), dtype_code(*t)};
}

cc1d_ssm_problem problem(const at::Tensor& x, const at::Tensor& dt, const at::Tensor& A, const at::Tensor& B,
                         const at::Tensor& C, const Opt& D, const Opt& z, const Opt& dt_bias, bool softplus,
                         const Opt& seq_idx, const Opt& init, bool one = false) {
  cc1d_ssm_problem q{};
  q.x = tokens(x, one), q.dt = tokens(dt, one), q.B = tokens(B, one), q.C = tokens(C, one);
  if (z.has_value()) q.z = tokens(*z, one);
  q.A = param(A), q.D = param(D), q.dt_bias = param(dt_bias), q.initial_states = param(init);
  q.seq_idx = ints(seq_idx);
  q.batch = x.size(0), q.seqlen = one ? 1 : x.size(1), q.dim = x.size(-1), q.dstate = A.size(1);
  q.groups = B.dim() == x.dim() + 1 ? B.size(-2) : 1;
  q.x_dtype = dtype_code(x), q.dt_softplus = softplus ? 1 : 0;
  return q;
}

// Shapes, element types and devices common to the scan and the update; `one` as above.
void check_operands(const at::Tensor& x, const at::Tensor& dt, const at::Tensor& A, const at::Tensor& B,
                    const at::Tensor& C, const Opt& D, const Opt& z, const Opt& dt_bias, bool one) {
  const int64_t lead = one ? 1 : 2, dim = x.size(lead);
  need(dt.sizes() == x.sizes(), "dt must have the shape of x");
  need(!z.has_value() || z->sizes() == x.sizes(), "z must have the shape of x");
  need(A.dim() == 2 && A.size(0) == dim && A.size(1) >= 1, "A must be (dim, dstate)");
  need(A.size(1) <= 64, "dstate must be at most 64");
  const char* form = one ? "B and C must be (batch, [groups,] dstate)" : "B and C must be (batch, seqlen, [groups,] dstate)";
  need(B.sizes() == C.sizes() && (B.dim() == lead + 1 || B.dim() == lead + 2), form);
  need(B.sizes().slice(0, lead) == x.sizes().slice(0, lead) && B.size(-1) == A.size(1), form);
  need(B.dim() == lead + 1 || (B.size(lead) >= 1 && dim % B.size(lead) == 0),
       "dim must be a multiple of the groups of B and C");
  need(!D.has_value() || (D->dim() == 1 && D->size(0) == dim), "D must be (dim,)");
  need(!dt_bias.has_value() || (dt_bias->dim() == 1 && dt_bias->size(0) == dim), "dt_bias must be (dim,)");
  auto here = [&](const at::Tensor& t) { need(t.device() == x.device(), "all operands must be on x's device"); };
  here(dt), here(A), here(B), here(C);
  for (const Opt* t : {&D, &z, &dt_bias})
    if (t->has_value()) here(**t);
  if (dtype_code(x) < 0) raise(PyExc_TypeError, std::string("x must be float32, float16 or bfloat16, got ") + name(x));
  auto same = [&](const at::Tensor& t) {
    if (t.scalar_type() != x.scalar_type())
      raise(PyExc_TypeError, std::string("dt, B, C and z must have x's dtype ") + name(x) + ", got " + name(t));
  };
  same(dt), same(B), same(C);
  if (z.has_value()) same(*z);
  auto floating = [&](const at::Tensor& t) {
    if (!t.is_floating_point()) raise(PyExc_TypeError, std::string("A, D and dt_bias must be floating point, got ") + name(t));
  };
  floating(A);
  for (const Opt* t : {&D, &dt_bias})
    if (t->has_value()) floating(**t);
  need(x.is_cuda(), "x must be on a CUDA device");
}

// Forward-mode derivatives: the kernels have none, and tensors that carry a tangent (torch.autograd.forward_ad)
// would come out without one, which reads as a derivative of zero. Tensors have tangents only inside a
// forward-mode level; torch allows one, of index 0, and asking for it costs less than asking every operand.
void refuse_tangents(std::initializer_list<const at::Tensor*> given, std::initializer_list<const Opt*> optional) {
  if (torch::autograd::ForwardADLevel::try_get_by_idx(0) == nullptr) return;
  auto check = [](const at::Tensor& t) {
    if (t._fw_grad(0).defined()) raise(PyExc_NotImplementedError, "the state-space operators have no forward-mode derivatives");
  };
  for (const at::Tensor* t : given) check(*t);
  for (const Opt* t : optional)
    if (t->has_value()) check(**t);
}

void check_cache(const at::Tensor& state, const at::Tensor& x, int64_t dstate) {
  need(state.dim() == 3 && state.size(1) == x.size(-1) && state.size(2) == dstate, "ssm_state must be (n_slots, dim, dstate)");
  need(state.device() == x.device(), "all operands must be on x's device");
  need(state.is_contiguous(), "ssm_state must be contiguous (it is updated in place)");
  if (dtype_code(state) < 0)
    raise(PyExc_TypeError, std::string("ssm_state must be float32, float16 or bfloat16, got ") + name(state));
}

// Parameters are passed as they are, contiguous; in a float type that the kernels do not read
// (float64) as fp32.
at::Tensor vector(const at::Tensor& t) { return (dtype_code(t) < 0 ? t.to(at::kFloat) : t).contiguous(); }
Opt vector(const Opt& t) { return t.has_value() ? Opt(vector(*t)) : t; }
at::Tensor rows(const at::Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }
Opt rows(const Opt& t) { return t.has_value() ? Opt(rows(*t)) : t; }
void need_integer(const at::Tensor& t, const char* what) {
  if (t.is_floating_point() || t.is_complex()) raise(PyExc_TypeError, std::string(what) + " must be integer, got " + name(t));
}
at::Tensor int32s(const at::Tensor& t, const at::Tensor& x) {
  return (t.scalar_type() == at::kInt && t.device() == x.device() ? t : t.to(x.device(), at::kInt)).contiguous();
}

// The kernels write a state through its address: autograd learns of it by the version, and then refuses a
// backward over a graph that saved the values before. Tensors made under inference mode have no version.
void written_in_place(const at::Tensor& state) {
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
}

at::Tensor floats(const at::Tensor& like, int64_t bytes) { return empty({std::max<int64_t>(1, bytes / 4)}, at::kFloat, like); }

// h after the last token of an input without tokens.
at::Tensor states_of_nothing(const at::Tensor& x, const at::Tensor& A, const Opt& init) {
  if (init.has_value()) return init->to(at::kFloat, false, true);
  return at::zeros({x.size(0), x.size(2), A.size(1)}, x.options().dtype(at::kFloat));
}

// (rc, out, final_states or None, kept states or None)
std::tuple<int, at::Tensor, Opt, Opt> ssm_fwd(const at::Tensor& x, const at::Tensor& dt, const at::Tensor& A,
                                              const at::Tensor& B, const at::Tensor& C, const Opt& D, const Opt& z,
                                              const Opt& dt_bias, bool softplus, const Opt& seq_idx, const Opt& init,
                                              bool return_final, bool keep, const Opt& packed_state,
                                              const Opt& packed_slots) {
  const c10::cuda::CUDAGuard guard(x.device());
  at::Tensor out = empty(x.sizes(), x.scalar_type(), x);
  Opt final, kept;
  if (x.numel() == 0) {
    if (return_final) final = states_of_nothing(x, A, init);
    return {CC1D_OK, out, final, kept};
  }
  const cc1d_ssm_problem q = problem(x, dt, A, B, C, D, z, dt_bias, softplus, seq_idx, init);
  if (return_final) final = empty({q.batch, q.dim, q.dstate}, at::kFloat, x);
  if (keep) {
    const int64_t bytes = cc1d_ssm_kept_bytes(q.batch, q.seqlen, q.dim, q.dstate);
    if (bytes < 0) return {q.dstate > 64 ? CC1D_ERR_UNSUPPORTED : CC1D_ERR_INVALID, out, final, kept};
    kept = floats(x, bytes);
  }
  const int64_t ws = cc1d_ssm_workspace_bytes(q.batch, q.seqlen, q.dim, q.dstate, q.groups, q.x_dtype, 0);
  at::Tensor workspace;
  if (ws > 0) workspace = floats(x, ws);
  const int rc = cc1d_ssm_fwd(&q, out.data_ptr(), final.has_value() ? final->data_ptr<float>() : nullptr,
                              kept.has_value() ? kept->data_ptr<float>() : nullptr,
                              packed_state.has_value() ? packed_state->data_ptr() : nullptr,
                              packed_state.has_value() ? dtype_code(*packed_state) : CC1D_F32,
                              packed_state.has_value() ? packed_state->size(0) : 0, ints(packed_slots),
                              packed_slots.has_value() ? packed_slots->size(-1) : 0,
                              ws > 0 ? workspace.data_ptr() : nullptr, ws, stream_of(x));
  return {rc, out, final, kept};
}

// Absent tensors come in as empty optionals, which the autograd machinery treats as non-tensor
// arguments, so that needs_input_grad counts only the tensors given.
struct SsmFn : public torch::autograd::Function<SsmFn> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x,
                                                const at::Tensor& dt, const at::Tensor& A, const at::Tensor& B,
                                                const at::Tensor& C, const Opt& D, const Opt& z, const Opt& dt_bias,
                                                bool softplus, const Opt& seq_idx, const Opt& init, bool return_final) {
    auto [rc, out, final, kept] =
        ssm_fwd(x, dt, A, B, C, D, z, dt_bias, softplus, seq_idx, init, return_final, true, c10::nullopt, c10::nullopt);
    TORCH_CHECK(rc == CC1D_OK, reason(rc, "ssm_scan forward"));
    auto t = [](const Opt& o) { return o.value_or(at::Tensor()); };
    ctx->save_for_backward({x, dt, A, B, C, t(D), t(z), t(dt_bias), t(seq_idx), t(init), t(kept)});
    ctx->saved_data["softplus"] = softplus;
    ctx->saved_data["init_edge"] = static_cast<int64_t>(5 + D.has_value() + z.has_value() + dt_bias.has_value() +
                                                        seq_idx.has_value());
    if (return_final) return {out, *final};
    return {out};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "ssm_scan: gradients of its gradients are not available (create_graph=True)");
    const auto s = ctx->get_saved_variables();
    const at::Tensor &x = s[0], &dt = s[1], &A = s[2], &B = s[3], &C = s[4];
    auto opt = [](const at::Tensor& t) { return t.defined() ? Opt(t) : c10::nullopt; };
    const Opt D = opt(s[5]), z = opt(s[6]), dt_bias = opt(s[7]), seq_idx = opt(s[8]), init = opt(s[9]);
    const bool softplus = ctx->saved_data["softplus"].toBool();
    const bool need_dinit =
        init.has_value() && ctx->needs_input_grad(static_cast<size_t>(ctx->saved_data["init_edge"].toInt()));
    Opt dfinal;
    if (grads.size() > 1 && grads[1].defined()) dfinal = grads[1].contiguous();
    const c10::cuda::CUDAGuard guard(x.device());
    const bool nothing = x.numel() == 0;
    auto make = [&](const at::Tensor& t) { return nothing ? at::zeros(t.sizes(), t.options()) : empty(t.sizes(), t.scalar_type(), t); };
    at::Tensor dx = make(x), ddt = make(dt), dA = make(A), dB = make(B), dC = make(C), dD, dz, dbias, dinit;
    if (D.has_value()) dD = make(*D);
    if (z.has_value()) dz = make(*z);
    if (dt_bias.has_value()) dbias = make(*dt_bias);
    if (need_dinit) dinit = make(*init);
    if (nothing) {
      if (need_dinit && dfinal.has_value()) dinit.copy_(*dfinal);
    } else {
      at::Tensor dout = grads[0].defined() ? grads[0] : at::zeros_like(x, at::MemoryFormat::Contiguous);
      if (dout.stride(2) != 1) dout = dout.contiguous();
      const cc1d_ssm_problem q = problem(x, dt, A, B, C, D, z, dt_bias, softplus, seq_idx, init);
      const cc1d_tokens g = tokens(dout);
      const cc1d_param df = param(dfinal);
      auto p = [](const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
      const cc1d_ssm_grads out{p(dx), p(ddt), p(dz), p(dB), p(dC), p(dA), p(dD), p(dbias), p(dinit)};
      const int64_t ws = cc1d_ssm_workspace_bytes(q.batch, q.seqlen, q.dim, q.dstate, q.groups, q.x_dtype, 1);
      const at::Tensor workspace = floats(x, ws);
      const int rc = cc1d_ssm_bwd(&q, &g, s[10].data_ptr<float>(), &df, &out, workspace.data_ptr(), ws, stream_of(x));
      TORCH_CHECK(rc == CC1D_OK, reason(rc, "ssm_scan backward"));
    }
    return {dx, ddt, dA, dB, dC, dD, dz, dbias, at::Tensor(), at::Tensor(), dinit, at::Tensor()};
  }
};

py::object ssm_scan(const at::Tensor& x0, const at::Tensor& dt0, const at::Tensor& A0, const at::Tensor& B0,
                    const at::Tensor& C0, const Opt& D0, const Opt& z0, const Opt& dt_bias0, bool softplus,
                    const Opt& seq_idx0, const Opt& init0, bool return_final, const Opt& state, const Opt& indices0) {
  refuse_tangents({&x0, &dt0, &A0, &B0, &C0}, {&D0, &z0, &dt_bias0, &init0, &state});
  need(x0.dim() == 3, "x must be (batch, seqlen, dim)");
  check_operands(x0, dt0, A0, B0, C0, D0, z0, dt_bias0, false);
  const int64_t batch = x0.size(0), seqlen = x0.size(1), dim = x0.size(2), dstate = A0.size(1);
  Opt seq_idx, indices;
  if (seq_idx0.has_value()) {
    need(!return_final, "cannot return final states if seq_idx is not None");
    need(seq_idx0->dim() == 2 && seq_idx0->size(0) == batch && seq_idx0->size(1) == seqlen, "seq_idx must be (batch, seqlen)");
    need(seq_idx0->device() == x0.device(), "all operands must be on x's device");
    need_integer(*seq_idx0, "seq_idx");
    seq_idx = int32s(*seq_idx0, x0);
  }
  if (init0.has_value()) {
    need(init0->dim() == 3 && init0->size(0) == batch && init0->size(1) == dim && init0->size(2) == dstate,
         "initial_states must be (batch, dim, dstate)");
    need(init0->device() == x0.device(), "all operands must be on x's device");
    if (!init0->is_floating_point())
      raise(PyExc_TypeError, std::string("initial_states must be floating point, got ") + name(*init0));
  }
  if (state.has_value()) {
    need(seq_idx.has_value() && indices0.has_value(), "ssm_state requires seq_idx and ssm_state_indices");
    check_cache(*state, x0, dstate);
    need(indices0->dim() == 1 ? batch == 1 : indices0->dim() == 2 && indices0->size(0) == batch,
         "ssm_state_indices must be (batch, n_seqs)");
    need_integer(*indices0, "ssm_state_indices");
    indices = int32s(*indices0, x0);
  } else {
    need(!indices0.has_value(), "ssm_state_indices requires ssm_state");
  }
  const at::Tensor x = rows(x0), dt = rows(dt0), A = vector(A0), B = rows(B0), C = rows(C0);
  const Opt D = vector(D0), z = rows(z0), dt_bias = vector(dt_bias0), init = vector(init0);
  bool grad = false;
  if (at::GradMode::is_enabled()) {
    grad = x.requires_grad() || dt.requires_grad() || A.requires_grad() || B.requires_grad() || C.requires_grad();
    for (const Opt* t : {&D, &z, &dt_bias, &init}) grad = grad || (t->has_value() && (*t)->requires_grad());
  }
  if (grad) {
    need(!state.has_value(), "ssm_state is not differentiable: call under torch.no_grad()");
    const auto r = SsmFn::apply(x, dt, A, B, C, D, z, dt_bias, softplus, seq_idx, init, return_final);
    if (return_final) return py::make_tuple(r[0], r[1]);
    return py::cast(r[0]);
  }
  auto [rc, out, final, kept] =
      ssm_fwd(x, dt, A, B, C, D, z, dt_bias, softplus, seq_idx, init, return_final, false, state, indices);
  check(rc, "ssm_scan");
  if (state.has_value()) written_in_place(*state);
  if (return_final) return py::make_tuple(out, *final);
  return py::cast(out);
}

at::Tensor ssm_update(const at::Tensor& x0, const at::Tensor& state, const at::Tensor& dt0, const at::Tensor& A0,
                      const at::Tensor& B0, const at::Tensor& C0, const Opt& D0, const Opt& z0, const Opt& dt_bias0,
                      bool softplus, const Opt& indices0) {
  refuse_tangents({&x0, &state, &dt0, &A0, &B0, &C0}, {&D0, &z0, &dt_bias0});
  need(x0.dim() == 2 || x0.dim() == 3, "x must be (batch, dim) or (batch, seqlen, dim)");
  const bool one = x0.dim() == 2;
  check_operands(x0, dt0, A0, B0, C0, D0, z0, dt_bias0, one);
  check_cache(state, x0, A0.size(1));
  Opt indices;
  if (indices0.has_value()) {
    need(indices0->dim() == 1 && indices0->size(0) == x0.size(0), "ssm_state_indices must be (batch,)");
    need_integer(*indices0, "ssm_state_indices");
    indices = int32s(*indices0, x0);
  } else {
    need(state.size(0) >= x0.size(0), "ssm_state has fewer slots than x has rows");
  }
  const c10::cuda::CUDAGuard guard(x0.device());
  const at::Tensor x = rows(x0), dt = rows(dt0), A = vector(A0), B = rows(B0), C = rows(C0);
  const Opt D = vector(D0), z = rows(z0), dt_bias = vector(dt_bias0);
  at::Tensor out = empty(x.sizes(), x.scalar_type(), x);
  if (x.numel() == 0) return out;
  const cc1d_ssm_problem q = problem(x, dt, A, B, C, D, z, dt_bias, softplus, c10::nullopt, c10::nullopt, one);
  check(cc1d_ssm_update(&q, state.data_ptr(), dtype_code(state), state.size(0), ints(indices), out.data_ptr(), stream_of(x)),
        "ssm_update");
  written_in_place(state);
  return out;
}

// A tensor over `sizes` int32 at `offset` of `storage`.
at::Tensor part(const at::Tensor& storage, at::IntArrayRef sizes, int64_t offset) {
  at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(storage.storage()), storage.key_set(), storage.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(offset);
  t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
  return t;
}

py::tuple slot_maps(const at::Tensor& lengths0, int64_t seqlen, int64_t width, const Opt& slots0, const Opt& free0,
                    const Opt& past0) {
  need(lengths0.dim() == 1, "lengths must be (n,)");
  need(width >= 1 && seqlen >= 0, "width must be at least 1 and seqlen at least 0");
  need(slots0.has_value() || !free0.has_value(), "free_slots requires slots");
  const int64_t n = lengths0.size(0);
  auto integer = [&](const at::Tensor& t, const char* what) {
    need_integer(t, what);
    if (t.dim() != 1) raise(PyExc_AssertionError, std::string(what) + " must be 1-D");
    if (t.device() != lengths0.device()) raise(PyExc_AssertionError, std::string(what) + " must be on the device of lengths");
  };
  integer(lengths0, "lengths");
  if (slots0.has_value()) integer(*slots0, "slots"), need(slots0->size(0) == n, "slots must be (n,)");
  if (past0.has_value()) integer(*past0, "past_lengths"), need(past0->size(0) == n, "past_lengths must be (n,)");
  if (free0.has_value()) integer(*free0, "free_slots");
  need(lengths0.is_cuda(), "lengths must be on a CUDA device");
  const c10::cuda::CUDAGuard guard(lengths0.device());
  auto conv = [&](const Opt& t) { return t.has_value() ? Opt(int32s(*t, lengths0)) : t; };
  const at::Tensor lengths = int32s(lengths0, lengths0);
  const Opt slots = conv(slots0), free_slots = conv(free0), past = conv(past0);

  // One allocation for all maps; the two that are written in 16-byte pieces come first, each at a multiple.
  const int64_t row = (seqlen + 3) / 4 * 4, tail = n * (width - 1);
  at::Tensor all = empty({2 * row + (n + 1) + tail + n + 1}, at::kInt, lengths);
  int32_t* base = all.data_ptr<int32_t>();
  const int64_t o_cu = 2 * row, o_tail = o_cu + n + 1, o_slots = o_tail + tail, o_taken = o_slots + n;
  const int rc = cc1d_slot_maps(lengths.data_ptr<int32_t>(), n, seqlen, width, ints(past), ints(slots), ints(free_slots),
                                free_slots.has_value() ? free_slots->size(0) : 0, base + o_cu, base, base + row,
                                base + o_tail, slots.has_value() ? base + o_slots : nullptr, base + o_taken,
                                stream_of(lengths));
  check(rc, "slot_maps_from_lengths");
  py::object slots_out = py::none();
  if (slots.has_value()) slots_out = py::cast(part(all, {n}, o_slots));
  return py::make_tuple(part(all, {n + 1}, o_cu), part(all, {1, seqlen}, 0), part(all, {1, seqlen}, row),
                        part(all, {n, width - 1}, o_tail), slots_out, part(all, {1}, o_taken));
}

}  // namespace

void bind_ssm(pybind11::module_& m) {
  m.def("set_error_class", [](py::object cls) { g_error = cls.release().ptr(); }, "class of the errors of failing library calls");
  m.def("ssm_scan", &ssm_scan,
        "out or (out, final_states) = ssm_scan(x, dt, A, B, C, D, z, dt_bias, dt_softplus, seq_idx, initial_states, "
        "return_final_states, ssm_state, ssm_state_indices)");
  m.def("ssm_update", &ssm_update,
        "out = ssm_update(x, ssm_state, dt, A, B, C, D, z, dt_bias, dt_softplus, ssm_state_indices)");
  m.def("slot_maps", &slot_maps,
        "(cu_seqlens, seq_idx, positions, tail_rows, slots, n_taken) = slot_maps(lengths, seqlen, width, slots, "
        "free_slots, past_lengths)");
}
