// Torch-side launchers of the state-space operators and the slot maps (part of the _cc1d_torch
// module): outputs and workspaces from torch's caching allocator, the device guard, torch's current
// stream, then the C ABI of include/causal_conv1d_b200.h. Arguments arrive checked by the package's
// Python layer (ssm.py). Each launcher returns the C ABI's result code first, or throws inside the
// autograd Function, where the code cannot be handed back.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <tuple>
#include <vector>

#include "causal_conv1d_b200.h"

namespace {

using Opt = c10::optional<at::Tensor>;

int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return CC1D_F32;
    case at::kHalf: return CC1D_F16;
    case at::kBFloat16: return CC1D_BF16;
    default: return -1;
  }
}

void* stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
const int32_t* ints(const Opt& t) { return t.has_value() ? t->data_ptr<int32_t>() : nullptr; }

cc1d_tokens tokens(const at::Tensor& t) {  // (batch, seqlen, channels) or (batch, seqlen, groups, dstate)
  return {t.data_ptr(), t.stride(0), t.stride(1), t.dim() == 4 ? t.stride(2) : 0};
}
cc1d_param param(const Opt& t) {
  if (!t.has_value()) return {nullptr, CC1D_F32};
  return {t->data_ptr(), dtype_code(*t)};
}

cc1d_ssm_problem problem(const at::Tensor& x, const at::Tensor& dt, const at::Tensor& A, const at::Tensor& B,
                         const at::Tensor& C, const Opt& D, const Opt& z, const Opt& dt_bias, bool softplus,
                         const Opt& seq_idx, const Opt& init) {
  cc1d_ssm_problem q{};
  q.x = tokens(x), q.dt = tokens(dt), q.B = tokens(B), q.C = tokens(C);
  if (z.has_value()) q.z = tokens(*z);
  q.A = param(A), q.D = param(D), q.dt_bias = param(dt_bias), q.initial_states = param(init);
  q.seq_idx = ints(seq_idx);
  q.batch = x.size(0), q.seqlen = x.size(1), q.dim = x.size(2), q.dstate = A.size(1);
  q.groups = B.dim() == 4 ? B.size(2) : 1;
  q.x_dtype = dtype_code(x), q.dt_softplus = softplus ? 1 : 0;
  return q;
}

at::Tensor floats(const at::Tensor& like, int64_t bytes) {
  return at::empty({std::max<int64_t>(1, bytes / 4)}, like.options().dtype(at::kFloat));
}

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
  at::Tensor out = at::empty(x.sizes(), x.options());
  Opt final, kept;
  if (x.numel() == 0) {
    if (return_final) final = states_of_nothing(x, A, init);
    return {CC1D_OK, out, final, kept};
  }
  const cc1d_ssm_problem q = problem(x, dt, A, B, C, D, z, dt_bias, softplus, seq_idx, init);
  if (return_final) final = at::empty({q.batch, q.dim, q.dstate}, x.options().dtype(at::kFloat));
  if (keep) {
    const int64_t bytes = cc1d_ssm_kept_bytes(q.batch, q.seqlen, q.dim, q.dstate);
    if (bytes < 0) return {q.dstate > 64 ? CC1D_ERR_UNSUPPORTED : CC1D_ERR_INVALID, out, final, kept};
    kept = floats(x, bytes);
  }
  const int64_t ws = cc1d_ssm_workspace_bytes(q.batch, q.seqlen, q.dim, q.dstate, q.groups, 0);
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

void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == CC1D_OK, what, ": ", cc1d_error_string(rc), rc == CC1D_ERR_CUDA ? " (cudaError " : "",
              rc == CC1D_ERR_CUDA ? std::to_string(cc1d_last_cuda_error()) + ")" : std::string());
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
    check_rc(rc, "ssm_scan forward");
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
    auto like = [](const at::Tensor& t) { return at::empty(t.sizes(), t.options()); };
    const bool nothing = x.numel() == 0;
    auto make = [&](const at::Tensor& t) { return nothing ? at::zeros(t.sizes(), t.options()) : like(t); };
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
      const int64_t ws = cc1d_ssm_workspace_bytes(q.batch, q.seqlen, q.dim, q.dstate, q.groups, 1);
      const at::Tensor workspace = floats(x, ws);
      check_rc(cc1d_ssm_bwd(&q, &g, s[10].data_ptr<float>(), &df, &out, workspace.data_ptr(), ws, stream_of(x)),
               "ssm_scan backward");
    }
    return {dx, ddt, dA, dB, dC, dD, dz, dbias, at::Tensor(), at::Tensor(), dinit, at::Tensor()};
  }
};

torch::autograd::variable_list ssm_fn(const at::Tensor& x, const at::Tensor& dt, const at::Tensor& A,
                                      const at::Tensor& B, const at::Tensor& C, const Opt& D, const Opt& z,
                                      const Opt& dt_bias, bool softplus, const Opt& seq_idx, const Opt& init,
                                      bool return_final) {
  return SsmFn::apply(x, dt, A, B, C, D, z, dt_bias, softplus, seq_idx, init, return_final);
}

// (rc, out); x, dt, z (batch, seqlen, dim), B and C (batch, seqlen, [groups,] dstate)
std::tuple<int, at::Tensor> ssm_update(const at::Tensor& x, const at::Tensor& state, const at::Tensor& dt,
                                       const at::Tensor& A, const at::Tensor& B, const at::Tensor& C, const Opt& D,
                                       const Opt& z, const Opt& dt_bias, bool softplus, const Opt& indices) {
  const c10::cuda::CUDAGuard guard(x.device());
  at::Tensor out = at::empty(x.sizes(), x.options());
  if (x.numel() == 0) return {CC1D_OK, out};
  const cc1d_ssm_problem q = problem(x, dt, A, B, C, D, z, dt_bias, softplus, c10::nullopt, c10::nullopt);
  const int rc = cc1d_ssm_update(&q, state.data_ptr(), dtype_code(state), state.size(0), ints(indices), out.data_ptr(),
                                 stream_of(x));
  return {rc, out};
}

// (rc, cu_seqlens, seq_idx, positions, tail_rows, slots or None, n_taken)
std::tuple<int, at::Tensor, at::Tensor, at::Tensor, at::Tensor, Opt, at::Tensor> slot_maps(
    const at::Tensor& lengths, int64_t seqlen, int64_t width, const Opt& past, const Opt& slots, const Opt& free_slots) {
  const c10::cuda::CUDAGuard guard(lengths.device());
  const int64_t n = lengths.size(0);
  const auto o = lengths.options();
  at::Tensor cu = at::empty({n + 1}, o), seq = at::empty({1, seqlen}, o), pos = at::empty({1, seqlen}, o);
  at::Tensor tail = at::empty({n, width - 1}, o), taken = at::empty({1}, o);
  Opt slots_out;
  if (slots.has_value()) slots_out = at::empty({n}, o);
  const int rc = cc1d_slot_maps(
      lengths.data_ptr<int32_t>(), n, seqlen, width, ints(past), ints(slots), ints(free_slots),
      free_slots.has_value() ? free_slots->size(0) : 0, cu.data_ptr<int32_t>(), seq.data_ptr<int32_t>(),
      pos.data_ptr<int32_t>(), tail.data_ptr<int32_t>(), slots_out.has_value() ? slots_out->data_ptr<int32_t>() : nullptr,
      taken.data_ptr<int32_t>(), stream_of(lengths));
  return {rc, cu, seq, pos, tail, slots_out, taken};
}

}  // namespace

void bind_ssm(pybind11::module_& m) {
  m.def("ssm_fwd", &ssm_fwd,
        "(rc, out, final_states, kept) = ssm_fwd(x, dt, A, B, C, D, z, dt_bias, softplus, seq_idx, initial_states, "
        "return_final, keep, packed_state, packed_slots)");
  m.def("ssm_fn", &ssm_fn,
        "[out] or [out, final_states] = ssm_fn(x, dt, A, B, C, D, z, dt_bias, softplus, seq_idx, initial_states, "
        "return_final): forward with autograd");
  m.def("ssm_update", &ssm_update,
        "(rc, out) = ssm_update(x, state, dt, A, B, C, D, z, dt_bias, softplus, indices)");
  m.def("slot_maps", &slot_maps,
        "(rc, cu_seqlens, seq_idx, positions, tail_rows, slots, n_taken) = slot_maps(lengths, seqlen, width, "
        "past_lengths, slots, free_slots)");
}
