// C entry points of the state-space operators and the slot maps: argument checks, the layout that the
// kernels find, how a sequence is cut in pieces, and the workspaces. Declared in
// include/causal_conv1d_b200.h.
#include <algorithm>
#include <initializer_list>

#include "causal_conv1d_b200.h"
#include "cc1d_device.cuh"
#include "cc1d_slot_maps.h"
#include "cc1d_ssm.h"

namespace cc1d {

int device_sms(int* sms);  // cc1d_api.cu

namespace {

constexpr int64_t kMaxInt = (int64_t(1) << 31) - 64;

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
int elem_size(int dtype) { return dtype == kF32 ? 4 : 2; }
bool valid_dtype(int dtype) { return dtype == kF32 || dtype == kF16 || dtype == kBF16; }
bool valid_param(const cc1d_param& q) { return q.ptr == nullptr || valid_dtype(q.dtype); }

// Up to this many pieces each piece works out what it receives from the ones before it, which spares a
// launch; the work grows with the square of their number, so above it the join kernel does it once
// (a prompt of 512 tokens and channels in 16 pieces: 22.5 us with the join kernel, 18.4 without).
constexpr int kFoldSegs = 16;

// How one direction runs: CTAs that cover a group's channels, pieces of the sequence and their length.
struct Plan {
  int nl, blocks, segs, seg_len;
};

// A sequence is cut in pieces when the rows and channels alone leave SMs idle; a pass over the pieces
// then has to find what each receives before the pass proper. The cheapest number of pieces is taken, in
// units of a token of one CTA alone on its SM. Measured at 64 channels of 16 states a CTA and 2048 tokens:
// a forward takes 150 us with one CTA on every SM and 239 with two (`full`), a backward 434 and 711; the
// pass over the pieces takes 0.75 and 0.28 of the pass it prepares (`pass`); its launch and the pieces'
// start 7 us (`launches`), and filling and draining a CTA's tiles 1 us (`fill`). Shared memory holds two
// CTAs an SM except in the backward of 32-bit operands or of more than 32 states.
Plan make_plan(int64_t batch, int64_t seqlen, int64_t dim, int64_t dstate, int64_t groups, int x_dtype, bool backward,
               int sms) {
  const double pass = backward ? 0.28 : 0.75, launches = backward ? 35 : 100, fill = backward ? 4 : 15;
  const double full = backward ? 1.64 : 1.59;
  Plan r;
  r.nl = ssm_lanes(static_cast<int>(dstate));
  r.blocks = static_cast<int>(cdiv(dim / groups, ssm_channels(r.nl)));
  r.segs = 1, r.seg_len = static_cast<int>(std::max<int64_t>(32, cdiv(seqlen, 32) * 32));
  const bool alone = backward && (x_dtype == kF32 || r.nl > 8);
  const int64_t ctas = batch * groups * r.blocks, room = (alone ? 1 : 2) * sms;
  const int64_t most = std::min<int64_t>(cdiv(4 * room, std::max<int64_t>(1, ctas)), cdiv(seqlen, 32));
  double best = -1;
  for (int64_t want = 1; want <= std::max<int64_t>(1, most); ++want) {
    const int64_t len = cdiv(cdiv(seqlen, want), 32) * 32, segs = cdiv(seqlen, len), n = ctas * segs, rest = n % room;
    const double waves = static_cast<double>(n / room) * (alone ? 1 : full) + (rest == 0 ? 0 : rest <= sms ? 1 : full);
    const double cost = (len + fill) * waves * (segs > 1 ? 1 + pass : 1) + (segs > 1 ? launches : 0);
    if (best < 0 || cost < best) best = cost, r.segs = static_cast<int>(segs), r.seg_len = static_cast<int>(len);
  }
  return r;
}

int check_sizes(int64_t batch, int64_t seqlen, int64_t dim, int64_t dstate, int64_t groups) {
  if (batch < 0 || seqlen < 0 || dim < 0 || dstate < 1 || groups < 1) return CC1D_ERR_INVALID;
  if (batch > kMaxInt || seqlen > kMaxInt || dim > kMaxInt || dim % groups != 0) return CC1D_ERR_INVALID;
  return dstate > kSsmMaxState ? CC1D_ERR_UNSUPPORTED : CC1D_OK;
}

int plan_for(int64_t batch, int64_t seqlen, int64_t dim, int64_t dstate, int64_t groups, int x_dtype, bool backward,
             Plan* plan) {
  int sms = 0;
  const int rc = device_sms(&sms);
  if (rc != CC1D_OK) return rc;
  // The last few plans of the thread: a layer asks for the same ones again, twice a call.
  struct Known {
    int64_t key[6];
    Plan plan;
  };
  thread_local Known known[8] = {};
  thread_local unsigned next = 0;
  const int64_t key[6] = {batch, seqlen, dim, dstate, (groups * 4 + x_dtype) * 2 + (backward ? 1 : 0), sms};
  bool found = false;
  for (const Known& k : known)
    if (k.plan.segs > 0 && std::equal(key, key + 6, k.key)) *plan = k.plan, found = true;
  if (!found) {
    *plan = make_plan(batch, seqlen, dim, dstate, groups, x_dtype, backward, sms);
    Known& k = known[next++ % 8];
    std::copy(key, key + 6, k.key), k.plan = *plan;
  }
  if (batch * plan->segs * groups * plan->blocks > kMaxInt) return CC1D_ERR_INVALID;
  return CC1D_OK;
}

int64_t pieces_floats(const Plan& plan, int64_t batch, int64_t dim) {
  return plan.segs > 1 ? 3 * batch * plan.segs * dim * 4 * plan.nl : 0;
}

int64_t bwd_floats(const Plan& plan, int64_t batch, int64_t seqlen, int64_t dim, int64_t groups) {
  const int64_t np = 4 * plan.nl, bs = batch * plan.segs;
  return pieces_floats(plan, batch, dim) + batch * seqlen * groups * plan.blocks * 2 * np + bs * dim * np + bs * 2 * dim;
}

bool empty(const cc1d_ssm_problem& q) { return q.batch == 0 || q.dim == 0 || q.seqlen == 0; }

// Whether runs of `n` elements starting at multiples of n (of a group) are aligned vectors.
int aligned(const cc1d_tokens& t, int n, int es, int64_t batch) {
  const int64_t bytes = std::min(16, n * es);
  if (reinterpret_cast<uintptr_t>(t.ptr) % bytes != 0 || (t.stride_time * es) % bytes != 0) return 0;
  return batch <= 1 || (t.stride_batch * es) % bytes == 0;
}

SsmTokens tokens(const cc1d_tokens& t, int n, int es, const cc1d_ssm_problem& q) {
  int vec = aligned(t, n, es, q.batch);
  if (q.groups > 1) vec = vec && (n == 8 ? (q.dim / q.groups) % 8 == 0 : (t.stride_group * es) % std::min(16, n * es) == 0);
  return {t.ptr, t.stride_batch, t.stride_time, t.stride_group, vec};
}

// Whether every row of the contiguous outputs, `dim` elements each, starts at a multiple of 16 bytes (a null
// output has no rows).
int aligned_rows(int64_t dim, int es, std::initializer_list<const void*> outs) {
  if (dim * es % 16 != 0) return 0;
  for (const void* o : outs)
    if (reinterpret_cast<uintptr_t>(o) % 16 != 0) return 0;
  return 1;
}

SsmParam param(const cc1d_param& q) { return {q.ptr, q.dtype}; }

int check_problem(const cc1d_ssm_problem* q) {
  if (q == nullptr || !valid_dtype(q->x_dtype)) return CC1D_ERR_INVALID;
  const int rc = check_sizes(q->batch, q->seqlen, q->dim, q->dstate, q->groups);
  if (rc != CC1D_OK) return rc;
  if (!valid_param(q->A) || !valid_param(q->D) || !valid_param(q->dt_bias) || !valid_param(q->initial_states))
    return CC1D_ERR_INVALID;
  if (!empty(*q) && (!q->x.ptr || !q->dt.ptr || !q->B.ptr || !q->C.ptr || !q->A.ptr)) return CC1D_ERR_INVALID;
  return CC1D_OK;
}

SsmParams common(const cc1d_ssm_problem& q, const Plan& plan) {
  const int es = elem_size(q.x_dtype);
  SsmParams p{};
  p.x = tokens(q.x, 8, es, q), p.dt = tokens(q.dt, 8, es, q), p.z = tokens(q.z, 8, es, q);
  p.Bm = tokens(q.B, 4, es, q), p.Cm = tokens(q.C, 4, es, q);
  p.A = param(q.A), p.D = param(q.D), p.dt_bias = param(q.dt_bias), p.init = param(q.initial_states);
  p.seq_idx = q.seq_idx;
  p.batch = static_cast<int>(q.batch), p.seqlen = static_cast<int>(q.seqlen), p.dim = static_cast<int>(q.dim);
  p.dstate = static_cast<int>(q.dstate), p.groups = static_cast<int>(q.groups);
  p.group_dim = static_cast<int>(q.dim / q.groups), p.softplus = q.dt_softplus != 0;
  p.segs = plan.segs, p.seg_len = plan.seg_len, p.blocks = plan.blocks;
  return p;
}

void set_pieces(SsmParams& p, float* ws, int64_t floats) {
  p.fold = p.segs <= kFoldSegs;
  p.seg_out = ws, p.seg_decay = ws + floats / 3, p.seg_in = ws + 2 * (floats / 3);
}

// The buffers that the kernels read and write in vectors whatever the operands' alignment.
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int done(cudaError_t e) { return e == cudaSuccess ? CC1D_OK : record_cuda_error(e); }

#define CC1D_TRY(call)              \
  do {                              \
    const int r_ = (call);          \
    if (r_ != CC1D_OK) return r_;   \
  } while (0)

}  // namespace
}  // namespace cc1d

using namespace cc1d;

extern "C" {

int64_t cc1d_ssm_kept_bytes(int64_t batch, int64_t seqlen, int64_t dim, int64_t dstate) {
  if (check_sizes(batch, seqlen, dim, dstate, 1) != CC1D_OK) return -1;
  return batch * cdiv(seqlen, kSsmTile) * dim * 4 * ssm_lanes(static_cast<int>(dstate)) * 4;
}

int64_t cc1d_ssm_workspace_bytes(int64_t batch, int64_t seqlen, int64_t dim, int64_t dstate, int64_t groups,
                                 int x_dtype, int backward) {
  if (check_sizes(batch, seqlen, dim, dstate, groups) != CC1D_OK || !valid_dtype(x_dtype)) return -1;
  if (batch == 0 || dim == 0 || seqlen == 0) return 0;
  Plan plan;
  if (plan_for(batch, seqlen, dim, dstate, groups, x_dtype, backward != 0, &plan) != CC1D_OK) return -1;
  return 4 * (backward ? bwd_floats(plan, batch, seqlen, dim, groups) : pieces_floats(plan, batch, dim));
}

int cc1d_ssm_fwd(const cc1d_ssm_problem* q, void* out, float* final_states, float* kept_states, void* packed_state,
                 int packed_state_dtype, int64_t n_slots, const int32_t* packed_slots, int64_t packed_slots_n,
                 void* workspace, int64_t workspace_bytes, void* stream) {
  CC1D_TRY(check_problem(q));
  if (packed_state && (!q->seq_idx || !packed_slots || packed_slots_n < 0 || !valid_dtype(packed_state_dtype)))
    return CC1D_ERR_INVALID;
  if (empty(*q)) return CC1D_OK;
  if (!out || !aligned16(kept_states) || !aligned16(workspace)) return CC1D_ERR_INVALID;
  Plan plan;
  CC1D_TRY(plan_for(q->batch, q->seqlen, q->dim, q->dstate, q->groups, q->x_dtype, false, &plan));
  const int64_t need = pieces_floats(plan, q->batch, q->dim);
  if (need > 0 && (!workspace || workspace_bytes < 4 * need)) return CC1D_ERR_WORKSPACE;
  SsmParams p = common(*q, plan);
  p.out_vec = aligned_rows(q->dim, elem_size(q->x_dtype), {out});
  p.out = out, p.final_states = final_states, p.kept = kept_states;
  p.cache = packed_state, p.cache_dtype = packed_state_dtype, p.cache_idx = packed_slots, p.cache_n = packed_slots_n;
  p.cache_slots = n_slots;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (plan.segs > 1) {
    set_pieces(p, static_cast<float*>(workspace), need);
    CC1D_TRY(done(launch_ssm_scan(p, kSsmPieceForward, q->x_dtype, s)));
    if (!p.fold) CC1D_TRY(done(launch_ssm_join(p, false, s)));
  }
  return done(launch_ssm_scan(p, kSsmForward, q->x_dtype, s));
}

int cc1d_ssm_bwd(const cc1d_ssm_problem* q, const cc1d_tokens* dout, const float* kept_states,
                 const cc1d_param* dfinal_states, const cc1d_ssm_grads* grads, void* workspace, int64_t workspace_bytes,
                 void* stream) {
  CC1D_TRY(check_problem(q));
  if (!dout || !grads || (dfinal_states && !valid_param(*dfinal_states))) return CC1D_ERR_INVALID;
  if (empty(*q)) return CC1D_OK;
  if (!dout->ptr || !kept_states || !grads->dx || !grads->ddt || !grads->dA || !grads->dB || !grads->dC ||
      (q->z.ptr && !grads->dz) || (q->D.ptr && !grads->dD) || (q->dt_bias.ptr && !grads->ddt_bias) ||
      (grads->dinitial_states && !q->initial_states.ptr) || !aligned16(kept_states) || !aligned16(workspace))
    return CC1D_ERR_INVALID;
  Plan plan;
  CC1D_TRY(plan_for(q->batch, q->seqlen, q->dim, q->dstate, q->groups, q->x_dtype, true, &plan));
  if (!workspace || workspace_bytes < 4 * bwd_floats(plan, q->batch, q->seqlen, q->dim, q->groups))
    return CC1D_ERR_WORKSPACE;
  SsmParams p = common(*q, plan);
  p.dout = tokens(*dout, 8, elem_size(q->x_dtype), *q);
  if (dfinal_states) p.dfinal = param(*dfinal_states);
  p.kept = const_cast<float*>(kept_states);
  p.out_vec = aligned_rows(q->dim, elem_size(q->x_dtype), {grads->dx, grads->ddt, q->z.ptr ? grads->dz : nullptr});
  p.dx = grads->dx, p.ddt = grads->ddt, p.dz = grads->dz, p.dB = grads->dB, p.dC = grads->dC;
  p.dA = grads->dA, p.dD = q->D.ptr ? grads->dD : nullptr, p.ddt_bias = q->dt_bias.ptr ? grads->ddt_bias : nullptr;
  p.dinit = grads->dinitial_states;
  const int64_t np = 4 * plan.nl, bs = q->batch * plan.segs, piece = pieces_floats(plan, q->batch, q->dim);
  float* ws = static_cast<float*>(workspace);
  set_pieces(p, ws, piece);
  p.part_bc = ws + piece;
  p.part_a = p.part_bc + q->batch * q->seqlen * q->groups * plan.blocks * 2 * np;
  p.part_d = p.part_a + bs * q->dim * np;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (plan.segs > 1) {
    CC1D_TRY(done(launch_ssm_scan(p, kSsmPieceBackward, q->x_dtype, s)));
    if (!p.fold) CC1D_TRY(done(launch_ssm_join(p, true, s)));
  }
  return done(launch_ssm_bwd(p, q->x_dtype, s));
}

int cc1d_ssm_update(const cc1d_ssm_problem* q, void* state, int state_dtype, int64_t n_slots,
                    const int32_t* state_indices, void* out, void* stream) {
  CC1D_TRY(check_problem(q));
  if (!valid_dtype(state_dtype) || (!state_indices && n_slots < q->batch)) return CC1D_ERR_INVALID;
  if (empty(*q)) return CC1D_OK;
  if (!state || !out) return CC1D_ERR_INVALID;
  SsmUpdateParams p{};
  const int es = elem_size(q->x_dtype);
  p.x = tokens(q->x, 8, es, *q), p.dt = tokens(q->dt, 8, es, *q), p.z = tokens(q->z, 8, es, *q);
  p.Bm = tokens(q->B, 4, es, *q), p.Cm = tokens(q->C, 4, es, *q);
  p.A = param(q->A), p.D = param(q->D), p.dt_bias = param(q->dt_bias);
  p.state = state, p.slots = n_slots, p.state_dtype = state_dtype, p.x_dtype = q->x_dtype, p.indices = state_indices, p.out = out;
  p.batch = static_cast<int>(q->batch), p.seqlen = static_cast<int>(q->seqlen), p.dim = static_cast<int>(q->dim);
  p.dstate = static_cast<int>(q->dstate), p.group_dim = static_cast<int>(q->dim / q->groups);
  p.softplus = q->dt_softplus != 0;
  CC1D_TRY(device_sms(&p.sms));
  if (cdiv(q->batch * q->dim * ssm_lanes(p.dstate), 256) > kMaxInt) return CC1D_ERR_INVALID;
  return done(launch_ssm_update(p, static_cast<cudaStream_t>(stream)));
}

int cc1d_slot_maps(const int32_t* lengths, int64_t n, int64_t seqlen, int64_t width, const int32_t* past_lengths,
                   const int32_t* slots, const int32_t* free_slots, int64_t n_free, int32_t* cu_seqlens, int32_t* seq_idx,
                   int32_t* positions, int32_t* tail_rows, int32_t* slots_out, int32_t* n_taken, void* stream) {
  if (n < 0 || seqlen < 0 || width < 1 || n_free < 0 || n > kMaxInt || seqlen > kMaxInt || width > kMaxInt)
    return CC1D_ERR_INVALID;
  if ((n > 0 && !lengths) || !cu_seqlens || !n_taken || (seqlen > 0 && (!seq_idx || !positions)) ||
      (n > 0 && width > 1 && !tail_rows) || (n > 0 && slots && !slots_out) || (slots && n_free > 0 && !free_slots))
    return CC1D_ERR_INVALID;
  SlotMapParams p{};
  p.lengths = lengths, p.past = past_lengths, p.slots = slots, p.free_slots = free_slots, p.n_free = n_free;
  p.cu_seqlens = cu_seqlens, p.seq_idx = seq_idx, p.positions = positions, p.tail_rows = tail_rows;
  p.slots_out = slots_out, p.n_taken = n_taken;
  p.n = static_cast<int>(n), p.seqlen = static_cast<int>(seqlen), p.width = static_cast<int>(width);
  p.vec = aligned16(seq_idx) && aligned16(positions);
  return done(launch_slot_maps(p, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
