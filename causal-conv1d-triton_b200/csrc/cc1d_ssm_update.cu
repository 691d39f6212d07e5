// Single-token form of the state-space recurrence: L new tokens per batch row (usually one) against
// a kept state (slots, dim, dstate) that is updated in place,
//   h = exp(delta A) h + delta x B,   out = (sum_n C h + D x) silu(z).
//
// One lane holds 4 states of one channel, so that the state moves in 16-byte (fp32) or 8-byte pieces
// with neighbouring lanes on neighbouring pieces, once in and once out; it is all but a few percent
// of the bytes, and what bounds a batch. A lane takes kRows batch rows of its channel: their loads are
// in flight together, A is read once, and the element-wise work (step size, gate) is shared out, each
// of four lanes doing one row for all the channel's lanes. The sums over states go across lanes with
// lane_sums, which leaves each row's on the lane that finishes it. Step, decay and state update are
// the forward's operations in the forward's order, so that decoding continues a prompt with the
// forward's bits.
#include "cc1d_ssm_device.cuh"

namespace cc1d {
namespace {

constexpr int kRows = 4;

template <typename T, typename ST, int NL>
__global__ void __launch_bounds__(256, 3) cc1d_ssm_update_kernel(const __grid_constant__ SsmUpdateParams p) {
  const int nl = threadIdx.x % NL, n0 = 4 * nl;
  const int ch = static_cast<int>(blockIdx.x % p.blocks) * (256 / NL) + static_cast<int>(threadIdx.x) / NL;
  const int b0 = static_cast<int>(blockIdx.x / p.blocks) * kRows;
  const bool in = ch < p.dim;
  const int g = in ? ch / p.group_dim : 0;
  const int nn = in ? p.dstate - n0 : 0;  // states of this lane
  const bool whole = p.state_vec && nn >= 4;

  // Slots of the rows; a negative one (or one past the end) marks a padded entry: nothing of it is
  // read or written.
  int64_t at[kRows];
  bool live[kRows];
  float2 h[kRows][2];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int b = b0 + r;
    const int64_t slot = b >= p.batch ? -1 : (p.indices != nullptr ? p.indices[b] : b);
    live[r] = in && slot >= 0 && slot < p.slots;
    at[r] = (slot * p.dim + ch) * p.dstate + n0;
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const ST* st = static_cast<const ST*>(p.state) + at[r];
    h[r][0] = h[r][1] = make_float2(0.f, 0.f);
    if (live[r]) {
      if (whole) {
        load_vec<ST, 4>(st, h[r]);
      } else {
        if (nn > 0) h[r][0].x = to_f<ST>(st[0]);
        if (nn > 1) h[r][0].y = to_f<ST>(st[1]);
        if (nn > 2) h[r][1].x = to_f<ST>(st[2]);
        if (nn > 3) h[r][1].y = to_f<ST>(st[3]);
      }
    }
  }
  float a[4];
#pragma unroll
  for (int m = 0; m < 4; ++m)
    a[m] = m < nn ? ld_any(p.A.ptr, static_cast<int64_t>(ch) * p.dstate + n0 + m, p.A.dtype) * kLog2e : 0.0f;
  const float2 A2[2] = {make_float2(a[0], a[1]), make_float2(a[2], a[3])};
  const float skip = in && p.D.ptr != nullptr ? ld_any(p.D.ptr, ch, p.D.dtype) : 0.0f;
  const float bias = in && p.dt_bias.ptr != nullptr ? ld_any(p.dt_bias.ptr, ch, p.dt_bias.dtype) : 0.0f;

  // The row whose element-wise work this lane does: the one that lane_sums leaves it.
  const int own = lane_share<kRows, NL, 1>(), ob = b0 + own;
  bool own_live = false;
#pragma unroll
  for (int r = 0; r < kRows; ++r) own_live = r == own ? live[r] : own_live;
  const int lead = threadIdx.x & 31 & ~(NL - 1);  // the channel's first lane
  const T* bp = static_cast<const T*>(p.Bm.ptr) + g * p.Bm.sg;
  const T* cp = static_cast<const T*>(p.Cm.ptr) + g * p.Cm.sg;

  for (int64_t l = 0; l < p.seqlen; ++l) {
    float x = 0.0f, delta = 0.0f, z = 0.0f;
    if (own_live) {
      x = to_f<T>(static_cast<const T*>(p.x.ptr)[ob * p.x.sb + l * p.x.st + ch]);
      delta = to_f<T>(static_cast<const T*>(p.dt.ptr)[ob * p.dt.sb + l * p.dt.st + ch]) + bias;
      if (p.z.ptr != nullptr) z = to_f<T>(static_cast<const T*>(p.z.ptr)[ob * p.z.sb + l * p.z.st + ch]);
    }
    Raw4<T> rB[kRows], rC[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      rB[r] = rC[r] = zero4<T>();
      if (live[r] && nn > 0) {
        rB[r] = load4(bp + (b0 + r) * p.Bm.sb + l * p.Bm.st, n0, p.dstate, p.Bm.vec);
        rC[r] = load4(cp + (b0 + r) * p.Cm.sb + l * p.Cm.st, n0, p.dstate, p.Cm.vec);
      }
    }
    if (p.softplus) delta = softplus(delta);
    const float u = delta * x;
    float y[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      // The lane with share r: bits 0 and 1 of its place hold the halves in that order.
      const int from = lead + ((r >> 1) | ((r & 1) << 1));
      const float2 d = splat(__shfl_sync(0xffffffffu, delta, from)), v = splat(__shfl_sync(0xffffffffu, u, from));
      const float4 B = unpack4(rB[r]), C = unpack4(rC[r]);
      const float2 a0 = exp2_approx2(fmul2(d, A2[0])), a1 = exp2_approx2(fmul2(d, A2[1]));
      h[r][0] = ffma2(a0, h[r][0], fmul2(v, make_float2(B.x, B.y)));
      h[r][1] = ffma2(a1, h[r][1], fmul2(v, make_float2(B.z, B.w)));
      const float2 s = ffma2(h[r][1], make_float2(C.z, C.w), fmul2(h[r][0], make_float2(C.x, C.y)));
      y[r] = s.x + s.y;
    }
    lane_sums<kRows, NL, 1>(y);
    if (own_live && nl < 4) {
      float o = fmaf(skip, x, y[0]);
      if (p.z.ptr != nullptr) o *= z * sigmoid(z);
      static_cast<T*>(p.out)[(static_cast<int64_t>(ob) * p.seqlen + l) * p.dim + ch] = from_f<T>(o);
    }
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    ST* st = static_cast<ST*>(p.state) + at[r];
    if (live[r]) {
      if (whole) {
        store_vec<ST, 4>(st, h[r]);
      } else {
        if (nn > 0) st[0] = from_f<ST>(h[r][0].x);
        if (nn > 1) st[1] = from_f<ST>(h[r][0].y);
        if (nn > 2) st[2] = from_f<ST>(h[r][1].x);
        if (nn > 3) st[3] = from_f<ST>(h[r][1].y);
      }
    }
  }
}

template <typename T, typename ST>
cudaError_t launch(SsmUpdateParams p, cudaStream_t s) {
  const int nl = ssm_lanes(p.dstate);
  p.blocks = static_cast<int>((static_cast<int64_t>(p.dim) * nl + 255) / 256);
  p.state_vec = p.dstate % 4 == 0 && reinterpret_cast<uintptr_t>(p.state) % (4 * sizeof(ST)) == 0;
  const unsigned grid = static_cast<unsigned>(p.blocks) * ((p.batch + kRows - 1) / kRows);
  if (nl == 4)
    cc1d_ssm_update_kernel<T, ST, 4><<<grid, 256, 0, s>>>(p);
  else if (nl == 8)
    cc1d_ssm_update_kernel<T, ST, 8><<<grid, 256, 0, s>>>(p);
  else
    cc1d_ssm_update_kernel<T, ST, 16><<<grid, 256, 0, s>>>(p);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch(const SsmUpdateParams& p, cudaStream_t s) {
  if (p.state_dtype == kBF16) return launch<T, __nv_bfloat16>(p, s);
  if (p.state_dtype == kF16) return launch<T, __half>(p, s);
  return launch<T, float>(p, s);
}

}  // namespace

cudaError_t launch_ssm_update(const SsmUpdateParams& p, cudaStream_t s) {
  if (p.x_dtype == kBF16) return launch<__nv_bfloat16>(p, s);
  if (p.x_dtype == kF16) return launch<__half>(p, s);
  return launch<float>(p, s);
}

}  // namespace cc1d
