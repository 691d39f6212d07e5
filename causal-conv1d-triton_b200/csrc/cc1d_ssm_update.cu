// Single-token form of the state-space recurrence: L new tokens per batch row (usually one) against
// a kept state (slots, dim, dstate) that is updated in place,
//   h = exp(delta A) h + delta x B,   out = (sum_n C h + D x) silu(z).
//
// One lane holds 4 states of one channel, so that the state moves in 16-byte (fp32) or 8-byte pieces
// with neighbouring lanes on neighbouring pieces, once in and once out; it is all but a few percent
// of the bytes, and what bounds a batch. The 4 to 16 lanes of a channel add their products with C by
// shuffles. Step, decay and state update are the forward's operations in the forward's order, so
// that decoding continues a prompt with the same bits in the state.
#include "cc1d_ssm_device.cuh"

namespace cc1d {
namespace {

template <typename ST, int NL>
__global__ void __launch_bounds__(256) cc1d_ssm_update_kernel(const __grid_constant__ SsmUpdateParams p) {
  const int64_t idx = blockIdx.x * 256ll + threadIdx.x;
  const int64_t row = idx / NL;  // (b, channel)
  const int n0 = 4 * static_cast<int>(idx % NL);
  const int b = static_cast<int>(row / p.dim), ch = static_cast<int>(row % p.dim);
  const int64_t slot = b >= p.batch ? -1 : (p.indices != nullptr ? p.indices[b] : b);
  const bool live = slot >= 0 && slot < p.slots;  // a negative slot marks a padded batch entry: nothing is read or written
  const int g = ch / p.group_dim;

  ST* st = static_cast<ST*>(p.state) + (slot * p.dim + ch) * p.dstate + n0;
  const bool whole = p.dstate % 4 == 0 && reinterpret_cast<uintptr_t>(p.state) % (4 * sizeof(ST)) == 0;
  const int nn = live ? p.dstate - n0 : 0;  // states of this lane
  float2 h[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)}, A2[2];
  if (whole && nn > 0) {
    load_vec<ST, 4>(st, h);
  } else {
    if (nn > 0) h[0].x = to_f<ST>(st[0]);
    if (nn > 1) h[0].y = to_f<ST>(st[1]);
    if (nn > 2) h[1].x = to_f<ST>(st[2]);
    if (nn > 3) h[1].y = to_f<ST>(st[3]);
  }
  float a[4], skip = 0.0f, bias = 0.0f;
#pragma unroll
  for (int m = 0; m < 4; ++m)
    a[m] = m < nn ? ld_any(p.A.ptr, static_cast<int64_t>(ch) * p.dstate + n0 + m, p.A.dtype) * kLog2e : 0.0f;
  A2[0] = make_float2(a[0], a[1]), A2[1] = make_float2(a[2], a[3]);
  if (live && p.D.ptr != nullptr) skip = ld_any(p.D.ptr, ch, p.D.dtype);
  if (live && p.dt_bias.ptr != nullptr) bias = ld_any(p.dt_bias.ptr, ch, p.dt_bias.dtype);

  for (int64_t l = 0; l < p.seqlen; ++l) {
    float x = 0.0f, delta = 0.0f, B[4], C[4];
    if (live) {
      x = ld_any(p.x.ptr, b * p.x.sb + l * p.x.st + ch, p.x_dtype);
      delta = ld_any(p.dt.ptr, b * p.dt.sb + l * p.dt.st + ch, p.x_dtype) + bias;
      if (p.softplus) delta = softplus(delta);
    }
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      B[m] = m < nn ? ld_any(p.Bm.ptr, b * p.Bm.sb + l * p.Bm.st + g * p.Bm.sg + n0 + m, p.x_dtype) : 0.0f;
      C[m] = m < nn ? ld_any(p.Cm.ptr, b * p.Cm.sb + l * p.Cm.st + g * p.Cm.sg + n0 + m, p.x_dtype) : 0.0f;
    }
    const float u = delta * x;
    const float2 a0 = exp2_approx2(fmul2(splat(delta), A2[0])), a1 = exp2_approx2(fmul2(splat(delta), A2[1]));
    h[0] = ffma2(a0, h[0], fmul2(splat(u), make_float2(B[0], B[1])));
    h[1] = ffma2(a1, h[1], fmul2(splat(u), make_float2(B[2], B[3])));
    const float2 s = ffma2(h[1], make_float2(C[2], C[3]), fmul2(h[0], make_float2(C[0], C[1])));
    float y = s.x + s.y;
#pragma unroll
    for (int o = 1; o < NL; o *= 2) y += __shfl_xor_sync(0xffffffffu, y, o);
    if (live && n0 == 0) {
      y = fmaf(skip, x, y);
      if (p.z.ptr != nullptr) {
        const float z = ld_any(p.z.ptr, b * p.z.sb + l * p.z.st + ch, p.x_dtype);
        y *= z * sigmoid(z);
      }
      st_any(p.out, (static_cast<int64_t>(b) * p.seqlen + l) * p.dim + ch, p.x_dtype, y);
    }
  }
  if (whole && nn > 0) {
    store_vec<ST, 4>(st, h);
  } else {
    if (nn > 0) st[0] = from_f<ST>(h[0].x);
    if (nn > 1) st[1] = from_f<ST>(h[0].y);
    if (nn > 2) st[2] = from_f<ST>(h[1].x);
    if (nn > 3) st[3] = from_f<ST>(h[1].y);
  }
}

template <typename ST>
cudaError_t launch(const SsmUpdateParams& p, cudaStream_t s) {
  const int nl = ssm_lanes(p.dstate);
  const int64_t n = static_cast<int64_t>(p.batch) * p.dim * nl;
  const unsigned grid = static_cast<unsigned>((n + 255) / 256);
  if (nl == 4)
    cc1d_ssm_update_kernel<ST, 4><<<grid, 256, 0, s>>>(p);
  else if (nl == 8)
    cc1d_ssm_update_kernel<ST, 8><<<grid, 256, 0, s>>>(p);
  else
    cc1d_ssm_update_kernel<ST, 16><<<grid, 256, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_ssm_update(const SsmUpdateParams& p, cudaStream_t s) {
  if (p.state_dtype == kBF16) return launch<__nv_bfloat16>(p, s);
  if (p.state_dtype == kF16) return launch<__half>(p, s);
  return launch<float>(p, s);
}

}  // namespace cc1d
