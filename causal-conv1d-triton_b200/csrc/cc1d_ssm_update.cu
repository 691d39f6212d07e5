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
// the forward's operations in the forward's order: against an fp32 state, tokens give the bits of a forward
// over them that runs in one piece. (Between pieces a forward carries states by one decay of the summed
// steps, and a 16-bit state is rounded at every call.)
#include <type_traits>

#include "cc1d_ssm_device.cuh"

namespace cc1d {
namespace {

constexpr int kRows = 4;
constexpr int kStep = 128;  // threads of a CTA of the one-token kernel

// 4 consecutive elements of a buffer whose type is given at run time, the first `n` of them.
__device__ __forceinline__ void ld_any4(const void* base, int64_t i, int dtype, int n, float (&v)[4]) {
#pragma unroll
  for (int m = 0; m < 4; ++m) v[m] = 0.0f;
  if (dtype == kF32) {
#pragma unroll
    for (int m = 0; m < 4; ++m)
      if (m < n) v[m] = static_cast<const float*>(base)[i + m];
  } else {
    for (int m = 0; m < n && m < 4; ++m) v[m] = ld_any(base, i + m, dtype);
  }
}

// One token of every row, dstate 16, 32 or 64, all of it in aligned vectors: what a decode step is. A CTA
// takes G groups of kRows rows of its channels and has all their states on the way at once, as
// asynchronous copies of each thread's own pieces (16 KB a CTA at G = 2, eight CTAs an SM: with 256 threads
// and four, 128 rows of 2048 channels take 9.2 us instead of 8.5). 256 rows of 4352 channels, fp32 states, 151 MB:
// 30.8 us between other calls, 28.5 in a row of such steps (5.3 TB/s, 0.81 of the measured copy
// bandwidth); 33.8 us with three groups, 35.4 with four (80 registers, three quarters of the threads), 41 with the
// loads of a group in registers. Issue slots are 69% taken (124 instructions a warp and row); addresses of one
// 32-bit product and B and C a group ahead are no faster.
template <typename T, typename ST, int NL, int G>
__global__ void __launch_bounds__(kStep, 1024 / kStep) cc1d_ssm_step_kernel(const __grid_constant__ SsmUpdateParams p) {
  constexpr int BYTES = 4 * static_cast<int>(sizeof(ST));
  extern __shared__ __align__(16) unsigned char staged[];  // [G][kRows][kStep] pieces
  const int nl = threadIdx.x % NL, n0 = 4 * nl;
  const int own_ch = static_cast<int>(blockIdx.x % p.blocks) * (kStep / NL) + static_cast<int>(threadIdx.x) / NL;
  const bool in = own_ch < p.dim;
  const int ch = in ? own_ch : p.dim - 1;  // lanes past the last channel compute it again, and write nothing
  const int b0 = static_cast<int>(blockIdx.x / p.blocks) * (G * kRows);
  ST* const state = static_cast<ST*>(p.state) + static_cast<int64_t>(ch) * p.dstate + n0;
  const int64_t slot_size = static_cast<int64_t>(p.dim) * p.dstate;
  const bool has_z = p.z.ptr != nullptr;

  // Slots of the rows; -1 for a padded entry (a negative slot, or one past the end), of which nothing is
  // read or written.
  int slot[G][kRows];
#pragma unroll
  for (int i = 0; i < G * kRows; ++i) {
    const int b = b0 + i;
    int v = b >= p.batch ? -1 : (p.indices != nullptr ? p.indices[b] : b);
    if (v >= p.slots) v = -1;
    slot[i / kRows][i % kRows] = v;
  }
#pragma unroll
  for (int q = 0; q < G; ++q) {
#pragma unroll
    for (int r = 0; r < kRows; ++r)
      if (slot[q][r] >= 0)
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(staged) + ((q * kRows + r) * kStep + threadIdx.x) * BYTES),
                     "l"(state + slot[q][r] * slot_size), "n"(BYTES)
                     : "memory");
    copies_issued();
  }

  // The row of four whose element-wise work this lane does: the one that lane_sums leaves it.
  const int own = lane_share<kRows, NL, 1>();
  const int lead = threadIdx.x & 31 & ~(NL - 1);  // the channel's first lane
  T x[G], dt[G], z[G];
#pragma unroll
  for (int q = 0; q < G; ++q) {
    const int64_t b = min(b0 + q * kRows + own, p.batch - 1);
    x[q] = static_cast<const T*>(p.x.ptr)[b * p.x.sb + ch];
    dt[q] = static_cast<const T*>(p.dt.ptr)[b * p.dt.sb + ch];
    z[q] = has_z ? static_cast<const T*>(p.z.ptr)[b * p.z.sb + ch] : from_f<T>(0.0f);
  }
  float a[4];
  ld_any4(p.A.ptr, static_cast<int64_t>(ch) * p.dstate + n0, p.A.dtype, 4, a);
  const float2 A2[2] = {make_float2(a[0] * kLog2e, a[1] * kLog2e), make_float2(a[2] * kLog2e, a[3] * kLog2e)};
  const float skip = p.D.ptr != nullptr ? ld_any(p.D.ptr, ch, p.D.dtype) : 0.0f;
  const float bias = p.dt_bias.ptr != nullptr ? ld_any(p.dt_bias.ptr, ch, p.dt_bias.dtype) : 0.0f;
  const int64_t g = ch / p.group_dim;
  const T* bp = static_cast<const T*>(p.Bm.ptr) + b0 * p.Bm.sb + g * p.Bm.sg + n0;
  const T* cp = static_cast<const T*>(p.Cm.ptr) + b0 * p.Cm.sb + g * p.Cm.sg + n0;
  T* op = static_cast<T*>(p.out) + static_cast<int64_t>(b0 + own) * p.dim + ch;

  auto group = [&](auto q_) {
    constexpr int q = decltype(q_)::value;
    Raw4<T> B[kRows], C[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r, bp += p.Bm.sb, cp += p.Cm.sb) {
      const bool there = b0 + q * kRows + r < p.batch;
      B[r] = there ? load4(bp, 0, 4, true) : zero4<T>();
      C[r] = there ? load4(cp, 0, 4, true) : zero4<T>();
    }
    float delta = to_f<T>(dt[q]) + bias;
    if (p.softplus) delta = softplus(delta);
    const float u = delta * to_f<T>(x[q]);
    copies_done<G - 1 - q>();
    float y[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      // The lane with share r: bits 0 and 1 of its place hold the halves in that order.
      const int from = lead + ((r >> 1) | ((r & 1) << 1));
      const float2 d = splat(__shfl_sync(0xffffffffu, delta, from)), v = splat(__shfl_sync(0xffffffffu, u, from));
      const float4 b = unpack4(B[r]), c = unpack4(C[r]);
      float2 h[2];
      load_vec<ST, 4>(reinterpret_cast<const ST*>(staged) + ((q * kRows + r) * kStep + threadIdx.x) * 4, h);
      const float2 a0 = decay2<T>(d, A2[0]), a1 = decay2<T>(d, A2[1]);
      h[0] = ffma2(a0, h[0], fmul2(v, make_float2(b.x, b.y)));
      h[1] = ffma2(a1, h[1], fmul2(v, make_float2(b.z, b.w)));
      const float2 s = ffma2(h[1], make_float2(c.z, c.w), fmul2(h[0], make_float2(c.x, c.y)));
      y[r] = s.x + s.y;
      if (slot[q][r] >= 0 && in) store_vec<ST, 4>(state + slot[q][r] * slot_size, h);
    }
    lane_sums<kRows, NL, 1>(y);
    bool live = false;
#pragma unroll
    for (int r = 0; r < kRows; ++r) live = r == own ? slot[q][r] >= 0 : live;
    if (live && in && nl < 4) {
      float o = fmaf(skip, to_f<T>(x[q]), y[0]);
      const float zf = to_f<T>(z[q]);
      if (has_z) o *= zf * sigmoid(zf);
      op[static_cast<int64_t>(q * kRows) * p.dim] = from_f<T>(o);
    }
  };
  static_for<0, G>(group);
}

// Any number of tokens, states and alignment, four rows a CTA. VEC: a lane's 4 states are one aligned
// vector, and so are its B and C. 256 rows of 4352 channels, 16 states, inputs partly in L2: 78 us for 4
// tokens, 131 us for 8; with a token's operands loaded where they are used and addressed by products 113 and 202.
// What bounds it is the issue and latency of a token's work at 16 warps an SM (125 registers). Three CTAs an SM
// spill, and are slower but for the longest calls (77 and 124; 21 against 19 at 64 rows).
template <typename T, typename ST, int NL, bool VEC>
__global__ void __launch_bounds__(256, 2) cc1d_ssm_update_kernel(const __grid_constant__ SsmUpdateParams p) {
  const int nl = threadIdx.x % NL, n0 = 4 * nl;
  const int ch = static_cast<int>(blockIdx.x % p.blocks) * (256 / NL) + static_cast<int>(threadIdx.x) / NL;
  const int b0 = static_cast<int>(blockIdx.x / p.blocks) * kRows;
  const bool in = ch < p.dim;
  const int nn = in ? p.dstate - n0 : 0;  // states of this lane

  // Slots of the rows; -1 for a padded entry, of which nothing is read or written, and past the last channel.
  int slot[kRows];
  float2 h[kRows][2];
  ST* const state = static_cast<ST*>(p.state) + static_cast<int64_t>(ch) * p.dstate + n0;
  const int64_t slot_size = static_cast<int64_t>(p.dim) * p.dstate;
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int b = b0 + r;
    const int v = b >= p.batch ? -1 : (p.indices != nullptr ? p.indices[b] : b);
    slot[r] = in && v < p.slots ? v : -1;
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    h[r][0] = h[r][1] = make_float2(0.f, 0.f);
    if (slot[r] >= 0) {
      ST* const at = state + slot[r] * slot_size;
      if (VEC) {
        if (nn > 0) load_vec<ST, 4>(at, h[r]);
      } else {
        if (nn > 0) h[r][0].x = to_f<ST>(at[0]);
        if (nn > 1) h[r][0].y = to_f<ST>(at[1]);
        if (nn > 2) h[r][1].x = to_f<ST>(at[2]);
        if (nn > 3) h[r][1].y = to_f<ST>(at[3]);
      }
    }
  }
  float a[4];
  ld_any4(p.A.ptr, static_cast<int64_t>(ch) * p.dstate + n0, p.A.dtype, nn, a);
  const float2 A2[2] = {make_float2(a[0] * kLog2e, a[1] * kLog2e), make_float2(a[2] * kLog2e, a[3] * kLog2e)};
  const float skip = in && p.D.ptr != nullptr ? ld_any(p.D.ptr, ch, p.D.dtype) : 0.0f;
  const float bias = in && p.dt_bias.ptr != nullptr ? ld_any(p.dt_bias.ptr, ch, p.dt_bias.dtype) : 0.0f;

  const int own = lane_share<kRows, NL, 1>(), lead = threadIdx.x & 31 & ~(NL - 1);
  const int64_t ob = b0 + own;
  bool own_live = false;
#pragma unroll
  for (int r = 0; r < kRows; ++r) own_live = r == own ? slot[r] >= 0 : own_live;
  const int64_t g = in ? ch / p.group_dim : 0;
  const T* bp = static_cast<const T*>(p.Bm.ptr) + b0 * p.Bm.sb + g * p.Bm.sg;
  const T* cp = static_cast<const T*>(p.Cm.ptr) + b0 * p.Cm.sb + g * p.Cm.sg;
  const T* xp = static_cast<const T*>(p.x.ptr) + ob * p.x.sb + ch;
  const T* dp = static_cast<const T*>(p.dt.ptr) + ob * p.dt.sb + ch;
  const T* zp = static_cast<const T*>(p.z.ptr) + ob * p.z.sb + ch;
  T* op = static_cast<T*>(p.out) + ob * p.seqlen * p.dim + ch;

  // A token's operands are on the way while the token before it is computed.
  T xt = from_f<T>(0.0f), dtt = xt, zt = xt;
  Raw4<T> Bt[kRows], Ct[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) Bt[r] = Ct[r] = zero4<T>();
  auto fetch = [&]() {
    if (own_live) {
      xt = *xp, dtt = *dp;
      if (p.z.ptr != nullptr) zt = *zp;
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (slot[r] >= 0 && nn > 0) {
        Bt[r] = load4(bp + r * p.Bm.sb, n0, VEC ? kSsmMaxState : p.dstate, VEC);
        Ct[r] = load4(cp + r * p.Cm.sb, n0, VEC ? kSsmMaxState : p.dstate, VEC);
      }
    }
    xp += p.x.st, dp += p.dt.st, zp += p.z.st, bp += p.Bm.st, cp += p.Cm.st;
  };
  if (p.seqlen > 0) fetch();

#pragma unroll 1
  for (int64_t l = 0; l < p.seqlen; ++l, op += p.dim) {
    const float x = own_live ? to_f<T>(xt) : 0.0f, z = to_f<T>(zt);
    float delta = own_live ? to_f<T>(dtt) + bias : 0.0f;
    Raw4<T> B[kRows], C[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) B[r] = Bt[r], C[r] = Ct[r];
    if (l + 1 < p.seqlen) fetch();
    if (p.softplus) delta = softplus(delta);
    const float u = delta * x;
    float y[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int from = lead + ((r >> 1) | ((r & 1) << 1));
      const float2 d = splat(__shfl_sync(0xffffffffu, delta, from)), v = splat(__shfl_sync(0xffffffffu, u, from));
      const float4 b = unpack4(B[r]), c = unpack4(C[r]);
      const float2 a0 = decay2<T>(d, A2[0]), a1 = decay2<T>(d, A2[1]);
      h[r][0] = ffma2(a0, h[r][0], fmul2(v, make_float2(b.x, b.y)));
      h[r][1] = ffma2(a1, h[r][1], fmul2(v, make_float2(b.z, b.w)));
      const float2 s = ffma2(h[r][1], make_float2(c.z, c.w), fmul2(h[r][0], make_float2(c.x, c.y)));
      y[r] = s.x + s.y;
    }
    lane_sums<kRows, NL, 1>(y);
    if (own_live && nl < 4) {
      float o = fmaf(skip, x, y[0]);
      if (p.z.ptr != nullptr) o *= z * sigmoid(z);
      *op = from_f<T>(o);
    }
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    if (slot[r] >= 0) {
      ST* const at = state + slot[r] * slot_size;
      if (VEC) {
        if (nn > 0) store_vec<ST, 4>(at, h[r]);
      } else {
        if (nn > 0) at[0] = from_f<ST>(h[r][0].x);
        if (nn > 1) at[1] = from_f<ST>(h[r][0].y);
        if (nn > 2) at[2] = from_f<ST>(h[r][1].x);
        if (nn > 3) at[3] = from_f<ST>(h[r][1].y);
      }
    }
  }
}

template <typename T, typename ST, int NL, int G>
cudaError_t launch_step(SsmUpdateParams p, cudaStream_t s) {
  p.blocks = static_cast<int>((static_cast<int64_t>(p.dim) * NL + kStep - 1) / kStep);
  constexpr int smem = G * kRows * kStep * 4 * static_cast<int>(sizeof(ST));
  const cudaError_t e = allow_smem<cc1d_ssm_step_kernel<T, ST, NL, G>>(smem);
  if (e != cudaSuccess) return e;
  const unsigned grid = static_cast<unsigned>(p.blocks) * ((p.batch + G * kRows - 1) / (G * kRows));
  cc1d_ssm_step_kernel<T, ST, NL, G><<<grid, kStep, smem, s>>>(p);
  return cudaGetLastError();
}

template <typename T, typename ST, int NL>
cudaError_t launch(const SsmUpdateParams& p, cudaStream_t s) {
  const bool vec = p.dstate % 4 == 0 && reinterpret_cast<uintptr_t>(p.state) % (4 * sizeof(ST)) == 0 && p.Bm.vec && p.Cm.vec;
  // The one-token kernel has no lane without states, which it would have to mask in its copies, stores and loads
  // of A, B and C: 4, 8, 12 or 20 states take the general kernel, also where they are aligned (256 rows of 4352
  // channels, fp32 states: 4 states 39 us, 8 42, 12 45, against 31 for 16).
  if (vec && p.seqlen == 1 && p.dstate == 4 * NL) {
    // Two groups a CTA where that leaves 512 threads for every SM, one for small batches. States out of the
    // caches, one group against two: 1 x 512 channels 2.1 and 2.7 us, 48 x 2048 4.1 and 4.4, 64 x 2048 5.2 and 5.8
    // (433 threads an SM); 96 x 2048 7.8 and 7.4 (649), 256 x 4352 30.0 and 28.5.
    const int64_t wide = static_cast<int64_t>(p.blocks) * ((p.batch + 2 * kRows - 1) / (2 * kRows));
    return wide >= 2 * p.sms ? launch_step<T, ST, NL, 2>(p, s) : launch_step<T, ST, NL, 1>(p, s);
  }
  const unsigned grid = static_cast<unsigned>(p.blocks) * ((p.batch + kRows - 1) / kRows);
  if (vec)
    cc1d_ssm_update_kernel<T, ST, NL, true><<<grid, 256, 0, s>>>(p);
  else
    cc1d_ssm_update_kernel<T, ST, NL, false><<<grid, 256, 0, s>>>(p);
  return cudaGetLastError();
}

template <typename T, typename ST>
cudaError_t launch(SsmUpdateParams p, cudaStream_t s) {
  const int nl = ssm_lanes(p.dstate);
  p.blocks = static_cast<int>((static_cast<int64_t>(p.dim) * nl + 255) / 256);
  if (nl == 4) return launch<T, ST, 4>(p, s);
  if (nl == 8) return launch<T, ST, 8>(p, s);
  return launch<T, ST, 16>(p, s);
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
