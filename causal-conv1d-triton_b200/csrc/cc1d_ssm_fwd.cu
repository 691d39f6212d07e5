// Forward of the input-dependent state-space recurrence, per channel d and state n:
//   h[t] = exp(delta[t] A[d, n]) h[t-1] + delta[t] x[t] B[t, n]
//   out[t] = (sum_n C[t, n] h[t] + D[d] x[t]) silu(z[t]),   delta = softplus(dt + dt_bias)
#include "cc1d_ssm_device.cuh"

namespace cc1d {
namespace {

constexpr int kThreads = 256;
constexpr int kTokens = 32;  // tokens staged at a time

// A lane holds one channel's 4 states, NL lanes a channel; a warp covers 32 / NL channels and walks
// the tokens. Per tile of 32 tokens the CTA first computes (delta, delta x) of its channels once,
// element-wise, into shared memory with B and C in fp32; then the walk reads them as broadcasts;
// then the y of the tile, summed over the lanes of a channel four tokens at a time (lane_sums), gets
// the skip, the gate and its rounding in the element-wise mapping again, with 16-byte loads and
// stores. The next tile's loads are in flight during the walk.
//
// PASS kSsmForward is that. The other two prepare a sequence cut in pieces: kSsmPieceForward finds
// the state that a piece leaves when it starts from zero, kSsmPieceBackward the gradient that it
// passes back when it receives none, each with the piece's decay exp(A sum delta); launch_ssm_join
// chains them.
template <typename T, int NL, int PASS>
__global__ void __launch_bounds__(kThreads, 2) cc1d_ssm_scan_kernel(const __grid_constant__ SsmParams p) {
  constexpr int CW = 32 / NL, CH = 8 * CW, NP = 4 * NL, VR = CH / 8;
  constexpr int VECS = kTokens * VR;                           // 8-channel vectors of a tile
  constexpr int QUADS = kTokens * NL;                          // 4-state vectors of a tile, for B and for C
  constexpr int NQ = (2 * QUADS + kThreads - 1) / kThreads;    // of both, per thread
  static_assert(VECS <= kThreads, "one vector per thread");
  constexpr bool FWD = PASS == kSsmForward, BACK = PASS == kSsmPieceBackward;
  __shared__ float2 du[kTokens][CH];     // (delta, delta x); backward: (delta, dy)
  __shared__ float ys[kTokens][CH + 8];  // + 8: four rows of a warp's channels fall in different banks
  __shared__ float4 bc[2][kTokens][NL];  // B, C
  __shared__ float sk[2][CH];            // D, dt_bias

  const SsmPlace w = ssm_place<CH>(p);
  if ((PASS == kSsmPieceForward && w.seg == p.segs - 1) || (BACK && w.seg == 0)) return;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cl = lane / NL, nl = lane % NL, n0 = 4 * nl;
  const int lc = warp * CW + cl;  // channel within the block
  const bool live = lc < w.nc;
  const int ch = w.c0 + lc;

  if (tid < CH) {
    const bool in = tid < w.nc;
    sk[0][tid] = in && p.D.ptr != nullptr ? ld_any(p.D.ptr, w.c0 + tid, p.D.dtype) : 0.0f;
    sk[1][tid] = in && p.dt_bias.ptr != nullptr ? ld_any(p.dt_bias.ptr, w.c0 + tid, p.dt_bias.dtype) : 0.0f;
  }
  float2 A2[2], h[2];
  {
    float a[4], s[4];
    const int64_t row = static_cast<int64_t>(w.b) * p.dim + ch;
    const int64_t piece = ((static_cast<int64_t>(w.b) * p.segs + w.seg) * p.dim + ch) * NP + n0;
    const bool from_init = BACK ? w.seg == p.segs - 1 : w.seg == 0;
    const SsmParam& start = BACK ? p.dfinal : p.init;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const bool in = live && n0 + m < p.dstate;
      a[m] = in ? ld_any(p.A.ptr, static_cast<int64_t>(ch) * p.dstate + n0 + m, p.A.dtype) * kLog2e : 0.0f;
      s[m] = 0.0f;
      if (in && from_init && start.ptr != nullptr) s[m] = ld_any(start.ptr, row * p.dstate + n0 + m, start.dtype);
      if (FWD && live && !from_init) s[m] = p.seg_state[piece + m];
    }
    A2[0] = make_float2(a[0], a[1]), A2[1] = make_float2(a[2], a[3]);
    h[0] = make_float2(s[0], s[1]), h[1] = make_float2(s[2], s[3]);
  }
  float sum_delta = 0.0f;
  bool cut = false;  // a sequence starts in the piece: nothing passes through it

  // The element-wise mapping: one vector of 8 channels of one token per thread.
  const int er = tid / VR, ec = (tid % VR) * 8, en = min(8, w.nc - ec);
  const bool ework = tid < VECS && en > 0;
  const T *xp = static_cast<const T*>(p.x.ptr) + w.b * p.x.sb + w.c0 + ec;
  const T *dp = static_cast<const T*>(p.dt.ptr) + w.b * p.dt.sb + w.c0 + ec;
  const T *zp = static_cast<const T*>(p.z.ptr) + w.b * p.z.sb + w.c0 + ec;
  const T *gp = static_cast<const T*>(p.dout.ptr) + w.b * p.dout.sb + w.c0 + ec;
  const T *bp = static_cast<const T*>(p.Bm.ptr) + w.b * p.Bm.sb + w.g * p.Bm.sg;
  const T *cp = static_cast<const T*>(p.Cm.ptr) + w.b * p.Cm.sb + w.g * p.Cm.sg;
  const bool has_z = p.z.ptr != nullptr;

  Raw8<T> rx = zero8<T>(), rd = zero8<T>(), rz = zero8<T>();
  float4 rq[NQ];
  auto load_tile = [&](int t) {
    const int64_t te = t + er;
    if (ework && te < w.t1) {
      rd = load8(dp + te * p.dt.st, en, p.dt.vec);
      if constexpr (BACK) rx = load8(gp + te * p.dout.st, en, p.dout.vec);
      else rx = load8(xp + te * p.x.st, en, p.x.vec);
      if (PASS != kSsmPieceForward && has_z) rz = load8(zp + te * p.z.st, en, p.z.vec);
    }
#pragma unroll
    for (int k = 0; k < NQ; ++k) {
      const int i = tid + k * kThreads, which = i / QUADS, tq = (i % QUADS) / NL, nq = 4 * (i % NL);
      const int64_t tk = t + tq;
      rq[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      // A piece's state needs no C, its gradient no B.
      if (i < 2 * QUADS && tk < w.t1 && (FWD || which == (BACK ? 1 : 0)))
        rq[k] = which ? load4(cp + tk * p.Cm.st, nq, p.dstate, p.Cm.vec) : load4(bp + tk * p.Bm.st, nq, p.dstate, p.Bm.vec);
    }
  };

  const int tiles = (w.t1 - w.t0 + kTokens - 1) / kTokens;
  const int64_t kept_tiles = (p.seqlen + kSsmTile - 1) / kSsmTile;
  load_tile(BACK ? w.t0 + (tiles - 1) * kTokens : w.t0);
  __syncthreads();  // sk

  for (int it = 0; it < tiles; ++it) {
    const int t = w.t0 + (BACK ? tiles - 1 - it : it) * kTokens;
    const SeqBits seq = seq_bits(p, w.b, t);
    const bool off = (seq.pad >> er) & 1u;  // padding: no step, no input, output 0
    const Raw8<T> cx = rx, cz = rz;
    if (tid < VECS) {
      float v[8], u[8];
      unpack8(rd, v), unpack8(cx, u);
      const bool in = ework && t + er < w.t1 && !off;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float raw = v[i] + sk[1][ec + i];
        const float delta = p.softplus ? softplus(raw) : raw;
        const float second = BACK ? u[i] : delta * u[i];
        v[i] = in ? delta : 0.0f, u[i] = in ? second : 0.0f;
      }
      if (BACK && has_z) {
        float z[8];
        unpack8(cz, z);
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] = in ? u[i] * z[i] * sigmoid(z[i]) : 0.0f;
      }
      float4* dst = reinterpret_cast<float4*>(&du[er][ec]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // Rotated by the vector's place, so that a warp's 16-byte stores spread over the banks.
        const int k = (i + (tid & 3)) & 3;
        float4 q = make_float4(v[0], u[0], v[1], u[1]);
        if (k == 1) q = make_float4(v[2], u[2], v[3], u[3]);
        if (k == 2) q = make_float4(v[4], u[4], v[5], u[5]);
        if (k == 3) q = make_float4(v[6], u[6], v[7], u[7]);
        dst[k] = q;
      }
    }
#pragma unroll
    for (int k = 0; k < NQ; ++k) {
      const int i = tid + k * kThreads, tq = (i % QUADS) / NL;
      if (i < 2 * QUADS) {
        const bool gone = (seq.pad >> tq) & 1u;
        bc[i / QUADS][tq][i % NL] = gone ? make_float4(0.f, 0.f, 0.f, 0.f) : rq[k];
      }
    }
    __syncthreads();
    if (it + 1 < tiles) load_tile(BACK ? t - kTokens : t + kTokens);

#pragma unroll 2
    for (int q = 0; q < kTokens / 4; ++q) {
      if constexpr (FWD) {
        if (p.kept != nullptr && (4 * q) % kSsmTile == 0 && live && t + 4 * q < w.t1) {
          const int64_t kt = static_cast<int64_t>(w.b) * kept_tiles + (t + 4 * q) / kSsmTile;
          *reinterpret_cast<float4*>(p.kept + (kt * p.dim + ch) * NP + n0) = make_float4(h[0].x, h[0].y, h[1].x, h[1].y);
        }
      }
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = BACK ? kTokens - 1 - 4 * q - j : 4 * q + j;
        const float2 e = du[i][lc];
        float delta = e.x;
        const bool start = (seq.start >> i) & 1u;
        if constexpr (BACK) {
          const float4 c = bc[1][i][nl];
          h[0] = ffma2(splat(e.y), make_float2(c.x, c.y), h[0]);
          h[1] = ffma2(splat(e.y), make_float2(c.z, c.w), h[1]);
          h[0] = fmul2(exp2_approx2(fmul2(splat(delta), A2[0])), h[0]);
          h[1] = fmul2(exp2_approx2(fmul2(splat(delta), A2[1])), h[1]);
          sum_delta += delta;
          if (start) h[0] = h[1] = make_float2(0.f, 0.f), cut = true;
        } else {
          if (start) h[0] = h[1] = make_float2(0.f, 0.f), delta = 0.0f, cut = true;
          const float4 b = bc[0][i][nl];
          const float2 a0 = exp2_approx2(fmul2(splat(delta), A2[0])), a1 = exp2_approx2(fmul2(splat(delta), A2[1]));
          h[0] = ffma2(a0, h[0], fmul2(splat(e.y), make_float2(b.x, b.y)));
          h[1] = ffma2(a1, h[1], fmul2(splat(e.y), make_float2(b.z, b.w)));
          if constexpr (FWD) {
            const float4 c = bc[1][i][nl];
            const float2 s = ffma2(h[1], make_float2(c.z, c.w), fmul2(h[0], make_float2(c.x, c.y)));
            v[j] = s.x + s.y;
            if (p.cache != nullptr && ((seq.last >> i) & 1u)) {
              const int id = p.seq_idx[static_cast<int64_t>(w.b) * p.seqlen + t + i];
              const int64_t slot = id < p.cache_n ? p.cache_idx[w.b * p.cache_n + id] : -1;
              if (slot >= 0 && slot < p.cache_slots && live) {
                const float s4[4] = {h[0].x, h[0].y, h[1].x, h[1].y};
#pragma unroll
                for (int m = 0; m < 4; ++m)
                  if (n0 + m < p.dstate)
                    st_any(p.cache, (slot * p.dim + ch) * p.dstate + n0 + m, p.cache_dtype, s4[m]);
              }
            }
          } else {
            sum_delta += delta;
          }
        }
      }
      if constexpr (FWD) {
        lane_sums<4, NL, 1>(v);
        static_assert(share_size<4, NL>() == 1, "four tokens over at least four lanes");
        if (nl < 4) ys[4 * q + lane_share<4, NL, 1>()][lc] = v[0];
      }
    }
    __syncthreads();
    if constexpr (FWD) {
      if (ework && t + er < w.t1) {
        float x[8], o[8];
        unpack8(cx, x);
#pragma unroll
        for (int i = 0; i < 8; i += 4) *reinterpret_cast<float4*>(&o[i]) = *reinterpret_cast<const float4*>(&ys[er][ec + i]);
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = fmaf(sk[0][ec + i], x[i], o[i]);
        if (has_z) {
          unpack8(cz, x);
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] *= x[i] * sigmoid(x[i]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = off ? 0.0f : o[i];
        T* dst = static_cast<T*>(p.out) + (static_cast<int64_t>(w.b) * p.seqlen + t + er) * p.dim + w.c0 + ec;
        store8(dst, o, en, (p.dim * sizeof(T)) % 16 == 0 && (w.c0 * sizeof(T)) % 16 == 0);
      }
    }
  }

  if (!live) return;
  const float s4[4] = {h[0].x, h[0].y, h[1].x, h[1].y};
  if constexpr (FWD) {
    if (p.final_states != nullptr && w.seg == p.segs - 1) {
      float* dst = p.final_states + (static_cast<int64_t>(w.b) * p.dim + ch) * p.dstate + n0;
#pragma unroll
      for (int m = 0; m < 4; ++m)
        if (n0 + m < p.dstate) dst[m] = s4[m];
    }
  } else {
    const int64_t i = ((static_cast<int64_t>(w.b) * p.segs + w.seg) * p.dim + ch) * NP + n0;
    float2 e0 = exp2_approx2(fmul2(splat(sum_delta), A2[0])), e1 = exp2_approx2(fmul2(splat(sum_delta), A2[1]));
    if (cut) e0 = e1 = make_float2(0.f, 0.f);
    *reinterpret_cast<float4*>(p.seg_state + i) = make_float4(s4[0], s4[1], s4[2], s4[3]);
    *reinterpret_cast<float4*>(p.seg_decay + i) = make_float4(e0.x, e0.y, e1.x, e1.y);
  }
}

// Replaces each piece's own result by what it receives: forward, the state that the pieces before
// leave it; backward, the gradient that the pieces after pass to it. One thread per state.
__global__ void __launch_bounds__(256) cc1d_ssm_join_kernel(float* state, const float* decay, int segs, int64_t row,
                                                            int64_t n, bool backward) {
  const int64_t i = blockIdx.x * 256ll + threadIdx.x;
  if (i >= n) return;
  const int64_t step = backward ? -row : row, first = (i / row) * segs * row + i % row;
  int64_t at = backward ? first + (segs - 1) * row : first;
  float carry = state[at];
#pragma unroll 4
  for (int s = 1; s < segs; ++s) {
    at += step;
    if (s + 1 < segs) {
      const float own = state[at], d = decay[at];
      state[at] = carry;
      carry = d == 0.0f ? own : fmaf(d, carry, own);
    } else {
      state[at] = carry;  // the last piece's own result is not needed and was not computed
    }
  }
}

template <typename T, int NL>
cudaError_t launch(const SsmParams& p, SsmPass pass, cudaStream_t s) {
  const unsigned grid = static_cast<unsigned>(p.batch) * p.segs * p.groups * p.blocks;
  if (pass == kSsmForward)
    cc1d_ssm_scan_kernel<T, NL, kSsmForward><<<grid, kThreads, 0, s>>>(p);
  else if (pass == kSsmPieceForward)
    cc1d_ssm_scan_kernel<T, NL, kSsmPieceForward><<<grid, kThreads, 0, s>>>(p);
  else
    cc1d_ssm_scan_kernel<T, NL, kSsmPieceBackward><<<grid, kThreads, 0, s>>>(p);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch(const SsmParams& p, SsmPass pass, cudaStream_t s) {
  switch (ssm_lanes(p.dstate)) {
    case 4: return launch<T, 4>(p, pass, s);
    case 8: return launch<T, 8>(p, pass, s);
    default: return launch<T, 16>(p, pass, s);
  }
}

}  // namespace

cudaError_t launch_ssm_scan(const SsmParams& p, SsmPass pass, int x_dtype, cudaStream_t s) {
  if (x_dtype == kBF16) return launch<__nv_bfloat16>(p, pass, s);
  if (x_dtype == kF16) return launch<__half>(p, pass, s);
  return launch<float>(p, pass, s);
}

cudaError_t launch_ssm_join(const SsmParams& p, bool backward, cudaStream_t s) {
  const int64_t row = static_cast<int64_t>(p.dim) * 4 * ssm_lanes(p.dstate), n = p.batch * row;
  cc1d_ssm_join_kernel<<<static_cast<unsigned>((n + 255) / 256), 256, 0, s>>>(p.seg_state, p.seg_decay, p.segs, row, n,
                                                                            backward);
  return cudaGetLastError();
}

}  // namespace cc1d
