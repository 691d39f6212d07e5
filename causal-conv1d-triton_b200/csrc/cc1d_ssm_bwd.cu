// Backward of the input-dependent state-space recurrence. With dy = dout silu(z) and g the gradient
// of the state, run backwards from the one after the last token (dfinal or zero):
//   g[t] = dy[t] C[t] + a[t+1] g[t+1]
//   dC[t, n] = sum_d dy h[t]            dB[t, n] = sum_d g[t] delta x
//   q = g[t] a[t] h[t-1]                (the gradient of delta A)
//   ddelta = x sum_n g B + sum_n q A    dx = delta sum_n g B + D dy      dA = sum_t q delta
//   dz = dout y silu'(z)                dD = sum_t dy x                  ddt = ddelta softplus'
// It needs every h[t], which the forward does not keep: it keeps the state before each 16th token,
// and the states between are computed again.
#include "cc1d_ssm_device.cuh"

namespace cc1d {
namespace {

constexpr int kThreads = 128, kWarps = 4;
constexpr int kTokens = kSsmTile;  // tokens staged at a time: from one kept state to the next
constexpr int kRun = 4;            // tokens whose decays and states a thread holds in registers

template <typename T>
__device__ __forceinline__ void copy_raw8(uint4* dst, const T* src, int n, bool vec, int stride) {
  constexpr int Q = static_cast<int>(sizeof(T)) / 2;  // 16-byte pieces of 8 channels
  if (vec && n == 8) {
#pragma unroll
    for (int i = 0; i < Q; ++i)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst + i * stride)),
                   "l"(reinterpret_cast<const uint4*>(src) + i)
                   : "memory");
  } else {
    const Raw8<T> r = load8(src, n, false);
#pragma unroll
    for (int i = 0; i < Q; ++i) dst[i * stride] = make_uint4(r.w[4 * i], r.w[4 * i + 1], r.w[4 * i + 2], r.w[4 * i + 3]);
  }
}

template <typename T>
__device__ __forceinline__ void read_raw8(const uint4* src, int stride, float (&v)[8]) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < Raw8<T>::NW / 4; ++i) {
    const uint4 q = src[i * stride];
    r.w[4 * i] = q.x, r.w[4 * i + 1] = q.y, r.w[4 * i + 2] = q.z, r.w[4 * i + 3] = q.w;
  }
  unpack8(r, v);
}

// Shared memory of one CTA.
template <typename T, int NL>
struct BwdSmem {
  static constexpr int CH = 512 / NL, NP = 4 * NL, VR = CH / 8;
  static constexpr int NV = (kTokens * VR + kThreads - 1) / kThreads;  // 8-channel vectors per thread of a tile
  static constexpr int Q = static_cast<int>(sizeof(T)) / 2;
  uint4 raw[2][4][NV][Q][kThreads];     // x, dt, z, dout as loaded; each thread reads only its own
  float f[3][kTokens][CH];              // delta, delta x, dy; each token's then replaced by sum C h, sum g B, sum q A
  float4 h[kTokens / kRun][4][kThreads];  // states before each run of kRun tokens, private to a thread
  float4 bc[2][kTokens][NL];            // B, C
  float dbc[kWarps][kTokens][2 * NP];   // each warp's dB and dC of the tile
  float sk[2][CH];                      // D, dt_bias
  float sum[16][kThreads];              // dD and ddt_bias of a thread's 8 channels
};

// A lane holds 4 channels x 4 states, NL lanes a channel's states and 32 / NL lanes the warp's
// channels: of each token's products, the sums over states (y, sum g B, sum q A) and over channels
// (dB, dC) are first formed inside the thread, then across lanes by lane_sums, 12 values over NL
// lanes and 8 over the rest, which leaves 16 shuffles per token for 16 (channel, state) pairs.
// Bounded by the MUFU and FMA pipes: 1.75 exponentials and about 15 multiply-adds a pair.
// SEQ: packed rows (seq_idx), where a step may have to drop what came before it.
template <typename T, int NL, bool SEQ>
__global__ void __launch_bounds__(kThreads, 2) cc1d_ssm_bwd_kernel(const __grid_constant__ SsmParams p) {
  using S = BwdSmem<T, NL>;
  constexpr int CL = 32 / NL, CH = S::CH, NP = S::NP, VR = S::VR, NV = S::NV;
  constexpr int QUADS = kTokens * NL, NQ = 2 * QUADS / kThreads;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  S& s = *reinterpret_cast<S*>(smem_raw);

  const SsmPlace w = ssm_place<CH>(p);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int nl = lane % NL, n0 = 4 * nl;
  const int lc = warp * 4 * CL + 4 * (lane / NL);  // first of the thread's channels, within the block
  const int64_t row_bs = static_cast<int64_t>(w.b) * p.segs + w.seg;

  for (int i = tid; i < CH; i += kThreads) {
    const bool in = i < w.nc;
    s.sk[0][i] = in && p.D.ptr != nullptr ? ld_any(p.D.ptr, w.c0 + i, p.D.dtype) : 0.0f;
    s.sk[1][i] = in && p.dt_bias.ptr != nullptr ? ld_any(p.dt_bias.ptr, w.c0 + i, p.dt_bias.dtype) : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) s.sum[i][tid] = 0.0f;

  float2 A2[4][2], g[4][2], dA[4][2];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    float a[4], v[4];
    const int ch = w.c0 + lc + c;
    const bool last = w.seg == p.segs - 1;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const bool in = lc + c < w.nc && n0 + m < p.dstate;
      a[m] = in ? ld_any(p.A.ptr, static_cast<int64_t>(ch) * p.dstate + n0 + m, p.A.dtype) * kLog2e : 0.0f;
      v[m] = 0.0f;
      if (in && last && p.dfinal.ptr != nullptr)
        v[m] = ld_any(p.dfinal.ptr, (static_cast<int64_t>(w.b) * p.dim + ch) * p.dstate + n0 + m, p.dfinal.dtype);
      if (in && !last) v[m] = p.seg_state[(row_bs * p.dim + ch) * NP + n0 + m];
    }
    A2[c][0] = make_float2(a[0], a[1]), A2[c][1] = make_float2(a[2], a[3]);
    g[c][0] = make_float2(v[0], v[1]), g[c][1] = make_float2(v[2], v[3]);
    dA[c][0] = dA[c][1] = make_float2(0.f, 0.f);
  }

  const bool has_z = p.z.ptr != nullptr;
  const int64_t kept_tiles = (p.seqlen + kSsmTile - 1) / kSsmTile;
  // Element-wise mapping: vector k of a thread is channels ec.. of token row k; the column is the
  // same for every k, so that a thread's channels are.
  const int ec = (tid % VR) * 8, en = min(8, w.nc - ec);
  auto row_of = [&](int k) { return (tid + k * kThreads) / VR; };
  const T* const src[4] = {static_cast<const T*>(p.x.ptr) + w.b * p.x.sb + w.c0 + ec,
                           static_cast<const T*>(p.dt.ptr) + w.b * p.dt.sb + w.c0 + ec,
                           static_cast<const T*>(p.z.ptr) + w.b * p.z.sb + w.c0 + ec,
                           static_cast<const T*>(p.dout.ptr) + w.b * p.dout.sb + w.c0 + ec};
  const int64_t step[4] = {p.x.st, p.dt.st, p.z.st, p.dout.st};
  const int vec[4] = {p.x.vec, p.dt.vec, p.z.vec, p.dout.vec};
  const T* bp = static_cast<const T*>(p.Bm.ptr) + w.b * p.Bm.sb + w.g * p.Bm.sg;
  const T* cp = static_cast<const T*>(p.Cm.ptr) + w.b * p.Cm.sb + w.g * p.Cm.sg;

  auto fetch = [&](int t, int buf) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int r = row_of(k);
      if (r < kTokens && en > 0 && t + r < w.t1) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i != 2 || has_z) copy_raw8(&s.raw[buf][i][k][0][tid], src[i] + static_cast<int64_t>(t + r) * step[i], en, vec[i], kThreads);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  const int tiles = (w.t1 - w.t0 + kTokens - 1) / kTokens;
  fetch(w.t0 + (tiles - 1) * kTokens, 0);
  __syncthreads();  // sk

  for (int it = tiles - 1; it >= 0; --it) {
    const int t = w.t0 + it * kTokens, buf = (tiles - 1 - it) & 1;
    const SeqBits seq = SEQ ? seq_bits(p, w.b, t) : SeqBits{0u, 0u, 0u};
    float4 kept[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      kept[c] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (lc + c < w.nc) {
        const int64_t kt = static_cast<int64_t>(w.b) * kept_tiles + t / kSsmTile;
        kept[c] = *reinterpret_cast<const float4*>(p.kept + (kt * p.dim + w.c0 + lc + c) * NP + n0);
      }
    }
#pragma unroll
    for (int k = 0; k < NQ; ++k) {
      const int i = tid + k * kThreads, tq = (i % QUADS) / NL, nq = 4 * (i % NL);
      const int64_t tk = t + tq;
      float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
      if (tk < w.t1 && !(SEQ && ((seq.pad >> tq) & 1u)))
        q = i < QUADS ? load4(bp + tk * p.Bm.st, nq, p.dstate, p.Bm.vec) : load4(cp + tk * p.Cm.st, nq, p.dstate, p.Cm.vec);
      s.bc[i / QUADS][tq][i % NL] = q;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int r = row_of(k);
      if (r < kTokens) {
        float x[8], d[8], z[8], o[8];
        read_raw8<T>(&s.raw[buf][0][k][0][tid], kThreads, x);
        read_raw8<T>(&s.raw[buf][1][k][0][tid], kThreads, d);
        read_raw8<T>(&s.raw[buf][3][k][0][tid], kThreads, o);
        const bool in = en > 0 && t + r < w.t1 && !(SEQ && ((seq.pad >> r) & 1u));
        if (has_z) {
          read_raw8<T>(&s.raw[buf][2][k][0][tid], kThreads, z);
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] *= z[i] * sigmoid(z[i]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float raw = d[i] + s.sk[1][ec + i];
          const float delta = p.softplus ? softplus(raw) : raw;
          d[i] = in ? delta : 0.0f, x[i] = in ? delta * x[i] : 0.0f, o[i] = in ? o[i] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          *reinterpret_cast<float4*>(&s.f[0][r][ec + i]) = make_float4(d[i], d[i + 1], d[i + 2], d[i + 3]);
          *reinterpret_cast<float4*>(&s.f[1][r][ec + i]) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
          *reinterpret_cast<float4*>(&s.f[2][r][ec + i]) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        }
      }
    }
    __syncthreads();
    if (it > 0) fetch(t - kTokens, buf ^ 1);

    // One step of the recurrence; `a` gets the decays.
    auto advance = [&](int i, float2 (&h)[4][2], float2 (&a)[4][2]) {
      const float4 d4 = *reinterpret_cast<const float4*>(&s.f[0][i][lc]), u4 = *reinterpret_cast<const float4*>(&s.f[1][i][lc]);
      const float4 b = s.bc[0][i][nl];
      float d[4] = {d4.x, d4.y, d4.z, d4.w};
      const float u[4] = {u4.x, u4.y, u4.z, u4.w};
      const float2 B[2] = {make_float2(b.x, b.y), make_float2(b.z, b.w)};
      if (SEQ && ((seq.start >> i) & 1u)) {
#pragma unroll
        for (int c = 0; c < 4; ++c) d[c] = 0.0f, h[c][0] = h[c][1] = make_float2(0.f, 0.f);
      }
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          a[c][m] = exp2_approx2(fmul2(splat(d[c]), A2[c][m]));
          h[c][m] = ffma2(a[c][m], h[c][m], fmul2(splat(u[c]), B[m]));
        }
    };

    {
      float2 h[4][2], a[4][2];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s.h[0][c][tid] = kept[c];
        h[c][0] = make_float2(kept[c].x, kept[c].y), h[c][1] = make_float2(kept[c].z, kept[c].w);
      }
#pragma unroll 1
      for (int r = 1; r < kTokens / kRun; ++r) {
#pragma unroll
        for (int j = 0; j < kRun; ++j) advance((r - 1) * kRun + j, h, a);
#pragma unroll
        for (int c = 0; c < 4; ++c) s.h[r][c][tid] = make_float4(h[c][0].x, h[c][0].y, h[c][1].x, h[c][1].y);
      }
    }

#pragma unroll 1
    for (int r = kTokens / kRun - 1; r >= 0; --r) {
      float2 h[kRun + 1][4][2], a[kRun][4][2];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float4 q = s.h[r][c][tid];
        h[0][c][0] = make_float2(q.x, q.y), h[0][c][1] = make_float2(q.z, q.w);
      }
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
#pragma unroll
        for (int c = 0; c < 4; ++c) h[j + 1][c][0] = h[j][c][0], h[j + 1][c][1] = h[j][c][1];
        advance(r * kRun + j, h[j + 1], a[j]);
      }
#pragma unroll
      for (int j = kRun - 1; j >= 0; --j) {
        const int i = r * kRun + j;
        const float4 d4 = *reinterpret_cast<const float4*>(&s.f[0][i][lc]), u4 = *reinterpret_cast<const float4*>(&s.f[1][i][lc]);
        const float4 o4 = *reinterpret_cast<const float4*>(&s.f[2][i][lc]), b4 = s.bc[0][i][nl], c4 = s.bc[1][i][nl];
        const float d[4] = {d4.x, d4.y, d4.z, d4.w}, u[4] = {u4.x, u4.y, u4.z, u4.w}, o[4] = {o4.x, o4.y, o4.z, o4.w};
        const float2 B[2] = {make_float2(b4.x, b4.y), make_float2(b4.z, b4.w)};
        const float2 C[2] = {make_float2(c4.x, c4.y), make_float2(c4.z, c4.w)};
        const bool start = SEQ && ((seq.start >> i) & 1u);
        float2 dB[2], dC[2];
        float v[12];
#pragma unroll
        for (int m = 0; m < 2; ++m) dB[m] = dC[m] = make_float2(0.f, 0.f);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float2 y = make_float2(0.f, 0.f), gb = y, qa = y;
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            const float2 gt = ffma2(splat(o[c]), C[m], g[c][m]), ht = h[j + 1][c][m];
            y = ffma2(ht, C[m], y);
            dC[m] = ffma2(splat(o[c]), ht, dC[m]);
            dB[m] = ffma2(splat(u[c]), gt, dB[m]);
            gb = ffma2(gt, B[m], gb);
            float2 back = fmul2(a[j][c][m], gt);  // what the token before receives
            float2 q = fmul2(back, h[j][c][m]);
            if (start) back = q = make_float2(0.f, 0.f);
            qa = ffma2(q, A2[c][m], qa);
            dA[c][m] = ffma2(q, splat(d[c]), dA[c][m]);
            g[c][m] = back;
          }
          v[3 * c] = y.x + y.y, v[3 * c + 1] = gb.x + gb.y, v[3 * c + 2] = qa.x + qa.y;
        }
        lane_sums<12, NL, 1>(v);
        static_assert(share_size<12, NL>() == 3, "each of four lanes gets one channel's three sums");
        __syncwarp();  // every lane has read token i's delta, delta x and dy
        if (nl < 4) {
          const int c = lc + lane_share<12, NL, 1>() / 3;
          s.f[0][i][c] = v[0], s.f[1][i][c] = v[1], s.f[2][i][c] = v[2];
        }
        float e[8] = {dB[0].x, dB[0].y, dB[1].x, dB[1].y, dC[0].x, dC[0].y, dC[1].x, dC[1].y};
        lane_sums<8, CL, NL>(e);
        const int first = lane_share<8, CL, NL>();
#pragma unroll
        for (int k = 0; k < share_size<8, CL>(); ++k)
          s.dbc[warp][i][((first + k) >> 2) * NP + n0 + ((first + k) & 3)] = e[k];
      }
    }
    __syncthreads();

#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int r = row_of(k);
      if (r < kTokens && en > 0 && t + r < w.t1) {
        float x[8], d[8], z[8], o[8], y[8], gb[8], qa[8];
        read_raw8<T>(&s.raw[buf][0][k][0][tid], kThreads, x);
        read_raw8<T>(&s.raw[buf][1][k][0][tid], kThreads, d);
        read_raw8<T>(&s.raw[buf][3][k][0][tid], kThreads, o);
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          *reinterpret_cast<float4*>(&y[i]) = *reinterpret_cast<const float4*>(&s.f[0][r][ec + i]);
          *reinterpret_cast<float4*>(&gb[i]) = *reinterpret_cast<const float4*>(&s.f[1][r][ec + i]);
          *reinterpret_cast<float4*>(&qa[i]) = *reinterpret_cast<const float4*>(&s.f[2][r][ec + i]);
        }
        const bool off = SEQ && ((seq.pad >> r) & 1u);
        const int64_t at = (static_cast<int64_t>(w.b) * p.seqlen + t + r) * p.dim + w.c0 + ec;
        const bool out_vec = (p.dim * sizeof(T)) % 16 == 0 && (w.c0 * sizeof(T)) % 16 == 0;
        if (has_z) {
          read_raw8<T>(&s.raw[buf][2][k][0][tid], kThreads, z);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float sg = sigmoid(z[i]), yt = fmaf(s.sk[0][ec + i], x[i], y[i]);
            y[i] = off ? 0.0f : o[i] * yt * sg * fmaf(z[i], 1.0f - sg, 1.0f);  // dz
            o[i] *= z[i] * sg;                                                  // dy
          }
          store8(static_cast<T*>(p.dz) + at, y, en, out_vec);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float raw = d[i] + s.sk[1][ec + i];
          float delta = raw, slope = 1.0f;
          if (p.softplus) delta = softplus(raw), slope = sigmoid(raw);
          const float dd = off ? 0.0f : slope * fmaf(x[i], gb[i], kLn2 * qa[i]);
          s.sum[i][tid] += off ? 0.0f : o[i] * x[i];
          s.sum[8 + i][tid] += dd;
          x[i] = off ? 0.0f : fmaf(delta, gb[i], s.sk[0][ec + i] * o[i]);
          d[i] = dd;
        }
        store8(static_cast<T*>(p.dx) + at, x, en, out_vec);
        store8(static_cast<T*>(p.ddt) + at, d, en, out_vec);
      }
    }
    const int64_t tok = static_cast<int64_t>(w.b) * p.seqlen + t;
    for (int i = tid; i < kTokens * 2 * NP; i += kThreads) {
      const int r = i / (2 * NP), k = i % (2 * NP);
      if (t + r < w.t1) {
        const float v = (s.dbc[0][r][k] + s.dbc[1][r][k]) + (s.dbc[2][r][k] + s.dbc[3][r][k]);
        p.part_bc[(((tok + r) * p.groups + w.g) * p.blocks + w.blk) * (2 * NP) + k] = v;
      }
    }
  }

#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int ch = w.c0 + lc + c;
    if (lc + c < w.nc) {
      *reinterpret_cast<float4*>(p.part_a + (row_bs * p.dim + ch) * NP + n0) =
          make_float4(dA[c][0].x, dA[c][0].y, dA[c][1].x, dA[c][1].y);
      if (p.dinit != nullptr && w.seg == 0) {
        const float v[4] = {g[c][0].x, g[c][0].y, g[c][1].x, g[c][1].y};
#pragma unroll
        for (int m = 0; m < 4; ++m)
          if (n0 + m < p.dstate)
            st_any(p.dinit, (static_cast<int64_t>(w.b) * p.dim + ch) * p.dstate + n0 + m, p.init.dtype, v[m]);
      }
    }
  }
  __syncthreads();
  for (int i = tid; i < 2 * CH; i += kThreads) {  // the threads of one column of vectors, in order
    const int k = i / CH, c = i % CH;
    if (c < w.nc) {
      float v = 0.0f;
      for (int q = c / 8; q < kThreads; q += VR) v += s.sum[8 * k + c % 8][q];
      p.part_d[(row_bs * 2 + k) * p.dim + w.c0 + c] = v;
    }
  }
}

// The sums over CTAs, in a fixed order, and their rounding: first dB and dC (one thread per token,
// group and state), then dA (per channel and state), then dD and ddt_bias (per channel).
template <typename T>
__global__ void __launch_bounds__(256) cc1d_ssm_finish_kernel(const __grid_constant__ SsmParams p, int np, int64_t n_bc, int64_t n_a) {
  int64_t i = blockIdx.x * 256ll + threadIdx.x;
  if (i < n_bc) {
    const int k = static_cast<int>(i % (2 * p.dstate)), which = k / p.dstate, n = k % p.dstate;
    const int64_t row = i / (2 * p.dstate);  // token and group
    const float* src = p.part_bc + row * p.blocks * (2 * np) + which * np + n;
    float v = 0.0f;
    for (int q = 0; q < p.blocks; ++q) v += src[static_cast<int64_t>(q) * 2 * np];
    static_cast<T*>(which ? p.dC : p.dB)[row * p.dstate + n] = from_f<T>(v);
    return;
  }
  i -= n_bc;
  const int rows = p.batch * p.segs;
  if (i < n_a) {
    const float* src = p.part_a + i / p.dstate * np + i % p.dstate;
    float v = 0.0f;
#pragma unroll 4
    for (int q = 0; q < rows; ++q) v += src[static_cast<int64_t>(q) * p.dim * np];
    st_any(p.dA, i, p.A.dtype, v);
    return;
  }
  i -= n_a;
  if (i < 2ll * p.dim) {
    const int k = static_cast<int>(i / p.dim), ch = static_cast<int>(i % p.dim);
    float v = 0.0f;
#pragma unroll 4
    for (int q = 0; q < rows; ++q) v += p.part_d[(static_cast<int64_t>(q) * 2 + k) * p.dim + ch];
    if (k == 0 && p.dD != nullptr) st_any(p.dD, ch, p.D.dtype, v);
    if (k == 1 && p.ddt_bias != nullptr) st_any(p.ddt_bias, ch, p.dt_bias.dtype, v);
  }
}

template <typename T, int NL, bool SEQ>
cudaError_t launch_main(const SsmParams& p, cudaStream_t s) {
  constexpr int smem = static_cast<int>(sizeof(BwdSmem<T, NL>));
  const auto kernel = cc1d_ssm_bwd_kernel<T, NL, SEQ>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  kernel<<<static_cast<unsigned>(p.batch) * p.segs * p.groups * p.blocks, kThreads, smem, s>>>(p);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch(const SsmParams& p, cudaStream_t s) {
  const int nl = ssm_lanes(p.dstate);
  const bool seq = p.seq_idx != nullptr;
  cudaError_t e;
  if (nl == 4)
    e = seq ? launch_main<T, 4, true>(p, s) : launch_main<T, 4, false>(p, s);
  else if (nl == 8)
    e = seq ? launch_main<T, 8, true>(p, s) : launch_main<T, 8, false>(p, s);
  else
    e = seq ? launch_main<T, 16, true>(p, s) : launch_main<T, 16, false>(p, s);
  if (e != cudaSuccess) return e;
  const int64_t n_bc = static_cast<int64_t>(p.batch) * p.seqlen * p.groups * 2 * p.dstate;
  const int64_t n_a = static_cast<int64_t>(p.dim) * p.dstate, n = n_bc + n_a + 2ll * p.dim;
  cc1d_ssm_finish_kernel<T><<<static_cast<unsigned>((n + 255) / 256), 256, 0, s>>>(p, 4 * nl, n_bc, n_a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_ssm_bwd(const SsmParams& p, int x_dtype, cudaStream_t s) {
  if (x_dtype == kBF16) return launch<__nv_bfloat16>(p, s);
  if (x_dtype == kF16) return launch<__half>(p, s);
  return launch<float>(p, s);
}

}  // namespace cc1d
