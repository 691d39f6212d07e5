// Forward of the input-dependent state-space recurrence, per channel d and state n:
//   h[t] = exp(delta[t] A[d, n]) h[t-1] + delta[t] x[t] B[t, n]
//   out[t] = (sum_n C[t, n] h[t] + D[d] x[t]) silu(z[t]),   delta = softplus(dt + dt_bias)
#include <type_traits>

#include "cc1d_ssm_device.cuh"

namespace cc1d {
namespace {

constexpr int kThreads = 2 * kSsmHalf;
constexpr int kTokens = kSsmTile;  // tokens of a tile

// Shared memory of one CTA.
template <typename T, int NL>
struct ScanSmem {
  static constexpr int CH = 256 / NL, NQ = 2 * kTokens * NL / kSsmHalf;  // channels; vectors of B and C a thread loads
  // Handed over. (delta, delta, u, u) of a channel pair, with u = delta x (backward: dy); a pair's place
  // within its vector of 8 channels is turned by the vector's, so that a warp's stores fall in different
  // banks.
  float4 du[kSsmStages][kTokens][CH / 2];
  float4 bc[kSsmStages][2][kTokens][NL];  // B, C
  float ys[kSsmStages][kTokens][CH + 8];  // + 8: four rows of a warp's channels fall in different banks
  uint32_t start[kSsmStages], last[kSsmStages];  // SeqBits of the tiles
  // The element-wise threads' own, as loaded: x (backward: dout), dt, z; B and C; sequence ids.
  uint4 raw[kSsmStages][3][sizeof(T) / 2][kSsmHalf];
  Raw4<T> raw_bc[kSsmStages][NQ][kSsmHalf];
  SeqIds ids[kSsmStages][kSsmHalf];
};

// The first four warps walk the tokens, the other four do what is element-wise, a tile ahead and a tile
// behind them. In the walk a lane holds 2 channels x 4 states, NL lanes a channel's states, a warp
// 64 / NL channels; (delta, delta x), B and C come from shared memory as broadcasts, and the y of four
// tokens at a time are summed over a channel's lanes by lane_sums. The element-wise half computes
// (delta, delta x) of the next tile, and gives the y of the last one their skip, gate and rounding,
// with 16-byte loads and stores; its own loads are asynchronous copies issued two tiles early.
//
// What bounds the walk is one exponential a (channel, state) pair on the MUFU pipe (8.1 cycles a warp
// instruction on each scheduler). A broadcast from shared memory costs the bandwidth of all the lanes
// that receive it, 128 bytes a cycle an SM: with one channel a lane (12 bytes a pair) that was the
// bound, with two it is 6 bytes. Done by the same warps in turn, the element-wise phases left the
// MUFU idle for half of the time at two warps a scheduler.
//
// PASS kSsmForward is that. The other two prepare a sequence cut in pieces: kSsmPieceForward finds
// the state that a piece leaves when it starts from zero, kSsmPieceBackward the gradient that it
// passes back when it receives none, each with the piece's decay exp(A sum delta), or kSsmCut where a
// sequence starts in it; launch_ssm_join or piece_in chains them. SEQ: packed rows (seq_idx).
template <typename T, int NL, int PASS, bool SEQ>
struct Scan {
  using S = ScanSmem<T, NL>;
  static constexpr int CL = 32 / NL, CH = S::CH, NP = 4 * NL, VR = CH / 8;
  static constexpr int QUADS = kTokens * NL, NQ = S::NQ;  // 4-state vectors of B (and of C)
  static constexpr bool FWD = PASS == kSsmForward, BACK = PASS == kSsmPieceBackward;

  static __device__ __forceinline__ int tile_start(const SsmPlace& w, int tiles, int it) {
    return w.t0 + (BACK ? tiles - 1 - it : it) * kTokens;
  }

  static __device__ __forceinline__ void elementwise(const SsmParams& p, const SsmPlace& w, S& s, int tiles) {
    const int tid = threadIdx.x - kSsmHalf;
    const int er = tid / VR, ec = (tid % VR) * 8, en = min(8, w.nc - ec);  // 8 channels of token er of a tile
    const bool work = er < kTokens && en > 0;
    const T* xp = static_cast<const T*>(BACK ? p.dout.ptr : p.x.ptr) + w.b * (BACK ? p.dout.sb : p.x.sb) + w.c0 + ec;
    const int64_t xs = BACK ? p.dout.st : p.x.st;
    const int xv = BACK ? p.dout.vec : p.x.vec;
    const T* dp = static_cast<const T*>(p.dt.ptr) + w.b * p.dt.sb + w.c0 + ec;
    const T* zp = static_cast<const T*>(p.z.ptr) + w.b * p.z.sb + w.c0 + ec;
    const T* bp = static_cast<const T*>(p.Bm.ptr) + w.b * p.Bm.sb + w.g * p.Bm.sg;
    const T* cp = static_cast<const T*>(p.Cm.ptr) + w.b * p.Cm.sb + w.g * p.Cm.sg;
    const bool has_z = PASS != kSsmPieceForward && p.z.ptr != nullptr;
    float2 skip[4], bias[4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float d = FWD && i < en && p.D.ptr != nullptr ? ld_any(p.D.ptr, w.c0 + ec + i, p.D.dtype) : 0.0f;
      const float b = i < en && p.dt_bias.ptr != nullptr ? ld_any(p.dt_bias.ptr, w.c0 + ec + i, p.dt_bias.dtype) : 0.0f;
      (i % 2 ? skip[i / 2].y : skip[i / 2].x) = d;
      (i % 2 ? bias[i / 2].y : bias[i / 2].x) = b;
    }
    const bool out_vec = p.out_vec && (w.c0 * sizeof(T)) % 16 == 0;
    T* const out = static_cast<T*>(p.out) + (static_cast<int64_t>(w.b) * p.seqlen + er) * p.dim + w.c0 + ec;

    auto fetch = [&](int it) {
      const int st = it % kSsmStages, t = tile_start(w, tiles, it);
      const int64_t te = t + er;
      if (work && te < w.t1) {
        copy8(&s.raw[st][0][0][tid], xp + te * xs, en, xv, kSsmHalf);
        copy8(&s.raw[st][1][0][tid], dp + te * p.dt.st, en, p.dt.vec, kSsmHalf);
        if (has_z) copy8(&s.raw[st][2][0][tid], zp + te * p.z.st, en, p.z.vec, kSsmHalf);
      }
#pragma unroll
      for (int k = 0; k < NQ; ++k) {
        const int i = tid + k * kSsmHalf, which = i / QUADS, nq = 4 * (i % NL);
        const int64_t tk = t + (i % QUADS) / NL;
        // A piece's state needs no C, its gradient no B.
        if (tk < w.t1 && (FWD || which == (BACK ? 1 : 0))) {
          if (which) copy4(&s.raw_bc[st][k][tid], cp + tk * p.Cm.st, nq, p.dstate, p.Cm.vec);
          else copy4(&s.raw_bc[st][k][tid], bp + tk * p.Bm.st, nq, p.dstate, p.Bm.vec);
        }
      }
      if (SEQ) copy_ids(&s.ids[st][tid], p, w.b, t);
    };
    fetch(0);
    copies_issued();
    if (tiles > 1) fetch(1);
    copies_issued();

    Raw8<T> x0 = zero8<T>(), z0 = x0, x1 = x0, z1 = x0, x2 = x0, z2 = x0;  // of this tile and the two before
    uint32_t off0 = 0, off1 = 0, off2 = 0;
    int st = 0;
    for (int it = 0; it < tiles + 2; ++it, st = next_stage(st)) {
      x2 = x1, z2 = z1, off2 = off1, x1 = x0, z1 = z0, off1 = off0;
      if (it < tiles) {
        const int t = tile_start(w, tiles, it);
        if (it + 2 < tiles) fetch(it + 2);
        copies_issued();
        copies_done<2>();
        SeqBits seq{0u, 0u, 0u};
        if (SEQ) seq = seq_bits(s.ids[st][tid], p, t);
        off0 = seq.pad;
        x0 = read8<T>(&s.raw[st][0][0][tid], kSsmHalf);
        z0 = read8<T>(&s.raw[st][2][0][tid], kSsmHalf);
        if (er < kTokens) {
          float4* const dst = &s.du[st][er][ec >> 1];
          const int turn = ec >> 4 & 3;
          // Padding takes no step and has no input; neither has what lies outside the piece.
          if (work && t + er < w.t1 && !(SEQ && ((seq.pad >> er) & 1u))) {
            float2 v[4], u[4];
            unpack8(read8<T>(&s.raw[st][1][0][tid], kSsmHalf), v), unpack8(x0, u);
            if (BACK && has_z) {
              float2 z[4];
              unpack8(z0, z);
#pragma unroll
              for (int i = 0; i < 4; ++i) u[i] = fmul2(u[i], fmul2(z[i], sigmoid2(z[i])));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float2 delta = fadd2(v[i], bias[i]);
              if (p.softplus) delta = softplus2(delta);
              const float2 second = BACK ? u[i] : fmul2(delta, u[i]);
              dst[i ^ turn] = make_float4(delta.x, delta.y, second.x, second.y);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) dst[i] = make_float4(0.f, 0.f, 0.f, 0.f);
          }
        }
#pragma unroll
        for (int k = 0; k < NQ; ++k) {
          const int i = tid + k * kSsmHalf, tq = (i % QUADS) / NL;
          const bool in = t + tq < w.t1 && (FWD || i / QUADS == (BACK ? 1 : 0)) && !(SEQ && ((seq.pad >> tq) & 1u));
          s.bc[st][i / QUADS][tq][i % NL] = in ? unpack4(s.raw_bc[st][k][tid]) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        if (SEQ && tid == 0) s.start[st] = seq.start, s.last[st] = seq.last;
        hand_over(full_barrier(st));
      }
      // Two tiles back: its sums are there, and its buffer is the next but one to be filled.
      if (it >= 2 && (FWD || it + 1 < tiles)) {
        const int back = next_stage(st);  // (st - 2) mod 3
        take_over(done_barrier(back));
        if constexpr (FWD) {
          const int t = tile_start(w, tiles, it - 2);
          if (work && t + er < w.t1) {
            float2 x[4], o[4];
            unpack8(x2, x), pairs8(&s.ys[back][er][ec], o);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = ffma2(skip[i], x[i], o[i]);
            if (has_z) {
              float2 z[4];
              unpack8(z2, z);
#pragma unroll
              for (int i = 0; i < 4; ++i) o[i] = fmul2(o[i], fmul2(z[i], sigmoid2(z[i])));
            }
            if (SEQ && ((off2 >> er) & 1u)) {
#pragma unroll
              for (int i = 0; i < 4; ++i) o[i] = make_float2(0.f, 0.f);
            }
            store8(out + static_cast<int64_t>(t) * p.dim, o, en, out_vec);
          }
        }
      }
    }
  }

  static __device__ __forceinline__ void walk(const SsmParams& p, const SsmPlace& w, S& s, int tiles) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int nl = lane % NL, n0 = 4 * nl;
    const int pair = warp * CL + lane / NL, lc = 2 * pair;  // the lane's channel pair, its first channel within the block
    const int place = (pair & ~3) | ((pair & 3) ^ (pair >> 3 & 3));
    const int64_t piece = (static_cast<int64_t>(w.b) * p.segs + w.seg) * p.dim;
    float2 A2[2][2], h[2][2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float a[4], v[4];
      const int ch = w.c0 + lc + c;
      const bool from_init = BACK ? w.seg == p.segs - 1 : w.seg == 0;
      const SsmParam& start = BACK ? p.dfinal : p.init;
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const bool in = lc + c < w.nc && n0 + m < p.dstate;
        a[m] = in ? ld_any(p.A.ptr, static_cast<int64_t>(ch) * p.dstate + n0 + m, p.A.dtype) * kLog2e : 0.0f;
        v[m] = 0.0f;
        if (in && from_init && start.ptr != nullptr)
          v[m] = ld_any(start.ptr, (static_cast<int64_t>(w.b) * p.dim + ch) * p.dstate + n0 + m, start.dtype);
      }
      A2[c][0] = make_float2(a[0], a[1]), A2[c][1] = make_float2(a[2], a[3]);
      h[c][0] = make_float2(v[0], v[1]), h[c][1] = make_float2(v[2], v[3]);
    }
    if (FWD && w.seg > 0) piece_in(p, w, NP, w.c0 + lc, n0, n0 + 2, false, h);
#pragma unroll
    for (int c = 0; c < 2; ++c)
      if (lc + c >= w.nc) h[c][0] = h[c][1] = make_float2(0.f, 0.f);  // no channel
    float sum_delta[2] = {0.0f, 0.0f};
    bool cut = false;  // a sequence starts in the piece: nothing passes through it
    const int64_t kept_tiles = (p.seqlen + kSsmTile - 1) / kSsmTile;

    int buf = 0;
#pragma unroll 1
    for (int it = 0; it < tiles; ++it, buf = next_stage(buf)) {
      const int t = tile_start(w, tiles, it);
      take_over(full_barrier(buf));
      const uint32_t starts = SEQ ? s.start[buf] : 0u, lasts = SEQ && p.cache != nullptr ? s.last[buf] : 0u;
      if constexpr (FWD) {
        if (p.kept != nullptr) {
          const int64_t kt = static_cast<int64_t>(w.b) * kept_tiles + t / kSsmTile;
#pragma unroll
          for (int c = 0; c < 2; ++c)
            if (lc + c < w.nc)
              *reinterpret_cast<float4*>(p.kept + (kt * p.dim + w.c0 + lc + c) * NP + n0) =
                  make_float4(h[c][0].x, h[c][0].y, h[c][1].x, h[c][1].y);
        }
      }
      // The tile's sums over states are stored at its end, so that nothing keeps the loads and the
      // exponentials of later tokens from being issued early.
      float v[kTokens / 4][8];  // [four tokens][token, channel]
      // CUTS: a sequence starts or ends in the tile.
      auto tokens = [&](auto cuts) {
        constexpr bool CUTS = decltype(cuts)::value;
        // The decays of a token are computed while the one before is worked on.
        float2 a[2][2][2];
        float4 e[2];
        auto decays = [&](int k) {
          const int i = BACK ? kTokens - 1 - k : k;
          e[k & 1] = s.du[buf][i][place];
          const bool start = !BACK && CUTS && ((starts >> i) & 1u);
          const float d[2] = {start ? 0.0f : e[k & 1].x, start ? 0.0f : e[k & 1].y};
#pragma unroll
          for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int m = 0; m < 2; ++m) a[k & 1][c][m] = decay2<T>(splat(d[c]), A2[c][m]);
            if constexpr (!FWD) sum_delta[c] += d[c];
          }
        };
        decays(0);
#pragma unroll
        for (int k = 0; k < kTokens; ++k) {
          const int i = BACK ? kTokens - 1 - k : k;
          if (k + 1 < kTokens) decays(k + 1);
          const float4 k4 = s.bc[buf][BACK ? 1 : 0][i][nl];
          const float u[2] = {e[k & 1].z, e[k & 1].w};
          const float2 K[2] = {make_float2(k4.x, k4.y), make_float2(k4.z, k4.w)};
          const bool start = CUTS && ((starts >> i) & 1u);
          if (!BACK && start) h[0][0] = h[0][1] = h[1][0] = h[1][1] = make_float2(0.f, 0.f);
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              if constexpr (BACK) h[c][m] = fmul2(a[k & 1][c][m], ffma2(splat(u[c]), K[m], h[c][m]));
              else h[c][m] = ffma2(a[k & 1][c][m], h[c][m], fmul2(splat(u[c]), K[m]));
            }
          if (BACK && start) h[0][0] = h[0][1] = h[1][0] = h[1][1] = make_float2(0.f, 0.f);
          if constexpr (FWD) {
            const float4 c4 = s.bc[buf][1][i][nl];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const float2 y = ffma2(h[c][1], make_float2(c4.z, c4.w), fmul2(h[c][0], make_float2(c4.x, c4.y)));
              v[k / 4][2 * (k % 4) + c] = y.x + y.y;
            }
            if (k % 4 == 3) lane_sums<8, NL, 1>(v[k / 4]);
            if (CUTS && ((lasts >> i) & 1u)) {
              const int id = p.seq_idx[static_cast<int64_t>(w.b) * p.seqlen + t + i];
              const int64_t slot = id < p.cache_n ? p.cache_idx[w.b * p.cache_n + id] : -1;
              if (slot >= 0 && slot < p.cache_slots) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                  const float s4[4] = {h[c][0].x, h[c][0].y, h[c][1].x, h[c][1].y};
#pragma unroll
                  for (int m = 0; m < 4; ++m)
                    if (lc + c < w.nc && n0 + m < p.dstate)
                      st_any(p.cache, (slot * p.dim + w.c0 + lc + c) * p.dstate + n0 + m, p.cache_dtype, s4[m]);
                }
              }
            }
          }
        }
      };
      if (SEQ && (starts | lasts) != 0u) {
        cut = cut || starts != 0u;
        tokens(std::true_type{});
      } else {
        tokens(std::false_type{});
      }
      if constexpr (FWD) {
        const int at = lane_share<8, NL, 1>();
#pragma unroll
        for (int q = 0; q < kTokens / 4; ++q) {
          if constexpr (share_size<8, NL>() == 2)
            *reinterpret_cast<float2*>(&s.ys[buf][4 * q + at / 2][lc]) = make_float2(v[q][0], v[q][1]);
          else if (nl < share_lanes<8, NL>())
            s.ys[buf][4 * q + at / 2][lc + at % 2] = v[q][0];
        }
      }
      // The element-wise half waits for every tile forward, for those whose buffer it fills again otherwise.
      if (FWD || it + 3 < tiles) hand_over(done_barrier(buf));
    }

#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int ch = w.c0 + lc + c;
      if (lc + c >= w.nc) continue;
      const float4 s4 = make_float4(h[c][0].x, h[c][0].y, h[c][1].x, h[c][1].y);
      if constexpr (FWD) {
        if (p.final_states != nullptr && w.seg == p.segs - 1) {
          float* dst = p.final_states + (static_cast<int64_t>(w.b) * p.dim + ch) * p.dstate + n0;
          const float v[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
          for (int m = 0; m < 4; ++m)
            if (n0 + m < p.dstate) dst[m] = v[m];
        }
      } else {
        const int64_t i = (piece + ch) * NP + n0;
        const float2 e0 = decay2<T>(splat(sum_delta[c]), A2[c][0]), e1 = decay2<T>(splat(sum_delta[c]), A2[c][1]);
        *reinterpret_cast<float4*>(p.seg_out + i) = s4;
        *reinterpret_cast<float4*>(p.seg_decay + i) = cut ? make_float4(kSsmCut, kSsmCut, kSsmCut, kSsmCut) : make_float4(e0.x, e0.y, e1.x, e1.y);
      }
    }
  }
};

template <typename T, int NL, int PASS, bool SEQ>
__global__ void __launch_bounds__(kThreads, 2) cc1d_ssm_scan_kernel(const __grid_constant__ SsmParams p) {
  using K = Scan<T, NL, PASS, SEQ>;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  typename K::S& s = *reinterpret_cast<typename K::S*>(smem_raw);
  const SsmPlace w = ssm_place<K::CH>(p);
  if ((PASS == kSsmPieceForward && w.seg == p.segs - 1) || (PASS == kSsmPieceBackward && w.seg == 0)) return;
  const int tiles = (w.t1 - w.t0 + kTokens - 1) / kTokens;
  if (threadIdx.x < kSsmHalf)
    K::walk(p, w, s, tiles);
  else
    K::elementwise(p, w, s, tiles);
}

// What each piece receives, from the pieces' own results: forward, the state that the pieces before
// leave it; backward, the gradient that the pieces after pass to it. One thread per state; its loads
// are independent of the chain, and those of eight pieces are gathered before pass_piece's branches, which
// would keep them from being issued early (83.5 us instead of 82.0 for 21230 tokens x 171 channels).
__global__ void __launch_bounds__(128) cc1d_ssm_join_kernel(const float* __restrict__ own, const float* __restrict__ decay,
                                                            float* __restrict__ in, int segs, int64_t row, int64_t n,
                                                            bool backward) {
  const int64_t i = blockIdx.x * 128ll + threadIdx.x;
  if (i >= n) return;
  const int64_t step = backward ? -row : row, first = (i / row) * segs * row + i % row;
  const int64_t at = backward ? first + (segs - 1) * row : first;
  float carry = own[at];
  constexpr int N = 8;
  int s = 1;
  for (; s + N <= segs - 1; s += N) {
    float o[N], d[N];
#pragma unroll
    for (int k = 0; k < N; ++k) o[k] = own[at + (s + k) * step], d[k] = decay[at + (s + k) * step];
#pragma unroll
    for (int k = 0; k < N; ++k) in[at + (s + k) * step] = carry, carry = pass_piece(d[k], carry, o[k]);
  }
  for (; s < segs - 1; ++s) in[at + s * step] = carry, carry = pass_piece(decay[at + s * step], carry, own[at + s * step]);
  in[at + (segs - 1) * step] = carry;  // the last piece's own result is not needed and was not computed
}

template <typename T, int NL, int PASS, bool SEQ>
cudaError_t launch(const SsmParams& p, cudaStream_t s) {
  constexpr int smem = static_cast<int>(sizeof(ScanSmem<T, NL>));
  const cudaError_t e = allow_smem<cc1d_ssm_scan_kernel<T, NL, PASS, SEQ>>(smem);
  if (e != cudaSuccess) return e;
  cc1d_ssm_scan_kernel<T, NL, PASS, SEQ><<<static_cast<unsigned>(p.batch) * p.segs * p.groups * p.blocks, kThreads, smem, s>>>(p);
  return cudaGetLastError();
}

template <typename T, int NL, bool SEQ>
cudaError_t launch(const SsmParams& p, SsmPass pass, cudaStream_t s) {
  if (pass == kSsmForward) return launch<T, NL, kSsmForward, SEQ>(p, s);
  if (pass == kSsmPieceForward) return launch<T, NL, kSsmPieceForward, SEQ>(p, s);
  return launch<T, NL, kSsmPieceBackward, SEQ>(p, s);
}

template <typename T>
cudaError_t launch(const SsmParams& p, SsmPass pass, cudaStream_t s) {
  const bool seq = p.seq_idx != nullptr;
  switch (ssm_lanes(p.dstate)) {
    case 4: return seq ? launch<T, 4, true>(p, pass, s) : launch<T, 4, false>(p, pass, s);
    case 8: return seq ? launch<T, 8, true>(p, pass, s) : launch<T, 8, false>(p, pass, s);
    default: return seq ? launch<T, 16, true>(p, pass, s) : launch<T, 16, false>(p, pass, s);
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
  cc1d_ssm_join_kernel<<<static_cast<unsigned>((n + 127) / 128), 128, 0, s>>>(p.seg_out, p.seg_decay, p.seg_in, p.segs, row, n,
                                                                            backward);
  return cudaGetLastError();
}

}  // namespace cc1d
