// Backward of the input-dependent state-space recurrence. With dy = dout silu(z) and g the gradient
// of the state, run backwards from the one after the last token (dfinal or zero):
//   g[t] = dy[t] C[t] + a[t+1] g[t+1]
//   dC[t, n] = sum_d dy h[t]            dB[t, n] = sum_d g[t] delta x
//   q = g[t] a[t] h[t-1]                (the gradient of delta A)
//   ddelta = x sum_n g B + sum_n q A    dx = delta sum_n g B + D dy      dA = sum_t q delta
//   dz = dout y silu'(z)                dD = sum_t dy x                  ddt = ddelta softplus'
// It needs every h[t], which the forward does not keep: it keeps the state before each 16th token,
// and the states between are computed again.
#include <type_traits>

#include "cc1d_ssm_device.cuh"

namespace cc1d {
namespace {

constexpr int kThreads = 2 * kSsmHalf, kWarps = 4;  // warps of the walk
constexpr int kTokens = kSsmTile;                  // tokens of a tile: from one kept state to the next
constexpr int kRun = 4;                            // tokens whose decays and states a thread holds in registers
constexpr int kBuffers = 2;                        // tiles handed over
// Registers of a thread of each half after setmaxnreg; together twice what the launch gives each (128).
constexpr int kWalkRegs = 152, kElementRegs = 104;
static_assert(kWalkRegs + kElementRegs == 2 * 128, "the split draws on the registers of the launch");

// Shared memory of one CTA.
template <typename T, int NL>
struct BwdSmem {
  static constexpr int CH = 256 / NL, NP = 4 * NL, NQ = 2 * kTokens * NL / kSsmHalf;
  // Handed over.
  float4 du[kBuffers][kTokens][CH / 2];          // (delta, delta, delta x, delta x) of a channel pair
  float f[kBuffers][3][kTokens][CH];             // dy, then sum C h; sum g B; sum q A
  static constexpr int ORDERS = NL == 4 ? 2 : 1;  // above, a second copy would leave room for one CTA an SM only
  float4 bc[kBuffers][2][kTokens][ORDERS][NL];   // B, C; and with their pairs of states exchanged
  float dbc[kBuffers][kWarps][kTokens][2 * NP];  // each warp's dB and dC of the tile
  uint32_t start[kBuffers];                      // SeqBits of the tile
  // The walk's own, private to a thread: states before each run but the first, and before the tile.
  float4 h[kTokens / kRun - 1][2][kSsmHalf];
  float4 kept[2][2][kSsmHalf];
  // The element-wise threads' own, as loaded: x, dt, z, dout; B and C; sequence ids.
  uint4 raw[3][4][sizeof(T) / 2][kSsmHalf];
  Raw4<T> raw_bc[2][NQ][kSsmHalf];
  SeqIds ids[2][kWarps][kTokens];
  float sk[2][CH];                               // D, dt_bias
};

// The first four warps walk the tokens back, the other four do what is element-wise around them: dy,
// (delta, delta x), B and C of the next tile, and from the sums of the last one dx, ddt, dz and the
// CTA's dB and dC.
//
// In the walk a lane holds 2 channels x 4 states, NL lanes a channel's states and 32 / NL lanes the
// warp's channels: of each token's products, the sums over states (y, sum g B, sum q A) and over
// channels (dB, dC) are first formed inside the lane, then across lanes by lane_sums: 12 values of two
// tokens over NL lanes, 8 of each token over the rest. A tile's states are first walked through,
// keeping those before every 4th token, and each run of 4 tokens is then computed once more into
// registers and walked back. Half of the channel lanes hold their two pairs of states in exchanged
// order: what a lane sends in the first stage of the dB and dC sums is then its second pair and what it
// keeps its first, in every lane, without the selections that the other stages need. All stores to shared memory of a run are at its end, so that nothing
// keeps the loads of its next token from being issued early.
// SEQ: packed rows (seq_idx), where a step may have to drop what came before it.
template <typename T, int NL, bool SEQ>
struct Bwd {
  using S = BwdSmem<T, NL>;
  static constexpr int CL = 32 / NL, CH = S::CH, NP = S::NP, VR = CH / 8;
  static constexpr int QUADS = kTokens * NL, NQ = S::NQ;

  static __device__ __forceinline__ void elementwise(const SsmParams& p, const SsmPlace& w, S& s, int tiles) {
    const int tid = threadIdx.x - kSsmHalf;
    const int er = tid / VR, ec = (tid % VR) * 8, en = min(8, w.nc - ec);  // 8 channels of token er of a tile
    const bool work = er < kTokens && en > 0;
    const bool has_z = p.z.ptr != nullptr;
    const T* const src[4] = {static_cast<const T*>(p.x.ptr) + w.b * p.x.sb + w.c0 + ec,
                             static_cast<const T*>(p.dt.ptr) + w.b * p.dt.sb + w.c0 + ec,
                             static_cast<const T*>(p.z.ptr) + w.b * p.z.sb + w.c0 + ec,
                             static_cast<const T*>(p.dout.ptr) + w.b * p.dout.sb + w.c0 + ec};
    const int64_t step[4] = {p.x.st, p.dt.st, p.z.st, p.dout.st};
    const int vec[4] = {p.x.vec, p.dt.vec, p.z.vec, p.dout.vec};
    const T* bp = static_cast<const T*>(p.Bm.ptr) + w.b * p.Bm.sb + w.g * p.Bm.sg;
    const T* cp = static_cast<const T*>(p.Cm.ptr) + w.b * p.Cm.sb + w.g * p.Cm.sg;
    SeqIds* const ids[2] = {&s.ids[0][tid >> 5][tid & 15], &s.ids[1][tid >> 5][tid & 15]};

    auto fetch = [&](int it, int ring) {
      const int t = w.t0 + (tiles - 1 - it) * kTokens;
      if (work && t + er < w.t1) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i != 2 || has_z) copy8(&s.raw[ring][i][0][tid], src[i] + static_cast<int64_t>(t + er) * step[i], en, vec[i], kSsmHalf);
      }
#pragma unroll
      for (int k = 0; k < NQ; ++k) {
        const int i = tid + k * kSsmHalf, nq = 4 * (i % NL);
        const int64_t tk = t + (i % QUADS) / NL;
        if (tk < w.t1) {
          if (i < QUADS) copy4(&s.raw_bc[it & 1][k][tid], bp + tk * p.Bm.st, nq, p.dstate, p.Bm.vec);
          else copy4(&s.raw_bc[it & 1][k][tid], cp + tk * p.Cm.st, nq, p.dstate, p.Cm.vec);
        }
      }
      if (SEQ) copy_ids(ids[it & 1], p, w.b, t);
      copies_issued();
    };
    fetch(0, 0);

    // dB and dC of the CTA: element tid + k * 128 of a tile's rows of 2 NP.
    constexpr int SUMS = kTokens * 2 * NP / kSsmHalf, ROWS = kSsmHalf / (2 * NP);  // per thread; rows between two of them
    static_assert(kSsmHalf % (2 * NP) == 0 && SUMS * kSsmHalf == kTokens * 2 * NP, "");
    const int br = tid / (2 * NP), bk = tid % (2 * NP);
    const int64_t bc_row = static_cast<int64_t>(p.groups) * p.blocks * (2 * NP);
    float* const part_bc = p.part_bc + (static_cast<int64_t>(w.b) * p.seqlen + br) * bc_row +
                           (static_cast<int64_t>(w.g) * p.blocks + w.blk) * (2 * NP) + bk;
    const bool out_vec = p.out_vec && (w.c0 * sizeof(T)) % 16 == 0;
    const int64_t out = (static_cast<int64_t>(w.b) * p.seqlen + er) * p.dim + w.c0 + ec;
    const int turn = ec >> 4 & 3;

    float2 sums[2][4];  // dD and ddt_bias of the thread's channels
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[0][i] = sums[1][i] = make_float2(0.f, 0.f);
    uint32_t off0 = 0, off1 = 0, off2 = 0;
    int ring = 0;
    for (int it = 0; it < tiles + 2; ++it, ring = next_stage(ring)) {
      const int buf = it & 1;
      off2 = off1, off1 = off0;
      if (it >= 2) {
        const int t = w.t0 + (tiles + 1 - it) * kTokens, old = next_stage(ring);  // two tiles ago
        take_over(done_barrier(buf));
        if (work && t + er < w.t1) {
          const int64_t at = out + static_cast<int64_t>(t) * p.dim;
          float2 dx[4], dd[4], dz[4];
          if (SEQ && ((off2 >> er) & 1u)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) dx[i] = dd[i] = dz[i] = make_float2(0.f, 0.f);
          } else {
            float2 x[4], o[4], v[4], skip[4];
            unpack8(read8<T>(&s.raw[old][0][0][tid], kSsmHalf), x);
            unpack8(read8<T>(&s.raw[old][3][0][tid], kSsmHalf), o);
            pairs8(&s.sk[0][ec], skip);
            if (has_z) {
              float2 z[4];
              unpack8(read8<T>(&s.raw[old][2][0][tid], kSsmHalf), z);
              pairs8(&s.f[buf][0][er][ec], v);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float2 sg = sigmoid2(z[i]), y = ffma2(skip[i], x[i], v[i]);
                const float2 rest = make_float2(1.0f - sg.x, 1.0f - sg.y);  // silu' = sg (1 + z (1 - sg))
                dz[i] = fmul2(fmul2(o[i], y), fmul2(sg, ffma2(z[i], rest, splat(1.0f))));
                o[i] = fmul2(o[i], fmul2(z[i], sg));  // dy
              }
            }
            float2 gb[4], qa[4], bias[4];
            unpack8(read8<T>(&s.raw[old][1][0][tid], kSsmHalf), v);
            pairs8(&s.f[buf][1][er][ec], gb), pairs8(&s.f[buf][2][er][ec], qa), pairs8(&s.sk[1][ec], bias);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 delta = *reinterpret_cast<const float2*>(&s.du[buf][er][(ec >> 1) + (i ^ turn)]);
              dd[i] = ffma2(x[i], gb[i], fmul2(qa[i], splat(kLn2)));
              if (p.softplus) dd[i] = fmul2(dd[i], sigmoid2(fadd2(v[i], bias[i])));
              dx[i] = ffma2(delta, gb[i], fmul2(skip[i], o[i]));
              sums[0][i] = ffma2(o[i], x[i], sums[0][i]);
              sums[1][i] = fadd2(sums[1][i], dd[i]);
            }
          }
          if (has_z) store8(static_cast<T*>(p.dz) + at, dz, en, out_vec);
          store8(static_cast<T*>(p.dx) + at, dx, en, out_vec);
          store8(static_cast<T*>(p.ddt) + at, dd, en, out_vec);
        }
        const float* d = &s.dbc[buf][0][br][bk];
#pragma unroll
        for (int k = 0; k < SUMS; ++k, d += ROWS * 2 * NP) {
          constexpr int W = kTokens * 2 * NP;  // from one warp's to the next one's
          const float v = (d[0] + d[W]) + (d[2 * W] + d[3 * W]);
          if (t + br + k * ROWS < w.t1) part_bc[(t + k * ROWS) * bc_row] = v;
        }
      }
      if (it < tiles) {
        const int t = w.t0 + (tiles - 1 - it) * kTokens;
        copies_done<0>();
        SeqBits seq{0u, 0u, 0u};
        if (SEQ) seq = seq_bits(*ids[buf], p, t);
        off0 = seq.pad;
        if (er < kTokens) {
          float4* const dst = &s.du[buf][er][ec >> 1];  // a pair's place within its vector is turned as in the forward
          float4* const dy = reinterpret_cast<float4*>(&s.f[buf][0][er][ec]);
          // Padding takes no step and has no input; neither has what lies outside the piece.
          if (work && t + er < w.t1 && !(SEQ && ((seq.pad >> er) & 1u))) {
            float2 x[4], d[4], o[4], bias[4];
            unpack8(read8<T>(&s.raw[ring][0][0][tid], kSsmHalf), x);
            unpack8(read8<T>(&s.raw[ring][1][0][tid], kSsmHalf), d);
            unpack8(read8<T>(&s.raw[ring][3][0][tid], kSsmHalf), o);
            pairs8(&s.sk[1][ec], bias);
            if (has_z) {
              float2 z[4];
              unpack8(read8<T>(&s.raw[ring][2][0][tid], kSsmHalf), z);
#pragma unroll
              for (int i = 0; i < 4; ++i) o[i] = fmul2(o[i], fmul2(z[i], sigmoid2(z[i])));
            }
            dy[0] = make_float4(o[0].x, o[0].y, o[1].x, o[1].y), dy[1] = make_float4(o[2].x, o[2].y, o[3].x, o[3].y);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float2 delta = fadd2(d[i], bias[i]);
              if (p.softplus) delta = softplus2(delta);
              const float2 u = fmul2(delta, x[i]);
              dst[i ^ turn] = make_float4(delta.x, delta.y, u.x, u.y);
            }
          } else {
            dy[0] = dy[1] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int i = 0; i < 4; ++i) dst[i] = make_float4(0.f, 0.f, 0.f, 0.f);
          }
        }
#pragma unroll
        for (int k = 0; k < NQ; ++k) {
          const int i = tid + k * kSsmHalf, tq = (i % QUADS) / NL;
          const bool in = t + tq < w.t1 && !(SEQ && ((seq.pad >> tq) & 1u));
          const float4 q = in ? unpack4(s.raw_bc[buf][k][tid]) : make_float4(0.f, 0.f, 0.f, 0.f);
          s.bc[buf][i / QUADS][tq][0][i % NL] = q;
          if (S::ORDERS == 2) s.bc[buf][i / QUADS][tq][S::ORDERS - 1][i % NL] = make_float4(q.z, q.w, q.x, q.y);
        }
        if (SEQ && tid == 0) s.start[buf] = seq.start;
        hand_over(full_barrier(buf));
        if (it + 1 < tiles) fetch(it + 1, next_stage(ring));
      }
    }

    // dD and ddt_bias of the CTA: over the threads of one column of vectors, in order. The walk is done
    // with the buffers (the last tile was taken over).
    float* col = &s.f[0][0][0][0];
    static_assert(sizeof(s.f) >= 8 * kSsmHalf * sizeof(float), "room for 8 values of each thread");
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      named_sync(7, kSsmHalf);
#pragma unroll
      for (int i = 0; i < 8; ++i) col[i * kSsmHalf + tid] = i % 2 ? sums[k][i / 2].y : sums[k][i / 2].x;
      named_sync(7, kSsmHalf);
      for (int c = tid; c < w.nc; c += kSsmHalf) {
        float v = 0.0f;
        for (int q = c / 8; q < kSsmHalf; q += VR) v += col[(c % 8) * kSsmHalf + q];
        p.part_d[((static_cast<int64_t>(w.b) * p.segs + w.seg) * 2 + k) * p.dim + w.c0 + c] = v;
      }
    }
  }

  // One tile of the walk. CUTS: a sequence starts in it (bits of `starts`).
  template <typename Cuts>
  static __device__ __forceinline__ void tile(S& s, int buf, uint32_t starts, const float2 (&A2)[2][2],
                                              float2 (&g)[2][2], float2 (&dA)[2][2], Cuts) {
    constexpr bool CUTS = Cuts::value;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nl = lane % NL;
    const int pair = warp * CL + lane / NL, lc = 2 * pair, place = (pair & ~3) | ((pair & 3) ^ (pair >> 3 & 3));
    const int turn = (lane & NL) ? 1 : 0;

    // B (k = 0) or C of token i, the lane's first pair of states first.
    auto four = [&](int k, int i, float2 (&v)[2]) {
      if constexpr (S::ORDERS == 2) {
        const float4 q = s.bc[buf][k][i][turn][nl];
        v[0] = make_float2(q.x, q.y), v[1] = make_float2(q.z, q.w);
      } else {
        const float2* q = reinterpret_cast<const float2*>(&s.bc[buf][k][i][0][nl]);
        v[0] = q[turn], v[1] = q[1 - turn];
      }
    };
    // One step of the recurrence; `a` gets the decays.
    auto advance = [&](int i, float2 (&h)[2][2], float2 (&a)[2][2]) {
      const float4 e = s.du[buf][i][place];
      float d[2] = {e.x, e.y};
      const float u[2] = {e.z, e.w};
      float2 B[2];
      four(0, i, B);
      if (CUTS && ((starts >> i) & 1u)) d[0] = d[1] = 0.0f, h[0][0] = h[0][1] = h[1][0] = h[1][1] = make_float2(0.f, 0.f);
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          a[c][m] = decay2<T>(splat(d[c]), A2[c][m]);
          h[c][m] = ffma2(a[c][m], h[c][m], fmul2(splat(u[c]), B[m]));
        }
    };
    // The states before run r.
    auto get = [&](int r, float2 (&h)[2][2]) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float4 q = r == 0 ? s.kept[buf][c][tid] : s.h[r - 1][c][tid];
        h[c][0] = make_float2(q.x, q.y), h[c][1] = make_float2(q.z, q.w);
      }
    };

    {
      float2 h[2][2], a[2][2];
      get(0, h);
#pragma unroll 1
      for (int r = 1; r < kTokens / kRun; ++r) {
#pragma unroll
        for (int j = 0; j < kRun; ++j) advance((r - 1) * kRun + j, h, a);
#pragma unroll
        for (int c = 0; c < 2; ++c) s.h[r - 1][c][tid] = make_float4(h[c][0].x, h[c][0].y, h[c][1].x, h[c][1].y);
      }
    }

#pragma unroll 1
    for (int r = kTokens / kRun - 1; r >= 0; --r) {
      float2 h[kRun + 1][2][2], a[kRun][2][2];
      get(r, h[0]);
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
#pragma unroll
        for (int c = 0; c < 2; ++c) h[j + 1][c][0] = h[j][c][0], h[j + 1][c][1] = h[j][c][1];
        advance(r * kRun + j, h[j + 1], a[j]);
      }
      float v[kRun / 2][12];  // [two tokens][token, channel, (y, sum g B, sum q A)]
      float e[kRun][8];       // [pair of states][dB, dC][state]
#pragma unroll
      for (int j = kRun - 1; j >= 0; --j) {
        const int i = r * kRun + j;
        const float4 e4 = s.du[buf][i][place];
        const float2 o2 = *reinterpret_cast<const float2*>(&s.f[buf][0][i][lc]);
        const float d[2] = {e4.x, e4.y}, u[2] = {e4.z, e4.w}, o[2] = {o2.x, o2.y};
        float2 B[2], C[2];
        four(0, i, B), four(1, i, C);
        const bool start = CUTS && ((starts >> i) & 1u);
        float2 dB[2], dC[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float2 y, gb, qa;
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            const float2 gt = ffma2(splat(o[c]), C[m], g[c][m]), ht = h[j + 1][c][m];
            y = m ? ffma2(ht, C[m], y) : fmul2(ht, C[m]);
            gb = m ? ffma2(gt, B[m], gb) : fmul2(gt, B[m]);
            dC[m] = c ? ffma2(splat(o[c]), ht, dC[m]) : fmul2(splat(o[c]), ht);
            dB[m] = c ? ffma2(splat(u[c]), gt, dB[m]) : fmul2(splat(u[c]), gt);
            float2 back = fmul2(a[j][c][m], gt);  // what the token before receives
            float2 q = fmul2(back, h[j][c][m]);
            if (start) back = q = make_float2(0.f, 0.f);
            qa = m ? ffma2(q, A2[c][m], qa) : fmul2(q, A2[c][m]);
            dA[c][m] = ffma2(q, splat(d[c]), dA[c][m]);
            g[c][m] = back;
          }
          float* vv = &v[j / 2][6 * (j % 2) + 3 * c];
          vv[0] = y.x + y.y, vv[1] = gb.x + gb.y, vv[2] = qa.x + qa.y;
        }
#pragma unroll
        for (int m = 0; m < 2; ++m)
          e[j][4 * m] = dB[m].x, e[j][4 * m + 1] = dB[m].y, e[j][4 * m + 2] = dC[m].x, e[j][4 * m + 3] = dC[m].y;
      }
      // The sums of the whole run together, so that the shuffles of one token do not wait for each other. The
      // lane across NL holds the pairs of states the other way round: its second is this lane's first.
#pragma unroll
      for (int j = 0; j < kRun; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) e[j][k] += __shfl_xor_sync(0xffffffffu, e[j][4 + k], NL);
      lane_sums_of<12, NL, 1>(v);
      lane_sums_of<4, CL / 2, 2 * NL>(e);
      static_assert(share_size<12, NL>() == 3, "each of four lanes gets three sums of a token's channel");
      __syncwarp();  // every lane has read the run's dy
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
        const int i = r * kRun + j, first = lane_share<4, CL / 2, 2 * NL>();
#pragma unroll
        for (int k = 0; k < share_size<4, CL / 2>(); ++k)
          s.dbc[buf][warp][i][((first + k) >> 1) * NP + 4 * nl + 2 * turn + ((first + k) & 1)] = e[j][k];
        if (j % 2 == 0 && nl < 4) {
          const int at = lane_share<12, NL, 1>() / 3;
          s.f[buf][0][i + at / 2][lc + at % 2] = v[j / 2][0];
          s.f[buf][1][i + at / 2][lc + at % 2] = v[j / 2][1];
          s.f[buf][2][i + at / 2][lc + at % 2] = v[j / 2][2];
        }
      }
    }
  }

  static __device__ __forceinline__ void walk(const SsmParams& p, const SsmPlace& w, S& s, int tiles) {
    const int tid = threadIdx.x, lane = tid & 31, n0 = 4 * (lane % NL);
    const int lc = 2 * ((tid >> 5) * CL + lane / NL);  // first of the lane's channels, within the block
    const int turn = (lane & NL) ? 1 : 0, n1 = n0 + 2 * turn, n2 = n0 + 2 - 2 * turn;  // first state of either pair
    auto state = [&](int m) { return (m < 2 ? n1 : n2) + (m & 1); };
    const int64_t row_bs = static_cast<int64_t>(w.b) * p.segs + w.seg;
    const int64_t kept_tiles = (p.seqlen + kSsmTile - 1) / kSsmTile;

    // The lane's states before the tile at t, as the forward kept them.
    auto fetch = [&](int t, int buf) {
      const int64_t kt = static_cast<int64_t>(w.b) * kept_tiles + t / kSsmTile;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if (lc + c < w.nc)
          for (int m = 0; m < 2; ++m)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(&s.kept[buf][c][tid]) + 8 * m),
                         "l"(p.kept + (kt * p.dim + w.c0 + lc + c) * NP + state(2 * m))
                         : "memory");
        else
          s.kept[buf][c][tid] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
      copies_issued();
    };
    fetch(w.t0 + (tiles - 1) * kTokens, 0);

    float2 A2[2][2], g[2][2], dA[2][2];
    const bool last = w.seg == p.segs - 1;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float a[4], v[4];
      const int ch = w.c0 + lc + c;
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const int n = state(m);
        const bool in = lc + c < w.nc && n < p.dstate;
        a[m] = in ? ld_any(p.A.ptr, static_cast<int64_t>(ch) * p.dstate + n, p.A.dtype) * kLog2e : 0.0f;
        v[m] = 0.0f;
        if (in && last && p.dfinal.ptr != nullptr)
          v[m] = ld_any(p.dfinal.ptr, (static_cast<int64_t>(w.b) * p.dim + ch) * p.dstate + n, p.dfinal.dtype);
      }
      A2[c][0] = make_float2(a[0], a[1]), A2[c][1] = make_float2(a[2], a[3]);
      g[c][0] = make_float2(v[0], v[1]), g[c][1] = make_float2(v[2], v[3]);
      dA[c][0] = dA[c][1] = make_float2(0.f, 0.f);
    }
    if (!last) piece_in(p, w, NP, w.c0 + lc, n1, n2, true, g);
#pragma unroll
    for (int c = 0; c < 2; ++c)
      if (lc + c >= w.nc) g[c][0] = g[c][1] = make_float2(0.f, 0.f);  // no channel: nothing for the sums over channels

#pragma unroll 1
    for (int it = 0; it < tiles; ++it) {
      const int t = w.t0 + (tiles - 1 - it) * kTokens, buf = it & 1;
      if (it + 1 < tiles) fetch(t - kTokens, buf ^ 1);
      else copies_issued();
      copies_done<1>();
      take_over(full_barrier(buf));
      const uint32_t starts = SEQ ? s.start[buf] : 0u;
      if (SEQ && starts != 0u) tile(s, buf, starts, A2, g, dA, std::true_type{});
      else tile(s, buf, 0u, A2, g, dA, std::false_type{});
      hand_over(done_barrier(buf));
    }

#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int ch = w.c0 + lc + c;
      if (lc + c < w.nc) {
#pragma unroll
        for (int m = 0; m < 2; ++m) *reinterpret_cast<float2*>(p.part_a + (row_bs * p.dim + ch) * NP + state(2 * m)) = dA[c][m];
        if (p.dinit != nullptr && w.seg == 0) {
          const float v[4] = {g[c][0].x, g[c][0].y, g[c][1].x, g[c][1].y};
#pragma unroll
          for (int m = 0; m < 4; ++m)
            if (state(m) < p.dstate)
              st_any(p.dinit, (static_cast<int64_t>(w.b) * p.dim + ch) * p.dstate + state(m), p.init.dtype, v[m]);
        }
      }
    }
  }
};

template <typename T, int NL, bool SEQ>
__global__ void __launch_bounds__(kThreads, 2) cc1d_ssm_bwd_kernel(const __grid_constant__ SsmParams p) {
  using K = Bwd<T, NL, SEQ>;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  typename K::S& s = *reinterpret_cast<typename K::S*>(smem_raw);
  const SsmPlace w = ssm_place<K::CH>(p);
  for (int i = threadIdx.x; i < 2 * K::CH; i += kThreads) {
    const int c = i % K::CH;
    const SsmParam& q = i < K::CH ? p.D : p.dt_bias;
    s.sk[i / K::CH][c] = c < w.nc && q.ptr != nullptr ? ld_any(q.ptr, w.c0 + c, q.dtype) : 0.0f;
  }
  __syncthreads();
  const int tiles = (w.t1 - w.t0 + kTokens - 1) / kTokens;
  if (threadIdx.x < kSsmHalf) {
    setmaxnreg_inc<kWalkRegs>();
    K::walk(p, w, s, tiles);
  } else {
    setmaxnreg_dec<kElementRegs>();
    K::elementwise(p, w, s, tiles);
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
#pragma unroll 8
    for (int q = 0; q < p.blocks; ++q) v += src[static_cast<int64_t>(q) * 2 * np];
    static_cast<T*>(which ? p.dC : p.dB)[row * p.dstate + n] = from_f<T>(v);
    return;
  }
  i -= n_bc;
  const int rows = p.batch * p.segs;
  if (i < n_a) {
    const float* src = p.part_a + i / p.dstate * np + i % p.dstate;
    float v = 0.0f;
#pragma unroll 8
    for (int q = 0; q < rows; ++q) v += src[static_cast<int64_t>(q) * p.dim * np];
    st_any(p.dA, i, p.A.dtype, v);
    return;
  }
  i -= n_a;
  if (i < 2ll * p.dim) {
    const int k = static_cast<int>(i / p.dim), ch = static_cast<int>(i % p.dim);
    float v = 0.0f;
#pragma unroll 8
    for (int q = 0; q < rows; ++q) v += p.part_d[(static_cast<int64_t>(q) * 2 + k) * p.dim + ch];
    if (k == 0 && p.dD != nullptr) st_any(p.dD, ch, p.D.dtype, v);
    if (k == 1 && p.ddt_bias != nullptr) st_any(p.ddt_bias, ch, p.dt_bias.dtype, v);
  }
}

template <typename T, int NL, bool SEQ>
cudaError_t launch_main(const SsmParams& p, cudaStream_t s) {
  constexpr int smem = static_cast<int>(sizeof(BwdSmem<T, NL>));
  const auto kernel = cc1d_ssm_bwd_kernel<T, NL, SEQ>;
  const cudaError_t e = allow_smem<cc1d_ssm_bwd_kernel<T, NL, SEQ>>(smem);
  if (e != cudaSuccess) return e;
  // setmaxnreg would wait for registers that a launch with fewer of them does not have.
  static const bool holds_split = [&] {
    cudaFuncAttributes a{};
    return cudaFuncGetAttributes(&a, kernel) == cudaSuccess && 2 * a.numRegs >= kWalkRegs + kElementRegs;
  }();
  if (!holds_split) return cudaErrorLaunchOutOfResources;
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
