// Device-side building blocks of the state-space kernels: the step's elementwise functions, token
// vectors of 8 channels, and sums across lanes that leave each lane with its own share.
#pragma once

#include "cc1d_device.cuh"
#include "cc1d_ssm.h"

namespace cc1d {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// 2^x, one MUFU operation (measured against 64 bits over -16 < x < 0: at most 1.5e-7 off).
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 exp2_approx2(float2 x) { return make_float2(exp2_approx(x.x), exp2_approx(x.y)); }

__device__ __forceinline__ float2 splat(float v) { return make_float2(v, v); }

// log(1 + exp(v)) = max(v, 0) + log1p(w) with w = exp(-|v|) in (0, 1]. log1p(w) = 2 atanh(s) with
// s = w / (2 + w) <= 1/3, whose series 2 s (1 + s^2/3 + s^4/5 + ...) after seven terms is 3e-8 off
// at most (s = 1/3) and keeps its relative accuracy as w goes to 0, where the step size is small.
__device__ __forceinline__ float softplus(float v) {
  const float w = __expf(-fabsf(v));
  const float s = __fdividef(w, 2.0f + w), q = s * s;
  float r = fmaf(q, 1.0f / 13, 1.0f / 11);
  r = fmaf(r, q, 1.0f / 9);
  r = fmaf(r, q, 1.0f / 7);
  r = fmaf(r, q, 1.0f / 5);
  r = fmaf(r, q, 1.0f / 3);
  r = fmaf(r, q, 1.0f);
  return fmaf(s + s, r, fmaxf(v, 0.0f));  // NaN: through s
}

__device__ __forceinline__ float sigmoid(float v) { return __fdividef(1.0f, 1.0f + __expf(-v)); }

// 8 channels of one token as loaded, before conversion: a thread keeps the next tile's in registers.
template <typename T>
struct Raw8 {
  static constexpr int NW = 2 * static_cast<int>(sizeof(T));
  uint32_t w[NW];
};

// Loads channels [0, n) of `src` (n <= 8), zero beyond. `vec`: src + 8 channels is one aligned vector.
template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T* src, int n, bool vec) {
  Raw8<T> r;
  if (vec && n == 8) {
#pragma unroll
    for (int i = 0; i < Raw8<T>::NW; i += 4) {
      const uint4 q = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(src) + i);
      r.w[i] = q.x, r.w[i + 1] = q.y, r.w[i + 2] = q.z, r.w[i + 3] = q.w;
    }
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.w[i] = i < n ? reinterpret_cast<const uint32_t*>(src)[i] : 0u;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint16_t* s = reinterpret_cast<const uint16_t*>(src);
      const uint32_t lo = 2 * i < n ? s[2 * i] : 0u, hi = 2 * i + 1 < n ? s[2 * i + 1] : 0u;
      r.w[i] = lo | (hi << 16);
    }
  }
  return r;
}

template <typename T>
__device__ __forceinline__ Raw8<T> zero8() {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < Raw8<T>::NW; ++i) r.w[i] = 0u;
  return r;
}

template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r.w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = word_to_f2<T>(r.w[i]);
      v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
  }
}

// Rounds and stores channels [0, n) of 8.
template <typename T>
__device__ __forceinline__ void store8(T* dst, const float (&v)[8], int n, bool vec) {
  if (vec && n == 8) {
#pragma unroll
    for (int i = 0; i < 8; i += 16 / static_cast<int>(sizeof(T))) {
      constexpr int C = 16 / static_cast<int>(sizeof(T));
      float2 f[C / 2];
#pragma unroll
      for (int k = 0; k < C / 2; ++k) f[k] = make_float2(v[i + 2 * k], v[i + 2 * k + 1]);
      store_vec<T, C>(dst + i, f);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) dst[i] = from_f<T>(v[i]);
  }
}

// States [n0, n0 + 4) of one token's B or C, zero at and beyond `n`.
template <typename T>
__device__ __forceinline__ float4 load4(const T* src, int n0, int n, bool vec) {
  if (vec && n0 + 4 <= n) {
    float2 f[2];
    load_vec<T, 4>(src + n0, f);
    return make_float4(f[0].x, f[0].y, f[1].x, f[1].y);
  }
  float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
  if (n0 < n) r.x = to_f<T>(src[n0]);
  if (n0 + 1 < n) r.y = to_f<T>(src[n0 + 1]);
  if (n0 + 2 < n) r.z = to_f<T>(src[n0 + 2]);
  if (n0 + 3 < n) r.w = to_f<T>(src[n0 + 3]);
  return r;
}

// Sums v[0..V) over the L lanes of a warp that differ in lane bits BIT, 2 BIT, ... While the number
// of values is even, a stage halves it: each lane sends the half that its partner keeps, so V values
// over L lanes cost about V (1 - 1/L) shuffles instead of V log2 L. A lane with bit BIT set ends with
// the upper half, and so on; once one value (or an odd number) is left, all lanes get the sum.
// Returns how many values are left, in v[0..).
template <int V, int L, int BIT, int N>
__device__ __forceinline__ void lane_sums(float (&v)[N]) {
  if constexpr (L > 1) {
    if constexpr (V % 2 == 0) {
      const bool up = (threadIdx.x & BIT) != 0;
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const float send = up ? v[i] : v[i + V / 2];
        const float keep = up ? v[i + V / 2] : v[i];
        v[i] = keep + __shfl_xor_sync(0xffffffffu, send, BIT);
      }
      lane_sums<V / 2, L / 2, 2 * BIT>(v);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], BIT);
      lane_sums<V, L / 2, 2 * BIT>(v);
    }
  }
}

// Position of this lane's share among the V values that lane_sums started from, and its length.
template <int V, int L, int BIT>
__device__ __forceinline__ int lane_share() {
  if constexpr (L > 1 && V % 2 == 0)
    return ((threadIdx.x & BIT) ? V / 2 : 0) + lane_share<V / 2, L / 2, 2 * BIT>();
  else
    return 0;
}
template <int V, int L>
constexpr int share_size() {
  if constexpr (L > 1 && V % 2 == 0)
    return share_size<V / 2, L / 2>();
  else
    return V;
}
// Stages of lane_sums that halved (lanes that differ only in later bits hold the same share).
template <int V, int L>
constexpr int share_lanes() {
  if constexpr (L > 1 && V % 2 == 0)
    return 2 * share_lanes<V / 2, L / 2>();
  else
    return 1;
}

// What a CTA works on: batch row, piece of the sequence, group and its block of channels. The
// channel blocks of one piece are neighbours in the grid, so that they share its B and C in L2.
struct SsmPlace {
  int b, seg, g, blk;
  int c0, nc;  // first channel, and channels of the block
  int t0, t1;  // tokens
};
template <int CH>
__device__ __forceinline__ SsmPlace ssm_place(const SsmParams& p) {
  SsmPlace w;
  unsigned i = blockIdx.x;
  w.blk = i % p.blocks, i /= p.blocks;
  w.g = i % p.groups, i /= p.groups;
  w.seg = i % p.segs;
  w.b = i / p.segs;
  w.c0 = w.g * p.group_dim + w.blk * CH;
  w.nc = min(CH, p.group_dim - w.blk * CH);
  w.t0 = w.seg * p.seg_len;
  w.t1 = min(p.seqlen, w.t0 + p.seg_len);
  return w;
}

// The 32 tokens from t (bit i: token t + i) of row b: those whose state starts from zero because the
// sequence id differs from the token before (the row's first token continues initial_states),
// the padding ones, and the last ones of their sequence.
struct SeqBits {
  uint32_t start, pad, last;
};
__device__ __forceinline__ SeqBits seq_bits(const SsmParams& p, int b, int t) {
  SeqBits r{0u, 0u, 0u};
  if (p.seq_idx != nullptr) {
    const int32_t* s = p.seq_idx + static_cast<int64_t>(b) * p.seqlen;
    const int i = t + static_cast<int>(threadIdx.x & 31);
    const bool in = i < p.seqlen;
    const int cur = in ? s[i] : -1;
    const int prev = in && i > 0 ? s[i - 1] : cur;
    const int next = i + 1 < p.seqlen ? s[i + 1] : -1;
    r.start = __ballot_sync(0xffffffffu, in && prev != cur);
    r.pad = __ballot_sync(0xffffffffu, in && cur < 0);
    r.last = __ballot_sync(0xffffffffu, in && cur >= 0 && (i + 1 == p.seqlen || next != cur));
  }
  return r;
}

}  // namespace cc1d
