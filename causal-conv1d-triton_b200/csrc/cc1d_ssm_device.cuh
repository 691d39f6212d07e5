// Device-side building blocks of the state-space kernels: the step's elementwise functions, token
// vectors of 8 channels, and sums across lanes that leave each lane with its own share.
#pragma once

#include <atomic>

#include "cc1d_device.cuh"
#include "cc1d_ssm.h"

namespace cc1d {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float2 splat(float v) { return make_float2(v, v); }

// 2^x, one MUFU operation. Measured against 64 bits over -16 < x < 0 it is at most 1.4e-7 off, and low on
// average: 5e-8 for x < -1, about 2e-8 between -2^-1 and -2^-8, 6e-9 from -2^-10 on.
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 exp2_approx2(float2 x) { return make_float2(exp2_approx(x.x), exp2_approx(x.y)); }

// x limited to [lo, hi]; a NaN stays one.
__device__ __forceinline__ float within(float x, float lo, float hi) {
  asm("max.NaN.f32 %0, %0, %1;\n\tmin.NaN.f32 %0, %0, %2;" : "+f"(x) : "f"(lo), "f"(hi));
  return x;
}

// 2^x = 2^i 2^f with i the nearest integer (found by adding and taking off 1.5 2^23) and 2^f, |f| <= 1/2, by
// its Taylor polynomial of degree 6 (ln2^k / k!, below 2e-7 off at |f| = 1/2 and exact to rounding for small
// f). Arguments below -126 give 2^-126, above 127.5 infinity. A NaN gives a NaN: it passes the limits, and the
// power of two, which means nothing then, is multiplied and not added to the exponent's bits.
__device__ __forceinline__ float2 exp2_exact2(float2 x) {
  x = make_float2(within(x.x, -126.0f, 128.0f), within(x.y, -126.0f, 128.0f));
  const float2 t = fadd2(x, splat(12582912.0f)), f = fadd2(x, fmul2(fadd2(t, splat(-12582912.0f)), splat(-1.0f)));
  float2 q = ffma2(f, splat(1.5403530e-4f), splat(1.3333558e-3f));
  q = ffma2(q, f, splat(9.6181291e-3f));
  q = ffma2(q, f, splat(5.5504109e-2f));
  q = ffma2(q, f, splat(2.4022651e-1f));
  q = ffma2(q, f, splat(6.9314718e-1f));
  q = ffma2(q, f, splat(1.0f));
  return fmul2(q, make_float2(__int_as_float((__float_as_int(t.x) << 23) + 0x3f800000),
                              __int_as_float((__float_as_int(t.y) << 23) + 0x3f800000)));
}

// The decay of a step, for operands of type T. A one-sided error adds up over as many tokens as a state
// remembers. The MUFU's is met by an addend to the exponent, which comes free with the product: with 2e-8 the mean
// is below 1.2e-8 either way for |x| < 2^-2 (a multiply-add rounds small arguments finely enough to keep it; 2^2e-8
// itself is 1, so that a step of 0 changes nothing). 3e-8 would leave less at 2^-7 and twice as much at 2^-10, where the
// memory is longest. dA of 4 x 2048 tokens is then 8.3e-7 off in norm (1.8e-6 without the addend; the same sums in
// 32 bits with a library exponential 9.8e-7), at the same speed. Operands in 32 bits take the polynomial, whose
// error has no side.
constexpr float kExp2Addend = 2e-8f;
template <typename T>
__device__ __forceinline__ float2 decay2(float2 delta, float2 A2) {
  if constexpr (sizeof(T) == 4) return exp2_exact2(fmul2(delta, A2));
  else return exp2_approx2(ffma2(delta, A2, splat(kExp2Addend)));
}

// log(1 + exp(v)) = max(v, 0) + log1p(w) with w = exp(-|v|) in (0, 1]. log1p(w) = 2 atanh(s) with
// s = w / (2 + w) <= 1/3, whose series 2 s (1 + s^2/3 + s^4/5 + ...) after seven terms is 3e-8 off
// at most (s = 1/3) and keeps its relative accuracy as w goes to 0, where the step size is small.
// A NaN comes through s.
__device__ __forceinline__ float2 softplus2(float2 v) {
  const float2 w = exp2_approx2(fmul2(make_float2(fabsf(v.x), fabsf(v.y)), splat(-kLog2e)));
  const float2 s = make_float2(__fdividef(w.x, 2.0f + w.x), __fdividef(w.y, 2.0f + w.y)), q = fmul2(s, s);
  float2 r = ffma2(q, splat(1.0f / 13), splat(1.0f / 11));
  r = ffma2(r, q, splat(1.0f / 9));
  r = ffma2(r, q, splat(1.0f / 7));
  r = ffma2(r, q, splat(1.0f / 5));
  r = ffma2(r, q, splat(1.0f / 3));
  r = ffma2(r, q, splat(1.0f));
  return ffma2(fadd2(s, s), r, make_float2(fmaxf(v.x, 0.0f), fmaxf(v.y, 0.0f)));
}
__device__ __forceinline__ float softplus(float v) { return softplus2(splat(v)).x; }

__device__ __forceinline__ float2 sigmoid2(float2 v) {
  const float2 w = exp2_approx2(fmul2(v, splat(-kLog2e))), d = fadd2(w, splat(1.0f));
  return make_float2(__fdividef(1.0f, d.x), __fdividef(1.0f, d.y));
}
__device__ __forceinline__ float sigmoid(float v) { return sigmoid2(splat(v)).x; }

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
__device__ __forceinline__ void unpack8(const Raw8<T>& r, float2 (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) v[i] = make_float2(__uint_as_float(r.w[2 * i]), __uint_as_float(r.w[2 * i + 1]));
    else v[i] = word_to_f2<T>(r.w[i]);
  }
}

// Rounds and stores channels [0, n) of 8.
template <typename T>
__device__ __forceinline__ void store8(T* dst, const float2 (&v)[4], int n, bool vec) {
  if (vec && n == 8) {
    constexpr int C = 16 / static_cast<int>(sizeof(T));
#pragma unroll
    for (int i = 0; i < 8; i += C) {
      float2 f[C / 2];
#pragma unroll
      for (int k = 0; k < C / 2; ++k) f[k] = v[i / 2 + k];
      store_vec<T, C>(dst + i, f);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (2 * i < n) dst[2 * i] = from_f<T>(v[i].x);
      if (2 * i + 1 < n) dst[2 * i + 1] = from_f<T>(v[i].y);
    }
  }
}
// 8 consecutive floats of shared memory at a multiple of 8.
__device__ __forceinline__ void pairs8(const float* src, float2 (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 q = reinterpret_cast<const float4*>(src)[i];
    v[2 * i] = make_float2(q.x, q.y), v[2 * i + 1] = make_float2(q.z, q.w);
  }
}

// States [n0, n0 + 4) of one token's B or C as loaded, zero at and beyond `n`.
template <typename T>
struct alignas(4 * sizeof(T)) Raw4 {
  static constexpr int NW = static_cast<int>(sizeof(T));
  uint32_t w[NW];
};
template <typename T>
__device__ __forceinline__ Raw4<T> zero4() {
  Raw4<T> r;
#pragma unroll
  for (int i = 0; i < Raw4<T>::NW; ++i) r.w[i] = 0u;
  return r;
}
template <typename T>
__device__ __forceinline__ Raw4<T> load4(const T* src, int n0, int n, bool vec) {
  Raw4<T> r;
  if (vec && n0 + 4 <= n) {
    if constexpr (sizeof(T) == 4) {
      const uint4 q = *reinterpret_cast<const uint4*>(src + n0);
      r.w[0] = q.x, r.w[1] = q.y, r.w[2] = q.z, r.w[3] = q.w;
    } else {
      const uint2 q = *reinterpret_cast<const uint2*>(src + n0);
      r.w[0] = q.x, r.w[1] = q.y;
    }
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = n0 + i < n ? reinterpret_cast<const uint32_t*>(src)[n0 + i] : 0u;
  } else {
    const uint16_t* s = reinterpret_cast<const uint16_t*>(src) + n0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t lo = n0 + 2 * i < n ? s[2 * i] : 0u, hi = n0 + 2 * i + 1 < n ? s[2 * i + 1] : 0u;
      r.w[i] = lo | (hi << 16);
    }
  }
  return r;
}
template <typename T>
__device__ __forceinline__ float4 unpack4(const Raw4<T>& r) {
  if constexpr (sizeof(T) == 4) {
    return make_float4(__uint_as_float(r.w[0]), __uint_as_float(r.w[1]), __uint_as_float(r.w[2]), __uint_as_float(r.w[3]));
  } else {
    const float2 a = word_to_f2<T>(r.w[0]), b = word_to_f2<T>(r.w[1]);
    return make_float4(a.x, a.y, b.x, b.y);
  }
}

// The same two through shared memory, as asynchronous copies of the calling thread's own vectors where
// these are aligned (each thread waits for and reads only its own). dst + i * stride is the vector's
// i-th 16-byte piece.
template <typename T>
__device__ __forceinline__ void copy8(uint4* dst, const T* src, int n, bool vec, int stride) {
  constexpr int Q = static_cast<int>(sizeof(T)) / 2;
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
__device__ __forceinline__ Raw8<T> read8(const uint4* src, int stride) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < Raw8<T>::NW / 4; ++i) {
    const uint4 q = src[i * stride];
    r.w[4 * i] = q.x, r.w[4 * i + 1] = q.y, r.w[4 * i + 2] = q.z, r.w[4 * i + 3] = q.w;
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void copy4(Raw4<T>* dst, const T* src, int n0, int n, bool vec) {
  if (vec && n0 + 4 <= n)
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(dst)), "l"(src + n0), "n"(4 * sizeof(T)) : "memory");
  else
    *dst = load4(src, n0, n, false);
}
__device__ __forceinline__ void copies_issued() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>  // waits for all groups but the last N
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

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

// The same for K sets of values side by side, stage by stage, so that their shuffles overlap.
template <int V, int L, int BIT, int K, int N>
__device__ __forceinline__ void lane_sums_of(float (&v)[K][N]) {
  if constexpr (L > 1) {
    if constexpr (V % 2 == 0) {
      const bool up = (threadIdx.x & BIT) != 0;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          const float send = up ? v[k][i] : v[k][i + V / 2];
          const float keep = up ? v[k][i + V / 2] : v[k][i];
          v[k][i] = keep + __shfl_xor_sync(0xffffffffu, send, BIT);
        }
      lane_sums_of<V / 2, L / 2, 2 * BIT>(v);
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) v[k][i] += __shfl_xor_sync(0xffffffffu, v[k][i], BIT);
      lane_sums_of<V, L / 2, 2 * BIT>(v);
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

// Raises a kernel's dynamic shared memory limit, once per device and kernel (one flag per template
// instance of the caller). Repeating it would be harmless; it costs a microsecond.
template <auto KERNEL>
cudaError_t allow_smem(int bytes) {
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (ready.load(std::memory_order_acquire) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) ready.fetch_or(bit, std::memory_order_release);
  return e;
}

// A CTA's two halves, a walk and the element-wise work around it, hand tiles to each other in
// kSsmStages buffers through two named barriers each: `full` (element-wise arrives, walk waits) and
// `done` (the reverse). Both halves pass the same ones for the same tiles, so every wait ends.
constexpr int kSsmHalf = 128;  // threads of each
constexpr int kSsmStages = 3;
__device__ __forceinline__ void hand_over(int id) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(2 * kSsmHalf) : "memory"); }
__device__ __forceinline__ void take_over(int id) { named_sync(id, 2 * kSsmHalf); }
__device__ __forceinline__ int full_barrier(int stage) { return 1 + stage; }
__device__ __forceinline__ int done_barrier(int stage) { return 1 + kSsmStages + stage; }
__device__ __forceinline__ int next_stage(int stage) { return stage + 1 == kSsmStages ? 0 : stage + 1; }

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
  w.t1 = w.t0 + min(p.seqlen - w.t0, p.seg_len);  // the last piece's t0 + seg_len may pass 2^31
  return w;
}

// What leaves a piece of decay d and own result o that receives `carry`. A piece in which a sequence starts,
// through which nothing passes, is marked by a negative decay: a decay itself may underflow to 0, after which a
// state is still infinite or NaN if it was before, and overflow (A > 0), after which a zero is still zero.
// fmaf(d, carry, o) alone is right unless it gives a NaN.
constexpr float kSsmCut = -1.0f;
__device__ __forceinline__ float pass_piece(float d, float carry, float o) {
  if (d < 0.0f || carry == 0.0f) return o;
  return fmaf(d == 0.0f && isinf(carry) ? 1.0f : d, carry, o);
}

// What piece w.seg of the sequence receives, into h: of channels ch and ch + 1 the pairs of states that
// start at n1 and n2. From the join kernel, or, with few pieces, by the same chain over the pieces before
// (after) it, whose loads are independent of it.
__device__ __forceinline__ void piece_in(const SsmParams& p, const SsmPlace& w, int np, int ch, int n1, int n2, bool backward,
                                         float2 (&h)[2][2]) {
  const int64_t row = static_cast<int64_t>(p.dim) * np;
  int64_t at[2][2];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    // A channel past the last one reads the last one's.
    const int64_t q = w.b * p.segs * row + static_cast<int64_t>(min(ch + c, p.dim - 1)) * np;
    at[c][0] = q + n1, at[c][1] = q + n2;
  }
  auto read = [&](const float* base, int seg, float2 (&v)[2][2]) {
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int m = 0; m < 2; ++m) v[c][m] = *reinterpret_cast<const float2*>(base + at[c][m] + seg * row);
  };
  if (!p.fold) return read(p.seg_in, w.seg, h);
  const int from = backward ? p.segs - 1 : 0, step = backward ? -1 : 1, n = backward ? p.segs - 1 - w.seg : w.seg;
  read(p.seg_out, from, h);
#pragma unroll 4
  for (int i = 1; i < n; ++i) {
    float2 o[2][2], d[2][2];
    read(p.seg_out, from + i * step, o), read(p.seg_decay, from + i * step, d);
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        h[c][m].x = d[c][m].x < 0.0f ? o[c][m].x : fmaf(d[c][m].x, h[c][m].x, o[c][m].x);
        h[c][m].y = d[c][m].y < 0.0f ? o[c][m].y : fmaf(d[c][m].y, h[c][m].y, o[c][m].y);
      }
  }
  // A NaN may be one of 0 times infinity: then the chain once more, by pass_piece (whose tests at every step
  // cost a chain of 15 pieces 2 us, and its branches, which keep loads from being issued early, 7).
  bool nan = false;
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int m = 0; m < 2; ++m) nan = nan || isnan(h[c][m].x) || isnan(h[c][m].y);
  if (nan) {
    read(p.seg_out, from, h);
#pragma unroll 1
    for (int i = 1; i < n; ++i) {
      float2 o[2][2], d[2][2];
      read(p.seg_out, from + i * step, o), read(p.seg_decay, from + i * step, d);
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          h[c][m].x = pass_piece(d[c][m].x, h[c][m].x, o[c][m].x);
          h[c][m].y = pass_piece(d[c][m].y, h[c][m].y, o[c][m].y);
        }
    }
  }
}

// Tokens of a tile (bit i: token t + i of row b) whose state starts from zero because the sequence id
// differs from the token before (the row's first token continues initial_states), the padding ones,
// and the last ones of their sequence. From lane i's ids of token t + i and its neighbours, loaded
// early; whole warps call it.
struct SeqIds {
  int32_t prev, cur, next;
};
struct SeqBits {
  uint32_t start, pad, last;
};
__device__ __forceinline__ void copy_ids(SeqIds* dst, const SsmParams& p, int b, int t) {
  const int i = t + static_cast<int>(threadIdx.x & 31);
  if ((threadIdx.x & 31) < kSsmTile && i < p.seqlen) {
    const int32_t* s = p.seq_idx + static_cast<int64_t>(b) * p.seqlen + i;
    const int32_t* from[3] = {i > 0 ? s - 1 : s, s, i + 1 < p.seqlen ? s + 1 : s};
    int32_t* to[3] = {&dst->prev, &dst->cur, &dst->next};
#pragma unroll
    for (int k = 0; k < 3; ++k)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(to[k])), "l"(from[k]) : "memory");
  }
}
__device__ __forceinline__ SeqBits seq_bits(const SeqIds& id, const SsmParams& p, int t) {
  const int lane = threadIdx.x & 31, i = t + lane;
  const bool in = lane < kSsmTile && i < p.seqlen;
  SeqBits r;
  r.start = __ballot_sync(0xffffffffu, in && id.prev != id.cur);
  r.pad = __ballot_sync(0xffffffffu, in && id.cur < 0);
  r.last = __ballot_sync(0xffffffffu, in && id.cur >= 0 && (i + 1 == p.seqlen || id.next != id.cur));
  return r;
}

}  // namespace cc1d
