// Maps of a serving step, built on the device from the requests' lengths: where each request lies in
// the packed row, each token's request and position, the rows that a convolution keeps of each
// request, and the state slots, new ones handed out from a free list in request order.
//
// Latency decides at every size that a step has (8 bytes a token; 1 MB at 131072 tokens), so there is one launch:
// every CTA computes the requests' edges for itself in shared memory (a block-wide sum over lengths
// that are in L2 after the first CTA) and writes its own 1024 tokens. Above kInOne requests the edges
// do not fit, and a first kernel of one CTA writes them for a second to search.
#include <cuda_runtime.h>
#include <stdint.h>

#include "cc1d_slot_maps.h"

namespace cc1d {
namespace {

constexpr int kThreads = 256, kPer = 16, kInOne = kThreads * kPer, kTokensPerCta = 4 * kThreads;

// Inclusive sum over the CTA's threads, in thread order; `total` gets the whole sum.
template <int THREADS>
__device__ __forceinline__ int64_t block_sum(int64_t v, int64_t* total, int64_t* shared) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) shared[warp] = v;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) {
    if (i < warp) before += shared[i];
    all += shared[i];
  }
  __syncthreads();
  *total = all;
  return v + before;
}

// One request's edges, and its slot; `end` is past its last token, `rank` counts the new requests before it.
__device__ __forceinline__ int32_t clip(int64_t v, int seqlen) { return static_cast<int32_t>(v < seqlen ? v : seqlen); }
__device__ __forceinline__ bool wants_slot(const SlotMapParams& p, int r, int32_t len) {
  return p.slots != nullptr && p.slots[r] < 0 && len > 0;
}
__device__ __forceinline__ void put_slot(const SlotMapParams& p, int r, bool fresh, int64_t rank) {
  if (p.slots != nullptr) p.slots_out[r] = !fresh ? p.slots[r] : (rank < p.n_free ? p.free_slots[rank] : -1);
}

// seq_idx and positions of 4 tokens from `pos`, and this thread's share of the kept rows.
__device__ __forceinline__ void put_tokens(const SlotMapParams& p, const int32_t* edges, int64_t thread, int64_t threads) {
  const int64_t pos = 4 * thread;
  if (pos < p.seqlen) {
    int lo = 0, hi = p.n;  // the first request whose end is past pos
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (edges[mid + 1] <= pos) lo = mid + 1;
      else hi = mid;
    }
    int32_t id[4], at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      while (lo < p.n && edges[lo + 1] <= pos + i) ++lo;
      id[i] = lo < p.n ? lo : -1;
      at[i] = lo < p.n ? static_cast<int32_t>(pos + i) - edges[lo] + (p.past != nullptr ? p.past[lo] : 0) : -1;
    }
    if (p.vec && pos + 4 <= p.seqlen) {
      *reinterpret_cast<int4*>(p.seq_idx + pos) = make_int4(id[0], id[1], id[2], id[3]);
      *reinterpret_cast<int4*>(p.positions + pos) = make_int4(at[0], at[1], at[2], at[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (pos + i < p.seqlen) p.seq_idx[pos + i] = id[i], p.positions[pos + i] = at[i];
    }
  }
  const int rows = p.width - 1;
  for (int64_t i = thread; i < static_cast<int64_t>(p.n) * rows; i += threads) {
    const int r = static_cast<int>(i / rows), row = edges[r + 1] - rows + static_cast<int>(i % rows);
    p.tail_rows[i] = row >= edges[r] ? row : -1;
  }
}

__global__ void __launch_bounds__(kThreads) cc1d_slot_maps_kernel(const __grid_constant__ SlotMapParams p) {
  __shared__ int32_t edges[kInOne + 1];
  __shared__ int64_t shared[kThreads / 32];
  const int tid = threadIdx.x, per = (p.n + kThreads - 1) / kThreads, r0 = tid * per;
  int64_t sum = 0, fresh = 0, total;
  for (int r = r0; r < min(r0 + per, p.n); ++r) {
    const int32_t len = max(p.lengths[r], 0);
    sum += len;
    if (blockIdx.x == 0) fresh += wants_slot(p, r, len);
  }
  int64_t end = block_sum<kThreads>(sum, &total, shared) - sum;
  for (int r = r0; r < min(r0 + per, p.n); ++r) {
    edges[r] = clip(end, p.seqlen);
    end += max(p.lengths[r], 0);
  }
  if (tid == 0) edges[p.n] = clip(total, p.seqlen);
  if (blockIdx.x == 0) {
    int64_t rank = block_sum<kThreads>(fresh, &total, shared) - fresh;
    for (int r = r0; r < min(r0 + per, p.n); ++r) {
      const bool is = wants_slot(p, r, max(p.lengths[r], 0));
      put_slot(p, r, is, rank);
      rank += is;
    }
    if (tid == 0) *p.n_taken = static_cast<int32_t>(total);
  }
  __syncthreads();
  if (blockIdx.x == 0)
    for (int r = tid; r <= p.n; r += kThreads) p.cu_seqlens[r] = edges[r];
  put_tokens(p, edges, static_cast<int64_t>(blockIdx.x) * kThreads + tid, static_cast<int64_t>(gridDim.x) * kThreads);
}

__global__ void __launch_bounds__(1024) cc1d_slot_edges_kernel(const __grid_constant__ SlotMapParams p) {
  __shared__ int64_t shared[32];
  int64_t end = 0, rank = 0, total;
  for (int base = 0; base < p.n; base += 1024) {
    const int r = base + threadIdx.x;
    const int32_t len = r < p.n ? max(p.lengths[r], 0) : 0;
    const int64_t e = end + block_sum<1024>(len, &total, shared);
    end += total;
    if (r < p.n) p.cu_seqlens[r] = clip(e - len, p.seqlen);
    const bool is = r < p.n && wants_slot(p, r, len);
    const int64_t k = rank + block_sum<1024>(is, &total, shared) - is;
    rank += total;
    if (r < p.n) put_slot(p, r, is, k);
  }
  if (threadIdx.x == 0) p.cu_seqlens[p.n] = clip(end, p.seqlen), *p.n_taken = static_cast<int32_t>(rank);
}

__global__ void __launch_bounds__(kThreads) cc1d_slot_tokens_kernel(const __grid_constant__ SlotMapParams p) {
  put_tokens(p, p.cu_seqlens, static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x,
             static_cast<int64_t>(gridDim.x) * kThreads);
}

}  // namespace

cudaError_t launch_slot_maps(const SlotMapParams& p, cudaStream_t s) {
  const int64_t ctas = (static_cast<int64_t>(p.seqlen) + kTokensPerCta - 1) / kTokensPerCta;
  const unsigned grid = static_cast<unsigned>(ctas < 1 ? 1 : ctas);
  if (p.n <= kInOne) {
    cc1d_slot_maps_kernel<<<grid, kThreads, 0, s>>>(p);
  } else {
    cc1d_slot_edges_kernel<<<1, 1024, 0, s>>>(p);
    cc1d_slot_tokens_kernel<<<grid, kThreads, 0, s>>>(p);
  }
  return cudaGetLastError();
}

}  // namespace cc1d
