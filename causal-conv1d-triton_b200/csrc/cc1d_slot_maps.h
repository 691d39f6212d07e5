// Internal: launch parameters of the slot-map kernels (cc1d_slot_maps.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace cc1d {

struct SlotMapParams {
  const int32_t *lengths, *past, *slots, *free_slots;  // past and slots may be null
  int32_t *cu_seqlens, *seq_idx, *positions, *tail_rows, *slots_out, *n_taken;
  int n, seqlen, width;
  int vec;  // seq_idx and positions start at multiples of 16 bytes
  int64_t n_free;
};

cudaError_t launch_slot_maps(const SlotMapParams& p, cudaStream_t s);

}  // namespace cc1d
