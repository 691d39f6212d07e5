// Internal: launch parameters of the state-space kernels (cc1d_ssm_fwd.cu, cc1d_ssm_bwd.cu,
// cc1d_ssm_update.cu), filled by the C entry points in cc1d_ssm_api.cu.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace cc1d {

constexpr int kSsmTile = 16;      // tokens between two kept states (and of one backward tile)
constexpr int kSsmMaxState = 64;  // states per channel: 4 per lane, at most 16 lanes per channel

// A (batch, seqlen, channels) operand: element (b, t, c) at ptr + b * sb + t * st + c. `vec` says
// that every run of 8 channels starting at a multiple of 8 (of 4 states, for B and C) of a group is
// one aligned vector.
struct SsmTokens {
  const void* ptr;
  int64_t sb, st, sg;  // sg: stride of the group (B and C)
  int vec;
};

// A parameter whose element type is given at run time.
struct SsmParam {
  const void* ptr;
  int dtype;
};

struct SsmParams {
  SsmTokens x, dt, z, Bm, Cm;  // z.ptr null: no gate
  SsmParam A, D, dt_bias;      // (dim, dstate), (dim), (dim); D and dt_bias may be null
  SsmParam init;               // (batch, dim, dstate) or null
  const int32_t* seq_idx;      // (batch, seqlen) or null
  int batch, seqlen, dim, dstate, groups, group_dim;
  int softplus;
  int segs, seg_len;  // the sequence in `segs` pieces of `seg_len` tokens (a multiple of 32)
  int blocks;         // CTAs that cover one group's channels
  int out_vec;        // out (backward: dx, ddt and dz) and the rows in it start at multiples of 16 bytes
  // Forward
  void* out;                   // (batch, seqlen, dim) contiguous, type of x
  float* final_states;         // (batch, dim, dstate) or null
  float* kept;                 // (batch, ceil(seqlen / kSsmTile), dim, 4 NL): state before each tile, or null
  void* cache;                 // (slots, dim, dstate): state after each packed sequence, or null
  int cache_dtype;
  const int32_t* cache_idx;    // (batch, cache_n) slot of each sequence id
  int64_t cache_n, cache_slots;  // ids per row that cache_idx covers; rows of cache (a slot outside is skipped)
  // Sequences in pieces, (batch, segs, dim, 4 NL) each: the state (gradient) that a piece leaves when it
  // receives none, its decay, and what it receives.
  float *seg_out, *seg_decay, *seg_in;
  int fold;  // no join kernel ran: each piece works out what it receives
  // Backward
  SsmTokens dout;
  SsmParam dfinal;             // (batch, dim, dstate) or null
  void *dx, *ddt, *dz;         // (batch, seqlen, dim) contiguous, type of x
  void *dB, *dC;               // (batch, seqlen, groups, dstate) contiguous, type of x
  void *dA, *dD, *ddt_bias;    // types of A, D, dt_bias; null where those are
  void* dinit;                 // type of init, or null
  float* part_bc;              // (batch, seqlen, groups, blocks, 2, 4 NL): dB and dC over one CTA's channels
  float* part_a;               // (batch, segs, dim, 4 NL)
  float* part_d;               // (batch, segs, 2, dim): dD, ddt_bias
};

struct SsmUpdateParams {
  SsmTokens x, dt, z, Bm, Cm;
  SsmParam A, D, dt_bias;
  void* state;             // (slots, dim, dstate), updated in place
  int64_t slots;           // rows of state
  int state_dtype;
  int x_dtype;
  const int32_t* indices;  // (batch) slot of each row, or null
  void* out;               // (batch, seqlen, dim) contiguous
  int batch, seqlen, dim, dstate, group_dim;
  int softplus;
  int sms;                 // of the device
  int blocks;              // set by the launcher: CTAs over the channels
};

int record_cuda_error(cudaError_t e);  // sets cc1d_last_cuda_error(), returns CC1D_ERR_CUDA

// Lanes of a warp that share a channel, 4 states each: 4, 8 or 16. Fewer than 13 states run as 16
// with zeros.
inline int ssm_lanes(int dstate) { return dstate <= 16 ? 4 : dstate <= 32 ? 8 : 16; }
// Channels of a CTA: 128 threads of two channels each, NL of them alike.
inline int ssm_channels(int nl) { return 256 / nl; }

enum SsmPass : int { kSsmForward = 0, kSsmPieceForward = 1, kSsmPieceBackward = 2 };

cudaError_t launch_ssm_scan(const SsmParams& p, SsmPass pass, int x_dtype, cudaStream_t s);
cudaError_t launch_ssm_join(const SsmParams& p, bool backward, cudaStream_t s);
cudaError_t launch_ssm_bwd(const SsmParams& p, int x_dtype, cudaStream_t s);
cudaError_t launch_ssm_update(const SsmUpdateParams& p, cudaStream_t s);

}  // namespace cc1d
