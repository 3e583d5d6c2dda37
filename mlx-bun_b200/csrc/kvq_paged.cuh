#pragma once
// kvq_paged.cuh — the paged quantized cache's geometry, shared by its append
// and attention kernels.
//
// Why a tile of 16 rows with K and V together: the attention kernels work on
// 16 key rows at a time (one MMA tile) and need their K and V codes, scales
// and biases, so one bulk copy of one contiguous block brings everything, and
// consecutive tiles of a page are one longer block.  A (scale, bias) pair is
// one 32-bit word, read with one load.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kvq_internal.h"

namespace kvq {
namespace paged {

constexpr int kTileRows = 16;

// What a kernel knows about the pool and the step's batch.
struct View {
  uint8_t* pool;
  int* status;
  int num_pages, page_shift, page_mask;  // page_size = 1 << page_shift
  int tiles_shift;                       // tiles per page = 1 << tiles_shift
  int Hkv, D, bits, gs;
  int tile_bytes;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* seq_lens;
  const int32_t* cu;  // nullable: one row per sequence
  int B, max_pages, rows;
};

// Bytes of the parts of a tile.
__host__ __device__ inline int code_row_bytes(int D, int bits) { return D * bits / 8; }
__host__ __device__ inline int pair_row_bytes(int D, int gs) { return D / gs * 4; }
__host__ __device__ inline int half_tile_bytes(int D, int bits, int gs) {
  return kTileRows * (code_row_bytes(D, bits) + pair_row_bytes(D, gs));
}

__device__ __forceinline__ uint8_t* tile_ptr(const View& v, int page, int h, int tile) {
  return v.pool + ((((int64_t)page * v.Hkv + h) << v.tiles_shift) + tile) * v.tile_bytes;
}

// The pool's error flag: a row, page or length that makes no sense (1), a bounded
// wait that ran out (2).
__device__ __forceinline__ void raise(const View& v) { atomicOr(v.status, 1); }
__device__ __forceinline__ void gave_up(const View& v) { atomicOr(v.status, 2); }

// Rows of sequence b, `n` of them from `row0`, and its length.
__device__ __forceinline__ void seq_rows(const View& v, int b, int& row0, int& n, int& len) {
  row0 = v.cu ? v.cu[b] : b;
  n = v.cu ? v.cu[b + 1] - row0 : 1;
  len = v.seq_lens[b];
}

// Host launchers.
struct RopeArgs {
  int dims, half;
  bool traditional;
  double base, scale, pre;
  const float* freqs;
};
struct AppendArgs {
  View v;
  const uint16_t *k, *q, *val;
  int64_t k_row, k_head, v_row, v_head, q_row, q_head;
  uint16_t* q_out;
  int Hq;
  RopeArgs rope;
  bool bf16;
};
int32_t launch_paged_append(const AppendArgs& a, cudaStream_t st);

struct AttnArgs {
  View v;
  const uint16_t* q;
  int64_t q_row, q_head;
  uint16_t* out;
  int out_align;  // rows start at 16-byte (2), 4-byte (1) or element (0) borders
  int Hq, rep;
  float scale;
  int window, sinks;
  bool bf16;
};
size_t paged_attn_workspace(const AttnArgs& a);
int32_t launch_paged_attn(const AttnArgs& a, void* ws, size_t ws_bytes, cudaStream_t st);

}  // namespace paged
}  // namespace kvq
