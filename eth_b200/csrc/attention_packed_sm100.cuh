// C++ launchers of the packed-document flash attention kernels (see attention_packed_sm100.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace ethb {

// One unit of work: `tile` counts 128-row tiles (256-row blocks in the forward table of single
// heads) inside the document that starts at row `start` and has `len` rows.
struct PackedTile {
  int start, len, tile, reserved;
};

// q/o (and their gradients) are [rows, heads, head_dim] views, k/v [rows, kv_heads, head_dim], with
// head_dim contiguous; strides[] = element strides of (row, head). head_dim is 64 or 128, heads a
// multiple of kv_heads. Rows from `used` on belong to no document: outputs, lse and gradients there are 0.
struct PackedAttnArgs {
  int rows, used, heads, kv_heads, head_dim;
  const void *q, *k, *v;
  void* o;
  const void* d_o;
  void *dq, *dk, *dv;
  int64_t q_strides[2], k_strides[2], v_strides[2], o_strides[2];
  int64_t do_strides[2], dq_strides[2], dk_strides[2], dv_strides[2];
  float* lse;       // [heads, rows]  log-sum-exp of the scaled scores (natural log)
  float* delta;     // [heads, rows]  rowsum(dO * O), written by the backward
  void* residue;    // [rows, heads, head_dim] contiguous, type of q, or null: what rounding took off `o`
  const PackedTile* tiles;       // forward: work list, heaviest first
  int num_tiles;
  const PackedTile* q_tiles;     // backward: query tiles / key tiles, heaviest first
  int num_q_tiles;
  const PackedTile* k_tiles;
  int num_k_tiles;
  int* counters;                 // backward: two ints of scratch
  int splits;                    // backward: attention_packed_splits
  float* parts;                  // backward, splits > 1: fp32 [splits, 2, used, kv_heads, head_dim] of scratch
  float scale;
  int causal;
  int dtype;        // kF16 / kBF16
  int* status;
};

// true: the forward pairs two heads of a group on one 128-row tile, false: two tiles of one head
bool attention_packed_pairs_heads(int heads, int kv_heads);
// Into how many parts (a divisor of the group) the heads of a group are split in the dK / dV kernel: enough
// for two and a half units of work per SM, so that the heaviest does not decide the time. About 4000 tokens in 40
// documents, 16 / 2 heads of 64: 44 us without splitting, 30 and 4 us for the join with it (26 and 4 by now). With
// units enough the parts' traffic (8 bytes an element and part each way) is not worth it.
int attention_packed_splits(int num_k_tiles, int heads, int kv_heads);
cudaError_t attention_packed_fwd(const PackedAttnArgs& a, cudaStream_t st);
cudaError_t attention_packed_bwd(const PackedAttnArgs& a, cudaStream_t st);

}  // namespace ethb
