// C launch interface of the operators on packed documents: causal attention over documents that lie
// one behind the other in a token axis, and the rotary embedding at each document's own positions.
#pragma once

#include <cuda_runtime.h>

extern "C" {

// Operands shared by the forward and the backward pass.  Token t of head h starts at
// base + t * <x>_tok + h * <x>_head (elements); the features of a head are contiguous.
typedef struct {
  const void* q;  // [rows, heads, dim]
  const void* k;  // [rows, kv_heads, dim]
  const void* v;  // [rows, kv_heads, dim]
  long q_tok, q_head, k_tok, k_head, v_tok, v_head;
  const int* first_key;    // [rows]: first key that row t attends (its document's first token); t + 1: none
  const int* end_query;    // [rows]: one past the last row that attends key j; j: none
  // Tiles of 128 rows, most work first, four numbers each, 16-byte aligned:
  const int* query_tiles;  // [ceil(rows / 128)]: first row, its first key, the last row's first key, last key + 1
  const int* query_pairs;  // [ceil(rows / 256)][2]: the same for pairs of neighbouring tiles
  const int* key_tiles;    // [ceil(rows / 128)]: first key, last query + 1, last query + 1 of the first key, 0
  int rows;                // rows of the tensors
  int pitch;               // rows rounded up to a multiple of 128: floats to a head of bias2 and delta
  int valid;               // rows that belong to documents; the ones behind give zeros
  int heads, kv_heads, dim;
  int type;                // 0 = fp16, 1 = bf16, 2 = fp32
  float scale;             // > 0
  int* gave_up;            // a word of the host's, set to 1 where a kernel gives up on a wait (besides its status)
} BgnPackedAttention;

// o [rows, heads, dim] contiguous and bias2 [heads, pitch]: minus the base-2 logarithm of the softmax
// denominator of scale * log2(e) * q.k (for fp16 with 10 added); -inf where a row attends nothing,
// unset from `rows` on.  The backward pass reads it.
// o_rest, like o: what rounding to 16 bits took from o; null where no backward pass follows, and for fp32.
int bgn_packed_attention_fwd(const BgnPackedAttention* a, void* o, void* o_rest, float* bias2, int* status, cudaStream_t stream);

// Gradients of the operands (contiguous) from the output's gradient d_o [rows, heads, dim] (strides in
// elements), the forward's o, o_rest and bias2.  Scratch: delta [heads, pitch]; for fp16 ds_bounds [3 heads + kv_heads, pitch].
int bgn_packed_attention_bwd(const BgnPackedAttention* a, const void* o, const void* o_rest, const float* bias2,
                             const void* d_o, long do_tok, long do_head, float* delta, float* ds_bounds, void* dq, void* dk, void* dv, int* status,
                             cudaStream_t stream);

typedef struct {
  const void* q;  // [rows, heads, dim], strides in elements, contiguous features
  const void* k;  // [rows, kv_heads, dim]
  long q_tok, q_head, k_tok, k_head;
  const int* position;  // [rows]: row of the tables
  const float* cos;     // [positions, rot / 2]
  const float* sin;
  void* q_out;  // contiguous
  void* k_out;
  int rows, heads, kv_heads, dim, rot;
  int type;    // 0 = fp16, 1 = bf16, 2 = fp32
  float sign;  // 1: turn, -1: turn back
} BgnPackedRotary;

int bgn_packed_rotary(const BgnPackedRotary* a, cudaStream_t stream);
}
