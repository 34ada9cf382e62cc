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
  const int* query_order;  // [ceil(rows / 128)]: query tiles of 128 rows, most keys first
  const int* query_pair_order;  // [ceil(rows / 256)]: pairs of neighbouring query tiles, most keys first
  const int* key_order;    // [ceil(rows / 128)]: key tiles of 128 rows, most queries first
  int rows;                // rows of the tensors
  int pitch;               // rows rounded up to a multiple of 128: floats to a head of lse2 and delta
  int valid;               // rows that belong to documents; the ones behind give zeros
  int heads, kv_heads, dim;
  int type;                // 0 = fp16, 1 = bf16, 2 = fp32
  float scale;             // > 0
} BgnPackedAttention;

// o [rows, heads, dim] contiguous and lse2 [heads, pitch]: base-2 logarithm of the softmax denominator of
// scale * log2(e) * q.k; +inf where a row attends nothing, unset from `rows` on.
int bgn_packed_attention_fwd(const BgnPackedAttention* a, void* o, float* lse2, int* status, cudaStream_t stream);

// Gradients of the operands (contiguous) from the output's gradient d_o [rows, heads, dim] (strides in
// elements), the forward's o and lse2.  Scratch: delta [heads, pitch], do_max [heads, pitch / 32].
int bgn_packed_attention_bwd(const BgnPackedAttention* a, const void* o, const float* lse2, const void* d_o, long do_tok,
                             long do_head, float* delta, float* do_max, void* dq, void* dk, void* dv, int* status,
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
