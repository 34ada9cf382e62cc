// C launch interface of the distillation loss against a teacher's top logits.
#pragma once

#include <cuda_runtime.h>

extern "C" {

typedef struct {
  const void* logits;   // [tokens, vocab], row pitch `pitch` elements
  const void* ids;      // [tokens, top]: int64 or int32; an id outside [0, vocab) is no entry
  const void* teacher;  // [tokens, top]: the teacher's logits of those ids
  long pitch;
  long tokens;
  int vocab, top;     // top <= kDistillMaxTop
  int type;           // logits and their gradient: 0 = fp16, 1 = bf16, 2 = fp32
  int teacher_type;   // the same codes
  int ids_64;         // 1: int64 ids
  float temperature;  // > 0
} BgnDistill;

enum { kDistillMaxTop = 1024 };

// loss [tokens]; stats [tokens, 2]: the row's maximum logit m and log2 of its sum of
// e^((z - m) / temperature).
int bgn_distill_fwd(const BgnDistill* a, float* loss, float* stats, cudaStream_t stream);

// dlogits with row pitch `d_pitch` from dloss [tokens].
int bgn_distill_bwd(const BgnDistill* a, const float* stats, const float* dloss, void* dlogits, long d_pitch,
                    cudaStream_t stream);
}
