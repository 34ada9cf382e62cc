// Rotary embedding of q and k on packed documents, one launch for both.
//
// Feature pair (i, i + rot / 2) of token t turns by the angle of the token's position in its own
// document: (a, b) -> (a cos - b sin, b cos + a sin); the inverse turn is the gradient.  Every element
// is read once and written once, so HBM bounds it.  A thread keeps its slice of a token's cosine and sine
// rows and applies it to one head after the other; small blocks, a head at a time, keep the loads of many
// threads in flight: 62 us (5410 GB/s; a copy of the same bytes takes 54) for 16384 tokens of 32 + 8 heads
// of 128 in bf16, where blocks of 256 took 70 and two heads at a time 89.
#include "common.cuh"
#include "kernels_packed.h"

namespace bgn {

constexpr int kRotaryThreads = 128;  // twice that where a head has more packets

// N consecutive floats, 16 bytes at a time where N allows.
template <int N>
__device__ __forceinline__ void load_floats(float (&x)[N], const float* p) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int e = 0; e < N; e += 4) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(p + e));
      x[e] = v.x;
      x[e + 1] = v.y;
      x[e + 2] = v.z;
      x[e + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = __ldg(p + e);
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(2 * kRotaryThreads) packed_rotary_kernel(BgnPackedRotary a, int groups, int tokens) {
  const int half = a.rot / 2;
  const int turns = half / V, per_head = turns + (a.dim - a.rot) / V;  // packets: pairs, then untouched ones
  const int per_token = per_head * groups;
  const int x = threadIdx.x % per_token, group = x / per_head, p = x % per_head;
  const long t = long(blockIdx.x) * tokens + threadIdx.x / per_token;
  if (t >= a.rows || int(threadIdx.x) >= per_token * tokens) return;
  struct alignas(sizeof(T) * V) Packet { T v[V]; };
  const bool turn = p < turns;
  const int d_lo = turn ? p * V : a.rot + (p - turns) * V, d_hi = half + p * V;
  const int heads = a.heads + a.kv_heads;
  const T* q = static_cast<const T*>(a.q) + t * a.q_tok;
  const T* k = static_cast<const T*>(a.k) + t * a.k_tok;
  T* q_out = static_cast<T*>(a.q_out) + t * a.heads * a.dim;
  T* k_out = static_cast<T*>(a.k_out) + t * a.kv_heads * a.dim;
  float c[V], s[V];
  if (turn) {
    const long at = long(__ldg(a.position + t)) * half + p * V;
    load_floats<V>(c, a.cos + at);
    load_floats<V>(s, a.sin + at);
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] *= a.sign;
  }
  for (int h = group; h < heads; h += groups) {
    const T* from = h < a.heads ? q + h * a.q_head : k + (h - a.heads) * a.k_head;
    T* to = h < a.heads ? q_out + h * a.dim : k_out + (h - a.heads) * a.dim;
    const Packet lo = *reinterpret_cast<const Packet*>(from + d_lo);
    if (turn) {
      const Packet hi = *reinterpret_cast<const Packet*>(from + d_hi);
      Packet o_lo, o_hi;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float x = to_float<T>(lo.v[e]), y = to_float<T>(hi.v[e]);
        o_lo.v[e] = from_float<T>(x * c[e] - y * s[e]);
        o_hi.v[e] = from_float<T>(y * c[e] + x * s[e]);
      }
      *reinterpret_cast<Packet*>(to + d_lo) = o_lo;
      *reinterpret_cast<Packet*>(to + d_hi) = o_hi;
    } else {
      *reinterpret_cast<Packet*>(to + d_lo) = lo;
    }
  }
}

template <typename T>
static cudaError_t launch_rotary(const BgnPackedRotary& a, cudaStream_t stream) {
  constexpr int V = 16 / int(sizeof(T));
  // 16-byte packets where pairs, the untouched features and every head begin on their boundaries.
  const auto aligned = [](const void* p, long tok, long head) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && tok % V == 0 && head % V == 0;
  };
  const bool wide = (a.rot / 2) % V == 0 && a.dim % V == 0 && (reinterpret_cast<uintptr_t>(a.cos) & 15) == 0 &&
                    (reinterpret_cast<uintptr_t>(a.sin) & 15) == 0 && aligned(a.q, a.q_tok, a.q_head) &&
                    aligned(a.k, a.k_tok, a.k_head);
  const int per_head = (a.rot / 2 + a.dim - a.rot) / (wide ? V : 1);
  // About half a block to a token, as far as its heads go: each thread then has a few of them.
  const int heads = a.heads + a.kv_heads;
  const int threads = per_head > kRotaryThreads ? 2 * kRotaryThreads : kRotaryThreads;
  int groups = threads / 2 / per_head;
  groups = groups < 1 ? 1 : (groups > heads ? heads : groups);
  const int tokens = threads / (groups * per_head);
  const unsigned grid = unsigned((a.rows + tokens - 1) / tokens);
  if (wide) packed_rotary_kernel<T, V><<<grid, threads, 0, stream>>>(a, groups, tokens);
  else packed_rotary_kernel<T, 1><<<grid, threads, 0, stream>>>(a, groups, tokens);
  return cudaGetLastError();
}

}  // namespace bgn

extern "C" int bgn_packed_rotary(const BgnPackedRotary* a, cudaStream_t stream) {
  if (a->rows <= 0 || a->heads <= 0 || a->kv_heads <= 0 || a->rot < 0 || a->rot % 2 || a->rot > a->dim ||
      a->dim > 256)
    return int(cudaErrorInvalidValue);
  if (a->type == 2) return int(bgn::launch_rotary<float>(*a, stream));
  if (a->type == 1) return int(bgn::launch_rotary<__nv_bfloat16>(*a, stream));
  return int(bgn::launch_rotary<__half>(*a, stream));
}
