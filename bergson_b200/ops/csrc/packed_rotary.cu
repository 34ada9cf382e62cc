// Rotary embedding of q and k on packed documents, one launch for both.
//
// Feature pair (i, i + rot / 2) of token t turns by the angle of the token's position in its own
// document: (a, b) -> (a cos - b sin, b cos + a sin); the inverse turn is the gradient.  Every element
// is read once and written once, so HBM bounds it.  A block takes one token: a thread keeps its slice
// of the cosine and sine rows in registers and applies it to one head after the other.
#include "common.cuh"
#include "kernels_packed.h"

namespace bgn {

constexpr int kRotaryThreads = 512;

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
__global__ void __launch_bounds__(kRotaryThreads) packed_rotary_kernel(BgnPackedRotary a) {
  const int half = a.rot / 2;
  const int turns = half / V, per_head = turns + (a.dim - a.rot) / V;  // packets: pairs, then untouched ones
  const int lanes = blockDim.x / per_head;                             // heads at a time
  const int h0 = threadIdx.x / per_head, p = threadIdx.x % per_head;
  struct alignas(sizeof(T) * V) Packet { T v[V]; };
  const long t = blockIdx.x;
  const int position = __ldg(a.position + t);
  const bool turn = p < turns;
  const int d_lo = turn ? p * V : a.rot + (p - turns) * V, d_hi = half + p * V;
  const auto place = [&](int h, bool out) {
    const bool is_q = h < a.heads;
    const int g = is_q ? h : h - a.heads;
    if (out) return static_cast<T*>(is_q ? a.q_out : a.k_out) + (t * (is_q ? a.heads : a.kv_heads) + g) * a.dim;
    return const_cast<T*>(static_cast<const T*>(is_q ? a.q : a.k)) +
           (is_q ? t * a.q_tok + g * a.q_head : t * a.k_tok + g * a.k_head);
  };
  // The first head's features are asked for before the tables, whose rows hang on the position.
  const int heads = a.heads + a.kv_heads;
  Packet lo, hi;
  const auto fetch = [&](int h) {
    const T* x = place(h, false);
    lo = *reinterpret_cast<const Packet*>(x + d_lo);
    if (turn) hi = *reinterpret_cast<const Packet*>(x + d_hi);
  };
  if (h0 < heads) fetch(h0);
  float c[V], s[V];
  if (turn) {
    const long at = long(position) * half + p * V;
    load_floats<V>(c, a.cos + at);
    load_floats<V>(s, a.sin + at);
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] *= a.sign;
  }
  for (int h = h0; h < heads; h += lanes) {
    T* y = place(h, true);
    if (turn) {
      Packet o_lo, o_hi;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float u = to_float<T>(lo.v[e]), w = to_float<T>(hi.v[e]);
        o_lo.v[e] = from_float<T>(u * c[e] - w * s[e]);
        o_hi.v[e] = from_float<T>(w * c[e] + u * s[e]);
      }
      *reinterpret_cast<Packet*>(y + d_lo) = o_lo;
      *reinterpret_cast<Packet*>(y + d_hi) = o_hi;
    } else {
      *reinterpret_cast<Packet*>(y + d_lo) = lo;
    }
    if (h + lanes < heads) fetch(h + lanes);
  }
}

template <typename T>
static cudaError_t launch_rotary(const BgnPackedRotary& a, cudaStream_t stream) {
  constexpr int V = 16 / int(sizeof(T));
  // 16-byte packets where pairs, the untouched features and every head begin on such a boundary.
  const auto aligned = [](const void* p, long tok, long head) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && tok % V == 0 && head % V == 0;
  };
  const bool wide = (a.rot / 2) % V == 0 && (reinterpret_cast<uintptr_t>(a.cos) & 15) == 0 &&
                    (reinterpret_cast<uintptr_t>(a.sin) & 15) == 0 && a.dim % V == 0 && aligned(a.q, a.q_tok, a.q_head) &&
                    aligned(a.k, a.k_tok, a.k_head);
  const int packets = wide ? (a.rot / 2 + a.dim - a.rot) / V : a.rot / 2 + a.dim - a.rot;
  // As few passes over the heads as the block allows, and the heads spread evenly over them: 40 heads of
  // 8 packets take one pass of 320 threads (with 256 threads a second pass ran at a quarter).
  const int heads = a.heads + a.kv_heads;
  const int passes = (packets * heads + kRotaryThreads - 1) / kRotaryThreads;
  const int threads = packets * ((heads + passes - 1) / passes);
  if (wide) packed_rotary_kernel<T, V><<<unsigned(a.rows), threads, 0, stream>>>(a);
  else packed_rotary_kernel<T, 1><<<unsigned(a.rows), threads, 0, stream>>>(a);
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
