// Causal attention over packed documents in fp32 on the FMA units: forward and backward.
//
// Token t attends the keys first_key[t] .. t.  Tiles are cut from the packed token axis without
// regard to documents: a tile of 64 queries visits the keys from its first row's first key to its
// last row, and a per-row range masks the rest, so short documents share tiles.
//
//   S = scale q k^T, P = softmax(S), O = P v                         (one pass, running max and sum)
//   delta_t = do_t . o_t,  dS = P (do v^T - delta)
//   dQ = scale dS k,  dK = scale dS^T q (summed over the heads of a group),  dV = P^T do
//
// The scaled score is rounded on its own in both directions, so that a row with one key has P = 1 exactly.
// dQ and dK/dV are two kernels that recompute P from the stored log-sum-exp: sums stay in one block
// and one order, so results do not depend on scheduling.
//
// Bound by the FMA units and the shared memory that feeds them (a thread's 8 x 4 scores take three 16-byte loads
// to 32 operations): 8 documents of 1024 tokens, 12 heads of 64, forward 435 us (30 TFLOP/s), backward
// 1363 us.  Small batches wait for one block's chain of tiles; two rows to a thread did not shorten it.
// Fetching a tile into registers while the one before it is at work was slower (540 and 1715 against 500 and
// 1510 us, with four rows to a thread): the registers leave room for one block on an SM instead of two.
#pragma once

#include "common.cuh"
#include "kernels_packed.h"

namespace bgn {

constexpr int kSimpleTile = 64;              // queries and keys of a tile
constexpr int kSimplePitch = kSimpleTile + 4;  // floats between the rows of a tile in shared memory

// R: rows of a tile that a thread has, 4 or 8; 16 threads share a row, with 4 scores each.
template <int R>
constexpr int simple_threads() {
  return 16 * kSimpleTile / R;
}
constexpr float kLog2e = 1.4426950408889634f;

// Tiles of `kSimpleTile` tokens of two operands (or one) in shared memory, as [feature][token]; rows at or past
// `limit` and features at or past `dim` are zero.  All loads are on their way before the first store.
template <int DP, int R, bool TWO = true>
__device__ __forceinline__ void simple_load(float* dst_x, const float* x, long x_tok, float* dst_y, const float* y,
                                            long y_tok, int t0, int limit, int dim) {
  constexpr int kPackets = kSimpleTile * (DP / 4) / simple_threads<R>();
  float4 held[2][kPackets];
  // Neighbouring threads take neighbouring tokens, so that the transposed stores fall into different banks.
#pragma unroll
  for (int n = 0; n < (TWO ? 2 : 1) * kPackets; ++n) {
    const int i = threadIdx.x + n % kPackets * simple_threads<R>(), tok = i % kSimpleTile, d = (i / kSimpleTile) * 4;
    const float* from = n < kPackets ? x + long(t0 + tok) * x_tok : y + long(t0 + tok) * y_tok;
    float4& to = held[n / kPackets][n % kPackets];
    to = make_float4(0.f, 0.f, 0.f, 0.f);
    if (t0 + tok < limit && d < dim) to = *reinterpret_cast<const float4*>(from + d);
  }
#pragma unroll
  for (int n = 0; n < (TWO ? 2 : 1) * kPackets; ++n) {
    const int i = threadIdx.x + n % kPackets * simple_threads<R>();
    const float4 p = held[n / kPackets][n % kPackets];
    float* to = (n < kPackets ? dst_x : dst_y) + (i / kSimpleTile) * 4 * kSimplePitch + i % kSimpleTile;
    to[0] = p.x;
    to[kSimplePitch] = p.y;
    to[2 * kSimplePitch] = p.z;
    to[3 * kSimplePitch] = p.w;
  }
}

// acc[i][j] += sum_d a[d][4 ty + i] b[d][4 tx + j]
template <int DP, int R>
__device__ __forceinline__ void simple_scores(float (&acc)[R][4], const float* a, const float* b, int ty, int tx) {
#pragma unroll 8
  for (int d = 0; d < DP; ++d) {
    struct alignas(16) Rows { float v[R]; };
    const Rows x = *reinterpret_cast<const Rows*>(a + d * kSimplePitch + R * ty);
    const float4 y = *reinterpret_cast<const float4*>(b + d * kSimplePitch + 4 * tx);
    const float ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(x.v[i], ys[j], acc[i][j]);
  }
}

__device__ __forceinline__ void store_scores(float* p, const float (&s)[4], int row, int tx) {
  *reinterpret_cast<float4*>(p + row * kSimplePitch + 4 * tx) = make_float4(s[0], s[1], s[2], s[3]);
}

// out[i][c] += sum_j p[4 ty + i][j] x[tx + 16 c][j].  `careful`: only the columns inside(i) = [x, y] of a row take part,
// for what stands in a masked one may be infinite or NaN (a zero of p inside makes NaN of that, as it must).  That is
// slow, and only done over again when a result has turned out not to be finite.
template <int DP, int R, typename Range>
__device__ __forceinline__ void simple_product(float (&out)[R][DP / 16], const float* p, const float* x, int ty, int tx,
                                               bool careful, Range inside) {
  if (!careful) {
#pragma unroll 4
    for (int j = 0; j < kSimpleTile; j += 4) {
      float4 a[R];
#pragma unroll
      for (int i = 0; i < R; ++i) a[i] = *reinterpret_cast<const float4*>(p + (R * ty + i) * kSimplePitch + j);
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) {
        const float4 b = *reinterpret_cast<const float4*>(x + (tx + 16 * c) * kSimplePitch + j);
#pragma unroll
        for (int i = 0; i < R; ++i)
          out[i][c] = fmaf(a[i].x, b.x, fmaf(a[i].y, b.y, fmaf(a[i].z, b.z, fmaf(a[i].w, b.w, out[i][c]))));
      }
    }
  } else {
    for (int j = 0; j < kSimpleTile; ++j) {
      float a[R];
#pragma unroll
      for (int i = 0; i < R; ++i) a[i] = p[(R * ty + i) * kSimplePitch + j];
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) {
        const float b = x[(tx + 16 * c) * kSimplePitch + j];
#pragma unroll
        for (int i = 0; i < R; ++i)
          if (j >= inside(i).x && j <= inside(i).y) out[i][c] = fmaf(a[i], b, out[i][c]);
      }
    }
  }
}

template <int R, int N>
__device__ __forceinline__ bool some_not_finite(const float (&x)[R][N]) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int d = 0; d < N; ++d) bad |= !(fabsf(x[i][d]) < INFINITY);
  return bad;
}

// Sum / maximum over the 16 threads that share a row group (half a warp).
__device__ __forceinline__ float half_warp_sum(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float half_warp_max(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

template <int DP, int R>
__global__ void __launch_bounds__(simple_threads<R>()) packed_fwd_simple_kernel(BgnPackedAttention a, float* o, float* bias2) {
  extern __shared__ float smem[];
  float* qs = smem;
  float* ks = qs + DP * kSimplePitch;
  float* vs = ks + DP * kSimplePitch;
  float* ps = vs + DP * kSimplePitch;  // [query][key]
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  const int head = blockIdx.x % a.heads, slot = blockIdx.x / a.heads;
  const int kv_head = head / (a.heads / a.kv_heads);
  const int q0 = a.query_tiles[4 * (slot / 2)] + (slot & 1) * kSimpleTile;
  if (q0 >= a.rows) return;
  const float c = a.scale * kLog2e;

  const float* q = static_cast<const float*>(a.q) + long(head) * a.q_head;
  simple_load<DP, R, false>(qs, q, a.q_tok, nullptr, nullptr, 0, q0, a.valid, a.dim);
  int first[R];
  float m[R], l[R], out[R][DP / 16];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = q0 + R * ty + i;
    first[i] = row < a.valid ? a.first_key[row] : 0x7fffffff;
  }
  const float* k = static_cast<const float*>(a.k) + long(kv_head) * a.k_head;
  const float* v = static_cast<const float*>(a.v) + long(kv_head) * a.v_head;
  const int q1 = min(q0 + kSimpleTile, a.valid);
  bool careful = false;
again:
#pragma unroll
  for (int i = 0; i < R; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) out[i][d] = 0.f;
  }
  for (int k0 = q1 > q0 ? a.first_key[q0] : q1; k0 < q1; k0 += kSimpleTile) {
    __syncthreads();
    simple_load<DP, R>(ks, k, a.k_tok, vs, v, a.v_tok, k0, a.valid, a.dim);
    __syncthreads();
    float s[R][4] = {};
    simple_scores<DP, R>(s, qs, ks, ty, tx);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int row = q0 + R * ty + i;
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = k0 + 4 * tx + j;
        s[i][j] = (key >= first[i] && key <= row) ? s[i][j] * c : -INFINITY;
        mx = fmaxf(mx, s[i][j]);
      }
      mx = fmaxf(half_warp_max(mx), m[i]);
      const float base = mx == -INFINITY ? 0.f : mx;  // nothing attended yet
      const float old = exp2f(m[i] - base);
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = exp2f(s[i][j] - base);
        sum += s[i][j];
      }
      store_scores(ps, s[i], R * ty + i, tx);
      l[i] = l[i] * old + half_warp_sum(sum);
      m[i] = mx;
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) out[i][d] *= old;
    }
    __syncthreads();
    simple_product<DP, R>(out, ps, vs, ty, tx, careful, [&](int i) { return make_int2(first[i] - k0, q0 + R * ty + i - k0); });
  }
  if (!careful && __syncthreads_or(some_not_finite(out))) {
    careful = true;
    goto again;
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = q0 + R * ty + i;
    if (row >= a.rows) continue;
    const bool some = row < a.valid && first[i] <= row;
    const float inv = some ? 1.f / l[i] : 0.f;
    if (tx == 0) bias2[long(head) * a.pitch + row] = some ? -(m[i] + log2f(l[i])) : -INFINITY;
    float* dst = o + (long(row) * a.heads + head) * a.dim;
#pragma unroll
    for (int d = 0; d < DP / 16; ++d)
      if (tx + 16 * d < a.dim) dst[tx + 16 * d] = some ? out[i][d] * inv : 0.f;
  }
}

template <int DP, int R>
__global__ void __launch_bounds__(simple_threads<R>())
packed_dq_simple_kernel(BgnPackedAttention a, const float* o, const float* bias2, const float* d_o, long do_tok, long do_head,
                        float* delta, float* dq) {
  extern __shared__ float smem[];
  float* qs = smem;
  float* gs = qs + DP * kSimplePitch;
  float* ks = gs + DP * kSimplePitch;
  float* vs = ks + DP * kSimplePitch;
  float* ds = vs + DP * kSimplePitch;  // [query][key]
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  const int head = blockIdx.x % a.heads, slot = blockIdx.x / a.heads;
  const int kv_head = head / (a.heads / a.kv_heads);
  const int q0 = a.query_tiles[4 * (slot / 2)] + (slot & 1) * kSimpleTile;
  if (q0 >= a.rows) return;
  const float c = a.scale * kLog2e;

  const float* q = static_cast<const float*>(a.q) + long(head) * a.q_head;
  simple_load<DP, R>(qs, q, a.q_tok, gs, d_o + long(head) * do_head, do_tok, q0, a.valid, a.dim);
  __syncthreads();
  int first[R];
  float bias[R], dl[R], out[R][DP / 16];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = q0 + R * ty + i;
    const bool in = row < a.valid;
    first[i] = in ? a.first_key[row] : 0x7fffffff;
    bias[i] = in ? bias2[long(head) * a.pitch + row] : -INFINITY;
    float sum = 0.f;
    if (in) {
      const float* orow = o + (long(row) * a.heads + head) * a.dim;
      for (int d = tx; d < a.dim; d += 16) sum = fmaf(orow[d], gs[d * kSimplePitch + R * ty + i], sum);
    }
    dl[i] = half_warp_sum(sum);
    if (tx == 0 && row < a.rows) delta[long(head) * a.pitch + row] = dl[i];
  }
  const float* k = static_cast<const float*>(a.k) + long(kv_head) * a.k_head;
  const float* v = static_cast<const float*>(a.v) + long(kv_head) * a.v_head;
  const int q1 = min(q0 + kSimpleTile, a.valid);
  bool careful = false;
again:
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) out[i][d] = 0.f;
  for (int k0 = q1 > q0 ? a.first_key[q0] : q1; k0 < q1; k0 += kSimpleTile) {
    __syncthreads();
    simple_load<DP, R>(ks, k, a.k_tok, vs, v, a.v_tok, k0, a.valid, a.dim);
    __syncthreads();
    float s[R][4] = {}, dp[R][4] = {};
    simple_scores<DP, R>(s, qs, ks, ty, tx);
    simple_scores<DP, R>(dp, gs, vs, ty, tx);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int row = q0 + R * ty + i;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = k0 + 4 * tx + j;
        // A row with one key has P = 1 and no gradient through the softmax: exactly zero.
        const bool in = key >= first[i] && key <= row && first[i] < row;
        s[i][j] = in ? exp2f(__fmul_rn(s[i][j], c) + bias[i]) * (dp[i][j] - dl[i]) : 0.f;
      }
      store_scores(ds, s[i], R * ty + i, tx);
    }
    __syncthreads();
    simple_product<DP, R>(out, ds, ks, ty, tx, careful, [&](int i) {
      const int row = q0 + R * ty + i;
      return make_int2(first[i] < row ? first[i] - k0 : 0x7fffffff, row - k0);
    });
  }
  if (!careful && __syncthreads_or(some_not_finite(out))) {
    careful = true;
    goto again;
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = q0 + R * ty + i;
    if (row >= a.rows) continue;
    float* dst = dq + (long(row) * a.heads + head) * a.dim;
#pragma unroll
    for (int d = 0; d < DP / 16; ++d)
      if (tx + 16 * d < a.dim) dst[tx + 16 * d] = out[i][d] * a.scale;
  }
}

template <int DP, int R>
__global__ void __launch_bounds__(simple_threads<R>())
packed_dkv_simple_kernel(BgnPackedAttention a, const float* bias2, const float* d_o, long do_tok, long do_head,
                         const float* delta, float* dk, float* dv) {
  extern __shared__ float smem[];
  float* ks = smem;
  float* vs = ks + DP * kSimplePitch;
  float* qs = vs + DP * kSimplePitch;
  float* gs = qs + DP * kSimplePitch;
  float* ps = gs + DP * kSimplePitch;  // [key][query]
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  const int kv_head = blockIdx.x % a.kv_heads, slot = blockIdx.x / a.kv_heads;
  const int group = a.heads / a.kv_heads;
  const int k0 = a.key_tiles[4 * (slot / 2)] + (slot & 1) * kSimpleTile;
  if (k0 >= a.rows) return;
  const float c = a.scale * kLog2e;

  simple_load<DP, R>(ks, static_cast<const float*>(a.k) + long(kv_head) * a.k_head, a.k_tok, vs,
                  static_cast<const float*>(a.v) + long(kv_head) * a.v_head, a.v_tok, k0, a.valid, a.dim);
  int end[R], own_first[R];
  float out_k[R][DP / 16], out_v[R][DP / 16];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int key = k0 + R * ty + i;
    end[i] = key < a.valid ? a.end_query[key] : 0;
    own_first[i] = key < a.valid ? a.first_key[key] : 0;
  }
  const int k1 = min(k0 + kSimpleTile, a.valid);
  const int q_end = k1 > k0 ? min(a.end_query[k1 - 1], a.valid) : 0;
  bool careful = false;
again:
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) out_k[i][d] = out_v[i][d] = 0.f;
  for (int head = kv_head * group; head < (kv_head + 1) * group; ++head) {
    for (int q0 = k0; q0 < q_end; q0 += kSimpleTile) {
      __syncthreads();
      const float* q = static_cast<const float*>(a.q) + long(head) * a.q_head;
      simple_load<DP, R>(qs, q, a.q_tok, gs, d_o + long(head) * do_head, do_tok, q0, a.valid, a.dim);
      __syncthreads();
      float s[R][4] = {}, dp[R][4] = {};
      simple_scores<DP, R>(s, ks, qs, ty, tx);
      simple_scores<DP, R>(dp, vs, gs, ty, tx);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = q0 + 4 * tx + j;
        const bool in_row = row < a.valid;
        const float bias = in_row ? bias2[long(head) * a.pitch + row] : -INFINITY;
        const float dl = in_row ? delta[long(head) * a.pitch + row] : 0.f;
#pragma unroll
        for (int i = 0; i < R; ++i) {
          const int key = k0 + R * ty + i;
          const bool in = row >= key && row < end[i];
          const float p = in ? exp2f(__fmul_rn(s[i][j], c) + bias) : 0.f;
          s[i][j] = p;
          dp[i][j] = in && own_first[i] < row ? p * (dp[i][j] - dl) : 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < R; ++i) store_scores(ps, s[i], R * ty + i, tx);
      __syncthreads();
      simple_product<DP, R>(out_v, ps, gs, ty, tx, careful,
                            [&](int i) { return make_int2(k0 + R * ty + i - q0, end[i] - 1 - q0); });
      __syncthreads();
#pragma unroll
      for (int i = 0; i < R; ++i) store_scores(ps, dp[i], R * ty + i, tx);
      __syncthreads();
      simple_product<DP, R>(out_k, ps, qs, ty, tx, careful, [&](int i) {
        return make_int2(max(k0 + R * ty + i, own_first[i] + 1) - q0, end[i] - 1 - q0);
      });
    }
  }
  if (!careful && __syncthreads_or(some_not_finite(out_k) || some_not_finite(out_v))) {
    careful = true;
    goto again;
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int key = k0 + R * ty + i;
    if (key >= a.rows) continue;
    const long at = (long(key) * a.kv_heads + kv_head) * a.dim;
#pragma unroll
    for (int d = 0; d < DP / 16; ++d)
      if (tx + 16 * d < a.dim) {
        dk[at + tx + 16 * d] = out_k[i][d] * a.scale;
        dv[at + tx + 16 * d] = out_v[i][d];
      }
  }
}

template <int DP>
constexpr int simple_smem(int tiles) {
  return (tiles * DP + kSimpleTile) * kSimplePitch * int(sizeof(float));
}

}  // namespace bgn
