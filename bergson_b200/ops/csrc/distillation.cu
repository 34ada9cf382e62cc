// Distillation from a teacher's top logits: loss and gradient over [tokens, vocab] student logits.
//
//   p = softmax(t / tau) over the row's entries,  q = softmax(z / tau) over the vocabulary
//   loss = tau^2 sum_k p_k (log p_k - log q[id_k]),   dz_v = g tau (q_v - sum_{k: id_k = v} p_k)
//
// With w_k = e^{(t_k - t_max) / tau}, W = sum w, m the maximum and s the sum of e^{(z - m) / tau}:
//   loss = tau^2 ( sum_k w_k ((t_k - t_max) - (z[id_k] - m)) / tau / W - log W + log s ),
// so one sweep over the row with a running maximum and sum is enough, and the large parts cancel
// before anything is rounded.  Exponents are taken to base 2.  HBM bounds both directions: the
// forward reads the logits once, the backward reads them once and writes the gradient once.  4096 tokens
// of 128256 bf16 logits: forward 185 us (5670 GB/s), backward 351 us (5990 GB/s); half of the rows
// without entries: 109 and 284 us.
#include <cooperative_groups.h>

#include "common.cuh"
#include "kernels_distill.h"
#include "packed_tc.cuh"

namespace bgn {

namespace cg = cooperative_groups;

constexpr int kDistillThreads = 256;
constexpr int kDistillUnroll = 4;  // packets a thread has in flight; with 2 the forward takes 214 us
constexpr int kDistillWarps = kDistillThreads / 32;
constexpr float kDistillLog2e = 1.4426950408889634f;
constexpr float kDistillLn2 = 0.6931471805599453f;

__device__ __forceinline__ float load_code(const void* p, long i, int type) {
  if (type == 2) return static_cast<const float*>(p)[i];
  if (type == 1) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

// Entry i of the teacher: its id, and -1 where there is none (an id outside the vocabulary, or a
// logit of -inf, which has no probability).
__device__ __forceinline__ int load_entry(const BgnDistill& a, long i, float* t) {
  const long id = a.ids_64 ? static_cast<const long*>(a.ids)[i] : long(static_cast<const int*>(a.ids)[i]);
  *t = load_code(a.teacher, i, a.teacher_type);
  return id >= 0 && id < a.vocab && *t != -INFINITY ? int(id) : -1;
}

// Reductions over the block, in the order of the warps; every thread gets the result.
template <int N, bool MAX>
__device__ __forceinline__ void block_reduce(float (&v)[N], float* red) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    v[n] = MAX ? warp_max(v[n]) : warp_sum(v[n]);
    if (lane == 0) red[n * kDistillWarps + warp] = v[n];
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) {
    float r = red[n * kDistillWarps];
#pragma unroll
    for (int w = 1; w < kDistillWarps; ++w) r = MAX ? fmaxf(r, red[n * kDistillWarps + w]) : r + red[n * kDistillWarps + w];
    v[n] = r;
  }
  __syncthreads();
}

template <typename T>
struct alignas(16) DistillPacket {
  static constexpr int N = 16 / int(sizeof(T));
  T v[N];
};

// Elements in front of the first 16-byte boundary.
template <typename T>
__device__ __forceinline__ int lead_of(const T* p, int n) {
  const int lead = int(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T));
  return lead < n ? lead : n;
}

// work(packet, index) for the packets of one part of a row, kDistillUnroll of them in flight for a thread;
// the first ones are asked for by fetch().  Many small blocks on an SM keep the memory busy while one of
// them computes or joins its sums.
template <typename T>
struct DistillStream {
  static constexpr int U = kDistillUnroll;
  const DistillPacket<T>* from;
  int packets;
  DistillPacket<T> held[U];

  __device__ __forceinline__ void fetch(int base) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (base + u * kDistillThreads < packets) held[u] = from[base + u * kDistillThreads];
  }
  template <typename F>
  __device__ __forceinline__ void run(F work) {
    for (int i = threadIdx.x; i < packets;) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u * kDistillThreads < packets) work(held[u], i + u * kDistillThreads);
      i += U * kDistillThreads;
      fetch(i);
    }
  }
};

// The larger value; NaN if there is one.
__device__ __forceinline__ float max_or_nan(float x, float y) {
  float z;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(x), "f"(y));
  return z;
}

// A packet's values in fp32, and the largest of them; NaN if one is: a packet of nothing but -inf adds nothing to the
// sum and is left out, one with a NaN among them must not be.
template <typename T>
__device__ __forceinline__ float unpack_max(const DistillPacket<T>& p, float2 (&f)[DistillPacket<T>::N / 2]);
template <>
__device__ __forceinline__ float unpack_max<float>(const DistillPacket<float>& p, float2 (&f)[2]) {
  f[0] = make_float2(p.v[0], p.v[1]);
  f[1] = make_float2(p.v[2], p.v[3]);
  return max_or_nan(max_or_nan(p.v[0], p.v[1]), max_or_nan(p.v[2], p.v[3]));
}
template <>
__device__ __forceinline__ float unpack_max<__nv_bfloat16>(const DistillPacket<__nv_bfloat16>& p, float2 (&f)[4]) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(p.v);
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] = __bfloat1622float2(h[e]);
  const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
  return max_or_nan(__low2float(m), __high2float(m));
}
template <>
__device__ __forceinline__ float unpack_max<__half>(const DistillPacket<__half>& p, float2 (&f)[4]) {
  const __half2* h = reinterpret_cast<const __half2*>(p.v);
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] = __half22float2(h[e]);
  const __half2 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
  return max_or_nan(__low2float(m), __high2float(m));
}

// A cluster of blocks shares one row: block r of it sweeps the r-th part of the columns, the first
// block joins the parts in rank order.  Six blocks to an SM cover each other's start, where a block waits for
// its teacher entries: 185 us, with five 195.
template <typename T>
__global__ void __launch_bounds__(kDistillThreads, 6) distill_fwd_kernel(BgnDistill a, float* loss, float* stats) {
  constexpr int V = DistillPacket<T>::N;
  __shared__ float red[3 * kDistillWarps];
  __shared__ float part[2];
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const long row = blockIdx.x / parts;
  const T* z = static_cast<const T*>(a.logits) + row * a.pitch;
  const float c = kDistillLog2e / a.temperature;

  const int per = ((a.vocab + parts - 1) / parts + V - 1) / V * V;
  const int begin = min(rank * per, a.vocab), n = min(begin + per, a.vocab) - begin;
  const T* x = z + begin;
  const int lead = lead_of(x, n);
  DistillStream<T> stream = {reinterpret_cast<const DistillPacket<T>*>(x + lead), (n - lead) / V};
  stream.fetch(threadIdx.x);

  // Teacher entries of the row and the student's logits there, while the first packets are on their way.
  __shared__ float t_of[kDistillMaxTop], z_of[kDistillMaxTop];
  float t_max = -INFINITY;
  bool some = false;
  if (rank == 0)
    for (int k = threadIdx.x; k < a.top; k += kDistillThreads) {
      float t;
      const int id = load_entry(a, row * a.top + k, &t);
      t_of[k] = id >= 0 ? t : -INFINITY;
      z_of[k] = id >= 0 ? to_float<T>(z[id]) : 0.f;
      t_max = fmaxf(t_max, t_of[k]);
      some = some || id >= 0;
    }
  // A row without entries, such as a prompt's, has no loss whatever its logits are: they are not read on.
  if (parts == 1 && !__syncthreads_or(some)) {
    if (threadIdx.x == 0) loss[row] = stats[2 * row] = stats[2 * row + 1] = 0.f;
    return;
  }

  // The difference to the maximum is taken before the factor, which could overflow a type's lowest value.
  float m = -INFINITY, s = 0.f;
  const auto one = [&](float v) {
    if (v > m) {
      s *= exp2f((m - v) * c);
      m = v;
    }
    // an entry of -inf adds nothing, and there may be no finite maximum yet
    if (v != -INFINITY) s += exp2f((v - m) * c);
  };
  if (int(threadIdx.x) < lead) one(to_float<T>(x[threadIdx.x]));
  stream.run([&](const DistillPacket<T>& p, int) {
    float2 f[V / 2];
    const float mx = unpack_max<T>(p, f);
    if (mx > m) {
      s *= exp2f((m - mx) * c);
      m = mx;
    }
    if (mx != -INFINITY) {
      float2 sum = make_float2(0.f, 0.f);
#pragma unroll
      for (int e = 0; e < V / 2; ++e) {
        const float2 d = mul2(add2(f[e], make_float2(-m, -m)), make_float2(c, c));
        sum = add2(sum, make_float2(fast_exp2(d.x), fast_exp2(d.y)));
      }
      s += sum.x + sum.y;
    }
  });
  for (int i = lead + stream.packets * V + threadIdx.x; i < n; i += kDistillThreads) one(to_float<T>(x[i]));

  float mx[2] = {m, t_max};
  block_reduce<2, true>(mx, red);
  float row_m = mx[0];
  if (m != -INFINITY) s *= exp2f((m - row_m) * c);
  if (parts > 1) {
    float sum[1] = {s};
    block_reduce<1, false>(sum, red);
    if (threadIdx.x == 0) {
      part[0] = row_m;
      part[1] = sum[0];
    }
    cluster.sync();
    s = 0.f;
    if (rank == 0) {
      for (int r = 1; r < parts; ++r) row_m = fmaxf(row_m, *cluster.map_shared_rank(&part[0], r));
      if (threadIdx.x == 0)
        for (int r = 0; r < parts; ++r) {
          const float pm = *cluster.map_shared_rank(&part[0], r), ps = *cluster.map_shared_rank(&part[1], r);
          s += pm == -INFINITY ? ps : ps * exp2f((pm - row_m) * c);
        }
    }
    cluster.sync();  // the parts stay until they are read
    if (rank != 0) return;
  }
  // s; W; sum of w (log2 w - log2 of the student's unnormalised value)
  float sums[3] = {s, 0.f, 0.f};
  if (rank == 0)
    for (int k = threadIdx.x; k < a.top; k += kDistillThreads) {
      if (t_of[k] == -INFINITY) continue;
      const float d = (t_of[k] - mx[1]) * c, w = exp2f(d);
      sums[1] += w;
      if (w != 0.f) sums[2] += w * (d - (z_of[k] - row_m) * c);
    }
  block_reduce<3, false>(sums, red);
  if (threadIdx.x == 0) {
    const float l2 = log2f(sums[0]);
    stats[2 * row] = row_m;
    stats[2 * row + 1] = l2;
    const float loss2 = sums[2] / sums[1] - log2f(sums[1]) + l2;
    // the largest entry has w = 1: no sum, no entry
    loss[row] = sums[1] == 0.f ? 0.f : a.temperature * a.temperature * kDistillLn2 * loss2;
  }
}

// Blocks parts * row ...: a block rewrites one part of a row's columns and puts its teacher entries right
// afterwards, each from the logit itself, so that every value is rounded once.  Five blocks to an SM: 351 us,
// six 354.
template <typename T>
__global__ void __launch_bounds__(kDistillThreads, 5)
distill_bwd_kernel(BgnDistill a, const float* stats, const float* dloss, T* dlogits, long d_pitch, int parts) {
  constexpr int V = DistillPacket<T>::N;
  __shared__ float red[kDistillWarps];
  __shared__ alignas(16) float p_of[kDistillMaxTop];
  __shared__ alignas(16) int id_of[kDistillMaxTop];
  const long row = blockIdx.x / parts;
  const int rank = int(blockIdx.x % parts);
  const float c = kDistillLog2e / a.temperature;
  const long k0 = row * a.top;
  const T* z = static_cast<const T*>(a.logits) + row * a.pitch;
  T* dz = dlogits + row * d_pitch;

  const int per = ((a.vocab + parts - 1) / parts + V - 1) / V * V;
  const int begin = min(rank * per, a.vocab), n = min(begin + per, a.vocab) - begin;
  const T* x = z + begin;
  T* y = dz + begin;
  // Packets need the same alignment on both sides.
  const bool same = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(y)) & 15) == 0;
  const int lead = same ? lead_of(x, n) : n;
  DistillStream<T> stream = {reinterpret_cast<const DistillPacket<T>*>(x + lead), (n - lead) / V};
  stream.fetch(threadIdx.x);

  float t_max[1] = {-INFINITY};
  for (int k = threadIdx.x; k < (a.top + 3) / 4 * 4; k += kDistillThreads) {
    float t = 0.f;
    id_of[k] = k < a.top ? load_entry(a, k0 + k, &t) : -1;
    p_of[k] = t;
    if (id_of[k] >= 0) t_max[0] = fmaxf(t_max[0], t);
  }
  block_reduce<1, true>(t_max, red);
  float w_sum[1] = {0.f};
  for (int k = threadIdx.x; k < a.top; k += kDistillThreads) {
    p_of[k] = id_of[k] >= 0 ? exp2f((p_of[k] - t_max[0]) * c) : 0.f;
    w_sum[0] += p_of[k];
  }
  block_reduce<1, false>(w_sum, red);
  const bool any = w_sum[0] != 0.f;
  const float inv_w = any ? 1.f / w_sum[0] : 0.f;
  const float g = any ? dloss[row] * a.temperature : 0.f;
  const float m = stats[2 * row], l2 = stats[2 * row + 1];
  const auto value = [&](float v) { return g * exp2f((v - m) * c - l2); };
  DistillPacket<T>* to = reinterpret_cast<DistillPacket<T>*>(y + lead);
  if (g == 0.f) {  // no entries, or a loss that does not count: zeros, whatever the logits are
    for (int i = threadIdx.x; i < lead; i += kDistillThreads) y[i] = from_float<T>(0.f);
    for (int i = threadIdx.x; i < stream.packets; i += kDistillThreads) to[i] = DistillPacket<T>{};
    for (int i = lead + stream.packets * V + threadIdx.x; i < n; i += kDistillThreads) y[i] = from_float<T>(0.f);
    return;
  }

  for (int i = threadIdx.x; i < lead; i += kDistillThreads) y[i] = from_float<T>(value(to_float<T>(x[i])));
  stream.run([&](const DistillPacket<T>& p, int i) {
    DistillPacket<T> o;
    float2 f[V / 2];
    unpack_max<T>(p, f);
#pragma unroll
    for (int e = 0; e < V / 2; ++e) {
      const float2 d = fma2(add2(f[e], make_float2(-m, -m)), make_float2(c, c), make_float2(-l2, -l2));
      const float2 q = mul2(make_float2(fast_exp2(d.x), fast_exp2(d.y)), make_float2(g, g));
      o.v[2 * e] = from_float<T>(q.x);
      o.v[2 * e + 1] = from_float<T>(q.y);
    }
    to[i] = o;
  });
  for (int i = lead + stream.packets * V + threadIdx.x; i < n; i += kDistillThreads) y[i] = from_float<T>(value(to_float<T>(x[i])));
  __syncthreads();
  // The teacher's entries: the first of equal ids takes the sum of all of them, in their order.
  for (int k = threadIdx.x; k < a.top; k += kDistillThreads) {
    const int id = id_of[k];
    if (id < begin || id >= begin + n) continue;
    bool first = true;
    float p = 0.f;
    for (int j = 0; j < a.top; j += 4) {  // the arrays are filled up to a multiple of four
      const int4 ids = *reinterpret_cast<const int4*>(id_of + j);
      const float4 ps = *reinterpret_cast<const float4*>(p_of + j);
      if (ids.x == id) p += ps.x;
      if (ids.y == id) p += ps.y;
      if (ids.z == id) p += ps.z;
      if (ids.w == id) p += ps.w;
      first = first && !((ids.x == id && j < k) || (ids.y == id && j + 1 < k) || (ids.z == id && j + 2 < k) ||
                         (ids.w == id && j + 3 < k));
    }
    if (first) dz[id] = from_float<T>(g * (exp2f((to_float<T>(z[id]) - m) * c - l2) - p * inv_w));
  }
}

template <typename T>
static cudaError_t launch_distill_fwd(const BgnDistill& a, float* loss, float* stats, int parts, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(a.tokens) * unsigned(parts));
  cfg.blockDim = dim3(kDistillThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = unsigned(parts);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, distill_fwd_kernel<T>, a, loss, stats);
}

// Blocks to a row: with few rows a row is shared, so that some four blocks per SM are at work, as
// long as each has a full group of packets for its threads.  One token of 50257 fp32 logits: forward 7.2 us,
// backward 6.9, where a block to a row takes 16.0 and 16.5; 300 of them 16.9 and 20.7, unshared 19.2 and
// 23.9, shared up to two blocks per SM 19.3 and 23.5.
static int row_parts(const BgnDistill& a, int most) {
  const int per_block = kDistillThreads * kDistillUnroll * (a.type == 2 ? 4 : 8);
  int parts = 1;
  while (parts < most && a.tokens * parts < 4 * 148 && a.vocab / (2 * parts) >= per_block) parts *= 2;
  return parts;
}

static bool distill_sound(const BgnDistill* a) {
  return a->tokens > 0 && a->tokens < (1l << 27) && a->vocab > 0 && a->top > 0 && a->top <= kDistillMaxTop &&
         a->pitch >= a->vocab && a->temperature > 0.f && a->type >= 0 && a->type <= 2 && a->teacher_type >= 0 &&
         a->teacher_type <= 2;
}

}  // namespace bgn

using namespace bgn;

extern "C" int bgn_distill_fwd(const BgnDistill* a, float* loss, float* stats, cudaStream_t stream) {
  if (!distill_sound(a)) return int(cudaErrorInvalidValue);
  const int parts = row_parts(*a, 8);
  if (a->type == 2) return int(launch_distill_fwd<float>(*a, loss, stats, parts, stream));
  if (a->type == 1) return int(launch_distill_fwd<__nv_bfloat16>(*a, loss, stats, parts, stream));
  return int(launch_distill_fwd<__half>(*a, loss, stats, parts, stream));
}

extern "C" int bgn_distill_bwd(const BgnDistill* a, const float* stats, const float* dloss, void* dlogits, long d_pitch,
                               cudaStream_t stream) {
  if (!distill_sound(a) || d_pitch < a->vocab) return int(cudaErrorInvalidValue);
  const int parts = row_parts(*a, 16);
  const unsigned grid = unsigned(a->tokens) * unsigned(parts);
  if (a->type == 2)
    distill_bwd_kernel<float><<<grid, kDistillThreads, 0, stream>>>(*a, stats, dloss, static_cast<float*>(dlogits), d_pitch, parts);
  else if (a->type == 1)
    distill_bwd_kernel<__nv_bfloat16><<<grid, kDistillThreads, 0, stream>>>(
        *a, stats, dloss, static_cast<__nv_bfloat16*>(dlogits), d_pitch, parts);
  else
    distill_bwd_kernel<__half><<<grid, kDistillThreads, 0, stream>>>(*a, stats, dloss, static_cast<__half*>(dlogits), d_pitch, parts);
  return int(cudaGetLastError());
}
