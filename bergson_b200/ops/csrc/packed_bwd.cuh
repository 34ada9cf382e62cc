// Backward pass of the causal attention over packed documents on the tensor cores (fp16, bf16).
//
//   P = 2^(c q.k + bias2),  delta_t = do_t . o_t,  dS = P (do.v - delta)
//   dQ = scale dS k,   dK = scale dS^T q,   dV = P^T do      (dK, dV summed over the heads of a group)
//
// After a small one for delta, two kernels, each of which keeps its sums in TMEM from the first to the last
// tile: one block for the rows of dQ, one for the rows of dK and dV.  P is computed in both: that is seven products for the
// five of the mathematics, and buys sums in one order (the results are the same in every run) without
// a fp32 copy of dQ in memory.  Tiles are cut from the packed axis as in the forward pass.
//
// P and dS are rounded to the operands' type for the tensor core; everything else is fp32.  fp16 has
// few small values and ends at 65504, so there P carries a factor 2^10 and dS the power of two that brings B, a bound of
// |do.v - delta|, to [2^14, 2^15): dS cannot overflow and uses what the type has below that.
//   dQ, row t:  B = sum|do_t| max|v_j| + |delta_t|,  over the row's own keys (to the end of its 32 rows)
//   dK, key j:  B = max sum|do_t| max|v| + max|delta_t|,  over the document's rows t from the key's 32 rows on, v of those 32
// Both factors are taken out of the fp32 sums at the end.  A row, or a key, is a thread of the softmax warps, so each
// has its own factor and no document sets the precision of another one.
//
// Rows whose results are not finite are put right after a block's last unit, as in the forward pass.
#pragma once

#include "packed_fwd.cuh"

namespace bgn {

constexpr int kBwdThreads = 320;

struct PackedBwdArgs {
  const int* first_key;
  const int* end_query;
  const int4* tiles;  // query_tiles or key_tiles
  int units;          // tiles x heads of queries or of keys
  int rows, valid, heads, kv_heads, dim;
  int pitch;  // floats between the heads of bias2 and neg_delta, a multiple of 128
  float scale;
  const void *q, *k, *v, *o, *o_rest, *d_o;
  long q_tok, q_head, k_tok, k_head, v_tok, v_head, do_tok, do_head;
  const float* bias2;
  float* neg_delta;
  // fp16, what bounds dS; what is not finite counts as zero.  "doc": the largest value of the row's group of 32 rows
  // (from a multiple of 32 on), as far as they are of its document.
  float* row_do;     // [heads, pitch]: sum |do|
  float* doc_do;     // [heads, pitch]: the same, doc
  float* doc_delta;  // [heads, pitch]: |delta|, doc
  float* doc_v;      // [kv_heads, pitch]: |v|, doc
  void *dq, *dk, *dv;
  int* gave_up;
};

// The power of two that brings `bound` to [2^14, 2^15); 1 where there is nothing to scale.
__device__ __forceinline__ float power_for(float bound) {
  if (!(bound > 0.f) || !(bound < INFINITY)) return 1.f;
  const int f = 268 - int(__float_as_uint(bound) >> 23);  // biased: bound in [2^(e-127), 2^(e-126)), factor 2^(141-e)
  return __uint_as_float(uint32_t(f < 253 ? f : 253) << 23);
}

// Each value becomes the largest of the lanes with the same `run`, which lie side by side.
template <int N>
__device__ __forceinline__ void max_of_run(float (&x)[N], int run) {
  if (__all_sync(0xffffffffu, run == __shfl_sync(0xffffffffu, run, 0))) {
#pragma unroll
    for (int n = 0; n < N; ++n) x[n] = warp_max(x[n]);
    return;
  }
  const int lane = threadIdx.x & 31;
  float behind[N];
#pragma unroll
  for (int n = 0; n < N; ++n) behind[n] = x[n];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const bool up = __shfl_up_sync(0xffffffffu, run, o) == run && lane >= o;
    const bool down = __shfl_down_sync(0xffffffffu, run, o) == run && lane + o < 32;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const float b = __shfl_up_sync(0xffffffffu, x[n], o), f = __shfl_down_sync(0xffffffffu, behind[n], o);
      if (up) x[n] = fmaxf(x[n], b);
      if (down) behind[n] = fmaxf(behind[n], f);
    }
  }
#pragma unroll
  for (int n = 0; n < N; ++n) x[n] = fmaxf(x[n], behind[n]);
}

__device__ __forceinline__ float finite_or_zero(float x) { return fabsf(x) < INFINITY ? x : 0.f; }

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// P (with its factor) of two columns in place: 2^(c s + bias).
__device__ __forceinline__ void prob_pair(uint32_t& s0, uint32_t& s1, float2 c2, float2 bias) {
  const float2 x = fma2(make_float2(__uint_as_float(s0), __uint_as_float(s1)), c2, bias);
  s0 = __float_as_uint(fast_exp2(x.x));
  s1 = __float_as_uint(fast_exp2(x.y));
}

// dS (with its factor) of two columns: P (dP - delta).
template <int FMT>
__device__ __forceinline__ float2 score_gradient(uint32_t p0, uint32_t p1, uint32_t d0, uint32_t d1, float2 neg_delta,
                                                 float2 factor) {
  float2 x = mul2(make_float2(__uint_as_float(p0), __uint_as_float(p1)),
                  add2(make_float2(__uint_as_float(d0), __uint_as_float(d1)), neg_delta));
  return FMT == 0 ? mul2(x, factor) : x;
}

// ---- delta ----------------------------------------------------------------------------
//
// delta = do . o, with what rounding took from o: dS is a difference against delta, and for rows with few
// keys that rounding would be its largest error.  A block has 32 rows of a head, LANES lanes to a row.
// HBM bounds it: o, its rest and do are read once (16384 tokens of 32 heads of 128: 61 us, 6600 GB/s).  For fp16 it also
// reads v, for what bounds dS.

// fp16: four rows to a thread and so small blocks, of which others read while one joins its rows' bounds (76 us at the
// same size over 8 key heads, 90 with a row to a thread); bf16 has nothing to join.
template <int FMT, int LANES>
constexpr int delta_threads() {
  return 32 * LANES / (FMT == 0 ? 4 : 1);
}

template <int FMT, int LANES>
__global__ void __launch_bounds__(delta_threads<FMT, LANES>()) packed_delta_kernel(const __grid_constant__ PackedBwdArgs p) {
  using T = typename Type16<FMT>::T;
  constexpr int kStep = delta_threads<FMT, LANES>() / LANES, kRows = 32 / kStep;
  __shared__ float of_row[3][32];  // sum |do|, |delta|, largest |v|
  next_kernel_may_come();
  const int head = blockIdx.x % p.heads, row0 = blockIdx.x / p.heads * 32, group = p.heads / p.kv_heads;
  const int lane = threadIdx.x % LANES, row1 = threadIdx.x / LANES, f = 8 * lane;
  const bool with_v = FMT == 0 && head % group == 0;  // one head of a group looks at v
  union Packet { uint4 u; T h[8]; };
  Packet o[kRows], rest[kRows], g[kRows], v[kRows];
#pragma unroll
  for (int n = 0; n < kRows; ++n) {
    const int row = row0 + row1 + n * kStep;
    o[n].u = rest[n].u = g[n].u = v[n].u = make_uint4(0, 0, 0, 0);
    if (row < p.valid && f < p.dim) {
      const long from = (long(row) * p.heads + head) * p.dim + f;
      o[n].u = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.o) + from));
      rest[n].u = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.o_rest) + from));
      g[n].u = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.d_o) + long(row) * p.do_tok + long(head) * p.do_head + f));
      if (with_v)
        v[n].u = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.v) + long(row) * p.v_tok + long(head / group) * p.v_head + f));
    }
  }
#pragma unroll
  for (int n = 0; n < kRows; ++n) {
    float sum = 0.f, size = 0.f, top_v = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = to_float<T>(g[n].h[e]);
      sum = fmaf(-to_float<T>(o[n].h[e]) - to_float<T>(rest[n].h[e]), x, sum);
      if (FMT == 0) size += fabsf(x);
    }
    if (with_v)
#pragma unroll
      for (int e = 0; e < 8; ++e) top_v = fmaxf(top_v, fabsf(finite_or_zero(to_float<T>(v[n].h[e]))));
#pragma unroll
    for (int x = LANES / 2; x > 0; x >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, x);
      if (FMT == 0) size += __shfl_xor_sync(0xffffffffu, size, x);
      if (with_v) top_v = fmaxf(top_v, __shfl_xor_sync(0xffffffffu, top_v, x));
    }
    const int r = row1 + n * kStep;
    if (lane == 0) {
      p.neg_delta[long(head) * p.pitch + row0 + r] = sum;  // zero where there is no row
      if (FMT == 0) {
        of_row[0][r] = finite_or_zero(size);
        of_row[1][r] = fabsf(finite_or_zero(sum));
        of_row[2][r] = top_v;
      }
    }
  }
  if (FMT == 0) {
    __syncthreads();
    if (threadIdx.x < 32) {  // a row to a lane
      const int own = row0 + threadIdx.x;
      const long to = long(head) * p.pitch + own;
      float x[3] = {of_row[0][threadIdx.x], of_row[1][threadIdx.x], of_row[2][threadIdx.x]};
      p.row_do[to] = x[0];
      max_of_run(x, own < p.valid ? __ldg(p.first_key + own) : -1);
      p.doc_do[to] = x[0];
      p.doc_delta[to] = x[1];
      if (with_v) p.doc_v[long(head / group) * p.pitch + own] = x[2];
    }
  }
}

// ---- dQ -------------------------------------------------------------------------------
//
// A unit is one tile of 128 query rows of a head.  Per key tile: S = q k^T and dP = do v^T, the softmax
// warps turn them into dS (P stays in registers), dQ += dS k.  S is free again as soon as it is read and
// dP has two places, so the two products of the next key tile run while this one's dS is formed.
//
// TMEM: dQ, S, dP twice (128 columns each; dS in 16 bits over its dP).  Shared memory: q, do, three
// key and two value tiles (7 tiles of 32 KB at 128 features).  Warps 0-7: softmax, warps 0-3 on the first
// 64 keys of a tile, 4-7 on the rest; two threads share a row.  8 TMA, 9 MMA.
//
// Delta comes from a kernel of its own: read here, by softmax warps or by others, o and do took as long as
// two to four key tiles, as loads through the first-level cache wait for the tensor core's operands.
//
// Bound by the tensor core (three products of 512 cycles a tile at 128 features) and the softmax warps in turn:
// 32 over 8 heads of 128 in bf16, one document of 8192 tokens 0.63 ms (1320 TFLOP/s of its three products).

constexpr int kDqKStages = 3;  // a key tile stays until dQ of its step, which comes after S and dP of the next
constexpr int kDqVStages = 2;
constexpr int kDqRowFloats = 2 * kTile;  // of a unit: -delta, bias2

template <int DP>
constexpr int dq_smem_bytes() {
  return (2 + kDqKStages + kDqVStages) * tile_bytes<DP>() + kDqRowFloats * 4 + 256;
}

// A warp puts right one half of the features of a row of dQ, in the tile at row0.
template <int FMT, int DP>
__device__ __noinline__ void exact_dq_row(const PackedBwdArgs& p, int row0, int row, int head, int half, int lane) {
  using T = typename Type16<FMT>::T;
  const int kv = head / (p.heads / p.kv_heads), first = p.first_key[row];
  const int f0 = half ? DP / 2 : 0, f1 = min(f0 + DP / 2, p.dim);
  const long at = (long(row) * p.heads + head) * p.dim, k_off = long(kv) * p.k_head;
  float q[DP / 32], g[DP / 32], dq[DP / 32] = {};
  load_row<FMT, DP>(q, p.dq, at, p.dim, lane);
  bool bad = false;
#pragma unroll
  for (int e = 0; e < DP / 32; ++e) bad |= lane + 32 * e >= f0 && lane + 32 * e < f1 && !(fabsf(q[e]) < INFINITY);
  if (!__any_sync(0xffffffffu, bad)) return;
  // see exact_forward_row; here the keys are visited from the first one of the tile's first row on
  if (first <= row0 && !some_not_finite<FMT, DP>(p.k, p.k_tok, k_off, row + 1, min(row0 + 2 * kTile, p.valid), p.dim, lane))
    return;
  const float c = p.scale * kPackedLog2e, bias2 = p.bias2[long(head) * p.pitch + row] - p_shift<FMT>();
  const float neg_delta = p.neg_delta[long(head) * p.pitch + row];
  load_row<FMT, DP>(q, p.q, long(row) * p.q_tok + long(head) * p.q_head, p.dim, lane);
  load_row<FMT, DP>(g, p.d_o, long(row) * p.do_tok + long(head) * p.do_head, p.dim, lane);
  for (int j0 = first; j0 <= row && first < row && !all_nan(dq, f0, f1, lane); j0 += 64) {
#pragma unroll 4
    for (int j = j0; j <= min(j0 + 63, row); ++j) {
      float k[DP / 32], v[DP / 32];
      load_row<FMT, DP>(k, p.k, long(j) * p.k_tok + k_off, p.dim, lane);
      load_row<FMT, DP>(v, p.v, long(j) * p.v_tok + long(kv) * p.v_head, p.dim, lane);
      const float ds = exp2f(warp_dot(q, k) * c + bias2) * (warp_dot(g, v) + neg_delta);
#pragma unroll
      for (int e = 0; e < DP / 32; ++e) dq[e] = fmaf(ds, k[e], dq[e]);
    }
  }
  T* dst = static_cast<T*>(p.dq) + at;
#pragma unroll
  for (int e = 0; e < DP / 32; ++e)
    if (lane + 32 * e >= f0 && lane + 32 * e < f1) dst[lane + 32 * e] = from_float<T>(dq[e] * p.scale);
}

template <int FMT, int DP>
__global__ void __launch_bounds__(kBwdThreads, 1)
packed_dq_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                 const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                 const __grid_constant__ PackedBwdArgs p, int* status) {
  constexpr int kTileBytes = tile_bytes<DP>();
  constexpr int kSlabs = DP / 64;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  // Nearly all of the shared memory is in use at 128 features: there is no room for moving up to a boundary.
  if ((smem_u32(smem_raw) & 1023u) != 0) {
    if (threadIdx.x == 0) record_give_up(status, p.gave_up, kStatusTimeoutProducer);
    return;
  }
  uint8_t* q_tile = smem_raw;
  uint8_t* g_tile = q_tile + kTileBytes;
  uint8_t* k_tiles = g_tile + kTileBytes;
  uint8_t* v_tiles = k_tiles + kDqKStages * kTileBytes;
  float* row_values = reinterpret_cast<float*>(v_tiles + kDqVStages * kTileBytes);
  uint64_t* bars = reinterpret_cast<uint64_t*>(row_values + kDqRowFloats);
  uint64_t* q_full = bars;  // q, do and the row values
  uint64_t* q_empty = q_full + 1;
  uint64_t* k_full = q_empty + 1;  // [3]
  uint64_t* k_empty = k_full + kDqKStages;
  uint64_t* v_full = k_empty + kDqKStages;  // [2]
  uint64_t* v_empty = v_full + kDqVStages;
  uint64_t* s_full = v_empty + kDqVStages;
  uint64_t* s_read = s_full + 1;
  uint64_t* dp_full = s_read + 1;   // [2]
  uint64_t* ds_full = dp_full + 2;  // [2]
  uint64_t* dq_full = ds_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(dq_full + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = p.heads / p.kv_heads;

  next_kernel_may_come();
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 9);  // the MMA warp's commit and the softmax warps, which read the row values
    for (int s = 0; s < kDqKStages; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&v_full[t], 1);
      mbar_init(&v_empty[t], 1);
      mbar_init(&dp_full[t], 1);
      mbar_init(&ds_full[t], 8);
    }
    mbar_init(s_full, 1);
    mbar_init(s_read, 8);
    mbar_init(dq_full, 1);
    fence_barrier_init();
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_do);
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  wait_for_last_kernel();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tmem_dq = tmem, tmem_s = tmem + 128, tmem_dp = tmem + 256;  // dp: two places

  int unit = nth_unit(0, p.units);
  int4 entry = unit >= 0 ? __ldg(p.tiles + unit / p.heads) : make_int4(0, 0, 0, 0);
  // Of the unit at hand: first row, first key, key tiles.
  const auto steps_of = [](const int4& e) { return e.w > e.y ? (e.w - e.y + kTile - 1) / kTile : 0; };

  if (warp == 8) {
    if (lane == 0) {
      bool ok = true;
      int j = 0, uses = 0;
      for (int r = 0; unit >= 0 && ok; ++r) {
        const int after = nth_unit(r + 1, p.units);
        const int4 next = after >= 0 ? __ldg(p.tiles + after / p.heads) : entry;
        const int head = unit % p.heads, kv_head = head / group, n = steps_of(entry);
        for (int i = 0; i < n && ok; ++i, ++j) {
          const int st = j % kDqKStages, vst = j % kDqVStages, key = entry.y + i * kTile;
          ok = mbar_wait_bounded(&k_empty[st], ((j / kDqKStages) & 1) ^ 1);
          if (!ok) break;
          mbar_expect_tx(&k_full[st], kTileBytes);
  #pragma unroll
          for (int s = 0; s < kSlabs; ++s)
            tma_load_3d(k_tiles + st * kTileBytes + s * kSlabBytes, &map_k, &k_full[st], 64 * s, kv_head, key);
          if (i == 0) {
            ok = mbar_wait_bounded(q_empty, (uses & 1) ^ 1);
            if (!ok) break;
            ++uses;
            mbar_expect_tx(q_full, 2 * kTileBytes + 4 * kDqRowFloats);
            // whole tiles of rows to a head, so the copies stay inside
            bulk_load(row_values, p.neg_delta + long(head) * p.pitch + entry.x, 4 * kTile, q_full);
            bulk_load(row_values + kTile, p.bias2 + long(head) * p.pitch + entry.x, 4 * kTile, q_full);
  #pragma unroll
            for (int s = 0; s < kSlabs; ++s) {
              tma_load_3d(q_tile + s * kSlabBytes, &map_q, q_full, 64 * s, head, entry.x);
              tma_load_3d(g_tile + s * kSlabBytes, &map_do, q_full, 64 * s, head, entry.x);
            }
          }
          ok = mbar_wait_bounded(&v_empty[vst], ((j / kDqVStages) & 1) ^ 1);
          if (!ok) break;
          mbar_expect_tx(&v_full[vst], kTileBytes);
  #pragma unroll
          for (int s = 0; s < kSlabs; ++s)
            tma_load_3d(v_tiles + vst * kTileBytes + s * kSlabBytes, &map_v, &v_full[vst], 64 * s, kv_head, key);
        }
        unit = after;
        entry = next;
      }
      if (!ok) {
        record_give_up(status, p.gave_up, kStatusTimeoutProducer);
        drain_copies();
      }
    }
    __syncwarp();
  } else if (warp == 9) {
    constexpr uint32_t idesc_s = make_idesc_f16(kTile, kTile, FMT, 0, 0);
    constexpr uint32_t idesc_dq = make_idesc_f16(kTile, DP, FMT, 0, 1);
    bool ok = true;
    int j = 0, uses = 0;
    const uint64_t dq = make_kmajor_sw128_desc(smem_u32(q_tile)), dg = make_kmajor_sw128_desc(smem_u32(g_tile));
    const uint64_t dk = make_kmajor_sw128_desc(smem_u32(k_tiles)), dv = make_kmajor_sw128_desc(smem_u32(v_tiles));
    const uint64_t dk_mn = make_mnmajor_sw128_desc(smem_u32(k_tiles), kSlabBytes);
    constexpr uint64_t kStage = kTileBytes >> 4;
    const auto scores = [&](uint32_t tmem_d, uint64_t a, uint64_t b) {  // one thread
  #pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        const uint64_t off = uint64_t(((k / 4) * kSlabBytes + (k % 4) * 32) >> 4);
        umma_f16(tmem_d, a + off, b + off, idesc_s, k > 0 ? 1u : 0u);
      }
    };
    // The two halves of the softmax warps leave their 64 keys over their own columns.
    const auto add_dq = [&](int jj, bool first) {
      const int st = jj % kDqKStages;
      ok = ok && warp_wait(&ds_full[jj & 1], (jj >> 1) & 1);
      if (!ok) return;
      tc_fence_after();
      const uint64_t b = dk_mn + st * kStage;
      const uint32_t a = tmem_dp + 128 * (jj & 1);
      if (elect_one()) {
  #pragma unroll
        for (int k = 0; k < kTile / 16; ++k)
          umma_f16_ts(tmem_dq, a + (k / 4) * 64 + (k % 4) * 8, b + uint64_t((2048 * k) >> 4), idesc_dq,
                      (!first || k > 0) ? 1u : 0u);
        umma_commit(&k_empty[st]);
      }
      __syncwarp();
    };
    for (int r = 0; unit >= 0 && ok; ++r) {
      const int after = nth_unit(r + 1, p.units);
      const int4 next = after >= 0 ? __ldg(p.tiles + after / p.heads) : entry;
      const int n = steps_of(entry);
      for (int i = 0; i < n && ok; ++i, ++j) {
        const int st = j % kDqKStages, vst = j % kDqVStages;
        if (i == 0) {
          ok = warp_wait(q_full, uses & 1);
          ++uses;
        }
        ok = ok && warp_wait(&k_full[st], (j / kDqKStages) & 1);
        ok = ok && (j == 0 || warp_wait(s_read, (j - 1) & 1));
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          scores(tmem_s, dq, dk + st * kStage);
          umma_commit(s_full);
        }
        __syncwarp();
        ok = warp_wait(&v_full[vst], (j / kDqVStages) & 1);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          scores(tmem_dp + 128 * (j & 1), dg, dv + vst * kStage);
          umma_commit(&dp_full[j & 1]);
          umma_commit(&v_empty[vst]);
          if (i == n - 1) umma_commit(q_empty);
        }
        __syncwarp();
        if (i > 0) add_dq(j - 1, i == 1);
      }
      if (n > 0 && ok) {
        add_dq(j - 1, n == 1);
        if (ok && elect_one()) umma_commit(dq_full);
        __syncwarp();
      }
      unit = after;
      entry = next;
    }
    if (!ok && lane == 0) record_give_up(status, p.gave_up, kStatusTimeoutMma);
  } else {
    using T = typename Type16<FMT>::T;
    const int half = warp >> 2, quad = warp & 3;
    const int tile_row = quad * 32 + lane;
    const uint32_t lane_base = uint32_t(quad * 32) << 16;
    const uint32_t ts = tmem_s + lane_base + 64 * half;
    const float c = p.scale * kPackedLog2e;
    bool ok = true, bad = false;
    int j = 0, count = 0;
    // fp16: what bounds dS of a unit.  Only the document of the warp's first row began before its 32 rows, and the groups
    // of 32 that it comes through end with it.
    float row_do = 0.f, own_v = 0.f, before_v = 0.f;
    const auto fetch_bounds = [&](const int4& e, int u) {
      if (FMT != 0 || u < 0 || steps_of(e) == 0) return;
      const int row32 = e.x + quad * 32, begin = row32 < p.valid ? __ldg(p.first_key + row32) : row32;
      const float* doc_v = p.doc_v + long(u % p.heads / group) * p.pitch;
      row_do = p.row_do[long(u % p.heads) * p.pitch + row32 + lane];
      own_v = doc_v[row32 + lane];
      before_v = 0.f;
      for (int r32 = (begin & ~31) + 32 * lane; r32 < row32; r32 += 1024) before_v = fmaxf(before_v, doc_v[r32 + 31]);
    };
    fetch_bounds(entry, unit);
    for (int r = 0; unit >= 0 && ok; ++r) {
      const int after = nth_unit(r + 1, p.units);
      const int4 next = after >= 0 ? __ldg(p.tiles + after / p.heads) : entry;
      const int head = unit % p.heads, n = steps_of(entry);
      const int warp_row0 = entry.x + quad * 32, row = warp_row0 + lane;
      const bool in = row < p.valid;
      const long at = (long(row) * p.heads + head) * p.dim;
      const int first = in ? __ldg(p.first_key + row) : 0x7fffffff;
      const int all_from = __shfl_sync(0xffffffffu, first, 31), any_from = __shfl_sync(0xffffffffu, first, 0);

      float neg_delta = 0.f, bias2 = -INFINITY, factor = 1.f;
      if (n > 0) {
        ok = warp_wait(q_full, count & 1);
        if (!ok) break;
        neg_delta = row_values[tile_row];
        bias2 = in ? row_values[kTile + tile_row] : -INFINITY;
        if (FMT == 0) {
          const float before = warp_max(before_v);
          factor = power_for(row_do * (first < warp_row0 ? fmaxf(own_v, before) : own_v) + fabsf(neg_delta));
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(q_empty);
      }
      const float ds_factor = FMT == 0 ? factor * (1.f / 1024.f) : 1.f;
      const bool lone = first == row;  // one key: P = 1, and nothing goes through the softmax
      const float2 c2 = make_float2(c, c), b2 = make_float2(bias2, bias2), d2 = make_float2(neg_delta, neg_delta);
      const float2 f2 = make_float2(ds_factor, ds_factor);

      for (int i = 0; i < n; ++i, ++j) {
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(s_full, j & 1));
        if (!ok) break;
        tc_fence_after();
        uint32_t s[2][32];
        tmem_ld_32(ts, s[0]);
        tmem_ld_32(ts + 32, s[1]);
        tmem_ld_wait();
        pin_32(s[0]);
        pin_32(s[1]);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_read);
        const int key = entry.y + i * kTile + 64 * half;  // first key of this half
        const bool masked = key + 63 > warp_row0 || key < all_from;
        // Chunks of 32 keys that some row of the warp attends: [g0, g1).  With short documents they are few.
        const int g0 = masked ? max(any_from - key, 0) >> 5 : 0, g1 = masked ? ((warp_row0 + 31 - key) >> 5) + 1 : 2;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          if (g < g0 || g >= g1) continue;
#pragma unroll
          for (int e = 0; e < 32; e += 2) prob_pair(s[g][e], s[g][e + 1], c2, b2);
        }
        const uint32_t tp = tmem_dp + 128 * (j & 1) + lane_base + 64 * half;
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(&dp_full[j & 1], (j >> 1) & 1));
        if (!ok) break;
        tc_fence_after();
        const int from = lone ? 0x7fffffff : first - key, upto = row - key;
        uint32_t d[2][32];
        tmem_ld_32(tp, d[0]);
        tmem_ld_32(tp + 32, d[1]);
        tmem_ld_wait();
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          pin_32(d[g]);
          if (g < g0 || g >= g1) {
            tmem_st_zero_16(tp + 16 * g);
            continue;
          }
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float2 x = score_gradient<FMT>(s[g][e], s[g][e + 1], d[g][e], d[g][e + 1], d2, f2);
            d[g][e] = __float_as_uint(x.x);
            d[g][e + 1] = __float_as_uint(x.y);
          }
          if (masked) hide(d[g], bit_range(from - 32 * g, upto - 32 * g), 0u);
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) w[e] = pack16<FMT>(__uint_as_float(d[g][2 * e]), __uint_as_float(d[g][2 * e + 1]));
          tmem_st_16(tp + 16 * g, w);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ds_full[j & 1]);
      }
      if (!ok) break;
      const bool some = in && first <= row;
      unit = after;
      entry = next;
      fetch_bounds(entry, unit);  // under what is left of this unit
      T* dst = static_cast<T*>(p.dq) + at;
      if (n > 0) {
        ok = warp_wait(dq_full, count & 1);
        ++count;
        if (!ok) break;
        tc_fence_after();
        // each of the two threads of a row stores one half of the features
        bad |= store_row<FMT, DP>(tmem_dq + lane_base, p.scale / factor, dst, p.dim, some, half);
        tc_fence_before();
      }
      if (!some && row < p.rows && half == 0)
        for (int d = 0; d < p.dim; d += 8) *reinterpret_cast<uint4*>(dst + d) = make_uint4(0, 0, 0, 0);
    }
    if (!ok && lane == 0) record_give_up(status, p.gave_up, kStatusTimeoutEpilogue);
    if (ok && __any_sync(0xffffffffu, bad)) {
      __syncwarp();  // the lanes' rows are read by all
      for (int r = 0; (unit = nth_unit(r, p.units)) >= 0; ++r) {
        const int row0 = p.tiles[unit / p.heads].x, begin = row0 + quad * 32;
        for (int row = begin; row < min(begin + 32, p.valid); ++row)
          exact_dq_row<FMT, DP>(p, row0, row, unit % p.heads, half, lane);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---- dK, dV ---------------------------------------------------------------------------
//
// A unit is 128 key rows of one key head: it goes through the query tiles that may attend them, for
// one head of the group after the other.  Scores are transposed, keys along the lanes:
//   S^T = k q^T -> P^T in 16 bits over S^T -> dV += P^T do;   dP^T = v do^T -> dS^T over dP^T -> dK += dS^T q.
// The tensor core takes dV of step j, S^T of j + 1, dK of j, dP^T of j + 1: the softmax warps turn S^T into
// P^T under dK and dP^T, and dP^T into dS^T under dV and S^T.
//
// TMEM: dV, dK (up to 128 columns each), S^T, dP^T (128 each).  Shared memory: k, v, three query tiles,
// two tiles of do with the rows' bias2 and delta.  Warps 0-7: softmax, warps 0-3 on the first 64
// queries of a tile, 4-7 on the rest; two threads share a key.  8 TMA, 9 MMA.
//
// Bound like dQ, with four products: 0.90 ms at the same sizes (1220 TFLOP/s of its four products).

constexpr int kDkvQStages = 3;
constexpr int kDkvGStages = 2;
constexpr int kDkvRowBytes = 2 * kTile * 4;  // bias2 and delta of a query tile

template <int DP>
constexpr int dkv_smem_bytes() {
  return (2 + kDkvQStages + kDkvGStages) * tile_bytes<DP>() + kDkvGStages * kDkvRowBytes + 512;
}

// A block of dK, dV that came early holds its TMEM until all of dQ has ended.  A block of dQ that had to wait for it on
// the same SM would wait for good, so there is no room for both (228 KB to an SM, 1 KB of them kept for each block).
static_assert(dq_smem_bytes<64>() + dkv_smem_bytes<64>() + 2 * 1024 > 228 * 1024, "dQ and dK, dV must not share an SM");

// A warp puts right a row of dV (half 0) or of dK, of the tile of keys whose queries are [row0, last).
template <int FMT, int DP>
__device__ __noinline__ void exact_dkv_row(const PackedBwdArgs& p, int row0, int last, int key, int kv, int half, int lane) {
  using T = typename Type16<FMT>::T;
  const int group = p.heads / p.kv_heads, end = p.end_query[key], first = p.first_key[key];
  T* dst = static_cast<T*>(half ? p.dk : p.dv) + (long(key) * p.kv_heads + kv) * p.dim;
  float k[DP / 32], v[DP / 32], sum[DP / 32] = {};
  load_row<FMT, DP>(k, dst, 0, p.dim, lane);
  bool bad = false;
#pragma unroll
  for (int e = 0; e < DP / 32; ++e) bad |= !(fabsf(k[e]) < INFINITY);
  if (!__any_sync(0xffffffffu, bad)) return;
  // A document that ends in the tile is short there; the others are left with few rows that do not attend them.
  if (end > row0 + kTile) {
    bad = false;
    for (int head = kv * group; head < (kv + 1) * group && !bad; ++head) {
      const void* x = half ? p.q : p.d_o;
      const long tok = half ? p.q_tok : p.do_tok, off = long(head) * (half ? p.q_head : p.do_head);
      bad = some_not_finite<FMT, DP>(x, tok, off, row0, key, p.dim, lane) ||
            some_not_finite<FMT, DP>(x, tok, off, end, min(last, p.valid), p.dim, lane);
    }
    if (!bad) return;
  }
  const float c = p.scale * kPackedLog2e;
  load_row<FMT, DP>(k, p.k, long(key) * p.k_tok + long(kv) * p.k_head, p.dim, lane);
  load_row<FMT, DP>(v, p.v, long(key) * p.v_tok + long(kv) * p.v_head, p.dim, lane);
  const int begin = half && key == first ? key + 1 : key;  // a document's first row has a single key, and no dS
  for (int head = kv * group; head < (kv + 1) * group; ++head) {
    const long at = long(head) * p.pitch;
    for (int i0 = begin; i0 < end && !all_nan(sum, 0, p.dim, lane); i0 += 64) {
#pragma unroll 4
      for (int row = i0; row < min(i0 + 64, end); ++row) {
        float q[DP / 32], g[DP / 32];
        load_row<FMT, DP>(q, p.q, long(row) * p.q_tok + long(head) * p.q_head, p.dim, lane);
        load_row<FMT, DP>(g, p.d_o, long(row) * p.do_tok + long(head) * p.do_head, p.dim, lane);
        float w = exp2f(warp_dot(q, k) * c + (p.bias2[at + row] - p_shift<FMT>()));
        if (half) w *= warp_dot(g, v) + p.neg_delta[at + row];
#pragma unroll
        for (int e = 0; e < DP / 32; ++e) sum[e] = fmaf(w, half ? q[e] : g[e], sum[e]);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < DP / 32; ++e)
    if (lane + 32 * e < p.dim) dst[lane + 32 * e] = from_float<T>(half ? sum[e] * p.scale : sum[e]);
}

template <int FMT, int DP>
__global__ void __launch_bounds__(kBwdThreads, 1)
packed_dkv_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                  const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                  const __grid_constant__ PackedBwdArgs p, int* status) {
  constexpr int kTileBytes = tile_bytes<DP>();
  constexpr int kSlabs = DP / 64;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  // All of the shared memory is in use at 128 features: there is no room for moving up to a boundary.
  if ((smem_u32(smem_raw) & 1023u) != 0) {
    if (threadIdx.x == 0) record_give_up(status, p.gave_up, kStatusTimeoutProducer);
    return;
  }
  uint8_t* k_tile = smem_raw;
  uint8_t* v_tile = k_tile + kTileBytes;
  uint8_t* q_tiles = v_tile + kTileBytes;
  uint8_t* g_tiles = q_tiles + kDkvQStages * kTileBytes;
  float* row_values = reinterpret_cast<float*>(g_tiles + kDkvGStages * kTileBytes);  // [stage][bias2, -delta][128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(row_values) + kDkvGStages * kDkvRowBytes);
  uint64_t* k_full = bars;
  uint64_t* k_empty = k_full + 1;
  uint64_t* v_full = k_empty + 1;
  uint64_t* v_empty = v_full + 1;
  uint64_t* q_full = v_empty + 1;            // [3]
  uint64_t* q_empty = q_full + kDkvQStages;  // [3]
  uint64_t* g_full = q_empty + kDkvQStages;  // [2]
  uint64_t* g_empty = g_full + kDkvGStages;  // [2]
  uint64_t* s_full = g_empty + kDkvGStages;
  uint64_t* p_full = s_full + 1;
  uint64_t* dp_full = p_full + 1;
  uint64_t* ds_full = dp_full + 1;
  uint64_t* done = ds_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = p.heads / p.kv_heads;

  if (threadIdx.x == 0) {
    mbar_init(k_full, 1);
    mbar_init(k_empty, 1);
    mbar_init(v_full, 1);
    mbar_init(v_empty, 1);
    for (int s = 0; s < kDkvQStages; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], 1);
    }
    for (int s = 0; s < kDkvGStages; ++s) {
      mbar_init(&g_full[s], 1);
      mbar_init(&g_empty[s], 9);  // commit and 8 softmax warps
    }
    mbar_init(s_full, 1);
    mbar_init(p_full, 8);
    mbar_init(dp_full, 1);
    mbar_init(ds_full, 8);
    mbar_init(done, 1);
    fence_barrier_init();
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_do);
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  wait_for_last_kernel();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tmem_dv = tmem, tmem_dk = tmem + 128, tmem_s = tmem + 256, tmem_dp = tmem + 384;

  int unit = nth_unit(0, p.units);
  int4 entry = unit >= 0 ? __ldg(p.tiles + unit / p.kv_heads) : make_int4(0, 0, 0, 0);
  const auto tiles_of = [](const int4& e) { return (e.y - e.x + kTile - 1) / kTile; };  // query tiles of a head

  if (warp == 8) {
    if (lane == 0) {
      bool ok = true;
      int base = 0, uses = 0;
      for (int r = 0; unit >= 0 && ok; ++r) {
        const int after = nth_unit(r + 1, p.units);
        const int4 next = after >= 0 ? __ldg(p.tiles + after / p.kv_heads) : entry;
        const int kv_head = unit % p.kv_heads, per_head = tiles_of(entry), n = per_head * group;
        for (int i = 0; i < n && ok; ++i) {
          const int j = base + i;
          const int h = kv_head * group + i / per_head, q0 = entry.x + (i % per_head) * kTile;
          const int qs = j % kDkvQStages, gs = j % kDkvGStages;
          if (i == 0) {
            ok = mbar_wait_bounded(k_empty, (uses & 1) ^ 1);
            if (!ok) break;
            mbar_expect_tx(k_full, kTileBytes);
#pragma unroll
            for (int s = 0; s < kSlabs; ++s)
              tma_load_3d(k_tile + s * kSlabBytes, &map_k, k_full, 64 * s, kv_head, entry.x);
          }
          ok = mbar_wait_bounded(&q_empty[qs], ((j / kDkvQStages) & 1) ^ 1);
          if (!ok) break;
          mbar_expect_tx(&q_full[qs], kTileBytes);
#pragma unroll
          for (int s = 0; s < kSlabs; ++s)
            tma_load_3d(q_tiles + qs * kTileBytes + s * kSlabBytes, &map_q, &q_full[qs], 64 * s, h, q0);
          if (i == 0) {
            ok = mbar_wait_bounded(v_empty, (uses & 1) ^ 1);
            if (!ok) break;
            ++uses;
            mbar_expect_tx(v_full, kTileBytes);
#pragma unroll
            for (int s = 0; s < kSlabs; ++s)
              tma_load_3d(v_tile + s * kSlabBytes, &map_v, v_full, 64 * s, kv_head, entry.x);
          }
          ok = mbar_wait_bounded(&g_empty[gs], ((j / kDkvGStages) & 1) ^ 1);
          if (!ok) break;
          mbar_expect_tx(&g_full[gs], kTileBytes + kDkvRowBytes);
#pragma unroll
          for (int s = 0; s < kSlabs; ++s)
            tma_load_3d(g_tiles + gs * kTileBytes + s * kSlabBytes, &map_do, &g_full[gs], 64 * s, h, q0);
          // bias2 and delta have whole tiles of rows to a head, so the copies stay inside
          bulk_load(row_values + gs * 2 * kTile, p.bias2 + long(h) * p.pitch + q0, kTile * 4, &g_full[gs]);
          bulk_load(row_values + gs * 2 * kTile + kTile, p.neg_delta + long(h) * p.pitch + q0, kTile * 4, &g_full[gs]);
        }
        base += n;
        unit = after;
        entry = next;
      }
      if (!ok) {
        record_give_up(status, p.gave_up, kStatusTimeoutProducer);
        drain_copies();
      }
    }
    __syncwarp();
  } else if (warp == 9) {
    constexpr uint32_t idesc_s = make_idesc_f16(kTile, kTile, FMT, 0, 0);
    constexpr uint32_t idesc_d = make_idesc_f16(kTile, DP, FMT, 0, 1);
    bool ok = true;
    const uint64_t dk = make_kmajor_sw128_desc(smem_u32(k_tile)), dv = make_kmajor_sw128_desc(smem_u32(v_tile));
    const uint64_t dq = make_kmajor_sw128_desc(smem_u32(q_tiles)), dg = make_kmajor_sw128_desc(smem_u32(g_tiles));
    const uint64_t dq_mn = make_mnmajor_sw128_desc(smem_u32(q_tiles), kSlabBytes);
    const uint64_t dg_mn = make_mnmajor_sw128_desc(smem_u32(g_tiles), kSlabBytes);
    constexpr uint64_t kStage = kTileBytes >> 4;
    const auto scores = [&](uint32_t tmem_d, uint64_t a, uint64_t b) {  // one thread
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        const uint64_t off = uint64_t(((k / 4) * kSlabBytes + (k % 4) * 32) >> 4);
        umma_f16(tmem_d, a + off, b + off, idesc_s, k > 0 ? 1u : 0u);
      }
    };
    // The two halves of the softmax warps leave their 64 queries over their own columns.
    const auto add = [&](uint32_t tmem_d, uint32_t tmem_a, uint64_t b, bool first) {  // one thread
#pragma unroll
      for (int k = 0; k < kTile / 16; ++k)
        umma_f16_ts(tmem_d, tmem_a + (k / 4) * 64 + (k % 4) * 8, b + uint64_t((2048 * k) >> 4), idesc_d,
                    (!first || k > 0) ? 1u : 0u);
    };
    int base = 0, uses = 0;
    for (int r = 0; unit >= 0 && ok; ++r) {
      const int after = nth_unit(r + 1, p.units);
      const int4 next = after >= 0 ? __ldg(p.tiles + after / p.kv_heads) : entry;
      const int n = tiles_of(entry) * group;
      const auto first_product = [&](int i) {
        const int j = base + i, qs = j % kDkvQStages;
        ok = ok && warp_wait(&q_full[qs], (j / kDkvQStages) & 1);
        if (!ok) return;
        tc_fence_after();
        if (elect_one()) {
          scores(tmem_s, dk, dq + qs * kStage);
          umma_commit(s_full);
          if (i == n - 1) umma_commit(k_empty);
        }
        __syncwarp();
      };
      const auto third_product = [&](int i) {
        const int j = base + i, gs = j % kDkvGStages;
        ok = ok && warp_wait(&g_full[gs], (j / kDkvGStages) & 1);
        if (!ok) return;
        tc_fence_after();
        if (elect_one()) {
          scores(tmem_dp, dv, dg + gs * kStage);
          umma_commit(dp_full);
          if (i == n - 1) umma_commit(v_empty);
        }
        __syncwarp();
      };
      if (n > 0) {
        ok = warp_wait(k_full, uses & 1);
        first_product(0);
        ok = ok && warp_wait(v_full, uses & 1);
        third_product(0);
        ++uses;
      }
      for (int i = 0; i < n && ok; ++i) {
        const int j = base + i;
        const int qs = j % kDkvQStages, gs = j % kDkvGStages;
        ok = warp_wait(p_full, j & 1);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          add(tmem_dv, tmem_s, dg_mn + gs * kStage, i == 0);
          umma_commit(&g_empty[gs]);
        }
        __syncwarp();
        if (i + 1 < n) first_product(i + 1);
        ok = ok && warp_wait(ds_full, j & 1);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          add(tmem_dk, tmem_dp, dq_mn + qs * kStage, i == 0);
          umma_commit(&q_empty[qs]);
          if (i == n - 1) umma_commit(done);
        }
        __syncwarp();
        if (i + 1 < n) third_product(i + 1);
      }
      base += n;
      unit = after;
      entry = next;
    }
    if (!ok && lane == 0) record_give_up(status, p.gave_up, kStatusTimeoutMma);
  } else {
    using T = typename Type16<FMT>::T;
    const int half = warp >> 2, quad = warp & 3;
    const uint32_t lane_base = uint32_t(quad * 32) << 16;
    const uint32_t ts = tmem_s + lane_base + 64 * half, tp = tmem_dp + lane_base + 64 * half;
    const float c = p.scale * kPackedLog2e;
    const float2 c2 = make_float2(c, c);
    bool ok = true, bad = false;
    int j = 0, count = 0;
    for (int r = 0; unit >= 0 && ok; ++r) {
      const int after = nth_unit(r + 1, p.units);
      const int4 next = after >= 0 ? __ldg(p.tiles + after / p.kv_heads) : entry;
      const int kv_head = unit % p.kv_heads, per_head = tiles_of(entry), n = per_head * group;
      const int warp_key0 = entry.x + quad * 32, key = warp_key0 + lane;
      const bool in = key < p.valid;
      const int end = in ? __ldg(p.end_query + key) : 0;
      const bool opens = in && __ldg(p.first_key + key) == key;  // its own row attends nothing else
      const int min_end = __reduce_min_sync(0xffffffffu, end), max_end = __reduce_max_sync(0xffffffffu, end);
      // fp16: what bounds dS.  Only the document of the warp's last key goes on behind its 32 rows, and every later
      // group of 32 that it reaches begins with it.  (Asked for under the end of the unit before, as in dQ: 37 instead
      // of 41 us for 211 facts of 12 heads of 64, but 56 instead of 51 for 16 over 2 heads.)
      float factor = 1.f;
      if (FMT == 0 && n > 0) {
        const int behind = warp_key0 + 32, later = max(__shfl_sync(0xffffffffu, end, 31) - behind + 31, 0) >> 5;
        const long head0 = long(kv_head) * group * p.pitch;
        float size = 0.f, delta = 0.f, later_size = 0.f, later_delta = 0.f;
#pragma unroll 4
        for (int h = 0; h < group; ++h) {
          size = fmaxf(size, p.doc_do[head0 + long(h) * p.pitch + key]);
          delta = fmaxf(delta, p.doc_delta[head0 + long(h) * p.pitch + key]);
        }
#pragma unroll 4
        for (int x = lane; x < later * group; x += 32) {
          const long from = head0 + long(x / later) * p.pitch + behind + 32 * (x % later);
          later_size = fmaxf(later_size, p.doc_do[from]);
          later_delta = fmaxf(later_delta, p.doc_delta[from]);
        }
        if (later > 0) {
          later_size = warp_max(later_size);
          later_delta = warp_max(later_delta);
          if (end > behind) {
            size = fmaxf(size, later_size);
            delta = fmaxf(delta, later_delta);
          }
        }
        factor = power_for(size * p.doc_v[long(kv_head) * p.pitch + key] + delta);
      }
      const float ds_factor = FMT == 0 ? factor * (1.f / 1024.f) : 1.f;
      const float2 f2 = make_float2(ds_factor, ds_factor);
      for (int i = 0; i < n; ++i, ++j) {
        const int gs = j % kDkvGStages;
        const int q0 = entry.x + (i % per_head) * kTile + 64 * half;  // first query of this half
        ok = mbar_wait_bounded(&g_full[gs], (j / kDkvGStages) & 1);
        ok = mbar_wait_bounded(s_full, j & 1) && ok;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const bool masked = q0 < warp_key0 + 31 || q0 + 64 > min_end;
        const int from = key - q0, upto = end - 1 - q0;  // columns that attend this key
        // Chunks of 32 queries of which some attend some key of the warp: [g0, g1).
        const int g0 = masked ? max(warp_key0 - q0, 0) >> 5 : 0, g1 = masked ? ((max_end - 1 - q0) >> 5) + 1 : 2;
        const float4* bias = reinterpret_cast<const float4*>(row_values + gs * 2 * kTile + 64 * half);
        uint32_t s[2][32];
        tmem_ld_32(ts, s[0]);
        tmem_ld_32(ts + 32, s[1]);
        tmem_ld_wait();
        pin_32(s[0]);
        pin_32(s[1]);
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          if (g < g0 || g >= g1) {
            tmem_st_zero_16(ts + 16 * g);
            continue;
          }
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 x = bias[g * 8 + e / 4];
            prob_pair(s[g][e], s[g][e + 1], c2, make_float2(x.x, x.y));
            prob_pair(s[g][e + 2], s[g][e + 3], c2, make_float2(x.z, x.w));
          }
          if (masked) hide(s[g], bit_range(from - 32 * g, upto - 32 * g), 0u);
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) w[e] = pack16<FMT>(__uint_as_float(s[g][2 * e]), __uint_as_float(s[g][2 * e + 1]));
          tmem_st_16(ts + 16 * g, w);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full);

        ok = __all_sync(0xffffffffu, mbar_wait_bounded(dp_full, j & 1));
        if (!ok) break;
        tc_fence_after();
        const float4* dl = reinterpret_cast<const float4*>(row_values + gs * 2 * kTile + kTile + 64 * half);
        uint32_t d[2][32];
        tmem_ld_32(tp, d[0]);
        tmem_ld_32(tp + 32, d[1]);
        tmem_ld_wait();
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          pin_32(d[g]);
          if (g < g0 || g >= g1) {
            tmem_st_zero_16(tp + 16 * g);
            continue;
          }
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 y = dl[g * 8 + e / 4];
            const float2 x0 = score_gradient<FMT>(s[g][e], s[g][e + 1], d[g][e], d[g][e + 1], make_float2(y.x, y.y), f2);
            const float2 x1 = score_gradient<FMT>(s[g][e + 2], s[g][e + 3], d[g][e + 2], d[g][e + 3], make_float2(y.z, y.w), f2);
            d[g][e] = __float_as_uint(x0.x);
            d[g][e + 1] = __float_as_uint(x0.y);
            d[g][e + 2] = __float_as_uint(x1.x);
            d[g][e + 3] = __float_as_uint(x1.y);
          }
          // what is masked may be infinite or NaN; the first row of a document has a single key
          if (masked) hide(d[g], bit_range(from + opens - 32 * g, upto - 32 * g), 0u);
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) w[e] = pack16<FMT>(__uint_as_float(d[g][2 * e]), __uint_as_float(d[g][2 * e + 1]));
          tmem_st_16(tp + 16 * g, w);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(ds_full);
          mbar_arrive(&g_empty[gs]);  // bias2 and delta are read
        }
      }
      if (!ok) break;
      unit = after;
      entry = next;
      T* dst = static_cast<T*>(half ? p.dk : p.dv) + (long(key) * p.kv_heads + kv_head) * p.dim;
      if (n > 0) {
        ok = warp_wait(done, count & 1);
        ++count;
        if (!ok) break;
        tc_fence_after();
        const float out = half ? p.scale / factor : (FMT == 0 ? 1.f / 1024.f : 1.f);
        bad |= store_row<FMT, DP>((half ? tmem_dk : tmem_dv) + lane_base, out, dst, p.dim, in);
        tc_fence_before();
      }
      if (!in && key < p.rows)
        for (int d = 0; d < p.dim; d += 8) *reinterpret_cast<uint4*>(dst + d) = make_uint4(0, 0, 0, 0);
    }
    if (!ok && lane == 0) record_give_up(status, p.gave_up, kStatusTimeoutEpilogue);
    if (ok && __any_sync(0xffffffffu, bad)) {
      __syncwarp();  // the lanes' rows are read by all
      for (int r = 0; (unit = nth_unit(r, p.units)) >= 0; ++r) {
        const int4 e = p.tiles[unit / p.kv_heads];
        const int begin = e.x + quad * 32;
        for (int key = begin; key < min(begin + 32, p.valid); ++key)
          exact_dkv_row<FMT, DP>(p, e.x, e.x + tiles_of(e) * kTile, key, unit % p.kv_heads, half, lane);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace bgn
