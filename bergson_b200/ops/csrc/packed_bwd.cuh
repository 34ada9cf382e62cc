// Backward pass of the causal attention over packed documents on the tensor cores (fp16, bf16).
//
//   P = 2^(c q.k - lse2),  delta_t = do_t . o_t,  dS = P (do.v - delta)
//   dQ = scale dS k,   dK = scale dS^T q,   dV = P^T do      (dK, dV summed over the heads of a group)
//
// Two kernels, each of which keeps its sums in TMEM from the first to the last tile: one block for the
// rows of dQ, one for the rows of dK and dV.  P is computed in both: that is seven products for the
// five of the mathematics, and buys sums in one order (the results are the same in every run) without
// a fp32 copy of dQ in memory.  Tiles are cut from the packed axis as in the forward pass.
//
// P and dS are rounded to the operands' type for the tensor core; everything else is fp32.  fp16 has
// few small values, so there P carries a factor 2^10 and dS the power of two that brings the largest
// |do| of the rows concerned to [1/2, 1): both are taken out of the fp32 sums at the end.
//
// Blocks look for infinities and NaN in operand tiles that are partly masked and then compute their
// rows again, row by row, as the forward pass does.
#pragma once

#include "packed_fwd.cuh"

namespace bgn {

constexpr int kBwdThreads = 384;

struct PackedBwdArgs {
  const int* first_key;
  const int* end_query;
  const int* order;
  int rows, valid, heads, kv_heads, dim;
  int head_pairs;  // dQ: as in the forward pass
  int pitch;       // floats between the heads of lse2 and delta, a multiple of 128
  float scale;
  const void *q, *k, *v, *o, *d_o;
  long q_tok, q_head, k_tok, k_head, v_tok, v_head, do_tok, do_head;
  const float* lse2;
  float* delta;
  float* do_max;  // [heads, pitch / 32]: largest |do| of 32 rows (fp16)
  void *dq, *dk, *dv;
};

// fp16 only: P carries 2^10.
template <int FMT>
constexpr float p_shift() {
  return FMT == 0 ? 10.f : 0.f;
}

// The power of two that brings `top` to [1/2, 1); 1 where there is nothing to scale.
__device__ __forceinline__ float power_below_one(float top) {
  if (!(top > 0.f) || !(top < INFINITY)) return 1.f;
  const int e = int((__float_as_uint(top) >> 23) & 0xff) - 126;  // top in [2^(e-1), 2^e)
  const int f = 127 - e;
  return __uint_as_float(uint32_t(f < 1 ? 1 : (f > 253 ? 253 : f)) << 23);
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// ---- dQ -------------------------------------------------------------------------------
//
// A block has two tiles of 128 query rows, as in the forward pass, and goes through their key tiles
// step by step (a step is one key tile for one of the two):
//   S = q k^T -> softmax warps of that tile: P in registers -> dP = do v^T -> dS over dP -> dQ += dS k.
// The tensor core takes S of step n, then dQ of step n - 1, then dP of step n, so that it has work while
// the softmax warps of either tile compute.
//
// TMEM: dQ of the two tiles (256 columns), S (128), dP (128; dS in 16 bits over its first half).
// Shared memory: q and do of the two tiles, two key tiles, one value tile (7 tiles of 32 KB at 128
// features).  Warps: as in the forward pass; warps 10-11 look through partly masked key tiles.

template <int DP>
constexpr int dq_smem_bytes() {
  return 7 * tile_bytes<DP>() + 1024 + 256;
}

template <int FMT, int DP>
__device__ __noinline__ void exact_dq_row(const PackedBwdArgs& p, int row, int head, float lse2, float delta, int lane) {
  using T = typename Type16<FMT>::T;
  const int kv = head / (p.heads / p.kv_heads), first = p.first_key[row];
  const float c = p.scale * kPackedLog2e;
  float q[DP / 32], g[DP / 32], dq[DP / 32] = {};
  load_row<FMT, DP>(q, p.q, long(row) * p.q_tok + long(head) * p.q_head, p.dim, lane);
  load_row<FMT, DP>(g, p.d_o, long(row) * p.do_tok + long(head) * p.do_head, p.dim, lane);
  for (int j = first; j <= row && first < row; ++j) {
    float k[DP / 32], v[DP / 32];
    load_row<FMT, DP>(k, p.k, long(j) * p.k_tok + long(kv) * p.k_head, p.dim, lane);
    load_row<FMT, DP>(v, p.v, long(j) * p.v_tok + long(kv) * p.v_head, p.dim, lane);
    const float ds = exp2f(warp_dot(q, k) * c - lse2) * (warp_dot(g, v) - delta);
#pragma unroll
    for (int e = 0; e < DP / 32; ++e) dq[e] = fmaf(ds, k[e], dq[e]);
  }
  T* dst = static_cast<T*>(p.dq) + (long(row) * p.heads + head) * p.dim;
#pragma unroll
  for (int e = 0; e < DP / 32; ++e)
    if (lane + 32 * e < p.dim) dst[lane + 32 * e] = from_float<T>(dq[e] * p.scale);
}

template <int FMT, int DP>
__global__ void __launch_bounds__(kBwdThreads, 1)
packed_dq_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                 const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                 const __grid_constant__ PackedBwdArgs p, int* status) {
  constexpr int kTileBytes = tile_bytes<DP>();
  constexpr int kSlabs = DP / 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* q_tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* g_tiles = q_tiles + 2 * kTileBytes;
  uint8_t* k_tiles = g_tiles + 2 * kTileBytes;  // two
  uint8_t* v_tile = k_tiles + 2 * kTileBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(v_tile + kTileBytes);
  uint64_t* q_full = bars;         // [2]: q and do of a tile
  uint64_t* k_full = q_full + 2;   // [2]
  uint64_t* k_empty = k_full + 2;  // [2]
  uint64_t* v_full = k_empty + 2;
  uint64_t* v_empty = v_full + 1;
  uint64_t* s_full = v_empty + 1;   // [2] per tile, as the following
  uint64_t* s_read = s_full + 2;
  uint64_t* dp_full = s_read + 2;
  uint64_t* ds_full = dp_full + 2;
  uint64_t* dq_full = ds_full + 2;  // [1]
  uint64_t* checked = dq_full + 1;  // [1]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(checked + 1);
  int* poison = reinterpret_cast<int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  int row0[2], head[2];
  {
    const int per = p.head_pairs ? p.heads / 2 : p.heads;
    const int slot = __ldg(p.order + blockIdx.x / per), h = blockIdx.x % per;
    if (p.head_pairs) {
      row0[0] = row0[1] = slot * kTile;
      head[0] = 2 * h;
      head[1] = 2 * h + 1;
    } else {
      row0[0] = 2 * slot * kTile;
      row0[1] = row0[0] + kTile;
      head[0] = head[1] = h;
    }
  }
  const int kv_head = head[0] / (p.heads / p.kv_heads);
  KeyRange range[2] = {key_range(p.first_key, row0[0], p.valid), key_range(p.first_key, row0[1], p.valid)};
  const bool some0 = range[0].hi > range[0].lo, some1 = range[1].hi > range[1].lo;
  const int base = some0 ? (some1 ? min(range[0].lo, range[1].lo) : range[0].lo) : range[1].lo;
  int i0[2], i1[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const bool some = t ? some1 : some0;
    i0[t] = some ? (range[t].lo - base) / kTile : 0;
    i1[t] = some ? (range[t].hi - base + kTile - 1) / kTile : 0;
  }
  const int n = max(i1[0], i1[1]);

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], 1);
      mbar_init(&k_full[t], 1);
      mbar_init(&k_empty[t], 3);  // the MMA warp's commit and the two looking warps
      mbar_init(&s_full[t], 1);
      mbar_init(&s_read[t], 4);
      mbar_init(&dp_full[t], 1);
      mbar_init(&ds_full[t], 4);
    }
    mbar_init(v_full, 1);
    mbar_init(v_empty, 1);
    mbar_init(dq_full, 1);
    mbar_init(checked, 2);
    *poison = 0;
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
  const uint32_t tmem = *tmem_slot;
  const uint32_t tmem_s = tmem + 256, tmem_dp = tmem + 384;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");  // 3 * 168 >= 2 * 208 + 80
    if (warp == 8) {
      if (lane == 0) {
        bool ok = true;
        for (int t = 0; t < 2; ++t) {
          if (i1[t] == 0) continue;
          mbar_expect_tx(&q_full[t], 2 * kTileBytes);
#pragma unroll
          for (int s = 0; s < kSlabs; ++s) {
            tma_load_3d(q_tiles + t * kTileBytes + s * kSlabBytes, &map_q, &q_full[t], 64 * s, head[t], row0[t]);
            tma_load_3d(g_tiles + t * kTileBytes + s * kSlabBytes, &map_do, &q_full[t], 64 * s, head[t], row0[t]);
          }
        }
        for (int i = 0; i < n && ok; ++i) {
          const int st = i & 1, key = base + i * kTile;
          ok = mbar_wait_bounded(&k_empty[st], ((i >> 1) & 1) ^ 1);
          if (!ok) break;
          mbar_expect_tx(&k_full[st], kTileBytes);
#pragma unroll
          for (int s = 0; s < kSlabs; ++s)
            tma_load_3d(k_tiles + st * kTileBytes + s * kSlabBytes, &map_k, &k_full[st], 64 * s, kv_head, key);
          ok = mbar_wait_bounded(v_empty, (i & 1) ^ 1);
          if (!ok) break;
          mbar_expect_tx(v_full, kTileBytes);
#pragma unroll
          for (int s = 0; s < kSlabs; ++s)
            tma_load_3d(v_tile + s * kSlabBytes, &map_v, v_full, 64 * s, kv_head, key);
        }
        if (!ok) {
          atomicCAS(status, kStatusOk, kStatusTimeoutProducer);
          drain_copies();
        }
      }
      __syncwarp();
    } else if (warp == 9) {
      constexpr uint32_t idesc_s = make_idesc_f16(kTile, kTile, FMT, 0, 0);
      constexpr uint32_t idesc_dq = make_idesc_f16(kTile, DP, FMT, 0, 1);
      if (lane == 0 && n > 0) {
        bool ok = true;
        int prev_t = -1, prev_i = 0;
        const auto add_dq = [&](int t, int i) {  // dQ of a finished step
          ok = ok && mbar_wait_bounded(&ds_full[t], (i - i0[t]) & 1);
          if (!ok) return;
          tc_fence_after();
          const uint64_t dk = make_mnmajor_sw128_desc(smem_u32(k_tiles + (i & 1) * kTileBytes), kSlabBytes);
#pragma unroll
          for (int k = 0; k < kTile / 16; ++k)
            umma_f16_ts(tmem + 128 * t, tmem_dp + 8 * k, dk + uint64_t((2048 * k) >> 4), idesc_dq,
                        (i > i0[t] || k > 0) ? 1u : 0u);
        };
        for (int i = 0; i < n && ok; ++i) {
          const uint32_t k_addr = smem_u32(k_tiles + (i & 1) * kTileBytes);
          ok = mbar_wait_bounded(&k_full[i & 1], (i >> 1) & 1);
          bool v_there = false;
          for (int t = 0; t < 2 && ok; ++t) {
            if (i < i0[t] || i >= i1[t]) continue;
            if (i == i0[t]) ok = mbar_wait_bounded(&q_full[t], 0);
            if (prev_t >= 0) ok = ok && mbar_wait_bounded(&s_read[prev_t], (prev_i - i0[prev_t]) & 1);
            if (!ok) break;
            tc_fence_after();
            const uint64_t dq = make_kmajor_sw128_desc(smem_u32(q_tiles + t * kTileBytes));
            const uint64_t dk = make_kmajor_sw128_desc(k_addr);
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
              const uint64_t off = uint64_t(((k / 4) * kSlabBytes + (k % 4) * 32) >> 4);
              umma_f16(tmem_s, dq + off, dk + off, idesc_s, k > 0 ? 1u : 0u);
            }
            umma_commit(&s_full[t]);
            if (prev_t >= 0) {
              add_dq(prev_t, prev_i);
              if (!ok) break;
              if (prev_i < i) umma_commit(&k_empty[prev_i & 1]);
            }
            if (!v_there) {
              ok = mbar_wait_bounded(v_full, i & 1);
              if (!ok) break;
              v_there = true;
            }
            tc_fence_after();
            const uint64_t dg = make_kmajor_sw128_desc(smem_u32(g_tiles + t * kTileBytes));
            const uint64_t dv = make_kmajor_sw128_desc(smem_u32(v_tile));
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
              const uint64_t off = uint64_t(((k / 4) * kSlabBytes + (k % 4) * 32) >> 4);
              umma_f16(tmem_dp, dg + off, dv + off, idesc_s, k > 0 ? 1u : 0u);
            }
            umma_commit(&dp_full[t]);
            prev_t = t;
            prev_i = i;
          }
          if (ok) umma_commit(v_empty);
        }
        if (ok) add_dq(prev_t, prev_i);
        if (ok) umma_commit(dq_full);
        if (!ok) atomicCAS(status, kStatusOk, kStatusTimeoutMma);
      }
      __syncwarp();
    } else {
      bool bad = false, ok = true;
      for (int i = 0; i < n && ok; ++i) {
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(&k_full[i & 1], (i >> 1) & 1));
        const int key = base + i * kTile;
        bool masked = false;
#pragma unroll
        for (int t = 0; t < 2; ++t)
          masked |= i >= i0[t] && i < i1[t] && (key + kTile - 1 > row0[t] || key < range[t].last_first);
        if (masked && ok) bad |= scan_not_finite<FMT>(k_tiles + (i & 1) * kTileBytes, kTileBytes, warp - 10, 2, lane);
        __syncwarp();
        if (lane == 0) mbar_arrive(&k_empty[i & 1]);
      }
      if (__any_sync(0xffffffffu, bad) && lane == 0) *poison = 1;
      __syncwarp();
      if (lane == 0) mbar_arrive(checked);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    using T = typename Type16<FMT>::T;
    const int t = warp >> 2, quad = warp & 3;
    const int my_i0 = t ? i0[1] : i0[0], my_i1 = t ? i1[1] : i1[0];
    const int warp_row0 = (t ? row0[1] : row0[0]) + quad * 32, my_head = t ? head[1] : head[0];
    const int row = warp_row0 + lane, tile_row = quad * 32 + lane;
    const bool in = row < p.valid;
    const int first = in ? __ldg(p.first_key + row) : 0x7fffffff;
    const int all_from = __shfl_sync(0xffffffffu, in ? first : 0x7fffffff, 31);
    const uint32_t lane_base = uint32_t(quad * 32) << 16;
    const uint32_t ts = tmem_s + lane_base, tp = tmem_dp + lane_base;
    const float c = p.scale * kPackedLog2e;
    const float lse2 = in ? p.lse2[long(my_head) * p.pitch + row] : INFINITY;
    bool ok = true;

    // delta = do . o; do from the tile in shared memory (swizzled rows of 128 bytes).
    float delta = 0.f, top = 0.f;
    if (my_i1 > my_i0) {
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(&q_full[t], 0));
      if (ok && in) {
        const uint8_t* g = g_tiles + t * kTileBytes + tile_row * 128;
        const T* orow = static_cast<const T*>(p.o) + (long(row) * p.heads + my_head) * p.dim;
#pragma unroll 4
        for (int d = 0; d < p.dim; d += 8) {
          union { uint4 u; T h[8]; } a, b;
          a.u = *reinterpret_cast<const uint4*>(orow + d);
          b.u = *reinterpret_cast<const uint4*>(g + (d / 64) * kSlabBytes + ((((d % 64) / 8) ^ (tile_row & 7)) << 4));
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float x = to_float<T>(b.h[e]);
            delta = fmaf(to_float<T>(a.h[e]), x, delta);
            top = fmaxf(top, fabsf(x));
          }
        }
      }
    }
    if (row < p.rows) p.delta[long(my_head) * p.pitch + row] = delta;
    float factor = 1.f;
    if (FMT == 0) {
      top = warp_max(top);
      if (lane == 0 && warp_row0 < p.pitch) p.do_max[(long(my_head) * p.pitch + warp_row0) / 32] = top;
      factor = power_below_one(top);
    }
    const float base2 = -(lse2 - p_shift<FMT>());
    const float ds_factor = FMT == 0 ? factor * (1.f / 1024.f) : 1.f;
    const bool lone = first == row;  // one key: P = 1, and nothing goes through the softmax

    for (int i = my_i0; i < my_i1 && ok; ++i) {
      const int parity = (i - my_i0) & 1;
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(&s_full[t], parity));
      if (!ok) break;
      tc_fence_after();
      uint32_t s[4][32];
#pragma unroll
      for (int g = 0; g < 4; ++g) tmem_ld_32(ts + 32 * g, s[g]);
      tmem_ld_wait();
#pragma unroll
      for (int g = 0; g < 4; ++g) pin_32(s[g]);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_read[t]);
      const int key = base + i * kTile;
      const bool masked = key + kTile - 1 > warp_row0 || key < all_from;
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int e = 0; e < 32; ++e)
          s[g][e] = __float_as_uint(fast_exp2(fmaf(__uint_as_float(s[g][e]), c, base2)));
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(&dp_full[t], parity));
      if (!ok) break;
      tc_fence_after();
      const int from = lone ? 0x7fffffff : first - key, upto = row - key;
#pragma unroll
      for (int g = 0; g < 4; g += 2) {
        uint32_t w[32];
#pragma unroll
        for (int gg = g; gg < g + 2; ++gg) {
          uint32_t d[32];
          tmem_ld_32(tp + 32 * gg, d);
          tmem_ld_wait();
          pin_32(d);
          float x[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            x[e] = __uint_as_float(s[gg][e]) * (__uint_as_float(d[e]) - delta);
            if (FMT == 0) x[e] *= ds_factor;
          }
          if (masked) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (32 * gg + e < from || 32 * gg + e > upto) x[e] = 0.f;
          }
#pragma unroll
          for (int e = 0; e < 32; e += 2) w[(gg - g) * 16 + e / 2] = pack16<FMT>(x[e], x[e + 1]);
        }
        tmem_st_32(tp + 16 * g, w);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ds_full[t]);
    }
    if (ok && my_i1 > my_i0) ok = __all_sync(0xffffffffu, mbar_wait_bounded(dq_full, 0));
    ok = __all_sync(0xffffffffu, mbar_wait_bounded(checked, 0)) && ok;
    if (!ok && lane == 0) atomicCAS(status, kStatusOk, kStatusTimeoutEpilogue);
    tc_fence_after();
    const bool some = in && first <= row;
    T* dst = static_cast<T*>(p.dq) + (long(row) * p.heads + my_head) * p.dim;
    const bool exact = *reinterpret_cast<volatile int*>(poison) != 0;
    if (my_i1 > my_i0 && ok) {
      if (!exact) store_row<FMT, DP>(tmem + 128 * t + lane_base, p.scale / factor, dst, p.dim, some);
      for (int r = 0; exact && r < 32; ++r) {
        const float lse_r = __shfl_sync(0xffffffffu, lse2, r), delta_r = __shfl_sync(0xffffffffu, delta, r);
        if (__shfl_sync(0xffffffffu, int(some), r)) exact_dq_row<FMT, DP>(p, warp_row0 + r, my_head, lse_r, delta_r, lane);
      }
    }
    if (!some && row < p.rows)
      for (int d = 0; d < p.dim; d += 8) *reinterpret_cast<uint4*>(dst + d) = make_uint4(0, 0, 0, 0);
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
// A block has 128 key rows of one key head and goes through the query tiles that may attend them, for
// one head of the group after the other.  Scores are transposed, keys along the lanes:
//   S^T = k q^T -> P^T in 16 bits over S^T -> dV += P^T do;   dP^T = v do^T -> dS^T over dP^T -> dK += dS^T q.
// The tensor core takes dV of step j, S^T of j + 1, dK of j, dP^T of j + 1: the softmax warps turn S^T into
// P^T under dK and dP^T, and dP^T into dS^T under dV and S^T.
//
// TMEM: dV, dK (up to 128 columns each), S^T, dP^T (128 each).  Shared memory: k, v, three query tiles,
// two tiles of do with the rows' lse2 and delta.  Warps 0-7: softmax, warps 0-3 on the first 64
// queries of a tile, 4-7 on the rest; a thread has a key.  8 TMA, 9 MMA, 10-11 look through partly
// masked tiles of q and do.

constexpr int kDkvQStages = 3;
constexpr int kDkvGStages = 2;
constexpr int kDkvRowBytes = 2 * kTile * 4;  // lse2 and delta of a query tile

template <int DP>
constexpr int dkv_smem_bytes() {
  return (2 + kDkvQStages + kDkvGStages) * tile_bytes<DP>() + kDkvGStages * kDkvRowBytes + 512;
}

template <int FMT, int DP>
__device__ __noinline__ void exact_dkv_row(const PackedBwdArgs& p, int key, int kv, int lane) {
  using T = typename Type16<FMT>::T;
  const int group = p.heads / p.kv_heads, end = p.end_query[key], first = p.first_key[key];
  const float c = p.scale * kPackedLog2e;
  float k[DP / 32], v[DP / 32], dk[DP / 32] = {}, dv[DP / 32] = {};
  load_row<FMT, DP>(k, p.k, long(key) * p.k_tok + long(kv) * p.k_head, p.dim, lane);
  load_row<FMT, DP>(v, p.v, long(key) * p.v_tok + long(kv) * p.v_head, p.dim, lane);
  for (int head = kv * group; head < (kv + 1) * group; ++head) {
    for (int row = key; row < end; ++row) {
      float q[DP / 32], g[DP / 32];
      load_row<FMT, DP>(q, p.q, long(row) * p.q_tok + long(head) * p.q_head, p.dim, lane);
      load_row<FMT, DP>(g, p.d_o, long(row) * p.do_tok + long(head) * p.do_head, p.dim, lane);
      const float w = exp2f(warp_dot(q, k) * c - p.lse2[long(head) * p.pitch + row]);
      const float ds = row == first ? 0.f : w * (warp_dot(g, v) - p.delta[long(head) * p.pitch + row]);
#pragma unroll
      for (int e = 0; e < DP / 32; ++e) {
        dv[e] = fmaf(w, g[e], dv[e]);
        if (row != first) dk[e] = fmaf(ds, q[e], dk[e]);
      }
    }
  }
  const long at = (long(key) * p.kv_heads + kv) * p.dim;
#pragma unroll
  for (int e = 0; e < DP / 32; ++e)
    if (lane + 32 * e < p.dim) {
      static_cast<T*>(p.dk)[at + lane + 32 * e] = from_float<T>(dk[e] * p.scale);
      static_cast<T*>(p.dv)[at + lane + 32 * e] = from_float<T>(dv[e]);
    }
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
    if (threadIdx.x == 0) atomicCAS(status, kStatusOk, kStatusTimeoutProducer);
    return;
  }
  uint8_t* k_tile = smem_raw;
  uint8_t* v_tile = k_tile + kTileBytes;
  uint8_t* q_tiles = v_tile + kTileBytes;
  uint8_t* g_tiles = q_tiles + kDkvQStages * kTileBytes;
  float* row_values = reinterpret_cast<float*>(g_tiles + kDkvGStages * kTileBytes);  // [stage][lse2, delta][128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(row_values) + kDkvGStages * kDkvRowBytes);
  uint64_t* kv_full = bars;
  uint64_t* q_full = kv_full + 1;            // [3]
  uint64_t* q_empty = q_full + kDkvQStages;  // [3]
  uint64_t* g_full = q_empty + kDkvQStages;  // [2]
  uint64_t* g_empty = g_full + kDkvGStages;  // [2]
  uint64_t* s_full = g_empty + kDkvGStages;
  uint64_t* p_full = s_full + 1;
  uint64_t* dp_full = p_full + 1;
  uint64_t* ds_full = dp_full + 1;
  uint64_t* done = ds_full + 1;
  uint64_t* checked = done + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(checked + 1);
  int* poison = reinterpret_cast<int*>(tmem_slot + 1);
  float* tops = reinterpret_cast<float*>(poison + 1);  // [12]: per warp

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kv_head = blockIdx.x % p.kv_heads, group = p.heads / p.kv_heads;
  const int k0 = __ldg(p.order + blockIdx.x / p.kv_heads) * kTile;
  const int k1 = min(k0 + kTile, p.valid);
  const int q_end = k1 > k0 ? min(__ldg(p.end_query + k1 - 1), p.valid) : k0;
  const int first_end = k1 > k0 ? __ldg(p.end_query + k0) : 0;
  const int per_head = (q_end - k0 + kTile - 1) / kTile;
  const int n = per_head * group;

  if (threadIdx.x == 0) {
    mbar_init(kv_full, 1);
    for (int s = 0; s < kDkvQStages; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], 3);
    }
    for (int s = 0; s < kDkvGStages; ++s) {
      mbar_init(&g_full[s], 1);
      mbar_init(&g_empty[s], 11);  // commit, 8 softmax warps, 2 looking warps
    }
    mbar_init(s_full, 1);
    mbar_init(p_full, 8);
    mbar_init(dp_full, 1);
    mbar_init(ds_full, 8);
    mbar_init(done, 1);
    mbar_init(checked, 2);
    *poison = 0;
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
  // fp16: the largest |do| among the rows of all steps sets the factor of dS.
  float factor = 1.f;
  if (FMT == 0) {
    float top = 0.f;
    for (int i = threadIdx.x; i < n * 4; i += kBwdThreads) {
      const int h = kv_head * group + i / (per_head * 4);
      top = fmaxf(top, p.do_max[(long(h) * p.pitch + k0) / 32 + i % (per_head * 4)]);
    }
    top = warp_max(top);
    if (lane == 0) tops[warp] = top;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (FMT == 0) {
    float top = 0.f;
    for (int w = 0; w < kBwdThreads / 32; ++w) top = fmaxf(top, tops[w]);
    factor = power_below_one(top);
  }
  const uint32_t tmem = *tmem_slot;
  const uint32_t tmem_dv = tmem, tmem_dk = tmem + 128, tmem_s = tmem + 256, tmem_dp = tmem + 384;

  if (warp == 8) {
    if (lane == 0 && n > 0) {
      bool ok = true;
      mbar_expect_tx(kv_full, 2 * kTileBytes);
#pragma unroll
      for (int s = 0; s < kSlabs; ++s) {
        tma_load_3d(k_tile + s * kSlabBytes, &map_k, kv_full, 64 * s, kv_head, k0);
        tma_load_3d(v_tile + s * kSlabBytes, &map_v, kv_full, 64 * s, kv_head, k0);
      }
      for (int j = 0; j < n && ok; ++j) {
        const int h = kv_head * group + j / per_head, q0 = k0 + (j % per_head) * kTile;
        const int qs = j % kDkvQStages, gs = j % kDkvGStages;
        ok = mbar_wait_bounded(&q_empty[qs], ((j / kDkvQStages) & 1) ^ 1);
        if (!ok) break;
        mbar_expect_tx(&q_full[qs], kTileBytes);
#pragma unroll
        for (int s = 0; s < kSlabs; ++s)
          tma_load_3d(q_tiles + qs * kTileBytes + s * kSlabBytes, &map_q, &q_full[qs], 64 * s, h, q0);
        ok = mbar_wait_bounded(&g_empty[gs], ((j / kDkvGStages) & 1) ^ 1);
        if (!ok) break;
        mbar_expect_tx(&g_full[gs], kTileBytes + kDkvRowBytes);
#pragma unroll
        for (int s = 0; s < kSlabs; ++s)
          tma_load_3d(g_tiles + gs * kTileBytes + s * kSlabBytes, &map_do, &g_full[gs], 64 * s, h, q0);
        // lse2 and delta have whole tiles of rows to a head, so the copy stays inside
        bulk_load(row_values + gs * 2 * kTile, p.lse2 + long(h) * p.pitch + q0, kTile * 4, &g_full[gs]);
        bulk_load(row_values + gs * 2 * kTile + kTile, p.delta + long(h) * p.pitch + q0, kTile * 4, &g_full[gs]);
      }
      if (!ok) {
        atomicCAS(status, kStatusOk, kStatusTimeoutProducer);
        drain_copies();
      }
    }
    __syncwarp();
  } else if (warp == 9) {
    constexpr uint32_t idesc_s = make_idesc_f16(kTile, kTile, FMT, 0, 0);
    constexpr uint32_t idesc_d = make_idesc_f16(kTile, DP, FMT, 0, 1);
    if (lane == 0 && n > 0) {
      bool ok = mbar_wait_bounded(kv_full, 0);
      const uint64_t dk = make_kmajor_sw128_desc(smem_u32(k_tile)), dv = make_kmajor_sw128_desc(smem_u32(v_tile));
      const auto scores = [&](uint32_t tmem_d, uint64_t a, const uint8_t* b_tile, uint64_t* bar) {
        tc_fence_after();
        const uint64_t b = make_kmajor_sw128_desc(smem_u32(b_tile));
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          const uint64_t off = uint64_t(((k / 4) * kSlabBytes + (k % 4) * 32) >> 4);
          umma_f16(tmem_d, a + off, b + off, idesc_s, k > 0 ? 1u : 0u);
        }
        umma_commit(bar);
      };
      // The two halves of the softmax warps leave their 64 queries over their own columns.
      const auto add = [&](uint32_t tmem_d, uint32_t tmem_a, const uint8_t* b_tile, bool first) {
        tc_fence_after();
        const uint64_t b = make_mnmajor_sw128_desc(smem_u32(b_tile), kSlabBytes);
#pragma unroll
        for (int k = 0; k < kTile / 16; ++k)
          umma_f16_ts(tmem_d, tmem_a + (k / 4) * 64 + (k % 4) * 8, b + uint64_t((2048 * k) >> 4), idesc_d,
                      (!first || k > 0) ? 1u : 0u);
      };
      ok = ok && mbar_wait_bounded(&q_full[0], 0);
      if (ok) scores(tmem_s, dk, q_tiles, s_full);
      ok = ok && mbar_wait_bounded(&g_full[0], 0);
      if (ok) scores(tmem_dp, dv, g_tiles, dp_full);
      for (int j = 0; j < n && ok; ++j) {
        const int qs = j % kDkvQStages, gs = j % kDkvGStages;
        const int qn = (j + 1) % kDkvQStages, gn = (j + 1) % kDkvGStages;
        ok = mbar_wait_bounded(p_full, j & 1);
        if (!ok) break;
        add(tmem_dv, tmem_s, g_tiles + gs * kTileBytes, j == 0);
        umma_commit(&g_empty[gs]);
        if (j + 1 < n) {
          ok = mbar_wait_bounded(&q_full[qn], ((j + 1) / kDkvQStages) & 1);
          if (!ok) break;
          scores(tmem_s, dk, q_tiles + qn * kTileBytes, s_full);
        }
        ok = mbar_wait_bounded(ds_full, j & 1);
        if (!ok) break;
        add(tmem_dk, tmem_dp, q_tiles + qs * kTileBytes, j == 0);
        umma_commit(&q_empty[qs]);
        if (j + 1 < n) {
          ok = mbar_wait_bounded(&g_full[gn], ((j + 1) / kDkvGStages) & 1);
          if (!ok) break;
          scores(tmem_dp, dv, g_tiles + gn * kTileBytes, dp_full);
        }
      }
      if (ok) umma_commit(done);
      if (!ok) atomicCAS(status, kStatusOk, kStatusTimeoutMma);
    }
    __syncwarp();
  } else if (warp >= 10) {
    bool bad = false, ok = true;
    for (int j = 0; j < n && ok; ++j) {
      const int q0 = k0 + (j % per_head) * kTile;
      const int qs = j % kDkvQStages, gs = j % kDkvGStages;
      const bool masked = q0 < k0 + kTile || q0 + kTile > first_end;
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(&q_full[qs], (j / kDkvQStages) & 1));
      if (masked && ok) bad |= scan_not_finite<FMT>(q_tiles + qs * kTileBytes, kTileBytes, warp - 10, 2, lane);
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_empty[qs]);
      ok = ok && __all_sync(0xffffffffu, mbar_wait_bounded(&g_full[gs], (j / kDkvGStages) & 1));
      if (masked && ok) bad |= scan_not_finite<FMT>(g_tiles + gs * kTileBytes, kTileBytes, warp - 10, 2, lane);
      __syncwarp();
      if (lane == 0) mbar_arrive(&g_empty[gs]);
    }
    if (__any_sync(0xffffffffu, bad) && lane == 0) *poison = 1;
    __syncwarp();
    if (lane == 0) mbar_arrive(checked);
  } else {
    using T = typename Type16<FMT>::T;
    const int half = warp >> 2, quad = warp & 3;
    const int key = k0 + quad * 32 + lane;
    const bool in = key < p.valid;
    const int end = in ? __ldg(p.end_query + key) : 0;
    const bool opens = in && __ldg(p.first_key + key) == key;  // its own row attends nothing else
    const int warp_key_last = k0 + quad * 32 + 31;
    const int min_end = __reduce_min_sync(0xffffffffu, end);
    const uint32_t lane_base = uint32_t(quad * 32) << 16;
    const uint32_t ts = tmem_s + lane_base + 64 * half, tp = tmem_dp + lane_base + 64 * half;
    const float c = p.scale * kPackedLog2e;
    const float ds_factor = FMT == 0 ? factor * (1.f / 1024.f) : 1.f;
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      const int gs = j % kDkvGStages;
      const int q0 = k0 + (j % per_head) * kTile + 64 * half;  // first query of this half
      ok = mbar_wait_bounded(&g_full[gs], (j / kDkvGStages) & 1);
      ok = mbar_wait_bounded(s_full, j & 1) && ok;
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      uint32_t s[2][32];
      tmem_ld_32(ts, s[0]);
      tmem_ld_32(ts + 32, s[1]);
      tmem_ld_wait();
      pin_32(s[0]);
      pin_32(s[1]);
      const bool masked = q0 < warp_key_last || q0 + 64 > min_end;
      const int from = key - q0, to = end - q0;  // columns [from, to) attend this key
      const float4* lse = reinterpret_cast<const float4*>(row_values + gs * 2 * kTile + 64 * half);
      uint32_t w[32];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 x = lse[g * 8 + e / 4];
          const float xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int u = 0; u < 4; ++u)
            s[g][e + u] = __float_as_uint(
                fast_exp2(fmaf(__uint_as_float(s[g][e + u]), c, FMT == 0 ? p_shift<FMT>() - xs[u] : -xs[u])));
        }
        if (masked) {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (32 * g + e < from || 32 * g + e >= to) s[g][e] = 0u;
        }
#pragma unroll
        for (int e = 0; e < 32; e += 2)
          w[16 * g + e / 2] = pack16<FMT>(__uint_as_float(s[g][e]), __uint_as_float(s[g][e + 1]));
      }
      tmem_st_32(ts, w);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full);

      ok = __all_sync(0xffffffffu, mbar_wait_bounded(dp_full, j & 1));
      if (!ok) break;
      tc_fence_after();
      const float4* dl = reinterpret_cast<const float4*>(row_values + gs * 2 * kTile + kTile + 64 * half);
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        uint32_t d[32];
        tmem_ld_32(tp + 32 * g, d);
        tmem_ld_wait();
        pin_32(d);
        float x[32];
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 y = dl[g * 8 + e / 4];
          const float ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            x[e + u] = __uint_as_float(s[g][e + u]) * (__uint_as_float(d[e + u]) - ys[u]);
            if (FMT == 0) x[e + u] *= ds_factor;
          }
        }
        if (masked) {
          // what is masked may be infinite or NaN; the first row of a document has a single key
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (32 * g + e < from || 32 * g + e >= to || (opens && 32 * g + e == from)) x[e] = 0.f;
        }
#pragma unroll
        for (int e = 0; e < 32; e += 2) w[16 * g + e / 2] = pack16<FMT>(x[e], x[e + 1]);
      }
      tmem_st_32(tp, w);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(ds_full);
        mbar_arrive(&g_empty[gs]);  // lse2 and delta are read
      }
    }
    if (ok && n > 0) ok = __all_sync(0xffffffffu, mbar_wait_bounded(done, 0));
    ok = __all_sync(0xffffffffu, mbar_wait_bounded(checked, 0)) && ok;
    if (!ok && lane == 0) atomicCAS(status, kStatusOk, kStatusTimeoutEpilogue);
    tc_fence_after();
    const long at = (long(key) * p.kv_heads + kv_head) * p.dim;
    T* dst = static_cast<T*>(half ? p.dk : p.dv) + at;
    const bool exact = *reinterpret_cast<volatile int*>(poison) != 0;
    if (n > 0 && ok) {
      const float factor_out = half ? p.scale / factor : (FMT == 0 ? 1.f / 1024.f : 1.f);
      if (!exact) store_row<FMT, DP>((half ? tmem_dk : tmem_dv) + lane_base, factor_out, dst, p.dim, in);
      // both halves share the rows: even ones here, odd ones there
      for (int r = half; exact && r < 32; r += 2)
        if (k0 + quad * 32 + r < p.valid) exact_dkv_row<FMT, DP>(p, k0 + quad * 32 + r, kv_head, lane);
    }
    if (!in && key < p.rows)
      for (int d = 0; d < p.dim; d += 8) *reinterpret_cast<uint4*>(dst + d) = make_uint4(0, 0, 0, 0);
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace bgn
