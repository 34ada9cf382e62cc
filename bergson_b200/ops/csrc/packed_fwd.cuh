// Forward pass of the causal attention over packed documents on the tensor cores (fp16, bf16).
//
//   S = q k^T,  P = 2^(c S - c m),  O = sum P v / sum P        (c = scale * log2 e, m: running maximum)
//
// A block works on two tiles of 128 query rows at once, so that the softmax of one runs under the
// products of the other: two heads of a group at the same rows (they share every key tile), or, where
// a group has an odd number of heads, two neighbouring row tiles of a head.  Tiles are cut from the
// packed axis without regard to documents; a tile of rows [r, r + 128) visits the keys from the first
// key of row r to its last row, and each row masks its own range [first_key, row].  Short documents
// so share tiles, and nothing depends on how documents lie in them.
//
// TMEM (512 columns): S of the two tiles (128 each, P in 16 bits over the first half of the same
// columns: the A operand of the second product) and O of the two (up to 128 each).
//
// Warps: 0-3 and 4-7 softmax of tile 0 and 1 (a thread has a row), 8 TMA, 9 MMA, 10-11 look for
// infinities and NaN in value tiles that are partly masked: 0 * NaN would carry them into rows that
// do not attend them.  If there are any, the block's rows are computed again, row by row.
//
// O is rescaled only when a row's maximum grew by more than 2^8 since the last time (P then stays
// below 2^8, which fp16 holds): the final division by the sum makes any base right.
//
// P is rounded to the operands' type, as the tensor core needs; the sum is taken from the unrounded
// values in fp32, and O is rounded once.
#pragma once

#include "packed_tc.cuh"

namespace bgn {

constexpr int kFwdThreads = 384;
constexpr int kFwdStages = 2;  // key tiles and value tiles in flight, each

template <int DP>
constexpr int fwd_smem_bytes() {
  return (2 + 2 * kFwdStages) * tile_bytes<DP>() + 1024 + 256;
}

struct PackedFwdArgs {
  const int* first_key;
  const int* order;  // tiles (head pairs) or pairs of tiles, most keys first
  int rows, valid, heads, kv_heads, dim;
  int pitch;       // floats between the heads of lse2
  int head_pairs;  // 1: a block takes two heads of a group; 0: two row tiles of a head
  float scale;
  const void *q, *k, *v;  // for the exact recomputation
  long q_tok, q_head, k_tok, k_head, v_tok, v_head;
  void* o;
  float* lse2;
};

// Key range of the rows [r0, r0 + 128): empty where hi <= lo.
struct KeyRange {
  int lo, hi;
  int last_first;  // first key of the last row: from there on every row may attend
};

__device__ __forceinline__ KeyRange key_range(const int* first_key, int r0, int valid) {
  KeyRange k = {0, 0, 0};
  if (r0 < valid) {
    k.hi = min(r0 + kTile, valid);
    k.lo = __ldg(first_key + r0);
    k.last_first = __ldg(first_key + k.hi - 1);
  }
  return k;
}

template <int FMT, int DP>
__device__ __noinline__ void exact_forward_row(const PackedFwdArgs& p, int row, int head, float lse2, int lane) {
  using T = typename Type16<FMT>::T;
  const int kv = head / (p.heads / p.kv_heads);
  const float c = p.scale * kPackedLog2e;
  float q[DP / 32], o[DP / 32] = {};
  load_row<FMT, DP>(q, p.q, long(row) * p.q_tok + long(head) * p.q_head, p.dim, lane);
  for (int j = p.first_key[row]; j <= row; ++j) {
    float k[DP / 32], v[DP / 32];
    load_row<FMT, DP>(k, p.k, long(j) * p.k_tok + long(kv) * p.k_head, p.dim, lane);
    load_row<FMT, DP>(v, p.v, long(j) * p.v_tok + long(kv) * p.v_head, p.dim, lane);
    const float w = exp2f(warp_dot(q, k) * c - lse2);
#pragma unroll
    for (int e = 0; e < DP / 32; ++e) o[e] = fmaf(w, v[e], o[e]);
  }
  T* dst = static_cast<T*>(p.o) + (long(row) * p.heads + head) * p.dim;
#pragma unroll
  for (int e = 0; e < DP / 32; ++e)
    if (lane + 32 * e < p.dim) dst[lane + 32 * e] = from_float<T>(o[e]);
}

template <int FMT, int DP>
__global__ void __launch_bounds__(kFwdThreads, 1)
packed_fwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const __grid_constant__ PackedFwdArgs p, int* status) {
  constexpr int kTileBytes = tile_bytes<DP>();
  constexpr int kSlabs = DP / 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* q_tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* k_tiles = q_tiles + 2 * kTileBytes;
  uint8_t* v_tiles = k_tiles + kFwdStages * kTileBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(v_tiles + kFwdStages * kTileBytes);
  uint64_t* q_full = bars;                     // [2]
  uint64_t* k_full = q_full + 2;               // [stages]
  uint64_t* k_empty = k_full + kFwdStages;
  uint64_t* v_full = k_empty + kFwdStages;
  uint64_t* v_empty = v_full + kFwdStages;
  uint64_t* s_full = v_empty + kFwdStages;     // [2]
  uint64_t* p_full = s_full + 2;               // [2]
  uint64_t* o_full = p_full + 2;               // [2]
  uint64_t* checked = o_full + 2;              // [1]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(checked + 1);
  int* poison = reinterpret_cast<int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // This block's two tiles.
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
  // Key tiles are counted from the lower of the two first keys; [i0, i1) are the ones a tile needs.
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
  const int begin = some0 && some1 ? min(i0[0], i0[1]) : (some0 ? i0[0] : i0[1]);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kFwdStages; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 3);  // the MMA warp's commit and the two looking warps
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], 1);
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_full[t], 1);
    }
    mbar_init(checked, 2);
    *poison = 0;
    fence_barrier_init();
    tma_prefetch_desc(&map_q);
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
  const uint32_t tmem_s[2] = {tmem, tmem + 128}, tmem_o[2] = {tmem + 256, tmem + 384};

  if (warp >= 8) {
    // 168 registers a thread at launch: 3 * 168 >= 2 * 208 + 80
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == 8) {
      if (lane == 0 && n > 0) {
        bool ok = true;
        for (int t = 0; t < 2; ++t) {
          if (i1[t] == 0) continue;
          mbar_expect_tx(&q_full[t], kTileBytes);
#pragma unroll
          for (int s = 0; s < kSlabs; ++s)
            tma_load_3d(q_tiles + t * kTileBytes + s * kSlabBytes, &map_q, &q_full[t], 64 * s, head[t], row0[t]);
        }
        for (int i = begin, j = 0; i < n && ok; ++i, ++j) {
          const int st = j % kFwdStages;
          const uint32_t parity = ((j / kFwdStages) & 1) ^ 1;
          const int key = base + i * kTile;
          ok = mbar_wait_bounded(&k_empty[st], parity);
          if (!ok) break;
          mbar_expect_tx(&k_full[st], kTileBytes);
#pragma unroll
          for (int s = 0; s < kSlabs; ++s)
            tma_load_3d(k_tiles + st * kTileBytes + s * kSlabBytes, &map_k, &k_full[st], 64 * s, kv_head, key);
          ok = mbar_wait_bounded(&v_empty[st], parity);
          if (!ok) break;
          mbar_expect_tx(&v_full[st], kTileBytes);
#pragma unroll
          for (int s = 0; s < kSlabs; ++s)
            tma_load_3d(v_tiles + st * kTileBytes + s * kSlabBytes, &map_v, &v_full[st], 64 * s, kv_head, key);
        }
        if (!ok) {
          atomicCAS(status, kStatusOk, kStatusTimeoutProducer);
          drain_copies();
        }
      }
      __syncwarp();
    } else if (warp == 9) {
      constexpr uint32_t idesc_s = make_idesc_f16(kTile, kTile, FMT, 0, 0);
      constexpr uint32_t idesc_o = make_idesc_f16(kTile, DP, FMT, 0, 1);
      if (lane == 0 && n > 0) {
        bool ok = true;
        // Step i: for each tile the second product of key tile i - 1, then the first product of i.
        for (int i = begin, j = 0; i <= n && ok; ++i, ++j) {
          const int st = j % kFwdStages, pst = (j + kFwdStages - 1) % kFwdStages;  // stages of i and i - 1
          bool k_there = false, v_there = false;
          for (int t = 0; t < 2 && ok; ++t) {
            if (i - 1 >= i0[t] && i - 1 < i1[t]) {
              if (!v_there) {
                ok = mbar_wait_bounded(&v_full[pst], ((j - 1) / kFwdStages) & 1);
                v_there = true;
              }
              ok = ok && mbar_wait_bounded(&p_full[t], (i - 1 - i0[t]) & 1);
              if (!ok) break;
              tc_fence_after();
              const uint64_t dv = make_mnmajor_sw128_desc(smem_u32(v_tiles + pst * kTileBytes), kSlabBytes);
#pragma unroll
              for (int k = 0; k < kTile / 16; ++k)
                umma_f16_ts(tmem_o[t], tmem_s[t] + 8 * k, dv + uint64_t((2048 * k) >> 4), idesc_o,
                            (i - 1 > i0[t] || k > 0) ? 1u : 0u);
              if (i == i1[t]) umma_commit(&o_full[t]);
            }
            if (i >= i0[t] && i < i1[t]) {
              if (!k_there) {
                ok = mbar_wait_bounded(&k_full[st], (j / kFwdStages) & 1);
                k_there = true;
              }
              if (i == i0[t]) ok = ok && mbar_wait_bounded(&q_full[t], 0);
              if (!ok) break;
              tc_fence_after();
              const uint64_t dq = make_kmajor_sw128_desc(smem_u32(q_tiles + t * kTileBytes));
              const uint64_t dk = make_kmajor_sw128_desc(smem_u32(k_tiles + st * kTileBytes));
#pragma unroll
              for (int k = 0; k < DP / 16; ++k) {
                const uint64_t off = uint64_t(((k / 4) * kSlabBytes + (k % 4) * 32) >> 4);
                umma_f16(tmem_s[t], dq + off, dk + off, idesc_s, k > 0 ? 1u : 0u);
              }
              umma_commit(&s_full[t]);
            }
          }
          if (ok) {
            // A stage that no tile needed is handed back the same way.
            if (i < n) {
              if (!k_there) ok = mbar_wait_bounded(&k_full[st], (j / kFwdStages) & 1);
              umma_commit(&k_empty[st]);
            }
            if (i > begin) {
              if (!v_there) ok = ok && mbar_wait_bounded(&v_full[pst], ((j - 1) / kFwdStages) & 1);
              umma_commit(&v_empty[pst]);
            }
          }
        }
        if (!ok) atomicCAS(status, kStatusOk, kStatusTimeoutMma);
      }
      __syncwarp();
    } else {
      bool bad = false, ok = true;
      for (int i = begin, j = 0; i < n && ok; ++i, ++j) {
        const int st = j % kFwdStages;
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(&v_full[st], (j / kFwdStages) & 1));
        const int key = base + i * kTile;
        bool masked = false;
#pragma unroll
        for (int t = 0; t < 2; ++t)
          masked |= i >= i0[t] && i < i1[t] && (key + kTile - 1 > row0[t] || key < range[t].last_first);
        if (masked && ok) bad |= scan_not_finite<FMT>(v_tiles + st * kTileBytes, kTileBytes, warp - 10, 2, lane);
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_empty[st]);
      }
      if (__any_sync(0xffffffffu, bad) && lane == 0) *poison = 1;
      __syncwarp();
      if (lane == 0) mbar_arrive(checked);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int t = warp >> 2, quad = warp & 3;
    const int my_i0 = t ? i0[1] : i0[0], my_i1 = t ? i1[1] : i1[0];
    const int r0 = t ? row0[1] : row0[0], my_head = t ? head[1] : head[0];
    const int row = r0 + quad * 32 + lane;
    const bool in = row < p.valid;
    const int first = in ? __ldg(p.first_key + row) : 0x7fffffff;
    // The warp's rows attend all of a key tile from `all_from` on, up to its first row.
    const int warp_row0 = r0 + quad * 32;
    const int all_from = __shfl_sync(0xffffffffu, in ? first : 0x7fffffff, 31);
    const uint32_t lane_base = uint32_t(quad * 32) << 16;
    const uint32_t ts = (t ? tmem_s[1] : tmem_s[0]) + lane_base, to = (t ? tmem_o[1] : tmem_o[0]) + lane_base;
    const float c = p.scale * kPackedLog2e;
    float m = -INFINITY, l = 0.f;  // m: the base in use, of the unscaled scores
    bool ok = true;
    for (int i = my_i0; i < my_i1; ++i) {
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(&s_full[t], (i - my_i0) & 1));
      if (!ok) break;
      tc_fence_after();
      uint32_t s[4][32];
#pragma unroll
      for (int g = 0; g < 4; ++g) tmem_ld_32(ts + 32 * g, s[g]);
      tmem_ld_wait();
#pragma unroll
      for (int g = 0; g < 4; ++g) pin_32(s[g]);
      const int key = base + i * kTile;
      if (key + kTile - 1 > warp_row0 || key < all_from) {
        const int from = first - key, to_ = row - key;  // columns of the row's own range
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (32 * g + e < from || 32 * g + e > to_) s[g][e] = 0xff800000u;  // -inf
      }
      float mx[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        mx[g] = __uint_as_float(s[g][0]);
#pragma unroll
        for (int e = 1; e < 32; ++e) mx[g] = fmaxf(mx[g], __uint_as_float(s[g][e]));
      }
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      // A new base where the maximum grew by more than 2^8 (or is the row's first).
      const bool grow = (top - m) * c > 8.f;
      if (__any_sync(0xffffffffu, grow)) {
        const float alpha = grow ? fast_exp2((m - top) * c) : 1.f;
        if (grow) m = top;
        l *= alpha;
        if (i > my_i0) {
#pragma unroll 1
          for (int d = 0; d < DP; d += 32) {
            uint32_t o[32];
            tmem_ld_32(to + d, o);
            tmem_ld_wait();
            pin_32(o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st_32(to + d, o);
          }
        }
      }
      const float mc = m == -INFINITY ? 0.f : m * c;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int g = 0; g < 4; g += 2) {
        uint32_t w[32];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float a0 = fast_exp2(fmaf(__uint_as_float(s[g][e]), c, -mc));
          const float a1 = fast_exp2(fmaf(__uint_as_float(s[g][e + 1]), c, -mc));
          const float b0 = fast_exp2(fmaf(__uint_as_float(s[g + 1][e]), c, -mc));
          const float b1 = fast_exp2(fmaf(__uint_as_float(s[g + 1][e + 1]), c, -mc));
          sum[0] += a0;
          sum[1] += a1;
          sum[2] += b0;
          sum[3] += b1;
          w[e / 2] = pack16<FMT>(a0, a1);
          w[16 + e / 2] = pack16<FMT>(b0, b1);
        }
        tmem_st_32(ts + 16 * g, w);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[t]);
    }
    if (ok && my_i1 > my_i0) ok = __all_sync(0xffffffffu, mbar_wait_bounded(&o_full[t], 0));
    ok = __all_sync(0xffffffffu, mbar_wait_bounded(checked, 0)) && ok;
    if (!ok && lane == 0) atomicCAS(status, kStatusOk, kStatusTimeoutEpilogue);
    tc_fence_after();
    const bool some = in && first <= row;
    const float lse2 = some ? fmaf(m, c, log2f(l)) : INFINITY;
    if (row < p.rows) p.lse2[long(my_head) * p.pitch + row] = lse2;
    using T = typename Type16<FMT>::T;
    T* dst = static_cast<T*>(p.o) + (long(row) * p.heads + my_head) * p.dim;
    const bool exact = *reinterpret_cast<volatile int*>(poison) != 0;
    if (my_i1 > my_i0 && ok) {
      if (!exact) store_row<FMT, DP>(to, some ? 1.f / l : 0.f, dst, p.dim, some);
      for (int r = 0; exact && r < 32; ++r) {
        const int row_r = warp_row0 + r;
        const float lse_r = __shfl_sync(0xffffffffu, lse2, r);
        if (__shfl_sync(0xffffffffu, int(some), r)) exact_forward_row<FMT, DP>(p, row_r, my_head, lse_r, lane);
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

}  // namespace bgn
