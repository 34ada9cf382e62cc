// Forward pass of the causal attention over packed documents on the tensor cores (fp16, bf16).
//
//   S = q k^T,  P = 2^(c S - c m),  O = sum P v / sum P        (c = scale * log2 e, m: running maximum)
//
// One block per SM works through its share of the units.  A unit is two tiles of 128 query rows, so
// that the softmax of one runs under the products of the other: two heads of a group at the same
// rows (they share every key tile), or, where a group has an odd number of heads, two neighbouring row
// tiles of a head.  Tiles are cut from the packed axis without regard to documents; a tile of rows
// [r, r + 128) visits the keys from the first key of row r to its last row, and each row masks its own
// range [first_key, row].  Short documents so share tiles, and nothing depends on how they lie.
//
// TMEM (512 columns): S of the two tiles (128 each, P in 16 bits over the first half of the same
// columns: the A operand of the second product) and O of the two (up to 128 each).
//
// Warps: 0-3 and 4-7 softmax of tile 0 and 1 (a thread has a row), 8 TMA, 9 and 10 MMA of tile 0 and 1.
//
// An infinity or NaN in a value row that some rows of a tile do not attend reaches them all the same, as
// 0 * NaN of the second product.  It shows as a NaN of the result: a row whose result is not finite is
// computed again over its own keys alone, unless the few value rows that it was multiplied with and does not
// attend are all finite.  That comes after a block's last unit, when no other warp waits for this one with
// a limit.  (Looking through the tiles in shared memory instead held up the pipeline: other reads wait
// long while the tensor core takes its operands from there.)
//
// What bounds it: a tile of 128 x 128 scores takes 1024 cycles of the tensor core at 128 features and
// 1024 of the exponential unit (twice that of the tensor core at 64), in a chain that the two tiles
// fill alternately.  The chain is kept short: a row's scores stay in registers, the second product starts
// on the first three quarters of the keys, fp32 arithmetic is packed in pairs.  Moving a quarter of the
// exponentials to a polynomial on the FMA units was slower (2.0 against 1.9 ms at 16384 tokens).
// 32 over 8 heads of 128 in bf16: one document of 16384 tokens 1.9 ms (1160 TFLOP/s), of 8192 0.55 ms (1000); 24 documents
// of 16321 tokens together 233 us, with two row tiles to a unit instead of two heads 260 us.
//
// O is rescaled only when a row's maximum grew by more than 2^8 since the last time (P then stays
// below 2^8, which fp16 holds): the final division by the sum makes any base right.
//
// P is rounded to the operands' type, as the tensor core needs; the sum is taken from the unrounded
// values in fp32, and O is rounded once.
#pragma once

#include <type_traits>

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
  const int4* tiles;  // query_tiles (head pairs) or query_pairs
  int units;          // what the blocks share out: tiles x head pairs, or pairs of tiles x heads
  int rows, valid, heads, kv_heads, dim;
  int pitch;       // floats between the heads of bias2
  int head_pairs;  // 1: a unit is two heads of a group at one tile; 0: two row tiles of a head
  float scale;
  const void *q, *k, *v;  // for the exact recomputation
  long q_tok, q_head, k_tok, k_head, v_tok, v_head;
  void* o;
  void* o_rest;  // what rounding took from o, for the backward pass (may be null)
  float* bias2;
  int* gave_up;
};

// The r-th unit of a block, -1 behind the last: units come most work first, so the blocks take them in
// rounds of alternating direction, which evens out what they get.
__device__ __forceinline__ int nth_unit(int r, int units) {
  const int g = gridDim.x;
  const int u = r * g + ((r & 1) ? g - 1 - int(blockIdx.x) : int(blockIdx.x));
  return u < units ? u : -1;
}

struct QueryUnit {
  int row0[2], head[2];
  int i0[2], i1[2];  // key tiles of each, counted from `base` in steps of 128
  int base, n, kv_head;
};

// The tile entries of a unit (most of a trip to L2: asked for one unit ahead).
__device__ __forceinline__ void fetch_unit(const int4* tiles, int head_pairs, int heads, int u, int4 (&e)[2]) {
  if (u < 0) return;
  if (head_pairs) {
    e[0] = e[1] = __ldg(tiles + u / (heads / 2));
  } else {
    e[0] = __ldg(tiles + 2 * (u / heads));
    e[1] = __ldg(tiles + 2 * (u / heads) + 1);
  }
}

__device__ __forceinline__ QueryUnit query_unit(const int4 (&e)[2], int head_pairs, int heads, int kv_heads, int u) {
  QueryUnit w;
  const int h = head_pairs ? 2 * (u % (heads / 2)) : u % heads;
  w.head[0] = h;
  w.head[1] = head_pairs ? h + 1 : h;
  w.kv_head = h / (heads / kv_heads);
  const bool some0 = e[0].w > e[0].y, some1 = e[1].w > e[1].y;
  // The second tile never begins before the first one does, and is empty if that is.
  w.base = e[0].y;
  w.row0[0] = e[0].x;
  w.row0[1] = e[1].x;
  w.i0[0] = 0;
  w.i1[0] = some0 ? (e[0].w - w.base + kTile - 1) / kTile : 0;
  w.i0[1] = some1 ? (e[1].y - w.base) / kTile : 0;
  w.i1[1] = some1 ? (e[1].w - w.base + kTile - 1) / kTile : 0;
  w.n = max(w.i1[0], w.i1[1]);
  return w;
}

// A warp puts right a row of the tile at row0.
template <int FMT, int DP>
__device__ __noinline__ void exact_forward_row(const PackedFwdArgs& p, int row0, int row, int head, int lane) {
  using T = typename Type16<FMT>::T;
  const int kv = head / (p.heads / p.kv_heads), first = p.first_key[row];
  float q[DP / 32], o[DP / 32] = {};
  const long v_off = long(kv) * p.v_head;
  load_row<FMT, DP>(q, p.o, (long(row) * p.heads + head) * p.dim, p.dim, lane);
  bool bad = false;
#pragma unroll
  for (int e = 0; e < DP / 32; ++e) bad |= !(fabsf(q[e]) < INFINITY);
  if (!__any_sync(0xffffffffu, bad)) return;
  // A document that begins in the tile is short there.  Another one begins less than a tile behind the first
  // key that was visited, and the last one visited is less than two tiles behind row0.
  if (first <= row0 && !some_not_finite<FMT, DP>(p.v, p.v_tok, v_off, max(first - kTile + 1, 0), first, p.dim, lane) &&
      !some_not_finite<FMT, DP>(p.v, p.v_tok, v_off, row + 1, min(row0 + 2 * kTile, p.valid), p.dim, lane))
    return;
  const float c = p.scale * kPackedLog2e, bias2 = p.bias2[long(head) * p.pitch + row] - p_shift<FMT>();
  load_row<FMT, DP>(q, p.q, long(row) * p.q_tok + long(head) * p.q_head, p.dim, lane);
  for (int j0 = first; j0 <= row && !all_nan(o, 0, p.dim, lane); j0 += 64) {
#pragma unroll 4
    for (int j = j0; j <= min(j0 + 63, row); ++j) {
      float k[DP / 32], v[DP / 32];
      load_row<FMT, DP>(k, p.k, long(j) * p.k_tok + long(kv) * p.k_head, p.dim, lane);
      load_row<FMT, DP>(v, p.v, long(j) * p.v_tok + v_off, p.dim, lane);
      const float w = exp2f(warp_dot(q, k) * c + bias2);
#pragma unroll
      for (int e = 0; e < DP / 32; ++e) o[e] = fmaf(w, v[e], o[e]);
    }
  }
  const long at = (long(row) * p.heads + head) * p.dim + lane;
#pragma unroll
  for (int e = 0; e < DP / 32; ++e)
    if (lane + 32 * e < p.dim) {
      const T kept = from_float<T>(o[e]);
      static_cast<T*>(p.o)[at + 32 * e] = kept;
      if (p.o_rest != nullptr) static_cast<T*>(p.o_rest)[at + 32 * e] = from_float<T>(o[e] - to_float<T>(kept));
    }
}

// Largest of 32 values and `top`.
__device__ __forceinline__ float max_chunk(const uint32_t (&s)[32], float top) {
  float a = __uint_as_float(s[0]), b = __uint_as_float(s[1]);
#pragma unroll
  for (int e = 2; e < 30; e += 4) {
    a = max3(a, __uint_as_float(s[e]), __uint_as_float(s[e + 1]));
    b = max3(b, __uint_as_float(s[e + 2]), __uint_as_float(s[e + 3]));
  }
  a = max3(a, __uint_as_float(s[30]), __uint_as_float(s[31]));
  return max3(top, a, b);
}

// P = 2^(c s - mc) of 32 columns, in 16 bits to TMEM; their sum is added to `sum`.
template <int FMT>
__device__ __forceinline__ void exp_chunk(uint32_t tmem, const uint32_t (&s)[32], float c, float mc, float2 (&sum)[2]) {
  const float2 c2 = make_float2(c, c), m2 = make_float2(-mc, -mc);
  uint32_t w[16];
#pragma unroll
  for (int e = 0; e < 32; e += 2) {
    const float2 x = fma2(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), c2, m2);
    const float2 p = make_float2(fast_exp2(x.x), fast_exp2(x.y));
    sum[(e / 2) & 1] = add2(sum[(e / 2) & 1], p);
    w[e / 2] = pack16<FMT>(p.x, p.y);
  }
  tmem_st_16(tmem, w);
}

// The MMA warp of one of the two tiles.
template <int FMT, int DP>
struct FwdMma {
  static_assert(kFwdStages == 2, "stages are addressed by the lowest bit of the step");
  uint32_t tmem_s, tmem_o;
  uint64_t q, k, v;  // descriptors; of stage 0 for k and v
  uint64_t *k_full, *k_empty, *v_full, *v_empty, *q_full, *q_empty, *s_full, *p_full, *o_full;
  uint32_t j = 0;  // key tiles so far
  uint32_t steps = 0, uses = 0;
  static constexpr uint64_t kStage = tile_bytes<DP>() >> 4;

  __device__ __forceinline__ bool scores(uint32_t jj) {
    constexpr uint32_t idesc = make_idesc_f16(kTile, kTile, FMT, 0, 0);
    if (!warp_wait(&k_full[jj & 1], (jj >> 1) & 1)) return false;
    tc_fence_after();
    const uint64_t b = k + (jj & 1) * kStage;
    if (elect_one()) {
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) {
        const uint64_t off = uint64_t(((i / 4) * kSlabBytes + (i % 4) * 32) >> 4);
        umma_f16(tmem_s, q + off, b + off, idesc, i > 0 ? 1u : 0u);
      }
      umma_commit(s_full);
      umma_commit(&k_empty[jj & 1]);
    }
    __syncwarp();
    return true;
  }
  __device__ __forceinline__ bool output(uint32_t jj, bool first) {
    constexpr uint32_t idesc = make_idesc_f16(kTile, DP, FMT, 0, 1);
    if (!warp_wait(&v_full[jj & 1], (jj >> 1) & 1)) return false;
    const uint64_t b = v + (jj & 1) * kStage;
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      if (!warp_wait(&p_full[part], steps & 1)) return false;
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int i = part ? 6 : 0; i < (part ? 8 : 6); ++i)
          umma_f16_ts(tmem_o, tmem_s + 8 * i, b + uint64_t((2048 * i) >> 4), idesc, (!first || i > 0) ? 1u : 0u);
        if (part == 1) umma_commit(&v_empty[jj & 1]);
      }
      __syncwarp();
    }
    ++steps;
    return true;
  }
  // Key tiles that only the other tile needs are handed back at once.
  __device__ __forceinline__ bool pass(uint32_t from, uint32_t to) {
    for (uint32_t jj = from; jj < to; ++jj) {
      if (!warp_wait(&k_full[jj & 1], (jj >> 1) & 1)) return false;
      if (elect_one()) mbar_arrive(&k_empty[jj & 1]);
      if (!warp_wait(&v_full[jj & 1], (jj >> 1) & 1)) return false;
      if (elect_one()) mbar_arrive(&v_empty[jj & 1]);
      __syncwarp();
    }
    return true;
  }
  // S of the first key tile, then by turns O of a tile and S of the next.
  __device__ __forceinline__ bool unit(int i0, int i1, int n) {
    const uint32_t begin = j, end = j + n;
    j = end;
    if (i1 <= i0) return pass(begin, end);
    const uint32_t a = begin + i0, z = begin + i1;
    if (!pass(begin, a) || !warp_wait(q_full, uses & 1) || !scores(a)) return false;
    ++uses;
    for (uint32_t jj = a; jj + 1 < z; ++jj)
      if (!output(jj, jj == a) || !scores(jj + 1)) return false;
    if (elect_one()) umma_commit(q_empty);
    if (!output(z - 1, z - 1 == a)) return false;
    if (elect_one()) umma_commit(o_full);
    return pass(z, end);
  }
};

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
  uint64_t* q_full = bars;                  // [2] per tile
  uint64_t* q_empty = q_full + 2;           // [2]
  uint64_t* k_full = q_empty + 2;           // [stages]
  uint64_t* k_empty = k_full + kFwdStages;
  uint64_t* v_full = k_empty + kFwdStages;
  uint64_t* v_empty = v_full + kFwdStages;
  uint64_t* s_full = v_empty + kFwdStages;  // [2] per tile
  uint64_t* p_full = s_full + 2;            // [2][2]: tile, first 96 and last 32 keys
  uint64_t* turn_over = p_full + 4;         // [2]
  uint64_t* o_full = turn_over + 2;         // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kFwdStages; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 2);  // the MMA warps
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 2);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], 1);
      mbar_init(&q_empty[t], 1);
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[2 * t], 4);
      mbar_init(&p_full[2 * t + 1], 4);
      mbar_init(&turn_over[t], 4);
      mbar_init(&o_full[t], 1);
    }
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
  const uint32_t tmem_s = tmem, tmem_o = tmem + 256;  // 128 columns each per tile

  // Every role goes through the block's units on its own; the barriers keep counting.
  int4 entry[2], next[2];
  int unit = nth_unit(0, p.units);
  fetch_unit(p.tiles, p.head_pairs, p.heads, unit, entry);

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");  // 168 a thread at launch: 3 * 168 = 2 * 208 + 88
    if (warp == 8) {
      if (lane == 0) {
        bool ok = true;
        int j = 0, uses[2] = {0, 0};
        for (int r = 0; unit >= 0 && ok; ++r) {
          const int after = nth_unit(r + 1, p.units);
          fetch_unit(p.tiles, p.head_pairs, p.heads, after, next);
          const QueryUnit u = query_unit(entry, p.head_pairs, p.heads, p.kv_heads, unit);
          for (int i = 0; i < u.n && ok; ++i, ++j) {
            const int st = j % kFwdStages;
            const uint32_t parity = ((j / kFwdStages) & 1) ^ 1;
            const int key = u.base + i * kTile;
            ok = mbar_wait_bounded(&k_empty[st], parity);
            if (!ok) break;
            mbar_expect_tx(&k_full[st], kTileBytes);
#pragma unroll
            for (int s = 0; s < kSlabs; ++s)
              tma_load_3d(k_tiles + st * kTileBytes + s * kSlabBytes, &map_k, &k_full[st], 64 * s, u.kv_head, key);
            for (int t = 0; t < 2 && i == 0 && ok; ++t) {
              if (u.i1[t] == 0) continue;
              ok = mbar_wait_bounded(&q_empty[t], (uses[t] & 1) ^ 1);
              if (!ok) break;
              ++uses[t];
              mbar_expect_tx(&q_full[t], kTileBytes);
#pragma unroll
              for (int s = 0; s < kSlabs; ++s)
                tma_load_3d(q_tiles + t * kTileBytes + s * kSlabBytes, &map_q, &q_full[t], 64 * s, u.head[t], u.row0[t]);
            }
            ok = ok && mbar_wait_bounded(&v_empty[st], parity);
            if (!ok) break;
            mbar_expect_tx(&v_full[st], kTileBytes);
#pragma unroll
            for (int s = 0; s < kSlabs; ++s)
              tma_load_3d(v_tiles + st * kTileBytes + s * kSlabBytes, &map_v, &v_full[st], 64 * s, u.kv_head, key);
          }
          unit = after;
          entry[0] = next[0];
          entry[1] = next[1];
        }
        if (!ok) {
          record_give_up(status, p.gave_up, kStatusTimeoutProducer);
          drain_copies();
        }
      }
      __syncwarp();
    } else if (warp < 11) {
      const int t = warp - 9;
      FwdMma<FMT, DP> mma;
      mma.tmem_s = tmem_s + 128 * t;
      mma.tmem_o = tmem_o + 128 * t;
      mma.q = make_kmajor_sw128_desc(smem_u32(q_tiles + t * kTileBytes));
      mma.k = make_kmajor_sw128_desc(smem_u32(k_tiles));
      mma.v = make_mnmajor_sw128_desc(smem_u32(v_tiles), kSlabBytes);
      mma.k_full = k_full;
      mma.k_empty = k_empty;
      mma.v_full = v_full;
      mma.v_empty = v_empty;
      mma.q_full = &q_full[t];
      mma.q_empty = &q_empty[t];
      mma.s_full = &s_full[t];
      mma.p_full = &p_full[2 * t];
      mma.o_full = &o_full[t];
      bool ok = true;
      for (int r = 0; unit >= 0 && ok; ++r) {
        const int after = nth_unit(r + 1, p.units);
        fetch_unit(p.tiles, p.head_pairs, p.heads, after, next);
        int i0, i1, n;
        {
          const QueryUnit u = query_unit(entry, p.head_pairs, p.heads, p.kv_heads, unit);
          i0 = t ? u.i0[1] : u.i0[0];
          i1 = t ? u.i1[1] : u.i1[0];
          n = u.n;
        }
        ok = mma.unit(i0, i1, n);
        unit = after;
        entry[0] = next[0];
        entry[1] = next[1];
      }
      if (!ok && lane == 0) record_give_up(status, p.gave_up, kStatusTimeoutMma);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    using T = typename Type16<FMT>::T;
    const int t = warp >> 2, quad = warp & 3;
    const uint32_t lane_base = uint32_t(quad * 32) << 16;
    const uint32_t ts = tmem_s + 128 * t + lane_base, to = tmem_o + 128 * t + lane_base;
    const float c = p.scale * kPackedLog2e;
    bool ok = true, bad = false;
    int steps = 0, uses = 0, turns = 0;
    // The two tiles take turns at the exponentials, tile 0 first: left alone they fall into step, and then
    // nobody computes under the products.  A tile takes its turn at every key tile of the unit, needed
    // or not, so neither is ever more than one ahead (a barrier tells only two phases apart).
    const auto my_turn = [&](int turn) {
      if (t == 0 && turn == 0) return true;
      return bool(__all_sync(0xffffffffu, mbar_wait_bounded(&turn_over[1 - t], (t ? turn : turn - 1) & 1)));
    };
    for (int r = 0; unit >= 0 && ok; ++r) {
      int i0, i1, warp_row0, head, base, n;
      {
        const QueryUnit u = query_unit(entry, p.head_pairs, p.heads, p.kv_heads, unit);
        i0 = t ? u.i0[1] : u.i0[0];
        i1 = t ? u.i1[1] : u.i1[0];
        warp_row0 = (t ? u.row0[1] : u.row0[0]) + quad * 32;
        head = t ? u.head[1] : u.head[0];
        base = u.base;
        n = u.n;
      }
      const int row = warp_row0 + lane;
      const bool in = row < p.valid;
      const int first = in ? __ldg(p.first_key + row) : 0x7fffffff;
      // The warp's rows attend all of a key tile from `all_from` on, up to its first row, and nothing of it
      // in front of `any_from`.
      const int all_from = __shfl_sync(0xffffffffu, first, 31), any_from = __shfl_sync(0xffffffffu, first, 0);
      float m = -INFINITY, l = 0.f;  // m: the base in use, of the unscaled scores
      for (int i = 0; i < n; ++i, ++turns) {
        if (i < i0 || i >= i1) {  // only the other tile needs this key tile
          ok = my_turn(turns);
          if (!ok) break;
          if (lane == 0) mbar_arrive(&turn_over[t]);
          continue;
        }
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(&s_full[t], steps & 1));
        if (!ok) break;
        tc_fence_after();
        const int key = base + i * kTile;
        const bool masked = key + kTile - 1 > warp_row0 || key < all_from;
        const int from = first - key, upto = row - key;  // columns of the row's own range
        uint32_t s[4][32];
#pragma unroll
        for (int g = 0; g < 4; ++g) tmem_ld_32(ts + 32 * g, s[g]);
        tmem_ld_wait();
#pragma unroll
        for (int g = 0; g < 4; ++g) pin_32(s[g]);
        // Chunks of 32 keys that some row of the warp attends: [g0, g1).  With short documents they are few.
        const int g0 = masked ? max(any_from - key, 0) >> 5 : 0, g1 = masked ? ((warp_row0 + 31 - key) >> 5) + 1 : 4;
        float top = -INFINITY;
        if (masked) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            if (g < g0 || g >= g1) continue;
            hide(s[g], bit_range(from - 32 * g, upto - 32 * g), 0xff800000u);  // -inf
            top = max_chunk(s[g], top);
          }
        } else {
#pragma unroll
          for (int g = 0; g < 4; ++g) top = max_chunk(s[g], top);
        }
        // A new base where the maximum grew by more than 2^8 (or is the row's first).
        const bool grow = (top - m) * c > 8.f;
        if (__any_sync(0xffffffffu, grow)) {
          const float alpha = grow ? fast_exp2((m - top) * c) : 1.f;
          if (grow) m = top;
          l *= alpha;
          if (i > i0) {
#pragma unroll 1
            for (int d = 0; d < DP; d += 16) {
              float o[16];
              uint32_t scaled[16];
              tmem_ld_32x16(to + d, o);
#pragma unroll
              for (int e = 0; e < 16; ++e) scaled[e] = __float_as_uint(o[e] * alpha);
              tmem_st_16(to + d, scaled);
            }
          }
        }
        const float mc = m == -INFINITY ? 0.f : m * c;
        ok = my_turn(turns);
        if (!ok) break;
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        // Two copies of the code: tests between the chunks keep the whole tiles' exponentials from overlapping.
        const auto exps = [&](auto part) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          if (!decltype(part)::value || (g >= g0 && g < g1)) exp_chunk<FMT>(ts + 16 * g, s[g], c, mc, sum);
          else tmem_st_zero_16(ts + 16 * g);
          if (g == 1) {  // early: the handover takes about as long as the other half
            __syncwarp();
            if (lane == 0) mbar_arrive(&turn_over[t]);
          }
          if (g >= 2) {  // the second product starts on three quarters of the keys
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[2 * t + g - 2]);
          }
        }
        };
        if (masked) exps(std::true_type());
        else exps(std::false_type());
        ++steps;
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      }
      if (!ok) break;
      // the next unit, under what is left of this one
      unit = nth_unit(r + 1, p.units);
      fetch_unit(p.tiles, p.head_pairs, p.heads, unit, entry);
      const bool some = in && first <= row;
      const float bias2 = some ? p_shift<FMT>() - fmaf(m, c, log2f(l)) : -INFINITY;
      if (row < p.rows) p.bias2[long(head) * p.pitch + row] = bias2;
      const long at = (long(row) * p.heads + head) * p.dim;
      T* dst = static_cast<T*>(p.o) + at;
      T* rest = p.o_rest != nullptr ? static_cast<T*>(p.o_rest) + at : nullptr;
      if (i1 > i0) {
        ok = warp_wait(&o_full[t], uses & 1);
        ++uses;
        if (!ok) break;
        tc_fence_after();
        bad |= store_row<FMT, DP>(to, some ? 1.f / l : 0.f, dst, p.dim, some, -1, rest);
        tc_fence_before();
      }
      if (!some && row < p.rows)
        for (int d = 0; d < p.dim; d += 8) *reinterpret_cast<uint4*>(dst + d) = make_uint4(0, 0, 0, 0);
    }
    if (!ok && lane == 0) record_give_up(status, p.gave_up, kStatusTimeoutEpilogue);
    if (ok && __any_sync(0xffffffffu, bad)) {
      __syncwarp();  // the lanes' rows are read by all
      for (int r = 0; (unit = nth_unit(r, p.units)) >= 0; ++r) {
        fetch_unit(p.tiles, p.head_pairs, p.heads, unit, entry);
        const QueryUnit u = query_unit(entry, p.head_pairs, p.heads, p.kv_heads, unit);
        const int row0 = t ? u.row0[1] : u.row0[0], begin = row0 + quad * 32;
        for (int row = begin; row < min(begin + 32, p.valid); ++row)
          exact_forward_row<FMT, DP>(p, row0, row, t ? u.head[1] : u.head[0], lane);
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
