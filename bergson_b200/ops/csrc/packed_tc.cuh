// What the tensor-core kernels of the packed attention share: TMEM accesses, the MMA form that reads
// its A operand from TMEM, operand maps, and the exact recomputation of a tile's rows.
#pragma once

#include "common.cuh"
#include "kernels_packed.h"

namespace bgn {

constexpr int kTile = 128;                  // rows (queries or keys) of a tile
constexpr float kPackedLog2e = 1.4426950408889634f;

// Bytes of a [128 rows, DP features] operand tile: slabs of 64 features in the 128-byte swizzle.
template <int DP>
constexpr int tile_bytes() {
  return kTile * DP * 2;
}
constexpr int kSlabBytes = kTile * 128;

// D[tmem] (+)= A[tmem] * B[smem]: A has one row per lane, two 16-bit values of the reduction per column.
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "}"
      :
      : "r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// One lane of a converged warp, the same one every time.  Code under it is known to run in one thread:
// the MMA instructions' operands then need no detour through the vector registers, and a warp that
// issues them next to busy arithmetic warps needs few issue slots (a branch on the lane number took
// several times as many, and the tensor core went idle).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t"
      ".reg .pred q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t"
      "}"
      : "=r"(p));
  return p != 0;
}

// All lanes of a warp wait; false if the time ran out.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity));
}

// 32 lanes x 32 columns without waiting; tmem_ld_wait() makes the values of all loads before it usable.
__device__ __forceinline__ void tmem_ld_32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Ties values to the place in the program: what reads them cannot be moved in front of it.
__device__ __forceinline__ void pin_32(uint32_t (&r)[32]) {
  asm volatile(""
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]));
  asm volatile(""
               : "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}

__device__ __forceinline__ void tmem_st_16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
      :
      : "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}

__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Two values rounded to the 16-bit type, the first in the low half.
template <int FMT>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t r;
  if (FMT == 1) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

template <int FMT>
__device__ __forceinline__ float2 unpack16(uint32_t h) {
  if (FMT == 1) return make_float2(__uint_as_float(h << 16), __uint_as_float(h & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

template <int FMT>
struct Type16;
template <>
struct Type16<0> { using T = __half; };
template <>
struct Type16<1> { using T = __nv_bfloat16; };

// What the forward pass hands to the backward pass: P of a row is 2^(c q.k + bias2), times 2^10 for fp16,
// whose small values are few (see packed_bwd.cuh).
template <int FMT>
constexpr float p_shift() {
  return FMT == 0 ? 10.f : 0.f;
}

// Features of a row that a lane holds when a warp works on whole rows.
template <int FMT, int DP>
__device__ __forceinline__ void load_row(float (&x)[DP / 32], const void* base, long offset, int dim, int lane) {
  using T = typename Type16<FMT>::T;
  const T* p = static_cast<const T*>(base) + offset;
#pragma unroll
  for (int e = 0; e < DP / 32; ++e) x[e] = lane + 32 * e < dim ? to_float<T>(p[lane + 32 * e]) : 0.f;
}

// Whether a value of the rows [from, to) is infinite or NaN.
template <int FMT, int DP>
__device__ __forceinline__ bool some_not_finite(const void* base, long tok, long offset, int from, int to, int dim, int lane) {
  bool bad = false;
#pragma unroll 4
  for (int j = from; j < to; ++j) {
    float x[DP / 32];
    load_row<FMT, DP>(x, base, long(j) * tok + offset, dim, lane);
#pragma unroll
    for (int e = 0; e < DP / 32; ++e) bad |= !(fabsf(x[e]) < INFINITY);
  }
  return __any_sync(0xffffffffu, bad);
}

// Whether every value that counts is NaN, which no further sum changes.
template <int N>
__device__ __forceinline__ bool all_nan(const float (&x)[N], int from, int to, int lane) {
  bool yes = true;
#pragma unroll
  for (int e = 0; e < N; ++e) yes &= lane + 32 * e < from || lane + 32 * e >= to || isnan(x[e]);
  return __all_sync(0xffffffffu, yes);
}

template <int N>
__device__ __forceinline__ float warp_dot(const float (&x)[N], const float (&y)[N]) {
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < N; ++e) s = fmaf(x[e], y[e], s);
  return warp_sum(s);
}

// The kernels of a backward pass follow one another closely: each lets the next one's blocks come as soon as there is
// room on an SM, and they wait for the end of the kernel before them when they have set up what they need.
// 8187 tokens in facts, 12 heads of 64 in fp16: 83 us instead of 87 (bf16: 69 and 75); 1024 tokens, 32 over 8 heads of 128
// in bf16: 91 instead of 95.
__device__ __forceinline__ void next_kernel_may_come() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_last_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Records a wait that ran out: in the status word, then where the host sees it without asking the device.
__device__ __forceinline__ void record_give_up(int* status, int* gave_up, int code) {
  atomicCAS(status, kStatusOk, code);
  __threadfence_system();
  *reinterpret_cast<volatile int*>(gave_up) = 1;
}

// Gives up after a wait that ran out: long enough for every copy in flight to land.
__device__ __forceinline__ void drain_copies() {
  const long long start = clock64();
  while (clock64() - start < 400000) {
  }
}

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;"
      : "=l"(*reinterpret_cast<uint64_t*>(&d))
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)), "l"(*reinterpret_cast<uint64_t*>(&c)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.ftz.f32x2 %0, %1, %2;"
      : "=l"(*reinterpret_cast<uint64_t*>(&d))
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.ftz.f32x2 %0, %1, %2;"
      : "=l"(*reinterpret_cast<uint64_t*>(&d))
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.ftz.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Bits lo .. hi (those inside 0 .. 31).
__device__ __forceinline__ uint32_t bit_range(int lo, int hi) {
  const int l = lo > 0 ? lo : 0, h = hi < 31 ? hi : 31;
  return l <= h ? (0xffffffffu << l) & (0xffffffffu >> (31 - h)) : 0u;
}

__device__ __forceinline__ void tmem_st_zero_16(uint32_t taddr) {
  const uint32_t zeros[16] = {};
  tmem_st_16(taddr, zeros);
}

// Puts `value` where a bit of `keep` is not set.
__device__ __forceinline__ void hide(uint32_t (&x)[32], uint32_t keep, uint32_t value) {
#pragma unroll
  for (int e = 0; e < 32; ++e)
    if (!(keep & (1u << e))) x[e] = value;
}

__device__ __forceinline__ void store_v8(void* ptr, const uint32_t* r) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(ptr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// A thread's row of an accumulator in TMEM, scaled, rounded and stored to `dst` (dim features,
// 16-byte aligned); with `half` 0 or 1 only that half of the features.  `rest`, if any, gets what the
// rounding took away, rounded in its turn.  Returns whether some value is infinite or NaN.
template <int FMT, int DP>
__device__ __forceinline__ bool store_row(uint32_t tmem, float scale, void* dst, int dim, bool write, int half = -1,
                                          void* rest = nullptr) {
  const bool wide = (dim & 15) == 0;  // every row begins on a 32-byte boundary then
  bool bad = false;
#pragma unroll 1
  for (int c = half == 1 ? DP / 2 : 0; c < (half == 0 ? DP / 2 : DP); c += 32) {
    if (c >= dim) break;
    uint32_t r[32];
    tmem_ld_32(tmem + c, r);
    tmem_ld_wait();
    pin_32(r);
    if (write) {
      uint32_t h[16];
      const auto store = [&](void* to) {
        uint8_t* at = static_cast<uint8_t*>(to) + c * 2;
        if (wide) {
          store_v8(at, h);
          if (c + 16 < dim) store_v8(at + 32, h + 8);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (c + 8 * i < dim)
              *reinterpret_cast<uint4*>(at + 16 * i) = make_uint4(h[4 * i], h[4 * i + 1], h[4 * i + 2], h[4 * i + 3]);
        }
      };
      float largest = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float x = __uint_as_float(r[2 * i]) * scale, y = __uint_as_float(r[2 * i + 1]) * scale;
        asm("max.NaN.ftz.f32 %0, %0, %1;" : "+f"(largest) : "f"(fabsf(x)));
        asm("max.NaN.ftz.f32 %0, %0, %1;" : "+f"(largest) : "f"(fabsf(y)));
        h[i] = pack16<FMT>(x, y);
      }
      bad |= !(largest < INFINITY);
      store(dst);
      if (rest != nullptr) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float2 kept = unpack16<FMT>(h[i]);
          h[i] = pack16<FMT>(fmaf(__uint_as_float(r[2 * i]), scale, -kept.x),
                             fmaf(__uint_as_float(r[2 * i + 1]), scale, -kept.y));
        }
        store(rest);
      }
    }
    __syncwarp();
  }
  return bad;
}

}  // namespace bgn
