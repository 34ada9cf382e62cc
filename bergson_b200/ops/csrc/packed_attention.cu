// Host side of the attention over packed documents.
#include "packed_simple.cuh"

using namespace bgn;

namespace {

// cudaFuncSetAttribute holds for the current device only.
cudaError_t allow_smem(const void* kernel, int bytes) {
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

template <typename T, int DP>
cudaError_t simple_fwd(const BgnPackedAttention& a, void* o, float* lse2, cudaStream_t stream) {
  constexpr int smem = simple_smem<DP>(3);
  auto kern = packed_fwd_simple_kernel<T, DP>;
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(kern), smem);
  if (e != cudaSuccess) return e;
  const unsigned grid = unsigned((a.rows + 127) / 128) * 2u * unsigned(a.heads);
  kern<<<grid, kSimpleThreads, smem, stream>>>(a, static_cast<T*>(o), lse2);
  return cudaGetLastError();
}

template <typename T, int DP>
cudaError_t simple_bwd(const BgnPackedAttention& a, const void* o, const float* lse2, const void* d_o, long do_tok,
                       long do_head, float* delta, void* dq, void* dk, void* dv, cudaStream_t stream) {
  constexpr int smem = simple_smem<DP>(4);
  auto kq = packed_dq_simple_kernel<T, DP>;
  auto kk = packed_dkv_simple_kernel<T, DP>;
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(kq), smem);
  if (e == cudaSuccess) e = allow_smem(reinterpret_cast<const void*>(kk), smem);
  if (e != cudaSuccess) return e;
  const unsigned tiles = unsigned((a.rows + 127) / 128) * 2u;
  kq<<<tiles * unsigned(a.heads), kSimpleThreads, smem, stream>>>(a, static_cast<const T*>(o), lse2,
                                                                  static_cast<const T*>(d_o), do_tok, do_head, delta,
                                                                  static_cast<T*>(dq));
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  kk<<<tiles * unsigned(a.kv_heads), kSimpleThreads, smem, stream>>>(a, lse2, static_cast<const T*>(d_o), do_tok,
                                                                     do_head, delta, static_cast<T*>(dk),
                                                                     static_cast<T*>(dv));
  return cudaGetLastError();
}

bool sound(const BgnPackedAttention* a) {
  return a->rows > 0 && a->valid >= 0 && a->valid <= a->rows && a->heads > 0 && a->kv_heads > 0 &&
         a->heads % a->kv_heads == 0 && a->dim >= 8 && a->dim <= 128 && a->dim % 8 == 0 && a->type >= 0 && a->type <= 2 &&
         a->scale > 0.f;
}

}  // namespace

extern "C" int bgn_packed_attention_fwd(const BgnPackedAttention* a, void* o, float* lse2, int* status,
                                        cudaStream_t stream) {
  if (!sound(a)) return int(cudaErrorInvalidValue);
  (void)status;
  if (a->type == 2) return int(a->dim <= 64 ? simple_fwd<float, 64>(*a, o, lse2, stream) : simple_fwd<float, 128>(*a, o, lse2, stream));
  if (a->type == 1)
    return int(a->dim <= 64 ? simple_fwd<__nv_bfloat16, 64>(*a, o, lse2, stream)
                            : simple_fwd<__nv_bfloat16, 128>(*a, o, lse2, stream));
  return int(a->dim <= 64 ? simple_fwd<__half, 64>(*a, o, lse2, stream) : simple_fwd<__half, 128>(*a, o, lse2, stream));
}

extern "C" int bgn_packed_attention_bwd(const BgnPackedAttention* a, const void* o, const float* lse2, const void* d_o,
                                        long do_tok, long do_head, float* delta, void* dq, void* dk, void* dv,
                                        int* status, cudaStream_t stream) {
  if (!sound(a)) return int(cudaErrorInvalidValue);
  (void)status;
#define SIMPLE(T) \
  return int(a->dim <= 64 ? simple_bwd<T, 64>(*a, o, lse2, d_o, do_tok, do_head, delta, dq, dk, dv, stream) \
                          : simple_bwd<T, 128>(*a, o, lse2, d_o, do_tok, do_head, delta, dq, dk, dv, stream))
  if (a->type == 2) SIMPLE(float);
  if (a->type == 1) SIMPLE(__nv_bfloat16);
  SIMPLE(__half);
#undef SIMPLE
}
