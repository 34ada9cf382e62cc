// Host side of the attention over packed documents.
#include <mutex>
#include <set>
#include <utility>

#include "packed_bwd.cuh"
#include "packed_fwd.cuh"
#include "packed_simple.cuh"

using namespace bgn;

namespace {

// What a launch has to know of the current device.
cudaError_t sm_count(int* n) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  return e == cudaSuccess ? cudaDeviceGetAttribute(n, cudaDevAttrMultiProcessorCount, device) : e;
}

// cudaFuncSetAttribute holds for the current device only; it is asked for once per kernel and device.
cudaError_t allow_smem(const void* kernel, int bytes) try {
  static std::mutex mu;
  static std::set<std::pair<const void*, int>> done;
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> lock(mu);
  if (done.count({kernel, device})) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.insert({kernel, device});
  return e;
} catch (...) {  // the entries are C
  return cudaErrorMemoryAllocation;
}

template <int DP, int R>
cudaError_t simple_fwd(const BgnPackedAttention& a, void* o, float* bias2, cudaStream_t stream) {
  constexpr int smem = simple_smem<DP>(3);
  auto kern = packed_fwd_simple_kernel<DP, R>;
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(kern), smem);
  if (e != cudaSuccess) return e;
  const unsigned grid = unsigned((a.rows + 127) / 128) * 2u * unsigned(a.heads);
  kern<<<grid, simple_threads<R>(), smem, stream>>>(a, static_cast<float*>(o), bias2);
  return cudaGetLastError();
}

template <int DP, int R>
cudaError_t simple_bwd(const BgnPackedAttention& a, const void* o, const float* bias2, const void* d_o, long do_tok,
                       long do_head, float* delta, void* dq, void* dk, void* dv, cudaStream_t stream) {
  constexpr int smem = simple_smem<DP>(4);
  auto kq = packed_dq_simple_kernel<DP, R>;
  auto kk = packed_dkv_simple_kernel<DP, R>;
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(kq), smem);
  if (e == cudaSuccess) e = allow_smem(reinterpret_cast<const void*>(kk), smem);
  if (e != cudaSuccess) return e;
  const unsigned tiles = unsigned((a.rows + 127) / 128) * 2u;
  kq<<<tiles * unsigned(a.heads), simple_threads<R>(), smem, stream>>>(a, static_cast<const float*>(o), bias2,
                                                                  static_cast<const float*>(d_o), do_tok, do_head, delta,
                                                                  static_cast<float*>(dq));
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  kk<<<tiles * unsigned(a.kv_heads), simple_threads<R>(), smem, stream>>>(a, bias2, static_cast<const float*>(d_o), do_tok,
                                                                     do_head, delta, static_cast<float*>(dk),
                                                                     static_cast<float*>(dv));
  return cudaGetLastError();
}

// fp32: eight rows to a thread take fewer loads from shared memory for the same operations than four, and half the
// threads.  Up to 64 features that is faster in the forward pass (8 documents of 1024, 12 heads of 64: 435 against
// 480 us; 7 of 2000 tokens together, 4 heads of 32: 30 against 34); in the backward pass where there are more than
// two blocks to an SM (1363 against 1462 us; but 91 against 86 for the small batch).  At 128 features the registers do
// not suffice (2 of 2048, 16 over 4 heads: forward 1706 against 1239 us).
bool many_blocks(const BgnPackedAttention& a) {
  return (a.rows + 127) / 128 * 2 * a.heads > 2 * 148;
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static const EncodeTiledFn fn = []() -> EncodeTiledFn {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q);
    return e == cudaSuccess && q == cudaDriverEntryPointSuccess ? reinterpret_cast<EncodeTiledFn>(ptr) : nullptr;
  }();
  return fn;
}

// [tokens, heads, dim] in boxes of 128 tokens x 64 features of one head.  Rows behind the last document
// and features past dim are outside the map and read as zeros, whatever stands there.
bool operand_map(CUtensorMap* map, const void* base, int fmt, int dim, int heads, int valid, long head, long tok) {
  EncodeTiledFn enc = encode_fn();
  if (!enc || (reinterpret_cast<uintptr_t>(base) & 15) || head % 8 || tok % 8) return false;
  cuuint64_t dims[3] = {cuuint64_t(dim), cuuint64_t(heads), cuuint64_t(valid > 0 ? valid : 1)};
  cuuint64_t strides[2] = {cuuint64_t(head) * 2, cuuint64_t(tok) * 2};
  cuuint32_t box[3] = {64, 1, cuuint32_t(kTile)};
  cuuint32_t one[3] = {1, 1, 1};
  return enc(map, fmt == 1 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
             const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int FMT, int DP>
cudaError_t tensor_fwd(const BgnPackedAttention& a, void* o, void* o_rest, float* bias2, int* status, cudaStream_t stream) {
  ensure_context_bound();
  CUtensorMap mq, mk, mv;
  if (!operand_map(&mq, a.q, FMT, a.dim, a.heads, a.valid, a.q_head, a.q_tok) ||
      !operand_map(&mk, a.k, FMT, a.dim, a.kv_heads, a.valid, a.k_head, a.k_tok) ||
      !operand_map(&mv, a.v, FMT, a.dim, a.kv_heads, a.valid, a.v_head, a.v_tok))
    return cudaErrorInvalidValue;
  PackedFwdArgs p = {};
  // Two heads of a group always see the same keys; two row tiles of a head do not.
  p.head_pairs = (a.heads / a.kv_heads) % 2 == 0;
  p.first_key = a.first_key;
  const int tiles = (a.rows + kTile - 1) / kTile;
  p.tiles = reinterpret_cast<const int4*>(p.head_pairs ? a.query_tiles : a.query_pairs);
  p.units = p.head_pairs ? tiles * (a.heads / 2) : (tiles + 1) / 2 * a.heads;
  p.rows = a.rows;
  p.valid = a.valid;
  p.pitch = a.pitch;
  p.heads = a.heads;
  p.kv_heads = a.kv_heads;
  p.dim = a.dim;
  p.scale = a.scale;
  p.q = a.q;
  p.k = a.k;
  p.v = a.v;
  p.q_tok = a.q_tok;
  p.q_head = a.q_head;
  p.k_tok = a.k_tok;
  p.k_head = a.k_head;
  p.v_tok = a.v_tok;
  p.v_head = a.v_head;
  p.o = o;
  p.o_rest = o_rest;
  p.bias2 = bias2;
  p.gave_up = a.gave_up;
  constexpr int smem = fwd_smem_bytes<DP>();
  auto kern = packed_fwd_kernel<FMT, DP>;
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(kern), smem);
  if (e != cudaSuccess) return e;
  int sms = 0;
  e = sm_count(&sms);
  if (e != cudaSuccess) return e;
  kern<<<unsigned(p.units < sms ? p.units : sms), kFwdThreads, smem, stream>>>(mq, mk, mv, p, status);
  return cudaGetLastError();
}

// Launches a kernel of the backward pass whose blocks may come before the one before it has ended.  For kernels
// with one block to an SM only: small blocks (fp32) that come early crowd on the SMs that were free first (242 against 177 us).
template <typename... Args>
cudaError_t launch_next(void (*kernel)(Args...), int blocks, int smem, cudaStream_t stream, Args... args) {
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(blocks));
  cfg.blockDim = dim3(kBwdThreads);
  cfg.dynamicSmemBytes = size_t(smem);
  cfg.stream = stream;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <int FMT, int DP>
cudaError_t tensor_bwd(const BgnPackedAttention& a, const void* o, const void* o_rest, const float* bias2, const void* d_o, long do_tok,
                       long do_head, float* delta, float* ds_bounds, void* dq, void* dk, void* dv, int* status,
                       cudaStream_t stream) {
  ensure_context_bound();
  CUtensorMap mq, mk, mv, mg;
  if (!operand_map(&mq, a.q, FMT, a.dim, a.heads, a.valid, a.q_head, a.q_tok) ||
      !operand_map(&mk, a.k, FMT, a.dim, a.kv_heads, a.valid, a.k_head, a.k_tok) ||
      !operand_map(&mv, a.v, FMT, a.dim, a.kv_heads, a.valid, a.v_head, a.v_tok) ||
      !operand_map(&mg, d_o, FMT, a.dim, a.heads, a.valid, do_head, do_tok))
    return cudaErrorInvalidValue;
  PackedBwdArgs p = {};
  p.first_key = a.first_key;
  p.end_query = a.end_query;
  p.rows = a.rows;
  p.valid = a.valid;
  p.heads = a.heads;
  p.kv_heads = a.kv_heads;
  p.dim = a.dim;
  p.pitch = a.pitch;
  p.scale = a.scale;
  p.q = a.q;
  p.k = a.k;
  p.v = a.v;
  p.o = o;
  p.o_rest = o_rest;
  p.d_o = d_o;
  p.q_tok = a.q_tok;
  p.q_head = a.q_head;
  p.k_tok = a.k_tok;
  p.k_head = a.k_head;
  p.v_tok = a.v_tok;
  p.v_head = a.v_head;
  p.do_tok = do_tok;
  p.do_head = do_head;
  p.bias2 = bias2;
  p.neg_delta = delta;
  if (FMT == 0) {
    const long heads = long(a.heads) * a.pitch;
    p.row_do = ds_bounds;
    p.doc_do = ds_bounds + heads;
    p.doc_delta = ds_bounds + 2 * heads;
    p.doc_v = ds_bounds + 3 * heads;
  }
  p.dq = dq;
  p.dk = dk;
  p.dv = dv;
  p.gave_up = a.gave_up;
  auto kq = packed_dq_kernel<FMT, DP>;
  auto kk = packed_dkv_kernel<FMT, DP>;
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(kq), dq_smem_bytes<DP>());
  if (e == cudaSuccess) e = allow_smem(reinterpret_cast<const void*>(kk), dkv_smem_bytes<DP>());
  if (e != cudaSuccess) return e;
  int sms = 0;
  e = sm_count(&sms);
  if (e != cudaSuccess) return e;
  const int tiles = (a.rows + kTile - 1) / kTile;
  constexpr int kLanes = DP / 8;
  packed_delta_kernel<FMT, kLanes><<<unsigned(4 * tiles) * unsigned(a.heads), delta_threads<FMT, kLanes>(), 0, stream>>>(p);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  p.tiles = reinterpret_cast<const int4*>(a.query_tiles);
  p.units = tiles * a.heads;
  e = launch_next(kq, p.units < sms ? p.units : sms, dq_smem_bytes<DP>(), stream, mq, mg, mk, mv, p, status);
  if (e != cudaSuccess) return e;
  p.tiles = reinterpret_cast<const int4*>(a.key_tiles);
  p.units = tiles * a.kv_heads;
  return launch_next(kk, p.units < sms ? p.units : sms, dkv_smem_bytes<DP>(), stream, mq, mg, mk, mv, p, status);
}

bool sound(const BgnPackedAttention* a) {
  return a->rows > 0 && a->pitch >= a->rows && a->pitch % kTile == 0 && a->valid >= 0 && a->valid <= a->rows && a->heads > 0 && a->kv_heads > 0 &&
         a->heads % a->kv_heads == 0 && a->dim >= 8 && a->dim <= 128 && a->dim % 8 == 0 && a->type >= 0 && a->type <= 2 &&
         a->scale > 0.f && a->gave_up != nullptr;
}

}  // namespace

extern "C" int bgn_packed_attention_fwd(const BgnPackedAttention* a, void* o, void* o_rest, float* bias2, int* status,
                                        cudaStream_t stream) {
  if (!sound(a)) return int(cudaErrorInvalidValue);
  const bool narrow = a->dim <= 64;
  if (a->type == 2) {
    auto run = a->dim <= 32 ? simple_fwd<32, 8> : narrow ? simple_fwd<64, 8> : simple_fwd<128, 4>;
    return int(run(*a, o, bias2, stream));
  }
  if (a->type == 1)
    return int(narrow ? tensor_fwd<1, 64>(*a, o, o_rest, bias2, status, stream) : tensor_fwd<1, 128>(*a, o, o_rest, bias2, status, stream));
  return int(narrow ? tensor_fwd<0, 64>(*a, o, o_rest, bias2, status, stream) : tensor_fwd<0, 128>(*a, o, o_rest, bias2, status, stream));
}

extern "C" int bgn_packed_attention_bwd(const BgnPackedAttention* a, const void* o, const void* o_rest,
                                        const float* bias2, const void* d_o,
                                        long do_tok, long do_head, float* delta, float* ds_bounds, void* dq, void* dk,
                                        void* dv, int* status, cudaStream_t stream) {
  if (!sound(a)) return int(cudaErrorInvalidValue);
  const bool narrow = a->dim <= 64;
  if (a->type == 2) {
    auto run = simple_bwd<128, 4>;
    if (narrow && many_blocks(*a)) run = a->dim <= 32 ? simple_bwd<32, 8> : simple_bwd<64, 8>;
    else if (narrow) run = a->dim <= 32 ? simple_bwd<32, 4> : simple_bwd<64, 4>;
    return int(run(*a, o, bias2, d_o, do_tok, do_head, delta, dq, dk, dv, stream));
  }
  auto run = a->type == 1 ? (narrow ? tensor_bwd<1, 64> : tensor_bwd<1, 128>)
                          : (narrow ? tensor_bwd<0, 64> : tensor_bwd<0, 128>);
  if (o_rest == nullptr || (a->type == 0 && ds_bounds == nullptr)) return int(cudaErrorInvalidValue);
  return int(run(*a, o, o_rest, bias2, d_o, do_tok, do_head, delta, ds_bounds, dq, dk, dv, status, stream));
}
