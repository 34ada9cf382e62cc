// Python bindings of the operators on packed documents and of the distillation loss: checks,
// allocation of outputs, current-stream lookup.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/CUDAGraphsUtils.cuh>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/extension.h>

#include <cstring>
#include <mutex>

#include "bindings.h"
#include "kernels_distill.h"
#include "kernels_packed.h"

namespace {

int type_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kHalf: return 0;
    case at::kBFloat16: return 1;
    case at::kFloat: return 2;
    default: TORCH_CHECK(false, "bergson_b200: unsupported dtype ", t.scalar_type());
  }
}

void ran(int err, const char* what) {
  TORCH_CHECK(err == 0, "bergson_b200: ", what, " failed: ", cudaGetErrorString(static_cast<cudaError_t>(err)));
}

cudaStream_t current() { return at::cuda::getCurrentCUDAStream().stream(); }

// [tokens, heads, dim] as the kernels read it: contiguous features, heads and tokens on 16-byte
// boundaries, the token stride a multiple of the head stride.  Anything else is copied.
at::Tensor readable(const at::Tensor& x) {
  const int64_t packet = 16 / x.element_size();
  const int64_t st = x.stride(0), sh = x.stride(1);
  const bool heads_ok = x.size(1) == 1 || (sh >= x.size(2) && sh % packet == 0);
  const int64_t head = x.size(1) == 1 ? x.size(2) : sh;
  const bool tokens_ok = !heads_ok || x.size(0) == 1 || (st >= head * x.size(1) && st % packet == 0 && st % head == 0);
  const bool aligned = reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
  return (x.stride(2) == 1 || x.size(2) == 1) && heads_ok && tokens_ok && aligned ? x : x.clone(at::MemoryFormat::Contiguous);
}

// Strides of a readable tensor; those of a single head or token are never used but must be sound.
std::pair<long, long> strides_of(const at::Tensor& x) {
  const long head = x.size(1) == 1 ? x.size(2) : x.stride(1);
  const long tok = x.size(0) == 1 ? head * x.size(1) : x.stride(0);
  return {tok, head};
}

void check_packed(const at::Tensor& q, const at::Tensor& k) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 3 && k.dim() == 3 && q.size(0) == k.size(0) && q.size(2) == k.size(2) &&
                  q.scalar_type() == k.scalar_type() && k.device() == q.device(),
              "bergson_b200: q [T, H, D] and k [T, H_kv, D] of one dtype and device expected");
}

// One word a device in the host's memory, which kernels that give up on a wait set: a call can look at it without
// asking the device.
int* gave_up_word(int device) {
  constexpr int kMost = 64;
  static std::mutex mu;
  static int* words = nullptr;
  TORCH_CHECK(device >= 0 && device < kMost, "bergson_b200: device ", device);
  std::lock_guard<std::mutex> lock(mu);
  if (words == nullptr) {
    c10::cuda::CUDAStreamCaptureModeGuard relaxed{cudaStreamCaptureModeRelaxed};  // the first call may be captured
    void* host = nullptr;
    C10_CUDA_CHECK(cudaHostAlloc(&host, kMost * sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped));
    std::memset(host, 0, kMost * sizeof(int));
    words = static_cast<int*>(host);
  }
  return words + device;
}

// Raises if an attention kernel on the device gave up since the status word was last cleared.
int* check_waits(const at::Tensor& like) {
  int* word = gave_up_word(like.get_device());
  volatile int* seen = word;
  if (*seen == 0) return word;
  int status = -1;
  if (at::cuda::currentStreamCaptureStatus() == at::cuda::CaptureStatus::None) {
    status = kernel_status(like.get_device()).item<int>();
    if (status == 0) {  // cleared by whoever looked into it
      *seen = 0;
      return word;
    }
  }
  TORCH_CHECK(false, "bergson_b200: a kernel of packed_causal_attention gave up on a bounded wait (status ", status,
              "); its results are incomplete.  ops.native.kernel_status(device).zero_() clears this.");
}

at::Tensor packed_gave_up(int64_t device) {
  return at::from_blob(gave_up_word(int(device)), {1}, at::TensorOptions().dtype(at::kInt));
}

// The plan's table was allocated on the stream that was current then and may be dropped while kernels of another one
// still read it.
void keep_plan(const at::Tensor& part) {
  c10::cuda::CUDACachingAllocator::recordStream(part.storage().data_ptr(), at::cuda::getCurrentCUDAStream());
}

void check_index(const at::Tensor& x, int64_t n, const at::Tensor& like) {
  TORCH_CHECK(x.scalar_type() == at::kInt && x.is_contiguous() && x.device() == like.device() && x.numel() == n,
              "bergson_b200: the packing does not fit the tensors");
}

BgnPackedAttention packed_args(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& first_key,
                               const at::Tensor& end_query, const at::Tensor& query_tiles,
                               const at::Tensor& query_pairs, const at::Tensor& key_tiles,
                               int64_t valid, double scale) {
  const int64_t rows = q.size(0), tiles = (rows + 127) / 128;
  check_packed(q, k);
  TORCH_CHECK(v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type() && v.device() == k.device(),
              "bergson_b200: k and v must be alike");
  TORCH_CHECK(rows < (int64_t(1) << 30) && valid >= 0 && valid <= rows, "bergson_b200: row count out of range");
  TORCH_CHECK(4 * tiles * q.size(1) < (int64_t(1) << 31), "bergson_b200: too many tiles for one launch");
  check_index(first_key, rows, q);
  check_index(end_query, rows, q);
  check_index(query_tiles, 4 * tiles, q);
  check_index(query_pairs, 8 * ((rows + 255) / 256), q);
  check_index(key_tiles, 4 * tiles, q);
  for (const auto* t : {&query_tiles, &query_pairs, &key_tiles})
    TORCH_CHECK(reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0, "bergson_b200: tile tables on 16-byte boundaries");
  BgnPackedAttention a = {};
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  std::tie(a.q_tok, a.q_head) = strides_of(q);
  std::tie(a.k_tok, a.k_head) = strides_of(k);
  std::tie(a.v_tok, a.v_head) = strides_of(v);
  a.first_key = first_key.data_ptr<int>();
  a.end_query = end_query.data_ptr<int>();
  a.query_tiles = query_tiles.data_ptr<int>();
  a.query_pairs = query_pairs.data_ptr<int>();
  a.key_tiles = key_tiles.data_ptr<int>();
  a.rows = int(rows);
  a.pitch = int(128 * tiles);
  a.valid = int(valid);
  a.heads = int(q.size(1));
  a.kv_heads = int(k.size(1));
  a.dim = int(q.size(2));
  a.type = type_of(q);
  a.scale = float(scale);
  keep_plan(first_key);  // one storage holds all of the plan
  return a;
}

std::vector<at::Tensor> packed_attention_fwd(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor first_key,
                                             at::Tensor end_query, at::Tensor query_tiles, at::Tensor query_pairs, at::Tensor key_tiles,
                                             int64_t valid, double scale, bool backward) {
  c10::cuda::CUDAGuard guard(q.device());
  check_packed(q, k);
  q = readable(q);
  k = readable(k);
  v = readable(v);
  auto a = packed_args(q, k, v, first_key, end_query, query_tiles, query_pairs, key_tiles, valid, scale);
  a.gave_up = check_waits(q);
  auto o = at::empty({q.size(0), q.size(1), q.size(2)}, q.options());
  auto bias2 = at::empty({q.size(1), a.pitch}, q.options().dtype(at::kFloat));
  at::Tensor rest;
  if (backward && a.type != 2) rest = at::empty_like(o);
  ran(bgn_packed_attention_fwd(&a, o.data_ptr(), rest.defined() ? rest.data_ptr() : nullptr, bias2.data_ptr<float>(),
                               bgn_status_word(q), current()),
      "packed_attention_fwd");
  if (rest.defined()) return {o, bias2, rest};
  return {o, bias2};
}

std::vector<at::Tensor> packed_attention_bwd(at::Tensor d_o, at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor o,
                                             at::Tensor bias2, c10::optional<at::Tensor> rest, at::Tensor first_key, at::Tensor end_query,
                                             at::Tensor query_tiles, at::Tensor query_pairs, at::Tensor key_tiles, int64_t valid, double scale) {
  c10::cuda::CUDAGuard guard(q.device());
  check_packed(q, k);
  q = readable(q);
  k = readable(k);
  v = readable(v);
  TORCH_CHECK(d_o.sizes() == q.sizes() && d_o.scalar_type() == q.scalar_type() && d_o.device() == q.device() &&
                  o.sizes() == q.sizes() && o.scalar_type() == q.scalar_type() && o.is_contiguous() &&
                  bias2.scalar_type() == at::kFloat && bias2.is_contiguous() && bias2.numel() == (q.size(0) + 127) / 128 * 128 * q.size(1),
              "bergson_b200: the output's gradient does not fit the operands");
  TORCH_CHECK(!rest.has_value() || (rest->sizes() == o.sizes() && rest->scalar_type() == o.scalar_type() &&
                                    rest->is_contiguous() && rest->device() == o.device()),
              "bergson_b200: the output's rest does not fit the output");
  d_o = readable(d_o);
  auto a = packed_args(q, k, v, first_key, end_query, query_tiles, query_pairs, key_tiles, valid, scale);
  a.gave_up = check_waits(q);
  auto delta = at::empty_like(bias2);
  auto ds_bounds = at::empty({a.type == 0 ? (3 * q.size(1) + k.size(1)) * a.pitch : 0}, bias2.options());
  auto dq = at::empty({q.size(0), q.size(1), q.size(2)}, q.options());
  auto dk = at::empty({k.size(0), k.size(1), k.size(2)}, k.options());
  auto dv = at::empty_like(dk);
  const auto [tok, head] = strides_of(d_o);
  ran(bgn_packed_attention_bwd(&a, o.data_ptr(), rest.has_value() ? rest->data_ptr() : nullptr, bias2.data_ptr<float>(), d_o.data_ptr(), tok, head,
                               delta.data_ptr<float>(), a.type == 0 ? ds_bounds.data_ptr<float>() : nullptr, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                               bgn_status_word(q), current()),
      "packed_attention_bwd");
  return {dq, dk, dv};
}

std::vector<at::Tensor> packed_rotary_turn(at::Tensor q, at::Tensor k, at::Tensor cos, at::Tensor sin,
                                           at::Tensor position, int64_t rot, bool inverse) {
  c10::cuda::CUDAGuard guard(q.device());
  check_packed(q, k);
  check_index(position, q.size(0), q);
  keep_plan(position);
  TORCH_CHECK(cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat && cos.is_contiguous() &&
                  sin.is_contiguous() && cos.sizes() == sin.sizes() && cos.dim() == 2 && cos.size(1) == rot / 2 &&
                  cos.device() == q.device() && sin.device() == q.device(),
              "bergson_b200: rotary tables [positions, rot / 2] in fp32 expected");
  const auto inner = [](const at::Tensor& x) {
    return x.size(2) == 1 || x.stride(2) == 1 ? x : x.clone(at::MemoryFormat::Contiguous);
  };
  q = inner(q);
  k = inner(k);
  BgnPackedRotary a = {};
  auto qo = at::empty({q.size(0), q.size(1), q.size(2)}, q.options());
  auto ko = at::empty({k.size(0), k.size(1), k.size(2)}, k.options());
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.q_tok = q.stride(0);
  a.q_head = q.stride(1);
  a.k_tok = k.stride(0);
  a.k_head = k.stride(1);
  a.position = position.data_ptr<int>();
  a.cos = cos.data_ptr<float>();
  a.sin = sin.data_ptr<float>();
  a.q_out = qo.data_ptr();
  a.k_out = ko.data_ptr();
  a.rows = int(q.size(0));
  a.heads = int(q.size(1));
  a.kv_heads = int(k.size(1));
  a.dim = int(q.size(2));
  a.rot = int(rot);
  a.type = type_of(q);
  a.sign = inverse ? -1.f : 1.f;
  ran(bgn_packed_rotary(&a, current()), "packed_rotary");
  return {qo, ko};
}

BgnDistill distill_args(const at::Tensor& logits, const at::Tensor& ids, const at::Tensor& teacher, double temperature) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && logits.stride(1) == 1 && logits.stride(0) >= logits.size(1),
              "bergson_b200: logits [T, V] with contiguous rows expected");
  TORCH_CHECK(ids.dim() == 2 && ids.sizes() == teacher.sizes() && ids.size(0) == logits.size(0) && ids.is_contiguous() &&
                  teacher.is_contiguous() && ids.device() == logits.device() && teacher.device() == logits.device() &&
                  (ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt),
              "bergson_b200: teacher ids and logits [T, K] expected");
  TORCH_CHECK(logits.size(1) < (int64_t(1) << 30), "bergson_b200: vocabulary out of range");
  BgnDistill a = {};
  a.logits = logits.data_ptr();
  a.ids = ids.data_ptr();
  a.teacher = teacher.data_ptr();
  a.pitch = logits.stride(0);
  a.tokens = logits.size(0);
  a.vocab = int(logits.size(1));
  a.top = int(ids.size(1));
  a.type = type_of(logits);
  a.teacher_type = type_of(teacher);
  a.ids_64 = ids.scalar_type() == at::kLong;
  a.temperature = float(temperature);
  return a;
}

// Rows the kernels can walk; a single row's pitch is of no account.
at::Tensor rows_of(const at::Tensor& x) {
  return x.stride(1) == 1 && x.stride(0) >= x.size(1) ? x : x.clone(at::MemoryFormat::Contiguous);
}

std::vector<at::Tensor> distill_fwd(at::Tensor logits, at::Tensor ids, at::Tensor teacher, double temperature) {
  c10::cuda::CUDAGuard guard(logits.device());
  logits = rows_of(logits);
  const auto a = distill_args(logits, ids, teacher, temperature);
  auto loss = at::empty({logits.size(0)}, logits.options().dtype(at::kFloat));
  auto stats = at::empty({logits.size(0), 2}, loss.options());
  ran(bgn_distill_fwd(&a, loss.data_ptr<float>(), stats.data_ptr<float>(), current()), "distill_fwd");
  return {loss, stats};
}

at::Tensor distill_bwd(at::Tensor logits, at::Tensor ids, at::Tensor teacher, at::Tensor stats, at::Tensor dloss,
                       double temperature) {
  c10::cuda::CUDAGuard guard(logits.device());
  logits = rows_of(logits);
  const auto a = distill_args(logits, ids, teacher, temperature);
  TORCH_CHECK(stats.scalar_type() == at::kFloat && stats.is_contiguous() && stats.numel() == 2 * logits.size(0) &&
                  dloss.scalar_type() == at::kFloat && dloss.is_contiguous() && dloss.numel() == logits.size(0) &&
                  stats.device() == logits.device() && dloss.device() == logits.device(),
              "bergson_b200: distill_bwd: stats [T, 2] and dloss [T] in fp32 expected");
  // The gradient's rows are aligned like the logits', so that both take the same packets.
  const int64_t packet = 16 / logits.element_size();
  const int64_t pitch = logits.size(1) + (logits.stride(0) - logits.size(1)) % packet;
  const int64_t shift = reinterpret_cast<uintptr_t>(logits.data_ptr()) % 16 / logits.element_size();
  auto dlogits = at::empty({logits.size(0) * pitch + shift}, logits.options())
                     .as_strided({logits.size(0), logits.size(1)}, {pitch, 1}, shift);
  ran(bgn_distill_bwd(&a, stats.data_ptr<float>(), dloss.data_ptr<float>(), dlogits.data_ptr(), pitch, current()),
      "distill_bwd");
  return dlogits;
}

// ---- autograd -------------------------------------------------------------------------
//
// The graph nodes are here and not in Python: for small batches their calls cost more than the kernels.

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The kernels have no forward-mode derivatives; a tangent that came along would be lost without a word.
void refuse_tangents(std::initializer_list<const at::Tensor*> inputs, const char* what) {
  for (const auto* t : inputs)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(0).defined(), "bergson_b200: ", what,
                                " on the kernels has no forward-mode derivative");
}

bool tracked(std::initializer_list<const at::Tensor*> inputs, const char* what) {
  if (!at::GradMode::is_enabled()) return false;
  bool any = false;
  for (const auto* t : inputs) any = any || t->requires_grad();
  if (!any || at::cuda::currentStreamCaptureStatus() == at::cuda::CaptureStatus::None) return any;
  // While an eager graph of a leaf lives, so does the leaf's accumulation node, bound to that graph's stream;
  // a captured backward pass would wait for the stream, which ends the process.
  const auto here = at::cuda::getCurrentCUDAStream().unwrap();
  for (const auto* t : inputs) {
    if (!t->requires_grad() || !t->is_leaf()) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
    const auto stream = node ? node->stream() : c10::nullopt;
    TORCH_CHECK(!stream || *stream == here, "bergson_b200: ", what,
                ": capturing a graph over a leaf whose eager graph on another stream is still alive; drop that graph first");
  }
  return true;
}

// Gradients that refuse to be differentiated: the backward kernels have none of their own.
variable_list once(variable_list grads, const char* what) {
  if (!at::GradMode::is_enabled()) return grads;
  auto refuse = std::make_shared<torch::autograd::DelayedError>(
      std::string("bergson_b200: the gradient of ") + what + " on the kernels cannot be differentiated again; use ops.composable()",
      int64_t(grads.size()));
  return (*refuse)(std::move(grads));
}

struct PackedAttentionFn : torch::autograd::Function<PackedAttentionFn> {
  static at::Tensor forward(AutogradContext* ctx, at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor first_key,
                            at::Tensor end_query, at::Tensor query_tiles, at::Tensor query_pairs, at::Tensor key_tiles,
                            int64_t valid, double scale) {
    auto out = packed_attention_fwd(q, k, v, first_key, end_query, query_tiles, query_pairs, key_tiles, valid, scale, true);
    if (out.size() < 3) out.emplace_back();
    ctx->save_for_backward({q, k, v, out[0], out[1], out[2], first_key, end_query, query_tiles, query_pairs, key_tiles});
    ctx->saved_data["valid"] = valid;
    ctx->saved_data["scale"] = scale;
    return out[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    variable_list out(3);
    {
      at::AutoGradMode off(false);
      c10::optional<at::Tensor> rest;
      if (s[5].defined()) rest = s[5];
      out = packed_attention_bwd(grads[0], s[0], s[1], s[2], s[3], s[4], rest, s[6], s[7], s[8], s[9], s[10],
                                 ctx->saved_data["valid"].toInt(), ctx->saved_data["scale"].toDouble());
    }
    out = once(std::move(out), "packed_causal_attention");
    out.resize(10);
    return out;
  }
};

at::Tensor packed_attention(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor first_key, at::Tensor end_query,
                            at::Tensor query_tiles, at::Tensor query_pairs, at::Tensor key_tiles, int64_t valid,
                            double scale) {
  refuse_tangents({&q, &k, &v}, "packed_causal_attention");
  if (tracked({&q, &k, &v}, "packed_causal_attention"))
    return PackedAttentionFn::apply(q, k, v, first_key, end_query, query_tiles, query_pairs, key_tiles, valid, scale);
  return packed_attention_fwd(q, k, v, first_key, end_query, query_tiles, query_pairs, key_tiles, valid, scale, false)[0];
}

struct PackedRotaryFn : torch::autograd::Function<PackedRotaryFn> {
  static variable_list forward(AutogradContext* ctx, at::Tensor q, at::Tensor k, at::Tensor cos, at::Tensor sin,
                               at::Tensor position, int64_t rot) {
    ctx->save_for_backward({cos, sin, position});
    ctx->saved_data["rot"] = rot;
    return packed_rotary_turn(q, k, cos, sin, position, rot, false);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    variable_list out(2);
    {
      at::AutoGradMode off(false);
      out = packed_rotary_turn(grads[0], grads[1], s[0], s[1], s[2], ctx->saved_data["rot"].toInt(), true);
    }
    out = once(std::move(out), "packed_rotary");
    out.resize(6);
    return out;
  }
};

std::tuple<at::Tensor, at::Tensor> packed_rotary(at::Tensor q, at::Tensor k, at::Tensor cos, at::Tensor sin,
                                                 at::Tensor position, int64_t rot) {
  refuse_tangents({&q, &k, &cos, &sin}, "packed_rotary");
  auto out = tracked({&q, &k}, "packed_rotary") ? PackedRotaryFn::apply(q, k, cos, sin, position, rot)
                               : packed_rotary_turn(q, k, cos, sin, position, rot, false);
  return {out[0], out[1]};
}

struct DistillFn : torch::autograd::Function<DistillFn> {
  static at::Tensor forward(AutogradContext* ctx, at::Tensor logits, at::Tensor ids, at::Tensor teacher, double temperature) {
    auto out = distill_fwd(logits, ids, teacher, temperature);
    ctx->save_for_backward({logits, ids, teacher, out[1]});
    ctx->saved_data["temperature"] = temperature;
    return out[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    variable_list out(1);
    {
      at::AutoGradMode off(false);
      out[0] = distill_bwd(s[0], s[1], s[2], s[3], grads[0].contiguous(), ctx->saved_data["temperature"].toDouble());
    }
    out = once(std::move(out), "token_distillation");
    out.resize(4);
    return out;
  }
};

at::Tensor distill(at::Tensor logits, at::Tensor ids, at::Tensor teacher, double temperature) {
  refuse_tangents({&logits, &teacher}, "token_distillation");
  ids = ids.contiguous();
  teacher = teacher.contiguous();
  if (tracked({&logits}, "token_distillation")) return DistillFn::apply(logits, ids, teacher, temperature);
  return distill_fwd(logits, ids, teacher, temperature)[0];
}

}  // namespace

void bgn_register_packed(pybind11::module& m) {
  m.def("packed_attention", &packed_attention);
  m.def("packed_rotary", &packed_rotary);
  m.def("distill", &distill);
  m.def("packed_gave_up", &packed_gave_up);
}
