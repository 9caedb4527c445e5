// Packed-document ops on CUDA tensors: checks of arguments, allocation of results, launches, and their
// autograd nodes in C++. A Python autograd function would hand the interpreter lock to the engine's
// thread and back in every backward; for these ops, which take a few microseconds on short inputs,
// that costs several times the kernels (attention over 4001 tokens, forward and backward: 160 us of
// host time with Python nodes).
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>

#include <cmath>
#include <tuple>

#include "attention_packed_sm100.cuh"
#include "gemm_sm100.cuh"
#include "token_loss.cuh"

namespace ethb {
namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }
void check(cudaError_t e, const char* what) {
  TORCH_CHECK(e == cudaSuccess, what, ": ", cudaGetErrorString(e), " [", last_error_detail(), "]");
}
int dtype_code(const Tensor& t) {   // the library's type tags
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kHalf: return 1;
    case at::kBFloat16: return 2;
    default: TORCH_CHECK_VALUE(false, "unsupported type ", t.scalar_type());
  }
}
// The gradients come from kernels that autograd cannot look into.
void refuse_double_backward() {
  TORCH_CHECK(!at::GradMode::is_enabled(), "packed ops: a backward pass cannot itself be differentiated");
}

// ---------------------------------------------------------------------------------------------
// attention over packed documents
// ---------------------------------------------------------------------------------------------
// Work lists of an ops.PackedLayout for one mask: 128-row tiles and 256-row blocks for the forward and
// the query side, key tiles for dK / dV.
struct Lists {
  Tensor tiles, blocks, keys;
  int64_t used, total;
};

bool addressable(const Tensor& t) {   // by a tensor map: 16-byte aligned, strides of 16 bytes
  if ((reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) != 0 || t.stride(2) != 1) return false;
  for (int d = 0; d < 2; ++d)
    if (t.size(d) > 1 && (t.stride(d) <= 0 || t.stride(d) % 8 != 0)) return false;
  return true;
}
Tensor tma_view(const Tensor& t) { return addressable(t) ? t : t.clone(at::MemoryFormat::Contiguous); }

// A dimension of size 1 has no stride of its own and gets one that a tensor map takes.
void rhd_strides(const Tensor& t, int64_t out[2]) {
  out[1] = t.size(1) == 1 ? t.size(2) : t.stride(1);
  out[0] = t.size(0) <= 1 ? t.size(1) * t.size(2) : t.stride(0);
}
// A layout may be let go of while a call on another stream than its own still runs: the allocator is told
// (it returns at once on the layout's own stream), as a kernel that met other data in its list would
// address memory by it.
const PackedTile* tile_list(const Tensor& t, const Tensor& like, int& n) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.get_device() == like.get_device(), "packed attention: layout on ", t.device(),
                    ", tensors on ", like.device());
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.dim() == 2 && t.size(1) == 4 && t.is_contiguous(),
                    "packed attention: work lists are int32 [n, 4]");
  n = static_cast<int>(t.size(0));
  c10::cuda::CUDACachingAllocator::recordStream(t.storage().data_ptr(), at::cuda::getCurrentCUDAStream());
  return reinterpret_cast<const PackedTile*>(t.data_ptr());
}

void check_packed(const Tensor& q, const Tensor& k, const Tensor& v, const Lists& l, double scale) {
  TORCH_CHECK_VALUE(q.dim() == 3 && k.dim() == 3 && k.sizes() == v.sizes() && q.size(0) == k.size(0) &&
                        q.size(2) == k.size(2),
                    "packed attention: q [total, heads, dim], k and v [total, kv_heads, dim]; got ", q.sizes(), ", ",
                    k.sizes(), ", ", v.sizes());
  TORCH_CHECK_VALUE(q.size(1) >= 1 && k.size(1) >= 1 && q.size(1) % k.size(1) == 0, "packed attention: ", q.size(1),
                    " heads cannot share ", k.size(1), " key/value heads evenly");
  TORCH_CHECK_VALUE(q.is_cuda() && q.device() == k.device() && q.device() == v.device() &&
                        q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(),
                    "packed attention: q, k and v must agree in type and device");
  TORCH_CHECK_VALUE((q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16) &&
                        (q.size(2) == 64 || q.size(2) == 128),
                    "packed attention: fp16 / bf16 with head_dim 64 or 128 only, got ", q.scalar_type(), ", ", q.size(2));
  TORCH_CHECK_VALUE(l.total == q.size(0), "packed attention: layout of ", l.total, " rows, tensors of ", q.size(0));
  TORCH_CHECK_VALUE(l.used >= 0 && l.used <= l.total && l.total < 0x7fffff00, "packed attention: rows of the layout");
  TORCH_CHECK_VALUE(scale >= 1e-30 && scale <= 1e3, "packed attention: scale must be between 1e-30 and 1e3, got ", scale);
}

double scale_of(const Tensor& q, c10::optional<double> scale) {
  return scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(q.dim() == 3 ? q.size(2) : 1));
}

PackedAttnArgs packed_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o, const Tensor& lse,
                           const Lists& l, double scale, bool causal, const Tensor& status) {
  PackedAttnArgs a{};
  a.rows = static_cast<int>(q.size(0)); a.used = static_cast<int>(l.used);
  a.heads = static_cast<int>(q.size(1)); a.kv_heads = static_cast<int>(k.size(1));
  a.head_dim = static_cast<int>(q.size(2));
  a.q = q.data_ptr(); a.k = k.data_ptr(); a.v = v.data_ptr(); a.o = o.data_ptr();
  rhd_strides(q, a.q_strides); rhd_strides(k, a.k_strides); rhd_strides(v, a.v_strides); rhd_strides(o, a.o_strides);
  a.lse = lse.data_ptr<float>();
  a.scale = static_cast<float>(scale);
  a.causal = causal;
  a.dtype = dtype_code(q);
  a.status = status.data_ptr<int>();
  return a;
}

// out, lse and, if asked for, what the rounding of out to 16 bits took off (the backward's rowsum(dO * O)
// takes the sum of both).
std::tuple<Tensor, Tensor, Tensor> packed_fwd(const Tensor& q0, const Tensor& k0, const Tensor& v0, const Lists& l,
                                              double scale, bool causal, const Tensor& status, bool with_residue) {
  check_packed(q0, k0, v0, l, scale);
  c10::cuda::CUDAGuard guard(q0.device());
  const Tensor q = tma_view(q0), k = tma_view(k0), v = tma_view(v0);
  Tensor out = at::empty(q.sizes(), q.options());
  Tensor lse = at::empty({q.size(1), q.size(0)}, q.options().dtype(at::kFloat));
  Tensor residue;
  auto a = packed_args(q, k, v, out, lse, l, scale, causal, status);
  if (with_residue) {
    residue = at::empty(q.sizes(), q.options());
    a.residue = residue.data_ptr();
  }
  a.tiles = tile_list(attention_packed_pairs_heads(a.heads, a.kv_heads) ? l.tiles : l.blocks, q, a.num_tiles);
  check(attention_packed_fwd(a, cur_stream()), "attention_packed_fwd");
  return {out, lse, residue};
}

std::tuple<Tensor, Tensor, Tensor> packed_bwd(const Tensor& d_out, const Tensor& q0, const Tensor& k0,
                                              const Tensor& v0, const Tensor& out, const Tensor& lse, const Lists& l,
                                              double scale, bool causal, const Tensor& status,
                                              const Tensor& residue) {
  check_packed(q0, k0, v0, l, scale);
  TORCH_CHECK_VALUE(!residue.defined() || (residue.device() == q0.device() && residue.scalar_type() == q0.scalar_type() &&
                                           residue.sizes() == q0.sizes() && residue.is_contiguous()),
                    "packed attention: the residue is a contiguous tensor like out");
  for (const Tensor& t : {d_out, out})
    TORCH_CHECK_VALUE(t.device() == q0.device() && t.scalar_type() == q0.scalar_type() && t.sizes() == q0.sizes(),
                      "packed attention: out and its gradient must match q");
  TORCH_CHECK_VALUE(lse.device() == q0.device() && lse.scalar_type() == at::kFloat && lse.is_contiguous() &&
                        lse.numel() == q0.size(0) * q0.size(1), "packed attention: lse must be fp32 [heads, total]");
  c10::cuda::CUDAGuard guard(q0.device());
  const Tensor q = tma_view(q0), k = tma_view(k0), v = tma_view(v0), d_o = tma_view(d_out), o = tma_view(out);
  Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), q.options());
  Tensor dv = at::empty(k.sizes(), q.options()), delta = at::empty_like(lse);
  auto a = packed_args(q, k, v, o, lse, l, scale, causal, status);
  a.d_o = d_o.data_ptr(); a.dq = dq.data_ptr(); a.dk = dk.data_ptr(); a.dv = dv.data_ptr();
  rhd_strides(d_o, a.do_strides); rhd_strides(dq, a.dq_strides);
  rhd_strides(dk, a.dk_strides); rhd_strides(dv, a.dv_strides);
  a.delta = delta.data_ptr<float>();
  a.residue = residue.defined() ? residue.data_ptr() : nullptr;
  a.q_tiles = tile_list(l.tiles, q, a.num_q_tiles);
  a.k_tiles = tile_list(l.keys, q, a.num_k_tiles);
  const Tensor counters = at::empty({2}, q.options().dtype(at::kInt));
  a.counters = counters.data_ptr<int>();
  a.splits = attention_packed_splits(a.num_k_tiles, a.heads, a.kv_heads);
  Tensor parts;
  if (a.splits > 1) {
    parts = at::empty({a.splits, 2, l.used, k.size(1), q.size(2)}, q.options().dtype(at::kFloat));
    a.parts = parts.data_ptr<float>();
  }
  check(attention_packed_bwd(a, cur_stream()), "attention_packed_bwd");
  return {dq, dk, dv};
}

struct PackedAttention : torch::autograd::Function<PackedAttention> {
  static Variable forward(AutogradContext* ctx, const Variable& q, const Variable& k, const Variable& v,
                          const Tensor& tiles, const Tensor& blocks, const Tensor& keys, int64_t used, int64_t total,
                          double scale, bool causal, const Tensor& status, bool needs_grad) {
    auto [out, lse, residue] =
        packed_fwd(q, k, v, Lists{tiles, blocks, keys, used, total}, scale, causal, status, needs_grad);
    ctx->save_for_backward({q, k, v, out, lse, residue});
    // the kernels' own data, no values of the graph: neither hooks on saved tensors nor their version checks
    // apply (the status word is cleared in place between steps)
    ctx->saved_data["tiles"] = tiles;
    ctx->saved_data["blocks"] = blocks;
    ctx->saved_data["keys"] = keys;
    ctx->saved_data["status"] = status;
    ctx->saved_data["used"] = used;
    ctx->saved_data["total"] = total;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["causal"] = causal;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_double_backward();
    const auto s = ctx->get_saved_variables();
    const Lists l{ctx->saved_data["tiles"].toTensor(), ctx->saved_data["blocks"].toTensor(),
                  ctx->saved_data["keys"].toTensor(), ctx->saved_data["used"].toInt(), ctx->saved_data["total"].toInt()};
    auto [dq, dk, dv] = packed_bwd(grads[0], s[0], s[1], s[2], s[3], s[4], l, ctx->saved_data["scale"].toDouble(),
                                   ctx->saved_data["causal"].toBool(), ctx->saved_data["status"].toTensor(), s[5]);
    return {dq, dk, dv, Variable(), Variable(), Variable(), Variable(), Variable(), Variable(), Variable(), Variable(), Variable()};
  }
};

// ---------------------------------------------------------------------------------------------
// per-token vocabulary ops
// ---------------------------------------------------------------------------------------------
LogitsView logits_view(const Tensor& z, int64_t vocab_start, double temperature) {
  LogitsView a{};
  a.z = z.data_ptr(); a.rows = z.size(0); a.ld = z.stride(0); a.vocab = static_cast<int>(z.size(1));
  a.v0 = vocab_start;
  a.dtype = dtype_code(z);
  a.inv_temperature = static_cast<float>(1.0 / temperature);
  return a;
}
// Checks the logits; returns them with unit inner stride and rows that do not overlap, any pitch.
Tensor unit_rows(const Tensor& z, double temperature) {
  TORCH_CHECK_VALUE(z.is_cuda() && z.dim() == 2 && z.size(1) >= 1, "logits must be [tokens, vocab], got ", z.sizes());
  TORCH_CHECK_VALUE(z.scalar_type() == at::kFloat || z.scalar_type() == at::kHalf || z.scalar_type() == at::kBFloat16,
                    "logits of type ", z.scalar_type(), " are not supported");
  TORCH_CHECK_VALUE(z.size(0) < 0x7fffffff && z.size(1) < (int64_t{1} << 30), "logits are too large: ", z.sizes());
  TORCH_CHECK_VALUE(temperature >= 1e-30 && temperature <= 1e30, "temperature must be between 1e-30 and 1e30, got ",
                    temperature);
  const bool bad = (z.size(1) > 1 && z.stride(1) != 1) || (z.size(0) > 1 && z.stride(0) < z.size(1));
  return bad ? z.contiguous() : z;
}
Tensor rows_of(const Tensor& t, const Tensor& z, at::ScalarType type, c10::IntArrayRef shape, const char* name) {
  TORCH_CHECK_VALUE(t.device() == z.device() && t.scalar_type() == type && t.sizes() == shape, name, " must be ", type,
                    " ", shape, " on ", z.device(), ", got ", t.scalar_type(), " ", t.sizes(), " on ", t.device());
  return t.contiguous();
}
// An uninitialised gradient whose rows sit at the same offsets from a 16-byte boundary as the rows of
// the logits: a slice of a padded vocabulary keeps vector accesses on both sides.
Tensor grad_rows(const Tensor& z) {
  const int64_t rows = z.size(0), vocab = z.size(1), per = 16 / z.element_size();
  const int64_t lead = static_cast<int64_t>(reinterpret_cast<uintptr_t>(z.data_ptr()) % 16) / z.element_size();
  const int64_t pitch = rows > 1 ? vocab + ((z.stride(0) - vocab) % per + per) % per : vocab;
  if (lead == 0 && pitch == vocab) return at::empty({rows, vocab}, z.options());
  return at::empty({lead + rows * pitch}, z.options()).as_strided({rows, vocab}, {pitch, 1}, lead);
}
float* fptr(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

using Scores = std::tuple<Tensor, Tensor, OptTensor, OptTensor, Tensor>;
struct ScoresBuffers {
  Tensor logprob, entropy, stats, top_logprob, top_index;
  ScoresBuffers(const Tensor& like, int64_t rows, int64_t k) {
    const auto f = like.options().dtype(at::kFloat);
    logprob = at::empty({rows}, f);
    entropy = at::empty({rows}, f);
    stats = at::empty({rows, 2}, f);
    if (k > 0) {
      top_logprob = at::empty({rows, k}, f);
      top_index = at::empty({rows, k}, like.options().dtype(at::kLong));
    }
  }
  TokenScoresOut out() const {
    return {fptr(logprob), fptr(entropy), fptr(top_logprob),
            top_index.defined() ? top_index.data_ptr<int64_t>() : nullptr, fptr(stats)};
  }
  Scores tuple() const {
    OptTensor a, b;
    if (top_index.defined()) { a = top_logprob; b = top_index; }
    return {logprob, entropy, a, b, stats};
  }
};
void check_top(int64_t top_k, int64_t vocab) {
  const int64_t most = std::min<int64_t>(kMaxTopAlternatives, vocab);
  TORCH_CHECK_VALUE(top_k >= 0 && top_k <= most, "top_k must be between 0 and ", most, ", got ", top_k);
}

Scores token_scores_fwd(const Tensor& logits, const Tensor& tokens0, int64_t top_k, double temperature,
                        int64_t vocab_start) {
  const Tensor z = unit_rows(logits, temperature);
  check_top(top_k, z.size(1));
  const Tensor tokens = rows_of(tokens0, z, at::kLong, {z.size(0)}, "tokens");
  c10::cuda::CUDAGuard guard(z.device());
  const ScoresBuffers b(z, z.size(0), top_k);
  check(token_scores(logits_view(z, vocab_start, temperature), tokens.data_ptr<int64_t>(), static_cast<int>(top_k),
                     b.out(), cur_stream()), "token_scores");
  return b.tuple();
}
Tensor token_scores_part(const Tensor& logits, const Tensor& tokens0, int64_t top_k, double temperature,
                         int64_t vocab_start) {
  const Tensor z = unit_rows(logits, temperature);
  check_top(top_k, z.size(1));
  const Tensor tokens = rows_of(tokens0, z, at::kLong, {z.size(0)}, "tokens");
  c10::cuda::CUDAGuard guard(z.device());
  Tensor part = at::empty({z.size(0), 4 + 2 * top_k}, z.options().dtype(at::kFloat));
  check(token_scores_partial(logits_view(z, vocab_start, temperature), tokens.data_ptr<int64_t>(),
                             static_cast<int>(top_k), fptr(part), cur_stream()), "token_scores_partial");
  return part;
}
int64_t check_parts(const Tensor& parts, int64_t rows, int64_t width) {
  TORCH_CHECK_VALUE(parts.is_cuda() && parts.scalar_type() == at::kFloat && parts.dim() == 3 && parts.size(0) >= 1 &&
                        parts.size(1) == rows && parts.size(2) == width && parts.is_contiguous(),
                    "gather_fn must return the [shards, ", rows, ", ", width, "] stack of its argument");
  return parts.size(0);
}
Scores token_scores_join(const Tensor& parts, const Tensor& tokens0, int64_t top_k, double temperature) {
  const int64_t rows = tokens0.size(0);
  const int64_t world = check_parts(parts, rows, 4 + 2 * top_k);
  const Tensor tokens = rows_of(tokens0, parts, at::kLong, {rows}, "tokens");
  c10::cuda::CUDAGuard guard(parts.device());
  const ScoresBuffers b(parts, rows, top_k);
  check(token_scores_combine(fptr(parts), static_cast<int>(world), rows, tokens.data_ptr<int64_t>(),
                             static_cast<int>(top_k), static_cast<float>(1.0 / temperature), b.out(), cur_stream()),
        "token_scores_combine");
  return b.tuple();
}
Tensor token_scores_grad(const Tensor& logits, const Tensor& tokens0, const Tensor& stats, const Tensor& entropy,
                         const OptTensor& top_index, const OptTensor& g, const OptTensor& h, const OptTensor& u,
                         double temperature, int64_t vocab_start) {
  const Tensor z = unit_rows(logits, temperature);
  const int64_t rows = z.size(0), k = top_index.has_value() ? top_index->size(1) : 0;
  const Tensor tokens = rows_of(tokens0, z, at::kLong, {rows}, "tokens");
  const Tensor st = rows_of(stats, z, at::kFloat, {rows, 2}, "stats");
  const Tensor en = rows_of(entropy, z, at::kFloat, {rows}, "entropy");
  Tensor index, gt, ht, ut;
  if (k > 0) index = rows_of(*top_index, z, at::kLong, {rows, k}, "top_index");
  if (g.has_value()) gt = rows_of(*g, z, at::kFloat, {rows}, "d_logprob");
  if (h.has_value()) ht = rows_of(*h, z, at::kFloat, {rows}, "d_entropy");
  if (u.has_value() && k > 0) ut = rows_of(*u, z, at::kFloat, {rows, k}, "d_top_logprob");
  c10::cuda::CUDAGuard guard(z.device());
  Tensor dz = grad_rows(z);
  check(token_scores_bwd(logits_view(z, vocab_start, temperature), tokens.data_ptr<int64_t>(), fptr(st), fptr(en),
                         index.defined() ? index.data_ptr<int64_t>() : nullptr, static_cast<int>(k), fptr(gt), fptr(ht),
                         fptr(ut), dz.data_ptr(), dz.stride(0), cur_stream()), "token_scores_bwd");
  return dz;
}

struct TokenScoresNode : torch::autograd::Function<TokenScoresNode> {
  static variable_list forward(AutogradContext* ctx, const Variable& logits, const Tensor& tokens, int64_t top_k,
                               double temperature, int64_t vocab_start) {
    auto [logprob, entropy, top_logprob, top_index, stats] =
        token_scores_fwd(logits, tokens, top_k, temperature, vocab_start);
    const Tensor index = top_index.value_or(Tensor());
    ctx->save_for_backward({logits, tokens, stats, entropy, index});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["vocab_start"] = vocab_start;
    ctx->set_materialize_grads(false);
    if (top_k == 0) return {logprob, entropy};
    ctx->mark_non_differentiable({index});
    return {logprob, entropy, *top_logprob, index};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_double_backward();
    const auto s = ctx->get_saved_variables();
    auto opt = [&](size_t i) { return i < grads.size() && grads[i].defined() ? OptTensor(grads[i]) : OptTensor(); };
    Tensor dz = token_scores_grad(s[0], s[1], s[2], s[3], s[4].defined() ? OptTensor(s[4]) : OptTensor(), opt(0), opt(1),
                                  opt(2), ctx->saved_data["temperature"].toDouble(),
                                  ctx->saved_data["vocab_start"].toInt());
    return {dz, Variable(), Variable(), Variable(), Variable()};
  }
};

struct Teacher {
  Tensor index, logit;
  Teacher(const Tensor& i, const Tensor& l, const Tensor& like, int64_t rows) {
    TORCH_CHECK_VALUE(i.dim() == 2 && i.size(1) >= 1 && i.size(1) <= kMaxTeacherEntries,
                      "teacher lists must be [tokens, 1..", kMaxTeacherEntries, "], got ", i.sizes());
    index = rows_of(i, like, at::kLong, {rows, i.size(1)}, "teacher_index");
    logit = rows_of(l, like, at::kFloat, {rows, i.size(1)}, "teacher_logit");
  }
  TeacherView view() const { return {index.data_ptr<int64_t>(), logit.data_ptr<float>(), static_cast<int>(index.size(1))}; }
};

std::tuple<Tensor, Tensor> distill_forward(const Tensor& logits, const Tensor& index, const Tensor& logit,
                                           double temperature, int64_t vocab_start) {
  const Tensor z = unit_rows(logits, temperature);
  const Teacher t(index, logit, z, z.size(0));
  c10::cuda::CUDAGuard guard(z.device());
  const auto f = z.options().dtype(at::kFloat);
  Tensor loss = at::empty({z.size(0)}, f), stats = at::empty({z.size(0), 2}, f);
  check(distill_fwd(logits_view(z, vocab_start, temperature), t.view(), fptr(loss), fptr(stats), cur_stream()),
        "distill_fwd");
  return {loss, stats};
}
Tensor distill_part(const Tensor& logits, const Tensor& index, const Tensor& logit, double temperature,
                    int64_t vocab_start) {
  const Tensor z = unit_rows(logits, temperature);
  const Teacher t(index, logit, z, z.size(0));
  c10::cuda::CUDAGuard guard(z.device());
  Tensor part = at::empty({z.size(0), kDistillParts}, z.options().dtype(at::kFloat));
  check(distill_partial(logits_view(z, vocab_start, temperature), t.view(), fptr(part), cur_stream()),
        "distill_partial");
  return part;
}
std::tuple<Tensor, Tensor> distill_join(const Tensor& parts, const Tensor& index, const Tensor& logit,
                                        double temperature) {
  const int64_t rows = index.size(0), world = check_parts(parts, rows, kDistillParts);
  const Teacher t(index, logit, parts, rows);
  c10::cuda::CUDAGuard guard(parts.device());
  Tensor loss = at::empty({rows}, parts.options()), stats = at::empty({rows, 2}, parts.options());
  check(distill_combine(fptr(parts), static_cast<int>(world), rows, t.view(), static_cast<float>(1.0 / temperature),
                        fptr(loss), fptr(stats), cur_stream()), "distill_combine");
  return {loss, stats};
}
Tensor distill_grad(const Tensor& logits, const Tensor& index, const Tensor& logit, const Tensor& stats,
                    const Tensor& dloss0, double temperature, int64_t vocab_start) {
  const Tensor z = unit_rows(logits, temperature);
  const Teacher t(index, logit, z, z.size(0));
  const Tensor st = rows_of(stats, z, at::kFloat, {z.size(0), 2}, "stats");
  const Tensor dloss = rows_of(dloss0, z, at::kFloat, {z.size(0)}, "dloss");
  c10::cuda::CUDAGuard guard(z.device());
  Tensor dz = grad_rows(z);
  check(distill_bwd(logits_view(z, vocab_start, temperature), t.view(), fptr(st), fptr(dloss), dz.data_ptr(),
                    dz.stride(0), cur_stream()), "distill_bwd");
  return dz;
}
std::tuple<Tensor, Tensor> distill_both(const Tensor& logits, const Tensor& index, const Tensor& logit,
                                        const Tensor& dloss0, double temperature, const OptTensor& out) {
  const Tensor z = unit_rows(logits, temperature);
  const Teacher t(index, logit, z, z.size(0));
  const Tensor dloss = rows_of(dloss0, z, at::kFloat, {z.size(0)}, "dloss");
  Tensor dz;
  c10::cuda::CUDAGuard guard(z.device());
  if (out.has_value()) {
    dz = *out;
    TORCH_CHECK_VALUE(dz.sizes() == logits.sizes() && dz.scalar_type() == z.scalar_type() && dz.device() == z.device() &&
                          (dz.size(1) <= 1 || dz.stride(1) == 1) && (dz.size(0) <= 1 || dz.stride(0) >= dz.size(1)),
                      "distill_step: out must match the logits and have contiguous rows that do not overlap");
    const bool same = dz.data_ptr() == logits.data_ptr() && dz.strides() == logits.strides();
    TORCH_CHECK_VALUE(same || dz.storage().data() != logits.storage().data(),
                      "distill_step: out may be the logits themselves or other memory, not an overlapping view");
    // a change in place: a node that has saved the logits and runs later raises, it does not read a gradient
    dz.unsafeGetTensorImpl()->bump_version();
  } else {
    dz = grad_rows(z);
  }
  Tensor loss = at::empty({z.size(0)}, z.options().dtype(at::kFloat));
  check(distill_step(logits_view(z, 0, temperature), t.view(), fptr(dloss), fptr(loss), dz.data_ptr(), dz.stride(0),
                     cur_stream()), "distill_step");
  return {loss, dz};
}

struct DistillNode : torch::autograd::Function<DistillNode> {
  static Variable forward(AutogradContext* ctx, const Variable& logits, const Tensor& index, const Tensor& logit,
                          double temperature, int64_t vocab_start) {
    auto [loss, stats] = distill_forward(logits, index, logit, temperature, vocab_start);
    ctx->save_for_backward({logits, index, logit, stats});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["vocab_start"] = vocab_start;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_double_backward();
    const auto s = ctx->get_saved_variables();
    Tensor dz = distill_grad(s[0], s[1], s[2], s[3], grads[0], ctx->saved_data["temperature"].toDouble(),
                             ctx->saved_data["vocab_start"].toInt());
    return {dz, Variable(), Variable(), Variable(), Variable()};
  }
};

}  // namespace

void bind_packed_ops(pybind11::module_& m) {
  namespace py = pybind11;
  using unlocked = py::call_guard<py::gil_scoped_release>;
  m.def("flash_attention_packed",
        [](const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& tiles, const Tensor& blocks,
           const Tensor& keys, int64_t used, int64_t total, c10::optional<double> scale, bool causal, const Tensor& status) {
          const bool needs_grad = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad());
          return PackedAttention::apply(q, k, v, tiles, blocks, keys, used, total, scale_of(q, scale), causal, status,
                                        needs_grad);
        }, unlocked());
  m.def("attention_packed_fwd",
        [](const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& tiles, const Tensor& blocks,
           const Tensor& keys, int64_t used, int64_t total, c10::optional<double> scale, bool causal, const Tensor& status,
           bool with_residue) {
          auto [out, lse, residue] = packed_fwd(q, k, v, Lists{tiles, blocks, keys, used, total}, scale_of(q, scale), causal,
                                                status, with_residue);
          return std::make_tuple(out, lse, residue.defined() ? OptTensor(residue) : OptTensor());
        }, unlocked());
  m.def("attention_packed_bwd",
        [](const Tensor& d_out, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out, const Tensor& lse,
           const Tensor& tiles, const Tensor& blocks, const Tensor& keys, int64_t used, int64_t total,
           c10::optional<double> scale, bool causal, const Tensor& status, const OptTensor& residue) {
          return packed_bwd(d_out, q, k, v, out, lse, Lists{tiles, blocks, keys, used, total}, scale_of(q, scale), causal,
                            status, residue.value_or(Tensor()));
        }, unlocked());
  m.def("token_logprobs",
        [](const Tensor& logits, const Tensor& tokens, int64_t top_k, double temperature, int64_t vocab_start) {
          return TokenScoresNode::apply(logits, tokens, top_k, temperature, vocab_start);
        }, unlocked());
  m.def("token_scores_fwd", &token_scores_fwd, unlocked());
  m.def("token_scores_partial", &token_scores_part, unlocked());
  m.def("token_scores_combine", &token_scores_join, unlocked());
  m.def("token_scores_bwd", &token_scores_grad, unlocked());
  m.def("topk_distillation_loss",
        [](const Tensor& logits, const Tensor& index, const Tensor& logit, double temperature, int64_t vocab_start) {
          return DistillNode::apply(logits, index, logit, temperature, vocab_start);
        }, unlocked());
  m.def("distill_fwd", &distill_forward, unlocked());
  m.def("distill_partial", &distill_part, unlocked());
  m.def("distill_combine", &distill_join, unlocked());
  m.def("distill_bwd", &distill_grad, unlocked());
  m.def("distill_step", &distill_both, unlocked());
}

}  // namespace ethb
