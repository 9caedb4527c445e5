// C++ launchers of the per-token vocabulary kernels (see token_loss.cu): log-probabilities of given
// tokens with entropy and top alternatives, and the loss against a teacher's top logits.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace ethb {

constexpr int kMaxTopAlternatives = 128;   // top_k of token_logprobs
constexpr int kMaxTeacherEntries = 512;    // entries per row of a teacher's list

// Logits are [rows, vocab] with unit inner stride and any row pitch `ld`; `v0` is the first global
// token id of this vocabulary shard. `world` > 1 in the *_combine calls merges the shards' statistics.
struct LogitsView {
  const void* z;
  int64_t rows, ld;
  int vocab;
  int64_t v0;
  int dtype;            // kF32 / kF16 / kBF16
  float inv_temperature;
};

// stats: [rows, 2] (subtracted maximum, sum of exponentials, negative where the token lies outside the vocabulary)
// kept for the backward pass.
struct TokenScoresOut {
  float *logprob, *entropy, *top_logprob;   // [rows], [rows], [rows, top_k]
  int64_t* top_index;                       // [rows, top_k] global token ids
  float* stats;
};
cudaError_t token_scores(const LogitsView& a, const int64_t* tokens, int top_k, const TokenScoresOut& out,
                         cudaStream_t st);
// one shard's part: [rows, 4 + 2 top_k] = max, sum, sum of e*t, token logit (NaN: not here), the
// top_k logits, the top_k global ids (int32 bits)
cudaError_t token_scores_partial(const LogitsView& a, const int64_t* tokens, int top_k, float* partial,
                                 cudaStream_t st);
cudaError_t token_scores_combine(const float* partials, int world, int64_t rows, const int64_t* tokens, int top_k,
                                 float inv_temperature, const TokenScoresOut& out, cudaStream_t st);
// g / h / u: gradients of logprob [rows], entropy [rows], top_logprob [rows, top_k]; any may be null
cudaError_t token_scores_bwd(const LogitsView& a, const int64_t* tokens, const float* stats, const float* entropy,
                             const int64_t* top_index, int top_k, const float* g, const float* h, const float* u,
                             void* dz, int64_t ldd, cudaStream_t st);

// A teacher's list: [rows, k] global ids and logits (log-probabilities do), -inf marks an unused entry.
struct TeacherView {
  const int64_t* index;
  const float* logit;
  int k;
};
cudaError_t distill_fwd(const LogitsView& a, const TeacherView& t, float* loss, float* stats, cudaStream_t st);
// one shard's part: [rows, kDistillParts] = max, sum, weighted sum of the listed logits found here, their
// weight, their number
constexpr int kDistillParts = 5;
cudaError_t distill_partial(const LogitsView& a, const TeacherView& t, float* partial, cudaStream_t st);
cudaError_t distill_combine(const float* partials, int world, int64_t rows, const TeacherView& t,
                            float inv_temperature, float* loss, float* stats, cudaStream_t st);
cudaError_t distill_bwd(const LogitsView& a, const TeacherView& t, const float* stats, const float* dloss, void* dz,
                        int64_t ldd, cudaStream_t st);
// loss and gradient in one launch; dz may be the logits themselves
cudaError_t distill_step(const LogitsView& a, const TeacherView& t, const float* dloss, float* loss, void* dz,
                         int64_t ldd, cudaStream_t st);

}  // namespace ethb
