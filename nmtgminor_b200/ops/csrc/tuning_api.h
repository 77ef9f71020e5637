// C launch API of preference tuning: log-probabilities of target words, paired and clipped policy losses (preference.cu), the embedding
// gradient by sorted tokens (embed_sorted.cu) and activations kept in 8 bits (kept8.cu).
// Every launcher returns nullptr on success or a static error string; nothing allocates.
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

extern "C" {

// ---- rows of logits (preference.cu) ----------------------------------------------------------------------------------
// dtype of logits and gradient: 0 = fp32, 1 = bf16, 2 = fp16.  Rows are `ld` elements apart, elements of a row adjacent; the gradient has
// the same `ld` and the same address modulo 16 bytes (it may be the logits themselves).  Rows whose label is `pad` or no word count as padding:
// log-probability, loss and gradient 0.
struct NmtgRows {
  const void* logits;
  void* grad;               // null: no gradient
  const int64_t* labels;    // [rows]
  int rows, vocab, dtype;
  long ld;
  float inv_temperature;
  long pad;
  float grad_scale;         // factor of the gradient of the two losses, times *grad_scale_at where that is not null
  const float* grad_scale_at;
  float* logprobs;          // [rows] out
  float2* stat;             // [rows] (largest logit, sum of exp((x - largest) / T)): out of the scores and, where not null, of the policy loss; in of their
                            // gradient
  void* workspace;          // nmtg_rows_workspace bytes (pairs: of the paired loss, otherwise 0), 16-byte aligned
};
long nmtg_rows_workspace(int rows, int vocab, int dtype, int pairs);
// log-probability of every label, and `stat` where it is not null
const char* nmtg_row_scores(const NmtgRows* r, cudaStream_t stream);
// grad = weight[row] * d logprob / d logits, from `stat`; times *grad_scale_at where that is not null
const char* nmtg_row_scores_grad(const NmtgRows* r, const float* weight, cudaStream_t stream);

struct NmtgPolicy {
  const float* old_logprobs;   // [rows]
  const float* advantages;     // [rows]
  const float* ref_logprobs;   // [rows] or null
  float clip_low, clip_high, kl_coef;
  float *loss, *kl, *clipped;  // [1] each, out: sums of losses and KL terms, number of clipped words
  float* coef;                 // [rows], there where r->stat is: d loss / d logprob, the weights of a gradient that is made later
};
const char* nmtg_policy_loss(const NmtgRows* r, const NmtgPolicy* p, cudaStream_t stream);

// Sequences 2i (preferred) and 2i + 1 (rejected) of `cu` are pair i.
struct NmtgPairs {
  const int* cu;               // [2 pairs + 1]
  const float* ref;            // [2 pairs] or null
  int pairs;
  int kind;                    // 0 sigmoid, 1 hinge, 2 squared distance to 1 / (2 beta)
  int average;
  float beta, smoothing, margin, nll_weight;
  float* seq_logprobs;         // [2 pairs] out
  float *loss, *ranked;        // [1] each, out: sum of losses, number of pairs ranked as preferred
};
const char* nmtg_preference_loss(const NmtgRows* r, const NmtgPairs* p, cudaStream_t stream);
// the gradient by itself, from the workspace that nmtg_preference_loss has left for the same logits and `pairs` pairs
const char* nmtg_preference_grad(const NmtgRows* r, int pairs, cudaStream_t stream);
// r->grad *= *factor, unless it is 1
const char* nmtg_scale_rows(const NmtgRows* r, const float* factor, cudaStream_t stream);

// ---- activations kept in 8 bits (kept8.cu) -----------------------------------------------------------------------------
// dtype as above.  codes: [rows, 32 * blocks] bytes, 8-byte aligned; scales: [rows, blocks]; blocks = ceil(width / 32).  Tensors other than `in` are
// dense [rows, width].
struct NmtgKept {
  const void* in;           // x (quantise), z (forward) or dy (backward), rows ld_in elements apart
  void* out;                // restore: x' or null; forward: dropout(act(z)); backward: dropout-mask(dy) act'(z')
  void* out2;               // restore: dropout(act(x')) or null
  uint8_t* codes;           // forward: null where nothing is to be kept
  uint8_t* scales;
  long rows, width, ld_in;
  int dtype, act;           // act: 0 none, 1 ReLU, 2 GELU (erf), 3 SiLU
  float p;                  // dropout of the activation: the mask of dropout_add for the same seed and stream
  unsigned long long seed, stream_id;
  const unsigned long long* seed_dev;
  cudaStream_t stream;
};
const char* nmtg_kept_quantise(const NmtgKept* k);
const char* nmtg_kept_restore(const NmtgKept* k);
const char* nmtg_kept_forward(const NmtgKept* k);
const char* nmtg_kept_backward(const NmtgKept* k);

// ---- embedding gradient by sorted tokens (embed_sorted.cu) ----------------------------------------------------------------
// grad[k] (+)= scale * sum over the rows r with key k, in the order of r, of dropout-mask(dy)[r].  Key of a row: its token, or with `positions` its
// position brought into [0, keys); none where the token is `pad` or outside [0, vocab).
struct NmtgEmbedGrad {
  const int64_t* tokens;    // [rows]
  const int64_t* positions; // [rows] or null
  const void* dy;           // dense [rows, width]
  void* grad;               // dense [keys, width]: fp32 added to (accumulate), or of dy's type and written whole
  int rows, vocab, keys, width;
  int dtype, accumulate;
  long pad;
  float scale, p;
  unsigned long long seed, stream_id;
  const unsigned long long* seed_dev;
  void* workspace;          // nmtg_embed_grad_workspace bytes, 16-byte aligned
  cudaStream_t stream;
};
long nmtg_embed_grad_workspace(int rows, int keys, int width);
const char* nmtg_embed_grad(const NmtgEmbedGrad* e);
// out[r] = table[tokens[r]] * scale, dense [rows, width] of the table's type; tokens outside the table read its first row
const char* nmtg_embed_rows(const int64_t* tokens, const void* table, void* out, int rows, int vocab, int width, int dtype, float scale,
                            cudaStream_t stream);
}
