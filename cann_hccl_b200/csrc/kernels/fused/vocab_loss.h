// Launch interface of the loss over the vocabulary (kernels/fused/vocab_loss.cu): the products, row sums and gradients of a chunk of
// tokens against one shard of the vocabulary.
#pragma once
#include "common/base.h"

namespace hcclb {

struct VocabLossCall {
    const void *x, *w;               // bf16 [tokens, hidden], [vocab, hidden]
    int64_t x_stride, w_stride;      // elements between rows
    const void *targets;
    bool wide;                       // 64-bit targets
    const float *weights;            // of the tokens; null: ones
    int64_t tokens, vocab, first, whole, ignore;  // first id of the shard, ids of all shards, target of tokens that do not count
    int32_t hidden;
    int64_t scratch_bytes;           // at the call's scratch; 0: not stated
    const float *losses;             // of the tokens, for the gradients; null: target - lse in their place
};
// Tokens whose exponentials fit the scratch of a call with gradients, or whose sums fit that of one without.
int64_t vocab_loss_chunk(int64_t vocab, bool grad);
// Scratch of a call of exactly `tokens`; a call of fewer may need more.
int64_t vocab_loss_scratch_bytes(int64_t tokens, int64_t vocab, int32_t hidden, bool grad);
// The same where a device has `sms` multiprocessors and runs `pairs` clusters of two CTAs at once.
int64_t vocab_loss_scratch_bytes_on(int sms, int pairs, int64_t tokens, int64_t vocab, int32_t hidden, bool grad);
// lse and target logit (-inf where another shard has it) of every token against this shard; losses (may be null) for a lone shard.
// grad: the exponentials stay in scratch for vocab_loss_grad.
HcclResult vocab_loss_scores(const VocabLossCall &c, bool grad, float *lse, float *target, float *losses, void *scratch, void *stream);
// From the shards' [shards][2][tokens] (lse, target): the joint lse and losses.
HcclResult vocab_loss_combine(const VocabLossCall &c, const float *parts, int shards, float *lse, float *losses, void *stream);
// *total = sum of the weights of the tokens that count.
HcclResult vocab_loss_total(const VocabLossCall &c, float *total, void *stream);
// *loss = sum of weights * losses (of the tokens that count), divided by *total where there is one (0 where it is 0).
HcclResult vocab_loss_sum(const VocabLossCall &c, const float *losses, const float *total, float *loss, void *stream);
// What becomes of dw: written in bf16; written or added to in fp32; added to an fp32 sum and written in bf16.
enum VocabLossOut : int { VL_BF16 = 0, VL_F32 = 1, VL_ADD = 2, VL_ADD_BF16 = 3 };
// Gradients of scale * loss after vocab_loss_scores with grad (and with the losses that it or vocab_loss_combine left): dx bf16 [tokens, hidden] (of this shard alone), dw by `out`: in dw_sum
// where it is fp32, in dw where it is bf16.
HcclResult vocab_loss_grad(const VocabLossCall &c, const float *lse, const float *target, const float *total, float scale, void *dx, void *dw, float *dw_sum,
                           int out, void *scratch, void *stream);

// Loss and gradients of at most kVocabStepMost tokens against the whole vocabulary, in five to seven launches.
constexpr int64_t kVocabStepMost = 65536;
int64_t vocab_loss_step_bytes(int64_t tokens, int64_t vocab, int32_t hidden);
HcclResult vocab_loss_step(const VocabLossCall &c, bool mean, float scale, float *loss, void *dx, void *dw, float *dw_sum, int out, void *scratch, void *stream);

}  // namespace hcclb
