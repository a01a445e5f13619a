// Launch interface of the router of a mixture-of-experts layer (kernels/moe_gate.cu).
#pragma once
#include "common/base.h"

namespace hcclb {

constexpr int kGateMaxExperts = 4096, kGateMaxTopk = 32;

struct GateShape {
    int64_t tokens;
    int32_t experts, topk;
    HcclDataType type;       // of the logits: FP32, FP16, BFP16
    int64_t stride;          // elements between rows of the logits
    bool normalize;          // gates of a token sum to one
    bool again;              // gradient: slots of a token may name an expert more than once
};
int64_t moe_gate_scratch_bytes(int64_t tokens, int32_t experts);
HcclResult moe_gate(const GateShape &s, const void *logits, const uint8_t *mask, int32_t *idx, float *gates, int32_t *counts, float *prob_sum,
                    int32_t *routed, float *balance, void *scratch, void *stream);
HcclResult moe_balance(const int32_t *counts, const float *prob_sum, const int32_t *routed, int32_t experts, int32_t topk, float *balance, void *stream);
// d_gates may be null (no gradient of the gates); coef: gradient of the balance loss.
HcclResult moe_gate_grad(const GateShape &s, const void *logits, const int32_t *idx, const float *d_gates, const int32_t *counts, const int32_t *routed,
                         const uint8_t *mask, float coef, void *d_logits, void *stream);

}  // namespace hcclb
