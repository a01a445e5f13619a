// Launch interface of the token embedding (kernels/vocab_embed.cu).
#pragma once
#include "common/base.h"

namespace hcclb {

// Tokens of one gradient: every tile of the sort reads the histograms of all of them.
constexpr int64_t kEmbedGradMost = 1 << 24;

// Rows of a vocabulary (or of one rank's shard of it, which holds the ids first .. first + vocab - 1).
struct EmbedTable {
    int64_t vocab, first;
    int32_t hidden;
    HcclDataType type;  // FP32, FP16, BFP16
};
struct EmbedIds {
    const void *ids;
    bool wide;          // 64-bit ids
    int64_t tokens;
};
HcclResult embed_lookup(const EmbedTable &t, const EmbedIds &ids, const void *weights, int64_t stride, float scale, void *out, void *stream);
int64_t embed_grad_scratch_bytes(int64_t tokens, int64_t vocab, int32_t hidden);
// add: out is fp32 and the sums are added to it; else out has the table's type and every row of it is written.
HcclResult embed_grad(const EmbedTable &t, const EmbedIds &ids, const void *grad, int64_t stride, float scale, void *out, bool add, void *scratch,
                      void *stream);

}  // namespace hcclb
