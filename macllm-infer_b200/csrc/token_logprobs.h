// Log probabilities of given tokens (see token_logprobs.cu).
#pragma once
#include "common.cuh"
#include "shared_attention.h"   // bits of the status word
#include "verify_drafts.h"

namespace mk {

constexpr int kLogprobMaxTop = 64;

struct LogprobArgs {
    const void* logits = nullptr;   // [rows] of vocab values, ld apart
    int64_t ld = 0;
    int kind = 0;                   // 0 f32, 1 f16, 2 bf16
    int rows = 0, vocab = 0, top = 0;
    const int32_t* tokens = nullptr;
    float *logprobs = nullptr, *entropy = nullptr;
    int32_t* ranks = nullptr;
    int32_t* top_tokens = nullptr;  // [rows][top]
    float* top_logprobs = nullptr;
    int32_t* status = nullptr;      // may be null
};
void launch_token_logprobs(const LogprobArgs& a, cudaStream_t s);

}  // namespace mk
