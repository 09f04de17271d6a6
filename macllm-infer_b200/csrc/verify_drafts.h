// Verification of drafted tokens against the target's distribution (see verify_drafts.cu).
#pragma once
#include "common.cuh"

namespace mk {

constexpr int kDevBadRow = 8;     // a row of logits without a distribution (NaN, +inf or nothing above -inf); bits 1 to 4 in shared_attention.h
constexpr int kVerifyMaxTopK = 1024;
constexpr int kVerifyMaxVocab = 416000;   // the best values of a row's threads fit shared memory, 32 tokens a thread

struct VerifyArgs {
    const void* logits = nullptr;      // [lanes][drafts + 1] rows of vocab values, ld values apart
    int64_t ld = 0;
    int type = 0;                      // 0 f32, 1 f16, 2 bf16
    int lanes = 0, n_drafts = 0, vocab = 0;
    const int32_t* drafts = nullptr;   // [lanes][n_drafts]; the first negative one ends a lane's
    const float* draft_probs = nullptr;// [lanes][n_drafts][vocab] or null: all on the drafted token
    const float* u = nullptr;          // [lanes][n_drafts + 1]
    const float* temperature = nullptr;// [lanes]
    const int32_t* top_k = nullptr;    // [lanes]
    const float* top_p = nullptr;      // [lanes]
    int32_t* tokens = nullptr;         // [lanes][n_drafts + 1]
    int32_t* accepted = nullptr;       // [lanes]
    int32_t* status = nullptr;
    // filled in by the launcher
    float* group_best = nullptr;       // [rows][runs][256] best value of each thread's tokens
    void* run_results = nullptr;       // [rows][runs]
    int2* rows = nullptr;              // (draft kept, token drawn in its place)
    int vpt = 0, runs = 0, list_at = 0, keys_at = 0;
};

// How a call is cut, and its workspace.
struct VerifyPlan {
    int vpt = 1, runs = 0;             // pieces of 16 bytes to a thread; runs of tokens, a CTA each, to a row
    int64_t results_at = 0, rows_at = 0, bytes = 0;
};
VerifyPlan verify_plan(int type, int lanes, int n_drafts, int vocab);
void launch_verify_drafts(VerifyArgs a, const VerifyPlan& p, uint8_t* workspace, cudaStream_t s);

}  // namespace mk
