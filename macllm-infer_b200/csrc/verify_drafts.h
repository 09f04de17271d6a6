// Verification of drafted tokens against the target's distribution (see verify_drafts.cu).
#pragma once
#include "common.cuh"

namespace mk {

constexpr int kDevBadRow = 8;     // a row of logits without a distribution (NaN, +inf or nothing above -inf); bits 1 to 4 in shared_attention.h
constexpr int kVerifyMaxTopK = 1024;
constexpr int kVerifyMaxVocab = 8 * 52000;   // eight CTAs' shared memory at 32 bits a value

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
    int2* rows = nullptr;              // scratch [lanes][n_drafts + 1]: (draft accepted, token drawn in its place)
    int32_t* status = nullptr;
    int list_at = 0;                   // filled in by the launcher: where a CTA's list of candidates begins in its shared memory
};
inline int64_t verify_scratch_bytes(int lanes, int n_drafts) { return (int64_t)lanes * (n_drafts + 1) * 8; }
void launch_verify_drafts(VerifyArgs a, cudaStream_t s);

}  // namespace mk
