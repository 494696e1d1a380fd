// lists.cuh — softmax operators over lists of candidates: log probabilities with alternatives (log_probs.cu) and
// distillation from a teacher's top logits (distill.cu). A list is a row of a dense matrix or a run of a flat array
// between two boundaries (a query's documents).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace sb2 {

constexpr uint32_t kMaxTop = 128;  // most alternatives of a list, and most entries of a teacher's top

struct ListsArgs {
    const void* scores;
    int32_t type;            // SB2_F32 / SB2_BF16 / SB2_F16
    uint32_t lists;
    uint64_t width;          // dense: entries of a list; with bounds: entries behind `scores`
    uint64_t stride;         // dense: entries from one list to the next
    const uint32_t* bounds;  // nullptr (dense), or lists + 1 boundaries
};

struct LogProbsArgs {
    ListsArgs l;
    float inv_t;             // 1 / temperature
    uint32_t sms;
    uint32_t num_given, top;
    const int32_t* given;    // [lists, num_given]
    float* given_out;        // [lists, num_given]
    float* entropy;          // [lists] or nullptr
    float* log_sum;          // [lists] or nullptr
    int32_t* top_ids;        // [lists, top]
    float* top_out;          // [lists, top]
};

// A teacher's top: `ids` and `logits` of `top` entries a list, `stride` entries from one list to the next.
struct TeacherArgs {
    const int32_t* ids;
    const void* logits;
    const float* log_sum;    // nullptr: renormalised over the top
    int32_t type;
    uint32_t top;
    uint64_t stride;
};

struct DistillArgs {
    ListsArgs l;
    TeacherArgs t;
    float inv_t;
    uint32_t sms;
    uint64_t grad_stride;      // dense: entries from one list's gradients to the next's
    const float* weight;       // [lists] or nullptr
    float* loss;               // [lists] or nullptr
    void* grad;                // scores' type and layout, or nullptr
    void* hess;                // scores' type and layout, or nullptr
    bool clear;                // with bounds: entries of no list have derivatives 0
    // a training iteration's gradients only (f32):
    const float* row_weight;   // per entry, or nullptr
    const int32_t* stopped;    // nothing is done when set
    unsigned long long* max_g; // atomicMax of the f64 bits of |grad| and |hess|, or nullptr
    unsigned long long* max_h;
};

// CTAs that share a list of `entries`, as a cluster: while the lists leave half of the SMs without a CTA and a share
// keeps 4096 entries, twice as many, 8 at most (the largest cluster every device of the architecture takes).
inline uint32_t list_shares(uint64_t entries, uint32_t lists, uint32_t sms) {
    uint32_t shares = 1;
    while (shares < 8 && static_cast<uint64_t>(lists) * shares * 2 <= 2 * sms && entries / (2 * shares) >= 4096) shares *= 2;
    return shares;
}

// One launch each; errors are left for the caller's cudaGetLastError.
void launch_log_probs(const LogProbsArgs& a, cudaStream_t s);
void launch_distill(const DistillArgs& a, cudaStream_t s);

}  // namespace sb2
