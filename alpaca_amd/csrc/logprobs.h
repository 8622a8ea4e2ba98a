// Log probabilities of tokens (kernels_logprobs.hip).
#pragma once

#include "common.h"

constexpr int kLogprobsMostTop = 32;
constexpr int kLogprobsMostSplitRows = 512;  // rows that may be split, a counter each at the front of the workspace
constexpr int kLogprobsParts = 2048;         // their parts in all

struct LogprobsArgs {
    const void* logits = nullptr;
    int64_t stride = 0;
    int rows = 0, vocab = 0, top = 0;
    const int* tokens = nullptr;
    float* logprobs = nullptr;
    float* entropy = nullptr;
    int* top_tokens = nullptr;
    float* top_logprobs = nullptr;
    // the launcher's
    int splits = 1, each = 0;
    int* counters = nullptr;
    float* parts = nullptr;
};
int64_t logprobs_workspace();
// workspace: of logprobs_workspace() bytes, its counters zero before and after every launch, or null (no row is split).
hipError_t launch_logprobs(bool f16_logits, LogprobsArgs p, void* workspace, hipStream_t st);
