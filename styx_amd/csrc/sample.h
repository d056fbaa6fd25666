// sample.h -- arguments of the sampling launches (sample.hip).
#pragma once

#include "common.h"

namespace styx {

// Most words of a row: 2^19 - 1 weights of at most 2^44 sum below 2^63.
constexpr int SAMPLE_MAX_N = (1 << 19) - 1;
constexpr int SAMPLE_BINS = 2048;

struct SampleArgs {
    const float *logits;
    int64_t ld;
    int rows, n;
    const styx_sample_params *params;
    int one_params;  // every row has params[0]
    const float *u;
    uint32_t *token;
    float *logprob;   // or null
    uint32_t *n_kept; // or null
    // workspace (filled by the launch), per row: per block of words the first
    // one's key, sum and number of those that surely stay, number of border
    // words; weights and numbers of the bins; border words, each block's at
    // its own place
    unsigned long long *top, *sum, *hw;
    uint32_t *cnt, *lcnt, *hc;
    uint16_t *list;
    int blocks, per, G;  // blocks of a row, of a workgroup; workgroups of a row
};

struct SampleWs {
    int blocks, per, G;
    int64_t bytes;
};
SampleWs sample_ws(int rows, int n);
// Places the workspace's arrays and launches.
hipError_t launch_sample(hipStream_t st, SampleArgs a, void *ws);

}  // namespace styx
