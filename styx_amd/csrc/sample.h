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
    // workspace, per row: the chunks' largest keys, sums and counts of kept
    // words; weights and counts of the bins; border words
    unsigned long long *cmax, *csum, *hw;
    uint32_t *ccnt, *hc, *nlist, *list;
    int G, ch;  // chunks of a row, words of a chunk
};

struct SampleWs {
    int G, ch;
    int64_t bytes;
};
SampleWs sample_ws(int rows, int n);
// Places the workspace's arrays and launches.
hipError_t launch_sample(hipStream_t st, SampleArgs a, void *ws);

}  // namespace styx
