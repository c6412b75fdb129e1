// sample.h -- the draw of a token from logits (sample.hip), for the entry point and the decoder.
#pragma once

#include "kv4.h"

namespace ojx {

struct SampleParams {
    const void *logits;                  // row r at logits + r * stride (elements)
    long stride;
    const float *uniform;                // [rows], or with step: of one row, entry *step
    const int *step;
    int *tokens;                         // [rows]
    int rows, vocab, slices;
    // one value for all rows, or an array of a value for each
    double temperature, top_p, min_p;
    int top_k;
    const float *temperatures, *top_ps, *min_ps;
    const int *top_ks;
};

long sample_workspace(int rows, int vocab);      // bytes, or an error code
int check_sampling(double temperature, double top_p, double min_p);
int launch_sample(SampleParams a, int dtype, void *workspace, hipStream_t st);

}  // namespace ojx
