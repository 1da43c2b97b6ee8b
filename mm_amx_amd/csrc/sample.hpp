// What the drawing of tokens is made of (sample.hip).
#pragma once

#include "common.hpp"

namespace mmx {

struct SampleArgs {
    const char* logits;  // rows of V fp32 or bf16, ld bytes apart
    int64_t ld;
    const float* u;
    const float *temperature, *top_p, *min_p;  // for each row, or NULL: the same for all
    const int32_t* top_k;
    double temperature_all, top_p_all, min_p_all;
    int top_k_all;
    int V;
    int shift;  // masses as whole numbers are multiples of 2^-shift: V of them stay below 2^62
    int slice;  // segments of a slice
    int32_t* ids;
    char* scratch;
};

}  // namespace mmx
