// jy_sample.h — launcher of the sampling kernels (jy_sample.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "jieyu_amd.h"

namespace jy {

// most logits of one row: keeps the fixed-point masses' sum under 2^63 with 40 bits of fraction
constexpr int SAMPLE_MAX_VOCAB = 1 << 22;

struct SampleArgs {
    const void* logits = nullptr;
    long long row_stride = 0;
    int type = 0, rows = 0, vocab = 0;
    const float* u = nullptr;
    const float* temperature = nullptr;  // each null: the filter is off (temperature: 1)
    const int* top_k = nullptr;
    const float* top_p = nullptr;
    const float* min_p = nullptr;
    int* ids = nullptr;
    unsigned char* ws = nullptr;
};
size_t sample_workspace_bytes(int rows, int vocab);
void launch_sample(const SampleArgs& A, hipStream_t st);
// a generation's device state after the token ids[at]: state[0] = at + 1, state[1] (stopped) = 0; where
// there was none to pick (-1), id 0 stands for it and state[2] is set
void launch_advance(int* ids, int* state, int at, hipStream_t st);

}  // namespace jy
