// jy_rope.h — launcher of the rotary kernel (jy_rope.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "jieyu_amd.h"

namespace jy {

constexpr int ROPE_MAX_HEAD = 1024;  // elements of a head

struct RopeArgs {
    jyhip_vectors q{}, k{}, q_out{}, k_out{};
    int q_heads = 0, k_heads = 0, rows = 0, hd = 0;
    const int* pos = nullptr;
    const double* freq = nullptr;  // [pairs]
    int pairs = 0;
    bool interleaved = false;
    float factor = 1.0f;
    int type = 0;
};
// workgroups of a launch
int64_t rope_blocks(const RopeArgs& A);
void launch_rope(const RopeArgs& A, hipStream_t st);

}  // namespace jy
