// jy_ruled.h — what the two kernels of attention under rules (jy_ruled_attention.hip, jy_tiled_attention.hip) share:
// the call with its plan and workspace, and which rows a workgroup takes.
#pragma once

#include "jy_device.h"
#include "jy_paged.h"

namespace jy {

struct Ruled {
    RuledAttn A;
    int ps_log2;
    int hpg, rpg;   // heads and rows of a column group
    int tiles;      // groups of heads per kv head
    int groups;     // groups of rows: the most there can be
    int chunk, splits;
    bool tiled = false;    // by jy_tiled_attention.hip
    bool aligned = false;  // its vectors start at multiples of 16 bytes
    int sstride;    // scores of one (row, head) in the workspace
    float* part_o;  // [rows][nh][splits][hd]
    float2* part_ml;
    int* part_live;  // [rows] chunks that a row's group had
    float2* ml;      // [rows][nh] the final maximum and sum
    float* scores;   // [rows][nh][sstride], from the group's first multiple of 32 on
};

// jy_tiled_attention.hip: the plan of runs of rows (false: not one for it), the launch
bool plan_tiled(Ruled& K);
void launch_tiled(const Ruled& K, unsigned grid, hipStream_t st);

namespace {

// smallest / largest over a row of 16 lanes, in each of them
template <int CTRL>
__device__ __forceinline__ int dpp_i(int v) {
    return __builtin_bit_cast(int, dpp_f<CTRL>(__builtin_bit_cast(float, v)));
}
__device__ __forceinline__ int cols_min(int v) {
    v = min(v, dpp_i<0xB1>(v));
    v = min(v, dpp_i<0x4E>(v));
    v = min(v, dpp_i<0x124>(v));
    return min(v, dpp_i<0x128>(v));
}
__device__ __forceinline__ int cols_max(int v) { return -cols_min(-v); }

// The run and group of rows that group number `at` of the launch is: (sequence, first row), sequence -1 past
// the last.  The lanes look at 64 runs at a time.
struct Run {
    int seq, row0, end;
};
__device__ __forceinline__ Run run_of(const Ruled& K, int at) {
    Run r{-1, 0, 0};
#if defined(__HIP_DEVICE_COMPILE__)
    const int lane = threadIdx.x & 63, n = K.A.M.nseq;
    for (int s0 = 0; s0 < n; s0 += 64) {
        const int s = s0 + lane;
        int a = 0, b = 0;
        if (s < n) {
            a = min(max(K.A.starts[s], 0), K.A.rows);
            b = min(max(K.A.starts[s + 1], a), K.A.rows);
        }
        int sum = (b - a + K.rpg - 1) / K.rpg;
        const int own = sum;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int v = __shfl_up(sum, d);
            if (lane >= d) sum += v;
        }
        const unsigned long long hit = __ballot(sum > at);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            r.seq = s0 + l;
            r.row0 = __builtin_amdgcn_readlane(a, l) + (at - __builtin_amdgcn_readlane(sum - own, l)) * K.rpg;
            r.end = __builtin_amdgcn_readlane(b, l);
            return r;
        }
        at -= __builtin_amdgcn_readlane(sum, 63);
    }
#endif
    return r;
}

}  // namespace

}  // namespace jy
