// jy_paged.h — launchers of the paged cache's kernels (jy_paged.hip, jy_paged_attention.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "jieyu_amd.h"

namespace jy {

// throws jy::Error where the kernels cannot run on these pages
void check_pages(const jyhip_pages* p);
// throws jy::Error where rows x heads is more than one launch of launch_paged_write / _read takes
void check_moved_size(int rows, int num_kv_heads);

// which position each row is, and where it lies (jyhip_page_tables with the rows' indices)
struct PageMap {
    const int* tables = nullptr;
    int nseq = 0, stride = 0;
    const int* seq = nullptr;
    const int* pos = nullptr;
};

void launch_paged_write(const jyhip_pages& P, const PageMap& M, int rows, const jyhip_vectors& k,
                        const jyhip_vectors& v, int type, hipStream_t st);
void launch_paged_read(const jyhip_pages& P, const PageMap& M, int rows, const jyhip_vectors& k,
                       const jyhip_vectors& v, int type, hipStream_t st);

// RoPE on the q and k heads of every row of qkv ([rows][width], q then k first) in place, row r at
// position pos[r], the rotated pairs in rope_pack's order; head_dim a multiple of 16
void launch_rope_rows(float* qkv, int rows, int width, const int* pos, int heads, int hd, const float* cos_t,
                      const float* sin_t, hipStream_t st);

struct PagedAttn {
    jyhip_pages P;
    PageMap M;                   // tables only: sequence s is row s
    const int* lens = nullptr;
    int max_len = 0;             // sizes the launch
    int cap = 0;                 // positions past it do not exist: the smaller of max_len and the table's
    int nh = 0;
    float scale = 1.0f;
    jyhip_vectors q{}, out{};
    int type = 0;
    float* part = nullptr;       // paged_attend_part_floats() floats
};
size_t paged_attend_part_floats(const jyhip_pages& P, int nseq, int nh, int max_len);
// workgroups of 256 threads of the larger of its launches
int64_t paged_attend_blocks(const jyhip_pages& P, int nseq, int nh, int max_len);
void launch_paged_attend(const PagedAttn& A, hipStream_t st);

}  // namespace jy
