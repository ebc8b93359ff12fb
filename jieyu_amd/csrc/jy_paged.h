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

// the same for 4-bit pages (jy_paged4.hip)
void launch_paged4_write(const jyhip_pages& P, const PageMap& M, int rows, const jyhip_vectors& k,
                         const jyhip_vectors& v, int type, hipStream_t st);
void launch_paged4_read(const jyhip_pages& P, const PageMap& M, int rows, const jyhip_vectors& k,
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

// Attention with rules for scores, of one row per sequence (starts null: row s is sequence s, its positions
// first[s] .. lens[s] - 1) or of runs of rows (sequence s has rows starts[s] .. starts[s + 1] - 1, row r at
// position pos[r] over first[r] .. last[r] - 1).
struct RuledAttn {
    jyhip_pages P;
    PageMap M;  // tables only
    const int* lens = nullptr;
    const int* starts = nullptr;
    const int* pos = nullptr;
    const int* first = nullptr;  // null: 0
    const int* last = nullptr;   // null: pos + 1
    int rows = 0;
    int span = 0;  // at least 1: most positions that a row (starts null) or a run of rows may see, sizes the launch
    int most = 0;  // with `first`, one row per sequence: positions past the first `most` do not count
    int cap = 0;   // positions past it do not exist
    int nh = 0;
    float scale = 1.0f;
    float soft = 0.0f;              // scores stay within +-soft (0: any)
    const float* slopes = nullptr;  // [nh] null: no bias
    jyhip_vectors q{}, out{};
    int type = 0;
    // one row per sequence: the weights of position j < weights_len are added to weights[s * seq_stride +
    // kv head * head_stride + j]
    float* weights = nullptr;
    long long seq_stride = 0, head_stride = 0;
    int weights_len = 0;
    float* part = nullptr;  // ruled_attend_part_floats() floats
};
// rows, runs, heads and span as launch_ruled_attend gets them
size_t ruled_attend_part_floats(const RuledAttn& A);
int64_t ruled_attend_blocks(const RuledAttn& A);
void launch_ruled_attend(const RuledAttn& A, hipStream_t st);

// Eviction: of each sequence's positions the last `recent` and the heaviest of the others, `keep` in all, to
// the front of the pages that new_tables names.
struct Eviction {
    jyhip_pages P;
    PageMap M, to;  // tables only
    const int* lens = nullptr;
    int* new_lens = nullptr;
    int cap = 0;  // positions past it do not exist
    int keep = 0, recent = 0;
    const float* weights = nullptr;  // [s * seq_stride + kv head * head_stride + position], weights_len of them
    float* new_weights = nullptr;    // null: not wanted
    long long seq_stride = 0, head_stride = 0, new_seq_stride = 0, new_head_stride = 0;
    int weights_len = 0, new_weights_len = 0;
    int* kept = nullptr;  // [nseq][kv heads][keep]
};
void launch_evict(const Eviction& E, hipStream_t st);

}  // namespace jy
