// jy_batch.cpp — the C entry points of include/jieyu_amd.h: argument checks, the launch on the
// caller's stream.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "jieyu_amd.h"
#include "jy_guard.h"
#include "jy_paged.h"
#include "jy_sample.h"

using namespace jy;

void jy::check_pages(const jyhip_pages* p) {
    if (!p) fail("pages is NULL");
    if (p->type != JYHIP_T_I8 && p->type != JYHIP_T_F16 && p->type != JYHIP_T_BF16)
        fail("pages: the type must be int8, fp16 or bf16");
    if (p->num_pages < 1 || p->num_kv_heads < 1) fail("pages: num_pages and num_kv_heads must be positive");
    const int ps = p->page_size;
    if (ps != 16 && ps != 32 && ps != 64 && ps != 128 && ps != 256)
        fail("pages: page_size must be 16, 32, 64, 128 or 256");
    if (p->head_dim < 16 || p->head_dim > 256 || p->head_dim % 16)
        fail("pages: head_dim must be a multiple of 16 up to 256");
    if (!p->k || !p->v) fail("pages: NULL k or v");
    if (((uintptr_t)p->k | (uintptr_t)p->v) % 16) fail("pages: k and v must be aligned to 16 bytes");
    if (p->type == JYHIP_T_I8) {
        if (!p->k_scale || !p->v_scale) fail("pages: int8 pages need scales");
        if (((uintptr_t)p->k_scale | (uintptr_t)p->v_scale) % 16) fail("pages: scales must be aligned to 16 bytes");
    } else if (p->k_scale || p->v_scale) {
        fail("pages: 16-bit pages have no scales");
    }
}

void jy::check_moved_size(int rows, int num_kv_heads) {
    // 16 threads a (row, head) in workgroups of 256, and a launch has less than 2^32 threads
    if ((int64_t)rows * num_kv_heads > (1 << 28) - 16) fail("rows x heads is too large for one call");
}

namespace {

constexpr int MAX_LEN = 1 << 30;  // (a position plus a chunk is an int in the kernels)

void check_tables(const jyhip_page_tables* t) {
    if (!t || !t->tables) fail("NULL page tables");
    if (t->num_seqs < 1 || t->table_stride < 1) fail("page tables: num_seqs and table_stride must be positive");
}

void check_type(int type) {
    if (type != JYHIP_T_F32 && type != JYHIP_T_F16 && type != JYHIP_T_BF16) fail("the type must be fp32, fp16 or bf16");
}

void check_vectors(const jyhip_vectors* x, int type, const char* name) {
    if (!x || !x->data) fail(std::string(name) + " is NULL");
    if ((uintptr_t)x->data % (type == JYHIP_T_F32 ? 4 : 2)) fail(std::string(name) + " is not aligned to its elements");
    if (x->row_stride < 0 || x->head_stride < 0) fail(std::string(name) + ": a negative stride");
}

// rows of jyhip_pages_write / _read; false when there is nothing to do
bool check_moved(const jyhip_pages* p, const jyhip_page_tables* t, int rows, const int* seq, const int* pos,
                 const jyhip_vectors* k, const jyhip_vectors* v, int type) {
    check_pages(p);
    check_tables(t);
    check_type(type);
    if (rows < 0) fail("rows must not be negative");
    if (rows == 0) return false;
    if (!pos) fail("pos is NULL");
    if (!seq && rows > t->num_seqs) fail("without seq there is one row per sequence: more rows than sequences");
    check_vectors(k, type, "k");
    check_vectors(v, type, "v");
    check_moved_size(rows, p->num_kv_heads);
    return true;
}

PageMap map_of(const jyhip_page_tables* t, const int* seq, const int* pos) {
    PageMap m;
    m.tables = t->tables;
    m.nseq = t->num_seqs;
    m.stride = t->table_stride;
    m.seq = seq;
    m.pos = pos;
    return m;
}

}  // namespace

extern "C" {

JYHIP_API int jyhip_pages_write(const jyhip_pages* pages, const jyhip_page_tables* tables, int rows, const int* seq,
                                const int* pos, const jyhip_vectors* k, const jyhip_vectors* v, int type,
                                void* stream) {
    return guarded([&]() {
        if (!check_moved(pages, tables, rows, seq, pos, k, v, type)) return 0;
        const OnDevice on(pages->device, (hipStream_t)stream);
        launch_paged_write(*pages, map_of(tables, seq, pos), rows, *k, *v, type, (hipStream_t)stream);
        CK(hipGetLastError());
        return 0;
    }, -1);
}

JYHIP_API int jyhip_pages_read(const jyhip_pages* pages, const jyhip_page_tables* tables, int rows, const int* seq,
                               const int* pos, const jyhip_vectors* k, const jyhip_vectors* v, int type, void* stream) {
    return guarded([&]() {
        if (!check_moved(pages, tables, rows, seq, pos, k, v, type)) return 0;
        const OnDevice on(pages->device, (hipStream_t)stream);
        launch_paged_read(*pages, map_of(tables, seq, pos), rows, *k, *v, type, (hipStream_t)stream);
        CK(hipGetLastError());
        return 0;
    }, -1);
}

JYHIP_API size_t jyhip_pages_attend_workspace(const jyhip_pages* pages, int num_seqs, int num_heads, int max_len) {
    if (!pages || num_seqs < 1 || num_heads < 1 || pages->num_kv_heads < 1 || max_len < 1 || max_len > MAX_LEN) return 0;
    if (num_heads % pages->num_kv_heads || pages->head_dim < 16 || pages->head_dim > 256) return 0;
    return paged_attend_part_floats(*pages, num_seqs, num_heads, max_len) * sizeof(float);
}

JYHIP_API int jyhip_pages_attend(const jyhip_pages* pages, const jyhip_page_tables* tables, const int* lens,
                                 int max_len, int num_heads, float scale, const jyhip_vectors* q,
                                 const jyhip_vectors* out, int type, void* workspace, size_t workspace_bytes,
                                 void* stream) {
    return guarded([&]() {
        check_pages(pages);
        check_tables(tables);
        check_type(type);
        if (!lens) fail("lens is NULL");
        if (max_len < 0 || max_len > MAX_LEN) fail("max_len must be between 0 and 2^30");
        if (num_heads < 1 || num_heads % pages->num_kv_heads)
            fail("the query heads must be a multiple of the key/value heads");
        if (!std::isfinite(scale)) fail("scale must be finite");
        check_vectors(q, type, "q");
        check_vectors(out, type, "out");
        PagedAttn A;
        A.P = *pages;
        A.M = map_of(tables, nullptr, nullptr);
        A.lens = lens;
        A.max_len = max_len;
        A.cap = (int)std::min<int64_t>(max_len, (int64_t)tables->table_stride * pages->page_size);
        A.nh = num_heads;
        A.scale = scale;
        A.q = *q;
        A.out = *out;
        A.type = type;
        A.part = static_cast<float*>(workspace);
        const size_t need = paged_attend_part_floats(*pages, tables->num_seqs, num_heads, max_len) * sizeof(float);
        if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
            fail("attend: the workspace must hold " + std::to_string(need) + " bytes, aligned to 16");
        if (paged_attend_blocks(*pages, tables->num_seqs, num_heads, max_len) >= (1 << 24))
            fail("attend: too many sequences and heads for one call");
        const OnDevice on(pages->device, (hipStream_t)stream);
        launch_paged_attend(A, (hipStream_t)stream);
        CK(hipGetLastError());
        return 0;
    }, -1);
}

JYHIP_API size_t jyhip_sample_workspace(int rows, int vocab) {
    if (rows < 1 || vocab < 1 || vocab > SAMPLE_MAX_VOCAB) return 0;
    return sample_workspace_bytes(rows, vocab);
}

JYHIP_API int jyhip_sample(const void* logits, int type, int rows, int vocab, long long row_stride, const float* u,
                           const float* temperature, const int* top_k, const float* top_p, const float* min_p,
                           int* ids, void* workspace, size_t workspace_bytes, int device, void* stream) {
    return guarded([&]() {
        check_type(type);
        if (rows < 0) fail("rows must not be negative");
        if (rows == 0) return 0;
        if (vocab < 1 || vocab > SAMPLE_MAX_VOCAB) fail("sample: vocab must be between 1 and 2^22");
        if (rows >= 1 << 20) fail("sample: too many rows for one call");
        if (!logits || !u || !ids) fail("sample: NULL logits, u or ids");
        if ((uintptr_t)logits % (type == JYHIP_T_F32 ? 4 : 2)) fail("sample: logits are not aligned to their elements");
        if (row_stride < 0) fail("sample: a negative row stride");
        SampleArgs A;
        A.logits = logits;
        A.row_stride = row_stride;
        A.type = type;
        A.rows = rows;
        A.vocab = vocab;
        A.u = u;
        A.temperature = temperature;
        A.top_k = top_k;
        A.top_p = top_p;
        A.min_p = min_p;
        A.ids = ids;
        A.ws = static_cast<unsigned char*>(workspace);
        const size_t need = sample_workspace_bytes(rows, vocab);
        if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
            fail("sample: the workspace must hold " + std::to_string(need) + " bytes, aligned to 16");
        const OnDevice on(device, (hipStream_t)stream);
        launch_sample(A, (hipStream_t)stream);
        CK(hipGetLastError());
        return 0;
    }, -1);
}

}  // extern "C"
