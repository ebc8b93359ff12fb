// jy_batch.cpp — the C entry points of include/jieyu_amd.h: argument checks, the launch on the
// caller's stream.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "jieyu_amd.h"
#include "jy_guard.h"
#include "jy_paged.h"
#include "jy_rope.h"
#include "jy_sample.h"

using namespace jy;

void jy::check_pages(const jyhip_pages* p) {
    if (!p) fail("pages is NULL");
    if (p->type != JYHIP_T_I8 && p->type != JYHIP_T_I4 && p->type != JYHIP_T_F16 && p->type != JYHIP_T_BF16)
        fail("pages: the type must be int8, 4-bit, fp16 or bf16");
    if (p->num_pages < 1 || p->num_kv_heads < 1) fail("pages: num_pages and num_kv_heads must be positive");
    const int ps = p->page_size;
    if (ps != 16 && ps != 32 && ps != 64 && ps != 128 && ps != 256)
        fail("pages: page_size must be 16, 32, 64, 128 or 256");
    if (p->head_dim < 16 || p->head_dim > 256 || p->head_dim % 16)
        fail("pages: head_dim must be a multiple of 16 up to 256");
    if (!p->k || !p->v) fail("pages: NULL k or v");
    if (((uintptr_t)p->k | (uintptr_t)p->v) % 16) fail("pages: k and v must be aligned to 16 bytes");
    if (p->type == JYHIP_T_I8 || p->type == JYHIP_T_I4) {
        if (!p->k_scale || !p->v_scale) fail("pages: int8 and 4-bit pages need scales");
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

// whether attention over these pages is one that a workspace is given for
bool shaped(const jyhip_pages& p, int num_heads, int max_len) {
    return num_heads >= 1 && p.num_kv_heads >= 1 && max_len >= 0 && max_len <= MAX_LEN && num_heads % p.num_kv_heads == 0 &&
           p.head_dim >= 16 && p.head_dim <= 256;
}

// what single rows and runs of rows have in common, checked
RuledAttn ruled_args(const jyhip_pages* pages, const jyhip_page_tables* tables, int max_len, int num_heads, float scale,
                     const jyhip_rules* rules, const jyhip_vectors* q, const jyhip_vectors* out, int type) {
    check_pages(pages);
    check_tables(tables);
    check_type(type);
    if (max_len < 0 || max_len > MAX_LEN) fail("max_len must be between 0 and 2^30");
    if (num_heads < 1 || num_heads % pages->num_kv_heads) fail("the query heads must be a multiple of the key/value heads");
    if (!std::isfinite(scale)) fail("scale must be finite");
    check_vectors(q, type, "q");
    check_vectors(out, type, "out");
    RuledAttn A;
    A.P = *pages;
    A.M = map_of(tables, nullptr, nullptr);
    A.span = std::max(max_len, 1);
    A.most = max_len;
    A.cap = (int)std::min<int64_t>(MAX_LEN, (int64_t)tables->table_stride * pages->page_size);
    A.nh = num_heads;
    A.scale = scale;
    if (rules) {
        if (!std::isfinite(rules->cap) || rules->cap < 0.0f) fail("the cap must be finite and not negative");
        if (rules->cap != 0.0f && !std::isfinite(scale / rules->cap * 4.0f)) fail("scale over the cap must be finite");
        if (((uintptr_t)rules->slopes | (uintptr_t)rules->first | (uintptr_t)rules->last) % 4)
            fail("slopes, first or last are not aligned to their elements");
        A.soft = std::min(rules->cap, 0x1p64f);
        A.slopes = rules->slopes;
        A.first = rules->first;
        A.last = rules->last;
    }
    A.q = *q;
    A.out = *out;
    A.type = type;
    return A;
}

// whether weights that are written [seqs][heads][len] have an element each
bool apart(long long seq_stride, int seqs, long long head_stride, int heads, int len) {
    if (len == 0) return true;
    auto nested = [len](long long inner, int a, long long outer, int b) {
        return (a == 1 || inner >= len) && (b == 1 || (__int128)outer >= (a == 1 ? 0 : (__int128)inner * (a - 1)) + len);
    };
    return nested(head_stride, heads, seq_stride, seqs) || nested(seq_stride, seqs, head_stride, heads);
}

void launch_checked(RuledAttn& A, void* workspace, size_t workspace_bytes, int device, hipStream_t st) {
    A.part = static_cast<float*>(workspace);
    const size_t need = ruled_attend_part_floats(A) * sizeof(float);
    if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
        fail("attend: the workspace must hold " + std::to_string(need) + " bytes, aligned to 16");
    if (ruled_attend_blocks(A) >= (1 << 24)) fail("attend: too many rows and heads for one call");
    const OnDevice on(device, st);
    launch_ruled_attend(A, st);
    CK(hipGetLastError());
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

JYHIP_API size_t jyhip_pages_attend_ruled_workspace(const jyhip_pages* pages, int num_seqs, int num_heads, int max_len,
                                                    int has_first, int has_weights) {
    if (!pages || num_seqs < 1 || !shaped(*pages, num_heads, max_len)) return 0;
    static const int some = 0;
    static float any = 0.0f;
    RuledAttn A;
    A.P = *pages;
    A.M.nseq = A.rows = num_seqs;
    A.nh = num_heads;
    A.span = std::max(max_len, 1);
    A.first = has_first ? &some : nullptr;
    A.weights = has_weights ? &any : nullptr;
    return ruled_attend_part_floats(A) * sizeof(float);
}

JYHIP_API int jyhip_pages_attend_ruled(const jyhip_pages* pages, const jyhip_page_tables* tables, const int* lens,
                                       int max_len, int num_heads, float scale, const jyhip_rules* rules,
                                       const jyhip_vectors* q, const jyhip_vectors* out, int type, float* weights,
                                       long long weights_seq_stride, long long weights_head_stride, int weights_len,
                                       void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&]() {
        RuledAttn A = ruled_args(pages, tables, max_len, num_heads, scale, rules, q, out, type);
        if (!lens) fail("lens is NULL");
        if (rules && rules->last) fail("attend: one row per sequence ends at its length: last is for runs of rows");
        if (weights && (weights_seq_stride < 0 || weights_head_stride < 0 || weights_len < 0))
            fail("attend: a negative stride or length of the weights");
        if ((uintptr_t)weights % 4) fail("attend: weights are not aligned to their elements");
        if (weights && !apart(weights_seq_stride, tables->num_seqs, weights_head_stride, pages->num_kv_heads, weights_len))
            fail("attend: the weights of two sequences or heads share elements");
        A.lens = lens;
        A.rows = tables->num_seqs;
        if (!A.first) A.cap = std::min(A.cap, max_len);
        A.weights = weights;
        A.seq_stride = weights_seq_stride;
        A.head_stride = weights_head_stride;
        A.weights_len = weights_len;
        launch_checked(A, workspace, workspace_bytes, pages->device, (hipStream_t)stream);
        return 0;
    }, -1);
}

JYHIP_API size_t jyhip_pages_attend_rows_workspace(const jyhip_pages* pages, int num_seqs, int rows, int num_heads,
                                                   int max_len, int type) {
    if (!pages || num_seqs < 1 || rows < 1 || !shaped(*pages, num_heads, max_len)) return 0;
    static const int some = 0;
    RuledAttn A;
    A.P = *pages;
    A.M.nseq = num_seqs;
    A.rows = rows;
    A.nh = num_heads;
    A.span = std::max(max_len, 1);
    A.starts = &some;
    A.type = type;
    return ruled_attend_part_floats(A) * sizeof(float);
}

JYHIP_API int jyhip_pages_attend_rows(const jyhip_pages* pages, const jyhip_page_tables* tables, const int* starts,
                                      const int* pos, int rows, int max_len, int num_heads, float scale,
                                      const jyhip_rules* rules, const jyhip_vectors* q, const jyhip_vectors* out, int type,
                                      void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&]() {
        if (rows < 0) fail("rows must not be negative");
        if (rows == 0) {
            check_pages(pages);
            check_tables(tables);
            check_type(type);
            return 0;
        }
        RuledAttn A = ruled_args(pages, tables, max_len, num_heads, scale, rules, q, out, type);
        if (!starts || !pos) fail("attend_rows: NULL starts or pos");
        A.starts = starts;
        A.pos = pos;
        A.rows = rows;
        A.cap = std::min(A.cap, max_len);
        launch_checked(A, workspace, workspace_bytes, pages->device, (hipStream_t)stream);
        return 0;
    }, -1);
}

JYHIP_API int jyhip_pages_evict(const jyhip_pages* pages, const jyhip_page_tables* tables, const jyhip_page_tables* to,
                                const int* lens, int* new_lens, int max_len, int keep, int recent, const float* weights,
                                long long weights_seq_stride, long long weights_head_stride, int weights_len,
                                float* new_weights, long long new_seq_stride, long long new_head_stride,
                                int new_weights_len, int* kept, void* stream) {
    return guarded([&]() {
        check_pages(pages);
        check_tables(tables);
        check_tables(to);
        if (tables->num_seqs != to->num_seqs) fail("evict: the new tables are of other sequences");
        if (!lens || !new_lens || (!weights && weights_len) || !kept) fail("evict: NULL lens, new_lens, weights or kept");
        if (lens == new_lens) fail("evict: lens and new_lens must be apart");
        if (((uintptr_t)lens | (uintptr_t)new_lens | (uintptr_t)weights | (uintptr_t)new_weights | (uintptr_t)kept) % 4)
            fail("evict: a buffer is not aligned to its elements");
        if (max_len < 0 || max_len > MAX_LEN) fail("max_len must be between 0 and 2^30");
        if (keep < 1 || keep > MAX_LEN) fail("evict: keep must be between 1 and 2^30");
        if (recent < 0 || recent > keep) fail("evict: recent must be between 0 and keep");
        if (weights_seq_stride < 0 || weights_head_stride < 0 || weights_len < 0 || new_seq_stride < 0 || new_head_stride < 0 ||
            new_weights_len < 0)
            fail("evict: a negative stride or length of weights");
        if (new_weights && !apart(new_seq_stride, tables->num_seqs, new_head_stride, pages->num_kv_heads, new_weights_len))
            fail("evict: the new weights of two sequences or heads share elements");
        Eviction E;
        E.P = *pages;
        E.M = map_of(tables, nullptr, nullptr);
        E.to = map_of(to, nullptr, nullptr);
        E.lens = lens;
        E.new_lens = new_lens;
        E.cap = (int)std::min<int64_t>(max_len, (int64_t)tables->table_stride * pages->page_size);
        E.keep = keep;
        E.recent = recent;
        if ((int64_t)to->table_stride * pages->page_size < std::min(keep, E.cap))
            fail("evict: the new tables have too few pages for what stays");
        const int64_t heads = (int64_t)tables->num_seqs * pages->num_kv_heads;
        if (heads >= 1 << 22 || heads * std::min(keep, std::max(E.cap, 1)) > (1 << 28) - 16)
            fail("evict: sequences x heads x keep is too large for one call");
        E.weights = weights;
        E.new_weights = new_weights;
        E.seq_stride = weights_seq_stride;
        E.head_stride = weights_head_stride;
        E.weights_len = weights_len;
        E.new_seq_stride = new_seq_stride;
        E.new_head_stride = new_head_stride;
        E.new_weights_len = new_weights_len;
        E.kept = kept;
        const OnDevice on(pages->device, (hipStream_t)stream);
        launch_evict(E, (hipStream_t)stream);
        CK(hipGetLastError());
        return 0;
    }, -1);
}

JYHIP_API int jyhip_rope(const jyhip_vectors* q, const jyhip_vectors* q_out, int q_heads, const jyhip_vectors* k,
                         const jyhip_vectors* k_out, int k_heads, int rows, int head_dim, const int* pos,
                         const double* freq, int pairs, int interleaved, float factor, int type, int device,
                         void* stream) {
    return guarded([&]() {
        check_type(type);
        if (rows < 0 || q_heads < 0 || k_heads < 0) fail("rope: rows and heads must not be negative");
        if (head_dim < 2 || head_dim > ROPE_MAX_HEAD) fail("rope: head_dim must be between 2 and 1024");
        if (pairs < 1 || 2 * (int64_t)pairs > head_dim) fail("rope: 2 * pairs must be between 2 and head_dim");
        if (((int64_t)q_heads + k_heads) * head_dim > 1 << 20) fail("rope: heads x head_dim is over 2^20");
        if (rows == 0 || q_heads + k_heads == 0) return 0;
        if (!pos || !freq) fail("rope: NULL pos or freq");
        if ((uintptr_t)freq % 8 || (uintptr_t)pos % 4) fail("rope: pos or freq is not aligned to its elements");
        RopeArgs A;
        if (q_heads) {
            check_vectors(q, type, "q");
            check_vectors(q_out, type, "q_out");
            A.q = *q;
            A.q_out = *q_out;
        }
        if (k_heads) {
            check_vectors(k, type, "k");
            check_vectors(k_out, type, "k_out");
            A.k = *k;
            A.k_out = *k_out;
        }
        A.q_heads = q_heads;
        A.k_heads = k_heads;
        A.rows = rows;
        A.hd = head_dim;
        A.pos = pos;
        A.freq = freq;
        A.pairs = pairs;
        A.interleaved = interleaved != 0;
        A.factor = factor;
        A.type = type;
        if (rope_blocks(A) >= (1 << 24)) fail("rope: too many rows for one call");
        const OnDevice on(device, (hipStream_t)stream);
        launch_rope(A, (hipStream_t)stream);
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
