// jy_paged.hip — writing and reading the paged key/value cache.
//
// A vector (one row's key or value of one head, head_dim elements) belongs to 16 lanes, DL
// consecutive elements each, so its absolute maximum takes four DPP moves within a row of
// lanes and its bytes leave as one contiguous run.  The lanes take the key and the value of a head
// together: one look-up of the slot, two vectors in flight.  Every byte moves once; small calls are
// bound by the launch and the look-up's chain (position, page id), large ones by memory:
//   1 row of 2 heads of 64, fp32 to int8          2.6 us written, 1.9 read
//   256 rows of 8 heads of 128, bf16 to int8      4.5 and 3.1
//   8191 rows of the same (51 MB each way)        17.4 (2.9 TB/s) and 11.3 (4.5 TB/s)
//   32770 rows of 4 heads of 128 read (101 MB)    20 (5.1 TB/s, some of it the infinity cache's)
// Sixteen rows of one head a workgroup, so that a page's vectors leave side by side, measured 17.3 and
// 11.1 us for the 8191 rows, but 3.2 and 2.5 for one: heads stay fastest.
#include <hip/hip_runtime.h>

#include "jy_device.h"
#include "jy_paged_device.h"

namespace jy {

namespace {

struct Moved {
    jyhip_pages P;
    PageMap M;
    int rows, ps_log2;
    jyhip_vectors k, v;
};

// the vectors of this group of 16 lanes: (row, head), heads fastest; false past the end
struct Item {
    int row, head;
};
__device__ __forceinline__ bool item_of(const Moved& A, Item& it) {
    const unsigned i = blockIdx.x * 16 + (threadIdx.x >> 4), nkv = A.P.num_kv_heads;
    it.row = (int)(i / nkv);
    it.head = (int)(i - it.row * nkv);
    return it.row < A.rows;
}

// where the item's vectors lie in the pool (-1: they do not exist)
__device__ __forceinline__ int64_t vector_of(const Moved& A, const Item& it) {
    const int64_t slot = slot_of(A.M, A.P.num_pages, A.ps_log2, A.M.seq ? A.M.seq[it.row] : it.row, A.M.pos[it.row]);
    if (slot < 0) return -1;
    return (((slot >> A.ps_log2) * A.P.num_kv_heads + it.head) << A.ps_log2) + (slot & ((1 << A.ps_log2) - 1));
}

template <class PE, int PT, int DL>
__device__ __forceinline__ void hold(PE* dst, float* scale, const float (&x)[DL], bool on) {
    if constexpr (PT == JYHIP_T_I8) {
        float a = 0.0f;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < DL; i++) {
            a = fmaxf(a, fabsf(x[i]));
            bad |= !(fabsf(x[i]) <= 3.402823466e38f);
        }
        a = fmaxf(a, dpp_f<0xB1>(a));
        a = fmaxf(a, dpp_f<0x4E>(a));
        a = fmaxf(a, dpp_f<0x124>(a));
        a = fmaxf(a, dpp_f<0x128>(a));
        const unsigned group = threadIdx.x & 48u;
        bad = ((__ballot(bad) >> group) & 0xffffull) != 0;
        const float inv = quant_inv(a);
        if (on) {
            int8_t q[DL];
#pragma unroll
            for (int i = 0; i < DL; i++) q[i] = bad ? (int8_t)0 : quant_i8(x[i], inv);
            typedef int words __attribute__((ext_vector_type(DL / 4)));
            *reinterpret_cast<words*>(dst) = __builtin_bit_cast(words, q);
        }
        if ((threadIdx.x & 15) == 0) *scale = bad ? __builtin_nanf("") : quant_scale(a);
    } else if (on) {
        store_n<PE, DL, true>(dst, x);
    }
}

template <int PT, int T, int DL, bool VEC>
__global__ __launch_bounds__(256) void paged_write_kernel(Moved A) {
    typedef elem_t<PT> PE;
    typedef elem_t<T> E;
    Item it;
    if (!item_of(A, it)) return;
    const jyhip_pages& P = A.P;
    const int d0 = (threadIdx.x & 15) * DL;
    const bool on = d0 < P.head_dim;
    float k[DL], v[DL];
    if (on) {
        load_n<E, DL, VEC>(static_cast<const E*>(A.k.data) + it.row * A.k.row_stride + it.head * A.k.head_stride + d0, k);
        load_n<E, DL, VEC>(static_cast<const E*>(A.v.data) + it.row * A.v.row_stride + it.head * A.v.head_stride + d0, v);
    } else {
#pragma unroll
        for (int i = 0; i < DL; i++) k[i] = v[i] = 0.0f;
    }
    const int64_t vec = vector_of(A, it);
    if (vec < 0) return;
    hold<PE, PT, DL>(static_cast<PE*>(P.k) + vec * P.head_dim + d0, P.k_scale + vec, k, on);
    hold<PE, PT, DL>(static_cast<PE*>(P.v) + vec * P.head_dim + d0, P.v_scale + vec, v, on);
}

template <int PT, int T, int DL, bool VEC>
__global__ __launch_bounds__(256) void paged_read_kernel(Moved A) {
    typedef elem_t<PT> PE;
    typedef elem_t<T> E;
    Item it;
    if (!item_of(A, it)) return;
    const jyhip_pages& P = A.P;
    const int d0 = (threadIdx.x & 15) * DL;
    if (d0 >= P.head_dim) return;
    const int64_t vec = vector_of(A, it);
    float k[DL], v[DL];
    if (vec >= 0) {
        load_n<PE, DL, true>(static_cast<const PE*>(P.k) + vec * P.head_dim + d0, k);
        load_n<PE, DL, true>(static_cast<const PE*>(P.v) + vec * P.head_dim + d0, v);
        if constexpr (PT == JYHIP_T_I8) {
            const float ks = P.k_scale[vec], vs = P.v_scale[vec];
#pragma unroll
            for (int i = 0; i < DL; i++) {
                k[i] *= ks;
                v[i] *= vs;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < DL; i++) k[i] = v[i] = 0.0f;
    }
    store_n<E, DL, VEC>(static_cast<E*>(A.k.data) + it.row * A.k.row_stride + it.head * A.k.head_stride + d0, k);
    store_n<E, DL, VEC>(static_cast<E*>(A.v.data) + it.row * A.v.row_stride + it.head * A.v.head_stride + d0, v);
}

// a thread takes 8 pairs, which is as far as the rotation moves them
__global__ __launch_bounds__(256) void rope_rows_kernel(float* qkv, int rows, int width, const int* pos, int heads, int hd,
                                                        const float* cos_t, const float* sin_t) {
    const int half = hd / 2, groups = half / 8;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= (int64_t)rows * heads * groups) return;
    const int g = (int)(id % groups), head = (int)(id / groups % heads);
    const int64_t row = id / groups / heads;
    float* const x = qkv + row * width + head * hd + g * 16;
    const size_t t = (size_t)pos[row] * half + g * 8;
    float v[16], y[16];
    load_n<float, 16, true>(x, v);
#pragma unroll
    for (int o = 0; o < 8; o++) {
        const float c = cos_t[t + o], s = sin_t[t + o];
        const int d = o == 2 || o == 3 ? o + 2 : o == 4 || o == 5 ? o - 2 : o;
        y[2 * d] = __builtin_fmaf(v[2 * o], c, -(v[2 * o + 1] * s));
        y[2 * d + 1] = __builtin_fmaf(v[2 * o], s, v[2 * o + 1] * c);
    }
    store_n<float, 16, true>(x, y);
}

// whether every vector starts at a multiple of 16 bytes
bool aligned(const jyhip_vectors& x, int type) {
    const long long e = type == JYHIP_T_F32 ? 4 : 2;
    return ((uintptr_t)x.data | (uintptr_t)(x.row_stride * e) | (uintptr_t)(x.head_stride * e)) % 16 == 0;
}

template <bool WRITE, int PT, int T, int DL>
void launch_vec(const Moved& A, bool vec, unsigned grid, hipStream_t st) {
    if constexpr (WRITE) {
        if (vec)
            paged_write_kernel<PT, T, DL, true><<<grid, 256, 0, st>>>(A);
        else
            paged_write_kernel<PT, T, DL, false><<<grid, 256, 0, st>>>(A);
    } else {
        if (vec)
            paged_read_kernel<PT, T, DL, true><<<grid, 256, 0, st>>>(A);
        else
            paged_read_kernel<PT, T, DL, false><<<grid, 256, 0, st>>>(A);
    }
}

template <bool WRITE, int PT, int T>
void launch_dl(const Moved& A, bool vec, unsigned grid, hipStream_t st) {
    if (A.P.head_dim <= 64)
        launch_vec<WRITE, PT, T, 4>(A, vec, grid, st);
    else if (A.P.head_dim <= 128)
        launch_vec<WRITE, PT, T, 8>(A, vec, grid, st);
    else
        launch_vec<WRITE, PT, T, 16>(A, vec, grid, st);
}

template <bool WRITE, int PT>
void launch_io(const Moved& A, int type, bool vec, unsigned grid, hipStream_t st) {
    if (type == JYHIP_T_F32)
        launch_dl<WRITE, PT, JYHIP_T_F32>(A, vec, grid, st);
    else if (type == JYHIP_T_F16)
        launch_dl<WRITE, PT, JYHIP_T_F16>(A, vec, grid, st);
    else
        launch_dl<WRITE, PT, JYHIP_T_BF16>(A, vec, grid, st);
}

template <bool WRITE>
void launch_moved(const jyhip_pages& P, const PageMap& M, int rows, const jyhip_vectors& k, const jyhip_vectors& v,
                  int type, hipStream_t st) {
    const Moved A{P, M, rows, __builtin_ctz(P.page_size), k, v};
    const bool vec = aligned(k, type) && aligned(v, type);
    const unsigned grid = (unsigned)(((int64_t)rows * P.num_kv_heads + 15) / 16);
    if (P.type == JYHIP_T_I8)
        launch_io<WRITE, JYHIP_T_I8>(A, type, vec, grid, st);
    else if (P.type == JYHIP_T_F16)
        launch_io<WRITE, JYHIP_T_F16>(A, type, vec, grid, st);
    else
        launch_io<WRITE, JYHIP_T_BF16>(A, type, vec, grid, st);
}

}  // namespace

void launch_rope_rows(float* qkv, int rows, int width, const int* pos, int heads, int hd, const float* cos_t,
                      const float* sin_t, hipStream_t st) {
    const int64_t n = (int64_t)rows * heads * (hd / 16);
    rope_rows_kernel<<<(unsigned)((n + 255) / 256), 256, 0, st>>>(qkv, rows, width, pos, heads, hd, cos_t, sin_t);
}

void launch_paged_write(const jyhip_pages& P, const PageMap& M, int rows, const jyhip_vectors& k,
                        const jyhip_vectors& v, int type, hipStream_t st) {
    if (P.type == JYHIP_T_I4) return launch_paged4_write(P, M, rows, k, v, type, st);
    launch_moved<true>(P, M, rows, k, v, type, st);
}

void launch_paged_read(const jyhip_pages& P, const PageMap& M, int rows, const jyhip_vectors& k,
                       const jyhip_vectors& v, int type, hipStream_t st) {
    if (P.type == JYHIP_T_I4) return launch_paged4_read(P, M, rows, k, v, type, st);
    launch_moved<false>(P, M, rows, k, v, type, st);
}

}  // namespace jy
