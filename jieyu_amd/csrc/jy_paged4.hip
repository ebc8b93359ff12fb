// jy_paged4.hip — writing and reading 4-bit pages.
//
// A vector's elements come in groups of 32, each with its lowest value and step in fp16:
//   low = fp16(min x), step = fp16((max x - low) / 15 in seven significant bits),
//   n = rint((x - low) / step) in 0 .. 15; value n step + low
// The numbers go by the rounded low and step, so those roundings bias nothing.  A step of seven bits times a
// number of four is exact in fp16: the attention's products take it so.
//
// 16 lanes take a vector, and lane r elements 32 g + 2 r and 32 g + 2 r + 1 of every group g: its byte of
// each group lies beside the others (byte r G + g of the vector, G groups), so a lane's bytes are one store,
// and the attention's lanes, which take a vector's dims in the same shares, one load.  A group's lowest and
// largest take four DPP moves within the row of lanes, and lane i works out the words of one of the key's and
// the value's groups (each lane dividing for itself took 16% longer).  8191 rows of 8 heads of 128 in bf16, which read
// 34 MB and write 10: 20.5 us from launch to launch, bound by vector instructions; two vectors a group of lanes, with more
// loads under way, took 25.7, and 91.6 against 76 for 32768 rows.  The same rows read back take 12 us, 3.6 TB/s.
#include <hip/hip_runtime.h>

#include "jy_device.h"
#include "jy_paged_device.h"

namespace jy {

namespace {

typedef _Float16 h2_t __attribute__((ext_vector_type(2)));

// elements past it make a vector NaN: 16 steps of a group stay finite in fp16
constexpr float kMax4 = 30000.0f;

struct Moved4 {
    jyhip_pages P;
    PageMap M;
    int rows, ps_log2;
    jyhip_vectors k, v;
};

// minimum / maximum over a row of 16 lanes, in each of them
__device__ __forceinline__ float row_min(float v) {
    v = fminf(v, dpp_f<0xB1>(v));
    v = fminf(v, dpp_f<0x4E>(v));
    v = fminf(v, dpp_f<0x124>(v));
    return fminf(v, dpp_f<0x128>(v));
}
__device__ __forceinline__ float row_max(float v) {
    v = fmaxf(v, dpp_f<0xB1>(v));
    v = fmaxf(v, dpp_f<0x4E>(v));
    v = fmaxf(v, dpp_f<0x124>(v));
    return fmaxf(v, dpp_f<0x128>(v));
}

// fp32 rounded to seven significant bits, ties to even
__device__ __forceinline__ float seven_bits(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    return __builtin_bit_cast(float, (u + 0xffffu + ((u >> 17) & 1u)) & ~0x1ffffu);
}

template <int G>
using bytes_t = uint8_t __attribute__((ext_vector_type(G)));

// (one branch around all loads: around each, every one is waited for before the next)
template <class E, int G>
__device__ __forceinline__ void load_pairs(const E* k, const E* v, int hd, bool pairs, float (&x)[2][2 * G]) {
    const int r2 = (threadIdx.x & 15) * 2;
    auto at = [&](int s, int g) {
        const int d = 32 * g + r2;
        return (s ? v : k) + (d < hd ? d : 0);  // (hd is a multiple of 16)
    };
    if (pairs) {
        typedef E two __attribute__((ext_vector_type(2)));
        two y[2][G];
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int g = 0; g < G; g++) y[s][g] = *reinterpret_cast<const two*>(at(s, g));
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int e = 0; e < 2 * G; e++) x[s][e] = (float)y[s][e / 2][e % 2];
    } else {
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int e = 0; e < 2 * G; e++) x[s][e] = (float)at(s, e / 2)[e % 2];
    }
}

// v of lane L of the row
template <int L>
__device__ __forceinline__ float from_lane(float v) {
    return dpp_f<0x150 + L>(v);  // row_newbcast
}

// the numbers of both sides' groups from group I on, by the lows and reciprocal steps that lane I of the row has
template <int G, int I>
__device__ __forceinline__ void numbers(const float (&x)[2][2 * G], float low, float inv, uint8_t (&bytes)[2][G]) {
    if constexpr (I < 2 * G) {
        const float lo = from_lane<I>(low), back = from_lane<I>(inv);
        uint32_t n[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const float y = __builtin_rintf((x[I / G][2 * (I % G) + e] - lo) * back);
            n[e] = (uint32_t)(int)fminf(fmaxf(y, 0.0f), 15.0f);
        }
        bytes[I / G][I % G] = (uint8_t)(n[0] | n[1] << 4);
        numbers<G, I + 1>(x, low, inv, bytes);
    }
}

// Hold the 2 G elements that this lane has of a key (x[0]) and of its value (x[1]) as the vectors at `vec`.  Lane i of
// the row works out the words of group i of the 2 G (the divisions once, not in every lane) and stores them.
template <int G>
__device__ __forceinline__ void hold4(const jyhip_pages& P, int64_t vec, const float (&x)[2][2 * G]) {
    const int r = threadIdx.x & 15, hd = P.head_dim;
    float lo = 0.0f, hi = 0.0f, past[2];
#pragma unroll
    for (int s = 0; s < 2; s++) {
        past[s] = 0.0f;
#pragma unroll
        for (int g = 0; g < G; g++) {
            const bool on = 32 * g + 2 * r < hd;
            const float a = x[s][2 * g], b = x[s][2 * g + 1];
            // (without branches)
            past[s] = on & !((fmaxf(fabsf(a), fabsf(b)) <= kMax4) & (a == a) & (b == b)) ? 1.0f : past[s];
            const float least = row_min(on ? fminf(a, b) : __builtin_inff());
            const float most = row_max(on ? fmaxf(a, b) : -__builtin_inff());
            lo = r == s * G + g ? least : lo;
            hi = r == s * G + g ? most : hi;
        }
        past[s] = row_max(past[s]);
    }
    const bool some = 32 * (r % G) < hd, second = r >= G;  // (lanes from 2 G on: anything)
    const bool bad = (second ? past[1] : past[0]) > 0.0f;  // the whole vector is NaN
    const _Float16 low = some ? (_Float16)lo : (_Float16)0.0f;
    const _Float16 step = some ? (_Float16)seven_bits((hi - (float)low) / 15.0f) : (_Float16)0.0f;
    const float inv = (float)step > 0.0f && !bad ? 1.0f / (float)step : 0.0f;
    const uint32_t word = bad && some ? 0x7e007e00u : __builtin_bit_cast(uint32_t, h2_t{step, low});
    uint8_t bytes[2][G];
    numbers<G, 0>(x, (float)low, inv, bytes);
#pragma unroll
    for (int s = 0; s < 2; s++) {
        bytes_t<G> b;
#pragma unroll
        for (int g = 0; g < G; g++) b[g] = (32 * g + 2 * r < hd) & !(past[s] > 0.0f) ? bytes[s][g] : (uint8_t)0;
        *reinterpret_cast<bytes_t<G>*>(static_cast<uint8_t*>(s ? P.v : P.k) + vec * (16 * G) + r * G) = b;
    }
    if (r < 2 * G) reinterpret_cast<uint32_t*>(second ? P.v_scale : P.k_scale)[vec * G + r % G] = word;
}

template <class E, int G>
__device__ __forceinline__ void give4(const void* pool, const void* scales, int64_t vec, int hd, E* out, bool pairs) {
    const int r = threadIdx.x & 15;
    uint8_t bytes[G] = {};
    uint32_t word[G] = {};
    if (vec >= 0) {
        const auto b = *reinterpret_cast<const bytes_t<G>*>(static_cast<const uint8_t*>(pool) + vec * (16 * G) + r * G);
#pragma unroll
        for (int g = 0; g < G; g++) bytes[g] = b[g];
        constexpr int W = G > 4 ? 4 : G;
        typedef uint32_t words __attribute__((ext_vector_type(W)));
#pragma unroll
        for (int c = 0; c < G; c += W) {
            const words w = *reinterpret_cast<const words*>(static_cast<const uint32_t*>(scales) + vec * G + c);
#pragma unroll
            for (int g = 0; g < W; g++) word[c + g] = w[g];
        }
    }
#pragma unroll
    for (int g = 0; g < G; g++) {
        const int d = 32 * g + 2 * r;
        if (d >= hd) continue;
        const h2_t s = __builtin_bit_cast(h2_t, word[g]);
        // (a number times a step is exact in fp32: one rounding)
        const float a = __builtin_fmaf((float)(bytes[g] & 15), (float)s.x, (float)s.y);
        const float b = __builtin_fmaf((float)(bytes[g] >> 4), (float)s.x, (float)s.y);
        if (pairs) {
            typedef E two __attribute__((ext_vector_type(2)));
            *reinterpret_cast<two*>(out + d) = two{(E)a, (E)b};
        } else {
            out[d] = (E)a;
            out[d + 1] = (E)b;
        }
    }
}

template <class E, int G, bool WRITE>
__global__ __launch_bounds__(256) void paged4_kernel(Moved4 A, bool pairs) {
    const jyhip_pages& P = A.P;
    const unsigned at = blockIdx.x * 16 + (threadIdx.x >> 4), nkv = P.num_kv_heads, total = A.rows * nkv;
    const unsigned i = min(at, total - 1);  // (lanes past the end look at the last vector)
    const int row = (int)(i / nkv), head = (int)(i - row * nkv);
    E* const k = static_cast<E*>(A.k.data) + row * A.k.row_stride + head * A.k.head_stride;
    E* const v = static_cast<E*>(A.v.data) + row * A.v.row_stride + head * A.v.head_stride;
    const int64_t slot = slot_of(A.M, P.num_pages, A.ps_log2, A.M.seq ? A.M.seq[row] : row, A.M.pos[row]);
    const int64_t vec =
        slot < 0 ? -1 : (((slot >> A.ps_log2) * nkv + head) << A.ps_log2) + (slot & ((1 << A.ps_log2) - 1));
    if constexpr (WRITE) {
        float x[2][2 * G];
        load_pairs<E, G>(k, v, P.head_dim, pairs, x);
        if (vec >= 0 && at < total) hold4<G>(P, vec, x);
    } else {
        if (at >= total) return;
        give4<E, G>(P.k, P.k_scale, vec, P.head_dim, k, pairs);
        give4<E, G>(P.v, P.v_scale, vec, P.head_dim, v, pairs);
    }
}

// whether every pair of elements starts at a multiple of its size
bool paired(const jyhip_vectors& x, int type) {
    const long long e = type == JYHIP_T_F32 ? 4 : 2;
    return ((uintptr_t)x.data | (uintptr_t)(x.row_stride * e) | (uintptr_t)(x.head_stride * e)) % (2 * e) == 0;
}

template <class E, bool WRITE>
void launch_groups(const Moved4& A, bool pairs, unsigned grid, hipStream_t st) {
    switch (groups4(A.P.head_dim)) {
        case 2: paged4_kernel<E, 2, WRITE><<<grid, 256, 0, st>>>(A, pairs); break;
        case 4: paged4_kernel<E, 4, WRITE><<<grid, 256, 0, st>>>(A, pairs); break;
        default: paged4_kernel<E, 8, WRITE><<<grid, 256, 0, st>>>(A, pairs);
    }
}

template <bool WRITE>
void launch_moved4(const jyhip_pages& P, const PageMap& M, int rows, const jyhip_vectors& k, const jyhip_vectors& v,
                   int type, hipStream_t st) {
    const Moved4 A{P, M, rows, __builtin_ctz(P.page_size), k, v};
    const bool pairs = paired(k, type) && paired(v, type);
    const unsigned grid = (unsigned)(((int64_t)rows * P.num_kv_heads + 15) / 16);
    if (type == JYHIP_T_F32)
        launch_groups<float, WRITE>(A, pairs, grid, st);
    else if (type == JYHIP_T_F16)
        launch_groups<_Float16, WRITE>(A, pairs, grid, st);
    else
        launch_groups<__bf16, WRITE>(A, pairs, grid, st);
}

}  // namespace

void launch_paged4_write(const jyhip_pages& P, const PageMap& M, int rows, const jyhip_vectors& k,
                         const jyhip_vectors& v, int type, hipStream_t st) {
    launch_moved4<true>(P, M, rows, k, v, type, st);
}

void launch_paged4_read(const jyhip_pages& P, const PageMap& M, int rows, const jyhip_vectors& k,
                        const jyhip_vectors& v, int type, hipStream_t st) {
    launch_moved4<false>(P, M, rows, k, v, type, st);
}

}  // namespace jy
