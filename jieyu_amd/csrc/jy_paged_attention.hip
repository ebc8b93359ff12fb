// jy_paged_attention.hip — attention of one new token per sequence over the paged cache.
//
// out = sum_j p_j v_j, p = softmax of the scores s_j = scale q . k_j, in one pass over the keys
// with a running maximum m and sum l: when m grows, the sum and the output so far shrink by
// 2^(m_old - m_new) (scores in units of log2 e).
//
// Every key and value byte is used once per group of query heads that share them, a dozen
// operations a byte, so memory bounds the kernel: the point is to keep enough bytes in flight and
// the vector unit out of the way.  One wave takes 32 positions at a time for up to 16 query heads
// of one kv head, all in registers, the next 32 positions' loads already issued:
//
//   q.k  keys as the 16 rows (A: lane l holds key l & 15, 16 bytes of it from dim 16 (l >> 4)),
//        heads as the columns.  int8 keys stay int8: the query is split into three base-256
//        digits relative to its largest element (23 bits), each digit's dot an exact int32 on
//        mfma_i32_16x16x64_i8.  fp16 keys take the query as two fp16 parts, bf16 keys as three
//        bf16 parts, accumulated in fp32; so split that an infinite key gives the score that the
//        whole query would.
//   p.v  o^T = V^T p^T: the weights come out of the first product in the very layout the second
//        takes as its B operand (lane: head l & 15, keys 4 (l >> 4) + i of two 16-key groups), so
//        they change no lane.  V is read row by row, lane l holding DL consecutive dims from
//        (l & 15) DL of its 8 keys, and transposed in registers: output tile t's row r is dim
//        r DL + t, and a byte permute pairs two keys of one dim.  int8 values become fp16 exactly
//        (their bytes read as subnormal halves, one packed fma gives (u - 128) / 512); a weight
//        times its value scale is carried as two fp16 parts (21 bits, relative to the running
//        maximum and to a power of two over the value scales seen), for bf16 values as three
//        bf16 parts, none of them 0 beside a first one that is not: 0 times an infinite value is NaN.
//
// A workgroup's four waves take the tiles of one chunk of a sequence in turn and join through
// LDS; chunks are joined by a second kernel where there is more than one.
//
// 64 sequences of 200 to 8190 positions, 32 / 8 heads of 128, bf16 (591 MB): 112 to 160 us from launch to
// launch, half of them within 136 (4.3 TB/s), and 4.8 of join.  One of 32769, 28 / 4 heads, int8 (34.6 MB):
// 12.6 us, of them 5 for the bytes (a wave per SIMD), and 5.2 of join.  32 of 1 to 1500, int8: 14.2 us, the
// chain of the longest chunk, and 3.9.  One of 61 positions, 14 / 2 heads of 64: 4.7 us, the start, one step
// and the end.  fp32 queries cost more than 16-bit ones against 16-bit pools, in products and in registers
// (some spilled from head size 128 on): 48 of 200 to 6000, 32 / 8 heads of 128, both kernels 128 us
// against 89 in bf16, 102 against 89 in fp16.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "jy_device.h"
#include "jy_mfma.h"
#include "jy_paged_device.h"

namespace jy {

namespace {

typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));

constexpr float kNone = -3.402823466e38f;  // the running maximum before any score: at most any finite one
constexpr int kMaxChunk = 4096;          // 64 groups of 16 positions per wave: one lane holds each one's page
constexpr float kLog2e = 1.4426950408889634f;

struct AttnPlan {
    int chunk = 0;   // positions per workgroup, a multiple of 32
    int splits = 1;  // chunks of the longest sequence the launch may see
    int tiles = 1;   // groups of 16 query heads per kv head
};

// The chunk by the launch's upper bound of its lengths (the lengths themselves are on the device).
// A workgroup's own start and end cost about as much as 300 positions, two run on a CU at a time,
// and chunks that one sequence has and another has not are what balances a ragged batch:
//   up to 1024 positions in one piece: no join (32 x 800 positions of int8 12.1 us, in two 13.7)
//   512 at least; 1024 where those still make 768 workgroups (16 x 6000 positions of 8 heads of 128
//   int8 46.3 us against 50.7 with 512; 32 of up to 1500 20.0 us against 18.2, so not there)
//   2048 workgroups where the batch is longer (64 of 200 to 8190 in bf16: 137 us, with half as
//   many 145, with twice as many 135; 16 x 12000 84, 81, 84 us)
AttnPlan plan_of(const jyhip_pages& P, int nseq, int nh, int max_len) {
    AttnPlan p;
    p.tiles = (nh / P.num_kv_heads + 15) / 16;
    const int64_t base = (int64_t)nseq * P.num_kv_heads * p.tiles;
    if (max_len <= 1024) {
        p.chunk = 1024;
        return p;
    }
    const int64_t want = std::max<int64_t>(1, 2048 / base);
    const int64_t least = base * ((max_len + 1023) / 1024) >= 768 ? 1024 : 512;
    const int64_t chunk = std::max<int64_t>(least, ((max_len + want - 1) / want + 31) / 32 * 32);
    p.chunk = (int)std::min<int64_t>(chunk, kMaxChunk);
    p.splits = (max_len + p.chunk - 1) / p.chunk;
    return p;
}

struct AttnKernelArgs {
    PagedAttn A;
    AttnPlan plan;
    int ps_log2;
    float* part_o;   // [nseq][nh][splits][hd]
    float2* part_ml; // [nseq][nh][splits]: running maximum and sum
};

// maximum / sum over the four lanes that hold one head (l, l ^ 16, l ^ 32, l ^ 48)
__device__ __forceinline__ float head_max(float v) {
#if defined(__HIP_DEVICE_COMPILE__)
    const int x = __builtin_bit_cast(int, v);
    const auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    v = fmaxf(__builtin_bit_cast(float, (int)a[0]), __builtin_bit_cast(float, (int)a[1]));
    const int y = __builtin_bit_cast(int, v);
    const auto b = __builtin_amdgcn_permlane16_swap(y, y, false, false);
    v = fmaxf(__builtin_bit_cast(float, (int)b[0]), __builtin_bit_cast(float, (int)b[1]));
#endif
    return v;
}
__device__ __forceinline__ float head_sum(float v) {
#if defined(__HIP_DEVICE_COMPILE__)
    const int x = __builtin_bit_cast(int, v);
    const auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    v = __builtin_bit_cast(float, (int)a[0]) + __builtin_bit_cast(float, (int)a[1]);
    const int y = __builtin_bit_cast(int, v);
    const auto b = __builtin_amdgcn_permlane16_swap(y, y, false, false);
    v = __builtin_bit_cast(float, (int)b[0]) + __builtin_bit_cast(float, (int)b[1]);
#endif
    return v;
}

// this lane's elements of a query row p: STEP from STEP (4 c + lane >> 4) for each c, zeros past hd
// (`on` false: all zeros)
template <class E, int KC, int STEP>
__device__ __forceinline__ void load_query(const E* p, int hd, bool on, float (&x)[KC * STEP]) {
    const int d0 = ((threadIdx.x & 63) >> 4) * STEP;
#pragma unroll
    for (int c = 0; c < KC; c++) {
        const int d = c * 4 * STEP + d0;
        const E* at = p + (d < hd ? d : 0);  // (hd is a multiple of 16)
        E v[STEP];
#pragma unroll
        for (int e = 0; e < STEP; e++) v[e] = at[e];
#pragma unroll
        for (int e = 0; e < STEP; e++) x[c * STEP + e] = on && d < hd ? (float)v[e] : 0.0f;
    }
}
// o / sum as dims d .. d + 3 of the output of head h of sequence b (zeros without any weight)
__device__ __forceinline__ void store_out(const PagedAttn& A, int b, int h, int d, const f4_t& o, float sum) {
    const int64_t at = b * A.out.row_stride + h * A.out.head_stride + d;
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = sum == 0.0f ? 0.0f : o[i] / sum;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (A.type == JYHIP_T_F32)
            static_cast<float*>(A.out.data)[at + i] = v[i];
        else if (A.type == JYHIP_T_F16)
            static_cast<_Float16*>(A.out.data)[at + i] = (_Float16)v[i];
        else
            static_cast<__bf16*>(A.out.data)[at + i] = (__bf16)v[i];
    }
}

// the top 16 bits of two fp32 values as a pair of bf16 (truncated): a in the low half
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
    return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, a), 0x07060302u);
}
__device__ __forceinline__ float bf16_cut(float a) {
    return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, a) & 0xffff0000u);
}

// the smaller / larger of two pairs of 16-bit numbers: of halves or bf16 that are not negative, too.
// The second and third parts of a weight are at least the type's smallest number wherever the first is not
// 0, so that an infinite value times them is that infinity and not NaN.
typedef unsigned short s2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t min16(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(s2_t, a), __builtin_bit_cast(s2_t, b)));
}
__device__ __forceinline__ uint32_t max16(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(s2_t, a), __builtin_bit_cast(s2_t, b)));
}

// The query of 16 heads as B operands of q.k, and the factor that turns their products into
// scores.  Without WIDE one 16-bit operand holds the query (fp16 or bf16 ones against fp16 keys:
// scaled, they lose only what lies 2^-40 below the largest element; bf16 ones against bf16 keys).
template <int PT, int KC, bool WIDE>
struct Query;

template <int KC, bool WIDE>
struct Query<JYHIP_T_I8, KC, WIDE> {
    i4_t q[KC][3];
    __device__ __forceinline__ void load(const float* x, float amax) {  // x: KC x 16 elements of this lane
        // 127 * 65536 over the largest, which is finite from 2^-104 on; a smaller query counts as zeros
        const float inv = amax >= 0x1p-104f ? 8323072.0f / amax : 0.0f;
#pragma unroll
        for (int c = 0; c < KC; c++) {
            uint32_t w[3][4] = {};
#pragma unroll
            for (int e = 0; e < 16; e++) {
                // bytes of value + 0x808080, each less 128: three digits in [-128, 127]
                const uint32_t u = (uint32_t)((int)__builtin_rintf(x[c * 16 + e] * inv) + 0x808080) ^ 0x808080u;
#pragma unroll
                for (int d = 0; d < 3; d++) w[d][e >> 2] |= ((u >> (8 * d)) & 255u) << (8 * (e & 3));
            }
#pragma unroll
            for (int d = 0; d < 3; d++) q[c][d] = i4_t{(int)w[d][0], (int)w[d][1], (int)w[d][2], (int)w[d][3]};
        }
    }
    static __device__ __forceinline__ float factor(float amax) { return amax * (1.0f / 8323072.0f); }
    __device__ __forceinline__ void dot(const i4_t (&k)[KC], float (&s)[4]) const {
        i4_t d[3] = {};
#pragma unroll
        for (int c = 0; c < KC; c++)
#pragma unroll
            for (int p = 0; p < 3; p++) d[p] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[c], q[c][p], d[p], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; i++)
            // (|d| <= 128 * 128 * 256 = 2^22, so the lower two digits add up in 31 bits)
            s[i] = __builtin_fmaf((float)d[2][i], 65536.0f, (float)(d[1][i] * 256 + d[0][i]));
    }
};

template <int KC, bool WIDE>
struct Query<JYHIP_T_F16, KC, WIDE> {
    static constexpr int PARTS = WIDE ? 2 : 1;
    h8_t q[KC][PARTS];
    // scaled by the power of two that puts the largest element in [2^14, 2^15)
    static __device__ __forceinline__ int exponent(float amax) {
        return amax > 0.0f ? 15 - (int)((__builtin_bit_cast(uint32_t, amax) >> 23) - 126) : 0;
    }
    __device__ __forceinline__ void load(const float* x, float amax) {
        const int e2 = exponent(amax);
#pragma unroll
        for (int c = 0; c < KC; c++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float v = __builtin_ldexpf(x[c * 8 + e], e2);
                const _Float16 hi = (_Float16)v;
                q[c][0][e] = hi;
                if constexpr (WIDE) q[c][1][e] = (_Float16)(v - (float)hi);
            }
    }
    static __device__ __forceinline__ float factor(float amax) { return __builtin_ldexpf(1.0f, -exponent(amax)); }
    // An infinite key: the first parts' product says which infinity (or NaN), the second ones', of any sign or
    // 0, have no say.
    __device__ __forceinline__ void dot(const i4_t (&k)[KC], float (&s)[4]) const {
#if defined(__HIP_DEVICE_COMPILE__)
        f4_t d[PARTS] = {};
#pragma unroll
        for (int p = PARTS - 1; p >= 0; p--)
#pragma unroll
            for (int c = 0; c < KC; c++)
                d[p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, k[c]), q[c][p], d[p], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            s[i] = d[0][i];
            if constexpr (WIDE) s[i] += __builtin_amdgcn_fmed3f(d[1][i], -3.402823466e38f, 3.402823466e38f);
        }
#endif
    }
};

template <int KC, bool WIDE>
struct Query<JYHIP_T_BF16, KC, WIDE> {
    static constexpr int PARTS = WIDE ? 3 : 1;
    b8_t q[KC][PARTS];
    __device__ __forceinline__ void load(const float* x, float) {
#pragma unroll
        for (int c = 0; c < KC; c++) {
            uint32_t w[PARTS][4];
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                float a = x[c * 8 + e], b = x[c * 8 + e + 1];
#pragma unroll
                for (int p = 0; p < PARTS; p++) {
                    w[p][e >> 1] = bf16_pair(a, b);
                    a -= bf16_cut(a);
                    b -= bf16_cut(b);
                }
                // parts of one sign, none of them 0 where the first is not: an infinite key times 0 would be NaN
                const uint32_t sign = w[0][e >> 1] & 0x80008000u;
                const uint32_t least = min16(w[0][e >> 1] & 0x7fff7fffu, 0x00800080u) | sign;
#pragma unroll
                for (int p = 1; p < PARTS; p++) w[p][e >> 1] = max16(w[p][e >> 1] | sign, least);
            }
#pragma unroll
            for (int p = 0; p < PARTS; p++) q[c][p] = __builtin_bit_cast(b8_t, u4_t{w[p][0], w[p][1], w[p][2], w[p][3]});
        }
    }
    static __device__ __forceinline__ float factor(float) { return 1.0f; }
    __device__ __forceinline__ void dot(const i4_t (&k)[KC], float (&s)[4]) const {
        f4_t d = {};
#pragma unroll
        for (int p = PARTS - 1; p >= 0; p--)
#pragma unroll
            for (int c = 0; c < KC; c++)
                d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8_t, k[c]), q[c][p], d, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; i++) s[i] = d[i];
    }
};

// 32 positions as a lane holds them: 16 bytes of key (l & 15) of both groups per step of the dot,
// and its dims of 8 values
template <int PT, int NC>
struct Tile {
    static constexpr int ES = PT == JYHIP_T_I8 ? 1 : 2;
    static constexpr int KC = NC * ES;  // 16-byte steps over a key
    static constexpr int VW = NC * ES;  // dwords of a value that a lane holds
    i4_t k[2][KC];
    uint32_t v[8][VW];
    f4_t ks[2], vs[2];
    int live[2];  // positions of each group that exist: the first ones
};

// Loads of 16 positions go through a buffer resource over just those that exist: the ones that do not
// (past the sequence's end, in a hole) read as zeros and are not fetched.  So do the lanes past the
// head's end, at an offset behind any resource: another dim's key in their place, against a query of
// zero, would make NaN of an infinity.
constexpr unsigned kNowhere = 1u << 30;
template <int PT, int NC>
struct Loader {
    typedef Tile<PT, NC> T;
    static constexpr int ES = T::ES, DL = 4 * NC;
    const char *k, *v;       // this head's first position in page 0
    const float *ks, *vs;
    unsigned koff[T::KC], voff[4];
    int64_t page_rows;       // positions (of all heads) per page
    int num_pages, ps, row_bytes;

    __device__ __forceinline__ void load(T& t, int page0, int page1, int key0, int n) const {
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
        for (int g = 0; g < 2; g++) {
            const int page = g ? page1 : page0, at = key0 + 16 * g;
            const bool here = (unsigned)page < (unsigned)num_pages;
            t.live[g] = __builtin_amdgcn_readfirstlane(here ? min(max(n - at, 0), 16) : 0);
            const int64_t row = (here ? page * page_rows : 0) + (at & (ps - 1));
            const auto kr = buffer(k + row * row_bytes, t.live[g] * row_bytes);
            const auto vr = buffer(v + row * row_bytes, t.live[g] * row_bytes);
#pragma unroll
            for (int c = 0; c < T::KC; c++)
                t.k[g][c] = __builtin_bit_cast(i4_t, __builtin_amdgcn_raw_buffer_load_b128(kr, koff[c], 0, 0));
#pragma unroll
            for (int j = 0; j < 4; j++) {
                uint32_t* const d = t.v[g * 4 + j];
                if constexpr (T::VW == 1) {
                    d[0] = __builtin_amdgcn_raw_buffer_load_b32(vr, voff[j], 0, 0);
                } else if constexpr (T::VW == 2) {
                    const i2_t x = __builtin_bit_cast(i2_t, __builtin_amdgcn_raw_buffer_load_b64(vr, voff[j], 0, 0));
                    d[0] = x[0];
                    d[1] = x[1];
                } else {
#pragma unroll
                    for (int w = 0; w < T::VW; w += 4) {
                        const i4_t x = __builtin_bit_cast(i4_t, __builtin_amdgcn_raw_buffer_load_b128(vr, voff[j] + 4 * w, 0, 0));
#pragma unroll
                        for (int i = 0; i < 4; i++) d[w + i] = x[i];
                    }
                }
            }
            if constexpr (PT == JYHIP_T_I8) {
                const unsigned o = ((threadIdx.x & 63) >> 4) * 16;
                t.ks[g] = __builtin_bit_cast(f4_t, __builtin_amdgcn_raw_buffer_load_b128(buffer(ks + row, t.live[g] * 4), o, 0, 0));
                t.vs[g] = __builtin_bit_cast(f4_t, __builtin_amdgcn_raw_buffer_load_b128(buffer(vs + row, t.live[g] * 4), o, 0, 0));
            }
        }
#endif
    }
#if defined(__HIP_DEVICE_COMPILE__)
    static __device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* p, int bytes) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, bytes, 0x00020000);
    }
#endif
};

// One head group's state in a wave: output tiles (lane: head l & 15, dim (4 (l >> 4) + i) DL + t),
// running maximum, the lane's part of the sum, and the power of two over the value scales
template <int PT, int NC>
struct State {
    static constexpr int DL = 4 * NC;
    f4_t o[DL] = {};
    float m = kNone, l = 0.0f;
    float vref = 0.0f, vinv = 0.0f;  // int8: o counts in units of vref / 2^15 * 512; vinv = 2^15 / vref

    template <class Q>
    __device__ __forceinline__ void add(const Q& q, float qf, Tile<PT, NC>& t) {
        const int kg = ((threadIdx.x & 63) >> 4) * 4;  // the lane's first key of each group
        float s[2][4];
#pragma unroll
        for (int g = 0; g < 2; g++) {
            q.dot(t.k[g], s[g]);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                s[g][i] *= qf;
                if constexpr (PT == JYHIP_T_I8) s[g][i] *= t.ks[g][i];
            }
        }
        if (t.live[0] + t.live[1] < 32) {  // no weight for what does not exist (its value and scale are 0)
            asm volatile("");              // (a branch: as selects this would cost every tile)
#pragma unroll
            for (int g = 0; g < 2; g++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (kg + i >= t.live[g]) s[g][i] = -__builtin_inff();
        }
        float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                          fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        float vtop = 0.0f;
        bool grow = top > m;
        if constexpr (PT == JYHIP_T_I8) {
#pragma unroll
            for (int g = 0; g < 2; g++)
#pragma unroll
                for (int i = 0; i < 4; i++) vtop = fmaxf(vtop, fabsf(t.vs[g][i]));
            grow |= vtop > vref;
        }
        if (__any(grow)) {
            const float mn = fmaxf(m, head_max(top));
            float a = exp2_hw(m - mn);
            m = mn;
            l *= a;
            if constexpr (PT == JYHIP_T_I8) {
                vtop = head_max(vtop);
                if (vtop > vref) {  // (the same in every lane)
                    // the power of two over vtop, within [2^-112, 2^126] (2^15 over it has to be finite)
                    const int e = min(max((int)(__builtin_bit_cast(uint32_t, vtop) >> 23) - 126, -112), 126);
                    const float next = __builtin_ldexpf(1.0f, e);
                    vinv = __builtin_ldexpf(1.0f, 15 - e);
                    a *= vref * __builtin_ldexpf(1.0f, -e);
                    vref = next;
                }
            }
#pragma unroll
            for (int d = 0; d < DL; d++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[d][i] *= a;
        }
        float p[8];
        float sum = 0.0f;
#pragma unroll
        for (int g = 0; g < 2; g++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float w = exp2_hw(s[g][i] - m);
                sum += w;
                if constexpr (PT == JYHIP_T_I8)
                    p[g * 4 + i] = w * (t.vs[g][i] * vinv);
                else if constexpr (PT == JYHIP_T_F16)
                    p[g * 4 + i] = w * 32768.0f;
                else
                    p[g * 4 + i] = w;
            }
        l += sum;
        if constexpr (PT == JYHIP_T_BF16) {
            uint32_t w[3][4];
#pragma unroll
            for (int j = 0; j < 8; j += 2)
#pragma unroll
                for (int c = 0; c < 3; c++) {
                    w[c][j >> 1] = bf16_pair(p[j], p[j + 1]);
                    p[j] -= bf16_cut(p[j]);
                    p[j + 1] -= bf16_cut(p[j + 1]);
                    if (c) w[c][j >> 1] = max16(w[c][j >> 1], min16(w[0][j >> 1], 0x00800080u));
                }
            b8_t pb[3];
#pragma unroll
            for (int c = 0; c < 3; c++) pb[c] = __builtin_bit_cast(b8_t, u4_t{w[c][0], w[c][1], w[c][2], w[c][3]});
#pragma unroll
            for (int d = 0; d < DL; d++) {
                const b8_t a = __builtin_bit_cast(b8_t, column16(t, d));
#pragma unroll
                for (int c = 2; c >= 0; c--) o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, pb[c], o[d], 0, 0, 0);
            }
        } else {
            h8_t hi, lo;
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const auto a = __builtin_amdgcn_cvt_pkrtz(p[j], p[j + 1]);
                const auto b = __builtin_amdgcn_cvt_pkrtz(__builtin_fmaf((float)a[0], -1.0f, p[j]),
                                                          __builtin_fmaf((float)a[1], -1.0f, p[j + 1]));
                hi[j] = (_Float16)a[0];
                hi[j + 1] = (_Float16)a[1];
                if constexpr (PT == JYHIP_T_F16) {
                    const uint32_t c = max16(__builtin_bit_cast(uint32_t, b), min16(__builtin_bit_cast(uint32_t, a), 0x00010001u));
                    const h2_t d = __builtin_bit_cast(h2_t, c);
                    lo[j] = d.x;
                    lo[j + 1] = d.y;
                } else {
                    lo[j] = (_Float16)b[0];
                    lo[j + 1] = (_Float16)b[1];
                }
            }
#pragma unroll
            for (int d = 0; d < DL; d++) {
                const h8_t a = PT == JYHIP_T_I8 ? column8(t, d) : __builtin_bit_cast(h8_t, column16(t, d));
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, lo, o[d], 0, 0, 0);
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, hi, o[d], 0, 0, 0);
            }
        }
    }

    // dim d of the lane's 8 keys: 16-bit values
    static __device__ __forceinline__ u4_t column16(const Tile<PT, NC>& t, int d) {
        const uint32_t sel = d & 1 ? 0x07060302u : 0x05040100u;
        u4_t r;
#pragma unroll
        for (int j = 0; j < 4; j++) r[j] = __builtin_amdgcn_perm(t.v[2 * j + 1][d >> 1], t.v[2 * j][d >> 1], sel);
        return r;
    }
    // int8 values as (v) / 512 in fp16: the byte u = v + 128 read as the subnormal half u 2^-24,
    // times 2^15, less 128 / 512
    static __device__ __forceinline__ h8_t column8(const Tile<PT, NC>& t, int d) {
        const uint32_t b = d & 3, sel = b | 0x0c00u | (4 + b) << 16 | 0x0c000000u;
        const h2_t mul = {(_Float16)32768.0f, (_Float16)32768.0f}, off = {(_Float16)-0.25f, (_Float16)-0.25f};
        h8_t r;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t u = __builtin_amdgcn_perm(t.v[2 * j + 1][d >> 2] ^ 0x80808080u, t.v[2 * j][d >> 2] ^ 0x80808080u, sel);
            const h2_t x = __builtin_elementwise_fma(__builtin_bit_cast(h2_t, u), mul, off);
            r[2 * j] = x.x;
            r[2 * j + 1] = x.y;
        }
        return r;
    }

    // what one count of o is worth
    __device__ __forceinline__ float unit() const {
        return PT == JYHIP_T_I8 ? vref * (512.0f / 32768.0f) : PT == JYHIP_T_F16 ? 1.0f / 32768.0f : 1.0f;
    }
    static __device__ __forceinline__ float exp2_hw(float x) {
#if defined(__HIP_DEVICE_COMPILE__)
        return __builtin_amdgcn_exp2f(x);
#else
        return x;
#endif
    }
};

template <int PT, int NC, bool WIDE>
__global__ __launch_bounds__(256, NC <= 2 ? 2 : 1) void paged_attend_kernel(AttnKernelArgs K) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef Tile<PT, NC> T;
    typedef Query<PT, T::KC, WIDE> Q;
    constexpr int DL = 4 * NC, ES = T::ES, STEP = 16 / ES;
    constexpr int ROW = 64 * NC + 4;
    __shared__ float so[4][16][ROW];
    __shared__ float sm[4][16], sl[4][16];
    const PagedAttn& A = K.A;
    const jyhip_pages& P = A.P;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int hd = P.head_dim, nkv = P.num_kv_heads, per = A.nh / nkv;
    // Blocks: heads fastest, then sequences, then chunks.  Blocks go round the XCDs in turn, and
    // short sequences have first chunks alone: with chunks fastest those met on two of the eight.
    unsigned id = blockIdx.x;
    const int hg = id % (nkv * K.plan.tiles);
    id /= nkv * K.plan.tiles;
    const int b = id % A.M.nseq, split = id / A.M.nseq;
    const int kvh = hg / K.plan.tiles, tile = hg % K.plan.tiles;
    const int c0 = split * K.plan.chunk;
    const int h0 = kvh * per + tile * 16, heads = min(16, per - tile * 16);

    // the page of each of the wave's groups of 16 positions: lane 2i + g has that of group g of its
    // i-th tile (past the sequence's end as well: whether a position exists is settled below)
    int ids = -1;
    {
        const int at = (c0 + (wave + 4 * (lane >> 1)) * 32 + 16 * (lane & 1)) >> K.ps_log2;
        if (at < A.M.stride) ids = A.M.tables[(int64_t)b * A.M.stride + at];
    }
    const int n = __builtin_amdgcn_readfirstlane(min(A.lens[b], A.cap));
    const bool on = (lane & 15) < heads;
    const int64_t qbase = b * A.q.row_stride + (h0 + (on ? lane & 15 : 0)) * A.q.head_stride;
    float x[T::KC * STEP];
    if (A.type == JYHIP_T_F32)
        load_query<float, T::KC, STEP>(static_cast<const float*>(A.q.data) + qbase, hd, on, x);
    else if (A.type == JYHIP_T_F16)
        load_query<_Float16, T::KC, STEP>(static_cast<const _Float16*>(A.q.data) + qbase, hd, on, x);
    else
        load_query<__bf16, T::KC, STEP>(static_cast<const __bf16*>(A.q.data) + qbase, hd, on, x);
    if (c0 >= n && split != 0) return;

    Loader<PT, NC> ld;
    const int64_t first = (int64_t)kvh * P.page_size;  // this head's first position in page 0
    ld.k = static_cast<const char*>(P.k) + first * (hd * ES);
    ld.v = static_cast<const char*>(P.v) + first * (hd * ES);
    ld.ks = PT == JYHIP_T_I8 ? P.k_scale + first : nullptr;
    ld.vs = PT == JYHIP_T_I8 ? P.v_scale + first : nullptr;
    ld.page_rows = (int64_t)nkv * P.page_size;
    ld.num_pages = P.num_pages;
    ld.ps = P.page_size;
    ld.row_bytes = hd * ES;
#pragma unroll
    for (int c = 0; c < T::KC; c++) {
        const int d = c * 4 * STEP + (lane >> 4) * STEP;
        // (the first half is inside any head of this form: one register and offsets in the loads)
        const bool in = (NC > 1 && (c + 1) * 4 * STEP <= 32 * NC) || d < hd;
        ld.koff[c] = in ? (unsigned)(((lane & 15) * hd + d) * ES) : kNowhere;
    }
    {
        const int d = (lane & 15) * DL;  // (outputs past the head's end are not stored)
#pragma unroll
        for (int j = 0; j < 4; j++) ld.voff[j] = d < hd ? (unsigned)((((lane >> 4) * 4 + j) * hd + d) * ES) : kNowhere;
    }
    const int end = min(n, c0 + K.plan.chunk);
    const int ntiles = end > c0 ? (end - c0 + 31) / 32 : 0;
    const int cnt = (ntiles - wave + 3) / 4;  // (not positive for a wave without any)
    auto load = [&](T& t, int i) {
        const int p0 = __builtin_amdgcn_readlane(ids, 2 * i), p1 = __builtin_amdgcn_readlane(ids, 2 * i + 1);
        ld.load(t, p0, p1, c0 + (wave + 4 * i) * 32, end);
    };
    T t0, t1;
    if (cnt > 0) load(t0, 0);
    if (cnt > 1) load(t1, 1);

    // the query as operands, while the first positions are on their way
    Q q;
    float qf;
    {
        float amax = 0.0f;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < T::KC * STEP; i++) {
            amax = fmaxf(amax, fabsf(x[i]));
            bad |= !(fabsf(x[i]) <= 3.402823466e38f);
        }
        amax = head_max(amax);
        bad = head_max(bad ? 1.0f : 0.0f) > 0.0f;
        if (bad) {
#pragma unroll
            for (int i = 0; i < T::KC * STEP; i++) x[i] = 0.0f;
            amax = 0.0f;
        }
        q.load(x, amax);
        qf = bad ? __builtin_nanf("") : q.factor(amax) * (A.scale * kLog2e);
    }
    State<PT, NC> st;
    for (int i = 0; i < cnt; i += 2) {
        st.add(q, qf, t0);
        if (i + 1 >= cnt) break;
        if (i + 2 < cnt) load(t0, i + 2);
        st.add(q, qf, t1);
        if (i + 3 < cnt) load(t1, i + 3);
    }

    // join the waves
    st.l = head_sum(st.l);
    const float unit = st.unit();
    const int g = lane & 15;
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int d = 0; d < DL; d++) so[wave][g][((lane >> 4) * 4 + i) * DL + d] = st.o[d][i] * unit;
    if (lane < 16) {
        sm[wave][g] = st.m;
        sl[wave][g] = st.l;
    }
    __syncthreads();
    const int quads = hd / 4;
    for (int e = threadIdx.x; e < heads * quads; e += 256) {
        const int r = e / quads, d = 4 * (e - r * quads);
        float m[4], f[4], sum = 0.0f, mx = kNone;
        f4_t acc = {};
#pragma unroll
        for (int w = 0; w < 4; w++) {
            m[w] = sm[w][r];
            mx = fmaxf(mx, m[w]);
        }
#pragma unroll
        for (int w = 0; w < 4; w++) {
            f[w] = State<PT, NC>::exp2_hw(m[w] - mx);
            sum += f[w] * sl[w][r];
            const f4_t o = *reinterpret_cast<const f4_t*>(&so[w][r][d]);
#pragma unroll
            for (int i = 0; i < 4; i++) acc[i] += f[w] * o[i];
        }
        const int64_t row = (int64_t)b * A.nh + h0 + r;
        if (K.plan.splits == 1) {
            store_out(A, b, h0 + r, d, acc, sum);
        } else {
            *reinterpret_cast<f4_t*>(K.part_o + (row * K.plan.splits + split) * hd + d) = acc;
            if (d == 0) K.part_ml[row * K.plan.splits + split] = float2{mx, sum};
        }
    }
#endif
}

// The join: a (sequence, query head)'s chunks, their outputs weighted by 2^(m - max m) over the sum of
// their weighted sums.  hd / 4 threads take one chunk's output, four consecutive dims each.  A thread
// goes through chunks gi, gi + groups, ... with a running maximum of its own, four read at once, the
// first ones before the sequence's length is known.
struct Joined {
    f4_t acc = {};
    float sum = 0.0f, m = kNone;
    __device__ __forceinline__ void add(float mo, float so, const f4_t& oo) {
#if defined(__HIP_DEVICE_COMPILE__)
        const float mn = fmaxf(m, mo);
        const float a = __builtin_amdgcn_exp2f(m - mn), f = __builtin_amdgcn_exp2f(mo - mn);
        m = mn;
        sum = sum * a + f * so;
#pragma unroll
        for (int c = 0; c < 4; c++) acc[c] = acc[c] * a + f * oo[c];
#endif
    }
    __device__ __forceinline__ void chunks(const AttnKernelArgs& K, int row, int b, int gi, int groups, int d) {
        const int splits = K.plan.splits, hd = K.A.P.head_dim;
        const float2* ml = K.part_ml + (int64_t)row * splits;
        const float* po = K.part_o + (int64_t)row * splits * hd + d;
        float2 x[4];
        f4_t o[4];
        auto read = [&](int i) {  // (those that are live are told apart in use)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int at = min(i + j * groups, splits - 1);
                x[j] = ml[at];
                o[j] = *reinterpret_cast<const f4_t*>(po + (int64_t)at * hd);
            }
        };
        read(gi);
        const int n = min(K.A.lens[b], K.A.cap);
        const int live = max(1, (max(n, 0) + K.plan.chunk - 1) / K.plan.chunk);
        for (int i = gi; i < live; i += 4 * groups) {
            if (i != gi) read(i);
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (i + j * groups < live) add(x[j].x, x[j].y, o[j]);
        }
    }
};

// few chunks: a thread takes all of them, nothing is exchanged
__global__ __launch_bounds__(256) void paged_join_few_kernel(AttnKernelArgs K) {
    const PagedAttn& A = K.A;
    const int quads = A.P.head_dim / 4;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t row = id / quads;
    if (row >= (int64_t)A.M.nseq * A.nh) return;
    const int d = 4 * (int)(id - row * quads), b = (int)(row / A.nh);
    Joined t;
    t.chunks(K, (int)row, b, 0, 1, d);
    store_out(A, b, (int)row - b * A.nh, d, t.acc, t.sum);
}

// many: one workgroup per row, the threads' parts joined through LDS in a fixed order
template <int NT>
__global__ __launch_bounds__(NT) void paged_join_kernel(AttnKernelArgs K) {
    __shared__ f4_t so[NT];
    __shared__ float sm[NT], ss[NT];
    const PagedAttn& A = K.A;
    const int row = blockIdx.x, b = row / A.nh, h = row % A.nh;
    const int quads = A.P.head_dim / 4, groups = NT / quads;
    const int gi = threadIdx.x / quads, d4 = threadIdx.x % quads;
    Joined t;
    if (gi < groups) t.chunks(K, row, b, gi, groups, 4 * d4);
    // rounds: every eighth group's threads take their seven neighbours'
    for (int step = 1; step < groups; step *= 8) {
        so[threadIdx.x] = t.acc;
        sm[threadIdx.x] = t.m;
        ss[threadIdx.x] = t.sum;
        __syncthreads();
        if (gi % (8 * step) == 0)
            for (int w = gi + step; w < min(gi + 8 * step, groups); w += step)
                t.add(sm[w * quads + d4], ss[w * quads + d4], so[w * quads + d4]);
        __syncthreads();
    }
    if (gi == 0) store_out(A, b, h, 4 * d4, t.acc, t.sum);
}

template <int PT, bool WIDE>
void launch_nc(const AttnKernelArgs& K, unsigned grid, hipStream_t st) {
    const int hd = K.A.P.head_dim;
    if (hd <= 64)
        paged_attend_kernel<PT, 1, WIDE><<<grid, 256, 0, st>>>(K);
    else if (hd <= 128)
        paged_attend_kernel<PT, 2, WIDE><<<grid, 256, 0, st>>>(K);
    else
        paged_attend_kernel<PT, 4, WIDE><<<grid, 256, 0, st>>>(K);
}

// WIDE: a query that one 16-bit operand cannot hold (fp32, and fp16 against bf16 keys); the int8
// form's digits hold any
template <int PT>
void launch_wide(const AttnKernelArgs& K, unsigned grid, hipStream_t st) {
    if (PT == JYHIP_T_I8 || K.A.type == JYHIP_T_F32 || (PT == JYHIP_T_BF16 && K.A.type == JYHIP_T_F16))
        launch_nc<PT, true>(K, grid, st);
    else if constexpr (PT != JYHIP_T_I8)
        launch_nc<PT, false>(K, grid, st);
}

}  // namespace

// (positions past max_len do not exist, so a launch over none still has one chunk: it writes zeros)
size_t paged_attend_part_floats(const jyhip_pages& P, int nseq, int nh, int max_len) {
    const AttnPlan p = plan_of(P, nseq, nh, std::max(max_len, 1));
    return p.splits == 1 ? 0 : (size_t)nseq * nh * p.splits * (P.head_dim + 2);
}

int64_t paged_attend_blocks(const jyhip_pages& P, int nseq, int nh, int max_len) {
    const AttnPlan p = plan_of(P, nseq, nh, std::max(max_len, 1));
    return std::max((int64_t)nseq * P.num_kv_heads * p.tiles * p.splits, (int64_t)nseq * nh * 4);
}

void launch_paged_attend(const PagedAttn& A, hipStream_t st) {
    AttnKernelArgs K;
    K.A = A;
    K.plan = plan_of(A.P, A.M.nseq, A.nh, std::max(A.max_len, 1));
    K.ps_log2 = __builtin_ctz(A.P.page_size);
    K.part_o = A.part;
    K.part_ml = reinterpret_cast<float2*>(A.part + (size_t)A.M.nseq * A.nh * K.plan.splits * A.P.head_dim);
    const unsigned grid = (unsigned)((int64_t)A.M.nseq * A.P.num_kv_heads * K.plan.tiles * K.plan.splits);
    if (A.P.type == JYHIP_T_I8)
        launch_wide<JYHIP_T_I8>(K, grid, st);
    else if (A.P.type == JYHIP_T_F16)
        launch_wide<JYHIP_T_F16>(K, grid, st);
    else
        launch_wide<JYHIP_T_BF16>(K, grid, st);
    if (K.plan.splits > 1) {
        // 32 sequences of up to 1500 positions, 32 heads of 128, 3 chunks: both kernels 18.5 us with a
        // workgroup a row, 17.5 us with a thread for four dims.  More chunks: four a thread are read
        // at once, so more threads where those are not all (one sequence of 32000, 14 heads of 64:
        // 11.6 us with 256 threads, 13.2 us with 1024).
        const int quads = A.P.head_dim / 4;
        const int64_t rows = (int64_t)A.M.nseq * A.nh;
        if (K.plan.splits <= 16)
            paged_join_few_kernel<<<(unsigned)((rows * quads + 255) / 256), 256, 0, st>>>(K);
        else if (K.plan.splits * quads <= 4 * 256)
            paged_join_kernel<256><<<(unsigned)rows, 256, 0, st>>>(K);
        else
            paged_join_kernel<1024><<<(unsigned)rows, 1024, 0, st>>>(K);
    }
}

}  // namespace jy
