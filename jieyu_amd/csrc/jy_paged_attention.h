// jy_paged_attention.h — the parts of the paged attention's kernels that run on a wave's registers: the
// query as matrix operands, the loads of 32 positions, and one group of heads' running softmax
// (jy_paged_attention.hip has the mathematics).
#pragma once

#include <hip/hip_runtime.h>

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
template <class ARGS>
__device__ __forceinline__ void store_out(const ARGS& A, int b, int h, int d, const f4_t& o, float sum) {
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

    // KEYS, VALUES: which of the two (a kernel may load them at different times)
    template <bool KEYS = true, bool VALUES = true>
    __device__ __forceinline__ void load(T& t, int page0, int page1, int key0, int n) const {
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
        for (int g = 0; g < 2; g++) {
            const int page = g ? page1 : page0, at = key0 + 16 * g;
            const bool here = (unsigned)page < (unsigned)num_pages;
            const int live = __builtin_amdgcn_readfirstlane(here ? min(max(n - at, 0), 16) : 0);
            const int64_t row = (here ? page * page_rows : 0) + (at & (ps - 1));
            const auto kr = buffer(k + row * row_bytes, live * row_bytes);
            const auto vr = buffer(v + row * row_bytes, live * row_bytes);
            if constexpr (KEYS) {
                t.live[g] = live;
#pragma unroll
                for (int c = 0; c < T::KC; c++)
                    t.k[g][c] = __builtin_bit_cast(i4_t, __builtin_amdgcn_raw_buffer_load_b128(kr, koff[c], 0, 0));
            }
#pragma unroll
            for (int j = 0; j < (VALUES ? 4 : 0); j++) {
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
                if constexpr (KEYS)
                    t.ks[g] = __builtin_bit_cast(f4_t, __builtin_amdgcn_raw_buffer_load_b128(buffer(ks + row, live * 4), o, 0, 0));
                if constexpr (VALUES)
                    t.vs[g] = __builtin_bit_cast(f4_t, __builtin_amdgcn_raw_buffer_load_b128(buffer(vs + row, live * 4), o, 0, 0));
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
        float s[2][4], p[8];
        scores(q, qf, t, s);
        only_live(t, s);
        weights(t, s, p);
        product(t, p, o);
    }

    template <class Q>
    static __device__ __forceinline__ void scores(const Q& q, float qf, const Tile<PT, NC>& t, float (&s)[2][4]) {
#pragma unroll
        for (int g = 0; g < 2; g++) {
            q.dot(t.k[g], s[g]);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                s[g][i] *= qf;
                if constexpr (PT == JYHIP_T_I8) s[g][i] *= t.ks[g][i];
            }
        }
    }

    static __device__ __forceinline__ void only_live(const Tile<PT, NC>& t, float (&s)[2][4]) {
        const int kg = ((threadIdx.x & 63) >> 4) * 4;  // the lane's first key of each group
        if (t.live[0] + t.live[1] < 32) {  // no weight for what does not exist (its value and scale are 0)
            asm volatile("");              // (a branch: as selects this would cost every tile)
#pragma unroll
            for (int g = 0; g < 2; g++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (kg + i >= t.live[g]) s[g][i] = -__builtin_inff();
        }
    }

    // the running maximum and sum with these scores, and the weights as the product takes them
    __device__ __forceinline__ void weights(const Tile<PT, NC>& t, const float (&s)[2][4], float (&p)[8]) {
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
    }

    // o + V^T p^T
    static __device__ __forceinline__ void product(const Tile<PT, NC>& t, float (&p)[8], f4_t (&o)[DL]) {
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

}  // namespace

}  // namespace jy
