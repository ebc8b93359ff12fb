// jy_paged_attention4.h — the parts of jy_paged_attention.h for 4-bit pages.
//
// An element of key j is n step_jg + low_jg in its group g of 32, so
//   q.k_j = sum_g (q_g . n_jg) step_jg + sum_g low_jg (sum of q_g)
// n step has eleven bits (four and seven): the keys' operand holds it exactly in fp16, built from the bytes as
// (1 + n / 16) in the mantissa and one packed fma, (1 + n / 16) 16 step - 16 step.  The second sum is one more
// matrix product over the groups: A the lows, B the query's sums in three fp16 parts.  And
//   sum_j p_j v_jd = sum_j (p_j step_jg) n_jd + sum_j p_j low_jg
// where the numbers' bytes, masked, are subnormal halves that one packed product makes n / 512 (as subnormal operands
// they cost fp32 sums five digits: 4e-5 measured against 1e-7); the weight times the step goes in as one fp16 part
// where queries and outputs are bf16 (at most 2^-11 of a term, of either sign: an eighth of what the outputs' rounding
// leaves, and 79 us against 85 for 64 sequences of 200 to 8190) and as two where they have more digits, relative to a
// power of two over the steps seen; and the second sum is one more product, the groups its rows.
//
// Lane l holds of key l & 15 the bytes of quarter l >> 4 (elements 8 (l >> 4) .. + 7 of every group) and that
// key's words; of its 8 values j the byte of every group for elements 32 g + 2 (l & 15), + 1, and their words.
#pragma once

#include "jy_paged_attention.h"

namespace jy {

namespace {

__device__ __forceinline__ h2_t as_h2(uint32_t w) { return __builtin_bit_cast(h2_t, w); }

// byte `at` of v[0 ..] and byte `at2` as the low bytes of two halves; both constants after unrolling
__device__ __forceinline__ uint32_t two_bytes(const uint32_t* v, int at, int at2) {
    const uint32_t sel = (uint32_t)(at & 3) | 0x0c00u | (uint32_t)(4 + (at2 & 3)) << 16 | 0x0c000000u;
    return __builtin_amdgcn_perm(v[at2 >> 2], v[at >> 2], sel);
}

template <int NC>
struct Tile<JYHIP_T_I4, NC> {
    static constexpr int G = 2 * NC;              // groups
    static constexpr int KC = G, VW = G > 4 ? 2 : 1;
    uint32_t k[2][G];        // 4 G bytes of key l & 15
    uint32_t kw[2][G];       // its words (step, low)
    uint32_t v[8][VW];       // G bytes of each value
    // The words of the 16 values, spread over the wave so that a row of 16 lanes holds those of its four values
    // (4 (l >> 4) + i): word_lane(i, g) has group g's of value i, in vw[.][g / 4] (two groups: lanes 8 .. 15 repeat 0 .. 7).
    static constexpr int VC = G > 4 ? 2 : 1;
    uint32_t vw[2][VC];
    static constexpr __device__ int word_lane(int i, int g) { return G == 2 ? 2 * i + g : 4 * i + (g & 3); }
    // which of the row's values lane l has words of
    static __device__ __forceinline__ int word_value(int lane) { return G == 2 ? lane >> 1 & 3 : lane >> 2 & 3; }
    int live[2];
};

template <int NC>
struct Loader<JYHIP_T_I4, NC> {
    typedef Tile<JYHIP_T_I4, NC> T;
    static constexpr int G = T::G, ROW = 16 * G;
    const char *k, *v, *kw, *vw;
    int64_t page_rows;
    int num_pages, ps;

#if defined(__HIP_DEVICE_COMPILE__)
    template <int N>
    static __device__ __forceinline__ void words(uint32_t* d, __amdgpu_buffer_rsrc_t r, unsigned off) {
        if constexpr (N == 1) {
            d[0] = __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0);
        } else if constexpr (N == 2) {
            const i2_t x = __builtin_bit_cast(i2_t, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0));
            d[0] = x[0];
            d[1] = x[1];
        } else {
#pragma unroll
            for (int w = 0; w < N; w += 4) {
                const i4_t x = __builtin_bit_cast(i4_t, __builtin_amdgcn_raw_buffer_load_b128(r, off + 4 * w, 0, 0));
#pragma unroll
                for (int i = 0; i < 4; i++) d[w + i] = x[i];
            }
        }
    }
#endif

    template <bool KEYS = true, bool VALUES = true>
    __device__ __forceinline__ void load(T& t, int page0, int page1, int key0, int n) const {
#if defined(__HIP_DEVICE_COMPILE__)
        const int lane = threadIdx.x & 63, key = lane & 15, kg = (lane >> 4) * 4;
#pragma unroll
        for (int g = 0; g < 2; g++) {
            const int page = g ? page1 : page0, at = key0 + 16 * g;
            const bool here = (unsigned)page < (unsigned)num_pages;
            const int live = __builtin_amdgcn_readfirstlane(here ? min(max(n - at, 0), 16) : 0);
            const int64_t row = (here ? page * page_rows : 0) + (at & (ps - 1));
            if constexpr (KEYS) {
                t.live[g] = live;
                words<G>(t.k[g], buffer(k + row * ROW, live * ROW), (unsigned)(key * ROW + kg * G));
                words<G>(t.kw[g], buffer(kw + row * (4 * G), live * (4 * G)), (unsigned)(key * 4 * G));
            }
            if constexpr (VALUES) {
                const auto vr = buffer(v + row * ROW, live * ROW), vwr = buffer(vw + row * (4 * G), live * (4 * G));
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const unsigned off = (unsigned)(kg * ROW + key * G) + j * ROW;
                    if constexpr (G == 2)
                        t.v[g * 4 + j][0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(vr, off, 0, 0);
                    else
                        words<T::VW>(t.v[g * 4 + j], vr, off);
                }
#pragma unroll
                for (int c = 0; c < T::VC; c++)
                    words<1>(&t.vw[g][c], vwr, (unsigned)(((kg + T::word_value(lane)) * G + (G == 2 ? key & 1 : key & 3) + 4 * c) * 4));
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

// the order of a lane's 8 elements of a group, as the operand's halves hold them
__device__ __forceinline__ constexpr int order4(int e) { return (e & 4) + (e & 1) * 2 + ((e >> 1) & 1); }

// the lane's elements of a query row: 8 from 32 g + 8 (lane >> 4) for each group, zeros past hd
template <class E, int G>
__device__ __forceinline__ void load_query4(const E* p, int hd, bool on, float (&x)[8 * G]) {
    const int d0 = ((threadIdx.x & 63) >> 4) * 8;
#pragma unroll
    for (int g = 0; g < G; g++) {
        const int d = 32 * g + d0;
        const E* at = p + (d < hd ? d : 0);  // (hd is a multiple of 16)
        E v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = at[e];
#pragma unroll
        for (int e = 0; e < 8; e++) x[8 * g + e] = on && d < hd ? (float)v[order4(e)] : 0.0f;
    }
}

template <int KC, bool WIDE>
struct Query<JYHIP_T_I4, KC, WIDE> {
    static constexpr int G = KC, PARTS = WIDE ? 2 : 1;
    h8_t q[G][PARTS];
    h8_t sums;  // of the groups, in three parts: lane quarter p holds part p
    // scaled by the power of two that puts the largest element in [2^8, 2^9): a group's sum stays under 2^14
    static __device__ __forceinline__ int exponent(float amax) {
        return amax > 0.0f ? 9 - (int)((__builtin_bit_cast(uint32_t, amax) >> 23) - 126) : 0;
    }
    __device__ __forceinline__ void load(const float* x, float amax) {
        const int e2 = exponent(amax), quarter = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int e = 0; e < 8; e++) sums[e] = (_Float16)0.0f;
#pragma unroll
        for (int g = 0; g < G; g++) {
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float v = __builtin_ldexpf(x[8 * g + e], e2);
                const _Float16 hi = (_Float16)v;
                q[g][0][e] = hi;
                if constexpr (WIDE) q[g][1][e] = (_Float16)(v - (float)hi);
                sum += v;
            }
            sum = head_sum(sum);
            asm volatile("" : "+v"(sum));  // (its parts are those of the rounded sum)
            const _Float16 a = (_Float16)sum, b = (_Float16)(sum - (float)a), c = (_Float16)(sum - (float)a - (float)b);
            sums[g] = quarter == 0 ? a : quarter == 1 ? b : quarter == 2 ? c : (_Float16)0.0f;
        }
    }
    static __device__ __forceinline__ float factor(float amax) { return __builtin_ldexpf(1.0f, -exponent(amax)); }

    __device__ __forceinline__ void dot(const uint32_t (&k)[G], const uint32_t (&kw)[G], float (&s)[4]) const {
#if defined(__HIP_DEVICE_COMPILE__)
        uint32_t w[4] = {};
#pragma unroll
        for (int g = 0; g < G; g += 2) w[g / 2] = __builtin_amdgcn_perm(kw[g + 1], kw[g], 0x07060302u);  // the lows
        f4_t d = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, i4_t{(int)w[0], (int)w[1], (int)w[2], (int)w[3]}),
                                                        sums, f4_t{}, 0, 0, 0);
#pragma unroll
        for (int g = 0; g < G; g++) {
            const _Float16 s1 = as_h2(kw[g]).x * (_Float16)16.0f;
            const h2_t s16 = {s1, s1};
            uint32_t a[4];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const uint32_t b = two_bytes(k, 2 * j * G + g, (2 * j + 1) * G + g);
                const uint32_t lo = (b & 0x000f000fu) << 6 | 0x3c003c00u, hi = (b & 0x00f000f0u) << 2 | 0x3c003c00u;
                a[2 * j] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(as_h2(lo), s16, -s16));
                a[2 * j + 1] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(as_h2(hi), s16, -s16));
            }
            const h8_t A = __builtin_bit_cast(h8_t, i4_t{(int)a[0], (int)a[1], (int)a[2], (int)a[3]});
#pragma unroll
            for (int p = PARTS - 1; p >= 0; p--) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(A, q[g][p], d, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) s[i] = d[i];
#endif
    }
};

// One head group's state over 4-bit pages: output tile 2 g + e holds elements 32 g + 2 r + e in row r
template <int NC, bool WIDE>
struct State4 {
    static constexpr int G = 2 * NC, DL = 2 * G;
    typedef Tile<JYHIP_T_I4, NC> T;
    f4_t o[DL] = {};
    f4_t low = {};  // row g (as in o): 2^15 sum p low of group g
    float m = kNone, l = 0.0f;
    float vref = 0.0f, vinv = 0.0f;  // o counts in units of vref / 2^15 * 2^9; vinv = 2^15 / vref

    template <class Q>
    static __device__ __forceinline__ void scores(const Q& q, float qf, const T& t, float (&s)[2][4]) {
#pragma unroll
        for (int g = 0; g < 2; g++) {
            q.dot(t.k[g], t.kw[g], s[g]);
#pragma unroll
            for (int i = 0; i < 4; i++) s[g][i] *= qf;
        }
    }

    __device__ __forceinline__ void weights(const T& t, const float (&s)[2][4], float (&p)[8]) {
        float most = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                           fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        float step = 0.0f;  // the largest this lane holds
#pragma unroll
        for (int g = 0; g < 2; g++)
#pragma unroll
            for (int i = 0; i < T::VC; i++) step = fmaxf(step, fabsf((float)as_h2(t.vw[g][i]).x));
        if (__any(most > m || step > vref)) {
            const float mn = fmaxf(m, head_max(most));
            float a = exp2_hw(m - mn);
            m = mn;
            l *= a;
#pragma unroll
            for (int i = 0; i < 4; i++) low[i] *= a;
            step = wave_max64(step);
            if (step > vref) {  // (the same in every lane)
                const int e = min((int)(__builtin_bit_cast(uint32_t, step) >> 23) - 126, 100);
                vinv = __builtin_ldexpf(1.0f, 15 - e);
                a *= vref * __builtin_ldexpf(1.0f, -e);
                vref = __builtin_ldexpf(1.0f, e);
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
                p[g * 4 + i] = exp2_hw(s[g][i] - m);
                sum += p[g * 4 + i];
            }
        l += sum;
    }

    // 8 numbers as one or two fp16 parts.  (Two are cut, not rounded: a conversion that the compiler joins with the
    // product that made the number rounds once where the remainder takes it as rounded twice.)
    static __device__ __forceinline__ void parts(const float (&w)[8], h8_t& hi, h8_t& lo) {
        if constexpr (WIDE) {
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const auto a = __builtin_amdgcn_cvt_pkrtz(w[j], w[j + 1]);
                const auto b = __builtin_amdgcn_cvt_pkrtz(w[j] - (float)a[0], w[j + 1] - (float)a[1]);
                hi[j] = (_Float16)a[0];
                hi[j + 1] = (_Float16)a[1];
                lo[j] = (_Float16)b[0];
                lo[j + 1] = (_Float16)b[1];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) hi[j] = (_Float16)w[j];
        }
    }

    // Where some words are not finite in a tile that not all columns see whole: they count as zeros, and the columns
    // that see them (`out`: which of its 8 positions this lane's does not) become NaN in all their dims, as such a vector is.
    __device__ __forceinline__ void take_infinite(T& t, uint32_t out) {
#if defined(__HIP_DEVICE_COMPILE__)
        const int lane = threadIdx.x & 63;
        bool hit = false;
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int c = 0; c < T::VC; c++) {
                const h2_t x = as_h2(t.vw[h][c]);
                const bool is = !(fabsf((float)x.x) <= 65504.0f) || !(fabsf((float)x.y) <= 65504.0f);
                const uint32_t row = (uint32_t)(__ballot(is) >> (lane & 48)) & 0xffffu;
                t.vw[h][c] = is ? 0u : t.vw[h][c];
#pragma unroll
                for (int i = 0; i < 4; i++)
                    hit |= !(out >> (4 * h + i) & 1u) && (row & (G == 2 ? 0x0303u << (2 * i) : 0xfu << (4 * i))) != 0;
            }
        if (head_max(hit ? 1.0f : 0.0f) > 0.0f)
#pragma unroll
            for (int d = 0; d < DL; d++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[d][i] = __builtin_nanf("");
#endif
    }

    // o and low with these weights
    __device__ __forceinline__ void product(const T& t, const float (&p)[8]) {
#if defined(__HIP_DEVICE_COMPILE__)
        // The lows: one product of the groups (its rows) by the weights.  Lane r of a row takes group r's words of the
        // row's values by rotations.
        {
            uint32_t x[8];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                x[4 * h] = first<0>(t.vw[h]);
                x[4 * h + 1] = first<1>(t.vw[h]);
                x[4 * h + 2] = first<2>(t.vw[h]);
                x[4 * h + 3] = first<3>(t.vw[h]);
            }
            i4_t A;
#pragma unroll
            for (int j = 0; j < 4; j++) A[j] = (int)__builtin_amdgcn_perm(x[2 * j + 1], x[2 * j], 0x07060302u);
            float w[8];
#pragma unroll
            for (int j = 0; j < 8; j++) w[j] = p[j] * 32768.0f;
            h8_t hi, lo;
            parts(w, hi, lo);
            if constexpr (WIDE) low = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, A), lo, low, 0, 0, 0);
            low = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, A), hi, low, 0, 0, 0);
        }
        // the steps in the product's units; a lane takes each from the one that has it, by a move within its row that
        // the multiplication does itself
        float steps[2][T::VC];
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < T::VC; i++) steps[h][i] = (float)as_h2(t.vw[h][i]).x * vinv;
#pragma unroll
        for (int g = 0; g < G; g++) {
            float w[8];
            values<0>(w, p, steps, g);
            h8_t hi, lo;
            parts(w, hi, lo);
            uint32_t b[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if constexpr (G > 4) {
                    const uint32_t x = t.v[2 * j][g >> 2], y = t.v[2 * j + 1][g >> 2], c = g & 3;
                    b[j] = __builtin_amdgcn_perm(y, x, c | 0x0c00u | (4 + c) << 16 | 0x0c000000u);
                } else {
                    const uint32_t c = g;
                    b[j] = __builtin_amdgcn_perm(t.v[2 * j + 1][0], t.v[2 * j][0], c | 0x0c00u | (4 + c) << 16 | 0x0c000000u);
                }
            }
#pragma unroll
            for (int e = 0; e < 2; e++) {
                // n 2^-24 (an odd element's 16 n 2^-24) as subnormal halves, to n 2^-9
                const uint32_t mask = e ? 0x00f000f0u : 0x000f000fu;
                const h2_t up = e ? h2_t{(_Float16)2048.0f, (_Float16)2048.0f} : h2_t{(_Float16)32768.0f, (_Float16)32768.0f};
                uint32_t a[4];
#pragma unroll
                for (int j = 0; j < 4; j++) a[j] = __builtin_bit_cast(uint32_t, as_h2(b[j] & mask) * up);
                const h8_t A = __builtin_bit_cast(h8_t, i4_t{(int)a[0], (int)a[1], (int)a[2], (int)a[3]});
                if constexpr (WIDE) o[2 * g + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A, lo, o[2 * g + e], 0, 0, 0);
                o[2 * g + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A, hi, o[2 * g + e], 0, 0, 0);
            }
        }
#endif
    }

    // lane r of a row: the word of group r of the row's value I (other lanes past the last group: anything)
    template <int I>
    static __device__ __forceinline__ uint32_t first(const uint32_t (&vw)[T::VC]) {
        constexpr int by = T::word_lane(I, 0), back = (16 - by) & 15;  // row_ror by 16 - n brings lane r + n's to lane r
        uint32_t x = rotated<back>(vw[0]);
        if constexpr (T::VC > 1) {
            const uint32_t y = rotated<(back + 4) & 15>(vw[1]);  // (moved by all lanes, those that have the word among them)
            x = (threadIdx.x & 15) < 4 ? x : y;
        }
        return x;
    }
    template <int N>
    static __device__ __forceinline__ uint32_t rotated(uint32_t v) {
        if constexpr (N == 0)
            return v;
        else
            return __builtin_bit_cast(uint32_t, dpp_f<0x120 + N>(__builtin_bit_cast(float, v)));
    }

    // w[J ..]: the weights times the steps of group g
    template <int J>
    __device__ __forceinline__ void values(float (&w)[8], const float (&p)[8], const float (&steps)[2][T::VC], int g) {
        if constexpr (J < 8) {
            switch (g) {
                case 0: value<J, 0>(w, p, steps); break;
                case 1: value<J, 1>(w, p, steps); break;
                case 2: value<J, 2>(w, p, steps); break;
                case 3: value<J, 3>(w, p, steps); break;
                case 4: value<J, 4>(w, p, steps); break;
                case 5: value<J, 5>(w, p, steps); break;
                case 6: value<J, 6>(w, p, steps); break;
                default: value<J, 7>(w, p, steps);
            }
            values<J + 1>(w, p, steps, g);
        }
    }
    template <int J, int GR>
    __device__ __forceinline__ void value(float (&w)[8], const float (&p)[8], const float (&steps)[2][T::VC]) {
        if constexpr (GR < G) w[J] = dpp_f<0x150 + T::word_lane(J & 3, GR)>(steps[J >> 2][GR / 4]) * p[J];  // row_newbcast
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
