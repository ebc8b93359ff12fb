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
//        bf16 parts, accumulated in fp32.
//   p.v  o^T = V^T p^T: the weights come out of the first product in the very layout the second
//        takes as its B operand (lane: head l & 15, keys 4 (l >> 4) + i of two 16-key groups), so
//        they change no lane.  V is read row by row, lane l holding DL consecutive dims from
//        (l & 15) DL of its 8 keys, and transposed in registers: output tile t's row r is dim
//        r DL + t, and a byte permute pairs two keys of one dim.  int8 values become fp16 exactly
//        (their bytes read as subnormal halves, one packed fma gives (u - 128) / 512); a weight
//        times its value scale is carried as two fp16 parts (21 bits, relative to the running
//        maximum and to a power of two over the value scales seen), for bf16 values as three
//        bf16 parts.
//
// A workgroup's four waves take the tiles of one chunk of a sequence in turn and join through
// LDS; chunks are joined by a second kernel where there is more than one.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "jy_device.h"
#include "jy_mfma.h"
#include "jy_paged_device.h"

namespace jy {

namespace {

typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));

constexpr float kNone = -3.0e38f;       // the running maximum before any score
constexpr float kLog2e = 1.4426950408889634f;

struct AttnPlan {
    int chunk = 0;   // positions per workgroup, a multiple of 128
    int splits = 1;  // chunks of the longest sequence the launch may see
    int tiles = 1;   // groups of 16 query heads per kv head
};

AttnPlan plan_of(const jyhip_pages& P, int nseq, int nh, int max_len) {
    AttnPlan p;
    p.tiles = (nh / P.num_kv_heads + 15) / 16;
    // chunks small enough that the launch has several workgroups per CU to balance sequences of
    // different lengths, not so small that the joining costs more than it spreads
    const int64_t base = (int64_t)nseq * P.num_kv_heads * p.tiles;
    const int64_t want = std::max<int64_t>(1, (2048 + base - 1) / base);
    const int64_t chunk = (max_len + want - 1) / want;
    p.chunk = (int)std::max<int64_t>(256, (chunk + 127) / 128 * 128);
    p.splits = std::max(1, (max_len + p.chunk - 1) / p.chunk);
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

__device__ __forceinline__ float load_io(const void* p, int64_t i, int type) {
    return type == JYHIP_T_F32   ? static_cast<const float*>(p)[i]
           : type == JYHIP_T_F16 ? (float)static_cast<const _Float16*>(p)[i]
                                 : (float)static_cast<const __bf16*>(p)[i];
}
__device__ __forceinline__ void store_io(void* p, int64_t i, int type, float v) {
    if (type == JYHIP_T_F32)
        static_cast<float*>(p)[i] = v;
    else if (type == JYHIP_T_F16)
        static_cast<_Float16*>(p)[i] = (_Float16)v;
    else
        static_cast<__bf16*>(p)[i] = (__bf16)v;
}

// the top 16 bits of two fp32 values as a pair of bf16 (truncated): a in the low half
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
    return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, a), 0x07060302u);
}
__device__ __forceinline__ float bf16_cut(float a) {
    return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, a) & 0xffff0000u);
}

// The query of 16 heads as B operands of q.k, and the factor that turns their products into
// scores: PARTS operands for each 16 bytes of a key.
template <int PT, int KC>
struct Query;

template <int KC>
struct Query<JYHIP_T_I8, KC> {
    static constexpr int PARTS = 3;
    i4_t q[KC][3];
    __device__ __forceinline__ void load(const float* x, float amax) {  // x: KC x 16 elements of this lane
        const float inv = amax > 0.0f ? 8323072.0f / amax : 0.0f;       // 127 * 65536
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
            s[i] = __builtin_fmaf((float)d[2][i], 65536.0f, __builtin_fmaf((float)d[1][i], 256.0f, (float)d[0][i]));
    }
};

template <int KC>
struct Query<JYHIP_T_F16, KC> {
    h8_t q[KC][2];
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
                q[c][1][e] = (_Float16)(v - (float)hi);
            }
    }
    static __device__ __forceinline__ float factor(float amax) { return __builtin_ldexpf(1.0f, -exponent(amax)); }
    __device__ __forceinline__ void dot(const i4_t (&k)[KC], float (&s)[4]) const {
        f4_t d = {};
#pragma unroll
        for (int p = 1; p >= 0; p--)
#pragma unroll
            for (int c = 0; c < KC; c++)
                d = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, k[c]), q[c][p], d, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; i++) s[i] = d[i];
    }
};

template <int KC>
struct Query<JYHIP_T_BF16, KC> {
    b8_t q[KC][3];
    __device__ __forceinline__ void load(const float* x, float) {
#pragma unroll
        for (int c = 0; c < KC; c++) {
            uint32_t w[3][4];
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                float a = x[c * 8 + e], b = x[c * 8 + e + 1];
#pragma unroll
                for (int p = 0; p < 3; p++) {
                    w[p][e >> 1] = bf16_pair(a, b);
                    a -= bf16_cut(a);
                    b -= bf16_cut(b);
                }
            }
#pragma unroll
            for (int p = 0; p < 3; p++) q[c][p] = __builtin_bit_cast(b8_t, u4_t{w[p][0], w[p][1], w[p][2], w[p][3]});
        }
    }
    static __device__ __forceinline__ float factor(float) { return 1.0f; }
    __device__ __forceinline__ void dot(const i4_t (&k)[KC], float (&s)[4]) const {
        f4_t d = {};
#pragma unroll
        for (int p = 2; p >= 0; p--)
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

template <int PT, int NC>
struct Loader {
    typedef Tile<PT, NC> T;
    static constexpr int ES = T::ES, DL = 4 * NC;
    const char *k, *v;
    const float *ks, *vs;
    unsigned koff[T::KC], voff;
    int64_t head_stride;     // positions between pages of one head: nkv * page_size
    int num_pages, ps, hd;

    __device__ __forceinline__ void load(T& t, int page0, int page1, int key0, int n) const {
#pragma unroll
        for (int g = 0; g < 2; g++) {
            int page = g ? page1 : page0;
            const int at = key0 + 16 * g;
            const bool here = (unsigned)page < (unsigned)num_pages;
            t.live[g] = here ? min(max(n - at, 0), 16) : 0;
            if (!here) page = 0;
            // (positions past the sequence's end are in the page all the same; they are masked)
            const int64_t row = page * head_stride + (at & (ps - 1));
            const char* kr = k + row * (hd * ES);
            const char* vr = v + row * (hd * ES);
#pragma unroll
            for (int c = 0; c < T::KC; c++) t.k[g][c] = *reinterpret_cast<const i4_t*>(kr + koff[c]);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const char* p = vr + voff + (unsigned)(j * hd * ES);
                typedef uint32_t words __attribute__((ext_vector_type(T::VW < 4 ? T::VW : 4)));
                constexpr int PER = T::VW < 4 ? T::VW : 4;
#pragma unroll
                for (int w = 0; w < T::VW / PER; w++) {
                    if constexpr (PER == 1) {
                        t.v[g * 4 + j][w] = reinterpret_cast<const uint32_t*>(p)[w];
                    } else {
                        const words x = reinterpret_cast<const words*>(p)[w];
#pragma unroll
                        for (int i = 0; i < PER; i++) t.v[g * 4 + j][w * PER + i] = x[i];
                    }
                }
            }
            if constexpr (PT == JYHIP_T_I8) {
                const int64_t sr = row + ((threadIdx.x & 63) >> 4) * 4;
                t.ks[g] = *reinterpret_cast<const f4_t*>(ks + sr);
                t.vs[g] = *reinterpret_cast<const f4_t*>(vs + sr);
            }
        }
    }
};

// One head group's state in a wave: output tiles (lane: head l & 15, dim (4 (l >> 4) + i) DL + t),
// running maximum, the lane's part of the sum, and the power of two over the value scales
template <int PT, int NC>
struct State {
    static constexpr int DL = 4 * NC;
    f4_t o[DL] = {};
    float m = kNone, l = 0.0f;
    float vref = 0.0f, vinv = 0.0f;  // int8: o counts in units of vref / 2^15 / 512

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
        if (t.live[0] + t.live[1] < 32) {  // what does not exist: weight 0, whatever its slot holds
#pragma unroll
            for (int g = 0; g < 2; g++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (kg + i >= t.live[g]) {
                        s[g][i] = -__builtin_inff();
                        if constexpr (PT == JYHIP_T_I8) {
                            t.vs[g][i] = 0.0f;
                        } else {
#pragma unroll
                            for (int w = 0; w < Tile<PT, NC>::VW; w++) t.v[g * 4 + i][w] = 0;
                        }
                    }
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
                    // the power of two over vtop, within [2^-120, 2^126]
                    const int e = min(max((int)(__builtin_bit_cast(uint32_t, vtop) >> 23) - 126, -120), 126);
                    const float next = __builtin_ldexpf(1.0f, e);
                    vinv = __builtin_ldexpf(1.0f, -e);
                    a *= vref * vinv;
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
                    p[g * 4 + i] = w * (t.vs[g][i] * vinv) * 32768.0f;
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
                const auto b = __builtin_amdgcn_cvt_pkrtz(p[j] - (float)a[0], p[j + 1] - (float)a[1]);
                hi[j] = (_Float16)a[0];
                hi[j + 1] = (_Float16)a[1];
                lo[j] = (_Float16)b[0];
                lo[j + 1] = (_Float16)b[1];
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

template <int PT, int NC>
__global__ __launch_bounds__(256) void paged_attend_kernel(AttnKernelArgs K) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef Tile<PT, NC> T;
    constexpr int DL = 4 * NC, ES = T::ES, STEP = 16 / ES;
    constexpr int ROW = 64 * NC + 4;
    __shared__ float so[4][16][ROW];
    __shared__ float sm[4][16], sl[4][16];
    const PagedAttn& A = K.A;
    const jyhip_pages& P = A.P;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int hd = P.head_dim, nkv = P.num_kv_heads, per = A.nh / nkv;
    // blocks: chunks fastest, then head groups, kv heads, sequences
    unsigned id = blockIdx.x;
    const int split = id % K.plan.splits;
    id /= K.plan.splits;
    const int tile = id % K.plan.tiles;
    id /= K.plan.tiles;
    const int kvh = id % nkv, b = id / nkv;
    const int n = min(A.lens[b], A.cap);
    const int c0 = split * K.plan.chunk;
    if (c0 >= n && !(split == 0)) return;
    const int end = min(n, c0 + K.plan.chunk);
    const int h0 = kvh * per + tile * 16, heads = min(16, per - tile * 16);

    // the query: this lane's head, its dims of every 16-byte step
    Query<PT, T::KC> q;
    float qf;
    {
        float x[T::KC * STEP];
        float amax = 0.0f;
        bool bad = false;
        const bool on = (lane & 15) < heads;
        const int64_t base = b * A.q.row_stride + (h0 + (on ? lane & 15 : 0)) * A.q.head_stride;
#pragma unroll
        for (int c = 0; c < T::KC; c++)
#pragma unroll
            for (int e = 0; e < STEP; e++) {
                const int d = c * 4 * STEP + (lane >> 4) * STEP + e;
                const float v = on && d < hd ? load_io(A.q.data, base + d, A.type) : 0.0f;
                x[c * STEP + e] = v;
                amax = fmaxf(amax, fabsf(v));
                bad |= !(fabsf(v) <= 3.402823466e38f);
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

    Loader<PT, NC> ld;
    ld.k = static_cast<const char*>(P.k);
    ld.v = static_cast<const char*>(P.v);
    ld.head_stride = (int64_t)nkv * P.page_size;
    ld.num_pages = P.num_pages;
    ld.ps = P.page_size;
    ld.hd = hd;
    const int64_t first = (int64_t)kvh * P.page_size;  // this head's first position in page 0
    ld.k += first * (hd * ES);
    ld.v += first * (hd * ES);
    ld.ks = PT == JYHIP_T_I8 ? P.k_scale + first : nullptr;
    ld.vs = PT == JYHIP_T_I8 ? P.v_scale + first : nullptr;
#pragma unroll
    for (int c = 0; c < T::KC; c++) {
        int d = c * 4 * STEP + (lane >> 4) * STEP;
        if (d >= hd) d = 0;  // (past the head's end the query is zero)
        ld.koff[c] = (unsigned)(((lane & 15) * hd + d) * ES);
    }
    {
        int d = (lane & 15) * DL;
        if (d >= hd) d = 0;  // (outputs past the head's end are not stored)
        ld.voff = (unsigned)(((lane >> 4) * 4 * hd + d) * ES);
    }

    State<PT, NC> st;
    const int ntiles = end > c0 ? (end - c0 + 31) / 32 : 0;
    const int* table = A.M.tables + (int64_t)b * A.M.stride;
    // 64 page ids at a time: lane 2i + g holds the page of group g of the wave's i-th tile
    int ids = -1;
    auto fetch_ids = [&](int t0) {
        const int key = c0 + (t0 + 4 * (lane >> 1)) * 32 + 16 * (lane & 1);
        ids = key < end ? table[key >> K.ps_log2] : -1;
    };
    auto load = [&](T& t, int i, int tl) {
        const int p0 = __builtin_amdgcn_readlane(ids, 2 * i), p1 = __builtin_amdgcn_readlane(ids, 2 * i + 1);
        ld.load(t, p0, p1, c0 + tl * 32, end);
    };
    for (int t0 = wave; t0 < ntiles; t0 += 128) {
        fetch_ids(t0);
        const int cnt = min(32, (ntiles - t0 + 3) / 4);
        T cur, nxt;
        load(cur, 0, t0);
        for (int i = 0; i < cnt; i++) {
            if (i + 1 < cnt) load(nxt, i + 1, t0 + 4 * (i + 1));
            st.add(q, qf, cur);
            cur = nxt;
        }
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
    for (int e = threadIdx.x; e < heads * hd; e += 256) {
        const int r = e / hd, d = e - r * hd;
        const float mx = fmaxf(fmaxf(sm[0][r], sm[1][r]), fmaxf(sm[2][r], sm[3][r]));
        float sum = 0.0f, acc = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float f = State<PT, NC>::exp2_hw(sm[w][r] - mx);
            sum += f * sl[w][r];
            acc += f * so[w][r][d];
        }
        const int64_t row = (int64_t)b * A.nh + h0 + r;
        if (K.plan.splits == 1) {
            store_io(A.out.data, b * A.out.row_stride + (h0 + r) * A.out.head_stride + d, A.type,
                     sum == 0.0f ? 0.0f : acc / sum);
        } else {
            K.part_o[(row * K.plan.splits + split) * hd + d] = acc;
            if (d == 0) K.part_ml[row * K.plan.splits + split] = float2{mx, sum};
        }
    }
#endif
}

// One workgroup per (sequence, query head): the chunks' outputs weighted by 2^(m - max m) over the
// sum of their weighted sums, in the chunks' order.  hd / 4 threads read one chunk's output, the
// others the next ones'.
__global__ __launch_bounds__(256) void paged_join_kernel(AttnKernelArgs K) {
#if defined(__HIP_DEVICE_COMPILE__)
    __shared__ float4 so[256];
    __shared__ float ss[256];
    const PagedAttn& A = K.A;
    const int row = blockIdx.x, b = row / A.nh, h = row % A.nh, hd = A.P.head_dim;
    const int n = min(A.lens[b], A.cap);
    const int live = max(1, (max(n, 0) + K.plan.chunk - 1) / K.plan.chunk);
    const int splits = K.plan.splits;
    const float2* ml = K.part_ml + (int64_t)row * splits;
    const float* po = K.part_o + (int64_t)row * splits * hd;
    float mx = kNone;
    for (int i = threadIdx.x & 63; i < live; i += 64) mx = fmaxf(mx, ml[i].x);
    mx = head_max(mx);
    mx = fmaxf(mx, dpp_f<0xB1>(mx));
    mx = fmaxf(mx, dpp_f<0x4E>(mx));
    mx = fmaxf(mx, dpp_f<0x124>(mx));
    mx = fmaxf(mx, dpp_f<0x128>(mx));
    const int quads = hd / 4, groups = 256 / quads;
    const int gi = threadIdx.x / quads, d4 = threadIdx.x % quads;
    float4 acc = {0, 0, 0, 0};
    float sum = 0.0f;
    if (gi < groups) {
#pragma unroll 4
        for (int i = gi; i < live; i += groups) {
            const float2 x = ml[i];
            const float f = __builtin_amdgcn_exp2f(x.x - mx);
            const float4 o = *reinterpret_cast<const float4*>(po + (int64_t)i * hd + 4 * d4);
            sum += f * x.y;
            acc.x += f * o.x;
            acc.y += f * o.y;
            acc.z += f * o.z;
            acc.w += f * o.w;
        }
    }
    so[threadIdx.x] = acc;
    ss[threadIdx.x] = sum;
    __syncthreads();
    if (gi == 0) {
        for (int w = 1; w < groups; w++) {
            const float4 o = so[w * quads + d4];
            sum += ss[w * quads + d4];
            acc.x += o.x;
            acc.y += o.y;
            acc.z += o.z;
            acc.w += o.w;
        }
        const int64_t at = b * A.out.row_stride + h * A.out.head_stride + 4 * d4;
        const float v[4] = {acc.x, acc.y, acc.z, acc.w};
#pragma unroll
        for (int i = 0; i < 4; i++) store_io(A.out.data, at + i, A.type, sum == 0.0f ? 0.0f : v[i] / sum);
    }
#endif
}

template <int PT>
void launch_nc(const AttnKernelArgs& K, unsigned grid, hipStream_t st) {
    const int hd = K.A.P.head_dim;
    if (hd <= 64)
        paged_attend_kernel<PT, 1><<<grid, 256, 0, st>>>(K);
    else if (hd <= 128)
        paged_attend_kernel<PT, 2><<<grid, 256, 0, st>>>(K);
    else
        paged_attend_kernel<PT, 4><<<grid, 256, 0, st>>>(K);
}

}  // namespace

// (positions past max_len do not exist, so a launch over none still has one chunk: it writes zeros)
size_t paged_attend_part_floats(const jyhip_pages& P, int nseq, int nh, int max_len) {
    const AttnPlan p = plan_of(P, nseq, nh, std::max(max_len, 1));
    return p.splits == 1 ? 0 : (size_t)nseq * nh * p.splits * (P.head_dim + 2);
}

int64_t paged_attend_blocks(const jyhip_pages& P, int nseq, int nh, int max_len) {
    const AttnPlan p = plan_of(P, nseq, nh, std::max(max_len, 1));
    return std::max((int64_t)nseq * P.num_kv_heads * p.tiles * p.splits, (int64_t)nseq * nh);
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
        launch_nc<JYHIP_T_I8>(K, grid, st);
    else if (A.P.type == JYHIP_T_F16)
        launch_nc<JYHIP_T_F16>(K, grid, st);
    else
        launch_nc<JYHIP_T_BF16>(K, grid, st);
    if (K.plan.splits > 1) paged_join_kernel<<<(unsigned)(A.M.nseq * A.nh), 256, 0, st>>>(K);
}

}  // namespace jy
