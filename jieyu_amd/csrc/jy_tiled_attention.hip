// jy_tiled_attention.hip — attention of long runs of 16-bit rows (prompts) over the paged cache, under the rules of
// jy_ruled_attention.hip.
//
// A workgroup's four waves take 128 columns, (row, query head) pairs of one kv head, 32 a wave, and go through
// the keys 64 at a time with a running maximum and sum (the maximum moves only when it grows by 2^6, so that few
// tiles rescale).  Both products on the matrix unit, 32 x 32 x 16:
//
//   s^T = K q^T   A: 32 keys from LDS, 8 elements a lane; B: the wave's queries, in registers throughout
//   o^T = V^T p^T a lane's scores are those of one column for keys 8 b + 4 h + i (h the lane's half), which is a B
//                 operand of 16 keys as they lie; A: V's columns, read from LDS transposed (ds_read_b64_tr_b16)
//
// so scores and outputs of a column never leave their lanes, and its maximum and sum take one exchange between
// the two halves of the wave.  Keys and values are staged in LDS as 16-bit numbers, the chunks of a row exchanged
// by its key's low bits against bank conflicts, in two buffers: the next tile's loads are under way while one
// is worked on, with one barrier a tile.
//
// Number types: fp16 and bf16 pages as they are, queries of the other type as fp16 by a power of two (bf16 queries) or
// in two bf16 parts (fp16 ones).  int8 pages: the whole numbers, exact in 16 bits; a key's scale multiplies its
// scores, a value's its weight, which is carried in bf16 (in two parts for fp16 outputs).  4-bit pages: a key's
// number times step, exact in fp16, its low by one more product with the query's sums over the groups; a value
// rounded to fp16, once more than its outputs are.  A weight is rounded to the product's 16 bits, and the sum adds up
// what was rounded (over int8 values the weights themselves), so that only the roundings' differences are left: for bf16
// outputs bf16 weights are off 2.1e-3 of the largest output from the formula in 64 bits where the outputs' own rounding
// alone leaves 1.6e-3.  Two bf16 parts leave 1.6e-3 and take 1111 us for 850 (the prompt below).
//
// What a row does not see has to leave it alone even where its values are not finite (0 times that is NaN).
// Positions that no row of the workgroup sees are staged as zeros.  Where some rows see a tile whole and others do not
// (on the diagonal) and a value in it is not finite, the workgroup starts again row by row, staging what each sees.
//
// A prompt of 8191 rows, 32 heads over 8 of 128, bf16, cap 30: 840 to 890 us from card to card, 620 to 655 TFLOP/s (a
// large product: 1335); over int8 without a cap 767.  A tile is 1024 cycles of matrix instructions a wave and 1950 of
// vector ones (15 a score with a cap), each wave reads all of it from LDS, and only the two workgroups of a CU cover
// each other.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "jy_paged_attention.h"
#include "jy_ruled.h"

namespace jy {

namespace {

typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
typedef short s4_t __attribute__((ext_vector_type(4)));

constexpr int NT = 256, COLS = 128, BN = 64;  // threads, columns, keys of a tile

__device__ __forceinline__ float exp2_hw(float x) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_exp2f(x);
#else
    return x;
#endif
}
// over the two lanes of a column (l, l ^ 32)
__device__ __forceinline__ float half_max(float v) {
#if defined(__HIP_DEVICE_COMPILE__)
    const int x = __builtin_bit_cast(int, v);
    const auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return fmaxf(__builtin_bit_cast(float, (int)a[0]), __builtin_bit_cast(float, (int)a[1]));
#else
    return v;
#endif
}
__device__ __forceinline__ float half_sum(float v) {
#if defined(__HIP_DEVICE_COMPILE__)
    const int x = __builtin_bit_cast(int, v);
    const auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return __builtin_bit_cast(float, (int)a[0]) + __builtin_bit_cast(float, (int)a[1]);
#else
    return v;
#endif
}

// 16-bit numbers of a product: what they are and the product itself
template <bool BF>
struct Half;
template <>
struct Half<false> {
    typedef _Float16 E;
    typedef h8_t V;
    static __device__ __forceinline__ f16_t mul(const u4_t& a, const u4_t& b, const f16_t& c) {
#if defined(__HIP_DEVICE_COMPILE__)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
#else
        return c;
#endif
    }
    // both numbers of a word added to l
    static __device__ __forceinline__ float both(uint32_t w, float l) {
#if defined(__HIP_DEVICE_COMPILE__)
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2_t, w), h2_t{(_Float16)1.0f, (_Float16)1.0f}, l, false);
#else
        return l;
#endif
    }
};
template <>
struct Half<true> {
    typedef __bf16 E;
    typedef b8_t V;
    static __device__ __forceinline__ f16_t mul(const u4_t& a, const u4_t& b, const f16_t& c) {
#if defined(__HIP_DEVICE_COMPILE__)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, b), c, 0, 0, 0);
#else
        return c;
#endif
    }
    static __device__ __forceinline__ float both(uint32_t w, float l) {
#if defined(__HIP_DEVICE_COMPILE__)
        typedef __bf16 b2_t __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2_t, w), b2_t{(__bf16)1.0f, (__bf16)1.0f}, l, false);
#else
        return l;
#endif
    }
};

// 8 numbers as two bf16 each, of one sign, the second not 0 where the first is not: an infinity times both is
// that infinity
template <bool SIGNED>
__device__ __forceinline__ void two_parts(const float (&x)[8], u4_t& a, u4_t& b) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const uint32_t hi = bf16_pair(x[e], x[e + 1]);
        const uint32_t lo = bf16_pair(x[e] - bf16_cut(x[e]), x[e + 1] - bf16_cut(x[e + 1]));
        const uint32_t sign = SIGNED ? hi & 0x80008000u : 0u;
        a[e >> 1] = hi;
        b[e >> 1] = max16(lo | sign, min16(hi & 0x7fff7fffu, 0x00800080u) | sign);
    }
}

// PT: the pages' type, HDT: 64 HDT elements hold a head, BIO: bf16 queries and outputs, else fp16
template <int PT, int HDT, bool BIO>
struct Form {
    static constexpr bool I8 = PT == JYHIP_T_I8, I4 = PT == JYHIP_T_I4, F16 = PT == JYHIP_T_F16, BF = PT == JYHIP_T_BF16;
    static constexpr bool KBF = BF || (I8 && BIO);             // the first product in bf16
    static constexpr bool VBF = BF || I8;                      // the second
    static constexpr int QP = BF && !BIO ? 2 : 1;              // parts of a query
    static constexpr int PP = (BF || I8) && !BIO ? 2 : 1;      // of a weight
    static constexpr bool SCALED = (F16 && BIO) || I4;         // queries by a power of two
    // Weights, at most 2^6 as the maximum moves late, by this power of two more, in outputs and sums alike: fp16 ones then
    // reach 2^15, and lose digits only from 2^-23 of the largest down; bf16 ones reach 1, so that they times a value stay
    // finite where the value is.
    static constexpr float LIFT = VBF ? -6.0f : 9.0f;
    static constexpr int HD = 64 * HDT, ROW = 2 * HD;          // elements and bytes of a staged row
    static constexpr int MASK = HDT == 1 ? 7 : 15;             // of a key's bits that move its chunks of 16 bytes
    static constexpr int G = HDT == 1 ? 2 : HDT == 2 ? 4 : 8;  // groups of a 4-bit vector
    static constexpr int STEPS = HD / 16, DT = HD / 32;        // steps of the first product, tiles of outputs
    static constexpr int BYTES = I8 ? HD : I4 ? 16 * G : 2 * HD;  // of a vector in its page, at most
    // where a chunk of key `key`'s values lies in its row: pairs of chunks side by side, those of 4 neighbouring keys apart
    static __host__ __device__ __forceinline__ constexpr int vchunk(int key, int chunk) { return chunk ^ (2 * key & MASK); }
    // what a thread brings of a tile's keys (and as much of its values), in 16-byte units (4 bits: a key's quarter)
    static constexpr int UNITS = I4 ? (G + 3) / 4 : BN * (BYTES / 16) / NT;
};

template <class F>
struct Staged {
    u4_t k[F::UNITS], v[F::UNITS];
    u4_t kw[F::I4 ? (F::G + 3) / 4 : 1], vw[F::I4 ? (F::G + 3) / 4 : 1];
    float ks, vs;  // int8: lane l < 16 of wave w has those of key 16 w + l
};

template <class F>
struct Shared {
    uint32_t k[2][BN * F::ROW / 4], v[2][BN * F::ROW / 4];
    _Float16 low[2][F::I4 ? BN : 1][8];
    float ks[2][F::I8 ? BN : 4], vs[2][F::I8 ? BN : 4];
    int bound[4][4];
    int odd[2];  // a value that is not finite in a tile that only some see whole
};

__device__ __forceinline__ bool infinite16(uint32_t w, bool bf) {
    const uint32_t e = bf ? 0x7f80u : 0x7c00u;
    return (w & e) == e || (w >> 16 & e) == e;
}

// FINE: tanh to 8 steps of itself.  1 - 2 / (e^2y + 1) cancels at small y and is off by 4 steps of 1, so scores under a cap c
// by c 2^-22: up to caps of 64 that is 2e-5 of a weight.  As a branch of one kernel the other form made those that do not
// take it 2 to 3% slower (slopes without a cap 849 -> 873 us, the prompt above).
constexpr float kFineCap = 64.0f;
template <int PT, int HDT, bool BIO, bool FINE>
__global__ __launch_bounds__(NT, HDT <= 2 ? 2 : 1) void tiled_attend_kernel(Ruled K) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef Form<PT, HDT, BIO> F;
    typedef Half<F::KBF> HK;
    typedef Half<F::VBF> HV;
    typedef typename Half<BIO>::E IO;
    typedef typename Half<BIO>::V vec8;
    typedef IO vec4 __attribute__((ext_vector_type(4)));
    __shared__ Shared<F> sh;
    const RuledAttn& A = K.A;
    const jyhip_pages& P = A.P;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int half = lane >> 5, hd = P.head_dim, nkv = P.num_kv_heads, per = A.nh / nkv;
    unsigned id = blockIdx.x;
    const int hg = id % (nkv * K.tiles);
    id /= nkv * K.tiles;
    const int at = id % K.groups, split = id / K.groups;
    const int kvh = hg / K.tiles, tile = hg % K.tiles;
    const int h0 = kvh * per + tile * K.hpg, heads = min(K.hpg, per - tile * K.hpg);
    const Run run = run_of(K, K.groups - 1 - at);  // the last rows of a run see most: first
    if (run.seq < 0) return;
    const int rows = min(K.rpg, run.end - run.row0);

    // this lane's column
    const int col = 32 * wave + (lane & 31), crow = col / K.hpg, chead = col - crow * K.hpg;
    const bool on = crow < rows && chead < heads;
    const int row = run.row0 + (on ? crow : 0), head = h0 + (on ? chead : 0);
    const int pos = A.pos[row];
    const int lo = A.first ? max(A.first[row], 0) : 0;
    const int hi = min(A.last ? A.last[row] : min(pos, A.cap) + 1, A.cap);
    const bool sees = on && hi > lo;
    // bounds of the wave's columns: what any sees, and what all that see anything see
    auto wave_min = [](int v) {
        v = cols_min(v);
        return min(min(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
                   min(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
    };
    const int w_from = wave_min(sees ? lo : 0x7fffffff), w_to = -wave_min(sees ? -hi : 0);
    const int w_all_lo = -wave_min(sees ? -lo : 0), w_all_hi = wave_min(sees ? hi : 0x7fffffff);
    if (lane < 4) sh.bound[wave][lane] = lane == 0 ? w_from : lane == 1 ? w_to : lane == 2 ? w_all_lo : w_all_hi;
    if (tid < 2) sh.odd[tid] = 0;
    __syncthreads();
    int from = 0x7fffffff, to = 0, all_lo = 0, all_hi = 0x7fffffff;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        from = min(from, sh.bound[w][0]);
        to = max(to, sh.bound[w][1]);
        all_lo = max(all_lo, sh.bound[w][2]);
        all_hi = min(all_hi, sh.bound[w][3]);
    }
    from = __builtin_amdgcn_readfirstlane(from);
    to = __builtin_amdgcn_readfirstlane(to);
    const int base = to > 0 ? from & ~31 : 0;
    // (both up to 2^30: their sum may pass 2^31)
    if (split != 0 && (unsigned)base + (unsigned)split * K.chunk >= (unsigned)to) return;
    const int c0 = base + split * K.chunk;
    if (K.splits > 1 && split == 0 && hg == 0)
        for (int r = tid; r < rows; r += NT) K.part_live[run.row0 + r] = max(1, (to - base + K.chunk - 1) / K.chunk);
    const int end = K.splits > 1 ? min(to, c0 + K.chunk) : to;

    // the query as operands: element e of step s is 16 s + 8 half + e
    u4_t q[F::STEPS][F::QP];
    u4_t sums = {};
    float qf;
    {
        const IO* const src = static_cast<const IO*>(A.q.data) + row * A.q.row_stride + head * A.q.head_stride;
        IO x[F::STEPS][8];
        float amax = 0.0f;
        bool bad = false;
#pragma unroll
        for (int s = 0; s < F::STEPS; s++) {
            const int d = 16 * s + 8 * half;
            const IO* const p = src + (d < hd ? d : 0);
            if (K.aligned) {
                const auto y = *reinterpret_cast<const vec8*>(p);
#pragma unroll
                for (int e = 0; e < 8; e++) x[s][e] = on && d < hd ? y[e] : (IO)0.0f;
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) x[s][e] = on && d < hd ? p[e] : (IO)0.0f;
            }
#pragma unroll
            for (int e = 0; e < 8; e++) {
                amax = fmaxf(amax, fabsf((float)x[s][e]));
                bad |= !(fabsf((float)x[s][e]) <= 3.402823466e38f);
            }
        }
        amax = half_max(amax);
        bad = half_max(bad ? 1.0f : 0.0f) > 0.0f;
        // 4 bits: the largest in [2^8, 2^9), so that a group's sum stays under 2^14; else in [2^14, 2^15)
        const int e2 = F::SCALED && amax > 0.0f ? (F::I4 ? 9 : 15) - (int)((__builtin_bit_cast(uint32_t, amax) >> 23) - 126) : 0;
        float sum[F::G] = {};
#pragma unroll
        for (int s = 0; s < F::STEPS; s++) {
            typename HK::V a;
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                y[e] = bad ? 0.0f : F::SCALED ? __builtin_ldexpf((float)x[s][e], e2) : (float)x[s][e];
                if (A.scale < 0.0f) y[e] = -y[e];
                a[e] = (typename HK::E)y[e];
                if constexpr (F::I4) sum[s / 2] += y[e];
            }
            q[s][0] = __builtin_bit_cast(u4_t, a);
            if constexpr (F::QP == 2) two_parts<true>(y, q[s][0], q[s][1]);
        }
        if constexpr (F::I4) {
            h8_t w;
#pragma unroll
            for (int g = 0; g < 8; g++) w[g] = (_Float16)0.0f;
#pragma unroll
            for (int g = 0; g < F::G; g++) {
                float t = half_sum(sum[g]);
                asm volatile("" : "+v"(t));  // (its parts are those of the rounded sum)
                const _Float16 hi16 = (_Float16)t;
                w[g] = half ? (_Float16)(t - (float)hi16) : hi16;
            }
            sums = __builtin_bit_cast(u4_t, w);
        }
        const float unit = F::SCALED ? __builtin_ldexpf(1.0f, -e2) : 1.0f;
        qf = unit * (A.soft != 0.0f ? fabsf(A.scale) / A.soft : fabsf(A.scale) * kLog2e);
        // Queries and scales so small that this would be 0, which a masked score of -infinity cannot be multiplied with: raw
        // scores are under 2^40 here, so these scores are 0 either way.
        if constexpr (F::SCALED) qf = fmaxf(qf, 0x1p-126f);
        qf = fminf(qf, 3.402823466e38f);  // (a small cap: an infinite factor would make NaN of a score of 0)
        if (bad) qf = __builtin_nanf("");
    }
    const bool simple = !(fabsf(A.scale) < 0x1p-60f);
    const float soft = A.soft * kLog2e, slope = A.slopes ? A.slopes[head] * kLog2e : 0.0f;

    // tanh y = y (1 + t1 y^2 + t2 y^4 + t3 y^6) for y up to 0.45, off by 2.9e-7 of itself at most (fitted; the first
    // coefficient is 1, so that scores that are a small part of the cap lose nothing), and its coefficients for raw scores:
    // cap tanh(qf x) = x (p0 + p1 x^2 + p2 x^4 + p3 x^6)
    constexpr float kSmall = 0.45f, t1 = -0.333304852f, t2 = 0.13246648f, t3 = -0.0463218503f;
    const float q2 = qf * qf, p0 = soft * qf, p1 = t1 * p0 * q2, p2 = t2 * p0 * q2 * q2, p3 = t3 * p0 * q2 * q2 * q2;

    // LDS addresses, in bytes: of a key's chunk of step 0 for the first product, and of the values' columns of tile 0
    // (for keys 0 .. 3 and 8 .. 11 of a half) for the second.  Step s and tile t lie an exclusive or with 32 s or 64 t away.
    const uint32_t koff = (uint32_t)((lane & 31) * F::ROW + ((half ^ (lane & F::MASK)) * 16));
    uint32_t voff[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
        const int key = 8 * e + 4 * half + (lane & 15) / 4;  // (a multiple of 16 further on in the reads)
        voff[e] = (uint32_t)(key * F::ROW + F::vchunk(key, 2 * (lane >> 4 & 1) + (lane & 3) / 2) * 16 + (lane & 1) * 8);
    }

    const int64_t first = (int64_t)kvh * P.page_size, page_rows = (int64_t)nkv * P.page_size;
    const int* const table = A.M.tables + (int64_t)run.seq * A.M.stride;
    const int row_bytes = F::I4 ? 16 * F::G : F::I8 ? hd : 2 * hd;
    const int units = row_bytes / 16;

    // The page of each of a tile's four groups of 16 positions, in lanes 0 .. 3 (and again behind them).
    auto pages = [&](int t0) -> int {
        const int i = (t0 + 16 * (lane & 3)) >> K.ps_log2;
        return i < A.M.stride ? table[i] : -1;
    };
    // A unit's loads lie within one group for all lanes of a wave, so they go through a buffer over the group's
    // positions below `to`: others read as zeros.
    constexpr int PER = F::I4 ? 4 : F::BYTES / 16;  // threads that share a key
    const int key16 = tid / PER & 15;
    const uint32_t voff_k = F::I4 ? (uint32_t)(key16 * row_bytes + (tid & 3) * 4 * F::G)
                            : tid % PER < units ? (uint32_t)(key16 * row_bytes + tid % PER * 16)
                                                : kNowhere;
    auto bring = [&](Staged<F>& g, int ids, int t0, int from, int to) {
        auto group = [&](int grp, int& live) -> int64_t {  // its first position among those of all pages and heads
            const int page = __builtin_amdgcn_readlane(ids, grp), at = t0 + 16 * grp;
            const bool here = (unsigned)page < (unsigned)P.num_pages;
            live = __builtin_amdgcn_readfirstlane(here ? min(max(to - at, 0), 16) : 0);
            return (here ? page * page_rows : 0) + first + (at & (P.page_size - 1));
        };
        auto buffer = [](const void* p, int bytes) {
            return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, bytes, 0x00020000);
        };
        auto load16 = [](auto r, uint32_t off) { return __builtin_bit_cast(u4_t, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0)); };
        auto load8 = [](auto r, uint32_t off) {
            const u2_t x = __builtin_bit_cast(u2_t, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0));
            return u4_t{x[0], x[1], 0, 0};
        };
        if constexpr (F::I4) {
            int live;
            const int64_t r = group(wave, live);
            const bool out = key16 < from - (t0 + 16 * wave);
            const uint32_t off = out ? kNowhere : voff_k, woff = out ? kNowhere : (uint32_t)(key16 * 4 * F::G);
            const auto kr = buffer(static_cast<const char*>(P.k) + r * row_bytes, live * row_bytes);
            const auto vr = buffer(static_cast<const char*>(P.v) + r * row_bytes, live * row_bytes);
            const auto kwr = buffer(reinterpret_cast<const char*>(P.k_scale) + r * (4 * F::G), live * (4 * F::G));
            const auto vwr = buffer(reinterpret_cast<const char*>(P.v_scale) + r * (4 * F::G), live * (4 * F::G));
            if constexpr (F::G == 2) {
                g.k[0] = load8(kr, off);
                g.v[0] = load8(vr, off);
                g.kw[0] = load8(kwr, woff);
                g.vw[0] = load8(vwr, woff);
            } else {
#pragma unroll
                for (int u = 0; u < F::UNITS; u++) {
                    g.k[u] = load16(kr, off + 16 * u);
                    g.v[u] = load16(vr, off + 16 * u);
                    g.kw[u] = load16(kwr, woff + 16 * u);
                    g.vw[u] = load16(vwr, woff + 16 * u);
                }
            }
        } else {
#pragma unroll
            for (int u = 0; u < F::UNITS; u++) {
                const int grp = (u * NT + 64 * wave) / PER / 16;
                int live;
                const int64_t r = group(grp, live);
                // (rows of 32 units: every other one is the group's second half)
                const int key = key16 + (PER == 32 && (u & 1) ? 8 : 0);
                const uint32_t off = key < from - (t0 + 16 * grp) ? kNowhere : voff_k + (uint32_t)(PER == 32 && (u & 1) ? 8 * row_bytes : 0);
                g.k[u] = load16(buffer(static_cast<const char*>(P.k) + r * row_bytes, live * row_bytes), off);
                g.v[u] = load16(buffer(static_cast<const char*>(P.v) + r * row_bytes, live * row_bytes), off);
            }
            if constexpr (F::I8) {
                int live;
                const int64_t r = group(wave, live);
                const uint32_t off = lane < 16 && lane >= from - (t0 + 16 * wave) ? (uint32_t)(4 * lane) : kNowhere;
                g.ks = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(buffer(P.k_scale + r, 4 * live), off, 0, 0));
                g.vs = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(buffer(P.v_scale + r, 4 * live), off, 0, 0));
            }
        }
    };
    // into LDS as the products take it; with `ask`, whether a value is not finite
    auto put = [&](const Staged<F>& g, int buf, bool ask) -> bool {
        char* const ks = reinterpret_cast<char*>(sh.k[buf]);
        char* const vs = reinterpret_cast<char*>(sh.v[buf]);
        bool odd = false;
        if constexpr (F::I4) {
            const int key = tid / 4, quarter = tid & 3;
            uint32_t k[4 * F::UNITS], v[4 * F::UNITS], kw[4 * ((F::G + 3) / 4)], vw[4 * ((F::G + 3) / 4)];
#pragma unroll
            for (int u = 0; u < F::UNITS; u++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    k[4 * u + i] = g.k[u][i];
                    v[4 * u + i] = g.v[u][i];
                    kw[4 * u + i] = g.kw[u][i];
                    vw[4 * u + i] = g.vw[u][i];
                }
#pragma unroll
            for (int c = 0; c < F::G; c++) {
                const h2_t x = __builtin_bit_cast(h2_t, kw[c]), y = __builtin_bit_cast(h2_t, vw[c]);
                const _Float16 s16 = x.x * (_Float16)16.0f;
                u4_t a, b;
#pragma unroll
                for (int j = 0; j < 4; j++) {  // byte j G + c: two elements side by side
                    const int at = j * F::G + c;
                    const uint32_t kb = k[at >> 2] >> (8 * (at & 3)), vb = v[at >> 2] >> (8 * (at & 3));
                    const uint32_t n = (kb << 6 & 0x3c0u) | (kb << 18 & 0x03c00000u) | 0x3c003c00u;  // 1 + n / 16
                    a[j] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(h2_t, n), h2_t{s16, s16}, h2_t{-s16, -s16}));
                    const float v0 = __builtin_fmaf((float)(vb & 15u), (float)y.x, (float)y.y);
                    const float v1 = __builtin_fmaf((float)(vb >> 4 & 15u), (float)y.x, (float)y.y);
                    b[j] = __builtin_bit_cast(uint32_t, h2_t{(_Float16)v0, (_Float16)v1});
                }
                if (32 * c + 8 * quarter >= hd) a = b = u4_t{};
                const uint32_t off = (uint32_t)(key * F::ROW + (((4 * c + quarter) ^ (key & F::MASK)) * 16));
                *reinterpret_cast<u4_t*>(ks + off) = a;
                *reinterpret_cast<u4_t*>(vs + key * F::ROW + F::vchunk(key, 4 * c + quarter) * 16) = b;
                if (ask)
#pragma unroll
                    for (int i = 0; i < 4; i++) odd |= infinite16(b[i], false);
                if (quarter == 0) sh.low[buf][key][c] = 32 * c < hd ? x.y : (_Float16)0.0f;
            }
            if (quarter == 0)
#pragma unroll
                for (int c = F::G; c < 8; c++) sh.low[buf][key][c] = (_Float16)0.0f;
        } else {
#pragma unroll
            for (int u = 0; u < F::UNITS; u++) {
                const int i = u * NT + tid, key = i / PER, c = i % PER;
                if constexpr (F::I8) {
                    // 16 whole numbers: two chunks
#pragma unroll
                    for (int p = 0; p < 2; p++) {
                        const uint32_t off = (uint32_t)(key * F::ROW + (((2 * c + p) ^ (key & F::MASK)) * 16));
                        auto wide = [](uint32_t w0, uint32_t w1, auto h) {
                            typename decltype(h)::V r;
#pragma unroll
                            for (int e = 0; e < 8; e++) r[e] = (typename decltype(h)::E)(float)(int8_t)((e < 4 ? w0 : w1) >> (8 * (e & 3)));
                            return __builtin_bit_cast(u4_t, r);
                        };
                        if constexpr (F::KBF)
                            *reinterpret_cast<u4_t*>(ks + off) = wide(g.k[u][2 * p], g.k[u][2 * p + 1], HK{});
                        else
                            *reinterpret_cast<u4_t*>(ks + off) = __builtin_bit_cast(u4_t, q8_to_h8(g.k[u][2 * p], g.k[u][2 * p + 1]));
                        *reinterpret_cast<u4_t*>(vs + key * F::ROW + F::vchunk(key, 2 * c + p) * 16) = wide(g.v[u][2 * p], g.v[u][2 * p + 1], HV{});
                    }
                } else {
                    const uint32_t off = (uint32_t)(key * F::ROW + ((c ^ (key & F::MASK)) * 16));
                    *reinterpret_cast<u4_t*>(ks + off) = g.k[u];
                    *reinterpret_cast<u4_t*>(vs + key * F::ROW + F::vchunk(key, c) * 16) = g.v[u];
                    if (ask)
#pragma unroll
                        for (int i = 0; i < 4; i++) odd |= infinite16(g.v[u][i], F::VBF);
                }
            }
            if constexpr (F::I8)
                if (lane < 16) {
                    sh.ks[buf][16 * wave + lane] = g.ks;
                    sh.vs[buf][16 * wave + lane] = g.vs;
                }
        }
        return odd;
    };

    f16_t o[F::DT];
    float m, l;
    bool far;  // the wave has a running maximum past 2^20
    // one tile from LDS
    auto work = [&](int buf, int t0, uint32_t there) {
        const char* const ks = reinterpret_cast<const char*>(sh.k[buf]);
        uint32_t ko = koff, vo[2] = {voff[0], voff[1]};
        asm volatile("" : "+v"(ko), "+v"(vo[0]), "+v"(vo[1]));  // (the addresses made from them are not kept in registers)
        f16_t s[2];
#pragma unroll
        for (int n = 0; n < 2; n++) {
            s[n] = f16_t{};
            if constexpr (F::I4) {
                const u4_t a = *reinterpret_cast<const u4_t*>(&sh.low[buf][32 * n + (lane & 31)][0]);
                s[n] = HK::mul(a, sums, s[n]);
            }
#pragma unroll
            for (int i = 0; i < F::STEPS; i++) {
                const u4_t a = *reinterpret_cast<const u4_t*>(ks + 32 * n * F::ROW + (ko ^ (32u * i)));
#pragma unroll
                for (int p = F::QP - 1; p >= 0; p--) s[n] = HK::mul(a, q[i][p], s[n]);
            }
        }
        const bool masked = t0 < w_all_lo || t0 + BN > w_all_hi || there != 15u;
        // whether the column does not see the position of its score s[n][i]
        auto outside = [&](int n, int i) {
            const int j = t0 + 32 * n + 8 * (i >> 2) + 4 * half + (i & 3);
            return j < lo || j >= hi || !(there >> (2 * n + (i >> 3)) & 1u);
        };
        auto mask = [&](float none) {
            asm volatile("");  // (a branch)
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int i = 0; i < 16; i++) s[n][i] = outside(n, i) ? none : s[n][i];
        };
        auto largest = [&](float sign) {
            float top = -__builtin_inff();
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int i = 0; i < 16; i++) top = fmaxf(top, sign * s[n][i]);
            return half_max(top);
        };
        if constexpr (F::I8) {
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int b = 0; b < 4; b++) {
                    const f4_t x = *reinterpret_cast<const f4_t*>(&sh.ks[buf][32 * n + 8 * b + 4 * half]);
#pragma unroll
                    for (int i = 0; i < 4; i++) s[n][4 * b + i] *= x[i];
                }
        }
        // s becomes the exponents, scores in units of log2 e less the running maximum: without cap or bias by one fma (but
        // where the scale is 0 or close to it, as -infinity cannot be multiplied with 0); capped ones that are all within
        // 0.45 of the cap by the polynomial in five operations; else step by step.
        float top = largest(1.0f);
        int way = A.slopes || (A.soft != 0.0f && masked) || !simple || far ? 2 : A.soft != 0.0f ? 1 : 0;
        // (between these the polynomial's coefficients are finite and normal numbers)
        if (way == 1 && __any(!(fmaxf(top, largest(-1.0f)) * qf <= kSmall && qf >= 0x1p-16f && qf <= 0x1p16f))) way = 2;
        way = __builtin_amdgcn_readfirstlane(way);
        auto capped = [&](float x, float less) {
            const float x2 = x * x;
            return __builtin_fmaf(x, __builtin_fmaf(x2, __builtin_fmaf(x2, __builtin_fmaf(x2, p3, p2), p1), p0), less);
        };
        if (way == 2) {
            const float twice = 2.0f * kLog2e;
#pragma unroll
            for (int n = 0; n < 2; n++) {
                if (FINE) {
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float y = s[n][i] * qf, y2 = y * y;
                        const float x = __builtin_fmaf(-2.0f * soft, __builtin_amdgcn_rcpf(exp2_hw(fabsf(y) * twice) + 1.0f), soft);
                        const float z = soft * y * __builtin_fmaf(y2, __builtin_fmaf(y2, __builtin_fmaf(y2, t3, t2), t1), 1.0f);
                        s[n][i] = fabsf(y) <= kSmall ? z : __builtin_copysignf(x, y);
                    }
                } else if (A.soft != 0.0f) {  // 1 - 2 / (e^2y + 1)
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        s[n][i] = __builtin_fmaf(-2.0f * soft, __builtin_amdgcn_rcpf(exp2_hw(s[n][i] * qf * twice) + 1.0f), soft);
                } else {
#pragma unroll
                    for (int i = 0; i < 16; i++) s[n][i] *= qf;
                }
                if (A.slopes) {
                    const float d = (float)(pos - t0 - 32 * n - 4 * half);
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        s[n][i] = __builtin_fmaf(-slope, fabsf(d - (float)(8 * (i >> 2) + (i & 3))), s[n][i]);
                }
            }
        }
        if (masked) mask(-__builtin_inff());
        if (way == 2 || masked) top = largest(1.0f);
        top = way == 2 ? top : way == 1 ? capped(top, 0.0f) : top * qf;
        // the running maximum moves when the tile's is over it by more than 2^6, and at first
        if (__any(top - m > 6.0f)) {
            const float mn = top - m > 6.0f ? top : m;
            const float a = exp2_hw(m - mn);
            m = mn;
            // Past 2^20 scores are rounded before the maximum is taken off: it is one of them, and what it lost by its own
            // rounding, which grows with it, must not be left over as an exponent.
            far = __any(fabsf(m) > 0x1p20f && m > kNone);
            if (__builtin_expect(far && way != 2, 0)) {
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int i = 0; i < 16; i++) s[n][i] = way == 1 ? capped(s[n][i], 0.0f) : s[n][i] * qf;
                way = 2;
            }
            l *= a;
#pragma unroll
            for (int t = 0; t < F::DT; t++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[t][i] *= a;
        }
        float less = F::LIFT - m;
        if (__builtin_expect(far, 0)) {  // (always way 2)
            less = F::LIFT;
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int i = 0; i < 16; i++) s[n][i] -= m;
        }
#pragma unroll
        for (int n = 0; n < 2; n++) {
            if (way == 0) {
#pragma unroll
                for (int i = 0; i < 16; i++) s[n][i] = __builtin_fmaf(s[n][i], qf, less);
            } else if (way == 1) {
#pragma unroll
                for (int i = 0; i < 16; i++) s[n][i] = capped(s[n][i], less);
            } else {
#pragma unroll
                for (int i = 0; i < 16; i++) s[n][i] += less;
            }
        }
        const char* const vs = reinterpret_cast<const char*>(sh.v[buf]);
#pragma unroll
        for (int n = 0; n < 2; n++) {
#pragma unroll
            for (int c = 0; c < 2; c++) {  // 16 keys
                u4_t p[F::PP];
                {
                    float w[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) w[e] = exp2_hw(s[n][8 * c + e]);
                    if constexpr (F::I8) {
#pragma unroll
                        for (int e = 0; e < 8; e++) l += w[e];
#pragma unroll
                        for (int b = 0; b < 2; b++) {
                            const f4_t x = *reinterpret_cast<const f4_t*>(&sh.vs[buf][32 * n + 16 * c + 8 * b + 4 * half]);
#pragma unroll
                            for (int i = 0; i < 4; i++) w[4 * b + i] *= x[i];
                        }
                        if (masked) {  // 0 times a scale that is NaN, where the row does not see it
                            asm volatile("");
#pragma unroll
                            for (int e = 0; e < 8; e++) w[e] = outside(n, 8 * c + e) ? 0.0f : w[e];
                        }
                    }
                    if constexpr (F::PP == 2) {
                        if constexpr (!F::I8)
#pragma unroll
                            for (int e = 0; e < 8; e++) l += w[e];
                        two_parts<false>(w, p[0], p[1]);
                    } else {
                        typename HV::V a;
#pragma unroll
                        for (int e = 0; e < 8; e++) a[e] = (typename HV::E)w[e];
                        p[0] = __builtin_bit_cast(u4_t, a);
                        if constexpr (!F::I8)
#pragma unroll
                            for (int e = 0; e < 4; e++) l = HV::both(p[0][e], l);
                    }
                }
#pragma unroll
                for (int t = 0; t < F::DT; t++) {
                    u4_t a;
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const auto x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (__attribute__((address_space(3))) s4_t*)(vs + (32 * n + 16 * c) * F::ROW + (vo[e] ^ (64u * t))));
                        const u2_t y = __builtin_bit_cast(u2_t, x);
                        a[2 * e] = y[0];
                        a[2 * e + 1] = y[1];
                    }
#pragma unroll
                    for (int i = F::PP - 1; i >= 0; i--) o[t] = HV::mul(a, p[i], o[t]);
                }
            }
        }
    };

    // all rows at once; where a value that is not finite meets rows that do not see it, row by row
    for (int only = -1; only < rows; only++) {
        int s_from = from, s_to = end;
        if (only >= 0) {
            const int r = run.row0 + only;
            s_from = A.first ? max(A.first[r], 0) : 0;
            s_to = min(A.last ? A.last[r] : min(A.pos[r], A.cap) + 1, end);
        }
#pragma unroll
        for (int t = 0; t < F::DT; t++) o[t] = f16_t{};
        m = kNone;
        l = 0.0f;
        far = false;
        bool odd = false;
        Staged<F> g;
        int ids = -1, next = -1;  // the pages of this tile and of the next
        if (c0 < end) {
            next = pages(c0);
            bring(g, next, c0, s_from, s_to);
        }
        for (int t0 = c0, buf = 0; t0 < end; t0 += BN, buf ^= 1) {
            ids = next;
            if (t0 + BN < end) next = pages(t0 + BN);
            const bool ask = !F::I8 && only < 0 && (t0 < all_lo || t0 + BN > all_hi);
            if (put(g, buf, ask)) sh.odd[buf] = 1;
            __syncthreads();
            if (ask && sh.odd[buf]) {  // (this buffer's flag is not set again before all have read it)
                odd = true;
                break;
            }
            if (t0 + BN < end) bring(g, next, t0 + BN, s_from, s_to);
            const uint32_t there = (uint32_t)__ballot((unsigned)ids < (unsigned)P.num_pages) & 15u;
            if (t0 < w_to && t0 + BN > w_from) work(buf, t0, there);
        }
        if (odd) {
            __syncthreads();
            continue;
        }

        // o / l, or both with m for the join
        l = half_sum(l);
        const float sum = sees ? l : 0.0f;
        const int64_t at_row = (int64_t)row * A.nh + head;
        if (on && (only < 0 || only == crow)) {
            if (K.splits == 1) {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                IO* const dst = static_cast<IO*>(A.out.data) + row * A.out.row_stride + head * A.out.head_stride;
#pragma unroll
                for (int t = 0; t < F::DT; t++)
#pragma unroll
                    for (int b = 0; b < 4; b++) {
                        const int d = 32 * t + 8 * b + 4 * half;
                        if (d >= hd) continue;
                        vec4 y;
#pragma unroll
                        for (int i = 0; i < 4; i++) y[i] = (IO)(sum == 0.0f ? 0.0f : o[t][4 * b + i] * inv);
                        if (K.aligned)
                            *reinterpret_cast<vec4*>(dst + d) = y;
                        else
#pragma unroll
                            for (int i = 0; i < 4; i++) dst[d + i] = y[i];
                    }
            } else {
                float* const dst = K.part_o + (at_row * K.splits + split) * hd;
#pragma unroll
                for (int t = 0; t < F::DT; t++)
#pragma unroll
                    for (int b = 0; b < 4; b++) {
                        const int d = 32 * t + 8 * b + 4 * half;
                        if (d < hd) *reinterpret_cast<f4_t*>(dst + d) = f4_t{o[t][4 * b], o[t][4 * b + 1], o[t][4 * b + 2], o[t][4 * b + 3]};
                    }
                if (half == 0) K.part_ml[at_row * K.splits + split] = float2{m, sum};
            }
        }
        if (only < 0) break;
        __syncthreads();
    }
#endif
}

template <int PT, bool BIO, bool FINE>
void launch_hd(const Ruled& K, unsigned grid, hipStream_t st) {
    const int hd = K.A.P.head_dim;
    if (hd <= 64)
        tiled_attend_kernel<PT, 1, BIO, FINE><<<grid, NT, 0, st>>>(K);
    else if (hd <= 128)
        tiled_attend_kernel<PT, 2, BIO, FINE><<<grid, NT, 0, st>>>(K);
    else
        tiled_attend_kernel<PT, 4, BIO, FINE><<<grid, NT, 0, st>>>(K);
}

template <int PT, bool FINE>
void launch_io(const Ruled& K, unsigned grid, hipStream_t st) {
    if (K.A.type == JYHIP_T_BF16)
        launch_hd<PT, true, FINE>(K, grid, st);
    else
        launch_hd<PT, false, FINE>(K, grid, st);
}

template <int PT>
void launch_fine(const Ruled& K, unsigned grid, hipStream_t st) {
    if (K.A.soft > kFineCap)
        launch_io<PT, true>(K, grid, st);
    else
        launch_io<PT, false>(K, grid, st);
}

}  // namespace

bool plan_tiled(Ruled& K) {
    const RuledAttn& A = K.A;
    if (!A.starts || A.type == JYHIP_T_F32) return false;
    const int per = A.nh / A.P.num_kv_heads;
    // Columns a run on average that pay for tiles of 128; the kernel of 16 columns reads a run's cache once for
    // each 16.  32 heads over 8 of 128, 16 runs behind 4000 positions: 8 rows each (32 columns) 48 us there and 62
    // here, 16 rows 66 and 74, 32 rows 95 and 91, 64 rows 155 and 132; prompts of 16 rows 17.5 and 12.9.  14 over 2
    // of 64: 4 rows (28 columns) 25 and 26, 8 rows (56) 29 and 27, 16 rows 36 and 31.
    const int pays = A.P.head_dim <= 64 ? 32 : 64;
    if ((int64_t)A.rows * per < (int64_t)pays * A.M.nseq) return false;
    K.hpg = std::min(per, COLS);
    K.tiles = (per + COLS - 1) / COLS;
    K.rpg = per <= COLS ? COLS / per : 1;
    K.groups = (int)std::min<int64_t>(A.rows, A.rows / K.rpg + (int64_t)A.M.nseq);
    const int64_t base = (int64_t)K.groups * A.P.num_kv_heads * K.tiles;
    K.chunk = (A.span + 31 + BN - 1) / BN * BN;
    K.splits = 1;
    if (base < 512 && A.span > 512) {
        const int64_t want = 1024 / base;
        K.chunk = (int)std::max<int64_t>(256, ((A.span + 31 + want - 1) / want + BN - 1) / BN * BN);
        K.splits = (A.span + 31 + K.chunk - 1) / K.chunk;
    }
    auto whole = [](const jyhip_vectors& x) { return ((uintptr_t)x.data | (uintptr_t)(x.row_stride * 2) | (uintptr_t)(x.head_stride * 2)) % 16 == 0; };
    K.aligned = whole(A.q) && whole(A.out);
    K.tiled = true;
    return true;
}

void launch_tiled(const Ruled& K, unsigned grid, hipStream_t st) {
    if (K.A.P.type == JYHIP_T_I4)
        launch_fine<JYHIP_T_I4>(K, grid, st);
    else if (K.A.P.type == JYHIP_T_I8)
        launch_fine<JYHIP_T_I8>(K, grid, st);
    else if (K.A.P.type == JYHIP_T_F16)
        launch_fine<JYHIP_T_F16>(K, grid, st);
    else
        launch_fine<JYHIP_T_BF16>(K, grid, st);
}

}  // namespace jy
