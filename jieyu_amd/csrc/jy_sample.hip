// jy_sample.hip — one token per row of logits: temperature, top-k, top-p, min-p, and a given
// random number.
//
// With M the row's largest logit, e_i = exp((x_i - M) / T) is token i's mass.  The filters keep a
// prefix of the tokens in order of falling logits (ties: the lowest index first), which is a
// threshold on the logit and a number of its ties; the token is the first one, in order of
// indices, whose running sum of kept masses exceeds u times their total.
//
// Masses are computed in fp64 and held as 64-bit whole numbers, e_i 2^s with V 2^s < 2^63: a sum of
// 150000 fp32 masses is off by more than many a token's share, and whole numbers add up to the
// same total in any order, so atomics do not change a result.
//
// A row is shared by up to 64 workgroups, in four kernels that each read what they need of it once:
//   1  the largest logit, and the maxima of 1024 parts of the row: the k-th largest of those is at
//      most the k-th largest logit, so it bounds the top-k candidates from below
//   2  top-k: the candidates into a list; else the masses of blocks of 2048 tokens, or with top-p a
//      histogram of mass over the distance to M (32 bins per factor of two)
//   3  top-p: the masses of the blocks above the bin that the border lies in, that bin's tokens
//      into the list
//   4  one workgroup per row: the border among the list's tokens, then the block and the token in
//      it
// A row whose candidates do not fit the list (k > 1024, thousands of equal logits at the border, and many a
// row with k = 1024, whose bound is the least of the parts' maxima) is done by its workgroup in kernel 4
// alone, by a radix descent over the logits' bits: 64 rows of 128256, fp32, all passes: k = 50 30 us,
// 500 40, 1000 43, 1024 490, 2000 580; one row 20, 28, 30, 420 and 410.
//
// Time of the kernels (1, 2, 3, 4), us: one row of 151936, fp32, k = 50: 3.8, 6.4, 1.7, 6.2: the launches
// and each kernel's chain of loads and barriers.  64 rows of 128256, fp32, all kinds of settings: 8.5,
// 14.5, 9.8, 17.1, the last for k = 1000: a step of a descent and an ordering for each border, two steps
// for the token, each some barriers and waits for LDS.  256 rows of 152064, bf16, top-p 0.9: 17, 32,
// 33, 16: the first is memory's time (4.7 TB/s); the next two have that and 15 us more, their start
// (the table, the cells or the border's bin) and end, which no other workgroup's work covers as all are
// resident at once (with half of them at a time it was more).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "jy_device.h"
#include "jy_paged_device.h"
#include "jy_sample.h"

namespace jy {

namespace {

constexpr int NP = 512;             // threads of a row's parts (kernels 1 to 3)
constexpr int NT = 1024;            // threads of a row's last workgroup
constexpr int BINS = 2048;
constexpr int LIST = 8192;          // tokens of a row's list
constexpr int BLOCK = 2048;         // tokens per partial mass
constexpr int STRIPES = 1024;       // parts whose maxima bound the k-th largest logit
constexpr int MAX_SEGS = 64;
constexpr int SEG_BLOCKS = 512;     // blocks of a segment at most
constexpr int STEP_BITS = 9;
constexpr int STEPS = 1 << STEP_BITS;  // table entries per factor of two of mass
constexpr int PER_BIN = 16;         // of them in a histogram bin: masses under 2^-52 are none, 53 * 512 / 16 < BINS
constexpr int STAGE = 1024;         // list entries a workgroup collects before it takes places for them

enum { ROW_GREEDY, ROW_TOPK, ROW_MASS, ROW_NUCLEUS, ROW_ALONE };

typedef unsigned long long u64;

struct SamplePlan {
    int segs = 1, seg_len = 0, blocks = 0;
    size_t row_bytes = 0;
};

SamplePlan plan_of(int rows, int vocab) {
    SamplePlan p;
    p.blocks = (vocab + BLOCK - 1) / BLOCK;
    // about 1024 workgroups, none of less than a block
    p.segs = 1;
    while (p.segs < MAX_SEGS && (((int64_t)rows * p.segs * 2 <= 1024 && p.segs * 2 <= p.blocks) ||
                                 (p.blocks + p.segs - 1) / p.segs > SEG_BLOCKS))
        p.segs *= 2;
    p.seg_len = (p.blocks + p.segs - 1) / p.segs * BLOCK;
    const size_t n = (size_t)BINS * 8 + (size_t)LIST * 8 + (size_t)p.blocks * 8 + MAX_SEGS * 8 + STRIPES * 4 + 16;
    p.row_bytes = (n + 255) / 256 * 256;
    return p;
}

// a row's part of the workspace
struct RowWs {
    u64* hist;      // [BINS]
    u64* list;      // [LIST] key << 32 | ~index
    u64* block;     // [blocks]
    u64* seg_top;   // [MAX_SEGS] the segment's first token in the order, as a list entry; 0: none
    float* stripe;  // [STRIPES]
    uint32_t* count;
};
__device__ __forceinline__ RowWs row_ws(const SampleArgs& A, const SamplePlan& P, int row) {
    RowWs w;
    unsigned char* p = A.ws + (size_t)row * P.row_bytes;
    w.hist = reinterpret_cast<u64*>(p);
    w.list = w.hist + BINS;
    w.block = w.list + LIST;
    w.seg_top = w.block + P.blocks;
    w.stripe = reinterpret_cast<float*>(w.seg_top + MAX_SEGS);
    w.count = reinterpret_cast<uint32_t*>(w.stripe + STRIPES);
    return w;
}

// order-preserving bits of a logit; NaN counts as the lowest, -0 as 0
__device__ __forceinline__ uint32_t key_of(float x) {
    if (x != x) return 0;
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
    return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// a row's settings
struct Set {
    float T, p;
    int k;
    double min_e;
    int mode;
};
__device__ __forceinline__ Set set_of(const SampleArgs& A, int row) {
    Set s;
    s.T = A.temperature ? A.temperature[row] : 1.0f;
    s.k = A.top_k ? A.top_k[row] : 0;
    s.p = A.top_p ? A.top_p[row] : 1.0f;
    const float m = A.min_p ? A.min_p[row] : 0.0f;
    s.min_e = m > 0.0f ? fmin((double)m, 1.0) : 0.0;
    const bool topk = s.k > 0 && s.k < A.vocab;
    s.mode = !(s.T > 0.0f) ? ROW_GREEDY : topk ? (s.k <= STRIPES ? ROW_TOPK : ROW_ALONE) : s.p < 1.0f ? ROW_NUCLEUS : ROW_MASS;
    return s;
}

// Masses of a row's logits, e 2^s.  With y = 512 (x - M) log2 e / T = k + r, k whole and |r| <= 1/2:
// 2^(k/512) from a table of 512 (2^s in it) and the exponent, times the Taylor terms of 2^(r/512) up to
// r^3 (the rest is under 9e-15).  The fp64 operations bound the passes that weigh every token, so
// few of them: with a table of 32 and two more terms kernel 2 took 41 us over 256 x 152064, 38 us so.
struct Masses {
    float M, low;    // low: the logit whose mass is far under 2^-52, standing for all below it and NaN
    double c;        // 512 log2 e / T
    double unit;     // 2^s
    const u64* tab;  // [STEPS]
    // false: the largest logit is infinite or T so large that no such logit is finite (then c is 0
    // or M infinite, and only pick_alone() takes the row)
    __device__ __forceinline__ bool set(float top, float T, int vocab, const u64* table) {
        M = top;
        c = STEPS * 1.4426950408889634074 / (double)T;
        // the largest logit 64 factors of two under M.  Where T is so small next to M that this is the
        // float before M, none lies between: a c of twice that keeps y within a whole number's bits.
        const double far = (double)M - 64.0 * STEPS / c;
        low = (float)far;
        if ((double)low > far || low == M) low = logit_of(key_of(low) - 1);
        if (key_of(low) + 1 == key_of(M)) c = fmin(c, 128.0 * STEPS / ((double)M - (double)low));
        int s = 51;
        while (s > 40 && (1ll << (62 - s)) < vocab) s--;
        unit = (double)(1ull << s);
        tab = table;
        return M < __builtin_inff() && low > -3.4e38f;
    }
    // entry i: 2^(i/512) 2^s, as the square root of two times the Taylor terms of e^x up to x^12, x = ln 2
    // (i/512 - 1/2) (the rest is under 2e-16)
    __device__ __forceinline__ void fill(u64* table) const {
        for (int i = threadIdx.x; i < STEPS; i += blockDim.x) {
            const double x = (i - STEPS / 2) * (0.69314718055994531 / STEPS);
            double q = 1.0;
#pragma unroll
            for (int n = 12; n > 0; n--) q = __builtin_fma(q, x * (1.0 / n), 1.0);
            table[i] = __builtin_bit_cast(u64, unit * 1.4142135623730951 * q);
        }
    }
    // 2^(r/512)
    static __device__ __forceinline__ double near(double r) {
        constexpr double L = 0.69314718055994531 / STEPS;
        double q = __builtin_fma(r, L * L * L / 6.0, L * L / 2.0);
        q = __builtin_fma(q, r, L);
        return __builtin_fma(q, r, 1.0);
    }
    struct At {
        double r;
        int k;  // <= 0
        __device__ __forceinline__ int bin() const { return (unsigned)-k / PER_BIN; }
    };
    // l within [low, M], NaN as low
    __device__ __forceinline__ float clamp(float l) const {
#if defined(__HIP_DEVICE_COMPILE__)
        return __builtin_amdgcn_fmed3f(l, low, M);
#else
        return l;
#endif
    }
    __device__ __forceinline__ At at(float l) const {
        const double y = ((double)clamp(l) - (double)M) * c;
        const double shift = 0x1.8p+52;
        const double kd = y + shift;
        return At{y - (kd - shift), (int)(uint32_t)__builtin_bit_cast(u64, kd)};
    }
    // the mass, rounded to a whole number by adding it to 2^52 (it is under that)
    __device__ __forceinline__ u64 mass(const At& a) const {
        const u64 t = tab[a.k & (STEPS - 1)] + ((u64)(uint32_t)((a.k >> STEP_BITS) << 20) << 32);
        return __builtin_bit_cast(u64, __builtin_fma(near(a.r), __builtin_bit_cast(double, t), 0x1p+52)) & 0xfffffffffffffull;
    }
    __device__ __forceinline__ u64 mass(float l) const { return mass(at(l)); }
    // min-p's least mass
    __device__ __forceinline__ u64 least(const Set& s) const { return (u64)__builtin_rint(s.min_e * unit); }
    // a logit at or under the least one of a bin
    __device__ __forceinline__ float under(int bin) const {
        const double l = (double)M - (bin + 1.0) * PER_BIN / c;
        return (float)(l - fabs(l) * 0x1p-20 - 0x1p-120);
    }
    // the same for any M and T
    __device__ __forceinline__ u64 mass_any(float l) const {
        if (l == M) return (u64)unit;
        if (!(l > -__builtin_inff()) || M == __builtin_inff()) return 0;
        const double y = ((double)l - (double)M) * c, k = __builtin_rint(y);
        if (!(y > -64.0 * STEPS)) return 0;
        const u64 t = tab[(int)k & (STEPS - 1)] + ((u64)(uint32_t)(((int)k >> STEP_BITS) << 20) << 32);
        return (u64)__builtin_rint(near(y - k) * __builtin_bit_cast(double, t));
    }
};

// the sum of v over the wave, in every lane (whole numbers: any order)
template <int CTRL>
__device__ __forceinline__ u64 dpp_u64(u64 v) {
#if defined(__HIP_DEVICE_COMPILE__)
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, 0xf, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, 0xf, 0xf, false);
    return (u64)hi << 32 | lo;
#else
    return v;
#endif
}
__device__ __forceinline__ u64 lane_u64(u64 v, int lane) {
#if defined(__HIP_DEVICE_COMPILE__)
    return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
#else
    return v;
#endif
}
__device__ __forceinline__ u64 wave_sum(u64 v) {
    v += dpp_u64<0xB1>(v);
    v += dpp_u64<0x4E>(v);
    v += dpp_u64<0x124>(v);
    v += dpp_u64<0x128>(v);  // every lane: its row of 16's sum
    return lane_u64(v, 0) + lane_u64(v, 16) + lane_u64(v, 32) + lane_u64(v, 48);
}

// the largest of v over the wave, in every lane
__device__ __forceinline__ u64 wave_max(u64 v) {
    v = max(v, dpp_u64<0xB1>(v));
    v = max(v, dpp_u64<0x4E>(v));
    v = max(v, dpp_u64<0x124>(v));
    v = max(v, dpp_u64<0x128>(v));
    return max(max(lane_u64(v, 0), lane_u64(v, 16)), max(lane_u64(v, 32), lane_u64(v, 48)));
}

// VL consecutive logits from index i (those at or past `end` as NaN, which has no mass)
template <class E>
struct Logits {
    static constexpr int VL = 16 / sizeof(E);
    typedef E vec __attribute__((ext_vector_type(VL)));
    const E* x;
    bool aligned;
    __device__ __forceinline__ void load(int i, int end, float (&l)[VL]) const {
        if (aligned && i + VL <= end) {
            const vec v = *reinterpret_cast<const vec*>(x + i);
#pragma unroll
            for (int e = 0; e < VL; e++) l[e] = (float)v[e];
        } else {
#pragma unroll
            for (int e = 0; e < VL; e++) l[e] = i + e < end ? (float)x[i + e] : __builtin_nanf("");
        }
    }
};
template <class E>
__device__ __forceinline__ Logits<E> row_logits(const SampleArgs& A, int row) {
    Logits<E> r;
    r.x = static_cast<const E*>(A.logits) + row * A.row_stride;
    r.aligned = reinterpret_cast<uintptr_t>(r.x) % 16 == 0;
    return r;
}

// f(l, i) for the workgroup's VL logits at a time of [i0, i1), all lanes of a wave together; the next
// ones are read before f takes the present ones.  The first ones: first(), for a caller with other
// work before.
template <class E>
struct First {
    float l[Logits<E>::VL];
};
template <class E>
__device__ __forceinline__ First<E> first(const Logits<E>& x, int i0, int i1) {
    First<E> a;
    x.load(i0 + (int)threadIdx.x * Logits<E>::VL, i1, a.l);
    return a;
}
template <class E, class F>
__device__ __forceinline__ void each(const Logits<E>& x, First<E> a, int i0, int i1, F&& f) {
    constexpr int VL = Logits<E>::VL, STEP = NP * VL;
    First<E> b;
    int i = i0 + (int)threadIdx.x * VL;
    for (int base = i0; base < i1; base += STEP, i += STEP) {
        if (base + STEP < i1) x.load(i + STEP, i1, b.l);
        f(a.l, i);
        a = b;
    }
}
template <class E, class F>
__device__ __forceinline__ void each(const Logits<E>& x, int i0, int i1, F&& f) {
    each(x, first(x, i0, i1), i0, i1, f);
}

// a token in the order: falling logits, equal ones by index
__device__ __forceinline__ u64 entry_of(uint32_t key, int i) { return (u64)key << 32 | (uint32_t)~i; }
constexpr uint32_t LEAST_KEY = 0x00800000u;  // after -infinity's

// the row's first token from its parts' (0: none above -infinity); every wave by itself
__device__ __forceinline__ u64 row_top(const RowWs& w, int segs) {
    const int lane = threadIdx.x & 63;
    return wave_max(lane < segs ? w.seg_top[lane] : 0);
}
__device__ __forceinline__ float top_logit(u64 top) { return logit_of((uint32_t)(top >> 32)); }

// list entries of a workgroup: collected in LDS (one atomic on the row's counter for all of them),
// the ones that find it full go to the list by themselves
struct Stage {
    u64 entry[STAGE];
    uint32_t n, at;
    __device__ __forceinline__ void clear() {
        if (threadIdx.x == 0) n = 0;
    }
    // those of a lane's N entries that are marked, from any of a wave's lanes: one place for each
    template <int N, class F>
    __device__ __forceinline__ void add(const RowWs& w, const bool (&mine)[N], F&& of) {
        u64 who[N];
        int total = 0;
#pragma unroll
        for (int e = 0; e < N; e++) {
            who[e] = __ballot(mine[e]);
            total += __popcll(who[e]);
        }
        if (!total) return;
        const u64 below = (1ull << (threadIdx.x & 63)) - 1;
        uint32_t i = 0;
        if ((threadIdx.x & 63) == 0) i = atomicAdd(&n, (uint32_t)total);
        i = __builtin_amdgcn_readfirstlane(i);
#pragma unroll
        for (int e = 0; e < N; e++) {
            if (mine[e]) {
                const uint32_t j = i + __popcll(who[e] & below);
                if (j < STAGE) {
                    entry[j] = of(e);
                } else {
                    const uint32_t g = atomicAdd(w.count, 1u);
                    if (g < LIST) w.list[g] = of(e);
                }
            }
            i += __popcll(who[e]);
        }
    }
    __device__ __forceinline__ void flush(const RowWs& w) {
        __syncthreads();
        const uint32_t m = min(n, (uint32_t)STAGE);
        if (threadIdx.x == 0 && m) at = atomicAdd(w.count, m);
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < m; i += NP)
            if (at + i < LIST) w.list[at + i] = entry[i];
    }
};

// ---- 1: the parts' largest logits
template <class E>
__global__ __launch_bounds__(NP) void sample_top_kernel(SampleArgs A, SamplePlan P) {
    constexpr int VL = Logits<E>::VL;
    __shared__ u64 first[NP / 64];
    const int row = blockIdx.x / P.segs, seg = blockIdx.x % P.segs;
    const RowWs w = row_ws(A, P, row);
    const Set s = set_of(A, row);
    const int i0 = seg * P.seg_len, i1 = min(i0 + P.seg_len, A.vocab);
    // each thread two maxima (even and odd elements): 1024 parts of the segment
    float top[2] = {-__builtin_inff(), -__builtin_inff()};
    int at = -1;
    each(row_logits<E>(A, row), i0, i1, [&](const float (&l)[VL], int i) {
#pragma unroll
        for (int e = 0; e < VL; e++) {
            if (l[e] > fmaxf(top[0], top[1])) at = i + e;
            top[e & 1] = fmaxf(top[e & 1], l[e]);
        }
    });
    const u64 mine = wave_max(at < 0 ? 0 : entry_of(key_of(fmaxf(top[0], top[1])), at));
    if ((threadIdx.x & 63) == 0) first[threadIdx.x >> 6] = mine;
    if (s.mode == ROW_TOPK) {
        // the segment's share of the row's 1024 maxima, each over 1024 / n of these
        const int n = STRIPES / P.segs;
        if (n == 2 * NP) {
            w.stripe[seg * n + threadIdx.x] = top[0];
            w.stripe[seg * n + NP + threadIdx.x] = top[1];
        } else {
            float m = fmaxf(top[0], top[1]);
            if (n < NP) m = fmaxf(m, dpp_f<0xB1>(m));       // 2 lanes
            if (n < NP / 2) m = fmaxf(m, dpp_f<0x4E>(m));   // 4
            if (n < NP / 4) m = fmaxf(m, dpp_f<0x141>(m));  // 8: the half row mirrored
            if (n < NP / 8) m = fmaxf(m, dpp_f<0x140>(m));  // 16: the row mirrored
            if (n < NP / 16) m = fmaxf(m, __shfl_xor(m, 16));
            const int lanes = NP / n;
            if (threadIdx.x % lanes == 0) w.stripe[seg * n + threadIdx.x / lanes] = m;
        }
        static_assert(STRIPES == 2 * NP && STRIPES / MAX_SEGS >= NP / 32, "groups of up to 32 lanes");
    }
    __syncthreads();
    if (s.mode == ROW_NUCLEUS)
        for (int i = seg * NP + threadIdx.x; i < BINS; i += P.segs * NP) w.hist[i] = 0;
    if (threadIdx.x == 0) {
        u64 t = first[0];
#pragma unroll
        for (int v = 1; v < NP / 64; v++) t = max(t, first[v]);
        w.seg_top[seg] = t;
        if (seg == 0) *w.count = 0;
    }
}

// A lower bound of the k-th largest of the row's stripe maxima, as a key: its leading 21 bits, the
// rest zero.  Every wave holds all maxima, 16 a lane, and counts those at or above one of seven
// thresholds: three bits a round.
struct Bound {
    int n[2][8];
};
__device__ __forceinline__ uint32_t stripe_bound(Bound& S, const RowWs& w, int k) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t key[STRIPES / 64];
#pragma unroll
    for (int j = 0; j < STRIPES / 64; j++) key[j] = key_of(w.stripe[j * 64 + lane]);
    uint32_t bound = 0;
    for (int round = 0; round < 7; round++) {
        const int shift = 29 - 3 * round;
        const uint32_t t = bound | (uint32_t)wave << shift;
        int n = 0;
#pragma unroll
        for (int j = 0; j < STRIPES / 64; j++) n += __popcll(__ballot(key[j] >= t));
        if (lane == 0) S.n[round & 1][wave] = n;
        __syncthreads();
        int best = 0;
        for (int v = 1; v < 8; v++)
            if (S.n[round & 1][v] >= k) best = v;
        bound |= (uint32_t)best << shift;
    }
    return bound;
}
static_assert(NP / 64 == 8, "a wave for each value of three bits");

// bf16 logits have few values: a workgroup counts its tokens by value and weighs each value once
// (256 x 152064: 38 us with every token weighed, 32 us so).
// A cell for every magnitude of the upper 16 powers of two of those with mass, either sign; the tokens
// nearer to zero are weighed one by one.
constexpr int SIDE = 16 << 7;
struct Cells {
    int base;  // the least magnitude with a cell (a bf16's bits)
    __device__ __forceinline__ Cells(const Masses& m) {
        const uint32_t low = __builtin_bit_cast(uint32_t, m.low) & 0x7fffffffu, M = __builtin_bit_cast(uint32_t, m.M) & 0x7fffffffu;
        base = max((int)(max(M, low + 0xffffu) >> 16) - (SIDE - 1), 0);
    }
    // the cell of l, SIDE or more: none
    __device__ __forceinline__ uint32_t magnitude(float l) const {
        return (__builtin_bit_cast(uint32_t, l) >> 16 & 0x7fffu) - (uint32_t)base;
    }
    static __device__ __forceinline__ uint32_t side(float l) { return __builtin_bit_cast(uint32_t, l) >> 31 ? SIDE : 0; }
    __device__ __forceinline__ float logit(int cell) const {
        return __builtin_bit_cast(float, (uint32_t)(base + cell % SIDE) << 16 | (cell >= SIDE ? 0x80000000u : 0));
    }
};

// ---- 2: top-k candidates, masses or the histogram
template <class E>
__global__ __launch_bounds__(NP, 8) void sample_mass_kernel(SampleArgs A, SamplePlan P) {
    constexpr int VL = Logits<E>::VL;
    __shared__ union {
        u64 hist[BINS];
        Stage stage;
    } U;
    __shared__ u64 tab[STEPS];
    __shared__ Bound bound;
    constexpr bool BF16 = __is_same(E, __bf16);
    __shared__ uint32_t cell[BF16 ? 2 * SIDE + 64 : 1];  // (64: for the tokens without a cell)
    u64* const hist = U.hist;
    const int row = blockIdx.x / P.segs, seg = blockIdx.x % P.segs;
    const Set s = set_of(A, row);
    if (s.mode == ROW_GREEDY || s.mode == ROW_ALONE) return;
    const RowWs w = row_ws(A, P, row);
    const int i0 = seg * P.seg_len, i1 = min(i0 + P.seg_len, A.vocab);
    const Logits<E> x = row_logits<E>(A, row);
    const First<E> f = first(x, i0, i1);
    if (s.mode == ROW_TOPK) {
        U.stage.clear();
        const uint32_t b = max(stripe_bound(bound, w, s.k), LEAST_KEY);  // (with barriers)
        each(x, f, i0, i1, [&](const float (&l)[VL], int i) {
            bool mine[VL];
            uint32_t k[VL];
#pragma unroll
            for (int e = 0; e < VL; e++) {
                k[e] = key_of(l[e]);  // (past the end NaN, whose key is under any bound)
                mine[e] = k[e] >= b;
            }
            U.stage.add(w, mine, [&](int e) { return entry_of(k[e], i + e); });
        });
        U.stage.flush(w);
        return;
    }
    const u64 top = row_top(w, P.segs);
    Masses m;
    if (!top || !m.set(top_logit(top), s.T, A.vocab, tab)) return;
    const bool bins = s.mode == ROW_NUCLEUS;
    const int nb = bins ? BINS : (i1 - i0 + BLOCK - 1) / BLOCK;
    for (int i = threadIdx.x; i < nb; i += NP) hist[i] = 0;
    m.fill(tab);
    // where the cells are fewer than the tokens
    const bool counted = BF16 && bins && P.seg_len > 2 * SIDE;
    if (counted)
        for (int i = threadIdx.x; i < 2 * SIDE; i += NP) cell[i] = 0;
    __syncthreads();
    if (counted) {
        const Cells cells(m);
        const uint32_t none = 2 * SIDE + (threadIdx.x & 63);
        each(x, f, i0, i1, [&](const float (&l)[VL], int) {
            bool far = false;
#pragma unroll
            for (int e = 0; e < VL; e++) {
                const uint32_t c = cells.magnitude(l[e]);
                atomicAdd(&cell[c < SIDE ? c + Cells::side(l[e]) : none], 1u);
                far |= c >= SIDE && l[e] > m.low;
            }
            if (__any(far)) {
#pragma unroll
                for (int e = 0; e < VL; e++) {
                    const Masses::At y = m.at(l[e]);
                    const u64 q = m.mass(y);
                    if (q && cells.magnitude(l[e]) >= SIDE) atomicAdd(&hist[y.bin()], q);
                }
            }
        });
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * SIDE; i += NP) {
            const uint32_t n = cell[i];
            if (!n) continue;
            const Masses::At y = m.at(cells.logit(i));
            const u64 q = m.mass(y);
            if (q) atomicAdd(&hist[y.bin()], n * q);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < BINS; i += NP)
            if (hist[i]) atomicAdd(&w.hist[i], hist[i]);
    } else if (bins) {
        each(x, f, i0, i1, [&](const float (&l)[VL], int) {
#pragma unroll
            for (int e = 0; e < VL; e++) {
                const Masses::At y = m.at(l[e]);
                const u64 q = m.mass(y);
                if (q) atomicAdd(&hist[y.bin()], q);
            }
        });
        __syncthreads();
        for (int i = threadIdx.x; i < BINS; i += NP)
            if (hist[i]) atomicAdd(&w.hist[i], hist[i]);
    } else {
        const u64 least = m.least(s);
        each(x, f, i0, i1, [&](const float (&l)[VL], int i) {
            u64 q = 0;
#pragma unroll
            for (int e = 0; e < VL; e++) {
                const u64 v = m.mass(l[e]);
                q += v >= least ? v : 0;
            }
            q = wave_sum(q);
            if ((threadIdx.x & 63) == 0 && q) atomicAdd(&hist[(i - i0) / BLOCK], q);
        });
        __syncthreads();
        for (int i = threadIdx.x; i < nb; i += NP) w.block[i0 / BLOCK + i] = hist[i];
    }
}

// the running sum of v over the wave's lanes up to and with this one
__device__ __forceinline__ u64 wave_scan(u64 v) {
    const int lane = threadIdx.x & 63;
    // within rows of 16 (row_shr:n brings zeros in from the left)
    v += dpp_u64<0x111>(v);
    v += dpp_u64<0x112>(v);
    v += dpp_u64<0x114>(v);
    v += dpp_u64<0x118>(v);
    const u64 r0 = lane_u64(v, 15), r1 = r0 + lane_u64(v, 31), r2 = r1 + lane_u64(v, 47);
    return v + (lane < 16 ? 0 : lane < 32 ? r0 : lane < 48 ? r1 : r2);
}

// Running sums over the first WT threads of a workgroup, one wave on each SIMD of the CU: the sums'
// instructions are what a step costs, and sixteen waves would issue them four times over.  One barrier
// (for all threads) each: the waves' sums go to the two halves of `part` in turn, and a half is
// written again only after the barrier of the call between.
constexpr int WT = 256;
struct Scan {
    u64 part[2][WT / 64];
    // (the sum before this one of the WT threads; the total, in every thread); `turn` is the caller's, 0 at
    // first
    __device__ __forceinline__ u64 before(int& turn, u64 v, u64& total) {
        const int wave = threadIdx.x >> 6;
        u64* const p = part[turn];
        turn ^= 1;
        u64 run = 0;
        if (threadIdx.x < WT) {
            run = wave_scan(v);
            if ((threadIdx.x & 63) == 63) p[wave] = run;
        }
        __syncthreads();
        u64 a = 0;
        total = 0;
#pragma unroll
        for (int w = 0; w < WT / 64; w++) {
            if (w == wave) a = total;
            total += p[w];
        }
        return a + run - v;
    }
};

// The bin that the last kept token lies in: the last one, from the top, with mass in it and less than
// `want` = ceil(p total) above; `above` that mass.  h: a worker's bins.  All threads return the same.
struct BorderBin {
    int bin;
    u64 above, want;
};
struct BorderFound {
    int bin;
    u64 above;
};
constexpr int BINS_EACH = BINS / WT;
__device__ __forceinline__ void load_bins(const u64* hist, u64 (&h)[BINS_EACH]) {
    if (threadIdx.x < WT)
#pragma unroll
        for (int j = 0; j < BINS_EACH; j++) h[j] = hist[threadIdx.x * BINS_EACH + j];
}
__device__ __forceinline__ BorderBin border_bin(const u64 (&h)[BINS_EACH], float p, Scan& scan, int& turn, BorderFound& found) {
    const bool worker = threadIdx.x < WT;
    u64 sum = 0, total;
    if (worker)
#pragma unroll
        for (int j = 0; j < BINS_EACH; j++) sum += h[j];
    u64 run = scan.before(turn, sum, total);
    BorderBin b;
    b.want = (u64)ceil((p > 0.0f ? (double)p : 0.0) * (double)total);
    if (worker && (run < b.want || run == 0) && run + sum >= b.want && sum)
#pragma unroll
        for (int j = 0; j < BINS_EACH; j++) {
            // (run == 0: the first token is always kept)
            if (h[j] && (run < b.want || run == 0) && run + h[j] >= b.want) {
                found.bin = threadIdx.x * BINS_EACH + j;
                found.above = run;
            }
            run += h[j];
        }
    __syncthreads();
    b.bin = found.bin;
    b.above = found.above;
    return b;
}

// ---- 3: top-p: the masses above the border's bin, its tokens into the list
constexpr int VALUES = 2048;  // values of 16-bit logits from the largest down that a table holds
constexpr u64 EDGE = 1ull << 63;
template <class E>
__global__ __launch_bounds__(NP, 8) void sample_border_kernel(SampleArgs A, SamplePlan P) {
    constexpr int VL = Logits<E>::VL, HALF = 4;  // elements packed at a time
    __shared__ u64 block[SEG_BLOCKS];
    __shared__ u64 tab[STEPS];
    __shared__ Stage stage;
    __shared__ union {
        uint2 mine[NP / 64][64 * (HALF + 1)];
        u64 value[VALUES + 1];
    } U;
    __shared__ Scan scan;
    __shared__ BorderFound found;
    const int row = blockIdx.x / P.segs, seg = blockIdx.x % P.segs;
    const Set s = set_of(A, row);
    if (s.mode != ROW_NUCLEUS) return;
    const RowWs w = row_ws(A, P, row);
    u64 h[BINS_EACH];
    load_bins(w.hist, h);
    const u64 top = row_top(w, P.segs);
    Masses m;
    if (!top || !m.set(top_logit(top), s.T, A.vocab, tab)) return;
    const int i0 = seg * P.seg_len, i1 = min(i0 + P.seg_len, A.vocab);
    const int nb = max(0, (i1 - i0 + BLOCK - 1) / BLOCK);
    for (int i = threadIdx.x; i < nb; i += NP) block[i] = 0;
    const Logits<E> x = row_logits<E>(A, row);
    const First<E> f = first(x, i0, i1);
    m.fill(tab);
    stage.clear();
    int turn = 0;
    const BorderBin b = border_bin(h, s.p, scan, turn, found);  // (with barriers)
    const u64 least = m.least(s);
    const float floor = m.under(b.bin);
    const int lane = threadIdx.x & 63;
    if constexpr (sizeof(E) == 2) {
        // 16-bit logits have few values above the border: their masses from a table, by the distance to
        // the largest one in steps of a value (EDGE for those of the border's bin).  256 x 152064 in
        // bf16: 33 us, 37 us as below.
        constexpr int SHIFT = __is_same(E, __bf16) ? 16 : 13;
        const uint32_t at_M = __builtin_bit_cast(uint32_t, m.M), at_floor = __builtin_bit_cast(uint32_t, floor);
        const uint32_t flip = at_M >> 31 ? 0u : ~0u;  // (of one sign they grow apart upwards or downwards)
        const uint32_t values = (((at_floor ^ flip) - (at_M ^ flip)) >> SHIFT) + 1;
        if ((at_M ^ at_floor) >> 31 == 0 && values <= VALUES) {
            for (uint32_t i = threadIdx.x; i <= values; i += NP) {
                const Masses::At y = m.at(__builtin_bit_cast(float, at_M + (at_M >> 31 ? i << SHIFT : -(i << SHIFT))));
                const u64 v = m.mass(y);
                U.value[i] = i == values || y.bin() > b.bin ? 0 : y.bin() == b.bin ? EDGE : v >= least ? v : 0;
            }
            __syncthreads();
            each(x, f, i0, i1, [&](const float (&l)[VL], int i) {
                u64 v[VL], q = 0;
#pragma unroll
                for (int e = 0; e < VL; e++) {
                    const uint32_t far = ((__builtin_bit_cast(uint32_t, l[e]) ^ flip) - (at_M ^ flip)) >> SHIFT;
                    v[e] = U.value[l[e] >= floor ? far : values];
                    q += v[e];
                }
#pragma unroll
                for (int e = 0; e < VL; e++) {
                    const bool edge[1] = {(v[e] & EDGE) != 0};
                    stage.add(w, edge, [&](int) { return entry_of(key_of(l[e]), i + e); });
                }
                q &= EDGE - 1;  // (an even or odd number of EDGEs, and masses under 2^55)
                if (__any(q != 0)) {
                    q = wave_sum(q);
                    if (lane == 0) atomicAdd(&block[(i - i0) / BLOCK], q);
                }
            });
            stage.flush(w);  // (with barriers)
            for (int i = threadIdx.x; i < nb; i += NP) w.block[i0 / BLOCK + i] = block[i];
            return;
        }
    }
    // Most tokens lie below the border.  Each wave packs those that may not, then takes them 64 at a
    // time: with a nucleus of 9 % of the tokens the masses of all lanes' every token cost 1.7 times as much.
    uint2* const pack = U.mine[threadIdx.x >> 6];
    each(x, f, i0, i1, [&](const float (&l)[VL], int i) {
        int n = 0;
        u64 q = 0;
        auto take = [&](bool have, int j) {
            const uint2 t = pack[have ? j : 0];
            const float tl = __builtin_bit_cast(float, t.x);
            const Masses::At y = m.at(tl);
            const u64 v = m.mass(y);
            q += have && y.bin() < b.bin && v >= least ? v : 0;
            const bool edge[1] = {have && y.bin() == b.bin};
            stage.add(w, edge, [&](int) { return entry_of(key_of(tl), (int)t.y); });
        };
#pragma unroll
        for (int h = 0; h < VL; h += HALF) {
#pragma unroll
            for (int e = h; e < h + HALF; e++) {
                const bool in = l[e] >= floor;
                const u64 who = __ballot(in);
                if (in) pack[n + __popcll(who & ((1ull << lane) - 1))] = uint2{__builtin_bit_cast(uint32_t, l[e]), (uint32_t)(i + e)};
                n += __popcll(who);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            for (; n >= 64; n -= 64) take(true, n - 64 + lane);
        }
        if (n) take(lane < n, lane);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (__any(q != 0)) {
            q = wave_sum(q);
            if (lane == 0) atomicAdd(&block[(i - i0) / BLOCK], q);
        }
    });
    stage.flush(w);  // (with barriers)
    for (int i = threadIdx.x; i < nb; i += NP) w.block[i0 / BLOCK + i] = block[i];
}

// ---- 4: the token

// how far down the order the filters keep tokens: those above `key`, and the first `ties` (by
// index) of those at it
constexpr uint32_t ALL = 0xffffffffu;
struct Border {
    uint32_t key = 0;
    uint32_t ties = ALL;
};

constexpr int WAY_BITS = 11;         // bits of key or index that one step of a descent in kernel 4 settles
constexpr int WAYS = 1 << WAY_BITS;
constexpr int WAYS_EACH = WAYS / WT;
constexpr int FEW = WT;              // tokens that are put in order by comparing each with each
constexpr int FEWER = 128;           // of several keys, where another step (1.3 us) may leave less (256: 2 us)
constexpr int BATCH = 4;             // of them at a time: one wait for LDS
// where a bin lies: a worker takes consecutive ones, but the workers' first ones lie side by side, then
// their second ones (consecutive ones side by side would put 64 lanes on four banks)
__device__ __forceinline__ uint32_t place(uint32_t bin) { return (bin & (WAYS_EACH - 1)) * WT + bin / WAYS_EACH; }
struct RowShared {
    uint32_t count[WAYS];           // at place(bin); zero between steps
    u64 sum[WAYS];                  // the same
    u64 list[LIST + BATCH];         // zeros behind the last entry
    u64 few[2][FEW + BATCH];
    u64 block[SAMPLE_MAX_VOCAB / BLOCK];
    Scan scan;
    u64 part[NT / 64];
    u64 tab[STEPS];
    uint32_t tpart[NT / 64], lo_part[NT / 64], hi_part[NT / 64];
    u64 above, edge;
    uint32_t bin, left, few_n;
    int found;
    BorderFound border;
};

struct Row {
    const void* x;
    int type, V;
    __device__ __forceinline__ float at(int i) const {
        return type == JYHIP_T_F32   ? static_cast<const float*>(x)[i]
               : type == JYHIP_T_F16 ? (float)static_cast<const _Float16*>(x)[i]
                                     : (float)static_cast<const __bf16*>(x)[i];
    }
};

// the sum of v over the workgroup, in every thread
__device__ __forceinline__ u64 block_sum(RowShared& S, u64 v) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) S.part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < NT / 64; w++) v += S.part[w];
    return v;
}

// how many of the n entries of a list are greater (zeros behind them up to a multiple of BATCH)
__device__ __forceinline__ int rank_of(const u64* list, int n, u64 entry) {
    int rank = 0;
    for (int i = 0; i < n; i += BATCH) {
        u64 x[BATCH];
#pragma unroll
        for (int j = 0; j < BATCH; j++) x[j] = list[i + j];
#pragma unroll
        for (int j = 0; j < BATCH; j++) rank += x[j] > entry;
    }
    return rank;
}

// One step of a descent: of the bins in S (bin 0 the first in the order), the last one with a token in it
// and less than `want` above it, `above` lying above the first; it is the one that reaches `want`.
// Leaves the bin, what lies above it and its count; the bins are zero again.
__device__ __forceinline__ void choose(RowShared& S, int& turn, bool by_mass, u64 above, u64 want) {
    constexpr int PER = WAYS_EACH;
    const bool worker = threadIdx.x < WT;
    __syncthreads();
    uint32_t n[PER];
    u64 v[PER], sum = 0, total;
    if (worker)
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int b = j * WT + threadIdx.x;
            n[j] = S.count[b];
            v[j] = by_mass ? S.sum[b] : n[j];
            sum += v[j];
            S.count[b] = 0;
            if (by_mass) S.sum[b] = 0;
        }
    u64 run = above + S.scan.before(turn, sum, total);
    if (worker && (run < want || run == 0) && run + sum >= want)
#pragma unroll
        for (int j = 0; j < PER; j++) {
            if (n[j] && (run < want || run == 0) && run + v[j] >= want) {
                S.bin = threadIdx.x * PER + j;
                S.above = run;
                S.left = n[j];
            }
            run += v[j];
        }
    if (threadIdx.x == 0) S.few_n = 0;
    __syncthreads();
}

// the border at key `key`, whose tokens S.left are, each of mass `one`, S.above before them
__device__ __forceinline__ Border border_at(RowShared& S, u64 one, uint32_t key, bool by_mass, u64 want) {
    Border r;
    r.key = key;
    const u64 left = S.left;
    u64 ties;
    if (by_mass) {
        ties = S.above >= want ? 0 : one ? (want - S.above + one - 1) / one : left;
    } else {
        ties = want - S.above;
    }
    r.ties = ties < left ? (uint32_t)ties : ALL;
    if (r.ties == 0) r.ties = 1;  // (want == 0: the first token is kept all the same)
    return r;
}

// The border of the `want` first tokens in the order (by_mass: of the tokens before which less
// than `want` of mass lies; ties share what is left), by a radix descent over the whole row's keys,
// 11 bits at a time
__device__ __forceinline__ Border descend(RowShared& S, int& turn, const Row& R, const Masses& m, bool by_mass, u64 want) {
    uint32_t prefix = 0;
    u64 above = 0;
    for (int shift = 32 - WAY_BITS, nb = WAY_BITS; nb; shift -= nb) {
        const uint32_t mask = (1u << nb) - 1;
        const bool step = shift + nb < 32;
        for (int i = threadIdx.x; i < R.V; i += NT) {
            const float l = R.at(i);
            const uint32_t k = key_of(l);
            if (step && (k >> (shift + nb)) != prefix) continue;
            const uint32_t b = place(mask - ((k >> shift) & mask));
            atomicAdd(&S.count[b], 1u);
            if (by_mass) {
                const u64 q = m.mass_any(l);
                if (q) atomicAdd(&S.sum[b], q);
            }
        }
        choose(S, turn, by_mass, above, want);
        prefix = (step ? prefix << nb : 0) | (mask - S.bin);
        above = S.above;
        nb = min(nb, shift);
    }
    return border_at(S, prefix ? m.mass_any(logit_of(prefix)) : 0, prefix, by_mass, want);
}

// The index of the last tie that B keeps among the list's n tokens (those at B's key)
constexpr int INDEX_BITS = 22;
static_assert(SAMPLE_MAX_VOCAB == 1 << INDEX_BITS && INDEX_BITS <= 2 * WAY_BITS, "two steps over an index");
constexpr int LOW_BITS = INDEX_BITS - WAY_BITS;
template <int PER>
__device__ __forceinline__ uint32_t last_tie(RowShared& S, int& turn, const Border& B, int n) {
    if (B.ties == ALL) return ALL;
    uint32_t high = 0;
    u64 above = 0;
    for (int step = 0; step < 2; step++) {
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int i = j * NT + threadIdx.x;
            if (i >= n || (uint32_t)(S.list[i] >> 32) != B.key) continue;
            const uint32_t at = ~(uint32_t)S.list[i];
            if (step == 0 || at >> LOW_BITS == high) atomicAdd(&S.count[place(step ? at & ((1u << LOW_BITS) - 1) : at >> LOW_BITS)], 1u);
        }
        choose(S, turn, false, above, B.ties);
        if (step) break;
        high = S.bin;
        above = S.above;
    }
    return high << LOW_BITS | S.bin;
}

// The last kept one of the n entries in `list` (FEW at most, zeros behind them), `above` before them
__device__ __forceinline__ u64 last_of_few(RowShared& S, int& turn, const Masses& m, const u64* list, int n, bool by_mass,
                                           u64 above, u64 want) {
    const int me = threadIdx.x;
    if (me < FEW) {
        const u64 entry = me < n ? list[me] : 0;
        const int rank = rank_of(list, n, entry);
        if (me < n) S.few[1][rank] = entry;
    }
    __syncthreads();
    const u64 mine = me < n ? S.few[1][me] : 0;
    if (by_mass) {
        const u64 q = me < n ? m.mass(logit_of((uint32_t)(mine >> 32))) : 0;
        u64 total;
        const u64 before = above + S.scan.before(turn, q, total);
        if (me < n && (me == 0 || before < want) && (me + 1 == n || before + q >= want)) S.edge = mine;
    } else if (me < n && above + me + 1 == want) {
        S.edge = mine;
    }
    __syncthreads();
    return S.edge;
}

// The last kept one of the n tokens of the list, of which the first `want` are kept (by_mass: those
// before which less than `want` of mass lies), with `above` before them: the keys' range is divided
// by up to 2048 until few tokens are left, or one key.  A thread has at most PER of them.  ORDER: few
// are put in order.  (For the border of top-p alone it costs registers and saves nothing: its tokens of
// 16-bit logits have one or two keys.)
template <int PER, bool ORDER>
__device__ __forceinline__ u64 last_kept(RowShared& S, int& turn, const Masses& m, int n, bool by_mass, u64 above, u64 want) {
    if constexpr (ORDER)
        if (n <= FEWER) return last_of_few(S, turn, m, S.list, n, by_mass, above, want);
    uint32_t key[PER], lo = 0xffffffffu, hi = 0;
    u64 q[PER];
#pragma unroll
    for (int j = 0; j < PER; j++) {
        const int i = j * NT + threadIdx.x;
        key[j] = i < n ? (uint32_t)(S.list[i] >> 32) : 0;
        q[j] = by_mass && key[j] ? m.mass(logit_of(key[j])) : 0;
        if (key[j]) {
            lo = min(lo, key[j]);
            hi = max(hi, key[j]);
        }
    }
    const u64 far = wave_max((u64)hi << 32), near = wave_max((u64)(uint32_t)~lo);
    if ((threadIdx.x & 63) == 0) {
        S.lo_part[threadIdx.x >> 6] = ~(uint32_t)near;
        S.hi_part[threadIdx.x >> 6] = (uint32_t)(far >> 32);
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 64; w++) {
        lo = min(lo, S.lo_part[w]);
        hi = max(hi, S.hi_part[w]);
    }
    for (;;) {
        int shift = 0;  // keys per bin, as a power of two
        while (((hi - lo) >> shift) >= WAYS) shift++;
#pragma unroll
        for (int j = 0; j < PER; j++)
            if (key[j] && key[j] >= lo && key[j] <= hi) {
                const uint32_t b = place((hi - key[j]) >> shift);
                atomicAdd(&S.count[b], 1u);
                if (q[j]) atomicAdd(&S.sum[b], q[j]);
            }
        choose(S, turn, by_mass, above, want);
        above = S.above;
        const uint32_t top = hi - (S.bin << shift), low = top - ((1u << shift) - 1);
        lo = low > lo && low <= top ? low : lo;
        hi = top;
        const int left = (int)S.left;
        if constexpr (ORDER)
            if (left <= (shift ? FEWER : FEW)) {
#pragma unroll
                for (int j = 0; j < PER; j++)
                    if (key[j] && key[j] >= lo && key[j] <= hi) S.few[0][atomicAdd(&S.few_n, 1u)] = S.list[j * NT + threadIdx.x];
                if (threadIdx.x < BATCH) S.few[0][left + threadIdx.x] = 0;
                __syncthreads();
                return last_of_few(S, turn, m, S.few[0], left, by_mass, above, want);
            }
        if (shift == 0) {
            const Border B = border_at(S, m.mass(logit_of(top)), top, by_mass, want);
            return (u64)B.key << 32 | ~last_tie<PER>(S, turn, B, n);
        }
    }
}

// the kept mass of tokens with indices in [i0, i1), per wave in steps of 64, `ties` the ties before
// i0; find: the index at which the running sum passes `target`
struct Kept {
    u64 sum;
    uint32_t ties;
    int at;
};
__device__ __forceinline__ Kept walk(const Row& R, const Masses& m, const Border& B, u64 least, int i0, int i1, uint32_t ties,
                     bool find, u64 target) {
    const int lane = threadIdx.x & 63;
    Kept r{0, ties, -1};
    for (int i = i0; i < i1; i += 64) {
        const int j = i + lane;
        const float l = j < i1 ? R.at(j) : __builtin_nanf("");
        const uint32_t k = key_of(l);
        const bool tie = j < i1 && k == B.key;
        const u64 tm = __ballot(tie);
        const uint32_t rank = r.ties + __popcll(tm & ((1ull << lane) - 1));
        r.ties += __popcll(tm);
        const u64 v = m.mass_any(l);
        const u64 q = j < i1 && (k > B.key || (tie && rank < B.ties)) && v >= least ? v : 0;
        if (find) {
            u64 run = q;
            for (int d = 1; d < 64; d <<= 1) {
                const u64 o = __shfl_up(run, d);
                if (lane >= d) run += o;
            }
            const u64 hit = __ballot(q && r.sum + run > target);
            if (hit) {
                r.at = i + __builtin_ctzll(hit);
                return r;
            }
            r.sum += __shfl(run, 63);
        } else {
            r.sum += q;
        }
    }
    if (!find) r.sum = wave_sum(r.sum);
    return r;
}

__device__ __forceinline__ u64 target_of(float u, u64 total) {
    const double v = u > 0.0f ? (double)fminf(u, 0x1.fffffep-1f) : 0.0;
    return (u64)(v * (double)total);
}

// the whole row by this workgroup
__device__ __forceinline__ int pick_alone(RowShared& S, int& turn, const Row& R, const Masses& m, const Set& s, float u) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const u64 least = m.least(s);
    Border B;
    if (s.k > 0 && s.k < R.V) B = descend(S, turn, R, m, false, (u64)s.k);
    if (s.p < 1.0f) {
        u64 z = 0;
        for (int i = threadIdx.x; i < R.V; i += NT) {
            const float l = R.at(i);
            const uint32_t k = key_of(l);
            if (k > B.key || (k == B.key && B.ties == ALL)) z += m.mass_any(l);
        }
        z = block_sum(S, z);
        if (B.ties != ALL) z += B.ties * (B.key ? m.mass_any(logit_of(B.key)) : 0);
        const u64 want = (u64)ceil((s.p > 0.0f ? (double)s.p : 0.0) * (double)z);
        const Border C = descend(S, turn, R, m, true, want);
        if (C.key > B.key || (C.key == B.key && C.ties < B.ties)) B = C;
    }
    // the kept mass of each wave's run of indices, then the run and the index in it
    const int per = ((R.V + NT / 64 - 1) / (NT / 64) + 63) / 64 * 64;
    uint32_t mine = 0;
    const int i0 = min(wave * per, R.V), i1 = min(i0 + per, R.V);
    for (int i = i0 + lane; i < i1; i += 64) mine += key_of(R.at(i)) == B.key;
    for (int d = 32; d; d >>= 1) mine += __shfl_xor(mine, d);
    __syncthreads();
    if (lane == 0) S.tpart[wave] = mine;
    __syncthreads();
    uint32_t before = 0;
    for (int w = 0; w < wave; w++) before += S.tpart[w];
    const Kept kept = walk(R, m, B, least, i0, i1, before, false, 0);
    if (lane == 0) S.part[wave] = kept.sum;
    if (threadIdx.x == 0) S.found = -1;
    __syncthreads();
    u64 z = 0;
    for (int w = 0; w < NT / 64; w++) z += S.part[w];
    const u64 target = target_of(u, z);
    u64 run = 0;
    for (int w = 0; w < NT / 64; w++) {
        if (run + S.part[w] > target) {
            if (w == wave) {
                const Kept f = walk(R, m, B, least, i0, i1, before, true, target - run);
                if (lane == 0) S.found = f.at;
            }
            break;
        }
        run += S.part[w];
    }
    __syncthreads();
    return S.found;
}

// top-k, few candidates: the n in S.list, a thread each, every one compared with every other
__device__ __forceinline__ int pick_few(RowShared& S, int& turn, const Masses& m, const Set& s, int n, float u) {
    const int me = threadIdx.x;
    if (me < FEW) {
        const u64 entry = me < n ? S.list[me] : 0;
        const int rank = rank_of(S.list, n, entry);
        if (me < n) S.block[rank] = entry;
    }
    if (me == 0) S.found = 0x7fffffff;
    __syncthreads();
    n = min(n, s.k);
    const u64 mine = me < n ? S.block[me] : 0;
    const u64 q = me < n ? m.mass(logit_of((uint32_t)(mine >> 32))) : 0;
    bool keep = me < n;
    u64 z;
    if (s.p < 1.0f) {
        const u64 before = S.scan.before(turn, q, z);
        keep &= before < (u64)ceil((s.p > 0.0f ? (double)s.p : 0.0) * (double)z);
    }
    keep = (keep && q >= m.least(s)) || me == 0;
    const u64 kept = keep ? q : 0;
    const uint32_t idx = ~(uint32_t)mine;
    if (me < FEW) {
        S.list[me] = kept;
        S.count[me] = idx;
    }
    S.scan.before(turn, kept, z);  // (with a barrier)
    const u64 target = target_of(u, z);
    // the running sum up to each kept token's index (of all FEW places those without a token are zero)
    if (me < FEW) {
        u64 run = 0;
        for (int i = 0; i < n; i += BATCH) {
            u64 v[BATCH];
            uint32_t at[BATCH];
#pragma unroll
            for (int j = 0; j < BATCH; j++) {
                v[j] = S.list[i + j];
                at[j] = S.count[i + j];
            }
#pragma unroll
            for (int j = 0; j < BATCH; j++) run += at[j] <= idx ? v[j] : 0;
        }
        if (kept && run > target) atomicMin(&S.found, (int)idx);
    }
    __syncthreads();
    return S.found;
}
static_assert(FEW <= WAYS && FEW <= LIST && FEW <= SAMPLE_MAX_VOCAB / BLOCK, "one place for each");

// top-k, many candidates: the k first of the n in S.list, the border of top-p among them, then the token
// by its index, in two steps
__device__ __forceinline__ int pick_list(RowShared& S, int& turn, const Masses& m, const Set& s, int n, float u) {
    constexpr int PER = LIST / NT;
    if (n > s.k) {
        const u64 last = last_kept<PER, true>(S, turn, m, n, false, 0, (u64)s.k);
        u64 mine[PER];
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int i = j * NT + threadIdx.x;
            mine[j] = i < n ? S.list[i] : 0;
        }
        __syncthreads();  // (everyone has read the list and S.left)
        if (threadIdx.x == 0) S.left = 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < PER; j++)
            if (mine[j] >= last) S.list[atomicAdd(&S.left, 1u)] = mine[j];
        __syncthreads();
        n = S.left;
        if (threadIdx.x < BATCH) S.list[n + threadIdx.x] = 0;  // (read after the next barrier)
    }
    static_assert(STRIPES <= NT, "at most one of the k a thread");
    const u64 e = (int)threadIdx.x < n ? S.list[threadIdx.x] : 0;
    const uint32_t key = (uint32_t)(e >> 32), at = ~(uint32_t)e;
    const u64 q = e ? m.mass(logit_of(key)) : 0;
    bool kept = q && q >= m.least(s);
    if (s.p < 1.0f) {
        const u64 z = block_sum(S, q);
        const u64 want = (u64)ceil((s.p > 0.0f ? (double)s.p : 0.0) * (double)z);
        const u64 last = last_kept<1, true>(S, turn, m, n, true, 0, want);  // (by all threads)
        kept = kept && e >= last;
    }
    const u64 target = target_of(u, block_sum(S, kept ? q : 0));
    u64 above = 0;
    uint32_t high = 0;
    for (int step = 0; step < 2; step++) {
        if (kept && (step == 0 || at >> LOW_BITS == high)) {
            const uint32_t b = place(step ? at & ((1u << LOW_BITS) - 1) : at >> LOW_BITS);
            atomicAdd(&S.count[b], 1u);
            atomicAdd(&S.sum[b], q);
        }
        choose(S, turn, true, above, target + 1);  // (the first bin whose running sum exceeds the target)
        if (step) break;
        high = S.bin;
        above = S.above;
    }
    return (int)(high << LOW_BITS | S.bin);
}

// no top-k: the blocks' masses are in the workspace (with top-p those above the border's bin, whose
// tokens are the n in S.list; h: this thread's bins)
__device__ __forceinline__ int pick_blocks(RowShared& S, int& turn, const Row& R, const Masses& m, const Set& s, const RowWs& w,
                           int blocks, int n, const u64 (&h)[BINS_EACH], float u) {
    constexpr int PER = LIST / NT;
    const u64 least = m.least(s);
    u64 last = 0;
    for (int i = threadIdx.x; i < blocks; i += NT) S.block[i] = w.block[i];
    if (s.mode == ROW_NUCLEUS) {
        const BorderBin b = border_bin(h, s.p, S.scan, turn, S.border);
        last = n <= NT ? last_kept<1, false>(S, turn, m, n, true, b.above, b.want)
                       : last_kept<PER, false>(S, turn, m, n, true, b.above, b.want);
        // the border's tokens
        for (int i = threadIdx.x; i < n; i += NT) {
            const u64 e = S.list[i];
            if (e < last) continue;
            const u64 q = m.mass(logit_of((uint32_t)(e >> 32)));
            if (q && q >= least) atomicAdd(&S.block[~(uint32_t)e / BLOCK], q);
        }
    }
    __syncthreads();
    constexpr int EACH = SAMPLE_MAX_VOCAB / BLOCK / WT;  // blocks a worker
    u64 v[EACH], sum = 0, z;
    const int b0 = threadIdx.x * EACH;
    if (threadIdx.x < WT)
#pragma unroll
        for (int j = 0; j < EACH; j++) {
            v[j] = b0 + j < blocks ? S.block[b0 + j] : 0;
            sum += v[j];
        }
    u64 run = S.scan.before(turn, sum, z);
    const u64 target = target_of(u, z);
    if (threadIdx.x < WT && run <= target && run + sum > target)
#pragma unroll
        for (int j = 0; j < EACH; j++) {
            if (run <= target && run + v[j] > target) {
                S.bin = b0 + j;
                S.above = run;
            }
            run += v[j];
        }
    __syncthreads();
    // the block's tokens, two a thread; the wave whose sum reaches the target looks closer
    static_assert(BLOCK == 2 * NT, "two tokens a thread");
    const int i = (int)S.bin * BLOCK + threadIdx.x * 2;
    const u64 left = target - S.above;
    u64 q[2];
    for (int j = 0; j < 2; j++) {
        const float l = i + j < R.V ? R.at(i + j) : __builtin_nanf("");
        const u64 q1 = m.mass(l);
        q[j] = entry_of(key_of(l), i + j) >= last && q1 >= least ? q1 : 0;
    }
    const u64 mine = wave_sum(q[0] + q[1]);
    if ((threadIdx.x & 63) == 0) S.part[threadIdx.x >> 6] = mine;
    __syncthreads();
    run = 0;
    for (int w = 0; w < (int)(threadIdx.x >> 6); w++) run += S.part[w];
    if (run <= left && run + mine > left) {
        run += wave_scan(q[0] + q[1]) - q[0] - q[1];
        for (int j = 0; j < 2; j++) {
            if (run <= left && run + q[j] > left) S.found = i + j;
            run += q[j];
        }
    }
    __syncthreads();
    return S.found;
}

__global__ __launch_bounds__(NT) void sample_pick_kernel(SampleArgs A, SamplePlan P) {
    __shared__ RowShared S;
    const int row = blockIdx.x;
    const RowWs w = row_ws(A, P, row);
    // (read with the rest, before it is known how many there are and whether they are needed)
    const u64 e0 = w.list[threadIdx.x];
    u64 h[BINS_EACH];
    load_bins(w.hist, h);
    const uint32_t count = *w.count;
    const float u = A.u[row];
    const u64 top = row_top(w, P.segs);
    const Set s = set_of(A, row);
    if (s.mode == ROW_GREEDY || !top) {
        if (threadIdx.x == 0) A.ids[row] = top ? (int)~(uint32_t)top : -1;
        return;
    }
    Masses m;
    const bool plain = m.set(top_logit(top), s.T, A.vocab, S.tab);
    m.fill(S.tab);
    for (int i = threadIdx.x; i < WAYS; i += NT) {
        S.count[i] = 0;
        S.sum[i] = 0;
    }
    int turn = 0;
    const int n = s.mode == ROW_TOPK || s.mode == ROW_NUCLEUS ? (int)min(count, (uint32_t)LIST + 1) : 0;
    if (n <= LIST) {
        if ((int)threadIdx.x < n) S.list[threadIdx.x] = e0;
        for (int i = NT + threadIdx.x; i < n; i += NT) S.list[i] = w.list[i];
        if (threadIdx.x < BATCH) S.list[n + threadIdx.x] = 0;
    }
    __syncthreads();
    Row R;
    R.x = static_cast<const char*>(A.logits) + row * A.row_stride * (A.type == JYHIP_T_F32 ? 4 : 2);
    R.type = A.type;
    R.V = A.vocab;
    int id;
    if (s.mode == ROW_ALONE || n > LIST || !plain)
        id = pick_alone(S, turn, R, m, s, u);
    else if (s.mode == ROW_TOPK)
        id = n <= FEW ? pick_few(S, turn, m, s, n, u) : pick_list(S, turn, m, s, n, u);
    else
        id = pick_blocks(S, turn, R, m, s, w, P.blocks, n, h, u);
    if (threadIdx.x == 0) A.ids[row] = id;
}

__global__ void advance_kernel(int* ids, int* state, int at) {
    if (ids[at] < 0) {
        ids[at] = 0;
        state[2] = 1;
    }
    state[0] = at + 1;
    state[1] = 0;
}

template <class E>
void launch_type(const SampleArgs& A, const SamplePlan& P, hipStream_t st) {
    const unsigned grid = (unsigned)(A.rows * P.segs);
    sample_top_kernel<E><<<grid, NP, 0, st>>>(A, P);
    sample_mass_kernel<E><<<grid, NP, 0, st>>>(A, P);
    if (A.top_p) sample_border_kernel<E><<<grid, NP, 0, st>>>(A, P);
    sample_pick_kernel<<<A.rows, NT, 0, st>>>(A, P);
}

}  // namespace

size_t sample_workspace_bytes(int rows, int vocab) { return (size_t)rows * plan_of(rows, vocab).row_bytes; }

void launch_sample(const SampleArgs& A, hipStream_t st) {
    const SamplePlan P = plan_of(A.rows, A.vocab);
    if (A.type == JYHIP_T_F32)
        launch_type<float>(A, P, st);
    else if (A.type == JYHIP_T_F16)
        launch_type<_Float16>(A, P, st);
    else
        launch_type<__bf16>(A, P, st);
}

void launch_advance(int* ids, int* state, int at, hipStream_t st) { advance_kernel<<<1, 1, 0, st>>>(ids, state, at); }

}  // namespace jy
