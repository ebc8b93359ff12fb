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
// A row whose candidates do not fit the list (k > 1024, or thousands of equal logits at the border)
// is done by its workgroup in kernel 4 alone, by a radix descent over the logits' bits.
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
constexpr int STEPS = 512;          // table entries per factor of two of mass
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
    while (p.segs < MAX_SEGS && (int64_t)rows * p.segs * 2 <= 1024 && p.segs * 2 <= p.blocks) p.segs *= 2;
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
    float* seg_max; // [MAX_SEGS]
    int* seg_arg;   // [MAX_SEGS]
    float* stripe;  // [STRIPES]
    uint32_t* count;
};
__device__ __forceinline__ RowWs row_ws(const SampleArgs& A, const SamplePlan& P, int row) {
    RowWs w;
    unsigned char* p = A.ws + (size_t)row * P.row_bytes;
    w.hist = reinterpret_cast<u64*>(p);
    w.list = w.hist + BINS;
    w.block = w.list + LIST;
    w.seg_max = reinterpret_cast<float*>(w.block + P.blocks);
    w.seg_arg = reinterpret_cast<int*>(w.seg_max + MAX_SEGS);
    w.stripe = reinterpret_cast<float*>(w.seg_arg + MAX_SEGS);
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

__device__ constexpr u64 kExp2[32] = JY_EXP2_TABLE;

// Masses of a row's logits, e 2^s.  With y = 512 (x - M) log2 e / T = k + r, k whole and |r| <= 1/2:
// 2^(k/512) from a table of 512 (2^s in it) and the exponent, times the Taylor terms of 2^(r/512) up
// to r^3 (the rest is under 9e-15).
struct Masses {
    float M, low;    // low: the logit whose mass is far under 2^-52, standing for all below it and NaN
    double c;        // 512 log2 e / T
    double unit;     // 2^s
    const u64* tab;  // [STEPS]
    // false: the largest logit is infinite or T so large that no such logit is finite (then c is 0
    // or M infinite, and only pick_alone() takes the row)
    __device__ __forceinline__ bool set(float top, float T, int vocab, const u64* table) {
        M = top;
        c = 512.0 * 1.4426950408889634074 / (double)T;
        low = (float)((double)M - 64.0 * 512.0 / c);
        int s = 51;
        while (s > 40 && (1ll << (62 - s)) < vocab) s--;
        unit = (double)(1ull << s);
        tab = table;
        return M < __builtin_inff() && low > -3.4e38f;
    }
    // entry i of the table: 2^(i/512) 2^s, from 2^(j/32) (its bits less j << 47, so adding any
    // j << 47 gives 2^(j/32)) and the Taylor terms of 2^r, |r| <= 1/64, up to r^5 (the rest is
    // under 2.3e-15)
    __device__ __forceinline__ void fill(u64* table) const {
        for (int i = threadIdx.x; i < STEPS; i += blockDim.x) table[i] = __builtin_bit_cast(u64, unit * exp2_slow(i / 512.0));
    }
    static __device__ __forceinline__ double exp2_slow(double y) {
        const double shift = 0x1.8p+52;
        double kd = __builtin_fma(y, 32.0, shift);
        const u64 ki = __builtin_bit_cast(u64, kd);
        kd -= shift;
        const double r = __builtin_fma(kd, -0.03125, y);
        double q = __builtin_fma(r, 0.0013333558146428443, 0.0096181291076284772);
        q = __builtin_fma(q, r, 0.055504108664821580);
        q = __builtin_fma(q, r, 0.24022650695910071);
        q = __builtin_fma(q, r, 0.69314718055994531);
        q = __builtin_fma(q, r, 1.0);
        return q * __builtin_bit_cast(double, kExp2[ki & 31u] + (ki << 47));
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
    __device__ __forceinline__ double scaled(const At& a) const {
        constexpr double L = 0.69314718055994531 / 512.0;
        double q = __builtin_fma(a.r, L * L * L / 6.0, L * L / 2.0);
        q = __builtin_fma(q, a.r, L);
        q = __builtin_fma(q, a.r, 1.0);
        const u64 t = tab[a.k & (STEPS - 1)] + ((u64)(uint32_t)((a.k >> 9) << 20) << 32);
        return q * __builtin_bit_cast(double, t);
    }
    __device__ __forceinline__ double scaled(float l) const { return scaled(at(l)); }
    // the nearest whole number of a scaled mass (under 2^52)
    static __device__ __forceinline__ u64 whole(double scaled) {
        return __builtin_bit_cast(u64, scaled + 0x1p+52) & 0xfffffffffffffull;
    }
    __device__ __forceinline__ u64 mass(float l) const { return whole(scaled(l)); }
    // the same for any M and T
    __device__ __forceinline__ double scaled_any(float l) const {
        if (l == M) return unit;
        if (!(l > -__builtin_inff()) || M == __builtin_inff()) return 0.0;
        const double y = ((double)l - (double)M) * (c / 512.0);
        return y > -64.0 ? unit * exp2_slow(y) : 0.0;
    }
    __device__ __forceinline__ u64 mass_any(float l) const { return whole(scaled_any(l)); }
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
// ones are read before f takes the present ones
template <class E, class F>
__device__ __forceinline__ void each(const Logits<E>& x, int i0, int i1, F&& f) {
    constexpr int VL = Logits<E>::VL, STEP = NP * VL;
    float a[VL], b[VL];
    int i = i0 + (int)threadIdx.x * VL;
    x.load(i, i1, a);
    for (int base = i0; base < i1; base += STEP, i += STEP) {
        if (base + STEP < i1) x.load(i + STEP, i1, b);
        f(a, i);
#pragma unroll
        for (int e = 0; e < VL; e++) a[e] = b[e];
    }
}

// the row's largest logit and its lowest index (-1: none), from its parts; every wave by itself
__device__ __forceinline__ void row_top(const RowWs& w, int segs, float& top, int& at) {
    const int lane = threadIdx.x & 63;
    top = lane < segs ? w.seg_max[lane] : -__builtin_inff();
    at = lane < segs ? w.seg_arg[lane] : -1;
    for (int d = 32; d; d >>= 1) {
        const float ot = __shfl_xor(top, d);
        const int oa = __shfl_xor(at, d);
        if (ot > top || (ot == top && oa >= 0 && (at < 0 || oa < at))) {
            top = ot;
            at = oa;
        }
    }
}

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
    __shared__ float part[2 * NP];
    __shared__ int arg[NP / 64];
    const int row = blockIdx.x / P.segs, seg = blockIdx.x % P.segs;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const RowWs w = row_ws(A, P, row);
    const Set s = set_of(A, row);
    const int i0 = seg * P.seg_len, i1 = min(i0 + P.seg_len, A.vocab);
    // each thread two maxima (even and odd elements): 1024 parts of the segment
    float top[2] = {-__builtin_inff(), -__builtin_inff()};
    int at = -1;
    const Logits<E> x = row_logits<E>(A, row);
    each<E>(x, i0, i1, [&](const float (&l)[VL], int i) {
#pragma unroll
        for (int e = 0; e < VL; e++) {
            if (l[e] > fmaxf(top[0], top[1])) at = i + e;
            top[e & 1] = fmaxf(top[e & 1], l[e]);
        }
    });
    if (s.mode == ROW_NUCLEUS)
        for (int i = seg * NP + threadIdx.x; i < BINS; i += P.segs * NP) w.hist[i] = 0;
    if (seg == 0 && threadIdx.x == 0) *w.count = 0;
    if (s.mode == ROW_TOPK) {
        part[threadIdx.x] = top[0];
        part[NP + threadIdx.x] = top[1];
        __syncthreads();
        const int mine = STRIPES / P.segs;
        for (int r = threadIdx.x; r < mine; r += NP) {
            float m = part[r];
            for (int j = r + mine; j < 2 * NP; j += mine) m = fmaxf(m, part[j]);
            w.stripe[seg * mine + r] = m;
        }
        __syncthreads();
    }
    float m = fmaxf(top[0], top[1]);
    for (int d = 32; d; d >>= 1) {
        const float om = __shfl_xor(m, d);
        const int oa = __shfl_xor(at, d);
        if (om > m || (om == m && oa >= 0 && (at < 0 || oa < at))) {
            m = om;
            at = oa;
        }
    }
    if (lane == 0) {
        part[wave] = m;
        arg[wave] = at;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int v = 1; v < NP / 64; v++)
            if (part[v] > m || (part[v] == m && arg[v] >= 0 && (at < 0 || arg[v] < at))) {
                m = part[v];
                at = arg[v];
            }
        w.seg_max[seg] = m;
        w.seg_arg[seg] = at;
    }
}

// A lower bound of the k-th largest of the row's stripe maxima, as a key: its leading 21 bits, the
// rest zero.  Every wave holds all maxima, 16 a lane, and counts those at or above one of seven
// thresholds: three bits a round.
struct Bound {
    int n[2][8];
};
__device__ uint32_t stripe_bound(Bound& S, const RowWs& w, int k) {
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

// ---- 2: top-k candidates, masses or the histogram
template <class E>
__global__ __launch_bounds__(NP) void sample_mass_kernel(SampleArgs A, SamplePlan P) {
    constexpr int VL = Logits<E>::VL;
    __shared__ union {
        u64 hist[BINS];
        Stage stage;
    } U;
    __shared__ u64 tab[STEPS];
    __shared__ Bound bound;
    u64* const hist = U.hist;
    const int row = blockIdx.x / P.segs, seg = blockIdx.x % P.segs;
    const Set s = set_of(A, row);
    if (s.mode == ROW_GREEDY || s.mode == ROW_ALONE) return;
    const RowWs w = row_ws(A, P, row);
    const int i0 = seg * P.seg_len, i1 = min(i0 + P.seg_len, A.vocab);
    const Logits<E> x = row_logits<E>(A, row);
    if (s.mode == ROW_TOPK) {
        U.stage.clear();
        const uint32_t b = max(stripe_bound(bound, w, s.k), 0x00800000u);  // (the key after -infinity's); has barriers
        each<E>(x, i0, i1, [&](const float (&l)[VL], int i) {
            bool mine[VL];
            uint32_t k[VL];
#pragma unroll
            for (int e = 0; e < VL; e++) {
                k[e] = key_of(l[e]);  // (past the end NaN, whose key is under any bound)
                mine[e] = k[e] >= b;
            }
            U.stage.add(w, mine, [&](int e) { return (u64)k[e] << 32 | (uint32_t)~(i + e); });
        });
        U.stage.flush(w);
        return;
    }
    float top;
    int at;
    row_top(w, P.segs, top, at);
    Masses m;
    if (at < 0 || !m.set(top, s.T, A.vocab, tab)) return;
    const bool bins = s.mode == ROW_NUCLEUS;
    const int nb = bins ? BINS : (i1 - i0 + BLOCK - 1) / BLOCK;
    for (int i = threadIdx.x; i < nb; i += NP) hist[i] = 0;
    m.fill(tab);
    __syncthreads();
    if (bins) {
        each<E>(x, i0, i1, [&](const float (&l)[VL], int) {
#pragma unroll
            for (int e = 0; e < VL; e++) {
                const Masses::At y = m.at(l[e]);
                const u64 q = Masses::whole(m.scaled(y));
                if (q) atomicAdd(&hist[y.bin()], q);
            }
        });
        __syncthreads();
        for (int i = threadIdx.x; i < BINS; i += NP)
            if (hist[i]) atomicAdd(&w.hist[i], hist[i]);
    } else {
        const double least = s.min_e * m.unit;
        each<E>(x, i0, i1, [&](const float (&l)[VL], int i) {
            u64 q = 0;
#pragma unroll
            for (int e = 0; e < VL; e++) {
                const double v = m.scaled(l[e]);
                q += v >= least ? Masses::whole(v) : 0;
            }
            q = wave_sum(q);
            if ((threadIdx.x & 63) == 0 && q) atomicAdd(&hist[(i - i0) / BLOCK], q);
        });
        __syncthreads();
        for (int i = threadIdx.x; i < nb; i += NP) w.block[i0 / BLOCK + i] = hist[i];
    }
}

// running sums over a workgroup of N threads
template <int N>
struct Scan {
    u64 part[N / 64];
    // (the sum before this thread, the total)
    __device__ __forceinline__ u64 before(u64 v, u64& total) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        u64 run = v;
        for (int d = 1; d < 64; d <<= 1) {
            const u64 o = __shfl_up(run, d);
            if (lane >= d) run += o;
        }
        __syncthreads();
        if (lane == 63) part[wave] = run;
        __syncthreads();
        u64 a = 0;
        total = 0;
        for (int i = 0; i < N / 64; i++) {
            if (i < wave) a += part[i];
            total += part[i];
        }
        return a + run - v;
    }
};

// The bin that the last kept token lies in: the last one, from the top, with mass in it and less than
// `want` = ceil(p total) above; `above` that mass, `total` all of it.  All threads return the same.
struct BorderBin {
    int bin;
    u64 above, want;
};
template <int N>
__device__ BorderBin border_bin(const u64* hist, float p, Scan<N>& scan, int* found, u64* found_above) {
    constexpr int PER = BINS / N;
    u64 h[PER], sum = 0, total;
#pragma unroll
    for (int j = 0; j < PER; j++) {
        h[j] = hist[threadIdx.x * PER + j];
        sum += h[j];
    }
    if (threadIdx.x == 0) *found = -1;
    u64 run = scan.before(sum, total);
    BorderBin b;
    b.want = (u64)ceil((p > 0.0f ? (double)p : 0.0) * (double)total);
    int mine = -1;
    u64 mine_above = 0;
#pragma unroll
    for (int j = 0; j < PER; j++) {
        if (h[j] && (run < b.want || run == 0)) {  // (run == 0: the first token is always kept)
            mine = threadIdx.x * PER + j;
            mine_above = run;
        }
        run += h[j];
    }
    if (mine >= 0) atomicMax(found, mine);
    __syncthreads();
    if (mine >= 0 && *found == mine) *found_above = mine_above;
    __syncthreads();
    b.bin = *found;
    b.above = *found_above;
    return b;
}

// ---- 3: top-p: the masses above the border's bin, its tokens into the list
template <class E>
__global__ __launch_bounds__(NP) void sample_border_kernel(SampleArgs A, SamplePlan P) {
    constexpr int VL = Logits<E>::VL;
    __shared__ u64 block[SAMPLE_MAX_VOCAB / BLOCK];
    __shared__ u64 tab[STEPS];
    __shared__ Stage stage;
    __shared__ Scan<NP> scan;
    __shared__ int found;
    __shared__ u64 found_above;
    const int row = blockIdx.x / P.segs, seg = blockIdx.x % P.segs;
    const Set s = set_of(A, row);
    if (s.mode != ROW_NUCLEUS) return;
    const RowWs w = row_ws(A, P, row);
    float top;
    int at;
    row_top(w, P.segs, top, at);
    Masses m;
    if (at < 0 || !m.set(top, s.T, A.vocab, tab)) return;
    const int i0 = seg * P.seg_len, i1 = min(i0 + P.seg_len, A.vocab);
    const int nb = max(0, (i1 - i0 + BLOCK - 1) / BLOCK);
    for (int i = threadIdx.x; i < nb; i += NP) block[i] = 0;
    m.fill(tab);
    stage.clear();
    const BorderBin b = border_bin<NP>(w.hist, s.p, scan, &found, &found_above);  // (with barriers)
    const double least = s.min_e * m.unit;
    const Logits<E> x = row_logits<E>(A, row);
    each<E>(x, i0, i1, [&](const float (&l)[VL], int i) {
        u64 q = 0;
        bool mine[VL];
#pragma unroll
        for (int e = 0; e < VL; e++) {
            const Masses::At y = m.at(l[e]);
            const int bin = y.bin();
            if (bin < b.bin) {
                const double v = m.scaled(y);
                q += v >= least ? Masses::whole(v) : 0;
            }
            mine[e] = bin == b.bin;
        }
        if (__any(q != 0)) {
            q = wave_sum(q);
            if ((threadIdx.x & 63) == 0) atomicAdd(&block[(i - i0) / BLOCK], q);
        }
        stage.add(w, mine, [&](int e) { return (u64)key_of(l[e]) << 32 | (uint32_t)~(i + e); });
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

struct RowShared {
    uint32_t count[BINS];
    u64 sum[BINS];
    u64 list[LIST];
    Scan<NT> scan;
    u64 part[NT / 64];
    u64 tab[STEPS];
    uint32_t tpart[NT / 64];
    u64 above;
    uint32_t bin, left;
    int found;
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

// One step of a descent: of the bins in S (bin 0 the highest keys), the last one with a token in it and
// less than `want` above it, `above` lying above the first.  Leaves bin, above and the bin's count.
__device__ void choose(RowShared& S, bool by_mass, u64 above, u64 want) {
    u64 v[2], total;
    const int b0 = threadIdx.x * 2;
    for (int j = 0; j < 2; j++) v[j] = by_mass ? S.sum[b0 + j] : S.count[b0 + j];
    u64 run = above + S.scan.before(v[0] + v[1], total);
    if (threadIdx.x == 0) S.found = -1;
    __syncthreads();
    int mine = -1;
    u64 mine_above = 0;
    for (int j = 0; j < 2; j++) {
        if (S.count[b0 + j] && (run < want || run == 0)) {
            mine = b0 + j;
            mine_above = run;
        }
        run += v[j];
    }
    if (mine >= 0) atomicMax(&S.found, mine);
    __syncthreads();
    if (mine >= 0 && S.found == mine) {
        S.bin = mine;
        S.above = mine_above;
        S.left = S.count[mine];
    }
    __syncthreads();
}

// the border at key `key`, whose tokens S.left are, each of mass `one`, S.above before them
__device__ Border border_at(RowShared& S, u64 one, uint32_t key, bool by_mass, u64 want) {
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
    __syncthreads();
    return r;
}

// The border of the `want` first tokens in the order (by_mass: of the tokens before which less
// than `want` of mass lies; ties share what is left), by a radix descent over the whole row's keys,
// 11, 11 and 10 bits at a time
__device__ Border descend(RowShared& S, const Row& R, const Masses& m, bool by_mass, u64 want) {
    uint32_t prefix = 0;
    u64 above = 0;
    const int bits[3] = {11, 11, 10};
    int shift = 32;
    for (int step = 0; step < 3; step++) {
        const int nb = bits[step];
        const uint32_t mask = (1u << nb) - 1;
        shift -= nb;
        __syncthreads();
        for (int i = threadIdx.x; i < BINS; i += NT) {
            S.count[i] = 0;
            S.sum[i] = 0;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < R.V; i += NT) {
            const float l = R.at(i);
            const uint32_t k = key_of(l);
            if (step && (k >> (shift + nb)) != prefix) continue;
            const uint32_t b = mask - ((k >> shift) & mask);
            atomicAdd(&S.count[b], 1u);
            if (by_mass) {
                const u64 q = m.mass_any(l);
                if (q) atomicAdd(&S.sum[b], q);
            }
        }
        __syncthreads();
        choose(S, by_mass, above, want);
        prefix = (step ? prefix << nb : 0) | (mask - S.bin);
        above = S.above;
    }
    return border_at(S, prefix ? m.mass_any(logit_of(prefix)) : 0, prefix, by_mass, want);
}

// the same border among the n tokens of the list, with `above` before them: the keys' range divided by
// up to 2048 until one key is left
__device__ Border descend_list(RowShared& S, const Masses& m, int n, bool by_mass, u64 above, u64 want) {
    uint32_t lo = 0xffffffffu, hi = 0;
    for (int i = threadIdx.x; i < n; i += NT) {
        const uint32_t k = (uint32_t)(S.list[i] >> 32);
        lo = min(lo, k);
        hi = max(hi, k);
    }
    for (int d = 32; d; d >>= 1) {
        lo = min(lo, (uint32_t)__shfl_xor((int)lo, d));
        hi = max(hi, (uint32_t)__shfl_xor((int)hi, d));
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        S.tpart[threadIdx.x >> 6] = lo;
        S.part[threadIdx.x >> 6] = hi;
    }
    __syncthreads();
    for (int w = 0; w < NT / 64; w++) {
        lo = min(lo, S.tpart[w]);
        hi = max(hi, (uint32_t)S.part[w]);
    }
    for (;;) {
        int shift = 0;  // keys per bin, as a power of two
        while (((hi - lo) >> shift) >= BINS) shift++;
        __syncthreads();
        for (int i = threadIdx.x; i < BINS; i += NT) {
            S.count[i] = 0;
            S.sum[i] = 0;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += NT) {
            const uint32_t k = (uint32_t)(S.list[i] >> 32);
            if (k < lo || k > hi) continue;
            const uint32_t b = (hi - k) >> shift;
            atomicAdd(&S.count[b], 1u);
            const u64 q = by_mass ? m.mass(logit_of(k)) : 0;
            if (q) atomicAdd(&S.sum[b], q);
        }
        __syncthreads();
        choose(S, by_mass, above, want);
        above = S.above;
        const uint32_t top = hi - (S.bin << shift);
        if (shift == 0) return border_at(S, m.mass(logit_of(top)), top, by_mass, want);
        const uint32_t low = top - ((1u << shift) - 1);
        lo = low > lo && low <= top ? low : lo;
        hi = top;
    }
}

// the index of the last tie that B keeps among the list's n tokens (those at B's key): the block of
// 2048 indices that it lies in, then the index
__device__ uint32_t last_tie(RowShared& S, const Border& B, int n) {
    if (B.ties == ALL) return ALL;
    uint32_t block = 0;
    u64 above = 0;
    for (int step = 0; step < 2; step++) {
        __syncthreads();
        for (int i = threadIdx.x; i < BINS; i += NT) S.count[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += NT) {
            const uint32_t at = ~(uint32_t)S.list[i];
            if ((uint32_t)(S.list[i] >> 32) == B.key && (step == 0 || at / BLOCK == block))
                atomicAdd(&S.count[step ? at % BLOCK : at / BLOCK], 1u);
        }
        __syncthreads();
        choose(S, false, above, B.ties);
        if (step) return block * BLOCK + S.bin;
        block = S.bin;
        above = S.above;
    }
    return 0;  // (not reached)
}

// the kept mass of tokens with indices in [i0, i1), per wave in steps of 64, `ties` the ties before
// i0; find: the index at which the running sum passes `target`
struct Kept {
    u64 sum;
    uint32_t ties;
    int at;
};
__device__ Kept walk(const Row& R, const Masses& m, const Border& B, double least, int i0, int i1, uint32_t ties,
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
        const double v = m.scaled_any(l);
        u64 q = 0;
        if (j < i1 && (k > B.key || (tie && rank < B.ties)) && v >= least) q = Masses::whole(v);
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
__device__ int pick_alone(RowShared& S, const Row& R, const Masses& m, const Set& s, float u) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const double least = s.min_e * m.unit;
    Border B;
    if (s.k > 0 && s.k < R.V) B = descend(S, R, m, false, (u64)s.k);
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
        const Border C = descend(S, R, m, true, want);
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
constexpr int FEW = 256;
__device__ int pick_few(RowShared& S, const Masses& m, const Set& s, int n, float u) {
    const int me = threadIdx.x;
    const u64 entry = me < n ? S.list[me] : 0;
    int rank = 0;
    if (me < n)
#pragma unroll 8
        for (int i = 0; i < n; i++) rank += S.list[i] > entry;
    __syncthreads();
    if (me < n) S.list[rank] = entry;
    __syncthreads();
    n = min(n, s.k);
    const u64 mine = me < n ? S.list[me] : 0;
    const double v = me < n ? m.scaled(logit_of((uint32_t)(mine >> 32))) : 0.0;
    const u64 q = Masses::whole(v);
    u64 z;
    const u64 before = S.scan.before(q, z);
    bool keep = me < n;
    if (s.p < 1.0f) keep &= before < (u64)ceil((s.p > 0.0f ? (double)s.p : 0.0) * (double)z);
    keep = (keep && v >= s.min_e * m.unit) || me == 0;
    const u64 kept = keep ? q : 0;
    const uint32_t idx = ~(uint32_t)mine;
    S.sum[me] = kept;
    S.count[me] = idx;
    if (me == 0) S.found = 0x7fffffff;
    S.scan.before(kept, z);  // (with barriers)
    const u64 target = target_of(u, z);
    // the running sum up to each kept token's index
    if (kept) {
        u64 run = 0;
#pragma unroll 8
        for (int i = 0; i < n; i++) run += S.count[i] <= idx ? S.sum[i] : 0;
        if (run > target) atomicMin(&S.found, (int)idx);
    }
    __syncthreads();
    return S.found;
}

// top-k, many candidates: the border among the n in S.list, then the token by histograms over the
// indices' blocks and within the block
__device__ int pick_list(RowShared& S, const Masses& m, const Set& s, int n, float u) {
    const double least = s.min_e * m.unit;
    Border B;
    if (n > s.k) B = descend_list(S, m, n, false, 0, (u64)s.k);
    uint32_t cut = last_tie(S, B, n);
    auto kept = [&](u64 e) {
        const uint32_t k = (uint32_t)(e >> 32);
        return k > B.key || (k == B.key && ~(uint32_t)e <= cut);
    };
    if (s.p < 1.0f) {
        u64 z = 0;
        for (int i = threadIdx.x; i < n; i += NT)
            if (kept(S.list[i])) z += m.mass(logit_of((uint32_t)(S.list[i] >> 32)));
        z = block_sum(S, z);
        const u64 want = (u64)ceil((s.p > 0.0f ? (double)s.p : 0.0) * (double)z);
        const Border C = descend_list(S, m, n, true, 0, want);
        if (C.key > B.key || (C.key == B.key && C.ties < B.ties)) {
            B = C;
            cut = last_tie(S, B, n);
        }
    }
    u64 target = 0, above = 0;
    uint32_t block = 0;
    for (int step = 0; step < 2; step++) {
        __syncthreads();
        for (int i = threadIdx.x; i < BINS; i += NT) S.sum[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += NT) {
            const u64 e = S.list[i];
            const uint32_t at = ~(uint32_t)e;
            if (!kept(e) || (step && at / BLOCK != block)) continue;
            const double v = m.scaled(logit_of((uint32_t)(e >> 32)));
            const u64 q = v >= least ? Masses::whole(v) : 0;
            if (q) atomicAdd(&S.sum[step ? at % BLOCK : at / BLOCK], q);
        }
        __syncthreads();
        u64 v[2], z;
        const int b0 = threadIdx.x * 2;
        for (int j = 0; j < 2; j++) v[j] = S.sum[b0 + j];
        u64 run = above + S.scan.before(v[0] + v[1], z);
        if (step == 0) target = target_of(u, z);
        for (int j = 0; j < 2; j++) {
            if (run <= target && run + v[j] > target) {
                S.bin = b0 + j;
                S.above = run;
            }
            run += v[j];
        }
        __syncthreads();
        if (step) break;
        block = S.bin;
        above = S.above;
    }
    return (int)(block * BLOCK + S.bin);
}

// no top-k: the blocks' masses are in the workspace (with top-p those above the border's bin, whose
// tokens are the n in S.list)
__device__ int pick_blocks(RowShared& S, const Row& R, const Masses& m, const Set& s, const RowWs& w, int blocks, int n,
                           float u) {
    const double least = s.min_e * m.unit;
    Border B;
    uint32_t cut = ALL;
    if (s.mode == ROW_NUCLEUS) {
        const BorderBin b = border_bin<NT>(w.hist, s.p, S.scan, &S.found, &S.above);
        B = descend_list(S, m, n, true, b.above, b.want);
        cut = last_tie(S, B, n);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < blocks; i += NT) S.sum[i] = w.block[i];
    __syncthreads();
    // the border's tokens
    if (s.mode == ROW_NUCLEUS) {
        for (int i = threadIdx.x; i < n; i += NT) {
            const uint32_t k = (uint32_t)(S.list[i] >> 32), i1 = ~(uint32_t)S.list[i];
            if (k < B.key || (k == B.key && i1 > cut)) continue;
            const double v = m.scaled(logit_of(k));
            const u64 q = v >= least ? Masses::whole(v) : 0;
            if (q) atomicAdd(&S.sum[i1 / BLOCK], q);
        }
        __syncthreads();
    }
    static_assert(SAMPLE_MAX_VOCAB / BLOCK <= 2 * NT && BINS >= 2 * NT, "two blocks a thread");
    u64 v[2], z;
    const int b0 = threadIdx.x * 2;
    for (int j = 0; j < 2; j++) v[j] = b0 + j < blocks ? S.sum[b0 + j] : 0;
    u64 run = S.scan.before(v[0] + v[1], z);
    const u64 target = target_of(u, z);
    for (int j = 0; j < 2; j++) {
        if (run <= target && run + v[j] > target) {
            S.bin = b0 + j;
            S.above = run;
        }
        run += v[j];
    }
    __syncthreads();
    const int i0 = (int)S.bin * BLOCK;
    const u64 left = target - S.above;
    const int i = i0 + threadIdx.x * 2;
    u64 q[2], total;
    for (int j = 0; j < 2; j++) {
        const float l = i + j < R.V ? R.at(i + j) : __builtin_nanf("");
        const uint32_t k = key_of(l);
        const double v = m.scaled(l);
        const bool keep = k > B.key || (k == B.key && (uint32_t)(i + j) <= cut);
        q[j] = keep && v >= least ? Masses::whole(v) : 0;
    }
    run = S.scan.before(q[0] + q[1], total);
    if (threadIdx.x == 0) S.found = -1;
    __syncthreads();
    for (int j = 0; j < 2; j++) {
        if (run <= left && run + q[j] > left) S.found = i + j;
        run += q[j];
    }
    __syncthreads();
    return S.found;
}

__global__ __launch_bounds__(NT) void sample_pick_kernel(SampleArgs A, SamplePlan P) {
    __shared__ RowShared S;
    const int row = blockIdx.x;
    const RowWs w = row_ws(A, P, row);
    const Set s = set_of(A, row);
    float top;
    int at;
    row_top(w, P.segs, top, at);
    if (s.mode == ROW_GREEDY || at < 0) {
        if (threadIdx.x == 0) A.ids[row] = at;
        return;
    }
    Masses m;
    const bool plain = m.set(top, s.T, A.vocab, S.tab);
    m.fill(S.tab);
    const int n = s.mode == ROW_TOPK || s.mode == ROW_NUCLEUS ? (int)min(*w.count, (uint32_t)LIST + 1) : 0;
    if (n <= LIST)
        for (int i = threadIdx.x; i < n; i += NT) S.list[i] = w.list[i];
    __syncthreads();
    Row R;
    R.x = static_cast<const char*>(A.logits) + row * A.row_stride * (A.type == JYHIP_T_F32 ? 4 : 2);
    R.type = A.type;
    R.V = A.vocab;
    const float u = A.u[row];
    int id;
    if (s.mode == ROW_ALONE || n > LIST || !plain)
        id = pick_alone(S, R, m, s, u);
    else if (s.mode == ROW_TOPK)
        id = n <= FEW ? pick_few(S, m, s, n, u) : pick_list(S, m, s, n, u);
    else
        id = pick_blocks(S, R, m, s, w, P.blocks, n, u);
    if (threadIdx.x == 0) A.ids[row] = id;
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

}  // namespace jy
