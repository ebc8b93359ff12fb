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
#include <hip/hip_runtime.h>

#include "jy_device.h"
#include "jy_paged_device.h"
#include "jy_sample.h"

namespace jy {

namespace {

constexpr int NT = 1024;            // threads of a row's workgroup
constexpr int BINS = 2048;          // of one step of the radix descent: 11, 11, 10 bits of the key

// order-preserving bits of a logit; NaN counts as the lowest, -0 as 0
__device__ __forceinline__ uint32_t key_of(float x) {
    if (x != x) return 0;
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct Row {
    const void* x;
    int type, V;
    float M;           // the largest logit
    double inv_t;      // 1 / T
    double unit;       // 2^s
    __device__ __forceinline__ float at(int i) const {
        return type == JYHIP_T_F32   ? static_cast<const float*>(x)[i]
               : type == JYHIP_T_F16 ? (float)static_cast<const _Float16*>(x)[i]
                                     : (float)static_cast<const __bf16*>(x)[i];
    }
    __device__ __forceinline__ double e(float l) const {
        if (l == M) return 1.0;
        if (!(l > -__builtin_inff()) || M == __builtin_inff()) return 0.0;
        return exp(((double)l - (double)M) * inv_t);
    }
    __device__ __forceinline__ uint64_t mass(double e) const { return (uint64_t)__builtin_rint(e * unit); }
};

// how far down the order the filters keep tokens: those above `key`, and the first `ties` (by
// index) of those at it
struct Border {
    uint32_t key = 0;
    uint32_t ties = 0xffffffffu;
};

struct RowShared {
    uint32_t count[BINS];
    unsigned long long sum[BINS];
    unsigned long long part[NT / 64];
    uint32_t tpart[NT / 64];
    float fpart[NT / 64];
    int ipart[NT / 64];
    unsigned long long above_sum;
    uint32_t above_count, bin, left;
};

__device__ __forceinline__ unsigned long long wave_sum_u64(unsigned long long v) {
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// the sum of v over the workgroup, in every thread
__device__ __forceinline__ unsigned long long block_sum_u64(RowShared& S, unsigned long long v) {
    v = wave_sum_u64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) S.part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < NT / 64; w++) v += S.part[w];
    return v;
}

// The border of the `want` first tokens in the order (by_mass: of the tokens before which less
// than `want` units of mass lie; ties share what is left).  A radix descent over the keys: at each
// step the histogram of those with the prefix found so far.
__device__ Border descend(RowShared& S, const Row& R, bool by_mass, unsigned long long want) {
    uint32_t prefix = 0;
    unsigned long long above = 0;  // counted or weighed, over everything before the prefix
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
            const uint32_t b = (k >> shift) & mask;
            atomicAdd(&S.count[b], 1u);
            if (by_mass) atomicAdd(&S.sum[b], R.mass(R.e(l)));
        }
        __syncthreads();
        // the lowest bin that still has a kept token: the last one, from the top, with less than
        // `want` above it
        if (threadIdx.x == 0) {
            unsigned long long a = above, best_above = above;
            int best = -1;
            for (int b = (int)mask; b >= 0; b--) {
                if (!S.count[b]) continue;
                if (a >= want && best >= 0) break;
                best = b;
                best_above = a;
                a += by_mass ? S.sum[b] : S.count[b];
            }
            S.bin = (uint32_t)best;
            S.above_sum = best_above;
            S.left = S.count[best];
        }
        __syncthreads();
        prefix = step ? prefix << nb | S.bin : S.bin;
        above = S.above_sum;
    }
    Border r;
    r.key = prefix;
    const uint32_t left = S.left;
    unsigned long long ties;
    if (by_mass) {
        const unsigned long long one = S.sum[S.bin] / left;  // (equal logits have equal masses)
        ties = above >= want ? 0 : one ? (want - above + one - 1) / one : left;
    } else {
        ties = want - above;
    }
    r.ties = (uint32_t)(ties < left ? ties : left);
    if (r.ties == 0) r.ties = 1;  // (want == 0: the first token is kept all the same)
    __syncthreads();
    return r;
}

// the mass of the kept tokens with indices in [i0, i1), per wave in steps of 64, `ties` the ties
// before i0; find: the index at which the running sum passes `target` (-1: it does not)
struct Kept {
    unsigned long long sum;
    uint32_t ties;
    int at;
};
__device__ Kept walk(const Row& R, const Border& B, double min_e, int i0, int i1, uint32_t ties, bool find,
                     unsigned long long target) {
    const int lane = threadIdx.x & 63;
    Kept r{0, ties, -1};
    for (int i = i0; i < i1; i += 64) {
        const int j = i + lane;
        const float l = j < i1 ? R.at(j) : __builtin_nanf("");
        const uint32_t k = key_of(l);
        const bool tie = j < i1 && k == B.key;
        const unsigned long long tm = __ballot(tie);
        const uint32_t rank = r.ties + __popcll(tm & ((1ull << lane) - 1));
        r.ties += __popcll(tm);
        const double e = R.e(l);
        unsigned long long m = 0;
        if (j < i1 && (k > B.key || (tie && rank < B.ties)) && e >= min_e) m = R.mass(e);
        if (find) {
            unsigned long long run = m;
            for (int d = 1; d < 64; d <<= 1) {
                const unsigned long long o = __shfl_up(run, d);
                if (lane >= d) run += o;
            }
            const unsigned long long hit = __ballot(m && r.sum + run > target);
            if (hit) {
                r.at = i + __builtin_ctzll(hit);
                return r;
            }
            r.sum += __shfl(run, 63);
        } else {
            r.sum += m;
        }
    }
    if (!find) r.sum = wave_sum_u64(r.sum);
    return r;
}

__global__ __launch_bounds__(NT) void sample_row_kernel(SampleArgs A) {
    __shared__ RowShared S;
    const int row = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Row R;
    R.x = static_cast<const char*>(A.logits) + row * A.row_stride * (A.type == JYHIP_T_F32 ? 4 : 2);
    R.type = A.type;
    R.V = A.vocab;
    // the largest logit and its lowest index
    float top = -__builtin_inff();
    int at = -1;
    for (int i = threadIdx.x; i < R.V; i += NT) {
        const float l = R.at(i);
        if (l > top) {
            top = l;
            at = i;
        }
    }
    for (int d = 32; d; d >>= 1) {
        const float ot = __shfl_xor(top, d);
        const int oa = __shfl_xor(at, d);
        if (ot > top || (ot == top && oa >= 0 && (at < 0 || oa < at))) {
            top = ot;
            at = oa;
        }
    }
    if (lane == 0) {
        S.fpart[wave] = top;
        S.ipart[wave] = at;
    }
    __syncthreads();
    for (int w = 0; w < NT / 64; w++)
        if (S.fpart[w] > top || (S.fpart[w] == top && S.ipart[w] >= 0 && (at < 0 || S.ipart[w] < at))) {
            top = S.fpart[w];
            at = S.ipart[w];
        }
    const float T = A.temperature ? A.temperature[row] : 1.0f;
    if (!(T > 0.0f) || at < 0) {
        if (threadIdx.x == 0) A.ids[row] = at;
        return;
    }
    R.M = top;
    R.inv_t = 1.0 / (double)T;
    int s = 62;
    while ((R.V - 1) >> (62 - s)) s--;
    R.unit = (double)(1ull << s);

    const int k = A.top_k ? A.top_k[row] : 0;
    const float p = A.top_p ? A.top_p[row] : 1.0f;
    const float mp = A.min_p ? A.min_p[row] : 0.0f;
    const double min_e = mp > 0.0f ? fmin((double)mp, 1.0) : 0.0;
    Border B;
    if (k > 0 && k < R.V) B = descend(S, R, false, (unsigned long long)k);
    if (p < 1.0f) {
        unsigned long long z = 0;
        uint32_t n = 0;
        for (int i = threadIdx.x; i < R.V; i += NT) {
            const float l = R.at(i);
            const uint32_t kk = key_of(l);
            if (kk > B.key || (kk == B.key && B.ties == 0xffffffffu)) z += R.mass(R.e(l));
            (void)n;
        }
        z = block_sum_u64(S, z);
        if (B.ties != 0xffffffffu) {
            const uint32_t b = B.key;
            const float l = __builtin_bit_cast(float, b & 0x80000000u ? b & 0x7fffffffu : ~b);
            z += B.ties * R.mass(b ? R.e(l) : 0.0);
        }
        const double want = (p > 0.0f ? (double)p : 0.0) * (double)z;
        const Border C = descend(S, R, true, (unsigned long long)ceil(want));
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
    const Kept kept = walk(R, B, min_e, i0, i1, before, false, 0);
    if (lane == 0) S.part[wave] = kept.sum;
    __syncthreads();
    unsigned long long z = 0;
    for (int w = 0; w < NT / 64; w++) z += S.part[w];
    const float uf = A.u[row];
    const double u = uf > 0.0f ? (double)fminf(uf, 0x1.fffffep-1f) : 0.0;
    const unsigned long long target = (unsigned long long)(u * (double)z);
    unsigned long long run = 0;
    for (int w = 0; w < NT / 64; w++) {
        if (run + S.part[w] > target) {
            if (w == wave) {
                const Kept f = walk(R, B, min_e, i0, i1, before, true, target - run);
                if (lane == 0) A.ids[row] = f.at;
            }
            break;
        }
        run += S.part[w];
    }
}

}  // namespace

size_t sample_workspace_bytes(int, int) { return 0; }

void launch_sample(const SampleArgs& A, hipStream_t st) { sample_row_kernel<<<A.rows, NT, 0, st>>>(A); }

}  // namespace jy
