// jy_evict.hip — which positions of a cache stay by their accumulated weights, and their way to new pages.
//
// Selection: a workgroup per (sequence, kv head).  A weight's bits become a number that rises with it, and the
// need-th largest is found by three counts over its digits (12, 10 and 10 bits, bins in LDS, whole numbers: the
// order of the atomics does not matter); the first digit is sign, exponent and three bits of the fraction, so
// that the weights of a sequence spread over dozens of bins.  A last pass over the positions in order takes
// what lies above that weight, of those equal to it the first, and the recent ones.  Up to 35840 positions the
// numbers stay in LDS and the weights are read once, 16 of a thread under way at a time.
// A chain of passes with barriers bounds it: 32 sequences of 1100 to 4099, 8 heads, 15 us; one of 32769, 4 heads, 35 us.
// Moving: 16 lanes a vector, key and value together, bytes as they are (1024 positions
// of those 32 sequences in int8: 138 MB in and out in 39 us, 3.5 TB/s).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "jy_device.h"
#include "jy_paged_device.h"

namespace jy {

namespace {

typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
typedef float f4_t __attribute__((ext_vector_type(4), aligned(4)));  // (four elements from any)

constexpr int NT = 1024, PER = 4;  // threads; positions a thread takes side by side
constexpr int AHEAD = 4;           // and so many times at once
constexpr int BINS = 4096;
constexpr int kHeld = 140 * 1024;  // bytes of LDS for ranks, beside the bins

struct EvictArgs {
    Eviction E;
    int ps_log2;
};

// rises with the weight, from 1 on: NaN lowest, then -infinity .. +infinity, both zeros the same; and back
__device__ __forceinline__ uint32_t rank_of(float w) {
    if (!(w == w)) return 1;
    const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float weight_of(uint32_t r) {
    return r == 1 ? __builtin_nanf("") : __builtin_bit_cast(float, r & 0x80000000u ? r ^ 0x80000000u : ~r);
}

// inclusive sum over the wave's lanes by DPP moves (within rows of 16, then each row's last to those behind it)
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
#if defined(__HIP_DEVICE_COMPILE__)
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);
#endif
    return v;
}

// exclusive sums over the workgroup's threads, of N numbers at once, and the whole
template <int N>
__device__ __forceinline__ void scan(uint32_t (&v)[N], uint32_t (*part)[NT / 64], uint32_t (&total)[N]) {
#if defined(__HIP_DEVICE_COMPILE__)
    static_assert(NT == 1024, "one row of lanes holds the waves' sums");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t s[N];
#pragma unroll
    for (int i = 0; i < N; i++) s[i] = wave_scan(v[i]);
    __syncthreads();  // (the last scan's parts are read)
    if (lane == 63)
#pragma unroll
        for (int i = 0; i < N; i++) part[i][wave] = s[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        const uint32_t all = wave_scan(part[i][lane & 15]);  // (lane 15 has the whole)
        total[i] = (uint32_t)__builtin_amdgcn_readlane((int)all, 15);
        const uint32_t before = wave ? (uint32_t)__builtin_amdgcn_readlane((int)all, wave - 1) : 0u;
        v[i] = before + s[i] - v[i];
    }
#endif
}

// The bin (into found[0]) in which the left-th largest lies, counted from the largest bin down; how many lie above it.
__device__ __forceinline__ uint32_t border(const uint32_t* bins, int size, uint32_t left, uint32_t (*part)[NT / 64], uint32_t* found) {
    const int per = (size + NT - 1) / NT;  // thread t has bins size - 1 - t per and down
    uint32_t own = 0;
    for (int i = 0; i < per; i++) {
        const int b = size - 1 - ((int)threadIdx.x * per + i);
        own += b >= 0 ? bins[b] : 0;
    }
    uint32_t at[1] = {own}, total[1];
    scan<1>(at, part, total);
    uint32_t above = at[0];
    if (above < left && above + own >= left) {
        for (int i = 0; i < per; i++) {
            const int b = size - 1 - ((int)threadIdx.x * per + i);
            if (above + bins[b] >= left) {
                found[0] = (uint32_t)b;
                found[1] = above;
                break;
            }
            above += bins[b];
        }
    }
    __syncthreads();
    return found[1];
}

// HELD: the ranks of all positions stay in LDS (n of them behind the bins), so the weights are read once; else each
// pass reads them again.
template <bool HELD>
__global__ __launch_bounds__(NT) void evict_select_kernel(EvictArgs K) {
    extern __shared__ uint32_t ranks[];
    __shared__ uint32_t bins[BINS];
    __shared__ uint32_t part[AHEAD][NT / 64];
    __shared__ uint32_t found[2];
    const Eviction& E = K.E;
    const int nkv = E.P.num_kv_heads, s = blockIdx.x / nkv, h = blockIdx.x - s * nkv;
    const int n = max(min(E.lens[s], E.cap), 0), late = max(n - E.recent, 0);
    const float* const w = E.weights + s * E.seq_stride + h * E.head_stride;
    const int* const table = E.M.tables + (int64_t)s * E.M.stride;

    // the ranks of positions j .. j + 3 (j a multiple of 4: one page), 0 where there is none
    struct Four {
        float w[4];
        int page;
    };
    auto ask = [&](int j) {
        Four f;
        f.page = j < n ? table[j >> K.ps_log2] : -1;
        if (j < n && j + 4 <= E.weights_len) {
            const f4_t v = *reinterpret_cast<const f4_t*>(w + j);
#pragma unroll
            for (int e = 0; e < 4; e++) f.w[e] = v[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) f.w[e] = j + e < min(n, E.weights_len) ? w[j + e] : 0.0f;
        }
        return f;
    };
    auto ranked = [&](const Four& f, int j, uint32_t (&r)[4]) {
#pragma unroll
        for (int e = 0; e < 4; e++) r[e] = j + e < n && (unsigned)f.page < (unsigned)E.P.num_pages ? rank_of(f.w[e]) : 0u;
    };
    auto get = [&](int j, uint32_t (&r)[4]) {
        if constexpr (HELD) {
            const u4_t v = *reinterpret_cast<const u4_t*>(ranks + j);
#pragma unroll
            for (int e = 0; e < 4; e++) r[e] = v[e];
        } else {
            ranked(ask(j), j, r);
        }
    };
    auto count = [&](uint32_t r, int shift, int bits) { atomicAdd(&bins[(r >> shift) & ((1u << bits) - 1u)], 1u); };

    // how many positions there are and how many of them are recent, and the first digits of the others: 12 bits
    for (int i = threadIdx.x; i < BINS; i += NT) bins[i] = 0;
    __syncthreads();
    uint32_t early = 0, latest = 0;
    for (int c0 = 0; c0 < n; c0 += NT * PER * AHEAD) {
        Four f[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; a++) f[a] = ask(c0 + (a * NT + (int)threadIdx.x) * PER);
#pragma unroll
        for (int a = 0; a < AHEAD; a++) {
            const int j = c0 + (a * NT + (int)threadIdx.x) * PER;
            if (j >= n) continue;
            uint32_t r[4];
            ranked(f[a], j, r);
            if constexpr (HELD) *reinterpret_cast<u4_t*>(ranks + j) = u4_t{r[0], r[1], r[2], r[3]};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (r[e] == 0) continue;
                if (j + e < late) {
                    early++;
                    count(r[e], 20, 12);
                } else {
                    latest++;
                }
            }
        }
    }
    uint32_t counts[2] = {early, latest}, sums[2];
    scan<2>(counts, part, sums);
    const uint32_t old = sums[0], recent = sums[1];
    const int there = (int)(old + recent), stay = min(E.keep, there);
    const bool all = there <= E.keep;

    // the need-th largest rank among the old positions: its digits from the top
    const uint32_t need = all ? 0 : (uint32_t)stay - recent;
    uint32_t top = 0, ties = 0;
    if (need > 0) {
        uint32_t left = need;
        left -= border(bins, BINS, left, part, found);
        top = found[0] << 20;
#pragma unroll
        for (int shift = 10; shift >= 0; shift -= 10) {
            __syncthreads();
            for (int i = threadIdx.x; i < 1024; i += NT) bins[i] = 0;
            __syncthreads();
            for (int c0 = 0; c0 < late; c0 += NT * PER * AHEAD) {
                uint32_t r[AHEAD][4];
#pragma unroll
                for (int c = 0; c < AHEAD; c++) {
                    const int j = c0 + (c * NT + (int)threadIdx.x) * PER;
#pragma unroll
                    for (int e = 0; e < 4; e++) r[c][e] = 0;
                    if (j < late) get(j, r[c]);
                }
#pragma unroll
                for (int c = 0; c < AHEAD; c++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (r[c][e] >> (shift + 10) == top >> (shift + 10) && r[c][e] &&
                            c0 + (c * NT + (int)threadIdx.x) * PER + e < late)
                            count(r[c][e], shift, 10);
            }
            __syncthreads();
            left -= border(bins, 1024, left, part, found);
            top |= found[0] << shift;
        }
        ties = left;  // of those whose rank is the border's, the first
    }

    int* const kept = E.kept + (int64_t)blockIdx.x * E.keep;
    float* const to = E.new_weights ? E.new_weights + s * E.new_seq_stride + h * E.new_head_stride : nullptr;
    uint32_t above = 0, equal = 0;  // positions over the border and on it, so far
    for (int c0 = 0; c0 < n; c0 += NT * PER * AHEAD) {
        uint32_t r[AHEAD][4], before[AHEAD], total[AHEAD];
        uint32_t over[AHEAD], on[AHEAD];  // a bit for each of the four
#pragma unroll
        for (int c = 0; c < AHEAD; c++) {
            const int j0 = c0 + (c * NT + (int)threadIdx.x) * PER;
#pragma unroll
            for (int e = 0; e < 4; e++) r[c][e] = 0;
            if (j0 < n) get(j0, r[c]);
            over[c] = on[c] = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const bool is = r[c][e] && (all || j0 + e >= late || (need > 0 && r[c][e] > top));
                over[c] |= (uint32_t)is << e;
                on[c] |= (uint32_t)(r[c][e] && !is && need > 0 && r[c][e] == top) << e;
            }
            before[c] = (uint32_t)__builtin_popcount(over[c]) | (uint32_t)__builtin_popcount(on[c]) << 16;  // (4096 of each at most)
        }
        scan<AHEAD>(before, part, total);  // (all of these positions' weights are read by now)
#pragma unroll
        for (int c = 0; c < AHEAD; c++) {
            const int j0 = c0 + (c * NT + (int)threadIdx.x) * PER;
            uint32_t a = above + (before[c] & 0xffffu), e0 = equal + (before[c] >> 16);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const bool is_over = over[c] >> e & 1, is_on = on[c] >> e & 1;
                if (is_over || (is_on && e0 < ties)) {
                    const uint32_t at = a + min(e0, ties);
                    if constexpr (HELD) {
                        ranks[at] = (uint32_t)(j0 + e);  // (over numbers that are used up: at is at most j0 + e)
                    } else {
                        kept[at] = j0 + e;
                        if (to && (int)at < E.new_weights_len) to[at] = weight_of(r[c][e]);
                    }
                }
                a += is_over;
                e0 += is_on;
            }
            above += total[c] & 0xffffu;
            equal += total[c] >> 16;
        }
    }
    __syncthreads();
    if constexpr (HELD) {  // the list as it lies: whole lines leave, where lanes scattered over the positions took 18 us for 32769
        for (int c0 = 0; c0 < stay; c0 += NT * AHEAD) {
            float x[AHEAD];
#pragma unroll
            for (int c = 0; c < AHEAD; c++) {
                const int i = c0 + c * NT + (int)threadIdx.x;
                x[c] = 0.0f;
                if (i < stay) {
                    const int j = (int)ranks[i];
                    kept[i] = j;
                    if (to && j < E.weights_len) x[c] = w[j];
                }
            }
            __syncthreads();  // (new weights may take the place of the old: they are read first, and later ones lie further on)
#pragma unroll
            for (int c = 0; c < AHEAD; c++) {
                const int i = c0 + c * NT + (int)threadIdx.x;
                if (to && i < min(stay, E.new_weights_len)) to[i] = x[c];
            }
        }
    }
    for (int i = stay + threadIdx.x; i < E.keep; i += NT) kept[i] = -1;
    if (to)
        for (int i = stay + threadIdx.x; i < E.new_weights_len; i += NT) to[i] = 0.0f;
    if (h == 0 && threadIdx.x == 0) E.new_lens[s] = stay;
}

// where a head's vector of a position lies in the pool (-1: nowhere)
__device__ __forceinline__ int64_t vector_at(const Eviction& E, const PageMap& M, int ps_log2, int s, int h, int pos) {
    const int64_t slot = slot_of(M, E.P.num_pages, ps_log2, s, pos);
    if (slot < 0) return -1;
    return (((slot >> ps_log2) * E.P.num_kv_heads + h) << ps_log2) + (slot & ((1 << ps_log2) - 1));
}

// 16 lanes take VECS vectors, keys and values, whose places are looked up together: a look-up is three loads, one
// after the other, and there has to be enough under way meanwhile.
constexpr int VECS = 2;
template <int UNITS>
__global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs K, int groups, int vec16, int words) {
    const Eviction& E = K.E;
    const unsigned id = blockIdx.x * 16 + (threadIdx.x >> 4);
    const unsigned head = id / groups, lane = threadIdx.x & 15;
    const int i0 = (int)(id - head * groups) * VECS, nkv = E.P.num_kv_heads, width = min(E.keep, E.cap);
    if (head >= (unsigned)E.M.nseq * nkv) return;
    const int s = head / nkv, h = head % nkv;
    int64_t from[VECS], to[VECS];
    int pos[VECS];
#pragma unroll
    for (int v = 0; v < VECS; v++) pos[v] = i0 + v < width ? E.kept[(int64_t)head * E.keep + i0 + v] : -1;
#pragma unroll
    for (int v = 0; v < VECS; v++) {
        from[v] = vector_at(E, E.M, K.ps_log2, s, h, pos[v]);
        to[v] = pos[v] < 0 ? -1 : vector_at(E, E.to, K.ps_log2, s, h, i0 + v);
    }
    // 16 bytes a lane, the key's first; scales as words
    u4_t x[VECS][UNITS];
    float y[VECS];
#pragma unroll
    for (int v = 0; v < VECS; v++) {
        const bool is = from[v] >= 0 && to[v] >= 0;
#pragma unroll
        for (int c = 0; c < UNITS; c++) {
            const int u = 16 * c + (int)lane;
            if (is && u < 2 * vec16)
                x[v][c] = static_cast<const u4_t*>(u < vec16 ? E.P.k : E.P.v)[from[v] * vec16 + (u < vec16 ? u : u - vec16)];
        }
        const int u = lane;  // (at most 8 words a vector)
        if (is && u < 2 * words) y[v] = (u < words ? E.P.k_scale : E.P.v_scale)[from[v] * words + (u < words ? u : u - words)];
    }
#pragma unroll
    for (int v = 0; v < VECS; v++) {
        const bool is = from[v] >= 0 && to[v] >= 0;
#pragma unroll
        for (int c = 0; c < UNITS; c++) {
            const int u = 16 * c + (int)lane;
            if (is && u < 2 * vec16)
                static_cast<u4_t*>(u < vec16 ? E.P.k : E.P.v)[to[v] * vec16 + (u < vec16 ? u : u - vec16)] = x[v][c];
        }
        const int u = lane;
        if (is && u < 2 * words) (u < words ? E.P.k_scale : E.P.v_scale)[to[v] * words + (u < words ? u : u - words)] = y[v];
    }
}

}  // namespace

void launch_evict(const Eviction& E, hipStream_t st) {
    const EvictArgs K{E, __builtin_ctz(E.P.page_size)};
    const unsigned heads = (unsigned)(E.M.nseq * E.P.num_kv_heads);
    const int64_t held = ((int64_t)E.cap + 3) / 4 * 16;  // bytes of the ranks
    if (held <= kHeld)
        evict_select_kernel<true><<<heads, NT, (unsigned)held, st>>>(K);
    else
        evict_select_kernel<false><<<heads, NT, 0, st>>>(K);
    const int width = std::min(E.keep, E.cap);
    if (width == 0) return;
    const bool b4 = E.P.type == JYHIP_T_I4;
    const int bytes = b4 ? 16 * groups4(E.P.head_dim) : E.P.type == JYHIP_T_I8 ? E.P.head_dim : 2 * E.P.head_dim;
    const int words = b4 ? groups4(E.P.head_dim) : E.P.type == JYHIP_T_I8 ? 1 : 0;
    const int groups = (width + VECS - 1) / VECS;
    const unsigned grid = (unsigned)(((int64_t)heads * groups + 15) / 16);
    const int units = (2 * bytes / 16 + 15) / 16;  // 1 to 4
    if (units == 1)
        evict_move_kernel<1><<<grid, 256, 0, st>>>(K, groups, bytes / 16, words);
    else if (units == 2)
        evict_move_kernel<2><<<grid, 256, 0, st>>>(K, groups, bytes / 16, words);
    else
        evict_move_kernel<4><<<grid, 256, 0, st>>>(K, groups, bytes / 16, words);
}

}  // namespace jy
