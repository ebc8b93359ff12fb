// jy_evict.hip — which positions of a cache stay by their accumulated weights, and their way to new pages.
//
// Selection: a workgroup per (sequence, kv head).  A weight's bits become a number that rises with it, and the
// need-th largest is found by three counts over its digits (12, 10 and 10 bits, bins in LDS, whole numbers: the
// order of the atomics does not matter); the first digit is sign, exponent and three bits of the fraction, so
// that the weights of a sequence spread over dozens of bins.  A last pass over the positions in order takes
// what lies above that weight, of those equal to it the first, and the recent ones.
// Moving: 16 lanes a vector, key and value together, bytes as they are.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "jy_device.h"
#include "jy_paged_device.h"

namespace jy {

namespace {

constexpr int NT = 1024, PER = 4;  // threads; positions a thread takes at a time
constexpr int BINS = 4096;

struct EvictArgs {
    Eviction E;
    int ps_log2;
};

// rises with the weight: NaN lowest, then -infinity .. +infinity, both zeros the same
__device__ __forceinline__ uint32_t rank_of(float w) {
    if (!(w == w)) return 0;
    const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// exclusive sum over the workgroup's threads, and the whole
__device__ __forceinline__ uint32_t scan(uint32_t v, uint32_t* part, uint32_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t s = v;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t x = __shfl_up(s, d);
        if (lane >= d) s += x;
    }
    __syncthreads();  // (the last scan's parts are read)
    if (lane == 63) part[wave] = s;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; w++) {
        const uint32_t x = part[w];
        before += w < wave ? x : 0;
        total += x;
    }
    return before + s - v;
}

__global__ __launch_bounds__(NT) void evict_select_kernel(EvictArgs K) {
    __shared__ uint32_t bins[BINS];
    __shared__ uint32_t part[NT / 64];
    __shared__ uint32_t found[2];
    const Eviction& E = K.E;
    const int nkv = E.P.num_kv_heads, s = blockIdx.x / nkv, h = blockIdx.x - s * nkv;
    const int n = max(min(E.lens[s], E.cap), 0);
    const int late = max(n - E.recent, 0);
    const float* const w = E.weights + s * E.seq_stride + h * E.head_stride;
    const int* const table = E.M.tables + (int64_t)s * E.M.stride;
    auto exists = [&](int j) { return (unsigned)table[j >> K.ps_log2] < (unsigned)E.P.num_pages; };
    auto weight = [&](int j) { return j < E.weights_len ? w[j] : 0.0f; };

    // how many positions there are, and how many of them are recent
    uint32_t count = 0;
    for (int at = threadIdx.x << K.ps_log2; at < n; at += NT << K.ps_log2) {
        if (!exists(at)) continue;
        const int end = min(at + (1 << K.ps_log2), n);
        count += (uint32_t)(end - at);
    }
    uint32_t there = 0, recent = 0;
    scan(count, part, there);
    count = 0;
    for (int j = late + threadIdx.x; j < n; j += NT) count += exists(j);
    scan(count, part, recent);
    const int stay = min(E.keep, (int)there);
    const bool all = (int)there <= E.keep;

    // the need-th largest rank among the old positions: its digits from the top
    uint32_t need = all ? 0 : (uint32_t)stay - recent, top = 0, ties = 0;
    if (need > 0) {
        int shift = 32;
        uint32_t left = need;
#pragma unroll
        for (int digit = 0; digit < 3; digit++) {
            const int bits = digit == 0 ? 12 : 10, size = 1 << bits;
            shift -= bits;
            for (int i = threadIdx.x; i < size; i += NT) bins[i] = 0;
            __syncthreads();
            for (int j = threadIdx.x; j < late; j += NT) {
                if (!exists(j)) continue;
                const uint32_t r = rank_of(weight(j));
                if (digit == 0 || r >> (shift + bits) == top >> (shift + bits)) atomicAdd(&bins[(r >> shift) & (size - 1)], 1u);
            }
            __syncthreads();
            // from the largest bin down: thread t has bins size - 1 - t per .. down
            const int per = (size + NT - 1) / NT;
            uint32_t own = 0;
            for (int i = 0; i < per; i++) {
                const int b = size - 1 - ((int)threadIdx.x * per + i);
                own += b >= 0 ? bins[b] : 0;
            }
            uint32_t total;
            uint32_t above = scan(own, part, total);
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
            top |= found[0] << shift;
            left -= found[1];
            __syncthreads();
        }
        ties = left;  // of those whose rank is the border's, the first
    }

    int* const kept = E.kept + (int64_t)blockIdx.x * E.keep;
    float* const to = E.new_weights ? E.new_weights + s * E.new_seq_stride + h * E.new_head_stride : nullptr;
    uint32_t above = 0, equal = 0;  // positions over the border and on it, so far
    for (int c0 = 0; c0 < n; c0 += NT * PER) {
        const int j0 = c0 + threadIdx.x * PER;
        float x[PER];
        bool over[PER], on[PER];
        uint32_t v = 0;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int j = j0 + i;
            const bool is = j < n && exists(j);
            x[i] = is ? weight(j) : 0.0f;
            const uint32_t r = rank_of(x[i]);
            over[i] = is && (all || j >= late || (need > 0 && r > top));
            on[i] = is && !over[i] && need > 0 && r == top;
            v += (over[i] ? 1u : 0u) + (on[i] ? 0x10000u : 0u);
        }
        uint32_t total;
        const uint32_t before = scan(v, part, total);
        uint32_t a = above + (before & 0xffffu), e = equal + (before >> 16);
#pragma unroll
        for (int i = 0; i < PER; i++) {
            if (over[i] || (on[i] && e < ties)) {
                const uint32_t at = a + min(e, ties);
                kept[at] = j0 + i;
                if (to && (int)at < E.new_weights_len) to[at] = x[i];
            }
            a += over[i];
            e += on[i];
        }
        above += total & 0xffffu;
        equal += total >> 16;
    }
    __syncthreads();
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

__global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs K, int width, int vec16, int words) {
    const Eviction& E = K.E;
    const unsigned id = blockIdx.x * 16 + (threadIdx.x >> 4);
    const unsigned head = id / width, lane = threadIdx.x & 15;
    const int i = (int)(id - head * width), nkv = E.P.num_kv_heads;
    if (head >= (unsigned)E.M.nseq * nkv) return;
    const int s = head / nkv, h = head % nkv;
    const int pos = E.kept[(int64_t)head * E.keep + i];
    const int64_t from = vector_at(E, E.M, K.ps_log2, s, h, pos), to = vector_at(E, E.to, K.ps_log2, s, h, i);
    if (from < 0 || to < 0) return;
    // 16 bytes a lane, the key's first; scales as words
    for (int u = lane; u < 2 * vec16; u += 16) {
        uint4* const p = static_cast<uint4*>(u < vec16 ? E.P.k : E.P.v);
        const int at = u < vec16 ? u : u - vec16;
        p[to * vec16 + at] = p[from * vec16 + at];
    }
    for (int u = lane; u < 2 * words; u += 16) {
        float* const p = u < words ? E.P.k_scale : E.P.v_scale;
        const int at = u < words ? u : u - words;
        p[to * words + at] = p[from * words + at];
    }
}

}  // namespace

void launch_evict(const Eviction& E, hipStream_t st) {
    const EvictArgs K{E, __builtin_ctz(E.P.page_size)};
    evict_select_kernel<<<(unsigned)(E.M.nseq * E.P.num_kv_heads), NT, 0, st>>>(K);
    const int width = std::min(E.keep, E.cap);
    if (width == 0) return;
    const bool b4 = E.P.type == JYHIP_T_I4;
    const int bytes = b4 ? 16 * groups4(E.P.head_dim) : E.P.type == JYHIP_T_I8 ? E.P.head_dim : 2 * E.P.head_dim;
    const int words = b4 ? groups4(E.P.head_dim) : E.P.type == JYHIP_T_I8 ? 1 : 0;
    const int64_t vectors = (int64_t)E.M.nseq * E.P.num_kv_heads * width;
    evict_move_kernel<<<(unsigned)((vectors + 15) / 16), 256, 0, st>>>(K, width, bytes / 16, words);
}

}  // namespace jy
