// jy_ruled_attention.hip — attention over the paged cache with capped and biased scores, masks and 4-bit
// pages: one row per sequence, or short runs of rows.
//
//   s_j = scale q . k_j;  with a cap c: s_j = c tanh(s_j / c);  with a slope: s_j -= slope_h |pos - j|
//   out = sum_j p_j v_j, p = softmax of s over positions first .. last - 1 (holes left out)
//
// The work is split as in jy_paged_attention.hip: a wave takes 32 positions at a time for up to 16 columns of
// one kv head, in registers, chunks are joined by a second kernel.  A column here is a (row, query head):
// where a kv head has fewer than 9 query heads, the rows of a run share a wave, so that a run of drafted tokens
// reads its keys and values once.  Each lane belongs to one column and has its bounds; a tile that all columns
// see whole (nearly all of them) skips the masks.  A position that some columns see and others do not has
// to leave the others alone even where its value is not finite (0 times it is NaN): the lanes' scales and words
// are their own, so they are cleared, and 16-bit values that are not finite are taken out of
// such a tile, and the rows that do see them get them at the end.
//
// The weights of single rows need the softmax's final maximum and sum: the scores go to the workspace (a
// sixteenth of an int8 cache's bytes at four query heads a kv head), and a last kernel adds up what they weigh.
//
// 64 sequences of 200 to 8190, 32 heads over 8 of 128, 4 bits: 71 to 81 us, 2.5 TB/s (4.1 where all are of one
// length: in the ragged batch the longest end alone); the vector instructions of a tile are as long as its loads.
// 8 of 1000 to 16001 in int8 with cap and weights: 46 us, 4.9 of join, 6.3 of weighing.  77 drafted rows of 16
// sequences behind 4000 positions in int8: 35 us.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "jy_paged_attention.h"
#include "jy_paged_attention4.h"
#include "jy_ruled.h"

namespace jy {

namespace {

constexpr int kPages = 4096;  // positions whose pages the lanes hold at once

// Rows of a group: what fills 16 columns.  Single rows are groups of one.
Ruled plan_of(const RuledAttn& A) {
    Ruled K;
    K.A = A;
    K.ps_log2 = A.P.page_size > 0 ? __builtin_ctz(A.P.page_size) : 0;  // (a workspace is asked for before pages are checked)
    K.sstride = 0;
    if (plan_tiled(K)) return K;
    const int per = A.nh / A.P.num_kv_heads;
    K.hpg = std::min(per, 16);
    K.tiles = (per + 15) / 16;
    K.rpg = A.starts && per <= 8 ? 16 / per : 1;
    K.groups = A.starts ? (int)std::min<int64_t>(A.rows, A.rows / K.rpg + (int64_t)A.M.nseq) : A.rows;
    // the chunks of jy_paged_attention.hip; runs whose groups fill the chip by themselves are not cut
    const int64_t base = (int64_t)K.groups * A.P.num_kv_heads * K.tiles;
    const int span = A.span + (A.first && !A.starts ? 31 : 0);  // (a window starts anywhere in its first tile)
    K.chunk = 1024;
    K.splits = 1;
    if (span > 1024) {
        const int64_t want = std::max<int64_t>(1, 2048 / base);
        const int64_t least = base * ((span + 1023) / 1024) >= 768 ? 1024 : 512;
        int64_t chunk = std::max<int64_t>(least, ((span + want - 1) / want + 31) / 32 * 32);
        if (!A.starts) chunk = std::min<int64_t>(chunk, kPages);
        K.chunk = (int)std::min<int64_t>(chunk, (int64_t)(span + 31) / 32 * 32);
        K.splits = (span + K.chunk - 1) / K.chunk;
    }
    K.sstride = A.weights ? (span + 31) / 32 * 32 : 0;
    return K;
}

// the workspace's parts from `at` on (null: their sizes alone); floats
size_t lay_out(Ruled& K, float* at) {
    const size_t rows = (size_t)K.A.rows * K.A.nh;
    size_t n = 0;
    auto take = [&](size_t floats) {
        float* const p = at ? at + n : nullptr;
        n += (floats + 3) / 4 * 4;
        return p;
    };
    const size_t split = K.splits > 1 ? K.splits : 0;
    K.part_o = take(rows * split * K.A.P.head_dim);
    K.part_ml = reinterpret_cast<float2*>(take(rows * split * 2));
    K.part_live = reinterpret_cast<int*>(take(split ? K.A.rows : 0));
    K.ml = reinterpret_cast<float2*>(take(K.A.weights ? rows * 2 : 0));
    K.scores = take(rows * K.sstride);
    return n;
}

// tanh: 1 - 2 / (e^2y + 1), where that cancels the series to y^11 (its remainder under 2^-26 of tanh there)
__device__ __forceinline__ float tanh_of(float y) {
#if defined(__HIP_DEVICE_COMPILE__)
    const float a = fabsf(y), y2 = y * y;
    const float big = __builtin_copysignf(
        __builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(a * (2.0f * kLog2e)) + 1.0f), 1.0f), y);
    float t = __builtin_fmaf(y2, -1382.0f / 155925.0f, 62.0f / 2835.0f);
    t = __builtin_fmaf(t, y2, -17.0f / 315.0f);
    t = __builtin_fmaf(t, y2, 2.0f / 15.0f);
    t = __builtin_fmaf(t, y2, -1.0f / 3.0f);
    t = __builtin_fmaf(t * y2, y, y);
    return a < 0.35f ? t : big;  // (NaN: big, which is NaN)
#else
    return y;
#endif
}

template <int PT, int NC, bool WIDE>
struct StateOf {
    typedef State<PT, NC> type;
};
template <int NC, bool WIDE>
struct StateOf<JYHIP_T_I4, NC, WIDE> {
    typedef State4<NC, WIDE> type;
};

// whether the tile's 16-bit values hold an infinity or a NaN
template <int PT, int NC>
__device__ __forceinline__ bool holds_infinite(const Tile<PT, NC>& t) {
    constexpr uint32_t e = PT == JYHIP_T_F16 ? 0x7c00u : 0x7f80u;
    bool any = false;
#pragma unroll
    for (int j = 0; j < 8; j++)
#pragma unroll
        for (int w = 0; w < Tile<PT, NC>::VW; w++)
            any |= (t.v[j][w] & e) == e || (t.v[j][w] >> 16 & e) == e;
    return __any(any);
}

// Takes the infinities and NaN out of the tile's values, and notes for each row that sees one of them
// what its dim becomes: bad[row][dim], a bit each for +infinity, -infinity and NaN, four dims a word.
template <int PT, int NC>
__device__ __forceinline__ void take_infinite(Tile<PT, NC>& t, uint32_t (*bad)[16 * NC], int key0, int rows, int hpg, int lo, int hi) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr uint32_t e = PT == JYHIP_T_F16 ? 0x7c00u : 0x7f80u, m = 0x7fffu ^ e;
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int at = key0 + 16 * (j >> 2) + (lane >> 4) * 4 + (j & 3);
#pragma unroll
        for (int w = 0; w < Tile<PT, NC>::VW; w++)
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const uint32_t x = t.v[j][w] >> (16 * half) & 0xffffu;
                const bool is = (x & e) == e;
                if (!__any(is)) continue;
                const int d = (lane & 15) * (4 * NC) + 2 * w + half;
                const uint32_t bit = (x & m ? 4u : x >> 15 ? 2u : 1u) << (8 * (d & 3));
                for (int r = 0; r < rows; r++) {
                    const int rlo = __builtin_amdgcn_readlane(lo, r * hpg), rhi = __builtin_amdgcn_readlane(hi, r * hpg);
                    if (is && at >= rlo && at < rhi) atomicOr(&bad[r][d >> 2], bit);
                }
                if (is) t.v[j][w] &= half ? 0x0000ffffu : 0xffff0000u;
            }
    }
#endif
}

// RUNS: several rows of a run share a wave, over 16-bit values
template <int PT, int NC, bool WIDE, bool RUNS>
__global__ __launch_bounds__(256, NC <= 2 ? 2 : 1) void ruled_attend_kernel(Ruled K) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr bool B4 = PT == JYHIP_T_I4, B16 = RUNS;
    typedef Tile<PT, NC> T;
    typedef Query<PT, T::KC, WIDE> Q;
    typedef typename StateOf<PT, NC, WIDE>::type S;
    constexpr int DL = S::DL, ES = PT == JYHIP_T_F16 || PT == JYHIP_T_BF16 ? 2 : 1, STEP = 16 / ES;
    constexpr int XN = B4 ? 8 * T::KC : T::KC * STEP;  // elements of a query row that a lane holds
    constexpr int ROW = 64 * NC + 4;
    __shared__ float so[4][16][ROW];
    __shared__ float sm[4][16], sl[4][16];
    __shared__ uint32_t bad[B16 ? 16 : 1][16 * NC];
    const RuledAttn& A = K.A;
    const jyhip_pages& P = A.P;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15;
    const int hd = P.head_dim, nkv = P.num_kv_heads, per = A.nh / nkv;
    // heads fastest, then groups of rows, the last (and longest) of a run first, then chunks
    unsigned id = blockIdx.x;
    const int hg = id % (nkv * K.tiles);
    id /= nkv * K.tiles;
    int at = id % K.groups;
    const int split = id / K.groups;
    const int kvh = hg / K.tiles, tile = hg % K.tiles;
    const int h0 = kvh * per + tile * 16, heads = min(K.hpg, per - tile * 16);
    // the page of each of the wave's groups of 16 positions from s0 on: lane 2i + g has that of group g of its i-th tile
    auto pages = [&](int b, int s0) {
        const int i = (s0 + (wave + 4 * (lane >> 1)) * 32 + 16 * (lane & 1)) >> K.ps_log2;
        return i < A.M.stride ? A.M.tables[(int64_t)b * A.M.stride + i] : -1;
    };
    Run run{at, at, at + 1};
    int early = -1;  // single rows from position 0 on: where their pages lie does not wait for their lengths
    if (A.starts) {
        run = run_of(K, K.groups - 1 - at);
        if (run.seq < 0) return;
    } else {
        // (a chunk that its sequence has not leaves at once: in a ragged batch those are most)
        if (!A.first) early = pages(at, split * K.chunk);
        const unsigned f = A.first ? max(A.first[at], 0) & ~31 : 0;
        if (split != 0 && f + (unsigned)split * K.chunk >= (unsigned)max(min(A.lens[at], A.cap), 0)) return;
    }
    const int b = run.seq, rows = min(K.rpg, run.end - run.row0);
    // this lane's column
    const int crow = col / K.hpg, chead = col - crow * K.hpg;
    const bool on = crow < rows && chead < heads;
    const int row = run.row0 + (on ? crow : 0), head = h0 + (on ? chead : 0);
    int pos, lo = A.first ? max(A.first[row], 0) : 0, hi;
    if (A.starts) {
        pos = A.pos[row];
        hi = A.last ? A.last[row] : min(pos, A.cap) + 1;
    } else {
        hi = A.lens[b];
        pos = hi - 1;
        if (A.first) hi = (int)min((int64_t)hi, (int64_t)lo + A.most);
    }
    hi = min(hi, A.cap);
    const bool sees = hi > lo;
    // the group's bounds: over all columns that see anything, and what all of those see
    const int from = __builtin_amdgcn_readfirstlane(cols_min(sees ? lo : 0x7fffffff));
    const int to = __builtin_amdgcn_readfirstlane(cols_max(sees ? hi : 0));
    const int all_lo = __builtin_amdgcn_readfirstlane(cols_max(sees ? lo : 0));
    const int all_hi = __builtin_amdgcn_readfirstlane(cols_min(sees ? hi : 0x7fffffff));
    const int base = to > 0 ? from & ~31 : 0;
    // (both up to 2^30: their sum may pass 2^31)
    if (split != 0 && (unsigned)base + (unsigned)split * K.chunk >= (unsigned)to) return;
    const int c0 = base + split * K.chunk;
    if (K.splits > 1 && split == 0 && hg == 0 && threadIdx.x < 16 && on && chead == 0)
        K.part_live[row] = max(1, (to - base + K.chunk - 1) / K.chunk);

    const int64_t qbase = row * A.q.row_stride + head * A.q.head_stride;
    float x[XN];
    auto query = [&](auto* p) {
        if constexpr (B4)
            load_query4<std::remove_const_t<std::remove_pointer_t<decltype(p)>>, T::KC>(p + qbase, hd, on, x);
        else
            load_query<std::remove_const_t<std::remove_pointer_t<decltype(p)>>, T::KC, STEP>(p + qbase, hd, on, x);
    };
    if (A.type == JYHIP_T_F32)
        query(static_cast<const float*>(A.q.data));
    else if (A.type == JYHIP_T_F16)
        query(static_cast<const _Float16*>(A.q.data));
    else
        query(static_cast<const __bf16*>(A.q.data));

    Loader<PT, NC> ld;
    const int64_t first = (int64_t)kvh * P.page_size;  // this head's first position in page 0
    ld.page_rows = (int64_t)nkv * P.page_size;
    ld.num_pages = P.num_pages;
    ld.ps = P.page_size;
    if constexpr (B4) {
        ld.k = static_cast<const char*>(P.k) + first * Loader<PT, NC>::ROW;
        ld.v = static_cast<const char*>(P.v) + first * Loader<PT, NC>::ROW;
        ld.kw = reinterpret_cast<const char*>(P.k_scale) + first * (4 * T::G);
        ld.vw = reinterpret_cast<const char*>(P.v_scale) + first * (4 * T::G);
    } else {
        ld.k = static_cast<const char*>(P.k) + first * (hd * ES);
        ld.v = static_cast<const char*>(P.v) + first * (hd * ES);
        ld.ks = PT == JYHIP_T_I8 ? P.k_scale + first : nullptr;
        ld.vs = PT == JYHIP_T_I8 ? P.v_scale + first : nullptr;
        ld.row_bytes = hd * ES;
#pragma unroll
        for (int c = 0; c < T::KC; c++) {
            const int d = c * 4 * STEP + (lane >> 4) * STEP;
            const bool in = (NC > 1 && (c + 1) * 4 * STEP <= 32 * NC) || d < hd;
            ld.koff[c] = in ? (unsigned)(((lane & 15) * hd + d) * ES) : kNowhere;
        }
        const int d = (lane & 15) * DL;  // (outputs past the head's end are not stored)
#pragma unroll
        for (int j = 0; j < 4; j++) ld.voff[j] = d < hd ? (unsigned)((((lane >> 4) * 4 + j) * hd + d) * ES) : kNowhere;
    }

    if constexpr (B16) {
        for (int i = threadIdx.x; i < 16 * 16 * NC; i += 256) bad[i / (16 * NC)][i % (16 * NC)] = 0;
        __syncthreads();
    }
    const int end = K.splits > 1 ? min(to, c0 + K.chunk) : to;
    Q q;
    float qf = 0.0f;
    S st;
    // how the raw products become scores in units of log2 e
    const float soft = A.soft * kLog2e;
    const float slope = A.slopes ? A.slopes[head] * kLog2e : 0.0f;
    float* const sc = K.sstride ? K.scores + ((int64_t)row * A.nh + head) * K.sstride - base : nullptr;
    bool asked = false;

    // One tile, its keys in t and its values in tv; the keys of a later one are asked for once these are used up, its
    // values at the end.  DK, DV: two tiles of keys, of values are in registers at a time (what fits them)
    constexpr bool DK = B4 || PT == JYHIP_T_I8 || (!WIDE && !RUNS && NC <= 2), DV = B4 && NC <= 2;
    T ta, tb;
    auto step = [&](T& t, T& tv, int key0, auto&& next_keys, auto&& next_values) {
        const int kg = (lane >> 4) * 4;
        uint32_t outs = 0;
        bool care = false;
        float s[2][4], p[8];
        S::scores(q, qf, t, s);
        const int live[2] = {t.live[0], t.live[1]};
        next_keys();
        if (A.soft != 0.0f) {
#pragma unroll
            for (int g = 0; g < 2; g++)
#pragma unroll
                for (int i = 0; i < 4; i++) s[g][i] = soft * tanh_of(s[g][i]);
        }
        if (A.slopes) {
            const float d = (float)(pos - key0 - kg);
#pragma unroll
            for (int g = 0; g < 2; g++)
#pragma unroll
                for (int i = 0; i < 4; i++) s[g][i] = __builtin_fmaf(-slope, fabsf(d - (float)(16 * g + i)), s[g][i]);
        }
        if (key0 < all_lo || key0 + 32 > all_hi || live[0] + live[1] < 32) {
            asm volatile("");  // (a branch)
#pragma unroll
            for (int g = 0; g < 2; g++) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int j = key0 + 16 * g + kg + i;
                    const bool out = j < lo || j >= hi || kg + i >= live[g];
                    s[g][i] = out ? -__builtin_inff() : s[g][i];
                    if constexpr (PT == JYHIP_T_I8) tv.vs[g][i] = out ? 0.0f : tv.vs[g][i];
                    if constexpr (B4) outs |= (uint32_t)out << (4 * g + i);
                    if constexpr (PT == JYHIP_T_F16 || PT == JYHIP_T_BF16) {
                        // a value in front of everybody's first position (the ones behind were not loaded)
#pragma unroll
                        for (int w = 0; w < T::VW; w++) tv.v[4 * g + i][w] = j < from ? 0u : tv.v[4 * g + i][w];
                    }
                }
                if constexpr (B4) {
#pragma unroll
                    for (int w = 0; w < T::VC; w++) {
                        // (what nobody sees has no say in the scale of the weights either)
                        tv.vw[g][w] = key0 + 16 * g + kg + T::word_value(lane) < from ? 0u : tv.vw[g][w];
                        const h2_t x = as_h2(tv.vw[g][w]);
                        care |= __any(!(fabsf((float)x.x) <= 65504.0f) || !(fabsf((float)x.y) <= 65504.0f));
                    }
                }
            }
            if constexpr (B16)
                if (rows > 1 && holds_infinite<PT, NC>(tv)) take_infinite<PT, NC>(tv, bad, key0, rows, K.hpg, lo, hi);
        }
        if (sc && on) {
#pragma unroll
            for (int g = 0; g < 2; g++)
                *reinterpret_cast<f4_t*>(sc + key0 + 16 * g + kg) = f4_t{s[g][0], s[g][1], s[g][2], s[g][3]};
        }
        st.weights(tv, s, p);
        if constexpr (B4) {
            if (care) st.take_infinite(tv, outs);
            st.product(tv, p);
        } else {
            S::product(tv, p, st.o);
        }
        next_values();
    };

    for (int s0 = c0; s0 < end || !asked; s0 += kPages) {
        const int stop = min(end, s0 + kPages);
        const int ids = !A.starts && !A.first && s0 == c0 ? early : pages(b, s0);
        const int ntiles = stop > s0 ? (stop - s0 + 31) / 32 : 0;
        const int cnt = (ntiles - wave + 3) / 4;
        // (Past the last tile nothing is fetched, but the loads are issued: were they under a condition, the waits for the
        // earlier ones could not count on them and would wait for the whole queue.)
        auto keys = [&](T& t, int i) {
            const int p0 = __builtin_amdgcn_readlane(ids, 2 * i & 63), p1 = __builtin_amdgcn_readlane(ids, (2 * i + 1) & 63);
            ld.template load<true, false>(t, p0, p1, s0 + (wave + 4 * i) * 32, stop);
        };
        auto values = [&](T& t, int i) {
            const int p0 = __builtin_amdgcn_readlane(ids, 2 * i & 63), p1 = __builtin_amdgcn_readlane(ids, (2 * i + 1) & 63);
            ld.template load<false, true>(t, p0, p1, s0 + (wave + 4 * i) * 32, stop);
        };
        keys(ta, 0);
        values(ta, 0);
        if constexpr (DK) keys(tb, 1);
        if constexpr (DV) values(tb, 1);
        if (!asked) {  // the query as operands, while the first positions are on their way
            asked = true;
            float amax = 0.0f;
            bool bad = false;
#pragma unroll
            for (int i = 0; i < XN; i++) {
                amax = fmaxf(amax, fabsf(x[i]));
                bad |= !(fabsf(x[i]) <= 3.402823466e38f);
            }
            amax = head_max(amax);
            bad = head_max(bad ? 1.0f : 0.0f) > 0.0f;
            if (bad) {
#pragma unroll
                for (int i = 0; i < XN; i++) x[i] = 0.0f;
                amax = 0.0f;
            }
            q.load(x, amax);
            qf = q.factor(amax) * (A.soft != 0.0f ? A.scale / A.soft : A.scale * kLog2e);
            // (a small cap: an infinite factor would make NaN of a score of 0)
            qf = bad ? __builtin_nanf("") : fminf(fmaxf(qf, -3.402823466e38f), 3.402823466e38f);
        }
        auto at = [&](int i) { return s0 + (wave + 4 * i) * 32; };
        if constexpr (DK) {
            T& vb = DV ? tb : ta;
            // (in pairs without a way out between them, for the same reason)
            int i = 0;
            for (; i + 1 < cnt; i += 2) {
                step(ta, ta, at(i), [&] { keys(ta, i + 2); }, [&] { values(ta, DV ? i + 2 : i + 1); });
                step(tb, vb, at(i + 1), [&] { keys(tb, i + 3); }, [&] { values(vb, DV ? i + 3 : i + 2); });
            }
            if (i < cnt) step(ta, ta, at(i), [] {}, [] {});
        } else {
            for (int i = 0; i < cnt; i++) step(ta, ta, at(i), [&] { keys(ta, i + 1); }, [&] { values(ta, i + 1); });
        }
    }

    // join the waves
    st.l = head_sum(st.l);
    if constexpr (B4) {
#pragma unroll
        for (int g = 0; g < T::G; g++) {
            const float low = __shfl(st.low[g & 3], (g >> 2) * 16 + col) * (1.0f / 32768.0f);
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float unit = st.vref * (512.0f / 32768.0f);
#pragma unroll
                for (int i = 0; i < 4; i++)
                    so[wave][col][32 * g + 2 * ((lane >> 4) * 4 + i) + e] = __builtin_fmaf(st.o[2 * g + e][i], unit, low);
            }
        }
    } else {
        const float unit = st.unit();
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int d = 0; d < DL; d++) so[wave][col][((lane >> 4) * 4 + i) * DL + d] = st.o[d][i] * unit;
    }
    if (lane < 16) {
        sm[wave][col] = st.m;
        sl[wave][col] = sees ? st.l : 0.0f;
    }
    __syncthreads();
    const int quads = hd / 4, ncols = rows * K.hpg;
    for (int e = threadIdx.x; e < ncols * quads; e += 256) {
        const int c = e / quads, d = 4 * (e - c * quads);
        const int r = c / K.hpg, h = c - r * K.hpg;
        if (h >= heads) continue;
        float m[4], f[4], sum = 0.0f, mx = kNone;
        f4_t acc = {};
#pragma unroll
        for (int w = 0; w < 4; w++) {
            m[w] = sm[w][c];
            mx = fmaxf(mx, m[w]);
        }
#pragma unroll
        for (int w = 0; w < 4; w++) {
            f[w] = S::exp2_hw(m[w] - mx);
            sum += f[w] * sl[w][c];
            const f4_t o = *reinterpret_cast<const f4_t*>(&so[w][c][d]);
#pragma unroll
            for (int i = 0; i < 4; i++) acc[i] += f[w] * o[i];
        }
        if constexpr (B16)
            if (bad[r][d >> 2]) {
                const uint32_t w = bad[r][d >> 2];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t x = w >> (8 * i) & 7u;
                    if (x) acc[i] = x == 1 ? __builtin_inff() : x == 2 ? -__builtin_inff() : __builtin_nanf("");
                }
            }
        const int64_t at_row = (int64_t)(run.row0 + r) * A.nh + h0 + h;
        if (K.splits == 1) {
            store_out(A, run.row0 + r, h0 + h, d, acc, sum);
            if (d == 0 && K.sstride) K.ml[at_row] = float2{mx, sum};
        } else {
            *reinterpret_cast<f4_t*>(K.part_o + (at_row * K.splits + split) * hd + d) = acc;
            if (d == 0) K.part_ml[at_row * K.splits + split] = float2{mx, sum};
        }
    }
#endif
}

// The join of a (row, query head)'s chunks, as in jy_paged_attention.hip: groups of hd / 4 threads go through
// chunks of their own with a running maximum, then through LDS in a fixed order.
struct Joining {
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
    __device__ __forceinline__ void chunks(const Ruled& K, int64_t at, int row, int gi, int groups, int d) {
        const int splits = K.splits, hd = K.A.P.head_dim;
        const float2* ml = K.part_ml + at * splits;
        const float* po = K.part_o + at * splits * hd + d;
        float2 x[4];
        f4_t o[4];
        auto read = [&](int i) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int c = min(i + j * groups, splits - 1);
                x[j] = ml[c];
                o[j] = *reinterpret_cast<const f4_t*>(po + (int64_t)c * hd);
            }
        };
        read(gi);
        const int live = min(K.part_live[row], splits);
        for (int i = gi; i < live; i += 4 * groups) {
            if (i != gi) read(i);
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (i + j * groups < live) add(x[j].x, x[j].y, o[j]);
        }
    }
    __device__ __forceinline__ void store(const Ruled& K, int64_t at, int row, int h, int d) {
        store_out(K.A, row, h, d, acc, sum);
        if (d == 0 && K.sstride) K.ml[at] = float2{m, sum};
    }
};

// whether a row belongs to a run (the others are left as they are)
__device__ __forceinline__ bool in_run(const RuledAttn& A, int row) {
    return !A.starts || (row >= A.starts[0] && row < A.starts[A.M.nseq]);
}

__global__ __launch_bounds__(256) void ruled_join_few_kernel(Ruled K) {
    const RuledAttn& A = K.A;
    const int quads = A.P.head_dim / 4;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t at = id / quads;
    if (at >= (int64_t)A.rows * A.nh) return;
    const int d = 4 * (int)(id - at * quads), row = (int)(at / A.nh);
    if (!in_run(A, row)) return;
    Joining t;
    t.chunks(K, at, row, 0, 1, d);
    t.store(K, at, row, (int)(at - (int64_t)row * A.nh), d);
}

template <int NT>
__global__ __launch_bounds__(NT) void ruled_join_kernel(Ruled K) {
    __shared__ f4_t so[NT];
    __shared__ float sm[NT], ss[NT];
    const RuledAttn& A = K.A;
    const int at = blockIdx.x, row = at / A.nh, h = at % A.nh;
    if (!in_run(A, row)) return;
    const int quads = A.P.head_dim / 4, groups = NT / quads;
    const int gi = threadIdx.x / quads, d4 = threadIdx.x % quads;
    Joining t;
    if (gi < groups) t.chunks(K, at, row, gi, groups, 4 * d4);
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
    if (gi == 0) t.store(K, at, row, h, 4 * d4);
}

// weights[s][kv head][j] += the heads' p_j: the scores are read once, four positions a thread
__global__ __launch_bounds__(256) void weigh_kernel(Ruled K) {
#if defined(__HIP_DEVICE_COMPILE__)
    const RuledAttn& A = K.A;
    const int nkv = A.P.num_kv_heads, per = A.nh / nkv;
    const unsigned parts = (K.sstride + 1023) / 1024, at_head = blockIdx.x / parts, part = blockIdx.x - at_head * parts;
    const int b = at_head / nkv, kvh = at_head % nkv;
    const int lo = A.first ? max(A.first[b], 0) : 0;
    int hi = A.lens[b];
    if (A.first) hi = (int)min((int64_t)hi, (int64_t)lo + A.most);
    hi = min(min(hi, A.cap), A.weights_len);
    if (hi <= lo) return;
    const int base = lo & ~31;
    const int j0 = base + (part * 256 + threadIdx.x) * 4;
    if (j0 >= hi) return;
    const int64_t at = (int64_t)b * A.nh + kvh * per;
    float w[4] = {};
    for (int h = 0; h < per; h++) {
        const f4_t s = *reinterpret_cast<const f4_t*>(K.scores + (at + h) * K.sstride + (j0 - base));
        const float2 ml = K.ml[at + h];
        const float inv = ml.y == 0.0f ? 0.0f : 1.0f / ml.y;
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] += __builtin_amdgcn_exp2f(s[i] - ml.x) * inv;
    }
    float* const to = A.weights + b * A.seq_stride + kvh * A.head_stride + j0;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (j0 + i >= lo && j0 + i < hi) to[i] += w[i];
#endif
}

template <int PT, int NC, bool WIDE>
void launch_runs(const Ruled& K, unsigned grid, hipStream_t st) {
    if constexpr (PT == JYHIP_T_F16 || PT == JYHIP_T_BF16) {
        if (K.rpg > 1) {
            ruled_attend_kernel<PT, NC, WIDE, true><<<grid, 256, 0, st>>>(K);
            return;
        }
    }
    ruled_attend_kernel<PT, NC, WIDE, false><<<grid, 256, 0, st>>>(K);
}

template <int PT, bool WIDE>
void launch_nc(const Ruled& K, unsigned grid, hipStream_t st) {
    const int hd = K.A.P.head_dim;
    if (hd <= 64)
        launch_runs<PT, 1, WIDE>(K, grid, st);
    else if (hd <= 128)
        launch_runs<PT, 2, WIDE>(K, grid, st);
    else
        launch_runs<PT, 4, WIDE>(K, grid, st);
}

template <int PT>
void launch_wide(const Ruled& K, unsigned grid, hipStream_t st) {
    // (4-bit pages: what fp16 outputs would show of a weight's rounding to fp16, bf16 ones do not)
    if (PT == JYHIP_T_I8 || K.A.type == JYHIP_T_F32 || ((PT == JYHIP_T_BF16 || PT == JYHIP_T_I4) && K.A.type == JYHIP_T_F16))
        launch_nc<PT, true>(K, grid, st);
    else if constexpr (PT != JYHIP_T_I8)
        launch_nc<PT, false>(K, grid, st);
}

}  // namespace

size_t ruled_attend_part_floats(const RuledAttn& A) {
    Ruled K = plan_of(A);
    return lay_out(K, nullptr);
}

int64_t ruled_attend_blocks(const RuledAttn& A) {
    const Ruled K = plan_of(A);
    const int64_t weigh = (int64_t)(K.sstride + 1023) / 1024 * A.rows * A.P.num_kv_heads;
    return std::max({(int64_t)K.groups * A.P.num_kv_heads * K.tiles * K.splits, (int64_t)A.rows * A.nh * 4, weigh});
}

void launch_ruled_attend(const RuledAttn& A, hipStream_t st) {
    Ruled K = plan_of(A);
    lay_out(K, A.part);
    const unsigned grid = (unsigned)((int64_t)K.groups * A.P.num_kv_heads * K.tiles * K.splits);
    if (K.tiled)
        launch_tiled(K, grid, st);
    else if (A.P.type == JYHIP_T_I4)
        launch_wide<JYHIP_T_I4>(K, grid, st);
    else if (A.P.type == JYHIP_T_I8)
        launch_wide<JYHIP_T_I8>(K, grid, st);
    else if (A.P.type == JYHIP_T_F16)
        launch_wide<JYHIP_T_F16>(K, grid, st);
    else
        launch_wide<JYHIP_T_BF16>(K, grid, st);
    if (K.splits > 1) {
        const int quads = A.P.head_dim / 4;
        const int64_t rows = (int64_t)A.rows * A.nh;
        // 8 sequences of 32 heads of 128: 16 chunks 4.7 us with a workgroup a row, 6.7 with a thread for four dims; the
        // latter takes 4.8 for 64 sequences of 8 chunks, with fewer workgroups to start
        if (K.splits <= 8)
            ruled_join_few_kernel<<<(unsigned)((rows * quads + 255) / 256), 256, 0, st>>>(K);
        else if (K.splits * quads <= 4 * 256)
            ruled_join_kernel<256><<<(unsigned)rows, 256, 0, st>>>(K);
        else
            ruled_join_kernel<1024><<<(unsigned)rows, 1024, 0, st>>>(K);
    }
    if (A.weights)
        weigh_kernel<<<(unsigned)((int64_t)(K.sstride + 1023) / 1024 * A.rows * A.P.num_kv_heads), 256, 0, st>>>(K);
}

}  // namespace jy
