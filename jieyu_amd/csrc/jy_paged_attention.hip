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
//        bf16 parts, accumulated in fp32; so split that an infinite key gives the score that the
//        whole query would.
//   p.v  o^T = V^T p^T: the weights come out of the first product in the very layout the second
//        takes as its B operand (lane: head l & 15, keys 4 (l >> 4) + i of two 16-key groups), so
//        they change no lane.  V is read row by row, lane l holding DL consecutive dims from
//        (l & 15) DL of its 8 keys, and transposed in registers: output tile t's row r is dim
//        r DL + t, and a byte permute pairs two keys of one dim.  int8 values become fp16 exactly
//        (their bytes read as subnormal halves, one packed fma gives (u - 128) / 512); a weight
//        times its value scale is carried as two fp16 parts (21 bits, relative to the running
//        maximum and to a power of two over the value scales seen), for bf16 values as three
//        bf16 parts, none of them 0 beside a first one that is not: 0 times an infinite value is NaN.
//
// A workgroup's four waves take the tiles of one chunk of a sequence in turn and join through
// LDS; chunks are joined by a second kernel where there is more than one.
//
// 64 sequences of 200 to 8190 positions, 32 / 8 heads of 128, bf16 (591 MB): 112 to 160 us from launch to
// launch, half of them within 136 (4.3 TB/s), and 4.8 of join.  One of 32769, 28 / 4 heads, int8 (34.6 MB):
// 12.6 us, of them 5 for the bytes (a wave per SIMD), and 5.2 of join.  32 of 1 to 1500, int8: 14.2 us, the
// chain of the longest chunk, and 3.9.  One of 61 positions, 14 / 2 heads of 64: 4.7 us, the start, one step
// and the end.  fp32 queries cost more than 16-bit ones against 16-bit pools, in products and in registers
// (some spilled from head size 128 on): 48 of 200 to 6000, 32 / 8 heads of 128, both kernels 128 us
// against 89 in bf16, 102 against 89 in fp16.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "jy_paged_attention.h"

namespace jy {

namespace {

struct AttnPlan {
    int chunk = 0;   // positions per workgroup, a multiple of 32
    int splits = 1;  // chunks of the longest sequence the launch may see
    int tiles = 1;   // groups of 16 query heads per kv head
};

// The chunk by the launch's upper bound of its lengths (the lengths themselves are on the device).
// A workgroup's own start and end cost about as much as 300 positions, two run on a CU at a time,
// and chunks that one sequence has and another has not are what balances a ragged batch:
//   up to 1024 positions in one piece: no join (32 x 800 positions of int8 12.1 us, in two 13.7)
//   512 at least; 1024 where those still make 768 workgroups (16 x 6000 positions of 8 heads of 128
//   int8 46.3 us against 50.7 with 512; 32 of up to 1500 20.0 us against 18.2, so not there)
//   2048 workgroups where the batch is longer (64 of 200 to 8190 in bf16: 137 us, with half as
//   many 145, with twice as many 135; 16 x 12000 84, 81, 84 us)
AttnPlan plan_of(const jyhip_pages& P, int nseq, int nh, int max_len) {
    AttnPlan p;
    p.tiles = (nh / P.num_kv_heads + 15) / 16;
    const int64_t base = (int64_t)nseq * P.num_kv_heads * p.tiles;
    if (max_len <= 1024) {
        p.chunk = 1024;
        return p;
    }
    const int64_t want = std::max<int64_t>(1, 2048 / base);
    const int64_t least = base * ((max_len + 1023) / 1024) >= 768 ? 1024 : 512;
    const int64_t chunk = std::max<int64_t>(least, ((max_len + want - 1) / want + 31) / 32 * 32);
    p.chunk = (int)std::min<int64_t>(chunk, kMaxChunk);
    p.splits = (max_len + p.chunk - 1) / p.chunk;
    return p;
}

struct AttnKernelArgs {
    PagedAttn A;
    AttnPlan plan;
    int ps_log2;
    float* part_o;   // [nseq][nh][splits][hd]
    float2* part_ml; // [nseq][nh][splits]: running maximum and sum
};

template <int PT, int NC, bool WIDE>
__global__ __launch_bounds__(256, NC <= 2 ? 2 : 1) void paged_attend_kernel(AttnKernelArgs K) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef Tile<PT, NC> T;
    typedef Query<PT, T::KC, WIDE> Q;
    constexpr int DL = 4 * NC, ES = T::ES, STEP = 16 / ES;
    constexpr int ROW = 64 * NC + 4;
    __shared__ float so[4][16][ROW];
    __shared__ float sm[4][16], sl[4][16];
    const PagedAttn& A = K.A;
    const jyhip_pages& P = A.P;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int hd = P.head_dim, nkv = P.num_kv_heads, per = A.nh / nkv;
    // Blocks: heads fastest, then sequences, then chunks.  Blocks go round the XCDs in turn, and
    // short sequences have first chunks alone: with chunks fastest those met on two of the eight.
    unsigned id = blockIdx.x;
    const int hg = id % (nkv * K.plan.tiles);
    id /= nkv * K.plan.tiles;
    const int b = id % A.M.nseq, split = id / A.M.nseq;
    const int kvh = hg / K.plan.tiles, tile = hg % K.plan.tiles;
    const int c0 = split * K.plan.chunk;
    const int h0 = kvh * per + tile * 16, heads = min(16, per - tile * 16);

    // the page of each of the wave's groups of 16 positions: lane 2i + g has that of group g of its
    // i-th tile (past the sequence's end as well: whether a position exists is settled below)
    int ids = -1;
    {
        const int at = (c0 + (wave + 4 * (lane >> 1)) * 32 + 16 * (lane & 1)) >> K.ps_log2;
        if (at < A.M.stride) ids = A.M.tables[(int64_t)b * A.M.stride + at];
    }
    const int n = __builtin_amdgcn_readfirstlane(min(A.lens[b], A.cap));
    const bool on = (lane & 15) < heads;
    const int64_t qbase = b * A.q.row_stride + (h0 + (on ? lane & 15 : 0)) * A.q.head_stride;
    float x[T::KC * STEP];
    if (A.type == JYHIP_T_F32)
        load_query<float, T::KC, STEP>(static_cast<const float*>(A.q.data) + qbase, hd, on, x);
    else if (A.type == JYHIP_T_F16)
        load_query<_Float16, T::KC, STEP>(static_cast<const _Float16*>(A.q.data) + qbase, hd, on, x);
    else
        load_query<__bf16, T::KC, STEP>(static_cast<const __bf16*>(A.q.data) + qbase, hd, on, x);
    if (c0 >= n && split != 0) return;

    Loader<PT, NC> ld;
    const int64_t first = (int64_t)kvh * P.page_size;  // this head's first position in page 0
    ld.k = static_cast<const char*>(P.k) + first * (hd * ES);
    ld.v = static_cast<const char*>(P.v) + first * (hd * ES);
    ld.ks = PT == JYHIP_T_I8 ? P.k_scale + first : nullptr;
    ld.vs = PT == JYHIP_T_I8 ? P.v_scale + first : nullptr;
    ld.page_rows = (int64_t)nkv * P.page_size;
    ld.num_pages = P.num_pages;
    ld.ps = P.page_size;
    ld.row_bytes = hd * ES;
#pragma unroll
    for (int c = 0; c < T::KC; c++) {
        const int d = c * 4 * STEP + (lane >> 4) * STEP;
        // (the first half is inside any head of this form: one register and offsets in the loads)
        const bool in = (NC > 1 && (c + 1) * 4 * STEP <= 32 * NC) || d < hd;
        ld.koff[c] = in ? (unsigned)(((lane & 15) * hd + d) * ES) : kNowhere;
    }
    {
        const int d = (lane & 15) * DL;  // (outputs past the head's end are not stored)
#pragma unroll
        for (int j = 0; j < 4; j++) ld.voff[j] = d < hd ? (unsigned)((((lane >> 4) * 4 + j) * hd + d) * ES) : kNowhere;
    }
    const int end = min(n, c0 + K.plan.chunk);
    const int ntiles = end > c0 ? (end - c0 + 31) / 32 : 0;
    const int cnt = (ntiles - wave + 3) / 4;  // (not positive for a wave without any)
    auto load = [&](T& t, int i) {
        const int p0 = __builtin_amdgcn_readlane(ids, 2 * i), p1 = __builtin_amdgcn_readlane(ids, 2 * i + 1);
        ld.load(t, p0, p1, c0 + (wave + 4 * i) * 32, end);
    };
    T t0, t1;
    if (cnt > 0) load(t0, 0);
    if (cnt > 1) load(t1, 1);

    // the query as operands, while the first positions are on their way
    Q q;
    float qf;
    {
        float amax = 0.0f;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < T::KC * STEP; i++) {
            amax = fmaxf(amax, fabsf(x[i]));
            bad |= !(fabsf(x[i]) <= 3.402823466e38f);
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
    State<PT, NC> st;
    for (int i = 0; i < cnt; i += 2) {
        st.add(q, qf, t0);
        if (i + 1 >= cnt) break;
        if (i + 2 < cnt) load(t0, i + 2);
        st.add(q, qf, t1);
        if (i + 3 < cnt) load(t1, i + 3);
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
    const int quads = hd / 4;
    for (int e = threadIdx.x; e < heads * quads; e += 256) {
        const int r = e / quads, d = 4 * (e - r * quads);
        float m[4], f[4], sum = 0.0f, mx = kNone;
        f4_t acc = {};
#pragma unroll
        for (int w = 0; w < 4; w++) {
            m[w] = sm[w][r];
            mx = fmaxf(mx, m[w]);
        }
#pragma unroll
        for (int w = 0; w < 4; w++) {
            f[w] = State<PT, NC>::exp2_hw(m[w] - mx);
            sum += f[w] * sl[w][r];
            const f4_t o = *reinterpret_cast<const f4_t*>(&so[w][r][d]);
#pragma unroll
            for (int i = 0; i < 4; i++) acc[i] += f[w] * o[i];
        }
        const int64_t row = (int64_t)b * A.nh + h0 + r;
        if (K.plan.splits == 1) {
            store_out(A, b, h0 + r, d, acc, sum);
        } else {
            *reinterpret_cast<f4_t*>(K.part_o + (row * K.plan.splits + split) * hd + d) = acc;
            if (d == 0) K.part_ml[row * K.plan.splits + split] = float2{mx, sum};
        }
    }
#endif
}

// The join: a (sequence, query head)'s chunks, their outputs weighted by 2^(m - max m) over the sum of
// their weighted sums.  hd / 4 threads take one chunk's output, four consecutive dims each.  A thread
// goes through chunks gi, gi + groups, ... with a running maximum of its own, four read at once, the
// first ones before the sequence's length is known.
struct Joined {
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
    __device__ __forceinline__ void chunks(const AttnKernelArgs& K, int row, int b, int gi, int groups, int d) {
        const int splits = K.plan.splits, hd = K.A.P.head_dim;
        const float2* ml = K.part_ml + (int64_t)row * splits;
        const float* po = K.part_o + (int64_t)row * splits * hd + d;
        float2 x[4];
        f4_t o[4];
        auto read = [&](int i) {  // (those that are live are told apart in use)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int at = min(i + j * groups, splits - 1);
                x[j] = ml[at];
                o[j] = *reinterpret_cast<const f4_t*>(po + (int64_t)at * hd);
            }
        };
        read(gi);
        const int n = min(K.A.lens[b], K.A.cap);
        const int live = max(1, (max(n, 0) + K.plan.chunk - 1) / K.plan.chunk);
        for (int i = gi; i < live; i += 4 * groups) {
            if (i != gi) read(i);
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (i + j * groups < live) add(x[j].x, x[j].y, o[j]);
        }
    }
};

// few chunks: a thread takes all of them, nothing is exchanged
__global__ __launch_bounds__(256) void paged_join_few_kernel(AttnKernelArgs K) {
    const PagedAttn& A = K.A;
    const int quads = A.P.head_dim / 4;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t row = id / quads;
    if (row >= (int64_t)A.M.nseq * A.nh) return;
    const int d = 4 * (int)(id - row * quads), b = (int)(row / A.nh);
    Joined t;
    t.chunks(K, (int)row, b, 0, 1, d);
    store_out(A, b, (int)row - b * A.nh, d, t.acc, t.sum);
}

// many: one workgroup per row, the threads' parts joined through LDS in a fixed order
template <int NT>
__global__ __launch_bounds__(NT) void paged_join_kernel(AttnKernelArgs K) {
    __shared__ f4_t so[NT];
    __shared__ float sm[NT], ss[NT];
    const PagedAttn& A = K.A;
    const int row = blockIdx.x, b = row / A.nh, h = row % A.nh;
    const int quads = A.P.head_dim / 4, groups = NT / quads;
    const int gi = threadIdx.x / quads, d4 = threadIdx.x % quads;
    Joined t;
    if (gi < groups) t.chunks(K, row, b, gi, groups, 4 * d4);
    // rounds: every eighth group's threads take their seven neighbours'
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
    if (gi == 0) store_out(A, b, h, 4 * d4, t.acc, t.sum);
}

template <int PT, bool WIDE>
void launch_nc(const AttnKernelArgs& K, unsigned grid, hipStream_t st) {
    const int hd = K.A.P.head_dim;
    if (hd <= 64)
        paged_attend_kernel<PT, 1, WIDE><<<grid, 256, 0, st>>>(K);
    else if (hd <= 128)
        paged_attend_kernel<PT, 2, WIDE><<<grid, 256, 0, st>>>(K);
    else
        paged_attend_kernel<PT, 4, WIDE><<<grid, 256, 0, st>>>(K);
}

// WIDE: a query that one 16-bit operand cannot hold (fp32, and fp16 against bf16 keys); the int8
// form's digits hold any
template <int PT>
void launch_wide(const AttnKernelArgs& K, unsigned grid, hipStream_t st) {
    if (PT == JYHIP_T_I8 || K.A.type == JYHIP_T_F32 || (PT == JYHIP_T_BF16 && K.A.type == JYHIP_T_F16))
        launch_nc<PT, true>(K, grid, st);
    else if constexpr (PT != JYHIP_T_I8)
        launch_nc<PT, false>(K, grid, st);
}

// 4-bit pages: the other kernel, without rules
RuledAttn ruled_of(const PagedAttn& A) {
    RuledAttn R;
    R.P = A.P;
    R.M = A.M;
    R.lens = A.lens;
    R.rows = A.M.nseq;
    R.span = std::max(A.max_len, 1);
    R.cap = A.cap;
    R.nh = A.nh;
    R.scale = A.scale;
    R.q = A.q;
    R.out = A.out;
    R.type = A.type;
    R.part = A.part;
    return R;
}
RuledAttn ruled_of(const jyhip_pages& P, int nseq, int nh, int max_len) {
    PagedAttn A;
    A.P = P;
    A.M.nseq = nseq;
    A.nh = nh;
    A.max_len = max_len;
    return ruled_of(A);
}

}  // namespace

// (positions past max_len do not exist, so a launch over none still has one chunk: it writes zeros)
size_t paged_attend_part_floats(const jyhip_pages& P, int nseq, int nh, int max_len) {
    if (P.type == JYHIP_T_I4) return ruled_attend_part_floats(ruled_of(P, nseq, nh, max_len));
    const AttnPlan p = plan_of(P, nseq, nh, std::max(max_len, 1));
    return p.splits == 1 ? 0 : (size_t)nseq * nh * p.splits * (P.head_dim + 2);
}

int64_t paged_attend_blocks(const jyhip_pages& P, int nseq, int nh, int max_len) {
    if (P.type == JYHIP_T_I4) return ruled_attend_blocks(ruled_of(P, nseq, nh, max_len));
    const AttnPlan p = plan_of(P, nseq, nh, std::max(max_len, 1));
    return std::max((int64_t)nseq * P.num_kv_heads * p.tiles * p.splits, (int64_t)nseq * nh * 4);
}

void launch_paged_attend(const PagedAttn& A, hipStream_t st) {
    if (A.P.type == JYHIP_T_I4) return launch_ruled_attend(ruled_of(A), st);
    AttnKernelArgs K;
    K.A = A;
    K.plan = plan_of(A.P, A.M.nseq, A.nh, std::max(A.max_len, 1));
    K.ps_log2 = __builtin_ctz(A.P.page_size);
    K.part_o = A.part;
    K.part_ml = reinterpret_cast<float2*>(A.part + (size_t)A.M.nseq * A.nh * K.plan.splits * A.P.head_dim);
    const unsigned grid = (unsigned)((int64_t)A.M.nseq * A.P.num_kv_heads * K.plan.tiles * K.plan.splits);
    if (A.P.type == JYHIP_T_I8)
        launch_wide<JYHIP_T_I8>(K, grid, st);
    else if (A.P.type == JYHIP_T_F16)
        launch_wide<JYHIP_T_F16>(K, grid, st);
    else
        launch_wide<JYHIP_T_BF16>(K, grid, st);
    if (K.plan.splits > 1) {
        // 32 sequences of up to 1500 positions, 32 heads of 128, 3 chunks: both kernels 18.5 us with a
        // workgroup a row, 17.5 us with a thread for four dims.  More chunks: four a thread are read
        // at once, so more threads where those are not all (one sequence of 32000, 14 heads of 64:
        // 11.6 us with 256 threads, 13.2 us with 1024).
        const int quads = A.P.head_dim / 4;
        const int64_t rows = (int64_t)A.M.nseq * A.nh;
        if (K.plan.splits <= 16)
            paged_join_few_kernel<<<(unsigned)((rows * quads + 255) / 256), 256, 0, st>>>(K);
        else if (K.plan.splits * quads <= 4 * 256)
            paged_join_kernel<256><<<(unsigned)rows, 256, 0, st>>>(K);
        else
            paged_join_kernel<1024><<<(unsigned)rows, 1024, 0, st>>>(K);
    }
}

}  // namespace jy
