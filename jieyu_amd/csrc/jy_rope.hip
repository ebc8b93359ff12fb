// jy_rope.hip — rotary positions on rows of query and key heads.
//
// Pair i of a row at position p turns by the angle p f_i:  (x, y) -> (x c - y s, x s + y c), c and s the
// factor times cos and sin.  A row's heads share its angles, so a workgroup takes all heads of a few rows:
// its threads first put the rows' cosines and sines into LDS, one pair each, then walk over the vectors.
//
// The angle is an fp64 product: at position 2^20 an fp32 one would be off by 2^-4.  It is reduced to
// [-pi/4, pi/4] in fp64 (pi/2 in two parts) and from there on fp32 Taylor polynomials do (their
// remainders are under 2^-27).  That is some fifteen fp64 operations a pair, for 32 to 64 pairs a row; everything
// else is one read and one write of the heads, so memory bounds long calls and the launch short ones: 8191 rows of
// 32 + 8 heads of 128 in bf16 30 us (168 MB, 5.6 TB/s), one row of 14 + 2 heads of 64 2 us.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "jy_paged_device.h"
#include "jy_rope.h"

namespace jy {

namespace {

constexpr int NT = 256;

struct RopeKernelArgs {
    RopeArgs A;
    int rb;      // rows of a workgroup
    int turned;  // items of a head that turn, the others are copied
    int items;   // items of a head
};

// cos and sin of an angle in radians
__device__ __forceinline__ float2 cos_sin(double a) {
    const double k = __builtin_rint(a * 0x1.45f306dc9c883p-1);  // 2 / pi
    const double r = __builtin_fma(k, -0x1.1a62633145c07p-54, __builtin_fma(k, -0x1.921fb54442d18p+0, a));
    const float x = (float)r, x2 = x * x;
    float s = __builtin_fmaf(x2, 1.0f / 362880.0f, -1.0f / 5040.0f);
    s = __builtin_fmaf(s, x2, 1.0f / 120.0f);
    s = __builtin_fmaf(s, x2, -1.0f / 6.0f);
    s = __builtin_fmaf(s * x2, x, x);
    float c = __builtin_fmaf(x2, -1.0f / 3628800.0f, 1.0f / 40320.0f);
    c = __builtin_fmaf(c, x2, -1.0f / 720.0f);
    c = __builtin_fmaf(c, x2, 1.0f / 24.0f);
    c = __builtin_fmaf(c, x2, -0.5f);
    c = __builtin_fmaf(c, x2, 1.0f);
    // the quadrant: k mod 4 (k is a whole number below 2^52 for any angle that has digits to reduce)
    const double q = k - 4.0 * __builtin_floor(k * 0.25);
    const bool swap = q == 1.0 || q == 3.0;
    const float cc = swap ? s : c, ss = swap ? c : s;
    return float2{q == 1.0 || q == 2.0 ? -cc : cc, q >= 2.0 ? -ss : ss};
}

// V elements an item: of each half of V pairs (HALF), or V / 2 pairs side by side; V = 1: one pair
template <class E, int V, bool HALF>
__global__ __launch_bounds__(NT) void rope_kernel(RopeKernelArgs K) {
    extern __shared__ float2 turn[];  // [rb][pairs]
    const RopeArgs& A = K.A;
    const int64_t row0 = (int64_t)blockIdx.x * K.rb;
    const int rows = (int)min((int64_t)K.rb, A.rows - row0);
    for (int i = threadIdx.x; i < rows * A.pairs; i += NT) {
        const int r = i / A.pairs;
        const float2 t = cos_sin((double)A.pos[row0 + r] * A.freq[i - r * A.pairs]);
        turn[i] = float2{t.x * A.factor, t.y * A.factor};
    }
    __syncthreads();
    const int heads = A.q_heads + A.k_heads, per_row = heads * K.items;
    // the y-th part of the heads' items (few rows: each has several workgroups)
    for (int id = blockIdx.y * NT + threadIdx.x; id < rows * per_row; id += gridDim.y * NT) {
        const int r = id / per_row, in_row = id - r * per_row, head = in_row / K.items, item = in_row - head * K.items;
        const bool key = head >= A.q_heads;
        const jyhip_vectors& in = key ? A.k : A.q;
        const jyhip_vectors& to = key ? A.k_out : A.q_out;
        const int64_t row = row0 + r;
        const int h = key ? head - A.q_heads : head;
        const E* const src = static_cast<const E*>(in.data) + row * in.row_stride + h * in.head_stride;
        E* const dst = static_cast<E*>(to.data) + row * to.row_stride + h * to.head_stride;
        const float2* const t = turn + r * A.pairs;
        constexpr bool VEC = V > 1;
        if (HALF || !VEC) {
            if (item < K.turned) {  // pairs item V ..
                const int i = HALF ? item * V : 2 * item, j = HALF ? i + A.pairs : i + 1;
                float x[V], y[V];
                load_n<E, V, VEC>(src + i, x);
                load_n<E, V, VEC>(src + j, y);
#pragma unroll
                for (int e = 0; e < V; e++) {
                    const float2 cs = t[item * V + e];
                    const float u = __builtin_fmaf(x[e], cs.x, -(y[e] * cs.y));
                    y[e] = __builtin_fmaf(x[e], cs.y, y[e] * cs.x);
                    x[e] = u;
                }
                store_n<E, V, VEC>(dst + i, x);
                store_n<E, V, VEC>(dst + j, y);
            } else {
                const int i = 2 * A.pairs + (item - K.turned) * V;
                float x[V];
                load_n<E, V, VEC>(src + i, x);
                store_n<E, V, VEC>(dst + i, x);
            }
        } else {
            float x[V];
            load_n<E, V, VEC>(src + item * V, x);
            if (item < K.turned) {
#pragma unroll
                for (int e = 0; e < V; e += 2) {
                    const float2 cs = t[(item * V + e) / 2];
                    const float u = __builtin_fmaf(x[e], cs.x, -(x[e + 1] * cs.y));
                    x[e + 1] = __builtin_fmaf(x[e], cs.y, x[e + 1] * cs.x);
                    x[e] = u;
                }
            }
            store_n<E, V, VEC>(dst + item * V, x);
        }
    }
}

bool aligned16(const jyhip_vectors& x, int type) {
    const long long e = type == JYHIP_T_F32 ? 4 : 2;
    return ((uintptr_t)x.data | (uintptr_t)(x.row_stride * e) | (uintptr_t)(x.head_stride * e)) % 16 == 0;
}

// Rows of a workgroup: as many as give each thread a pair, where that leaves four workgroups a CU; else
// one, its heads shared by several workgroups (which compute its angles again), two vectors of 16 bytes a
// thread.
struct Grid {
    int rb;
    unsigned x, y;
};
Grid grid_of(const RopeArgs& A) {
    Grid g;
    g.rb = std::max(1, NT / A.pairs);
    if ((A.rows + g.rb - 1) / g.rb < 1024) g.rb = 1;
    g.x = (unsigned)((A.rows + g.rb - 1) / g.rb);
    const int64_t bytes = (int64_t)(A.q_heads + A.k_heads) * A.hd * (A.type == JYHIP_T_F32 ? 4 : 2);
    g.y = g.rb > 1 ? 1 : (unsigned)std::min<int64_t>(64, std::max<int64_t>(1, bytes / (32 * NT)));
    return g;
}

template <class E, int V, bool HALF>
void launch_form(const RopeArgs& A, hipStream_t st) {
    RopeKernelArgs K;
    K.A = A;
    const Grid g = grid_of(A);
    K.rb = g.rb;
    K.turned = V == 1 || HALF ? A.pairs / V : 2 * A.pairs / V;
    K.items = K.turned + (A.hd - 2 * A.pairs) / V;
    rope_kernel<E, V, HALF><<<dim3(g.x, g.y), NT, K.rb * A.pairs * sizeof(float2), st>>>(K);
}

template <class E>
void launch_type(const RopeArgs& A, hipStream_t st) {
    constexpr int V = 16 / (int)sizeof(E);
    const bool whole = A.hd % V == 0 && (A.interleaved ? 2 * A.pairs : A.pairs) % V == 0;
    const bool vec = whole && aligned16(A.q, A.type) && aligned16(A.q_out, A.type) &&
                     aligned16(A.k, A.type) && aligned16(A.k_out, A.type);  // (zeros where there are no heads)
    if (A.interleaved)
        vec ? launch_form<E, V, false>(A, st) : launch_form<E, 1, false>(A, st);
    else
        vec ? launch_form<E, V, true>(A, st) : launch_form<E, 1, true>(A, st);
}

}  // namespace

int64_t rope_blocks(const RopeArgs& A) {
    const Grid g = grid_of(A);
    return (int64_t)g.x * g.y;
}

void launch_rope(const RopeArgs& A, hipStream_t st) {
    if (A.type == JYHIP_T_F32)
        launch_type<float>(A, st);
    else if (A.type == JYHIP_T_F16)
        launch_type<_Float16>(A, st);
    else
        launch_type<__bf16>(A, st);
}

}  // namespace jy
