// jy_paged_attention.hip — attention of one new token per sequence over the paged cache.
#include <hip/hip_runtime.h>

#include "jy_device.h"
#include "jy_paged_device.h"

namespace jy {

namespace {

// One workgroup per (query head, sequence); its four waves take every fourth position, a lane
// holding dims lane, lane + 64, ... of the query and of the wave's output.
template <int PT, int T>
__global__ __launch_bounds__(256) void paged_attend_kernel(PagedAttn A) {
    typedef elem_t<PT> PE;
    typedef elem_t<T> E;
    __shared__ float so[4][256], sm[4], sl[4];
    const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const jyhip_pages& P = A.P;
    const int hd = P.head_dim, g = h / (A.nh / P.num_kv_heads);
    const int n = min(A.lens[b], A.max_len);
    float q[4], o[4] = {0, 0, 0, 0}, m = -3.0e38f, l = 0.0f;
    for (int i = 0; i < 4; i++) {
        const int d = lane + 64 * i;
        q[i] = d < hd ? (float)(static_cast<const E*>(A.q.data) + b * A.q.row_stride + h * A.q.head_stride)[d] : 0.0f;
    }
    for (int j = wave; j < n; j += 4) {
        const int64_t slot = slot_of(A.M, P.num_pages, P.page_size, b, j);
        if (slot < 0) continue;
        const int64_t vec = ((slot / P.page_size) * P.num_kv_heads + g) * P.page_size + slot % P.page_size;
        float s = 0.0f;
        for (int i = 0; i < 4; i++) {
            const int d = lane + 64 * i;
            if (d < hd) s += q[i] * (float)static_cast<const PE*>(P.k)[vec * hd + d];
        }
        for (int x = 32; x; x >>= 1) s += __shfl_xor(s, x);
        s *= A.scale;
        float vs = 1.0f;
        if (PT == JYHIP_T_I8) {
            s *= P.k_scale[vec];
            vs = P.v_scale[vec];
        }
        const float mn = fmaxf(m, s), alpha = expf(m - mn), p = expf(s - mn);
        m = mn;
        l = l * alpha + p;
        for (int i = 0; i < 4; i++) {
            const int d = lane + 64 * i;
            if (d < hd) o[i] = o[i] * alpha + p * vs * (float)static_cast<const PE*>(P.v)[vec * hd + d];
        }
    }
    for (int i = 0; i < 4; i++) so[wave][lane + 64 * i] = o[i];
    if (lane == 0) {
        sm[wave] = m;
        sl[wave] = l;
    }
    __syncthreads();
    const int d = threadIdx.x;
    if (d >= hd) return;
    float mx = sm[0], sum = 0.0f, acc = 0.0f;
    for (int w = 1; w < 4; w++) mx = fmaxf(mx, sm[w]);
    for (int w = 0; w < 4; w++) {
        const float f = expf(sm[w] - mx);
        sum += f * sl[w];
        acc += f * so[w][d];
    }
    (static_cast<E*>(A.out.data) + b * A.out.row_stride + h * A.out.head_stride)[d] = (E)(sum == 0.0f ? 0.0f : acc / sum);
}

template <int PT>
void launch_io(const PagedAttn& A, hipStream_t st) {
    const dim3 grid(A.nh, A.M.nseq);
    if (A.type == JYHIP_T_F32)
        paged_attend_kernel<PT, JYHIP_T_F32><<<grid, 256, 0, st>>>(A);
    else if (A.type == JYHIP_T_F16)
        paged_attend_kernel<PT, JYHIP_T_F16><<<grid, 256, 0, st>>>(A);
    else
        paged_attend_kernel<PT, JYHIP_T_BF16><<<grid, 256, 0, st>>>(A);
}

}  // namespace

size_t paged_attend_part_floats(const jyhip_pages&, int, int, int) { return 0; }

void launch_paged_attend(const PagedAttn& A, hipStream_t st) {
    if (A.P.type == JYHIP_T_I8)
        launch_io<JYHIP_T_I8>(A, st);
    else if (A.P.type == JYHIP_T_F16)
        launch_io<JYHIP_T_F16>(A, st);
    else
        launch_io<JYHIP_T_BF16>(A, st);
}

}  // namespace jy
