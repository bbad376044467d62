// Attention of one new token a row over a paged cache.  One wave a (row, head): the cache's tokens one
// by one, their values over the lanes, with the running maximum and sum of the softmax in fp32.
#include "attention.h"

namespace qlin {
namespace {

template <int DT>
__global__ __launch_bounds__(64) void paged_attention_kernel(PagedAttentionArgs a) {
    const int lane = threadIdx.x;
    const int64_t b = blockIdx.x / a.H;
    const int h = (int)(blockIdx.x % a.H), g = h / (a.H / a.Hk);
    const int64_t len = min((int64_t)max(a.lengths[b], 0), a.W * a.page);
    const int64_t first = a.window && len > a.window ? len - a.window : 0;
    float q[4], o[4] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = lane + 64 * j < a.D ? load_rt(a.q.p, DT, b * a.q.st + h * a.q.sh + lane + 64 * j) : 0.0f;
    for (int64_t s = first; s < len; ++s) {
        const int64_t block = a.table[b * a.ldt + s / a.page];
        if (block < 0 || block >= a.blocks) continue;
        float dot = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (lane + 64 * j < a.D)
                dot += q[j] * load_rt(a.kc.p, DT, block * a.kc.sb + (s % a.page) * a.kc.sp + g * a.kc.sh + lane + 64 * j);
        dot = wave_sum(dot) * a.scale;
        const float mn = fmaxf(m, dot), base = mn == -INFINITY ? 0.0f : mn;
        const float keep = expf(m - base), p = expf(dot - base);
        m = mn;
        l = l * keep + p;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (lane + 64 * j < a.D)
                o[j] = o[j] * keep + p * load_rt(a.vc.p, DT, block * a.vc.sb + (s % a.page) * a.vc.sp + g * a.vc.sh + lane + 64 * j);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (lane + 64 * j < a.D)
            store_rt(a.out.p, DT, b * a.out.st + h * a.out.sh + lane + 64 * j, l == 0.0f ? 0.0f : o[j] / l);
}

}  // namespace

size_t ws_paged_attention(int64_t, int64_t, int64_t, int64_t) { return 0; }

hipError_t run_paged_attention(const PagedAttentionArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)(a.B * a.H));
    if (a.dtype == DT_F16) hipLaunchKernelGGL(paged_attention_kernel<DT_F16>, grid, dim3(64), 0, st, a);
    else hipLaunchKernelGGL(paged_attention_kernel<DT_BF16>, grid, dim3(64), 0, st, a);
    return hipGetLastError();
}

}  // namespace qlin
