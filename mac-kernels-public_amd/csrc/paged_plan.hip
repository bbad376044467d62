// The tables of one step over a paged cache, from request lengths on the GPU: pages for the new
// tokens, each token's slot, position and request.  All integers; what bounds it is the latency of
// one launch and three dependent reads (lengths, their sums, a token's page): 4.5 us on the GPU for 32 requests of one new token,
// 5.4 for 256 with 23487.
//
// Every workgroup adds up all requests' new tokens and missing pages in LDS (at most 4096 of each), so
// that no second launch and no exchange between workgroups is needed; then each takes a share of the
// new tokens and of the new pages, and finds the request of either by bisection of the sums.
#include "attention.h"

namespace qlin {
namespace {

constexpr int THREADS = 256;
constexpr int64_t MOST = 0x7FFFFFFF;

// Largest i with sum[i] <= x among sum[0] = 0 <= sum[1] <= ... <= sum[n - 1]; x >= 0.
template <typename T>
__device__ __forceinline__ int find(const T* sum, int n, T x) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (sum[mid] <= x) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__global__ __launch_bounds__(THREADS) void paged_plan_kernel(PagedPlanArgs a) {
    extern __shared__ int64_t lds[];
    int64_t* first = lds;                                   // [B + 1]: missing pages before request b
    int32_t* starts = reinterpret_cast<int32_t*>(lds + a.B + 1);  // [B + 1]: new tokens before request b
    __shared__ int64_t wave_tokens[THREADS / 64], wave_pages[THREADS / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = (a.B + THREADS - 1) / THREADS, b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);

    // running sums, in 64 bits; a start that does not fit 32 stays at the largest value, which no place reaches
    int64_t tokens = 0, pages = 0;
    for (int b = b0; b < b1; ++b) {
        const int64_t c = max(a.context[b], 0), n = max(a.added[b], 0);
        tokens += n;
        pages += (c + n + a.page - 1) / a.page - (c + a.page - 1) / a.page;
    }
    int64_t st = tokens, sp = pages;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const int64_t x = __shfl_up(st, m), y = __shfl_up(sp, m);
        if (lane >= m) {
            st += x;
            sp += y;
        }
    }
    if (lane == 63) {
        wave_tokens[wave] = st;
        wave_pages[wave] = sp;
    }
    __syncthreads();
    st -= tokens;
    sp -= pages;
    for (int w = 0; w < wave; ++w) {
        st += wave_tokens[w];
        sp += wave_pages[w];
    }
    for (int b = b0; b < b1; ++b) {
        const int64_t c = max(a.context[b], 0), n = max(a.added[b], 0);
        starts[b] = (int32_t)min(st, MOST);
        first[b] = sp;
        st += n;
        sp += (c + n + a.page - 1) / a.page - (c + a.page - 1) / a.page;
    }
    if (tid == THREADS - 1) {
        starts[a.B] = (int32_t)min(st, MOST);
        first[a.B] = sp;
    }
    __syncthreads();

    const int64_t all = (int64_t)gridDim.x * THREADS, me = (int64_t)blockIdx.x * THREADS + tid;
    for (int64_t b = me; b <= a.B; b += all) {
        a.starts[b] = starts[b];
        if (b < a.B) a.lengths[b] = (int32_t)min((int64_t)max(a.context[b], 0) + max(a.added[b], 0), MOST);
    }
    if (me == 0) a.used[0] = (int32_t)min(first[a.B], MOST);
    const int64_t needed = first[a.B];
    for (int64_t e = me; e < needed; e += all) {  // the new entries of the table
        const int b = find(first, a.B + 1, e);
        const int64_t at = ((int64_t)max(a.context[b], 0) + a.page - 1) / a.page + (e - first[b]);
        if (at < a.W) a.table[b * a.ldt + at] = e < a.F ? a.free_blocks[e] : -1;
        // the request's other pages have no entry either, and a length that is wrong by far must not take a step for each
        else e += (first[b + 1] - e - 1) / all * all;
    }
    const int total = starts[a.B];
    for (int64_t i = me; i < a.N; i += all) {
        int32_t row = -1, position = -1;
        int64_t slot = -1;
        if (i < total) {
            row = find(starts, a.B + 1, (int)i);
            const int64_t c = max(a.context[row], 0), p = c + (i - starts[row]), at = p / a.page, old = (c + a.page - 1) / a.page;
            position = (int32_t)min(p, MOST);
            int64_t block = -1;
            if (at < a.W) {
                const int64_t e = first[row] + (at - old);
                block = at < old ? a.table[row * a.ldt + at] : e < a.F ? a.free_blocks[e] : -1;
            }
            if (block >= 0) slot = block * a.page + (p - at * a.page);
        }
        a.rows[i] = row;
        a.positions[i] = position;
        a.slots[i] = slot;
    }
}

}  // namespace

hipError_t run_paged_plan(const PagedPlanArgs& a, hipStream_t st) {
    const int64_t work = std::max<int64_t>(a.N, a.B + 1);
    const unsigned grid = (unsigned)std::min<int64_t>((work + THREADS - 1) / THREADS, 256);
    hipLaunchKernelGGL(paged_plan_kernel, dim3(grid), dim3(THREADS), (size_t)12 * (a.B + 1), st, a);
    return hipGetLastError();
}

}  // namespace qlin
