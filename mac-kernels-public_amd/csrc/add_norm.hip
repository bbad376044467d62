// Root-mean-square norm with the residual's addition: h = x + r, y = w h rho, rho = (mean h^2 + eps)^-1/2, y in 16 or 32
// bits or in 8 with a scale a row, and its gradient.  Bound by memory: every value is read once and written once.
//
// A row stays in registers between its reads and its writes.  8 bits: the codes are rne(127 v / top) with v = w h
// (rotated, for weights that are stored so) and top the row's largest |v|; rho cancels in them, so that one
// exchange between a row's threads gives both the sum of squares and top, and the scale is top rho / 127.
#include <algorithm>

#include "mlp_rows.h"

namespace qlin {
namespace {

// The sum of a and the largest of b over the threads of a row: a wave's lanes, or all of a workgroup's.
template <bool WAVE>
__device__ __forceinline__ void row_sum_max(float& a, uint32_t& b) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        a += __shfl_xor(a, m, 64);
        b = max(b, (uint32_t)__shfl_xor((int)b, m, 64));
    }
    if constexpr (!WAVE) {
        __shared__ float sums[16];
        __shared__ uint32_t tops[16];
        if (lane == 0) {
            sums[wave] = a;
            tops[wave] = b;
        }
        __syncthreads();
        a = 0.0f;
        for (int i = 0; i < waves; ++i) {
            a += sums[i];
            b = max(b, tops[i]);
        }
    }
}

// A row a workgroup, or (WAVE) a wave; every thread holds SLOTS runs of RUN values.  SLOTS 0: rows of any length, read
// twice.  T: x and y, H: the residual and h.
template <typename T, typename H, int RUN, int SLOTS, bool INT8, bool WAVE>
__global__ __launch_bounds__(1024) void add_norm_kernel(AddNormArgs a, int64_t t0) {
    const int lane = threadIdx.x & 63;
    const int per = WAVE ? 64 : (int)blockDim.x, at = WAVE ? lane : (int)threadIdx.x;
    const int64_t t = t0 + (WAVE ? (int64_t)blockIdx.x * (blockDim.x >> 6) + (threadIdx.x >> 6) : (int64_t)blockIdx.x);
    if (t >= a.T) return;  // a whole wave's (WAVE), or no thread's
    const T* x = (const T*)a.x.p + t * a.x.ld;
    const H* r = a.r.p ? (const H*)a.r.p + t * a.r.ld : nullptr;
    H* h = a.r.p ? (H*)a.h.p + t * a.h.ld : nullptr;
    float ss = 0.0f;
    uint32_t top = 0;
    auto sum_of = [&](int e0, float* v) {
        const int n = a.W - e0;
        load_run<T, RUN>(x + e0, n, v);
        if (r) {
            float u[RUN];
            load_run<H, RUN>(r + e0, n, u);
#pragma unroll
            for (int i = 0; i < RUN; ++i) v[i] += u[i];
        }
    };
    // the weighted values, rotated: what the 8-bit output holds but for rho
    auto weigh = [&](int e0, float* v) {
        if (a.w) {
            float w[RUN];
            load_run_rt<RUN>(a.w, a.w_dt, e0, a.W - e0, w);
#pragma unroll
            for (int i = 0; i < RUN; ++i) v[i] *= w[i];
        }
        if constexpr (INT8 && RUN == 16) rotate_run(v, a.G, lane);
    };
    auto squares = [&](const float* v) {
#pragma unroll
        for (int i = 0; i < RUN; ++i) ss = __builtin_fmaf(v[i], v[i], ss);
    };
    auto largest = [&](const float* v) {
#pragma unroll
        for (int i = 0; i < RUN; ++i) top = max(top, abs_bits(v[i]));
    };
    auto emit = [&](int e0, float* v, float rho, float inv, float first) {
        const int n = a.W - e0;
        if constexpr (INT8) {
            if (first != 1.0f)
#pragma unroll
                for (int i = 0; i < RUN; ++i) v[i] *= first;
            if (n > 0) store_codes<RUN>(a.q + t * a.ldq + e0, n, v, inv);
        } else {
#pragma unroll
            for (int i = 0; i < RUN; ++i) v[i] *= rho;
            if (n > 0) store_run<T, RUN>((T*)a.y.p + t * a.y.ld + e0, n, v);
        }
    };
    auto finish = [&](float& rho, float& inv, float& first) {
        row_sum_max<WAVE>(ss, top);
        rho = 1.0f / sqrtf(ss / (float)a.W + a.eps);
        if constexpr (INT8) {
            const float largest_v = __uint_as_float(top);
            inv = code_factor(largest_v, first);
            if (at == 0) a.scale[t] = largest_v / 127.0f * rho;
        }
    };
    float rho, inv = 0.0f, first = 1.0f;
    if constexpr (SLOTS > 0) {
        float v[SLOTS][RUN];
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) sum_of((s * per + at) * RUN, v[s]);
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            const int e0 = (s * per + at) * RUN;
            if (h && e0 < a.W) store_run<H, RUN>(h + e0, a.W - e0, v[s]);
            squares(v[s]);
            weigh(e0, v[s]);
            if constexpr (INT8) largest(v[s]);
        }
        finish(rho, inv, first);
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) emit((s * per + at) * RUN, v[s], rho, inv, first);
    } else {
        float v[RUN];
        for (int c = 0; c < a.W; c += per * RUN) {
            sum_of(c + at * RUN, v);
            squares(v);
            if constexpr (INT8) {
                weigh(c + at * RUN, v);
                largest(v);
            }
        }
        finish(rho, inv, first);
        for (int c = 0; c < a.W; c += per * RUN) {
            const int e0 = c + at * RUN;
            sum_of(e0, v);
            if (h && e0 < a.W) store_run<H, RUN>(h + e0, a.W - e0, v);
            weigh(e0, v);
            emit(e0, v, rho, inv, first);
        }
    }
}

// dx = rho (g - h rho^2 mean(g h)) + dh with g = w dy, and a workgroup's part of dw = sum_t dy h rho.
template <typename T, typename H, int SLOTS>
__global__ __launch_bounds__(1024) void add_norm_grad_kernel(AddNormGradArgs a) {
    constexpr int RUN = 8;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int per = blockDim.x, at = threadIdx.x;
    __shared__ float red[2][16][2];
    float w[SLOTS][RUN], dw[SLOTS][RUN];
#pragma unroll
    for (int s = 0; s < SLOTS; ++s)
#pragma unroll
        for (int i = 0; i < RUN; ++i) {
            w[s][i] = 1.0f;
            dw[s][i] = 0.0f;
        }
    if (a.w)
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            const int e0 = (s * per + at) * RUN;
            load_run_rt<RUN>(a.w, a.w_dt, e0, a.W - e0, w[s]);
        }
    int turn = 0;
    for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x, turn ^= 1) {
        float g[SLOTS][RUN], h[SLOTS][RUN], d[SLOTS][RUN];
        float ss = 0.0f, gh = 0.0f;
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            const int e0 = (s * per + at) * RUN, n = a.W - e0;
            load_run<T, RUN>((const T*)a.dy.p + t * a.dy.ld + e0, n, g[s]);
            load_run<H, RUN>((const H*)a.h.p + t * a.h.ld + e0, n, h[s]);
            if (a.dh.p) load_run<H, RUN>((const H*)a.dh.p + t * a.dh.ld + e0, n, d[s]);
        }
#pragma unroll
        for (int s = 0; s < SLOTS; ++s)
#pragma unroll
            for (int i = 0; i < RUN; ++i) {
                ss = __builtin_fmaf(h[s][i], h[s][i], ss);
                gh = __builtin_fmaf(g[s][i] * w[s][i], h[s][i], gh);
            }
        ss = wave_sum(ss);
        gh = wave_sum(gh);
        if (lane == 0) {
            red[turn][wave][0] = ss;
            red[turn][wave][1] = gh;
        }
        __syncthreads();  // the other turn's sums were read before this barrier
        ss = gh = 0.0f;
        for (int i = 0; i < waves; ++i) {
            ss += red[turn][i][0];
            gh += red[turn][i][1];
        }
        const float rho = 1.0f / sqrtf(ss / (float)a.W + a.eps);
        const float c = rho * rho * (gh / (float)a.W);
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            const int e0 = (s * per + at) * RUN;
            float o[RUN];
#pragma unroll
            for (int i = 0; i < RUN; ++i) {
                dw[s][i] = __builtin_fmaf(g[s][i], h[s][i] * rho, dw[s][i]);
                o[i] = rho * (g[s][i] * w[s][i] - h[s][i] * c);
                if (a.dh.p) o[i] += d[s][i];
            }
            if (e0 < a.W) store_run<H, RUN>((H*)a.dx.p + t * a.dx.ld + e0, a.W - e0, o);
        }
    }
    if (a.dw)
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            const int e0 = (s * per + at) * RUN;
            if (e0 < a.W) store_run<float, RUN>(a.part + (int64_t)blockIdx.x * a.W + e0, a.W - e0, dw[s]);
        }
}

// Rows of any length: the row's sums, then its gradient; dw by add_norm_dw_kernel from rho.
template <typename T, typename H>
__global__ __launch_bounds__(1024) void add_norm_grad_long_kernel(AddNormGradArgs a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __shared__ float red[2][16][2];
    float* part = a.dw ? a.part + (int64_t)blockIdx.x * a.W : nullptr;
    int turn = 0;
    bool begun = false;
    for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x, turn ^= 1) {
        const T* dy = (const T*)a.dy.p + t * a.dy.ld;
        const H* h = (const H*)a.h.p + t * a.h.ld;
        const H* dh = a.dh.p ? (const H*)a.dh.p + t * a.dh.ld : nullptr;
        H* dx = (H*)a.dx.p + t * a.dx.ld;
        float ss = 0.0f, gh = 0.0f;
        for (int e = threadIdx.x; e < a.W; e += blockDim.x) {
            const float v = (float)h[e], g = (float)dy[e] * (a.w ? load_rt(a.w, a.w_dt, e) : 1.0f);
            ss = __builtin_fmaf(v, v, ss);
            gh = __builtin_fmaf(g, v, gh);
        }
        ss = wave_sum(ss);
        gh = wave_sum(gh);
        if (lane == 0) {
            red[turn][wave][0] = ss;
            red[turn][wave][1] = gh;
        }
        __syncthreads();
        ss = gh = 0.0f;
        for (int i = 0; i < (int)(blockDim.x >> 6); ++i) {
            ss += red[turn][i][0];
            gh += red[turn][i][1];
        }
        const float rho = 1.0f / sqrtf(ss / (float)a.W + a.eps);
        const float c = rho * rho * (gh / (float)a.W);
        for (int e = threadIdx.x; e < a.W; e += blockDim.x) {  // an element is the same thread's in every row
            const float v = (float)h[e], g = (float)dy[e], w = a.w ? load_rt(a.w, a.w_dt, e) : 1.0f;
            if (part) part[e] = __builtin_fmaf(g, v * rho, begun ? part[e] : 0.0f);
            dx[e] = (H)(rho * (g * w - v * c) + (dh ? (float)dh[e] : 0.0f));
        }
        begun = true;
    }
}

// dw[e] = the parts' sum: 16 threads add every 16th part of a column, then their sums, always in this order.
__global__ __launch_bounds__(256) void add_norm_dw_kernel(const float* part, int parts, int W, void* dw, int dw_dt) {
    __shared__ float sums[16][17];
    const int c = threadIdx.x & 15, i = threadIdx.x >> 4, e = blockIdx.x * 16 + c;
    float s = 0.0f;
    if (e < W)
        for (int p = i; p < parts; p += 16) s += part[(int64_t)p * W + e];
    sums[i][c] = s;
    __syncthreads();
    if (i || e >= W) return;
    for (int j = 1; j < 16; ++j) s += sums[j][c];
    store_rt(dw, dw_dt, e, s);
}

constexpr int GRAD_PARTS = 512;

int grad_parts(int64_t T) { return (int)std::min<int64_t>(T, GRAD_PARTS); }

template <typename T, typename H, int RUN, bool INT8>
hipError_t launch_norm(const AddNormArgs& a, hipStream_t st) {
    int slots = 0;
    const int n = row_threads(a.W, RUN, slots);
    const int64_t most = (int64_t)(0x7FFFFFFF / n);  // workgroups of one launch: a grid's threads count to 2^32
    for (int64_t t0 = 0; t0 < a.T; t0 += most) {
        const dim3 grid((unsigned)std::min<int64_t>(most, a.T - t0)), block((unsigned)n);
        switch (slots) {
            case 1: hipLaunchKernelGGL((add_norm_kernel<T, H, RUN, 1, INT8, false>), grid, block, 0, st, a, t0); break;
            case 2: hipLaunchKernelGGL((add_norm_kernel<T, H, RUN, 2, INT8, false>), grid, block, 0, st, a, t0); break;
            case 4: hipLaunchKernelGGL((add_norm_kernel<T, H, RUN, 4, INT8, false>), grid, block, 0, st, a, t0); break;
            default: hipLaunchKernelGGL((add_norm_kernel<T, H, RUN, 0, INT8, false>), grid, block, 0, st, a, t0); break;
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

template <typename T, typename H>
hipError_t norm_of(const AddNormArgs& a, hipStream_t st) {
    if (!a.q) return launch_norm<T, H, 8, false>(a, st);
    return a.G ? launch_norm<T, H, 16, true>(a, st) : launch_norm<T, H, 8, true>(a, st);
}

template <typename T, typename H>
hipError_t grad_of(const AddNormGradArgs& a, hipStream_t st) {
    int slots = 0;
    const int n = row_threads(a.W, 8, slots), parts = grad_parts(a.T);
    const dim3 grid((unsigned)parts), block((unsigned)n);
    switch (slots) {
        case 1: hipLaunchKernelGGL((add_norm_grad_kernel<T, H, 1>), grid, block, 0, st, a); break;
        case 2: hipLaunchKernelGGL((add_norm_grad_kernel<T, H, 2>), grid, block, 0, st, a); break;
        default: hipLaunchKernelGGL((add_norm_grad_long_kernel<T, H>), grid, block, 0, st, a); break;
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !a.dw) return e;
    hipLaunchKernelGGL(add_norm_dw_kernel, dim3((unsigned)((a.W + 15) / 16)), dim3(256), 0, st, a.part, parts, a.W, a.dw, a.dw_dt);
    return hipGetLastError();
}

template <typename Args, typename F>
hipError_t by_types(const Args& a, F&& f) {
    if (a.dtype == DT_F32) return f.template operator()<float, float>();
    if (a.dtype == DT_F16) return a.h_dtype == DT_F32 ? f.template operator()<f16, float>() : f.template operator()<f16, f16>();
    return a.h_dtype == DT_F32 ? f.template operator()<__bf16, float>() : f.template operator()<__bf16, __bf16>();
}

}  // namespace

hipError_t run_add_norm(const AddNormArgs& a, hipStream_t st) {
    if (a.T == 0 || a.W == 0) return hipSuccess;
    return by_types(a, [&]<typename T, typename H>() { return norm_of<T, H>(a, st); });
}

size_t ws_add_norm_grad(int64_t T, int64_t W) { return (size_t)grad_parts(T) * W * 4; }

hipError_t run_add_norm_grad(const AddNormGradArgs& a, hipStream_t st) {
    if (a.W == 0) return hipSuccess;
    if (a.T == 0 && !a.dw) return hipSuccess;
    if (a.T == 0) {  // a sum over no rows
        hipLaunchKernelGGL(add_norm_dw_kernel, dim3((unsigned)((a.W + 15) / 16)), dim3(256), 0, st, a.part, 0, a.W, a.dw, a.dw_dt);
        return hipGetLastError();
    }
    return by_types(a, [&]<typename T, typename H>() { return grad_of<T, H>(a, st); });
}

}  // namespace qlin
