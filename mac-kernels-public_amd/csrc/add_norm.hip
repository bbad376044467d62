// Root-mean-square norm with the residual's addition: h = x + r, y = w h rho, rho = (mean h^2 + eps)^-1/2, y in 16 or 32
// bits or in 8 with a scale a row, and its gradient.  Bound by memory: every value is read once and written once.
//
// A row stays in registers between its reads and its writes, 8 or 16 values a thread, a row (or a few short ones) a workgroup.  8
// bits: the codes are rne(127 v / top) with v = w h (rotated, for weights that are stored so) and top the row's largest |v|;
// rho cancels in them, so that one exchange between a row's threads gives both the sum of squares and top, and the scale is
// top rho / 127.  (Workgroups that take rows in turn, the next one's reads in flight, are no faster: 4608 x 6144 to bf16 50 us
// against 49 before either wrote nontemporally; the gradient is so because its workgroups keep partial sums.)
//
// 4608 x 6144 to bf16 41 us (36 at 6.3 TB/s), to int8 36 (31), rotated by 128 41; gradient of 9504 x 5120 75 (62).
#include "mlp_rows.h"

namespace qlin {
namespace {

// T: x and y, H: the residual and h.  RUN 4: rotated.  RES: with a residual.  ONCE: nontemporal reads and writes.
template <typename T, typename H, int RUN, int SLOTS, bool INT8, bool RES, bool ONCE>
__global__ __launch_bounds__(1024, SLOTS * RUN > 16 ? 4 : 6) void add_norm_kernel(AddNormArgs a, int64_t t0, int per, int groups) {
    const Group g(per);
    const Rotation turned(RUN == 4 ? a.G : 1, g.lane);
    const int64_t t = t0 + (int64_t)blockIdx.x * groups + g.wave / g.waves;
    const bool live = t < a.T;
    const int64_t from = live ? t : a.T - 1;
    const int e0 = g.place<RUN>(), apart = per * RUN;
    Run<T, RUN> x[SLOTS];
    Run<H, RUN> r[SLOTS];
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
        x[s] = load_piece<ONCE, T, RUN>((const T*)a.x.p + from * a.x.ld, e0 + s * apart, a.W);
        if constexpr (RES) r[s] = load_piece<ONCE, H, RUN>((const H*)a.r.p + from * a.r.ld, e0 + s * apart, a.W);
    }
    float v[SLOTS][RUN], w[SLOTS][RUN];
    if (a.w) load_pieces_rt<ONCE, RUN, SLOTS>(a.w, a.w_dt, e0, apart, a.W, w);
    float ss = 0.0f;
    float top = 0.0f;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
        const int e = e0 + s * apart;
        trimmed<ONCE, T, RUN>(x[s], e, a.W, v[s]);
        if constexpr (RES) {
            float u[RUN];
            trimmed<ONCE, H, RUN>(r[s], e, a.W, u);
#pragma unroll
            for (int i = 0; i < RUN; ++i) v[s][i] += u[i];
            if (live && e < a.W) store_run<ONCE, H, RUN>((H*)a.h.p + t * a.h.ld + e, a.W - e, v[s]);
        }
        float sq = 0.0f;
#pragma unroll
        for (int i = 0; i < RUN; ++i) sq = __builtin_fmaf(v[s][i], v[s][i], sq);
        ss += e < a.W ? sq : 0.0f;
        if (a.w)
#pragma unroll
            for (int i = 0; i < RUN; ++i) v[s][i] *= w[s][i];
        if constexpr (RUN == 4) turned(v[s]);
        if constexpr (INT8) top = larger(top, e < a.W ? largest<RUN>(v[s]) : 0.0f);
    }
    g.sums(ss, top, 0, larger);
    const float rho = 1.0f / sqrtf(ss / (float)a.W + a.eps);
    if (!live) return;
    if constexpr (INT8) {
        const float most = top;
        float first;
        const float inv = code_factor(most, first);
        if (g.at == 0) a.scale[t] = most * (RUN == 4 ? turned.left : 1.0f) / 127.0f * rho;
        if (first != 1.0f)
#pragma unroll
            for (int s = 0; s < SLOTS; ++s)
#pragma unroll
                for (int i = 0; i < RUN; ++i) v[s][i] *= first;
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            const int e = e0 + s * apart;
            if (e < a.W) store_codes<ONCE, RUN>(a.q + t * a.ldq + e, a.W - e, v[s], inv);
        }
    } else {
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            const int e = e0 + s * apart;
#pragma unroll
            for (int i = 0; i < RUN; ++i) v[s][i] *= rho;
            if (e < a.W) store_run<ONCE, T, RUN>((T*)a.y.p + t * a.y.ld + e, a.W - e, v[s]);
        }
    }
}

// A thread's sum of a row of any length: of runs, sixteen of them at a time, so that 2^20 values meet 52 roundings in turn (4 + 16 + 32), where
// one after the other they would 2048 (equal values: y off by 2^-16).
struct LongSum {
    float all = 0.0f, part = 0.0f;
    int runs = 0;
    __device__ __forceinline__ void add(float run) {
        part += run;
        if (++runs & 15) return;
        all += part;
        part = 0.0f;
    }
    __device__ __forceinline__ float sum() const { return all + part; }
};

// Rows of any length, read twice.
template <typename T, typename H, int RUN, bool INT8>
__global__ __launch_bounds__(512) void add_norm_long_kernel(AddNormArgs a) {
    const Group g(512);
    const Rotation turned(RUN == 4 ? a.G : 1, g.lane);
    int turn = 0;
    for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x, turn ^= 1) {
        const T* x = (const T*)a.x.p + t * a.x.ld;
        const H* r = a.r.p ? (const H*)a.r.p + t * a.r.ld : nullptr;
        float v[RUN];
        auto sum_of = [&](int e0) {
            load_run<T, RUN>(x + e0, a.W - e0, v);
            if (r) {
                float u[RUN];
                load_run<H, RUN>(r + e0, a.W - e0, u);
#pragma unroll
                for (int i = 0; i < RUN; ++i) v[i] += u[i];
            }
        };
        auto weigh = [&](int e0) {
            if (a.w) {
                float u[RUN];
                load_run_rt<RUN>(a.w, a.w_dt, e0, a.W - e0, u);
#pragma unroll
                for (int i = 0; i < RUN; ++i) v[i] *= u[i];
            }
            if constexpr (RUN == 4) turned(v);
        };
        LongSum squares;
        float top = 0.0f;
        for (int c = 0; c < a.W; c += 512 * RUN) {
            const int e0 = c + g.place<RUN>();
            sum_of(e0);
            float sq = 0.0f;
#pragma unroll
            for (int i = 0; i < RUN; ++i) sq = __builtin_fmaf(v[i], v[i], sq);
            squares.add(sq);
            if constexpr (INT8) {
                weigh(e0);
                top = larger(top, largest<RUN>(v));
            }
        }
        float ss = squares.sum();
        g.sums(ss, top, turn, larger);
        const float rho = 1.0f / sqrtf(ss / (float)a.W + a.eps), most = top;
        float first = 1.0f;
        const float inv = INT8 ? code_factor(most, first) : 0.0f;
        if (INT8 && g.at == 0) a.scale[t] = most * (RUN == 4 ? turned.left : 1.0f) / 127.0f * rho;
        for (int c = 0; c < a.W; c += 512 * RUN) {
            const int e0 = c + g.place<RUN>();
            sum_of(e0);
            if (r && e0 < a.W) store_run<false, H, RUN>((H*)a.h.p + t * a.h.ld + e0, a.W - e0, v);
            weigh(e0);
#pragma unroll
            for (int i = 0; i < RUN; ++i) v[i] *= INT8 ? first : rho;
            if (e0 >= a.W) continue;
            if constexpr (INT8) store_codes<false, RUN>(a.q + t * a.ldq + e0, a.W - e0, v, inv);
            else store_run<false, T, RUN>((T*)a.y.p + t * a.y.ld + e0, a.W - e0, v);
        }
    }
}

// dx = rho (g - h rho^2 mean(g h)) + dh with g = w dy, and a workgroup's part of dw = sum_t dy h rho.  h is taken as it was stored: x and the
// residual in its place would be 10 bytes a value where 8 are, and one tensor more to keep.  With h in bf16 that is 1.8e-3 of dw (1056
// rows of 6144 normal values, root mean square: 2.4e-3 with dw's rounding to bf16, which alone is 1.65e-3) and 2e-5 of dx.
template <typename T, typename H, int SLOTS, bool DH, bool ONCE, int THREADS>
__global__ __launch_bounds__(THREADS) void add_norm_grad_kernel(AddNormGradArgs a, int per, int groups) {
    constexpr int RUN = 8;
    const Group g(per);
    struct Raw {
        Run<T, RUN> dy;
        Run<H, RUN> h, dh;
    };
    const int e0 = g.at * RUN, apart = per * RUN;
    auto fetch = [&](int64_t t, Raw (&o)[SLOTS]) {
        t = min(t, a.T - 1);
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            o[s].dy = load_piece<ONCE, T, RUN>((const T*)a.dy.p + t * a.dy.ld, e0 + s * apart, a.W);
            o[s].h = load_piece<ONCE, H, RUN>((const H*)a.h.p + t * a.h.ld, e0 + s * apart, a.W);
            if constexpr (DH) o[s].dh = load_piece<ONCE, H, RUN>((const H*)a.dh.p + t * a.dh.ld, e0 + s * apart, a.W);
        }
    };
    const int64_t step = (int64_t)gridDim.x * groups;
    int64_t t = (int64_t)blockIdx.x * groups + g.wave / g.waves;
    Raw raw[SLOTS];
    fetch(t, raw);
    float w[SLOTS][RUN], dw[SLOTS][RUN];
    if (a.w) load_pieces_rt<ONCE, RUN, SLOTS>(a.w, a.w_dt, e0, apart, a.W, w);
#pragma unroll
    for (int s = 0; s < SLOTS; ++s)
#pragma unroll
        for (int i = 0; i < RUN; ++i) {
            if (!a.w) w[s][i] = 1.0f;
            dw[s][i] = 0.0f;
        }
    int turn = 0;
    for (int64_t base = (int64_t)blockIdx.x * groups; base < a.T; base += step, t += step, turn ^= 1) {
        float d[SLOTS][RUN], h[SLOTS][RUN];
        Run<H, RUN> dh[SLOTS];
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            trimmed<ONCE, T, RUN>(raw[s].dy, e0 + s * apart, a.W, d[s]);
            trimmed<ONCE, H, RUN>(raw[s].h, e0 + s * apart, a.W, h[s]);
            if constexpr (DH) dh[s] = raw[s].dh;
        }
        if (base + step < a.T) fetch(t + step, raw);
        float ss = 0.0f, gh = 0.0f;
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            float sq = 0.0f, pr = 0.0f;
#pragma unroll
            for (int i = 0; i < RUN; ++i) {
                sq = __builtin_fmaf(h[s][i], h[s][i], sq);
                pr = __builtin_fmaf(d[s][i] * w[s][i], h[s][i], pr);
            }
            const bool in = e0 + s * apart < a.W;
            ss += in ? sq : 0.0f;
            gh += in ? pr : 0.0f;
        }
        g.sums(ss, gh, turn, [](float p, float q) { return p + q; });
        const float rho = 1.0f / sqrtf(ss / (float)a.W + a.eps);
        const float c = rho * rho * (gh / (float)a.W);
        if (t >= a.T) continue;
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            const int e = e0 + s * apart;
            float o[RUN], more[RUN] = {};
            if constexpr (DH) trimmed<ONCE, H, RUN>(dh[s], e, a.W, more);
#pragma unroll
            for (int i = 0; i < RUN; ++i) {
                dw[s][i] = __builtin_fmaf(d[s][i], h[s][i] * rho, dw[s][i]);
                {
#pragma clang fp contract(off)
                    // the same operations in every variant: rows of any alignment give the same bits
                    const float in = __builtin_fmaf(d[s][i], w[s][i], -(h[s][i] * c));
                    o[i] = DH ? __builtin_fmaf(rho, in, more[i]) : rho * in;
                }
            }
            if (e < a.W) store_run<ONCE && SLOTS == 1, H, RUN>((H*)a.dx.p + t * a.dx.ld + e, a.W - e, o);  // see grad_cut
        }
    }
    if (!a.dw) return;
    // the groups' sums, in their order, are the workgroup's
    __shared__ float other[256 * RUN];  // groups of fewer than 256 threads: one slot
    for (int k = 1; k < groups; ++k) {
        __syncthreads();
        if (g.wave / g.waves == k)
#pragma unroll
            for (int i = 0; i < RUN; ++i) other[g.at * RUN + i] = dw[0][i];
        __syncthreads();
        if (g.wave / g.waves == 0)
#pragma unroll
            for (int i = 0; i < RUN; ++i) dw[0][i] += other[g.at * RUN + i];
    }
    if (g.wave / g.waves) return;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
        const int e = e0 + s * apart;
        if (e < a.W) store_run<false, float, RUN>(a.part + (int64_t)blockIdx.x * a.W + e, a.W - e, dw[s]);
    }
}

// Rows of any length: the row's sums, then its gradient.  The partial sums stay in memory, a run the same thread's in every row.
template <typename T, typename H>
__global__ __launch_bounds__(512) void add_norm_grad_long_kernel(AddNormGradArgs a) {
    constexpr int RUN = 8;
    const Group g(512);
    float* part = a.dw ? a.part + (int64_t)blockIdx.x * a.W : nullptr;
    int turn = 0;
    bool begun = false;
    for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x, turn ^= 1) {
        const T* dy = (const T*)a.dy.p + t * a.dy.ld;
        const H* h = (const H*)a.h.p + t * a.h.ld;
        const H* dh = a.dh.p ? (const H*)a.dh.p + t * a.dh.ld : nullptr;
        H* dx = (H*)a.dx.p + t * a.dx.ld;
        float v[RUN], d[RUN], w[RUN];
        auto load = [&](int e) {
            load_run<H, RUN>(h + e, a.W - e, v);
            load_run<T, RUN>(dy + e, a.W - e, d);
            if (a.w) load_run_rt<RUN>(a.w, a.w_dt, e, a.W - e, w);
            else
#pragma unroll
                for (int i = 0; i < RUN; ++i) w[i] = 1.0f;
        };
        LongSum squares, products;
        for (int e = threadIdx.x * RUN; e < a.W; e += 512 * RUN) {
            load(e);
            float sq = 0.0f, pr = 0.0f;
#pragma unroll
            for (int i = 0; i < RUN; ++i) {
                sq = __builtin_fmaf(v[i], v[i], sq);
                pr = __builtin_fmaf(d[i] * w[i], v[i], pr);
            }
            squares.add(sq);
            products.add(pr);
        }
        float ss = squares.sum(), gh = products.sum();
        g.sums(ss, gh, turn, [](float p, float q) { return p + q; });
        const float rho = 1.0f / sqrtf(ss / (float)a.W + a.eps);
        const float c = rho * rho * (gh / (float)a.W);
        for (int e = threadIdx.x * RUN; e < a.W; e += 512 * RUN) {
            float sum[RUN] = {}, more[RUN] = {}, o[RUN];
            if (part && begun) load_run<float, RUN>(part + e, a.W - e, sum);
            if (dh) load_run<H, RUN>(dh + e, a.W - e, more);
            load(e);
#pragma unroll
            for (int i = 0; i < RUN; ++i) {
                sum[i] = __builtin_fmaf(d[i], v[i] * rho, sum[i]);
                o[i] = __builtin_fmaf(rho, __builtin_fmaf(d[i], w[i], -(v[i] * c)), more[i]);
            }
            if (part) store_run<false, float, RUN>(part + e, a.W - e, sum);
            store_run<false, H, RUN>(dx + e, a.W - e, o);
        }
        begun = true;
    }
}

// dw[e] = the parts' sum: 16 threads add every 16th part of a column, then their sums, always in this order.
__global__ __launch_bounds__(256) void add_norm_dw_kernel(const float* part, int parts, int W, void* dw, int dw_dt) {
    __shared__ float sums[16][17];
    const int c = threadIdx.x & 15, i = threadIdx.x >> 4, e = blockIdx.x * 16 + c;
    float s = 0.0f;
    if (e < W) {
        const float* p = part + e;
        int k = i;
        for (; k + 7 * 16 < parts; k += 8 * 16) {  // eight in flight
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = p[(int64_t)(k + 16 * j) * W];
#pragma unroll
            for (int j = 0; j < 8; ++j) s += v[j];
        }
        for (; k < parts; k += 16) s += p[(int64_t)k * W];
    }
    sums[i][c] = s;
    __syncthreads();
    if (i || e >= W) return;
    for (int j = 1; j < 16; ++j) s += sums[j][c];
    store_rt(dw, dw_dt, e, s);
}

// The gradient's workgroups leave W partial sums each and take rows in turn: one a CU for wide rows, two of 256 threads for short
// ones (9504 x 5120: 251 workgroups 78 us, 501 84, 732 94; 9504 x 1024: 251 27, 501 22).  Wide rows are written through the
// caches (78 us; nontemporally 95), short ones not (9504 x 1024: 24.5, 22.3).
RowCut grad_cut(int64_t T, int W) { return cut_rows(T, W, 8, 2, 1024, 8); }

template <typename T, typename H, int RUN, bool INT8, bool RES>
hipError_t launch_norm(const AddNormArgs& a, hipStream_t st) {
    const RowCut c = cut_rows(a.T, a.W, RUN, RUN == 4 ? 4 : 2, 1024, 0);
    if (!c.slots) {
        hipLaunchKernelGGL((add_norm_long_kernel<T, H, RUN, INT8>), dim3(c.grid), c.block(), 0, st, a);
        return hipGetLastError();
    }
    const bool once = whole(a.x, a.W, RUN, sizeof(T)) && whole(a.r, a.W, RUN, sizeof(H)) && whole(a.h, a.W, RUN, sizeof(H)) &&
                      whole(a.y, a.W, RUN, sizeof(T)) && whole({a.q, a.ldq}, a.W, RUN, 1);
    return by_parts(c, a.T, [&](dim3 grid, int64_t t0) {
        auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, c.block(), 0, st, a, t0, c.per, c.groups); };
        if (RUN == 8 && c.slots == 1) once ? go(add_norm_kernel<T, H, 8, 1, INT8, RES, true>) : go(add_norm_kernel<T, H, 8, 1, INT8, RES, false>);
        else if constexpr (RUN == 4) once ? go(add_norm_kernel<T, H, 4, 4, INT8, RES, true>) : go(add_norm_kernel<T, H, 4, 4, INT8, RES, false>);
        else once ? go(add_norm_kernel<T, H, 8, 2, INT8, RES, true>) : go(add_norm_kernel<T, H, 8, 2, INT8, RES, false>);
    });
}

template <typename T, typename H>
hipError_t norm_of(const AddNormArgs& a, hipStream_t st) {
    auto by_res = [&]<int RUN, bool INT8>() {
        return a.r.p ? launch_norm<T, H, RUN, INT8, true>(a, st) : launch_norm<T, H, RUN, INT8, false>(a, st);
    };
    if (!a.q) return by_res.template operator()<8, false>();
    return a.G ? by_res.template operator()<4, true>() : by_res.template operator()<8, true>();
}

template <typename T, typename H>
hipError_t grad_of(const AddNormGradArgs& a, hipStream_t st) {
    const RowCut c = grad_cut(a.T, a.W);
    const bool once = whole(a.dy, a.W, 8, sizeof(T)) && whole(a.h, a.W, 8, sizeof(H)) && whole(a.dh, a.W, 8, sizeof(H)) &&
                      whole(a.dx, a.W, 8, sizeof(H));
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, dim3(c.grid), c.block(), 0, st, a, c.per, c.groups); };
    auto by_slots = [&]<int SLOTS, int THREADS>() {
        if (a.dh.p) once ? go(add_norm_grad_kernel<T, H, SLOTS, true, true, THREADS>) : go(add_norm_grad_kernel<T, H, SLOTS, true, false, THREADS>);
        else once ? go(add_norm_grad_kernel<T, H, SLOTS, false, true, THREADS>) : go(add_norm_grad_kernel<T, H, SLOTS, false, false, THREADS>);
    };
    switch (c.slots) {
        case 1: by_slots.template operator()<1, 512>(); break;
        case 2: c.per <= 512 ? by_slots.template operator()<2, 512>() : by_slots.template operator()<2, 1024>(); break;
        default: hipLaunchKernelGGL((add_norm_grad_long_kernel<T, H>), dim3(c.grid), c.block(), 0, st, a); break;
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !a.dw) return e;
    hipLaunchKernelGGL(add_norm_dw_kernel, dim3((unsigned)((a.W + 15) / 16)), dim3(256), 0, st, a.part, (int)c.grid, a.W, a.dw, a.dw_dt);
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

size_t ws_add_norm_grad(int64_t T, int64_t W) {
    return T <= 0 || W <= 0 || W > MLP_MAX_WIDTH ? 0 : (size_t)grad_cut(T, (int)W).grid * (size_t)W * 4;
}

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
