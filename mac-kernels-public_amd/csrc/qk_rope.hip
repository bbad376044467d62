// Rotation of q and k by positions on several axes, with the per-head norms in the same pass
// (y = rotate(w * x * rsqrt(mean(x^2) + eps))), into tensors or straight into a paged cache, and
// its gradient.  One wave a (token, head) row: every value is read once and written once.
#include "attention.h"

namespace qlin {
namespace {

template <int DT> struct HeadType;
template <> struct HeadType<DT_F32> { using T = float; };
template <> struct HeadType<DT_F16> { using T = f16; };
template <> struct HeadType<DT_BF16> { using T = bf16_t; };

// Values of row dimension a lane holds as pairs: lane l has pairs l, l + 64, ... of ROPE_MAX_DIM / 2.
constexpr int PAIRS = ROPE_MAX_DIM / 128;

__device__ __forceinline__ double position_at(const RopeTurn& r, int pair, int64_t t) {
    const int ax = r.axis ? min(max(r.axis[pair], 0), r.axes - 1) : 0;
    const int64_t i = ax * r.pos_sa + t * r.pos_st;
    if (r.pos_dt == DT_I32) return (double)((const int32_t*)r.pos)[i];
    if (r.pos_dt == DT_I64) return (double)((const int64_t*)r.pos)[i];
    return (double)((const float*)r.pos)[i];
}

// cos and sin of position * frequency: the product and its reduction to a turn in 64 bits, so that
// a position of a million loses nothing; then one fp32 evaluation on [-1/2, 1/2] turns.
__device__ __forceinline__ void turn_at(const RopeTurn& r, int pair, int64_t t, float& c, float& s) {
    double rev = position_at(r, pair, t) * (double)r.inv_freq[pair] * 0.15915494309189533577;
    rev -= rint(rev);
    sincospif(2.0f * (float)rev, &s, &c);
    if (r.inverse) s = -s;
}

// The two dimensions of pseudo-pair i: the P rotated pairs, then the values that pass through, two by
// two; -1 where there is none.
__device__ __forceinline__ void dims_of(const RopeTurn& r, int D, int i, int& a, int& b) {
    if (i < r.P) {
        a = r.interleaved ? 2 * i : i;
        b = r.interleaved ? 2 * i + 1 : i + r.P;
    } else {
        a = 2 * i < D ? 2 * i : -1;
        b = 2 * i + 1 < D ? 2 * i + 1 : -1;
    }
}

template <int DT>
__global__ __launch_bounds__(256) void head_rope_kernel(HeadRopeArgs a) {
    using T = typename HeadType<DT>::T;
    const int lane = threadIdx.x & 63;
    const int heads = a.Hq + a.Hk + (a.store ? a.Hk : 0);
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= a.T * heads) return;
    const int64_t t = row / heads;
    int h = (int)(row % heads);
    const int kind = h < a.Hq ? 0 : h < a.Hq + a.Hk ? 1 : 2;
    h -= kind == 0 ? 0 : kind == 1 ? a.Hq : a.Hq + a.Hk;
    const HeadView& in = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
    const T* x = (const T*)in.p + t * in.st + h * in.sh;
    T* y;
    if (kind == 0) {
        y = (T*)a.qo.p + t * a.qo.st + h * a.qo.sh;
    } else if (!a.store) {
        y = (T*)a.ko.p + t * a.ko.st + h * a.ko.sh;
    } else {
        const int64_t slot = a.slots_dt == DT_I64 ? ((const int64_t*)a.slots)[t * a.slots_st] : ((const int32_t*)a.slots)[t * a.slots_st];
        if (slot < 0 || slot >= a.blocks * a.page) return;
        const CacheView& c = kind == 1 ? a.kc : a.vc;
        y = (T*)c.p + (slot / a.page) * c.sb + (slot % a.page) * c.sp + h * c.sh;
    }
    float u[PAIRS], v[PAIRS], sum = 0.0f;
#pragma unroll
    for (int j = 0; j < PAIRS; ++j) {
        int da, db;
        dims_of(a.turn, a.D, lane + 64 * j, da, db);
        u[j] = da >= 0 ? load_f(x + da) : 0.0f;
        v[j] = db >= 0 ? load_f(x + db) : 0.0f;
        sum += u[j] * u[j] + v[j] * v[j];
    }
    float rstd = 1.0f;
    if (a.norm) rstd = 1.0f / sqrtf(wave_sum(sum) / (float)a.D + a.eps);
    const void* w = kind == 0 ? a.wq : a.wk;
    const int wdt = kind == 0 ? a.wq_dt : a.wk_dt;
#pragma unroll
    for (int j = 0; j < PAIRS; ++j) {
        const int i = lane + 64 * j;
        int da, db;
        dims_of(a.turn, a.D, i, da, db);
        if (kind < 2) {
            if (a.norm) {
                u[j] *= rstd;
                v[j] *= rstd;
                if (w && da >= 0) u[j] *= load_rt(w, wdt, da);
                if (w && db >= 0) v[j] *= load_rt(w, wdt, db);
            }
            if (i < a.turn.P) {
                float c, s;
                turn_at(a.turn, i, t, c, s);
                const float p = u[j] * c - v[j] * s;
                v[j] = u[j] * s + v[j] * c;
                u[j] = p;
            }
        }
        if (da >= 0) store_out(y + da, u[j]);
        if (db >= 0) store_out(y + db, v[j]);
    }
}

// One wave a workgroup; wave w takes rows w, w + grid, ... and keeps its sums of g x^ for q's and k's weights.
template <int DT>
__global__ __launch_bounds__(64) void head_grad_kernel(HeadGradArgs a) {
    using T = typename HeadType<DT>::T;
    const int lane = threadIdx.x;
    const int heads = a.Hq + a.Hk;
    const int64_t rows = a.T * heads;
    float du[2][PAIRS] = {}, dv[2][PAIRS] = {};
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const int64_t t = row / heads;
        int h = (int)(row % heads);
        const int kind = h < a.Hq ? 0 : 1;
        h -= kind ? a.Hq : 0;
        const HeadView &in = kind ? a.k : a.q, &gin = kind ? a.gk : a.gq, &dx = kind ? a.dk : a.dq;
        const T* x = (const T*)in.p + t * in.st + h * in.sh;
        const T* gy = (const T*)gin.p + t * gin.st + h * gin.sh;
        T* y = (T*)dx.p + t * dx.st + h * dx.sh;
        const void* w = kind ? a.wk : a.wq;
        const int wdt = kind ? a.wk_dt : a.wq_dt;
        float u[PAIRS], v[PAIRS], gu[PAIRS], gv[PAIRS], sum = 0.0f;
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) {
            const int i = lane + 64 * j;
            int da, db;
            dims_of(a.turn, a.D, i, da, db);
            u[j] = da >= 0 ? load_f(x + da) : 0.0f;
            v[j] = db >= 0 ? load_f(x + db) : 0.0f;
            gu[j] = da >= 0 ? load_f(gy + da) : 0.0f;
            gv[j] = db >= 0 ? load_f(gy + db) : 0.0f;
            sum += u[j] * u[j] + v[j] * v[j];
            if (i < a.turn.P) {
                float c, s;
                turn_at(a.turn, i, t, c, s);
                const float p = gu[j] * c + gv[j] * s;
                gv[j] = gv[j] * c - gu[j] * s;
                gu[j] = p;
            }
        }
        const float rstd = 1.0f / sqrtf(wave_sum(sum) / (float)a.D + a.eps);
        float dot = 0.0f;
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) {
            int da, db;
            dims_of(a.turn, a.D, lane + 64 * j, da, db);
            u[j] *= rstd;
            v[j] *= rstd;
            du[0][j] += kind == 0 ? gu[j] * u[j] : 0.0f;
            dv[0][j] += kind == 0 ? gv[j] * v[j] : 0.0f;
            du[1][j] += kind == 1 ? gu[j] * u[j] : 0.0f;
            dv[1][j] += kind == 1 ? gv[j] * v[j] : 0.0f;
            if (w && da >= 0) gu[j] *= load_rt(w, wdt, da);
            if (w && db >= 0) gv[j] *= load_rt(w, wdt, db);
            dot += gu[j] * u[j] + gv[j] * v[j];
        }
        dot = wave_sum(dot) / (float)a.D;
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) {
            int da, db;
            dims_of(a.turn, a.D, lane + 64 * j, da, db);
            if (da >= 0) store_out(y + da, rstd * (gu[j] - u[j] * dot));
            if (db >= 0) store_out(y + db, rstd * (gv[j] - v[j] * dot));
        }
    }
    if (!a.part) return;
#pragma unroll
    for (int kind = 0; kind < 2; ++kind)
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) {
            int da, db;
            dims_of(a.turn, a.D, lane + 64 * j, da, db);
            float* p = a.part + ((int64_t)blockIdx.x * 2 + kind) * a.D;
            if (da >= 0) p[da] = du[kind][j];
            if (db >= 0) p[db] = dv[kind][j];
        }
}

// Weight gradients from the partials: one workgroup a value of q's or k's weight.
__global__ __launch_bounds__(256) void head_grad_sum_kernel(HeadGradArgs a, int parts) {
    __shared__ float s[256];
    const int kind = blockIdx.x / a.D, d = blockIdx.x % a.D;
    float sum = 0.0f;
    for (int i = threadIdx.x; i < parts; i += 256) sum += a.part[((int64_t)i * 2 + kind) * a.D + d];
    s[threadIdx.x] = sum;
    __syncthreads();
    for (int n = 128; n; n >>= 1) {
        if (threadIdx.x < n) s[threadIdx.x] += s[threadIdx.x + n];
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        if (kind == 0 && a.dwq) store_rt(a.dwq, a.dwq_dt, d, s[0]);
        if (kind == 1 && a.dwk) store_rt(a.dwk, a.dwk_dt, d, s[0]);
    }
}

}  // namespace

hipError_t run_head_rope(const HeadRopeArgs& a, hipStream_t st) {
    const int64_t rows = a.T * (a.Hq + a.Hk + (a.store ? a.Hk : 0));
    const dim3 grid((unsigned)((rows + 3) / 4));
    if (a.dtype == DT_F32) hipLaunchKernelGGL(head_rope_kernel<DT_F32>, grid, dim3(256), 0, st, a);
    else if (a.dtype == DT_F16) hipLaunchKernelGGL(head_rope_kernel<DT_F16>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(head_rope_kernel<DT_BF16>, grid, dim3(256), 0, st, a);
    return hipGetLastError();
}

int head_grad_parts(int64_t T, int64_t heads) { return (int)std::min<int64_t>(std::max<int64_t>(T * heads, 1), 4096); }

size_t ws_head_grad(int64_t T, int64_t heads, int64_t D) { return (size_t)head_grad_parts(T, heads) * 2 * D * 4; }

hipError_t run_head_grad(const HeadGradArgs& a, hipStream_t st) {
    const int parts = head_grad_parts(a.T, a.Hq + a.Hk);
    if (a.dtype == DT_F32) hipLaunchKernelGGL(head_grad_kernel<DT_F32>, dim3(parts), dim3(64), 0, st, a);
    else if (a.dtype == DT_F16) hipLaunchKernelGGL(head_grad_kernel<DT_F16>, dim3(parts), dim3(64), 0, st, a);
    else hipLaunchKernelGGL(head_grad_kernel<DT_BF16>, dim3(parts), dim3(64), 0, st, a);
    if (hipError_t e = hipGetLastError()) return e;
    if (a.dwq || a.dwk) {
        hipLaunchKernelGGL(head_grad_sum_kernel, dim3(2 * a.D), dim3(256), 0, st, a, parts);
        return hipGetLastError();
    }
    return hipSuccess;
}

}  // namespace qlin
