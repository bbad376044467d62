// Gated activation: y = f(gate) up (up absent: f(gate)), f(z) = z sigma(t) with t = z (SiLU) or t = 2 sqrt(2/pi) (z + 0.044715
// z^3) (GELU in its tanh form), y in 16 or 32 bits or in 8 with a scale a row, and its gradient.  Bound by memory:
// every value is read once and written once.
//
// 8 bits: a row stays in registers until its largest |value| is known; the codes are rne(127 v / top), v rotated first for
// weights that are stored so, the scale is top / 127.
#include <algorithm>

#include "mlp_rows.h"

namespace qlin {
namespace {

constexpr float GELU_C = 1.5957691216057308f, GELU_A = 0.044715f;  // 2 sqrt(2/pi)

// sigma(t), and e^-t with 32 bits' precision for outputs of 32 bits, else by the exponential instruction: its argument's
// rounding leaves 2^-24 |t| of e^-t, at most 2^-18 where sigma is not yet below the smallest 16-bit fraction.
template <typename T>
__device__ __forceinline__ float sigma(float t) {
    if constexpr (sizeof(T) == 4) return 1.0f / (1.0f + expf(-t));
    else return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * t));
}

// s = sigma(t(z)) and dt = t'(z); f = z s, f' = s + z s (1 - s) dt.
template <typename T, int ACT>
__device__ __forceinline__ void gate_of(float z, float& s, float& dt) {
    if constexpr (ACT == QLIN_ACT_SILU) {
        s = sigma<T>(z);
        dt = 1.0f;
    } else {
        const float z2 = z * z;
        s = sigma<T>(GELU_C * z * __builtin_fmaf(GELU_A, z2, 1.0f));
        dt = GELU_C * __builtin_fmaf(3.0f * GELU_A, z2, 1.0f);
    }
}
// y = f(gate) up, 8 values a thread.
template <typename T, int ACT, bool GATED>
__global__ __launch_bounds__(256) void gated_act_kernel(GatedActArgs a, int64_t t0, uint32_t units, uint32_t per) {
    const uint32_t u = blockIdx.x * 256u + threadIdx.x;
    if (u >= units) return;
    const uint32_t row = u / per;
    const int e0 = (int)(u - row * per) * 8, n = a.W - e0;
    const int64_t t = t0 + row;
    float z[8], v[8];
    load_run<T, 8>((const T*)a.gate.p + t * a.gate.ld + e0, n, z);
    if constexpr (GATED) load_run<T, 8>((const T*)a.up.p + t * a.up.ld + e0, n, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float s, dt;
        gate_of<T, ACT>(z[i], s, dt);
        const float f = z[i] * s;
        v[i] = GATED ? f * v[i] : f;
    }
    store_run<T, 8>((T*)a.y.p + t * a.y.ld + e0, n, v);
}

template <typename T, int ACT, bool GATED>
__global__ __launch_bounds__(256) void gated_act_grad_kernel(GatedActArgs a, int64_t t0, uint32_t units, uint32_t per) {
    const uint32_t u = blockIdx.x * 256u + threadIdx.x;
    if (u >= units) return;
    const uint32_t row = u / per;
    const int e0 = (int)(u - row * per) * 8, n = a.W - e0;
    const int64_t t = t0 + row;
    float z[8], v[8], g[8];
    load_run<T, 8>((const T*)a.gate.p + t * a.gate.ld + e0, n, z);
    if constexpr (GATED) load_run<T, 8>((const T*)a.up.p + t * a.up.ld + e0, n, v);
    load_run<T, 8>((const T*)a.dy.p + t * a.dy.ld + e0, n, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float s, dt;
        gate_of<T, ACT>(z[i], s, dt);
        const float f = z[i] * s, p = s * (1.0f - s);
        const float df = p == 0.0f ? s : s + z[i] * p * dt;  // far from 0, where z dt may be infinite, sigma
        const float up = GATED ? v[i] : 1.0f;
        v[i] = g[i] * f;
        z[i] = g[i] * up * df;
    }
    store_run<T, 8>((T*)a.dgate.p + t * a.dgate.ld + e0, n, z);
    if constexpr (GATED) store_run<T, 8>((T*)a.dup.p + t * a.dup.ld + e0, n, v);
}

__device__ __forceinline__ uint32_t row_max(uint32_t b) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) b = max(b, (uint32_t)__shfl_xor((int)b, m, 64));
    __shared__ uint32_t tops[16];
    if (lane == 0) tops[wave] = b;
    __syncthreads();
    for (int i = 0; i < waves; ++i) b = max(b, tops[i]);
    return b;
}

// A row a workgroup, SLOTS runs of RUN values a thread (RUN 16: rotated); SLOTS 0: rows of any length, read twice.
template <typename T, int ACT, bool GATED, int RUN, int SLOTS>
__global__ __launch_bounds__(1024) void gated_act_int8_kernel(GatedActArgs a, int64_t t0) {
    const int per = blockDim.x, at = threadIdx.x, lane = threadIdx.x & 63;
    const int64_t t = t0 + blockIdx.x;
    const T* gate = (const T*)a.gate.p + t * a.gate.ld;
    const T* up = GATED ? (const T*)a.up.p + t * a.up.ld : nullptr;
    auto value = [&](int e0, float* v) {
        const int n = a.W - e0;
        float z[RUN];
        load_run<T, RUN>(gate + e0, n, z);
        if constexpr (GATED) load_run<T, RUN>(up + e0, n, v);
#pragma unroll
        for (int i = 0; i < RUN; ++i) {
            float s, dt;
            gate_of<T, ACT>(z[i], s, dt);
            const float f = z[i] * s;
            v[i] = GATED ? f * v[i] : f;
        }
        if constexpr (RUN == 16) rotate_run(v, a.G, lane);
    };
    uint32_t top = 0;
    float inv, first;
    auto finish = [&] {
        top = row_max(top);
        inv = code_factor(__uint_as_float(top), first);
        if (at == 0) a.scale[t] = __uint_as_float(top) / 127.0f;
    };
    auto emit = [&](int e0, float* v) {
        if (first != 1.0f)
#pragma unroll
            for (int i = 0; i < RUN; ++i) v[i] *= first;
        if (e0 < a.W) store_codes<RUN>(a.q + t * a.ldq + e0, a.W - e0, v, inv);
    };
    auto largest = [&](const float* v) {
#pragma unroll
        for (int i = 0; i < RUN; ++i) top = max(top, abs_bits(v[i]));
    };
    if constexpr (SLOTS > 0) {
        float v[SLOTS][RUN];
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            value((s * per + at) * RUN, v[s]);
            largest(v[s]);
        }
        finish();
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) emit((s * per + at) * RUN, v[s]);
    } else {
        float v[RUN];
        for (int c = 0; c < a.W; c += per * RUN) {
            value(c + at * RUN, v);
            largest(v);
        }
        finish();
        for (int c = 0; c < a.W; c += per * RUN) {
            value(c + at * RUN, v);
            emit(c + at * RUN, v);
        }
    }
}

template <typename F>
hipError_t by_kind(const GatedActArgs& a, F&& f) {
    auto gates = [&]<typename T, int ACT>() {
        return a.up.p ? f.template operator()<T, ACT, true>() : f.template operator()<T, ACT, false>();
    };
    auto acts = [&]<typename T>() {
        return a.act == QLIN_ACT_SILU ? gates.template operator()<T, QLIN_ACT_SILU>() : gates.template operator()<T, QLIN_ACT_GELU_TANH>();
    };
    if (a.dtype == DT_F32) return acts.template operator()<float>();
    return a.dtype == DT_F16 ? acts.template operator()<f16>() : acts.template operator()<__bf16>();
}

// f(first row, units, units a row) over parts of fewer than 2^31 units of 8 values.
template <typename F>
hipError_t by_units(const GatedActArgs& a, F&& f) {
    const int64_t per = (a.W + 7) / 8, most = 0x7FFFFF00 / per;
    for (int64_t t0 = 0; t0 < a.T; t0 += most) {
        const uint32_t units = (uint32_t)(std::min<int64_t>(most, a.T - t0) * per);
        f(dim3((units + 255) / 256), t0, units, (uint32_t)per);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

template <typename T, int ACT, bool GATED, int RUN>
hipError_t launch_int8(const GatedActArgs& a, hipStream_t st) {
    int slots = 0;
    const int n = row_threads(a.W, RUN, slots);
    const int64_t most = (int64_t)(0x7FFFFFFF / n);
    for (int64_t t0 = 0; t0 < a.T; t0 += most) {
        const dim3 grid((unsigned)std::min<int64_t>(most, a.T - t0)), block((unsigned)n);
        switch (slots) {
            case 1: hipLaunchKernelGGL((gated_act_int8_kernel<T, ACT, GATED, RUN, 1>), grid, block, 0, st, a, t0); break;
            case 2: hipLaunchKernelGGL((gated_act_int8_kernel<T, ACT, GATED, RUN, 2>), grid, block, 0, st, a, t0); break;
            default: hipLaunchKernelGGL((gated_act_int8_kernel<T, ACT, GATED, RUN, 0>), grid, block, 0, st, a, t0); break;
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace

hipError_t run_gated_act(const GatedActArgs& a, hipStream_t st) {
    if (a.T == 0 || a.W == 0) return hipSuccess;
    return by_kind(a, [&]<typename T, int ACT, bool GATED>() {
        if (a.q) return a.G ? launch_int8<T, ACT, GATED, 16>(a, st) : launch_int8<T, ACT, GATED, 8>(a, st);
        return by_units(a, [&](dim3 grid, int64_t t0, uint32_t units, uint32_t per) {
            hipLaunchKernelGGL((gated_act_kernel<T, ACT, GATED>), grid, dim3(256), 0, st, a, t0, units, per);
        });
    });
}

hipError_t run_gated_act_grad(const GatedActArgs& a, hipStream_t st) {
    if (a.T == 0 || a.W == 0) return hipSuccess;
    return by_kind(a, [&]<typename T, int ACT, bool GATED>() {
        return by_units(a, [&](dim3 grid, int64_t t0, uint32_t units, uint32_t per) {
            hipLaunchKernelGGL((gated_act_grad_kernel<T, ACT, GATED>), grid, dim3(256), 0, st, a, t0, units, per);
        });
    });
}

}  // namespace qlin
