// Rows held in a workgroup's registers: loads and stores of runs of values, the rotation, the codes of an 8-bit output.
#pragma once
#include "hadamard.h"
#include "mlp.h"

namespace qlin {

template <typename T, int N>
__device__ __forceinline__ void load_run(const T* p, int n, float* v) {
    if (n >= N) {  // rows of any alignment: global loads take any
        struct { T a[N]; } r;
        __builtin_memcpy(&r, p, sizeof r);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (float)r.a[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i < n ? (float)p[i] : 0.0f;
    }
}
template <int N>
__device__ __forceinline__ void load_run_rt(const void* p, int dt, int64_t e0, int n, float* v) {
    if (dt == DT_F32) load_run<float, N>((const float*)p + e0, n, v);
    else if (dt == DT_F16) load_run<f16, N>((const f16*)p + e0, n, v);
    else load_run<__bf16, N>((const __bf16*)p + e0, n, v);
}
template <typename T, int N>
__device__ __forceinline__ void store_run(T* p, int n, const float* v) {
    if (n >= N) {
        struct { T a[N]; } r;
#pragma unroll
        for (int i = 0; i < N; ++i) r.a[i] = (T)v[i];
        __builtin_memcpy(p, &r, sizeof r);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < n) p[i] = (T)v[i];
    }
}

// |v| as bits that order as the values do, a NaN above all.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// The codes rne(v * 127 / top) of a run, top the row's largest |v|, as bytes: v * inv added to 1.5 * 2^23 rounds once, to
// an integer in the low bits (|v * inv| <= 127 and an ulp).
template <int N>
__device__ __forceinline__ void store_codes(int8_t* p, int n, const float* v, float inv) {
    uint32_t b[N];
#pragma unroll
    for (int i = 0; i < N; ++i) b[i] = __float_as_uint(__builtin_fmaf(v[i], inv, 12582912.0f));
    struct { uint32_t w[N / 4]; } r;
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        const uint32_t lo = __builtin_amdgcn_perm(b[4 * i + 1], b[4 * i], 0x0C0C0400u);
        const uint32_t hi = __builtin_amdgcn_perm(b[4 * i + 3], b[4 * i + 2], 0x04000C0Cu);
        r.w[i] = lo | hi;
    }
    if (n >= N) {
        __builtin_memcpy(p, &r, sizeof r);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < n) p[i] = (int8_t)(r.w[i / 4] >> (8 * (i % 4)));
    }
}

// A row's code factor 127 / top and the power of two that its values are multiplied by first (so that the factor of
// a row of tiny values stays finite); 0 for a row of zeros.
__device__ __forceinline__ float code_factor(float top, float& first) {
    first = top < 0x1p-100f ? 0x1p100f : 1.0f;
    return top > 0.0f ? 127.0f / (top * first) : 0.0f;
}

// A run of 16 values through the rotation of its group, shared by a wave's lanes.
__device__ __forceinline__ void rotate_run(float* v, int G, int lane) {
    float n = 1.0f;
    auto by = [&]<int S>() {
        hadamard16<S>(v, lane);
        n = hadamard_norm<S>();
    };
    switch (G) {
        case 4: by.template operator()<4>(); break;
        case 8: by.template operator()<8>(); break;
        case 16: by.template operator()<16>(); break;
        case 32: by.template operator()<32>(); break;
        case 64: by.template operator()<64>(); break;
        case 128: by.template operator()<128>(); break;
        default: by.template operator()<256>(); break;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] *= n;
}

// Threads of a workgroup that holds a row, SLOTS runs of `run` values a thread; 0: longer than any.
inline int row_threads(int W, int run, int& slots) {
    const int runs = (W + run - 1) / run;
    for (int s : {1, 2, 4}) {
        const int n = ((runs + s - 1) / s + 63) / 64 * 64;
        if (n <= 1024) {
            slots = s;
            return n;
        }
    }
    slots = 0;
    return 1024;
}

}  // namespace qlin
