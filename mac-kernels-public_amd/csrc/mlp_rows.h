// Rows held in a workgroup's registers: loads and stores of runs of values, the rotation, the codes of an 8-bit output.
#pragma once
#include <algorithm>

#include "hadamard.h"
#include "mlp.h"

namespace qlin {

// N values as they are in memory, rows of any alignment (global loads take any); zeros past the n-th.  ONCE: read
// nontemporally, 16-byte aligned.
template <typename T, int N>
struct Run {
    T v[N];
};
template <bool ONCE, typename T, int N>
__device__ __forceinline__ Run<T, N> load_raw(const T* p, int n) {
    Run<T, N> r;
    if (n >= N) {
        if constexpr (ONCE) {
            constexpr int W = sizeof r / 16;
            struct { u32x4 w[W]; } q;
#pragma unroll
            for (int i = 0; i < W; ++i) q.w[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p) + i);
            r = __builtin_bit_cast(Run<T, N>, q);
        } else {
            __builtin_memcpy(&r, p, sizeof r);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) r.v[i] = i < n ? p[i] : (T)0.0f;
    }
    return r;
}
template <typename T, int N>
__device__ __forceinline__ void load_run(const T* p, int n, float* v) {
    const Run<T, N> r = load_raw<false, T, N>(p, n);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)r.v[i];
}
template <int N>
__device__ __forceinline__ void load_run_rt(const void* p, int dt, int64_t e0, int n, float* v) {
    if (dt == DT_F32) load_run<float, N>((const float*)p + e0, n, v);
    else if (dt == DT_F16) load_run<f16, N>((const f16*)p + e0, n, v);
    else load_run<__bf16, N>((const __bf16*)p + e0, n, v);
}
template <bool ONCE, typename T, int N>
__device__ __forceinline__ void store_raw(T* p, int n, const Run<T, N>& r) {
    if (n >= N) {
        if constexpr (ONCE) {
            constexpr int W = sizeof r / 16;
            struct Words { u32x4 w[W]; };
            const Words q = __builtin_bit_cast(Words, r);
#pragma unroll
            for (int i = 0; i < W; ++i) __builtin_nontemporal_store(q.w[i], reinterpret_cast<u32x4*>(p) + i);
        } else {
            __builtin_memcpy(p, &r, sizeof r);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < n) p[i] = r.v[i];
    }
}
template <bool ONCE, typename T, int N>
__device__ __forceinline__ void store_run(T* p, int n, const float* v) {
    Run<T, N> r;
#pragma unroll
    for (int i = 0; i < N; ++i) r.v[i] = (T)v[i];
    store_raw<ONCE, T, N>(p, n, r);
}

// |v| as bits that order as the values do, a NaN above all.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// The codes rne(v * 127 / top) of a run, top the row's largest |v|, as bytes: v * inv added to 1.5 * 2^23 rounds once, to
// an integer in the low bits (|v * inv| <= 127 and an ulp).
template <bool ONCE, int N>
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
        if constexpr (ONCE) {
            typedef uint32_t Words __attribute__((ext_vector_type(N / 4)));
            __builtin_nontemporal_store(__builtin_bit_cast(Words, r), reinterpret_cast<Words*>(p));
        } else {
            __builtin_memcpy(p, &r, sizeof r);
        }
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

// A run of 16 values through the rotation of its group of G, shared by a wave's lanes.  (Stage after stage, each under a condition of
// its own, the exchanges' latencies do not overlap: 9504 x 5120 to 8 bits 112 us against 74.)
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

// A row's threads: the waves of a group of the workgroup.  All of a workgroup's threads call sums() the same number of times; `turn`
// alternates, so that one barrier a call separates a buffer's writes from its next ones.
struct Group {
    int at, waves, wave, lane;  // the thread's place in the row; the group's waves, this one among the workgroup's
    __device__ __forceinline__ explicit Group(int per) {
        lane = threadIdx.x & 63;
        wave = threadIdx.x >> 6;
        waves = per >> 6;
        at = (int)threadIdx.x - wave / waves * per;
    }
    // a and b of all of the group's threads by the functions' rules
    template <typename B, typename F>
    __device__ __forceinline__ void sums(float& a, B& b, int turn, F&& join) const {
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            a += __shfl_xor(a, m, 64);
            b = join(b, __shfl_xor(b, m, 64));
        }
        if (waves == 1) return;
        __shared__ float as[2][16];
        __shared__ B bs[2][16];
        if (lane == 0) {
            as[turn][wave] = a;
            bs[turn][wave] = b;
        }
        lds_barrier();
        const int first = wave / waves * waves;
        a = as[turn][first];
        b = bs[turn][first];
        for (int i = 1; i < waves; ++i) {
            a += as[turn][first + i];
            b = join(b, bs[turn][first + i]);
        }
    }
};

// Whether 16-byte pieces of the rows are aligned.
inline bool aligned(const RowView& v, int es) { return !v.p || ((uintptr_t)v.p % 16 == 0 && v.ld * es % 16 == 0); }

// Calls that read more than this read and write nontemporally: what they touch is not in the caches when it is needed again (4608
// x 6144 norm to bf16, reads and writes: 56 us neither so, 49 the reads, 40 both).
constexpr int64_t ONCE_BYTES = 32 << 20;

// How rows are dealt: `per` threads hold a row, `slots` runs each; `groups` rows a workgroup; `grid` workgroups, each of which takes
// every grid-th of the row groups (by_parts: one each).  slots 0: rows longer than any.
struct RowCut {
    int per = 64, groups = 1, slots = 1;
    unsigned grid = 1;
    dim3 block() const { return dim3((unsigned)(per * groups)); }
};
// Rows of 8-value runs: up to 512 threads with one slot, 1024 with two; rotated ones, of 16-value runs: up to 1024 with one (more
// spill).  waves: that a CU is to hold, where workgroups take rows in turn.
inline RowCut cut_rows(int64_t T, int W, int run, int waves) {
    RowCut c;
    const int64_t runs = (W + run - 1) / run;
    c.slots = 0;
    c.per = 512;
    for (int s : {1, 2}) {
        const int64_t n = ((runs + s - 1) / s + 63) / 64 * 64;
        if (n > (s * run == 8 ? 512 : 1024) || s * run > 16) continue;
        c.slots = s;
        c.per = (int)n;
        break;
    }
    c.groups = c.slots && c.per < 256 ? 256 / c.per : 1;
    const int64_t blocks = (T + c.groups - 1) / c.groups, most = 256 * (int64_t)std::max(1, waves * 64 / (c.per * c.groups));
    const int64_t rounds = (blocks + most - 1) / most;
    c.grid = (unsigned)((blocks + rounds - 1) / rounds);
    return c;
}

// f(grid, first row): a row group a workgroup, in launches of fewer than 2^31 threads.
template <typename F>
hipError_t by_parts(const RowCut& c, int64_t T, F&& f) {
    const int64_t most = 0x7FFFFFFF / (c.per * c.groups);
    for (int64_t t0 = 0; t0 < T; t0 += most * c.groups) {
        f(dim3((unsigned)std::min<int64_t>(most, (T - t0 + c.groups - 1) / c.groups)), t0);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace qlin
