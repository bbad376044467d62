// Rows held in a workgroup's registers: loads and stores of runs of values, the rotation, the codes of an 8-bit output.
#pragma once
#include <algorithm>

#include "mlp.h"

namespace qlin {

// N values as they are in memory.
template <typename T, int N>
struct Run {
    T v[N];
};
// Values e0 .. e0 + N - 1 of a row of W >= N, at any alignment (global loads take any), without a branch, so that a thread's loads
// are in flight together: a run that reaches past the row's end gets its last N values, which trimmed() puts right once
// all loads have been issued.  ONCE: nontemporal, whole 16-byte (8-byte: RUN 4 of 16 bits) pieces: what is read and written once
// takes no place in the caches (norm 4608 x 6144 to bf16, one row a workgroup: 49 us, 40 with both).
template <bool ONCE, typename T, int N>
__device__ __forceinline__ Run<T, N> load_piece(const T* row, int e0, int W) {
    const T* p = row + min(e0, W - N);
    Run<T, N> r;
    if constexpr (ONCE) {
        typedef uint32_t Words __attribute__((ext_vector_type(sizeof r % 16 ? 2 : 4)));
        struct { Words w[sizeof r / sizeof(Words)]; } q;
#pragma unroll
        for (int i = 0; i < (int)(sizeof r / sizeof(Words)); ++i) q.w[i] = __builtin_nontemporal_load(reinterpret_cast<const Words*>(p) + i);
        r = __builtin_bit_cast(Run<T, N>, q);
    } else {
        __builtin_memcpy(&r, p, sizeof r);
    }
    return r;
}
// A piece's values in fp32, zeros past the row's end.  WHOLE: a piece is all in its row, or all behind it and then a copy of the row's
// last values, which the callers leave out of their sums.
template <bool WHOLE, typename T, int N>
__device__ __forceinline__ void trimmed(const Run<T, N>& r, int e0, int W, float* v) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)r.v[i];
    if (!WHOLE && e0 + N > W) {
        const int d = e0 - (W - N);  // value i is the piece's i + d
#pragma unroll
        for (int step = 1; step < N; step *= 2)
            if (d & step)
#pragma unroll
                for (int i = 0; i < N; ++i) v[i] = i + step < N ? v[i + step] : 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i + d < N ? v[i] : 0.0f;
    }
}
// The same of a vector of float32, float16 or bfloat16, S pieces `apart` values from one another.
template <bool WHOLE, int N, int S>
__device__ __forceinline__ void load_pieces_rt(const void* p, int dt, int e0, int apart, int W, float (&v)[S][N]) {
    auto of = [&]<typename T>() {
        Run<T, N> r[S];
#pragma unroll
        for (int s = 0; s < S; ++s) r[s] = load_piece<false, T, N>((const T*)p, e0 + s * apart, W);
#pragma unroll
        for (int s = 0; s < S; ++s) trimmed<WHOLE, T, N>(r[s], e0 + s * apart, W, v[s]);
    };
    if (dt == DT_F32) of.template operator()<float>();
    else if (dt == DT_F16) of.template operator()<f16>();
    else of.template operator()<__bf16>();
}

// Rows of any length, short ones too.
template <typename T, int N>
__device__ __forceinline__ void load_run(const T* p, int n, float* v) {
    if (n >= N) {
        Run<T, N> r;
        __builtin_memcpy(&r, p, sizeof r);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (float)r.v[i];
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
template <bool ONCE, typename T, int N>
__device__ __forceinline__ void store_raw(T* p, int n, const Run<T, N>& r) {
    if (n >= N) {
        if constexpr (ONCE) {
            typedef uint32_t Words __attribute__((ext_vector_type(sizeof r % 16 ? 2 : 4)));
            struct Pieces { Words w[sizeof r / sizeof(Words)]; };
            const Pieces q = __builtin_bit_cast(Pieces, r);
#pragma unroll
            for (int i = 0; i < (int)(sizeof r / sizeof(Words)); ++i) __builtin_nontemporal_store(q.w[i], reinterpret_cast<Words*>(p) + i);
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
    for (int i = 0; i < N; ++i) {
        float x = v[i];
        // fp16: a product and its rounding to 16 bits may become one instruction of another result, in some variants and not in others
        if constexpr (__is_same(T, f16)) asm("" : "+v"(x));
        r.v[i] = (T)x;
    }
    store_raw<ONCE, T, N>(p, n, r);
}

// The larger magnitude, NaN if there is one.
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(__builtin_fabsf(a), __builtin_fabsf(b)); }
template <int N>
__device__ __forceinline__ float largest(const float* v) {
    float m = __builtin_fabsf(v[0]);
#pragma unroll
    for (int i = 1; i < N; ++i) m = larger(m, v[i]);
    return m;
}

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
            if constexpr (N == 4) {
                __builtin_nontemporal_store(r.w[0], reinterpret_cast<uint32_t*>(p));
            } else {
                typedef uint32_t Words __attribute__((ext_vector_type(N / 4)));
                __builtin_nontemporal_store(__builtin_bit_cast(Words, r), reinterpret_cast<Words*>(p));
            }
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

// The rotation of 256 values on the matrix cores.  As a 16 x 16 matrix V[a][b] of values 16 a + b they become M_a V M_b with M_b the
// Hadamard matrix of the group's lowest (at most) two base-4 digits and M_a that of the higher ones, block diagonal where the
// group is smaller than 256 values: entries 0, 1 and -1 (M_b's times a power of two), exact in bf16.  Lane l holds values 16 (l % 16) + 4 (l / 16) .. + 3,
// which are its part of V as the first operand; the product's registers, taken as a first operand again, are its transpose, and the
// second product comes out in the layout of the values.
//
// The factor 1 / sqrt(G) is in the first product's entries, as the power of two at or below it; what is left, 1 or sqrt(2), is the
// scale's.  So no sum passes fp32's range where the rotated values stay below 2^126: among the values that take part in a first sum
// one is at least as large, and the partial sums of 16 terms are at most 4 times the largest of the 16 sums.  (The factor behind the
// sums gave finite rows infinite scales from 2^124 on.)
//
// A value enters a product as three bf16 parts that together are the value (8 bits of its 24 each), so that the rotation is as exact as
// fp32's sums.  Two rounded parts, off by 2^-18, would change one code in 10^4 (9504 x 13824 in fp16, with the gate: two
// parts 140 us, three 154; the matrix cores' fp32 products, of a 16th of the rate, 207; fp32 across the lanes 157).
typedef short bf16x4_bits __attribute__((ext_vector_type(4)));
struct RotationTable {
    // lane l's entries [4 (l / 16) + i][l % 16]: M_b by log2 G, its entries 2^-ceil(log2 G / 2), and M_a by log2 of its size
    uint64_t low[9][64], high[5][64];
    static constexpr int entry(int size, int r, int c) {
        if (r / size != c / size) return 0;
        r %= size;
        c %= size;
        int s = 1;
        for (; size >= 4; size /= 4, r /= 4, c /= 4) s = r % 4 + c % 4 == 3 ? -s : s;
        return size == 2 && r && c ? -s : s;
    }
    static constexpr uint64_t lane(int size, int halvings, int l) {
        uint64_t m = 0;
        for (int i = 0; i < 4; ++i) {
            const int e = entry(size, 4 * (l / 16) + i, l % 16), one = 0x3F80 - 0x80 * halvings;
            m |= (uint64_t)(e == 0 ? 0 : e == 1 ? one : one | 0x8000) << (16 * i);
        }
        return m;
    }
    constexpr RotationTable() : low(), high() {
        for (int l = 0; l < 64; ++l) {
            for (int k = 0; k < 9; ++k) low[k][l] = lane(1 << (k < 4 ? k : 4), (k + 1) / 2, l);
            for (int k = 0; k < 5; ++k) high[k][l] = lane(1 << k, 0, l);
        }
    }
};
__device__ const RotationTable rotation_table;

struct Rotation {
    bf16x4_bits low, high;  // M_b, M_a
    float left;             // what the rotated values lack
    __device__ __forceinline__ Rotation(int G, int lane) {
        const int k = 31 - __clz(G);
        low = __builtin_bit_cast(bf16x4_bits, rotation_table.low[k][lane]);
        high = __builtin_bit_cast(bf16x4_bits, rotation_table.high[max(k - 4, 0)][lane]);
        left = k % 2 ? 1.41421356237309505f : 1.0f;
    }
    static __device__ __forceinline__ f32x4 product(const f32x4 v, const bf16x4_bits m) {
        // the parts of two values side by side, as the product takes them: the upper halves of their words, those of what is left
        u32x2 part[3];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float a = v[2 * i], b = v[2 * i + 1];
#pragma unroll
            for (int p = 0; p < 3; ++p) {
                part[p][i] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
                a -= __uint_as_float(part[p][i] << 16);
                b -= __uint_as_float(part[p][i] & 0xFFFF0000u);
            }
        }
        f32x4 d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int p = 2; p >= 0; --p) d = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(bf16x4_bits, part[p]), m, d, 0, 0, 0);
        return d;
    }
    __device__ __forceinline__ void operator()(float* v) const {
        const f32x4 d = product(product(f32x4{v[0], v[1], v[2], v[3]}, low), high);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = d[i];
    }
};

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
    // Where the thread's first run of RUN values is: one thread's behind the other's, or (RUN 4) as Rotation has them.
    template <int RUN>
    __device__ __forceinline__ int place() const {
        return RUN == 4 ? 256 * (at >> 6) + 16 * (lane & 15) + 4 * (lane >> 4) : at * RUN;
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

// Whether rows of W values of es bytes divide into aligned pieces of `run` values; rows that are absent do.
inline bool whole(const RowView& v, int W, int run, int es) {
    const int piece = std::min(16, run * es);
    return !v.p || (W % run == 0 && (uintptr_t)v.p % piece == 0 && v.ld * es % piece == 0);
}

// How rows are dealt: `per` threads hold a row, `slots` runs each; `groups` rows a workgroup; `grid` workgroups, each of which takes
// every grid-th of the row groups (by_parts: one each).  slots 0: rows longer than any, or shorter than a
// run.
struct RowCut {
    int per = 64, groups = 1, slots = 1;
    unsigned grid = 1;
    dim3 block() const { return dim3((unsigned)(per * groups)); }
};
// 8-value runs: a slot more from 512 threads on (norm 4608 x 6144 to int8, 384 threads of two slots 35.5 us, 768 of one 38.2), up to
// `most` slots and, with these, 1024 threads; fewer slots hold up to `threads`.  4-value runs: four slots, and eight where
// `most` says so and a row has more than 20 times 256 values (activation 9504 x 13824 in bf16: four 144 us, eight 140; 9504 x 5120: both 56),
// which also holds rows of up to 32768 values.
// waves: that a CU is to hold, where workgroups take rows in turn.
inline RowCut cut_rows(int64_t T, int W, int run, int most, int threads, int waves) {
    RowCut c;
    const int64_t runs = run == 4 ? (W + 255) / 256 * 64 : (W + run - 1) / run;
    c.slots = 0;
    c.per = 512;
    for (int s = run == 4 ? (most == 8 && runs > 20 * 64 ? 8 : 4) : 1; s <= most && W >= run; s *= 2) {
        const int64_t n = ((runs + s - 1) / s + 63) / 64 * 64;
        if (n > (s == most ? 1024 : s == 1 ? 512 : threads)) continue;
        c.slots = s;
        c.per = (int)n;
        break;
    }
    c.groups = c.slots && c.per < 256 ? 256 / c.per : 1;
    if (!c.slots && !waves) waves = 32;  // rows longer than any slots hold, read twice (4096 x 20480 to int8: one workgroup a CU 261 us, four 158)
    const int64_t blocks = (T + c.groups - 1) / c.groups, held = 256 * (int64_t)std::max(1, waves * 64 / (c.per * c.groups));
    const int64_t rounds = (blocks + held - 1) / held;
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
