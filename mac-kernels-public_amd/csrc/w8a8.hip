// Product of int8 rows with scales for each token and channel: y[m, n] = sx[m] sw[n] sum_k x[m, k] w[n, k] + bias[n], then
// residual + residual_scale y.  The int32 sums are exact (K < 131072); the epilogue is fp32 with one rounding.
//
// Few rows stream the weights once from memory (w8a8_tile_kernel; w8a8_any_rows_kernel where rows are not whole 16-byte
// chunks).  More rows run in the int8 GEMM of gemm_i8.hip, whose rows are whole 128-value pieces at 16-byte aligned
// addresses; other operands are copied to such rows first, with zeros behind their K values.
#include <algorithm>

#include "mlp.h"

namespace qlin {
namespace {

constexpr size_t ALIGN = 256;
size_t align_up(size_t v) { return (v + ALIGN - 1) / ALIGN * ALIGN; }
int64_t whole(int64_t K) { return (K + 127) / 128 * 128; }

// [rows, K] of any row stride -> [rows, Kp], zeros behind K; 16 values a thread.
__global__ __launch_bounds__(256) void pack_rows_kernel(const int8_t* x, int64_t ld, int K, int8_t* out, int Kp, int64_t units) {
    const int per = Kp / 16;
    for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < units; u += (int64_t)gridDim.x * 256) {
        const int64_t row = u / per;
        const int k0 = (int)(u - row * per) * 16;
        const int8_t* src = x + row * ld + k0;
        u32x4 v = {0u, 0u, 0u, 0u};
        if (k0 + 16 <= K) {
            __builtin_memcpy(&v, src, 16);
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (k0 + i < K) v[i / 4] |= (uint32_t)(uint8_t)src[i] << (8 * (i % 4));
        }
        *reinterpret_cast<u32x4*>(out + row * Kp + k0) = v;
    }
}

hipError_t pack_rows(const int8_t* x, int64_t ld, int64_t rows, int64_t K, int8_t* out, hipStream_t st) {
    const int64_t Kp = whole(K), units = rows * (Kp / 16);
    const dim3 grid((unsigned)std::min<int64_t>((units + 255) / 256, 8192));
    hipLaunchKernelGGL(pack_rows_kernel, grid, dim3(256), 0, st, x, ld, (int)K, out, (int)Kp, units);
    return hipGetLastError();
}

// ((f32(sum) * sx) * sw) + bias, each operation rounded on its own, then residual + residual_scale * that: the int8 GEMM's
// arithmetic, to the bit.
__device__ __forceinline__ float scaled(int sum, float sx, float sw, bool bias, float b) {
#pragma clang fp contract(off)
    float y = (float)sum * sx;
    y = y * sw;
    return bias ? y + b : y;
}

// A tile of 16 MT rows x 16 NT outputs a workgroup, K split over its waves.  A wave works alone: it brings stages of 128 bytes of
// the tile's rows into a ring of its own in LDS (ST stages, by LDS DMA, a stage two instructions of 8 whole 128-byte lines for
// each 16 rows), and reads them as operands of v_mfma_i32_16x16x64_i8, the next half stage's while one is multiplied.  No
// barrier until the waves' sums meet in LDS.
//
// Why through LDS: lane l of an operand holds row l % 16, so that loads straight into operands touch 4 lines with every 4 lanes,
// and a CU gets 38 B/ns of them from L2 against 150 of whole lines (measured, 256 KB shared by all).  Why the K split:
// each byte passes the CU's LDS once on the way in and once on the way out, where waves that share a tile read it 2 to 4
// times.  A line's 16-byte chunks are XOR-swizzled by row / 2, so that 16 rows' reads meet all banks.  Stages start at another
// place of K in every workgroup: rows of 16384 bytes would meet in few channels otherwise (1 row, N 8192: 33 -> 24 us).
template <int MT, int NT, int WAVES, int ST>
__global__ __launch_bounds__(64 * WAVES) void w8a8_tile_kernel(W8A8Args a, int mtiles) {
    constexpr int TILES = MT + NT, SB = TILES * 2048, PER = 2 * TILES, R = 16 * MT, C = 16 * NT, LDC = C + 4;
    constexpr int LDS = WAVES * (ST * SB > R * LDC * 4 ? ST * SB : R * LDC * 4);
    static_assert(LDS <= 160 * 1024, "rings and sums must fit");
    __shared__ __attribute__((aligned(16))) uint8_t smem[LDS];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r16 = lane & 15, g = lane >> 4;
    // workgroup b runs on XCD b % 8: a contiguous run of tiles each, row tiles innermost, so that an XCD reads its weights once
    const int per = (int)gridDim.x / 8;
    const int b = (int)blockIdx.x < 8 * per ? (int)(blockIdx.x % 8) * per + (int)blockIdx.x / 8 : (int)blockIdx.x;
    const int64_t m0 = (int64_t)(b % mtiles) * R, n0 = (int64_t)(b / mtiles) * C;

    // the outputs of thread tid are 4 columns of rows (tid + T q) / (C / 4); what they need besides the sums is requested now
    constexpr int T = 64 * WAVES, C4 = C / 4, Q = (R * C4 + T - 1) / T;
    static_assert(T % C4 == 0, "a thread's columns are the same in every row");
    const int64_t nc = n0 + 4 * (tid % C4);
    float sx[Q], sw[4];
    uint32_t bias[4];
#pragma unroll
    for (int q = 0; q < Q; ++q) sx[q] = a.sx[min<int64_t>(m0 + (tid + T * q) / C4, a.M - 1)];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int64_t n = min<int64_t>(nc + e, a.N - 1);
        sw[e] = a.sw[n];
        bias[e] = a.bias ? load_bits_rt(a.bias, a.bias_dt, n) : 0u;
    }

    const int count = (int)max<int64_t>(0, min<int64_t>(4, a.N - nc));
    const int es = a.res.r_dt == DT_F32 ? 16 : 8;  // bytes of 4 residual values
    const bool res4 = a.res.r && a.res.ldr % 4 == 0 && (uintptr_t)a.res.r % es == 0;  // n0 is a multiple of 16
    u32x4 res[Q];
    if (res4 && count == 4)
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            const uint8_t* p = (const uint8_t*)a.res.r + (min<int64_t>(m0 + (tid + T * q) / C4, a.M - 1) * a.res.ldr + nc) * (es / 4);
            if (es == 16) {
                res[q] = *reinterpret_cast<const u32x4*>(p);
            } else {
                const u32x2 v = *reinterpret_cast<const u32x2*>(p);
                res[q] = u32x4{v.x & 0xFFFFu, v.x >> 16, v.y & 0xFFFFu, v.y >> 16};
            }
        }

    const int K = (int)a.K, stages = (K + 127) / 128;
    const int first = stages * wave / WAVES, n = stages * (wave + 1) / WAVES - first;
    uint8_t* ring = smem + wave * ST * SB;
    // DMA instruction i of 16 rows: rows 8 i + lane / 8, whose chunk lane % 8 in LDS is chunk (lane % 8) ^ (row / 2) % 8; chunks
    // past the row's end re-read its last one (K is a multiple of 16), and rows past the last one that one
    const int row8 = lane >> 3, most = K / 16 - 1;
    const int c0 = (lane & 7) ^ (row8 >> 1), c1 = (lane & 7) ^ ((8 + row8) >> 1);
    const int8_t *xs = a.x + m0 * a.ldx, *ws = a.w + n0 * a.ldw;
    const int xrows = (int)min<int64_t>(R, a.M - m0), wrows = (int)min<int64_t>(C, a.N - n0);
    uint32_t at[TILES][2];
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i)
            at[t][i] = t < MT ? (uint32_t)min(16 * t + 8 * i + row8, xrows - 1) * (uint32_t)a.ldx
                              : (uint32_t)min(16 * (t - MT) + 8 * i + row8, wrows - 1) * (uint32_t)a.ldw;
    const int start = n > 0 ? b / mtiles % n : 0;
    auto stage_of = [&](int i) {  // stage i in this workgroup's order; past the end the last one again
        i = min(i, n - 1) + start;
        return first + (i >= n ? i - n : i);
    };
    auto fetch = [&](int i, int buf) {
        const int st = stage_of(i);
        const uint32_t k0 = 16 * min(8 * st + c0, most), k1 = 16 * min(8 * st + c1, most);
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const int8_t* rows = t < MT ? xs : ws;
            lds_dma16(rows + (at[t][0] + k0), ring + buf * SB + t * 2048);
            lds_dma16(rows + (at[t][1] + k1), ring + buf * SB + t * 2048 + 1024);
        }
    };
    i32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
    const int sz = r16 >> 1;
    auto read = [&](int buf, int j, i32x4 (&f)[TILES]) {  // half j of a stage: lane l holds row l % 16, k = 64 j + 16 (l / 16) ..
        const uint8_t* p = ring + buf * SB + r16 * 128 + 16 * ((4 * j + g) ^ sz);
#pragma unroll
        for (int t = 0; t < TILES; ++t) f[t] = *reinterpret_cast<const i32x4*>(p + t * 2048);
    };
    auto multiply = [&](int i, int j, i32x4 (&f)[TILES]) {
        const int k = 128 * stage_of(i) + 64 * j;
        if (k + 64 > K && k + 16 * g >= K)  // behind K: nothing
#pragma unroll
            for (int t = 0; t < MT; ++t) f[t] = i32x4{0, 0, 0, 0};
#pragma unroll
        for (int p = 0; p < MT; ++p)
#pragma unroll
            for (int q = 0; q < NT; ++q) acc[p][q] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f[p], f[MT + q], acc[p][q], 0, 0, 0);
    };
    if (n > 0) {
        i32x4 f0[TILES], f1[TILES];
#pragma unroll
        for (int s = 0; s < ST; ++s) fetch(s, s);
        wait_vmcnt<(ST - 1) * PER>();  // stage 0 has landed
        __builtin_amdgcn_sched_barrier(0);
        read(0, 0, f0);
        for (int i = 0; i < n; i += ST) {
#pragma unroll
            for (int s = 0; s < ST; ++s) {
                if (i + s >= n) break;
                read(s, 1, f1);
                multiply(i + s, 0, f0);
                wait_lgkmcnt0();  // the stage has been read: its place is free
                __builtin_amdgcn_sched_barrier(0);
                fetch(i + s + ST, s);
                wait_vmcnt<(ST - 1) * PER>();  // the next stage has landed
                __builtin_amdgcn_sched_barrier(0);
                read((s + 1) % ST, 0, f0);
                multiply(i + s, 1, f1);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        wait_lgkmcnt0();
        wait_vmcnt<0>();
    }
    __syncthreads();  // the rings are no longer written or read

    // lane l, register v of a 16 x 16 product holds row 4 (l / 16) + v, column l % 16
    int* sums = reinterpret_cast<int*>(smem);
#pragma unroll
    for (int p = 0; p < MT; ++p)
#pragma unroll
        for (int q = 0; q < NT; ++q)
#pragma unroll
            for (int v = 0; v < 4; ++v) sums[(wave * R + 16 * p + 4 * g + v) * LDC + 16 * q + r16] = acc[p][q][v];
    __syncthreads();
    const bool vec = a.ldy % 4 == 0 && (uintptr_t)a.y % 16 == 0;
    float rs[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) rs[e] = a.res.rs ? load_rt(a.res.rs, a.res.rs_dt, min<int64_t>(nc + e, a.N - 1)) : 1.0f;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int row = (tid + T * q) / C4;
        const int64_t m = m0 + row;
        if (row >= R || m >= a.M || count == 0) continue;
        i32x4 sum = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < WAVES; ++w) sum += *reinterpret_cast<const i32x4*>(sums + (w * R + row) * LDC + 4 * (tid % C4));
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = scaled(sum[e], sx[q], sw[e], a.bias, bits_to_f32_rt(bias[e], a.bias_dt));
        if (a.res.r) {
            if (res4 && count == 4)
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = __builtin_fmaf(rs[e], y[e], bits_to_f32_rt(res[q][e], a.res.r_dt));
            else residual_apply4(a.res, m, nc, a.N, y);
        }
        store4_rt(a.y, a.y_dt, m * a.ldy + nc, y, count, vec);
    }
}

// Rows of any alignment, few of them.  A wave owns 16 weight rows and a part of K, which it takes in steps of 64 values straight into
// the operands; U steps are in flight.  The waves of one weight group, `parts` of the 8, add their sums through LDS.
constexpr int STREAM_ROWS = 64;

// 16 codes at k of a row of K; zeros behind it.
__device__ __forceinline__ i32x4 codes_at(const int8_t* row, int k, int K) {
    i32x4 v = {0, 0, 0, 0};
    if (k + 16 <= K) {
        __builtin_memcpy(&v, row + k, 16);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (k + i < K) v[i / 4] |= (int)((uint32_t)(uint8_t)row[k + i] << (8 * (i % 4)));
    }
    return v;
}

template <int MT>
__global__ __launch_bounds__(512) void w8a8_any_rows_kernel(W8A8Args a, int parts) {
    __shared__ int sums[8][MT][4][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r16 = lane & 15, g = lane >> 4;
    const int part = wave % parts, groups = 8 / parts, group = wave / parts;
    const int64_t n0 = ((int64_t)blockIdx.x * groups + group) * 16;
    const int K = (int)a.K, steps = K / 64;  // whole ones; the last part takes what is behind them
    const int first = steps * part / parts, end = steps * (part + 1) / parts, last = max(end - 1, first);
    const int8_t* wrow = a.w + min<int64_t>(n0 + r16, a.N - 1) * a.ldw;
    const int8_t* xrow[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) xrow[i] = a.x + min<int64_t>(16 * i + r16, a.M - 1) * a.ldx;
    i32x4 acc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = i32x4{0, 0, 0, 0};
    struct Step {
        i32x4 w, x[MT];
    };
    auto load = [&](int st, Step& s) {
        const int k = 64 * min(st, last) + 16 * g;
        __builtin_memcpy(&s.w, wrow + k, 16);
#pragma unroll
        for (int i = 0; i < MT; ++i) __builtin_memcpy(&s.x[i], xrow[i] + k, 16);
    };
    auto multiply = [&](const Step& s) {
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(s.x[i], s.w, acc[i], 0, 0, 0);
    };
    if (first < end) {
        constexpr int U = MT <= 2 ? 8 : 4;  // registers
        Step s[U];
#pragma unroll
        for (int u = 0; u < U; ++u) load(first + u, s[u]);
        int st = first;
        for (; st + U < end; st += U) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                multiply(s[u]);
                load(st + U + u, s[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (st + u < end) multiply(s[u]);
    }
    if (part == parts - 1 && 64 * steps < K) {
        Step s;
        const int k = 64 * steps + 16 * g;
        s.w = codes_at(wrow, k, K);
#pragma unroll
        for (int i = 0; i < MT; ++i) s.x[i] = codes_at(xrow[i], k, K);
        multiply(s);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v) sums[wave][i][v][lane] = acc[i][v];
    __syncthreads();
    for (int e = tid; e < groups * MT * 256; e += 512) {
        const int gr = e / (MT * 256), i = e / 256 % MT, v = e / 64 % 4, l = e % 64;
        const int64_t m = 16 * i + 4 * (l >> 4) + v, n = ((int64_t)blockIdx.x * groups + gr) * 16 + (l & 15);
        if (m >= a.M || n >= a.N) continue;
        int sum = 0;
        for (int p = 0; p < parts; ++p) sum += sums[gr * parts + p][i][v][l];
        float y = scaled(sum, a.sx[m], a.sw[n], a.bias, a.bias ? load_rt(a.bias, a.bias_dt, n) : 0.0f);
        if (a.res.r) y = __builtin_fmaf(a.res.rs ? load_rt(a.res.rs, a.res.rs_dt, n) : 1.0f, y, load_rt(a.res.r, a.res.r_dt, m * a.res.ldr + n));
        store_rt(a.y, a.y_dt, m * a.ldy + n, y);
    }
}

hipError_t run_any_rows(const W8A8Args& a, hipStream_t st) {
    const int64_t groups = (a.N + 15) / 16;
    int parts = 8;  // of K: at least four steps each
    while (parts > 1 && a.K / 64 < 4 * parts) parts /= 2;
    const dim3 grid((unsigned)((groups + 8 / parts - 1) / (8 / parts)));
    switch ((a.M + 15) / 16) {
        case 1: hipLaunchKernelGGL(w8a8_any_rows_kernel<1>, grid, dim3(512), 0, st, a, parts); break;
        case 2: hipLaunchKernelGGL(w8a8_any_rows_kernel<2>, grid, dim3(512), 0, st, a, parts); break;
        case 3: hipLaunchKernelGGL(w8a8_any_rows_kernel<3>, grid, dim3(512), 0, st, a, parts); break;
        default: hipLaunchKernelGGL(w8a8_any_rows_kernel<4>, grid, dim3(512), 0, st, a, parts); break;
    }
    return hipGetLastError();
}

template <int MT, int NT, int WAVES, int ST>
hipError_t launch_tiles(const W8A8Args& a, hipStream_t st) {
    const int64_t mt = (a.M + 16 * MT - 1) / (16 * MT), nt = (a.N + 16 * NT - 1) / (16 * NT);
    hipLaunchKernelGGL((w8a8_tile_kernel<MT, NT, WAVES, ST>), dim3((unsigned)(mt * nt)), dim3(64 * WAVES), 0, st, a, (int)mt);
    return hipGetLastError();
}

// What computes a call, and what is copied to rows of its own before it.
enum Path { ANY_ROWS = -1, GEMM = 100 };  // GEMM + i: GEMM_SHAPES[i]
struct Plan {
    int path;
    int packs;
};

// A round of workgroups takes about `us` for each 128 values of K (measured at K = 4096 .. 16384, weights from memory); a call is
// taken to need 5 us and that for every started round of 256 workgroups.  Of 70 calls (M 1 .. 2048, six weights)
// the choice was the fastest measured or within 10% of it in all but four, which lost 15%.
struct Shape {
    int m, n;
    float us;
};
constexpr Shape TILE_SHAPES[] = {{16, 16, 0.06f}, {16, 32, 0.09f}, {16, 64, 0.17f}, {32, 16, 0.11f}, {32, 32, 0.14f},
                                 {32, 64, 0.21f}, {64, 32, 0.21f}, {48, 64, 0.26f}, {64, 64, 0.32f}, {96, 64, 0.38f}};
constexpr Shape GEMM_SHAPES[] = {{128, 64, 0.43f}, {128, 128, 0.6f}, {256, 128, 0.95f}, {128, 256, 1.0f}, {256, 256, 1.22f}};
constexpr int GEMM_TILES[] = {I8_128x64, I8_128x128, I8_256x128, I8_128x256, I8_256x256};

// Tiles of up to 512 threads in a launch of fewer than 2^32.
constexpr int64_t MOST_TILES = 1 << 23;

float cost(const Shape& s, int64_t M, int64_t N, int64_t K) {
    const int64_t tiles = ((M + s.m - 1) / s.m) * ((N + s.n - 1) / s.n);
    if (tiles >= MOST_TILES) return 1e20f;
    return 5.0f + s.us * (float)((K + 127) / 128) * (float)((tiles + 255) / 256);
}

Plan plan_of(int64_t M, int64_t N, int64_t K, int apart) {
    const int all = W8A8_X_ROWS | W8A8_W_ROWS;
    const int packs = K % 128 ? all : ((apart & W8A8_X_ROWS) | (apart & (W8A8_W_ROWS | W8A8_W_APART) ? W8A8_W_ROWS : 0));
    const bool chunks = K % 16 == 0 && !(apart & all);  // the tile kernel takes the rows as they are
    if (!chunks && M <= STREAM_ROWS) return {ANY_ROWS, 0};
    // copying: two launches at most, read and written at 4 TB/s
    const float copy = packs ? 6.0f + 0.5e-6f * (float)whole(K) * ((packs & W8A8_X_ROWS ? (float)M : 0.0f) + (packs & W8A8_W_ROWS ? (float)N : 0.0f)) : 0.0f;
    Plan best{GEMM, packs};
    float least = 1e30f;
    for (int i = 0; i < (int)(sizeof GEMM_SHAPES / sizeof(Shape)); ++i) {
        const float c = copy + cost(GEMM_SHAPES[i], M, N, K);
        if (c < least) {
            least = c;
            best = {GEMM + i, packs};
        }
    }
    for (int i = 0; i < (int)(sizeof TILE_SHAPES / sizeof(Shape)); ++i) {
        const float c = (chunks ? 0.0f : copy) + cost(TILE_SHAPES[i], M, N, K);
        if (c < least) {
            least = c;
            best = {i, chunks ? 0 : packs};
        }
    }
    return best;
}

hipError_t run_tiles(const W8A8Args& a, int shape, hipStream_t st) {
    switch (shape) {
        case 0: return launch_tiles<1, 1, 4, 4>(a, st);
        case 1: return launch_tiles<1, 2, 4, 2>(a, st);
        case 2: return launch_tiles<1, 4, 4, 2>(a, st);
        case 3: return launch_tiles<2, 1, 4, 3>(a, st);
        case 4: return launch_tiles<2, 2, 4, 2>(a, st);
        case 5: return launch_tiles<2, 4, 4, 2>(a, st);
        case 6: return launch_tiles<4, 2, 8, 1>(a, st);
        case 7: return launch_tiles<3, 4, 4, 2>(a, st);
        case 8: return launch_tiles<4, 4, 8, 1>(a, st);
        case 9: return launch_tiles<6, 4, 4, 2>(a, st);
    }
    return hipErrorInvalidValue;
}

// Operands as the path takes them.
hipError_t run_shape(const W8A8Args& a, int path, hipStream_t st) {
    if (path < GEMM) return run_tiles(a, path, st);
    const int shape = GEMM_TILES[path - GEMM];
    // Whole rounds of 256 x 256 tiles, and a call of their own for the rows that would start another of few tiles (9504 rows,
    // 5120 -> 13824: the last 32 rows 15.4 us in tiles of 32 x 64, 34.6 in the GEMM's of 128 x 64).
    if (const int64_t top = shape == I8_256x256 ? tail_split_rows(a.M, a.N) : 0) {
        W8A8Args first = a, rest = a;
        first.M = top;
        rest.M = a.M - top;
        rest.x = a.x + top * a.ldx;
        rest.sx = a.sx + top;
        rest.y = (uint8_t*)a.y + top * a.ldy * dt_bytes(a.y_dt);
        if (a.res.r) rest.res.r = (const uint8_t*)a.res.r + top * a.res.ldr * dt_bytes(a.res.r_dt);
        if (hipError_t e = run_shape(first, path, st)) return e;
        return run_shape(rest, plan_of(rest.M, rest.N, rest.K, 0).path, st);
    }
    GemmI8Args p;
    p.xq = a.x; p.ldx = a.ldx; p.sx = a.sx; p.M = a.M; p.N = a.N; p.K = a.K;
    p.w8 = const_cast<int8_t*>(a.w); p.s_ch = a.sw;
    p.bias = a.bias; p.bias_dtype = a.bias_dt; p.res = a.res;
    p.y = a.y; p.y_dtype = a.y_dt; p.ldy = a.ldy;
    return run_gemm_i8_dense(p, shape, st);
}

}  // namespace

int w8a8_apart(const W8A8Args& a) {
    const auto off = [](const int8_t* p, int64_t ld) { return ld % 16 || (uintptr_t)p % 16 || ld >= W8A8_MOST_APART; };
    return (off(a.x, a.ldx) && a.K % 16 == 0 ? W8A8_X_ROWS : 0) | (off(a.w, a.ldw) && a.K % 16 == 0 ? W8A8_W_ROWS : 0) |
           (a.ldw != a.K ? W8A8_W_APART : 0);
}

size_t ws_w8a8(int64_t M, int64_t N, int64_t K, int apart) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    const int packs = plan_of(M, N, K, apart).packs;
    return (packs & W8A8_X_ROWS ? align_up((size_t)(M * whole(K))) : 0) + (packs & W8A8_W_ROWS ? align_up((size_t)(N * whole(K))) : 0);
}

hipError_t run_w8a8(const W8A8Args& call, hipStream_t st) {
    if (call.M == 0 || call.N == 0) return hipSuccess;
    W8A8Args a = call;
    const Plan plan = plan_of(a.M, a.N, a.K, w8a8_apart(a));
    if (plan.path == ANY_ROWS) return run_any_rows(a, st);
    uint8_t* ws = (uint8_t*)a.ws;
    const int64_t Kp = whole(a.K);
    if (plan.packs & W8A8_X_ROWS) {
        if (hipError_t e = pack_rows(a.x, a.ldx, a.M, a.K, (int8_t*)ws, st)) return e;
        a.x = (int8_t*)ws;
        a.ldx = Kp;
        ws += align_up((size_t)(a.M * Kp));
    }
    if (plan.packs & W8A8_W_ROWS) {
        if (hipError_t e = pack_rows(a.w, a.ldw, a.N, a.K, (int8_t*)ws, st)) return e;
        a.w = (int8_t*)ws;
        a.ldw = Kp;
    }
    if (plan.packs == (W8A8_X_ROWS | W8A8_W_ROWS)) a.K = Kp;
    return run_shape(a, plan.path, st);
}

}  // namespace qlin
