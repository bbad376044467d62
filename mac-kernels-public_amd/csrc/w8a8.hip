// Product of int8 rows with scales for each token and channel: y[m, n] = sx[m] sw[n] sum_k x[m, k] w[n, k] + bias[n], then
// residual + residual_scale y.  The int32 sums are exact (K < 131072); the epilogue is fp32 with one rounding.
//
// Up to STREAM_ROWS rows the weights are streamed once from memory straight into the matrix cores' operands
// (w8a8_stream_kernel).  More rows run in the int8 GEMM of gemm_i8.hip, whose rows are whole 128-value pieces at 16-byte aligned
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

// Few rows.  A wave owns 16 weight rows and a part of K, which it takes in steps of 64 values: lane l loads 16 codes of
// weight row l % 16 at k = 16 (l / 16) of the step, which are its part of v_mfma_i32_16x16x64_i8's B operand, and the same of
// activation rows l % 16 (A; MT of them, rows behind the last one repeat it).  STEPS steps are in flight a wave, enough for
// 4096 values over 8 waves to be requested at once.  The waves of one weight group, `parts` of the 8, add their sums through LDS.
constexpr int STREAM_ROWS = 64, STEPS = 8;

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
__global__ __launch_bounds__(512) void w8a8_stream_kernel(W8A8Args a, int parts) {
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
        constexpr int U = MT <= 2 ? STEPS : STEPS / 2;  // registers
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
    // lane l, register v of a 16 x 16 product holds row 4 (l / 16) + v, column l % 16
    for (int e = tid; e < groups * MT * 256; e += 512) {
        const int gr = e / (MT * 256), i = e / 256 % MT, v = e / 64 % 4, l = e % 64;
        const int64_t m = 16 * i + 4 * (l >> 4) + v, n = ((int64_t)blockIdx.x * groups + gr) * 16 + (l & 15);
        if (m >= a.M || n >= a.N) continue;
        int sum = 0;
        for (int p = 0; p < parts; ++p) sum += sums[gr * parts + p][i][v][l];
        float y = (float)sum * a.sx[m] * a.sw[n];
        if (a.bias) y += load_rt(a.bias, a.bias_dt, n);
        if (a.res.r) y = __builtin_fmaf(a.res.rs ? load_rt(a.res.rs, a.res.rs_dt, n) : 1.0f, y, load_rt(a.res.r, a.res.r_dt, m * a.res.ldr + n));
        store_rt(a.y, a.y_dt, m * a.ldy + n, y);
    }
}

hipError_t run_stream(const W8A8Args& a, hipStream_t st) {
    const int64_t groups = (a.N + 15) / 16;
    int parts = 8;  // of K: at least four steps each
    while (parts > 1 && a.K / 64 < 4 * parts) parts /= 2;
    const dim3 grid((unsigned)((groups + 8 / parts - 1) / (8 / parts)));
    switch ((a.M + 15) / 16) {
        case 1: hipLaunchKernelGGL(w8a8_stream_kernel<1>, grid, dim3(512), 0, st, a, parts); break;
        case 2: hipLaunchKernelGGL(w8a8_stream_kernel<2>, grid, dim3(512), 0, st, a, parts); break;
        case 3: hipLaunchKernelGGL(w8a8_stream_kernel<3>, grid, dim3(512), 0, st, a, parts); break;
        default: hipLaunchKernelGGL(w8a8_stream_kernel<4>, grid, dim3(512), 0, st, a, parts); break;
    }
    return hipGetLastError();
}

}  // namespace

int w8a8_packs(const W8A8Args& a) {
    if (a.M <= STREAM_ROWS) return 0;
    if (a.K % 128) return W8A8_PACK_X | W8A8_PACK_W;
    const bool x = a.ldx % 16 || (uintptr_t)a.x % 16;
    const bool w = a.ldw != a.K || (uintptr_t)a.w % 16;
    return (x ? W8A8_PACK_X : 0) | (w ? W8A8_PACK_W : 0);
}

size_t ws_w8a8(int64_t M, int64_t N, int64_t K, int packs) {
    if (M <= STREAM_ROWS) return 0;
    if (K % 128) packs = W8A8_PACK_X | W8A8_PACK_W;
    size_t n = 0;
    if (packs & W8A8_PACK_X) n += align_up((size_t)(M * whole(K)));
    if (packs & W8A8_PACK_W) n += align_up((size_t)(N * whole(K)));
    return n;
}

hipError_t run_w8a8(const W8A8Args& a, hipStream_t st) {
    if (a.M == 0 || a.N == 0) return hipSuccess;
    if (a.M <= STREAM_ROWS) return run_stream(a, st);
    GemmI8Args p;
    p.xq = a.x; p.ldx = a.ldx; p.sx = a.sx; p.M = a.M; p.N = a.N; p.K = whole(a.K);
    p.w8 = const_cast<int8_t*>(a.w); p.s_ch = a.sw;
    p.bias = a.bias; p.bias_dtype = a.bias_dt; p.res = a.res;
    p.y = a.y; p.y_dtype = a.y_dt; p.ldy = a.ldy;
    const int packs = w8a8_packs(a);
    uint8_t* ws = (uint8_t*)a.ws;
    if (packs & W8A8_PACK_X) {
        if (hipError_t e = pack_rows(a.x, a.ldx, a.M, a.K, (int8_t*)ws, st)) return e;
        p.xq = (int8_t*)ws;
        p.ldx = p.K;
        ws += align_up((size_t)(a.M * p.K));
    }
    if (packs & W8A8_PACK_W) {
        if (hipError_t e = pack_rows(a.w, a.ldw, a.N, a.K, (int8_t*)ws, st)) return e;
        p.w8 = (int8_t*)ws;
    }
    return run_gemm_i8_dense(p, st);
}

}  // namespace qlin
