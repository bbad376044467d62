// Product of int8 rows with scales for each token and channel: y[m, n] = sx[m] sw[n] sum_k x[m, k] w[n, k] + bias[n], then
// residual + residual_scale y.  The int32 sums are exact (K < 131072); the epilogue is fp32 with one rounding.
//
// The products run in the int8 GEMM of gemm_i8.hip, whose rows are whole 128-value pieces at 16-byte aligned addresses;
// other operands are copied to such rows first, with zeros behind their K values.
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

}  // namespace

int w8a8_packs(const W8A8Args& a) {
    if (a.K % 128) return W8A8_PACK_X | W8A8_PACK_W;
    const bool x = a.ldx % 16 || (uintptr_t)a.x % 16;
    const bool w = a.ldw != a.K || (uintptr_t)a.w % 16;
    return (x ? W8A8_PACK_X : 0) | (w ? W8A8_PACK_W : 0);
}

size_t ws_w8a8(int64_t M, int64_t N, int64_t K, int packs) {
    if (K % 128) packs = W8A8_PACK_X | W8A8_PACK_W;
    size_t n = 0;
    if (packs & W8A8_PACK_X) n += align_up((size_t)(M * whole(K)));
    if (packs & W8A8_PACK_W) n += align_up((size_t)(N * whole(K)));
    return n;
}

hipError_t run_w8a8(const W8A8Args& a, hipStream_t st) {
    if (a.M == 0 || a.N == 0) return hipSuccess;
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
