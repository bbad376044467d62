// Launcher interfaces of the MLP side: norm with the residual's addition (add_norm.hip), gated
// activation (gated_act.hip), int8 product (w8a8.hip); C ABI in capi_mlp.hip.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "qlin.h"
#include "qlin_internal.h"

namespace qlin {

// [rows, values] with unit stride along the values; ld in elements.
struct RowView {
    void* p = nullptr;
    int64_t ld = 0;
};

constexpr int MLP_MAX_WIDTH = 1 << 20;  // values of a row

// ---- norm with the residual's addition (add_norm.hip) ----
struct AddNormArgs {
    int dtype = DT_F16;                // x, y
    int h_dtype = DT_F16;              // residual, h: dtype, or f32
    int64_t T = 0;
    int W = 0;
    RowView x, r, h, y;                // r.p == nullptr: no residual, h is not written
    const void* w = nullptr;           // [W] or nullptr (1)
    int w_dt = DT_F16;
    float eps = 0.0f;
    int8_t* q = nullptr;               // 8-bit output instead of y, with its scales [T]
    int64_t ldq = 0;
    float* scale = nullptr;
    int G = 0;                         // ConvRot group of the 8-bit output, 0 = none
};
hipError_t run_add_norm(const AddNormArgs& a, hipStream_t st);

struct AddNormGradArgs {
    int dtype = DT_F16;                // dy
    int h_dtype = DT_F16;              // h, dh, dx
    int64_t T = 0;
    int W = 0;
    RowView dy, dh, h, dx;             // dh.p == nullptr: none
    const void* w = nullptr;
    int w_dt = DT_F16;
    float eps = 0.0f;
    void* dw = nullptr;                // [W] or nullptr (not formed)
    int dw_dt = DT_F32;
    float* part = nullptr;             // ws_add_norm_grad() bytes: a row of W partial sums a workgroup
};
hipError_t run_add_norm_grad(const AddNormGradArgs& a, hipStream_t st);
size_t ws_add_norm_grad(int64_t T, int64_t W);

// ---- gated activation (gated_act.hip) ----
struct GatedActArgs {
    int dtype = DT_F16;                // of all
    int act = QLIN_ACT_SILU;
    int64_t T = 0;
    int W = 0;
    RowView gate, up, y;               // up.p == nullptr: not gated
    int8_t* q = nullptr;               // 8-bit output instead of y, with its scales [T]
    int64_t ldq = 0;
    float* scale = nullptr;
    int G = 0;
    RowView dy, dgate, dup;            // the gradient
};
hipError_t run_gated_act(const GatedActArgs& a, hipStream_t st);
hipError_t run_gated_act_grad(const GatedActArgs& a, hipStream_t st);

// ---- int8 product (w8a8.hip) ----
// Longest contraction: 128 * 128 * K < 2^31, both sides may hold -128.
constexpr int W8A8_MAX_K = 131071;
struct W8A8Args {
    const int8_t* x = nullptr;         // [M, K]
    int64_t ldx = 0;
    const float* sx = nullptr;         // [M]
    const int8_t* w = nullptr;         // [N, K]
    int64_t ldw = 0;
    const float* sw = nullptr;         // [N]
    int64_t M = 0, N = 0, K = 0;
    const void* bias = nullptr;        // [N] or nullptr
    int bias_dt = DT_NONE;
    ResidualTile res;
    void* y = nullptr;
    int y_dt = DT_F16;
    int64_t ldy = 0;
    void* ws = nullptr;                // ws_w8a8() bytes, 256-byte aligned
};
// What keeps a call's operands from being taken as they are (bits of `param`).
enum { W8A8_X_ROWS = QLIN_W8A8_X_ROWS, W8A8_W_ROWS = QLIN_W8A8_W_ROWS, W8A8_W_APART = QLIN_W8A8_W_APART };
// Rows and outputs of a call below these, and at most 2^36 results: 256 x 256 tiles are then fewer than 2^22, and shapes whose launch would have
// 2^32 threads or more are not chosen (cost() in w8a8.hip).
constexpr int64_t W8A8_MOST_ROWS = 1 << 28, W8A8_MOST_OUTPUTS = 1 << 26, W8A8_MOST_RESULTS = (int64_t)1 << 36;
constexpr int64_t W8A8_MOST_APART = 1 << 24;  // row strides below it: the kernels' offsets in a tile, of up to 256 rows, are 32 bits
int w8a8_apart(const W8A8Args& a);
size_t ws_w8a8(int64_t M, int64_t N, int64_t K, int apart);
hipError_t run_w8a8(const W8A8Args& a, hipStream_t st);

// The int8 GEMM over whole rows of K values, K a multiple of 128, 16-byte aligned rows, weights K
// apart (gemm_i8.hip): p.xq, p.sx, p.w8, p.s_ch, bias, residual and y, in tiles of the given shape.  256 x 256: as the decoded grids
// take them, with the rows past whole rounds in smaller ones.
enum { I8_128x64, I8_128x128, I8_256x128, I8_128x256, I8_256x256 };
hipError_t run_gemm_i8_dense(const GemmI8Args& p, int shape, hipStream_t st);

}  // namespace qlin
