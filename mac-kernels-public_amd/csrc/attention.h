// Launcher interfaces of the attention side: rotation and head norms (qk_rope.hip), the tables of a
// step (paged_plan.hip), attention over the paged cache (paged_attention.hip); C ABI in
// capi_attention.hip.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "qlin.h"
#include "qlin_internal.h"

namespace qlin {

// Sets the calling thread's error message and returns s (capi.hip).
qlin_status report(qlin_status s, const char* message);

// [tokens, heads, D] with unit stride along D; strides in elements.
struct HeadView {
    void* p = nullptr;
    int64_t st = 0, sh = 0;
};

// [blocks, page, kv heads, D] with unit stride along D; strides in elements.
struct CacheView {
    void* p = nullptr;
    int64_t sb = 0, sp = 0, sh = 0;
};

// The rotation of a call: pair i turns by positions[axis[i], t] * inv_freq[i].
struct RopeTurn {
    const float* inv_freq = nullptr;
    const int32_t* axis = nullptr;     // nullptr: row 0
    const void* pos = nullptr;
    int pos_dt = DT_I32;
    int64_t pos_sa = 0, pos_st = 0;    // strides of positions along axes and tokens
    int axes = 1;
    int P = 0;                         // pairs
    bool interleaved = false, inverse = false;
};

// ---- rotation and head norms (qk_rope.hip) ----
constexpr int ROPE_MAX_DIM = 512;
constexpr int ROPE_MAX_HEADS = 16384;  // of q, of k; the kernels' division of rows by heads is exact up to 3 x that
struct HeadRopeArgs {
    int dtype = DT_F16;
    int64_t T = 0;
    int Hq = 0, Hk = 0, D = 0;
    HeadView q, k, v;                  // v only with `store`
    HeadView qo, ko;                   // ko unused with `store`
    bool norm = false;
    float eps = 0.0f;
    const void* wq = nullptr;          // [D] or nullptr (1)
    const void* wk = nullptr;
    int wq_dt = DT_F16, wk_dt = DT_F16;
    RopeTurn turn;
    bool store = false;
    CacheView kc, vc;
    int64_t blocks = 0, page = 1;
    const void* slots = nullptr;
    int slots_dt = DT_I64;
    int64_t slots_st = 1;
};
hipError_t run_head_rope(const HeadRopeArgs& a, hipStream_t st);

struct HeadGradArgs {
    int dtype = DT_F16;
    int64_t T = 0;
    int Hq = 0, Hk = 0, D = 0;
    HeadView q, k, gq, gk, dq, dk;
    float eps = 0.0f;
    const void* wq = nullptr;
    const void* wk = nullptr;
    int wq_dt = DT_F16, wk_dt = DT_F16;
    RopeTurn turn;
    void* dwq = nullptr;               // [D] or nullptr (not formed)
    void* dwk = nullptr;
    int dwq_dt = DT_F32, dwk_dt = DT_F32;
    float* part = nullptr;             // head_grad_parts() x [D] partial sums, q's then k's
};
// Workgroups of the gradient kernel, each of which leaves one partial [D].
int head_grad_parts(int64_t T, int64_t heads);
hipError_t run_head_grad(const HeadGradArgs& a, hipStream_t st);
size_t ws_head_grad(int64_t T, int64_t heads, int64_t D);

// ---- the tables of a step (paged_plan.hip) ----
struct PagedPlanArgs {
    const int32_t* context = nullptr;
    const int32_t* added = nullptr;
    const int32_t* free_blocks = nullptr;
    int32_t* table = nullptr;
    int64_t* slots = nullptr;
    int32_t* positions = nullptr;
    int32_t* rows = nullptr;
    int32_t* starts = nullptr;
    int32_t* lengths = nullptr;
    int32_t* used = nullptr;
    int B = 0;
    int64_t F = 0, W = 0, ldt = 0, N = 0, page = 1;
};
hipError_t run_paged_plan(const PagedPlanArgs& a, hipStream_t st);

// ---- attention over the paged cache (paged_attention.hip) ----
constexpr int PAGED_MAX_DIM = 256;
struct PagedAttentionArgs {
    int dtype = DT_F16;
    int64_t B = 0;
    int H = 0, Hk = 0, D = 0;
    HeadView q, out;
    CacheView kc, vc;
    int64_t blocks = 0, page = 1;
    const int32_t* table = nullptr;
    int64_t W = 0, ldt = 0;
    const int32_t* lengths = nullptr;
    float scale = 1.0f;
    int64_t window = 0;
    void* ws = nullptr;
};
hipError_t run_paged_attention(const PagedAttentionArgs& a, hipStream_t st);
size_t ws_paged_attention(int64_t B, int64_t H, int64_t Hk, int64_t D);

}  // namespace qlin
