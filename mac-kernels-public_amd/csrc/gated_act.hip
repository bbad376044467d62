// Gated activation: y = f(gate) up (up absent: f(gate)), f(z) = z sigma(t) with t = z (SiLU) or t = 2 sqrt(2/pi) (z + 0.044715
// z^3) (GELU in its tanh form), y in 16 or 32 bits or in 8 with a scale a row, and its gradient.  Bound by memory:
// every value is read once and written once.
//
// 8 bits: a row stays in registers until its largest |value| is known; the codes are rne(127 v / top), v rotated first for
// weights that are stored so, the scale is top / 127.
//
// 9504 x 13824 with up: to bf16 127 us (125 at 6.3 TB/s), to int8 105 (104), rotated by 256 140 (the rotation's vector instructions,
// and in fp16 the activation's conversions, 154); its gradient 217 (209).
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
// Where a thread of an elementwise kernel works: 8 values of a row.  Rows shorter than that are read value by value.
template <bool ONCE, typename T>
struct Values {
    Run<T, 8> r;
    const T* row;
    __device__ __forceinline__ Values(const RowView& v, int64_t t, int e0, int W) : row((const T*)v.p + t * v.ld) {
        if (W >= 8) r = load_piece<ONCE, T, 8>(row, e0, W);
    }
    __device__ __forceinline__ void to(int e0, int W, float* v) const {
        if (W >= 8) trimmed<ONCE, T, 8>(r, e0, W, v);
        else load_run<T, 8>(row + e0, W - e0, v);
    }
};

// y = f(gate) up, 8 values a thread.  ONCE: nontemporal reads and writes.
template <typename T, int ACT, bool GATED, bool ONCE>
__global__ __launch_bounds__(256) void gated_act_kernel(GatedActArgs a, int64_t t0, uint32_t units, uint32_t per) {
    const uint32_t u = blockIdx.x * 256u + threadIdx.x;
    if (u >= units) return;
    const uint32_t row = u / per;
    const int e0 = (int)(u - row * per) * 8;
    const int64_t t = t0 + row;
    const Values<ONCE, T> gate(a.gate, t, e0, a.W), up(GATED ? a.up : a.gate, t, e0, a.W);
    float z[8], v[8];
    gate.to(e0, a.W, z);
    if constexpr (GATED) up.to(e0, a.W, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float s, dt;
        gate_of<T, ACT>(z[i], s, dt);
        v[i] = GATED ? z[i] * s * v[i] : z[i] * s;
    }
    store_run<ONCE, T, 8>((T*)a.y.p + t * a.y.ld + e0, a.W - e0, v);
}

template <typename T, int ACT, bool GATED, bool ONCE>
__global__ __launch_bounds__(256) void gated_act_grad_kernel(GatedActArgs a, int64_t t0, uint32_t units, uint32_t per) {
    const uint32_t u = blockIdx.x * 256u + threadIdx.x;
    if (u >= units) return;
    const uint32_t row = u / per;
    const int e0 = (int)(u - row * per) * 8;
    const int64_t t = t0 + row;
    const Values<ONCE, T> gate(a.gate, t, e0, a.W), up(GATED ? a.up : a.gate, t, e0, a.W), dy(a.dy, t, e0, a.W);
    float z[8], v[8], g[8];
    gate.to(e0, a.W, z);
    if constexpr (GATED) up.to(e0, a.W, v);
    dy.to(e0, a.W, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float s, dt;
        gate_of<T, ACT>(z[i], s, dt);
        const float p = s * (1.0f - s), f = z[i] * s;
        const float df = p == 0.0f ? s : __builtin_fmaf(z[i] * p, dt, s);  // far from 0, where z dt may be infinite, sigma
        z[i] = g[i] * (GATED ? v[i] : 1.0f) * df;
        v[i] = g[i] * f;
    }
    store_run<ONCE, T, 8>((T*)a.dgate.p + t * a.dgate.ld + e0, a.W - e0, z);
    if constexpr (GATED) store_run<ONCE, T, 8>((T*)a.dup.p + t * a.dup.ld + e0, a.W - e0, v);
}

// f(z) w of a run into w, rotated (RUN 4).
template <typename T, int ACT, bool GATED, int RUN>
__device__ __forceinline__ void values_of(const float* z, float* w, const Rotation& turned) {
#pragma unroll
    for (int i = 0; i < RUN; ++i) {
        float s, dt;
        gate_of<T, ACT>(z[i], s, dt);
        w[i] = GATED ? z[i] * s * w[i] : z[i] * s;
    }
    if constexpr (RUN == 4) turned(w);
}

template <typename T, int ACT, bool GATED, int RUN, int SLOTS, bool ONCE>
__global__ __launch_bounds__(1024, SLOTS * RUN > 16 ? 4 : 6) void gated_act_int8_kernel(GatedActArgs a, int64_t t0, int per, int groups) {
    const Group g(per);
    const Rotation turned(RUN == 4 ? a.G : 1, g.lane);
    const int64_t t = t0 + (int64_t)blockIdx.x * groups + g.wave / g.waves;
    const bool live = t < a.T;
    const int64_t from = live ? t : a.T - 1;
    const int e0 = g.place<RUN>(), apart = per * RUN;
    Run<T, RUN> gate[SLOTS], up[SLOTS];
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
        gate[s] = load_piece<ONCE, T, RUN>((const T*)a.gate.p + from * a.gate.ld, e0 + s * apart, a.W);
        if constexpr (GATED) up[s] = load_piece<ONCE, T, RUN>((const T*)a.up.p + from * a.up.ld, e0 + s * apart, a.W);
    }
    float v[SLOTS][RUN], none = 0.0f;
    float top = 0.0f;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
        float z[RUN];
        trimmed<ONCE, T, RUN>(gate[s], e0 + s * apart, a.W, z);
        if constexpr (GATED) trimmed<ONCE, T, RUN>(up[s], e0 + s * apart, a.W, v[s]);
        values_of<T, ACT, GATED, RUN>(z, v[s], turned);
        top = larger(top, e0 + s * apart < a.W ? largest<RUN>(v[s]) : 0.0f);
    }
    g.sums(none, top, 0, larger);
    if (!live) return;
    float first;
    const float inv = code_factor(top, first);
    if (g.at == 0) a.scale[t] = top * (RUN == 4 ? turned.left : 1.0f) / 127.0f;
    if (first != 1.0f)
#pragma unroll
        for (int s = 0; s < SLOTS; ++s)
#pragma unroll
            for (int i = 0; i < RUN; ++i) v[s][i] *= first;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
        const int e = e0 + s * apart;
        if (e < a.W) store_codes<ONCE, RUN>(a.q + t * a.ldq + e, a.W - e, v[s], inv);
    }
}

// Rows of any length, read twice.
template <typename T, int ACT, bool GATED, int RUN>
__global__ __launch_bounds__(512) void gated_act_int8_long_kernel(GatedActArgs a) {
    const Group g(512);
    const Rotation turned(RUN == 4 ? a.G : 1, g.lane);
    int turn = 0;
    for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x, turn ^= 1) {
        const T *gate = (const T*)a.gate.p + t * a.gate.ld, *up = GATED ? (const T*)a.up.p + t * a.up.ld : nullptr;
        float v[RUN], none = 0.0f;
        float top = 0.0f;
        auto value = [&](int e0) {
            float z[RUN];
            load_run<T, RUN>(gate + e0, a.W - e0, z);
            if constexpr (GATED) load_run<T, RUN>(up + e0, a.W - e0, v);
            values_of<T, ACT, GATED, RUN>(z, v, turned);
        };
        for (int c = 0; c < a.W; c += 512 * RUN) {
            value(c + g.place<RUN>());
            top = larger(top, largest<RUN>(v));
        }
        g.sums(none, top, turn, larger);
        float first;
        const float inv = code_factor(top, first);
        if (g.at == 0) a.scale[t] = top * (RUN == 4 ? turned.left : 1.0f) / 127.0f;
        for (int c = 0; c < a.W; c += 512 * RUN) {
            const int e0 = c + g.place<RUN>();
            value(e0);
#pragma unroll
            for (int i = 0; i < RUN; ++i) v[i] *= first;
            if (e0 < a.W) store_codes<false, RUN>(a.q + t * a.ldq + e0, a.W - e0, v, inv);
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
    const RowCut c = cut_rows(a.T, a.W, RUN, RUN == 4 ? 8 : 4, 640, 0);
    if (!c.slots) {
        hipLaunchKernelGGL((gated_act_int8_long_kernel<T, ACT, GATED, RUN>), dim3(c.grid), c.block(), 0, st, a);
        return hipGetLastError();
    }
    const bool once = whole(a.gate, a.W, RUN, sizeof(T)) && whole(a.up, a.W, RUN, sizeof(T)) && whole({a.q, a.ldq}, a.W, RUN, 1);
    return by_parts(c, a.T, [&](dim3 grid, int64_t t0) {
        auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, c.block(), 0, st, a, t0, c.per, c.groups); };
        auto by_slots = [&]<int SLOTS>() {
            once ? go(gated_act_int8_kernel<T, ACT, GATED, RUN, SLOTS, true>) : go(gated_act_int8_kernel<T, ACT, GATED, RUN, SLOTS, false>);
        };
        switch (c.slots) {
            case 1: if constexpr (RUN == 8) by_slots.template operator()<1>(); break;
            case 2: if constexpr (RUN == 8) by_slots.template operator()<2>(); break;
            case 4: by_slots.template operator()<4>(); break;
            case 8: if constexpr (RUN == 4) by_slots.template operator()<8>(); break;
        }
    });
}

}  // namespace

hipError_t run_gated_act(const GatedActArgs& a, hipStream_t st) {
    if (a.T == 0 || a.W == 0) return hipSuccess;
    return by_kind(a, [&]<typename T, int ACT, bool GATED>() {
        if (a.q) return a.G ? launch_int8<T, ACT, GATED, 4>(a, st) : launch_int8<T, ACT, GATED, 8>(a, st);
        const bool once = whole(a.gate, a.W, 8, sizeof(T)) && whole(a.up, a.W, 8, sizeof(T)) && whole(a.y, a.W, 8, sizeof(T));
        return by_units(a, [&](dim3 grid, int64_t t0, uint32_t units, uint32_t per) {
            auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(256), 0, st, a, t0, units, per); };
            once ? go(gated_act_kernel<T, ACT, GATED, true>) : go(gated_act_kernel<T, ACT, GATED, false>);
        });
    });
}

hipError_t run_gated_act_grad(const GatedActArgs& a, hipStream_t st) {
    if (a.T == 0 || a.W == 0) return hipSuccess;
    return by_kind(a, [&]<typename T, int ACT, bool GATED>() {
        const bool once = whole(a.gate, a.W, 8, sizeof(T)) && whole(a.up, a.W, 8, sizeof(T)) && whole(a.dy, a.W, 8, sizeof(T)) &&
                          whole(a.dgate, a.W, 8, sizeof(T)) && whole(a.dup, a.W, 8, sizeof(T));
        return by_units(a, [&](dim3 grid, int64_t t0, uint32_t units, uint32_t per) {
            auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(256), 0, st, a, t0, units, per); };
            once ? go(gated_act_grad_kernel<T, ACT, GATED, true>) : go(gated_act_grad_kernel<T, ACT, GATED, false>);
        });
    });
}

}  // namespace qlin
