// Rotation of q and k by positions on several axes, with the per-head norms in the same pass
// (y = rotate(w * x * rsqrt(mean(x^2) + eps))), into tensors or straight into a paged cache, and
// its gradient.  Bound by memory: every value is read once and written once.
//
// A row (one head of one token) is held by the smallest power of two of lanes that has 2 * VW values a lane: VW pairs,
// as two vectors (i .. and i + P .., or 2 i .. and the next), so that a pair never leaves its lane.  A
// workgroup takes all or some heads of a few tokens: their cosines and sines are formed once, a pair a thread, and
// shared through LDS, as are the weights in fp32; the next row's loads are in flight while one is computed.
#include <algorithm>

#include "attention.h"

namespace qlin {
namespace {

constexpr int THREADS = 256;
constexpr int MAX_TOKENS = 8;         // tokens of one workgroup
constexpr int WORKGROUPS = 2048;      // that a large call is cut into at least (8 on a compute unit)
constexpr int GRAD_WORKGROUPS = 1024;
constexpr int MOST_ROUNDS = 12;       // rows of one lane group, at most

template <int DT> struct HeadType;
template <> struct HeadType<DT_F32> { using T = float; };
template <> struct HeadType<DT_F16> { using T = f16; };
template <> struct HeadType<DT_BF16> { using T = __bf16; };

__device__ __forceinline__ double position_at(const RopeTurn& r, int pair, int64_t t) {
    const int ax = r.axis ? min(max(r.axis[pair], 0), r.axes - 1) : 0;
    const int64_t i = ax * r.pos_sa + t * r.pos_st;
    if (r.pos_dt == DT_I32) return (double)((const int32_t*)r.pos)[i];
    if (r.pos_dt == DT_I64) return (double)((const int64_t*)r.pos)[i];
    return (double)((const float*)r.pos)[i];
}

// cos and sin of position * frequency: the product and its reduction to a turn in 64 bits, so that
// a position of a million loses nothing; then one fp32 evaluation on [-1/2, 1/2] turns.
__device__ __forceinline__ void turn_at(const RopeTurn& r, int pair, int64_t t, float& c, float& s) {
    double rev = position_at(r, pair, t) * (double)r.inv_freq[pair] * 0.15915494309189533577;
    rev -= rint(rev);
    sincospif(2.0f * (float)rev, &s, &c);
    if (r.inverse) s = -s;
}

// How a call is cut: `lanes` a row, `heads` rows a token (store: v's too), `tokens` tokens and `span` rows of
// them a workgroup (span < heads: one token over several workgroups).
struct Cut {
    int lanes = 1, heads = 0, tokens = 1, span = 0;
    uint32_t magic = 0;   // ceil(2^32 / heads), for row / heads of two and more
};

// The values a lane holds of a row: x[e] and x[VW + e] are a pair, or x[2 e] and x[2 e + 1] of interleaved ones.
// VEC: two vectors; else value by value (any D and P).  A lane past the row's end holds zeros.
template <typename T, int VW, bool VEC, bool INTER>
struct Piece {
    static constexpr int N = 2 * VW;
    struct alignas(sizeof(T) * VW < 16 ? sizeof(T) * VW : 16) Vector { T v[VW]; };
    int first, second;    // VEC: where the vectors start
    int pair;             // the first pair's number
    int D, P;
    bool inside;
    __device__ __forceinline__ Piece(int unit, int D_, int P_) : pair(VW * unit), D(D_), P(P_) {
        if (INTER || pair >= P) {
            first = N * unit;
            second = first + VW;
        } else {
            first = VW * unit;
            second = P + first;
        }
        inside = 2 * pair < D;
    }
    // Where value j is in the row; -1 for none.
    __device__ __forceinline__ int at(int j) const {
        if (VEC && !INTER && pair >= P) return inside ? first + j : -1;
        const int i = pair + (INTER ? j / 2 : j % VW), half = INTER ? j % 2 : j / VW;
        const int d = i < P && !INTER ? i + half * P : 2 * i + half;
        return d < D ? d : -1;
    }
    struct Raw { Vector a, b; };
    __device__ __forceinline__ Raw load(const T* row, bool wanted) const {
        Raw r = {};
        if constexpr (VEC) {
            if (wanted && inside) {
                r.a = *reinterpret_cast<const Vector*>(row + first);
                r.b = *reinterpret_cast<const Vector*>(row + second);
            }
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (wanted && at(j) >= 0) (j < VW ? r.a.v[j] : r.b.v[j - VW]) = row[at(j)];
        }
        return r;
    }
    static __device__ __forceinline__ void values(const Raw& r, float* x) {
#pragma unroll
        for (int e = 0; e < VW; ++e) {
            x[e] = (float)r.a.v[e];
            x[VW + e] = (float)r.b.v[e];
        }
    }
    __device__ __forceinline__ void store(T* row, const float* x) const {
        if constexpr (VEC) {
            Vector a, b;
#pragma unroll
            for (int e = 0; e < VW; ++e) {
                a.v[e] = (T)x[e];
                b.v[e] = (T)x[VW + e];
            }
            if (inside) {
                *reinterpret_cast<Vector*>(row + first) = a;
                *reinterpret_cast<Vector*>(row + second) = b;
            }
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (at(j) >= 0) row[at(j)] = (T)x[j];
        }
    }
    // (u, v) of pair e
    static __device__ __forceinline__ float& u(float* x, int e) { return x[INTER ? 2 * e : e]; }
    static __device__ __forceinline__ float& v(float* x, int e) { return x[INTER ? 2 * e + 1 : VW + e]; }
};

// Sum over the lanes of a row.
__device__ __forceinline__ float row_sum(float v, int lanes) {
    if (lanes > 1) v += lane_xor<1>(v);
    if (lanes > 2) v += lane_xor<2>(v);
    if (lanes > 4) v += lane_xor<4>(v);
    if (lanes > 8) v += lane_xor<8>(v);
    if (lanes > 16) v += lane_xor<16>(v);
    if (lanes > 32) v += lane_xor<32>(v);
    return v;
}

// In LDS: the weights of q and k as the pieces hold them (1 where there are none), then cosines and
// sines [tokens][P] each, padded to whole pieces.
struct Shared {
    float* w;       // [2][units][2 VW]
    float* c;
    float* s;
    int stride;     // of a token's cosines
};

template <typename PC, int VW>
__device__ __forceinline__ Shared shared_part(float* lds, int units, int tokens) {
    Shared h;
    h.stride = units * VW;
    h.w = lds;
    h.c = lds + 2 * units * 2 * VW;
    h.s = h.c + tokens * h.stride;
    return h;
}

template <typename PC, int VW>
__device__ __forceinline__ void fill_weights(const Shared& h, int units, int D, int P, const void* wq, int wq_dt,
                                             const void* wk, int wk_dt) {
    for (int i = threadIdx.x; i < 2 * units * 2 * VW; i += THREADS) {
        const int kind = i / (units * 2 * VW), j = i % (units * 2 * VW), d = PC(j / (2 * VW), D, P).at(j % (2 * VW));
        const void* w = kind ? wk : wq;
        h.w[i] = w && d >= 0 ? load_rt(w, kind ? wk_dt : wq_dt, d) : 1.0f;
    }
}

// Cosines and sines of `count` tokens from t0 on; the pairs behind P turn by nothing.
__device__ __forceinline__ void fill_turns(const Shared& h, const RopeTurn& r, int64_t t0, int count) {
    for (int i = threadIdx.x; i < count * h.stride; i += THREADS) {
        const int t = i / h.stride, pair = i - t * h.stride;
        float c = 1.0f, s = 0.0f;
        if (pair < r.P) turn_at(r, pair, t0 + t, c, s);
        h.c[i] = c;
        h.s[i] = s;
    }
}

template <int VW>
__device__ __forceinline__ void read_row(const float* p, float* x) {
#pragma unroll
    for (int e = 0; e < VW; e += 4) *reinterpret_cast<f32x4*>(x + e) = *reinterpret_cast<const f32x4*>(p + e);
}

extern __shared__ __align__(16) float lds[];

template <int DT, int VW, bool VEC, bool INTER>
__global__ __launch_bounds__(THREADS) void head_rope_kernel(HeadRopeArgs a, Cut cut) {
    using T = typename HeadType<DT>::T;
    using PC = Piece<T, VW, VEC, INTER>;
    __shared__ int64_t to_k[MAX_TOKENS], to_v[MAX_TOKENS];
    __shared__ bool stored[MAX_TOKENS];
    const int units = (a.D + 2 * VW - 1) / (2 * VW);
    const int unit = threadIdx.x & (cut.lanes - 1), group = threadIdx.x / cut.lanes, groups = THREADS / cut.lanes;
    const int64_t t0 = (int64_t)blockIdx.x * cut.tokens;
    const int tokens = (int)min<int64_t>(cut.tokens, a.T - t0);
    const int begin = blockIdx.y * cut.span, end = min(begin + cut.span, tokens * cut.heads);
    const PC piece(unit, a.D, a.turn.P);

    // the place of a row of this workgroup's
    struct Row {
        int token, h, kind;
    };
    const auto row_of = [&](int r) {
        Row x;
        // the magic number of one head would be 2^32
        x.token = cut.tokens == 1 ? 0 : cut.heads == 1 ? r : (int)__umulhi((uint32_t)r, cut.magic);
        x.h = r - x.token * cut.heads;
        x.kind = x.h < a.Hq ? 0 : x.h < a.Hq + a.Hk ? 1 : 2;
        x.h -= x.kind == 0 ? 0 : x.kind == 1 ? a.Hq : a.Hq + a.Hk;
        return x;
    };
    const auto load = [&](int r, Row& x) {
        x = row_of(r);
        const T* base = (const T*)(x.kind == 0 ? a.q.p : x.kind == 1 ? a.k.p : a.v.p);
        const int64_t st = x.kind == 0 ? a.q.st : x.kind == 1 ? a.k.st : a.v.st, sh = x.kind == 0 ? a.q.sh : x.kind == 1 ? a.k.sh : a.v.sh;
        return piece.load(base + (t0 + x.token) * st + x.h * sh, r < end);
    };
    int r = begin + group;
    Row row;
    typename PC::Raw raw = load(r, row);

    const Shared h = shared_part<PC, VW>(lds, units, cut.tokens);
    if (a.norm) fill_weights<PC, VW>(h, units, a.D, a.turn.P, a.wq, a.wq_dt, a.wk, a.wk_dt);
    fill_turns(h, a.turn, t0, tokens);
    if (a.store && threadIdx.x < tokens) {
        const int64_t i = (t0 + threadIdx.x) * a.slots_st;
        const int64_t slot = a.slots_dt == DT_I64 ? ((const int64_t*)a.slots)[i] : ((const int32_t*)a.slots)[i];
        const bool there = slot >= 0 && slot < a.blocks * a.page;
        const int64_t block = there ? slot / a.page : 0, place = there ? slot - block * a.page : 0;
        to_k[threadIdx.x] = block * a.kc.sb + place * a.kc.sp;
        to_v[threadIdx.x] = block * a.vc.sb + place * a.vc.sp;
        stored[threadIdx.x] = there;
    }
    __syncthreads();

    for (; r < end; r += groups) {
        Row next;
        const typename PC::Raw ahead = load(r + groups, next);
        float x[PC::N];
        PC::values(raw, x);
        T* y;
        bool there = true;
        if (row.kind == 0) {
            y = (T*)a.qo.p + (t0 + row.token) * a.qo.st + row.h * a.qo.sh;
        } else if (!a.store) {
            y = (T*)a.ko.p + (t0 + row.token) * a.ko.st + row.h * a.ko.sh;
        } else {
            const int64_t to = row.kind == 1 ? to_k[row.token] : to_v[row.token];
            there = stored[row.token];
            y = (T*)(row.kind == 1 ? a.kc.p : a.vc.p) + to + row.h * (row.kind == 1 ? a.kc.sh : a.vc.sh);
        }
        if (row.kind < 2) {
            if (a.norm) {
                float sum = 0.0f;
#pragma unroll
                for (int j = 0; j < PC::N; ++j) sum = __builtin_fmaf(x[j], x[j], sum);
                const float rstd = 1.0f / sqrtf(row_sum(sum, cut.lanes) / (float)a.D + a.eps);
                if (piece.inside) {
                    float w[PC::N];
                    read_row<PC::N>(h.w + (row.kind * units + unit) * PC::N, w);
#pragma unroll
                    for (int j = 0; j < PC::N; ++j) x[j] *= rstd * w[j];
                }
            }
            if (piece.inside) {
                float c[VW], s[VW];
                read_row<VW>(h.c + row.token * h.stride + piece.pair, c);
                read_row<VW>(h.s + row.token * h.stride + piece.pair, s);
#pragma unroll
                for (int e = 0; e < VW; ++e) {
                    const float u = PC::u(x, e), v = PC::v(x, e);
                    PC::u(x, e) = u * c[e] - v * s[e];
                    PC::v(x, e) = u * s[e] + v * c[e];
                }
            }
        }
        if (there) piece.store(y, x);
        raw = ahead;
        row = next;
    }
}

// Sums of the weights' gradients stay in a lane over all its rows and are added up over the workgroup at
// the end, in a fixed order; every workgroup leaves one partial [2][D].
template <int DT, int VW, bool VEC, bool INTER>
__global__ __launch_bounds__(THREADS) void head_grad_kernel(HeadGradArgs a, Cut cut) {
    using T = typename HeadType<DT>::T;
    using PC = Piece<T, VW, VEC, INTER>;
    const int units = (a.D + 2 * VW - 1) / (2 * VW);
    const int unit = threadIdx.x & (cut.lanes - 1), group = threadIdx.x / cut.lanes, groups = THREADS / cut.lanes;
    const PC piece(unit, a.D, a.turn.P);
    const Shared h = shared_part<PC, VW>(lds, units, cut.tokens);
    fill_weights<PC, VW>(h, units, a.D, a.turn.P, a.wq, a.wq_dt, a.wk, a.wk_dt);
    float dw[2][PC::N] = {};
    for (int64_t t0 = (int64_t)blockIdx.x * cut.tokens; t0 < a.T; t0 += (int64_t)gridDim.x * cut.tokens) {
        const int tokens = (int)min<int64_t>(cut.tokens, a.T - t0);
        __syncthreads();
        fill_turns(h, a.turn, t0, tokens);
        __syncthreads();
#pragma unroll
        for (int kind = 0; kind < 2; ++kind) {
            const HeadView &in = kind ? a.k : a.q, &gin = kind ? a.gk : a.gq, &out = kind ? a.dk : a.dq;
            const int heads = kind ? a.Hk : a.Hq, end = tokens * heads;
            struct Two {
                typename PC::Raw x, g;
                int token, h;
            };
            const auto load = [&](int r) {
                Two w;
                w.token = heads > 0 ? r / heads : 0;
                w.h = r - w.token * heads;
                w.x = piece.load((const T*)in.p + (t0 + w.token) * in.st + w.h * in.sh, r < end);
                w.g = piece.load((const T*)gin.p + (t0 + w.token) * gin.st + w.h * gin.sh, r < end);
                return w;
            };
            int r = group;
            Two two = load(r);
            for (; r < end; r += groups) {
                const Two ahead = load(r + groups);
                float x[PC::N], g[PC::N];
                PC::values(two.x, x);
                PC::values(two.g, g);
                float sum = 0.0f;
#pragma unroll
                for (int j = 0; j < PC::N; ++j) sum = __builtin_fmaf(x[j], x[j], sum);
                const float rstd = 1.0f / sqrtf(row_sum(sum, cut.lanes) / (float)a.D + a.eps);
                float w[PC::N] = {};
                if (piece.inside) {
                    float c[VW], s[VW];
                    read_row<PC::N>(h.w + (kind * units + unit) * PC::N, w);
                    read_row<VW>(h.c + two.token * h.stride + piece.pair, c);
                    read_row<VW>(h.s + two.token * h.stride + piece.pair, s);
#pragma unroll
                    for (int e = 0; e < VW; ++e) {
                        const float u = PC::u(g, e), v = PC::v(g, e);
                        PC::u(g, e) = u * c[e] + v * s[e];
                        PC::v(g, e) = v * c[e] - u * s[e];
                    }
                }
                float dot = 0.0f;
#pragma unroll
                for (int j = 0; j < PC::N; ++j) {
                    x[j] *= rstd;
                    dw[kind][j] = __builtin_fmaf(g[j], x[j], dw[kind][j]);
                    g[j] *= w[j];
                    dot = __builtin_fmaf(g[j], x[j], dot);
                }
                dot = row_sum(dot, cut.lanes) / (float)a.D;
#pragma unroll
                for (int j = 0; j < PC::N; ++j) g[j] = rstd * (g[j] - x[j] * dot);
                piece.store((T*)out.p + (t0 + two.token) * out.st + two.h * out.sh, g);
                two = ahead;
            }
        }
    }
    if (!a.part) return;
    // the wave's rows, then the workgroup's waves
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __syncthreads();
#pragma unroll
    for (int kind = 0; kind < 2; ++kind)
#pragma unroll
        for (int j = 0; j < PC::N; ++j) {
            float v = dw[kind][j];
            for (int m = cut.lanes; m < 64; m <<= 1) v += __shfl_xor(v, m);
            if (lane < cut.lanes && unit < units) lds[((wave * 2 + kind) * units + unit) * PC::N + j] = v;
        }
    __syncthreads();
    const int all = 2 * units * PC::N;
    for (int i = threadIdx.x; i < all; i += THREADS) {
        const int kind = i / (units * PC::N), j = i % (units * PC::N), d = PC(j / PC::N, a.D, a.turn.P).at(j % PC::N);
        const float v = (lds[i] + lds[all + i]) + (lds[2 * all + i] + lds[3 * all + i]);
        if (d >= 0) a.part[((int64_t)blockIdx.x * 2 + kind) * a.D + d] = v;
    }
}

// Weight gradients from the partials: a workgroup takes 16 values of q's or k's weight, 16 partials at a time.
__global__ __launch_bounds__(THREADS) void head_grad_sum_kernel(HeadGradArgs a, int parts) {
    __shared__ float s[16][17];
    const int col = threadIdx.x & 15, row = threadIdx.x >> 4, i = blockIdx.x * 16 + col;
    float sum = 0.0f;
    if (i < 2 * a.D) {
#pragma unroll 8
        for (int p = row; p < parts; p += 16) sum += a.part[(int64_t)p * 2 * a.D + i];
    }
    s[row][col] = sum;
    __syncthreads();
    if (row == 0 && i < 2 * a.D) {
#pragma unroll
        for (int p = 1; p < 16; ++p) sum += s[p][col];
        const int kind = i / a.D, d = i - kind * a.D;
        if (kind == 0 && a.dwq) store_rt(a.dwq, a.dwq_dt, d, sum);
        if (kind == 1 && a.dwk) store_rt(a.dwk, a.dwk_dt, d, sum);
    }
}

// Whether rows of these views move in pieces of `bytes` (8 or 16).
bool aligned(const void* p, std::initializer_list<int64_t> strides, int es, int bytes) {
    if ((uintptr_t)p % bytes) return false;
    for (int64_t s : strides)
        if (s * es % bytes) return false;
    return true;
}

// The pieces of a call: 8 pairs a lane where both sizes allow 8-value vectors and all rows are aligned to them, else 4,
// else 8 value by value.
struct Kind {
    int VW;
    bool vec;
};
template <typename ALIGNED>
Kind kind_of(int D, int P, int dtype, const ALIGNED& all_aligned) {
    const int es = dtype == DT_F32 ? 4 : 2;
    if (D % 16 == 0 && P % 8 == 0 && all_aligned(es, 16)) return {8, true};
    if (D % 8 == 0 && P % 4 == 0 && all_aligned(es, 4 * es)) return {4, true};
    return {8, false};
}

Cut cut_of(const Kind& k, int D, int heads) {
    Cut c;
    const int units = (D + 2 * k.VW - 1) / (2 * k.VW);
    while (c.lanes < units) c.lanes *= 2;
    c.heads = heads;
    return c;
}

// Rounds of a workgroup's lane groups: few where the call is small, so that it spreads over the chip; more where it
// is large, so that cosines and the launch are shared by more rows.
int rounds_of(const Cut& c, int64_t T, int workgroups) {
    const int64_t groups = THREADS / c.lanes, rounds = T * c.heads / (groups * workgroups);
    return (int)std::max<int64_t>(1, std::min<int64_t>(rounds, MOST_ROUNDS));
}

size_t lds_bytes(const Kind& k, int D, int tokens, bool grad) {
    const size_t units = (D + 2 * k.VW - 1) / (2 * k.VW), w = 2 * units * 2 * k.VW, turns = 2 * (size_t)tokens * units * k.VW;
    return 4 * (grad ? std::max(w + turns, 4 * w) : w + turns);
}

template <int DT, bool INTER>
hipError_t launch_rope(const HeadRopeArgs& a, const Kind& k, const Cut& c, dim3 grid, hipStream_t st) {
    const size_t bytes = lds_bytes(k, a.D, c.tokens, false);
    if (!k.vec) hipLaunchKernelGGL((head_rope_kernel<DT, 8, false, INTER>), grid, dim3(THREADS), bytes, st, a, c);
    else if (k.VW == 8) hipLaunchKernelGGL((head_rope_kernel<DT, 8, true, INTER>), grid, dim3(THREADS), bytes, st, a, c);
    else hipLaunchKernelGGL((head_rope_kernel<DT, 4, true, INTER>), grid, dim3(THREADS), bytes, st, a, c);
    return hipGetLastError();
}

template <int DT, bool INTER>
hipError_t launch_grad(const HeadGradArgs& a, const Kind& k, const Cut& c, dim3 grid, hipStream_t st) {
    const size_t bytes = lds_bytes(k, a.D, c.tokens, true);
    if (!k.vec) hipLaunchKernelGGL((head_grad_kernel<DT, 8, false, INTER>), grid, dim3(THREADS), bytes, st, a, c);
    else if (k.VW == 8) hipLaunchKernelGGL((head_grad_kernel<DT, 8, true, INTER>), grid, dim3(THREADS), bytes, st, a, c);
    else hipLaunchKernelGGL((head_grad_kernel<DT, 4, true, INTER>), grid, dim3(THREADS), bytes, st, a, c);
    return hipGetLastError();
}

}  // namespace

hipError_t run_head_rope(const HeadRopeArgs& a, hipStream_t st) {
    const Kind k = kind_of(a.D, a.turn.P, a.dtype, [&](int es, int bytes) {
        if (!aligned(a.q.p, {a.q.st, a.q.sh}, es, bytes) || !aligned(a.qo.p, {a.qo.st, a.qo.sh}, es, bytes)) return false;
        if (a.Hk == 0) return true;
        if (!aligned(a.k.p, {a.k.st, a.k.sh}, es, bytes)) return false;
        if (!a.store) return aligned(a.ko.p, {a.ko.st, a.ko.sh}, es, bytes);
        return aligned(a.v.p, {a.v.st, a.v.sh}, es, bytes) && aligned(a.kc.p, {a.kc.sb, a.kc.sp, a.kc.sh}, es, bytes) &&
               aligned(a.vc.p, {a.vc.sb, a.vc.sp, a.vc.sh}, es, bytes);
    });
    Cut c = cut_of(k, a.D, a.Hq + a.Hk + (a.store ? a.Hk : 0));
    const int rows = rounds_of(c, a.T, WORKGROUPS) * (THREADS / c.lanes);
    c.tokens = std::max(1, std::min(MAX_TOKENS, rows / c.heads));
    c.span = c.tokens > 1 ? c.tokens * c.heads : std::min(rows, c.heads);
    c.magic = (uint32_t)((0x100000000ull + c.heads - 1) / c.heads);
    const dim3 grid((unsigned)((a.T + c.tokens - 1) / c.tokens), (unsigned)((c.tokens * c.heads + c.span - 1) / c.span));
    const bool i = a.turn.interleaved;
    if (a.dtype == DT_F32) return i ? launch_rope<DT_F32, true>(a, k, c, grid, st) : launch_rope<DT_F32, false>(a, k, c, grid, st);
    if (a.dtype == DT_F16) return i ? launch_rope<DT_F16, true>(a, k, c, grid, st) : launch_rope<DT_F16, false>(a, k, c, grid, st);
    return i ? launch_rope<DT_BF16, true>(a, k, c, grid, st) : launch_rope<DT_BF16, false>(a, k, c, grid, st);
}

// At most one token a workgroup less than there are, GRAD_WORKGROUPS of them at most.
int head_grad_parts(int64_t T, int64_t) { return (int)std::max<int64_t>(1, std::min<int64_t>(T, GRAD_WORKGROUPS)); }

size_t ws_head_grad(int64_t T, int64_t heads, int64_t D) { return (size_t)head_grad_parts(T, heads) * 2 * D * 4; }

hipError_t run_head_grad(const HeadGradArgs& a, hipStream_t st) {
    const Kind k = kind_of(a.D, a.turn.P, a.dtype, [&](int es, int bytes) {
        for (const HeadView* v : {&a.q, &a.gq, &a.dq})
            if (!aligned(v->p, {v->st, v->sh}, es, bytes)) return false;
        if (a.Hk > 0)
            for (const HeadView* v : {&a.k, &a.gk, &a.dk})
                if (!aligned(v->p, {v->st, v->sh}, es, bytes)) return false;
        return true;
    });
    Cut c = cut_of(k, a.D, a.Hq + a.Hk);
    // several tokens where one has fewer heads than a workgroup lane groups
    const int groups = THREADS / c.lanes, least = std::max(1, std::min(a.Hq, a.Hk > 0 ? a.Hk : a.Hq));
    const int parts = head_grad_parts(a.T, a.Hq + a.Hk);
    c.tokens = (int)std::max<int64_t>(1, std::min<int64_t>({MAX_TOKENS, groups / least, a.T / parts}));
    const dim3 grid((unsigned)parts);
    const bool i = a.turn.interleaved;
    hipError_t e;
    if (a.dtype == DT_F32) e = i ? launch_grad<DT_F32, true>(a, k, c, grid, st) : launch_grad<DT_F32, false>(a, k, c, grid, st);
    else if (a.dtype == DT_F16) e = i ? launch_grad<DT_F16, true>(a, k, c, grid, st) : launch_grad<DT_F16, false>(a, k, c, grid, st);
    else e = i ? launch_grad<DT_BF16, true>(a, k, c, grid, st) : launch_grad<DT_BF16, false>(a, k, c, grid, st);
    if (e != hipSuccess || (!a.dwq && !a.dwk)) return e;
    hipLaunchKernelGGL(head_grad_sum_kernel, dim3((unsigned)((2 * a.D + 15) / 16)), dim3(THREADS), 0, st, a, parts);
    return hipGetLastError();
}

}  // namespace qlin
