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
constexpr int MAX_TOKENS = 64;        // tokens that a workgroup's rows belong to, at most: see most_tokens()
constexpr int WORKGROUPS = 2048;      // that a call is spread over, once or several times
constexpr int GRAD_WORKGROUPS = 1024; // of head_grad_kernel that the chip holds at once
constexpr int MOST_ROUNDS = 5;        // rows of one lane group, at most
constexpr int GRAD_TOKENS = 8;        // tokens of one block of the gradient

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

// row / heads for the rows of a few tokens (row * heads < 2^32), by ceil(2^32 / heads).
struct Divisor {
    int heads = 1;
    uint32_t magic = 0;
    Divisor() = default;
    explicit Divisor(int h) : heads(h), magic(h > 1 ? (uint32_t)((0x100000000ull + h - 1) / h) : 0) {}
    // the magic number of one head would be 2^32
    __device__ __forceinline__ int operator()(int r) const { return heads <= 1 ? r : (int)__umulhi((uint32_t)r, magic); }
};

// How a call is cut: `lanes` a row, `heads` rows a token (store: v's too).  Forward: all rows laid end to end, `span` of
// them a workgroup, of `tokens` tokens at most.  Gradient: blocks of `tokens` tokens.
struct Cut {
    int lanes = 1, heads = 0, tokens = 1, span = 0;
    Divisor by_heads;
};

// The values a lane holds of a row: x[e] and x[VW + e] are a pair, or x[2 e] and x[2 e + 1] of interleaved ones.
// VEC: two vectors, which neighbouring lanes continue (ONCE: read nontemporally); else value by value (any D and P).  A
// lane past the row's end holds zeros.
enum { SCALAR = 0, VECTORS = 1, ONCE = 2 };
// INTER: pairs of neighbours; SOME_PAIRS: not all of a row's (vectors).
enum { HALVES = 0, PAIRS = 1, SOME_PAIRS = 2 };
template <typename T, int VW, int VEC, int INTER>
struct Piece {
    static constexpr int N = 2 * VW;
    struct alignas(sizeof(T) * VW < 16 ? sizeof(T) * VW : 16) Vector { T v[VW]; };
    int first, second;    // VEC: where the vectors start
    int pair;             // the first pair's number; VEC INTER: the second vector's first pair is pair2
    int pair2;
    int D, P;
    bool inside;
    __device__ __forceinline__ Piece(int unit, int D_, int P_) : pair(VW * unit), pair2(VW * unit + VW / 2), D(D_), P(P_) {
        inside = 2 * pair < D;
        if (INTER) {
            first = VW * unit;
            second = D / 2 + first;
            if (VEC) {
                pair = first / 2;
                pair2 = second / 2;
            }
        } else if (pair >= P) {
            first = N * unit;
            second = first + VW;
        } else {
            first = VW * unit;
            second = P + first;
        }
    }
    // Where value j is in the row; -1 for none.
    __device__ __forceinline__ int at(int j) const {
        if (VEC) return inside ? (j < VW ? first + j : second + j - VW) : -1;
        const int i = pair + (INTER ? j / 2 : j % VW), half = INTER ? j % 2 : j / VW;
        const int d = i < P && !INTER ? i + half * P : 2 * i + half;
        return d < D ? d : -1;
    }
    // The VW pairs' entries of a table of all pairs.
    __device__ __forceinline__ void turns(const float* table, float* x) const {
        typedef float V __attribute__((ext_vector_type(VW / 2)));
        *reinterpret_cast<V*>(x) = *reinterpret_cast<const V*>(table + pair);
        *reinterpret_cast<V*>(x + VW / 2) = *reinterpret_cast<const V*>(table + (VEC && INTER ? pair2 : pair + VW / 2));
    }
    static __device__ __forceinline__ Vector vector_at(const T* p) {
        typedef uint32_t Words __attribute__((ext_vector_type(sizeof(Vector) % 16 ? 2 : 4)));
        if constexpr (VEC != ONCE) {
            return *reinterpret_cast<const Vector*>(p);
        } else if constexpr (sizeof(Vector) == sizeof(Words)) {
            return __builtin_bit_cast(Vector, __builtin_nontemporal_load(reinterpret_cast<const Words*>(p)));
        } else {
            struct Two { Words a, b; };
            static_assert(sizeof(Vector) == sizeof(Two), "8 fp32 values");
            const Words* q = reinterpret_cast<const Words*>(p);
            return __builtin_bit_cast(Vector, Two{__builtin_nontemporal_load(q), __builtin_nontemporal_load(q + 1)});
        }
    }
    struct Raw { Vector a, b; };
    __device__ __forceinline__ Raw load(const T* row, bool wanted) const {
        Raw r = {};
        if constexpr (VEC) {
            if (wanted && inside) {
                r.a = vector_at(row + first);
                r.b = vector_at(row + second);
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
    // Turns the pairs by (c, s), or BACK.  Values behind the P pairs pass as they are: 0 times an infinity beside them would
    // be a NaN.  In halves a vector turns whole or not at all; pairs of neighbours are looked at one by one where not all of
    // them turn, in a kernel of its own: with that test 1056 tokens x 96 heads take 13.6 us, without 13.1.
    template <bool BACK>
    __device__ __forceinline__ void rotate(float* x, const float* c, const float* s) const {
        if (VEC && INTER == HALVES && pair >= P) return;
#pragma unroll
        for (int e = 0; e < VW; ++e) {
            if ((!VEC || INTER == SOME_PAIRS) && (VEC && e >= VW / 2 ? pair2 + e - VW / 2 : pair + e) >= P) continue;
            const float a = u(x, e), b = v(x, e);
            u(x, e) = __builtin_fmaf(a, c[e], BACK ? b * s[e] : -(b * s[e]));
            v(x, e) = BACK ? __builtin_fmaf(b, c[e], -(a * s[e])) : __builtin_fmaf(a, s[e], b * c[e]);
        }
    }
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

template <int DT, int VW, int VEC, int INTER>
__global__ __launch_bounds__(THREADS) void head_rope_kernel(HeadRopeArgs a, Cut cut) {
    using T = typename HeadType<DT>::T;
    using PC = Piece<T, VW, VEC, INTER>;
    __shared__ int64_t to_k[MAX_TOKENS], to_v[MAX_TOKENS];
    __shared__ bool stored[MAX_TOKENS];
    const int units = (a.D + 2 * VW - 1) / (2 * VW);
    const int unit = threadIdx.x & (cut.lanes - 1), group = threadIdx.x / cut.lanes, groups = THREADS / cut.lanes;
    const int64_t from = (int64_t)blockIdx.x * cut.span, t0 = from / cut.heads;
    const int begin = (int)(from - t0 * cut.heads);  // rows count from the first head of token t0
    const int end = begin + (int)min<int64_t>(cut.span, a.T * cut.heads - from), tokens = cut.by_heads(end - 1) + 1;
    const PC piece(unit, a.D, a.turn.P);

    // the place of a row of this workgroup's
    struct Row {
        int token, h, kind;
    };
    const auto row_of = [&](int r) {
        Row x;
        x.token = cut.by_heads(r);
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
                piece.turns(h.c + row.token * h.stride, c);
                piece.turns(h.s + row.token * h.stride, s);
                piece.template rotate<false>(x, c, s);
            }
        }
        if (there) piece.store(y, x);
        raw = ahead;
        row = next;
    }
}

// A workgroup takes q's rows (workgroups below parts_q) or k's.  Sums of the weight's gradient stay in a lane over all
// its rows and are added up over the workgroup at the end, in a fixed order; every workgroup leaves one partial [D].
template <int DT, int VW, int VEC, int INTER>
__global__ __launch_bounds__(THREADS, VEC ? 4 : 1) void head_grad_kernel(HeadGradArgs a, Cut cut, Divisor by_q, Divisor by_k, int parts_q) {
    using T = typename HeadType<DT>::T;
    using PC = Piece<T, VW, VEC, INTER>;
    const bool of_k = (int)blockIdx.x >= parts_q;
    const int units = (a.D + 2 * VW - 1) / (2 * VW), heads = of_k ? a.Hk : a.Hq;
    const Divisor by_heads = of_k ? by_k : by_q;
    const int unit = threadIdx.x & (cut.lanes - 1), group = threadIdx.x / cut.lanes, groups = THREADS / cut.lanes;
    const int part = of_k ? blockIdx.x - parts_q : blockIdx.x, parts = of_k ? gridDim.x - parts_q : parts_q;
    const HeadView in = of_k ? a.k : a.q, gin = of_k ? a.gk : a.gq, out = of_k ? a.dk : a.dq;
    const PC piece(unit, a.D, a.turn.P);
    const Shared h = shared_part<PC, VW>(lds, units, cut.tokens);
    fill_weights<PC, VW>(h, units, a.D, a.turn.P, of_k ? a.wk : a.wq, of_k ? a.wk_dt : a.wq_dt, nullptr, 0);
    float dw[PC::N] = {};
    const int64_t past = heads > 0 ? a.T : 0;  // the one workgroup of a side without heads leaves its sum of zeros at once
    for (int64_t t0 = (int64_t)part * cut.tokens; t0 < past; t0 += (int64_t)parts * cut.tokens) {
        const int tokens = (int)min<int64_t>(cut.tokens, a.T - t0), end = tokens * heads;
        __syncthreads();
        fill_turns(h, a.turn, t0, tokens);
        __syncthreads();
        for (int r = group; r < end; r += groups) {
            const int token = cut.tokens == 1 ? 0 : by_heads(r), head = r - token * heads;
            const typename PC::Raw rx = piece.load((const T*)in.p + (t0 + token) * in.st + head * in.sh, true);
            const typename PC::Raw rg = piece.load((const T*)gin.p + (t0 + token) * gin.st + head * gin.sh, true);
            float x[PC::N], g[PC::N];
            PC::values(rx, x);
            PC::values(rg, g);
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < PC::N; ++j) sum = __builtin_fmaf(x[j], x[j], sum);
            const float rstd = 1.0f / sqrtf(row_sum(sum, cut.lanes) / (float)a.D + a.eps);
            float w[PC::N] = {};
            if (piece.inside) {
                float c[VW], s[VW];
                piece.turns(h.c + token * h.stride, c);
                piece.turns(h.s + token * h.stride, s);
                piece.template rotate<true>(g, c, s);
                read_row<PC::N>(h.w + unit * PC::N, w);
            }
            float dot = 0.0f;
#pragma unroll
            for (int j = 0; j < PC::N; ++j) {
                x[j] *= rstd;
                dw[j] = __builtin_fmaf(g[j], x[j], dw[j]);
                g[j] *= w[j];
                dot = __builtin_fmaf(g[j], x[j], dot);
            }
            dot = row_sum(dot, cut.lanes) / (float)a.D;
#pragma unroll
            for (int j = 0; j < PC::N; ++j) g[j] = rstd * (g[j] - x[j] * dot);
            piece.store((T*)out.p + (t0 + token) * out.st + head * out.sh, g);
        }
    }
    if (!a.part) return;
    // the wave's rows, then the workgroup's waves
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, all = units * PC::N;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PC::N; ++j) {
        for (int m = cut.lanes; m < 64; m <<= 1) dw[j] += __shfl_xor(dw[j], m);
        if (lane < cut.lanes && unit < units) lds[wave * all + unit * PC::N + j] = dw[j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < all; i += THREADS) {
        const int d = PC(i / PC::N, a.D, a.turn.P).at(i % PC::N);
        const float v = (lds[i] + lds[all + i]) + (lds[2 * all + i] + lds[3 * all + i]);
        if (d >= 0) a.part[(int64_t)blockIdx.x * a.D + d] = v;
    }
}

// Weight gradients from the partials: a workgroup takes 16 values of q's weight or of k's, SUM_ROWS partials at a time.
constexpr int SUM_ROWS = 64;
__global__ __launch_bounds__(16 * SUM_ROWS) void head_grad_sum_kernel(HeadGradArgs a, int parts_q, int parts) {
    __shared__ float s[SUM_ROWS][17];
    const int col = threadIdx.x & 15, row = threadIdx.x >> 4, d = blockIdx.x * 16 + col;
    const bool of_k = blockIdx.y;
    void* dw = of_k ? a.dwk : a.dwq;
    if (!dw) return;
    float sum = 0.0f;
    if (d < a.D) {
#pragma unroll 8
        for (int p = (of_k ? parts_q : 0) + row; p < (of_k ? parts : parts_q); p += SUM_ROWS) sum += a.part[(int64_t)p * a.D + d];
    }
    s[row][col] = sum;
    __syncthreads();
    for (int n = SUM_ROWS / 2; n >= 1; n >>= 1) {
        if (row < n) s[row][col] += s[row + n][col];
        __syncthreads();
    }
    if (row == 0 && d < a.D) store_rt(dw, of_k ? a.dwk_dt : a.dwq_dt, d, s[0][col]);
}

// Whether rows of these views move in pieces of `bytes` (8 or 16).
bool aligned(const void* p, std::initializer_list<int64_t> strides, int es, int bytes) {
    if ((uintptr_t)p % bytes) return false;
    for (int64_t s : strides)
        if (s * es % bytes) return false;
    return true;
}

// The pieces of a call: 8 pairs a lane where both sizes allow 8-value vectors and all rows are aligned to them, else 4,
// else 8 value by value.  Vectors of interleaved pairs hold whole pairs whatever P is.
//
// Rows of more than MUCH bytes in all are read nontemporally: what they would take of the caches is left to the outputs,
// which the next kernel reads.  Measured between a kernel that writes the rows and one that reads the outputs (us, all three;
// nontemporal / not): 9504 tokens x 80 heads of 128 (195 MB) 186 / 202, 4608 x 96 (113) 109 / 108, 6000 x 40 (61) 65.3 / 65.8, 3000 x
// 128 of 64 (49) 54.3 / 53.3, 1056 x 96 (26) 32.2 / 32.6; the gradient 228 / 257, 139 / 144, 89.4 / 87.7, 74.7 / 70.7, 48.6 / 45.3.  Rows
// that come from memory, normalized into a cache: 4095 x 48 of 128 (50) 23.7 / 25.2.  So 32 to 64 MB gain or lose by up to 6%
// with what is around them; below, plain loads win, above, the others.  Nontemporal stores gain nothing.
constexpr int64_t MUCH = 32 << 20;

struct Kind {
    int VW;
    int vec;
};
template <typename ALIGNED>
Kind kind_of(int64_t rows, int D, const RopeTurn& turn, int dtype, const ALIGNED& all_aligned) {
    const int es = dtype == DT_F32 ? 4 : 2, P = turn.interleaved ? 0 : turn.P;
    const int vec = rows * D * es > MUCH ? ONCE : VECTORS;
    if (D % 16 == 0 && P % 8 == 0 && all_aligned(es, 16)) return {8, vec};
    if (D % 8 == 0 && P % 4 == 0 && all_aligned(es, 4 * es)) return {4, vec};
    return {8, SCALAR};
}

// Tokens whose cosines and sines a workgroup holds in LDS, at most: 32 KB of them, or two tokens.
int64_t most_tokens(int64_t D) { return std::max<int64_t>(2, std::min<int64_t>(MAX_TOKENS, 8192 / (D + 15))); }

Cut cut_of(const Kind& k, int D, int heads) {
    Cut c;
    const int units = (D + 2 * k.VW - 1) / (2 * k.VW);
    while (c.lanes < units) c.lanes *= 2;
    c.heads = heads;
    c.by_heads = Divisor(heads);
    return c;
}

// Tokens of a workgroup, at most `most`: the fewest whose rows leave the least of the lane groups' last round idle
// (to a twentieth).
int tokens_of(int heads, int groups, int most) {
    int best = 1;
    double held = 0.0;
    for (int t = 1; t <= most; ++t) {
        const int64_t rows = (int64_t)t * heads, rounds = (rows + groups - 1) / groups;
        const double share = (double)rows / (double)(rounds * groups);
        if (share > held + 0.05) {
            held = share;
            best = t;
        }
    }
    return best;
}

size_t lds_bytes(const Kind& k, int D, int tokens, bool grad) {
    const size_t units = (D + 2 * k.VW - 1) / (2 * k.VW), w = 2 * units * 2 * k.VW, turns = 2 * (size_t)tokens * units * k.VW;
    return 4 * (grad ? std::max(w + turns, 2 * w) : w + turns);
}

template <int DT, int INTER>
hipError_t launch_rope(const HeadRopeArgs& a, const Kind& k, const Cut& c, dim3 grid, hipStream_t st) {
    const size_t bytes = lds_bytes(k, a.D, c.tokens, false);
    const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(THREADS), bytes, st, a, c); };
    if (k.vec == SCALAR) go(head_rope_kernel<DT, 8, SCALAR, INTER != HALVES>);
    else if (k.VW == 8 && k.vec == ONCE) go(head_rope_kernel<DT, 8, ONCE, INTER>);
    else if (k.VW == 8) go(head_rope_kernel<DT, 8, VECTORS, INTER>);
    else if (k.vec == ONCE) go(head_rope_kernel<DT, 4, ONCE, INTER>);
    else go(head_rope_kernel<DT, 4, VECTORS, INTER>);
    return hipGetLastError();
}

template <int DT, int INTER>
hipError_t launch_grad(const HeadGradArgs& a, const Kind& k, const Cut& c, dim3 grid, int parts_q, hipStream_t st) {
    const size_t bytes = lds_bytes(k, a.D, c.tokens, true);
    const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(THREADS), bytes, st, a, c, Divisor(a.Hq), Divisor(a.Hk), parts_q); };
    if (k.vec == SCALAR) go(head_grad_kernel<DT, 8, SCALAR, INTER != HALVES>);
    else if (k.VW == 8 && k.vec == ONCE) go(head_grad_kernel<DT, 8, ONCE, INTER>);
    else if (k.VW == 8) go(head_grad_kernel<DT, 8, VECTORS, INTER>);
    else if (k.vec == ONCE) go(head_grad_kernel<DT, 4, ONCE, INTER>);
    else go(head_grad_kernel<DT, 4, VECTORS, INTER>);
    return hipGetLastError();
}

template <typename F>
hipError_t of_type(int dtype, const F& typed) {
    if (dtype == DT_F32) return typed(std::integral_constant<int, DT_F32>{});
    if (dtype == DT_F16) return typed(std::integral_constant<int, DT_F16>{});
    return typed(std::integral_constant<int, DT_BF16>{});
}

}  // namespace

hipError_t run_head_rope(const HeadRopeArgs& a, hipStream_t st) {
    const Kind k = kind_of(a.T * (a.Hq + a.Hk), a.D, a.turn, a.dtype, [&](int es, int bytes) {
        if (!aligned(a.q.p, {a.q.st, a.q.sh}, es, bytes) || !aligned(a.qo.p, {a.qo.st, a.qo.sh}, es, bytes)) return false;
        if (a.Hk == 0) return true;
        if (!aligned(a.k.p, {a.k.st, a.k.sh}, es, bytes)) return false;
        if (!a.store) return aligned(a.ko.p, {a.ko.st, a.ko.sh}, es, bytes);
        return aligned(a.v.p, {a.v.st, a.v.sh}, es, bytes) && aligned(a.kc.p, {a.kc.sb, a.kc.sp, a.kc.sh}, es, bytes) &&
               aligned(a.vc.p, {a.vc.sb, a.vc.sp, a.vc.sh}, es, bytes);
    });
    Cut c = cut_of(k, a.D, a.Hq + a.Hk + (a.store ? a.Hk : 0));
    // Equal runs of rows, in whole rounds of the lane groups: a small call is spread over the chip, a row a lane group; a
    // large one over WORKGROUPS at a time, which share a token's cosines among up to 5 rounds.  Measured (us, at
    // most 3 / 5 / 8 / 16 rounds): 4095 tokens x 56 rows into a cache 29.7 / 26.4 / 26.8 / 26.1, 4608 x 96 40.9 /
    // 40.3 / 47.4 / 47.2, 9504 x 80 66.9 / 65.0 / 67.3 / 76.7, 5000 x 20 of 256 values 25.4 / 23.7 / 23.7 / 23.7, 6000 x 40 27.2 / 27.9 /
    // 27.9 / 27.8, 3000 x 128 of 64 25.5 / 25.6 / 25.6 / 25.5.
    const int64_t groups = THREADS / c.lanes, rows = a.T * c.heads, round = groups * WORKGROUPS;
    const int64_t times = std::max<int64_t>(1, (rows + MOST_ROUNDS * round - 1) / (MOST_ROUNDS * round));
    int64_t span = std::max<int64_t>(1, (rows + times * round - 1) / (times * round)) * groups;
    span = std::min(span, (most_tokens(a.D) - 1) * c.heads);
    c.span = (int)std::min(span, rows);
    c.tokens = (int)std::min<int64_t>(a.T, (c.span - 1) / c.heads + 2);
    const dim3 grid((unsigned)((rows + c.span - 1) / c.span));
    const auto typed = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (!a.turn.interleaved) return launch_rope<DT, HALVES>(a, k, c, grid, st);
        return 2 * a.turn.P < a.D ? launch_rope<DT, SOME_PAIRS>(a, k, c, grid, st) : launch_rope<DT, PAIRS>(a, k, c, grid, st);
    };
    return of_type(a.dtype, typed);
}

int head_grad_parts(int64_t T, int64_t) { return (int)std::max<int64_t>(2, std::min<int64_t>(2 * T, GRAD_WORKGROUPS)); }

size_t ws_head_grad(int64_t T, int64_t heads, int64_t D) { return (size_t)head_grad_parts(T, heads) * D * 4; }

hipError_t run_head_grad(const HeadGradArgs& a, hipStream_t st) {
    const Kind k = kind_of(a.T * (a.Hq + a.Hk), a.D, a.turn, a.dtype, [&](int es, int bytes) {
        for (const HeadView* v : {&a.q, &a.gq, &a.dq})
            if (!aligned(v->p, {v->st, v->sh}, es, bytes)) return false;
        if (a.Hk > 0)
            for (const HeadView* v : {&a.k, &a.gk, &a.dk})
                if (!aligned(v->p, {v->st, v->sh}, es, bytes)) return false;
        return true;
    });
    Cut c = cut_of(k, a.D, a.Hq + a.Hk);
    // workgroups for q's rows and for k's as their heads are, each with the same number of token blocks or one less
    const int groups = THREADS / c.lanes, most = head_grad_parts(a.T, c.heads);
    const int most_k = std::max(1, std::min<int>(most - 1, (int)((int64_t)most * a.Hk / std::max(c.heads, 1)))), most_q = most - most_k;
    c.tokens = tokens_of(std::max(1, std::min(a.Hq, a.Hk > 0 ? a.Hk : a.Hq)), groups, (int)std::min<int64_t>(GRAD_TOKENS, std::max<int64_t>(1, 4 * a.T / most)));
    const int64_t blocks = std::max<int64_t>(1, (a.T + c.tokens - 1) / c.tokens);
    const auto even = [&](int n) { const int64_t each = (blocks + n - 1) / n; return (int)((blocks + each - 1) / each); };
    const int parts_q = even(most_q), parts = parts_q + even(most_k);
    const dim3 grid((unsigned)parts);
    const auto typed = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (!a.turn.interleaved) return launch_grad<DT, HALVES>(a, k, c, grid, parts_q, st);
        return 2 * a.turn.P < a.D ? launch_grad<DT, SOME_PAIRS>(a, k, c, grid, parts_q, st) : launch_grad<DT, PAIRS>(a, k, c, grid, parts_q, st);
    };
    const hipError_t e = of_type(a.dtype, typed);
    if (e != hipSuccess || (!a.dwq && !a.dwk)) return e;
    hipLaunchKernelGGL(head_grad_sum_kernel, dim3((unsigned)((a.D + 15) / 16), 2), dim3(16 * SUM_ROWS), 0, st, a, parts_q, parts);
    return hipGetLastError();
}

}  // namespace qlin
