// Attention of one new token a row over a paged cache: out = softmax(scale q K^T) V, one pass over the
// cache with the running maximum m and sum l of the softmax.
//
// What bounds it is the cache's bytes: 2 * 2 * D a token and kv head against 4 * D flops for each query
// head that shares it.  So the query heads of one kv head (up to 16) are computed together by matrix
// instructions whose operands the loads bring in as they are, without LDS:
//   S^T = K Q^T    16 tokens x 16 heads, A = K: a lane has 8 values of one token's row (16 bytes loaded);
//   O^T += V^T P^T  16 dims x 16 heads over 32 tokens, A = V^T: a lane has 8 tokens' pieces of one row (16 bytes
//                  each), whose 16-bit values one v_perm a pair turns into 8 tokens of one dim.
// The order of tokens in the second product is free, so it is the order in which a lane holds S^T: the weights
// go from one to the other in their lane, and m, l and the rescaling are per lane (its column is a head).
//
// The weights p enter the second product as two 16-bit parts (p rounded, and what is left of it), or a row's
// output would carry their rounding on top of its own.  Up to 8 heads the second part rides in the 8 columns that the
// heads leave free; 9 to 16 heads take a second instruction.
//
// Work split: a row's tokens in units of 128 (4 waves x 32), joined in LDS; rows of more than `per` units are split
// over workgroups that leave (O, m, l) in fp32 for a second kernel.  `per` follows on the GPU from all
// rows' lengths, which the host does not know: about TARGET workgroups for the whole batch, so that one long
// row among short ones is spread like the rest.  Every workgroup forms the same plan from the lengths.
#include "attention.h"

namespace qlin {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr int THREADS = 256, WAVES = 4, TILE = 32, UNIT = WAVES * TILE;
constexpr int MAX_ROWS = 1024;       // rows of one launch (their lengths are summed by every workgroup)
constexpr int TARGET = 1024;         // workgroups that a batch is split into

struct Launch {
    PagedAttentionArgs a;
    int ng;                 // head groups of a kv head
    int hpg;                // heads of a group (the last one may have fewer)
    int per_group;          // chunks to aim for, for each head group
    uint64_t page_magic;    // floor(2^64 / d) + 1 for d = page / 16 or page; 0 for d = 1
    float* part_o;          // [chunk][kv head, group][head][D]
    float* part_ml;         // [chunk][kv head, group][head][2]
    int2* meta;             // [rows]: chunks, the first one's place
    bool join;
};

template <int DT> struct Mma;
template <> struct Mma<DT_F16> {
    static __device__ __forceinline__ f32x4 mul(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ float rounded(float v) { return (float)(f16)v; }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const f16x2 h = {(f16)a, (f16)b};
        return __builtin_bit_cast(uint32_t, h);
    }
};
template <> struct Mma<DT_BF16> {
    static __device__ __forceinline__ f32x4 mul(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ float rounded(float v) { return (float)(__bf16)v; }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const bf16x2 h = {(__bf16)a, (__bf16)b};
        return __builtin_bit_cast(uint32_t, h);
    }
};

// n / d for the d of `magic` (any 32-bit n and d).
__device__ __forceinline__ uint32_t divided(uint32_t n, uint64_t magic) {
    if (magic == 0) return n;
    const uint64_t lo = (uint64_t)n * (uint32_t)magic, hi = (uint64_t)n * (uint32_t)(magic >> 32);
    return (uint32_t)((hi + (lo >> 32)) >> 32);
}

// The range of row b's tokens that count.
__device__ __forceinline__ void range_of(const PagedAttentionArgs& a, int b, int& lo, int& hi) {
    const int64_t n = min((int64_t)max(a.lengths[b], 0), a.W * a.page);
    hi = (int)n;
    lo = a.window && n > a.window ? (int)(n - a.window) : 0;
}
__device__ __forceinline__ int units_of(int lo, int hi) { return (hi - (lo & ~(TILE - 1)) + UNIT - 1) / UNIT; }

// What a workgroup computes: tokens [start, end) of row b, which counts [lo, hi).
struct Item {
    int b, chunk, chunks, place, lo, hi, start, end;
};

// The plan from all rows' lengths: `per` units a chunk, and the item of this number; false past the last.
__device__ bool find_item(const Launch& p, int item, Item& it) {
    __shared__ int64_t sum_units[WAVES];
    __shared__ int sum_chunks[WAVES], sum_split[WAVES];
    __shared__ int found[5];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int rows = (int)p.a.B, each = (rows + THREADS - 1) / THREADS;
    int units[MAX_ROWS / THREADS];
    int64_t mine = 0;
#pragma unroll
    for (int i = 0; i < MAX_ROWS / THREADS; ++i) {
        const int b = tid * each + i;
        units[i] = 0;
        if (i < each && b < rows) {
            int lo, hi;
            range_of(p.a, b, lo, hi);
            units[i] = units_of(lo, hi);
        }
        mine += units[i];
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) mine += __shfl_xor(mine, m);
    if (lane == 0) sum_units[wave] = mine;
    if (tid == 0) found[0] = -1;
    __syncthreads();
    int64_t total = 0;
    for (int w = 0; w < WAVES; ++w) total += sum_units[w];
    const int per = (int)max<int64_t>(1, (total + p.per_group - 1) / p.per_group);
    int chunks = 0, split = 0;
#pragma unroll
    for (int i = 0; i < MAX_ROWS / THREADS; ++i)
        if (i < each && tid * each + i < rows) {
            const int c = max(1, (units[i] + per - 1) / per);
            chunks += c;
            split += c > 1 ? c : 0;
        }
    int before = chunks, place = split;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const int x = __shfl_up(before, m), y = __shfl_up(place, m);
        if (lane >= m) {
            before += x;
            place += y;
        }
    }
    if (lane == 63) {
        sum_chunks[wave] = before;
        sum_split[wave] = place;
    }
    __syncthreads();
    before -= chunks;
    place -= split;
    for (int w = 0; w < wave; ++w) {
        before += sum_chunks[w];
        place += sum_split[w];
    }
#pragma unroll
    for (int i = 0; i < MAX_ROWS / THREADS; ++i)
        if (i < each && tid * each + i < rows) {
            const int c = max(1, (units[i] + per - 1) / per);
            if (item >= before && item < before + c) {
                found[0] = tid * each + i;
                found[1] = item - before;
                found[2] = c;
                found[3] = place;
            }
            before += c;
            place += c > 1 ? c : 0;
        }
    __syncthreads();
    it.b = __builtin_amdgcn_readfirstlane(found[0]);
    if (it.b < 0) return false;
    it.chunk = __builtin_amdgcn_readfirstlane(found[1]);
    it.chunks = __builtin_amdgcn_readfirstlane(found[2]);
    it.place = __builtin_amdgcn_readfirstlane(found[3]);
    range_of(p.a, it.b, it.lo, it.hi);
    it.lo = __builtin_amdgcn_readfirstlane(it.lo);
    it.hi = __builtin_amdgcn_readfirstlane(it.hi);
    const int64_t start = (it.lo & ~(TILE - 1)) + (int64_t)it.chunk * per * UNIT;
    it.start = (int)min<int64_t>(start, it.hi);
    it.end = (int)min<int64_t>(start + (int64_t)per * UNIT, it.hi);
    return true;
}

// Bits of the tokens t .. t + 31 that lie in [lo, hi).
__device__ __forceinline__ uint32_t bits_in(int t, int lo, int hi) {
    uint32_t m = ~0u;
    if (t < lo) m &= lo - t < 32 ? ~0u << (lo - t) : 0u;
    if (hi - t < 32) m &= hi > t ? ~(~0u << (hi - t)) : 0u;
    return m;
}

constexpr uint32_t NOWHERE = 0x80000000u;  // a buffer offset past every range: the load gives 0 and reads nothing

template <typename V>
__device__ __forceinline__ V load_from(__amdgpu_buffer_rsrc_t r, uint32_t offset) {
    if constexpr (sizeof(V) == 16) return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b128(r, offset, 0, 0));
    else return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b64(r, offset, 0, 0));
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_at(const void* p) {
    const uint64_t v = (uint64_t)p;
    // readfirstlane gives an int: without the casts a low half of 2^31 and more would fill the upper one with its sign
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32));
    const uint64_t u = (uint64_t)hi << 32 | lo;
    return __builtin_amdgcn_make_buffer_rsrc((void*)u, 0, 0x7FFFFFFF, 0x00027000);
}

// DP: the head size's room (64, 128, 256).  P16: pages of whole 16-token tiles, so that a tile's base address is
// uniform; else every token's address is looked up by itself.  WIDE: 9 to 16 heads.
template <int DT, int DP, bool P16, bool WIDE>
__global__ __launch_bounds__(THREADS, DP == 256 ? 1 : 2) void paged_attention_kernel(Launch p) {
    constexpr int KS = DP / 32;              // 32-value steps of a score
    constexpr int EPL = DP / 16;             // values of a V row that a lane holds
    constexpr int VL = EPL > 8 ? 2 : 1;      // loads they take
    using VT = typename std::conditional<EPL == 4, u32x2, u32x4>::type;
    constexpr int OS = DP + 4;               // row stride of the join in LDS
    constexpr int OH = WIDE ? 16 : 8;
    __shared__ float lds_o[WAVES][OH][OS];
    __shared__ float lds_m[WAVES][16], lds_l[WAVES][16];
    const PagedAttentionArgs& a = p.a;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;  // column (a head) and row group
    const int hg = a.Hk * p.ng, hgi = blockIdx.x % hg;
    Item it;
    if (!find_item(p, blockIdx.x / hg, it)) return;
    const int kvh = hgi / p.ng, G = a.H / a.Hk, h0 = (hgi % p.ng) * p.hpg, heads = min(p.hpg, G - h0);
    if (p.join && hgi == 0 && it.chunk == 0 && threadIdx.x == 0) p.meta[it.b] = make_int2(it.chunks, it.place);

    // Q^T: column n is a head; up to 8 heads the columns 8 .. 15 repeat them for the weights' second part
    const int col = WIDE ? n : n & 7;
    u32x4 q[KS];
#pragma unroll
    for (int j = 0; j < KS; ++j) {
        q[j] = u32x4{0, 0, 0, 0};
        if (col < heads && 32 * j + 8 * g < a.D)
            q[j] = *reinterpret_cast<const u32x4*>((const uint16_t*)a.q.p + it.b * a.q.st +
                                                   (int64_t)(kvh * G + h0 + col) * a.q.sh + 32 * j + 8 * g);
    }
    const uint16_t* kbase = (const uint16_t*)a.kc.p + kvh * a.kc.sh;
    const uint16_t* vbase = (const uint16_t*)a.vc.p + kvh * a.vc.sh;
    const int32_t* table = a.table + it.b * a.ldt;

    // byte offsets within 16 tokens of a page
    uint32_t kofs[KS], vofs[VL];
#pragma unroll
    for (int j = 0; j < KS; ++j) kofs[j] = 32 * j + 8 * g < a.D ? (uint32_t)(n * (int)a.kc.sp + 32 * j + 8 * g) * 2u : NOWHERE;
#pragma unroll
    for (int j = 0; j < VL; ++j) {
        const int d = (EPL < 8 ? EPL : 8) * n + 128 * j;
        vofs[j] = d < a.D ? (uint32_t)(4 * g * (int)a.vc.sp + d) * 2u : NOWHERE;
    }
    const uint32_t vstep = (uint32_t)((int)a.vc.sp * 2);

    u32x4 kr[2][KS];
    VT vr[8][VL];
    // A tile's place: P16 the two halves' block and first place in it; else lane t & 31 has token t's.
    struct Tile {
        int block[2], place[2];
        uint32_t mask;
    };
    auto locate = [&](int t) {
        Tile x;
        x.mask = bits_in(t, it.lo, it.hi);
        if constexpr (P16) {
            const uint32_t per_page = (uint32_t)(a.page >> 4);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t s = (uint32_t)t / 16 + h, pg = divided(s, p.page_magic);
                x.place[h] = (int)(s - pg * per_page) * 16;
                x.block[h] = -1;
                if ((x.mask >> (16 * h)) & 0xFFFFu) x.block[h] = __builtin_amdgcn_readfirstlane(table[pg]);
                if ((uint32_t)x.block[h] >= (uint32_t)a.blocks) {
                    x.block[h] = 0;
                    x.place[h] = 0;
                    x.mask &= h ? 0x0000FFFFu : 0xFFFF0000u;
                }
            }
        } else {
            const int tok = lane & 31;
            const uint32_t s = (uint32_t)t + tok, pg = divided(s, p.page_magic);
            int block = -1;
            if ((x.mask >> tok) & 1) block = table[pg];
            const bool ok = (uint32_t)block < (uint32_t)a.blocks;
            x.block[0] = ok ? block : 0;
            x.place[0] = ok ? (int)(s - pg * (uint32_t)a.page) : 0;
            x.mask = (uint32_t)__ballot(ok);
        }
        return x;
    };
    auto load_k = [&](const Tile& x) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if constexpr (P16) {
                const auto r = buffer_at(kbase + x.block[h] * a.kc.sb + x.place[h] * a.kc.sp);
#pragma unroll
                for (int j = 0; j < KS; ++j) kr[h][j] = load_from<u32x4>(r, kofs[j]);
            } else {
                const int src = 16 * h + n;
                const uint16_t* r = kbase + __shfl(x.block[0], src) * a.kc.sb + __shfl(x.place[0], src) * a.kc.sp + 8 * g;
#pragma unroll
                for (int j = 0; j < KS; ++j) {
                    kr[h][j] = u32x4{0, 0, 0, 0};
                    if (32 * j + 8 * g < a.D) kr[h][j] = *reinterpret_cast<const u32x4*>(r + 32 * j);
                }
            }
        }
    };
    // V's rows in the order of S^T: e = 0 .. 7 are tokens 4 g + e and 16 + 4 g + (e - 4); absent ones are zeros
    auto load_v = [&](const Tile& x) {
        if constexpr (P16) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const auto r = buffer_at(vbase + x.block[h] * a.vc.sb + x.place[h] * a.vc.sp);
                if (((x.mask >> (16 * h)) & 0xFFFFu) == 0xFFFFu) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int j = 0; j < VL; ++j) vr[4 * h + e][j] = load_from<VT>(r, vofs[j] + e * vstep);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int j = 0; j < VL; ++j)
                            vr[4 * h + e][j] = load_from<VT>(r, (x.mask >> (16 * h + 4 * g + e)) & 1 ? vofs[j] + e * vstep : NOWHERE);
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int src = 16 * (e / 4) + 4 * g + e % 4;
                const uint16_t* r = vbase + __shfl(x.block[0], src) * a.vc.sb + __shfl(x.place[0], src) * a.vc.sp;
#pragma unroll
                for (int j = 0; j < VL; ++j) {
                    const int d = (EPL < 8 ? EPL : 8) * n + 128 * j;
                    vr[e][j] = VT{};
                    if (d < a.D && ((x.mask >> src) & 1)) vr[e][j] = *reinterpret_cast<const VT*>(r + d);
                }
            }
        }
    };

    const float c = a.scale * 1.4426950408889634f;  // weights are powers of two
    f32x4 acc[EPL] = {};
    float m = -INFINITY, l = 0.0f;
    int t = it.start + wave * TILE;
    if (t < it.end) {
        Tile x = locate(t);
        load_k(x);
        load_v(x);
        while (true) {
            f32x4 s0 = {}, s1 = {};
#pragma unroll
            for (int j = 0; j < KS; ++j) {
                s0 = Mma<DT>::mul(kr[0][j], q[j], s0);
                s1 = Mma<DT>::mul(kr[1][j], q[j], s1);
            }
            const int tn = t + UNIT;
            const bool more = tn < it.end;
            Tile y = x;
            if (more) {
                y = locate(tn);
                load_k(y);
            }
            float s[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[i] = s0[i] * c;
                s[4 + i] = s1[i] * c;
            }
            if (x.mask != ~0u) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (!((x.mask >> (16 * (i / 4) + 4 * g + i % 4)) & 1)) s[i] = -INFINITY;
            }
            float mt = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
            mt = fmaxf(mt, __shfl_xor(mt, 16));
            mt = fmaxf(mt, __shfl_xor(mt, 32));
            const float mn = fmaxf(m, mt), base = mn == -INFINITY ? 0.0f : mn;
            const float keep = __builtin_amdgcn_exp2f(m - base);
            m = mn;
            float w[8], sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                w[i] = __builtin_amdgcn_exp2f(s[i] - base);
                sum += w[i];
            }
            l = l * keep + sum;
            u32x4 ph, pl;
            if constexpr (WIDE) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    ph[i] = Mma<DT>::pack(w[2 * i], w[2 * i + 1]);
                    pl[i] = Mma<DT>::pack(w[2 * i] - Mma<DT>::rounded(w[2 * i]), w[2 * i + 1] - Mma<DT>::rounded(w[2 * i + 1]));
                }
            } else {
                const bool second = n & 8;
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] -= second ? Mma<DT>::rounded(w[i]) : 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) ph[i] = Mma<DT>::pack(w[2 * i], w[2 * i + 1]);
            }
            if (__ballot(keep != 1.0f)) {
#pragma unroll
                for (int j = 0; j < EPL; ++j) acc[j] *= keep;
            }
#pragma unroll
            for (int j = 0; j < EPL; ++j) {
                const int ld = j / 8, word = (j % 8) / 2;  // values j of the lane's 16 bytes, over its 8 tokens
                const uint32_t sel = j & 1 ? 0x07060302u : 0x05040100u;
                u32x4 vt;
#pragma unroll
                for (int i = 0; i < 4; ++i) vt[i] = __builtin_amdgcn_perm(vr[2 * i + 1][ld][word], vr[2 * i][ld][word], sel);
                acc[j] = Mma<DT>::mul(vt, ph, acc[j]);
                if constexpr (WIDE) acc[j] = Mma<DT>::mul(vt, pl, acc[j]);
            }
            if (!more) break;
            load_v(y);
            x = y;
            t = tn;
        }
    }

    // join of the four waves: lane (n, g) has dims of rows 4 g + i of its head: EPL (or 8 + 8) consecutive ones each
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if constexpr (!WIDE) {
#pragma unroll
        for (int j = 0; j < EPL; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[j][i] += __shfl_xor(acc[j][i], 8);
    }
    if (n < OH) {
        if (g == 0) {
            lds_m[wave][n] = m;
            lds_l[wave][n] = l;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < EPL; j += 4) {
                const int d = (EPL < 8 ? EPL : 8) * (4 * g + i) + (j / 8) * 128 + j % 8;
                *reinterpret_cast<f32x4*>(&lds_o[wave][n][d]) = f32x4{acc[j][i], acc[j + 1][i], acc[j + 2][i], acc[j + 3][i]};
            }
    }
    __syncthreads();
    const int quads = a.D / 4;
    for (int idx = threadIdx.x; idx < heads * quads; idx += THREADS) {
        const int h = idx / quads, d = (idx - h * quads) * 4;
        float mm = lds_m[0][h];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) mm = fmaxf(mm, lds_m[w][h]);
        const float base = mm == -INFINITY ? 0.0f : mm;
        float ll = 0.0f;
        f32x4 o = {};
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float f = __builtin_amdgcn_exp2f(lds_m[w][h] - base);
            ll += lds_l[w][h] * f;
            o += *reinterpret_cast<const f32x4*>(&lds_o[w][h][d]) * f;
        }
        const int head = kvh * G + h0 + h;
        if (it.chunks == 1) {
            const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
            const float v[4] = {ll == 0.0f ? 0.0f : o[0] * inv, ll == 0.0f ? 0.0f : o[1] * inv, ll == 0.0f ? 0.0f : o[2] * inv,
                                ll == 0.0f ? 0.0f : o[3] * inv};
            store4_rt(a.out.p, DT, it.b * a.out.st + head * a.out.sh + d, v, 4, true);
        } else {
            const int64_t at = ((int64_t)(it.place + it.chunk) * hg + hgi) * p.hpg + h;
            *reinterpret_cast<f32x4*>(p.part_o + at * a.D + d) = o;
            if (d == 0) {
                p.part_ml[2 * at] = mm;
                p.part_ml[2 * at + 1] = ll;
            }
        }
    }
}

// out of a split row from its chunks' (O, m, l): a workgroup takes `each` heads of one row, its groups of D / 4 threads
// the chunks in turn.
__global__ __launch_bounds__(THREADS) void paged_join_kernel(Launch p, int each) {
    __shared__ f32x4 lds_o[THREADS];
    __shared__ float lds_m[THREADS], lds_l[THREADS];
    const PagedAttentionArgs& a = p.a;
    const int2 meta = p.meta[blockIdx.x];
    if (meta.x <= 1) return;
    const int quads = a.D / 4, groups = THREADS / quads, grp = threadIdx.x / quads, dq = threadIdx.x % quads;
    const int G = a.H / a.Hk, hg = a.Hk * p.ng;
    for (int head = blockIdx.y * each; head < min(a.H, (int)(blockIdx.y + 1) * each); ++head) {
        const int kvh = head / G, in = head - kvh * G, hgi = kvh * p.ng + in / p.hpg, h = in % p.hpg;
        float m = -INFINITY, l = 0.0f;
        f32x4 o = {};
        if (grp < groups)
            for (int i = grp; i < meta.x; i += groups) {
                const int64_t at = ((int64_t)(meta.y + i) * hg + hgi) * p.hpg + h;
                const float mi = p.part_ml[2 * at], li = p.part_ml[2 * at + 1];
                const f32x4 oi = *reinterpret_cast<const f32x4*>(p.part_o + at * a.D + 4 * dq);
                const float mn = fmaxf(m, mi), base = mn == -INFINITY ? 0.0f : mn;
                const float f = __builtin_amdgcn_exp2f(m - base), fi = __builtin_amdgcn_exp2f(mi - base);
                l = l * f + li * fi;
                o = o * f + oi * fi;
                m = mn;
            }
        lds_o[threadIdx.x] = o;
        lds_m[threadIdx.x] = m;
        lds_l[threadIdx.x] = l;
        __syncthreads();
        if (threadIdx.x < quads) {
            float mm = -INFINITY;
            for (int i = 0; i < groups; ++i) mm = fmaxf(mm, lds_m[i * quads + dq]);
            const float base = mm == -INFINITY ? 0.0f : mm;
            float ll = 0.0f;
            f32x4 s = {};
            for (int i = 0; i < groups; ++i) {
                const float f = __builtin_amdgcn_exp2f(lds_m[i * quads + dq] - base);
                ll += lds_l[i * quads + dq] * f;
                s += lds_o[i * quads + dq] * f;
            }
            const float inv = 1.0f / ll;
            const float v[4] = {ll == 0.0f ? 0.0f : s[0] * inv, ll == 0.0f ? 0.0f : s[1] * inv, ll == 0.0f ? 0.0f : s[2] * inv,
                                ll == 0.0f ? 0.0f : s[3] * inv};
            store4_rt(a.out.p, a.dtype, blockIdx.x * a.out.st + head * a.out.sh + 4 * dq, v, 4, true);
        }
        __syncthreads();
    }
}

// Head groups of a kv head, and the heads of one.
void head_groups(int64_t G, int& ng, int& hpg) {
    ng = (int)((G + 15) / 16);
    hpg = (int)((G + ng - 1) / ng);
}
int64_t chunks_per_group(int64_t hg) { return std::max<int64_t>(1, TARGET / hg); }

template <int DT, int DP>
hipError_t launch(const Launch& p, bool p16, unsigned grid, hipStream_t st) {
    const bool wide = p.hpg > 8;
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(grid), dim3(THREADS), 0, st, p); };
    if (p16 && wide) go(paged_attention_kernel<DT, DP, true, true>);
    else if (p16) go(paged_attention_kernel<DT, DP, true, false>);
    else if (wide) go(paged_attention_kernel<DT, DP, false, true>);
    else go(paged_attention_kernel<DT, DP, false, false>);
    return hipGetLastError();
}

template <int DT>
hipError_t launch_dim(const Launch& p, bool p16, unsigned grid, hipStream_t st) {
    if (p.a.D <= 64) return launch<DT, 64>(p, p16, grid, st);
    if (p.a.D <= 128) return launch<DT, 128>(p, p16, grid, st);
    return launch<DT, 256>(p, p16, grid, st);
}

constexpr size_t META_BYTES = MAX_ROWS * sizeof(int2);

}  // namespace

size_t ws_paged_attention(int64_t, int64_t H, int64_t Hk, int64_t D) {
    if (Hk < 1 || H < Hk) return 0;
    int ng, hpg;
    head_groups(H / Hk, ng, hpg);
    const size_t heads = (size_t)(2 * chunks_per_group(Hk * ng) * Hk * ng) * hpg;
    return META_BYTES + heads * 8 + heads * D * 4 + 256;
}

hipError_t run_paged_attention(const PagedAttentionArgs& a, hipStream_t st) {
    Launch p;
    head_groups(a.H / a.Hk, p.ng, p.hpg);
    const int64_t hg = (int64_t)a.Hk * p.ng;
    p.per_group = (int)chunks_per_group(hg);
    // 16-token tiles whose places are reached by 32-bit offsets from a uniform address
    const auto near = [](int64_t sp) { return sp >= 0 && sp < (1 << 24); };
    const bool p16 = a.page % 16 == 0 && near(a.kc.sp) && near(a.vc.sp);
    const uint64_t d = (uint64_t)(p16 ? a.page / 16 : a.page);
    p.page_magic = d == 1 ? 0 : ~0ull / d + 1;
    const size_t heads = (size_t)(2 * p.per_group * hg) * p.hpg;
    uint8_t* ws = (uint8_t*)a.ws;
    p.meta = (int2*)ws;
    p.part_ml = (float*)(ws + META_BYTES);
    p.part_o = (float*)(ws + META_BYTES + (heads * 8 + 255) / 256 * 256);
    const int64_t rows = std::min<int64_t>(MAX_ROWS, (1 << 23) / hg);  // a grid holds 2^32 threads
    for (int64_t b0 = 0; b0 < a.B; b0 += rows) {
        p.a = a;
        p.a.B = std::min<int64_t>(rows, a.B - b0);
        p.a.q.p = (uint16_t*)a.q.p + b0 * a.q.st;
        p.a.out.p = (uint16_t*)a.out.p + b0 * a.out.st;
        p.a.table = a.table + b0 * a.ldt;
        p.a.lengths = a.lengths + b0;
        if (a.blocks == 0) p.a.W = 0;
        p.a.W = std::min<int64_t>(p.a.W, 0x7FFFFF00 / a.page);  // positions stay 32-bit
        // units a row can have at most: a row that cannot be split needs no second kernel
        int64_t most = (p.a.W * a.page + UNIT - 1) / UNIT;
        if (a.window) most = std::min<int64_t>(most, (a.window + TILE - 1 + UNIT - 1) / UNIT);
        most = std::max<int64_t>(most, 1);
        p.join = most > 1;
        const int64_t items = std::min<int64_t>(p.per_group + p.a.B, most * p.a.B);
        const unsigned grid = (unsigned)(items * hg);
        hipError_t e = a.dtype == DT_F16 ? launch_dim<DT_F16>(p, p16, grid, st) : launch_dim<DT_BF16>(p, p16, grid, st);
        if (e != hipSuccess) return e;
        if (p.join) {
            const int each = (int)std::max<int64_t>(1, std::min<int64_t>(a.H, p.a.B * a.H / 1024));
            hipLaunchKernelGGL(paged_join_kernel, dim3((unsigned)p.a.B, (unsigned)((a.H + each - 1) / each)), dim3(THREADS), 0, st,
                               p, each);
            if ((e = hipGetLastError()) != hipSuccess) return e;
        }
    }
    return hipSuccess;
}

}  // namespace qlin
