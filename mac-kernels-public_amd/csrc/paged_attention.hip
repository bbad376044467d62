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
// The weights p enter the second product as two 16-bit parts (p cut off, and what is left of it), or a row's
// output would carry their rounding on top of its own.  Up to 8 heads the second part rides in the 8 columns that the
// heads leave free; 9 to 16 heads take a second instruction.  The second part is never negative, and at least the type's
// least: an infinite value gives its infinity with both parts (0 times it would be a NaN).  fp16 has no exponents below
// 2^-24, and weights that far below a row's largest add up over a long row: there p is 2^15 exp(s - m), the second part 2^11
// times what is left, and the parts' sums are kept apart until the end, so that a weight keeps 16 bits down to 2^-35 of the
// largest and counts down to 2^-50.  O and l have the factor alike.
//
// Work split: a row's tokens count in units of 128 (4 waves x 32), all rows' units are laid end to end and every
// workgroup takes an equal run of them, as many workgroups as the chip holds at once.  So one long row among short ones
// is spread like the rest, and the host need not know the lengths: every workgroup forms the running sum from them.
// A row that crosses from one workgroup's run into the next leaves its parts as (O, m, l) in fp32, and a second
// kernel joins them.  Where the table has no room for rows longer than whole_rows(), a workgroup takes one row, whatever the
// others have.
//
// Measured on one MI355X (calls back to back, inputs that are not in the caches, bytes of the cache over the whole call):
// 1 row of 131071 tokens, 40 heads over 8 of 128 values 89 us, 6.0 TB/s; 64 rows of 100 to 16384, 32 over 8 141 us, 6.1 TB/s;
// 8 rows of 3000 to 4096 29.0 us, 4.0 TB/s, of which the first loads take some 5 us and the second kernel with its launch 6;
// 1 row of 77 5.6 us.  Tried and slower: more workgroups than the chip holds, a join by the last workgroup (its agent fences
// write back and drop the L2: 105 us for the 8 rows), 3 waves a SIMD (spills), the next row's loads before this row's join, loads
// without branches around them (the waits are exact then; 3% faster for 64 values, 2 to 5% slower for 128).
#include "attention.h"

namespace qlin {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr int THREADS = 256, WAVES = 4, TILE = 32, UNIT = WAVES * TILE;
constexpr int MAX_ROWS = 1024;       // rows of one launch (their lengths are summed by every workgroup)
constexpr int CUS = 256;
constexpr int MOST_GROUPS = 4 * CUS;  // of any head size: see held()

// Workgroups of the kernel for this head size that the chip holds at once (registers: 4, 2 and 1 on a compute unit; 3 of
// small heads in groups of 9 to 16, `wide`: 8 rows of 8000 to 16384 tokens, 64 over 4 heads of 64 values 26.8 us so, 29.8 with 4).
int64_t held(int64_t D, bool wide) { return CUS * (D <= 64 ? wide ? 3 : 4 : D <= 128 ? 2 : 1); }

// Units up to which rows are not split: a workgroup takes one whole row, without the running sum and the second kernel.
// Where that fills the chip rows may be longer.  Measured on equal rows that are not in the caches, not split / split (us, 32
// over 8 heads; 1 unit = 128 tokens): D = 128, 1 row of 2 units 8.2 / 11.5, of 4 12.3 / 11.9, of 6 15.9 / 12.1; 64 rows of 4
// 27.6 / 30.0, of 8 49.1 / 51.7, of 16 93.1 / 96.0, of 24 137 / 140; D = 64, 8 rows of 4 10.9 / 11.7, of 8 17.2 / 13.2; 64 rows of 16
// 52.5 / 61.7, of 32 100 / 114; D = 256, 8 rows of 2 12.9 / 15.3, of 4 18.7 / 17.0; 64 rows of 8 88.1 / 89.0, of 16 165 / 166.
// The host knows the table's room alone, and unequal rows lose by it: D = 128, one row of 1024 tokens among 63 of 60 20.2 /
// 18.4, of 2048 34.5 / 19.2.
int64_t whole_rows(int64_t D, int64_t workgroups) {
    return workgroups >= 2 * CUS ? std::min<int64_t>(16, 2048 / D) : D <= 128 ? 4 : 2;
}

// Whether whole rows of at most `longest` tokens take a wave each instead of a workgroup of four: many rows that leave some
// of four waves without a tile.  Measured as above, one wave / four (us, 8 kv heads of 128 values): 200 rows of 30 tokens 8.9 /
// 19.5, of 60 13.8 / 21.4, of 120 22.6 / 28.7, of 250 40.7 / 46.0, of 500 76.2 / 80.6; 64 rows of 60 7.9 / 8.0, of 120 12.4 / 10.6,
// of 250 20.7 / 16.0; of 256 values, 64 rows of 120 19.2 / 21.7, of 250 29.7 / 31.3; of 64, 300 rows of 60 11.7 / 16.0.
bool one_wave_rows(int64_t D, int64_t longest, int64_t workgroups) {
    return longest <= 512 && 2 * workgroups >= held(D, false) * (longest <= 64 ? 2 : longest <= 128 ? 3 : 6);
}

struct Launch {
    PagedAttentionArgs a;
    int ng;                 // head groups of a kv head
    int hpg;                // heads of a group (the last one may have fewer)
    int shares;             // workgroups of a head group
    uint64_t page_magic;    // floor(2^64 / d) + 1 for d = page / 16 or page; 0 for d = 1
    float* part_o;          // [share, first or last row][kv head, group][head][D]
    float* part_ml;         // [share, first or last row][kv head, group][head][2]
    int4* meta;             // [rows]: the first share, shares, whether the row is not the first of its first share
    bool split;             // shares of equal runs, joined; else a workgroup takes one row
};

// What no kernel writes while this one runs is read through the scalar cache: its loads do not queue with
// those of keys and values.
typedef const __attribute__((address_space(4))) int32_t* ScalarInts;

// The weights' parts, in pairs.  RAISE: the largest weight is 2^RAISE.  LOW: factor of a weight's second part.
template <int DT> struct Mma;
template <> struct Mma<DT_F16> {
    static constexpr float RAISE = 15.0f, LOW = 2048.0f, LEAST = 0x1p-24f;
    static __device__ __forceinline__ f32x4 mul(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t first(float a, float b) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
    }
    static __device__ __forceinline__ uint32_t second(float a, float b, uint32_t of) {
        const f16x2 h = __builtin_bit_cast(f16x2, of);
        return first(__builtin_fmaf(a - (float)h[0], LOW, LEAST), __builtin_fmaf(b - (float)h[1], LOW, LEAST));
    }
};
template <> struct Mma<DT_BF16> {
    static constexpr float RAISE = 0.0f, LOW = 1.0f, LEAST = 0x1p-126f;
    static __device__ __forceinline__ f32x4 mul(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t first(float a, float b) {
        return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
    }
    static __device__ __forceinline__ uint32_t second(float a, float b, uint32_t of) {
        const bf16x2 h = {(__bf16)(a - __uint_as_float(of << 16) + LEAST), (__bf16)(b - __uint_as_float(of & 0xFFFF0000u) + LEAST)};
        return __builtin_bit_cast(uint32_t, h);
    }
};

// n / d for the d of `magic` (any 32-bit n and d).
__device__ __forceinline__ uint32_t divided(uint32_t n, uint64_t magic) {
    if (magic == 0) return n;
    const uint64_t lo = (uint64_t)n * (uint32_t)magic, hi = (uint64_t)n * (uint32_t)(magic >> 32);
    return (uint32_t)((hi + (lo >> 32)) >> 32);
}

// The range of row b's tokens that count, LAST at most: positions of a whole tile behind it stay 32-bit.
constexpr int64_t LAST = 0x7FFFFF00;
__device__ __forceinline__ void range_of(const PagedAttentionArgs& a, int length, int& lo, int& hi) {
    const int64_t n = min((int64_t)max(length, 0), min(a.W * a.page, LAST));
    hi = (int)n;
    lo = a.window && n > a.window ? (int)(n - a.window) : 0;
}
// Units of a row; one, of no token, for an empty row.
__device__ __forceinline__ int units_of(const PagedAttentionArgs& a, int length) {
    int lo, hi;
    range_of(a, length, lo, hi);
    return max(1, (hi - (lo & ~(TILE - 1)) + UNIT - 1) / UNIT);
}

// A workgroup's run of units, [unit, end) in the running sum; the row of its first one, which starts at `first`.
struct Share {
    int b, first, unit, end, per;
    int length;   // up to 64 rows: lane b has row b's length
};

// Running sum over a wave, this lane's own value included.
__device__ __forceinline__ int scan(int a, int lane) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const int x = __shfl_up(a, m);
        if (lane >= m) a += x;
    }
    return a;
}

__device__ __forceinline__ bool set_share(const Launch& p, int w, int total, Share& s) {
    s.per = (total + p.shares - 1) / p.shares;
    s.unit = w * s.per;
    s.end = min(s.unit + s.per, total);
    return s.unit < total;
}

// The share of this number; false past the last.  Up to 64 rows every wave forms the sums for itself, a row a lane,
// without a barrier.
__device__ __forceinline__ bool find_share_wave(const Launch& p, int w, Share& s) {
    const int lane = threadIdx.x & 63;
    s.length = lane < p.a.B ? p.a.lengths[lane] : 0;
    const int units = lane < p.a.B ? units_of(p.a, s.length) : 0;
    const int sum = scan(units, lane);
    if (!set_share(p, w, __builtin_amdgcn_readlane(sum, 63), s)) return false;
    const uint64_t here = __ballot(s.unit < sum && s.unit >= sum - units);
    s.b = __ffsll((unsigned long long)here) - 1;
    s.first = __builtin_amdgcn_readlane(sum, s.b) - __builtin_amdgcn_readlane(units, s.b);
    return true;
}

// The same for up to MAX_ROWS rows, over the workgroup.
__device__ bool find_share(const Launch& p, int w, Share& s) {
    __shared__ int sums[WAVES], found[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int rows = (int)p.a.B, each = (rows + THREADS - 1) / THREADS;
    int units[MAX_ROWS / THREADS], mine = 0;
#pragma unroll
    for (int i = 0; i < MAX_ROWS / THREADS; ++i) {
        const int b = tid * each + i;
        units[i] = i < each && b < rows ? units_of(p.a, p.a.lengths[b]) : 0;
        mine += units[i];
    }
    const int sum = scan(mine, lane);
    if (lane == 63) sums[wave] = sum;
    __syncthreads();
    int total = 0, at = sum - mine;
    for (int v = 0; v < WAVES; ++v) {
        at += v < wave ? sums[v] : 0;
        total += sums[v];
    }
    if (!set_share(p, w, total, s)) return false;
#pragma unroll
    for (int i = 0; i < MAX_ROWS / THREADS; ++i) {
        if (s.unit >= at && s.unit < at + units[i]) {
            found[0] = tid * each + i;
            found[1] = at;
        }
        at += units[i];
    }
    __syncthreads();
    s.b = __builtin_amdgcn_readfirstlane(found[0]);
    s.first = __builtin_amdgcn_readfirstlane(found[1]);
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

// Cache policy of a load: V's rows are read whole by one instruction and never again, so they are not kept (nontemporal); K's
// come 64 bytes at a time, and the other half of their lines has to stay until the next instruction.  Measured, none /
// V / K / both nontemporal (us): 8 rows of 3000 to 4096 32.2 / 28.7 / 30.6 / 32.5, 1 of 131071 100 / 89.9 / 93.4 / 90.7,
// 64 of 100 to 16384 157 / 142 / 147 / 143, 8 of 4000 to 9000 of 64 values 34.0 / 30.9 / 33.2 / 35.9.
constexpr int KEPT = 0, READ_ONCE = 2;

template <typename V, int POLICY>
__device__ __forceinline__ V load_from(__amdgpu_buffer_rsrc_t r, uint32_t offset) {
    if constexpr (sizeof(V) == 16) return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b128(r, offset, 0, POLICY));
    else return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b64(r, offset, 0, POLICY));
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
// W: waves of a workgroup, 4, or 1 for many short rows (not split).
template <int DT, int DP, bool P16, bool WIDE, int W>
__global__ __launch_bounds__(64 * W, DP == 256 ? 1 : 2) void paged_attention_kernel(Launch p) {
    static_assert(W == WAVES || W == 1, "rows are split in units of 4 waves' tiles");
    constexpr int STEP = W * TILE;
    const bool split = W == WAVES && p.split;
    constexpr int KS = DP / 32;              // 32-value steps of a score
    constexpr int EPL = DP / 16;             // values of a V row that a lane holds
    constexpr int VL = EPL > 8 ? 2 : 1;      // loads they take
    using VT = typename std::conditional<EPL == 4, u32x2, u32x4>::type;
    constexpr int OS = DP + 4;               // row stride of the join in LDS
    constexpr int OH = WIDE ? 16 : 8;
    constexpr bool APART = WIDE && Mma<DT>::LOW != 1.0f;  // the second parts have sums of their own
    __shared__ float lds_o[W][OH][OS];
    __shared__ float lds_m[W][16], lds_l[W][16];
    const PagedAttentionArgs& a = p.a;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;  // column (a head) and row group
    const int hg = a.Hk * p.ng, hgi = blockIdx.x % hg, share = blockIdx.x / hg;
    Share sh;
    if (!split) {
        sh = Share{share, 0, 0, 1, 1, 0};
    } else if constexpr (W == WAVES) {
        if (a.B <= 64 ? !find_share_wave(p, share, sh) : !find_share(p, share, sh)) return;
    }
    const int kvh = hgi / p.ng, G = a.H / a.Hk, h0 = (hgi % p.ng) * p.hpg, heads = min(p.hpg, G - h0);
    const uint16_t* kbase = (const uint16_t*)a.kc.p + kvh * a.kc.sh;
    const uint16_t* vbase = (const uint16_t*)a.vc.p + kvh * a.vc.sh;

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
    int lo = 0, hi = 0;                  // the row's tokens that count
    int64_t row = 0;                     // the row's entries in the table
    // A tile's table entries: P16 the two halves'; else lane t & 31 has token t's.  Read a tile ahead of their use.
    struct Entries {
        int block[2];
    };
    auto entries = [&](int t) {
        Entries x;
        if constexpr (P16) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                x.block[h] = ((ScalarInts)a.table)[row + min((int64_t)divided((uint32_t)t / 16 + h, p.page_magic), a.W - 1)];
        } else {
            x.block[0] = a.table[row + min((int64_t)divided((uint32_t)t + (lane & 31), p.page_magic), a.W - 1)];
        }
        return x;
    };
    // Its places in the cache: block and first place in it, tokens that are there.
    struct Tile {
        int block[2], place[2];
        uint32_t mask;
    };
    auto locate = [&](int t, const Entries& from) {
        Tile x;
        x.mask = bits_in(t, lo, hi);
        if constexpr (P16) {
            const uint32_t per_page = (uint32_t)(a.page >> 4);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t s = (uint32_t)t / 16 + h;
                x.place[h] = (int)(s - divided(s, p.page_magic) * per_page) * 16;
                x.block[h] = from.block[h];
                if (!((x.mask >> (16 * h)) & 0xFFFFu) || (uint32_t)x.block[h] >= (uint32_t)a.blocks) {
                    x.block[h] = 0;
                    x.place[h] = 0;
                    x.mask &= h ? 0x0000FFFFu : 0xFFFF0000u;
                }
            }
        } else {
            const int tok = lane & 31;
            const uint32_t s = (uint32_t)t + tok;
            const bool ok = ((x.mask >> tok) & 1) && (uint32_t)from.block[0] < (uint32_t)a.blocks;
            x.block[0] = ok ? from.block[0] : 0;
            x.place[0] = ok ? (int)(s - divided(s, p.page_magic) * (uint32_t)a.page) : 0;
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
                for (int j = 0; j < KS; ++j) kr[h][j] = load_from<u32x4, KEPT>(r, kofs[j]);
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
                        for (int j = 0; j < VL; ++j) vr[4 * h + e][j] = load_from<VT, READ_ONCE>(r, vofs[j] + e * vstep);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int j = 0; j < VL; ++j)
                            vr[4 * h + e][j] = load_from<VT, READ_ONCE>(r, (x.mask >> (16 * h + 4 * g + e)) & 1 ? vofs[j] + e * vstep : NOWHERE);
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
                    if (d < a.D && ((x.mask >> src) & 1)) vr[e][j] = __builtin_nontemporal_load(reinterpret_cast<const VT*>(r + d));
                }
            }
        }
    };

    const float c = a.scale * 1.4426950408889634f;  // weights are powers of two
    for (; sh.unit < sh.end; ++sh.b) {
        const int length = split && a.B <= 64 ? __builtin_amdgcn_readlane(sh.length, sh.b) : ((ScalarInts)a.lengths)[sh.b];
        range_of(a, length, lo, hi);
        row = sh.b * a.ldt;
        const int units = split ? units_of(a, length) : 1, last = min(sh.end, sh.first + units);
        const int start = (lo & ~(TILE - 1)) + (sh.unit - sh.first) * UNIT;
        const int end = split ? (int)min((int64_t)start + (int64_t)(last - sh.unit) * UNIT, (int64_t)hi) : hi;
        const int share0 = sh.first / sh.per, shares = (sh.first + units - 1) / sh.per - share0 + 1;
        if (split && hgi == 0 && sh.unit == sh.first && threadIdx.x == 0)
            p.meta[sh.b] = make_int4(share0, shares, sh.first != share0 * sh.per, 0);

        // Q^T: column n is a head; up to 8 heads the columns 8 .. 15 repeat them for the weights' second part
        const int col = WIDE ? n : n & 7;
        u32x4 q[KS];
#pragma unroll
        for (int j = 0; j < KS; ++j) {
            q[j] = u32x4{0, 0, 0, 0};
            if (col < heads && 32 * j + 8 * g < a.D)
                q[j] = *reinterpret_cast<const u32x4*>((const uint16_t*)a.q.p + sh.b * a.q.st +
                                                       (int64_t)(kvh * G + h0 + col) * a.q.sh + 32 * j + 8 * g);
        }
        f32x4 acc[EPL] = {}, low[APART ? EPL : 1] = {};
        float m = -INFINITY, l = 0.0f;
        int t = start + wave * TILE;
        if (t < end) {
            Tile x = locate(t, entries(t));
            Entries ahead = entries(t + STEP);
            load_k(x);
            load_v(x);
            while (true) {
                f32x4 s0 = {}, s1 = {};
#pragma unroll
                for (int j = 0; j < KS; ++j) {
                    s0 = Mma<DT>::mul(kr[0][j], q[j], s0);
                    s1 = Mma<DT>::mul(kr[1][j], q[j], s1);
                }
                const int tn = t + STEP;
                const bool more = tn < end;
                Tile y = x;
                if (more) {
                    y = locate(tn, ahead);
                    ahead = entries(tn + STEP);
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
                    w[i] = s[i] - base;
                    if constexpr (Mma<DT>::RAISE != 0.0f) w[i] += Mma<DT>::RAISE;
                    w[i] = __builtin_amdgcn_exp2f(w[i]);
                    sum += w[i];
                }
                l = l * keep + sum;
                u32x4 ph, pl;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    ph[i] = Mma<DT>::first(w[2 * i], w[2 * i + 1]);
                    pl[i] = Mma<DT>::second(w[2 * i], w[2 * i + 1], ph[i]);
                    if (!WIDE && (n & 8)) ph[i] = pl[i];
                }
                if (__ballot(keep != 1.0f)) {
#pragma unroll
                    for (int j = 0; j < EPL; ++j) {
                        acc[j] *= keep;
                        if constexpr (APART) low[j] *= keep;
                    }
                }
#pragma unroll
                for (int j = 0; j < EPL; ++j) {
                    const int ld = j / 8, word = (j % 8) / 2;  // values j of the lane's 16 bytes, over its 8 tokens
                    const uint32_t sel = j & 1 ? 0x07060302u : 0x05040100u;
                    u32x4 vt;
#pragma unroll
                    for (int i = 0; i < 4; ++i) vt[i] = __builtin_amdgcn_perm(vr[2 * i + 1][ld][word], vr[2 * i][ld][word], sel);
                    acc[j] = Mma<DT>::mul(vt, ph, acc[j]);
                    if constexpr (APART) low[j] = Mma<DT>::mul(vt, pl, low[j]);
                    else if constexpr (WIDE) acc[j] = Mma<DT>::mul(vt, pl, acc[j]);
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
        if constexpr (!WIDE || APART) {
#pragma unroll
            for (int j = 0; j < EPL; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    acc[j][i] = __builtin_fmaf(APART ? low[APART ? j : 0][i] : __shfl_xor(acc[j][i], 8), 1.0f / Mma<DT>::LOW, acc[j][i]);
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
        for (int idx = threadIdx.x; idx < heads * quads; idx += 64 * W) {
            const int h = idx / quads, d = (idx - h * quads) * 4;
            float mm = lds_m[0][h];
#pragma unroll
            for (int w = 1; w < W; ++w) mm = fmaxf(mm, lds_m[w][h]);
            const float base = mm == -INFINITY ? 0.0f : mm;
            float ll = 0.0f;
            f32x4 o = {};
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const float f = __builtin_amdgcn_exp2f(lds_m[w][h] - base);
                ll += lds_l[w][h] * f;
                o += *reinterpret_cast<const f32x4*>(&lds_o[w][h][d]) * f;
            }
            const int head = kvh * G + h0 + h;
            if (shares == 1) {
                const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
                const float v[4] = {ll == 0.0f ? 0.0f : o[0] * inv, ll == 0.0f ? 0.0f : o[1] * inv, ll == 0.0f ? 0.0f : o[2] * inv,
                                    ll == 0.0f ? 0.0f : o[3] * inv};
                store4_rt(a.out.p, DT, sh.b * a.out.st + head * a.out.sh + d, v, 4, true);
            } else {
                // of one share only the first and the last row can be split
                const int place = 2 * share + (sh.unit != share * sh.per);
                const int64_t at = ((int64_t)place * hg + hgi) * p.hpg + h;
                *reinterpret_cast<f32x4*>(p.part_o + at * a.D + d) = o;
                if (d == 0) {
                    p.part_ml[2 * at] = mm;
                    p.part_ml[2 * at + 1] = ll;
                }
            }
        }
        __syncthreads();
        sh.unit = last;
        sh.first += units;
    }
}

// out of a split row from its parts' (O, m, l): a workgroup a (row, head), groups of D / 4 threads over the parts, JOIN
// parts a group in flight; the first of them are on their way while the weights are formed.  One wave where there
// are many (row, head)s, which have few parts each, else four: 64 rows x 32 heads 8.1 us with four waves, 4.9 with one;
// 1 x 40 with 64 parts each 5.3 with four, some 3 us more with one.
constexpr int JOIN = 8;
template <int N>
__global__ __launch_bounds__(N) void paged_join_kernel(Launch p) {
    __shared__ f32x4 lds_o[N];
    __shared__ float lds_w[MOST_GROUPS];
    const PagedAttentionArgs& a = p.a;
    const int b = blockIdx.x, head = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    const int4 meta = p.meta[b];
    const int parts = meta.y;
    if (parts <= 1) return;
    const int quads = a.D / 4, groups = N / quads, grp = tid / quads, dq = tid % quads;
    const int G = a.H / a.Hk, hg = a.Hk * p.ng, kvh = head / G, in = head - kvh * G, hgi = kvh * p.ng + in / p.hpg;
    // the row's part in share i: the share's first, but for the row that starts within its first share
    const int64_t one = (int64_t)hg * p.hpg, from = (int64_t)hgi * p.hpg + in % p.hpg;
    const auto place = [&](int i) { return (2 * (meta.x + i) + (i == 0 ? meta.z : 0)) * one + from; };
    const float* part = p.part_o + 4 * dq;
    f32x4 x[JOIN];
    const auto fetch = [&](int i) {
#pragma unroll
        for (int u = 0; u < JOIN; ++u) {
            x[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if (grp < groups && i + u * groups < parts) x[u] = *reinterpret_cast<const f32x4*>(part + place(i + u * groups) * a.D);
        }
    };
    fetch(grp);
    float m = -INFINITY, l = 0.0f;  // every wave forms them for itself
    for (int i = lane; i < parts; i += 64) m = fmaxf(m, p.part_ml[2 * place(i)]);
    m = wave_max(m);
    const float base = m == -INFINITY ? 0.0f : m;
    for (int i = lane; i < parts; i += 64) {
        const float w = __builtin_amdgcn_exp2f(p.part_ml[2 * place(i)] - base);
        if (tid < 64) lds_w[i] = w;
        l += w * p.part_ml[2 * place(i) + 1];
    }
    l = wave_sum(l);
    __syncthreads();
    f32x4 o = {};
    for (int i = grp; i < parts; i += JOIN * groups) {
        if (i != grp) fetch(i);
#pragma unroll
        for (int u = 0; u < JOIN; ++u)
            if (i + u * groups < parts) o += x[u] * lds_w[i + u * groups];
    }
    lds_o[tid] = o;
    __syncthreads();
    if (tid < quads) {
        for (int i = 1; i < groups; ++i) o += lds_o[i * quads + tid];
        const float inv = 1.0f / l;
        const float v[4] = {l == 0.0f ? 0.0f : o[0] * inv, l == 0.0f ? 0.0f : o[1] * inv, l == 0.0f ? 0.0f : o[2] * inv,
                            l == 0.0f ? 0.0f : o[3] * inv};
        store4_rt(a.out.p, a.dtype, b * a.out.st + head * a.out.sh + 4 * tid, v, 4, true);
    }
}

// Head groups of a kv head, and the heads of one.
void head_groups(int64_t G, int& ng, int& hpg) {
    ng = (int)((G + 15) / 16);
    hpg = (int)((G + ng - 1) / ng);
}
int64_t shares_of(int64_t hg, int64_t hpg, int64_t D) { return std::max<int64_t>(1, held(D, hpg > 8) / hg); }

template <int DT, int DP>
hipError_t launch(const Launch& p, bool p16, bool one_wave, unsigned grid, hipStream_t st) {
    const bool wide = p.hpg > 8;
    auto go = [&](auto kernel, int threads) { hipLaunchKernelGGL(kernel, dim3(grid), dim3(threads), 0, st, p); };
    if (one_wave && wide) go(paged_attention_kernel<DT, DP, true, true, 1>, 64);
    else if (one_wave) go(paged_attention_kernel<DT, DP, true, false, 1>, 64);
    else if (p16 && wide) go(paged_attention_kernel<DT, DP, true, true, WAVES>, THREADS);
    else if (p16) go(paged_attention_kernel<DT, DP, true, false, WAVES>, THREADS);
    else if (wide) go(paged_attention_kernel<DT, DP, false, true, WAVES>, THREADS);
    else go(paged_attention_kernel<DT, DP, false, false, WAVES>, THREADS);
    return hipGetLastError();
}

template <int DT>
hipError_t launch_dim(const Launch& p, bool p16, bool one_wave, unsigned grid, hipStream_t st) {
    if (p.a.D <= 64) return launch<DT, 64>(p, p16, one_wave, grid, st);
    if (p.a.D <= 128) return launch<DT, 128>(p, p16, one_wave, grid, st);
    return launch<DT, 256>(p, p16, one_wave, grid, st);
}

constexpr size_t META_BYTES = MAX_ROWS * sizeof(int4);

}  // namespace

size_t ws_paged_attention(int64_t, int64_t H, int64_t Hk, int64_t D) {
    if (Hk < 1 || H < Hk) return 0;
    int ng, hpg;
    head_groups(H / Hk, ng, hpg);
    const size_t heads = (size_t)(2 * shares_of(Hk * ng, hpg, D) * Hk * ng) * hpg;
    return META_BYTES + heads * 8 + heads * D * 4 + 256;
}

hipError_t run_paged_attention(const PagedAttentionArgs& a, hipStream_t st) {
    Launch p;
    head_groups(a.H / a.Hk, p.ng, p.hpg);
    const int64_t hg = (int64_t)a.Hk * p.ng;
    p.shares = (int)shares_of(hg, p.hpg, a.D);
    // 16-token tiles whose places are reached by 32-bit offsets from a uniform address
    const auto near = [](int64_t sp) { return sp >= 0 && sp < (1 << 24); };
    const bool p16 = a.page % 16 == 0 && near(a.kc.sp) && near(a.vc.sp);
    const uint64_t d = (uint64_t)(p16 ? a.page / 16 : a.page);
    p.page_magic = d == 1 ? 0 : ~0ull / d + 1;
    const size_t heads = (size_t)(2 * p.shares * hg) * p.hpg;
    uint8_t* ws = (uint8_t*)a.ws;
    p.meta = (int4*)ws;
    p.part_ml = (float*)(ws + META_BYTES);
    p.part_o = (float*)(ws + META_BYTES + (heads * 8 + 255) / 256 * 256);
    const int64_t W = a.blocks == 0 ? 0 : std::min<int64_t>(a.W, (LAST + a.page - 1) / a.page), room = std::min(W * a.page, LAST);
    // units a row can have at most
    int64_t most = (room + UNIT - 1) / UNIT;
    if (a.window) most = std::min<int64_t>(most, a.window / UNIT + 2);
    most = std::max<int64_t>(most, 1);
    const int64_t longest = a.window ? std::min<int64_t>(room, std::min(a.window, room) + TILE) : room;
    // of one launch: sums of units stay 32-bit, and a workgroup a row and head group below the 2^32 threads of a launch
    const int64_t rows = std::min<int64_t>({MAX_ROWS, (1 << 30) / most, 0xFFFFFFFFll / THREADS / hg});
    for (int64_t b0 = 0; b0 < a.B; b0 += rows) {
        p.a = a;
        p.a.W = W;
        p.a.B = std::min<int64_t>(rows, a.B - b0);
        p.a.q.p = (uint16_t*)a.q.p + b0 * a.q.st;
        p.a.out.p = (uint16_t*)a.out.p + b0 * a.out.st;
        p.a.table = a.table + b0 * a.ldt;
        p.a.lengths = a.lengths + b0;
        p.split = most > whole_rows(a.D, p.a.B * hg);
        const unsigned grid = (unsigned)((p.split ? std::min<int64_t>(p.shares, most * p.a.B) : p.a.B) * hg);
        const bool one_wave = p16 && !p.split && one_wave_rows(a.D, longest, p.a.B * hg);
        hipError_t e = a.dtype == DT_F16 ? launch_dim<DT_F16>(p, p16, one_wave, grid, st) : launch_dim<DT_BF16>(p, p16, one_wave, grid, st);
        if (e != hipSuccess) return e;
        if (p.split) {
            const dim3 each((unsigned)p.a.B, (unsigned)a.H);
            if (p.a.B * a.H > 2 * CUS) hipLaunchKernelGGL(paged_join_kernel<64>, each, dim3(64), 0, st, p);
            else hipLaunchKernelGGL(paged_join_kernel<256>, each, dim3(256), 0, st, p);
            if ((e = hipGetLastError()) != hipSuccess) return e;
        }
    }
    return hipSuccess;
}

}  // namespace qlin
