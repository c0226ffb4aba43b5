// Causal attention of the sequences' new tokens over a paged f16 cache, gfx950.
//
// Sequence s has L = context_lens[s] tokens in the cache, the last n of them new
// (n = row_starts[s + 1] - row_starts[s]), and n rows of q. Row i is the token at
// place L - n + i and sees the tokens from max(0, that - window + 1) up to itself:
//   out[i, h] = sum_j softmax_j(scale * q[i, h] . k[j, h / G]) v[j, h / G]
// A row that sees nothing gives zeros.
//
// The rows of a (sequence, kv head) are its new tokens x the group's heads; an item is
// a block of them. A sequence that decodes has a few and is bound by one read of its
// keys and values, a piece of a prompt has hundreds and is bound by the matrix cores,
// and a batch holds both. So one launch runs two forms, chosen for each sequence:
//  * up to 64 rows: a workgroup takes 32 rows, its four waves 32-key tiles in turn,
//    straight from the pages into registers, a tile ahead; the waves merge at the end;
//  * more: a workgroup takes 128 rows, 32 a wave, and the waves share 64-key tiles (32
//    above 128 dims) in LDS, double-buffered and loaded straight from the pages.
// Both compute S^T = K . Q^T and O^T += V^T . P^T, so a lane holds one row's scores.
//
// P meets V in f16, as the matrix cores take it, and a second product adds what that rounding
// took off (22 bits in all): a result is off by 2.07e-4 of its size, all of it its own rounding,
// instead of 2.9e-4. With few rows the tiles wait for HBM, and 32 sequences decoding take 113 us
// with it and without. With many the products are the bound, so there a caller may choose to do
// without (us, with it and without: 2048 over 16384 with heads of 64 513, 386; 128 826, 644; 192
// 627, 481; 256 577, 514; 31 tokens + 600 150, 144; 9 x 13..701 51.6, 47.5).
//
// Items differ by orders of magnitude in keys, and only the device knows the lengths. So
// every workgroup works out the same plan from them: how many tiles a workgroup takes
// so that all run at once, and from that the partitions of every sequence's keys (with
// more than 64 sequences a launch before does it, and they look it up; there the workgroups go
// in the order of the sequences, not longest first: 65 over 512..8192 take 226 to 239 us, 64 of
// them 212). The last of an item's partitions to arrive joins them, in the order of their keys,
// whichever it is. (Joined in a second launch, whose code has to come from memory when the keys
// have gone through the caches, 31 tokens + 600 took 20 us more.)
//
// Measured, 32/8 heads of 128 unless said, with inputs that were just used and with others each
// time: 1 token over 1500 10.3 and 13.4 us, the plan and one chain of latencies; 32 sequences
// decoding over 512..8192 113 us (4.9 TB/s over random pages); 31 of those beside a piece of 600
// tokens 150 to 162 and 198 us; 2048 over 16384 826 to 835 and 879 us, the three products at 1.0
// to 1.06 PFLOP/s, nearly a large library product's rate (1.09); nine pieces of 13..701 with 4/1
// heads of 256 and a window of 1024 52 to 53 and 56 us (one wave a SIMD).
#include <algorithm>
#include <type_traits>

#include "paged_wave.hpp"

namespace tlh {

constexpr int CA_WAVES = 4;
constexpr int CA_NARROW = 64;      // rows of a (sequence, kv head) up to which a workgroup takes 32
// A partition costs a partial written and read, and the join waits for eight of them at a
// time. So at most 32 of an item (1 token over 8000, us: 15.4 with 32, 17.5 with 42), each
// of at least 2 tiles of 64 keys, a round of the four waves, or with more than 8 rows of 8
// (4 x 16 tokens over 100..3000, us, with 3, 6, 9: 22.0, 21.5, 18.3; 1 token over 1500 with 3,
// 6, 9: 10.2, 11.0, 11.9); with more than 64 rows of an eighth of the tiles, from 4 to 8 (32
// tokens with 4, 6, 8, heads of 128: over 992 20.3, 22.5, 24.0; over 4000 35.4, 32.9, 31.3; heads
// of 256: over 992 34, 38, 41; over 2016 42, 43, 45; over 4000 57, 54, 53).
constexpr int CA_MAX_PARTS = 32, CA_MIN_TILES = 2, CA_MIN_TILES_ROWS = 8, CA_MIN_TILES_MANY = 4;
constexpr int CA_NO_WINDOW = 1 << 30;
// Sequences up to which every workgroup works out the plan; of more, one does in a launch
// before, and the others look it up.
constexpr int CA_PLAN_HERE = 64;

// n / d for 0 <= n < 2^31 by a product. What every workgroup runs before its first load is
// kept short: its code comes from memory where another kernel's was last.
struct CaDiv {
    uint32_t mul, shift, by;
    __device__ __forceinline__ int operator()(int n) const { return (int)(((uint64_t)(uint32_t)n * mul) >> shift); }
    __device__ __forceinline__ int rest(int n) const { return n - (*this)(n) * (int)by; }
};
static CaDiv ca_div(int d) {
    int s = 0;
    while ((1ll << s) < d) ++s;
    return {(uint32_t)((1ull << (31 + s)) / (uint64_t)d + 1), (uint32_t)(31 + s), (uint32_t)d};
}

struct CaArgs : PagedArgs {
    uint8_t *out;
    const uint8_t *q;
    int64_t so, sq;  // bytes from token to token
    const int32_t *lens, *starts;
    float *part;     // units of 4 rows of ca_row(D) floats
    unsigned *counters;  // of an item's partitions that have arrived; 0 before and after a call
    int4 *plan;          // of more than CA_PLAN_HERE sequences, else null
    int S, rows, max_rows, max_ctx, window;
    int lg_wgs;          // workgroups that fill the machine, a power of two
    int span_few, span_many;  // keys that some row of a block of 32 and of 128 rows sees
    int f16_weights;
    CaDiv G, kv;
};

struct CaSeq {
    int b, n, L;  // first row, new tokens (below 0: the sequence ends before it starts), tokens in the cache
};
__device__ __forceinline__ CaSeq ca_seq(const CaArgs &a, int s) {
    CaSeq q;
    q.b = max(0, min(a.starts[s], a.rows));
    q.n = min(max(0, min(a.starts[s + 1], a.rows)) - q.b, a.max_rows);
    q.L = a.num_blocks > 0 ? max(0, min(a.lens[s], a.max_ctx)) : 0;
    return q;
}

// A sequence's items a kv head and the 64-key tiles that the largest of them sees
struct CaWork {
    int items, tiles, wide, units;  // units of 4 rows of an item's partial
    CaSeq q;
};
__host__ __device__ __forceinline__ int ca_tiles(int L, int span) { return L <= span ? (L + 63) >> 6 : ((span + 63) >> 6) + 1; }
__device__ __forceinline__ CaWork ca_work(const CaArgs &a, int s) {
    CaWork w = {};
    if (s >= a.S) return w;
    const CaSeq q = w.q = ca_seq(a, s);
    const int R = max(q.n, 0) * (int)a.G.by;
    w.wide = R > CA_NARROW;
    w.items = w.wide ? (R + 127) >> 7 : (R + 31) >> 5;
    w.units = w.wide ? 32 : (min(R, 32) + 3) >> 2;
    w.tiles = ca_tiles(q.L, w.wide ? a.span_many : a.span_few);
    return w;
}

// The sum of the lanes up to each (the last lane holds that of all), within the vector
// unit: a shuffle through LDS for each of the six steps would make the plan 4 us long.
__device__ __forceinline__ int ca_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);   // the lane 1 before, in rows of 16
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);   // 2
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);   // 4
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);   // 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // rows 1 and 3: the last lane of the row before
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // rows 2 and 3: lane 31
    return v;
}
__device__ __forceinline__ int ca_sum(int v) { return __builtin_amdgcn_readlane(ca_scan(v), 63); }
// a sequence's partitions of at most `each` tiles: ceil(tiles / each), within the bounds
__device__ __forceinline__ int ca_parts(const CaWork &w, int each) {
    const int least = w.wide ? max(CA_MIN_TILES_MANY, min(w.tiles >> 3, CA_MIN_TILES_ROWS)) : w.units > 2 ? CA_MIN_TILES_ROWS : CA_MIN_TILES;
    const int n = max(each, least);
    if (w.tiles >= (int64_t)CA_MAX_PARTS * n) return CA_MAX_PARTS;
    const int q = (int)((float)w.tiles * __builtin_amdgcn_rcpf((float)n));  // off by at most 1
    const int r = w.tiles - q * n;
    return max(1, q + (r > 0) + (r > n) - (r <= -n));
}

// What a workgroup does. Every lane calls; a lane looks at one sequence.
struct CaPlan {
    int s, local, parts, items, wide, units;  // s < 0: nothing
    int unit, counter;  // the first ones of the sequence's
    CaSeq q;
};
// how many tiles one of 2^lg workgroups takes of all
__device__ __forceinline__ int ca_share(uint64_t tiles, int lg) {
    return (int)min(max((tiles + (1u << lg) - 1) >> lg, (uint64_t)CA_MIN_TILES), (uint64_t)1 << 26);
}
// Few rows: no workgroup takes more than 1.5 even shares. (us with 0.5, 1, 1.5, 2: 32
// tokens over 512..8192 120, 123, 113, 117; 8 over 8000 57, 50, 47, 45; 24 over 100..30000
// 282, 283, 267, 290; 1 over 100000 85, 85, 90, 79.)
__device__ __forceinline__ int ca_few_share(int even) { return (even * 3 + 1) >> 1; }
// Many rows: partitions are whole, so with an even share some workgroups are left over,
// to run alone after the others: the first of a few larger shares, up to twice the even
// one, that leaves none. With more items than workgroups none does, and the last one
// splits only what is much longer than the others. In eighths of the even share: 8, 9, 10, 12, 16.
__device__ __forceinline__ int ca_next_share(int eighths) { return eighths + (eighths < 10 ? 1 : eighths == 10 ? 2 : 4); }
__device__ __forceinline__ int ca_many_share(int even, int eighths) { return (even * eighths + 7) >> 3; }
// a sequence's workgroups, for that choice
__device__ __forceinline__ int ca_count(const CaArgs &a, const CaWork &w, int each) {
    return min((w.wide ? (int)min((int64_t)w.items * (int)a.kv.by, (int64_t)1 << 18) : 0) * ca_parts(w, each), 1 << 18);
}

// The plan of many sequences, by one workgroup: of each its first workgroup, unit and counter
// and its partitions, and behind them, as if of one more, the number of workgroups. (Worked
// out by every workgroup, the time grows with the square of the sequences: a token each over
// 100, us: 256 sequences 47.5, so 43; 1024 336, 155; 4096 3658, 579.)
constexpr int CA_PLANNERS = 1024;
// the sum over the workgroup; called by all
template <typename T> __device__ __forceinline__ T ca_block_sum(T v, T *s_wave) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s_wave[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < CA_PLANNERS / 64; ++w) v += s_wave[w];
    return v;
}
__global__ void __launch_bounds__(CA_PLANNERS) k_chunk_plan(const CaArgs a) {
    __shared__ uint64_t s_long[CA_PLANNERS / 64];
    __shared__ int s_upto[3][CA_PLANNERS / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, KV = (int)a.kv.by, wgs = 1 << a.lg_wgs;
    uint64_t few = 0, many = 0, bad = 0;
    for (int s = threadIdx.x; s < a.S; s += CA_PLANNERS) {
        const CaWork w = ca_work(a, s);
        bad += w.q.n < 0;
        (w.wide ? many : few) += (uint64_t)w.items * (uint32_t)w.tiles;
    }
    bad = ca_block_sum(bad, s_long), few = ca_block_sum(few, s_long), many = ca_block_sum(many, s_long);
    if (bad != 0) {  // (as in ca_plan)
        if (threadIdx.x == 0) a.plan[a.S] = make_int4(0, 0, 0, 0);
        return;
    }
    const int even = ca_share((few + many) * KV, a.lg_wgs), each_few = ca_few_share(even);
    int each_many = even;
    if (many > 0) {
        for (int eighths = 8;; eighths = ca_next_share(eighths)) {
            each_many = ca_many_share(even, eighths);
            uint64_t count = 0;
            for (int s = threadIdx.x; s < a.S; s += CA_PLANNERS) count += ca_count(a, ca_work(a, s), each_many);
            if (ca_block_sum(count, s_long) <= (uint64_t)wgs || eighths == 16) break;
        }
    }
    int at[3] = {0, 0, 0};  // workgroups, units, counters before the next 1024 sequences
    for (int s0 = 0; s0 < a.S; s0 += CA_PLANNERS) {
        const int s = s0 + (int)threadIdx.x;
        const CaWork w = ca_work(a, s);
        const int parts = ca_parts(w, w.wide ? each_many : each_few), n = w.items * KV;
        const int mine[3] = {n * parts, parts > 1 ? n * parts * w.units : 0, parts > 1 ? n : 0};
        int upto[3];
#pragma unroll
        for (int i = 0; i < 3; ++i) upto[i] = ca_scan(mine[i]);
        __syncthreads();
        if (lane == 63) {
#pragma unroll
            for (int i = 0; i < 3; ++i) s_upto[i][wave] = upto[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            upto[i] += at[i] - mine[i];
            for (int v = 0; v < CA_PLANNERS / 64; ++v) {
                if (v < wave) upto[i] += s_upto[i][v];
                at[i] += s_upto[i][v];
            }
        }
        if (s < a.S) a.plan[s] = make_int4(upto[0], upto[1], upto[2], parts);
    }
    if (threadIdx.x == 0) a.plan[a.S] = make_int4(at[0], 0, 0, 0);
}
__device__ __forceinline__ CaPlan ca_planned(const CaArgs &a, int block, int lane) {
    CaPlan p = {};
    p.s = -1;
    if (block >= __builtin_amdgcn_readfirstlane(a.plan[a.S].x)) return p;
    int lo = 0, len = a.S;  // the last sequence that begins at `block` or before it
    while (len > 1) {
        const int stride = (len + 63) >> 6, s = lo + lane * stride;
        const bool in = s < lo + len && a.plan[min(s, a.S)].x <= block;
        const int n = max(1, (int)__popcll(__builtin_amdgcn_ballot_w64(in)));
        const int next = lo + (n - 1) * stride;
        len = min(stride, lo + len - next);
        lo = next;
    }
    p.s = __builtin_amdgcn_readfirstlane(lo);
    const int4 x = a.plan[p.s];
    const CaWork w = ca_work(a, p.s);
    p.local = block - __builtin_amdgcn_readfirstlane(x.x);
    p.unit = __builtin_amdgcn_readfirstlane(x.y), p.counter = __builtin_amdgcn_readfirstlane(x.z);
    p.parts = __builtin_amdgcn_readfirstlane(x.w);
    p.items = __builtin_amdgcn_readfirstlane(w.items), p.wide = __builtin_amdgcn_readfirstlane(w.wide);
    p.units = __builtin_amdgcn_readfirstlane(w.units);
    p.q.b = __builtin_amdgcn_readfirstlane(w.q.b), p.q.n = __builtin_amdgcn_readfirstlane(w.q.n);
    p.q.L = __builtin_amdgcn_readfirstlane(w.q.L);
    return p;
}

__device__ __forceinline__ CaPlan ca_plan(const CaArgs &a, int block, int lane) {
    if (a.plan) return ca_planned(a, block, lane);
    const CaWork w = ca_work(a, lane);
    const int KV = (int)a.kv.by, wgs = 1 << a.lg_wgs;
    CaPlan p = {};
    p.s = -1;
    // Starts that decrease make sequences overlap, and more work than there is room for:
    // then nothing is computed.
    if (__builtin_amdgcn_ballot_w64(w.q.n < 0) != 0) return p;
    // tiles, of the sequences with few rows and of the others, summed in two parts: 64 of either fit 32 bits
    const uint64_t mine_all = (uint64_t)w.items * (uint32_t)w.tiles;
    const int lo = (int)(mine_all & 0xffffff), hi = (int)(mine_all >> 24);
    const uint64_t few = (uint64_t)(uint32_t)ca_sum(w.wide ? 0 : lo) + ((uint64_t)(uint32_t)ca_sum(w.wide ? 0 : hi) << 24);
    const uint64_t many = (uint64_t)(uint32_t)ca_sum(w.wide ? lo : 0) + ((uint64_t)(uint32_t)ca_sum(w.wide ? hi : 0) << 24);
    const uint64_t total = (few + many) * KV;
    const int even = ca_share(total, a.lg_wgs), each_few = ca_few_share(even);
    int each_many = even, count = 0;
    if (many > 0)
#pragma unroll 1
        for (int eighths = 8;; eighths = ca_next_share(eighths)) {
            each_many = ca_many_share(even, eighths);
            count = ca_sum(ca_count(a, w, each_many));
            if (count <= wgs || eighths == 16) break;
        }
    // all run at once: their order does not matter
    const bool all = few == 0 ? count <= wgs : total <= (uint64_t)(wgs * CA_MIN_TILES);

    const int parts = ca_parts(w, w.wide ? each_many : each_few), n = w.items * KV;
    const int mine = n * parts, units = parts > 1 ? mine * w.units : 0, counters = parts > 1 ? n : 0;
    const int units_upto = ca_scan(units), counters_upto = ca_scan(counters);
    int off = ca_scan(mine) - mine;
    if (!all) {  // longest workgroups first: one that starts last would end alone
        const int key = (int)((float)w.tiles / (float)parts) << w.wide;
        off = 0;
        for (int j = 0; j < a.S; ++j) {
            const int kj = __builtin_amdgcn_readlane(key, j), mj = __builtin_amdgcn_readlane(mine, j);
            if (kj > key || (kj == key && j < lane)) off += mj;
        }
    }
    const uint64_t who = __builtin_amdgcn_ballot_w64(block >= off && block - off < mine);
    if (who == 0) return p;
    const int l = p.s = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)who) - 1);
    p.local = block - __builtin_amdgcn_readlane(off, l);
    p.parts = __builtin_amdgcn_readlane(parts, l);
    p.items = __builtin_amdgcn_readlane(w.items, l);
    p.wide = __builtin_amdgcn_readlane(w.wide, l);
    p.units = __builtin_amdgcn_readlane(w.units, l);
    p.unit = __builtin_amdgcn_readlane(units_upto - units, l);
    p.counter = __builtin_amdgcn_readlane(counters_upto - counters, l);
    p.q.b = __builtin_amdgcn_readlane(w.q.b, l);
    p.q.n = __builtin_amdgcn_readlane(w.q.n, l);
    p.q.L = __builtin_amdgcn_readlane(w.q.L, l);
    return p;
}

// A row sees keys lo .. hi; all rows of the wave see all_lo .. all_hi.
struct CaRule {
    int lo, hi, all_lo, all_hi;
    __device__ __forceinline__ bool whole(int base) const { return base >= all_lo && base + 31 <= all_hi; }
    __device__ __forceinline__ uint32_t sees(int base) const {
        const int u = hi - base, d = lo - base;
        const uint32_t upto = u >= 31 ? ~0u : u < 0 ? 0u : (2u << u) - 1;
        return d <= 0 ? upto : d > 31 ? 0u : upto & (~0u << d);
    }
};

// Floats of a row of a partial: of few rows [m, l, -, -, D], of many the lanes' registers as
// they are (whole blocks of 32 dims), which 64 lanes write and read in one piece.
__host__ __device__ constexpr int ca_row(int D) { return (D + 31) / 32 * 32 + 4; }

// One partition of an item: rows r0 .. (of R), keys k0 .. k1 - 1, k0 a multiple of 64
struct CaJob {
    int s, hk, r0, R, k0, k1;
    int part, parts;
    float *slots;       // the item's partials, `step` floats apart
    int step;
    unsigned *counter;  // the item's
};
__device__ __forceinline__ CaJob ca_job(const CaArgs &a, const CaPlan &p, int D) {
    const CaSeq &q = p.q;
    CaJob j;
    j.s = p.s;
    const int r = a.kv(p.local);
    j.hk = p.local - r * a.KV;  // with 8 kv heads a head's workgroups share an XCD
    const int part = (uint32_t)r / (uint32_t)p.items, rb = p.items - 1 - (r - part * p.items);  // last rows first: they see the most
    const int per = p.wide ? 128 : 32;
    j.R = q.n * (int)a.G.by;
    j.r0 = per * rb;
    const int last = a.G(min(j.r0 + per, j.R) - 1);  // tokens r0 / G .. last
    const int lo = max(0, q.L - q.n + a.G(j.r0) - a.window + 1) & ~63, hi = q.L - q.n + last + 1;
    const uint32_t tiles = hi > lo ? (hi - lo + 63) >> 6 : 0, parts = p.parts;  // < 2^25, <= CA_MAX_PARTS
    j.k0 = lo + 64 * (int)(tiles * part / parts);
    j.k1 = min(hi, lo + 64 * (int)(tiles * (part + 1) / parts));
    const int item = rb * a.KV + j.hk;
    j.part = part, j.parts = p.parts;
    j.step = p.units * 4 * ca_row(D);
    j.slots = a.part + (int64_t)(p.unit + item * p.parts * p.units) * 4 * ca_row(D);
    j.counter = a.counters + p.counter + item;
    return j;
}

// Partials pass between workgroups, which may run on different XCDs: relaxed agent-scope
// stores and loads, which on gfx950 go past the XCD's L2 (no write-back or invalidation
// of all of it, which would cost the others the pages that they share).
__device__ __forceinline__ void ca_put(float *p, float x, float y) {
    __hip_atomic_store((uint64_t *)p, (uint64_t)__float_as_uint(y) << 32 | __float_as_uint(x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 ca_get(const float *p) {
    const uint64_t v = __hip_atomic_load((const uint64_t *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}
// Whether this workgroup is the last of its item's to have written its partial. That each
// wave's stores are complete (its wait) before the counter moves (behind the barrier), and
// that the loads behind it do not look in an older copy, rests on the above.
__device__ __forceinline__ bool ca_last(const CaJob &j, int *flag) {
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0) {
        const bool last = __hip_atomic_fetch_add(j.counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == (unsigned)j.parts;
        if (last) __hip_atomic_store(j.counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *flag = last;
    }
    __syncthreads();
    return *flag != 0;
}
__device__ __forceinline__ CaRule ca_rule(const CaArgs &a, const CaSeq &q, int first, int last, int row) {
    const int p = q.L - q.n;
    const int at = p + a.G(row);
    return {at - a.window + 1, at, p + a.G(last) - a.window + 1, p + a.G(first)};
}
template <int D> __device__ __forceinline__ const uint8_t *ca_q(const CaArgs &a, const CaSeq &q, int hk, int row) {
    return a.q + (int64_t)(q.b + a.G(row)) * a.sq + (int64_t)(hk * (int)a.G.by + a.G.rest(row)) * D * 2;
}
template <int D> __device__ __forceinline__ uint8_t *ca_out(const CaArgs &a, const CaSeq &q, int hk, int row) {
    return a.out + (int64_t)(q.b + a.G(row)) * a.so + (int64_t)(hk * (int)a.G.by + a.G.rest(row)) * D * 2;
}

// LDS of a workgroup, in two parts that the compiler can tell apart (a tile is loaded
// into one while the other is read)
template <int D> struct CaLds {
    static constexpr int MD = D > 32 ? 64 : 32;                  // dims merged at a time
    static constexpr int WAVE = 32 * (MD + 4) * 4;               // a wave's O in the merge
    static constexpr int HALF = std::max(PagedTile<D>::TILE, 2 * WAVE);
    static constexpr int AUX = std::max(D / 16 * 1024, CA_WAVES * 2048);  // Q, or the careful pass's P
};

// --------------------------------------------------------------- few rows
template <int D, int BS>
__device__ __forceinline__ void ca_few(const CaArgs &a, const CaSeq &sq, const CaJob &j, uint8_t *T0, uint8_t *T1, uint8_t *aux,
                                       int *flag, int lane, int wave) {
    using W = PagedWave<D, BS, CaRule>;
    constexpr int NS = W::NS, NB = W::NB, MD = CaLds<D>::MD;
    // Loads a tile ahead, where two waves' registers hold O, the keys and the values; above
    // 128 dims a tile's values are requested when its keys have been multiplied.
    constexpr bool AHEAD = D <= 128;
    __shared__ float s_m[CA_WAVES][32], s_l[CA_WAVES][32];
    uint4 *s_q = (uint4 *)aux;  // Q^T as the lanes take it: 16 bytes a lane, in order
    auto merge_at = [&](int w) { return (float *)((w & 2 ? T1 : T0) + (w & 1) * CaLds<D>::WAVE); };
    const int t0 = j.k0, ntiles = j.k1 > t0 ? (j.k1 - t0 + 31) / 32 : 0;
    const int c = lane & 31, h = lane >> 5, row = min(j.r0 + c, j.R - 1);
    W w(a, lane, j.s, j.hk, sq.L, ca_rule(a, sq, j.r0, min(j.r0 + 31, j.R - 1), row));
    {
        const uint8_t *qr = ca_q<D>(a, sq, j.hk, row) + 16 * h;
        for (int st = wave; st < NS; st += CA_WAVES) s_q[64 * st + lane] = w.signed_q(*(const uint4 *)(qr + 32 * st));
    }
    uint4 kf[NS], vf[NB][2];
    auto load_k = [&](const typename W::Pages &p) {
        const uint8_t *kp = w.k_at(p);
#pragma unroll
        for (int st = 0; st < NS; ++st) kf[st] = *(const uint4 *)(kp + W::k_step(st));
    };
    auto load_v = [&](const typename W::Pages &p) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint8_t *vp = w.v_at(p, i);
#pragma unroll
            for (int d = 0; d < NB; ++d) vf[d][i] = *(const uint4 *)(vp + w.v_step(d));
        }
    };
    __syncthreads();
    // (a loop for each kind of pass: in one, the rare kind's registers spill the other's above 128 dims)
    auto pass = [&](auto careful) {
        w.reset();
        typename W::Pages pg = {}, pn = {};
        if (wave < ntiles) {
            pg = w.checked(w.ids_of(t0 + 32 * wave));
            pn = w.ids_of(t0 + 32 * (wave + CA_WAVES));
            if (AHEAD) {
                load_k(pg);
                load_v(pg);
            }
        }
        for (int k = wave; k < ntiles; k += CA_WAVES) {
            const int base = t0 + 32 * k;
            pn = w.checked(pn);
            const typename W::Pages after = w.ids_of(base + 64 * CA_WAVES);
            if (!AHEAD) load_k(pg);
            f32x16 S[1] = {(f32x16){}};
#pragma unroll
            for (int st = 0; st < NS; ++st) S[0] = mfma32<false>(kf[st], s_q[64 * st + lane], S[0]);
            if (AHEAD) load_k(pn);  // past the last tile: the last page again
            else {
                __builtin_amdgcn_sched_barrier(0);  // into the keys' registers
                load_v(pg);
            }
            const PagedSeen sees[1] = {w.seen(base, pg.good)}, &see = sees[0];
            uint4 pf[2], rest[2];
            w.template softmax<true>(S, sees, pf, rest);
            if (see.there != ~0u) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int d = 0; d < NB; ++d) vf[d][i] = w.live_v(vf[d][i], i, see.there);
            }
            if (careful() && !see.whole) {
                // through the wave's part of the merge buffer, which is free until the end
                uint4 *sp = (uint4 *)merge_at(wave), *sv = sp + 128;
                static_assert(192 * 16 <= CaLds<D>::WAVE, "operands of 16 keys and a dim block");
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int d = 0; d < NB; ++d) {
                        __builtin_amdgcn_wave_barrier();
                        sp[lane] = pf[i], sp[64 + lane] = rest[i], sv[lane] = vf[d][i];
                        __builtin_amdgcn_wave_barrier();
                        w.careful_rest_pv(d, see, i, (const uint32_t *)sp, (const uint32_t *)sv);
                    }
            } else {
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int d = 0; d < NB; ++d) {
                        w.O[d] = mfma32<false>(vf[d][i], pf[i], w.O[d]);
                        w.O[d] = mfma32<false>(careful() ? W::finite_v(vf[d][i]) : vf[d][i], rest[i], w.O[d]);
                    }
            }
            if (AHEAD) load_v(pn);
            pg = pn;
            pn = after;
        }
    };
    pass(std::false_type());
    if (__builtin_amdgcn_ballot_w64(w.bad()) != 0) pass(std::true_type());

    // merge the waves, MD dims at a time
    const float lt = sum_halves(w.l);
    if (h == 0) s_m[wave][c] = w.m, s_l[wave][c] = lt;
#pragma unroll
    for (int d0 = 0; d0 < NB; d0 += MD / 32) {
        if (d0 > 0) lds_barrier();  // the last part has been read
        float *mine = merge_at(wave);
#pragma unroll
        for (int d = d0; d < d0 + MD / 32 && d < NB; ++d)
#pragma unroll
            for (int x = 0; x < 4; ++x)
                *(float4 *)&mine[c * (MD + 4) + 32 * (d - d0) + 8 * x + 4 * h] =
                    make_float4(w.O[d][4 * x], w.O[d][4 * x + 1], w.O[d][4 * x + 2], w.O[d][4 * x + 3]);
        lds_barrier();
        for (int e = threadIdx.x; e < 32 * (MD / 4); e += 64 * CA_WAVES) {
            const int r = e / (MD / 4), dd = 4 * (e % (MD / 4)), dim = 32 * d0 + dd, rr = j.r0 + r;
            if (rr >= j.R || dim >= D) continue;
            float M = -INFINITY;
#pragma unroll
            for (int x = 0; x < CA_WAVES; ++x) M = fmaxf(M, s_m[x][r]);
            float sum = 0.0f;
            float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int x = 0; x < CA_WAVES; ++x) {
                const float mw = s_m[x][r];
                const float f = mw == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((mw - M) * a.cs);
                const float4 v = *(const float4 *)&merge_at(x)[r * (MD + 4) + dd];
                if (mw == -INFINITY && !(s_l[x][r] != 0.0f)) continue;  // saw nothing
                sum += f * s_l[x][r];
                o.x += f * v.x, o.y += f * v.y, o.z += f * v.z, o.w += f * v.w;
            }
            if (j.parts == 1) {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                const float x[8] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv, 0, 0, 0, 0};
                const uint4 v = pack8<false>(x);
                *(uint2 *)(ca_out<D>(a, sq, j.hk, rr) + 2 * dim) = make_uint2(v.x, v.y);
            } else {
                float *dst = j.slots + j.part * j.step + r * ca_row(D);
                ca_put(dst + 4 + dim, o.x, o.y), ca_put(dst + 6 + dim, o.z, o.w);
                if (dim == 0) ca_put(dst, M, sum);
            }
        }
    }
    if (j.parts == 1 || !ca_last(j, flag)) return;
    // a thread takes four dims of a row
#pragma unroll 1
    for (int e = threadIdx.x; e < min(32, j.R - j.r0) * (D / 4); e += 64 * CA_WAVES) {
        const int r = e / (D / 4), dim = 4 * (e % (D / 4));
        const float *src = j.slots + r * ca_row(D);
        float M = -INFINITY, sum = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        constexpr int AT_ONCE = 8;
#pragma unroll 1
        for (int p0 = 0; p0 < j.parts; p0 += AT_ONCE) {
            float2 ml[AT_ONCE], lo[AT_ONCE], hi[AT_ONCE];
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                const float *x = src + min(p0 + i, j.parts - 1) * j.step;
                ml[i] = ca_get(x), lo[i] = ca_get(x + 4 + dim), hi[i] = ca_get(x + 6 + dim);
            }
            float top = M;
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) top = fmaxf(top, ml[i].x);
            const float f = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((M - top) * a.cs);
            M = top;
            sum *= f, o.x *= f, o.y *= f, o.z *= f, o.w *= f;
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                if (p0 + i >= j.parts) break;
                if (ml[i].x == -INFINITY && !(ml[i].y != 0.0f)) continue;  // saw nothing
                const float w = ml[i].x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((ml[i].x - M) * a.cs);
                sum += w * ml[i].y;
                o.x += w * lo[i].x, o.y += w * lo[i].y, o.z += w * hi[i].x, o.w += w * hi[i].y;
            }
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        const float x[8] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv, 0, 0, 0, 0};
        const uint4 v = pack8<false>(x);
        *(uint2 *)(ca_out<D>(a, sq, j.hk, j.r0 + r) + 2 * dim) = make_uint2(v.x, v.y);
    }
}

// -------------------------------------------------------------- many rows
// use(f, fragment f) for N 1-KiB fragments in LDS, read BATCH at a time and a batch
// ahead of their use: left to itself the compiler reads each right before its product.
template <int N, int BATCH, typename Use> __device__ __forceinline__ void ca_stream(const uint8_t *at, Use use) {
    uint4 f[2][BATCH];
    auto read = [&](int b) {
#pragma unroll
        for (int i = 0; i < BATCH; ++i)
            if (BATCH * b + i < N) f[b & 1][i] = *(const uint4 *)(at + (BATCH * b + i) * 1024);
    };
    read(0);
#pragma unroll
    for (int b = 0; BATCH * b < N; ++b) {
        read(b + 1);
        __builtin_amdgcn_sched_barrier(0x6);  // vector and scalar arithmetic may pass, reads and products not
#pragma unroll
        for (int i = 0; i < BATCH; ++i)
            if (BATCH * b + i < N) use(BATCH * b + i, f[b & 1][i]);
        __builtin_amdgcn_sched_barrier(0x6);
    }
}

template <int D, int BS>
__device__ __forceinline__ void ca_many(const CaArgs &a, const CaSeq &sq, const CaJob &j, uint8_t *T0, uint8_t *T1, uint8_t *aux,
                                        int *flag, int lane, int wave) {
    using W = PagedWave<D, BS, CaRule>;
    using Sh = PagedTile<D>;
    constexpr int NS = W::NS, NB = W::NB, KT = Sh::KT, SUBS = KT / 32, KF = SUBS * NS;
    // At 192 dims a batch of four leaves O and Q four registers too few, and reading those back
    // from memory waits for the next tile's loads, which are before it in line (2048 over 16384,
    // 16/4 heads, f16_weights, with four and two: 737, 485 us).
    constexpr int BATCH = D == 192 ? 2 : 4;
    __shared__ int s_flag[CA_WAVES];
    const int c = lane & 31, h = lane >> 5;
    const int r0 = j.r0 + 32 * wave, row = min(r0 + c, j.R - 1);
    const int ntiles = j.k1 > j.k0 ? (j.k1 - j.k0 + KT - 1) / KT : 0;
    const bool mine = r0 < j.R;  // some wave of the workgroup has rows, this one may not
    const int last = min(r0 + 31, j.R - 1);
    W w(a, lane, j.s, j.hk, sq.L, ca_rule(a, sq, min(r0, last), last, row));
    const int any_lo = w.rule.all_hi - a.window + 1, any_hi = w.rule.all_lo + a.window - 1;  // keys that some row sees
    typename W::Pages pg[SUBS], pn[SUBS];  // of the tile in turn and the next one
    auto ids = [&](int t, typename W::Pages (&p)[SUBS]) {
#pragma unroll
        for (int u = 0; u < SUBS; ++u) p[u] = w.ids_of(j.k0 + KT * t + 32 * u);
    };
    // wave w loads the fragments w, w + 4, ... of K and of V
    auto load_tile = [&](const typename W::Pages *p, uint8_t *T) {
#pragma unroll
        for (int u = 0; u < SUBS; ++u) {
            const uint8_t *kp = w.k_at(p[u]);
#pragma unroll
            for (int x = 0; x < (NS + CA_WAVES - 1) / CA_WAVES; ++x) {
                const int st = CA_WAVES * x + wave;
                if (NS % CA_WAVES == 0 || st < NS) to_lds(kp + W::k_step(st), T + (u * NS + st) * 1024);
            }
#pragma unroll
            for (int x = 0; x < (2 * NB + CA_WAVES - 1) / CA_WAVES; ++x) {
                const int f = CA_WAVES * x + wave, i = f & 1, d = f >> 1;
                if (2 * NB % CA_WAVES == 0 || f < 2 * NB)
                    to_lds(w.v_at(p[u], i) + w.v_step(d), T + (KF + (2 * u + i) * NB + d) * 1024);
            }
        }
    };
    uint4 qf[NS];
    {
        const uint8_t *qr = ca_q<D>(a, sq, j.hk, row) + 16 * h;
#pragma unroll
        for (int st = 0; st < NS; ++st) qf[st] = w.signed_q(*(const uint4 *)(qr + 32 * st));
    }
    auto tile = [&](auto careful, auto rests, int t, uint8_t *T, uint8_t *Tn) {
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): tile t has landed
        lds_barrier();                       // for every wave, and the other buffer is free
        const int k0 = j.k0 + KT * t;
        uint32_t good[SUBS], there[SUBS];
        bool gaps = false;
#pragma unroll
        for (int u = 0; u < SUBS; ++u) {
            good[u] = pg[u].good;
            there[u] = w.there(k0 + 32 * u, good[u]);
            gaps = gaps || there[u] != ~0u;
        }
        if (t + 1 < ntiles) {
#pragma unroll
            for (int u = 0; u < SUBS; ++u) pg[u] = w.checked(pn[u]);
            load_tile(pg, Tn);
            ids(t + 2, pn);
        }
        // Places that hold no token's value may hold anything: zeroed, by whichever wave, since behind
        // the barrier above every wave's loads of this tile have landed.
        if (gaps) {
#pragma unroll 1
            for (int f = wave; f < 2 * SUBS * NB; f += CA_WAVES) {
                uint4 *v = (uint4 *)(T + (KF + f) * 1024) + lane;
                const int i = f / NB;
                *v = w.live_v(*v, i & 1, SUBS == 1 || i < 2 ? there[0] : there[SUBS - 1]);
            }
            lds_barrier();
        }
        if (!mine || k0 > any_hi || k0 + KT - 1 < any_lo) return;  // nothing visible to the wave's rows
        f32x16 S[SUBS];
        bool whole = true;
#pragma unroll
        for (int u = 0; u < SUBS; ++u) {
            S[u] = (f32x16){};
            whole = whole && w.rule.whole(k0 + 32 * u) && good[u] == ~0u;
        }
        ca_stream<KF, BATCH>(T + 16 * lane, [&](int f, uint4 k) { S[f / NS] = mfma32<false>(k, qf[f % NS], S[f / NS]); });
        if (!whole) {
            int k = k0;
            asm volatile("" : "+s"(k));  // the masks formed here, not before every tile
#pragma unroll
            for (int u = 0; u < SUBS; ++u) w.hide(S[u], w.rule.sees(k + 32 * u) & there[u]);
        }
        uint4 pf[2 * SUBS], rest[2 * SUBS];
        PagedSeen see[SUBS];
#pragma unroll
        for (int u = 0; u < SUBS; ++u) see[u] = {true, ~0u, ~0u};
        w.template softmax<rests()>(S, see, pf, rest);
        if (careful() && !whole) {
            uint4 *sp = (uint4 *)aux + 128 * wave;
#pragma unroll
            for (int u = 0; u < SUBS; ++u) {
                see[u].vis = w.rule.sees(k0 + 32 * u) & there[u];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    __builtin_amdgcn_wave_barrier();
                    sp[lane] = pf[2 * u + i], sp[64 + lane] = rest[2 * u + i];
                    __builtin_amdgcn_wave_barrier();
#pragma unroll
                    for (int d = 0; d < NB; ++d)
                        w.careful_rest_pv(d, see[u], i, (const uint32_t *)sp, (const uint32_t *)(T + (KF + (2 * u + i) * NB + d) * 1024));
                }
            }
            return;
        }
        ca_stream<2 * SUBS * NB, BATCH>(T + KF * 1024 + 16 * lane, [&](int f, uint4 v) {
            w.O[f % NB] = mfma32<false>(v, pf[f / NB], w.O[f % NB]);
            if (rests()) w.O[f % NB] = mfma32<false>(careful() ? W::finite_v(v) : v, rest[f / NB], w.O[f % NB]);
        });
    };
    auto begin = [&] {
        w.reset();
        if (ntiles > 0) {
            int first = 0;
            asm volatile("" : "+s"(first));  // its addresses formed here: kept for another pass, they spill
            ids(first, pg);
            ids(1, pn);
#pragma unroll
            for (int u = 0; u < SUBS; ++u) pg[u] = w.checked(pg[u]);
            load_tile(pg, T0);
        }
    };
    begin();
    auto all = [&](auto rests) {
        for (int t = 0; t < ntiles; t += 2) {
            tile(std::false_type(), rests, t, T0, T1);
            if (t + 1 < ntiles) tile(std::false_type(), rests, t + 1, T1, T0);
        }
    };
    if (a.f16_weights) all(std::false_type());
    else all(std::true_type());
    const bool again = mine && __builtin_amdgcn_ballot_w64(w.bad() && r0 + c < j.R) != 0;
    if (lane == 0) s_flag[wave] = again;
    lds_barrier();  // and every wave is done with both buffers
    if ((s_flag[0] | s_flag[1] | s_flag[2] | s_flag[3]) != 0) {
        // (a loop of its own: with both kinds of tile in one, every tile moved O to other registers)
        begin();
#pragma unroll 1
        for (int t = 0; t < ntiles; ++t) tile(std::true_type(), std::true_type(), t, t & 1 ? T1 : T0, t & 1 ? T0 : T1);
    }
    const int rr = r0 + c;
    float sum = sum_halves(w.l);
    if (j.parts > 1) {
        // register pair x of lane l at 64 x + l, m and the sum behind the last
        const int at = 32 * wave * ca_row(D) + 2 * lane;
        float *dst = j.slots + j.part * j.step + at;
#pragma unroll
        for (int d = 0; d < NB; ++d)
#pragma unroll
            for (int x = 0; x < 8; ++x) ca_put(dst + 128 * (8 * d + x), w.O[d][2 * x], w.O[d][2 * x + 1]);
        ca_put(dst + 128 * 8 * NB, w.m, sum);
        static_assert(128 * (8 * NB + 1) <= 32 * ca_row(D), "a wave's registers");
        if (!ca_last(j, flag)) return;
        const float *src = j.slots + at;
        float M = -INFINITY;
#pragma unroll 4
        for (int p = 0; p < j.parts; ++p) M = fmaxf(M, ca_get(src + p * j.step + 128 * 8 * NB).x);
        f32x16 O[NB];
#pragma unroll
        for (int d = 0; d < NB; ++d) O[d] = (f32x16){};
        float all = 0.0f;
#pragma unroll 1
        for (int p = 0; p < j.parts; ++p) {
            const float *from = src + p * j.step;
            const float2 ml = ca_get(from + 128 * 8 * NB);
            const bool none = ml.x == -INFINITY && !(ml.y != 0.0f);  // saw nothing
            const float f = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((ml.x - M) * a.cs);
            all += none ? 0.0f : f * ml.y;
#pragma unroll
            for (int d = 0; d < NB; ++d) {
                float2 v[8];
#pragma unroll
                for (int x = 0; x < 8; ++x) v[x] = ca_get(from + 128 * (8 * d + x));
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    O[d][2 * x] += none ? 0.0f : f * v[x].x;
                    O[d][2 * x + 1] += none ? 0.0f : f * v[x].y;
                }
            }
        }
        sum = all;
#pragma unroll
        for (int d = 0; d < NB; ++d) w.O[d] = O[d];
    }
    if (rr >= j.R) return;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    uint8_t *dst = ca_out<D>(a, sq, j.hk, rr) + 8 * h;
#pragma unroll
    for (int d = 0; d < NB; ++d)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            if (32 * d + 8 * x >= D) continue;
            const float v[8] = {w.O[d][4 * x] * inv, w.O[d][4 * x + 1] * inv, w.O[d][4 * x + 2] * inv, w.O[d][4 * x + 3] * inv,
                                0, 0, 0, 0};
            const uint4 p = pack8<false>(v);
            *(uint2 *)(dst + 64 * d + 16 * x) = make_uint2(p.x, p.y);
        }
}

// Two workgroups a CU up to 192 dims (there with spills, around the loops over tiles and in those
// of the careful pass: heads of 192, 16/4, f16_weights, with one and two, us: 2048 over 16384 861,
// 485; nine pieces of 13..701 behind up to 5000 256, 182; 32 decoding over 512..8192 110, 91; 8 x
// 12 tokens over 2000 34, 32). Pages of 8 keep a tile's page ids in memory of the lane's own, in
// the loops too: 2048 over 16384, heads of 128, 893 us where pages of 16 take 826; 32 decoding 151
// and 113. (Three workgroups a CU at 64 dims gained 4% of 2048 over 16384 and lost 16% of it with
// f16_weights.)
template <int D, int BS>
__global__ void __launch_bounds__(64 * CA_WAVES, D <= 192 ? 2 : 1) k_chunk_attn(const CaArgs a) {
    __shared__ __attribute__((aligned(16))) uint8_t T0[CaLds<D>::HALF], T1[CaLds<D>::HALF], aux[CaLds<D>::AUX];
    __shared__ int flag;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const CaPlan p = ca_plan(a, blockIdx.x, lane);
    if (p.s < 0) return;
    const CaSeq &sq = p.q;
    const CaJob j = ca_job(a, p, D);
    if (p.wide) ca_many<D, BS>(a, sq, j, T0, T1, aux, &flag, lane, wave);
    else ca_few<D, BS>(a, sq, j, T0, T1, aux, &flag, lane, wave);
}

// What the host knows of the plan: bounds of the items, the partitions, the workgroups and
// the partials that any lengths and starts within the arguments can lead to.
// Of each kind of sequence: a share of t tiles makes a split sequence's partitions fewer
// than 2 / t of its tiles, and the shares are 1.5 / wgs of all tiles or more (few rows), and
// 2 / wgs or more if more than wgs partitions would come of less (many rows).
struct CaBounds {
    int64_t items, parts, wgs, units, blocks;
    int span_few, span_many;
};
static CaBounds ca_bounds(const tlh_chunk_attention_args &a) {
    CaBounds b;
    const int64_t G = a.num_heads / a.num_kv_heads, most = (int64_t)std::min(a.max_rows, a.num_rows) * G;
    const bool wide = most > CA_NARROW;
    // a sequence's last block of rows may be short, and 33 to 64 rows take two
    b.items = a.num_kv_heads * (std::min<int64_t>(a.num_seqs, a.num_rows) * (most > 32 ? 2 : 1) + a.num_rows * G / 128);
    b.wgs = a.head_size <= 192 ? 512 : 256;  // workgroups that fill the machine
    const int window = a.window > 0 ? std::min(a.window, CA_NO_WINDOW) : CA_NO_WINDOW;
    b.span_few = window + 31 / (int)G + 1, b.span_many = window + 127 / (int)G + 1;
    // (a context just past what a block sees may count a tile more than one just within; a call
    // that may hold many rows may hold few)
    const int64_t tiles = std::max(ca_tiles(a.max_context_len, b.span_few), wide ? ca_tiles(a.max_context_len, b.span_many) : 0);
    b.parts = std::max<int64_t>(1, std::min<int64_t>(CA_MAX_PARTS, (tiles + CA_MIN_TILES - 1) / CA_MIN_TILES));
    const int64_t few = (std::min<int64_t>(most, 32) + 3) / 4, many = wide ? 32 : 0;
    b.units = b.parts == 1 ? 0 : std::min(2 * b.wgs * few + b.wgs * many, b.items * b.parts * std::max(few, many));
    b.blocks = b.parts == 1 ? b.items : std::min(b.items * b.parts, 2 * b.wgs + b.items);
    return b;
}

// The counters, always in the same place and as many as any call may need (a split item has
// two partitions at least), then the plan of many sequences and the partials.
static_assert(TLH_CHUNK_COUNTER_BYTES >= 4 * (512 + 512 / 2), "split items");
static size_t ca_plan_bytes(const tlh_chunk_attention_args &a) {
    return a.num_seqs > CA_PLAN_HERE ? sizeof(int4) * ((size_t)a.num_seqs + 1) : 0;
}
size_t chunk_attention_scratch_bytes(const tlh_chunk_attention_args &a) {
    const CaBounds b = ca_bounds(a);
    const size_t plan = ca_plan_bytes(a);
    return b.parts == 1 && plan == 0 ? 0 : TLH_CHUNK_COUNTER_BYTES + plan + (size_t)b.units * 4 * ca_row(a.head_size) * sizeof(float);
}

template <int D> static void launch_ca(const CaArgs &c, int bs, const CaBounds &b, hipStream_t stream) {
    const dim3 grid((unsigned)b.blocks), threads(64 * CA_WAVES);
    switch (bs) {
    case 8: hipLaunchKernelGGL((k_chunk_attn<D, 8>), grid, threads, 0, stream, c); break;
    case 16: hipLaunchKernelGGL((k_chunk_attn<D, 16>), grid, threads, 0, stream, c); break;
    default: hipLaunchKernelGGL((k_chunk_attn<D, 32>), grid, threads, 0, stream, c); break;
    }
}

tlh_status launch_chunk_attention(const tlh_chunk_attention_args &a, void *scratch, hipStream_t stream) {
    const CaBounds b = ca_bounds(a);
    CaArgs c = {};
    c.out = (uint8_t *)a.out, c.q = (const uint8_t *)a.q, c.so = 2 * a.out_stride, c.sq = 2 * a.q_stride;
    c.kc = (const uint16_t *)a.k_cache, c.vc = (const uint16_t *)a.v_cache;
    c.tables = a.block_tables, c.lens = a.context_lens, c.starts = a.row_starts;
    c.counters = (unsigned *)scratch;
    c.part = (float *)((uint8_t *)scratch + TLH_CHUNK_COUNTER_BYTES + ca_plan_bytes(a));
    c.plan = a.num_seqs > CA_PLAN_HERE ? (int4 *)((uint8_t *)scratch + TLH_CHUNK_COUNTER_BYTES) : nullptr;
    c.num_blocks = a.num_blocks;
    c.S = a.num_seqs, c.KV = a.num_kv_heads, c.kv = ca_div(a.num_kv_heads), c.G = ca_div(a.num_heads / a.num_kv_heads);
    c.rows = a.num_rows, c.max_rows = a.max_rows, c.max_blocks = a.max_blocks_per_seq, c.max_ctx = a.max_context_len;
    c.window = a.window > 0 ? std::min(a.window, CA_NO_WINDOW) : CA_NO_WINDOW;
    c.lg_wgs = b.wgs == 512 ? 9 : 8, c.span_few = b.span_few, c.span_many = b.span_many;
    c.f16_weights = a.f16_weights;
    set_scale(c, a.scale);
    if (b.blocks >= 1 << 24)  // x 256 threads
        return set_error(TLH_INVALID, "chunk_attention: too many rows and heads for one launch");
    if (c.plan) hipLaunchKernelGGL(k_chunk_plan, dim3(1), dim3(CA_PLANNERS), 0, stream, c);
    switch (a.head_size) {
    case 64: launch_ca<64>(c, a.block_size, b, stream); break;
    case 80: launch_ca<80>(c, a.block_size, b, stream); break;
    case 96: launch_ca<96>(c, a.block_size, b, stream); break;
    case 112: launch_ca<112>(c, a.block_size, b, stream); break;
    case 128: launch_ca<128>(c, a.block_size, b, stream); break;
    case 192: launch_ca<192>(c, a.block_size, b, stream); break;
    default: launch_ca<256>(c, a.block_size, b, stream); break;
    }
    return check_launch("chunk_attention");
}

}  // namespace tlh
