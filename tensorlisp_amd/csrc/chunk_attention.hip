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
// Items differ by orders of magnitude in keys, and only the device knows the lengths. So
// every workgroup works out the same plan from them: how many tiles a workgroup takes
// so that all run at once, and from that the partitions of every sequence's keys. The
// partitions are joined in a second launch.
#include <algorithm>

#include "paged_wave.hpp"

namespace tlh {

constexpr int CA_WAVES = 4;
constexpr int CA_NARROW = 64;      // rows of a (sequence, kv head) up to which a workgroup takes 32
constexpr int CA_MAX_PARTS = 64;   // a lane each in the merge
constexpr int CA_MIN_TILES = 2;    // 64-key tiles of a partition, at least: a round of the four waves
constexpr int CA_NO_WINDOW = 1 << 30;

struct CaArgs : PagedArgs {
    uint8_t *out;
    const uint8_t *q;
    int64_t so, sq;  // bytes from token to token
    const int32_t *lens, *starts;
    float *part;     // [slot][slot_rows][m, l, -, -, D]
    struct CaItem *list;
    int S, G, rows, max_rows, max_ctx, window, wgs, slots, slot_rows;
};

struct CaSeq {
    int b, n, L;  // first row, new tokens, tokens in the cache
};
__device__ __forceinline__ CaSeq ca_seq(const CaArgs &a, int s) {
    CaSeq q;
    q.b = max(0, min(a.starts[s], a.rows));
    const int e = max(q.b, min(a.starts[s + 1], a.rows));
    q.n = min(e - q.b, a.max_rows);
    q.L = a.num_blocks > 0 ? max(0, min(a.lens[s], a.max_ctx)) : 0;
    return q;
}

// A sequence's items a kv head and the 64-key tiles that the largest of them sees
struct CaWork {
    int items, tiles, wide;
    CaSeq q;
};
__host__ __device__ __forceinline__ int ca_tiles(int L, int G, int window, int rows) {
    const int64_t span = (int64_t)window + (rows - 1) / G + 1;  // keys that some row of a block of `rows` sees
    return L <= span ? (L + 63) / 64 : (int)((span + 63) / 64) + 1;
}
__device__ __forceinline__ CaWork ca_work(const CaArgs &a, int s) {
    CaWork w = {};
    if (s >= a.S) return w;
    const CaSeq q = w.q = ca_seq(a, s);
    const int R = q.n * a.G;
    w.wide = R > CA_NARROW;
    const int per = w.wide ? 128 : 32;
    w.items = (R + per - 1) / per;
    w.tiles = ca_tiles(q.L, a.G, a.window, per);
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
// ceil(tiles / each), at least 1 and at most CA_MAX_PARTS
__device__ __forceinline__ int ca_parts(int tiles, int each, float inv) {
    if (tiles >= (int64_t)CA_MAX_PARTS * each) return CA_MAX_PARTS;
    const int q = (int)((float)tiles * inv);  // off by at most 1
    const int r = tiles - q * each;
    return max(1, q + (r > 0) + (r > each) - (r <= -each));
}

// What a workgroup does. Every lane calls; a lane looks at one sequence of 64 at a time.
struct CaPlan {
    int s, local, parts, items, wide, slot;  // s < 0: nothing; slot: the sequence's first
    int list, lists;                         // the first of the sequence's split items, and how many there are in all
    CaSeq q;
};
__device__ __forceinline__ CaPlan ca_plan(const CaArgs &a, int block, int lane) {
    const CaWork first = ca_work(a, lane);
    auto work = [&](int g) { return g == 0 ? first : ca_work(a, g + lane); };
    // tiles of a workgroup if all had as many
    uint64_t total = 0;
    for (int g = 0; g < a.S; g += 64) {
        const CaWork w = work(g);
        const uint64_t n = (uint64_t)w.items * (uint64_t)w.tiles;  // in two parts: 64 of either fit 32 bits
        total += (uint64_t)(uint32_t)ca_sum((int)(n & 0xffffff)) + ((uint64_t)(uint32_t)ca_sum((int)(n >> 24)) << 24);
    }
    const int even = (int)min(max((total * a.KV + a.wgs - 1) / a.wgs, (uint64_t)CA_MIN_TILES), (uint64_t)1 << 26);
    // Partitions are whole, so with that many some workgroups are left over, to run alone
    // after the others: the first of a few larger numbers that leaves none. With more
    // items than workgroups none does, and the last one splits only what is much longer
    // than the others.
    constexpr int TRIES = 5;
    const int eighths[TRIES] = {8, 9, 10, 12, 16};
    int each[TRIES], count[TRIES] = {};
    float inv[TRIES];
#pragma unroll
    for (int i = 0; i < TRIES; ++i) each[i] = (even * eighths[i] + 7) / 8, inv[i] = 1.0f / (float)each[i];
    for (int g = 0; g < a.S; g += 64) {
        const CaWork w = work(g);
        const int n = (int)min((int64_t)w.items * a.KV, (int64_t)1 << 18);
#pragma unroll
        for (int i = 0; i < TRIES; ++i)
            count[i] = min(count[i] + ca_sum(min(n * ca_parts(w.tiles, each[i], inv[i]), 1 << 18)), 1 << 24);
    }
    int take = each[TRIES - 1];
    float take_inv = inv[TRIES - 1];
    bool all = false;
#pragma unroll
    for (int i = TRIES - 1; i >= 0; --i)
        if (count[i] <= a.wgs) take = each[i], take_inv = inv[i], all = true;

    CaPlan p = {};
    p.s = -1;
    int at = 0, slot = 0, list = 0;
    for (int g = 0; g < a.S; g += 64) {
        const CaWork w = work(g);
        const int parts = ca_parts(w.tiles, take, take_inv), n = w.items * a.KV;
        const int mine = n * parts, slots = parts > 1 ? mine : 0, lists = parts > 1 ? n : 0;
        const int upto = ca_scan(mine), slots_upto = ca_scan(slots), lists_upto = ca_scan(lists);
        int off = at + upto - mine;
        if (!all && a.S <= 64) {  // longest workgroups first: one that starts last would end alone
            const int key = (w.tiles + parts - 1) / parts << w.wide;
            off = 0;
            for (int j = 0; j < a.S; ++j) {
                const int kj = __builtin_amdgcn_readlane(key, j), mj = __builtin_amdgcn_readlane(mine, j);
                if (kj > key || (kj == key && j < lane)) off += mj;
            }
        }
        const uint64_t who = __builtin_amdgcn_ballot_w64(block >= off && block - off < mine);
        if (who != 0) {
            const int l = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)who) - 1);
            p.s = g + l;
            p.local = block - __builtin_amdgcn_readlane(off, l);
            p.parts = __builtin_amdgcn_readlane(parts, l);
            p.items = __builtin_amdgcn_readlane(w.items, l);
            p.wide = __builtin_amdgcn_readlane(w.wide, l);
            p.slot = slot + __builtin_amdgcn_readlane(slots_upto - slots, l);
            p.list = list + __builtin_amdgcn_readlane(lists_upto - lists, l);
            p.q.b = __builtin_amdgcn_readlane(w.q.b, l);
            p.q.n = __builtin_amdgcn_readlane(w.q.n, l);
            p.q.L = __builtin_amdgcn_readlane(w.q.L, l);
            // sequences whose rows overlap, against the documentation, may ask for more slots than there are
            if (p.parts > 1 && p.slot + p.items * a.KV * p.parts > a.slots) p.s = -1;
            if (block > 0) break;
        }
        at += __builtin_amdgcn_readlane(upto, 63);
        slot += __builtin_amdgcn_readlane(slots_upto, 63);
        list += __builtin_amdgcn_readlane(lists_upto, 63);
    }
    p.lists = list;  // (of the whole launch in workgroup 0 only)
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

// One partition of an item: rows r0 .. (of R), keys k0 .. k1 - 1, k0 a multiple of 64
struct CaJob {
    int s, hk, r0, R, k0, k1;
    bool split;
    float *slot;  // where its partial goes
};
// What the merge needs of a split item: rows first .. end - 1 of the sequence whose first
// token is `token`. (The list's entry 0 counts the others, in `first`.)
struct CaItem {
    int first, end, hk, parts, slot, token, pad[2];
};
__device__ __forceinline__ CaJob ca_job(const CaArgs &a, const CaPlan &p, int D) {
    const CaSeq &q = p.q;
    CaJob j;
    j.s = p.s;
    j.hk = p.local % a.KV;  // with 8 kv heads a head's workgroups share an XCD
    const int r = p.local / a.KV, rb = p.items - 1 - r % p.items, part = r / p.items;  // last rows first: they see the most
    const int per = p.wide ? 128 : 32;
    j.R = q.n * a.G;
    j.r0 = per * rb;
    const int last = (min(j.r0 + per, j.R) - 1) / a.G;  // tokens r0 / G .. last
    const int lo = max(0, q.L - q.n + j.r0 / a.G - a.window + 1) & ~63, hi = q.L - q.n + last + 1;
    const int tiles = hi > lo ? (hi - lo + 63) / 64 : 0;
    j.k0 = lo + 64 * (int)((int64_t)tiles * part / p.parts);
    j.k1 = min(hi, lo + 64 * (int)((int64_t)tiles * (part + 1) / p.parts));
    j.split = p.parts > 1;
    const int slot = p.slot + (rb * a.KV + j.hk) * p.parts;
    j.slot = a.part + (int64_t)(slot + part) * a.slot_rows * (D + 4);
    if (j.split && part == 0 && threadIdx.x == 0)
        a.list[1 + p.list + rb * a.KV + j.hk] = {j.r0, min(j.r0 + per, j.R), j.hk, p.parts, slot, q.b, {}};
    return j;
}
__device__ __forceinline__ CaRule ca_rule(const CaArgs &a, const CaSeq &q, int first, int last, int row) {
    const int p = q.L - q.n;
    const int at = p + row / a.G;
    return {at - a.window + 1, at, p + last / a.G - a.window + 1, p + first / a.G};
}
template <int D> __device__ __forceinline__ const uint8_t *ca_q(const CaArgs &a, const CaSeq &q, int hk, int row) {
    return a.q + (int64_t)(q.b + row / a.G) * a.sq + (int64_t)(hk * a.G + row % a.G) * D * 2;
}
template <int D> __device__ __forceinline__ uint8_t *ca_out(const CaArgs &a, const CaSeq &q, int hk, int row) {
    return a.out + (int64_t)(q.b + row / a.G) * a.so + (int64_t)(hk * a.G + row % a.G) * D * 2;
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
                                       int lane, int wave) {
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
    bool careful = false;
    for (;;) {
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
            else load_v(pg);
            const PagedSeen sees[1] = {w.seen(base, pg.good)}, &see = sees[0];
            uint4 pf[2];
            w.softmax(S, sees, pf);
            if (see.there != ~0u) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int d = 0; d < NB; ++d) vf[d][i] = w.live_v(vf[d][i], i, see.there);
            }
            if (careful && !see.whole) {
                // through the wave's part of the merge buffer, which is free until the end
                uint4 *sp = (uint4 *)merge_at(wave), *sv = sp + 128;
                static_assert(256 * 16 <= CaLds<D>::WAVE, "operands of one dim block");
                sp[lane] = pf[0], sp[64 + lane] = pf[1];
#pragma unroll
                for (int d = 0; d < NB; ++d) {
                    __builtin_amdgcn_wave_barrier();
                    sv[lane] = vf[d][0], sv[64 + lane] = vf[d][1];
                    __builtin_amdgcn_wave_barrier();
                    w.careful_pv(d, see, (const uint32_t *)sp, (const uint32_t *)sv, 256);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int d = 0; d < NB; ++d) w.O[d] = mfma32<false>(vf[d][i], pf[i], w.O[d]);
            }
            if (AHEAD) load_v(pn);
            pg = pn;
            pn = after;
        }
        if (careful || !w.some_masked || __builtin_amdgcn_ballot_w64(w.bad()) == 0) break;
        careful = true;
    }

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
            if (!j.split) {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                const float x[8] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv, 0, 0, 0, 0};
                const uint4 v = pack8<false>(x);
                *(uint2 *)(ca_out<D>(a, sq, j.hk, rr) + 2 * dim) = make_uint2(v.x, v.y);
            } else {
                float *dst = j.slot + r * (D + 4);
                *(float4 *)(dst + 4 + dim) = o;
                if (dim == 0) *(float2 *)dst = make_float2(M, sum);
            }
        }
    }
}

// -------------------------------------------------------------- many rows
template <int D, int BS>
__device__ __forceinline__ void ca_many(const CaArgs &a, const CaSeq &sq, const CaJob &j, uint8_t *T0, uint8_t *T1, uint8_t *aux,
                                        int lane, int wave) {
    using W = PagedWave<D, BS, CaRule>;
    using Sh = PagedTile<D>;
    constexpr int NS = W::NS, NB = W::NB, KT = Sh::KT, SUBS = KT / 32, KF = SUBS * NS;
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
    bool careful = false;
    auto tile = [&](int t, uint8_t *T, uint8_t *Tn) {
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
        if (gaps) {  // places that hold no token's value may hold anything: zeroed by the waves that loaded them
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
#pragma unroll
            for (int st = 0; st < NS; ++st)
                S[u] = mfma32<false>(*(const uint4 *)(T + (u * NS + st) * 1024 + 16 * lane), qf[st], S[u]);
            whole = whole && w.rule.whole(k0 + 32 * u) && good[u] == ~0u;
        }
        if (!whole) {
            w.some_masked = true;
#pragma unroll
            for (int u = 0; u < SUBS; ++u) w.hide(S[u], w.rule.sees(k0 + 32 * u) & there[u]);
        }
        uint4 pf[2 * SUBS];
        PagedSeen see[SUBS];
#pragma unroll
        for (int u = 0; u < SUBS; ++u) see[u] = {true, ~0u, ~0u};
        w.softmax(S, see, pf);
        if (careful && !whole) {
            uint4 *sp = (uint4 *)aux + 128 * wave;
#pragma unroll
            for (int u = 0; u < SUBS; ++u) {
                see[u].vis = w.rule.sees(k0 + 32 * u) & there[u];
                __builtin_amdgcn_wave_barrier();
                sp[lane] = pf[2 * u], sp[64 + lane] = pf[2 * u + 1];
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int d = 0; d < NB; ++d)
                    w.careful_pv(d, see[u], (const uint32_t *)sp, (const uint32_t *)(T + (KF + u * 2 * NB + d) * 1024), 256 * NB);
            }
            return;
        }
#pragma unroll
        for (int u = 0; u < SUBS; ++u)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int d = 0; d < NB; ++d)
                    w.O[d] = mfma32<false>(*(const uint4 *)(T + (KF + (2 * u + i) * NB + d) * 1024 + 16 * lane), pf[2 * u + i], w.O[d]);
    };
    for (;;) {
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
        for (int t = 0; t < ntiles; t += 2) {
            tile(t, T0, T1);
            if (t + 1 < ntiles) tile(t + 1, T1, T0);
        }
        if (careful) break;
        const bool again = mine && w.some_masked && __builtin_amdgcn_ballot_w64(w.bad() && r0 + c < j.R) != 0;
        if (lane == 0) s_flag[wave] = again;
        lds_barrier();  // and every wave is done with both buffers
        careful = (s_flag[0] | s_flag[1] | s_flag[2] | s_flag[3]) != 0;
        if (!careful) break;
    }
    const int rr = r0 + c;
    const float sum = sum_halves(w.l);
    if (rr >= j.R) return;
    if (j.split) {
        float *dst = j.slot + (32 * wave + c) * (D + 4);
        if (h == 0) *(float2 *)dst = make_float2(w.m, sum);
#pragma unroll
        for (int d = 0; d < NB; ++d)
#pragma unroll
            for (int x = 0; x < 4; ++x)
                if (32 * d + 8 * x < D)
                    *(float4 *)(dst + 4 + 32 * d + 8 * x + 4 * h) =
                        make_float4(w.O[d][4 * x], w.O[d][4 * x + 1], w.O[d][4 * x + 2], w.O[d][4 * x + 3]);
        return;
    }
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

template <int D, int BS>
__global__ void __launch_bounds__(64 * CA_WAVES, D <= 128 ? 2 : 1) k_chunk_attn(const CaArgs a) {
    __shared__ __attribute__((aligned(16))) uint8_t T0[CaLds<D>::HALF], T1[CaLds<D>::HALF], aux[CaLds<D>::AUX];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const CaPlan p = ca_plan(a, blockIdx.x, lane);
    if (blockIdx.x == 0 && threadIdx.x == 0 && a.slots > 0) a.list[0].first = min(p.lists, a.slots / 2);
    if (p.s < 0) return;
    const CaSeq &sq = p.q;
    const CaJob j = ca_job(a, p, D);
    if (p.wide) ca_many<D, BS>(a, sq, j, T0, T1, aux, lane, wave);
    else ca_few<D, BS>(a, sq, j, T0, T1, aux, lane, wave);
}

// Joins an item's partitions, a wave a row: lane p holds partition p's weight, the lanes
// then take the dims.
constexpr int CA_MERGE_ROWS = 8;  // of a workgroup
template <int D> __global__ void __launch_bounds__(256) k_chunk_attn_merge(const CaArgs a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int count = a.list[0].first;
    const CaItem it = a.list[1 + blockIdx.x];
    if ((int)blockIdx.x >= count) return;
    const CaSeq sq = {it.token, 0, 0};
    const int np = it.parts;
    const int64_t step = (int64_t)a.slot_rows * (D + 4);
    constexpr int E = (D + 63) / 64, AT_ONCE = 8;
    for (int r = blockIdx.y * CA_MERGE_ROWS + wave; r < (int)(blockIdx.y + 1) * CA_MERGE_ROWS; r += 4) {
        const int row = it.first + r;
        if (row >= it.end) return;
        const float *base = a.part + it.slot * step + r * (D + 4);
        // the first partitions' sums are on their way while the weights are formed
        float o[AT_ONCE][E];
        auto load = [&](int p0) {
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
                for (int e = 0; e < E; ++e)  // (past the last partition or dim: an element that gets no weight, or no place)
                    o[i][e] = base[min(p0 + i, np - 1) * step + 4 + min(lane + 64 * e, D - 1)];
        };
        float2 ml = make_float2(-INFINITY, 0.0f);
        if (lane < np) ml = *(const float2 *)(base + lane * step);
        load(0);
        float M = ml.x;
        for (int i = 1; i < 64; i <<= 1) M = fmaxf(M, __shfl_xor(M, i, 64));
        const float w = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((ml.x - M) * a.cs);
        float sum = w * ml.y;
        for (int i = 1; i < 64; i <<= 1) sum += __shfl_xor(sum, i, 64);
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        float acc[E] = {};
        for (int p0 = 0; p0 < np; p0 += AT_ONCE) {
            if (p0 > 0) load(p0);
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                if (p0 + i >= np) break;
                const float wp = __shfl(w, p0 + i, 64);
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] += wp * o[i][e];
            }
        }
        uint16_t *dst = (uint16_t *)ca_out<D>(a, sq, it.hk, row);
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (lane + 64 * e < D) dst[lane + 64 * e] = f2h(acc[e] * inv);
    }
}

// What the host knows of the plan: bounds of the items, the partitions, the workgroups
// and the slots that any lengths and starts within the arguments can lead to.
struct CaBounds {
    int64_t items, parts, wgs, slots, slot_rows, blocks;
};
static CaBounds ca_bounds(const tlh_chunk_attention_args &a) {
    CaBounds b;
    const int64_t G = a.num_heads / a.num_kv_heads, most = (int64_t)std::min(a.max_rows, a.num_rows) * G;
    // a sequence's last block of rows may be short, and 33 to 64 rows take two
    b.items = a.num_kv_heads * (std::min<int64_t>(a.num_seqs, a.num_rows) * (most > 32 ? 2 : 1) + a.num_rows * G / 128);
    b.wgs = a.head_size <= 128 ? 512 : 256;  // workgroups that fill the machine
    const int window = a.window > 0 ? std::min(a.window, CA_NO_WINDOW) : CA_NO_WINDOW;
    const int64_t tiles = ca_tiles(a.max_context_len, (int)G, window, most > CA_NARROW ? 128 : 32);
    b.parts = std::max<int64_t>(1, std::min<int64_t>(CA_MAX_PARTS, (tiles + CA_MIN_TILES - 1) / CA_MIN_TILES));
    b.slots = b.parts == 1 ? 0 : std::min(b.wgs, b.items * b.parts);
    b.slot_rows = most > CA_NARROW ? 128 : 32;
    b.blocks = b.parts == 1 ? b.items : std::min(b.items * b.parts, std::max(b.wgs, b.items + b.wgs / 2));
    return b;
}

// The list of split items (each has two slots at least), then the slots.
static int64_t ca_list_bytes(const CaBounds &b) { return b.slots == 0 ? 0 : (int64_t)sizeof(CaItem) * (1 + b.slots / 2); }
size_t chunk_attention_scratch_bytes(const tlh_chunk_attention_args &a) {
    const CaBounds b = ca_bounds(a);
    return (size_t)(ca_list_bytes(b) + b.slots * b.slot_rows * (a.head_size + 4) * (int64_t)sizeof(float));
}

template <int D> static void launch_ca(const CaArgs &c, int bs, const CaBounds &b, hipStream_t stream) {
    const dim3 grid((unsigned)b.blocks), threads(64 * CA_WAVES);
    switch (bs) {
    case 8: hipLaunchKernelGGL((k_chunk_attn<D, 8>), grid, threads, 0, stream, c); break;
    case 16: hipLaunchKernelGGL((k_chunk_attn<D, 16>), grid, threads, 0, stream, c); break;
    default: hipLaunchKernelGGL((k_chunk_attn<D, 32>), grid, threads, 0, stream, c); break;
    }
    if (b.parts > 1)
        hipLaunchKernelGGL((k_chunk_attn_merge<D>), dim3((unsigned)std::min(b.items, b.slots / 2), (unsigned)(b.slot_rows / CA_MERGE_ROWS)),
                           dim3(256), 0, stream, c);
}

tlh_status launch_chunk_attention(const tlh_chunk_attention_args &a, void *scratch, hipStream_t stream) {
    const CaBounds b = ca_bounds(a);
    CaArgs c = {};
    c.out = (uint8_t *)a.out, c.q = (const uint8_t *)a.q, c.so = 2 * a.out_stride, c.sq = 2 * a.q_stride;
    c.kc = (const uint16_t *)a.k_cache, c.vc = (const uint16_t *)a.v_cache;
    c.tables = a.block_tables, c.lens = a.context_lens, c.starts = a.row_starts;
    c.list = (CaItem *)scratch;
    c.part = (float *)((uint8_t *)scratch + ca_list_bytes(b));
    c.num_blocks = a.num_blocks;
    c.S = a.num_seqs, c.KV = a.num_kv_heads, c.G = a.num_heads / a.num_kv_heads;
    c.rows = a.num_rows, c.max_rows = a.max_rows, c.max_blocks = a.max_blocks_per_seq, c.max_ctx = a.max_context_len;
    c.window = a.window > 0 ? std::min(a.window, CA_NO_WINDOW) : CA_NO_WINDOW;
    c.wgs = (int)b.wgs, c.slots = (int)b.slots, c.slot_rows = (int)b.slot_rows;
    set_scale(c, a.scale);
    if (b.blocks >= 1 << 24)  // x 256 threads
        return set_error(TLH_INVALID, "chunk_attention: too many rows and heads for one launch");
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
