// What the attentions over a paged f16 cache share: a wave's 32 rows of one (sequence,
// kv head), whose keys and values it takes from the pages as they are,
//   key   [blocks][kv_heads][D/8][block_size][8]
//   value [blocks][kv_heads][D][block_size]
// A `Rule` says what the rows see: whole(base) whether all of them see the 32 keys at
// `base`, sees(base) the bits of those that this lane's row sees.
#pragma once

#include "mfma32.hpp"

namespace tlh {

struct PagedArgs {
    const uint16_t *kc, *vc;
    const int32_t *tables;
    int64_t num_blocks;
    int KV, max_blocks;
    float cs;             // |scale| * log2(e); 1 where the scale is 0
    float lift;           // how far below the maximum the exponents' reference is set, in scores
    uint32_t qand, qxor;  // q's words: negated where the scale is negative, zeroed where it is 0
};
inline void set_scale(PagedArgs &a, float scale) {
    a.cs = scale == 0.0f ? 1.0f : fabsf(scale) * 1.4426950408889634f;
    a.lift = f16_lift(a.cs);
    a.qand = scale == 0.0f ? 0u : ~0u, a.qxor = scale < 0.0f ? 0x80008000u : 0u;
}

struct PagedSeen {
    bool whole;      // every row sees every key of the tile
    uint32_t there;  // keys that are in the cache
    uint32_t vis;    // keys that this lane's row sees
};

template <int D, int BS, class Rule> struct PagedWave {
    static constexpr int NS = D / 16, NB = (D + 31) / 32, PAGES = 32 / BS;
    const PagedArgs &a;
    const int lane, h, c;
    const int32_t *table;
    const uint32_t page_bytes;  // at most 65535 x 256 x 32 x 2
    const uint8_t *kbase, *vbase;
    const int kappa;  // the key of S^T's row c: bits 2 and 3 of c exchanged
    const int L;  // tokens in the cache
    Rule rule;

    __device__ __forceinline__ PagedWave(const PagedArgs &a_, int lane_, int s, int hk, int L_, const Rule &rule_)
        : a(a_), lane(lane_), h(lane_ >> 5), c(lane_ & 31), table(a_.tables + (int64_t)s * a_.max_blocks),
          page_bytes((uint32_t)a_.KV * D * BS * 2), kbase((const uint8_t *)a_.kc + (int64_t)hk * D * BS * 2),
          vbase((const uint8_t *)a_.vc + (int64_t)hk * D * BS * 2),
          kappa((c & 0x13) | (c & 4) << 1 | (c & 8) >> 1), L(L_), rule(rule_) {}

    // The pages of the tile at key `base` (past the context its last one again). Their
    // ids are read ahead of their use, so that no tile waits for the table; one
    // outside the pools is taken as page 0, its keys as not there.
    struct Pages {
        int id[PAGES];
        uint32_t good;  // bits of the tile's keys whose page is inside
    };
    __device__ __forceinline__ Pages ids_of(int base) const {
        Pages p = {};
#pragma unroll
        for (int i = 0; i < PAGES; ++i)
            p.id[i] = table[__builtin_amdgcn_readfirstlane(min(base / BS + i, (L - 1) / BS))];
        return p;
    }
    __device__ __forceinline__ Pages checked(Pages p) const {
        p.good = 0;
#pragma unroll
        for (int i = 0; i < PAGES; ++i) {
            const bool ok = p.id[i] >= 0 && p.id[i] < a.num_blocks;
            p.id[i] = ok ? p.id[i] : 0;
            p.good |= ok ? (BS == 32 ? ~0u : ((1u << (BS & 31)) - 1) << (BS * i)) : 0u;
        }
        return p;
    }
    __device__ __forceinline__ int64_t page_at(const Pages &p, int key) const {  // of key `key` of the tile
        int id = p.id[0];
#pragma unroll
        for (int i = 1; i < PAGES; ++i) id = key / BS == i ? p.id[i] : id;
        return (int64_t)((uint64_t)(uint32_t)id * page_bytes);
    }
    // this lane's 16 bytes of the keys' step st are k_at() + k_step(st), of the values'
    // keys 16 i + 8 h .. + 7 and dims 32 d .. + 31 v_at(i) + v_step(d)
    __device__ __forceinline__ const uint8_t *k_at(const Pages &p) const {
        return kbase + page_at(p, kappa) + h * BS * 16 + (kappa % BS) * 16;
    }
    static __device__ __forceinline__ int k_step(int st) { return st * BS * 32; }
    __device__ __forceinline__ const uint8_t *v_at(const Pages &p, int i) const {
        const int key = 16 * i + 8 * h;
        return vbase + page_at(p, key) + (key % BS) * 2 + c * BS * 2;
    }
    __device__ __forceinline__ int v_step(int d) const {  // dims past the last repeat it
        return (32 * d + 31 < D ? 32 * d : min(32 * d + c, D - 1) - c) * BS * 2;
    }

    __device__ __forceinline__ uint4 signed_q(uint4 w) const {
        return make_uint4((w.x & a.qand) ^ a.qxor, (w.y & a.qand) ^ a.qxor, (w.z & a.qand) ^ a.qxor, (w.w & a.qand) ^ a.qxor);
    }

    f32x16 O[NB];
    float m, l;  // the exponents' reference (an unscaled score), this half's sum
    // A value that is not finite would turn the zero weight of a key that a row does
    // not see into NaN, and an infinite one the rest of a weight. So where a wave's sums come
    // out not finite, it takes its tiles again, carefully: in those with masked keys it adds
    // each seen key's product by itself, in the others rests meet finite values only.
    bool some_masked = false;
    __device__ __forceinline__ void reset() {
#pragma unroll
        for (int d = 0; d < NB; ++d) O[d] = (f32x16){};
        m = -INFINITY;
        l = 0.0f;
    }
    __device__ __forceinline__ bool bad() const {
        bool x = false;
#pragma unroll
        for (int d = 0; d < NB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) x = x || !(fabsf(O[d][i]) < INFINITY);
        return x;
    }

    // which of the 32 keys at `base` are in the cache
    __device__ __forceinline__ uint32_t there(int base, uint32_t good) const {
        return L <= base ? 0u : good & (L - base >= 32 ? ~0u : (1u << (L - base)) - 1);
    }
    // what the wave's rows see of them
    __device__ __forceinline__ PagedSeen seen(int base, uint32_t good) {
        PagedSeen s = {rule.whole(base) && good == ~0u, ~0u, ~0u};
        if (!s.whole) {
            some_masked = true;
            s.there = there(base, good);
            s.vis = rule.sees(base) & s.there;
        }
        return s;
    }
    __device__ __forceinline__ void hide(f32x16 &S, uint32_t vis) const {
        const uint32_t mine = vis >> (8 * h);
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (!((mine >> (16 * (i / 8) + i % 8)) & 1)) S[i] = -INFINITY;
    }
    // scores of U x 32 keys -> numerators (f16), with REST what that rounding took off them (f16
    // as well: the two add up to 22 bits), the running maximum and sum
    template <bool REST = false, int U>
    __device__ __forceinline__ void softmax(f32x16 (&S)[U], const PagedSeen (&s)[U], uint4 (&pf)[2 * U], uint4 *rest = nullptr) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (!s[u].whole) hide(S[u], s[u].vis);
        float mx = S[0][0];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, S[u][i]);
        mx = max_halves(mx);
        // the reference moves only when the maximum has grown by more than 2^8
        const bool grow = mx > m && !((mx - m) * a.cs <= 8.0f + F16_LIFT);
        if (__builtin_amdgcn_ballot_w64(grow) != 0) {
            const float ref = mx - a.lift;
            const float alpha = grow ? __builtin_amdgcn_exp2f((m - ref) * a.cs) : 1.0f;
            m = grow ? ref : m;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < NB; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) O[d][i] *= alpha;
        }
        const float mc = m == -INFINITY ? 0.0f : m * a.cs;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float p[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(S[u][8 * i + e] * a.cs - mc);
                l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
                pf[2 * u + i] = pack8<false>(p);
                if (REST) {
                    // one mixed instruction each, from the packed halves (left to itself the compiler
                    // rounds every weight once more: chunk attention of 2048 over 16384 844 us, not 826)
                    uint4 &w = pf[2 * u + i];
                    asm("" : "+v"(w.x), "+v"(w.y), "+v"(w.z), "+v"(w.w));
                    float minus = -1.0f;
                    asm("" : "+s"(minus));
                    const f16x8 f = __builtin_bit_cast(f16x8, w);
#pragma unroll
                    for (int e = 0; e < 8; ++e) p[e] = fmaf((float)f[e], minus, p[e]);
                    rest[2 * u + i] = pack8<false>(p);
                }
            }
    }
    // places that hold no token's value may hold anything
    __device__ __forceinline__ uint4 live_v(uint4 v, int i, uint32_t there) const {
        const uint32_t on = there >> (16 * i + 8 * h);
        auto keep = [&](int e) { return ((on >> e) & 1 ? 0xffffu : 0u) | ((on >> e) & 2 ? 0xffff0000u : 0u); };
        return make_uint4(v.x & keep(0), v.y & keep(2), v.z & keep(4), v.w & keep(6));
    }
    // the values that are finite: an infinity times a weight's rest would be NaN
    static __device__ __forceinline__ uint4 finite_v(uint4 v) {
        auto keep = [](uint32_t w) {
            return w & (((w & 0x7c00u) == 0x7c00u ? 0u : 0xffffu) | ((w & 0x7c000000u) == 0x7c000000u ? 0u : 0xffff0000u));
        };
        return make_uint4(keep(v.x), keep(v.y), keep(v.z), keep(v.w));
    }
    // One dim block's products key by key: sp and sv hold the lanes' P and V^T operands
    // ([i][lane], 16 bytes each, sv's parts sv_step words apart).
    __device__ __forceinline__ void careful_pv(int d, const PagedSeen &s, const uint32_t *sp, const uint32_t *sv, int sv_step) {
#pragma unroll 1
        for (int key = 0; key < 32; ++key) {
            const int i = key >> 4, from = 32 * ((key >> 3) & 1), w = (key & 7) >> 1, sh = 16 * (key & 1);
            if (!((s.vis >> key) & 1)) continue;
            const float p = h2f((uint16_t)(sp[256 * i + 4 * (from + c) + w] >> sh));
#pragma unroll
            for (int x = 0; x < 16; ++x)
                O[d][x] += p * h2f((uint16_t)(sv[sv_step * i + 4 * (from + 8 * (x / 4) + 4 * h + x % 4) + w] >> sh));
        }
    }
    // ... of the keys 16 i .. + 15 alone, the weights' rests behind P
    __device__ __forceinline__ void careful_rest_pv(int d, const PagedSeen &s, int i, const uint32_t *sp, const uint32_t *sv) {
#pragma unroll 1
        for (int key = 0; key < 16; ++key) {
            const int from = 32 * (key >> 3), w = (key & 7) >> 1, sh = 16 * (key & 1);
            if (!((s.vis >> (16 * i + key)) & 1)) continue;
            const uint32_t *at = sp + 4 * (from + c) + w;
            const float p = h2f((uint16_t)(at[0] >> sh)) + h2f((uint16_t)(at[256] >> sh));
#pragma unroll
            for (int x = 0; x < 16; ++x) O[d][x] += p * h2f((uint16_t)(sv[4 * (from + 8 * (x / 4) + 4 * h + x % 4) + w] >> sh));
        }
    }
};

// Tiles of KT keys that four waves share in LDS, as the operands' 1-KiB fragments
// (64 lanes x 16 bytes): of every 32 keys the NS steps of K, then of V^T the two
// halves of keys x NB dim blocks.
template <int D> struct PagedTile {
    static constexpr int KT = D <= 128 ? 64 : 32;
    static constexpr int TILE = KT / 32 * (D / 16 + 2 * ((D + 31) / 32)) * 1024;
};

}  // namespace tlh
