// Attention of drafted tokens over a paged f16 cache, gfx950.
//
// Sequence s has L = context_lens[s] tokens in the cache, the last n of them
// drafted (n = draft_starts[s + 1] - draft_starts[s]), and n rows of q. Row i
// sees every token before L - n and drafted token j where bit j of its mask is
// set; the caches are the paged-attention layouts
//   key   [blocks][kv_heads][D/8][block_size][8]
//   value [blocks][kv_heads][D][block_size]
// A row that sees nothing gives zeros.
//
// Bound by one read of the keys and values while the rows are few; by the
// matrix cores and the exponentials with a tree of tens of tokens. The rows of a
// (sequence, kv head) are its drafted tokens x the group's heads; a wave owns 32:
//   S^T = K . Q^T     a lane's key row is one of 32, taken in an order that
//                     makes S^T's registers 8 i .. 8 i + 7 the keys 16 i + 8 h ..
//                     + 7 of the tile, in order;
//   O^T += V^T . P^T  so P is the operand as it is, and V^T's is 8 consecutive
//                     places of one dim.
// Either operand is 16 bytes a lane that lie together in the page, so the pages
// are read as they are. Two forms:
//  * a workgroup takes 32 rows and one partition of the context, its four waves
//    32-key tiles in turn, straight into registers: the next tile's keys are
//    requested when this one's have been multiplied, its values when this one's
//    have, so with two waves a SIMD a tile is always in flight; the waves merge
//    at the end, the partitions in a second launch;
//  * with many rows, and sequences enough to fill the machine without a split: a
//    workgroup takes 128 rows, and its four waves share 64-key tiles in LDS
//    (double-buffered, loaded straight from the pages in the order in which the
//    lanes take them), so a page is read a quarter as often.
//
// Measured, 32/8 heads of 128: 32 trees of 1..8 tokens over 512..8192 127 us (4.5 TB/s);
// 16 of 63 over 512..4096 84 to 89 us; 32 of 64 over 4096 200 to 217 us (shared tiles, 640
// to 700 TFLOP/s); 1 of 7 over 600 10 to 12 us in two launches. These are of nodes made for
// the longest context; made for 131072 tokens the first takes 5% more, the last 3 us.
#include <algorithm>

#include "paged_wave.hpp"

namespace tlh {

constexpr int TA_WAVES = 4, TA_KEYS = 32 * TA_WAVES;  // keys a workgroup takes a round
constexpr int TA_WGS = 1024;                          // workgroups a split aims for
constexpr int TA_WGS_SHARED = 512;                    // workgroups that fill the machine (two a CU)
constexpr int TA_MAX_PARTS = 64;                      // a lane each in the merge

struct TaArgs : PagedArgs {
    uint16_t *out;
    const uint16_t *q;
    const int32_t *lens, *starts;
    const int64_t *masks;
    float *part;  // [s][kv head][block of 32 rows][partition][row][m, l, -, -, D]
    int S, H, G, rows, max_drafts, max_ctx, P, part_len, RB;  // RB: blocks of 32 rows
    int sort;  // sequences go longest first
};

struct TaSeq {
    int b, n, L;  // first row, drafted tokens, tokens in the cache
};
__device__ __forceinline__ TaSeq ta_seq(const TaArgs &a, int s) {
    TaSeq q;
    q.b = max(0, min(a.starts[s], a.rows));
    const int e = max(q.b, min(a.starts[s + 1], a.rows));
    q.n = min(e - q.b, a.max_drafts);
    q.L = a.num_blocks > 0 ? max(0, min(a.lens[s], a.max_ctx)) : 0;
    return q;
}

// The o-th longest sequence's index (the o-th, without a.sort): with more workgroups
// than run at once, long sequences that start last would end alone. Every lane of the
// wave calls; lane i ranks sequence i (S <= 64).
__device__ __forceinline__ int ta_pick(const TaArgs &a, int o, int lane) {
    if (!a.sort) return o;
    int key = -1;
    if (lane < a.S) {
        const TaSeq q = ta_seq(a, lane);
        key = q.n > 0 ? q.L : 0;
    }
    int rank = 0;
    for (int j = 0; j < a.S; ++j) {
        const int other = __builtin_amdgcn_readlane(key, j);
        rank += other > key || (other == key && j < lane);
    }
    const uint64_t who = __builtin_amdgcn_ballot_w64(lane < a.S && rank == o);
    return __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)who) - 1);
}

// Row i of a sequence sees the `prefix` tokens before the drafted ones and drafted token j
// where bit j of its mask is set.
struct TaRule {
    int prefix;
    uint64_t mask = 0;  // of this lane's row
    __device__ __forceinline__ bool whole(int base) const { return base + 32 <= prefix; }
    __device__ __forceinline__ uint32_t sees(int base) const {
        const int d = base - prefix;
        return d >= 64    ? 0u
               : d >= 0   ? (uint32_t)(mask >> d)
               : d <= -32 ? ~0u
                          : (uint32_t)(mask << -d) | ((1u << -d) - 1);
    }
};
template <int D, int BS> using TaWave = PagedWave<D, BS, TaRule>;
// -> this lane's part of the row's q
template <int D> __device__ __forceinline__ const uint8_t *ta_row(const TaArgs &a, TaRule &rule, int half, int b, int hk, int row) {
    const int i = row / a.G;
    rule.mask = (uint64_t)a.masks[b + i];
    return (const uint8_t *)(a.q + ((int64_t)(b + i) * a.H + hk * a.G + row % a.G) * D) + 16 * half;
}

template <int D, int BS>
__global__ void __launch_bounds__(64 * TA_WAVES, D <= 128 ? 2 : 1) k_tree_attn(const TaArgs a) {
    using W = TaWave<D, BS>;
    constexpr int NS = W::NS, NB = W::NB;
    constexpr int MD = NB > 1 ? 64 : 32;  // dims merged at a time
    // Loads a tile ahead, where two waves' registers hold O, the keys and the values; above
    // 128 dims a tile's values are requested when its keys have been multiplied.
    constexpr bool AHEAD = D <= 128;
    __shared__ __attribute__((aligned(16))) float s_o[TA_WAVES][32][MD + 4];
    __shared__ float s_m[TA_WAVES][32], s_l[TA_WAVES][32];
    __shared__ uint4 s_q[NS][64];  // Q^T as the lanes take it: 16 bytes a lane, in order
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // with 8 kv heads a head's workgroups share an XCD, row blocks next to each other
    const int hk = blockIdx.x % a.KV;
    const int rb = (blockIdx.x / a.KV) % a.RB;
    const int s = ta_pick(a, (blockIdx.x / a.KV / a.RB) % a.S, lane);
    const int part = blockIdx.x / a.KV / a.RB / a.S;
    const TaSeq sq = ta_seq(a, s);
    const int L = sq.L, R = sq.n * a.G, r0 = 32 * rb;
    const int t0 = part * a.part_len;
    if (r0 >= R || (part > 0 && t0 >= L)) return;
    const int ntiles = (min(L, t0 + a.part_len) - t0 + 31) / 32;
    W w(a, lane, s, hk, L, TaRule{L - sq.n});
    const int c = w.c, h = w.h;
    {
        // the four waves share Q in LDS: in registers it would leave too few for two waves a SIMD
        const uint8_t *qr = ta_row<D>(a, w.rule, h, sq.b, hk, min(r0 + c, R - 1));
        for (int st = wave; st < NS; st += TA_WAVES) s_q[st][lane] = w.signed_q(*(const uint4 *)(qr + 32 * st));
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
            pn = w.ids_of(t0 + 32 * (wave + TA_WAVES));
            if (AHEAD) {
                load_k(pg);
                load_v(pg);
            }
        }
        for (int k = wave; k < ntiles; k += TA_WAVES) {
            const int base = t0 + 32 * k;
            pn = w.checked(pn);
            const typename W::Pages after = w.ids_of(base + 64 * TA_WAVES);
            if (!AHEAD) load_k(pg);
            f32x16 S[1] = {(f32x16){}};
#pragma unroll
            for (int st = 0; st < NS; ++st) S[0] = mfma32<false>(kf[st], s_q[st][lane], S[0]);
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
                uint4 *sp = (uint4 *)&s_o[wave][0][0], *sv = sp + 128;
                static_assert(256 * 16 <= sizeof(s_o[0]), "operands of one dim block");
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
    float *slot = a.part + ((((int64_t)s * a.KV + hk) * a.RB + rb) * a.P + part) * 32 * (D + 4);
#pragma unroll
    for (int d0 = 0; d0 < NB; d0 += MD / 32) {
        if (d0 > 0) lds_barrier();  // the last part has been read
#pragma unroll
        for (int d = d0; d < d0 + MD / 32 && d < NB; ++d)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *(float4 *)&s_o[wave][c][32 * (d - d0) + 8 * j + 4 * h] =
                    make_float4(w.O[d][4 * j], w.O[d][4 * j + 1], w.O[d][4 * j + 2], w.O[d][4 * j + 3]);
        lds_barrier();
        for (int e = threadIdx.x; e < 32 * (MD / 4); e += 64 * TA_WAVES) {
            const int row = e / (MD / 4), dd = 4 * (e % (MD / 4)), dim = 32 * d0 + dd, rr = r0 + row;
            if (rr >= R || dim >= D) continue;
            float M = -INFINITY;
#pragma unroll
            for (int x = 0; x < TA_WAVES; ++x) M = fmaxf(M, s_m[x][row]);
            float sum = 0.0f;
            float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int x = 0; x < TA_WAVES; ++x) {
                const float mw = s_m[x][row];
                const float f = mw == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((mw - M) * a.cs);
                const float4 v = *(const float4 *)&s_o[x][row][dd];
                if (mw == -INFINITY && !(s_l[x][row] != 0.0f)) continue;  // saw nothing
                sum += f * s_l[x][row];
                o.x += f * v.x, o.y += f * v.y, o.z += f * v.z, o.w += f * v.w;
            }
            if (a.P == 1) {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                uint16_t *dst = a.out + ((int64_t)(sq.b + rr / a.G) * a.H + hk * a.G + rr % a.G) * D + dim;
                const float x[8] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv, 0, 0, 0, 0};
                const uint4 v = pack8<false>(x);
                *(uint2 *)dst = make_uint2(v.x, v.y);
            } else {
                float *dst = slot + (int64_t)row * (D + 4);
                *(float4 *)(dst + 4 + dim) = o;
                if (dim == 0) *(float2 *)dst = make_float2(M, sum);
            }
        }
    }
}

template <int D, int BS>
__global__ void __launch_bounds__(64 * TA_WAVES, D <= 128 ? 2 : 1) k_tree_attn_shared(const TaArgs a) {
    using W = TaWave<D, BS>;
    constexpr int NS = W::NS, NB = W::NB;
    using Sh = PagedTile<D>;
    constexpr int KT = Sh::KT, SUBS = KT / 32, KF = SUBS * NS;
    __shared__ __attribute__((aligned(16))) uint8_t T0[Sh::TILE], T1[Sh::TILE];
    __shared__ uint4 s_p[TA_WAVES][128];  // the careful pass's P
    __shared__ int s_flag[TA_WAVES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row_groups = (a.RB + TA_WAVES - 1) / TA_WAVES;
    const int hk = blockIdx.x % a.KV;
    const int rg = (blockIdx.x / a.KV) % row_groups;
    const int s = ta_pick(a, (blockIdx.x / a.KV / row_groups) % a.S, lane);
    const TaSeq sq = ta_seq(a, s);
    const int L = sq.L, R = sq.n * a.G, r0 = 32 * (rg * TA_WAVES + wave);
    if (rg * TA_WAVES * 32 >= R) return;
    const int ntiles = (L + KT - 1) / KT;
    const bool mine = r0 < R;  // some wave of the workgroup has rows, this one may not
    W w(a, lane, s, hk, L, TaRule{L - sq.n});
    const int c = w.c, h = w.h;
    typename W::Pages pg[SUBS], pn[SUBS];  // of the tile in turn and the next one
    auto ids = [&](int t, typename W::Pages (&p)[SUBS]) {
#pragma unroll
        for (int u = 0; u < SUBS; ++u) p[u] = w.ids_of(KT * t + 32 * u);
    };
    // wave w loads the fragments w, w + 4, ... of K and of V
    auto load_tile = [&](const typename W::Pages *p, uint8_t *T) {
#pragma unroll
        for (int u = 0; u < SUBS; ++u) {
            const uint8_t *kp = w.k_at(p[u]);
#pragma unroll
            for (int x = 0; x < (NS + TA_WAVES - 1) / TA_WAVES; ++x) {
                const int st = TA_WAVES * x + wave;
                if (NS % TA_WAVES == 0 || st < NS)
                    to_lds(kp + W::k_step(st), T + (u * NS + st) * 1024);
            }
#pragma unroll
            for (int x = 0; x < (2 * NB + TA_WAVES - 1) / TA_WAVES; ++x) {
                const int f = TA_WAVES * x + wave, i = f & 1, d = f >> 1;
                if (2 * NB % TA_WAVES == 0 || f < 2 * NB)
                    to_lds(w.v_at(p[u], i) + w.v_step(d), T + (KF + (2 * u + i) * NB + d) * 1024);
            }
        }
    };
    uint4 qf[NS];
    {
        const uint8_t *qr = ta_row<D>(a, w.rule, h, sq.b, hk, min(r0 + c, R - 1));
#pragma unroll
        for (int st = 0; st < NS; ++st) qf[st] = w.signed_q(*(const uint4 *)(qr + 32 * st));
    }
    bool careful = false;
    auto tile = [&](int t, const uint8_t (&T)[Sh::TILE], uint8_t (&Tn)[Sh::TILE]) {
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): tile t has landed
        lds_barrier();                       // for every wave, and the other buffer is free
        uint32_t good[SUBS];
#pragma unroll
        for (int u = 0; u < SUBS; ++u) good[u] = pg[u].good;
        if (t + 1 < ntiles) {
#pragma unroll
            for (int u = 0; u < SUBS; ++u) pg[u] = w.checked(pn[u]);
            load_tile(pg, Tn);
            ids(t + 2, pn);
        }
        if (!mine) return;
        f32x16 S[SUBS];
        PagedSeen see[SUBS];
#pragma unroll
        for (int u = 0; u < SUBS; ++u) {
            S[u] = (f32x16){};
#pragma unroll
            for (int st = 0; st < NS; ++st)
                S[u] = mfma32<false>(*(const uint4 *)(T + (u * NS + st) * 1024 + 16 * lane), qf[st], S[u]);
            see[u] = w.seen(KT * t + 32 * u, good[u]);
        }
        uint4 pf[2 * SUBS];
        w.softmax(S, see, pf);
#pragma unroll
        for (int u = 0; u < SUBS; ++u) {
            const uint8_t *V = T + (KF + u * 2 * NB) * 1024;
            if (careful && !see[u].whole) {
                __builtin_amdgcn_wave_barrier();
                s_p[wave][lane] = pf[2 * u], s_p[wave][64 + lane] = pf[2 * u + 1];
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int d = 0; d < NB; ++d)
                    w.careful_pv(d, see[u], (const uint32_t *)s_p[wave], (const uint32_t *)(V + d * 1024), 256 * NB);
            } else if (see[u].there != ~0u) {
#pragma unroll 1
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int d = 0; d < NB; ++d)
                        w.O[d] = mfma32<false>(w.live_v(*(const uint4 *)(V + (i * NB + d) * 1024 + 16 * lane), i, see[u].there),
                                               i ? pf[2 * u + 1] : pf[2 * u], w.O[d]);
            } else {
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int d = 0; d < NB; ++d)
                        w.O[d] = mfma32<false>(*(const uint4 *)(V + (i * NB + d) * 1024 + 16 * lane), pf[2 * u + i], w.O[d]);
            }
        }
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
        const bool again = mine && w.some_masked && __builtin_amdgcn_ballot_w64(w.bad() && r0 + c < R) != 0;
        if (lane == 0) s_flag[wave] = again;
        lds_barrier();  // and every wave is done with both buffers
        careful = (s_flag[0] | s_flag[1] | s_flag[2] | s_flag[3]) != 0;
        if (!careful) break;
    }
    const int rr = r0 + c;
    const float sum = sum_halves(w.l);
    if (rr >= R) return;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    uint16_t *dst = a.out + ((int64_t)(sq.b + rr / a.G) * a.H + hk * a.G + rr % a.G) * D + 4 * h;
#pragma unroll
    for (int d = 0; d < NB; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (32 * d + 8 * j >= D) continue;
            const float x[8] = {w.O[d][4 * j] * inv, w.O[d][4 * j + 1] * inv, w.O[d][4 * j + 2] * inv,
                                w.O[d][4 * j + 3] * inv, 0, 0, 0, 0};
            const uint4 v = pack8<false>(x);
            *(uint2 *)(dst + 32 * d + 8 * j) = make_uint2(v.x, v.y);
        }
}

// One wave a row: lane p holds partition p's weight, the lanes then take the dims.
template <int D>
__global__ void __launch_bounds__(256) k_tree_attn_merge(const TaArgs a) {
    const int lane = threadIdx.x & 63;
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6), hk = blockIdx.y, s = blockIdx.z;
    const TaSeq sq = ta_seq(a, s);
    if (row >= sq.n * a.G) return;
    const int np = (sq.L + a.part_len - 1) / a.part_len;
    const int64_t step = 32 * (D + 4);
    const float *base = a.part + ((((int64_t)s * a.KV + hk) * a.RB + row / 32) * a.P) * step + (row % 32) * (D + 4);
    constexpr int E = (D + 63) / 64, AT_ONCE = 8;
    // the first partitions' sums are on their way while the weights are formed
    float o[AT_ONCE][E];
    auto load = [&](int p0) {
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e)  // (past the last partition or dim: an element that gets no weight, or no place)
                o[i][e] = base[max(min(p0 + i, np - 1), 0) * step + 4 + min(lane + 64 * e, D - 1)];
    };
    float2 ml = make_float2(-INFINITY, 0.0f);
    if (lane < np) ml = *(const float2 *)(base + lane * step);
    if (np > 0) load(0);
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
    uint16_t *dst = a.out + ((int64_t)(sq.b + row / a.G) * a.H + hk * a.G + row % a.G) * D;
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (lane + 64 * e < D) dst[lane + 64 * e] = f2h(acc[e] * inv);
}

static int64_t ta_max_rows(const tlh_tree_attention_args &a) { return (int64_t)a.max_drafts * (a.num_heads / a.num_kv_heads); }
static int64_t ta_row_blocks(const tlh_tree_attention_args &a) { return (ta_max_rows(a) + 31) / 32; }
static int64_t ta_shared_wgs(const tlh_tree_attention_args &a) {
    return (int64_t)a.num_seqs * a.num_kv_heads * ((ta_row_blocks(a) + TA_WAVES - 1) / TA_WAVES);
}
// Shared tiles for more than two blocks of 32 rows, where they make two workgroups a
// CU without a split. 32/8 heads of 128, trees of 64, us (shared, own tiles): 32
// sequences of 4096 200, 259, of 512..4096 172, 159; 64 of 1000 123, 177. With fewer
// workgroups a split's partials cost more than the shared reads save: 16 of 512..4096
// 102, 83, 8 of 100..8000 97, 85.
static bool ta_shared(const tlh_tree_attention_args &a) {
    return ta_row_blocks(a) > 2 && ta_shared_wgs(a) >= TA_WGS_SHARED;
}
static int64_t ta_rounds(const tlh_tree_attention_args &a) { return ((int64_t)a.max_context_len + TA_KEYS - 1) / TA_KEYS; }
// partitions: as many as make no more than TA_WGS workgroups, each of at least one round of keys
static int ta_parts(const tlh_tree_attention_args &a, int &part_len) {
    const int64_t base = (int64_t)a.num_seqs * a.num_kv_heads * ta_row_blocks(a);
    const int64_t rounds = std::max<int64_t>(ta_rounds(a), 1);
    const int64_t want = ta_shared(a) ? 1
                                      : std::max<int64_t>(1, std::min<int64_t>({TA_WGS / std::max<int64_t>(base, 1),
                                                                                TA_MAX_PARTS, rounds}));
    const int64_t each = (rounds + want - 1) / want;
    part_len = (int)(each * TA_KEYS);
    return (int)((rounds + each - 1) / each);
}

// A slot of 32 rows for every block of rows and partition, at most TA_WGS of them
// where there are several partitions. The size never shrinks as any of the counts
// grows: one buffer for the largest call serves every smaller one.
size_t tree_attention_scratch_bytes(const tlh_tree_attention_args &a) {
    if (ta_rounds(a) <= 1) return 0;
    const int64_t base = (int64_t)a.num_seqs * a.num_kv_heads * ta_row_blocks(a);
    const int64_t slots = std::min<int64_t>(base * std::min<int64_t>(ta_rounds(a), TA_MAX_PARTS), TA_WGS);
    return (size_t)slots * 32 * (a.head_size + 4) * sizeof(float);
}

template <int D, int BS> static void launch_ta2(const TaArgs &t, bool shared, unsigned blocks, hipStream_t stream) {
    if (shared) hipLaunchKernelGGL((k_tree_attn_shared<D, BS>), dim3(blocks), dim3(64 * TA_WAVES), 0, stream, t);
    else hipLaunchKernelGGL((k_tree_attn<D, BS>), dim3(blocks), dim3(64 * TA_WAVES), 0, stream, t);
}
template <int D> static void launch_ta(const TaArgs &t, int bs, bool shared, unsigned blocks, hipStream_t stream) {
    switch (bs) {
    case 8: launch_ta2<D, 8>(t, shared, blocks, stream); break;
    case 16: launch_ta2<D, 16>(t, shared, blocks, stream); break;
    default: launch_ta2<D, 32>(t, shared, blocks, stream); break;
    }
    if (t.P > 1)
        hipLaunchKernelGGL((k_tree_attn_merge<D>), dim3((t.max_drafts * t.G + 3) / 4, t.KV, t.S), dim3(256), 0, stream, t);
}

tlh_status launch_tree_attention(const tlh_tree_attention_args &a, void *scratch, hipStream_t stream) {
    TaArgs t = {};
    t.out = (uint16_t *)a.out, t.q = (const uint16_t *)a.q;
    t.kc = (const uint16_t *)a.k_cache, t.vc = (const uint16_t *)a.v_cache;
    t.tables = a.block_tables, t.lens = a.context_lens, t.starts = a.draft_starts, t.masks = a.draft_masks;
    t.part = (float *)scratch;
    t.num_blocks = a.num_blocks;
    t.S = a.num_seqs, t.H = a.num_heads, t.KV = a.num_kv_heads, t.G = a.num_heads / a.num_kv_heads;
    t.rows = a.num_rows, t.max_drafts = a.max_drafts, t.max_blocks = a.max_blocks_per_seq, t.max_ctx = a.max_context_len;
    const bool sh = ta_shared(a);
    const int64_t rb = ta_row_blocks(a);
    t.P = ta_parts(a, t.part_len);
    t.RB = (int)rb;
    set_scale(t, a.scale);
    const int64_t blocks = sh ? ta_shared_wgs(a) : (int64_t)t.P * t.S * rb * t.KV;
    t.sort = t.S > 1 && t.S <= 64 && blocks > 2 * device_cus();
    if (blocks >= 1 << 24)  // x 256 threads
        return set_error(TLH_INVALID, "tree_attention: too many sequences and heads for one launch");
    switch (a.head_size) {
    case 64: launch_ta<64>(t, a.block_size, sh, (unsigned)blocks, stream); break;
    case 80: launch_ta<80>(t, a.block_size, sh, (unsigned)blocks, stream); break;
    case 96: launch_ta<96>(t, a.block_size, sh, (unsigned)blocks, stream); break;
    case 112: launch_ta<112>(t, a.block_size, sh, (unsigned)blocks, stream); break;
    case 128: launch_ta<128>(t, a.block_size, sh, (unsigned)blocks, stream); break;
    case 192: launch_ta<192>(t, a.block_size, sh, (unsigned)blocks, stream); break;
    default: launch_ta<256>(t, a.block_size, sh, (unsigned)blocks, stream); break;
    }
    return check_launch("tree_attention");
}

}  // namespace tlh
