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
// matrix cores with a tree of tens of tokens. A workgroup of four waves takes up
// to 32 RT rows that share a kv head (drafted tokens x the group's heads) and
// one partition of the context; its waves take 32-key tiles in turn. Both
// products' operands come from the pages straight into registers, 16 bytes a
// lane:
//   S^T = K . Q^T     a lane's key row is one of 32, taken in an order that
//                     makes S^T's registers 8 i .. 8 i + 7 the keys 16 i + 8 h ..
//                     + 7 of the tile, in order;
//   O^T += V^T . P^T  so P is the operand as it is, and V^T's is 8 consecutive
//                     places of one dim.
// The next tile's keys are requested when this one's have been multiplied, its
// values when this one's have, so that with two waves a SIMD a tile is always
// in flight. Partitions are merged by a second launch.
#include <algorithm>

#include "mfma32.hpp"

namespace tlh {

constexpr int TA_WAVES = 4, TA_KEYS = 32 * TA_WAVES;  // keys a workgroup takes a round
constexpr int TA_WGS = 1024;                          // workgroups a split aims for
constexpr int TA_MAX_PARTS = 64;                      // a lane each in the merge

struct TaArgs {
    uint16_t *out;
    const uint16_t *q, *kc, *vc;
    const int32_t *tables, *lens, *starts;
    const int64_t *masks;
    float *part;  // [s][kv head][row block][partition][row][m, l, -, -, D]
    int64_t num_blocks;
    int S, H, KV, G, rows, max_drafts, max_blocks, max_ctx, P, part_len, RB;
    float cs;             // |scale| * log2(e); 1 where the scale is 0
    uint32_t qand, qxor;  // q's words: negated where the scale is negative, zeroed where it is 0
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

template <int D, int BS, int RT>
__global__ void __launch_bounds__(64 * TA_WAVES, D <= 128 && RT == 1 ? 2 : 1) k_tree_attn(const TaArgs a) {
    constexpr int NS = D / 16, NB = (D + 31) / 32, PAGES = 32 / BS;
    constexpr int MD = NB > 1 ? 64 : 32;  // dims merged at a time
    __shared__ __attribute__((aligned(16))) float s_o[TA_WAVES][32][MD + 4];
    __shared__ float s_m[TA_WAVES][32 * RT], s_l[TA_WAVES][32 * RT];
    __shared__ uint4 s_q[RT][NS][64];  // Q^T as the lanes take it: 16 bytes a lane, in order
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = lane >> 5, c = lane & 31;
    // with 8 kv heads a head's workgroups share an XCD, row blocks next to each other
    const int hk = blockIdx.x % a.KV;
    const int rb = (blockIdx.x / a.KV) % a.RB;
    const int s = (blockIdx.x / a.KV / a.RB) % a.S;
    const int part = blockIdx.x / a.KV / a.RB / a.S;
    const TaSeq sq = ta_seq(a, s);
    const int n = sq.n, L = sq.L, R = n * a.G, r0 = rb * 32 * RT;
    const int t0 = part * a.part_len;
    if (r0 >= R || (part > 0 && t0 >= L)) return;
    const int t1 = min(L, t0 + a.part_len);
    const int prefix = L - n;
    const int ntiles = (t1 - t0 + 31) / 32;
    const int32_t *table = a.tables + (int64_t)s * a.max_blocks;

    // this lane's rows: drafted token row / G, head row % G of the group. The four
    // waves share Q in LDS: in registers it would leave too few for two waves a SIMD
    uint64_t mask[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int row = min(r0 + 32 * t + c, R - 1), i = row / a.G;
        const uint8_t *qr = (const uint8_t *)(a.q + ((int64_t)(sq.b + i) * a.H + hk * a.G + row % a.G) * D) + 16 * h;
        mask[t] = (uint64_t)a.masks[sq.b + i];
        for (int st = wave; st < NS; st += TA_WAVES) {
            const uint4 w = *(const uint4 *)(qr + 32 * st);
            s_q[t][st][lane] = make_uint4((w.x & a.qand) ^ a.qxor, (w.y & a.qand) ^ a.qxor, (w.z & a.qand) ^ a.qxor,
                                          (w.w & a.qand) ^ a.qxor);
        }
    }

    const int64_t page_bytes = (int64_t)a.KV * D * BS * 2;
    const uint8_t *kbase = (const uint8_t *)a.kc + (int64_t)hk * D * BS * 2;
    const uint8_t *vbase = (const uint8_t *)a.vc + (int64_t)hk * D * BS * 2;
    // the key of S^T's row c: bits 2 and 3 of c exchanged
    const int kappa = (c & 0x13) | (c & 4) << 1 | (c & 8) >> 1;
    // a tile's pages (the last one's again past the context), and whether any is outside the pools
    struct Pages {
        int id[PAGES];
        uint32_t good;  // bits of the tile's keys whose page is inside
    };
    // their ids are read two tiles ahead, so that no tile waits for the table
    auto ids_of = [&](int k) {
        Pages p = {};
#pragma unroll
        for (int i = 0; i < PAGES; ++i)
            p.id[i] = table[__builtin_amdgcn_readfirstlane(min((t0 + 32 * k) / BS + i, (L - 1) / BS))];
        return p;
    };
    auto checked = [&](Pages p) {
        p.good = 0;
#pragma unroll
        for (int i = 0; i < PAGES; ++i) {
            const bool ok = p.id[i] >= 0 && p.id[i] < a.num_blocks;
            p.id[i] = ok ? p.id[i] : 0;
            p.good |= ok ? (BS == 32 ? ~0u : ((1u << (BS & 31)) - 1) << (BS * i)) : 0u;
        }
        return p;
    };
    auto page_at = [&](const Pages &p, int key) {  // of key `key` of the tile
        int id = p.id[0];
#pragma unroll
        for (int i = 1; i < PAGES; ++i) id = key / BS == i ? p.id[i] : id;
        return (int64_t)id * page_bytes;
    };
    uint4 kf[NS], vf[NB][2];
    auto load_k = [&](const Pages &p) {
        const uint8_t *kp = kbase + page_at(p, kappa) + h * BS * 16 + (kappa % BS) * 16;
#pragma unroll
        for (int st = 0; st < NS; ++st) kf[st] = *(const uint4 *)(kp + st * BS * 32);
    };
    auto load_v = [&](const Pages &p) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int key = 16 * i + 8 * h;
            const uint8_t *vp = vbase + page_at(p, key) + (key % BS) * 2 + c * BS * 2;
#pragma unroll
            for (int d = 0; d < NB; ++d)  // dims past the last repeat it
                vf[d][i] = *(const uint4 *)(vp + (32 * d + 31 < D ? 32 * d : min(32 * d + c, D - 1) - c) * BS * 2);
        }
    };

    __syncthreads();
    f32x16 O[RT][NB];
    float m[RT], l[RT];
    // A value that is not finite would turn the zero weight of a key that a row does
    // not see into NaN. So where a wave's sums come out not finite, it takes its tiles
    // again, carefully: in those with masked keys it adds each seen key's product by itself.
    bool careful = false, some_masked = false;
    for (;;) {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            m[t] = -INFINITY;
            l[t] = 0.0f;
#pragma unroll
            for (int d = 0; d < NB; ++d) O[t][d] = (f32x16){};
        }
        Pages pg = {}, pn = {};
        if (wave < ntiles) {
            pg = checked(ids_of(wave));
            pn = ids_of(wave + TA_WAVES);
            load_k(pg);
            load_v(pg);
        }
        for (int k = wave; k < ntiles; k += TA_WAVES) {
            const int base = t0 + 32 * k;
            pn = checked(pn);
            const Pages after = ids_of(k + 2 * TA_WAVES);
            f32x16 S[RT];
#pragma unroll
            for (int t = 0; t < RT; ++t) S[t] = (f32x16){};
#pragma unroll
            for (int st = 0; st < NS; ++st)
#pragma unroll
                for (int t = 0; t < RT; ++t) S[t] = mfma32<false>(kf[st], s_q[t][st][lane], S[t]);
            load_k(pn);  // past the last tile: the last page again
            const bool whole = base + 32 <= prefix && pg.good == ~0u;
            uint32_t vis[RT];
            uint32_t there = ~0u;  // keys that are in the cache
            if (!whole) {
                some_masked = true;
                there = pg.good & (L - base >= 32 ? ~0u : (1u << (L - base)) - 1);
                const int d = base - prefix;
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    const uint32_t see = d >= 64    ? 0u
                                         : d >= 0   ? (uint32_t)(mask[t] >> d)
                                         : d <= -32 ? ~0u
                                                    : (uint32_t)(mask[t] << -d) | ((1u << -d) - 1);
                    vis[t] = see & there;
                    const uint32_t mine = vis[t] >> (8 * h);
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (!((mine >> (16 * (i / 8) + i % 8)) & 1)) S[t][i] = -INFINITY;
                }
            }
            uint4 pf[RT][2];
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                float mx = S[t][0];
#pragma unroll
                for (int i = 1; i < 16; ++i) mx = fmaxf(mx, S[t][i]);
                mx = max_halves(mx);
                // the reference moves only when the maximum has grown by more than 2^8
                const bool grow = mx > m[t] && !((mx - m[t]) * a.cs <= 8.0f);
                if (__builtin_amdgcn_ballot_w64(grow) != 0) {
                    const float alpha = grow ? __builtin_amdgcn_exp2f((m[t] - mx) * a.cs) : 1.0f;
                    m[t] = grow ? mx : m[t];
                    l[t] *= alpha;
#pragma unroll
                    for (int d = 0; d < NB; ++d)
#pragma unroll
                        for (int i = 0; i < 16; ++i) O[t][d][i] *= alpha;
                }
                const float mc = m[t] == -INFINITY ? 0.0f : m[t] * a.cs;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float p[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(S[t][8 * i + e] * a.cs - mc);
                    l[t] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
                    pf[t][i] = pack8<false>(p);
                }
            }
            if (!whole && there != ~0u) {  // places that hold no token's value may hold anything
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t live = there >> (16 * i + 8 * h);
                    auto keep = [&](int e) { return ((live >> e) & 1 ? 0xffffu : 0u) | ((live >> e) & 2 ? 0xffff0000u : 0u); };
#pragma unroll
                    for (int d = 0; d < NB; ++d) {
                        vf[d][i].x &= keep(0);
                        vf[d][i].y &= keep(2);
                        vf[d][i].z &= keep(4);
                        vf[d][i].w &= keep(6);
                    }
                }
            }
            if (careful && !whole) {
// through the wave's part of the merge buffer, which is free until the end
                uint32_t *sp = (uint32_t *)&s_o[wave][0][0], *sv = sp + RT * 512;
                static_assert((RT + 1) * 512 * 4 <= sizeof(s_o[0]), "operands of one dim block");
#pragma unroll
                for (int t = 0; t < RT; ++t)
#pragma unroll
                    for (int x = 0; x < 8; ++x) sp[512 * t + 64 * x + lane] = word4(pf[t][x / 4], x % 4);
#pragma unroll
                for (int d = 0; d < NB; ++d) {
                    __builtin_amdgcn_wave_barrier();
#pragma unroll
                    for (int x = 0; x < 8; ++x) sv[64 * x + lane] = word4(vf[d][x / 4], x % 4);
                    __builtin_amdgcn_wave_barrier();
#pragma unroll 1
                    for (int key = 0; key < 32; ++key) {
                        const int at = 64 * (4 * (key >> 4) + ((key & 7) >> 1)) + 32 * ((key >> 3) & 1), sh = 16 * (key & 1);
#pragma unroll
                        for (int t = 0; t < RT; ++t) {
                            const float p = h2f((uint16_t)(sp[512 * t + at + c] >> sh));
                            if ((vis[t] >> key) & 1)
#pragma unroll
                                for (int i = 0; i < 16; ++i)
                                    O[t][d][i] += p * h2f((uint16_t)(sv[at + 8 * (i / 4) + 4 * h + i % 4] >> sh));
                        }
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int d = 0; d < NB; ++d)
#pragma unroll
                        for (int t = 0; t < RT; ++t) O[t][d] = mfma32<false>(vf[d][i], pf[t][i], O[t][d]);
            }
            load_v(pn);
            pg = pn;
            pn = after;
        }
        if (careful || !some_masked) break;
        bool bad = false;
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int d = 0; d < NB; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) bad = bad || !(fabsf(O[t][d][i]) < INFINITY);
        if (__builtin_amdgcn_ballot_w64(bad) == 0) break;
        careful = true;
    }

    // merge the waves: row c of row tile t, MD dims at a time
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const float lt = sum_halves(l[t]);
        if (h == 0) s_m[wave][32 * t + c] = m[t], s_l[wave][32 * t + c] = lt;
    }
    float *slot = a.part + ((((int64_t)s * a.KV + hk) * a.RB + rb) * a.P + part) * (32 * RT) * (D + 4);
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int d0 = 0; d0 < NB; d0 += MD / 32) {
            if (t + d0 > 0) lds_barrier();  // the last part has been read
#pragma unroll
            for (int d = d0; d < d0 + MD / 32 && d < NB; ++d)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    *(float4 *)&s_o[wave][c][32 * (d - d0) + 8 * j + 4 * h] =
                        make_float4(O[t][d][4 * j], O[t][d][4 * j + 1], O[t][d][4 * j + 2], O[t][d][4 * j + 3]);
            lds_barrier();
            for (int e = threadIdx.x; e < 32 * (MD / 4); e += 64 * TA_WAVES) {
                const int row = e / (MD / 4), dd = 4 * (e % (MD / 4)), dim = 32 * d0 + dd, rr = r0 + 32 * t + row;
                if (rr >= R || dim >= D) continue;
                float M = -INFINITY;
#pragma unroll
                for (int w = 0; w < TA_WAVES; ++w) M = fmaxf(M, s_m[w][32 * t + row]);
                float sum = 0.0f;
                float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < TA_WAVES; ++w) {
                    const float mw = s_m[w][32 * t + row];
                    const float f = mw == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((mw - M) * a.cs);
                    const float4 x = *(const float4 *)&s_o[w][row][dd];
                    if (mw == -INFINITY && !(s_l[w][32 * t + row] != 0.0f)) continue;  // saw nothing
                    sum += f * s_l[w][32 * t + row];
                    o.x += f * x.x, o.y += f * x.y, o.z += f * x.z, o.w += f * x.w;
                }
                if (a.P == 1) {
                    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                    uint16_t *dst = a.out + ((int64_t)(sq.b + rr / a.G) * a.H + hk * a.G + rr % a.G) * D + dim;
                    const float x[8] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv, 0, 0, 0, 0};
                    const uint4 w = pack8<false>(x);
                    *(uint2 *)dst = make_uint2(w.x, w.y);
                } else {
                    float *dst = slot + (int64_t)(32 * t + row) * (D + 4);
                    *(float4 *)(dst + 4 + dim) = o;
                    if (dim == 0) *(float2 *)dst = make_float2(M, sum);
                }
            }
        }
}

// One wave a row: lane p holds partition p's weight, the lanes then take the dims.
template <int D>
__global__ void __launch_bounds__(256) k_tree_attn_merge(const TaArgs a, int rows_a_block) {
    const int lane = threadIdx.x & 63;
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6), hk = blockIdx.y, s = blockIdx.z;
    const TaSeq sq = ta_seq(a, s);
    if (row >= sq.n * a.G) return;
    const int np = (sq.L + a.part_len - 1) / a.part_len;
    const int64_t step = (int64_t)rows_a_block * (D + 4);
    const float *base = a.part + ((((int64_t)s * a.KV + hk) * a.RB + row / rows_a_block) * a.P) * step +
                        (int64_t)(row % rows_a_block) * (D + 4);
    float2 ml = make_float2(-INFINITY, 0.0f);
    if (lane < np) ml = *(const float2 *)(base + lane * step);
    float M = ml.x;
    for (int o = 1; o < 64; o <<= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    const float w = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((ml.x - M) * a.cs);
    float sum = w * ml.y;
    for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    constexpr int E = (D + 63) / 64;
    float acc[E] = {};
    for (int p = 0; p < np; ++p) {
        const float wp = __shfl(w, p, 64);
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (lane + 64 * e < D) acc[e] += wp * base[p * step + 4 + lane + 64 * e];
    }
    uint16_t *dst = a.out + ((int64_t)(sq.b + row / a.G) * a.H + hk * a.G + row % a.G) * D;
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (lane + 64 * e < D) dst[lane + 64 * e] = f2h(acc[e] * inv);
}

// Row tiles a wave: two where a sequence may have more than 32 rows (the second
// one's products use the same key and value registers), if they fit.
static int ta_row_tiles(const tlh_tree_attention_args &a) {
    return a.head_size <= 128 && a.max_drafts * (a.num_heads / a.num_kv_heads) > 32 ? 2 : 1;
}
static int64_t ta_row_blocks(const tlh_tree_attention_args &a) {
    const int64_t per = 32 * ta_row_tiles(a);
    return ((int64_t)a.max_drafts * (a.num_heads / a.num_kv_heads) + per - 1) / per;
}
static int64_t ta_rounds(const tlh_tree_attention_args &a) { return ((int64_t)a.max_context_len + TA_KEYS - 1) / TA_KEYS; }
// partitions: as many as make TA_WGS workgroups, each of at least one round of keys
static int ta_parts(const tlh_tree_attention_args &a, int &part_len) {
    const int64_t base = (int64_t)a.num_seqs * a.num_kv_heads * ta_row_blocks(a);
    const int64_t rounds = std::max<int64_t>(ta_rounds(a), 1);
    const int64_t want = std::max<int64_t>(1, std::min<int64_t>({TA_WGS / std::max<int64_t>(base, 1), TA_MAX_PARTS, rounds}));
    const int64_t each = (rounds + want - 1) / want;
    part_len = (int)(each * TA_KEYS);
    return (int)((rounds + each - 1) / each);
}

// A slot of 32 RT rows a workgroup. Counted so that the size never shrinks as
// any of the counts grows: one buffer for the largest call serves every smaller one.
size_t tree_attention_scratch_bytes(const tlh_tree_attention_args &a) {
    if (ta_rounds(a) <= 1) return 0;
    const int64_t base = (int64_t)a.num_seqs * a.num_kv_heads * ta_row_blocks(a);
    const int64_t slots = std::min(base * std::min<int64_t>(ta_rounds(a), TA_MAX_PARTS), base + TA_WGS);
    return (size_t)slots * 32 * ta_row_tiles(a) * (a.head_size + 4) * sizeof(float);
}

template <int D, int BS, int RT> static void launch_ta3(const TaArgs &t, unsigned blocks, hipStream_t stream) {
    hipLaunchKernelGGL((k_tree_attn<D, BS, RT>), dim3(blocks), dim3(64 * TA_WAVES), 0, stream, t);
}
template <int D, int BS> static void launch_ta2(const TaArgs &t, int rt, unsigned blocks, hipStream_t stream) {
    if constexpr (D <= 128) {
        if (rt == 2) return launch_ta3<D, BS, 2>(t, blocks, stream);
    }
    launch_ta3<D, BS, 1>(t, blocks, stream);
}
template <int D> static void launch_ta(const TaArgs &t, int bs, int rt, unsigned blocks, hipStream_t stream) {
    switch (bs) {
    case 8: launch_ta2<D, 8>(t, rt, blocks, stream); break;
    case 16: launch_ta2<D, 16>(t, rt, blocks, stream); break;
    default: launch_ta2<D, 32>(t, rt, blocks, stream); break;
    }
    if (t.P > 1)
        hipLaunchKernelGGL((k_tree_attn_merge<D>), dim3((t.max_drafts * t.G + 3) / 4, t.KV, t.S), dim3(256), 0, stream, t,
                           32 * rt);
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
    const int rt = ta_row_tiles(a);
    const int64_t rb = ta_row_blocks(a);
    t.P = ta_parts(a, t.part_len);
    t.RB = (int)rb;
    t.cs = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * 1.4426950408889634f;
    t.qand = a.scale == 0.0f ? 0u : ~0u, t.qxor = a.scale < 0.0f ? 0x80008000u : 0u;
    const int64_t blocks = (int64_t)t.P * t.S * rb * t.KV;
    if (blocks > INT32_MAX) return set_error(TLH_INVALID, "tree_attention: too many sequences and heads for one launch");
    switch (a.head_size) {
    case 64: launch_ta<64>(t, a.block_size, rt, (unsigned)blocks, stream); break;
    case 80: launch_ta<80>(t, a.block_size, rt, (unsigned)blocks, stream); break;
    case 96: launch_ta<96>(t, a.block_size, rt, (unsigned)blocks, stream); break;
    case 112: launch_ta<112>(t, a.block_size, rt, (unsigned)blocks, stream); break;
    case 128: launch_ta<128>(t, a.block_size, rt, (unsigned)blocks, stream); break;
    case 192: launch_ta<192>(t, a.block_size, rt, (unsigned)blocks, stream); break;
    default: launch_ta<256>(t, a.block_size, rt, (unsigned)blocks, stream); break;
    }
    return check_launch("tree_attention");
}

}  // namespace tlh
