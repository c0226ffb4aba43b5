// Causal attention of whole prompts packed one after another, gfx950.
//
//   q [tokens][heads][D], k and v [tokens][kv_heads][D], out as q (f16 or bf16;
//   rows of heads contiguous, any token stride), seq_starts [num_seqs + 1]:
//   out[t, h] = sum_j softmax_j(scale * q[t, h] . k[j, h / G]) v[j, h / G]
//   over the tokens j <= t of t's own sequence.
//
// Bound by the matrix cores and, beside them, by the exponentials: 4 D flops a
// visible (query, key) pair. A workgroup of four waves takes gw heads of one kv
// head (gw = 4, 2 or 1, what divides the group) and 4 / gw blocks of 32 queries;
// a wave owns 32 query rows of one head. The keys come in tiles that all four
// waves read from LDS, double-buffered and loaded straight from global memory
// (no registers between), the 16-byte chunks of a row permuted so that both
// products' operands are read without bank conflicts:
//   S^T = K . Q^T   a lane holds one query's scores, so the running maximum and
//                   sum cost one exchange with lane l ^ 32 a tile;
//   O^T += V^T . P^T  P comes from S^T's registers as they are; V^T from LDS by
//                   transposing reads of four keys x 16 dims.
// Workgroups are ordered by sequence, then by query position, last first (they see
// the most keys), then by kv head: those that run together read the same K and V,
// and with 8 kv heads a head's stay in one XCD's L2. (By position first, which
// ends more evenly, 16 prompts of 100..2000 took 400 us instead of 300.)
//
// Measured: one prompt of 8191 tokens, 32/8 heads of 128, bf16, 559 to 608 us, 900 to 980
// TFLOP/s (a library product of 8192^3 reaches 1145 on this card); 16 prompts of
// 100..2000 264 to 279 us, 690 TFLOP/s, in any order of their lengths; heads of 64 (8191
// tokens) 334 to 353 us, 780 to 820; of 256 (4000 tokens, 16/8 heads) 252 us, 520.
//
// The softmax is lazy: the exponents' reference moves only when a row's maximum
// has grown by more than 2^8, so most tiles rescale nothing. In f16 it is set below
// the maximum (F16_LIFT): numerators of up to 2^15. It does not change the quotient
// (bf16's sums of products that leave f32's range for it are taken again, smaller).
#include <algorithm>

#include "mfma32.hpp"

namespace tlh {

constexpr float PK_LOG2E = 1.4426950408889634f;
constexpr float PK_BF_DROP = 40.0f;  // see the careful pass

template <int D> struct PkGeom {
    static constexpr int KT = D <= 128 ? 64 : 32;                 // keys per tile
    static constexpr int CP = D <= 64 ? 8 : D <= 128 ? 16 : 32;  // 16-byte chunks of a row in LDS (a power of two)
    static constexpr int C = D / 8;                              // ... and in memory
    static constexpr int TILE = KT * CP * 16;                    // bytes of a tile's K or V
    static constexpr int NB = (D + 31) / 32;                     // 32-dim blocks of O^T
    static constexpr int ND = TILE / 4096;                       // 1-KiB loads a wave makes for K (or V)
    // The chunk of key kk's row that position pos holds is pos ^ swizzle. K: eight consecutive
    // keys' reads of one chunk fall on eight different 16-byte bank groups.
    __device__ static int kswz(int kk) { return CP == 8 ? (kk >> 1) & 7 : kk & 15; }
    // V: the 32-byte pieces that 32 lanes read (four keys, two neighbouring pieces) likewise.
    __device__ static int vswz(int kk) { return CP == 8 ? ((kk >> 1) & 1) << 2 : (kk & 3) << 2; }
};

struct PkArgs {
    uint8_t *out;
    const uint8_t *q, *k, *v;
    const int32_t *starts;
    int64_t so, sq, sk, sv;  // bytes from token to token
    int S, tokens, max_len, G, gw, HG, levels;
    float cs;             // |scale| * log2(e); 1 where the scale is 0
    float lift;           // how far below the maximum the exponents' reference is set, in scores (bf16: carefully)
    uint32_t qand, qxor;  // q's words: negated where the scale is negative, zeroed where it is 0
};

template <int D, bool BF>
__global__ void __launch_bounds__(256, D <= 128 ? 2 : 1) k_packed_attn(const PkArgs a) {
    using Gm = PkGeom<D>;
    constexpr int KT = Gm::KT, CP = Gm::CP, KB = KT / 32, NB = Gm::NB, NS = D / 16;
    __shared__ __attribute__((aligned(16))) uint8_t T0[2 * Gm::TILE], T1[2 * Gm::TILE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = lane >> 5, c = lane & 31;
    // workgroup -> (sequence; query tile, last first; group of heads)
    const int hg = blockIdx.x % a.HG;
    const int qt = a.levels - 1 - (int)(blockIdx.x / a.HG);
    const int s = blockIdx.y;
    const int b0 = max(0, min(a.starts[s], a.tokens)), b1 = max(0, min(a.starts[s + 1], a.tokens));
    const int n = min(b1 - b0, a.max_len);
    const int qpw = 32 * (4 / a.gw);
    if (qt * qpw >= n) return;
    const int per = a.G / a.gw;  // workgroups of a kv head
    const int hk = hg / per, head = hk * a.G + (hg % per) * a.gw + wave % a.gw;
    const int q0 = qt * qpw + 32 * (wave / a.gw);  // the wave's first query
    const int qi = q0 + c;                         // this lane's
    const uint8_t *kb = a.k + (int64_t)b0 * a.sk + (int64_t)hk * D * 2;
    const uint8_t *vb = a.v + (int64_t)b0 * a.sv + (int64_t)hk * D * 2;
    const int ntiles = (min(n, qt * qpw + qpw) + KT - 1) / KT;

    // Tile loads: load i of wave w fills 1 KiB: keys from (4 i + w) 64 / CP on, lane l
    // key l / CP of them at position l % CP. Positions past a row's last chunk
    // repeat chunk 0 (read only into output dims that are not stored); keys past
    // the sequence repeat its last (masked).
    const int lk = lane / CP, lp = lane % CP;
    auto load_tile = [&](int t, uint8_t *T) {
#pragma unroll
        for (int i = 0; i < Gm::ND; ++i) {
            const int kk = (4 * i + wave) * (64 / CP) + lk;
            const int64_t key = min(t * KT + kk, n - 1);
            int ck = lp ^ Gm::kswz(kk), cv = lp ^ Gm::vswz(kk);
            if (Gm::C < CP) ck = ck < Gm::C ? ck : 0, cv = cv < Gm::C ? cv : 0;
            to_lds(kb + key * a.sk + 16 * ck, T + (4 * i + wave) * 1024);
            to_lds(vb + key * a.sv + 16 * cv, T + Gm::TILE + (4 * i + wave) * 1024);
        }
    };

    f32x16 O[NB];
    float m, l;  // this lane's query: the exponents' reference (an unscaled score); this half's sum
    load_tile(0, T0);
    // Q as the lanes take it: in registers, above 192 dims (where O leaves none: 4000
    // tokens, 16/8 heads of 256, 392 us with it in registers, 256 without) in LDS
    constexpr bool QREG = D <= 192;
    __shared__ uint4 s_q[QREG ? 1 : 4][QREG ? 1 : NS][QREG ? 1 : 64];
    uint4 qf[QREG ? NS : 1];
    {
        const uint8_t *qr = a.q + (int64_t)(b0 + min(qi, n - 1)) * a.sq + (int64_t)head * D * 2 + 16 * h;
#pragma unroll
        for (int st = 0; st < NS; ++st) {
            const uint4 w = *(const uint4 *)(qr + 32 * st);
            const uint4 q = make_uint4((w.x & a.qand) ^ a.qxor, (w.y & a.qand) ^ a.qxor, (w.z & a.qand) ^ a.qxor,
                                       (w.w & a.qand) ^ a.qxor);
            if constexpr (QREG) qf[st] = q;
            else s_q[wave][st][lane] = q;
        }
    }
    // a transposing read takes key tr_key of four and 4 of 16 dims from each of 16
    // lanes and gives a lane one dim of the four keys
    const int tr_key = (lane & 15) >> 2;
    const int tr_chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    const int tr_at = (4 * h + tr_key) * CP * 16 + 8 * (lane & 1);
    // A value that is not finite would turn the zero weight of a masked key into NaN.
    // So where a result comes out not finite, the pass is run again, carefully: tiles
    // with masked keys then add each visible key's product by itself. In bf16, whose
    // values reach the end of f32's range, the sums of products may also have left it:
    // the reference is then set 40 above a row's maximum, so that the numerators of 2^31
    // keys, each below 2^-32, come to less than 1, and no sum to more than the largest value.
    bool careful = false;
    float lift = BF ? 0.0f : a.lift, top = BF ? 8.0f : 8.0f + F16_LIFT;

    auto tile = [&](int t, const uint8_t (&T)[2 * Gm::TILE], uint8_t (&Tn)[2 * Gm::TILE]) {
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): tile t has landed
        lds_barrier();                       // for every wave, and the other buffer is free
        if (t + 1 < ntiles) load_tile(t + 1, Tn);
        const int k0 = t * KT;
        if (k0 > q0 + 31) return;  // nothing visible to the wave's queries
        f32x16 S[KB];
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            S[b] = (f32x16){};
            const int kk = 32 * b + c;
#pragma unroll
            for (int st = 0; st < NS; ++st)
                S[b] = mfma32<BF>(*(const uint4 *)(T + kk * CP * 16 + 16 * ((2 * st + h) ^ Gm::kswz(kk))),
                                  QREG ? qf[QREG ? st : 0] : s_q[QREG ? 0 : wave][QREG ? 0 : st][QREG ? 0 : lane], S[b]);
        }
        const bool diagonal = k0 + KT - 1 > q0;  // some key lies after some query
        if (diagonal) {
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (k0 + 32 * b + 8 * (i / 4) + 4 * h + i % 4 > qi) S[b][i] = -INFINITY;
        }
        float mx = S[0][0];
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, S[b][i]);
        mx = max_halves(mx);
        const bool grow = mx > -INFINITY && !((mx - m) * a.cs <= top);
        if (__builtin_amdgcn_ballot_w64(grow) != 0) {
            const float ref = mx - lift;
            const float alpha = grow ? __builtin_amdgcn_exp2f((m - ref) * a.cs) : 1.0f;
            m = grow ? ref : m;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < NB; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) O[d][i] *= alpha;
        }
        const float mc = m == -INFINITY ? 0.0f : m * a.cs;
        uint4 pf[2 * KB];
        float sum = 0.0f;
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int i = 0; i < 16; i += 8) {
                float p[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(S[b][i + e] * a.cs - mc);
                sum += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
                pf[2 * b + i / 8] = pack8<BF>(p);
            }
        l += sum;
        if (careful && diagonal) {
#pragma unroll 1
            for (int kk = 0; kk < KT; ++kk) {
                const int e = 4 * ((kk >> 3) & 1) + (kk & 3), w = 4 * (kk >> 4) + (e >> 1);
                uint32_t pw = 0;
#pragma unroll
                for (int x = 0; x < 8 * KB; ++x) pw = x == w ? word4(pf[x / 4], x % 4) : pw;
                pw = __shfl(pw, c + 32 * ((kk >> 2) & 1), 64);
                const float p = unpack16<BF>(e & 1 ? pw >> 16 : pw & 0xffffu);
                if (k0 + kk > qi) continue;
#pragma unroll
                for (int d = 0; d < NB; ++d)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint2 v = *(const uint2 *)(T + Gm::TILE + kk * CP * 16 +
                                                         16 * ((4 * d + j) ^ Gm::vswz(kk)) + 8 * h);
                        O[d][4 * j] += p * unpack16<BF>(v.x & 0xffffu);
                        O[d][4 * j + 1] += p * unpack16<BF>(v.x >> 16);
                        O[d][4 * j + 2] += p * unpack16<BF>(v.y & 0xffffu);
                        O[d][4 * j + 3] += p * unpack16<BF>(v.y >> 16);
                    }
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < 2 * KB; ++i)
#pragma unroll
            for (int d = 0; d < NB; ++d) {
                const uint8_t *va = T + Gm::TILE + tr_at + 16 * ((4 * d + tr_chunk) ^ Gm::vswz(tr_key)) + 16 * i * CP * 16;
                const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)va);
                const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(va + 8 * CP * 16));
                const uint2 vl = __builtin_bit_cast(uint2, lo), vh = __builtin_bit_cast(uint2, hi);
                O[d] = mfma32<BF>(make_uint4(vl.x, vl.y, vh.x, vh.y), pf[i], O[d]);
            }
    };

    for (;;) {
#pragma unroll
        for (int d = 0; d < NB; ++d) O[d] = (f32x16){};
        m = -INFINITY;
        l = 0.0f;
        for (int t = 0; t < ntiles; t += 2) {
            tile(t, T0, T1);
            if (t + 1 < ntiles) tile(t + 1, T1, T0);
        }
        const float inv = 1.0f / sum_halves(l);
        bool bad = false;
#pragma unroll
        for (int d = 0; d < NB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                O[d][i] *= inv;
                // (past the last dim: repeats of other dims' values)
                if (32 * d + 8 * (i / 4) < D) bad = bad || !(fabsf(O[d][i]) < INFINITY);
            }
        if (careful) {
            lds_barrier();
            break;
        }
        int *flags = (int *)T0;
        const int mine = __builtin_amdgcn_ballot_w64(bad && qi < n) != 0;
        lds_barrier();
        if (lane == 0) flags[wave] = mine;
        lds_barrier();
        const bool any = (flags[0] | flags[1] | flags[2] | flags[3]) != 0;
        lds_barrier();
        if (!any) break;
        careful = true;
        if (BF) lift = a.lift, top = 8.0f - PK_BF_DROP;
        int again = 0;
        asm volatile("" : "+s"(again));  // its addresses formed here: kept from the start, they spill
        load_tile(again, T0);
    }
    // The wave's 32 rows leave through its quarter of the buffers (free since the
    // flags' barriers), so that a row is written in one piece: 16-byte chunks of row r
    // at position chunk ^ (r % CP), then whole rows, 64 / CP at a time.
    uint8_t *R = (wave & 2 ? T1 : T0) + (wave & 1) * Gm::TILE;
    static_assert(32 * CP * 16 <= Gm::TILE, "a wave's rows");
#pragma unroll
    for (int d = 0; d < NB; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (32 * d + 8 * j >= D) continue;
            const float x[8] = {O[d][4 * j], O[d][4 * j + 1], O[d][4 * j + 2], O[d][4 * j + 3], 0, 0, 0, 0};
            const uint4 w = pack8<BF>(x);
            *(uint2 *)(R + c * CP * 16 + 16 * ((4 * d + j) ^ (c & (CP - 1))) + 8 * h) = make_uint2(w.x, w.y);
        }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < CP / 2; ++i) {
        const int r = i * (64 / CP) + lk, chunk = lp ^ (r & (CP - 1));
        if (q0 + r < n && (Gm::C == CP || chunk < Gm::C))
            *(uint4 *)(a.out + (int64_t)(b0 + q0 + r) * a.so + (int64_t)head * D * 2 + 16 * chunk) =
                *(const uint4 *)(R + r * CP * 16 + 16 * lp);
    }
}

template <int D> static tlh_status launch_pk(PkArgs p, bool bf, hipStream_t stream) {
    for (int left = p.S; left > 0; left -= 65535, p.starts += 65535) {  // grid y
        const dim3 grid((unsigned)(p.HG * p.levels), std::min(left, 65535));
        if (bf) hipLaunchKernelGGL((k_packed_attn<D, true>), grid, dim3(256), 0, stream, p);
        else hipLaunchKernelGGL((k_packed_attn<D, false>), grid, dim3(256), 0, stream, p);
        const tlh_status st = check_launch("packed_attention");
        if (st != TLH_OK) return st;
    }
    return TLH_OK;
}

tlh_status launch_packed_attention(const tlh_packed_attention_args &a, hipStream_t stream) {
    const int G = a.num_heads / a.num_kv_heads;
    PkArgs p = {};
    p.out = (uint8_t *)a.out, p.q = (const uint8_t *)a.q, p.k = (const uint8_t *)a.k, p.v = (const uint8_t *)a.v;
    p.starts = a.seq_starts;
    p.so = 2 * a.out_stride, p.sq = 2 * a.q_stride, p.sk = 2 * a.k_stride, p.sv = 2 * a.v_stride;
    p.S = a.num_seqs, p.tokens = a.num_tokens, p.G = G;
    p.max_len = std::min(a.max_seq_len, a.num_tokens);
    p.gw = G % 4 == 0 ? 4 : G % 2 == 0 ? 2 : 1;
    p.HG = a.num_heads / p.gw;
    const int qpw = 32 * (4 / p.gw);
    p.levels = (p.max_len - 1) / qpw + 1;
    p.cs = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * PK_LOG2E;
    p.lift = a.type == TLH_TYPE_BF16 ? -std::min(PK_BF_DROP / p.cs, 1e30f) : f16_lift(p.cs);
    p.qand = a.scale == 0.0f ? 0u : ~0u, p.qxor = a.scale < 0.0f ? 0x80008000u : 0u;
    if ((int64_t)p.levels * p.HG >= 1 << 24)  // x 256 threads
        return set_error(TLH_INVALID, "packed_attention: max_seq_len x num_heads too large for one launch");
    const bool bf = a.type == TLH_TYPE_BF16;
    switch (a.head_size) {
    case 64: return launch_pk<64>(p, bf, stream);
    case 80: return launch_pk<80>(p, bf, stream);
    case 96: return launch_pk<96>(p, bf, stream);
    case 112: return launch_pk<112>(p, bf, stream);
    case 128: return launch_pk<128>(p, bf, stream);
    case 192: return launch_pk<192>(p, bf, stream);
    default: return launch_pk<256>(p, bf, stream);
    }
}

}  // namespace tlh
