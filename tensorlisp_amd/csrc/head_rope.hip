// The norms of query and key heads, their rotation by the tokens' positions and the
// write of keys and values to a paged cache, in one pass, gfx950. A head x of D dims:
//   y = x / sqrt(mean(x^2) + eps) * w   (with a norm; else y = x)
//   (y_a, y_b) -> (y_a cos t - y_b sin t, y_a sin t + y_b cos t), times attn_factor,
//   for the pairs p < n_dims / 2 of its dims, t = positions[pair_axis[p]][token] freqs[p].
//
// Bound by HBM: every head is read once and written once. A workgroup takes a few
// consecutive tokens and a group of heads, a head a power of two of lanes:
//  * a lane holds dims 4 c .. + 3 and D / 2 + 4 c .. + 3, so that the two of a pair are in
//    one lane in either mode (rotating a part of the dims in mode 2, they pass through LDS);
//  * a lane's angles are formed once for all its heads. t reaches 10^5 and more, where f32
//    leaves hundredths of a radian: it is formed in turns in 64 bits (t / 2 pi), reduced to
//    its fraction there and only then taken to f32;
//  * a value page holds a dim's tokens next to each other: the values pass through LDS, and
//    consecutive lanes write consecutive tokens.
// Norms and rotation are f32, and a head is rounded once, to the type it is written in.
// Measured against a wave for a (token, head), which forms its angles for each and writes
// values two bytes a page line, with the same inputs again: 2501 tokens of 28 + 4 + 4 heads of
// 128 in bf16 (46 MB) 37 -> 13 us; 8192 tokens of 32 + 8 + 8 of 128 in f32 (302 MB) 230 -> 74 us.
// With inputs that no cache holds 19 us (2.4 TB/s: the angles, formed anew for each group of
// heads, are not hidden) and 86 us (3.5 TB/s, where a large copy reaches 4.9). 2048 tokens of
// 32 + 8 + 8 in bf16 take 15 and 22 us, rotating half of a head in mode 2, where each of a
// pair's lanes forms its angle, 17 and 23.
#include <algorithm>

#include "kernels.hpp"
#include "wave_ops.hpp"

namespace tlh {

// Workgroups that the heads are split for: more of them form the same angles more often,
// fewer leave CUs empty (from memory, us, with 512, 1024, 2048, 4096: 512 tokens of 32 + 8 +
// 8 heads of 128 in f32 10.9, 9.9, 9.8, 9.8; 2501 31.7, 25.6, 28.5, 27.5; 8192 107, 73, 74, 68;
// 2501 of 28 + 4 + 4 in bf16 23.8, 19.4, 18.1, 21.6).
constexpr int HR_WGS = 1024;

struct HrArgs {
    const uint8_t *q, *k, *v;
    uint8_t *qo, *ko, *vo;
    uint16_t *kc, *vc;
    const int32_t *positions;
    const float *freqs, *qw, *kw;
    const int64_t *slots;
    int64_t sq, sk, sv, soq, sok, sov;  // bytes from token to token
    int64_t pool_slots;
    int64_t first;                      // the launch's first token
    int tokens, H, KV, D, lg_bs, pairs, mode;
    int lg_tg;                          // tokens of a workgroup, a power of two
    int per, groups, per_v;             // query and key heads of a workgroup, their groups; value heads
    int heads;                          // query heads, and key heads where they go anywhere
    float eps, factor;
    uint8_t axis[128];
};

// four elements from element d on
template <int TY> __device__ __forceinline__ void hr_load4(const uint8_t *p, int d, float *x) {
    if constexpr (TY == TLH_TYPE_F32) {
        const float4 w = *(const float4 *)(p + 4 * d);
        x[0] = w.x, x[1] = w.y, x[2] = w.z, x[3] = w.w;
    } else {
        const uint2 w = *(const uint2 *)(p + 2 * d);
        const uint32_t ws[2] = {w.x, w.y};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint16_t h = (uint16_t)(ws[i / 2] >> (16 * (i & 1)));
            x[i] = TY == TLH_TYPE_F16 ? h2f(h) : bf16_to_f32(h);
        }
    }
}
template <bool BF> __device__ __forceinline__ uint2 hr_pack4(const float *x) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        w[i] = BF ? (uint32_t)f32_to_bf16(x[2 * i]) | (uint32_t)f32_to_bf16(x[2 * i + 1]) << 16
                  : (uint32_t)f2h(x[2 * i]) | (uint32_t)f2h(x[2 * i + 1]) << 16;
    return make_uint2(w[0], w[1]);
}

// LANES: of a head, the least power of two of at least D / 8. PART: mode 2 that rotates
// less than the whole head.
template <int TY, bool BF, int LANES, bool PART> __global__ void __launch_bounds__(256) k_head_rope(const HrArgs a) {
    constexpr int AT_ONCE = 256 / LANES, ROW = 8 * LANES + 4;  // heads that the workgroup takes at a time
    __shared__ __attribute__((aligned(16))) float s_x[AT_ONCE][ROW];
    const int col = threadIdx.x % LANES, g = threadIdx.x / LANES, D = a.D;
    const int t = g & ((1 << a.lg_tg) - 1), step = AT_ONCE >> a.lg_tg;
    const int64_t token = a.first + ((int64_t)blockIdx.x << a.lg_tg) + t;
    const int da = 4 * col, db = D / 2 + 4 * col;
    const bool live = token < a.tokens && da < D / 2;

    if ((int)blockIdx.y >= a.groups) {  // values
        constexpr int VROW = 8 * LANES + 2;  // 16-bit elements; consecutive rows in different banks
        static_assert(VROW * 2 <= ROW * 4, "a row of values");
        uint16_t *s_v = (uint16_t *)&s_x[0][0];
        const int h0 = (blockIdx.y - a.groups) * a.per_v, h1 = min(h0 + a.per_v, a.KV), tg = 1 << a.lg_tg;
        // of the place that this thread writes, the token in the workgroup
        const int wt = threadIdx.x & (tg - 1);
        const int64_t wtoken = token - t + wt;
        int64_t slot = -1;
        if (a.vc && wtoken < a.tokens) slot = a.slots[wtoken];
        if (slot >= a.pool_slots) slot = -1;
        for (int h = h0; h < h1; h += step) {
            const int mine = h + (g >> a.lg_tg);
            float x[8] = {};
            if (live && mine < h1) {
                const uint8_t *p = a.v + token * a.sv + (int64_t)mine * D * (TY == TLH_TYPE_F32 ? 4 : 2);
                hr_load4<TY>(p, da, x);
                hr_load4<TY>(p, db, x + 4);
            }
            const uint2 lo = hr_pack4<BF>(x), hi = hr_pack4<BF>(x + 4);
            if (a.vo && live && mine < h1) {
                uint8_t *o = a.vo + token * a.sov + (int64_t)mine * D * 2;
                *(uint2 *)(o + 2 * da) = lo;
                *(uint2 *)(o + 2 * db) = hi;
            }
            if (!a.vc) continue;
            if (h > h0) __syncthreads();
            if (da < D / 2) {
                uint32_t *row = (uint32_t *)(s_v + g * VROW);
                row[da / 2] = lo.x, row[da / 2 + 1] = lo.y, row[db / 2] = hi.x, row[db / 2 + 1] = hi.y;
            }
            __syncthreads();
            if (slot < 0) continue;
            uint16_t *page = a.vc + ((slot >> a.lg_bs) * a.KV * D << a.lg_bs) + (slot & ((1 << a.lg_bs) - 1));
            for (int i = threadIdx.x >> a.lg_tg; i < step * 8 * LANES; i += 256 >> a.lg_tg) {
                const int hs = i / (8 * LANES), d = i % (8 * LANES);
                if (d < D && h + hs < h1) page[((int64_t)(h + hs) * D + d) << a.lg_bs] = s_v[((hs << a.lg_tg) + wt) * VROW + d];
            }
        }
        return;
    }

    // this lane's angles: of the pairs (x[i], x[i + 4]) in mode 2, of (x[2 i], x[2 i + 1]) in
    // mode 0; PART: of each of its elements
    constexpr int ANGLES = PART ? 8 : 4;
    float cs[ANGLES], sn[ANGLES];
#pragma unroll
    for (int i = 0; i < ANGLES; ++i) {
        int p;
        if (PART) {
            const int d = (i < 4 ? da : db - 4) + i;
            p = d < a.pairs ? d : d - a.pairs;
        } else p = a.mode ? da + i : (i < 2 ? da : db - 4) / 2 + i;
        cs[i] = 1.0f, sn[i] = 0.0f;
        if (live && p < a.pairs) {
            const int position = a.positions[(int64_t)a.axis[p] * a.tokens + token];
            const double turns = (double)position * ((double)a.freqs[p] * 0.15915494309189533577);
            sincospif(2.0f * (float)(turns - rint(turns)), &sn[i], &cs[i]);
            sn[i] *= a.factor, cs[i] *= a.factor;
        }
    }
    int64_t slot = -1;
    if (a.kc && live) slot = a.slots[token];
    if (slot >= a.pool_slots) slot = -1;
    const int h0 = blockIdx.y * a.per, h1 = min(h0 + a.per, a.heads);
    const float rD = 1.0f / (float)D;
    float next[8] = {};
    auto load = [&](int h) {
        if (!live || h >= h1) return;
        const bool query = h < a.H;
        const uint8_t *p = query ? a.q + token * a.sq : a.k + token * a.sk;
        p += (int64_t)(query ? h : h - a.H) * D * (TY == TLH_TYPE_F32 ? 4 : 2);
        hr_load4<TY>(p, da, next);
        hr_load4<TY>(p, db, next + 4);
    };
    load(h0 + (g >> a.lg_tg));
    for (int hb = h0; hb < h1; hb += step) {
        const int h = hb + (g >> a.lg_tg);
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = next[i];
        load(h + step);
        const bool query = h < a.H;
        const float *w = query ? a.qw : a.kw;
        if (w) {
            float s = ((x[0] * x[0] + x[1] * x[1]) + (x[2] * x[2] + x[3] * x[3])) + ((x[4] * x[4] + x[5] * x[5]) + (x[6] * x[6] + x[7] * x[7]));
            s = wave_all(s, LANES, [](float u, float v) { return u + v; });
            const float inv = 1.0f / sqrtf(s * rD + a.eps);
            if (live) {
                const float4 wa = *(const float4 *)(w + da), wb = *(const float4 *)(w + db);
                x[0] *= inv * wa.x, x[1] *= inv * wa.y, x[2] *= inv * wa.z, x[3] *= inv * wa.w;
                x[4] *= inv * wb.x, x[5] *= inv * wb.y, x[6] *= inv * wb.z, x[7] *= inv * wb.w;
            }
        }
        float y[8];
        if constexpr (PART) {
            float *row = s_x[g];
            __builtin_amdgcn_wave_barrier();
            if (da < D / 2) {
                *(float4 *)(row + da) = make_float4(x[0], x[1], x[2], x[3]);
                *(float4 *)(row + db) = make_float4(x[4], x[5], x[6], x[7]);
            }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int d = (i < 4 ? da : db - 4) + i;
                const float o = d < 2 * a.pairs ? row[d < a.pairs ? d + a.pairs : d - a.pairs] : 0.0f;
                y[i] = d < a.pairs ? x[i] * cs[i] - o * sn[i] : d < 2 * a.pairs ? o * sn[i] + x[i] * cs[i] : x[i];
            }
        } else if (a.mode) {
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = x[i] * cs[i] - x[i + 4] * sn[i], y[i + 4] = x[i] * sn[i] + x[i + 4] * cs[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // (one that is not rotated passes through: 0 times an infinity beside it would be NaN)
                const bool turns = (i < 2 ? da : db - 4) / 2 + i < a.pairs;
                y[2 * i] = turns ? x[2 * i] * cs[i] - x[2 * i + 1] * sn[i] : x[2 * i];
                y[2 * i + 1] = turns ? x[2 * i] * sn[i] + x[2 * i + 1] * cs[i] : x[2 * i + 1];
            }
        }
        if (!live || h >= h1) continue;
        const uint2 lo = hr_pack4<BF>(y), hi = hr_pack4<BF>(y + 4);
        uint8_t *o = query ? a.qo + token * a.soq + (int64_t)h * D * 2 : a.ko ? a.ko + token * a.sok + (int64_t)(h - a.H) * D * 2 : nullptr;
        if (o) {
            *(uint2 *)(o + 2 * da) = lo;
            *(uint2 *)(o + 2 * db) = hi;
        }
        if (!query && slot >= 0) {
            uint16_t *page = a.kc + (((slot >> a.lg_bs) * a.KV + (h - a.H)) * D << a.lg_bs) + 8 * (slot & ((1 << a.lg_bs) - 1));
            *(uint2 *)(page + ((da >> 3) << (a.lg_bs + 3)) + (da & 4)) = lo;
            *(uint2 *)(page + ((db >> 3) << (a.lg_bs + 3)) + (db & 4)) = hi;
        }
    }
}

template <int TY, bool BF, int LANES> static void launch_hr(const HrArgs &a, dim3 grid, hipStream_t stream) {
    if (a.mode == 2 && 2 * a.pairs < a.D) hipLaunchKernelGGL((k_head_rope<TY, BF, LANES, true>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((k_head_rope<TY, BF, LANES, false>), grid, dim3(256), 0, stream, a);
}
template <int TY, bool BF> static void launch_hr(const HrArgs &a, int lanes, dim3 grid, hipStream_t stream) {
    switch (lanes) {
    case 8: launch_hr<TY, BF, 8>(a, grid, stream); break;
    case 16: launch_hr<TY, BF, 16>(a, grid, stream); break;
    default: launch_hr<TY, BF, 32>(a, grid, stream); break;
    }
}

tlh_status launch_head_rope(const tlh_head_rope_args &a, hipStream_t stream) {
    const int es = a.type == TLH_TYPE_F32 ? 4 : 2;
    HrArgs r = {};
    r.q = (const uint8_t *)a.q, r.k = (const uint8_t *)a.k, r.v = (const uint8_t *)a.v;
    r.qo = (uint8_t *)a.q_out, r.ko = (uint8_t *)a.k_out, r.vo = (uint8_t *)a.v_out;
    r.kc = (uint16_t *)a.k_cache, r.vc = (uint16_t *)a.v_cache;
    r.positions = a.positions, r.freqs = a.freqs, r.qw = a.q_norm, r.kw = a.k_norm, r.slots = a.slots;
    r.sq = a.q_stride * es, r.sk = a.k_stride * es, r.sv = a.v_stride * es;
    r.soq = 2 * a.q_out_stride, r.sok = 2 * a.k_out_stride, r.sov = 2 * a.v_out_stride;
    r.pool_slots = a.k_cache ? a.num_blocks * a.block_size : 0;
    r.tokens = a.num_tokens, r.H = a.num_heads, r.KV = a.num_kv_heads, r.D = a.head_size, r.pairs = a.n_dims / 2, r.mode = a.mode;
    r.lg_bs = a.block_size == 8 ? 3 : a.block_size == 16 ? 4 : 5;
    r.eps = a.eps, r.factor = a.attn_factor;
    std::copy(a.pair_axis, a.pair_axis + 128, r.axis);
    const int lanes = a.head_size <= 64 ? 8 : a.head_size <= 128 ? 16 : 32, at_once = 256 / lanes;
    // few tokens: heads side by side instead
    while ((2 << r.lg_tg) <= std::min(a.num_tokens, at_once)) ++r.lg_tg;
    const int step = at_once >> r.lg_tg;
    const bool keys = a.k_out || a.k_cache, values = a.v_out || a.v_cache;
    r.heads = a.num_heads + (keys ? a.num_kv_heads : 0);
    const int64_t tiles = ((int64_t)a.num_tokens + (1 << r.lg_tg) - 1) >> r.lg_tg;
    auto split = [&](int heads, int &per) {  // into enough groups of whole steps to fill the machine
        const int64_t want = std::min<int64_t>((heads + step - 1) / step, (HR_WGS + tiles - 1) / tiles);
        per = (int)((heads + want - 1) / want + step - 1) / step * step;
        return (heads + per - 1) / per;
    };
    r.groups = split(r.heads, r.per);
    const int groups = r.groups + (values ? split(a.num_kv_heads, r.per_v) : 0);
    for (int64_t x0 = 0; x0 < tiles; x0 += 1 << 20) {  // grid x, times 256 threads
        const dim3 grid((unsigned)std::min<int64_t>(tiles - x0, 1 << 20), (unsigned)groups);
        r.first = x0 << r.lg_tg;
        const bool bf = a.out_type == TLH_TYPE_BF16;
        switch (a.type) {
        case TLH_TYPE_F32:
            if (bf) launch_hr<TLH_TYPE_F32, true>(r, lanes, grid, stream);
            else launch_hr<TLH_TYPE_F32, false>(r, lanes, grid, stream);
            break;
        case TLH_TYPE_F16:
            if (bf) launch_hr<TLH_TYPE_F16, true>(r, lanes, grid, stream);
            else launch_hr<TLH_TYPE_F16, false>(r, lanes, grid, stream);
            break;
        default:
            if (bf) launch_hr<TLH_TYPE_BF16, true>(r, lanes, grid, stream);
            else launch_hr<TLH_TYPE_BF16, false>(r, lanes, grid, stream);
        }
        const tlh_status st = check_launch("head_rope");
        if (st != TLH_OK) return st;
    }
    return TLH_OK;
}

}  // namespace tlh
