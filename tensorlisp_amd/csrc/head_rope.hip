// The norms of query and key heads, their rotation by the tokens' positions and the
// write of keys and values to a paged cache, in one pass, gfx950. A head x of D dims:
//   y = x / sqrt(mean(x^2) + eps) * w   (with a norm; else y = x)
//   (y_a, y_b) -> (y_a cos t - y_b sin t, y_a sin t + y_b cos t), times attn_factor,
//   for the pairs p < n_dims / 2 of its dims, t = positions[pair_axis[p]][token] freqs[p].
//
// t reaches 10^5 and more, where f32 leaves hundredths of a radian. It is formed in
// turns in 64 bits (t / 2 pi), reduced to its fraction there and only then taken to f32.
#include <algorithm>

#include "kernels.hpp"

namespace tlh {

template <int TY> __device__ __forceinline__ float hr_load(const void *p, int64_t i) {
    if constexpr (TY == TLH_TYPE_F32) return ((const float *)p)[i];
    else if constexpr (TY == TLH_TYPE_F16) return h2f(((const uint16_t *)p)[i]);
    else return bf16_to_f32(((const uint16_t *)p)[i]);
}

// cos and sin of position * freq
__device__ __forceinline__ void hr_angle(int position, float freq, float factor, float &cs, float &sn) {
    const double turns = (double)position * ((double)freq * 0.15915494309189533577);
    const float part = (float)(turns - rint(turns));
    sincospif(2.0f * part, &sn, &cs);
    cs *= factor, sn *= factor;
}

// One wave a (token, head): q's heads, then k's, then v's.
template <int TY>
__global__ void __launch_bounds__(64) k_head_rope(const tlh_head_rope_args a) {
    const int lane = threadIdx.x, D = a.head_size, t = blockIdx.x, hh = blockIdx.y;
    const int kind = hh < a.num_heads ? 0 : hh < a.num_heads + a.num_kv_heads ? 1 : 2;
    const int h = hh - (kind > 0 ? a.num_heads : 0) - (kind > 1 ? a.num_kv_heads : 0);
    const void *src = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
    const int64_t from = (int64_t)t * (kind == 0 ? a.q_stride : kind == 1 ? a.k_stride : a.v_stride) + (int64_t)h * D;
    __shared__ float s_x[256], s_y[256];
    float sq = 0.0f;
    for (int d = lane; d < D; d += 64) {
        s_x[d] = hr_load<TY>(src, from + d);
        sq += s_x[d] * s_x[d];
    }
    const float *w = kind == 0 ? a.q_norm : kind == 1 ? a.k_norm : nullptr;
    if (w) {
        for (int o = 1; o < 64; o <<= 1) sq += __shfl_xor(sq, o, 64);
        const float inv = 1.0f / sqrtf(sq / D + a.eps);
        for (int d = lane; d < D; d += 64) s_x[d] *= inv * w[d];
    }
    __syncthreads();
    const int pairs = kind == 2 ? 0 : a.n_dims / 2;
    for (int p = lane; p < pairs; p += 64) {
        float cs, sn;
        hr_angle(a.positions[(int64_t)a.pair_axis[p] * a.num_tokens + t], a.freqs[p], a.attn_factor, cs, sn);
        const int i = a.mode == 0 ? 2 * p : p, j = a.mode == 0 ? 2 * p + 1 : p + pairs;
        s_y[i] = s_x[i] * cs - s_x[j] * sn;
        s_y[j] = s_x[i] * sn + s_x[j] * cs;
    }
    for (int d = lane + 2 * pairs; d < D; d += 64) s_y[d] = s_x[d];
    __syncthreads();
    void *dst = kind == 0 ? a.q_out : kind == 1 ? a.k_out : a.v_out;
    const int64_t to = (int64_t)t * (kind == 0 ? a.q_out_stride : kind == 1 ? a.k_out_stride : a.v_out_stride) + (int64_t)h * D;
    const int64_t slot = a.slots && kind > 0 ? a.slots[t] : -1;
    const int BS = a.block_size;
    for (int d = lane; d < D; d += 64) {
        const uint16_t y = a.out_type == TLH_TYPE_F16 ? f2h(s_y[d]) : f32_to_bf16(s_y[d]);
        if (dst) ((uint16_t *)dst)[to + d] = y;
        if (slot < 0 || slot >= a.num_blocks * BS) continue;
        const int64_t head = (slot / BS * a.num_kv_heads + h) * D * BS, at = slot % BS;
        if (kind == 1) ((uint16_t *)a.k_cache)[head + (d / 8 * BS + at) * 8 + d % 8] = y;
        else ((uint16_t *)a.v_cache)[head + d * BS + at] = y;
    }
}

tlh_status launch_head_rope(const tlh_head_rope_args &a, hipStream_t stream) {
    for (int t0 = 0; t0 < a.num_tokens; t0 += 1 << 24) {
        tlh_head_rope_args b = a;  // (num_tokens stays: it is positions' stride)
        const int es = a.type == TLH_TYPE_F32 ? 4 : 2;
        b.q = (const char *)a.q + t0 * a.q_stride * es, b.k = (const char *)a.k + t0 * a.k_stride * es;
        b.v = (const char *)a.v + t0 * a.v_stride * es;
        b.q_out = (char *)a.q_out + 2 * t0 * a.q_out_stride;
        if (a.k_out) b.k_out = (char *)a.k_out + 2 * t0 * a.k_out_stride;
        if (a.v_out) b.v_out = (char *)a.v_out + 2 * t0 * a.v_out_stride;
        if (a.positions) b.positions = a.positions + t0;
        if (a.slots) b.slots = a.slots + t0;
        const dim3 grid(std::min(a.num_tokens - t0, 1 << 24), a.num_heads + 2 * a.num_kv_heads);
        switch (a.type) {
        case TLH_TYPE_F32: hipLaunchKernelGGL((k_head_rope<TLH_TYPE_F32>), grid, dim3(64), 0, stream, b); break;
        case TLH_TYPE_F16: hipLaunchKernelGGL((k_head_rope<TLH_TYPE_F16>), grid, dim3(64), 0, stream, b); break;
        default: hipLaunchKernelGGL((k_head_rope<TLH_TYPE_BF16>), grid, dim3(64), 0, stream, b); break;
        }
        const tlh_status st = check_launch("head_rope");
        if (st != TLH_OK) return st;
        if (a.num_tokens - t0 <= 1 << 24) break;
    }
    return TLH_OK;
}

}  // namespace tlh
