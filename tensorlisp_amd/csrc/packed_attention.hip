// Causal attention of whole prompts packed one after another, gfx950.
//
//   q [tokens][heads][D], k and v [tokens][kv_heads][D], out as q (f16 or bf16;
//   rows of heads contiguous, any token stride), seq_starts [num_seqs + 1]:
//   out[t, h] = sum_j softmax_j(scale * q[t, h] . k[j, h / G]) v[j, h / G]
//   over the tokens j <= t of t's own sequence.
#include <algorithm>

#include "kernels.hpp"

namespace tlh {

template <bool BF> __device__ __forceinline__ float pk_load(uint16_t x) { return BF ? bf16_to_f32(x) : h2f(x); }
template <bool BF> __device__ __forceinline__ uint16_t pk_round(float x) { return BF ? f32_to_bf16(x) : f2h(x); }

// One wave per (token, head): 64 keys at a time, one a lane; the running
// maximum and sum in f32; then the lanes take the output dims.
template <bool BF>
__global__ void __launch_bounds__(64) k_packed_attn(const tlh_packed_attention_args a) {
    __shared__ float sq[256], sp[64];
    const int lane = threadIdx.x, D = a.head_size;
    const int h = blockIdx.x, hk = h / (a.num_heads / a.num_kv_heads), s = blockIdx.z;
    const int b = max(0, min(a.seq_starts[s], a.num_tokens)), e = min(a.seq_starts[s + 1], a.num_tokens);
    const uint16_t *K = (const uint16_t *)a.k + (int64_t)hk * D, *V = (const uint16_t *)a.v + (int64_t)hk * D;
    for (int i = blockIdx.y; i < min(e - b, a.max_seq_len); i += gridDim.y) {
        const int64_t t = b + i;
        const uint16_t *q = (const uint16_t *)a.q + t * a.q_stride + (int64_t)h * D;
        __syncthreads();
        for (int d = lane; d < D; d += 64) sq[d] = pk_load<BF>(q[d]);
        __syncthreads();
        float m = -INFINITY, l = 0.0f, acc[4] = {};
        for (int j0 = 0; j0 <= i; j0 += 64) {
            float x = -INFINITY;
            if (j0 + lane <= i) {
                const uint16_t *k = K + (int64_t)(b + j0 + lane) * a.k_stride;
                float dot = 0.0f;
                for (int d = 0; d < D; ++d) dot += sq[d] * pk_load<BF>(k[d]);
                x = dot * a.scale;
            }
            float mx = x;
            for (int o = 1; o < 64; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
            const float mn = fmaxf(m, mx), alpha = mn == -INFINITY ? 1.0f : __expf(m - mn);
            const float p = j0 + lane <= i && mn != -INFINITY ? __expf(x - mn) : 0.0f;
            m = mn;
            float ps = p;
            for (int o = 1; o < 64; o <<= 1) ps += __shfl_xor(ps, o, 64);
            l = l * alpha + ps;
            __syncthreads();
            sp[lane] = p;
            __syncthreads();
            for (int c = 0; c < 4; ++c) acc[c] *= alpha;
            for (int j = j0; j <= min(i, j0 + 63); ++j)
                for (int c = 0; c < 4; ++c)
                    if (lane + 64 * c < D) acc[c] += sp[j - j0] * pk_load<BF>(V[(int64_t)(b + j) * a.v_stride + lane + 64 * c]);
        }
        uint16_t *o = (uint16_t *)a.out + t * a.out_stride + (int64_t)h * D;
        for (int c = 0; c < 4; ++c)
            if (lane + 64 * c < D) o[lane + 64 * c] = pk_round<BF>(acc[c] / l);
    }
}

tlh_status launch_packed_attention(const tlh_packed_attention_args &a, hipStream_t stream) {
    const dim3 grid(a.num_heads, std::min(a.max_seq_len, 1024), a.num_seqs);
    if (a.type == TLH_TYPE_BF16) hipLaunchKernelGGL(k_packed_attn<true>, grid, dim3(64), 0, stream, a);
    else hipLaunchKernelGGL(k_packed_attn<false>, grid, dim3(64), 0, stream, a);
    return check_launch("packed_attention");
}

}  // namespace tlh
