// Causal attention of the sequences' new tokens over a paged f16 cache, gfx950.
//
// Sequence s has L = context_lens[s] tokens in the cache, the last n of them new
// (n = row_starts[s + 1] - row_starts[s]), and n rows of q. Row i is the token at
// place L - n + i and sees the tokens from max(0, that - window + 1) up to itself:
//   out[i, h] = sum_j softmax_j(scale * q[i, h] . k[j, h / G]) v[j, h / G]
// The caches are the paged-attention layouts
//   key   [blocks][kv_heads][D/8][block_size][8]
//   value [blocks][kv_heads][D][block_size]
// A row that sees nothing gives zeros.
#include <algorithm>

#include "mfma32.hpp"

namespace tlh {

// One wave a (row, head): a lane scores one of 64 keys, then takes the sums of D / 64 dims.
template <int D>
__global__ void __launch_bounds__(64) k_chunk_attn(const tlh_chunk_attention_args a) {
    constexpr int E = (D + 63) / 64;
    __shared__ float s_q[D], s_p[64];
    __shared__ int64_t s_v[64];
    const int lane = threadIdx.x, s = blockIdx.y, H = a.num_heads, KV = a.num_kv_heads, BS = a.block_size;
    const int b = max(0, min(a.row_starts[s], a.num_rows));
    const int n = min(max(b, min(a.row_starts[s + 1], a.num_rows)) - b, a.max_rows);
    const int L = a.num_blocks > 0 ? max(0, min(a.context_lens[s], a.max_context_len)) : 0;
    const int32_t *table = a.block_tables + (int64_t)s * a.max_blocks_per_seq;
    for (int64_t x = blockIdx.x; x < (int64_t)n * H; x += gridDim.x) {
        const int i = (int)(x / H), h = (int)(x % H), hk = h / (H / KV), pos = L - n + i;
        const int first = a.window > 0 ? max(0, pos - a.window + 1) : 0;
        const uint16_t *q = (const uint16_t *)a.q + (b + i) * a.q_stride + (int64_t)h * D;
        __syncthreads();
        for (int d = lane; d < D; d += 64) s_q[d] = h2f(q[d]) * a.scale;
        __syncthreads();
        float m = -INFINITY, l = 0.0f, o[E] = {};
        for (int k0 = first; k0 <= pos; k0 += 64) {
            const int j = k0 + lane;
            float sc = -INFINITY;
            int64_t va = -1;
            if (j <= pos) {
                const int page = table[j / BS];
                if (page >= 0 && page < a.num_blocks) {
                    const int64_t at = ((int64_t)page * KV + hk) * D * BS;
                    const uint16_t *k = (const uint16_t *)a.k_cache + at + (j % BS) * 8;
                    float dot = 0.0f;
                    for (int d = 0; d < D; ++d) dot += s_q[d] * h2f(k[(int64_t)(d / 8) * BS * 8 + d % 8]);
                    sc = dot;
                    va = at + j % BS;
                }
            }
            float top = sc;
            for (int e = 1; e < 64; e <<= 1) top = fmaxf(top, __shfl_xor(top, e, 64));
            const float to = fmaxf(m, top);
            if (__builtin_amdgcn_ballot_w64(va >= 0) == 0) continue;
            const float f = m == -INFINITY ? 0.0f : expf(m - to);
            const float p = va >= 0 ? expf(sc - to) : 0.0f;
            m = to;
            __syncthreads();
            s_p[lane] = p, s_v[lane] = va;
            __syncthreads();
            l *= f;
            for (int e = 0; e < E; ++e) o[e] *= f;
            for (int t = 0; t < 64; ++t) {
                if (s_v[t] < 0) continue;
                l += s_p[t];
                for (int e = 0; e < E; ++e)
                    if (lane + 64 * e < D)
                        o[e] += s_p[t] * h2f(((const uint16_t *)a.v_cache)[s_v[t] + (int64_t)(lane + 64 * e) * BS]);
            }
        }
        uint16_t *out = (uint16_t *)a.out + (b + i) * a.out_stride + (int64_t)h * D;
        for (int e = 0; e < E; ++e)
            if (lane + 64 * e < D) out[lane + 64 * e] = f2h(l == 0.0f ? 0.0f : o[e] / l);
    }
}

size_t chunk_attention_scratch_bytes(const tlh_chunk_attention_args &a) { return 0; }

template <int D> static void launch_ca(const tlh_chunk_attention_args &a, hipStream_t stream) {
    const int64_t rows = (int64_t)std::min(a.max_rows, a.num_rows) * a.num_heads;
    hipLaunchKernelGGL((k_chunk_attn<D>), dim3((unsigned)std::min<int64_t>(rows, 1 << 20), a.num_seqs), dim3(64), 0, stream, a);
}

tlh_status launch_chunk_attention(const tlh_chunk_attention_args &a, void *scratch, hipStream_t stream) {
    switch (a.head_size) {
    case 64: launch_ca<64>(a, stream); break;
    case 80: launch_ca<80>(a, stream); break;
    case 96: launch_ca<96>(a, stream); break;
    case 112: launch_ca<112>(a, stream); break;
    case 128: launch_ca<128>(a, stream); break;
    case 192: launch_ca<192>(a, stream); break;
    default: launch_ca<256>(a, stream); break;
    }
    return check_launch("chunk_attention");
}

}  // namespace tlh
