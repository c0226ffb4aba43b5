// Attention of drafted tokens over a paged f16 cache, gfx950.
//
// Sequence s has L = context_lens[s] tokens in the cache, the last n of them
// drafted (n = draft_starts[s + 1] - draft_starts[s]), and n rows of q. Row i
// sees every token before L - n and drafted token j where bit j of its mask is
// set; the caches are the paged-attention layouts
//   key   [blocks][kv_heads][D/8][block_size][8]
//   value [blocks][kv_heads][D][block_size]
// A row that sees nothing gives zeros.
#include "kernels.hpp"

namespace tlh {

// One wave per (row, head): 64 keys at a time, one a lane; the running maximum
// and sum in f32; then the lanes take the output dims.
__global__ void __launch_bounds__(64) k_tree_attn(const tlh_tree_attention_args a) {
    __shared__ float sq[256], sp[64];
    __shared__ int64_t sv[64];
    const int lane = threadIdx.x, D = a.head_size, bs = a.block_size;
    const int h = blockIdx.x, hk = h / (a.num_heads / a.num_kv_heads), s = blockIdx.z, i = blockIdx.y;
    const int b = max(0, min(a.draft_starts[s], a.num_rows)), e = max(b, min(a.draft_starts[s + 1], a.num_rows));
    const int n = min(e - b, a.max_drafts);
    if (i >= n) return;
    const int L = max(0, min(a.context_lens[s], a.max_context_len));
    const int64_t t = b + i, row = (t * a.num_heads + h) * D;
    const uint64_t mask = (uint64_t)a.draft_masks[t];
    for (int d = lane; d < D; d += 64) sq[d] = h2f(((const uint16_t *)a.q)[row + d]);
    __syncthreads();
    float m = -INFINITY, l = 0.0f, acc[4] = {};
    for (int j0 = 0; j0 < L; j0 += 64) {
        const int j = j0 + lane;
        bool see = j < L && (j < L - n || ((mask >> (j - (L - n))) & 1));
        int64_t page = 0;
        if (see) page = a.block_tables[(int64_t)s * a.max_blocks_per_seq + j / bs];
        see = see && page >= 0 && page < a.num_blocks;
        float x = -INFINITY;
        if (see) {
            const uint16_t *k = (const uint16_t *)a.k_cache + (page * a.num_kv_heads + hk) * D * bs + (j % bs) * 8;
            float dot = 0.0f;
            for (int d = 0; d < D; ++d) dot += sq[d] * h2f(k[(d / 8) * bs * 8 + d % 8]);
            x = dot * a.scale;
        }
        float mx = x;
        for (int o = 1; o < 64; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
        const float mn = fmaxf(m, mx), alpha = mn == -INFINITY ? 1.0f : __expf(m - mn);
        const float p = see && mn != -INFINITY ? __expf(x - mn) : 0.0f;
        m = mn;
        float ps = p;
        for (int o = 1; o < 64; o <<= 1) ps += __shfl_xor(ps, o, 64);
        l = l * alpha + ps;
        __syncthreads();
        sp[lane] = p;
        sv[lane] = see ? (page * a.num_kv_heads + hk) * D * bs + j % bs : -1;
        __syncthreads();
        for (int c = 0; c < 4; ++c) acc[c] *= alpha;
        for (int jj = 0; jj < 64; ++jj)
            for (int c = 0; c < 4; ++c)
                if (sv[jj] >= 0 && lane + 64 * c < D)
                    acc[c] += sp[jj] * h2f(((const uint16_t *)a.v_cache)[sv[jj] + (lane + 64 * c) * bs]);
        __syncthreads();
    }
    for (int c = 0; c < 4; ++c)
        if (lane + 64 * c < D) ((uint16_t *)a.out)[row + lane + 64 * c] = f2h(l == 0.0f ? 0.0f : acc[c] / l);
}

size_t tree_attention_scratch_bytes(const tlh_tree_attention_args &) { return 0; }

tlh_status launch_tree_attention(const tlh_tree_attention_args &a, void *scratch, hipStream_t stream) {
    hipLaunchKernelGGL(k_tree_attn, dim3(a.num_heads, a.max_drafts, a.num_seqs), dim3(64), 0, stream, a);
    return check_launch("tree_attention");
}

}  // namespace tlh
