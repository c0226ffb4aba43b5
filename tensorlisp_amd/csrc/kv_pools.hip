// Moves inside the pools of a paged KV cache, every layer in one launch, gfx950:
// copying whole pages (a fork's copy-on-write, a defragmentation), and closing
// the gaps that rejected drafted tokens leave.
#include <algorithm>

#include "kernels.hpp"

namespace tlh {

// Pool base addresses travel in the kernel arguments, so a captured launch
// keeps them; more pools than fit take further launches.
constexpr int POOLS_A_LAUNCH = 128;
struct PoolPtrs {
    uint8_t *p[POOLS_A_LAUNCH];
};

// One workgroup moves up to COPY_PIECE bytes of one page in one pool. The
// bound is HBM: every byte is read once and written once.
constexpr int COPY_PIECE = 16384;

__global__ void __launch_bounds__(256) k_copy_blocks(const PoolPtrs pools, int64_t block_bytes, int64_t num_blocks,
                                                     const int64_t *__restrict__ pairs) {
    const int64_t src = pairs[2 * (int64_t)blockIdx.x], dst = pairs[2 * (int64_t)blockIdx.x + 1];
    if (src < 0 || src >= num_blocks || dst < 0 || dst >= num_blocks || src == dst) return;
    uint8_t *base = pools.p[blockIdx.y];
    const int64_t at = (int64_t)blockIdx.z * COPY_PIECE;
    const int len = (int)min((int64_t)COPY_PIECE, block_bytes - at);
    const uint4 *from = (const uint4 *)(base + src * block_bytes + at);
    uint4 *to = (uint4 *)(base + dst * block_bytes + at);
    for (int i = threadIdx.x; i < len / 16; i += 256) to[i] = from[i];
}

tlh_status launch_copy_blocks(void *const *pools, int num_pools, int64_t block_bytes, int64_t num_blocks,
                              const int64_t *pairs, int num_pairs, hipStream_t stream) {
    for (int p0 = 0; p0 < num_pools; p0 += POOLS_A_LAUNCH) {
        const int n = std::min(POOLS_A_LAUNCH, num_pools - p0);
        PoolPtrs pp = {};
        for (int i = 0; i < n; ++i) pp.p[i] = (uint8_t *)pools[p0 + i];
        const dim3 grid(num_pairs, n, (unsigned)((block_bytes + COPY_PIECE - 1) / COPY_PIECE));
        hipLaunchKernelGGL(k_copy_blocks, grid, dim3(256), 0, stream, pp, block_bytes, num_blocks, pairs);
        const tlh_status st = check_launch("copy_blocks");
        if (st != TLH_OK) return st;
    }
    return TLH_OK;
}

// ---------------------------------------------------------------- compaction
// The kept drafted tokens of a sequence, in order, move to the places right
// behind its committed ones. A place may be the source of one token and the
// destination of another (token 2 to place 1, token 3 to place 2), so a
// workgroup, which owns one head of one sequence in one pool, reads all the
// moving tokens into LDS before it writes any: no other workgroup touches
// those bytes, and nothing depends on the order of workgroups.
struct CompactArgs {
    const int32_t *tables, *lens, *starts;
    const int64_t *keep;
    int32_t *new_lens;
    int64_t num_blocks;
    int num_seqs, max_drafts, kvh, hs, bs, max_blocks, n_k;  // pools below n_k hold keys, the others values
};

__global__ void __launch_bounds__(256) k_compact_cache(const PoolPtrs pools, const CompactArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint16_t stage[];  // [moving tokens][hs]
    __shared__ int64_t s_src[64], s_dst[64];  // element offsets of the moving tokens' places, -1: not moved
    const int s = blockIdx.x, pool = blockIdx.y, h = blockIdx.z;
    const int span = a.starts[s + 1] - a.starts[s];
    const int n = max(0, min(span, a.max_drafts));
    const int L = max(0, min(a.lens[s], a.max_blocks * a.bs));
    const int first = L - n;  // the first drafted token's place; those at negative places are not there
    uint64_t keep = (uint64_t)a.keep[s];
    if (n < 64) keep &= ((uint64_t)1 << n) - 1;
    if (first < 0) keep = -first < 64 ? keep >> -first << -first : 0;
    const int kept = __popcll(keep), to0 = max(first, 0);
    if (pool == 0 && h == 0 && threadIdx.x == 0 && a.new_lens) a.new_lens[s] = to0 + kept;
    const bool key = pool < a.n_k;
    const int ts = key ? 8 : 1;  // elements between two tokens of a page's run
    if (threadIdx.x < 64) {
        // lane j: drafted token j
        const int j = threadIdx.x;
        const bool mine = (keep >> j) & 1;
        const int rank = __popcll(keep & (((uint64_t)1 << j) - 1));
        const int from = first + j, to = to0 + rank;
        if (mine) {
            int64_t sp = -1, dp = -1;
            if (from != to) {
                sp = a.tables[(int64_t)s * a.max_blocks + from / a.bs];
                dp = a.tables[(int64_t)s * a.max_blocks + to / a.bs];
            }
            const bool ok = sp >= 0 && sp < a.num_blocks && dp >= 0 && dp < a.num_blocks;
            s_src[rank] = ok ? (sp * a.kvh + h) * a.hs * a.bs + (from % a.bs) * ts : -1;
            s_dst[rank] = ok ? (dp * a.kvh + h) * a.hs * a.bs + (to % a.bs) * ts : -1;
        }
    }
    __syncthreads();
    uint16_t *base = (uint16_t *)pools.p[pool];
    if (key) {  // runs of 8 dims
        const int chunks = a.hs / 8;
        for (int i = threadIdx.x; i < kept * chunks; i += 256)
            if (s_src[i / chunks] >= 0)
                ((uint4 *)stage)[i] = *(const uint4 *)(base + s_src[i / chunks] + (int64_t)(i % chunks) * a.bs * 8);
        __syncthreads();
        for (int i = threadIdx.x; i < kept * chunks; i += 256)
            if (s_src[i / chunks] >= 0)
                *(uint4 *)(base + s_dst[i / chunks] + (int64_t)(i % chunks) * a.bs * 8) = ((uint4 *)stage)[i];
    } else {
        for (int i = threadIdx.x; i < kept * a.hs; i += 256)
            if (s_src[i / a.hs] >= 0) stage[i] = base[s_src[i / a.hs] + (int64_t)(i % a.hs) * a.bs];
        __syncthreads();
        for (int i = threadIdx.x; i < kept * a.hs; i += 256)
            if (s_src[i / a.hs] >= 0) base[s_dst[i / a.hs] + (int64_t)(i % a.hs) * a.bs] = stage[i];
    }
}

tlh_status launch_compact_cache(const tlh_compact_cache_args &c, hipStream_t stream) {
    const int half = POOLS_A_LAUNCH / 2;
    for (int l0 = 0; l0 < c.num_layers; l0 += half) {
        const int n = std::min(half, c.num_layers - l0);
        PoolPtrs pp = {};
        for (int i = 0; i < n; ++i) pp.p[i] = (uint8_t *)c.k_caches[l0 + i], pp.p[n + i] = (uint8_t *)c.v_caches[l0 + i];
        CompactArgs a = {c.block_tables, c.context_lens, c.draft_starts, c.keep, l0 == 0 ? c.new_lens : nullptr,
                         c.num_blocks, c.num_seqs, c.max_drafts, c.num_kv_heads, c.head_size, c.block_size,
                         c.max_blocks_per_seq, n};
        hipLaunchKernelGGL(k_compact_cache, dim3(c.num_seqs, 2 * n, c.num_kv_heads), dim3(256),
                           (size_t)c.max_drafts * c.head_size * 2, stream, pp, a);
        const tlh_status st = check_launch("compact_cache");
        if (st != TLH_OK) return st;
    }
    return TLH_OK;
}

}  // namespace tlh
