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
// bound is HBM: every byte is read once and written once (300 pages of 32 KiB in
// 32 pools 99 us, 6.4 TB/s with a third of the sources repeated; one page in 64
// pools 3.2 us).
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
        for (int r0 = 0; r0 < num_pairs; r0 += 1 << 22) {  // grid x
            const dim3 grid(std::min(num_pairs - r0, 1 << 22), n, (unsigned)((block_bytes + COPY_PIECE - 1) / COPY_PIECE));
            hipLaunchKernelGGL(k_copy_blocks, grid, dim3(256), 0, stream, pp, block_bytes, num_blocks,
                               pairs + 2 * (int64_t)r0);
            const tlh_status st = check_launch("copy_blocks");
            if (st != TLH_OK) return st;
            if (num_pairs - r0 <= 1 << 22) break;
        }
    }
    return TLH_OK;
}

// ---------------------------------------------------------------- compaction
// The kept drafted tokens of a sequence, in order, move to the places right
// behind its committed ones. A place may be the source of one token and the
// destination of another (token 2 to place 1, token 3 to place 2), so a
// workgroup, which owns some heads of one sequence in one pool, reads all the
// moving tokens of a head into LDS before it writes any: no other workgroup
// touches those bytes, and nothing depends on the order of workgroups.
//
// The bytes are few (a token's keys and values in a head), so the call is
// bound by the latency of its chain (counts, page ids, data) and by the
// 2-byte places of a value page: consecutive lanes take consecutive tokens,
// which lie next to each other in a page, and a workgroup takes as many heads
// at a time as fit its buffer (32 sequences with trees of 1..63, 32 pools: 12.6 us,
// 27 with a workgroup a head; 1 sequence, 64 pools 2.2 us).
constexpr int COMPACT_STAGE = 32768;    // bytes; 64 tokens of 256 dims fit
constexpr int COMPACT_WGS = 1024;       // workgroups that a launch splits the heads for

struct CompactArgs {
    const int32_t *tables, *lens, *starts;
    const int64_t *keep;
    int32_t *new_lens;
    int64_t num_blocks;
    int max_drafts, kvh, hs, bs, max_blocks, n_k;  // pools below n_k hold keys, the others values
    int heads;                                     // of a workgroup
};

// unit: elements of a move, step: elements from one move of a token to its next
template <typename T, int PER>
__device__ __forceinline__ void compact_moves(uint16_t *base, const int64_t *src, const int64_t *dst, int moved, int h0,
                                              int h1, int hs, int bs, T *stage) {
    const int lg = moved > 1 ? 32 - __clz(moved - 1) : 0;  // lanes a token run takes, a power of two
    const int pieces = hs / PER;                           // moves of a token in a head
    const int at_once = max(1, COMPACT_STAGE / ((int)sizeof(T) * (pieces << lg)));
    for (int ha = h0; ha < h1; ha += at_once) {
        const int items = (min(h1 - ha, at_once) * pieces) << lg;
        uint16_t *at = base + (int64_t)ha * hs * bs;
        if (ha > h0) __syncthreads();  // the last heads' moves are out of the buffer
#pragma unroll 4
        for (int i = threadIdx.x; i < items; i += 256) {
            const int tok = i & ((1 << lg) - 1);
            if (tok < moved) stage[i] = *(const T *)(at + src[tok] + (int64_t)(i >> lg) * bs * PER);
        }
        __syncthreads();
#pragma unroll 4
        for (int i = threadIdx.x; i < items; i += 256) {
            const int tok = i & ((1 << lg) - 1);
            if (tok < moved) *(T *)(at + dst[tok] + (int64_t)(i >> lg) * bs * PER) = stage[i];
        }
    }
}

__global__ void __launch_bounds__(256) k_compact_cache(const PoolPtrs pools, const CompactArgs a) {
    __shared__ __attribute__((aligned(16))) uint8_t stage[COMPACT_STAGE];
    __shared__ int64_t s_src[64], s_dst[64];  // element offsets of the moving tokens' places in head 0
    __shared__ int s_moved;
    const int s = blockIdx.x, pool = blockIdx.y, h0 = blockIdx.z * a.heads;
    const int n = max(0, min(a.starts[s + 1] - a.starts[s], a.max_drafts));
    const int L = max(0, min(a.lens[s], a.max_blocks * a.bs));
    const int first = L - n;  // the first drafted token's place; those at negative places are not there
    uint64_t keep = (uint64_t)a.keep[s];
    if (n < 64) keep &= ((uint64_t)1 << n) - 1;
    if (first < 0) keep = -first < 64 ? keep >> -first << -first : 0;
    const int to0 = max(first, 0);
    if (pool == 0 && h0 == 0 && threadIdx.x == 0 && a.new_lens) a.new_lens[s] = to0 + __popcll(keep);
    const bool key = pool < a.n_k;
    if (threadIdx.x < 64) {
        // lane j: drafted token j
        const int j = threadIdx.x;
        const int from = first + j, to = to0 + __popcll(keep & (((uint64_t)1 << j) - 1));
        int64_t sp = -1, dp = -1;
        if ((keep >> j) & 1 && from != to) {
            sp = a.tables[(int64_t)s * a.max_blocks + from / a.bs];
            dp = a.tables[(int64_t)s * a.max_blocks + to / a.bs];
        }
        const bool moves = sp >= 0 && sp < a.num_blocks && dp >= 0 && dp < a.num_blocks;
        const uint64_t who = __builtin_amdgcn_ballot_w64(moves);
        const int rank = __popcll(who & (((uint64_t)1 << j) - 1));
        const int64_t block = (int64_t)a.kvh * a.hs * a.bs;
        if (moves) {
            s_src[rank] = sp * block + (from % a.bs) * (key ? 8 : 1);
            s_dst[rank] = dp * block + (to % a.bs) * (key ? 8 : 1);
        }
        if (j == 0) s_moved = __popcll(who);
    }
    __syncthreads();
    const int moved = s_moved, h1 = min(h0 + a.heads, a.kvh);
    if (moved == 0) return;
    uint16_t *base = (uint16_t *)pools.p[pool];
    if (key) compact_moves<uint4, 8>(base, s_src, s_dst, moved, h0, h1, a.hs, a.bs, (uint4 *)stage);
    else compact_moves<uint16_t, 1>(base, s_src, s_dst, moved, h0, h1, a.hs, a.bs, (uint16_t *)stage);
}

tlh_status launch_compact_cache(const tlh_compact_cache_args &c, hipStream_t stream) {
    const int half = POOLS_A_LAUNCH / 2;
    for (int l0 = 0; l0 < c.num_layers; l0 += half) {
        const int n = std::min(half, c.num_layers - l0);
        PoolPtrs pp = {};
        for (int i = 0; i < n; ++i) pp.p[i] = (uint8_t *)c.k_caches[l0 + i], pp.p[n + i] = (uint8_t *)c.v_caches[l0 + i];
        CompactArgs a = {};
        a.tables = c.block_tables, a.lens = c.context_lens, a.starts = c.draft_starts, a.keep = c.keep;
        a.new_lens = l0 == 0 ? c.new_lens : nullptr;
        a.num_blocks = c.num_blocks, a.max_drafts = c.max_drafts, a.max_blocks = c.max_blocks_per_seq;
        a.kvh = c.num_kv_heads, a.hs = c.head_size, a.bs = c.block_size, a.n_k = n;
        const int64_t wgs = (int64_t)c.num_seqs * 2 * n;
        const int split = (int)std::min<int64_t>(c.num_kv_heads, (COMPACT_WGS + wgs - 1) / wgs);
        a.heads = (c.num_kv_heads + split - 1) / split;
        hipLaunchKernelGGL(k_compact_cache, dim3(c.num_seqs, 2 * n, (c.num_kv_heads + a.heads - 1) / a.heads), dim3(256), 0,
                           stream, pp, a);
        const tlh_status st = check_launch("compact_cache");
        if (st != TLH_OK) return st;
    }
    return TLH_OK;
}

}  // namespace tlh
