// Log probabilities of given tokens, the distributions' entropies and the
// likeliest alternatives, gfx950. For a row x of V logits with m = max x,
// S = sum exp(x - m), T = sum exp(x - m) (x - m):
//   log p(t) = (x_t - m) - log S,   H = log S - T / S,
// and the `top` largest x, equal ones by the lowest index.
//
// The bound is one read of the logits. A workgroup takes a chunk of a row into
// registers, so the chunk's maximum is known before its exponentials (one pass,
// no rescaling) and its largest elements are found without a second read:
//  * the top-th largest of the 256 lanes' maxima is a threshold: at least `top`
//    elements of the chunk reach it, and few more do. Every wave lists its own, and the
//    listed ones are ranked by counting (a threshold from each wave's 64 maxima lists
//    four times as many: 777 x 128256, top 20, 130 us instead of 86; without the
//    alternatives it is 70);
//  * where more reach it than the list holds, as in a vocabulary-wide run of equal
//    logits (a grammar's -inf mask), ties are taken in index order and only up to
//    `top` (109 us with 999 of 1000 masked);
//  * more elements above the threshold than the list holds (the largest ones
//    crowded into few lanes) are taken one maximum at a time instead, read again.
// A second launch folds the chunks' sums and merges their sorted lists the same
// way, one wave a row with one list a lane.
#include <algorithm>

#include "kernels.hpp"

namespace tlh {

constexpr int LP_MAX_TOP = 32;
constexpr int LP_FEW = 64;        // elements that reach the threshold, a wave: listed as they are
constexpr int LP_CAP = 256;       // elements above it, where more reach it
constexpr int LP_MERGE = 256;     // listed entries of a row in the merge
constexpr int LP_AHEAD = 4;       // entries of a list that make the merge's threshold
constexpr int LP_LISTS = 64;      // chunks of a row, at most: a lane each in the merge
// elements of a chunk: 64 (or 16, for few rows) of each of 256 lanes
constexpr int LP_CHUNK = 64 * 256, LP_CHUNK_SMALL = 16 * 256;

// An order-preserving integer of a logit: larger is likelier, -0 equals 0, a
// NaN is above everything; 0 is free for an element that is not there.
__device__ __forceinline__ uint32_t lp_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    const uint32_t k = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
    return x != x ? 0xffffffffu : k;
}
__device__ __forceinline__ float lp_value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
// (key, lowest index first) in one integer
__device__ __forceinline__ uint64_t lp_entry(uint32_t key, uint32_t idx) { return (uint64_t)key << 32 | (uint32_t)~idx; }

// the maximum of the first `lanes` lanes, in all of those
template <typename T> __device__ __forceinline__ T lp_wave_max(T v, int lanes = 64) {
    for (int o = 1; o < lanes; o <<= 1) v = max(v, (T)__shfl_xor(v, o, 64));
    return v;
}
__device__ __forceinline__ float lp_wave_sum(float v) {
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
}
__device__ __forceinline__ float lp_wave_maxf(float v) {
    for (int o = 1; o < 64; o <<= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}
// x - m, whose exponential is 0 below -1000 anyway: a -inf (x, or the difference of
// numbers far apart) must not reach the product with it
__device__ __forceinline__ float lp_apart(float x, float m) {
    const float d = x - m;
    return d < -1000.0f ? -1000.0f : d;
}
// set bits of b below this lane
__device__ __forceinline__ int lp_below(uint64_t b) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0));
}

template <int TY> __device__ __forceinline__ float lp_elem(const void *p, int64_t i) {
    if constexpr (TY == TLH_TYPE_F32) return ((const float *)p)[i];
    else if constexpr (TY == TLH_TYPE_F16) return h2f(((const uint16_t *)p)[i]);
    else return bf16_to_f32(((const uint16_t *)p)[i]);
}

// Scratch of chunk p of a row: m, S, T, one free word, then `top` entries.
__host__ __device__ constexpr size_t lp_slot(int top) { return 16 + 8 * (size_t)top; }

// One wave's part of a chunk: NV vectors of C elements a lane, the first of vector
// i at element e0 + 256 C i of the row. EDGE: some elements may lie outside [0, V)
// (they hold -inf, and are told from a row's own -inf by their index).
template <int TY, int C, int NV, bool EDGE> struct LpWave {
    const float (&x)[NV][C];
    const void *base;  // the row
    const int e0, V, lane;
    __device__ int elem(int i, int c) const { return e0 + 256 * C * i + c; }
    __device__ bool there(int i, int c) const { return !EDGE || (uint32_t)elem(i, c) < (uint32_t)V; }

    // Lists the elements that reach thr (a value); where they are more than a few, those
    // above it and the first `top` that equal it; -> how many. A wave with a NaN or
    // +inf (plain = false) and one with too many above thr take their `top` largest one
    // maximum at a time instead.
    __device__ __forceinline__ int list_top(float thr, int top, bool plain, uint64_t *list) const {
        if (plain) {
            int n = 0;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                uint64_t any = 0;
#pragma unroll
                for (int c = 0; c < C; ++c) any |= __builtin_amdgcn_ballot_w64(x[i][c] >= thr);
                if (any == 0 || n > LP_FEW) continue;
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const uint64_t who = __builtin_amdgcn_ballot_w64(x[i][c] >= thr && there(i, c));
                    const int at = n + lp_below(who);
                    if ((who >> lane) & 1 && at < LP_FEW) list[at] = lp_entry(lp_key(x[i][c]), elem(i, c));
                    n += __popcll(who);
                }
            }
            if (n <= LP_FEW) return n;
            int above = 0, equal = 0;
            const float over = lp_value(lp_key(thr) + 1);  // the next number
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                uint64_t any = 0;
                const float bar = equal < top ? thr : over;  // enough ties: those to come have higher indices
#pragma unroll
                for (int c = 0; c < C; ++c) any |= __builtin_amdgcn_ballot_w64(x[i][c] >= bar);
                if (any == 0) continue;
                int before = 0;  // of the lanes below: elements of the vector that equal thr
                uint64_t eq[C];
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    eq[c] = __builtin_amdgcn_ballot_w64(x[i][c] == thr && there(i, c));
                    before += lp_below(eq[c]);
                }
                int eqs = 0;
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const uint64_t gt = __builtin_amdgcn_ballot_w64(x[i][c] > thr);
                    const uint64_t entry = lp_entry(lp_key(x[i][c]), elem(i, c));
                    const int ga = above + lp_below(gt);
                    if ((gt >> lane) & 1 && ga < LP_CAP) list[ga] = entry;
                    above += __popcll(gt);
                    if ((eq[c] >> lane) & 1) {
                        if (equal + before < top) list[LP_CAP + equal + before] = entry;
                        ++before;
                    }
                    eqs += __popcll(eq[c]);
                }
                equal += eqs;
            }
            if (above <= LP_CAP) {  // the ties behind the others
                const int ne = min(equal, top);
                __builtin_amdgcn_wave_barrier();
                if (lane < ne && above < LP_CAP) list[above + lane] = list[LP_CAP + lane];
                return above + ne;
            }
        }
        uint64_t last = ~(uint64_t)0;
        for (int r = 0; r < top; ++r) {
            uint64_t b = 0;
#pragma unroll 1
            for (int i = 0; i < NV * C; ++i) {  // read again: rare, and registers cannot be indexed in a loop
                const int e = e0 + 256 * C * (i / C) + i % C;
                if (e < 0 || e >= V) continue;
                const uint64_t entry = lp_entry(lp_key(lp_elem<TY>(base, e)), e);
                if (entry < last && entry > b) b = entry;
            }
            last = lp_wave_max(b);
            if (last == 0) return r;
            if (lane == 0) list[r] = last;
        }
        return top;
    }
};

template <int TY, int EPT>
__global__ void __launch_bounds__(256) k_token_logprobs(const void *__restrict__ logits, int64_t row_stride, int V,
                                                        int top, int P, uint8_t *__restrict__ scratch) {
    constexpr int C = TY == TLH_TYPE_F32 ? 4 : 8;  // elements of a 16-byte load
    constexpr int ES = 16 / C, NV = EPT / C;
    __shared__ uint64_t s_list[4][LP_CAP + LP_MAX_TOP];
    __shared__ uint32_t s_best[256], s_thr;
    __shared__ int s_n[4];
    __shared__ float s_sum[4][3];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int row = blockIdx.y, p = blockIdx.x;
    const char *base = (const char *)logits + (int64_t)row * row_stride * ES;
    // Loads are aligned whatever the row's address: element 0 of the chunks'
    // numbering lies up to C - 1 elements before the row.
    const int mis = (int)(((uintptr_t)base & 15) / ES);
    const int first = p * 256 * EPT - mis;
    const int e0 = first + threadIdx.x * C;
    const bool edge = first < 0 || first + 256 * EPT > V;  // the chunk holds places outside the row
    float x[NV][C];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int e = e0 + 256 * C * i;
        if (!edge || (e >= 0 && e + C <= V)) {
            const uint4 w = *(const uint4 *)(base + (int64_t)e * ES);
            const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int c = 0; c < C; ++c)
                x[i][c] = TY == TLH_TYPE_F32   ? __uint_as_float(ws[c % 4])
                          : TY == TLH_TYPE_F16 ? h2f((uint16_t)(ws[c / 2 % 4] >> (16 * (c & 1))))
                                               : bf16_to_f32((uint16_t)(ws[c / 2 % 4] >> (16 * (c & 1))));
        } else {
#pragma unroll
            for (int c = 0; c < C; ++c) x[i][c] = e + c >= 0 && e + c < V ? lp_elem<TY>(base, e + c) : -INFINITY;
        }
    }
    float best = -INFINITY;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int c = 0; c < C; ++c) best = fmaxf(best, x[i][c]);
    const float m = lp_wave_maxf(best);
    // exp(x - m) as 2^((x - m) log2 e). A NaN among the logits is not in m; it passes
    // both maxima and makes S NaN.
    float S = 0.0f, T = 0.0f;
    if (m != -INFINITY) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const float d = lp_apart(x[i][c], m);
                const float e = __builtin_amdgcn_exp2f(d * 1.4426950408889634f);
                S += e;
                T += e * d;
            }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int c = 0; c < C; ++c) S += x[i][c] == -INFINITY ? 0.0f : x[i][c];  // a NaN
    }
    S = lp_wave_sum(S);
    T = lp_wave_sum(T);
    if (lane == 0) s_sum[wave][0] = m, s_sum[wave][1] = S, s_sum[wave][2] = T;
    if (top > 0) {
        s_best[threadIdx.x] = lp_key(best);
        __syncthreads();
        // thr: the top-th largest of the lanes' maxima, bit by bit (-inf with fewer lanes than
        // that), by one wave
        if (wave == 0) {
            uint32_t k[4], t = 0;
#pragma unroll
            for (int w = 0; w < 4; ++w) k[w] = s_best[64 * w + lane];
            for (int bit = 31; bit >= 0; --bit) {
                const uint32_t cand = t | 1u << bit;
                int n = 0;
#pragma unroll
                for (int w = 0; w < 4; ++w) n += __popcll(__builtin_amdgcn_ballot_w64(k[w] >= cand));
                if (n >= top) t = cand;
            }
            if (lane == 0) s_thr = t;
        }
        __syncthreads();
        const uint32_t thr = s_thr;
        const bool plain = S == S;  // no NaN and no +inf
        const int n = edge ? LpWave<TY, C, NV, true>{x, base, e0, V, lane}.list_top(lp_value(thr), top, plain, s_list[wave])
                           : LpWave<TY, C, NV, false>{x, base, e0, V, lane}.list_top(lp_value(thr), top, plain, s_list[wave]);
        if (lane == 0) s_n[wave] = n;
    }
    __syncthreads();
    uint8_t *slot = scratch + ((int64_t)row * P + p) * lp_slot(top);
    if (threadIdx.x == 255) {
        float M = -INFINITY, SS = 0.0f, TT = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) M = fmaxf(M, s_sum[w][0]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float d = lp_apart(s_sum[w][0], M), f = __expf(d);
            const bool none = s_sum[w][0] == -INFINITY;  // S is 0, or NaN
            SS += none ? s_sum[w][1] : f * s_sum[w][1];
            TT += none ? 0.0f : f * s_sum[w][2] + f * d * s_sum[w][1];
        }
        *(float4 *)slot = make_float4(M, SS, TT, 0.0f);
    }
    if (top == 0) return;
    // an entry's rank is the number of larger ones; the first `top` leave, 0 past the last
    uint64_t *out = (uint64_t *)(slot + 16);
    const int total = s_n[0] + s_n[1] + s_n[2] + s_n[3];
    for (int e = threadIdx.x; e < total; e += 256) {
        int w = 0, f = e;
        while (f >= s_n[w]) f -= s_n[w++];
        const uint64_t mine = s_list[w][f];
        int rank = 0;
        for (int o = 0; o < 4; ++o) {
            const int n = s_n[o];
#pragma unroll 8
            for (int g = 0; g < n; ++g) rank += s_list[o][g] > mine;
        }
        if (rank < top) out[rank] = mine;
    }
    if (threadIdx.x >= total && threadIdx.x < top) out[threadIdx.x] = 0;
}

template <int TY>
__global__ void __launch_bounds__(256) k_token_logprobs_merge(const tlh_token_logprobs_args a, int P,
                                                              const uint8_t *__restrict__ scratch) {
    const int lane = threadIdx.x & 63;
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= a.rows) return;
    const int top = a.top;
    const uint8_t *slot = scratch + ((int64_t)row * P + min(lane, P - 1)) * lp_slot(top);
    const float4 st = *(const float4 *)slot;
    // what is needed later starts on its way here
    const uint64_t *list = (const uint64_t *)(slot + 16);
    auto entry = [&](int i) { return lane < P && i < top ? list[i] : (uint64_t)0; };
    uint64_t ahead[LP_AHEAD];
#pragma unroll
    for (int i = 0; i < LP_AHEAD; ++i) ahead[i] = entry(i);
    const int token = a.logprobs ? a.tokens[row] : -1;
    const bool known = token >= 0 && token < a.vocab;
    const float x = known ? lp_elem<TY>(a.logits, (int64_t)row * a.row_stride + token) : 0.0f;
    float M = lane < P ? st.x : -INFINITY;
    for (int o = 1; o < 64; o <<= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    float S = 0.0f, T = 0.0f;
    if (lane < P) {
        if (st.x == -INFINITY) {
            S = st.y;  // 0, or NaN
        } else {
            const float d = lp_apart(st.x, M), f = __expf(d);
            S = f * st.y;
            T = f * st.z + f * d * st.y;
        }
    }
    S = lp_wave_sum(S);
    T = lp_wave_sum(T);
    const float lse = logf(S);
    if (lane == 0) {
        if (a.entropy) a.entropy[row] = lse - T / S;
        if (a.logprobs) a.logprobs[row] = known ? (x - M) - lse : __uint_as_float(0x7fc00000u);
    }
    // The lanes' lists are sorted. As in a chunk: the top-th largest of their first
    // entries is a threshold (0 with fewer of them), and the few that reach it are ranked
    // by counting.
    __shared__ uint64_t s_list[4][LP_MERGE];
    uint64_t *l = s_list[threadIdx.x >> 6];
    auto put = [&](int r, uint64_t e) {
        a.top_logprobs[(int64_t)row * top + r] = (lp_value((uint32_t)(e >> 32)) - M) - lse;
        a.top_ids[(int64_t)row * top + r] = (int32_t)~(uint32_t)e;
    };
    if (top == 0) return;
    uint32_t thr = 0;
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t cand = thr | 1u << bit;
        int reach = 0;
#pragma unroll
        for (int i = 0; i < LP_AHEAD; ++i) reach += __popcll(__builtin_amdgcn_ballot_w64((uint32_t)(ahead[i] >> 32) >= cand));
        if (reach >= top) thr = cand;
    }
    int n = 0;
    for (int i = 0; i < top && n <= LP_MERGE; ++i) {
        const uint64_t e = ahead[0];
        const bool in = e != 0 && (uint32_t)(e >> 32) >= thr;
        const uint64_t who = __builtin_amdgcn_ballot_w64(in);
        if (who == 0) break;
        const int at = n + lp_below(who);
        if (in && at < LP_MERGE) l[at] = e;
        n += __popcll(who);
#pragma unroll
        for (int j = 0; j + 1 < LP_AHEAD; ++j) ahead[j] = ahead[j + 1];
        ahead[LP_AHEAD - 1] = entry(i + LP_AHEAD);
    }
    if (n <= LP_MERGE) {
        __builtin_amdgcn_wave_barrier();
        for (int e = lane; e < n; e += 64) {
            const uint64_t mine = l[e];
            int rank = 0;
#pragma unroll 8
            for (int f = 0; f < n; ++f) rank += l[f] > mine;
            if (rank < top) put(rank, mine);
        }
        return;
    }
    // Many (equal logits): the largest head is the next entry; the two entries behind
    // each head are on their way while it is compared.
    uint64_t head = entry(0), next = entry(1), after = entry(2);
    int at = 2;
    for (int r = 0; r < top; ++r) {
        const uint32_t best = lp_wave_max((uint32_t)(head >> 32), P);
        bool mine = lane < P && head != 0 && (uint32_t)(head >> 32) == best;
        if (__popcll(__builtin_amdgcn_ballot_w64(mine)) > 1) {  // equal logits: the lowest index, the largest complement
            const uint32_t first = lp_wave_max(mine ? (uint32_t)head : 0u, P);
            mine = mine && (uint32_t)head == first;
        }
        if (mine) {
            put(r, head);
            head = next;
            next = after;
            after = entry(++at);
        }
    }
}

// A small vocabulary's chunk of 64 a lane would be mostly empty: 1393 rows of 2601, 29
// us with it, 16 with 16.
static bool lp_small(int64_t vocab) { return vocab <= 2 * LP_CHUNK_SMALL; }
static int lp_ept(int64_t rows, int64_t vocab) {
    // few rows: shorter chunks, so that more CUs share them
    return lp_small(vocab) || (rows * ((vocab + LP_CHUNK - 1) / LP_CHUNK) < 256 &&
                               vocab + 7 <= (int64_t)LP_CHUNK_SMALL * LP_LISTS)
               ? 16
               : 64;
}
static int lp_chunks(int64_t vocab, int ept) {
    return (int)((vocab + 7 + 256 * ept - 1) / (256 * ept));  // up to 7 places before a row that is not aligned
}

// Room for either chunk length, so that the size grows with the rows and one
// buffer for the largest batch serves every smaller one.
size_t token_logprobs_scratch_bytes(int64_t rows, int64_t vocab, int top) {
    const size_t chunks = lp_small(vocab) ? (size_t)rows * lp_chunks(vocab, 16)
                                          : (size_t)rows * lp_chunks(vocab, 64) +
                                                (size_t)std::min<int64_t>(rows, 256) * lp_chunks(vocab, 16);
    return chunks * lp_slot(top);
}

template <int TY> static void launch_lp(const tlh_token_logprobs_args &a, void *scratch, hipStream_t stream) {
    const int P = lp_chunks(a.vocab, lp_ept(a.rows, a.vocab));
    auto k = lp_ept(a.rows, a.vocab) == 16 ? k_token_logprobs<TY, 16> : k_token_logprobs<TY, 64>;
    for (int r0 = 0; r0 < a.rows; r0 += 65535) {  // grid y
        const int n = std::min(65535, a.rows - r0);
        hipLaunchKernelGGL(k, dim3(P, n), dim3(256), 0, stream,
                           (const char *)a.logits + (int64_t)r0 * a.row_stride * (TY == TLH_TYPE_F32 ? 4 : 2), a.row_stride,
                           a.vocab, a.top, P, (uint8_t *)scratch + (int64_t)r0 * P * lp_slot(a.top));
    }
    hipLaunchKernelGGL((k_token_logprobs_merge<TY>), dim3((a.rows + 3) / 4), dim3(256), 0, stream, a, P,
                       (const uint8_t *)scratch);
}

tlh_status launch_token_logprobs(const tlh_token_logprobs_args &a, void *scratch, hipStream_t stream) {
    switch (a.type) {
    case TLH_TYPE_F32: launch_lp<TLH_TYPE_F32>(a, scratch, stream); break;
    case TLH_TYPE_F16: launch_lp<TLH_TYPE_F16>(a, scratch, stream); break;
    default: launch_lp<TLH_TYPE_BF16>(a, scratch, stream); break;
    }
    return check_launch("token_logprobs");
}

}  // namespace tlh
