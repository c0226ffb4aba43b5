// Log probabilities of given tokens, the distributions' entropies and the
// likeliest alternatives, gfx950. For a row x of V logits with m = max x,
// S = sum exp(x - m), T = sum exp(x - m) (x - m):
//   log p(t) = (x_t - m) - log S,   H = log S - T / S,
// and the `top` largest x, equal ones by the lowest index.
//
// The bound is one read of the logits. A workgroup takes a chunk of a row into
// registers, so the chunk's maximum is known before its exponentials (one pass,
// no rescaling) and its largest elements are found without a second read:
//  * every wave takes the top-th largest of its lanes' maxima as a threshold
//    (at least `top` elements reach it, few more do), lists the elements above
//    it and the first `top` that equal it, and ranks them by counting;
//  * a vocabulary-wide run of equal logits (a grammar's -inf mask) costs no
//    more: ties are taken in index order and only up to `top`;
//  * more elements above the threshold than the list holds (the largest ones
//    crowded into few lanes) are taken one maximum at a time instead.
// A second launch folds the chunks' sums and merges their sorted lists, one
// wave a row with one list a lane.
#include <algorithm>

#include "kernels.hpp"

namespace tlh {

constexpr int LP_MAX_TOP = 32;
constexpr int LP_CAP = 256;       // listed elements above a wave's threshold
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

template <typename T> __device__ __forceinline__ T lp_wave_max(T v) {
    for (int o = 1; o < 64; o <<= 1) v = max(v, (T)__shfl_xor(v, o, 64));
    return v;
}
__device__ __forceinline__ float lp_wave_sum(float v) {
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
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

template <int TY, int EPT>
__global__ void __launch_bounds__(256) k_token_logprobs(const void *__restrict__ logits, int64_t row_stride, int V,
                                                        int top, int P, uint8_t *__restrict__ scratch) {
    constexpr int C = TY == TLH_TYPE_F32 ? 4 : 8;  // elements of a 16-byte load
    constexpr int ES = 16 / C, NV = EPT / C;
    __shared__ uint64_t s_list[4][LP_CAP + LP_MAX_TOP];
    __shared__ uint64_t s_top[4][LP_MAX_TOP];
    __shared__ float s_sum[4][3];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int row = blockIdx.y, p = blockIdx.x;
    const char *base = (const char *)logits + (int64_t)row * row_stride * ES;
    // Loads are aligned whatever the row's address: element 0 of the chunks'
    // numbering lies up to C - 1 elements before the row.
    const int mis = (int)(((uintptr_t)base & 15) / ES);
    const int v0 = p * 256 * EPT + threadIdx.x * C - mis;  // the first of vector i's elements: v0 + 256 * C * i
    float x[NV][C];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int e = v0 + 256 * C * i;
        if (e >= 0 && e + C <= V) {
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
    auto there = [&](int i, int c) {
        const int e = v0 + 256 * C * i + c;
        return e >= 0 && e < V;
    };
    auto key_of = [&](int i, int c) { return there(i, c) ? lp_key(x[i][c]) : 0u; };

    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int c = 0; c < C; ++c) m = fmaxf(m, x[i][c]);
    for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    float S = 0.0f, T = 0.0f;
    // all -inf: S = 0. A NaN is not in the maximum, and makes S NaN unless m is -inf
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const float d = x[i][c] - m, e = __expf(d);
            S += x[i][c] == -INFINITY ? 0.0f : e;
            T += e > 0.0f && x[i][c] != -INFINITY ? e * d : 0.0f;
        }
    S = lp_wave_sum(S);
    T = lp_wave_sum(T);
    if (lane == 0) s_sum[wave][0] = m, s_sum[wave][1] = S, s_sum[wave][2] = T;

    if (top > 0) {
        uint32_t best = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int c = 0; c < C; ++c) best = max(best, key_of(i, c));
        // the top-th largest lane maximum, bit by bit
        uint32_t thr = 0;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t cand = thr | 1u << bit;
            if (__popcll(__builtin_amdgcn_ballot_w64(best >= cand)) >= top) thr = cand;
        }
        int above = 0, equal = 0;
        uint64_t *list = s_list[wave];  // the elements above thr, and from LP_CAP on those that equal it
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            uint64_t gt[C], eq[C];
            uint64_t any = 0;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const uint32_t k = key_of(i, c);
                gt[c] = __builtin_amdgcn_ballot_w64(k > thr);
                eq[c] = __builtin_amdgcn_ballot_w64(k == thr && k != 0);
                any |= gt[c] | eq[c];
            }
            if (any) {
                int before = 0, gts = 0, eqs = 0;  // of the lanes below: elements equal to thr
#pragma unroll
                for (int c = 0; c < C; ++c) before += lp_below(eq[c]);
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const uint64_t entry = lp_entry(key_of(i, c), v0 + 256 * C * i + c);
                    const int ga = above + gts + lp_below(gt[c]);
                    if ((gt[c] >> lane) & 1 && ga < LP_CAP) list[ga] = entry;
                    gts += __popcll(gt[c]);
                    if ((eq[c] >> lane) & 1) {
                        if (equal + before < top) list[LP_CAP + equal + before] = entry;
                        ++before;
                    }
                    eqs += __popcll(eq[c]);
                }
                above += gts;
                equal += eqs;
            }
        }
        if (lane < LP_MAX_TOP) s_top[wave][lane] = 0;
        if (above <= LP_CAP) {
            const int ne = min(equal, top), n = above + ne;
            __builtin_amdgcn_wave_barrier();
            for (int e = lane; e < n; e += 64) {
                const uint64_t mine = list[e < above ? e : LP_CAP + e - above];
                int rank = 0;
                for (int f = 0; f < n; ++f) rank += list[f < above ? f : LP_CAP + f - above] > mine;
                if (rank < top) s_top[wave][rank] = mine;
            }
        } else {  // one maximum at a time, each below the last
            uint64_t last = ~(uint64_t)0;
            for (int r = 0; r < top; ++r) {
                uint64_t b = 0;
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int c = 0; c < C; ++c) {
                        const uint32_t k = key_of(i, c);
                        const uint64_t entry = k ? lp_entry(k, v0 + 256 * C * i + c) : 0;
                        if (entry < last && entry > b) b = entry;
                    }
                last = lp_wave_max(b);
                if (lane == 0) s_top[wave][r] = last;
            }
        }
    }
    __syncthreads();
    uint8_t *slot = scratch + ((int64_t)row * P + p) * lp_slot(top);
    if (threadIdx.x == 0) {
        float M = -INFINITY, SS = 0.0f, TT = 0.0f;
        for (int w = 0; w < 4; ++w) M = fmaxf(M, s_sum[w][0]);
        for (int w = 0; w < 4; ++w) {
            const float d = s_sum[w][0] - M, f = __expf(d);
            if (s_sum[w][0] == -INFINITY) {
                SS += s_sum[w][1];  // 0, or NaN
                continue;
            }
            SS += f * s_sum[w][1];
            TT += f * s_sum[w][2] + f * d * s_sum[w][1];
        }
        *(float4 *)slot = make_float4(M, SS, TT, 0.0f);
    }
    // merge the waves' sorted lists: an entry's rank is its place in its own
    // list and the larger ones of the others
    for (int e = threadIdx.x; e < 4 * top; e += 256) {
        const int w = e / top, r = e % top;
        const uint64_t mine = s_top[w][r];
        int rank = r;
        for (int o = 1; o < 4; ++o)
            for (int f = 0; f < top; ++f) rank += s_top[(w + o) & 3][f] > mine;
        if (mine && rank < top) ((uint64_t *)(slot + 16))[rank] = mine;
    }
    // places past the chunk's last element
    int present = 0;
    for (int w = 0; w < 4; ++w)
        for (int f = 0; f < top; ++f) present += s_top[w][f] != 0;
    for (int r = present + threadIdx.x; r < top; r += 256) ((uint64_t *)(slot + 16))[r] = 0;
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
    float M = lane < P ? st.x : -INFINITY;
    for (int o = 1; o < 64; o <<= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    float S = 0.0f, T = 0.0f;
    if (lane < P) {
        if (st.x == -INFINITY) {
            S = st.y;  // 0, or NaN
        } else {
            const float d = st.x - M, f = __expf(d);
            S = f * st.y;
            T = f * st.z + f * d * st.y;
        }
    }
    S = lp_wave_sum(S);
    T = lp_wave_sum(T);
    const float lse = logf(S);
    if (lane == 0) {
        if (a.entropy) a.entropy[row] = lse - T / S;
        if (a.logprobs) {
            const int t = a.tokens[row];
            float lp = __uint_as_float(0x7fc00000u);
            if (t >= 0 && t < a.vocab) lp = (lp_elem<TY>(a.logits, (int64_t)row * a.row_stride + t) - M) - lse;
            a.logprobs[row] = lp;
        }
    }
    const uint64_t *list = (const uint64_t *)(slot + 16);
    int at = 0;
    uint64_t head = lane < P && top > 0 ? list[0] : 0;
    for (int r = 0; r < top; ++r) {
        const uint64_t best = lp_wave_max(head);
        if (head == best && best) {  // entries are unique
            a.top_logprobs[(int64_t)row * top + r] = (lp_value((uint32_t)(best >> 32)) - M) - lse;
            a.top_ids[(int64_t)row * top + r] = (int32_t)~(uint32_t)best;
            ++at;
            head = at < top ? list[at] : 0;
        }
    }
}

static int lp_ept(int64_t rows, int64_t vocab) {
    // few rows: shorter chunks, so that more CUs share them
    return rows * ((vocab + LP_CHUNK - 1) / LP_CHUNK) < 256 && vocab + 7 <= (int64_t)LP_CHUNK_SMALL * LP_LISTS ? 16 : 64;
}
static int lp_chunks(int64_t vocab, int ept) {
    return (int)((vocab + 7 + 256 * ept - 1) / (256 * ept));  // up to 7 places before a row that is not aligned
}

// Room for either chunk length, so that the size grows with the rows and one
// buffer for the largest batch serves every smaller one.
size_t token_logprobs_scratch_bytes(int64_t rows, int64_t vocab, int top) {
    return ((size_t)rows * lp_chunks(vocab, 64) + (size_t)std::min<int64_t>(rows, 256) * lp_chunks(vocab, 16)) * lp_slot(top);
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
