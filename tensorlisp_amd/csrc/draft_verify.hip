// Verification of drafted tokens from given random numbers, gfx950. With p and q the
// softmax of the target's and the drafter's logits over the temperature, draft i with
// token x is accepted where u_i q(x) < p(x); the first one refused is replaced by a
// token drawn from max(p - q, 0), and behind the last one accepted a token is drawn from p.
//
// Everything is f64. A drawn token is the first whose running sum exceeds r times the
// whole: with f32 terms (off by 2^-24 of themselves) the sums would be off by more than
// most of a vocabulary's tokens weigh, and the token would depend on the order of additions.
#include <algorithm>

#include "kernels.hpp"

namespace tlh {

struct DvRow {  // of a row of logits
    double sum;  // of exp((x - top) / T); 0 where the row is no distribution
    float top;   // its largest logit
    int at;      // the lowest index of that
};

template <int TY> __device__ __forceinline__ float dv_load(const void *p, int64_t i) {
    if constexpr (TY == TLH_TYPE_F32) return ((const float *)p)[i];
    else if constexpr (TY == TLH_TYPE_F16) return h2f(((const uint16_t *)p)[i]);
    else return bf16_to_f32(((const uint16_t *)p)[i]);
}

struct DvSeq {
    int b, n;  // first draft, drafts
};
__device__ __forceinline__ DvSeq dv_seq(const tlh_draft_verify_args &a, int s) {
    DvSeq q;
    q.b = max(0, min(a.draft_starts[s], a.num_drafts));
    q.n = min(max(q.b, min(a.draft_starts[s + 1], a.num_drafts)) - q.b, a.max_drafts);
    return q;
}

// p(x) of element x of a row
__device__ __forceinline__ double dv_weight(float x, float top, double inv_t) {
    return x == -INFINITY ? 0.0 : exp(((double)x - (double)top) * inv_t);
}

// One workgroup a (sequence; draft or the row behind them; target or draft row).
template <int TY>
__global__ void __launch_bounds__(256) k_draft_rows(const tlh_draft_verify_args a, DvRow *rows) {
    const int s = blockIdx.y, which = blockIdx.z;
    const DvSeq q = dv_seq(a, s);
    const float T = a.temperatures[s];
    const bool greedy = !(T > 0.0f);
    __shared__ float s_m[256];
    __shared__ int s_at[256];
    __shared__ double s_s[256];
    for (int i = blockIdx.x; i < q.n + 1 - which; i += gridDim.x) {
        const void *logits = which ? a.draft : a.target;
        const int64_t base = which ? (q.b + i) * a.draft_stride : ((int64_t)q.b + s + i) * a.target_stride;
        float m = -INFINITY;
        int at = 0;
        bool bad = false;
        for (int e = threadIdx.x; e < a.vocab; e += 256) {
            const float x = dv_load<TY>(logits, base + e);
            if (x > m) m = x, at = e;
            bad |= x != x || (x == INFINITY && !greedy);
        }
        __syncthreads();
        s_m[threadIdx.x] = bad ? NAN : m, s_at[threadIdx.x] = at;
        __syncthreads();
        m = -INFINITY, at = 0x7fffffff, bad = false;
        for (int t = 0; t < 256; ++t) {
            bad |= s_m[t] != s_m[t];
            if (s_m[t] > m || (s_m[t] == m && s_at[t] < at)) m = s_m[t], at = s_at[t];
        }
        bad |= m == -INFINITY;
        double sum = 0.0;
        if (!bad && !greedy)
            for (int e = threadIdx.x; e < a.vocab; e += 256) sum += dv_weight(dv_load<TY>(logits, base + e), m, 1.0 / (double)T);
        s_s[threadIdx.x] = sum;
        __syncthreads();
        if (threadIdx.x == 0) {
            DvRow r = {bad ? 0.0 : 1.0, m, at};
            if (!bad && !greedy) {
                r.sum = 0.0;
                for (int t = 0; t < 256; ++t) r.sum += s_s[t];
            }
            rows[which ? a.num_drafts + a.num_seqs + q.b + i : q.b + s + i] = r;
        }
    }
}

// One workgroup a sequence: the tests, then the token.
template <int TY>
__global__ void __launch_bounds__(256) k_draft_decide(const tlh_draft_verify_args a, const DvRow *rows) {
    const int s = blockIdx.x;
    const DvSeq sq = dv_seq(a, s);
    const float T = a.temperatures[s];
    const bool greedy = !(T > 0.0f);
    const double inv_t = 1.0 / (double)T;
    const DvRow *target = rows + sq.b + s, *draft = rows + a.num_drafts + a.num_seqs + sq.b;
    auto weight = [&](const void *logits, int64_t base, const DvRow &r, int x) {
        if (x < 0 || x >= a.vocab) return 0.0;
        if (greedy) return x == r.at ? 1.0 : 0.0;
        return dv_weight(dv_load<TY>(logits, base + x), r.top, inv_t) / r.sum;
    };
    auto p_of = [&](int i, int x) { return weight(a.target, ((int64_t)sq.b + s + i) * a.target_stride, target[i], x); };
    auto q_of = [&](int i, int x) {
        if (!a.draft) return x == a.tokens[sq.b + i] && x >= 0 && x < a.vocab ? 1.0 : 0.0;
        return weight(a.draft, (int64_t)(sq.b + i) * a.draft_stride, draft[i], x);
    };
    int stop = sq.n;
    bool none = false;  // no distribution where it stops
    for (int i = sq.n - 1; i >= 0; --i) {
        const int x = a.tokens[sq.b + i];
        const bool bad = target[i].sum == 0.0 || (a.draft && !greedy && draft[i].sum == 0.0);
        const double p = bad ? 0.0 : p_of(i, x), q = bad ? 0.0 : greedy ? 1.0 : q_of(i, x);
        const bool ok = !bad && (greedy ? p == 1.0 : (double)a.accept_at[sq.b + i] * q < p);
        if (threadIdx.x == 0 && a.accept_probs)
            a.accept_probs[sq.b + i] = bad ? NAN : q > 0.0 ? (float)fmin(1.0, p / q) : p > 0.0 ? 1.0f : 0.0f;
        if (!ok) stop = i, none = bad;
    }
    if (stop == sq.n) none = target[stop].sum == 0.0;
    int next = -1;
    if (!none && greedy) next = target[stop].at;
    if (!none && !greedy) {
        __shared__ double s_s[256];
        __shared__ int s_last[256], s_next;
        const int each = (a.vocab + 255) / 256, e0 = threadIdx.x * each, e1 = min(e0 + each, a.vocab);
        for (int whole = stop == sq.n; whole < 2; ++whole) {  // from p where p - q has nothing
            auto mass = [&](int x) { return whole ? p_of(stop, x) : fmax(p_of(stop, x) - q_of(stop, x), 0.0); };
            double sum = 0.0;
            int last = -1;
            for (int e = e0; e < e1; ++e) {
                const double w = mass(e);
                sum += w;
                if (w > 0.0) last = e;
            }
            __syncthreads();
            s_s[threadIdx.x] = sum, s_last[threadIdx.x] = last;
            if (threadIdx.x == 0) s_next = 0x7fffffff;
            __syncthreads();
            double before = 0.0, total = 0.0;
            last = -1;
            for (int t = 0; t < 256; ++t) {
                if (t == threadIdx.x) before = total;
                total += s_s[t];
                last = max(last, s_last[t]);
            }
            if (total == 0.0) continue;
            const double reach = (double)a.sample_at[s] * total;
            if (before + sum > reach) {
                for (int e = e0; e < e1; ++e) {
                    before += mass(e);
                    if (before > reach) {
                        atomicMin(&s_next, e);
                        break;
                    }
                }
            }
            __syncthreads();
            next = s_next == 0x7fffffff ? last : s_next;
            break;
        }
    }
    int32_t *out = a.out_tokens + (int64_t)s * (a.max_drafts + 1);
    for (int i = threadIdx.x; i <= a.max_drafts; i += 256) out[i] = i < stop ? a.tokens[sq.b + i] : i == stop ? next : -1;
    if (threadIdx.x == 0) a.accepted[s] = stop;
}

size_t draft_verify_scratch_bytes(const tlh_draft_verify_args &a) {
    return sizeof(DvRow) * ((size_t)a.num_drafts + a.num_seqs + (a.draft ? a.num_drafts : 0));
}

template <int TY> static void launch_dv(const tlh_draft_verify_args &a, void *scratch, hipStream_t stream) {
    const int n = std::min(a.max_drafts, a.num_drafts) + 1;
    hipLaunchKernelGGL((k_draft_rows<TY>), dim3(n, a.num_seqs, a.draft ? 2 : 1), dim3(256), 0, stream, a, (DvRow *)scratch);
    hipLaunchKernelGGL((k_draft_decide<TY>), dim3(a.num_seqs), dim3(256), 0, stream, a, (const DvRow *)scratch);
}

tlh_status launch_draft_verify(const tlh_draft_verify_args &a, void *scratch, hipStream_t stream) {
    switch (a.type) {
    case TLH_TYPE_F32: launch_dv<TLH_TYPE_F32>(a, scratch, stream); break;
    case TLH_TYPE_F16: launch_dv<TLH_TYPE_F16>(a, scratch, stream); break;
    default: launch_dv<TLH_TYPE_BF16>(a, scratch, stream); break;
    }
    return check_launch("draft_verify");
}

}  // namespace tlh
