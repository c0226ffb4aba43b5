// Verification of drafted tokens from given random numbers, gfx950. With p and q the
// softmax of the target's and the drafter's logits over the temperature, draft i with
// token x is accepted where u_i q(x) < p(x); the first one refused is replaced by a
// token drawn from max(p - q, 0), and behind the last one accepted a token is drawn from p.
//
// Everything is f64. A drawn token is the first whose running sum exceeds r times the
// whole: with f32 terms (off by 2^-24 of themselves) the sums would be off by more than
// most of a vocabulary's tokens weigh, and the token would depend on the order of
// additions. f64 products run at f32's rate here, so the bound is one read of the logits.
//
// Three launches: the sums of chunks of all rows, a chunk a workgroup; then every workgroup
// of a sequence finds where it stops, and sums its chunk of what the token there is drawn
// from; then one workgroup a sequence finds the chunk and the token in it.
// Measured, us (the three launches, with the same logits again): 1 x 4 drafts of 128256 f32 5.6
// + 7.9 + 5.7, of which 4.5 + 5 + 5 are there with 1000 tokens, chains of latencies; 32 x 1..8
// of 128256 f32, 149 MB, 40.2 (f64, as long as a read from memory) + 16.5 + 10.0; 48 x 10 of
// 32003 bf16, proposed outright, 25.4 (f64: half the bytes an element) + 9.4 + 8.4. With logits
// that no cache holds the calls take 24, 75 and 48 us, with the same ones 19.4, 65 and 41; all
// greedy, 1 x 4 and 32 x 1..8 15 and 34 (26 with the same).
#include <algorithm>
#include <type_traits>

#include "kernels.hpp"
#include "wave_ops.hpp"

namespace tlh {

constexpr int DV_MAX_CHUNKS = 64;  // of a row: a lane each
// elements of a chunk: 64 (or 16, for few rows) of each of 256 lanes
constexpr int DV_CHUNK = 64 * 256, DV_CHUNK_SMALL = 16 * 256;

// Sums of exp((x - ref) / T) need no running maximum: f64 holds 2^900 times a term as well
// as the term, so `ref` is some early element, and only a chunk with one further above it
// is taken again.
constexpr double DV_ABOVE = 900.0;  // powers of 2

struct DvPart {  // of a chunk of a row
    double sum;  // of exp((x - ref) / T); NaN where the chunk rules a distribution out
    float ref;   // (greedy: its largest logit; -inf: it holds nothing else)
    int at;      // greedy: the lowest index of that
};
struct DvMass {  // of a chunk of what is drawn from
    double sum, whole;  // of max(p - q, 0), of p
};
struct DvStop {  // of a sequence
    double zp, zq;    // the sums of the rows drawn from
    float mp, mq;     // ... and what their exponents are taken from
    int stop, draws;  // drafts accepted; whether a token is to be drawn
};

template <int TY> __device__ __forceinline__ float dv_elem(const void *p, int64_t i) {
    if constexpr (TY == TLH_TYPE_F32) return ((const float *)p)[i];
    else if constexpr (TY == TLH_TYPE_F16) return h2f(((const uint16_t *)p)[i]);
    else return bf16_to_f32(((const uint16_t *)p)[i]);
}

// exp((x - ref) / T) with c = log2(e) / T, off by less than 2^-45 of it (and 2^-52 times the
// exponent): 2^k times the polynomial that agrees with 2^f, |f| <= 1/2, at the ten Chebyshev
// nodes. The instructions that convert between f64 and integers, round or scale are slow
// beside its additions and products: k is the low word of the sum with 1.5 x 2^52, and is
// added to the result's exponent. Nothing is left below 2^-1000, and nothing of a masked
// logit (-inf), at any temperature. (32 x 1..8, the rows' sums, us: with rint, ldexp and a
// Taylor series up to f^12 56, up to f^11 without them 43, this 40.)
struct DvExp {
    double k[10];  // from f^9 down, in vector registers: else each would be moved there for every use
    __device__ __forceinline__ DvExp()
        : k{1.0205905413765595e-07, 1.325964524488711e-06, 1.5252672924850737e-05, 0.0001540343375125101, 0.0013333558200794592,
            0.009618129193934313, 0.05550410866465167, 0.2402265069564034, 0.6931471805599462, 1.0000000000000135} {
#pragma unroll
        for (int i = 0; i < 10; ++i) asm("" : "+v"(k[i]));
    }
    __device__ __forceinline__ double operator()(float x, float ref, double c) const {
        const double t = ((double)x - (double)ref) * c;
        const double big = t + 6755399441055744.0, f = t - (big - 6755399441055744.0);
        double e = k[0];
#pragma unroll
        for (int i = 1; i < 10; ++i) e = fma(e, f, k[i]);
        const uint64_t bits = __builtin_bit_cast(uint64_t, e);
        const uint32_t hi = (uint32_t)(bits >> 32) + ((uint32_t)__builtin_bit_cast(uint64_t, big) << 20);
        const bool some = t >= -1000.0;  // (no NaN: 0 times an infinity)
        return __builtin_bit_cast(double, some ? (uint64_t)hi << 32 | (uint32_t)bits : 0);
    }
};
constexpr double DV_LOG2E = 1.4426950408889634074;
// what p = wp ip has above q = wq iq: of equal distributions exactly 0
__device__ __forceinline__ double dv_above(double wp, double ip, double wq, double iq) {
#pragma clang fp contract(off)
    return fmax(wp * ip - wq * iq, 0.0);
}
// ... and a sum of those that equal distributions in another order of additions may leave
constexpr double DV_NOTHING = 0x1p-40;

__device__ __forceinline__ double dv_sum(double v, int lanes = 64) {
    return wave_all(v, lanes, [](double a, double b) { return a + b; });
}
__device__ __forceinline__ float dv_max(float v, int lanes = 64) { return wave_all(v, lanes, [](float a, float b) { return fmaxf(a, b); }); }
__device__ __forceinline__ int dv_min(int v, int lanes = 64) { return wave_all(v, lanes, [](int a, int b) { return min(a, b); }); }

struct DvSeq {
    int b, n;  // first draft, drafts that are looked at
};
__device__ __forceinline__ int dv_start(const tlh_draft_verify_args &a, int s) { return max(0, min(a.draft_starts[s], a.num_drafts)); }
__device__ __forceinline__ DvSeq dv_seq(const tlh_draft_verify_args &a, int s) {
    DvSeq q;
    q.b = dv_start(a, s);
    q.n = min(max(q.b, dv_start(a, s + 1)) - q.b, a.max_drafts);
    return q;
}
// The last sequence whose first row (of drafts: its first draft, else with one more row a
// sequence) is `row` or before it; starts are looked at 64 at a time. Where they decrease it is
// some sequence, and what follows from it is not used (dv_alone).
__device__ __forceinline__ int dv_find(const tlh_draft_verify_args &a, int row, bool target, int lane) {
    int lo = 0, len = a.num_seqs;
    while (len > 1) {
        const int stride = (len + 63) / 64, s = lo + lane * stride;
        const bool in = s < lo + len && dv_start(a, s) + (target ? s : 0) <= row;
        const int n = max(1, (int)__popcll(__builtin_amdgcn_ballot_w64(in)));
        const int next = lo + (n - 1) * stride;
        len = min(stride, lo + len - next);
        lo = next;
    }
    return lo;
}

// C consecutive elements of a row in 16 bytes, from element e on; what lies outside it is
// -inf. Loads are aligned whatever the row's address (`shift` elements past 16 bytes): a
// chunk's numbering begins up to C - 1 elements before the row.
template <int TY> struct DvLoad {
    static constexpr int C = TY == TLH_TYPE_F32 ? 4 : 8, ES = 16 / C;
    const char *base;
    int V, shift;
    __device__ __forceinline__ DvLoad(const void *logits, int64_t row, int64_t stride, int vocab)
        : base((const char *)logits + row * stride * ES), V(vocab), shift((int)(((uintptr_t)base & 15) / ES)) {}
    __device__ __forceinline__ void whole(int e, float (&x)[C]) const {
        const uint4 w = *(const uint4 *)(base + (int64_t)e * ES);
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int c = 0; c < C; ++c)
            x[c] = TY == TLH_TYPE_F32   ? __uint_as_float(ws[c % 4])
                   : TY == TLH_TYPE_F16 ? h2f((uint16_t)(ws[c / 2 % 4] >> (16 * (c & 1))))
                                        : bf16_to_f32((uint16_t)(ws[c / 2 % 4] >> (16 * (c & 1))));
    }
    __device__ __forceinline__ void vec(int e, bool aligned, float (&x)[C]) const {
        if (aligned && e >= 0 && e + C <= V) whole(e, x);
        else {
#pragma unroll
            for (int c = 0; c < C; ++c) x[c] = e + c >= 0 && e + c < V ? dv_elem<TY>(base, e + c) : -INFINITY;
        }
    }
};

// the larger one, or a NaN
__device__ __forceinline__ float dv_top(float a, float b) { return __builtin_elementwise_maximum(a, b); }

template <int TY>
__global__ void __launch_bounds__(256) k_draft_rows(const tlh_draft_verify_args a, int r0, int rows, int P, int chunk, int *__restrict__ odd,
                                                    DvPart *__restrict__ parts) {
    using L = DvLoad<TY>;
    constexpr int C = L::C, AT_ONCE = 16 / C, STEP = 256 * C * AT_ONCE;  // vectors on their way at a time
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, p = blockIdx.x;
    const int r = r0 + blockIdx.y, targets = a.num_drafts + a.num_seqs;
    if (r == rows) {  // behind the rows: whether a start is below the one before it
        if (p > 0) return;
        int any = 0;
        for (int s = threadIdx.x; s < a.num_seqs; s += 256) any |= dv_start(a, s + 1) < dv_start(a, s);
        any = __syncthreads_or(any);
        if (threadIdx.x == 0) *odd = any;
        return;
    }
    const bool target = r < targets;
    const int row = target ? r : r - targets;
    const int s = __builtin_amdgcn_readfirstlane(dv_find(a, row, target, lane));
    const DvSeq q = dv_seq(a, s);
    const float T = a.temperatures[s];
    const bool greedy = !(T > 0.0f);
    const int i = row - q.b - (target ? s : 0);
    if (i < 0 || i >= q.n + (target ? 1 : 0) || (greedy && !target)) return;  // nobody looks at the row
    const L load(target ? a.target : a.draft, row, target ? a.target_stride : a.draft_stride, a.vocab);
    const int begin = p * chunk - load.shift, end = min(begin + chunk, a.vocab), first = begin + threadIdx.x * C;
    const double c_t = greedy ? 0.0 : DV_LOG2E / (double)T;
    float top = -INFINITY, ref = -INFINITY;
    int at = 0x7fffffff;
    double sum = 0.0;
    // (edge: the chunk reaches past the row)
    const DvExp weight;
    auto get = [&](auto edge, int e, float (&x)[AT_ONCE][C]) {
#pragma unroll
        for (int v = 0; v < AT_ONCE; ++v) {
            if constexpr (edge()) load.vec(e + 256 * C * v, true, x[v]);
            else load.whole(e + 256 * C * v, x[v]);
        }
    };
    auto pass = [&](auto edge) {
        top = -INFINITY, sum = 0.0;
        float next[AT_ONCE][C];
        get(edge, first, next);
#pragma unroll 1
        for (int e = first; e - (int)threadIdx.x * C < end; e += STEP) {
            float x[AT_ONCE][C];
#pragma unroll
            for (int v = 0; v < AT_ONCE; ++v)
#pragma unroll
                for (int c = 0; c < C; ++c) x[v][c] = next[v][c];
            if (e - (int)threadIdx.x * C + STEP < end) get(edge, e + STEP, next);
            float m = x[0][0];
#pragma unroll
            for (int v = 0; v < AT_ONCE; ++v)
#pragma unroll
                for (int c = 0; c < C; ++c) m = dv_top(m, x[v][c]);
            if (greedy) {
                if (m > top) {
#pragma unroll
                    for (int v = AT_ONCE - 1; v >= 0; --v)
#pragma unroll
                        for (int c = C - 1; c >= 0; --c) at = x[v][c] == m ? e + 256 * C * v + c : at;
                }
                top = dv_top(top, m);
                continue;
            }
            top = dv_top(top, m);
            ref = ref == -INFINITY ? top : ref;
            if (__builtin_amdgcn_ballot_w64(ref != -INFINITY) == 0) continue;  // masked so far
#pragma unroll
            for (int v = 0; v < AT_ONCE; ++v)
#pragma unroll
                for (int c = 0; c < C; ++c) sum += weight(x[v][c], ref, c_t);
        }
    };
    for (;;) {
        if (begin < 0 || begin + chunk > a.vocab) pass(std::true_type());
        else pass(std::false_type());
        if (greedy || !(((double)top - (double)ref) * c_t > DV_ABOVE)) break;
        ref = top;
    }
    const bool bad = greedy ? top != top : !(top < INFINITY);
    __shared__ float s_ref[4];
    __shared__ double s_sum[4];
    __shared__ int s_at[4];
    if (greedy) ref = top;
    const float all = dv_max(ref);
    if (lane == 0) s_ref[wave] = all;
    __syncthreads();
    const float R = fmaxf(fmaxf(s_ref[0], s_ref[1]), fmaxf(s_ref[2], s_ref[3]));
    if (greedy) at = dv_min(ref == R ? at : 0x7fffffff);
    else sum = dv_sum(sum * weight(ref, R, c_t));  // (no element but -inf: 0)
    if (__builtin_amdgcn_ballot_w64(bad) != 0) sum = NAN;
    if (lane == 0) s_sum[wave] = sum, s_at[wave] = at;
    __syncthreads();
    if (threadIdx.x == 0)
        parts[(int64_t)r * P + p] = {(s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]), R, min(min(s_at[0], s_at[1]), min(s_at[2], s_at[3]))};
}

// A row's parts joined by `lanes` lanes, one a chunk
struct DvRow {
    double z;  // the sum of exp((x - m) / T); NaN: no distribution
    float m;
    int at;    // greedy: the likeliest token
};
__device__ __forceinline__ DvRow dv_row(const DvExp &weight, const DvPart *parts, int P, int c, int lanes, bool greedy, double c_t) {
    DvPart x = {0.0, -INFINITY, 0x7fffffff};
    if (c < P) x = parts[c];
    DvRow r;
    r.m = dv_max(x.ref, lanes);
    double z = x.ref == -INFINITY ? 0.0 : x.sum * (greedy ? 0.0 : weight(x.ref, r.m, c_t));
    if (x.sum != x.sum) z = NAN;
    r.z = dv_sum(z, lanes);
    r.at = greedy ? dv_min(x.ref == r.m ? x.at : 0x7fffffff, lanes) : 0;
    if (r.m == -INFINITY) r.z = NAN;
    return r;
}

// Whether draft x is accepted, and the probability of that; tx and dx: its logits
struct DvTest {
    bool ok;
    float prob;
};
__device__ __forceinline__ DvTest dv_test(const DvExp &weight, const DvRow &t, const DvRow &d, int x, bool known, bool drawn, float tx, float dx,
                                          float u, bool greedy, double c_t) {
    const bool bad = t.z != t.z || d.z != d.z;
    const double px = greedy ? (known && x == t.at ? 1.0 : 0.0) : known ? weight(tx, t.m, c_t) / t.z : 0.0;
    const double qx = !known ? 0.0 : drawn ? weight(dx, d.m, c_t) / d.z : 1.0;
    return {!bad && (greedy ? px == 1.0 : (double)u * qx < px),
            bad ? NAN : qx > 0.0 ? (float)fmin(1.0, px / qx) : px > 0.0 ? 1.0f : 0.0f};
}

template <int TY>
__global__ void __launch_bounds__(256) k_draft_masses(const tlh_draft_verify_args a, int P, int M, int chunk, int lanes,
                                                      const DvPart *__restrict__ parts, DvStop *__restrict__ stops,
                                                      DvMass *__restrict__ masses) {
    using L = DvLoad<TY>;
    constexpr int C = L::C;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, s = blockIdx.y, p = blockIdx.x;
    const DvSeq q = dv_seq(a, s);
    const float T = a.temperatures[s];
    const bool greedy = !(T > 0.0f);
    const double c_t = DV_LOG2E / (double)T;
    const int64_t t0 = q.b + s;                                      // the target's first row
    const DvPart *tp = parts + t0 * P, *dp = parts + ((int64_t)a.num_drafts + a.num_seqs + q.b) * P;
    const DvExp weight;
    __shared__ int s_stop;
    if (threadIdx.x == 0) s_stop = q.n;
    __syncthreads();
    // `lanes` lanes a draft
    const int each = 256 / lanes, c = threadIdx.x & (lanes - 1);
    for (int i0 = 0; i0 < q.n; i0 += each) {
        const int i = min(i0 + (int)threadIdx.x / lanes, q.n - 1);
        const int x = a.tokens[q.b + i];
        const bool known = x >= 0 && x < a.vocab, drawn = a.draft && !greedy;
        const float u = a.accept_at[q.b + i];
        const float tx = known ? dv_elem<TY>(a.target, (t0 + i) * a.target_stride + x) : -INFINITY;
        const float dx = known && drawn ? dv_elem<TY>(a.draft, (int64_t)(q.b + i) * a.draft_stride + x) : -INFINITY;
        const DvRow t = dv_row(weight, tp + (int64_t)i * P, P, c, lanes, greedy, c_t);
        const DvRow d = drawn ? dv_row(weight, dp + (int64_t)i * P, P, c, lanes, false, c_t) : DvRow{1.0, 0.0f, 0};
        const DvTest test = dv_test(weight, t, d, x, known, drawn, tx, dx, u, greedy, c_t);
        if (c == 0 && !test.ok) atomicMin(&s_stop, i);
        if (p == 0 && c == 0 && a.accept_probs) a.accept_probs[q.b + i] = test.prob;
    }
    __syncthreads();
    const int stop = s_stop;
    const bool minus = stop < q.n && a.draft && !greedy;  // a refused draft: its drafter's weights are taken off
    const DvRow t = dv_row(weight, tp + (int64_t)stop * P, P, lane, 64, greedy, c_t);
    const DvRow d = minus ? dv_row(weight, dp + (int64_t)stop * P, P, lane, 64, false, c_t) : DvRow{0.0, 0.0f, 0};
    const bool bad = t.z != t.z || d.z != d.z;
    const int outright = stop < q.n && !a.draft && !greedy ? a.tokens[q.b + stop] : -1;  // and of one proposed outright, itself
    if (p == 0) {
        int32_t *out = a.out_tokens + (int64_t)s * (a.max_drafts + 1);
        for (int i = threadIdx.x; i <= a.max_drafts; i += 256)
            out[i] = i < stop ? a.tokens[q.b + i] : i == stop && greedy && !bad ? t.at : -1;
        if (threadIdx.x == 0) {
            a.accepted[s] = stop;
            stops[s] = {t.z, d.z, t.m, d.m, stop, !greedy && !bad};
        }
    }
    if (greedy || bad) return;
    const L lt(a.target, t0 + stop, a.target_stride, a.vocab);
    const L ld(minus ? a.draft : a.target, minus ? (int64_t)q.b + stop : 0, minus ? a.draft_stride : 0, a.vocab);
    const bool alike = lt.shift == ld.shift;  // else the drafter's row is read element by element
    const int first = p * chunk - lt.shift + threadIdx.x * C, end = min((p + 1) * chunk - lt.shift, a.vocab);
    const double ip = 1.0 / t.z, iq = minus ? 1.0 / d.z : 0.0;
    double sum = 0.0, whole = 0.0;
#pragma unroll 1
    for (int e = first; e < end; e += 256 * C) {
        float x[C], y[C];
        lt.vec(e, true, x);
        if (minus) ld.vec(e, alike, y);
#pragma unroll
        for (int k = 0; k < C; ++k) {
            const double w = weight(x[k], t.m, c_t), above = minus ? dv_above(w, ip, weight(y[k], d.m, c_t), iq) : w * ip;
            whole += w * ip;
            sum += e + k == outright ? 0.0 : above;
        }
    }
    sum = dv_sum(sum), whole = dv_sum(whole);
    __shared__ DvMass s_mass[4];
    if (lane == 0) s_mass[wave] = {sum, whole};
    __syncthreads();
    if (threadIdx.x == 0)
        masses[(int64_t)s * M + p] = {(s_mass[0].sum + s_mass[1].sum) + (s_mass[2].sum + s_mass[3].sum),
                                      (s_mass[0].whole + s_mass[1].whole) + (s_mass[2].whole + s_mass[3].whole)};
}

// One workgroup a sequence: the chunk, then the token in it, a thread a run of elements.
constexpr int DV_DRAW = 1024;

// Starts that decrease: rows and sequences no longer follow from each other, a row may be
// several sequences', each at its own temperature. Then this workgroup does its sequence from
// its logits alone, whatever the launches before have left: the slow way, for what no batch
// that was laid out has. A sequence that shares drafts with another has no answer, so the
// others' rows are no more than a batch has.
template <typename T, typename F> __device__ __forceinline__ T dv_block(T v, T *s_wave, F f) {
    v = wave_all(v, 64, f);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s_wave[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s_wave[0];
    for (int w = 1; w < DV_DRAW / 64; ++w) v = f(v, s_wave[w]);
    return v;
}
template <int TY>
__device__ __forceinline__ DvRow dv_whole(const DvExp &weight, const void *logits, int64_t base, int V, bool greedy, double c_t, void *s_wave) {
    DvRow r = {0.0, -INFINITY, 0x7fffffff};
    for (int e = threadIdx.x; e < V; e += DV_DRAW) {
        const float x = dv_elem<TY>(logits, base + e);
        if (x > r.m) r.at = e;
        r.m = dv_top(r.m, x);
    }
    const float top = dv_block(r.m, (float *)s_wave, [](float u, float v) { return dv_top(u, v); });
    r.at = dv_block(r.m == top ? r.at : 0x7fffffff, (int *)s_wave, [](int u, int v) { return min(u, v); });
    r.m = top;
    if (!(top > -INFINITY) || (top == INFINITY && !greedy)) r.z = NAN;
    else if (!greedy) {
        for (int e = threadIdx.x; e < V; e += DV_DRAW) r.z += weight(dv_elem<TY>(logits, base + e), top, c_t);
        r.z = dv_block(r.z, (double *)s_wave, [](double u, double v) { return u + v; });
    }
    return r;
}
template <int TY>
__device__ __forceinline__ DvStop dv_alone(const tlh_draft_verify_args &a, int s, int M, int chunk, DvMass *s_mass) {
    constexpr int ES = TY == TLH_TYPE_F32 ? 4 : 2;
    __shared__ double s_wave[DV_DRAW / 64];
    const DvSeq q = dv_seq(a, s);
    const float T = a.temperatures[s];
    const bool greedy = !(T > 0.0f), drawn = a.draft && !greedy;
    const double c_t = DV_LOG2E / (double)T;
    const DvExp weight;
    int shares = 0;
    for (int o = threadIdx.x; o < a.num_seqs; o += DV_DRAW) {
        const DvSeq x = dv_seq(a, o);
        shares |= o != s && max(x.b, q.b) < min(x.b + x.n, q.b + q.n);
    }
    shares = __syncthreads_or(shares);
    auto target = [&](int i) { return dv_whole<TY>(weight, a.target, ((int64_t)q.b + s + i) * a.target_stride, a.vocab, greedy, c_t, s_wave); };
    int stop = shares ? 0 : q.n;
    DvRow t = {NAN, 0.0f, 0}, d = {0.0, 0.0f, 0};
    for (int i = 0; i < q.n; ++i) {
        DvTest test = {false, NAN};
        if (!shares) {
            const int x = a.tokens[q.b + i];
            const bool known = x >= 0 && x < a.vocab;
            const int64_t row = (int64_t)(q.b + i) * a.draft_stride;
            const DvRow ti = target(i), di = drawn ? dv_whole<TY>(weight, a.draft, row, a.vocab, false, c_t, s_wave) : DvRow{1.0, 0.0f, 0};
            const float tx = known ? dv_elem<TY>(a.target, ((int64_t)q.b + s + i) * a.target_stride + x) : -INFINITY;
            const float dx = known && drawn ? dv_elem<TY>(a.draft, row + x) : -INFINITY;
            test = dv_test(weight, ti, di, x, known, drawn, tx, dx, a.accept_at[q.b + i], greedy, c_t);
            if (!test.ok && stop == q.n) stop = i, t = ti, d = di;
        }
        if (threadIdx.x == 0 && a.accept_probs) a.accept_probs[q.b + i] = test.prob;
    }
    if (stop == q.n && !shares) t = target(q.n);
    const bool bad = t.z != t.z || d.z != d.z, minus = stop < q.n && drawn;
    int32_t *out = a.out_tokens + (int64_t)s * (a.max_drafts + 1);
    for (int i = threadIdx.x; i <= a.max_drafts; i += DV_DRAW) out[i] = i < stop ? a.tokens[q.b + i] : i == stop && greedy && !bad ? t.at : -1;
    if (threadIdx.x == 0) a.accepted[s] = stop;
    const DvStop st = {t.z, d.z, t.m, d.m, stop, !greedy && !bad};
    if (!st.draws) return st;
    // the chunks' sums, as k_draft_masses has them
    const int64_t row = ((int64_t)q.b + s + stop) * a.target_stride, drow = (int64_t)(q.b + stop) * a.draft_stride;
    const int shift = (int)(((uintptr_t)((const char *)a.target + row * ES) & 15) / ES);
    const int outright = stop < q.n && !a.draft ? a.tokens[q.b + stop] : -1;
    const double ip = 1.0 / t.z, iq = minus ? 1.0 / d.z : 0.0;
    for (int p = 0; p < M; ++p) {
        DvMass m = {0.0, 0.0};
        for (int e = max(p * chunk - shift, 0) + threadIdx.x; e < min((p + 1) * chunk - shift, a.vocab); e += DV_DRAW) {
            const double w = weight(dv_elem<TY>(a.target, row + e), t.m, c_t);
            const double above = minus ? dv_above(w, ip, weight(dv_elem<TY>(a.draft, drow + e), d.m, c_t), iq) : w * ip;
            m.whole += w * ip;
            m.sum += e == outright ? 0.0 : above;
        }
        auto add = [](double u, double v) { return u + v; };
        m.sum = dv_block(m.sum, s_wave, add), m.whole = dv_block(m.whole, s_wave, add);
        if (threadIdx.x == 0) s_mass[p] = m;
    }
    __syncthreads();
    return st;
}

template <int TY>
__device__ __forceinline__ void dv_draw(const tlh_draft_verify_args &a, int s, int M, int chunk, const DvStop &st, const DvMass *masses) {
    constexpr int ES = TY == TLH_TYPE_F32 ? 4 : 2;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (!st.draws) return;
    const DvSeq q = dv_seq(a, s);
    const double c_t = DV_LOG2E / (double)a.temperatures[s];
    const int64_t row = q.b + s + st.stop;
    bool minus = st.stop < q.n && a.draft;
    int outright = st.stop < q.n && !a.draft ? a.tokens[q.b + st.stop] : -1;
    const DvExp weight;
    DvMass m = {};
    if (lane < M) m = masses[lane];
    if (dv_sum(m.sum) <= DV_NOTHING) {  // nothing above the drafter's: from p alone
        minus = false;
        outright = -1;
        m.sum = m.whole;
    }
    double run = m.sum;
    for (int o = 1; o < 64; o <<= 1) {
        const double before = __shfl_up(run, o, 64);
        run += lane >= o ? before : 0.0;
    }
    const double total = __shfl(run, 63, 64);
    const double reach = (double)a.sample_at[s] * total;
    // Sums in another order may pass `reach` a rounding earlier, at a place without a weight:
    // it is no answer (but below 0 the first place is, whatever it weighs).
    const bool first_place = reach < 0.0;
    const uint64_t any = __builtin_amdgcn_ballot_w64(m.sum > 0.0);
    const uint64_t over = __builtin_amdgcn_ballot_w64(lane < M && run > reach && (m.sum > 0.0 || first_place));
    const int p = over != 0 ? __ffsll((unsigned long long)over) - 1 : 63 - __clzll((unsigned long long)any);  // else the last with a weight
    double from = __shfl(run - m.sum, p, 64);

    const char *base = (const char *)a.target + row * a.target_stride * ES;
    const int first = p * chunk - (int)(((uintptr_t)base & 15) / ES);
    const int each = chunk / DV_DRAW, e0 = max(first + (int)threadIdx.x * each, 0), e1 = min(first + ((int)threadIdx.x + 1) * each, a.vocab);
    const double ip = 1.0 / st.zp, iq = minus ? 1.0 / st.zq : 0.0;
    auto mass = [&](int e) {
        const double w = weight(dv_elem<TY>(base, e), st.mp, c_t);
        if (e == outright) return 0.0;
        if (!minus) return w * ip;
        return dv_above(w, ip, weight(dv_elem<TY>(a.draft, (int64_t)(q.b + st.stop) * a.draft_stride + e), st.mq, c_t), iq);
    };
    double sum = 0.0;
    int lead = 0x7fffffff, last = -1;  // the first and the last with a weight
    for (int e = e0; e < e1; ++e) {
        const double w = mass(e);
        sum += w;
        if (w > 0.0) lead = min(lead, e), last = e;
    }
    if (first_place && e0 < e1) lead = e0;
    __shared__ double s_sum[DV_DRAW / 64];
    __shared__ int s_last[DV_DRAW / 64], s_next;
    double upto = sum;
    for (int o = 1; o < 64; o <<= 1) {
        const double before = __shfl_up(upto, o, 64);
        upto += lane >= o ? before : 0.0;
    }
    const int wlast = -dv_min(-last);
    if (lane == 63) s_sum[wave] = upto;
    if (lane == 0) s_last[wave] = wlast;
    if (threadIdx.x == 0) s_next = 0x7fffffff;
    __syncthreads();
    last = -1;
    for (int w = 0; w < DV_DRAW / 64; ++w) {
        if (w < wave) from += s_sum[w];
        last = max(last, s_last[w]);
    }
    from += upto - sum;
    if (from > reach) atomicMin(&s_next, lead);
    else if (from + sum > reach) {
        for (int e = e0; e < e1; ++e) {
            from += mass(e);
            if (from > reach) {
                atomicMin(&s_next, e);
                break;
            }
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) a.out_tokens[(int64_t)s * (a.max_drafts + 1) + st.stop] = s_next == 0x7fffffff ? last : s_next;
}
template <int TY>
__global__ void __launch_bounds__(DV_DRAW) k_draft_draw(const tlh_draft_verify_args a, int M, int chunk, const int *__restrict__ odd,
                                                        const DvStop *__restrict__ stops, const DvMass *__restrict__ masses) {
    __shared__ DvMass s_alone[DV_MAX_CHUNKS];
    const int s = blockIdx.x;
    const bool alone = *odd != 0;
    DvStop st = stops[s];
    if (alone) st = dv_alone<TY>(a, s, M, chunk, s_alone);
    dv_draw<TY>(a, s, M, chunk, st, alone ? s_alone : masses + (int64_t)s * M);
}

// A small vocabulary's chunk of 64 a lane would be mostly empty; few rows: shorter chunks,
// so that more CUs share them.
static bool dv_small(int64_t vocab) { return vocab <= 2 * DV_CHUNK_SMALL; }
static int dv_ept(int64_t rows, int64_t vocab) {
    return dv_small(vocab) ||
                   (rows * ((vocab + DV_CHUNK - 1) / DV_CHUNK) < 256 && vocab + 7 <= (int64_t)DV_CHUNK_SMALL * DV_MAX_CHUNKS)
               ? 16
               : 64;
}
static int dv_chunks(int64_t vocab, int ept) {
    return (int)((vocab + 7 + 256 * ept - 1) / (256 * ept));  // up to 7 places before a row that is not aligned
}
// What is drawn from is one row a sequence: in short chunks wherever a lane each are enough,
// and shorter still where that makes four workgroups a CU at most, whose 5 us of reading the
// rows' parts go unseen. (Sums and draw with 8 and 16, us: 1 x 4 of 128256 13.6, 18.5; 48 of
// 32003 17.9, 18.8; 32 of 128256, 2016 workgroups with 8, 28.0, 26.7.)
constexpr int DV_SHORT_WGS = 1024;
static int dv_mass_ept(int64_t seqs, int64_t vocab) {
    if (vocab + 7 <= 8 * 256 * DV_MAX_CHUNKS && seqs * dv_chunks(vocab, 8) <= DV_SHORT_WGS) return 8;
    return vocab + 7 <= (int64_t)DV_CHUNK_SMALL * DV_MAX_CHUNKS ? 16 : 64;
}
static int64_t dv_rows(const tlh_draft_verify_args &a) { return (int64_t)a.num_drafts + a.num_seqs + (a.draft ? a.num_drafts : 0); }

// Room for any chunk length, so that the size grows with the rows and one buffer for
// the largest batch serves every smaller one: whether starts decrease, the sequences' stops,
// masses, the rows' parts.
constexpr size_t DV_ODD_BYTES = 16;
static size_t dv_most_chunks(int64_t rows, int64_t vocab) {
    return dv_small(vocab) ? (size_t)rows * dv_chunks(vocab, 16)
                           : (size_t)rows * dv_chunks(vocab, 64) + (size_t)std::min<int64_t>(rows, 256) * dv_chunks(vocab, 16);
}
size_t draft_verify_scratch_bytes(const tlh_draft_verify_args &a) {
    // of as many sequences as take short chunks, or of all in longer ones
    const int64_t longer = (int64_t)a.num_seqs * dv_chunks(a.vocab, dv_mass_ept(DV_SHORT_WGS + 1, a.vocab));
    const int64_t masses = std::max(longer, std::min<int64_t>((int64_t)a.num_seqs * dv_chunks(a.vocab, 8), DV_SHORT_WGS));
    return DV_ODD_BYTES + sizeof(DvStop) * (size_t)a.num_seqs + sizeof(DvMass) * (size_t)masses +
           sizeof(DvPart) * dv_most_chunks(dv_rows(a), a.vocab);
}

template <int TY> static void launch_dv(const tlh_draft_verify_args &a, void *scratch, hipStream_t stream) {
    const int64_t rows = dv_rows(a);
    const int ept = dv_ept(rows, a.vocab), chunk = 256 * ept, P = dv_chunks(a.vocab, ept);
    const int mass_ept = dv_mass_ept(a.num_seqs, a.vocab), M = dv_chunks(a.vocab, mass_ept), mass_chunk = 256 * mass_ept;
    int lanes = 1;
    while (lanes < P) lanes <<= 1;
    int *odd = (int *)scratch;
    DvStop *stops = (DvStop *)((uint8_t *)scratch + DV_ODD_BYTES);
    DvMass *masses = (DvMass *)(stops + a.num_seqs);
    DvPart *parts = (DvPart *)(masses + (size_t)a.num_seqs * M);
    for (int64_t r0 = 0; r0 <= rows; r0 += 65535)  // grid y
        hipLaunchKernelGGL((k_draft_rows<TY>), dim3(P, (unsigned)std::min<int64_t>(rows + 1 - r0, 65535)), dim3(256), 0, stream, a, (int)r0,
                           (int)rows, P, chunk, odd, parts);
    hipLaunchKernelGGL((k_draft_masses<TY>), dim3(M, a.num_seqs), dim3(256), 0, stream, a, P, M, mass_chunk, lanes, parts, stops, masses);
    hipLaunchKernelGGL((k_draft_draw<TY>), dim3(a.num_seqs), dim3(DV_DRAW), 0, stream, a, M, mass_chunk, odd, stops, masses);
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
