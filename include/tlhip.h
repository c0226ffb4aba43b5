/*
 * tlhip.h — C ABI of the MI355X (gfx950) executor for tensorlisp's quantized
 * hot path: GGML_OP_MUL_MAT over GGUF block-quantized weights (Q8_0, Q4_0,
 * Q4_K, Q5_K, Q6_K; decode GEMV for N <= 16 columns, MFMA GEMM for prefill),
 * paged-attention decode over an f16 block-table KV cache, dense
 * GGML_OP_FLASH_ATTN_EXT over f16 K/V, and what a server that mixes prompts,
 * single and drafted tokens needs beside them (packed prompts, pieces of prompts
 * over pages, drafted trees, heads' norms and rotation with the cache write,
 * page moves, log probabilities, verification of drafts).
 *
 * This is the surface a `native-hip` feature binds from Rust
 * (crates/kernels/src/hip/ + crates/tensorlisp/src/native_hip.rs), in place of
 * the NVRTC launcher of crates/kernels/src/cuda/{mod,exec,lower}.rs. Plain C:
 * pointers, sizes and PODs; no torch or HIP types in the signatures (a stream
 * is an opaque `void*` that is a hipStream_t, NULL = the null stream).
 *
 * Conventions (mirroring crates/kernels/src/lib.rs:44-61 and
 * crates/kernels/src/cuda/mod.rs):
 *  - every call returns a tlh_status; tlh_last_error() gives this thread's
 *    text for the last failure;
 *  - work calls are stream-ordered and asynchronous; nothing allocates behind
 *    the caller's back except where a function says so (tlh_alloc);
 *  - device pointers are plain device addresses on the current device.
 */
#ifndef TLHIP_H
#define TLHIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Error kinds of tensorlisp_kernels::Error (crates/kernels/src/lib.rs:44-61):
 * NoDevice, Unsupported{op,node,why}, Invalid, Alloc(bytes), Execution(msg). */
typedef enum tlh_status {
    TLH_OK = 0,
    TLH_NO_DEVICE = 1,
    TLH_UNSUPPORTED = 2,
    TLH_INVALID = 3,
    TLH_ALLOC = 4,
    TLH_EXECUTION = 5
} tlh_status;

/* ggml type numbers (vendor/ggml/include/ggml.h:390-417). */
enum {
    TLH_TYPE_F32 = 0,
    TLH_TYPE_F16 = 1,
    TLH_TYPE_Q4_0 = 2,
    TLH_TYPE_Q4_1 = 3,
    TLH_TYPE_Q5_0 = 6,
    TLH_TYPE_Q5_1 = 7,
    TLH_TYPE_Q8_0 = 8,
    TLH_TYPE_Q8_1 = 9,
    TLH_TYPE_Q2_K = 10,
    TLH_TYPE_Q3_K = 11,
    TLH_TYPE_Q4_K = 12,
    TLH_TYPE_Q5_K = 13,
    TLH_TYPE_Q6_K = 14,
    TLH_TYPE_Q8_K = 15,
    TLH_TYPE_I32 = 26,
    TLH_TYPE_I64 = 27,
    TLH_TYPE_BF16 = 30
};

/* Thread-local text of the last failure on this thread ("" if none). */
const char *tlh_last_error(void);
const char *tlh_status_name(tlh_status s);
/* Library version string, e.g. "tlhip 0.1 gfx950". */
const char *tlh_version(void);

/* ------------------------------------------------------------------ device
 * Replaces Device::system_default / name (crates/kernels/src/cuda/mod.rs:244-277):
 * TLH_NO_DEVICE when no GPU is present (not fatal at probe time). Opening
 * makes the device current on the calling thread. */
typedef struct tlh_device_props {
    char name[64];
    char arch[32];       /* e.g. "gfx950" */
    int compute_units;
    int wave_size;       /* 64 on CDNA */
    int lds_bytes;       /* per workgroup */
    int clock_khz;
    int64_t hbm_bytes;
} tlh_device_props;

tlh_status tlh_device_count(int *count);
tlh_status tlh_device_open(int ordinal, tlh_device_props *props);

/* ------------------------------------------------------------------ memory
 * Replaces Buffer (crates/kernels/src/cuda/mod.rs:39-133): alloc/free and
 * blocking copies, plus a stream-ordered sync (mod.rs:544-548). */
tlh_status tlh_alloc(size_t bytes, void **ptr);
tlh_status tlh_free(void *ptr);
tlh_status tlh_h2d(void *dst, const void *src, size_t bytes);
tlh_status tlh_d2h(void *dst, const void *src, size_t bytes);
tlh_status tlh_stream_sync(void *stream);

/* ---------------------------------------------------------- op descriptor
 * struct T / struct Op of crates/kernels/src/cuda/native/common.cuh:14-26, as
 * packed by OpBlob (crates/kernels/src/cuda/lower.rs:67-99): 5 tensors (slots
 * 0..3 sources, 4 the destination) of ggml ne/nb/type, then 12 scalar slots
 * (ints, or floats as their bit pattern). 456 bytes. */
typedef struct tlh_tensor {
    int64_t ne[4];
    int64_t nb[4];
    int32_t ty;
    int32_t pad_;
} tlh_tensor;

typedef struct tlh_op {
    tlh_tensor t[5];
    int64_t x[12];
} tlh_op;

/* --------------------------------------------------------------- MUL_MAT
 * GGML_OP_MUL_MAT, replacing Ctx::mul_mat (crates/kernels/src/cuda/lower.rs:543-571)
 * and its mm_vec / mm_tile kernels (crates/kernels/src/cuda/native/mm.cu:16-103),
 * computed the way the ggml CPU backend does (vendor/ggml/src/ggml-cpu/ggml-cpu.c:1254-1457):
 *   op->t[0] src0: weights, type Q4_0 | Q4_1 | Q5_0 | Q5_1 | Q8_0 | Q4_K | Q5_K | Q6_K |
 *                  F32 | F16 | BF16,
 *                  ne [K, M, ne02, ne03], nb[0] = block (element) bytes (rows must
 *                  not be transposed);
 *   op->t[1] src1: f32 activations (or, for F16 / BF16 weights, already of the
 *                  weight type), ne [K, N, ne12, ne13], nb[0] = element bytes;
 *   op->t[4] dst:  f32 [M, N, ne12, ne13], nb[0] = 4;
 *   op->x[0] = r2 = ne12 / ne02, op->x[1] = r3 = ne13 / ne03 (broadcast).
 * src1 is first quantized to the weight type's vec_dot type (Q8_0 for Q4_0, Q5_0
 * and Q8_0, Q8_1 for Q4_1 and Q5_1, Q8_K for Q4_K, Q5_K and Q6_K) into `scratch`
 * (at least tlh_mul_mat_scratch_bytes);
 * then N <= 16 runs the decode GEMV (register kernel for N <= 2, int8-MFMA
 * few-column kernel above), larger N the MFMA GEMM. Integer block
 * sums are exact; the f32 result agrees with the CPU backend to rounding of
 * the f32 accumulation order. F32 / F16 / BF16 weights follow the CPU's float
 * rows (ggml-cpu.c:215-226, :394-399): src1 rounded to the weight type, f32
 * products summed in f32, one launch (tlh_mul_mat_scratch_bytes still counts
 * the converted src1 rows, which only the split form below writes).
 * TLH_UNSUPPORTED (with the reason in tlh_last_error) for any
 * other type or layout. */
tlh_status tlh_mul_mat_scratch_bytes(const tlh_op *op, size_t *bytes);
tlh_status tlh_mul_mat(const tlh_op *op, const void *src0, const void *src1, void *dst, void *scratch,
                       size_t scratch_bytes, void *stream);

/* tlh_mul_mat with no caller scratch and no allocation, for callers that
 * cannot allocate device memory per call: code under HIP graph capture, tight
 * serving loops, harnesses that forbid hipMalloc. No counterpart in the
 * reference (its launcher allocates nothing per call but always passes
 * buffers it owns). Same kernels, descriptor and results as tlh_mul_mat; the
 * scratch is a static device array of TLH_NOALLOC_SCRATCH_BYTES that each GPU
 * holds for the life of the process, resolved on tlh_device_open (or on the
 * first call on a device). A node whose tlh_mul_mat_scratch_bytes exceeds it
 * is refused with TLH_INVALID (nothing is launched). The array keeps the last
 * call's contents and nothing in it has to start at zero; all calls on one GPU
 * share it, so calls that overlap in time on one GPU (other streams, other
 * threads) race: order them on one stream. Calls no hipMalloc/hipFree. */
#define TLH_NOALLOC_SCRATCH_BYTES ((size_t)64 << 20)
tlh_status tlh_mul_mat_noalloc(const tlh_op *op, const void *src0, const void *src1, void *dst, void *stream);

/* The two phases of tlh_mul_mat, which the CPU backend separates with a
 * barrier (ggml-cpu.c:1318-1359 quantize src1 into wdata; :1366 barrier;
 * :1426-1451 the dot products). Splitting them lets an executor quantize an
 * activation once for several weights that consume it (e.g. Q, K and V
 * projections of one input: same src1 shape and weight type, one scratch).
 * tlh_mul_mat_compute reads the scratch a matching tlh_mul_mat_quantize
 * filled (same op shape for src1, same vec_dot type). */
tlh_status tlh_mul_mat_quantize(const tlh_op *op, const void *src1, void *scratch, size_t scratch_bytes,
                                void *stream);
tlh_status tlh_mul_mat_compute(const tlh_op *op, const void *src0, const void *scratch, size_t scratch_bytes,
                               void *dst, void *stream);

/* GGML_OP_MUL_MAT_ID (vendor/ggml/src/ggml.c:3329-3353; CPU
 * ggml_compute_forward_mul_mat_id, ggml-cpu/ggml-cpu.c:1460-1640), which the
 * reference's native lowering has no kernel for (docs/design/kernel-launcher.md:326)
 * and runs on the CPU backend. Descriptor slots: t[0] = as, the expert
 * matrices [K, M, n_as] (q4_0 | q8_0 | q4_K | q5_K | q6_K); t[1] = b f32
 * [K, n_b1, n_tokens] with n_used % n_b1 == 0; t[2] = ids i32 [n_used, n_tokens];
 * t[4] = dst f32 [M, n_used, n_tokens]. dst[:, e, t] = as[:, :, ids[e, t]] times
 * b row (e % n_b1, t), each element the CPU's vec_dot of the quantized row
 * (so within the MUL_MAT tolerance of the CPU backend). An id outside
 * [0, n_as) yields NaN in its column (the CPU backend aborts there). With few
 * (expert, token) pairs each streams its expert's matrix once. With many and
 * k-quant weights they are sorted by expert on the device first, and an expert's
 * matrix is read once for a tile of its pairs; that takes the whole scratch of
 * tlh_mul_mat_id_scratch_bytes. A smaller one that holds the quantized rows (and
 * for K > 4096 their K-chunk sums) is taken too, with a matrix read a pair. */
tlh_status tlh_mul_mat_id_scratch_bytes(const tlh_op *op, size_t *bytes);
tlh_status tlh_mul_mat_id(const tlh_op *op, const void *src0, const void *src1, const void *ids, void *dst,
                          void *scratch, size_t scratch_bytes, void *stream);

/* Activation quantizer alone: `rows` rows of `k` f32 (row stride x_row_bytes)
 * into ggml's block layout of the vec_dot type of `wtype` — the from_float the
 * CPU mul_mat applies (quantize_row_q8_0 / quantize_row_q8_K:
 * vendor/ggml/src/ggml-cpu/arch/x86/quants.c:302-398, :505-507), bit-exact.
 * Output: rows * row_size(vec_dot_type, k) bytes, rows packed. A block whose
 * values are all zero gets d = 0, zero codes and zero bsums (the reference
 * leaves a zero Q8_K block's bsums unwritten). */
tlh_status tlh_quantize_act(int wtype, const float *x, int64_t k, int64_t rows, int64_t x_row_bytes, void *y,
                            void *stream);

/* dequantize_row_{q4_0,q8_0,q4_K,q5_K,q6_K} (vendor/ggml/src/ggml-quants.c:459-476,
 * :553-565, :1529-1550, :1731-1756, :1939-1968), bit-exact: `rows` rows of `k` elements (row stride
 * w_row_bytes) into f32 [rows][k]. The to_f32 of DType (crates/tensorlisp/src/dtype.rs:80-95). */
tlh_status tlh_dequantize(int type, const void *w, int64_t k, int64_t rows, int64_t w_row_bytes, float *y,
                          void *stream);

/* ------------------------------------------------------- FLASH_ATTN_EXT
 * GGML_OP_FLASH_ATTN_EXT, replacing Ctx::flash_attn_ext and its fa_main /
 * fa_split + fa_reduce kernels (crates/kernels/src/cuda/lower.rs:575-657,
 * split plan :764-792; crates/kernels/src/cuda/native/fa.cu:21-232), computed
 * as the ggml CPU backend does (vendor/ggml/src/ggml-cpu/ops.cpp:8468-8700):
 *   op->t[0] q:    f32 [D, nq, nh, nb], nb[0] = 4;
 *   op->t[1] k:    f16 [D, L, nhkv, nbk], nb[0] = 2, nh % nhkv == 0, nb % nbk == 0;
 *   op->t[2] v:    f16 [DV, L, nhkv, nbk], nb[0] = 2;
 *   op->t[3] mask: f16 [>= L, >= nq, mne2, mne3] (read only when `mask` is
 *                  non-NULL), broadcast over heads (nh % mne2 == 0) and batch;
 *   op->t[4] dst:  f32 [DV, nh, nq, nb], nb[0] = 4;
 *   op->x[0] scale (divided by softcap when softcap != 0), x[1] max_bias,
 *   x[2] m0, x[3] m1 (floats as their bit pattern, sign-extended), x[4]
 *   n_head_log2, x[5] softcap: the OpBlob lower.rs:615-620 packs.
 * K/V base pointers and strides must be 16-byte multiples; head sizes D = DV
 * in {32, 40, 64, 72, 80, 96, 112, 128, 192, 256} or D = 192, DV = 128. No
 * attention sinks (the reference lowering refuses them too). q is rounded to
 * f16 (as the CPU backend does for f16 keys); scores and the softmax are f32,
 * P.V accumulates in f32 (the CPU backend accumulates P.V in f16), so the
 * result agrees with the CPU backend to f16 rounding. Keys with a -inf mask are
 * skipped; a row with every key masked gives 0. `scratch` holds split-key
 * partials (tlh_flash_attn_ext_scratch_bytes; may be NULL when that is 0). */
tlh_status tlh_flash_attn_ext_scratch_bytes(const tlh_op *op, size_t *bytes);
tlh_status tlh_flash_attn_ext(const tlh_op *op, const void *q, const void *k, const void *v, const void *mask,
                              void *dst, void *scratch, size_t scratch_bytes, void *stream);

/* ------------------------------------------------------------ core ops
 * The ggml ops around MUL_MAT and attention in a decoder step (token
 * embedding, norms, residuals, activations, RoPE, KV-cache writes, softmax,
 * greedy sampling), replacing the reference's core kernels
 * (crates/kernels/src/cuda/native/core.cu) as Ctx::lower dispatches them
 * (crates/kernels/src/cuda/lower.rs:175-213, 219-500), computed as the ggml CPU
 * backend does (vendor/ggml/src/ggml-cpu/binary-ops.cpp, unary-ops.cpp,
 * ops.cpp). `op` is the blob the reference's lowering packs: t[0..2] sources,
 * t[4] the destination, x[] the op's parameters (floats as their bit
 * pattern). Data types f32 / f16; index tensors i32 / i64. Results are
 * bit-exact for BIN, CPY, GET_ROWS, SET_ROWS, ARGMAX and the unary ops
 * without a transcendental function; NORM sums in double like the CPU (equal
 * up to the order of the double additions); the others use the GPU's
 * expf/sinf/... (within a few ulp of the CPU's libm; GELU and GELU_QUICK go
 * through f16 like the CPU's tables). A SOFT_MAX row whose every entry is -inf
 * gives zeros (the CPU gives NaN).
 * tlh_core_check validates a node without launching (for planning);
 * tlh_core runs it. A GET_ROWS index outside src0 reads the nearest row and a
 * SET_ROWS index outside dst writes nothing (ggml asserts instead). */
typedef enum tlh_core_kind {
    TLH_CORE_BIN = 1,      /* ADD/SUB/MUL/DIV: x0 = 0/1/2/3; t0 op t1, t1 repeated to t0's shape */
    TLH_CORE_UNARY = 2,    /* UNARY (x0 = ggml_unary_op) and SCALE 100 (x1 s, x2 b), FILL 101 (x1),
                              CLAMP 102 (x1, x2), LEAKY_RELU 103 (x1), SQR 104, SQRT 105, SIN 106,
                              COS 107, LOG 108 (lower.rs:250-290) */
    TLH_CORE_NORM = 3,     /* NORM (x0 = 0) / RMS_NORM (x0 = 1), x1 = eps; f32 rows, unit element stride */
    TLH_CORE_GET_ROWS = 4, /* t0 f32/f16/q4_0/q8_0/q4_K/q5_K/q6_K rows, t1 indices -> t4 f32/f16 */
    TLH_CORE_SET_ROWS = 5, /* t0 f32/f16 rows to the t4 rows named by t1 */
    TLH_CORE_CPY = 6,      /* DUP/CPY/CONT: equal element counts, any shapes/strides */
    TLH_CORE_ROPE = 7,     /* x0 n_dims, x1 mode (0 normal, 2 neox), x2 freq_scale, x3 ext_factor,
                              x4 attn_factor, x5 freq_base^(-2/n_dims), x6/x7 YaRN corr dims,
                              x8 = 1 with f32 frequency factors in src2; t1 i32 positions */
    TLH_CORE_SOFT_MAX = 8, /* x0 scale, x1 max_bias, x2 m0, x3 m1, x4 n_head_log2; t0 f32; mask src1
                              f32/f16, optional (lower.rs:314-341) */
    TLH_CORE_ARGMAX = 9,   /* t0 f32 [n, rows] -> t4 i32 [rows] (last index of the maximum) */
    TLH_CORE_GLU = 10      /* GGML_OP_GLU, f32: x0 = ggml_glu_op (0 reglu, 1 geglu, 2 swiglu, 4 geglu_erf,
                              5 geglu_quick), x1 = swapped; t0 [2n, ...] halves, or t0 and t1 [n, ...]
                              (split form). No counterpart in the reference's lowering, which leaves
                              GLU unsupported; computed as ops.cpp ggml_compute_forward_glu does */
} tlh_core_kind;

tlh_status tlh_core_check(int kind, const tlh_op *op, int has_src1, int has_src2);
tlh_status tlh_core(int kind, const tlh_op *op, const void *src0, const void *src1, const void *src2, void *dst,
                    void *stream);

/* ------------------------------------------------------- paged attention
 * The `paged-attention` custom node (crates/tensorlisp/src/scheme/core.ss:251-258),
 * lowered by Ctx::custom kind 1 (crates/kernels/src/cuda/lower.rs:672-731) to
 * vLLM's paged_attention_v1/v2 (crates/kernels/src/cuda/paged_attn.rs:326-417).
 * Layouts (f16 elements, x = 8):
 *   q        [num_seqs][num_heads][head_size] (contiguous)
 *   k_cache  [num_blocks][num_kv_heads][head_size/8][block_size][8]
 *   v_cache  [num_blocks][num_kv_heads][head_size][block_size]
 *   block_tables i32 [num_seqs][max_blocks_per_seq], context_lens i32 [num_seqs]
 *   out      [num_seqs][num_heads][head_size]
 * head_size in {64, 80, 96, 112, 128, 192, 256}, block_size in {8, 16, 32},
 * num_heads % num_kv_heads == 0, context lens <= max_context_len.
 * `scratch` holds split-context partials (tlh_paged_attention_scratch_bytes,
 * which never shrinks as num_seqs or max_context_len grow, so one buffer sized
 * for the largest batch and context serves every smaller call); it may be
 * NULL when that size is 0. */
typedef struct tlh_paged_attention_args {
    void *out;
    const void *q;
    const void *k_cache;
    const void *v_cache;
    const int32_t *block_tables;
    const int32_t *context_lens;
    int32_t num_seqs;
    int32_t num_heads;
    int32_t num_kv_heads;
    int32_t head_size;
    int32_t block_size;
    int32_t max_blocks_per_seq;
    int32_t max_context_len;
    float scale;
} tlh_paged_attention_args;

tlh_status tlh_paged_attention_scratch_bytes(const tlh_paged_attention_args *a, size_t *bytes);
tlh_status tlh_paged_attention(const tlh_paged_attention_args *a, void *scratch, size_t scratch_bytes,
                               void *stream);

/* The `paged-cache-write` custom node (core.ss:265-272), Ctx::custom kind 2
 * (lower.rs:732-753) -> reshape_and_cache (crates/kernels/src/cuda/shaders/
 * reshape_and_cache_kernel.cu:31-84): key/value f16 [num_tokens][num_kv_heads*head_size]
 * into the caches at slot = block * block_size + offset; negative slots skip.
 * num_blocks is the pools' length in blocks (the caller's pool tensors give
 * it): a slot at or past num_blocks * block_size writes nothing, so a bad
 * slot cannot write outside the pools. */
tlh_status tlh_reshape_and_cache(const void *key, const void *value, void *k_cache, void *v_cache,
                                 const int64_t *slots, int32_t num_tokens, int32_t num_kv_heads, int32_t head_size,
                                 int32_t block_size, int64_t num_blocks, void *stream);

/* ------------------------------------------------------ packed attention
 * Causal attention of whole prompts packed one after another (a prefill of
 * several sequences in one call, with no mask tensor and no padding). No
 * counterpart in the reference, whose FLASH_ATTN_EXT takes a padded batch and a
 * mask. `type` is TLH_TYPE_F16 or TLH_TYPE_BF16, of all four tensors:
 *   q, out  [num_tokens][num_heads][head_size]
 *   k, v    [num_tokens][num_kv_heads][head_size]
 * a token's heads are contiguous, and q_stride, k_stride, v_stride and
 * out_stride are the elements from one token to the next (multiples of 8; views
 * of a fused QKV projection need no copy). Sequence s is the tokens
 * seq_starts[s] .. seq_starts[s + 1] - 1 (i32 [num_seqs + 1] on the device, not
 * decreasing; a sequence may be empty):
 *   out[t, h] = sum_j softmax_j(scale * q[t, h] . k[j, h / (num_heads / num_kv_heads)]) v[j, ..]
 * over the tokens j <= t of t's sequence. Scores, softmax and sums are f32; the
 * softmax's numerators are rounded to the type for the product with v (in f16
 * those below 2^-21 of the row's largest change by up to 2^-32 of it), the
 * result once. A token sees nothing of the ones it does not attend to, whatever
 * they hold (infinities and NaN too). Tokens behind the last sequence, and a
 * sequence's tokens from max_seq_len on, are left as they were; starts outside
 * [0, num_tokens] are taken as the nearer end. Pointers are 16-byte aligned;
 * no row of out may overlap one of q, k or v (other columns of the same rows
 * do not). head_size as for paged attention. */
typedef struct tlh_packed_attention_args {
    void *out;
    const void *q;
    const void *k;
    const void *v;
    const int32_t *seq_starts;
    int64_t out_stride;
    int64_t q_stride;
    int64_t k_stride;
    int64_t v_stride;
    int32_t type;
    int32_t num_seqs;
    int32_t num_tokens;
    int32_t max_seq_len;
    int32_t num_heads;
    int32_t num_kv_heads;
    int32_t head_size;
    float scale;
} tlh_packed_attention_args;

tlh_status tlh_packed_attention(const tlh_packed_attention_args *a, void *stream);

/* -------------------------------------------------------- tree attention
 * Attention of a tree of drafted tokens over the paged cache (the verification
 * step of speculative decoding; a chain of drafts is a tree too, and so is the
 * next few tokens of a prompt). No counterpart in the reference. Layouts and
 * geometry as for paged attention, the drafted tokens' keys and values already
 * written to the cache (tlh_reshape_and_cache) as the last of context_lens:
 *   q, out       f16 [num_rows][num_heads][head_size]
 *   draft_starts i32 [num_seqs + 1]: sequence s has the rows draft_starts[s] ..
 *                draft_starts[s + 1] - 1, n of them, at most max_drafts <= 64;
 *                rows behind the last sequence are left as they were
 *   draft_masks  i64 [num_rows]: bit j of a row's mask says that it sees its
 *                sequence's drafted token j (its ancestors and itself)
 * With L = context_lens[s], every row sees the tokens before L - n, and drafted
 * token j at place L - n + j where its mask says so. f32 scores, softmax and
 * sums, its numerators rounded to f16 for the product with v (those below 2^-21
 * of the row's largest change by up to 2^-32 of it); a row that sees
 * nothing gives zeros, and what a row does not see does not reach it, whatever
 * it holds. num_blocks is the pools' length in blocks: tokens of a page
 * outside it are not seen. Lengths are bounded by max_context_len (at most
 * 2^30), starts by num_rows. Of a sequence with more than max_drafts rows the
 * first max_drafts are computed, as if it had no others (n = max_drafts: their
 * drafted places are the context's last max_drafts), and the rest are left as
 * they were. out must not overlap the inputs. `scratch` holds the partials of a
 * split context (tlh_tree_attention_scratch_bytes, 16-byte aligned; it may be
 * NULL when that is 0); calls that share one must be stream-ordered. */
typedef struct tlh_tree_attention_args {
    void *out;
    const void *q;
    const void *k_cache;
    const void *v_cache;
    const int32_t *block_tables;
    const int32_t *context_lens;
    const int32_t *draft_starts;
    const int64_t *draft_masks;
    int64_t num_blocks;
    int32_t num_seqs;
    int32_t num_rows;
    int32_t max_drafts;
    int32_t num_heads;
    int32_t num_kv_heads;
    int32_t head_size;
    int32_t block_size;
    int32_t max_blocks_per_seq;
    int32_t max_context_len;
    float scale;
} tlh_tree_attention_args;

tlh_status tlh_tree_attention_scratch_bytes(const tlh_tree_attention_args *a, size_t *bytes);
tlh_status tlh_tree_attention(const tlh_tree_attention_args *a, void *scratch, size_t scratch_bytes, void *stream);

/* --------------------------------------------------------- cache moves
 * Copies of whole pages in every layer's pools in one launch (a fork's
 * copy-on-write, a defragmentation), as the reference's copy_blocks
 * (crates/kernels/src/cuda/paged_attn.rs:423-504) does a layer at a time.
 * `pools` is a host array of num_pools pool addresses (a layer's key pool and
 * its value pool count as two), each of num_blocks blocks of block_bytes bytes
 * (a multiple of 16; pools 16-byte aligned); pairs i64 [num_pairs][2] on the
 * device: block src to block dst in each pool. A block may be the source of
 * several pairs, but a destination must be neither another pair's destination
 * nor any pair's source: pairs run in no order. A pair with a block outside
 * [0, num_blocks) does nothing. */
tlh_status tlh_copy_blocks(void *const *pools, int32_t num_pools, int64_t block_bytes, int64_t num_blocks,
                           const int64_t *pairs, int32_t num_pairs, void *stream);

/* Closes the gaps that rejected drafted tokens leave in a paged cache, in every
 * layer in one launch (no counterpart in the reference). context_lens,
 * draft_starts and max_drafts as tlh_tree_attention took them; bit j of
 * keep[s] (i64 [num_seqs]) says that drafted token j of sequence s was
 * accepted. The kept tokens' keys and values move, in order, to the places from
 * L - n on, and new_lens[s] (i32, apart from what is read) becomes the length
 * with them. The drafted places must lie in pages that no other sequence of
 * the call shares. A move from or to a page outside [0, num_blocks) is left
 * out. k_caches and v_caches are host arrays of num_layers pool addresses in
 * the paged-attention layouts (f16). */
typedef struct tlh_compact_cache_args {
    void *const *k_caches;
    void *const *v_caches;
    const int32_t *block_tables;
    const int32_t *context_lens;
    const int32_t *draft_starts;
    const int64_t *keep;
    int32_t *new_lens;
    int64_t num_blocks;
    int32_t num_layers;
    int32_t num_seqs;
    int32_t max_drafts;
    int32_t num_kv_heads;
    int32_t head_size;
    int32_t block_size;
    int32_t max_blocks_per_seq;
} tlh_compact_cache_args;

tlh_status tlh_compact_cache(const tlh_compact_cache_args *a, void *stream);

/* ------------------------------------------------------- token logprobs
 * What a server answers and accepts by, from the logits of `rows` positions
 * (f32, f16 or bf16 [rows][vocab], row_stride elements from row to row, any
 * alignment of the type; vocab <= 1000000). No counterpart in the reference.
 *   logprobs[r]       log softmax(logits[r])[tokens[r]] (NaN for a token outside [0, vocab))
 *   entropy[r]        -sum p log p, natural logarithm
 *   top_ids[r][i], top_logprobs[r][i], i < top: the `top` largest logits from the
 *                     largest down, equal ones by the lowest index (top <= 32, <= vocab)
 * tokens and logprobs may be NULL together, entropy may be NULL, and the top
 * arrays where top is 0. Logits may be -inf (a grammar's mask): those tokens
 * have the log probability -inf. A row that is -inf throughout, or that holds
 * +inf or NaN, has NaN for what is not defined; a NaN ranks above every number.
 * `scratch` holds the rows' partial results (16-byte aligned); calls that share
 * one must be stream-ordered. */
typedef struct tlh_token_logprobs_args {
    const void *logits;
    const int32_t *tokens;
    float *logprobs;
    float *entropy;
    float *top_logprobs;
    int32_t *top_ids;
    int64_t row_stride;
    int32_t type;
    int32_t rows;
    int32_t vocab;
    int32_t top;
} tlh_token_logprobs_args;

tlh_status tlh_token_logprobs_scratch_bytes(const tlh_token_logprobs_args *a, size_t *bytes);
tlh_status tlh_token_logprobs(const tlh_token_logprobs_args *a, void *scratch, size_t scratch_bytes, void *stream);

/* ------------------------------------------------------- chunk attention
 * Causal attention of the sequences' new tokens over the paged cache: one token
 * of a sequence that decodes, or any number of a prompt that comes in pieces or
 * follows a cached prefix, mixed in one call. No counterpart in the reference.
 * Layouts and geometry as for paged attention, the new tokens' keys and values
 * already written to the cache as the last of context_lens:
 *   q, out       f16 [num_rows][num_heads][head_size], a token's heads contiguous,
 *                q_stride and out_stride elements from token to token (multiples of 8)
 *   row_starts   i32 [num_seqs + 1]: sequence s has the rows row_starts[s] ..
 *                row_starts[s + 1] - 1, n of them, at most max_rows (starts do not
 *                decrease, or nothing is computed); rows behind the last sequence
 *                are left as they were
 * With L = context_lens[s], row i of the sequence is the token at place L - n + i and
 * sees the tokens up to itself, with window > 0 the last `window` of them. f32 scores,
 * softmax and sums; for the product with v its numerators keep 22 bits (those below 2^-10 of
 * the row's largest change by up to 2^-32 of it). With f16_weights 1 (else 0) they are rounded
 * to f16 (those below 2^-21 alike) where a sequence has more than 64 rows of q a kv head, which
 * saves one of three products there. A row that sees nothing (a
 * place below 0, pages that are not there) gives zeros, and what a row does not see does
 * not reach it, whatever it holds. num_blocks is the pools' length in blocks: tokens
 * of a page outside it are not seen. Lengths are bounded by max_context_len (at most
 * 2^30), starts by num_rows. Of a sequence with more than max_rows rows the first
 * max_rows are computed, as if it had no others, and the rest are left as they were.
 * No row of out may overlap a row of q (other columns of the same rows do not), and out not
 * the caches, tables, lengths or starts; nothing may overlap the scratch. `scratch` holds the
 * partials of split contexts and the plan of many sequences (tlh_chunk_attention_scratch_bytes,
 * which never shrinks as a count grows, 16-byte aligned; it may be NULL when that is
 * 0). Its first TLH_CHUNK_COUNTER_BYTES must be zero before its first call, and every call
 * leaves them zero; calls that share one must be stream-ordered. */
#define TLH_CHUNK_COUNTER_BYTES ((size_t)8192)
typedef struct tlh_chunk_attention_args {
    void *out;
    const void *q;
    const void *k_cache;
    const void *v_cache;
    const int32_t *block_tables;
    const int32_t *context_lens;
    const int32_t *row_starts;
    int64_t out_stride;
    int64_t q_stride;
    int64_t num_blocks;
    int32_t num_seqs;
    int32_t num_rows;
    int32_t max_rows;
    int32_t num_heads;
    int32_t num_kv_heads;
    int32_t head_size;
    int32_t block_size;
    int32_t max_blocks_per_seq;
    int32_t max_context_len;
    int32_t window;
    float scale;
    int32_t f16_weights;
} tlh_chunk_attention_args;

tlh_status tlh_chunk_attention_scratch_bytes(const tlh_chunk_attention_args *a, size_t *bytes);
tlh_status tlh_chunk_attention(const tlh_chunk_attention_args *a, void *scratch, size_t scratch_bytes, void *stream);

/* ------------------------------------------------------------- head rope
 * What lies between the Q, K, V projections and attention, in one pass: the norms
 * of the query and key heads, their rotation by the tokens' positions, and the
 * write of keys and values to the paged cache. No counterpart in the reference,
 * which runs RMS_NORM, ROPE and the cache write as nodes of their own.
 *   q      [num_tokens][num_heads][head_size], k, v [num_tokens][num_kv_heads][head_size],
 *          of `type` (f32, f16 or bf16), a token's heads contiguous, *_stride elements
 *          from token to token
 *   q_norm, k_norm  f32 [head_size] or NULL: a head x becomes
 *          x / sqrt(mean(x^2) + eps) * norm
 *   then its first n_dims dims are rotated in pairs (mode 0: 2p and 2p + 1, mode 2:
 *          p and p + n_dims / 2, as TLH_CORE_ROPE): pair p by the angle
 *          positions[pair_axis[p]][token] * freqs[p], cos and sin times attn_factor;
 *          positions i32 [num_axes][num_tokens] (1 axis: text; 2 to 4: images, video),
 *          freqs f32 [n_dims / 2]; n_dims 0 rotates nothing. The angle is formed and
 *          reduced in 64 bits, so far positions keep their fraction.
 *   q_out  out_type (f16 or bf16) [num_tokens][num_heads][head_size]; k_out and v_out
 *          alike, each may be NULL: rounded once from f32
 *   k_cache, v_cache, slots: all NULL, or (out_type f16) the pools of
 *          tlh_reshape_and_cache and each token's slot there, num_blocks blocks long; a
 *          negative slot or one past the pools writes nothing; slots must differ
 * head_size as for paged attention; tensors 16-byte aligned, strides multiples of 16
 * bytes. No output may overlap an input or another output (columns of the same
 * rows that differ do not). */
typedef struct tlh_head_rope_args {
    const void *q;
    const void *k;
    const void *v;
    const int32_t *positions;
    const float *freqs;
    const float *q_norm;
    const float *k_norm;
    void *q_out;
    void *k_out;
    void *v_out;
    void *k_cache;
    void *v_cache;
    const int64_t *slots;
    int64_t q_stride;
    int64_t k_stride;
    int64_t v_stride;
    int64_t q_out_stride;
    int64_t k_out_stride;
    int64_t v_out_stride;
    int64_t num_blocks;
    int32_t type;
    int32_t out_type;
    int32_t num_tokens;
    int32_t num_heads;
    int32_t num_kv_heads;
    int32_t head_size;
    int32_t block_size;
    int32_t n_dims;
    int32_t mode;
    int32_t num_axes;
    float eps;
    float attn_factor;
    uint8_t pair_axis[128];
} tlh_head_rope_args;

tlh_status tlh_head_rope(const tlh_head_rope_args *a, void *stream);

/* ---------------------------------------------------------- draft verify
 * Verification of drafted tokens against the model's probabilities from given random
 * numbers, so that what is answered is distributed as the model alone would have it
 * (a chain of drafts a sequence). No counterpart in the reference.
 *   target  logits (f32, f16 or bf16) [num_drafts + num_seqs][vocab]: sequence s with
 *           the drafted tokens b = draft_starts[s] .. draft_starts[s + 1] - 1, n of
 *           them, at most max_drafts, has the rows b + s .. b + s + n: row b + s + i is
 *           what the model says at the place of its draft i, the last one behind them
 *   draft   logits of the drafting model, same type [num_drafts][vocab], or NULL where
 *           tokens were proposed outright (copied from the prompt): q is then 1 at them
 *   p, q    softmax(logits / temperatures[s]); a temperature that is not above 0 is
 *           greedy: p is 1 at the largest logit, the lowest index among equal ones,
 *           that token alone is accepted, and the drafter's logits are not looked at
 * Draft i with token x is accepted if accept_at[b + i] * q(x) < p(x) and those before it
 * are; accept_probs[b + i] = min(1, p(x) / q(x)) (NULL: not wanted; p(x) > 0 where q(x)
 * is 0). accepted[s] counts them. The next token is drawn from what p has above q at the first one
 * refused (from p where that is nothing: less than 2^-40), or from the row behind the drafts: the
 * lowest index where the running sum exceeds sample_at[s] times the whole (the last with
 * a weight above 0 where none does). out_tokens[s], i32 [max_drafts + 1], receives the
 * accepted ones, this one, and -1 behind them. All of it is computed in 64 bits: a running sum over
 * a vocabulary decides between neighbours that f32 cannot tell apart.
 * Logits may be -inf (a mask). A row with a NaN, with +inf at a temperature above 0, or
 * with nothing but -inf is no distribution: a draft that needs it is refused (accept
 * probability NaN), and a token that would be drawn from it is -1. A token outside
 * [0, vocab) has p = q = 0. A sequence that ends before it starts has no drafts; one that
 * shares drafts with another (starts that decrease) is not verified: accepted 0, tokens -1, accept
 * probabilities NaN. Starts are bounded by num_drafts. Of a sequence with more than max_drafts drafts the first max_drafts are
 * looked at, as if it had no others. Row strides in elements, any alignment of the type;
 * vocab <= 1000000, max_drafts <= 1024. `scratch` (16-byte aligned) holds the rows'
 * sums; calls that share one must be stream-ordered. The outputs must not overlap the
 * inputs or each other, and nothing the scratch. */
typedef struct tlh_draft_verify_args {
    const void *target;
    const void *draft;
    const int32_t *tokens;
    const int32_t *draft_starts;
    const float *temperatures;
    const float *accept_at;
    const float *sample_at;
    int32_t *accepted;
    int32_t *out_tokens;
    float *accept_probs;
    int64_t target_stride;
    int64_t draft_stride;
    int32_t type;
    int32_t num_seqs;
    int32_t num_drafts;
    int32_t max_drafts;
    int32_t vocab;
} tlh_draft_verify_args;

tlh_status tlh_draft_verify_scratch_bytes(const tlh_draft_verify_args *a, size_t *bytes);
tlh_status tlh_draft_verify(const tlh_draft_verify_args *a, void *scratch, size_t scratch_bytes, void *stream);

/* ------------------------------------------------------------ executor
 * A graph of ggml nodes compiled once into a recorded list of launches on this
 * library's kernels and replayed per run, replacing the reference's
 * Executor::compile / Program::run (crates/kernels/src/cuda/exec.rs:27-226)
 * over its IR (crates/kernels/src/graph.rs:72-229) and memory plan
 * (crates/kernels/src/plan.rs:56-189). The caller hands over the IR the
 * reference builds from a ggml graph (native_ir.rs lower_graph): one record
 * per tensor, the node order and the tensors that must outlive the run.
 *
 * Memory: weights stay where the caller put them (a device pointer per weight
 * index); state tensors live in one caller buffer at fixed byte offsets (per
 * state index), handed over per run so sessions can swap blocks; inputs live
 * in an io buffer and temporaries in an arena, both owned by the program. The
 * arena reuses a tensor's bytes once its last reader has run (first fit by
 * start position, 256-byte alignment), and holds each node's scratch.
 * MUL_MAT nodes that read the same activation with the same weight type
 * quantize it once: the first one writes the q8 blocks into a scratch block
 * that lives until the last of them has run (when the activation has more
 * than two columns; at one or two the GEMV quantizes on the fly, which saves
 * a launch).
 *
 * Lowering follows the reference's Ctx::lower (lower.rs:175-213): view ops
 * and empty tensors produce nothing; MUL_MAT, FLASH_ATTN_EXT and the core ops
 * go to the entry points above with the blobs Ctx packs. Every node is lowered
 * before failing, and one TLH_UNSUPPORTED names each missing op with a count
 * and an example, as exec.rs:39-58 reports them.
 *
 * Runs: tlh_program_run enqueues the launches on `stream`; with `graph` != 0
 * the launches are captured once into a hipGraph (per state buffer and stream)
 * and replayed with one hipGraphLaunch. Calls on one program must not overlap. */
typedef enum tlh_storage {
    TLH_STORE_TEMP = 0,   /* computed in the arena */
    TLH_STORE_WEIGHT = 1, /* weights[storage_index] */
    TLH_STORE_STATE = 2,  /* state buffer + state_offsets[storage_index] */
    TLH_STORE_INPUT = 3   /* input storage_index, in the program's io buffer */
} tlh_storage;

typedef struct tlh_ir_tensor {
    char op[24];            /* ggml op name ("MUL_MAT", "RMS_NORM", ...; "NONE" for leaves) */
    int32_t ty;             /* ggml type */
    int32_t storage;        /* tlh_storage; meaningful for roots */
    int32_t storage_index;
    int32_t view_src;       /* -1, or the root tensor whose storage this view aliases */
    int64_t view_offs;      /* byte offset into view_src */
    int64_t ne[4];
    int64_t nb[4];
    int32_t op_params[16];  /* as ggml stores them */
    int32_t src[10];        /* tensor ids, -1 = none */
} tlh_ir_tensor;

typedef struct tlh_program tlh_program;

/* Plans and lowers; allocates the arena and io buffer on the current device.
 * weights: n_weights device pointers; state_offsets: byte offset of each state
 * tensor in the state buffer given to tlh_program_run. */
tlh_status tlh_program_compile(const tlh_ir_tensor *tensors, int32_t n_tensors, const int32_t *nodes,
                               int32_t n_nodes, const int32_t *keep, int32_t n_keep, const void *const *weights,
                               int32_t n_weights, const int64_t *state_offsets, int32_t n_states,
                               tlh_program **program);
tlh_status tlh_program_destroy(tlh_program *p);
/* Stream-ordered copy between any two device (or pinned host) addresses. */
tlh_status tlh_copy(void *dst, const void *src, size_t bytes, void *stream);
/* Stream-ordered fill of `bytes` device bytes at dst with the low 8 bits of
   `value`, by a kernel (so it may be captured in a hipGraph). Replaces the
   CUDA backend's cuMemsetD8Async zero fill (Backend::zero,
   crates/kernels/src/cuda/backend.rs:334-343). */
tlh_status tlh_memset(void *dst, int value, size_t bytes, void *stream);
/* No counterpart in the reference: a plain streaming read of `bytes` bytes
   (16-byte aligned; `grid` workgroups of 256 lanes, `loads` = 1 or 4 16-byte
   loads in flight per lane) that writes nothing. For measurement only: the
   floor a kernel that must read the same bytes cannot beat, timed beside the
   GEMVs by bench.py. */
tlh_status tlh_read_floor(const void *src, size_t bytes, int32_t grid, int32_t loads, void *stream);
/* Device address and byte size of graph input i in the io buffer. */
tlh_status tlh_program_input(const tlh_program *p, int32_t i, void **ptr, size_t *bytes);
/* Device address of tensor `id` (any storage; `state` is the run's state buffer). */
tlh_status tlh_program_tensor(const tlh_program *p, int32_t id, void *state, void **ptr);
tlh_status tlh_program_run(tlh_program *p, void *state, void *stream, int32_t graph);
/* Sizes: arena bytes, io bytes, and the number of recorded dispatches (one
 * per lowered node, plus one quantization per MUL_MAT group; a dispatch may
 * launch more than one kernel). */
tlh_status tlh_program_stats(const tlh_program *p, size_t *arena_bytes, size_t *io_bytes, int32_t *launches);
/* Per-dispatch timing, in place of the reference's TL_NATIVE_PROFILE per-op
 * times (crates/kernels/src/cuda/exec.rs:186-216): one eager run of the program
 * on `stream` with an event after every dispatch; ms[i] = GPU milliseconds of
 * dispatch i (n >= the dispatch count of tlh_program_stats). Synchronous.
 * With the environment variable TLH_NATIVE_PROFILE set, every eager
 * tlh_program_run does the same and prints the ops with the most time to
 * stderr, as the reference does. */
tlh_status tlh_program_profile(tlh_program *p, void *state, void *stream, float *ms, int32_t n);
/* One eager run of the program on `stream` that records which kernels each
 * dispatch launched (no counterpart in the reference; its exec.rs labels
 * dispatches only by op). `text` receives one line per dispatch:
 * "<index>\t<ggml op of its first node>\t<launch labels, comma-separated>\n"
 * (labels as the launch sites name them: "gemv", "gemv_mfma", "gemv_cols",
 * "gemm_q4k", "gemm_q8", "flash_attn_ext", "flash_attn_ext (rows)",
 * "paged_attention", "norm_chain", ...), NUL-terminated and truncated to `cap`
 * bytes; *len (optional) = the bytes the whole text needs. Not synchronous. */
tlh_status tlh_program_trace(tlh_program *p, void *state, void *stream, char *text, size_t cap, size_t *len);
/* The plan without a device (for checking it): arena offset per tensor (-1 if
 * not in the arena), per-node scratch offset (-1 if none) and the arena size.
 * Scratch sizes come from the same entry points compile uses. */
tlh_status tlh_program_plan(const tlh_ir_tensor *tensors, int32_t n_tensors, const int32_t *nodes, int32_t n_nodes,
                            const int32_t *keep, int32_t n_keep, int64_t *tensor_offsets, int64_t *scratch_offsets,
                            size_t *arena_bytes);

/* ------------------------------------------------------------------ GGUF
 * Reading a GGUF model and loading its tensors into device memory, in place
 * of the reference's load for its native executors
 * (crates/tensorlisp/src/native_cuda.rs:44-82, reading through ggml's
 * gguf.cpp as crates/tensorlisp/src/gguf.rs:79-320 does). The file is checked
 * with ggml's rules (versions 2-3; general.alignment a u32 power of two,
 * default 32; tensor names under 64 bytes, unique; at most 4 dimensions; rows
 * of whole blocks; tensor offsets consecutive at the alignment); a refusal is
 * TLH_INVALID (TLH_UNSUPPORTED for a ggml type this loader cannot size) with
 * the reason. Key-value pairs keep their GGUF types (gguf_type numbering);
 * numeric values and arrays come back as their raw little-endian bytes.
 * tlh_gguf_layout places every tensor 256-byte aligned in one buffer of
 * `total` bytes; tlh_gguf_upload copies the file's tensor data there through
 * pinned staging buffers (a synchronous call on `stream`). */
typedef struct tlh_gguf tlh_gguf;
typedef struct tlh_gguf_tensor_info {
    char name[64];
    int32_t ty;      /* ggml type */
    int32_t n_dims;
    int64_t ne[4];
    uint64_t offset; /* in the data section */
    uint64_t bytes;
} tlh_gguf_tensor_info;

tlh_status tlh_gguf_open(const char *path, tlh_gguf **g);
tlh_status tlh_gguf_close(tlh_gguf *g);
tlh_status tlh_gguf_counts(const tlh_gguf *g, uint32_t *version, int64_t *n_tensors, int64_t *n_kv,
                           uint64_t *alignment, uint64_t *data_offset);
tlh_status tlh_gguf_tensor(const tlh_gguf *g, int64_t i, tlh_gguf_tensor_info *info);
tlh_status tlh_gguf_find_tensor(const tlh_gguf *g, const char *name, int64_t *i); /* -1 when absent */
tlh_status tlh_gguf_find_key(const tlh_gguf *g, const char *key, int64_t *i);     /* -1 when absent */
/* type: gguf_type of the value; for arrays (9) also the element type and count */
tlh_status tlh_gguf_key(const tlh_gguf *g, int64_t i, const char **key, int32_t *type, int32_t *arr_type,
                        uint64_t *n);
tlh_status tlh_gguf_value(const tlh_gguf *g, int64_t i, const void **data, size_t *bytes); /* numeric / bool */
tlh_status tlh_gguf_string(const tlh_gguf *g, int64_t i, uint64_t j, const char **s, uint64_t *len);
tlh_status tlh_gguf_layout(const tlh_gguf *g, uint64_t *offsets, uint64_t *total);
tlh_status tlh_gguf_upload(const tlh_gguf *g, void *dev, const uint64_t *offsets, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* TLHIP_H */
