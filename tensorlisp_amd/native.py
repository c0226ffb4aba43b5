"""Python binding of the gfx950 executor's C ABI (``include/tlhip.h``).

This mirrors, for tests and the benchmark, what a ``native-hip`` Rust binding
would do: build the 456-byte op descriptor of a ggml node (the ``struct Op``
of crates/kernels/src/cuda/native/common.cuh:14-26, packed like OpBlob in
crates/kernels/src/cuda/lower.rs:67-99) and call the library on a stream.
PyTorch only supplies device memory and the current stream.

The library must be built (``python -m tensorlisp_amd.build``); importing this
module without it raises, there is no fallback path.
"""
from __future__ import annotations

import ctypes as C
from pathlib import Path

PKG = Path(__file__).resolve().parent
LIB_PATH = PKG / "libtlhip.so"

# ggml type numbers (vendor/ggml/include/ggml.h:390-405)
F32, F16, Q4_0, Q8_0, Q4_K, Q5_K, Q6_K, Q8_K, BF16 = 0, 1, 2, 8, 12, 13, 14, 15, 30
Q4_1, Q5_0, Q5_1, Q8_1 = 3, 6, 7, 9
Q2_K, Q3_K = 10, 11
BLOCK = {Q4_0: (32, 18), Q8_0: (32, 34), Q4_K: (256, 144), Q5_K: (256, 176), Q6_K: (256, 210), Q8_K: (256, 292),
         Q4_1: (32, 20), Q5_0: (32, 22), Q5_1: (32, 24), Q8_1: (32, 36), F32: (1, 4), F16: (1, 2), BF16: (1, 2),
         Q2_K: (256, 84), Q3_K: (256, 110)}
# ggml's vec_dot_type: what src1 is converted to (float weights: their own type)
VEC_DOT_TYPE = {Q4_0: Q8_0, Q8_0: Q8_0, Q4_K: Q8_K, Q5_K: Q8_K, Q6_K: Q8_K, Q4_1: Q8_1, Q5_0: Q8_0, Q5_1: Q8_1,
                F32: F32, F16: F16, BF16: BF16, Q2_K: Q8_K, Q3_K: Q8_K}
TYPE_NAMES = {F32: "f32", F16: "f16", Q4_0: "q4_0", Q8_0: "q8_0", Q4_K: "q4_K", Q5_K: "q5_K", Q6_K: "q6_K", Q8_K: "q8_K",
              BF16: "bf16", Q4_1: "q4_1", Q5_0: "q5_0", Q5_1: "q5_1", Q8_1: "q8_1", Q2_K: "q2_K", Q3_K: "q3_K"}
TYPES_BY_NAME = {v: k for k, v in TYPE_NAMES.items()}

STATUS = {0: "OK", 1: "NO_DEVICE", 2: "UNSUPPORTED", 3: "INVALID", 4: "ALLOC", 5: "EXECUTION"}

# Every symbol include/tlhip.h declares.
EXPORTS = (
    "tlh_last_error", "tlh_status_name", "tlh_version", "tlh_device_count", "tlh_device_open", "tlh_alloc",
    "tlh_free", "tlh_h2d", "tlh_d2h", "tlh_stream_sync", "tlh_mul_mat_scratch_bytes", "tlh_mul_mat",
    "tlh_mul_mat_noalloc", "tlh_mul_mat_quantize", "tlh_mul_mat_compute", "tlh_mul_mat_id_scratch_bytes", "tlh_mul_mat_id",
    "tlh_quantize_act", "tlh_dequantize", "tlh_flash_attn_ext_scratch_bytes", "tlh_flash_attn_ext",
    "tlh_paged_attention_scratch_bytes", "tlh_paged_attention", "tlh_reshape_and_cache",
    "tlh_packed_attention", "tlh_tree_attention_scratch_bytes", "tlh_tree_attention", "tlh_copy_blocks",
    "tlh_compact_cache", "tlh_token_logprobs_scratch_bytes", "tlh_token_logprobs",
    "tlh_chunk_attention_scratch_bytes", "tlh_chunk_attention", "tlh_head_rope", "tlh_draft_verify_scratch_bytes",
    "tlh_draft_verify",
    "tlh_core_check", "tlh_core", "tlh_program_compile", "tlh_program_destroy", "tlh_copy", "tlh_memset",
    "tlh_read_floor",
    "tlh_program_input",
    "tlh_program_tensor", "tlh_program_run", "tlh_program_stats", "tlh_program_profile", "tlh_program_trace",
    "tlh_program_plan",
    "tlh_gguf_open", "tlh_gguf_close", "tlh_gguf_counts", "tlh_gguf_tensor", "tlh_gguf_find_tensor",
    "tlh_gguf_find_key", "tlh_gguf_key", "tlh_gguf_value", "tlh_gguf_string", "tlh_gguf_layout", "tlh_gguf_upload",
)


class TlhError(RuntimeError):
    """A failed call: .status is the tlh_status name (mirrors tensorlisp_kernels::Error)."""

    def __init__(self, status: int, msg: str):
        self.status = STATUS.get(status, str(status))
        super().__init__(f"{self.status}: {msg}")


class TlhTensor(C.Structure):
    _fields_ = [("ne", C.c_int64 * 4), ("nb", C.c_int64 * 4), ("ty", C.c_int32), ("pad_", C.c_int32)]


class TlhOp(C.Structure):
    _fields_ = [("t", TlhTensor * 5), ("x", C.c_int64 * 12)]


class TlhDeviceProps(C.Structure):
    _fields_ = [("name", C.c_char * 64), ("arch", C.c_char * 32), ("compute_units", C.c_int),
                ("wave_size", C.c_int), ("lds_bytes", C.c_int), ("clock_khz", C.c_int), ("hbm_bytes", C.c_int64)]


class TlhPagedArgs(C.Structure):
    _fields_ = [("out", C.c_void_p), ("q", C.c_void_p), ("k_cache", C.c_void_p), ("v_cache", C.c_void_p),
                ("block_tables", C.c_void_p), ("context_lens", C.c_void_p), ("num_seqs", C.c_int32),
                ("num_heads", C.c_int32), ("num_kv_heads", C.c_int32), ("head_size", C.c_int32),
                ("block_size", C.c_int32), ("max_blocks_per_seq", C.c_int32), ("max_context_len", C.c_int32),
                ("scale", C.c_float)]


class TlhPackedArgs(C.Structure):
    _fields_ = [("out", C.c_void_p), ("q", C.c_void_p), ("k", C.c_void_p), ("v", C.c_void_p),
                ("seq_starts", C.c_void_p), ("out_stride", C.c_int64), ("q_stride", C.c_int64),
                ("k_stride", C.c_int64), ("v_stride", C.c_int64), ("type", C.c_int32), ("num_seqs", C.c_int32),
                ("num_tokens", C.c_int32), ("max_seq_len", C.c_int32), ("num_heads", C.c_int32),
                ("num_kv_heads", C.c_int32), ("head_size", C.c_int32), ("scale", C.c_float)]


class TlhTreeArgs(C.Structure):
    _fields_ = [("out", C.c_void_p), ("q", C.c_void_p), ("k_cache", C.c_void_p), ("v_cache", C.c_void_p),
                ("block_tables", C.c_void_p), ("context_lens", C.c_void_p), ("draft_starts", C.c_void_p),
                ("draft_masks", C.c_void_p), ("num_blocks", C.c_int64), ("num_seqs", C.c_int32),
                ("num_rows", C.c_int32), ("max_drafts", C.c_int32), ("num_heads", C.c_int32),
                ("num_kv_heads", C.c_int32), ("head_size", C.c_int32), ("block_size", C.c_int32),
                ("max_blocks_per_seq", C.c_int32), ("max_context_len", C.c_int32), ("scale", C.c_float)]


class TlhCompactArgs(C.Structure):
    _fields_ = [("k_caches", C.POINTER(C.c_void_p)), ("v_caches", C.POINTER(C.c_void_p)),
                ("block_tables", C.c_void_p), ("context_lens", C.c_void_p), ("draft_starts", C.c_void_p),
                ("keep", C.c_void_p), ("new_lens", C.c_void_p), ("num_blocks", C.c_int64), ("num_layers", C.c_int32),
                ("num_seqs", C.c_int32), ("max_drafts", C.c_int32), ("num_kv_heads", C.c_int32),
                ("head_size", C.c_int32), ("block_size", C.c_int32), ("max_blocks_per_seq", C.c_int32)]


class TlhLogprobsArgs(C.Structure):
    _fields_ = [("logits", C.c_void_p), ("tokens", C.c_void_p), ("logprobs", C.c_void_p), ("entropy", C.c_void_p),
                ("top_logprobs", C.c_void_p), ("top_ids", C.c_void_p), ("row_stride", C.c_int64), ("type", C.c_int32),
                ("rows", C.c_int32), ("vocab", C.c_int32), ("top", C.c_int32)]


class TlhChunkArgs(C.Structure):
    _fields_ = [("out", C.c_void_p), ("q", C.c_void_p), ("k_cache", C.c_void_p), ("v_cache", C.c_void_p),
                ("block_tables", C.c_void_p), ("context_lens", C.c_void_p), ("row_starts", C.c_void_p),
                ("out_stride", C.c_int64), ("q_stride", C.c_int64), ("num_blocks", C.c_int64), ("num_seqs", C.c_int32),
                ("num_rows", C.c_int32), ("max_rows", C.c_int32), ("num_heads", C.c_int32), ("num_kv_heads", C.c_int32),
                ("head_size", C.c_int32), ("block_size", C.c_int32), ("max_blocks_per_seq", C.c_int32),
                ("max_context_len", C.c_int32), ("window", C.c_int32), ("scale", C.c_float), ("f16_weights", C.c_int32)]


class TlhHeadRopeArgs(C.Structure):
    _fields_ = [(f, C.c_void_p) for f in ("q", "k", "v", "positions", "freqs", "q_norm", "k_norm", "q_out", "k_out", "v_out",
                                          "k_cache", "v_cache", "slots")] + \
               [(f, C.c_int64) for f in ("q_stride", "k_stride", "v_stride", "q_out_stride", "k_out_stride", "v_out_stride",
                                         "num_blocks")] + \
               [(f, C.c_int32) for f in ("type", "out_type", "num_tokens", "num_heads", "num_kv_heads", "head_size",
                                         "block_size", "n_dims", "mode", "num_axes")] + \
               [("eps", C.c_float), ("attn_factor", C.c_float), ("pair_axis", C.c_uint8 * 128)]


class TlhVerifyArgs(C.Structure):
    _fields_ = [(f, C.c_void_p) for f in ("target", "draft", "tokens", "draft_starts", "temperatures", "accept_at",
                                          "sample_at", "accepted", "out_tokens", "accept_probs")] + \
               [("target_stride", C.c_int64), ("draft_stride", C.c_int64)] + \
               [(f, C.c_int32) for f in ("type", "num_seqs", "num_drafts", "max_drafts", "vocab")]


assert C.sizeof(TlhOp) == 456, C.sizeof(TlhOp)


def load_library(path: Path = LIB_PATH) -> C.CDLL:
    if not path.exists():
        raise ImportError(f"{path} is missing: build it with `python -m tensorlisp_amd.build` (no fallback exists)")
    L = C.CDLL(str(path))
    vp, i64, st = C.c_void_p, C.c_int64, C.c_int
    L.tlh_last_error.restype = C.c_char_p
    L.tlh_status_name.restype = C.c_char_p
    L.tlh_status_name.argtypes = [C.c_int]
    L.tlh_version.restype = C.c_char_p
    L.tlh_device_count.argtypes = [C.POINTER(C.c_int)]
    L.tlh_device_open.argtypes = [C.c_int, C.POINTER(TlhDeviceProps)]
    L.tlh_alloc.argtypes = [C.c_size_t, C.POINTER(C.c_void_p)]
    L.tlh_free.argtypes = [vp]
    L.tlh_h2d.argtypes = [vp, vp, C.c_size_t]
    L.tlh_d2h.argtypes = [vp, vp, C.c_size_t]
    L.tlh_stream_sync.argtypes = [vp]
    L.tlh_mul_mat_scratch_bytes.argtypes = [C.POINTER(TlhOp), C.POINTER(C.c_size_t)]
    L.tlh_mul_mat.argtypes = [C.POINTER(TlhOp), vp, vp, vp, vp, C.c_size_t, vp]
    L.tlh_mul_mat_noalloc.argtypes = [C.POINTER(TlhOp), vp, vp, vp, vp]
    L.tlh_mul_mat_quantize.argtypes = [C.POINTER(TlhOp), vp, vp, C.c_size_t, vp]
    L.tlh_mul_mat_compute.argtypes = [C.POINTER(TlhOp), vp, vp, C.c_size_t, vp, vp]
    L.tlh_mul_mat_id_scratch_bytes.argtypes = [C.POINTER(TlhOp), C.POINTER(C.c_size_t)]
    L.tlh_mul_mat_id.argtypes = [C.POINTER(TlhOp), vp, vp, vp, vp, vp, C.c_size_t, vp]
    L.tlh_quantize_act.argtypes = [C.c_int, vp, i64, i64, i64, vp, vp]
    L.tlh_dequantize.argtypes = [C.c_int, vp, i64, i64, i64, vp, vp]
    L.tlh_flash_attn_ext_scratch_bytes.argtypes = [C.POINTER(TlhOp), C.POINTER(C.c_size_t)]
    L.tlh_flash_attn_ext.argtypes = [C.POINTER(TlhOp), vp, vp, vp, vp, vp, vp, C.c_size_t, vp]
    L.tlh_paged_attention_scratch_bytes.argtypes = [C.POINTER(TlhPagedArgs), C.POINTER(C.c_size_t)]
    L.tlh_paged_attention.argtypes = [C.POINTER(TlhPagedArgs), vp, C.c_size_t, vp]
    L.tlh_reshape_and_cache.argtypes = [vp, vp, vp, vp, vp, C.c_int32, C.c_int32, C.c_int32, C.c_int32, C.c_int64, vp]
    L.tlh_packed_attention.argtypes = [C.POINTER(TlhPackedArgs), vp]
    L.tlh_tree_attention_scratch_bytes.argtypes = [C.POINTER(TlhTreeArgs), C.POINTER(C.c_size_t)]
    L.tlh_tree_attention.argtypes = [C.POINTER(TlhTreeArgs), vp, C.c_size_t, vp]
    L.tlh_copy_blocks.argtypes = [C.POINTER(C.c_void_p), C.c_int32, i64, i64, vp, C.c_int32, vp]
    L.tlh_compact_cache.argtypes = [C.POINTER(TlhCompactArgs), vp]
    L.tlh_token_logprobs_scratch_bytes.argtypes = [C.POINTER(TlhLogprobsArgs), C.POINTER(C.c_size_t)]
    L.tlh_token_logprobs.argtypes = [C.POINTER(TlhLogprobsArgs), vp, C.c_size_t, vp]
    L.tlh_chunk_attention_scratch_bytes.argtypes = [C.POINTER(TlhChunkArgs), C.POINTER(C.c_size_t)]
    L.tlh_chunk_attention.argtypes = [C.POINTER(TlhChunkArgs), vp, C.c_size_t, vp]
    L.tlh_head_rope.argtypes = [C.POINTER(TlhHeadRopeArgs), vp]
    L.tlh_draft_verify_scratch_bytes.argtypes = [C.POINTER(TlhVerifyArgs), C.POINTER(C.c_size_t)]
    L.tlh_draft_verify.argtypes = [C.POINTER(TlhVerifyArgs), vp, C.c_size_t, vp]
    L.tlh_core_check.argtypes = [C.c_int, C.POINTER(TlhOp), C.c_int, C.c_int]
    L.tlh_core.argtypes = [C.c_int, C.POINTER(TlhOp), vp, vp, vp, vp, vp]
    i32p, i64p = C.POINTER(C.c_int32), C.POINTER(C.c_int64)
    L.tlh_program_compile.argtypes = [vp, C.c_int32, i32p, C.c_int32, i32p, C.c_int32, C.POINTER(C.c_void_p),
                                      C.c_int32, i64p, C.c_int32, C.POINTER(C.c_void_p)]
    L.tlh_program_destroy.argtypes = [vp]
    L.tlh_copy.argtypes = [vp, vp, C.c_size_t, vp]
    L.tlh_memset.argtypes = [vp, C.c_int, C.c_size_t, vp]
    L.tlh_read_floor.argtypes = [vp, C.c_size_t, C.c_int32, C.c_int32, vp]
    L.tlh_program_input.argtypes = [vp, C.c_int32, C.POINTER(C.c_void_p), C.POINTER(C.c_size_t)]
    L.tlh_program_tensor.argtypes = [vp, C.c_int32, vp, C.POINTER(C.c_void_p)]
    L.tlh_program_run.argtypes = [vp, vp, vp, C.c_int32]
    L.tlh_program_stats.argtypes = [vp, C.POINTER(C.c_size_t), C.POINTER(C.c_size_t), C.POINTER(C.c_int32)]
    L.tlh_program_profile.argtypes = [vp, vp, vp, C.POINTER(C.c_float), C.c_int32]
    L.tlh_program_trace.argtypes = [vp, vp, vp, C.c_char_p, C.c_size_t, C.POINTER(C.c_size_t)]
    L.tlh_program_plan.argtypes = [vp, C.c_int32, i32p, C.c_int32, i32p, C.c_int32, i64p, i64p,
                                   C.POINTER(C.c_size_t)]
    u64p, cpp = C.POINTER(C.c_uint64), C.POINTER(C.c_char_p)
    L.tlh_gguf_open.argtypes = [C.c_char_p, C.POINTER(C.c_void_p)]
    L.tlh_gguf_close.argtypes = [vp]
    L.tlh_gguf_counts.argtypes = [vp, C.POINTER(C.c_uint32), i64p, i64p, u64p, u64p]
    L.tlh_gguf_tensor.argtypes = [vp, C.c_int64, vp]
    L.tlh_gguf_find_tensor.argtypes = [vp, C.c_char_p, i64p]
    L.tlh_gguf_find_key.argtypes = [vp, C.c_char_p, i64p]
    L.tlh_gguf_key.argtypes = [vp, C.c_int64, cpp, C.POINTER(C.c_int32), C.POINTER(C.c_int32), u64p]
    L.tlh_gguf_value.argtypes = [vp, C.c_int64, C.POINTER(C.c_void_p), C.POINTER(C.c_size_t)]
    L.tlh_gguf_string.argtypes = [vp, C.c_int64, C.c_uint64, cpp, u64p]
    L.tlh_gguf_layout.argtypes = [vp, u64p, u64p]
    L.tlh_gguf_upload.argtypes = [vp, vp, u64p, vp]
    for name in EXPORTS:
        if name not in ("tlh_last_error", "tlh_status_name", "tlh_version"):
            getattr(L, name).restype = st
    return L


_lib = None


def lib() -> C.CDLL:
    global _lib
    if _lib is None:
        _lib = load_library()
    return _lib


def check(status: int) -> None:
    if status != 0:
        raise TlhError(status, lib().tlh_last_error().decode())


def row_bytes(t: int, k: int) -> int:
    be, bb = BLOCK[t]
    if k % be:
        raise ValueError(f"k={k} is not a multiple of the {TYPE_NAMES[t]} block ({be})")
    return k // be * bb


def ggml_tensor(ty: int, ne, nb=None) -> TlhTensor:
    """A ggml-style tensor descriptor; nb defaults to the contiguous strides of `ty`."""
    ne = list(ne) + [1] * (4 - len(ne))
    t = TlhTensor()
    if nb is None:
        if ty in BLOCK:
            be, bb = BLOCK[ty]
            nb0, nb1 = bb, ne[0] // be * bb
        else:
            nb0 = {F32: 4, F16: 2, 26: 4, 27: 8}[ty]  # f32, f16, i32, i64
            nb1 = nb0 * ne[0]
        nb = [nb0, nb1, nb1 * ne[1], nb1 * ne[1] * ne[2]]
    for i in range(4):
        t.ne[i] = int(ne[i])
        t.nb[i] = int(nb[i])
    t.ty = int(ty)
    return t


def mul_mat_op(wtype: int, M: int, K: int, N: int, ne2: int = 1, ne3: int = 1, w_ne2: int = 1,
               w_ne3: int = 1, x_nb=None, w_nb=None, d_nb=None, xtype: int = F32) -> TlhOp:
    """The MUL_MAT descriptor of Ctx::mul_mat (lower.rs:543-571): t0 weights [K, M], t1 [K, N] (f32, or the
    f16 / bf16 of f16 / bf16 weights), t4 f32 [M, N]."""
    op = TlhOp()
    op.t[0] = ggml_tensor(wtype, [K, M, w_ne2, w_ne3], w_nb)
    op.t[1] = ggml_tensor(xtype, [K, N, ne2, ne3], x_nb)
    op.t[4] = ggml_tensor(F32, [M, N, ne2, ne3], d_nb)
    op.x[0] = ne2 // w_ne2
    op.x[1] = ne3 // w_ne3
    return op


def _stream(stream):
    import torch

    if stream is None:
        return C.c_void_p(torch.cuda.current_stream().cuda_stream)
    return C.c_void_p(getattr(stream, "cuda_stream", stream))


def _ptr(t) -> C.c_void_p:
    return C.c_void_p(t.data_ptr())


def device_props(ordinal: int = 0) -> dict:
    p = TlhDeviceProps()
    check(lib().tlh_device_open(ordinal, C.byref(p)))
    return {"name": p.name.decode(), "arch": p.arch.decode(), "compute_units": p.compute_units,
            "wave_size": p.wave_size, "lds_bytes": p.lds_bytes, "clock_khz": p.clock_khz, "hbm_bytes": p.hbm_bytes}


def device_count() -> int:
    n = C.c_int()
    check(lib().tlh_device_count(C.byref(n)))
    return n.value


def mul_mat_scratch_bytes(op: TlhOp) -> int:
    n = C.c_size_t()
    check(lib().tlh_mul_mat_scratch_bytes(C.byref(op), C.byref(n)))
    return n.value


class MulMat:
    """One GGML_OP_MUL_MAT node with its scratch, launched many times (what a lowered
    Dispatch is in crates/kernels/src/cuda/exec.rs:186-225)."""

    def __init__(self, wtype: int, M: int, K: int, N: int, device="cuda", op: TlhOp = None):
        import torch

        self.wtype, self.M, self.K, self.N = wtype, M, K, N
        self.op = mul_mat_op(wtype, M, K, N) if op is None else op
        self.scratch_bytes = mul_mat_scratch_bytes(self.op)
        self.scratch = torch.empty(max(self.scratch_bytes, 256) + 256, dtype=torch.uint8, device=device)
        off = (-self.scratch.data_ptr()) % 256
        self.scratch_ptr = C.c_void_p(self.scratch.data_ptr() + off)

    def __call__(self, w, x, y, stream=None):
        check(lib().tlh_mul_mat(C.byref(self.op), _ptr(w), _ptr(x), _ptr(y), self.scratch_ptr,
                                self.scratch_bytes, _stream(stream)))
        return y

    def quantize(self, x, stream=None):
        """Phase 1 only: x -> the node's scratch."""
        check(lib().tlh_mul_mat_quantize(C.byref(self.op), _ptr(x), self.scratch_ptr, self.scratch_bytes,
                                         _stream(stream)))

    def compute(self, w, y, stream=None):
        """Phase 2 only: the products from the scratch the last quantize() filled."""
        check(lib().tlh_mul_mat_compute(C.byref(self.op), _ptr(w), self.scratch_ptr, self.scratch_bytes, _ptr(y),
                                        _stream(stream)))
        return y


def mul_mat(wtype: int, w, M: int, K: int, x, stream=None):
    """y [N, M] f32 = x [N, K] @ dequant(W [M rows of K])^T, computed as ggml's CPU mul_mat does."""
    import torch

    x = x.contiguous()
    N = x.shape[0]
    y = torch.empty((N, M), dtype=torch.float32, device=x.device)
    MulMat(wtype, M, K, N, device=x.device)(w, x, y, stream)
    return y


def mul_mat_views(w, x, out=None, stream=None, split: bool = False):
    """ggml_mul_mat on torch views of float weights: w (w3, w2, M, K) f32 / f16 /
    bf16, x (n3, n2, N, K) f32 or w's dtype, out (n3, n2, N, M) f32 (ggml's ne
    reversed; fewer leading dims are 1). Any element-aligned strides with K
    contiguous; w's batch dims broadcast over x's (r2 = n2 / w2, r3 = n3 / w3).
    split: src1's conversion and the products as two launches
    (tlh_mul_mat_quantize + tlh_mul_mat_compute) instead of one."""
    import torch

    wt, xt = _ggml_type(w), _ggml_type(x)
    lead = lambda t: [1] * (4 - t.dim()) + list(t.shape[:-2])  # noqa: E731
    n3, n2 = lead(x)[-2:]
    if out is None:
        out = torch.empty((n3, n2, x.shape[-2], w.shape[-2]), dtype=torch.float32, device=x.device)
    op = TlhOp()
    op.t[0], op.t[1], op.t[4] = tensor_desc(w, wt), tensor_desc(x, xt), tensor_desc(out, F32)
    w3, w2 = lead(w)[-2:]
    op.x[0], op.x[1] = n2 // max(w2, 1), n3 // max(w3, 1)
    mm = MulMat(wt, w.shape[-2], w.shape[-1], x.shape[-2], device=x.device, op=op)
    if split:
        mm.quantize(x, stream)
        mm.compute(w, out, stream)
    else:
        mm(w, x, out, stream)
    return out


def quantize_act(wtype: int, x, stream=None):
    """x [rows, k] f32 -> uint8 [rows, row_bytes(vec_dot_type, k)] in ggml's block layout."""
    import torch

    rows, k = x.shape
    assert x.dtype == torch.float32 and x.stride(1) == 1
    out = torch.empty((rows, row_bytes(VEC_DOT_TYPE[wtype], k)), dtype=torch.uint8, device=x.device)
    check(lib().tlh_quantize_act(wtype, _ptr(x), k, rows, x.stride(0) * 4, _ptr(out), _stream(stream)))
    return out


def memset(t, value: int, nbytes: int = None, offset: int = 0, stream=None) -> None:
    """Fill `nbytes` bytes of device tensor t (from byte `offset`; all of it by
    default) with the low 8 bits of value, on `stream` (tlh_memset)."""
    n = t.numel() * t.element_size() - offset if nbytes is None else nbytes
    check(lib().tlh_memset(C.c_void_p(t.data_ptr() + offset), int(value), n, _stream(stream)))


def dequantize(wtype: int, w, k: int, stream=None):
    """uint8 [rows, row_bytes] -> f32 [rows, k]."""
    import torch

    rows = w.shape[0]
    y = torch.empty((rows, k), dtype=torch.float32, device=w.device)
    check(lib().tlh_dequantize(wtype, _ptr(w), k, rows, w.stride(0), _ptr(y), _stream(stream)))
    return y


def _f32_bits(x: float) -> int:
    """A float op parameter as OpBlob::float stores it (lower.rs:96-98): the f32
    bit pattern, sign-extended to 64 bits."""
    import struct

    return struct.unpack("<i", struct.pack("<f", x))[0]


def flash_attn_params(n_head: int, scale: float, max_bias: float = 0.0, softcap: float = 0.0):
    """(scale, max_bias, m0, m1, n_head_log2, softcap) as Ctx::flash_attn_ext derives
    them (lower.rs:604-620), in f32 arithmetic."""
    import numpy as np

    f = np.float32
    scale, max_bias, softcap = f(scale), f(max_bias), f(softcap)
    if softcap != 0:
        scale = f(scale / softcap)
    nhl2 = 1 << int(np.floor(np.log2(f(n_head))))
    m0 = f(np.power(f(2.0), f(-max_bias / f(nhl2))))
    m1 = f(np.power(f(2.0), f(-(max_bias / f(2.0)) / f(nhl2))))
    return float(scale), float(max_bias), float(m0), float(m1), nhl2, float(softcap)


def _ggml_type(t) -> int:
    import torch

    return {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}.get(t.dtype, -1)


def tensor_desc(t, ty: int) -> TlhTensor:
    """The ggml descriptor of a torch tensor whose shape is ggml's ne reversed
    (torch (n3, n2, n1, n0) <-> ggml [n0, n1, n2, n3]); strides follow the view."""
    shape = list(t.shape)[::-1] + [1] * (4 - t.dim())
    if t.numel() == 0:  # an empty view's strides are arbitrary: use ggml's contiguous ones
        strides = [t.element_size()]
        for i in range(1, 4):
            strides.append(strides[-1] * max(shape[i - 1], 1))
        return ggml_tensor(ty, shape, strides)
    strides = [s * t.element_size() for s in list(t.stride())[::-1]]
    for i in range(t.dim(), 4):
        strides.append(strides[-1] * shape[i - 1] if strides else t.element_size())
    return ggml_tensor(ty, shape, strides)


def flash_attn_op(q, k, v, mask, dst, scale: float, max_bias: float = 0.0, softcap: float = 0.0) -> TlhOp:
    """The FLASH_ATTN_EXT descriptor Ctx::flash_attn_ext packs (lower.rs:611-621):
    t0 q, t1 k, t2 v, t3 mask (zeros when absent), t4 dst; x0..x5 the parameters."""
    op = TlhOp()
    op.t[0] = tensor_desc(q, _ggml_type(q))
    op.t[1] = tensor_desc(k, _ggml_type(k))
    op.t[2] = tensor_desc(v, _ggml_type(v))
    if mask is not None:
        op.t[3] = tensor_desc(mask, _ggml_type(mask))
    op.t[4] = tensor_desc(dst, _ggml_type(dst))
    sc, mb, m0, m1, nhl2, cap = flash_attn_params(int(op.t[0].ne[2]), scale, max_bias, softcap)
    op.x[0], op.x[1], op.x[2], op.x[3] = _f32_bits(sc), _f32_bits(mb), _f32_bits(m0), _f32_bits(m1)
    op.x[4] = nhl2
    op.x[5] = _f32_bits(cap)
    return op


def flash_attn_scratch_bytes(op: TlhOp) -> int:
    n = C.c_size_t()
    check(lib().tlh_flash_attn_ext_scratch_bytes(C.byref(op), C.byref(n)))
    return n.value


class FlashAttnExt:
    """One GGML_OP_FLASH_ATTN_EXT node with its split-key scratch. Tensors are torch
    views whose shapes are ggml's ne reversed: q f32 (nb, nh, nq, D), k f16
    (nbk, nhkv, L, D), v f16 (nbk, nhkv, L, DV), mask f16 (mne3, mne2, >= nq, >= L)
    or None, dst f32 (nb, nq, nh, DV)."""

    def __init__(self, q, k, v, mask, dst, scale: float, max_bias: float = 0.0, softcap: float = 0.0):
        import torch

        self.op = flash_attn_op(q, k, v, mask, dst, scale, max_bias, softcap)
        self.scratch_bytes = flash_attn_scratch_bytes(self.op)
        self.scratch = torch.empty(max(self.scratch_bytes, 4), dtype=torch.uint8, device=q.device)

    def __call__(self, q, k, v, mask, dst, stream=None):
        check(lib().tlh_flash_attn_ext(C.byref(self.op), _ptr(q), _ptr(k), _ptr(v),
                                       _ptr(mask) if mask is not None else None, _ptr(dst), _ptr(self.scratch),
                                       self.scratch_bytes, _stream(stream)))
        return dst


def flash_attn_ext(q, k, v, mask=None, scale: float = 1.0, max_bias: float = 0.0, softcap: float = 0.0,
                   stream=None):
    """ggml_flash_attn_ext(q, k, v, mask, scale, max_bias, softcap) on torch views
    (shapes as in FlashAttnExt) -> dst f32 (nb, nq, nh, DV), ggml [DV, nh, nq, nb]."""
    import torch

    nb, nh, nq, _ = q.shape
    dst = torch.empty((nb, nq, nh, v.shape[-1]), dtype=torch.float32, device=q.device)
    return FlashAttnExt(q, k, v, mask, dst, scale, max_bias, softcap)(q, k, v, mask, dst, stream)


class PagedAttention:
    """The `paged-attention` node (crates/tensorlisp/src/scheme/core.ss:251-258) with its scratch."""

    def __init__(self, num_seqs, num_heads, num_kv_heads, head_size, block_size, max_blocks_per_seq,
                 max_context_len, scale, device="cuda"):
        import torch

        self.args = TlhPagedArgs()
        a = self.args
        a.num_seqs, a.num_heads, a.num_kv_heads = num_seqs, num_heads, num_kv_heads
        a.head_size, a.block_size = head_size, block_size
        a.max_blocks_per_seq, a.max_context_len, a.scale = max_blocks_per_seq, max_context_len, scale
        n = C.c_size_t()
        check(lib().tlh_paged_attention_scratch_bytes(C.byref(a), C.byref(n)))
        self.scratch_bytes = n.value
        self.scratch = torch.empty(max(n.value, 4), dtype=torch.uint8, device=device)

    def __call__(self, out, q, k_cache, v_cache, block_tables, context_lens, stream=None):
        a = self.args
        a.out, a.q, a.k_cache, a.v_cache = out.data_ptr(), q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
        a.block_tables, a.context_lens = block_tables.data_ptr(), context_lens.data_ptr()
        check(lib().tlh_paged_attention(C.byref(a), _ptr(self.scratch), self.scratch_bytes, _stream(stream)))
        return out


def paged_attention(q, k_cache, v_cache, block_tables, context_lens, block_size, max_context_len, scale,
                    num_kv_heads, stream=None):
    """q f16 [seqs, heads, hs] -> out f16 [seqs, heads, hs] (vLLM cache layouts)."""
    import torch

    seqs, heads, hs = q.shape
    out = torch.empty_like(q)
    pa = PagedAttention(seqs, heads, num_kv_heads, hs, block_size, block_tables.shape[1], max_context_len, scale,
                        device=q.device)
    return pa(out, q.contiguous(), k_cache, v_cache, block_tables.contiguous(), context_lens.contiguous(), stream)


def reshape_and_cache(key, value, k_cache, v_cache, slots, num_kv_heads, block_size, stream=None):
    """key/value f16 [tokens, kv_heads*hs] scattered into the caches; slots i64 [tokens] (negative = skip;
    at or past the pools' end = dropped)."""
    tokens = key.shape[0]
    hs = key.shape[1] // num_kv_heads
    num_blocks = min(k_cache.numel(), v_cache.numel()) // (num_kv_heads * hs * block_size)
    check(lib().tlh_reshape_and_cache(_ptr(key), _ptr(value), _ptr(k_cache), _ptr(v_cache), _ptr(slots), tokens,
                                      num_kv_heads, hs, block_size, num_blocks, _stream(stream)))


# --------------------------------------------------------- serving operators
def _tensor(t, dtype, shape, name: str, device):
    """The address of a contiguous tensor of this dtype and shape on `device`."""
    if t.dtype != dtype or t.shape != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name}: {t.dtype} {tuple(t.shape)} on {t.device}, not contiguous {dtype} {shape} on {device}")
    return t.data_ptr()


def _extent(t) -> int:
    """The first extent of a tensor that may have any."""
    return t.shape[0] if t.dim() else 0


def _int32(value, name: str) -> int:
    """A count as the calls take it: ctypes would cut a larger one to 32 bits without a word."""
    if not -(1 << 31) <= value < 1 << 31:
        raise ValueError(f"{name} {value} does not fit 32 bits")
    return value


def _current(device) -> int:
    """current_stream's number, without the 2.7 us its Stream object takes."""
    import torch

    return torch._C._cuda_getCurrentRawStream(device.index)


class _on:
    """Runs a call on the tensors' device, on `stream` or that device's current stream: that stream's number."""

    def __init__(self, device, stream):
        self.device, self.stream, self.guard = device, stream, None

    def __enter__(self):
        import torch

        if self.device.type != "cuda":
            raise ValueError(f"tensors must be on the GPU, not on {self.device}")
        if self.stream is not None and getattr(self.stream, "device", self.device) != self.device:
            raise ValueError(f"the stream is on {self.stream.device}, the tensors are on {self.device}")
        if self.device.index != torch.cuda.current_device():
            self.guard = torch.cuda.device(self.device)
            self.guard.__enter__()
        if self.stream is None:
            return _current(self.device)
        return int(getattr(self.stream, "cuda_stream", self.stream))

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _torch_stream(stream, device):
    """A stream as the calls take it (torch's, or a hipStream_t) as torch's."""
    import torch

    if isinstance(stream, torch.cuda.Stream):
        return stream
    if not stream:  # the default stream's number, which ExternalStream takes for none and makes a new stream
        return torch.cuda.default_stream(device)
    return torch.cuda.ExternalStream(stream, device=device)


def _behind_current(stream, device):
    """A call's own tensors come from the current stream's pool, where queued work may still use the memory they were
    given: the call's `stream` waits for that work. -> the stream as torch's, None for the current one."""
    import torch

    if stream is None:
        return None
    side, current = _torch_stream(stream, device), torch.cuda.current_stream(device)
    if side != current:
        side.wait_stream(current)
    return side


def _use_on(stream, *tensors):
    """Tensors allocated on the current stream but used on another: the allocator must wait for that one."""
    if stream is not None:
        s = _torch_stream(stream, tensors[0].device)
        for t in tensors:
            t.record_stream(s)


def _token_rows(t, heads: int, hs: int, name: str, device):
    """(address, token stride) of a (tokens, heads, head size) view whose tokens' heads are contiguous."""
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    one = heads * hs
    if t.is_contiguous():
        return t.data_ptr(), one
    st = t.stride()
    if t.shape[0] <= 1:  # the stride of a single token means nothing
        st = (one, st[1], st[2])
    if t.numel() and ((hs > 1 and st[2] != 1) or (heads > 1 and st[1] != hs)):
        raise ValueError(f"{name}: a token's heads must be contiguous")
    return t.data_ptr(), st[0] if t.numel() else one


def packed_attention(q, k, v, seq_starts, max_seq_len: int, scale: float, out=None, stream=None):
    """Causal attention of prompts packed one after another: q (tokens, heads,
    head size), k and v (tokens, kv heads, head size) f16 or bf16, tokens at any
    stride that is a multiple of 8 elements (views of a fused projection),
    seq_starts i32 (sequences + 1,) -> out (tokens, heads, head size). No
    sequence may be longer than max_seq_len, and `out` must be apart from the
    others (other columns of one buffer's rows are). Tokens behind the last sequence are
    left as they were in `out` (without one, as the new tensor holds them, and
    `stream` waits for the current stream's work, which may still use its memory)."""
    import torch

    (tokens, heads, hs), dtype, dev = q.shape, q.dtype, q.device
    if dtype not in (torch.float16, torch.bfloat16) or k.dtype != dtype or v.dtype != dtype:
        raise ValueError(f"q, k and v must be f16 or all bf16, not {dtype}, {k.dtype}, {v.dtype}")
    kv = k.shape[1] if k.dim() == 3 else 0
    if k.shape != (tokens, kv, hs) or v.shape != k.shape:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not match")
    fresh = out is None
    if fresh:
        out = torch.empty((tokens, heads, hs), dtype=dtype, device=dev)
    elif out.shape != q.shape or out.dtype != dtype:
        raise ValueError("out must have q's shape and type")
    a = TlhPackedArgs()
    a.q, a.q_stride = _token_rows(q, heads, hs, "q", dev)
    a.k, a.k_stride = _token_rows(k, kv, hs, "k", dev)
    a.v, a.v_stride = _token_rows(v, kv, hs, "v", dev)
    a.out, a.out_stride = _token_rows(out, heads, hs, "out", dev)
    n = _extent(seq_starts)
    a.seq_starts = _tensor(seq_starts, torch.int32, (n,), "seq_starts", dev)
    if n < 1:
        raise ValueError("seq_starts must hold at least one start")
    a.type = F16 if dtype == torch.float16 else BF16
    a.num_seqs, a.num_tokens, a.max_seq_len = n - 1, _int32(tokens, "tokens"), _int32(max_seq_len, "max_seq_len")
    a.num_heads, a.num_kv_heads, a.head_size, a.scale = heads, kv, hs, scale
    with _on(dev, stream) as s:
        if fresh:
            _behind_current(stream, dev)
        check(lib().tlh_packed_attention(C.byref(a), s))
    if fresh:
        _use_on(stream, out)
    return out


class _ScratchNode:
    """A node that owns its scratch, which it allocates on the current stream; its calls may run on others. Calls
    of one node must be stream-ordered, and a captured call keeps using the scratch: keep the node with the graph."""

    def _allocate(self, nbytes: int, device):
        import torch

        self.scratch_bytes = nbytes
        self.scratch = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=device)
        self.device, self.scratch_ptr = self.scratch.device, self.scratch.data_ptr()
        self._home = _current(self.device) if self.device.type == "cuda" else 0
        self._streams = {self._home}  # those that may use it

    def _use_scratch(self, stream: int):
        """Called before a launch on `stream`. On another stream's first call, that one waits for the work queued on
        the scratch's own, which may still use its memory, and the allocator learns that it uses the scratch."""
        if stream in self._streams:
            return
        side, home = (_torch_stream(n, self.device) for n in (stream, self._home))
        # (a capture cannot wait for work outside it, and begins with the device idle)
        if not _capturing(side) and not _capturing(home):
            side.wait_stream(home)
            self._streams.add(stream)
        self.scratch.record_stream(side)


def _capturing(stream) -> bool:
    import torch

    with torch.cuda.stream(stream):  # (the default stream cannot be captured, nor asked while others are)
        return stream.cuda_stream != 0 and torch.cuda.is_current_stream_capturing()


class TreeAttention(_ScratchNode):
    """Attention of drafted tokens over the paged cache, with its scratch, launched many times. A call
    takes up to num_seqs sequences and num_rows drafted tokens in all, at most max_drafts (<= 64) of one
    sequence; calls of one object must be stream-ordered (they share the scratch)."""

    def __init__(self, num_seqs, num_rows, max_drafts, num_heads, num_kv_heads, head_size, block_size,
                 max_blocks_per_seq, max_context_len, scale, device="cuda"):
        a = self.args = TlhTreeArgs()
        counts = dict(num_seqs=num_seqs, num_rows=num_rows, max_drafts=max_drafts, num_heads=num_heads,
                      num_kv_heads=num_kv_heads, head_size=head_size, block_size=block_size,
                      max_blocks_per_seq=max_blocks_per_seq, max_context_len=max_context_len)
        for name, value in counts.items():
            setattr(a, name, _int32(value, name))
        a.scale = scale
        n = C.c_size_t()
        check(lib().tlh_tree_attention_scratch_bytes(C.byref(a), C.byref(n)))
        self._allocate(n.value, device)

    def __call__(self, out, q, k_cache, v_cache, block_tables, context_lens, draft_starts, draft_masks, stream=None):
        """q and out f16 (rows, heads, head size) with rows <= num_rows, the caches in the paged-attention
        layouts, block_tables i32 (sequences, max_blocks_per_seq) with sequences <= num_seqs, context_lens
        i32 (sequences,) with the drafted tokens, draft_starts i32 (sequences + 1,), draft_masks i64
        (rows,): bit j = sees draft j."""
        import torch

        a, dev = TlhTreeArgs.from_buffer_copy(self.args), self.device  # a call's own: threads may share the node
        rows, S, KV, D, bs = _extent(out), _extent(block_tables), a.num_kv_heads, a.head_size, a.block_size
        if rows > a.num_rows or S > a.num_seqs:
            raise ValueError(f"out of {rows} rows and block_tables of {S} sequences, for up to {a.num_rows} and {a.num_seqs}")
        a.num_rows, a.num_seqs = rows, S
        a.q = _tensor(q, torch.float16, (rows, a.num_heads, D), "q", dev)
        a.out = _tensor(out, torch.float16, (rows, a.num_heads, D), "out", dev)
        a.num_blocks = blocks = _extent(k_cache)
        a.k_cache = _tensor(k_cache, torch.float16, (blocks, KV, D // 8, bs, 8), "k_cache", dev)
        a.v_cache = _tensor(v_cache, torch.float16, (blocks, KV, D, bs), "v_cache", dev)
        a.block_tables = _tensor(block_tables, torch.int32, (S, a.max_blocks_per_seq), "block_tables", dev)
        a.context_lens = _tensor(context_lens, torch.int32, (S,), "context_lens", dev)
        a.draft_starts = _tensor(draft_starts, torch.int32, (S + 1,), "draft_starts", dev)
        a.draft_masks = _tensor(draft_masks, torch.int64, (rows,), "draft_masks", dev)
        with _on(dev, stream) as s:
            self._use_scratch(s)
            check(lib().tlh_tree_attention(C.byref(a), self.scratch_ptr, self.scratch_bytes, s))
        return out


def tree_attention(q, k_cache, v_cache, block_tables, context_lens, draft_starts, draft_masks, max_drafts: int,
                   max_context_len: int, scale: float, stream=None):
    """One TreeAttention call: q f16 (rows, heads, head size) -> out alike (zeros in rows behind the last sequence).
    `stream` waits for the current stream's work."""
    import torch

    rows, heads, hs = q.shape
    node = TreeAttention(block_tables.shape[0], rows, max_drafts, heads, v_cache.shape[1], hs, v_cache.shape[3],
                         block_tables.shape[1], max_context_len, scale, device=q.device)
    out = torch.zeros((rows, heads, hs), dtype=q.dtype, device=q.device)
    # the zeros come from the current stream; the copies are the call's, on its own
    with torch.cuda.stream(_behind_current(stream, q.device)):
        q, block_tables = q.contiguous(), block_tables.contiguous()
    node(out, q, k_cache, v_cache, block_tables, context_lens, draft_starts, draft_masks, stream)
    _use_on(stream, out)
    return out


class KVPools:
    """The key and value pools of a cache's layers (lists of f16 tensors in the
    paged-attention layouts, one length in blocks), moved in all layers at once."""

    def __init__(self, k_caches, v_caches, num_kv_heads: int, head_size: int, block_size: int):
        import torch

        if len(k_caches) != len(v_caches) or not k_caches:
            raise ValueError("as many key as value pools, at least one")
        self.device, self.num_blocks = k_caches[0].device, k_caches[0].shape[0]
        self.kv_heads, self.head_size, self.block_size = num_kv_heads, head_size, block_size
        self.block_bytes = num_kv_heads * head_size * block_size * 2
        n, self.layers = self.num_blocks, len(k_caches)
        ks = [_tensor(t, torch.float16, (n, num_kv_heads, head_size // 8, block_size, 8), "k_cache", self.device)
              for t in k_caches]
        vs = [_tensor(t, torch.float16, (n, num_kv_heads, head_size, block_size), "v_cache", self.device)
              for t in v_caches]
        self.tensors = (list(k_caches), list(v_caches))  # the pools live as long as their addresses are used
        self._all = (C.c_void_p * (2 * self.layers))(*ks, *vs)
        self._k, self._v = (C.c_void_p * self.layers)(*ks), (C.c_void_p * self.layers)(*vs)

    def copy_blocks(self, pairs, stream=None) -> None:
        """Block pairs[i, 0] to block pairs[i, 1] in every pool; pairs i64 (n, 2). No destination may be
        another pair's destination or any pair's source; a pair outside the pools does nothing."""
        import torch

        n = _int32(_extent(pairs), "pairs")
        p = _tensor(pairs, torch.int64, (n, 2), "pairs", self.device)
        with _on(self.device, stream) as s:
            check(lib().tlh_copy_blocks(self._all, 2 * self.layers, self.block_bytes, self.num_blocks, p, n, s))

    def compact(self, block_tables, context_lens, draft_starts, keep, new_lens, max_drafts: int, stream=None):
        """Moves the kept drafted tokens (bit j of keep[s], i64 (sequences,)) of every sequence right behind
        its committed ones in every layer; new_lens i32 (sequences,) receives the lengths with them."""
        import torch

        a, dev = TlhCompactArgs(), self.device
        S, width = _extent(context_lens), block_tables.shape[-1]
        a.k_caches, a.v_caches = self._k, self._v
        a.block_tables = _tensor(block_tables, torch.int32, (S, width), "block_tables", dev)
        a.context_lens = _tensor(context_lens, torch.int32, (S,), "context_lens", dev)
        a.draft_starts = _tensor(draft_starts, torch.int32, (S + 1,), "draft_starts", dev)
        a.keep = _tensor(keep, torch.int64, (S,), "keep", dev)
        a.new_lens = _tensor(new_lens, torch.int32, (S,), "new_lens", dev)
        a.num_blocks, a.num_layers, a.num_seqs = self.num_blocks, self.layers, S
        a.max_drafts = _int32(max_drafts, "max_drafts")
        a.num_kv_heads, a.head_size, a.block_size = self.kv_heads, self.head_size, self.block_size
        a.max_blocks_per_seq = width
        with _on(dev, stream) as s:
            check(lib().tlh_compact_cache(C.byref(a), s))
        return new_lens


class TokenLogprobs(_ScratchNode):
    """Log probabilities of given tokens, entropies and the `top` likeliest tokens of up to `rows` rows of
    logits, with the scratch; calls of one object must be stream-ordered (they share it)."""

    def __init__(self, rows: int, vocab: int, top: int = 0, dtype=None, device="cuda"):
        import torch

        self.rows, self.vocab, self.dtype = rows, vocab, dtype or torch.float32
        a = self.args = TlhLogprobsArgs()
        a.type = _ggml_type(torch.empty(0, dtype=self.dtype))
        a.rows, a.vocab, a.top = _int32(rows, "rows"), _int32(vocab, "vocab"), _int32(top, "top")
        a.row_stride = vocab
        n = C.c_size_t()
        check(lib().tlh_token_logprobs_scratch_bytes(C.byref(a), C.byref(n)))
        self._allocate(n.value, device)

    def __call__(self, logits, tokens, logprobs, entropy, top_logprobs=None, top_ids=None, stream=None):
        """logits (n, vocab) with n <= rows, any row stride; tokens i32 (n,); logprobs and entropy f32 (n,);
        top_logprobs f32 and top_ids i32 (n, top). tokens and logprobs, or entropy, may be None."""
        import torch

        a, dev, n, vocab = TlhLogprobsArgs.from_buffer_copy(self.args), self.device, _extent(logits), self.vocab
        if (logits.dtype != self.dtype or logits.shape != (n, vocab) or n > self.rows or logits.device != dev or
                (vocab > 1 and logits.stride(1) != 1)):
            raise ValueError(f"logits {logits.dtype} {tuple(logits.shape)} on {logits.device}, strides {logits.stride()}, "
                             f"for up to {self.rows} rows of {vocab} {self.dtype} on {dev}")
        a.rows, a.logits = n, logits.data_ptr()
        a.row_stride = logits.stride(0) if n > 1 else vocab
        a.tokens = _tensor(tokens, torch.int32, (n,), "tokens", dev) if tokens is not None else None
        a.logprobs = _tensor(logprobs, torch.float32, (n,), "logprobs", dev) if logprobs is not None else None
        a.entropy = _tensor(entropy, torch.float32, (n,), "entropy", dev) if entropy is not None else None
        if a.top:
            if top_logprobs is None or top_ids is None:
                raise ValueError("top_logprobs and top_ids are needed where top > 0")
            a.top_logprobs = _tensor(top_logprobs, torch.float32, (n, a.top), "top_logprobs", dev)
            a.top_ids = _tensor(top_ids, torch.int32, (n, a.top), "top_ids", dev)
        with _on(dev, stream) as s:
            self._use_scratch(s)
            check(lib().tlh_token_logprobs(C.byref(a), self.scratch_ptr, self.scratch_bytes, s))
        return logprobs, entropy, top_logprobs, top_ids


def token_logprobs(logits, tokens, top: int = 0, stream=None):
    """logits (rows, vocab) f32 / f16 / bf16, tokens i32 (rows,) -> (logprobs (rows,), entropy (rows,),
    top_logprobs (rows, top), top_ids i32 (rows, top)). `stream` waits for the current stream's work, which
    may still use the new tensors' memory."""
    import torch

    n, dev = logits.shape[0], logits.device
    node = TokenLogprobs(n, logits.shape[1], top, logits.dtype, device=dev)
    f = lambda *s: torch.empty(s, dtype=torch.float32, device=dev)  # noqa: E731
    outs = (f(n), f(n), f(n, top), torch.empty((n, top), dtype=torch.int32, device=dev))
    _behind_current(stream, dev)
    node(logits, tokens, *outs, stream=stream)
    _use_on(stream, *outs)
    return outs


CHUNK_COUNTER_BYTES = 8192


class ChunkAttention(_ScratchNode):
    """Causal attention of the sequences' new tokens over the paged cache, one or thousands a sequence, with its
    scratch, launched many times; window > 0: a token sees the last `window` tokens up to itself. f16_weights: sequences
    with more than 64 rows of q a kv head round the softmax's weights to f16 before they meet v, as tree
    attention does (less exact, and a quarter faster where many rows see long contexts). A call takes up to
    num_seqs sequences and num_rows new tokens in all, at most max_rows of one sequence; calls of one object must be
    stream-ordered (they share the scratch). One made while a graph is captured is for captured calls alone: each
    clears the counters in its own graph."""

    def __init__(self, num_seqs, num_rows, max_rows, num_heads, num_kv_heads, head_size, block_size,
                 max_blocks_per_seq, max_context_len, scale, window: int = 0, device="cuda", f16_weights: bool = False):
        a = self.args = TlhChunkArgs()
        counts = dict(num_seqs=num_seqs, num_rows=num_rows, max_rows=max_rows, num_heads=num_heads,
                      num_kv_heads=num_kv_heads, head_size=head_size, block_size=block_size,
                      max_blocks_per_seq=max_blocks_per_seq, max_context_len=max_context_len, window=window)
        for name, value in counts.items():
            setattr(a, name, _int32(value, name))
        a.scale, a.f16_weights = scale, bool(f16_weights)
        n = C.c_size_t()
        check(lib().tlh_chunk_attention_scratch_bytes(C.byref(a), C.byref(n)))
        self._allocate(n.value, device)
        self._captured = self.device.type == "cuda" and _capturing(_torch_stream(self._home, self.device))
        if not self._captured:
            self.scratch[:CHUNK_COUNTER_BYTES].zero_()  # and every call leaves them so

    def __call__(self, out, q, k_cache, v_cache, block_tables, context_lens, row_starts, stream=None):
        """q and out f16 (rows, heads, head size) with rows <= num_rows, tokens at any stride that is a multiple of 8
        elements, the caches in the paged-attention layouts, block_tables i32 (sequences, max_blocks_per_seq) with
        sequences <= num_seqs, context_lens i32 (sequences,) with the new tokens, row_starts i32 (sequences + 1,)."""
        import torch

        a, dev = TlhChunkArgs.from_buffer_copy(self.args), self.device  # a call's own: threads may share the node
        rows, S, H, KV, D, bs = (_extent(out), _extent(block_tables), a.num_heads, a.num_kv_heads, a.head_size,
                                 a.block_size)
        if rows > a.num_rows or S > a.num_seqs:
            raise ValueError(f"out of {rows} rows and block_tables of {S} sequences, for up to {a.num_rows} and {a.num_seqs}")
        for name, t in (("q", q), ("out", out)):
            if t.dtype != torch.float16 or t.shape != (rows, H, D):
                raise ValueError(f"{name}: {t.dtype} {tuple(t.shape)}, not {torch.float16} {(rows, H, D)}")
        a.num_rows, a.num_seqs = rows, S
        a.q, a.q_stride = _token_rows(q, H, D, "q", dev)
        a.out, a.out_stride = _token_rows(out, H, D, "out", dev)
        a.num_blocks = blocks = _extent(k_cache)
        a.k_cache = _tensor(k_cache, torch.float16, (blocks, KV, D // 8, bs, 8), "k_cache", dev)
        a.v_cache = _tensor(v_cache, torch.float16, (blocks, KV, D, bs), "v_cache", dev)
        a.block_tables = _tensor(block_tables, torch.int32, (S, a.max_blocks_per_seq), "block_tables", dev)
        a.context_lens = _tensor(context_lens, torch.int32, (S,), "context_lens", dev)
        a.row_starts = _tensor(row_starts, torch.int32, (S + 1,), "row_starts", dev)
        with _on(dev, stream) as s:
            if self._captured:
                side, home = (_torch_stream(n, dev) for n in (s, self._home))
                if not _capturing(home):
                    raise ValueError("the node was made while a graph was captured: it is for calls in that graph or in others")
                if side != home:
                    side.wait_stream(home)
                with torch.cuda.stream(side):  # in this call's graph: another's clearing may not have been replayed
                    self.scratch[:CHUNK_COUNTER_BYTES].zero_()
            self._use_scratch(s)
            check(lib().tlh_chunk_attention(C.byref(a), self.scratch_ptr, self.scratch_bytes, s))
        return out


def chunk_attention(q, k_cache, v_cache, block_tables, context_lens, row_starts, max_rows: int, max_context_len: int,
                    scale: float, window: int = 0, stream=None, f16_weights: bool = False):
    """One ChunkAttention call: q f16 (rows, heads, head size) -> out alike, contiguous (zeros in rows behind the last
    sequence). `stream` waits for the current stream's work."""
    import torch

    rows, heads, hs = q.shape
    node = ChunkAttention(block_tables.shape[0], rows, max_rows, heads, v_cache.shape[1], hs, v_cache.shape[3],
                          block_tables.shape[1], max_context_len, scale, window, device=q.device, f16_weights=f16_weights)
    out = torch.zeros((rows, heads, hs), dtype=q.dtype, device=q.device)
    # the zeros come from the current stream; the copy is the call's, on its own
    with torch.cuda.stream(_behind_current(stream, q.device)):
        block_tables = block_tables.contiguous()
    node(out, q, k_cache, v_cache, block_tables, context_lens, row_starts, stream)
    _use_on(stream, out)
    return out


def rope_freqs(n_dims: int, freq_base: float = 10000.0, freq_scale: float = 1.0, freq_factors=None, device="cuda"):
    """HeadRope's frequencies, f32 (n_dims / 2,): freq_scale * freq_base^(-2 p / n_dims) / freq_factors[p]."""
    import torch

    p = torch.arange(n_dims // 2, dtype=torch.float64)
    f = freq_scale * float(freq_base) ** (-2.0 * p / n_dims)
    if freq_factors is not None:
        f = f / freq_factors.detach().cpu().double()
    return f.float().to(device)


def rope_sections(sections, interleaved: bool = False):
    """HeadRope's pair_axes where sections[a] pairs take axis a: one section after another, or in turn (pair p takes
    axis p % axes while that has pairs left, axis 0 then)."""
    axes = len(sections)
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    return [p % axes if p < axes * sections[p % axes] else 0 for p in range(sum(sections))]


class HeadRope:
    """The norms of the query and key heads, their rotation by the tokens' positions and the write of keys and values
    to the paged cache, in one launch. freqs f32 (n_dims / 2,) on the GPU: pair p turns by its position times freqs[p];
    pair_axes: the axis each pair takes its position from (None: one axis); mode 0 pairs dims 2p and 2p + 1, 2 (neox)
    p and p + n_dims / 2; dims from n_dims on are not rotated. attn_factor multiplies cos and sin."""

    def __init__(self, num_heads: int, num_kv_heads: int, head_size: int, freqs, pair_axes=None, mode: int = 2,
                 eps: float = 1e-6, attn_factor: float = 1.0):
        import torch

        pairs = _extent(freqs)
        a = self.args = TlhHeadRopeArgs()
        a.num_heads, a.num_kv_heads = _int32(num_heads, "num_heads"), _int32(num_kv_heads, "num_kv_heads")
        a.head_size, a.n_dims, a.mode = _int32(head_size, "head_size"), 2 * pairs, _int32(mode, "mode")
        a.eps, a.attn_factor = eps, attn_factor
        self.device, self.freqs = freqs.device, freqs  # freqs live as long as their address is used
        a.freqs = _tensor(freqs, torch.float32, (pairs,), "freqs", self.device)
        axes = [0] * pairs if pair_axes is None else [int(x) for x in pair_axes]
        if len(axes) != pairs or pairs > 128 or any(not 0 <= x < 4 for x in axes):
            raise ValueError(f"pair_axes must give one of four axes for each of {pairs} (at most 128) pairs")
        a.num_axes = max(axes, default=0) + 1
        a.pair_axis = (C.c_uint8 * 128)(*axes)

    def _out(self, t, like, q_out, name: str):
        if t.dtype != q_out.dtype or t.shape != like.shape:
            raise ValueError(f"{name}: {t.dtype} {tuple(t.shape)}, not {q_out.dtype} {tuple(like.shape)}")
        return _token_rows(t, self.args.num_kv_heads, self.args.head_size, name, self.device)

    def __call__(self, q, k, v, positions, q_out, q_norm=None, k_norm=None, k_out=None, v_out=None, k_cache=None,
                 v_cache=None, slots=None, stream=None):
        """q (tokens, heads, head size), k and v (tokens, kv heads, head size) f32, f16 or bf16, tokens at any stride
        that is a multiple of 16 bytes (views of a fused projection), positions i32 (tokens,) or (axes, tokens); q_norm
        and k_norm f32 (head size,) or None -> q_out, and k_out and v_out where given (f16 or bf16); k_cache, v_cache
        and slots i64 (tokens,) as reshape_and_cache takes them (then the outputs are f16)."""
        import torch

        a, dev = TlhHeadRopeArgs.from_buffer_copy(self.args), self.device
        H, KV, D, n = a.num_heads, a.num_kv_heads, a.head_size, _extent(q)
        if q.dtype != k.dtype or q.dtype != v.dtype or q.shape != (n, H, D) or k.shape != (n, KV, D) or v.shape != k.shape:
            raise ValueError(f"q {q.dtype} {tuple(q.shape)}, k {k.dtype} {tuple(k.shape)} and v {v.dtype} {tuple(v.shape)}, "
                             f"for {H} heads and {KV} kv heads of {D}")
        a.num_tokens, a.type, a.out_type = _int32(n, "tokens"), _ggml_type(q), _ggml_type(q_out)
        a.q, a.q_stride = _token_rows(q, H, D, "q", dev)
        a.k, a.k_stride = _token_rows(k, KV, D, "k", dev)
        a.v, a.v_stride = _token_rows(v, KV, D, "v", dev)
        if q_out.shape != q.shape:
            raise ValueError(f"q_out: {tuple(q_out.shape)}, not {tuple(q.shape)}")
        a.q_out, a.q_out_stride = _token_rows(q_out, H, D, "q_out", dev)
        a.k_out_stride = a.v_out_stride = KV * D
        if k_out is not None:
            a.k_out, a.k_out_stride = self._out(k_out, k, q_out, "k_out")
        if v_out is not None:
            a.v_out, a.v_out_stride = self._out(v_out, k, q_out, "v_out")
        if a.n_dims:
            one = positions.dim() == 1 and a.num_axes == 1
            a.positions = _tensor(positions, torch.int32, (n,) if one else (a.num_axes, n), "positions", dev)
        if q_norm is not None:
            a.q_norm = _tensor(q_norm, torch.float32, (D,), "q_norm", dev)
        if k_norm is not None:
            a.k_norm = _tensor(k_norm, torch.float32, (D,), "k_norm", dev)
        if k_cache is not None or v_cache is not None or slots is not None:
            if k_cache is None or v_cache is None or slots is None:
                raise ValueError("k_cache, v_cache and slots go together")
            a.num_blocks = blocks = _extent(k_cache)
            a.block_size = bs = v_cache.shape[-1] if v_cache.dim() else 0
            a.k_cache = _tensor(k_cache, torch.float16, (blocks, KV, D // 8, bs, 8), "k_cache", dev)
            a.v_cache = _tensor(v_cache, torch.float16, (blocks, KV, D, bs), "v_cache", dev)
            a.slots = _tensor(slots, torch.int64, (n,), "slots", dev)
        with _on(dev, stream) as s:
            check(lib().tlh_head_rope(C.byref(a), s))
        return q_out


class DraftVerify(_ScratchNode):
    """Verification of drafted tokens (a chain a sequence) against the model's probabilities from given random numbers,
    with the scratch. A call takes up to num_seqs sequences and num_drafts drafted tokens in all, at most max_drafts of
    one sequence; drafter: whether a drafting model's logits come with them (else tokens were proposed outright). Calls
    of one object must be stream-ordered (they share the scratch)."""

    def __init__(self, num_seqs: int, num_drafts: int, max_drafts: int, vocab: int, dtype=None, drafter: bool = True,
                 device="cuda"):
        import torch

        self.dtype, self.vocab, self.drafter = dtype or torch.float32, vocab, drafter
        a = self.args = TlhVerifyArgs()
        a.type = _ggml_type(torch.empty(0, dtype=self.dtype))
        for name, value in dict(num_seqs=num_seqs, num_drafts=num_drafts, max_drafts=max_drafts, vocab=vocab).items():
            setattr(a, name, _int32(value, name))
        a.target_stride = a.draft_stride = vocab
        a.draft = 16 if drafter else None  # (the size asks only whether there is one)
        n = C.c_size_t()
        check(lib().tlh_draft_verify_scratch_bytes(C.byref(a), C.byref(n)))
        self._allocate(n.value, device)

    def _logits(self, t, rows: int, name: str):
        if (t.dtype != self.dtype or t.shape != (rows, self.vocab) or t.device != self.device or
                (self.vocab > 1 and t.numel() and t.stride(1) != 1)):
            raise ValueError(f"{name} {t.dtype} {tuple(t.shape)} on {t.device}, strides {t.stride()}, "
                             f"not {rows} rows of {self.vocab} {self.dtype} on {self.device}")
        return t.data_ptr(), t.stride(0) if rows > 1 else self.vocab

    def __call__(self, target, draft, tokens, draft_starts, temperatures, accept_at, sample_at, accepted, out_tokens,
                 accept_probs=None, stream=None):
        """target (drafts + sequences, vocab): sequence s has the rows of its n drafted tokens and one more, from
        draft_starts[s] + s on; draft (drafts, vocab) or None; tokens i32 (drafts,), draft_starts i32 (sequences + 1,)
        (a sequence that shares drafts with another is not verified: 0 accepted, tokens -1, probabilities NaN),
        temperatures f32 (sequences,) (0: greedy), accept_at f32 (drafts,) and sample_at f32 (sequences,) uniform in
        [0, 1) -> accepted i32 (sequences,), out_tokens i32 (sequences, max_drafts + 1): the accepted tokens, the next
        one, -1 behind; accept_probs f32 (drafts,) or None."""
        import torch

        a, dev = TlhVerifyArgs.from_buffer_copy(self.args), self.device
        R, S = _extent(tokens), _extent(temperatures)
        if R > a.num_drafts or S > a.num_seqs:
            raise ValueError(f"{R} drafted tokens of {S} sequences, for up to {a.num_drafts} and {a.num_seqs}")
        if (draft is not None) != self.drafter:
            raise ValueError("a drafting model's logits come with every call of a node made for them, and with no other")
        a.num_drafts, a.num_seqs = R, S
        a.target, a.target_stride = self._logits(target, R + S, "target")
        if draft is not None:
            a.draft, a.draft_stride = self._logits(draft, R, "draft")
        a.tokens = _tensor(tokens, torch.int32, (R,), "tokens", dev)
        a.draft_starts = _tensor(draft_starts, torch.int32, (S + 1,), "draft_starts", dev)
        a.temperatures = _tensor(temperatures, torch.float32, (S,), "temperatures", dev)
        a.accept_at = _tensor(accept_at, torch.float32, (R,), "accept_at", dev)
        a.sample_at = _tensor(sample_at, torch.float32, (S,), "sample_at", dev)
        a.accepted = _tensor(accepted, torch.int32, (S,), "accepted", dev)
        a.out_tokens = _tensor(out_tokens, torch.int32, (S, a.max_drafts + 1), "out_tokens", dev)
        a.accept_probs = _tensor(accept_probs, torch.float32, (R,), "accept_probs", dev) if accept_probs is not None else None
        with _on(dev, stream) as s:
            self._use_scratch(s)
            check(lib().tlh_draft_verify(C.byref(a), self.scratch_ptr, self.scratch_bytes, s))
        return accepted, out_tokens, accept_probs


def draft_verify(target, draft, tokens, draft_starts, temperatures, accept_at, sample_at, max_drafts: int, stream=None):
    """One DraftVerify call -> (accepted i32 (sequences,), out_tokens i32 (sequences, max_drafts + 1), accept_probs f32
    (drafts,), NaN for drafts of no sequence). `stream` waits for the current stream's work, which may still use the
    new tensors' memory."""
    import torch

    S, R, dev = temperatures.shape[0], tokens.shape[0], target.device
    node = DraftVerify(S, R, max_drafts, target.shape[1], target.dtype, draft is not None, device=dev)
    outs = (torch.empty(S, dtype=torch.int32, device=dev), torch.empty((S, max_drafts + 1), dtype=torch.int32, device=dev),
            torch.full((R,), float("nan"), device=dev))
    _behind_current(stream, dev)
    node(target, draft, tokens, draft_starts, temperatures, accept_at, sample_at, *outs, stream=stream)
    _use_on(stream, *outs)
    return outs


# ------------------------------------------------------------------ core ops
# The ops around MUL_MAT and attention in a decoder step, packed as the
# reference's lowering packs them for its core kernels
# (crates/kernels/src/cuda/lower.rs:175-500) and run by tlh_core.
(CORE_BIN, CORE_UNARY, CORE_NORM, CORE_GET_ROWS, CORE_SET_ROWS, CORE_CPY, CORE_ROPE, CORE_SOFT_MAX, CORE_ARGMAX,
 CORE_GLU) = range(1, 11)
I32, I64 = 26, 27
# ggml_unary_op codes (ggml.h) and the lowering's extra element-wise codes
UNARY = {"abs": 0, "sgn": 1, "neg": 2, "step": 3, "tanh": 4, "elu": 5, "relu": 6, "sigmoid": 7, "gelu": 8,
         "gelu_quick": 9, "silu": 10, "hardswish": 11, "hardsigmoid": 12, "exp": 13, "expm1": 14, "softplus": 15,
         "gelu_erf": 16, "floor": 18, "ceil": 19, "round": 20, "trunc": 21, "scale": 100, "fill": 101,
         "clamp": 102, "leaky_relu": 103, "sqr": 104, "sqrt": 105, "sin": 106, "cos": 107, "log": 108}
# ggml_glu_op codes (ggml.h:623-630); swiglu_oai is not supported
GLU = {"reglu": 0, "geglu": 1, "swiglu": 2, "geglu_erf": 4, "geglu_quick": 5}

_libm = None


def _f32_fn(name: str):
    """The C library's single-precision `name` (powf, logf, ...): the host-side
    parameters below are derived with the same f32 functions the CPU backend
    and the reference's lowering call, so they match bit for bit."""
    global _libm
    if _libm is None:
        _libm = C.CDLL("libm.so.6")
    f = getattr(_libm, name)
    f.restype = C.c_float
    f.argtypes = [C.c_float] * (2 if name == "powf" else 1)
    return f


def _f32(x) -> float:
    import struct

    return struct.unpack("<f", struct.pack("<f", x))[0]


def core_type(t) -> int:
    import torch

    return {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16, torch.int32: I32,
            torch.int64: I64}.get(t.dtype, -1)


def quant_desc(t, wtype: int, k: int) -> TlhTensor:
    """The ggml descriptor of quantized rows held as a uint8 torch tensor of shape
    (..., rows, row_bytes): ne [k, rows, ...], nb from the tensor's byte strides."""
    rb = row_bytes(wtype, k)
    if t.shape[-1] != rb or t.stride(-1) != 1:
        raise ValueError(f"rows must be {rb} contiguous bytes for {TYPE_NAMES[wtype]} k={k}")
    lead = list(t.shape[:-1])[::-1] + [1] * (4 - t.dim())
    nbs = [s for s in list(t.stride()[:-1])[::-1]]
    while len(nbs) < 3:
        nbs.append(nbs[-1] * lead[len(nbs) - 1] if nbs else rb)
    return ggml_tensor(wtype, [k] + lead[:3], [BLOCK[wtype][1]] + nbs[:3])


def core_op(srcs, dst, x=()) -> TlhOp:
    """t[0..2] = the sources (torch tensors, TlhTensor descriptors or None),
    t[4] = dst, x[] = the op's parameters."""
    op = TlhOp()
    for i, t in enumerate(srcs):
        if t is None:
            continue
        op.t[i] = t if isinstance(t, TlhTensor) else tensor_desc(t, core_type(t))
    op.t[4] = dst if isinstance(dst, TlhTensor) else tensor_desc(dst, core_type(dst))
    for i, v in enumerate(x):
        op.x[i] = v
    return op


class CoreOp:
    """One core node, validated once (tlh_core_check) and run on each call."""

    def __init__(self, kind: int, op: TlhOp, has_src1: bool, has_src2: bool):
        self.kind, self.op = kind, op
        check(lib().tlh_core_check(kind, C.byref(op), int(has_src1), int(has_src2)))

    def __call__(self, src0, src1, src2, dst, stream=None):
        p = lambda t: _ptr(t) if t is not None else None  # noqa: E731
        check(lib().tlh_core(self.kind, C.byref(self.op), p(src0), p(src1), p(src2), _ptr(dst), _stream(stream)))
        return dst


def _run(kind, srcs, dst, x=(), descs=None, stream=None):
    op = core_op(descs if descs is not None else srcs, dst, x)
    s = list(srcs) + [None] * (3 - len(srcs))
    return CoreOp(kind, op, s[1] is not None, s[2] is not None)(s[0], s[1], s[2], dst, stream)


def _out(like, out, dtype=None):
    import torch

    return out if out is not None else torch.empty(like.shape, dtype=dtype or like.dtype, device=like.device)


def binary(code: int, a, b, out=None, stream=None):
    """ADD/SUB/MUL/DIV (code 0..3) with b repeated to a's shape (lower.rs:219-248)."""
    return _run(CORE_BIN, [a, b], _out(a, out), (code,), stream=stream)


def add(a, b, out=None, stream=None):
    return binary(0, a, b, out, stream)


def mul(a, b, out=None, stream=None):
    return binary(2, a, b, out, stream)


def unary(op, a, p1: float = 0.0, p2: float = 0.0, out=None, stream=None):
    """A ggml unary op or the lowering's element-wise extras (lower.rs:250-290),
    by name or code: scale (p1 s, p2 b), fill (p1), clamp (p1 min, p2 max),
    leaky_relu (p1 slope)."""
    code = UNARY[op] if isinstance(op, str) else int(op)
    return _run(CORE_UNARY, [a], _out(a, out), (code, _f32_bits(p1), _f32_bits(p2)), stream=stream)


def norm(a, eps: float, rms: bool = False, out=None, stream=None):
    """ggml_norm / ggml_rms_norm over ne0 (lower.rs:292-312)."""
    return _run(CORE_NORM, [a], _out(a, out), (int(rms), _f32_bits(eps)), stream=stream)


def rms_norm(a, eps: float, out=None, stream=None):
    return norm(a, eps, True, out, stream)


def get_rows(a, idx, wtype: int = None, k: int = None, out=None, stream=None):
    """ggml_get_rows: out (i3, i2, i1) row = a's row idx[i3, i2, i1] of plane
    (i2, i3). `a` is f32/f16, or quantized rows (uint8, (..., rows, row_bytes))
    with `wtype` and their element count `k`. out is f32 (..., n_idx, ne0)."""
    import torch

    ad = quant_desc(a, wtype, k) if wtype is not None else tensor_desc(a, core_type(a))
    ne0 = k if wtype is not None else a.shape[-1]
    if out is None:
        out = torch.empty(tuple(idx.shape) + (ne0,), dtype=torch.float32, device=idx.device)
    return _run(CORE_GET_ROWS, [a, idx], out, descs=[ad, idx], stream=stream)


def set_rows(dst, src, idx, stream=None):
    """ggml_set_rows: src row (i3, i2, i1) to dst row idx[i3 % n2, i2 % n1, i1]."""
    return _run(CORE_SET_ROWS, [src, idx], dst, stream=stream)


def cpy(src, dst, wtype: int = None, k: int = None, stream=None):
    """ggml_cpy / ggml_cont / ggml_dup: element i of src (row-major over ggml's
    ne) to element i of dst, converted to dst's type."""
    sd = quant_desc(src, wtype, k) if wtype is not None else tensor_desc(src, core_type(src))
    return _run(CORE_CPY, [src], dst, descs=[sd], stream=stream)


def rope_params(n_dims: int, mode: int, n_ctx_orig: int, freq_base: float, freq_scale: float, ext_factor: float,
                attn_factor: float, beta_fast: float, beta_slow: float, has_ff: bool):
    """x[] of Ctx::rope (lower.rs:422-466): the YaRN corr dims of
    ggml_rope_yarn_corr_dims (ggml.c:4369-4381) and theta_scale =
    freq_base^(-2/n_dims), all in f32."""
    import numpy as np

    powf, logf = _f32_fn("powf"), _f32_fn("logf")
    f = np.float32
    with np.errstate(all="ignore"):  # beta 0 or n_ctx_orig 0 give inf / nan, as in C
        def corr(beta):
            ratio = f(n_ctx_orig) / (f(beta) * f(2.0) * f(np.pi))
            return f(f(n_dims) * f(logf(float(ratio)))) / f(f(2.0) * f(logf(freq_base)))

        start, end = np.floor(corr(beta_fast)), np.ceil(corr(beta_slow))
    c0 = 0.0 if 0.0 > start else float(start)  # MAX(0, start) and MIN(n_dims - 1, end) of ggml.c
    c1 = float(n_dims - 1) if n_dims - 1 < end else float(end)
    ts = powf(freq_base, _f32(-2.0 / n_dims))
    return (n_dims, mode, _f32_bits(freq_scale), _f32_bits(ext_factor), _f32_bits(attn_factor), _f32_bits(ts),
            _f32_bits(c0), _f32_bits(c1), int(has_ff))


def rope(a, pos, n_dims: int, mode: int = 0, n_ctx_orig: int = 0, freq_base: float = 10000.0,
         freq_scale: float = 1.0, ext_factor: float = 0.0, attn_factor: float = 1.0, beta_fast: float = 32.0,
         beta_slow: float = 1.0, freq_factors=None, out=None, stream=None):
    """ggml_rope_ext on a (ggml [ne0, heads, tokens, ne3]) with i32 positions [tokens]."""
    x = rope_params(n_dims, mode, n_ctx_orig, freq_base, freq_scale, ext_factor, attn_factor, beta_fast,
                    beta_slow, freq_factors is not None)
    return _run(CORE_ROPE, [a, pos, freq_factors], _out(a, out), x, stream=stream)


def soft_max_params(n_head: int, scale: float, max_bias: float):
    """x[] of Ctx::soft_max (lower.rs:314-341): scale, max_bias, m0, m1, n_head_log2."""
    import math

    powf = _f32_fn("powf")
    nhl2 = 1 << int(math.floor(math.log2(n_head))) if n_head > 0 else 1
    m0 = powf(2.0, _f32(_f32(-max_bias) / nhl2))
    m1 = powf(2.0, _f32(_f32(-_f32(max_bias / 2.0)) / nhl2))
    return (_f32_bits(scale), _f32_bits(max_bias), _f32_bits(m0), _f32_bits(m1), nhl2)


def soft_max(a, mask=None, scale: float = 1.0, max_bias: float = 0.0, out=None, stream=None):
    """ggml_soft_max_ext over ne0 of f32 a, with an optional f16/f32 mask
    (ggml [ne0, >= rows, broadcast over heads / batches])."""
    n_head = a.shape[-3] if a.dim() >= 3 else 1
    return _run(CORE_SOFT_MAX, [a, mask], _out(a, out), soft_max_params(n_head, scale, max_bias), stream=stream)


def argmax(a, out=None, stream=None):
    """ggml_argmax of f32 a (rows, n) -> i32 (rows,): the last index of each row's maximum."""
    import torch

    if out is None:
        out = torch.empty((a.shape[0],), dtype=torch.int32, device=a.device)
    return _run(CORE_ARGMAX, [a], out, stream=stream)


def glu(op, a, b=None, swapped: bool = False, out=None, stream=None):
    """GGML_OP_GLU on f32 rows: act(x) * g with x, g = a, b (ggml_glu_split) or
    the two halves of a's rows (ggml_glu; x first unless swapped)."""
    import torch

    code = GLU[op] if isinstance(op, str) else int(op)
    if out is None:
        shape = tuple(a.shape) if b is not None else tuple(a.shape[:-1]) + (a.shape[-1] // 2,)
        out = torch.empty(shape, dtype=torch.float32, device=a.device)
    return _run(CORE_GLU, [a, b], out, (code, int(swapped)), stream=stream)
