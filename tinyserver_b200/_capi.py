"""ctypes binding of libqwen3fused.so (declared in include/qwen3fused.h).

The library is built in-tree (``python -m tinyserver_b200.build``).  If it is
missing or older than its sources it is rebuilt once per process; if that
fails, every op raises -- there is no CPU or torch fallback.
"""

from __future__ import annotations

import ctypes
import os
import struct
import threading

from . import build as _build

c_i64 = ctypes.c_int64
c_int = ctypes.c_int
c_vp = ctypes.c_void_p
c_float = ctypes.c_float
I64P = ctypes.POINTER(ctypes.c_int64)

QF_F32, QF_F16, QF_BF16 = 0, 1, 2
QF_I32, QF_I64 = 0, 1
QF_OK, QF_ERR_INVALID, QF_ERR_UNSUPPORTED, QF_ERR_LAUNCH, QF_ERR_DEVICE = 0, 1, 2, 3, 4
QF_ERR_SCRATCH = 5
QF_FLAG_BAD_BLOCK, QF_FLAG_BAD_SLOT, QF_FLAG_BAD_TOKEN, QF_FLAG_BAD_TABLE = 1, 2, 4, 8
QF_FLAG_TIMEOUT = 16
QF_FLAG_BAD_TREE = 32
QF_CACHE_PLAIN, QF_CACHE_E4M3, QF_CACHE_INT8 = 0, 1, 2

FLAG_NAMES = {QF_FLAG_BAD_BLOCK: "block index outside the cache",
              QF_FLAG_BAD_SLOT: "slot index outside the block",
              QF_FLAG_BAD_TOKEN: "token id outside the vocabulary",
              QF_FLAG_BAD_TABLE: "position beyond the block table",
              QF_FLAG_TIMEOUT: "a kernel timed out waiting on its tensor-core work",
              QF_FLAG_BAD_TREE: "a tree node's parent is no earlier node, or the tree exceeds "
                                "max_tree"}


class QkNormRopeArgs(ctypes.Structure):
    """Mirror of qf_qk_norm_rope_args (field order and types must match)."""

    _fields_ = [
        ("q", c_vp), ("q_stride_token", c_i64), ("q_stride_head", c_i64),
        ("k", c_vp), ("k_stride_token", c_i64), ("k_stride_head", c_i64),
        ("v", c_vp), ("v_stride_token", c_i64), ("v_stride_head", c_i64),
        ("q_weight", c_vp), ("k_weight", c_vp), ("eps", c_float),
        ("cos", c_vp), ("sin", c_vp), ("cos_sin_token_stride", c_i64),
        ("positions", c_vp), ("positions_type", c_int), ("inv_freq", c_vp),
        ("q_out", c_vp), ("q_out_stride_token", c_i64), ("q_out_stride_head", c_i64),
        ("k_out", c_vp), ("k_out_stride_token", c_i64), ("k_out_stride_head", c_i64),
        ("k_cache", c_vp), ("v_cache", c_vp), ("cache_strides", c_i64 * 4),
        ("num_blocks", c_i64), ("block_size", c_i64),
        ("block_mapping", c_vp), ("slot_mapping", c_vp), ("index_type", c_int),
        ("num_tokens", c_i64), ("num_q_heads", c_i64), ("num_kv_heads", c_i64),
        ("head_dim", c_i64),
        ("dtype", c_int),
        ("status", c_vp),
    ]


class PagedAttentionArgs(ctypes.Structure):
    """Mirror of qf_paged_attention_args (field order and types must match)."""

    _fields_ = [
        ("q", c_vp), ("q_stride_seq", c_i64), ("q_stride_head", c_i64),
        ("k_cache", c_vp), ("v_cache", c_vp), ("cache_strides", c_i64 * 4),
        ("num_blocks", c_i64), ("block_size", c_i64),
        ("block_tables", c_vp), ("block_tables_row_stride", c_i64),
        ("max_blocks_per_seq", c_i64),
        ("seq_lens", c_vp),
        ("num_seqs", c_i64), ("num_q_heads", c_i64), ("num_kv_heads", c_i64),
        ("head_dim", c_i64),
        ("scale", c_float),
        ("out", c_vp), ("out_stride_seq", c_i64), ("out_stride_head", c_i64),
        ("workspace", c_vp), ("workspace_bytes", c_i64),
        ("dtype", c_int),
        ("status", c_vp),
    ]


class PackedArgs:
    """An argument struct of the C side as bytes, packed by position in one call (a few
    microseconds less than a ctypes Structure's fields).  Native sizes and alignment:
    the order and the types must match the header; NULL is 0."""

    def __init__(self, *fields: tuple[str, str]):
        self.names = tuple(name for name, code in fields for _ in range(int(code[:-1] or 1)))
        # "0q" at the end: padded to the size of its widest member
        self._struct = struct.Struct("@" + "".join(code for _, code in fields) + "0q")
        self.pack = self._struct.pack
        self.size = self._struct.size

    def named(self, **values) -> bytes:
        """Packed from names, the rest 0 (a name of several members takes a tuple)."""
        left = {k: list(v) if isinstance(v, tuple) else [v] for k, v in values.items()}
        return self.pack(*(left[n].pop(0) if left.get(n) else 0 for n in self.names))


# qf_kv_quantized_args
KvQuantizedArgs = PackedArgs(
    ("k_rows", "q"), ("k_row_strides", "3q"), ("v_rows", "q"), ("v_row_strides", "3q"),
    ("k_cache", "q"), ("k_cache_strides", "4q"), ("v_cache", "q"), ("v_cache_strides", "4q"),
    ("k_scale", "q"), ("k_scale_strides", "3q"), ("v_scale", "q"), ("v_scale_strides", "3q"),
    ("block_mapping", "q"), ("slot_mapping", "q"),
    ("num_tokens", "q"), ("num_kv_heads", "q"), ("head_dim", "q"), ("num_blocks", "q"),
    ("block_size", "q"),
    ("index_type", "i"), ("dtype", "i"), ("format", "i"),
    ("status", "q"))

# qf_tree_mask_args
TreeMaskArgs = PackedArgs(
    ("parents", "q"), ("cu_seqlens", "q"), ("num_seqs", "q"), ("num_nodes", "q"),
    ("max_tree", "q"), ("mask_words", "q"), ("mask", "q"), ("depths", "q"), ("index_type", "i"),
    ("status", "q"))

# qf_paged_tree_attention_args
PagedTreeAttentionArgs = PackedArgs(
    ("q", "q"), ("q_stride_token", "q"), ("q_stride_head", "q"),
    ("k_cache", "q"), ("v_cache", "q"), ("cache_strides", "4q"),
    ("k_scale", "q"), ("v_scale", "q"), ("scale_strides", "3q"),
    ("num_blocks", "q"), ("block_size", "q"),
    ("block_tables", "q"), ("block_tables_row_stride", "q"), ("max_blocks_per_seq", "q"),
    ("context_lens", "q"), ("cu_seqlens_q", "q"),
    ("tree_mask", "q"), ("mask_words", "q"),
    ("num_seqs", "q"), ("num_tokens", "q"), ("max_tree", "q"),
    ("num_q_heads", "q"), ("num_kv_heads", "q"), ("head_dim", "q"),
    ("scale", "f"),
    ("out", "q"), ("out_stride_token", "q"), ("out_stride_head", "q"),
    ("workspace", "q"), ("workspace_bytes", "q"),
    ("dtype", "i"), ("cache_format", "i"),
    ("status", "q"))


class VarlenAttentionArgs(ctypes.Structure):
    """Mirror of qf_varlen_attention_args (field order and types must match)."""

    _fields_ = [
        ("q", c_vp), ("q_stride_token", c_i64), ("q_stride_head", c_i64),
        ("k", c_vp), ("k_stride_token", c_i64), ("k_stride_head", c_i64),
        ("v", c_vp), ("v_stride_token", c_i64), ("v_stride_head", c_i64),
        ("out", c_vp), ("out_stride_token", c_i64), ("out_stride_head", c_i64),
        ("cu_seqlens_q", c_vp), ("cu_seqlens_k", c_vp),
        ("batch", c_i64), ("max_seqlen_q", c_i64), ("num_q_heads", c_i64),
        ("num_kv_heads", c_i64), ("head_dim", c_i64),
        ("causal", c_int),
        ("scale", c_float),
        ("dtype", c_int),
        ("status", c_vp),
        ("total_q", c_i64), ("total_k", c_i64),
        ("work_counter", c_vp),
    ]


class SampleArgs(ctypes.Structure):
    """Mirror of qf_sample_args (field order and types must match)."""

    _fields_ = [
        ("logits", c_vp), ("logits_row_stride", c_i64),
        ("batch", c_i64), ("vocab", c_i64),
        ("dtype", c_int),
        ("temperature", c_vp),
        ("top_k", c_vp), ("top_k_type", c_int),
        ("top_p", c_vp),
        ("uniforms", c_vp),
        ("seeds", c_vp), ("steps", c_vp),
        ("out", c_vp),
        ("workspace", c_vp), ("workspace_bytes", c_i64),
        ("path", c_int),
    ]


# name -> argtypes of every exported entry point (restype int unless listed below)
SIGNATURES: dict[str, list] = {
    "qf_kv_store_batched": [c_vp, I64P, c_vp, I64P, c_vp, I64P, c_vp, I64P, c_vp, c_vp, c_int,
                            c_i64, c_i64, c_i64, c_i64, c_i64, c_i64, c_vp, c_vp],
    "qf_kv_store_seq": [c_i64, c_vp, c_i64, c_int, c_vp, I64P, c_vp, I64P, c_vp, I64P, c_vp,
                        I64P, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64, c_vp, c_vp],
    "qf_rmsnorm": [c_vp, c_i64, c_vp, c_vp, c_i64, c_i64, c_i64, c_float, c_int, c_vp],
    "qf_add_rmsnorm": [c_vp, c_i64, c_vp, c_i64, c_vp, c_vp, c_i64, c_vp, c_i64, c_i64, c_i64,
                       c_float, c_int, c_vp],
    "qf_rope_cos_sin": [c_vp, c_int, c_vp, c_i64, c_i64, c_float, c_int, c_vp, c_vp, c_vp],
    "qf_qk_norm_rope_store": [ctypes.POINTER(QkNormRopeArgs), c_vp],
    "qf_qk_norm_rope_args_size": [],
    "qf_silu_and_mul": [c_vp, c_i64, c_vp, c_i64, c_vp, c_i64, c_i64, c_i64, c_int, c_vp],
    "qf_embedding": [c_vp, c_int, c_vp, c_i64, c_i64, c_vp, c_i64, c_i64, c_i64, c_i64, c_vp,
                     c_vp],
    "qf_build_slot_mapping": [c_vp, c_i64, c_vp, c_i64, c_vp, c_i64, c_i64, c_i64, c_vp, c_vp,
                              c_vp, c_vp],
    "qf_paged_attention_decode": [ctypes.POINTER(PagedAttentionArgs), c_vp],
    "qf_paged_attention_workspace_bytes": [c_i64, c_i64, c_i64, c_i64],
    "qf_paged_attention_args_size": [],
    "qf_paged_attention_decode_noalloc": [ctypes.POINTER(PagedAttentionArgs), c_vp],
    "qf_paged_attention_noalloc_capacity": [],
    "qf_kv_store_quantized": [c_vp, c_vp],
    "qf_kv_load_quantized": [c_vp, c_vp],
    "qf_kv_quantized_args_size": [],
    "qf_paged_tree_attention": [c_vp, c_vp],
    "qf_paged_tree_attention_workspace_bytes": [c_vp],
    "qf_paged_tree_attention_args_size": [],
    "qf_build_tree_mask": [c_vp, c_vp],
    "qf_tree_mask_args_size": [],
    "qf_varlen_attention": [ctypes.POINTER(VarlenAttentionArgs), c_vp],
    "qf_varlen_attention_args_size": [],
    "qf_sample_tokens": [ctypes.POINTER(SampleArgs), c_vp],
    "qf_sample_workspace_bytes": [c_i64],
    "qf_sample_args_size": [],
    "qf_uniforms_from_seeds": [c_vp, c_vp, c_i64, c_vp, c_vp],
    "qf_read_status": [c_vp, ctypes.POINTER(ctypes.c_int32), c_int, c_vp],
    "qf_last_cuda_error": [],
    "qf_version": [],
}
RESTYPES = {"qf_last_cuda_error": ctypes.c_char_p, "qf_version": ctypes.c_char_p,
            "qf_qk_norm_rope_args_size": ctypes.c_size_t,
            "qf_paged_attention_args_size": ctypes.c_size_t,
            "qf_paged_attention_workspace_bytes": ctypes.c_size_t,
            "qf_paged_tree_attention_workspace_bytes": ctypes.c_size_t,
            "qf_paged_tree_attention_args_size": ctypes.c_size_t,
            "qf_kv_quantized_args_size": ctypes.c_size_t,
            "qf_tree_mask_args_size": ctypes.c_size_t,
            "qf_paged_attention_noalloc_capacity": ctypes.c_size_t,
            "qf_sample_workspace_bytes": c_i64,
            "qf_varlen_attention_args_size": ctypes.c_size_t,
            "qf_sample_args_size": ctypes.c_size_t}

_lock = threading.Lock()
_lib: ctypes.CDLL | None = None


def ensure_built() -> str:
    """Return the library path, (re)building it when its sources changed (the
    sources' hash decides; concurrent processes take turns, see build.build)."""
    if _build.is_stale():
        _build.build()
    return _build.LIB


def lib() -> ctypes.CDLL:
    """Load libqwen3fused.so once (building it first if needed)."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            path = ensure_built()
            handle = ctypes.CDLL(path)
            for name, argtypes in SIGNATURES.items():
                fn = getattr(handle, name)
                fn.argtypes = argtypes
                fn.restype = RESTYPES.get(name, c_int)
            for fn, mirror in (("qf_qk_norm_rope_args_size", QkNormRopeArgs),
                               ("qf_paged_attention_args_size", PagedAttentionArgs),
                               ("qf_varlen_attention_args_size", VarlenAttentionArgs),
                               ("qf_sample_args_size", SampleArgs)):
                size = getattr(handle, fn)()
                if size != ctypes.sizeof(mirror):
                    raise RuntimeError(f"{fn}: ABI mismatch, library {size} bytes, binding "
                                       f"{ctypes.sizeof(mirror)} bytes")
            for fn, packed in (("qf_kv_quantized_args_size", KvQuantizedArgs),
                               ("qf_tree_mask_args_size", TreeMaskArgs),
                               ("qf_paged_tree_attention_args_size", PagedTreeAttentionArgs)):
                size = getattr(handle, fn)()
                if size != packed.size:
                    raise RuntimeError(f"{fn}: ABI mismatch, library {size} bytes, binding "
                                       f"{packed.size} bytes")
            _lib = handle
    return _lib


def lib_path() -> str:
    return _build.LIB


def check(rc: int, what: str) -> None:
    """Turn a QF_* return code into the exception the reference would raise."""
    if rc == QF_OK:
        return
    if rc == QF_ERR_INVALID:
        raise ValueError(f"{what}: invalid argument")
    if rc == QF_ERR_UNSUPPORTED:
        raise ValueError(f"{what}: unsupported shape, stride or alignment")
    if rc == QF_ERR_LAUNCH:
        err = lib().qf_last_cuda_error().decode()
        raise RuntimeError(f"{what}: CUDA launch failed: {err}")
    raise RuntimeError(f"{what}: error code {rc}")


def i64_array(vals) -> ctypes.Array:
    return (c_i64 * len(vals))(*[int(v) for v in vals])
