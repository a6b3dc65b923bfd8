"""A paged KV cache of 8-bit rows: quantised as it is written, read back as dense
rows, and attended to in place (CUDA only, no fallback).

The pages keep the reference's layout (num_blocks, num_kv_heads, block_size,
head_dim), as ``torch.float8_e4m3fn`` or ``torch.int8``, beside one float32
scale per row, (num_blocks, num_kv_heads, block_size):

    amax  = max(max |x|, 2**-100)            over the row, in fp32
    scale = amax / Q                         Q = 448 (e4m3) or 127 (int8)
    code  = round-to-nearest-even(x * (Q / amax))
    value = code * scale

A row that holds an infinity or a NaN is stored with scale NaN and reads back as
NaN.  Half the bytes of a 16-bit cache, plus 4 per row.  The reference keeps its
cache in the model's dtype; the stores here have the arguments of its
``store_kv_cache_batched`` (server/model/kernels/kv_cache.py:194-251).
"""

from __future__ import annotations

import torch

from .. import _capi
from .._runtime import after_launch, device_index, dtype_tag, index_tag, launch, status_ptr
from .tree import attend, check_quantized_cache

__all__ = ["load_kv_cache_quantized", "paged_attention_quantized", "store_kv_cache_quantized"]


def _mappings(what: str, block_mapping: torch.Tensor, slot_mapping: torch.Tensor):
    if block_mapping.dim() != 1 or slot_mapping.shape != block_mapping.shape:
        raise ValueError(f"{what}: block_mapping and slot_mapping must be 1D of one length, got "
                         f"{tuple(block_mapping.shape)} and {tuple(slot_mapping.shape)}")
    itag = index_tag(block_mapping, f"{what} block_mapping")
    if index_tag(slot_mapping, f"{what} slot_mapping") != itag:  # both as the wider
        itag = _capi.QF_I64
        block_mapping, slot_mapping = block_mapping.long(), slot_mapping.long()
    if not block_mapping.is_contiguous():
        block_mapping = block_mapping.contiguous()
    if not slot_mapping.is_contiguous():
        slot_mapping = slot_mapping.contiguous()
    return block_mapping, slot_mapping, itag


def store_kv_cache_quantized(k_src: torch.Tensor, v_src: torch.Tensor, k_cache: torch.Tensor,
                             v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                             block_mapping: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """Quantise a batch's K/V rows into their pages: token t of ``k_src``/``v_src``
    (num_kv_heads, num_tokens, head_dim), float32, float16 or bfloat16, any
    strides, goes to ``cache[block_mapping[t], :, slot_mapping[t]]`` and its scales
    to ``scale[block_mapping[t], :, slot_mapping[t]]``.

    A place outside the cache is skipped and reported through
    :func:`tinyserver_b200.check_errors`.  The places of one call must be
    distinct: of two tokens sent to one place, codes and scale may come from
    different ones."""
    what = "store_kv_cache_quantized"
    if k_src.dim() != 3 or v_src.shape != k_src.shape:
        raise ValueError(f"{what}: k_src and v_src must be 3D tensors of one shape, but got "
                         f"{tuple(k_src.shape)} and {tuple(v_src.shape)}")
    if v_src.dtype != k_src.dtype:
        raise ValueError(f"{what}: k_src and v_src dtypes differ: {k_src.dtype} and {v_src.dtype}")
    fmt = check_quantized_cache(what, k_cache, v_cache, k_scale, v_scale)
    H, T, D = k_src.shape
    if k_cache.shape[1] != H or k_cache.shape[3] != D:
        raise ValueError(f"{what}: cache shape {tuple(k_cache.shape)} does not match k_src "
                         f"(num_kv_heads={H}, head_dim={D})")
    bm, sm, itag = _mappings(what, block_mapping, slot_mapping)
    if bm.numel() != T:
        raise ValueError(f"{what}: {bm.numel()} places for {T} tokens")
    tag = dtype_tag(k_src, what)
    dev = device_index(what, k_src, v_src, k_cache, v_cache, k_scale, v_scale, bm, sm)
    N, _, B, _ = k_cache.shape
    rc = launch(dev, _capi.lib().qf_kv_store_quantized, _capi.KvQuantizedArgs.pack(
        k_src.data_ptr(), *k_src.stride(), v_src.data_ptr(), *v_src.stride(),
        k_cache.data_ptr(), *k_cache.stride(), v_cache.data_ptr(), *v_cache.stride(),
        k_scale.data_ptr(), *k_scale.stride(), v_scale.data_ptr(), *v_scale.stride(),
        bm.data_ptr(), sm.data_ptr(), T, H, D, N, B, itag, tag, fmt, status_ptr(dev)))
    if rc:
        _capi.check(rc, what)
    after_launch(dev)


def load_kv_cache_quantized(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                            v_scale: torch.Tensor, block_mapping: torch.Tensor,
                            slot_mapping: torch.Tensor,
                            dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """The K and V rows at ``(block_mapping[t], slot_mapping[t])``, dequantised to
    ``dtype``: two new (num_kv_heads, num_tokens, head_dim) tensors, the shape the
    stores take, over token-major memory, so that ``k.transpose(0, 1)`` is the
    contiguous (T, H, D) that :func:`~tinyserver_b200.flash_attn_varlen_func`
    takes.  A place outside the cache reads as zeros and is reported through
    :func:`tinyserver_b200.check_errors`."""
    what = "load_kv_cache_quantized"
    fmt = check_quantized_cache(what, k_cache, v_cache, k_scale, v_scale)
    bm, sm, itag = _mappings(what, block_mapping, slot_mapping)
    N, H, B, D = k_cache.shape
    T = bm.numel()
    dev = device_index(what, k_cache, v_cache, k_scale, v_scale, bm, sm)
    k = torch.empty_strided((H, T, D), (D, H * D, 1), dtype=dtype, device=k_cache.device)
    v = torch.empty_strided((H, T, D), (D, H * D, 1), dtype=dtype, device=k_cache.device)
    tag = dtype_tag(k, what)
    rc = launch(dev, _capi.lib().qf_kv_load_quantized, _capi.KvQuantizedArgs.pack(
        k.data_ptr(), D, H * D, 1, v.data_ptr(), D, H * D, 1,
        k_cache.data_ptr(), *k_cache.stride(), v_cache.data_ptr(), *v_cache.stride(),
        k_scale.data_ptr(), *k_scale.stride(), v_scale.data_ptr(), *v_scale.stride(),
        bm.data_ptr(), sm.data_ptr(), T, H, D, N, B, itag, tag, fmt, status_ptr(dev)))
    if rc:
        _capi.check(rc, what)
    after_launch(dev)
    return k, v


def paged_attention_quantized(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                              k_scale: torch.Tensor, v_scale: torch.Tensor,
                              block_tables: torch.Tensor, block_size: int,
                              seq_lens: torch.Tensor, *, softmax_scale: float | None = None,
                              workspace: torch.Tensor | None = None,
                              split: bool = True) -> torch.Tensor:
    """:func:`~tinyserver_b200.paged_attention_forward` over a quantised cache:
    one query token per sequence, ``query`` (num_seqs, Hq, D), against the
    first ``seq_lens[s]`` cached tokens of sequence s, their rows dequantised as
    they are read.  Any Hq / Hkv; a sequence of no tokens gives zeros.  Scales are
    what the store writes, not negative; one of V below 2**-126 reads as 0."""
    what = "paged_attention_quantized"
    if query.dim() == 3 and (seq_lens.dim() != 1 or seq_lens.numel() != query.shape[0]):
        raise ValueError(f"{what}: seq_lens must be (num_seqs,) for {query.shape[0]} queries, got "
                         f"{tuple(seq_lens.shape)}")
    if k_scale is None or v_scale is None:
        raise ValueError(f"{what}: k_scale and v_scale are needed (paged_attention_forward reads a "
                         "cache of the query's dtype)")
    return attend(what, query, k_cache, v_cache, k_scale, v_scale, block_tables, block_size,
                  seq_lens, None, None, 1, softmax_scale, workspace, split)
