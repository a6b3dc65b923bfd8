"""Attention for a tree of drafted tokens over the paged KV cache (CUDA only, no
fallback), and the tree's visibility mask.

Speculative decoding drafts several continuations of a sequence at once, a tree
whose nodes share prefixes, and verifies them in one forward: every node
attends to the whole context and to its own ancestors among the drafted
tokens.  The steps of one layer of such a forward, with this library:

1. :func:`build_tree_mask` once per forward, from the nodes' parents;
2. ``positions = context_lens[seq] + depths``; the nodes' K/V stored at slots
   ``context_lens[seq] + node`` by :func:`~tinyserver_b200.qk_norm_rope_store`,
   :func:`~tinyserver_b200.store_kv_cache_batched` or
   :func:`~tinyserver_b200.store_kv_cache_quantized`;
3. :func:`paged_tree_attention` over the pages.

The reference has no counterpart: it decodes one token per sequence and step.
"""

from __future__ import annotations

import functools
import math

import torch

from .. import _capi
from .._runtime import (after_launch, device_index, dtype_tag, index_tag, launch, status_ptr)

__all__ = ["build_tree_mask", "paged_tree_attention", "paged_tree_attention_workspace_bytes"]

CACHE_FORMATS = {torch.float8_e4m3fn: _capi.QF_CACHE_E4M3, torch.int8: _capi.QF_CACHE_INT8}


def _narrow(t: torch.Tensor) -> torch.Tensor:
    """``t`` (int32 or int64) as int32.  What int32 does not hold becomes its least or
    largest number, which the kernels cut and report, not another one in range."""
    return t if t.dtype == torch.int32 else t.clamp(-(1 << 31), (1 << 31) - 1).to(torch.int32)


def _int32(t: torch.Tensor) -> torch.Tensor:
    """:func:`_narrow`, contiguous."""
    t = _narrow(t)
    return t if t.is_contiguous() else t.contiguous()


def build_tree_mask(parents: torch.Tensor, cu_seqlens: torch.Tensor,
                    max_tree: int) -> tuple[torch.Tensor, torch.Tensor]:
    """(tree_mask, depths) of packed trees: sequence s owns nodes
    ``cu_seqlens[s] .. cu_seqlens[s + 1] - 1``; ``parents[t]`` (int32 or int64)
    is the index within the sequence of an earlier node, or -1 for a child of
    the last context token.

    ``tree_mask`` (num_nodes, ceil(max_tree / 64)) int64: bit ``i % 64`` of word
    ``i // 64`` of row t is set iff node i of its sequence is t itself or one of
    its ancestors.  ``depths`` (num_nodes,) int32: the number of ancestors, so a
    node's position is its sequence's context length plus its depth.

    A parent that is not an earlier node is read as -1, and a node past
    ``max_tree`` gets an empty row; both are reported through
    :func:`tinyserver_b200.check_errors`.  Nodes that no sequence owns (a padded
    batch) get empty rows too."""
    if parents.dim() != 1 or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
        raise ValueError("parents must be (num_nodes,) and cu_seqlens (num_seqs + 1,), got "
                         f"{tuple(parents.shape)} and {tuple(cu_seqlens.shape)}")
    max_tree = int(max_tree)
    if max_tree < 1:
        raise ValueError(f"max_tree must be >= 1, got {max_tree}")
    itag = index_tag(parents, "build_tree_mask parents")
    index_tag(cu_seqlens, "build_tree_mask cu_seqlens")
    dev = device_index("build_tree_mask", parents, cu_seqlens)
    if not parents.is_contiguous():
        parents = parents.contiguous()
    cu = _int32(cu_seqlens)
    n, words, seqs = parents.numel(), (max_tree + 63) // 64, cu.numel() - 1
    if n and seqs < 1:
        raise ValueError(f"build_tree_mask: {n} nodes but no sequence")
    # (empty_strided: a microsecond less a call than empty)
    mask = torch.empty_strided((n, words), (words, 1), dtype=torch.int64, device=parents.device)
    depths = torch.empty_strided((n,), (1,), dtype=torch.int32, device=parents.device)
    rc = launch(dev, _capi.lib().qf_build_tree_mask, _capi.TreeMaskArgs.pack(
        parents.data_ptr(), cu.data_ptr(), seqs, n, max_tree, words, mask.data_ptr(),
        depths.data_ptr(), itag, status_ptr(dev)))
    if rc:
        _capi.check(rc, "build_tree_mask")
    after_launch(dev)
    return mask, depths


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(dev: int, num_tokens: int, num_seqs: int, max_tree: int, num_q_heads: int,
                     num_kv_heads: int, head_dim: int, block_size: int, max_blocks_per_seq: int,
                     tag: int, fmt: int, decode: bool) -> int:
    args = _capi.PagedTreeAttentionArgs.named(
        cu_seqlens_q=0 if decode else 1,  # (whether there is one is all that is read)
        num_tokens=num_tokens, num_seqs=num_seqs, max_tree=max_tree, num_q_heads=num_q_heads,
        num_kv_heads=num_kv_heads, head_dim=head_dim, block_size=block_size,
        max_blocks_per_seq=max_blocks_per_seq, dtype=tag, cache_format=fmt)
    with torch.cuda.device(dev):  # (its number of SMs counts; dev < 0: no GPU, no switch)
        return int(_capi.lib().qf_paged_tree_attention_workspace_bytes(args))


def paged_tree_attention_workspace_bytes(num_tokens: int, num_seqs: int, max_tree: int,
                                         num_q_heads: int, num_kv_heads: int, head_dim: int,
                                         block_size: int, max_blocks_per_seq: int,
                                         dtype: torch.dtype) -> int:
    """Bytes of fp32 scratch that let :func:`paged_tree_attention` split long
    sequences over several CTAs (0 when nothing needs splitting), for a cache of any
    format; a decode call (:func:`~tinyserver_b200.paged_attention_quantized`) counts
    as max_tree 1.  It depends on the GPU: ask with the call's device current."""
    tag = dtype_tag(torch.empty(0, dtype=dtype), "paged_tree_attention_workspace_bytes")
    dev = torch.cuda.current_device() if torch.cuda.is_available() else -1
    sizes = (dev, num_tokens, num_seqs, max_tree, num_q_heads, num_kv_heads, head_dim, block_size,
             max_blocks_per_seq, tag)
    return max(_workspace_bytes(*sizes, fmt, decode) for decode in {False, max_tree == 1}
               for fmt in (_capi.QF_CACHE_PLAIN, *CACHE_FORMATS.values()))


def check_quantized_cache(what: str, k_cache: torch.Tensor, v_cache: torch.Tensor,
                          k_scale: torch.Tensor, v_scale: torch.Tensor) -> int:
    """The cache format of a quantised cache; ValueError unless codes and scales fit."""
    shape, dtype = k_cache.shape, k_cache.dtype
    fmt, rows = CACHE_FORMATS.get(dtype), shape[:3]
    if (fmt is not None and len(shape) == 4 and v_cache.shape == shape and v_cache.dtype == dtype
            and k_scale.shape == rows and v_scale.shape == rows
            and k_scale.dtype is torch.float32 and v_scale.dtype is torch.float32):
        return fmt
    if len(shape) != 4 or v_cache.shape != shape:
        raise ValueError(f"{what}: k_cache/v_cache must be (num_blocks, num_kv_heads, block_size, "
                         f"head_dim), got {tuple(k_cache.shape)} and {tuple(v_cache.shape)}")
    if fmt is None or v_cache.dtype != dtype:
        raise ValueError(f"{what}: a quantised cache holds float8_e4m3fn or int8 rows, got "
                         f"{k_cache.dtype} and {v_cache.dtype}")
    if k_scale.shape != rows or v_scale.shape != rows:
        raise ValueError(f"{what}: k_scale/v_scale must be (num_blocks, num_kv_heads, block_size) "
                         f"= {tuple(rows)}, got {tuple(k_scale.shape)} and "
                         f"{tuple(v_scale.shape)}")
    raise ValueError(f"{what}: scales must be float32, got {k_scale.dtype} and {v_scale.dtype}")


def attend(what: str, query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
           k_scale: torch.Tensor | None, v_scale: torch.Tensor | None,
           block_tables: torch.Tensor, block_size: int, lens: torch.Tensor,
           cu_seqlens: torch.Tensor | None, tree_mask: torch.Tensor | None, max_tree: int,
           softmax_scale: float | None, workspace: torch.Tensor | None,
           split: bool) -> torch.Tensor:
    """The call both public forms make (``cu_seqlens`` None: decode)."""
    if query.dim() != 3:
        raise ValueError(f"{what}: query must be a 3D tensor, but got shape {tuple(query.shape)}")
    if workspace is not None and not workspace.is_contiguous():
        raise ValueError(f"{what}: workspace must be contiguous, got strides {workspace.stride()}")
    if (k_scale is None) != (v_scale is None):
        raise ValueError(f"{what}: k_scale and v_scale come together")
    if k_scale is not None:
        fmt = check_quantized_cache(what, k_cache, v_cache, k_scale, v_scale)
        if k_scale.stride() != v_scale.stride():
            raise ValueError(f"{what}: k_scale and v_scale strides differ")
    else:
        fmt = _capi.QF_CACHE_PLAIN
        if k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
            raise ValueError(f"{what}: k_cache/v_cache must be (num_blocks, num_kv_heads, "
                             f"block_size, head_dim), got {tuple(k_cache.shape)} and "
                             f"{tuple(v_cache.shape)}")
        if not (query.dtype == k_cache.dtype == v_cache.dtype):
            raise ValueError(f"{what}: query dtype {query.dtype} != cache dtypes {k_cache.dtype}, "
                             f"{v_cache.dtype} (a quantised cache needs k_scale and v_scale)")
    strides = k_cache.stride()
    if strides != v_cache.stride():
        raise ValueError(f"{what}: k_cache and v_cache strides differ")
    T, Hq, D = query.shape
    N, Hkv, B, Dc = k_cache.shape
    if Dc != D or B != block_size:
        raise ValueError(f"{what}: cache geometry {tuple(k_cache.shape)} does not match head_dim "
                         f"{D} / block_size {block_size}")
    if Hkv == 0 or Hq % Hkv:
        raise ValueError(f"{what}: num_heads {Hq} is not a multiple of num_kv_heads {Hkv}")
    S = lens.numel()
    if lens.dim() != 1 or block_tables.dim() != 2 or block_tables.shape[0] != S:
        raise ValueError(f"{what}: block_tables must be (num_seqs, max_blocks) and the lengths "
                         f"(num_seqs,), got {tuple(block_tables.shape)} and {tuple(lens.shape)}")
    tag = dtype_tag(query, what)
    for index in (block_tables, lens, cu_seqlens):
        if index is not None:
            index_tag(index, what)
    dev = device_index(what, query, k_cache, v_cache, block_tables, lens, k_scale, v_scale,
                       cu_seqlens, tree_mask, workspace)
    q = query
    es = q.element_size()
    sq = q.stride()
    if sq[2] != 1 or (sq[0] * es) % 16 or (sq[1] * es) % 16 or q.data_ptr() % 16:
        q = torch.empty(q.shape, dtype=q.dtype, device=q.device).copy_(q)  # the kernels' alignment
        sq = q.stride()
    bt = _narrow(block_tables)
    max_blocks = bt.shape[1]
    if max_blocks > 1 and bt.stride(1) != 1:
        bt = bt.contiguous()
    lens = _int32(lens)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    cu = mask = None
    words = 0
    if cu_seqlens is not None:
        cu = _int32(cu_seqlens)
        mask = tree_mask if tree_mask.is_contiguous() else tree_mask.contiguous()
        words = mask.shape[1]
    space = 0
    if split:
        if workspace is None:
            space = _workspace_bytes(dev, T, S, max_tree, Hq, Hkv, D, B, max_blocks, tag, fmt, cu is None)
            if space:
                workspace = torch.empty_strided((space // 4,), (1,), dtype=torch.float32,
                                                device=q.device)
        else:
            space = workspace.numel() * workspace.element_size()
    scaled = k_scale is not None
    rc = launch(dev, _capi.lib().qf_paged_tree_attention, _capi.PagedTreeAttentionArgs.pack(
        q.data_ptr(), sq[0], sq[1],
        k_cache.data_ptr(), v_cache.data_ptr(), *strides,
        k_scale.data_ptr() if scaled else 0, v_scale.data_ptr() if scaled else 0,
        *(k_scale.stride() if scaled else (0, 0, 0)),
        N, B,
        bt.data_ptr(), bt.stride(0), max_blocks,
        lens.data_ptr(), 0 if cu is None else cu.data_ptr(),
        0 if mask is None else mask.data_ptr(), words,
        S, T, max_tree, Hq, Hkv, D,
        1.0 / math.sqrt(D) if softmax_scale is None else float(softmax_scale),
        out.data_ptr(), Hq * D, D,
        workspace.data_ptr() if space else 0, space,
        tag, fmt,
        status_ptr(dev)))
    if rc:
        _capi.check(rc, what)
    after_launch(dev)
    return out


def paged_tree_attention(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                         block_tables: torch.Tensor, block_size: int, context_lens: torch.Tensor,
                         cu_seqlens: torch.Tensor, tree_mask: torch.Tensor, max_tree: int, *,
                         k_scale: torch.Tensor | None = None,
                         v_scale: torch.Tensor | None = None,
                         softmax_scale: float | None = None,
                         workspace: torch.Tensor | None = None,
                         split: bool = True) -> torch.Tensor:
    """Attention of packed trees of drafted tokens: ``query`` (T, Hq, D) holds
    sequence s's nodes at rows ``cu_seqlens[s] .. cu_seqlens[s + 1] - 1``; its
    ``context_lens[s]`` context tokens and, behind them, the nodes' own K/V rows
    are in the cache, through ``block_tables[s]``.  Node t sees every context
    key and the node keys whose bits its row of ``tree_mask`` has
    (:func:`build_tree_mask`, or any other mask of that layout):

        out[t, h] = softmax(query[t, h] @ K.T * softmax_scale, seen keys) @ V

    Returns a new (T, Hq, D) tensor; a node that sees no key, and a row that no
    sequence owns, is zero.  What an unseen key's K and V hold never matters.

    ``max_tree`` bounds the nodes of any one sequence.  ``k_scale``/``v_scale``
    (num_blocks, num_kv_heads, block_size) read a quantised cache
    (:func:`~tinyserver_b200.store_kv_cache_quantized`).  ``softmax_scale``
    defaults to 1/sqrt(D).  ``split`` lets long sequences spread over several
    CTAs through an fp32 workspace (allocated here unless ``workspace`` is
    given, :func:`paged_tree_attention_workspace_bytes`).

    Fewer keys than claimed (context + nodes beyond the block table's row,
    blocks outside the cache) are left out and reported through
    :func:`tinyserver_b200.check_errors`."""
    what = "paged_tree_attention"
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() != context_lens.numel() + 1:
        raise ValueError(f"{what}: cu_seqlens must be (num_seqs + 1,) with context_lens "
                         f"(num_seqs,), got {tuple(cu_seqlens.shape)} and "
                         f"{tuple(context_lens.shape)}")
    max_tree = int(max_tree)
    if max_tree < 1:
        raise ValueError(f"{what}: max_tree must be >= 1, got {max_tree}")
    if tree_mask.dim() != 2 or tree_mask.dtype != torch.int64 or \
            tree_mask.shape[0] != query.shape[0] or tree_mask.shape[1] * 64 < max_tree:
        raise ValueError(f"{what}: tree_mask must be int64 (num_tokens, at least "
                         f"{(max_tree + 63) // 64}) for {query.shape[0]} tokens, got "
                         f"{tree_mask.dtype} {tuple(tree_mask.shape)}")
    if context_lens.numel() == 0 and query.shape[0]:
        raise ValueError(f"{what}: {query.shape[0]} tokens but no sequence")
    return attend(what, query, k_cache, v_cache, k_scale, v_scale, block_tables, block_size,
                  context_lens, cu_seqlens, tree_mask, max_tree, softmax_scale, workspace, split)
