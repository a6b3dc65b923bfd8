"""Attention for drafted token trees on the GPU against its definition in 64 bits, within bounds
counted from its roundings (tree_reference); the visibility mask bit for bit."""

import pytest
import torch

import tinyserver_b200 as tsb
from tests import tree_reference as ref
from tests.test_gpu_quantized import DTYPES, paged

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3 = torch.float8_e4m3fn


def _cu(sizes):
    return torch.tensor([0] + sizes).cumsum(0).int().to(DEV)


@pytest.mark.parametrize("sizes,max_tree", [([1], 1), ([7, 0, 64], 64), ([65, 1, 127, 128], 128), ([300], 300),
                                            ([5, 5], 200)])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_mask_against_walks(sizes, max_tree, index):
    g = torch.Generator().manual_seed(sum(sizes))
    parents = ref.random_parents(sizes, g)
    mask, depths = tsb.build_tree_mask(parents.to(DEV, index), _cu(sizes), max_tree)
    tsb.check_errors()
    want = ref.mask_of(parents, sizes, max_tree)
    assert torch.equal(mask.cpu(), want[0]) and torch.equal(depths.cpu(), want[1])


def test_mask_of_bad_parents_large_trees_and_padding():
    """A parent that is no earlier node (itself, a later one, below -1) reads as a root; nodes past max_tree and
    nodes outside every sequence get empty rows."""
    parents = torch.tensor([-1, 1, 5, -7, 2, 3, 0, 0], device=DEV)
    mask, depths = tsb.build_tree_mask(parents, torch.tensor([1, 7], device=DEV), 8)
    with pytest.raises(IndexError, match="earlier node"):
        tsb.check_errors()
    # nodes of the sequence: parents 1, 5, -7, 2, 3, 0
    assert mask[:, 0].tolist() == [0, 1, 2, 4, 12, 28, 33, 0]
    assert depths.tolist() == [0, 0, 0, 0, 1, 2, 1, 0]
    chain = torch.arange(-1, 5, device=DEV, dtype=torch.int32)
    mask, depths = tsb.build_tree_mask(chain, _cu([6]), 4)
    with pytest.raises(IndexError, match="max_tree"):
        tsb.check_errors()
    assert mask[:, 0].tolist() == [1, 3, 7, 15, 0, 0] and depths.tolist() == [0, 1, 2, 3, 0, 0]


def _case(sizes, contexts, hq, hkv, D, block, dtype, fmt, seed, mask=None):
    k, v, ks, vs, bt = paged([c + n for c, n in zip(contexts, sizes)], hkv, D, block, fmt, dtype, seed)
    g = torch.Generator().manual_seed(seed + 1)
    if mask is None:
        mask = ref.mask_of(ref.random_parents(sizes, g), sizes, max(sizes + [1]))[0]
    q = torch.randn(sum(sizes), hq, D, generator=g).to(dtype).to(DEV)
    return q, k, v, ks, vs, bt, mask.to(DEV)


def _run(q, k, v, ks, vs, bt, mask, block, contexts, sizes, max_tree=None, **kw):
    got = tsb.paged_tree_attention(q, k, v, bt, block, torch.tensor(contexts, dtype=torch.int32, device=DEV),
                                   _cu(sizes), mask, max_tree or max(sizes + [1]), k_scale=ks, v_scale=vs, **kw)
    return got


def _check(sizes, contexts, hq, hkv, D, block, dtype, fmt, seed, mask=None, **kw):
    q, k, v, ks, vs, bt, mask = _case(sizes, contexts, hq, hkv, D, block, dtype, fmt, seed, mask)
    out, bound = ref.attention(q, k, v, bt, block, contexts, sizes, mask, ks, vs,
                               p_type=torch.float16 if fmt else None)
    for split in (True, False):
        got = _run(q, k, v, ks, vs, bt, mask, block, contexts, sizes, split=split, **kw)
        tsb.check_errors()
        ref.assert_within(got, out, bound, f"split={split}")


SIZES = [1, 0, 3, 9, 17, 64, 70]
CONTEXTS = [0, 40, 1, 127, 128, 700, 1290]


@pytest.mark.parametrize("fmt", [None, *ref.FORMATS])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,D,block", [(8, 8, 128, 16), (6, 2, 64, 8), (32, 8, 128, 16), (8, 1, 256, 24),
                                            (20, 1, 128, 256), (4, 1, 128, 5)])
def test_trees_against_64_bits(fmt, dtype, hq, hkv, D, block):
    _check(SIZES, CONTEXTS, hq, hkv, D, block, dtype, fmt, seed=hq + D)


@pytest.mark.parametrize("fmt", [None, E4M3])
@pytest.mark.parametrize("n", [1, 2, 4, 5, 16, 31, 33, 64, 128, 129])
def test_tree_sizes(fmt, n):
    """Row counts around every tile border of the kernels, at a context that ends inside a tile."""
    _check([n], [333], 16, 4, 128, 16, torch.bfloat16, fmt, seed=n)
    _check([n, 1], [0, 5], 16, 4, 128, 16, torch.float16, fmt, seed=n + 1)


@pytest.mark.parametrize("dtype", DTYPES)
def test_any_mask_and_rows_that_see_nothing(dtype):
    """Random masks (not a tree's), with bits past the tree set; a query that sees none of its nodes and has no
    context is zero."""
    sizes, contexts = [40, 12], [0, 77]
    g = torch.Generator().manual_seed(3)
    mask = torch.randint(-2 ** 62, 2 ** 62, (52, 2), generator=g)
    mask[3] = 0
    mask[5, 0] = -1 << 40  # bits past the tree only
    mask[45] = 0
    for hq, hkv in ((2, 2), (16, 2)):
        _check(sizes, contexts, hq, hkv, 128, 16, dtype, None, 5, mask)
        q, k, v, ks, vs, bt, m = _case(sizes, contexts, hq, hkv, 128, 16, dtype, None, 5, mask)
        got = _run(q, k, v, ks, vs, bt, m, 16, contexts, sizes)
        assert not got[3].any() and not got[5].any() and got[45].any()


@pytest.mark.parametrize("fmt", [None, E4M3])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,hq", [(3, 2), (9, 8), (40, 8)])
def test_unseen_keys_never_matter(fmt, dtype, n, hq):
    """NaN and infinities in the K and V of a drafted node reach its descendants alone; past the last key they
    reach nobody."""
    sizes, contexts = [n, n], [50, 0]
    parents = torch.tensor(([-1, 0, 0] + list(range(-1, n - 4)))[:n] * 2, dtype=torch.int32)
    mask = ref.mask_of(parents, sizes, n)[0]
    q, k, v, ks, vs, bt, mask = _case(sizes, contexts, hq, 2, 128, 16, dtype, fmt, 7, mask)
    for s in (0, 1):
        for node, (kval, vval) in ((1, (1.0, float("nan"))), (2, (float("inf"), 1.0))):
            j = contexts[s] + node
            at = int(bt[s, j // 16]), 0, j % 16
            if fmt is None:
                v[at][..., 5] = vval
                k[at][..., 7] = kval
            else:
                v.view(torch.uint8)[at][..., 5] = 0x7f if vval != vval else 0x10
                if kval != 1.0:
                    ks[at] = float("nan")
        j = contexts[s] + n
        last = int(bt[s, j // 16]) if j % 16 else None
        if last is not None:
            (k if fmt is None else k.view(torch.uint8))[last, :, j % 16:] = float("nan") if fmt is None else 0x7f
            (v if fmt is None else v.view(torch.uint8))[last, :, j % 16:] = float("nan") if fmt is None else 0x7f
            if fmt is not None:
                ks[last, :, j % 16:] = vs[last, :, j % 16:] = float("nan")
    got = _run(q, k, v, ks, vs, bt, mask, 16, contexts, sizes)
    tsb.check_errors()
    sees = lambda t, node: bool((int(mask[t, 0]) >> node) & 1)  # noqa: E731
    clean_k, clean_v, clean_ks = k.clone(), v.clone(), None if ks is None else ks.clone()
    for s in (0, 1):
        for node in (1, 2):
            j = contexts[s] + node
            at = int(bt[s, j // 16]), 0, j % 16
            (clean_k if fmt is None else clean_k.view(torch.uint8))[at] = 0
            (clean_v if fmt is None else clean_v.view(torch.uint8))[at] = 0
            if fmt is not None:
                clean_ks[at] = 1.0
    out, bound = ref.attention(q, clean_k, clean_v, bt, 16, contexts, sizes, mask, clean_ks, vs,
                               p_type=torch.float16 if fmt else None)
    without = ref.attention(q, clean_k, clean_v, bt, 16, contexts, sizes, mask & ~4, clean_ks, vs,
                            p_type=torch.float16 if fmt else None)
    for t in range(2 * n):
        heads = slice(hq // 2, hq)  # kv head 1 is clean throughout
        ref.assert_within(got[t, heads], out[t, heads], bound[t, heads], f"row {t}, other head")
        if sees(t, 2):
            # K = +inf in dim 7: a score of +inf (NaN after the softmax's inf - inf) where the query is positive
            # there, of -inf (a weight of 0) where it is negative; a NaN scale makes NaN of both
            up = q[t, :hq // 2, 7] > 0 if fmt is None else torch.ones(hq // 2, dtype=torch.bool, device=DEV)
            assert torch.equal(torch.isnan(got[t, :hq // 2]).all(-1), up), t
            ref.assert_within(got[t, :hq // 2][~up], without[0][t, :hq // 2][~up], without[1][t, :hq // 2][~up])
        elif sees(t, 1):
            assert torch.isnan(got[t, :hq // 2, 5]).all(), t
            assert int(torch.isnan(got[t, :hq // 2]).sum()) == hq // 2, t
        else:
            ref.assert_within(got[t, :hq // 2], out[t, :hq // 2], bound[t, :hq // 2], f"row {t}")


@pytest.mark.parametrize("hq", [2, 32])
def test_rows_outside_every_tree_are_zero(hq):
    """A padded batch: rows before the first sequence, behind the last, and past max_tree."""
    sizes, contexts = [4, 3], [30, 200]
    q, k, v, ks, vs, bt, mask = _case(sizes, contexts, hq, 2, 128, 16, torch.bfloat16, None, 4)
    want = _run(q, k, v, ks, vs, bt, mask, 16, contexts, sizes)
    pad = torch.randn(15, hq, 128, device=DEV).to(torch.bfloat16)
    pad[5:12] = q
    pmask = torch.full((15, 1), -1, dtype=torch.int64, device=DEV)
    pmask[5:12] = mask
    cu = torch.tensor([5, 9, 12], dtype=torch.int32, device=DEV)
    lens = torch.tensor(contexts, device=DEV)
    for fill in range(2):  # whatever the allocator hands out
        junk = torch.full((15, hq, 128), float("nan"), device=DEV, dtype=torch.bfloat16)
        del junk
        got = tsb.paged_tree_attention(pad, k, v, bt, 16, lens, cu, pmask, 4)
        tsb.check_errors()
        assert torch.equal(got[5:12], want) and not got[:5].any() and not got[12:].any()
    got = tsb.paged_tree_attention(pad, k, v, bt, 16, lens, cu, pmask, 3)
    with pytest.raises(IndexError, match="max_tree"):
        tsb.check_errors()
    assert not got[8].any() and got[7].any()
    got = tsb.paged_tree_attention(pad, k, v, bt, 16, lens, torch.tensor([5, 9, 400], device=DEV), pmask, 64)
    with pytest.raises(IndexError, match="block table"):
        tsb.check_errors()
    assert torch.isfinite(got).all()


def test_a_chain_is_a_sequence_of_decode_steps():
    """A chain of drafts (each node sees all before it) gives what one-token decode gives at each length."""
    n, ctx = 6, 150
    parents = torch.arange(-1, n - 1, device=DEV, dtype=torch.int32)
    mask, depths = tsb.build_tree_mask(parents, _cu([n]), n)
    assert depths.tolist() == list(range(n))
    q, k, v, ks, vs, bt, _ = _case([n], [ctx], 32, 8, 128, 16, torch.bfloat16, None, 6)
    got = _run(q, k, v, ks, vs, bt, mask, 16, [ctx], [n])
    lens = torch.arange(ctx + 1, ctx + n + 1, device=DEV)
    steps = tsb.paged_attention_forward(q, k, v, bt.expand(n, -1).contiguous(), 16, lens)
    tsb.check_errors()
    out, bound = ref.attention(q, k, v, bt, 16, [ctx], [n], mask)
    ref.assert_within(got, out, bound)
    ref.assert_within(steps, out, bound)


def test_a_verification_step_over_a_quantised_cache():
    """The operators together, as a server calls them: mask and depths from the parents, positions and slots
    from them, q/k norm + RoPE, the rows quantised into their pages, attention of the trees."""
    sizes, contexts, Hq, Hkv, D, B = [7, 5], [90, 33], 32, 8, 128, 16
    T = sum(sizes)
    q, k, v, ks, vs, bt, _ = _case(sizes, contexts, Hq, Hkv, D, B, torch.bfloat16, E4M3, 11)
    g = torch.Generator().manual_seed(12)
    parents = ref.random_parents(sizes, g).to(DEV)
    cu = _cu(sizes)
    mask, depths = tsb.build_tree_mask(parents, cu, 8)
    of = torch.repeat_interleave(torch.arange(2, device=DEV), torch.tensor(sizes, device=DEV))
    lens = torch.tensor(contexts, device=DEV)
    slots = lens[of] + torch.arange(T, device=DEV) - cu[:-1].long()[of]
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g).to(torch.bfloat16).to(DEV)
    qp, kp, vp = (x.unflatten(1, (-1, D)) for x in qkv.split([Hq * D, Hkv * D, Hkv * D], 1))
    w = torch.ones(D, dtype=torch.bfloat16, device=DEV)
    cos, sin = tsb.rope_cos_sin(lens[of] + depths, tsb.rope_inv_freq(D, 1e6, DEV), D, torch.bfloat16)
    qr, kr = tsb.qk_norm_rope_store(qp, kp, vp, w, w, 1e-6, cos, sin)
    bm, sm = tsb.build_slot_mapping(cu, slots, bt, B)
    tsb.store_kv_cache_quantized(kr.transpose(0, 1), vp.transpose(0, 1), k, v, ks, vs, bm, sm)
    got = tsb.paged_tree_attention(qr, k, v, bt, B, lens, cu, mask, 8, k_scale=ks, v_scale=vs)
    tsb.check_errors()
    out, bound = ref.attention(qr, k, v, bt, B, contexts, sizes, mask, ks, vs)
    ref.assert_within(got, out, bound)


def test_bad_blocks_and_short_tables_are_cut_and_flagged():
    for dtype, hq in ((torch.bfloat16, 2), (torch.bfloat16, 32), (torch.float32, 4)):
        sizes, contexts = [6, 6], [100, 40]
        q, k, v, ks, vs, bt, mask = _case(sizes, contexts, hq, 2, 128, 16, dtype, None, 4)
        bad = bt.clone()
        bad[0, 2], bad[1, 0] = k.shape[0], -5
        got = _run(q, k, v, ks, vs, bad, mask, 16, contexts, sizes)
        with pytest.raises(IndexError, match="block index"):
            tsb.check_errors()
        assert torch.isfinite(got).all()
        got = _run(q, k, v, ks, vs, bt[:, :3], mask, 16, contexts, sizes)
        with pytest.raises(IndexError, match="block table"):
            tsb.check_errors()
        assert torch.isfinite(got).all()
        none = torch.zeros(2, 0, dtype=torch.int32, device=DEV)
        got = _run(q, k, v, ks, vs, none, mask, 16, contexts, sizes)
        with pytest.raises(IndexError, match="block table"):
            tsb.check_errors()
        assert not got.any()


def test_strided_inputs_scale_and_layer_views():
    sizes, contexts = [20, 3], [60, 10]
    q, k, v, ks, vs, bt, mask = _case(sizes, contexts, 16, 2, 128, 16, torch.bfloat16, None, 4)
    want = _run(q, k, v, ks, vs, bt, mask, 16, contexts, sizes, softmax_scale=0.3)
    out, bound = ref.attention(q, k, v, bt, 16, contexts, sizes, mask, scale=0.3)
    ref.assert_within(want, out, bound)
    pool = torch.zeros(2, 3, *k.shape, dtype=k.dtype, device=DEV)
    pool[0, 1], pool[1, 1] = k, v
    wide = torch.zeros(23, 16, 200, dtype=q.dtype, device=DEV)
    for at in (0, 8, 3):  # 3: rows that start off a 16-byte boundary are copied
        wide[:, :, at:at + 128] = q
        view = wide[:, :, at:at + 128]
        wide_bt = torch.zeros(2, 2 * bt.shape[1], dtype=torch.int32, device=DEV)
        wide_bt[:, ::2] = bt
        got = _run(view, pool[0, 1], pool[1, 1], None, None, wide_bt[:, ::2], mask, 16, contexts, sizes,
                   softmax_scale=0.3)
        assert torch.equal(got, want)


@pytest.mark.parametrize("fmt", ref.FORMATS)
@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
@pytest.mark.parametrize("n,hq", [(8, 2), (12, 16), (40, 16)])
def test_scales_over_eight_decades_and_none(fmt, dtype, n, hq):
    """V's row scales from 1e-6 to 1e2 beside each other (none brings them all near 1), whole pages of one
    size, and scales of 0 (rows never written, which stand for zeros but have their weight)."""
    sizes, contexts = [n, 3], [1500, 130]
    q, k, v, ks, vs, bt, mask = _case(sizes, contexts, hq, 2, 128, 16, dtype, fmt, 21)
    g = torch.Generator().manual_seed(3)
    vs *= (10.0 ** torch.randint(-4, 5, vs.shape, generator=g)).to(DEV)
    vs[bt[0, 8:24].long()] = 0.02
    ks[bt[0, 40].long()] = 0.0
    vs[bt[0, 40].long()] = 0.0
    out, bound = ref.attention(q, k, v, bt, 16, contexts, sizes, mask, ks, vs, p_type=torch.float16)
    for split in (True, False):
        got = _run(q, k, v, ks, vs, bt, mask, 16, contexts, sizes, split=split)
        tsb.check_errors()
        ref.assert_within(got, out, bound, f"split={split}")


@pytest.mark.parametrize("fmt", ref.FORMATS)
@pytest.mark.parametrize("dtype", (torch.float32, torch.float16, torch.bfloat16))
@pytest.mark.parametrize("n,hq", [(1, 2), (8, 4), (40, 8)])
def test_rows_never_written_ahead_of_the_others(fmt, dtype, n, hq):
    """Keys whose codes and scales are 0 score 0, have that weight, and add nothing: 700 of them first, so that
    they alone set a maximum and a sum before any other key does, alone in a sequence, and all of it."""
    sizes, contexts = [n, 2, 1], [1500, 0, 520]
    q, k, v, ks, vs, bt, mask = _case(sizes, contexts, hq, 2, 128, 16, dtype, fmt, 12)
    for blocks in (bt[0, :44].long(), bt[2, :20].long()):
        for t in (k.view(torch.uint8), v.view(torch.uint8), ks, vs):
            t[blocks] = 0
    out, bound = ref.attention(q, k, v, bt, 16, contexts, sizes, mask, ks, vs,
                               p_type=torch.float16 if dtype != torch.float32 else None)
    for split in (True, False):
        ref.assert_within(_run(q, k, v, ks, vs, bt, mask, 16, contexts, sizes, split=split), out, bound, f"split={split}")


@pytest.mark.parametrize("dtype", (torch.float32, torch.float16, torch.bfloat16))
@pytest.mark.parametrize("scale", [-0.2, 0.0])
def test_negative_and_zero_softmax_scale(dtype, scale):
    """The definition holds for any scale: least scores first, and a plain mean of the seen values."""
    for hq, fmt in ((2, None), (20, None), (20, E4M3)):
        q, k, v, ks, vs, bt, mask = _case([9, 40], [300, 0], hq, 1, 128, 16, dtype, fmt, 8)
        out, bound = ref.attention(q, k, v, bt, 16, [300, 0], [9, 40], mask, ks, vs, scale=scale,
                                   p_type=torch.float16 if fmt else None)
        ref.assert_within(_run(q, k, v, ks, vs, bt, mask, 16, [300, 0], [9, 40], softmax_scale=scale), out, bound)


@pytest.mark.parametrize("hq,hkv", [(2, 2), (32, 2), (64, 2)])
def test_many_sequences_of_every_length(hq, hkv):
    """More sequences than a CTA has threads, empty ones among them: each CTA's stretch of the work begins and
    ends where it should; twice, with the same bits."""
    g = torch.Generator().manual_seed(5)
    n = 400
    sizes = torch.randint(0, 6, (n,), generator=g).tolist()
    contexts = [int(x) if i % 7 else 0 for i, x in enumerate(torch.randint(0, 300, (n,), generator=g))]
    contexts[77], contexts[399] = 5000, 2222
    for fmt in (None, E4M3):
        q, k, v, ks, vs, bt, mask = _case(sizes, contexts, hq, hkv, 128, 16, torch.bfloat16, fmt, 3)
        out, bound = ref.attention(q, k, v, bt, 16, contexts, sizes, mask, ks, vs,
                                   p_type=torch.float16 if fmt else None)
        got = _run(q, k, v, ks, vs, bt, mask, 16, contexts, sizes)
        tsb.check_errors()
        ref.assert_within(got, out, bound)
        assert torch.equal(got, _run(q, k, v, ks, vs, bt, mask, 16, contexts, sizes))


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("hq,hkv", [(2, 2), (16, 2), (64, 2)])
def test_one_long_sequence_among_short_ones(dtype, hq, hkv):
    """The long one is shared by most CTAs, however few a sequence gets on average."""
    sizes = [1 + i % 3 for i in range(150)]
    contexts = [i % 20 for i in range(150)]
    contexts[40] = 30000
    for fmt in (None, E4M3):
        q, k, v, ks, vs, bt, mask = _case(sizes, contexts, hq, hkv, 128, 16, dtype, fmt, 6)
        out, bound = ref.attention(q, k, v, bt, 16, contexts, sizes, mask, ks, vs,
                                   p_type=torch.float16 if fmt and dtype != torch.float32 else None)
        ref.assert_within(_run(q, k, v, ks, vs, bt, mask, 16, contexts, sizes), out, bound)


@pytest.mark.parametrize("fmt,block", [(None, 16), (None, 12), (E4M3, 16), (E4M3, 6)])
def test_caches_past_32_bit_offsets(fmt, block):
    """Rows by TMA boxes and one by one, from blocks more than 2^31 elements behind the first."""
    sizes, contexts = [3, 40], [50, 200]
    q, k, v, ks, vs, bt, mask = _case(sizes, contexts, 8, 2, 128, block, torch.bfloat16, fmt, 8)
    first = (1 << 31) // (2 * block * 128) + 1

    def far(t):
        if t is None:
            return None
        big = torch.empty((first + t.shape[0], *t.shape[1:]), dtype=t.dtype, device=DEV)
        big[first:] = t
        return big
    out, bound = ref.attention(q, k, v, bt, block, contexts, sizes, mask, ks, vs,
                               p_type=torch.float16 if fmt else None)
    got = _run(q, far(k), far(v), far(ks), far(vs), bt + first, mask, block, contexts, sizes)
    tsb.check_errors()
    ref.assert_within(got, out, bound)


def test_two_graphs_share_nothing():
    sizes, contexts = [30, 8], [2000, 700]
    cases = [_case(sizes, contexts, 16, 2, 128, 16, torch.bfloat16, f, 4) for f in (None, E4M3)]
    lens, cu = torch.tensor(contexts, dtype=torch.int32, device=DEV), _cu(sizes)
    run = lambda q, k, v, ks, vs, bt, m: tsb.paged_tree_attention(  # noqa: E731
        q, k, v, bt, 16, lens, cu, m, 30, k_scale=ks, v_scale=vs)
    eager = [run(*c) for c in cases]
    graphs, outs = [], []
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(*c))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    tsb.check_errors()
    for o, e in zip(outs, eager):
        assert torch.equal(o, e)


def test_large_scores_and_minus_infinity():
    """Scores in the thousands and a drafted K row of the type's lowest value: the running maximum moves far."""
    sizes, contexts = [12], [400]
    for hq in (2, 16):
        q, k, v, ks, vs, bt, mask = _case(sizes, contexts, hq, 2, 128, 16, torch.bfloat16, None, 4)
        q = q * 30
        out, bound = ref.attention(q, k, v, bt, 16, contexts, sizes, mask)
        ref.assert_within(_run(q, k, v, ks, vs, bt, mask, 16, contexts, sizes), out, bound)
        low = torch.finfo(torch.bfloat16).min
        k[int(bt[0, 25]), :, 2] = low  # node 2: scores of +-inf or NaN for its descendants alone
        got = _run(q, k, v, ks, vs, bt, mask, 16, contexts, sizes)
        clean = [t for t in range(12) if not (int(mask[t, 0]) >> 2) & 1]
        ref.assert_within(got[clean], out[clean], bound[clean])


def test_registered_ops_match_their_fakes_and_run_in_a_graph():
    """opcheck on real launches, and one verification step under torch.compile, caches included."""
    Q = torch.ops.qwen3fused
    sizes, contexts, B = [4, 3], [30, 9], 16
    q, k, v, ks, vs, bt, mask = _case(sizes, contexts, 8, 2, 128, B, torch.bfloat16, E4M3, 15)
    g = torch.Generator().manual_seed(2)
    parents, cu = ref.random_parents(sizes, g).to(DEV), _cu(sizes)
    lens = torch.tensor(contexts, dtype=torch.int32, device=DEV)
    kn, vn = (torch.randn(2, 7, 128, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    of = torch.tensor([0] * 4 + [1] * 3, device=DEV)
    at = lens[of].long() + torch.tensor([0, 1, 2, 3, 0, 1, 2], device=DEV)
    bm, sm = bt[of, at // B].long(), at % B
    checks = ("test_schema", "test_faketensor")
    i8 = torch.zeros(k.shape[0], 2, B, 128, dtype=torch.int8, device=DEV)
    sc = torch.ones(k.shape[0], 2, B, device=DEV)
    torch.library.opcheck(Q.store_kv_cache_quantized, (kn, vn, i8, i8.clone(), sc, sc.clone(), bm, sm),
                          test_utils=checks)
    torch.library.opcheck(Q.load_kv_cache_quantized, (i8, i8.clone(), sc, sc.clone(), bm, sm, torch.float16),
                          test_utils=checks)
    torch.library.opcheck(Q.build_tree_mask, (parents, cu, 5), test_utils=checks)
    torch.library.opcheck(Q.paged_attention_quantized, (q[:2], i8, i8.clone(), sc, sc.clone(), bt, B, lens),
                          test_utils=checks)
    torch.library.opcheck(Q.paged_tree_attention, (q, i8, i8.clone(), bt, B, lens, cu, mask, 4, sc, sc.clone()),
                          test_utils=checks)

    def step(q, kn, vn, k, v, ks, vs):
        m, _ = Q.build_tree_mask(parents, cu, 4)
        Q.store_kv_cache_quantized(kn, vn, k, v, ks, vs, bm, sm)
        return Q.paged_tree_attention(q, k, v, bt, B, lens, cu, m, 4, ks, vs) * 2

    caches = [[x.clone() for x in (k, v, ks, vs)] for _ in range(2)]
    want = step(q, kn, vn, *caches[0])
    got = torch.compile(step, fullgraph=True, backend="aot_eager")(q, kn, vn, *caches[1])
    tsb.check_errors()
    assert torch.equal(got, want)
    for a, b in zip(*caches):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("fmt", [None, *ref.FORMATS])
@pytest.mark.parametrize("n,hq,D,parts", [(1, 2, 128, 4), (12, 1, 64, 4), (5, 1, 256, 4), (40, 1, 128, 2),
                                          (150, 1, 128, 1)])
def test_small_weights_beside_keys_without_a_value(fmt, n, hq, D, parts):
    """A key of a large score and a V of zeros outweighs each of 2^18 others 2^25.5 times, and those make the whole
    output: they count in the product as they do in the sum, whatever 16-bit type the probabilities are held in.
    As many such keys as a row has partial sums in a CTA (the mma.sync kernel's warps, which take 16 keys in turn;
    the tcgen05 kernel's warpgroups, 128 in turn), one for each of them."""
    block, pages = 64, parts << 12
    L = pages * block
    k, v = torch.zeros(5, 1, block, D), -torch.ones(5, 1, block, D)
    for j in [i * (16 if parts == 4 else 128) for i in range(parts)]:
        k[j // block, 0, j % block, 0] = 4.42
        v[j // block, 0, j % block] = 0

    def cache(c):  # four pages, and the fifth again and again
        return None if c is None else torch.cat([c.to(DEV)[:4], c.to(DEV)[4:].expand(pages - 4, *c.shape[1:])])

    (k, ks), (v, vs) = (map(cache, ref.quantise(c, fmt) if fmt else (c.half(), None)) for c in (k, v))
    if vs is not None:  # codes of 0 at the scale of the others, so that it is no part of the weight's range
        vs[:] = vs[4, 0, 0]
    q = torch.zeros(n, hq, D, dtype=torch.float16, device=DEV)
    q[..., 0] = 4
    bt = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    mask = ref.mask_of([-1] * n, [n], n)[0].to(DEV)
    out, _ = ref.attention(q, k, v, bt, block, [L - n], [n], mask, ks, vs, scale=1.0)
    # Counted as in tree_reference, A being |out|; the sums' part by what is added up, 2^18 / 16 steps of an
    # accumulator that may cut off what it cannot hold, 2^-23 of it.  And half a probability's least step, 2^-25
    # where a row's largest is 2^4 (the tcgen05 kernel over codes), |v| being 1, for each of 2^18 keys.
    u = 2.0 ** -11
    c = 2 * ((D + 8) * 2.0 ** -24 * 17.7 + 2.0 ** -16) + 2.0 ** 14 * 2.0 ** -23
    bound = (u + (u + c) * (1 + u)) * out.abs() + 2.0 ** 18 * 2.0 ** -29
    for split in (True, False):
        got = _run(q, k, v, ks, vs, bt, mask, block, [L - n], [n], split=split, softmax_scale=1.0)
        tsb.check_errors()
        ref.assert_within(got, out, bound, f"split={split}")


@pytest.mark.parametrize("fmt", ref.FORMATS)
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("n,hq", [(1, 2), (8, 4), (40, 8), (80, 8)])
def test_the_least_scales_that_the_store_writes(fmt, dtype, n, hq):
    """V rows of 2^-108 to 2^-90, whose scales go down to 2^-100 / Q: attention reads them as the load does."""
    sizes, contexts = [n, 1], [1100, 40]
    q, k, v, ks, vs, bt, mask = _case(sizes, contexts, hq, 2, 128, 16, dtype, fmt, 13)
    g = torch.Generator().manual_seed(2)
    rows = torch.randn(v.shape, generator=g) * 2.0 ** torch.randint(-108, -90, (*v.shape[:3], 1), generator=g)
    rows[bt[0, 20:40].cpu().long()] *= 2.0 ** -10  # pages of the least of them alone
    rows[bt[1].cpu().long()] *= 2.0 ** -10
    v, vs = (x.to(DEV) for x in ref.quantise(rows, fmt))
    out, bound = ref.attention(q, k, v, bt, 16, contexts, sizes, mask, ks, vs, p_type=torch.float16)
    for split in (True, False):
        got = _run(q, k, v, ks, vs, bt, mask, 16, contexts, sizes, split=split)
        tsb.check_errors()
        ref.assert_within(got, out, bound, f"split={split}")


@pytest.mark.parametrize("fmt,block", [(None, 8), (None, 24), (None, 32), (None, 64)] +
                         [(f, b) for f in ref.FORMATS for b in (4, 8, 12, 32, 64)])
def test_pages_of_every_power_of_two(fmt, block):
    """Boxes of 4 to 64 slots, a page in one or several, with ends inside them; one tile of rows and two."""
    for hq in (4, 8):
        _check([9, 40, 1], [333, 127, 1029], hq, 2, 128, block, torch.bfloat16, fmt, seed=block + hq)
