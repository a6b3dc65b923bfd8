"""The quantised paged KV cache on the GPU against its definition: stores and loads bit
for bit, decode attention within bounds counted from its roundings (tree_reference)."""

import pytest
import torch

import tinyserver_b200 as tsb
from tests import tree_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def _bits(t):
    return t.view(torch.uint8)


def _places(tokens, blocks, block, g):
    at = torch.randperm(blocks * block, generator=g)[:tokens]
    return at // block, at % block


def _empty_cache(shape, fmt, device=DEV):
    codes = torch.full(shape, 0x55, dtype=torch.uint8, device=device).view(fmt)
    return codes, torch.full(shape[:3], 7.0, device=device)


def _check_store(k, v, fmt, block, blocks, g, index=torch.int64, view=None):
    """Store (H, T, D) rows; every place equals the definition, or is as it was."""
    H, T, D = k.shape
    bm, sm = _places(T, blocks, block, g)
    pools = [_empty_cache((blocks, H, block, D), fmt) for _ in range(2)]
    if view:
        pools = [view(*p) for p in pools]
    tsb.store_kv_cache_quantized(k.to(DEV), v.to(DEV), pools[0][0],
                                 pools[1][0], pools[0][1], pools[1][1], bm.to(DEV, index),
                                 sm.to(DEV, index))
    tsb.check_errors()
    for src, (codes, scales) in zip((k, v), pools):
        want_codes, want_scales = _empty_cache((blocks, H, block, D), fmt, "cpu")
        c, s = ref.quantise(src.transpose(0, 1), fmt)
        _bits(want_codes)[bm, :, sm] = _bits(c)
        want_scales[bm, :, sm] = s
        assert torch.equal(_bits(codes.contiguous()).cpu(), _bits(want_codes))
        assert torch.equal(scales.contiguous().cpu().view(torch.int32), want_scales.view(torch.int32)) or \
            torch.equal(scales.cpu().nan_to_num(-1.0), want_scales.nan_to_num(-1.0))
    return pools, bm, sm


@pytest.mark.parametrize("fmt", ref.FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256, 80, 1])
def test_store_and_load_are_the_definition(fmt, dtype, D):
    g = torch.Generator().manual_seed(D)
    for T in (1, 33, 130):
        k, v = (torch.randn(3, T, D, generator=g).mul_(10.0 ** torch.randint(-3, 4, (3, T, 1), generator=g))
                .to(dtype) for _ in range(2))
        k[0, 0] = 0  # an all-zero row
        pools, bm, sm = _check_store(k, v, fmt, 16, 12, g, torch.int32 if T == 33 else torch.int64)
        for out in DTYPES:
            got = tsb.load_kv_cache_quantized(pools[0][0], pools[1][0], pools[0][1], pools[1][1],
                                              bm.to(DEV), sm.to(DEV), out)
            for x, src in zip(got, (k, v)):
                c, s = ref.quantise(src, fmt)
                assert x.shape == src.shape and x.transpose(0, 1).is_contiguous()
                assert torch.equal(x.cpu(), (c.float() * s[..., None]).to(out))
    # half a step of the code, relative to the row's largest value, and what the type holds
    back = x.float().cpu() if out == torch.float32 else (c.float() * s[..., None])
    step = 0.5 / 127 if fmt == torch.int8 else 2.0 ** -4
    near = (back - src.float()).abs()
    top = src.float().abs().amax(-1, keepdim=True)
    assert (near <= step * (1 + 1e-5) * (top if fmt == torch.int8 else src.float().abs()) + top * 2.0 ** -9 / 448).all()


@pytest.mark.parametrize("fmt", ref.FORMATS)
def test_store_odd_values(fmt):
    """Infinities and NaN poison their own row's scale only; subnormal and tiny rows; the largest values."""
    g = torch.Generator().manual_seed(1)
    for dtype in DTYPES:
        k = torch.randn(2, 9, 128, generator=g).to(dtype)
        k[0, 1, 5], k[1, 2, 127], k[0, 3, 0] = float("nan"), float("inf"), -float("inf")
        k[0, 4] = torch.finfo(dtype).tiny / 8
        k[1, 5] = torch.finfo(dtype).max
        k[1, 6, ::2] = -torch.finfo(dtype).max
        pools, bm, sm = _check_store(k, k.flip(1), fmt, 8, 4, g)
        x, _ = tsb.load_kv_cache_quantized(pools[0][0], pools[1][0], pools[0][1], pools[1][1], bm.to(DEV),
                                           sm.to(DEV), dtype)
        assert torch.equal(torch.isnan(x).all(-1).cpu(), ~torch.isfinite(k).all(-1))


def test_store_strides_and_layer_views():
    """Sources as views of a merged projection, with odd offsets and a strided last dim; a layer of a pool."""
    g = torch.Generator().manual_seed(2)
    qkv = torch.randn(40, 5 * 128 + 3, generator=g).to(torch.bfloat16).to(DEV)
    aligned = qkv[:, :640].unflatten(1, (5, 128)).transpose(0, 1)
    odd = qkv[:, 3:643].unflatten(1, (5, 128)).transpose(0, 1)
    wide = torch.randn(5, 40, 256, generator=g).to(DEV)[:, :, ::2]
    for src in (aligned, odd, wide):
        _check_store(src, src.cpu().flip(1), torch.int8, 16, 5, g)

    def layer(codes, scales):
        n, h, b, d = codes.shape
        pool = torch.full((n, 3, h, b, d), 0x55, dtype=torch.uint8, device=DEV).view(codes.dtype)
        sc = torch.full((h, n, b, 2), 7.0, device=DEV)
        return pool[:, 1], sc[..., 1].transpose(0, 1)

    _check_store(aligned, aligned.cpu().flip(1), torch.float8_e4m3fn, 16, 5, g, view=layer)


def test_places_outside_the_cache_are_skipped_and_flagged():
    k = torch.ones(2, 3, 128, dtype=torch.bfloat16, device=DEV)
    codes, scales = _empty_cache((4, 2, 8, 128), torch.int8)
    before = codes.clone(), scales.clone()
    for bm, sm, match in (([-1, 4, 1 << 40], [0, 0, 0], "block"), ([1, 1, 1], [-1, 8, 1 << 33], "slot")):
        bm, sm = torch.tensor(bm, device=DEV), torch.tensor(sm, device=DEV)
        tsb.store_kv_cache_quantized(k, k, codes, codes, scales, scales, bm, sm)
        with pytest.raises(IndexError, match=match):
            tsb.check_errors()
        assert torch.equal(codes, before[0]) and torch.equal(scales, before[1])
        x, _ = tsb.load_kv_cache_quantized(codes, codes, scales, scales, bm, sm, torch.float16)
        assert not x.any()
        with pytest.raises(IndexError, match=match):
            tsb.check_errors()


def test_no_tokens():
    codes, scales = _empty_cache((4, 2, 8, 128), torch.int8)
    none = torch.zeros(0, dtype=torch.int64, device=DEV)
    k = torch.zeros(2, 0, 128, device=DEV)
    tsb.store_kv_cache_quantized(k, k, codes, codes, scales, scales, none, none)
    x, _ = tsb.load_kv_cache_quantized(codes, codes, scales, scales, none, none, torch.float32)
    assert x.shape == (2, 0, 128)
    q = torch.zeros(0, 4, 128, device=DEV)
    bt = torch.zeros(0, 3, dtype=torch.int32, device=DEV)
    assert tsb.paged_attention_quantized(q, codes, codes, scales, scales, bt, 8, none).shape == q.shape
    tsb.check_errors()


def paged(lens, hkv, D, block, fmt, dtype, seed, extra=3, spread=False):
    """Caches (quantised when fmt is given) holding lens[s] keys per sequence, and block tables."""
    g = torch.Generator().manual_seed(seed)
    pages = [-(-n // block) for n in lens]
    N = sum(pages) + extra
    got = []
    for _ in range(2):
        x = torch.randn(N, hkv, block, D, generator=g)
        if spread:
            x *= 10.0 ** torch.randint(-4, 5, (N, hkv, block, 1), generator=g)
        got.append(ref.quantise(x, fmt) if fmt else (x.to(dtype), None))
    order = torch.randperm(N, generator=g)[:sum(pages)].int()
    bt = torch.zeros(len(lens), max(pages + [1]) + 1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(pages):
        bt[s, :n] = order[at:at + n]
        at += n
    (k, ks), (v, vs) = got
    put = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    return put(k), put(v), put(ks), put(vs), bt.to(DEV)


@pytest.mark.parametrize("fmt", ref.FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,D,block", [(8, 8, 128, 16), (6, 2, 64, 8), (32, 8, 128, 16), (16, 2, 256, 24),
                                            (20, 1, 128, 256), (64, 8, 64, 16), (9, 1, 256, 5)])
def test_decode_against_64_bits(fmt, dtype, hq, hkv, D, block):
    lens = [0, 1, 2, 15, 16, 17, 63, 64, 65, 300, 1029]
    k, v, ks, vs, bt = paged(lens, hkv, D, block, fmt, dtype, seed=hq * D + block)
    q = torch.randn(len(lens), hq, D, generator=torch.Generator().manual_seed(5)).to(dtype).to(DEV)
    out, bound = ref.attention(q, k, v, bt, block, lens, k_scale=ks, v_scale=vs)
    sl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    for split in (True, False):
        got = tsb.paged_attention_quantized(q, k, v, ks, vs, bt, block, sl, split=split)
        tsb.check_errors()
        assert got.dtype == dtype and not got[0].any()
        ref.assert_within(got, out, bound, f"split={split}")


@pytest.mark.parametrize("fmt", ref.FORMATS)
@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
def test_decode_with_scales_over_eight_decades(fmt, dtype):
    """Rows from 1e-4 to 1e4: V's scale is in the exponent, so no probability under- or overflows; queries of
    very different sizes; a long split sequence."""
    lens = [700, 4000]
    k, v, ks, vs, bt = paged(lens, 2, 128, 16, fmt, dtype, seed=3, spread=True)
    ks = ks.clamp_max(0.02)
    q = torch.randn(2, 8, 128, generator=torch.Generator().manual_seed(6)).to(DEV)
    q *= torch.logspace(-7, 1, 8, device=DEV)[:, None]
    q = q.to(dtype)
    out, bound = ref.attention(q, k, v, bt, 16, lens, k_scale=ks, v_scale=vs)
    # queries below fp16's normal range lose bits in the type itself, not in the kernel
    got = tsb.paged_attention_quantized(q, k, v, ks, vs, bt, 16, torch.tensor(lens, device=DEV))
    tsb.check_errors()
    ref.assert_within(got, out, bound)


@pytest.mark.parametrize("fmt", ref.FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_masked_places_never_matter(fmt, dtype):
    """Slots past the end hold NaN scales and e4m3 NaN codes; a key of NaN scale inside gives NaN for its
    sequence alone; an infinite query for its head alone."""
    lens = [5, 21, 700, 33]
    k, v, ks, vs, bt = paged(lens, 2, 128, 16, fmt, dtype, seed=9)
    for s, n in enumerate(lens):
        last = int(bt[s, (n - 1) // 16])
        for c, sc in ((k, ks), (v, vs)):
            sc[last, :, (n - 1) % 16 + 1:] = float("nan")
            _bits(c)[last, :, (n - 1) % 16 + 1:] = 0x7f
    q = torch.randn(4, 8, 128, generator=torch.Generator().manual_seed(6)).to(dtype).to(DEV)
    out, bound = ref.attention(q, k, v, bt, 16, lens, k_scale=ks, v_scale=vs)
    sl = torch.tensor(lens, dtype=torch.int64, device=DEV)
    got = tsb.paged_attention_quantized(q, k, v, ks, vs, bt, 16, sl)
    tsb.check_errors()
    assert torch.isfinite(got).all()
    ref.assert_within(got, out, bound)
    vs[int(bt[3, 0]), 1, 3] = float("nan")
    q[0, 2, 7] = float("inf")
    got = tsb.paged_attention_quantized(q, k, v, ks, vs, bt, 16, sl)
    bad = torch.isnan(got).all(-1)
    want = torch.zeros(4, 8, dtype=torch.bool, device=DEV)
    want[3, 4:] = True
    want[0, 2] = True
    assert torch.equal(bad, want) and torch.isfinite(got[~want]).all()


def test_decode_bad_lengths_and_blocks_are_cut_and_flagged():
    lens = [40, 100, 30]
    k, v, ks, vs, bt = paged(lens, 2, 128, 16, torch.int8, torch.bfloat16, seed=12)
    q = torch.randn(3, 8, 128, device=DEV).to(torch.bfloat16)
    run = lambda b, n: tsb.paged_attention_quantized(q, k, v, ks, vs, b, 16, torch.tensor(n, device=DEV))  # noqa: E731
    cap = bt.shape[1] * 16
    cut = run(bt, [40, cap, 0])
    tsb.check_errors()
    got = run(bt, [40, cap + 5000, -3])
    with pytest.raises(IndexError, match="block table"):
        tsb.check_errors()
    assert torch.equal(got, cut) and not got[2].any()
    bad = bt.clone()
    bad[0, 1] = k.shape[0] + 1000
    got = run(bad, lens)
    with pytest.raises(IndexError, match="block index"):
        tsb.check_errors()
    keep = torch.tensor([int(b) for i, b in enumerate(bt[0, :3]) if i != 1] + [0], device=DEV, dtype=torch.int32)
    want = tsb.paged_attention_quantized(q[:1], k, v, ks, vs, keep[None], 16, torch.tensor([24], device=DEV))
    assert torch.allclose(got[0].float(), want[0].float(), atol=2e-2)  # the other keys, in other tiles


def test_offsets_past_32_bits():
    """A cache of more than 2^32 codes: the last blocks are written, read back and attended to."""
    N, H, B, D = 270000, 8, 16, 128
    assert N * H * B * D > 1 << 32
    k = torch.zeros(N, H, B, D, dtype=torch.int8, device=DEV)
    v = torch.zeros_like(k)
    ks, vs = (torch.zeros(N, H, B, device=DEV) for _ in range(2))
    g = torch.Generator().manual_seed(4)
    rows = [torch.randn(H, 90, D, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2)]
    at = N * B - 1 - torch.arange(96, device=DEV)
    bt = (N - 1 - torch.arange(6, device=DEV)).int()[None]
    j = torch.arange(90, device=DEV)
    bm, sm = bt[0][j // 16].long(), j % 16
    assert int(at.max()) * H * D > 1 << 31
    tsb.store_kv_cache_quantized(*rows, k, v, ks, vs, bm, sm)
    back = tsb.load_kv_cache_quantized(k, v, ks, vs, bm, sm, torch.float32)
    for x, src in zip(back, rows):
        c, s = ref.quantise(src, torch.int8)
        assert torch.equal(x.cpu(), c.float() * s[..., None])
    q = torch.randn(1, 32, D, generator=g).to(torch.bfloat16).to(DEV)
    got = tsb.paged_attention_quantized(q, k, v, ks, vs, bt, B, torch.tensor([90], device=DEV))
    tsb.check_errors()
    small = slice(N - 8, N)
    out, bound = ref.attention(q, k[small], v[small], bt - (N - 8), B, [90], k_scale=ks[small], v_scale=vs[small])
    ref.assert_within(got, out, bound)


def test_two_graphs_another_stream_and_a_given_workspace():
    """Two captured graphs replayed on two streams give what eager calls give; same bits every time."""
    lens = [900, 3000]
    k, v, ks, vs, bt = paged(lens, 2, 128, 16, torch.float8_e4m3fn, torch.bfloat16, seed=2)
    sl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    qs = [torch.randn(2, 8, 128, device=DEV).to(torch.bfloat16) for _ in range(2)]
    run = lambda q, **kw: tsb.paged_attention_quantized(q, k, v, ks, vs, bt, 16, sl, **kw)  # noqa: E731
    eager = [run(q) for q in qs]
    need = tsb.paged_tree_attention_workspace_bytes(2, 2, 1, 8, 2, 128, 16, bt.shape[1], torch.bfloat16)
    assert need > 0
    ws = torch.full((need // 4,), float("nan"), device=DEV)
    assert torch.equal(run(qs[0], workspace=ws), eager[0])
    with pytest.raises(ValueError):
        run(qs[0], workspace=ws[:need // 4 - 1])
    graphs, outs = [], []
    for q in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(q))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for o, e in zip(outs, eager):
        assert torch.equal(o, e)


def test_a_prefix_cached_quantised_then_prefilled_and_decoded():
    """The operators together: store a prefix quantised, load it back for the prefill kernel, and decode
    over it in place: prefill over the loaded rows and decode over the codes agree on the last token."""
    H, Hq, D, T, B = 8, 32, 128, 200, 16
    g = torch.Generator().manual_seed(8)
    k, v = (torch.randn(T, H, D, generator=g).to(torch.bfloat16).to(DEV).transpose(0, 1) for _ in range(2))
    N = 20
    pools = [_empty_cache((N, H, B, D), torch.float8_e4m3fn) for _ in range(2)]
    bt = torch.randperm(N, generator=g)[:13].int().to(DEV)[None]
    j = torch.arange(T, device=DEV)
    bm, sm = tsb.build_slot_mapping(torch.tensor([0, T], dtype=torch.int32, device=DEV), j, bt, B)
    tsb.store_kv_cache_quantized(k, v, pools[0][0], pools[1][0], pools[0][1], pools[1][1], bm, sm)
    kd, vd = tsb.load_kv_cache_quantized(pools[0][0], pools[1][0], pools[0][1], pools[1][1], bm, sm, torch.bfloat16)
    q = torch.randn(1, Hq, D, generator=g).to(torch.bfloat16).to(DEV)
    cu1, cuT = (torch.tensor([0, n], dtype=torch.int32, device=DEV) for n in (1, T))
    full = tsb.flash_attn_varlen_func(q, kd.transpose(0, 1), vd.transpose(0, 1), cu1, cuT, 1, T, False)
    got = tsb.paged_attention_quantized(q, pools[0][0], pools[1][0], pools[0][1], pools[1][1], bt, B,
                                        torch.tensor([T], device=DEV))
    tsb.check_errors()
    out, bound = ref.attention(q, pools[0][0], pools[1][0], bt, B, [T], k_scale=pools[0][1], v_scale=pools[1][1])
    ref.assert_within(got, out, bound)
    # the prefill's K and V are rounded to bf16 on loading: u in the scores (times E ~ 20) and in V
    u = 2.0 ** -8
    assert ((full.double() - out).abs() <= bound + (2 * 20 * u + u) * 1.0).all()


@pytest.mark.parametrize("fmt", ref.FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq", [8, 64])
def test_keys_of_nan_scales_alone_give_nan(fmt, dtype, hq):
    """Every V row that a head sees was stored from an infinity or a NaN: its output is NaN, not the zeros of a
    sequence of no keys; one key, several tiles, and partials none of which has a weight."""
    lens = [1, 70, 4000, 0]
    k, v, ks, vs, bt = paged(lens, 2, 128, 16, fmt, dtype, seed=14)
    vs[:, 1] = float("nan")
    _bits(v)[:, 1] = 0
    q = torch.randn(4, hq, 128, generator=torch.Generator().manual_seed(6)).to(dtype).to(DEV)
    want = torch.zeros(4, hq, dtype=torch.bool, device=DEV)
    want[:3, hq // 2:] = True
    for split in (True, False):
        got = tsb.paged_attention_quantized(q, k, v, ks, vs, bt, 16, torch.tensor(lens, device=DEV), split=split)
        tsb.check_errors()
        assert torch.equal(torch.isnan(got).all(-1), want) and torch.isfinite(got[~want]).all(), split
        assert not got[3].any()


def test_int64_lengths_and_blocks_past_32_bits_are_cut_and_flagged():
    """2^32 + 5 keys are more than the table describes, not 5; block 2^32 + 1 is no block of the cache, not 1."""
    lens = [40, 30]
    k, v, ks, vs, bt = paged(lens, 2, 128, 16, torch.int8, torch.bfloat16, seed=12)
    q = torch.randn(2, 8, 128, device=DEV).to(torch.bfloat16)
    run = lambda b, n: tsb.paged_attention_quantized(q, k, v, ks, vs, b, 16, torch.tensor(n, device=DEV))  # noqa: E731
    cap = bt.shape[1] * 16
    want = run(bt, [cap, 30])
    tsb.check_errors()
    got = run(bt, [(1 << 32) + 5, 30])
    with pytest.raises(IndexError, match="block table"):
        tsb.check_errors()
    assert torch.equal(got, want)
    far = bt.long()
    far[1, :2] += 1 << 32
    got = run(far, lens)
    with pytest.raises(IndexError, match="block index"):
        tsb.check_errors()
    assert not got[1].any()


def test_int64_slots_beside_int32_blocks_keep_their_values():
    """Slot 2^32 + 3 is no slot of the page, whatever the type of the block mapping."""
    k = torch.ones(2, 2, 128, dtype=torch.bfloat16, device=DEV)
    codes, scales = _empty_cache((4, 2, 8, 128), torch.int8)
    before = codes.clone(), scales.clone()
    bm = torch.tensor([1, 2], dtype=torch.int32, device=DEV)
    sm = torch.tensor([(1 << 32) + 3, -(1 << 32)], device=DEV)
    tsb.store_kv_cache_quantized(k, k, codes, codes, scales, scales, bm, sm)
    with pytest.raises(IndexError, match="slot"):
        tsb.check_errors()
    assert torch.equal(codes, before[0]) and torch.equal(scales, before[1])


@pytest.mark.parametrize("fmt", ref.FORMATS)
@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
@pytest.mark.parametrize("hq,hkv,block", [(32, 1, 16), (71, 1, 24), (160, 1, 16), (100, 2, 4), (60, 2, 5)])
def test_decode_of_many_heads_per_kv_head(fmt, dtype, hq, hkv, block):
    """More than 24 query heads a kv head: one node a sequence and no mask in the tcgen05 kernel."""
    lens = [0, 1, 127, 128, 129, 1029, 5000]
    k, v, ks, vs, bt = paged(lens, hkv, 128, block, fmt, dtype, seed=hq + block)
    q = torch.randn(len(lens), hq, 128, generator=torch.Generator().manual_seed(5)).to(dtype).to(DEV)
    out, bound = ref.attention(q, k, v, bt, block, lens, k_scale=ks, v_scale=vs, p_type=torch.float16)
    sl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    for split in (True, False):
        got = tsb.paged_attention_quantized(q, k, v, ks, vs, bt, block, sl, split=split)
        tsb.check_errors()
        assert not got[0].any()
        ref.assert_within(got, out, bound, f"split={split}")


@pytest.mark.parametrize("fmt", ref.FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256, 80, 1])
def test_rows_come_back_within_half_a_step(fmt, dtype, D):
    """What the kernels stored and loaded, K and V: half a step of the code from the source, 1 / 127 of the row's
    largest value for int8; 2^-3 of the value, or 2^-9 codes below 2^-6 of them, for e4m3.  Two roundings of 2^-24
    on the way to the code, and two on the way back."""
    g = torch.Generator().manual_seed(D + 1)
    for T in (1, 33, 130):
        k, v = (torch.randn(3, T, D, generator=g).mul_(10.0 ** torch.randint(-3, 4, (3, T, 1), generator=g))
                .to(dtype) for _ in range(2))
        pools, bm, sm = _check_store(k, v, fmt, 16, 12, g)
        got = tsb.load_kv_cache_quantized(pools[0][0], pools[1][0], pools[0][1], pools[1][1], bm.to(DEV),
                                          sm.to(DEV), torch.float32)
        for x, src in zip(got, (k.double(), v.double())):
            top = src.abs().amax(-1, keepdim=True)
            half = (0.5 / 127 * top).expand_as(src) if fmt == torch.int8 else \
                torch.maximum(2.0 ** -4 * src.abs(), 2.0 ** -10 * top / 448)
            assert ((x.double().cpu() - src).abs() <= half + 4 * 2.0 ** -24 * top).all()
