"""Host-side contract of the quantised cache and the token-tree operators (CPU only): what they refuse,
that they have no CPU path, their schemas and fakes, the argument structs, and the definitions that the
GPU tests compare with."""

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import tinyserver_b200 as tsb
from tests import tree_reference as ref
from tinyserver_b200 import _capi, ops

E4M3 = torch.float8_e4m3fn


def _cache(N=4, H=2, B=8, D=128, fmt=E4M3):
    return (torch.zeros(N, H, B, D, dtype=torch.uint8).view(fmt), torch.zeros(N, H, B))


def _store(k=None, v=None, kc=None, vc=None, ks=None, vs=None, bm=None, sm=None):
    codes, scales = _cache()
    k = torch.zeros(2, 3, 128) if k is None else k
    n = torch.zeros(3, dtype=torch.long)
    return tsb.store_kv_cache_quantized(k, k if v is None else v, codes if kc is None else kc,
                                        codes if vc is None else vc, scales if ks is None else ks,
                                        scales if vs is None else vs, n if bm is None else bm, n if sm is None else sm)


@pytest.mark.parametrize("kw,match", [
    (dict(k=torch.zeros(3, 128)), "3D"),
    (dict(v=torch.zeros(2, 4, 128)), "one shape"),
    (dict(v=torch.zeros(2, 3, 128, dtype=torch.float16)), "dtypes differ"),
    (dict(k=torch.zeros(2, 3, 64)), "does not match"),
    (dict(k=torch.zeros(3, 3, 128)), "does not match"),
    (dict(kc=torch.zeros(4, 2, 8, 128)), "float8_e4m3fn or int8"),
    (dict(kc=_cache(fmt=torch.int8)[0]), "float8_e4m3fn or int8"),
    (dict(vc=torch.zeros(4, 2, 128).to(E4M3)), "must be"),
    (dict(ks=torch.zeros(4, 2, 7)), "k_scale/v_scale"),
    (dict(vs=torch.zeros(4, 2, 8, dtype=torch.float16)), "float32"),
    (dict(bm=torch.zeros(4, dtype=torch.long)), "one length"),
    (dict(bm=torch.zeros(2, dtype=torch.long), sm=torch.zeros(2, dtype=torch.long)), "2 places for 3"),
    (dict(bm=torch.zeros(3), sm=torch.zeros(3)), "index dtype"),
    (dict(k=torch.zeros(2, 3, 128, dtype=torch.float64)), "not supported"),
    (dict(), "CUDA tensors only"),
])
def test_store_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        _store(**kw)


def test_load_refusals():
    codes, scales = _cache()
    n = torch.zeros(3, dtype=torch.long)
    with pytest.raises(ValueError, match="float8_e4m3fn or int8"):
        tsb.load_kv_cache_quantized(codes.float(), codes, scales, scales, n, n)
    with pytest.raises(ValueError, match="one length"):
        tsb.load_kv_cache_quantized(codes, codes, scales, scales, n, n[:2])
    with pytest.raises(ValueError, match="CUDA tensors only"):
        tsb.load_kv_cache_quantized(codes, codes, scales, scales, n, n)


def _attend(decode=False, **kw):
    codes, scales = _cache()
    a = dict(query=torch.zeros(5, 4, 128, dtype=torch.bfloat16), k_cache=codes, v_cache=codes, k_scale=scales,
             v_scale=scales, block_tables=torch.zeros(2, 3, dtype=torch.int32), block_size=8,
             lens=torch.zeros(2, dtype=torch.int32), cu=torch.tensor([0, 2, 5], dtype=torch.int32),
             mask=torch.zeros(5, 1, dtype=torch.int64), max_tree=3)
    if decode:
        a["query"] = a["query"][:2]
    a.update(kw)
    if decode:
        return tsb.paged_attention_quantized(a["query"], a["k_cache"], a["v_cache"], a["k_scale"], a["v_scale"],
                                             a["block_tables"], a["block_size"], a["lens"])
    return tsb.paged_tree_attention(a["query"], a["k_cache"], a["v_cache"], a["block_tables"], a["block_size"],
                                    a["lens"], a["cu"], a["mask"], a["max_tree"], k_scale=a["k_scale"],
                                    v_scale=a["v_scale"])


PLAIN = torch.zeros(4, 2, 8, 128, dtype=torch.bfloat16)


@pytest.mark.parametrize("decode", [False, True])
@pytest.mark.parametrize("kw,match", [
    (dict(query=torch.zeros(5, 128)), "3D|num_tokens"),
    (dict(k_scale=None), "come together|are needed"),
    (dict(k_cache=PLAIN, v_cache=PLAIN), "float8_e4m3fn or int8"),
    (dict(v_cache=_cache(B=16)[0]), "must be"),
    (dict(v_scale=torch.zeros(4, 2, 16)[..., ::2]), "strides differ"),
    (dict(block_size=16), "does not match"),
    (dict(block_tables=torch.zeros(3, 3, dtype=torch.int32)), "block_tables"),
    (dict(), "CUDA tensors only"),
])
def test_attention_refusals(kw, match, decode):
    with pytest.raises(ValueError, match=match):
        _attend(decode, **kw)


@pytest.mark.parametrize("kw,match", [
    (dict(query=torch.zeros(5, 3, 128, dtype=torch.bfloat16)), "multiple"),
    (dict(query=torch.zeros(5, 4, 64, dtype=torch.bfloat16)), "does not match"),
    (dict(k_scale=None, v_scale=None), "dtype"),
    (dict(k_scale=None, v_scale=None, k_cache=PLAIN, v_cache=PLAIN.half()), "dtype"),
    (dict(cu=torch.zeros(2, dtype=torch.int32)), "cu_seqlens"),
    (dict(max_tree=0), "max_tree"),
    (dict(max_tree=65), "tree_mask"),
    (dict(mask=torch.zeros(4, 1, dtype=torch.int64)), "tree_mask"),
    (dict(mask=torch.zeros(5, 1, dtype=torch.int32)), "tree_mask"),
    (dict(mask=torch.zeros(5, dtype=torch.int64)), "tree_mask"),
    (dict(lens=torch.zeros(0), cu=torch.zeros(1), block_tables=torch.zeros(0, 1)), "no sequence"),
])
def test_tree_attention_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        _attend(**kw)


def test_decode_refuses_other_lengths():
    with pytest.raises(ValueError, match="seq_lens"):
        _attend(True, lens=torch.zeros(3, dtype=torch.int32), block_tables=torch.zeros(3, 3, dtype=torch.int32))


@pytest.mark.parametrize("workspace", [torch.zeros(1).expand(1 << 20), torch.zeros(64)[::2]])
def test_workspace_in_one_piece(workspace):
    q, lens, bt = torch.zeros(1, 4, 128, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32), \
        torch.zeros(1, 3, dtype=torch.int32)
    cu, mask = torch.zeros(2, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int64)
    with pytest.raises(ValueError, match="contiguous"):
        tsb.paged_tree_attention(q, PLAIN, PLAIN, bt, 8, lens, cu, mask, 1, workspace=workspace)
    codes, scales = _cache()
    with pytest.raises(ValueError, match="contiguous"):
        tsb.paged_attention_quantized(q, codes, codes, scales, scales, bt, 8, lens, workspace=workspace)


def test_mask_refusals():
    p, cu = torch.zeros(3, dtype=torch.int32), torch.tensor([0, 3])
    for bad, match in (((p[None], cu, 3), "parents must"), ((p, cu, 0), "max_tree"), ((p.float(), cu, 3), "index dtype"),
                       ((p, cu.float(), 3), "index dtype"), ((p, cu, 3), "CUDA tensors only")):
        with pytest.raises(ValueError, match=match):
            tsb.build_tree_mask(*bad)


def _tree_args(**kw):
    base = dict(q=4096, q_stride_token=512, q_stride_head=128, k_cache=4096, v_cache=4096,
                cache_strides=(2048, 1024, 128, 1), k_scale=4096, v_scale=4096, scale_strides=(16, 8, 1),
                num_blocks=4, block_size=8, block_tables=4096, block_tables_row_stride=3, max_blocks_per_seq=300,
                context_lens=4096, cu_seqlens_q=4096, tree_mask=4096, mask_words=1, num_seqs=2, num_tokens=5,
                max_tree=3, num_q_heads=4, num_kv_heads=2, head_dim=128, scale=1.0, out=4096, out_stride_token=512,
                out_stride_head=128, dtype=_capi.QF_BF16, cache_format=_capi.QF_CACHE_E4M3)
    base.update(kw)
    return _capi.PagedTreeAttentionArgs.named(**base)


@pytest.mark.parametrize("kw,rc", [
    (dict(num_seqs=-1), 1), (dict(num_q_heads=3), 1), (dict(dtype=9), 1), (dict(cache_format=7), 1), (dict(q=0), 1),
    (dict(k_scale=0), 1), (dict(tree_mask=0), 1), (dict(mask_words=0), 1), (dict(max_tree=65), 1),
    (dict(max_tree=0), 1), (dict(num_seqs=0), 1), (dict(cu_seqlens_q=0), 1), (dict(out=0), 1),
    (dict(head_dim=96), 2), (dict(q=4104), 2), (dict(q_stride_token=516), 2), (dict(cache_strides=(2048, 1024, 8, 1)), 2),
    (dict(cache_strides=(2048, 1024, 128, 2)), 2), (dict(out=4100), 2), (dict(out_stride_head=4), 2),
    (dict(max_blocks_per_seq=1 << 28), 2), (dict(max_tree=70000, mask_words=2000), 2), (dict(num_seqs=70000), 2),
    (dict(num_seqs=65535, max_blocks_per_seq=1 << 26), 2), (dict(workspace=4096, workspace_bytes=16), 1),
    (dict(workspace=4104, workspace_bytes=1 << 40), 2), (dict(num_tokens=0), 0),
])
def test_c_entry_refuses_before_any_launch(kw, rc):
    assert _capi.lib().qf_paged_tree_attention(_tree_args(**kw), None) == rc


def test_other_c_entries_refuse_before_any_launch():
    lib = _capi.lib()
    for fn in (lib.qf_kv_store_quantized, lib.qf_kv_load_quantized):
        pack = _capi.KvQuantizedArgs.named
        ok = dict(num_tokens=3, num_kv_heads=2, head_dim=128, num_blocks=4, block_size=8, index_type=1, dtype=2,
                  format=1)
        assert fn(None, None) == 1
        assert fn(pack(**ok), None) == 1  # null pointers
        for bad in (dict(num_tokens=-1), dict(index_type=5), dict(dtype=4), dict(format=0), dict(head_dim=-2)):
            assert fn(pack(**{**ok, **bad}), None) == 1
        assert fn(pack(**{**ok, "num_tokens": 0}), None) == 0
    pack = _capi.TreeMaskArgs.named
    ok = dict(num_seqs=2, num_nodes=5, max_tree=3, mask_words=1)
    for bad in ({}, dict(max_tree=0), dict(max_tree=65), dict(index_type=2), dict(num_nodes=-1)):
        assert lib.qf_build_tree_mask(pack(**{**ok, **bad}), None) == 1
    assert lib.qf_build_tree_mask(pack(**{**ok, "num_nodes": 0}), None) == 0
    assert lib.qf_paged_tree_attention(None, None) == 1
    assert lib.qf_paged_tree_attention_workspace_bytes(None) == 0


def test_packed_structs_have_the_headers_layout():
    """Sizes as the library was compiled; a float and two ints leave the padding that C does."""
    lib = _capi.lib()
    assert lib.qf_kv_quantized_args_size() == _capi.KvQuantizedArgs.size
    assert lib.qf_tree_mask_args_size() == _capi.TreeMaskArgs.size
    assert lib.qf_paged_tree_attention_args_size() == _capi.PagedTreeAttentionArgs.size
    data = _capi.PagedTreeAttentionArgs.named(scale=1.5, out=7, status=9)
    at = data.index(b"\x00\x00\xc0\x3f")
    assert ctypes.c_int64.from_buffer_copy(data[at + 8:at + 16]).value == 7
    assert data.endswith(b"\x09" + 7 * b"\x00")


def test_workspace_grows_with_what_is_cut():
    ws = tsb.paged_tree_attention_workspace_bytes
    assert ws(4, 4, 1, 8, 2, 128, 16, 4, torch.bfloat16) == 0  # too short to be cut
    short, long = (ws(64, 1, 64, 32, 8, 128, 16, n, torch.bfloat16) for n in (64, 8192))
    assert 0 < short <= long < 1 << 30


def test_schemas_declare_the_cache_writes():
    for name, mutated in (("store_kv_cache_quantized", {"k_cache", "v_cache", "k_scale", "v_scale"}),
                          ("load_kv_cache_quantized", set()), ("paged_attention_quantized", set()),
                          ("build_tree_mask", set()), ("paged_tree_attention", set())):
        assert name in ops.OPS
        s = getattr(torch.ops.qwen3fused, name).default._schema
        assert {a.name for a in s.arguments if a.alias_info is not None and a.alias_info.is_write} == mutated
        assert all(r.alias_info is None for r in s.returns)


def test_fakes():
    Q = torch.ops.qwen3fused
    with FakeTensorMode():
        new = lambda *s, dtype=torch.bfloat16: torch.empty(*s, dtype=dtype, device="cuda")  # noqa: E731
        codes, scales = new(4, 2, 8, 128, dtype=E4M3), new(4, 2, 8, dtype=torch.float32)
        n = new(7, dtype=torch.long)
        assert Q.store_kv_cache_quantized(new(2, 7, 128), new(2, 7, 128), codes, codes, scales, scales, n, n) is None
        k, v = Q.load_kv_cache_quantized(codes, codes, scales, scales, n, n, torch.float16)
        assert k.shape == v.shape == (2, 7, 128) and k.dtype == torch.float16
        assert k.transpose(0, 1).is_contiguous()
        bt, lens = new(5, 3, dtype=torch.int32), new(5, dtype=torch.int32)
        q = new(5, 4, 128)
        assert Q.paged_attention_quantized(q, codes, codes, scales, scales, bt, 8, lens).shape == q.shape
        cu = new(6, dtype=torch.int32)
        mask, depths = Q.build_tree_mask(new(7, dtype=torch.int32), cu, 100)
        assert mask.shape == (7, 2) and mask.dtype == torch.int64 and depths.dtype == torch.int32
        out = Q.paged_tree_attention(new(7, 4, 128), codes, codes, bt, 8, lens, cu, mask, 100, scales, scales)
        assert out.shape == (7, 4, 128) and out.is_contiguous()


@pytest.mark.parametrize("fmt", ref.FORMATS)
def test_definition_of_a_quantised_row(fmt):
    """Codes are the nearest to x / scale (half a step), scales the row's amax over the top code."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(50, 128, generator=g) * 10.0 ** torch.randint(-5, 6, (50, 1), generator=g)
    codes, scales = ref.quantise(x, fmt)
    assert torch.allclose(scales.double(), x.abs().amax(-1).double() / ref.TOP[fmt], rtol=2.0 ** -23, atol=0)
    y = x.double() / (x.abs().amax(-1, keepdim=True).double() / ref.TOP[fmt])
    off = (codes.double() - y).abs()
    half = torch.full_like(y, 0.5) if fmt == torch.int8 else \
        torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 4)
    assert (off <= half * (1 + 1e-5)).all()
    zero, scale = ref.quantise(torch.zeros(1, 128), fmt)
    assert not zero.float().any() and scale[0] > 0
    bad, scale = ref.quantise(torch.tensor([[1.0, float("inf")]]), fmt)
    assert not bad.float().any() and torch.isnan(scale[0])


def test_reference_attention_against_a_softmax():
    """The 64-bit definition that the kernels are held to, against torch's softmax on a dense cache."""
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(6, 2, 8, 16, generator=g, dtype=torch.float64) for _ in range(2))
    q = torch.randn(5, 4, 16, generator=g)
    tables = torch.tensor([[3, 1, 5, 0], [2, 4, 0, 0]])
    mask, _ = ref.mask_of(torch.tensor([-1, 0, 0, -1, 0]), [3, 2], 3)
    out, _ = ref.attention(q, k, v, tables, 8, [20, 9], [3, 2], mask)
    rows = lambda c, s, n: c[tables[s]].transpose(1, 2).flatten(0, 1)[:n]  # noqa: E731
    for t, (s, seen) in enumerate([(0, [*range(20), 20]), (0, [*range(20), 20, 21]), (0, [*range(20), 20, 22]),
                                   (1, [*range(9), 9]), (1, [*range(9), 9, 10])]):
        kk, vv = (rows(c, s, 32)[seen] for c in (k, v))
        for h in range(4):
            p = torch.softmax(q[t, h].double() @ kk[:, h // 2].T / 4, -1)
            assert torch.allclose(out[t, h], p @ vv[:, h // 2])


@pytest.mark.parametrize("kw,decode", [(dict(lens=torch.zeros(2)), True), (dict(lens=torch.zeros(2)), False),
                                       (dict(block_tables=torch.zeros(2, 3)), True),
                                       (dict(block_tables=torch.zeros(2, 3, dtype=torch.int16)), False),
                                       (dict(cu=torch.tensor([0., 2., 5.])), False)])
def test_attention_refuses_lengths_and_tables_of_other_types(kw, decode):
    with pytest.raises(ValueError, match="index dtype"):
        _attend(decode, **kw)


def test_int64_lengths_stay_out_of_range_as_int32():
    """What is beyond int32 is the least or the largest of it, which the kernels cut and report: never a small
    number that it happens to equal modulo 2^32."""
    from tinyserver_b200.kernels.tree import _int32

    got = _int32(torch.tensor([(1 << 32) + 5, -(1 << 32) + 5, 1 << 31, 7, -3, (1 << 31) - 1]))
    assert got.dtype == torch.int32
    assert got.tolist() == [(1 << 31) - 1, -(1 << 31), (1 << 31) - 1, 7, -3, (1 << 31) - 1]
    for t in (torch.tensor([3, 4], dtype=torch.int32), torch.tensor([[1, 2], [3, 4]], dtype=torch.int32)):
        assert _int32(t) is t


def test_mappings_of_two_types_keep_their_values():
    from tinyserver_b200.kernels.quantized import _mappings

    small, large = torch.tensor([1, 2], dtype=torch.int32), torch.tensor([3, (1 << 32) + 4])
    for pair in ((small, large), (large, small)):
        bm, sm, tag = _mappings("test", *pair)
        assert bm.tolist() == pair[0].tolist() and sm.tolist() == pair[1].tolist()
        assert bm.dtype == sm.dtype == torch.int64 and tag == _capi.QF_I64
    bm, sm, tag = _mappings("test", small, small)
    assert bm is small and sm is small and tag == _capi.QF_I32


def test_workspace_sizes_before_the_arrays_exist():
    """cu_seqlens_q NULL: enough for the trees' call, and for a decode call of the same sizes."""
    size = lambda **kw: _capi.lib().qf_paged_tree_attention_workspace_bytes(_tree_args(**kw))  # noqa: E731
    for fmt in (_capi.QF_CACHE_PLAIN, _capi.QF_CACHE_E4M3):
        for dtype in (_capi.QF_F32, _capi.QF_BF16):
            for max_tree in (1, 3, 64):
                kw = dict(cache_format=fmt, dtype=dtype, max_tree=max_tree)
                trees, decode = size(**kw), size(**kw, cu_seqlens_q=0)
                assert 0 < trees <= decode
                assert size(**{**kw, "max_tree": 1}, cu_seqlens_q=0) <= decode
