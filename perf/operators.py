"""What is measured of the operators on a quantised KV cache and of attention for drafted token trees.

Four operators, in the order a serving step meets them: K/V rows quantised as they are written to their
pages (``store``), rows read back as dense tensors (``load``), one query token per sequence over such a cache
(``decode``), and a tree of drafted tokens per sequence over a cache (``tree``), with the tree's visibility
mask built from the nodes' parents (``mask``, alone and within a ``tree`` pass).

A quantised row holds head_dim 8-bit codes (float8 e4m3 or int8) and one float32 scale, amax / 448 or
amax / 127 of that row.
"""

import math
import random

import torch

own = False

_TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
_TOP = {"e4m3": 448.0, "int8": 127.0}
_FLOOR = 2.0 ** -100  # the least amax a row's scale is made from


def _store(name, fmt, dtype, tokens, hkv, d, block, blocks):
    return {"name": name, "op": "store", "fmt": fmt, "dtype": dtype, "tokens": tokens, "hkv": hkv, "d": d,
            "block": block, "blocks": blocks}


def _load(name, fmt, dtype, tokens, hkv, d, block, blocks):
    return dict(_store(name, fmt, dtype, tokens, hkv, d, block, blocks), op="load")


def _decode(name, fmt, dtype, seqs, lo, hi, hq, hkv, d, block):
    return {"name": name, "op": "decode", "fmt": fmt, "dtype": dtype, "seqs": seqs, "lo": lo, "hi": hi, "hq": hq,
            "hkv": hkv, "d": d, "block": block}


def _tree(name, fmt, dtype, seqs, lo, hi, tree_lo, tree, hq, hkv, d, block, parents=False):
    return dict(_decode(name, fmt, dtype, seqs, lo, hi, hq, hkv, d, block), op="tree", tree_lo=tree_lo, tree=tree,
                parents=parents)


def listed():
    return [
        # the mixed prefill + decode batch of an 8B layer: 8192 K and V rows of 8 heads to their pages
        _store("store e4m3 mixed 8192", "e4m3", "bfloat16", 8192, 8, 128, 16, 4096),
        # a decode step of 256 sequences: one row each, where the call's latency counts
        _store("store int8 decode 256", "int8", "bfloat16", 256, 8, 128, 16, 2048),
        # a cached prefix brought back for chunked prefill
        _load("load e4m3 prefix 16411", "e4m3", "bfloat16", 16411, 8, 128, 16, 4096),
        # a short prefix of an fp32 model, large pages
        _load("load int8 short 484", "int8", "float32", 484, 8, 64, 256, 64),
        # an 8B model's decode step, 256 sequences of 1 to 8191 tokens
        _decode("decode e4m3 256 x 8191", "e4m3", "bfloat16", 256, 1, 8191, 32, 8, 128, 16),
        # one long conversation
        _decode("decode int8 1 x 131071", "int8", "float16", 1, 131071, 131071, 64, 8, 128, 16),
        # a few short chats: latency
        _decode("decode e4m3 4 x 700", "e4m3", "bfloat16", 4, 37, 700, 16, 8, 128, 16),
        # verification of 64-token trees for 64 sequences of an 8B model
        _tree("tree bf16 64 x 8191 + 64", "none", "bfloat16", 64, 1024, 8191, 64, 64, 32, 8, 128, 16),
        # smaller ragged trees of a 1.7B model
        _tree("tree fp16 16 x 4095 + 16", "none", "float16", 16, 1, 4095, 5, 16, 16, 8, 128, 16),
        # trees over a quantised cache
        _tree("tree e4m3 32 x 8191 + 32", "e4m3", "bfloat16", 32, 512, 8191, 9, 32, 32, 8, 128, 16),
        # one interactive user of a 32B model: mask and attention of a tree of 7 nodes
        _tree("tree + mask bf16 1 x 300 + 7", "none", "bfloat16", 1, 300, 300, 7, 7, 64, 8, 128, 16, True),
        # the masks of a large batch of dynamic trees
        {"name": "mask 256 x 127", "op": "mask", "seqs": 256, "tree_lo": 1, "tree": 127},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["store", "load", "decode", "decode", "tree", "tree", "tree", "mask"])
    if op == "mask":
        return {"op": op, "seqs": _log(rng, 1, 256), "tree_lo": 1, "tree": _log(rng, 1, 127)}
    d = rng.choice([64, 128, 128, 128, 256])
    hkv = rng.choice([1, 2, 4, 8, 8])
    block = rng.choice([8, 16, 16, 24, 32, 64, 256])
    fmt = rng.choice(["e4m3", "int8"])
    if op in ("store", "load"):
        tokens = _log(rng, 1, 8192)
        case = {"op": op, "fmt": fmt, "dtype": rng.choice(list(_TYPES)), "tokens": tokens, "hkv": hkv, "d": d,
                "block": block, "blocks": -(-tokens // block) + rng.randrange(1, 100)}
        return case
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    hq = hkv * rng.choice([1, 2, 3, 4, 8])
    seqs = _log(rng, 1, 64)
    # keys x heads x width stay within the largest listed decode step, and the plain form's padded copies
    # within a tenth of the card
    top = min(131071, max(64, (1 << 28) // (seqs * hkv * d)))
    if op == "decode":
        hi = _log(rng, 1, top)
        return {"op": op, "fmt": fmt, "dtype": dtype, "seqs": seqs, "lo": rng.randrange(1, hi + 1), "hi": hi, "hq": hq,
                "hkv": hkv, "d": d, "block": block}
    tree = _log(rng, 1, 128)
    hi = _log(rng, 1, max(1, min(top, (1 << 31) // (seqs * hq * tree * d // 16))))
    return {"op": op, "fmt": rng.choice([fmt, "none", "none"]), "dtype": dtype, "seqs": seqs, "lo": rng.randrange(0, hi + 1),
            "hi": hi, "tree_lo": rng.randrange(1, tree + 1), "tree": tree, "hq": hq, "hkv": hkv, "d": d, "block": block,
            "parents": rng.random() < 0.3}


# ---------------------------------------------------------------------------------------------------------------
# sizes: a case's lengths are the case's own (work() counts them); values, pages and trees come from the seed
def _lengths(case, lo, hi, what):
    r = random.Random("%s %s" % (what, sorted((k, str(v)) for k, v in case.items() if k != "name")))
    n = [r.randint(lo, hi) for _ in range(case["seqs"])]
    n[0] = hi
    return n


def _contexts(case):
    return _lengths(case, case["lo"], case["hi"], "context")


def _trees(case):
    return _lengths(case, case["tree_lo"], case["tree"], "tree")


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _values(shape, g, dtype):
    """Normal values, one in a thousand 20 times as large, as the projections' outputs have them."""
    x = torch.randn(shape, generator=g, device="cuda")
    return torch.where(torch.rand(shape, generator=g, device="cuda") < 1e-3, x * 20, x).to(dtype)


def _cache(blocks, case, g, kept):
    """One page pool of keys or values: (rows, scales), scales None where the rows are kept as they are."""
    shape = (blocks, case["hkv"], case["block"], case["d"])
    if not kept:
        return torch.randn(shape, generator=g, device="cuda", dtype=_TYPES[case["dtype"]]), None
    scales = torch.rand(shape[:3], generator=g, device="cuda") * 0.02 + 0.002
    if case["fmt"] == "int8":
        return torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8), scales
    rows = torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16).mul_(120).clamp_(-448, 448)
    return rows.to(torch.float8_e4m3fn), scales


def _parents(sizes, r):
    """Parents of every node: the one before it (a chain) half of the time, else any earlier one or none (-1)."""
    got = []
    for n in sizes:
        got += [i - 1 if r.random() < 0.5 else r.randrange(-1, i) for i in range(n)]
    return got


def prepare(case, seed):
    g, r = _generator(seed), random.Random(seed)
    if case["op"] == "mask":
        return _with_trees({"case": case}, case, r)
    if case["op"] in ("store", "load"):
        s = {"case": case}
        for x in "kv":
            s[x + "_cache"], s[x + "_scale"] = _cache(case["blocks"], case, g, True)
        at = torch.randperm(case["blocks"] * case["block"], generator=g, device="cuda")[: case["tokens"]]
        s["blocks"], s["slots"] = at // case["block"], at % case["block"]
        if case["op"] == "store":  # token-major projections, seen head-major as the store takes them
            for x in "kv":
                rows = _values((case["tokens"], case["hkv"], case["d"]), g, _TYPES[case["dtype"]])
                s[x + "_rows"] = rows.transpose(0, 1)
        return s
    contexts = _contexts(case)
    trees = _trees(case) if case["op"] == "tree" else [0] * case["seqs"]
    pages = [-(-(c + t) // case["block"]) for c, t in zip(contexts, trees)]
    total = sum(pages) + 3
    s = {"case": case}
    for x in "kv":
        s[x + "_cache"], s[x + "_scale"] = _cache(total, case, g, case["fmt"] != "none")
    order = torch.randperm(total, generator=g, device="cuda")[: sum(pages)].to(torch.int32)
    s["tables"] = torch.zeros(case["seqs"], max(1, max(pages)), dtype=torch.int32, device="cuda")
    of = torch.repeat_interleave(torch.arange(case["seqs"]), torch.tensor(pages)).cuda()
    first = torch.tensor([0] + pages).cumsum(0).cuda()
    s["tables"][of, torch.arange(sum(pages), device="cuda") - first[of]] = order
    s["lens"] = torch.tensor(contexts, dtype=torch.int32, device="cuda")
    if case["op"] == "tree":
        _with_trees(s, case, r)
    n = sum(trees) if case["op"] == "tree" else case["seqs"]
    s["q"] = torch.randn((n, case["hq"], case["d"]), generator=g, device="cuda").to(_TYPES[case["dtype"]])
    return s


def _with_trees(s, case, r):
    sizes = _trees(case)
    s["cu"] = torch.tensor([0] + sizes, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
    s["parents"] = torch.tensor(_parents(sizes, r), dtype=torch.int32, device="cuda")
    s["mask"] = _plain_mask(s)[0] if case["op"] == "tree" and not case["parents"] else None
    return s


def run(state):
    if own:
        return _own(state)
    return {"store": _plain_store, "load": _plain_load, "decode": _plain_decode, "tree": _plain_tree,
            "mask": _plain_mask}[state["case"]["op"]](state)


def _own(s):
    import tinyserver_b200 as tsb

    case = s["case"]
    if case["op"] == "mask":
        return tsb.build_tree_mask(s["parents"], s["cu"], case["tree"])
    pools = (s["k_cache"], s["v_cache"])
    scales = (s["k_scale"], s["v_scale"])
    if case["op"] == "store":
        tsb.store_kv_cache_quantized(s["k_rows"], s["v_rows"], *pools, *scales, s["blocks"], s["slots"])
        return (*pools, *scales)
    if case["op"] == "load":
        return tsb.load_kv_cache_quantized(*pools, *scales, s["blocks"], s["slots"], _TYPES[case["dtype"]])
    if case["op"] == "decode":
        return tsb.paged_attention_quantized(s["q"], *pools, *scales, s["tables"], case["block"], s["lens"])
    mask, depths = (s["mask"], None) if s["mask"] is not None else tsb.build_tree_mask(s["parents"], s["cu"], case["tree"])
    out = tsb.paged_tree_attention(s["q"], *pools, s["tables"], case["block"], s["lens"], s["cu"], mask, case["tree"],
                                   k_scale=scales[0], v_scale=scales[1])
    return out if depths is None else (out, mask, depths)


# ---------------------------------------------------------------------------------------------------------------
# the plain forms
def _bits(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def _plain_store(s):
    case = s["case"]
    top = torch.tensor(_TOP[case["fmt"]], device="cuda")
    _quantise_into(s["k_rows"], s["k_cache"], s["k_scale"], s, top)
    _quantise_into(s["v_rows"], s["v_cache"], s["v_scale"], s, top)
    return s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]


def _quantise_into(rows, cache, scales, s, top):
    x = rows.transpose(0, 1).float()
    amax = x.abs().amax(-1).clamp_min(_FLOOR)
    y = (x * torch.div(top, amax)[..., None]).clamp(-top, top)
    codes = y.round().to(torch.int8) if cache.dtype == torch.int8 else y.to(cache.dtype)
    _bits(cache)[s["blocks"], :, s["slots"]] = _bits(codes)
    scales[s["blocks"], :, s["slots"]] = torch.div(amax, top)


def _plain_load(s):
    dtype = _TYPES[s["case"]["dtype"]]
    return (_rows(s["k_cache"], s["k_scale"], s["blocks"], s["slots"]).to(dtype).transpose(0, 1),
            _rows(s["v_cache"], s["v_scale"], s["blocks"], s["slots"]).to(dtype).transpose(0, 1))


def _rows(cache, scales, blocks, slots):
    """The rows at (blocks, slots) in 32 bits: (..., heads, width)."""
    x = _bits(cache)[blocks, :, slots].view(cache.dtype).float()
    return x if scales is None else x * scales[blocks, :, slots][..., None]


def _keys(s, longest):
    """Every sequence's keys and values, padded to the longest: (sequences, heads, longest, width)."""
    at = torch.arange(longest, device="cuda")
    blocks = s["tables"][:, at // s["case"]["block"]].long()
    slots = (at % s["case"]["block"]).expand_as(blocks)
    return (_rows(s["k_cache"], s["k_scale"], blocks, slots).transpose(1, 2),
            _rows(s["v_cache"], s["v_scale"], blocks, slots).transpose(1, 2))


def _attend(q, k, v, seen):
    """softmax(q k^T / sqrt(width)) v over the keys that are seen; a row that sees none is zero."""
    x = (q @ k.transpose(-1, -2) * (1 / math.sqrt(q.shape[-1]))).masked_fill_(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = x.sub_(top.masked_fill(top == -math.inf, 0)).exp_()
    total = p.sum(-1, keepdim=True)
    return torch.where(total > 0, p @ v / total.clamp_min(1e-30), 0)


def _plain_decode(s):
    case = s["case"]
    k, v = _keys(s, case["hi"])
    q = s["q"].float().view(case["seqs"], case["hkv"], -1, case["d"])
    seen = torch.arange(case["hi"], device="cuda") < s["lens"][:, None]
    return _attend(q, k, v, seen[:, None, None]).reshape(s["q"].shape).to(s["q"].dtype)


def _where(s):
    """(sequence, place within its tree) of every drafted token."""
    cu = s["cu"].long()
    t = torch.arange(s["parents"].numel(), device="cuda")
    of = torch.searchsorted(cu[1:], t, right=True)
    return of, t - cu[of]


def _plain_mask(s):
    """Bit i of a node's row: node i of its tree is the node itself or above it.  The relation "parent or self",
    squared until it spans the deepest tree.  Also each node's depth."""
    case = s["case"]
    n = case["tree"]
    of, at = _where(s)
    above = torch.zeros(case["seqs"], n, n, device="cuda")
    above[of, at, at] = 1
    inner = s["parents"] >= 0
    above[of, at, s["parents"].clamp_min(0).long()] += inner.float()
    for _ in range(max(1, (n - 1).bit_length())):
        above = (above @ above).clamp_max(1)
    sees = above[of, at].long()
    words = torch.nn.functional.pad(sees, (0, -n % 64)).view(sees.shape[0], -1, 64)
    mask = (words << torch.arange(64, device="cuda")).sum(-1)
    return mask, sees.sum(-1).sub(1).to(torch.int32)


def _plain_tree(s):
    case = s["case"]
    mask, depths = (s["mask"], None) if s["mask"] is not None else _plain_mask(s)
    longest = case["hi"] + case["tree"]
    longest = min(longest, s["tables"].shape[1] * case["block"])
    k, v = _keys(s, longest)
    of, at = _where(s)
    q = torch.zeros(case["seqs"], case["tree"], case["hq"], case["d"], device="cuda")
    q[of, at] = s["q"].float()
    group = case["hq"] // case["hkv"]
    q = q.view(case["seqs"], case["tree"], case["hkv"], group, case["d"]).transpose(1, 2).flatten(2, 3)
    key = torch.arange(longest, device="cuda")
    lens = s["lens"].long()
    node = key - lens[:, None]  # (sequences, longest): which node of the tree a key is
    bits = torch.zeros(case["seqs"], case["tree"], mask.shape[1], dtype=torch.int64, device="cuda")
    bits[of, at] = mask
    word = (node.clamp_min(0) // 64).clamp_max(mask.shape[1] - 1)[:, None].expand(-1, case["tree"], -1)
    bit = (bits.gather(2, word) >> (node.clamp_min(0) % 64)[:, None]) & 1
    size = (s["cu"][1:] - s["cu"][:-1]).long()
    seen = (node < 0)[:, None] | ((node < size[:, None])[:, None] & (bit == 1))
    seen = seen[:, None, :, None].expand(-1, 1, -1, group, -1).flatten(2, 3)
    out = _attend(q, k, v, seen)
    out = out.view(case["seqs"], case["hkv"], case["tree"], group, case["d"]).transpose(1, 2).flatten(2, 3)
    out = out[of, at].to(s["q"].dtype)
    return out if depths is None else (out, mask, depths)


# ---------------------------------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "mask":
        n = sum(_trees(case))
        return {"bytes": n * (4 + 4 + 8 * -(-case["tree"] // 64)) + 4 * (case["seqs"] + 1), "flops": 0}
    wide = _TYPES[case["dtype"]].itemsize
    if op in ("store", "load"):  # K and V: rows of the type, codes, scales; block and slot of each token
        row = case["d"] * wide + case["d"] + 4
        return {"bytes": case["tokens"] * (2 * case["hkv"] * row + 16), "flops": 0}
    contexts = _contexts(case)
    trees = _trees(case) if op == "tree" else [0] * case["seqs"]
    row = case["d"] * wide if case["fmt"] == "none" else case["d"] + 4
    keys = sum(contexts) + sum(trees)
    queries = sum(trees) if op == "tree" else case["seqs"]
    moved = 2 * keys * case["hkv"] * row + 2 * queries * case["hq"] * case["d"] * wide
    pages = sum(-(-(c + t) // case["block"]) for c, t in zip(contexts, trees))
    moved += 4 * pages + 4 * case["seqs"]
    pairs = sum((c + t) * max(1, t) for c, t in zip(contexts, trees))
    if op == "tree":
        moved += sum(trees) * 8 * -(-case["tree"] // 64) + (8 * sum(trees) if case["parents"] else 0)
    return {"bytes": moved, "flops": 4 * pairs * case["hq"] * case["d"]}


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits, sequence by sequence
def _nearest_e4m3(y):
    """The nearest value with 4 significant bits, exponents from -6 (steps of 2^-9 below it), ties to even."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(y / step) * step).clamp(-448, 448)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "mask":
        return None
    if case["op"] == "store":
        got = []
        for x in "kv":
            src = s[x + "_rows"].double().permute(1, 0, 2)
            amax = torch.maximum(src.abs().max(-1).values, torch.tensor(_FLOOR, dtype=torch.float64, device="cuda"))
            scales = s[x + "_scale"].double()
            scales[s["blocks"], :, s["slots"]] = amax / _TOP[case["fmt"]]
            if case["fmt"] == "int8":
                got.append((None, scales))
                continue
            codes = s[x + "_cache"].double()
            codes[s["blocks"], :, s["slots"]] = _nearest_e4m3(src / (amax / 448.0)[..., None])
            got.append((codes, scales))
        return got[0][0], got[1][0], got[0][1], got[1][1]

    def dense(x, blocks, slots):
        rows = s[x + "_cache"]
        rows = rows.view(torch.uint8)[blocks, :, slots].view(rows.dtype) if rows.element_size() == 1 else rows[blocks, :, slots]
        rows = rows.double()
        return rows if s[x + "_scale"] is None else rows * s[x + "_scale"][blocks, :, slots].double().unsqueeze(-1)

    if case["op"] == "load":
        return tuple(dense(x, s["blocks"], s["slots"]).permute(1, 0, 2) for x in "kv")
    contexts = _contexts(case)
    trees = _trees(case) if case["op"] == "tree" else [1] * case["seqs"]
    drafted = trees if case["op"] == "tree" else [0] * case["seqs"]
    group = case["hq"] // case["hkv"]
    parents = s["parents"].tolist() if case["op"] == "tree" else []
    out, begin = [], 0
    for i in range(case["seqs"]):
        total, n = contexts[i] + drafted[i], trees[i]
        at = torch.arange(total, device="cuda")
        blocks, slots = s["tables"][i].long()[at // case["block"]], at % case["block"]
        k, v = dense("k", blocks, slots), dense("v", blocks, slots)
        q = s["q"][begin:begin + n].double()
        sees = torch.ones(n, total, dtype=torch.bool)
        for t in range(drafted[i]):
            sees[t, contexts[i]:] = False
            node = t
            while node >= 0:
                sees[t, contexts[i] + node] = True
                node = parents[begin + node]
        sees = sees.cuda()
        heads = []
        for h in range(case["hkv"]):
            scores = torch.einsum("tgd,jd->tgj", q[:, h * group:(h + 1) * group], k[:, h]) / math.sqrt(case["d"])
            w = torch.softmax(scores.masked_fill(~sees[:, None], -math.inf), -1)
            heads.append(torch.einsum("tgj,jd->tgd", w, v[:, h]))
        out.append(torch.cat(heads, 1))
        begin += n
    out = torch.cat(out)
    return (out, None, None) if case["op"] == "tree" and case["parents"] else out
