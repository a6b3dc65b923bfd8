"""Plain forms of the quantised cache and of attention for drafted token trees, in
64 bits, and the error bounds their kernels are held to.

The bound of an attention output is counted from its roundings.  With u the half
step (eps / 2) of a type, A = sum_j p_j |v_j| and E = max_j sum_d |q_d k_jd| *
scale for the row:
* the output's own rounding: u_out * |out|;
* the products' probabilities, held in the operand type by the tcgen05 kernel:
  u_p * A (the other kernels keep a remainder, u_p**2, and are well inside);
* the scores: D products and as many sums in fp32, a factor or two, and the
  exponential of a number up to ~100: (D + 8) * 2**-24 * E absolute in the
  exponent, and 2**-16 relative for exp2 / log2 of such numbers, which numerator
  and denominator both carry;
* the sums over L keys in fp32: L * 2**-24 each.
"""

import math

import torch

TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
FORMATS = (torch.float8_e4m3fn, torch.int8)


def quantise(rows, fmt):
    """(codes, scales) of (..., D) rows on the CPU in IEEE fp32, the definition's own order."""
    x = rows.float().cpu()
    top = torch.tensor(TOP[fmt])
    amax = x.abs().amax(-1)
    bad = ~torch.isfinite(x).all(-1)
    amax = torch.where(bad, torch.ones_like(amax), amax).clamp_min(2.0 ** -100)
    scales = torch.div(amax, top.expand_as(amax))
    y = (x * torch.div(top.expand_as(amax), amax)[..., None]).clamp(-top, top)
    y = torch.where(bad[..., None], torch.zeros_like(y), y)
    codes = y.round().to(torch.int8) if fmt == torch.int8 else y.to(fmt)
    return codes, torch.where(bad, torch.full_like(scales, float("nan")), scales)


def mask_of(parents, sizes, max_tree):
    """(mask, depths) by walking every node's parents."""
    words = (max_tree + 63) // 64
    mask, depths, at = [], [], 0
    for n in sizes:
        for i in range(n):
            row, node, depth = [0] * words, i, -1
            while node >= 0:
                row[node // 64] |= 1 << (node % 64)
                node, depth = int(parents[at + node]), depth + 1
            mask.append([x - (1 << 64) if x >> 63 else x for x in row])
            depths.append(depth)
        at += n
    return (torch.tensor(mask, dtype=torch.int64).view(-1, words),
            torch.tensor(depths, dtype=torch.int32))


def random_parents(sizes, g):
    got = []
    for n in sizes:
        for i in range(n):
            chain = bool(torch.rand((), generator=g) < 0.5)
            got.append(i - 1 if chain else int(torch.randint(-1, i, (), generator=g)) if i else -1)
    return torch.tensor(got, dtype=torch.int32)


def attention(q, k_cache, v_cache, tables, block, contexts, sizes=None, mask=None, k_scale=None,
              v_scale=None, scale=None, p_type=None):
    """(out, bound) in 64 bits, sequence by sequence on q's device.  ``sizes`` None: decode."""
    D, Hq, Hkv = q.shape[2], q.shape[1], k_cache.shape[1]
    group = Hq // Hkv
    scale = 1 / math.sqrt(D) if scale is None else scale
    u_out = torch.finfo(q.dtype).eps / 2
    u_p = torch.finfo(p_type or q.dtype).eps / 2 if q.dtype != torch.float32 else 0.0
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    begin = 0

    def dense(cache, sc, blocks, slots):
        rows = cache.view(torch.uint8)[blocks, :, slots].view(cache.dtype) \
            if cache.element_size() == 1 else cache[blocks, :, slots]
        rows = rows.double()
        return rows if sc is None else rows * sc[blocks, :, slots].double()[..., None]

    for s, ctx in enumerate(contexts):
        n = 1 if sizes is None else sizes[s]
        L = ctx + (0 if sizes is None else n)
        if n and L:
            at = torch.arange(L, device=q.device)
            blocks, slots = tables[s].long()[at // block], at % block
            k, v = (dense(c, sc, blocks, slots) for c, sc in ((k_cache, k_scale), (v_cache, v_scale)))
            qs = q[begin:begin + n].double().view(n, Hkv, group, D)
            x = torch.einsum("thgd,jhd->thgj", qs, k) * scale
            e = torch.einsum("thgd,jhd->thgj", qs.abs(), k.abs()) * abs(scale)
            if sizes is not None:
                seen = torch.ones(n, L, dtype=torch.bool, device=q.device)
                node = torch.arange(n, device=q.device)
                bits = mask[begin:begin + n].to(q.device)
                seen[:, ctx:] = ((bits[:, node // 64] >> (node % 64)) & 1).bool()
            else:
                seen = torch.ones(n, L, dtype=torch.bool, device=q.device)
            sm = seen[:, None, None, :].expand_as(x)
            x = x.masked_fill(~sm, -math.inf)
            top = x.amax(-1, keepdim=True)
            p = torch.where(sm, torch.exp(x - torch.where(top == -math.inf, 0.0, top)), 0.0)
            total = p.sum(-1, keepdim=True)
            p = torch.where(total == 0, torch.zeros_like(p), p / total)

            def times_v(weights, values):  # unseen keys left out whatever they hold
                if torch.isfinite(values).all():
                    return torch.einsum("thgj,jhd->thgd", weights, values)
                got = torch.zeros(n, Hkv, group, D, dtype=torch.float64, device=q.device)
                for t in range(n):
                    js = seen[t].nonzero()[:, 0]
                    got[t] = torch.einsum("hgj,jhd->hgd", weights[t][:, :, js], values[js])
                return got

            o = times_v(p, v)
            a = times_v(p, v.abs())
            worst = torch.where(sm, e, 0.0).amax(-1, keepdim=True)
            c = 2 * ((D + 8) * 2.0 ** -24 * worst + 2.0 ** -16 + L * 2.0 ** -24)
            out[begin:begin + n] = o.reshape(n, Hq, D)
            bound[begin:begin + n] = (u_out * o.abs() + (u_p + c) * (1 + u_out) * a).reshape(n, Hq, D)
        begin += n
    return out, bound


def assert_within(actual, out, bound, what=""):
    """Every element within its bound; NaN exactly where the definition has NaN."""
    a, tiny = actual.double(), torch.finfo(actual.dtype).smallest_normal
    nan = torch.isnan(out)
    assert torch.equal(torch.isnan(a), nan), f"{what}: NaN in other places"
    inf = torch.isinf(out)
    assert torch.equal(a[inf], out[inf]), f"{what}: infinities"
    fine = ~(nan | inf)
    off = (a - out).abs()[fine] - bound[fine] - tiny
    assert off.numel() == 0 or float(off.max()) <= 0, (
        f"{what}: {int((off > 0).sum())} of {off.numel()} outside, worst by {float(off.max()):.3g}; "
        f"max error {float((a - out).abs()[fine].max()):.3g}")
