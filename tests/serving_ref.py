"""Plain 64-bit forms of the serving-step operators, request by request, and the
tolerances that follow from the kernels' arithmetic."""
from __future__ import annotations

import torch

PAGE, D = 16, 128
HALF_BF16 = 2.0 ** -8          # half a step of bf16, relative
INF = float("inf")


def plan(lens, new, table, free, taken, cap, page=PAGE):
    """Python integers and lists; returns what the device call leaves."""
    table = [list(r) for r in table]
    cu, slots, pos, out = [0], [-1] * cap, [0] * cap, []
    refused = False
    upto = 0                       # blocks the served and the refused takers ask for
    last = 0
    for r, (length, n) in enumerate(zip(lens, new)):
        length, n = max(length, 0), max(n, 0)
        t0 = cu[-1]
        cu.append(t0 + n)
        old, end = -(-length // page), -(-(length + n) // page)
        fits = end <= len(table[r]) and t0 + n <= cap
        need = end - old if fits else 0
        upto += need
        ok = fits and (need == 0 or taken + upto <= len(free))
        refused |= not ok
        if ok and need:
            for j in range(need):
                table[r][old + j] = free[taken + upto - need + j]
            last = upto
        for i in range(n):
            if t0 + i < cap:
                pos[t0 + i] = length + i
                if ok:
                    b = table[r][(length + i) // page]
                    slots[t0 + i] = b * page + (length + i) % page if b >= 0 else -1
        out.append(length + n if ok else length)
    return dict(cu=cu, slots=slots, pos=pos, lens=out, taken=taken + last, table=table,
                refused=refused)


def norm_rope(x, weight, eps, cs, rot, neox):
    """x (T, h, d) -> fp64; cs (T, rot) cos half | sin half or None."""
    x = x.double()
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    if cs is None:
        return x
    y, half = x.clone(), rot // 2
    for j in range(half):
        a, b = (j, j + half) if neox else (2 * j, 2 * j + 1)
        c, s = cs[:, None, j].double(), cs[:, None, half + j].double()
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def attend(q, k, v, seen, scale):
    """q (n, H, d), k and v (j, n_kv, d), seen (n, j).  Returns out, lse, the
    weighted mean of |v| and the largest sum of |q_d k_d| * scale of a row."""
    n, H, d = q.shape
    G = H // k.shape[1]
    q = q.double()
    k, v = (t.double().repeat_interleave(G, 1) for t in (k, v))
    x = torch.einsum("nhd,jhd->nhj", q, k) * scale
    size = torch.einsum("nhd,jhd->nhj", q.abs(), k.abs()) * abs(scale)
    hidden = ~seen[:, None].expand_as(x)
    x = x.masked_fill(hidden, -INF)
    size = size.masked_fill(hidden, 0.0)
    m = x.amax(-1, keepdim=True) if x.shape[-1] else x.new_full((n, H, 1), -INF)
    p = torch.exp(x - m.clamp(min=-1e300))
    s = p.sum(-1, keepdim=True)
    w = torch.where(s > 0, p / s.clamp(min=1e-300), 0.0)
    out, mean = torch.einsum("nhj,jhd->nhd", w, v), torch.einsum("nhj,jhd->nhd", w, v.abs())
    lse = torch.where(s > 0, m + s.clamp(min=1e-300).log(), -INF)[..., 0]
    return out, lse, mean, size.amax(-1) if x.shape[-1] else size.new_zeros(n, H)


def gather(plane, row, n):
    """First n tokens of a table row from a (NB, page, n_kv, d) plane."""
    j = torch.arange(n, device=plane.device)
    return plane[row.long()[j // PAGE], j % PAGE]


def out_tolerance(out, mean, size):
    """|error| of a bf16 output: half a step for its own rounding, and for the
    weights one more half step (they meet V in bf16) plus their relative error.
    A score is a sum of 128 fp32 products: at most 130 roundings of 2^-24 of the sum
    of magnitudes; scaling, the running maximum and exp2 add 2^-20.  Numerator and
    denominator both carry it: twice."""
    score = 130 * 2.0 ** -24 * size[..., None] + 2.0 ** -20
    return HALF_BF16 * out.abs() + (HALF_BF16 + 2 * score) * mean * (1 + HALF_BF16) + 1e-30


def lse_tolerance(lse, size):
    return 130 * 2.0 ** -24 * size + 2.0 ** -20 + lse.abs().clamp(max=1e9) * 2.0 ** -21
