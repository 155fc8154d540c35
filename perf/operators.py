"""Workloads of the serving-step operators around the paged KV cache: their inputs, their plain form and
their definition in 64 bits.

  plan     slots, positions, block-table entries and lengths of a step's new tokens, from request lengths
  norm     RMS norm of every query and key head, position rotation, K and V into the paged cache
  window   attention over the paged cache with a sliding window and a few first tokens that stay visible
  prefix   single-token attention of a batch whose requests share long prefixes

`run` computes the plain form with elementary torch operations where `own` is false, and calls the
framework where it is true.  Cache geometry: pages of 16 tokens, heads of 128 channels, bf16.
"""
import math
import os
import random
import sys

import torch

own = False

PAGE, D = 16, 128
SCALE = D ** -0.5
ROPE_THETA = 500000.0


# ---- cases ------------------------------------------------------------------------------------
def listed():
    return [
        # one token for each of a few requests: the bookkeeping of a small decode step (latency)
        dict(name="plan_decode", op="plan", reqs=16, new_lo=1, new_hi=1, len_lo=0, len_hi=131072, pad=0, layout=1),
        # prompts of many requests arriving at once, ragged, with padding behind the last token
        dict(name="plan_prompts", op="plan", reqs=256, new_lo=0, new_hi=512, len_lo=0, len_hi=4096, pad=1000, layout=2),
        # the single-token call of a decode step of one request
        dict(name="norm_decode", op="norm", tokens=1, n_kv=8, G=4, rot=128, neox=True, f32=False, skip=0, layout=3),
        # a prompt chunk with an odd token count, a few tokens without a slot
        dict(name="norm_chunk", op="norm", tokens=2053, n_kv=8, G=4, rot=128, neox=True, f32=False, skip=5, layout=4),
        # a large prefill step, two KV heads, half of the channels rotated in interleaved pairs, 32-bit weights
        dict(name="norm_prefill", op="norm", tokens=16384, n_kv=2, G=16, rot=64, neox=False, f32=True, skip=0, layout=5),
        # one request at 128K tokens decoding with a 4096-token window (latency)
        dict(name="window_decode", op="window", reqs=1, q_lo=1, q_hi=1, len_lo=131072, len_hi=131072, window=4096, sinks=4, n_kv=8, G=4, layout=6),
        # a ragged decode batch of the benchmark's range of lengths
        dict(name="window_decode_batch", op="window", reqs=64, q_lo=1, q_hi=1, len_lo=4096, len_hi=262144, window=2048, sinks=16, n_kv=8, G=4, layout=7),
        # a step that mixes single tokens and odd chunks, eight query heads on each KV head
        dict(name="window_mixed", op="window", reqs=33, q_lo=1, q_hi=193, len_lo=200, len_hi=5000, window=1000, sinks=5, n_kv=2, G=8, layout=8),
        # a whole prompt: the attention-bound end of the range
        dict(name="window_prompt", op="window", reqs=1, q_lo=8192, q_hi=8192, len_lo=8192, len_hi=8192, window=4096, sinks=4, n_kv=8, G=4, layout=9),
        # a few requests behind a short common prompt (latency)
        dict(name="prefix_few", op="prefix", groups=1, reqs=4, pre_lo=1000, pre_hi=1000, suf_lo=1, suf_hi=40, n_kv=2, G=8, layout=10),
        # a batch that shares one long document
        dict(name="prefix_document", op="prefix", groups=1, reqs=64, pre_lo=32768, pre_hi=32768, suf_lo=16, suf_hi=1024, n_kv=8, G=4, layout=11),
        # three groups with prefixes of their own, ends inside a page, sixteen query heads on each KV head
        dict(name="prefix_groups", op="prefix", groups=3, reqs=96, pre_lo=4000, pre_hi=16500, suf_lo=1, suf_hi=500, n_kv=2, G=16, layout=12),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    layout = rng.randrange(1 << 30)
    op = rng.choice(["plan", "norm", "window", "window", "prefix", "prefix"])
    n_kv, G = rng.choice([(8, 4), (2, 8), (2, 16), (4, 4), (8, 1), (4, 5), (2, 3), (1, 12), (4, 2)])
    if op == "plan":
        new_hi = _log_int(rng, 1, 512)
        return dict(op=op, reqs=_log_int(rng, 1, 256), new_lo=rng.choice([0, 1]), new_hi=new_hi, len_lo=0,
                    len_hi=_log_int(rng, 16, 131072), pad=rng.choice([0, 0, rng.randrange(1, 500)]), layout=layout)
    if op == "norm":
        return dict(op=op, tokens=_log_int(rng, 1, 16384 * 36 // (n_kv * (G + 2))), n_kv=n_kv, G=G, rot=rng.choice([128, 64, 32, 96, 20]),
                    neox=rng.choice([True, False]), f32=rng.choice([True, False]), skip=rng.choice([0, 0, 1, 3]), layout=layout)
    if op == "window":
        # (a padded plain form holds reqs x heads x longest query x visible keys in 32 bits)
        while True:
            reqs, q_hi = _log_int(rng, 1, 64), rng.choice([1, 1, _log_int(rng, 2, 8192)])
            window, sinks = _log_int(rng, 64, 8192), rng.choice([0, 1, 4, 16, 37, 128])
            len_hi = max(q_hi, _log_int(rng, 16, 131072))
            keys = sinks + min(len_hi, window + q_hi - 1)
            if reqs * n_kv * G * q_hi * keys <= 2 ** 31 and reqs * keys * n_kv <= 2 ** 20 * 2:
                break
        return dict(op=op, reqs=reqs, q_lo=1 if q_hi < 512 else q_hi // 2, q_hi=q_hi, len_lo=max(1, len_hi // 16), len_hi=len_hi,
                    window=window, sinks=sinks, n_kv=n_kv, G=G, layout=layout)
    while True:
        groups, reqs = rng.choice([1, 1, 2, 3, 5]), _log_int(rng, 2, 128)
        pre_hi, suf_hi = _log_int(rng, 32, 32768), _log_int(rng, 1, 1024)
        if groups <= reqs and groups * pre_hi * reqs * n_kv * G <= 2 ** 27 and groups * pre_hi * n_kv <= 2 ** 18 and reqs * suf_hi * n_kv <= 2 ** 19:
            return dict(op=op, groups=groups, reqs=reqs, pre_lo=max(1, pre_hi // 4), pre_hi=pre_hi, suf_lo=1, suf_hi=suf_hi, n_kv=n_kv, G=G, layout=layout)


# ---- lengths and layouts: fixed by the case -----------------------------------------------------
def _plan_lens(case):
    r = random.Random(case["layout"])
    lens = [r.randint(case["len_lo"], case["len_hi"]) for _ in range(case["reqs"])]
    new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(case["reqs"])]
    return lens, new


def _window_lens(case):
    r = random.Random(case["layout"])
    n_q, lens = [], []
    for _ in range(case["reqs"]):
        n_q.append(_log_int(r, case["q_lo"], case["q_hi"]))
        lens.append(max(n_q[-1], _log_int(r, case["len_lo"], case["len_hi"])))
    return n_q, lens


def _prefix_lens(case):
    r = random.Random(case["layout"])
    cuts = sorted(r.sample(range(1, case["reqs"]), case["groups"] - 1)) if case["groups"] > 1 else []
    cu = [0] + cuts + [case["reqs"]]
    pre = [_log_int(r, case["pre_lo"], case["pre_hi"]) for _ in range(case["groups"])]
    lens = []
    for g in range(case["groups"]):
        lens += [pre[g] + _log_int(r, case["suf_lo"], case["suf_hi"]) for _ in range(cu[g + 1] - cu[g])]
    return cu, pre, lens


def _visible(p, window, sinks):
    """How many keys the query at position p sees: positions up to p that are recent or among the first."""
    lo = max(p - window + 1, 0)
    return p + 1 - lo + min(sinks, lo)


def work(case):
    op = case["op"]
    if op == "plan":
        lens, new = _plan_lens(case)
        fresh = sum(-(-(a + b) // PAGE) + -a // PAGE for a, b in zip(lens, new))
        return {"bytes": 16 * (sum(new) + case["pad"]) + 20 * case["reqs"] + 8 * fresh, "flops": 0}
    if op == "norm":
        t, h, n_kv = case["tokens"], case["n_kv"] * case["G"], case["n_kv"]
        rows = 2 * D * (h + 2 * n_kv)
        return {"bytes": t * (2 * rows + case["rot"] * (4 if case["f32"] else 2) + 16), "flops": t * (h + n_kv) * (4 * D + 3 * case["rot"])}
    n_kv, h = case["n_kv"], case["n_kv"] * case["G"]
    if op == "window":
        n_q, lens = _window_lens(case)
        w, s = case["window"], case["sinks"]
        seen = sum(_visible(p, w, s) for n, l in zip(n_q, lens) for p in range(l - n, l))
        keys = 0
        for n, l in zip(n_q, lens):
            lo = max(l - n - w + 1, 0)
            keys += l - lo + min(s, lo)
        return {"bytes": sum(n_q) * h * (4 * D + 4) + keys * n_kv * 4 * D, "flops": 4 * D * h * seen}
    cu, pre, lens = _prefix_lens(case)
    own_keys = sum(lens[r] - pre[g] for g in range(case["groups"]) for r in range(cu[g], cu[g + 1]))
    return {"bytes": case["reqs"] * h * (4 * D + 4) + (sum(pre) + own_keys) * n_kv * 4 * D, "flops": 4 * D * h * sum(lens)}


# ---- inputs -------------------------------------------------------------------------------------
def _cache(gen, blocks, n_kv):
    """A paged cache (blocks, K | V, 16, n_kv, 128): unit normal, four loud key channels a head, as rotated keys have."""
    c = torch.randn(blocks, 2, PAGE, n_kv, D, generator=gen, device="cuda", dtype=torch.bfloat16)
    loud = torch.ones(n_kv, D, device="cuda")
    at = torch.rand(n_kv, D, generator=gen, device="cuda").argsort(1)[:, :4]
    loud.scatter_(1, at, 8.0)
    c[:, 0] *= loud.to(torch.bfloat16)
    return c


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _angles(rows, rot):
    inv = ROPE_THETA ** (-torch.arange(rot // 2, device="cuda", dtype=torch.float64) * 2 / rot)
    a = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], 1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op = case["op"]
    s = dict(op=op)
    if op == "plan":
        lens, new = _plan_lens(case)
        wide = (case["len_hi"] + case["new_hi"]) // PAGE + 2
        pages = sum(-(-a // PAGE) for a in lens)
        fresh = sum(-(-(a + b) // PAGE) for a, b in zip(lens, new)) - pages
        ids = torch.randperm(pages + fresh + 7, generator=gen, device="cuda").to(torch.int32) + 1
        col = torch.arange(wide, device="cuda")
        used = col < torch.tensor([-(-a // PAGE) for a in lens], device="cuda")[:, None]
        s["table"] = torch.full((case["reqs"], wide), -1, dtype=torch.int32, device="cuda")
        s["table"][used] = ids[:pages]
        # the free list, some of it taken already
        s["free"] = ids[pages:].contiguous()
        s["taken"] = _i32([3])
        s["lens"], s["new"] = _i32(lens), _i32(new)
        s["tokens"] = sum(new) + case["pad"]
        s["width"], s["reqs"] = wide, case["reqs"]
        s["out"] = dict(slots=torch.empty(s["tokens"], dtype=torch.int64, device="cuda"), positions=torch.empty(s["tokens"], dtype=torch.int64, device="cuda"),
                        cu=torch.empty(case["reqs"] + 1, dtype=torch.int32, device="cuda"), lens=torch.empty(case["reqs"], dtype=torch.int32, device="cuda"),
                        taken=torch.empty(1, dtype=torch.int32, device="cuda"))
        return s
    n_kv, G = case["n_kv"], case["G"]
    h = n_kv * G
    s.update(n_kv=n_kv, G=G)
    if op == "norm":
        t, rot = case["tokens"], case["rot"]
        kind = torch.float32 if case["f32"] else torch.bfloat16
        # the projection's output: queries, keys and values of a token side by side
        qkv = torch.randn(t, h + 2 * n_kv, D, generator=gen, device="cuda", dtype=torch.bfloat16)
        s["q"], s["k"], s["v"] = qkv[:, :h], qkv[:, h:h + n_kv], qkv[:, h + n_kv:]
        s["q_weight"] = (1 + 0.2 * torch.randn(D, generator=gen, device="cuda")).to(kind)
        s["k_weight"] = (1 + 0.2 * torch.randn(D, generator=gen, device="cuda")).to(kind)
        first = random.Random(case["layout"]).randrange(0, 4096)
        s["cos_sin"] = _angles(first + t + 1, rot).to(kind)
        s["positions"] = torch.arange(first, first + t, device="cuda")
        blocks = -(-t // PAGE) + 3
        s["cache"] = _cache(gen, blocks, n_kv)
        # scattered slots; block 0 belongs to nobody (what has no slot is sent there by the plain form)
        slots = torch.randperm((blocks - 1) * PAGE, generator=gen, device="cuda")[:t] + PAGE
        slots[t - min(case["skip"], t):] = -1
        s["slots"], s["neox"], s["rot"], s["eps"] = slots, case["neox"], rot, 1e-6
        s["out"] = torch.empty(t, h, D, device="cuda", dtype=torch.bfloat16)
        return s
    if op == "window":
        n_q, lens = _window_lens(case)
        w, sk = case["window"], case["sinks"]
        reqs, wide = case["reqs"], -(-max(lens) // PAGE)
        # pages that no query of the step sees are gone: their entries name a page of somebody else
        live = torch.zeros(reqs, wide, dtype=torch.bool)
        for r in range(reqs):
            live[r, max(lens[r] - n_q[r] - w + 1, 0) // PAGE:-(-lens[r] // PAGE)] = True
            live[r, :min(-(-sk // PAGE), -(-lens[r] // PAGE))] = True
        blocks = max(int(live.sum()) + 1, 3)
        live = live.cuda()
        s["table"] = torch.randint(0, blocks, (reqs, wide), generator=gen, device="cuda", dtype=torch.int32)
        s["table"][live] = torch.randperm(blocks, generator=gen, device="cuda")[:int(live.sum())].to(torch.int32)
        s["cache"] = _cache(gen, blocks, n_kv)
        cu = [0]
        for n in n_q:
            cu.append(cu[-1] + n)
        s.update(cu=_i32(cu), lens=_i32(lens), window=w, sinks=sk, max_q=max(n_q), max_len=max(lens))
        s["q"] = torch.randn(cu[-1], h, D, generator=gen, device="cuda", dtype=torch.bfloat16)
    else:
        cu, pre, lens = _prefix_lens(case)
        reqs, wide = case["reqs"], -(-max(lens) // PAGE)
        table = torch.zeros(reqs, wide, dtype=torch.int64)
        n = 0
        for g in range(case["groups"]):
            whole = pre[g] // PAGE      # whole pages are shared; the page in which the prefix ends is copied
            table[cu[g]:cu[g + 1], :whole] = torch.arange(n, n + whole)
            n += whole
            for r in range(cu[g], cu[g + 1]):
                m = -(-lens[r] // PAGE) - whole
                table[r, whole:whole + m] = torch.arange(n, n + m)
                n += m
        s["table"] = torch.randperm(n, generator=gen, device="cuda").to(torch.int32)[table.cuda()]
        s["cache"] = _cache(gen, max(n, 3), n_kv)
        first = torch.tensor(cu[:-1], device="cuda")
        group = torch.bucketize(torch.arange(reqs, device="cuda"), torch.tensor(cu[1:], device="cuda"), right=True)
        # the copied part of a prefix's last page holds the same tokens in every request of the group
        tail = torch.tensor(pre, device="cuda")
        blk = s["table"].gather(1, (tail[group] // PAGE).clamp(max=wide - 1)[:, None])[:, 0].long()
        src = blk[first[group]]
        common = (torch.arange(PAGE, device="cuda") < (tail[group] % PAGE)[:, None])[:, None, :, None, None]
        s["cache"][blk] = torch.where(common, s["cache"][src], s["cache"][blk])
        s.update(cu=_i32(cu), pre=_i32(pre), lens=_i32(lens), max_pre=max(pre), max_own=max(lens[r] - pre[g] for g in range(case["groups"]) for r in range(cu[g], cu[g + 1])),
                 max_rows=max(b - a for a, b in zip(cu, cu[1:])), max_len=max(lens))
        s["q"] = torch.randn(reqs, h, D, generator=gen, device="cuda", dtype=torch.bfloat16)
    s["out"] = torch.empty_like(s["q"])
    s["lse"] = torch.empty(s["q"].shape[:2], device="cuda", dtype=torch.float32)
    # what a step's split partials go to: as large as any step of this shape asks for
    s["scratch"] = torch.empty(16 * 2 ** 20, device="cuda", dtype=torch.float32)
    return s


# ---- the plain form -------------------------------------------------------------------------------
def _plain_plan(s):
    old, new = (s["lens"].long() + PAGE - 1) // PAGE, (s["lens"].long() + s["new"] + PAGE - 1) // PAGE
    fits = new <= s["width"]
    need = torch.where(fits, new - old, 0)
    upto = need.cumsum(0)
    granted = fits & ((need == 0) | (s["taken"] + upto <= s["free"].shape[0]))
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device="cuda"), s["new"].long().cumsum(0)])
    t = torch.arange(s["tokens"], device="cuda")
    r = torch.bucketize(t, cu[1:], right=True).clamp(max=s["reqs"] - 1)
    inside = t < cu[-1]
    live = inside & granted[r]
    pos = torch.where(inside, s["lens"][r] + t - cu[r], 0)
    page = pos // PAGE
    fresh = page - old[r]
    blk = torch.where(fresh >= 0, s["free"][(s["taken"] + (upto - need)[r] + fresh).clamp(0, s["free"].shape[0] - 1)],
                      s["table"][r, page.clamp(max=s["width"] - 1)])
    slots = torch.where(live, blk.long() * PAGE + pos % PAGE, -1)
    entry = torch.where(live & (fresh >= 0) & (pos % PAGE == 0), r * s["width"] + page, s["reqs"] * s["width"])
    table = torch.cat([s["table"].reshape(-1), s["table"].new_zeros(1)])
    table[entry] = blk.to(torch.int32)
    lens = torch.where(granted, s["lens"] + s["new"], s["lens"])
    taken = s["taken"] + torch.where(granted, upto, 0).max().to(torch.int32)
    return dict(slots=slots, positions=pos, cu=cu.to(torch.int32), lens=lens, taken=taken.to(torch.int32), table=table[:-1].view(s["reqs"], s["width"]))


def _plain_norm_rotate(x, weight, s):
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * weight.float()
    half = s["rot"] // 2
    cs = s["cos_sin"][s["positions"]].float()[:, None]
    c, n = cs[..., :half], cs[..., half:]
    if s["neox"]:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat([a * c - b * n, b * c + a * n], -1)
    else:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)
    return torch.cat([turned, x[..., 2 * half:]], -1)


def _plain_norm(s):
    q = _plain_norm_rotate(s["q"], s["q_weight"], s).to(torch.bfloat16)
    k = _plain_norm_rotate(s["k"], s["k_weight"], s).to(torch.bfloat16)
    at = s["slots"].clamp(min=0)
    here = (s["slots"] >= 0)[:, None, None]
    blk, tok, cache = at // PAGE, at % PAGE, s["cache"]
    cache[blk, 0, tok] = torch.where(here, k, cache[blk, 0, tok])
    cache[blk, 1, tok] = torch.where(here, s["v"], cache[blk, 1, tok])
    return dict(q=q, cache=cache)


def _rows(table, keys):
    """Block and token of key positions `keys` (rows, n) of the table's rows; positions behind the table read its last column."""
    page = (keys // PAGE).clamp(0, table.shape[1] - 1)
    return table.gather(1, page).long(), keys % PAGE


def _plain_attend(q, cache, blk, tok, seen, n_kv):
    """q (rows, n, heads, 128) over keys (rows, j): maximum, sum and weighted values of the softmax, 32 bits throughout."""
    rows, n, h, _ = q.shape
    k, v = cache[blk, 0, tok].float(), cache[blk, 1, tok].float()
    x = torch.einsum("rnagd,rjad->ragnj", q.float().view(rows, n, n_kv, h // n_kv, D), k) * SCALE
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - m.clamp(min=-1e30))
    return m[..., 0].permute(0, 3, 1, 2).flatten(2), p.sum(-1).permute(0, 3, 1, 2).flatten(2), torch.einsum("ragnj,rjad->rnagd", p, v).flatten(2, 3)


def _plain_window(s):
    cu, lens = s["cu"].long(), s["lens"].long()
    n_q = cu[1:] - cu[:-1]
    reqs, n_kv = lens.shape[0], s["n_kv"]
    i = torch.arange(s["max_q"], device="cuda")
    q = s["q"][(cu[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)]
    pos = (lens - n_q)[:, None] + i                                     # (reqs, n)
    first = torch.arange(s["sinks"], device="cuda").expand(reqs, -1)
    lo = (lens - n_q - s["window"] + 1).clamp(min=0)
    recent = lo[:, None] + torch.arange(min(s["window"] + s["max_q"] - 1, s["max_len"]), device="cuda")
    keys = torch.cat([first, recent], 1)                                # (reqs, j)
    is_first = torch.arange(keys.shape[1], device="cuda") < s["sinks"]
    fresh = is_first | (keys >= s["sinks"])                             # a first token counts once
    kk, pp = keys[:, None, :], pos[:, :, None]
    seen = (fresh & (keys < lens[:, None]))[:, None] & (kk <= pp) & (is_first | (kk > pp - s["window"]))
    blk, tok = _rows(s["table"], keys)
    m, l, o = _plain_attend(q, s["cache"], blk, tok, seen, n_kv)
    o = torch.where(l[..., None] > 0, o / l[..., None], 0).to(torch.bfloat16)
    lse = m + torch.log(l)
    t = torch.arange(s["q"].shape[0], device="cuda")
    r = torch.bucketize(t, cu[1:], right=True)
    return dict(out=o[r, t - cu[r]], lse=lse[r, t - cu[r]])


def _plain_prefix(s):
    cu, pre, lens = s["cu"].long(), s["pre"].long(), s["lens"].long()
    reqs, n_kv = lens.shape[0], s["n_kv"]
    row = torch.arange(reqs, device="cuda")
    group = torch.bucketize(row, cu[1:], right=True)
    # the shared part: every group's rows as the queries of one attention over its first row's table
    at = (cu[:-1, None] + torch.arange(s["max_rows"], device="cuda")).clamp(max=reqs - 1)
    keys = torch.arange(s["max_pre"], device="cuda").expand(pre.shape[0], -1)
    blk, tok = _rows(s["table"][cu[:-1]], keys)
    m1, l1, o1 = (x[group, row - cu[group]] for x in _plain_attend(s["q"][at], s["cache"], blk, tok, (keys < pre[:, None])[:, None].expand(-1, s["max_rows"], -1), n_kv))
    # each request's own part
    keys = pre[group][:, None] + torch.arange(s["max_own"], device="cuda")
    blk, tok = _rows(s["table"], keys)
    m2, l2, o2 = (x[:, 0] for x in _plain_attend(s["q"][:, None], s["cache"], blk, tok, (keys < lens[:, None])[:, None], n_kv))
    m = torch.maximum(m1, m2)
    a, b = torch.exp(m1 - m), torch.exp(m2 - m)
    l = a * l1 + b * l2
    return dict(out=((a[..., None] * o1 + b[..., None] * o2) / l[..., None]).to(torch.bfloat16), lse=m + torch.log(l))


# ---- the framework's calls ------------------------------------------------------------------------
def _own_attention():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "locks-kv_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import locks.attention as attention
    return attention


def _own_run(s):
    att, op = _own_attention(), s["op"]
    if op == "plan":
        o = s["out"]
        att.append_plan(s["lens"], s["new"], s["table"], s["free"], s["taken"], slot_mapping=o["slots"], positions=o["positions"],
                        cu_tokens=o["cu"], lens_out=o["lens"], taken_out=o["taken"])
        return dict(o, table=s["table"])
    if op == "norm":
        att.norm_rope_and_cache(s["q"], s["k"], s["v"], s["cache"], s["slots"], s["positions"], s["cos_sin"], q_weight=s["q_weight"],
                                k_weight=s["k_weight"], eps=s["eps"], q_out=s["out"], neox=s["neox"])
        return dict(q=s["out"], cache=s["cache"])
    if op == "window":
        att.window_paged_attention(s["q"], s["cache"], s["table"], s["cu"], s["lens"], s["out"], n_kv=s["n_kv"], G=s["G"], window=s["window"],
                                   sinks=s["sinks"], scale=SCALE, max_q=s["max_q"], scratch=s["scratch"], lse=s["lse"])
    else:
        att.shared_prefix_paged_decode(s["q"], s["cache"], s["table"], s["lens"], s["cu"], s["pre"], s["out"], n_kv=s["n_kv"], G=s["G"],
                                       scale=SCALE, scratch=s["scratch"], lse=s["lse"])
    return dict(out=s["out"], lse=s["lse"])


def run(state):
    if own:
        return _own_run(state)
    return {"plan": _plain_plan, "norm": _plain_norm, "window": _plain_window, "prefix": _plain_prefix}[state["op"]](state)


# ---- the definition in 64 bits ----------------------------------------------------------------------
def _exact_softmax(q, k, v, seen):
    """q (n, G, 128), k and v (j, 128) of one KV head, seen (n, j): outputs and log-sum-exp."""
    x = torch.tensordot(q, k, dims=([2], [1])) * SCALE
    x = torch.where(seen[:, None], x, -math.inf)
    lse = torch.logsumexp(x, -1)
    w = torch.exp(x - torch.where(lse.isinf(), 0.0, lse)[..., None])
    return torch.tensordot(w, v, dims=([2], [0])), lse


def exact(case, seed):
    op = case["op"]
    if op == "plan":
        return None     # whole numbers: the plain form is exact
    s = prepare(case, seed)
    if op == "norm":
        done = []
        half = s["rot"] // 2
        lo = torch.arange(half, device="cuda")
        i, j = (lo, lo + half) if s["neox"] else (2 * lo, 2 * lo + 1)
        table = s["cos_sin"].double()[s["positions"]][:, None]
        for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
            x = x.double()
            x = x / (x.square().sum(-1, keepdim=True) / D + s["eps"]).sqrt() * w.double()
            y = x.clone()
            y[..., i] = x[..., i] * table[..., :half] - x[..., j] * table[..., half:]
            y[..., j] = x[..., j] * table[..., :half] + x[..., i] * table[..., half:]
            done.append(y)
        cache = s["cache"].double()
        for slot, k, v in zip(s["slots"].tolist(), done[1], s["v"]):
            if slot >= 0:
                cache[slot // PAGE, 0, slot % PAGE] = k
                cache[slot // PAGE, 1, slot % PAGE] = v.double()
        return dict(q=done[0], cache=cache)
    n_kv, G = s["n_kv"], s["G"]
    if op == "window":
        n_q, lens = _window_lens(case)
        start = s["cu"].tolist()
    else:
        lens = _prefix_lens(case)[2]
        n_q, start = [1] * len(lens), list(range(len(lens) + 1))
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["lse"].shape, dtype=torch.float64, device="cuda")
    for r, (n, length) in enumerate(zip(n_q, lens)):
        pos = torch.arange(length - n, length, device="cuda")
        at = torch.arange(length, device="cuda")
        if op == "window":
            at = at[(at < s["sinks"]) | (at > length - n - s["window"])]
        seen = at <= pos[:, None]
        if op == "window":
            seen = seen & ((at < s["sinks"]) | (at > pos[:, None] - s["window"]))
        blk = s["table"][r].long()[at // PAGE]
        for a in range(n_kv):
            k, v = (s["cache"][blk, i, at % PAGE, a].double() for i in (0, 1))
            for b in range(0, n, 1024):
                c = slice(start[r] + b, start[r] + min(b + 1024, n))
                out[c, a * G:(a + 1) * G], lse[c, a * G:(a + 1) * G] = _exact_softmax(s["q"][c, a * G:(a + 1) * G].double(), k, v, seen[b:b + 1024])
    return dict(out=out, lse=lse)
