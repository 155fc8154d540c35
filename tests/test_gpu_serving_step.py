"""The serving step's operators against plain 64-bit forms: slot plan, head norms with
rotation into the cache, windowed attention, shared-prefix decode, and all of them
together, eager and captured."""
from __future__ import annotations

import math
import random

import pytest
import torch

import serving_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, I32, I64 = torch.bfloat16, torch.int32, torch.int64
SCALE = 128 ** -0.5


def i32(x):
    return torch.tensor(x, dtype=I32, device=DEV)


# ---- slot plan ---------------------------------------------------------------------
def run_plan(lens, new, table, free, taken, cap, *, page=16, in_place=False):
    from locks.attention import append_plan
    R = len(lens)
    t = dict(lens=i32(lens), new=i32(new), table=i32(table).reshape(R, len(table[0])), free=i32(free),
             taken=i32([taken]), status=i32([0]))
    o = dict(slots=torch.full((cap,), 77, dtype=I64, device=DEV),
             pos=torch.full((cap,), 77, dtype=I64, device=DEV),
             cu=i32([77] * (R + 1)), lens=t["lens"] if in_place else i32([77] * R),
             taken=t["taken"] if in_place else i32([77]))
    append_plan(t["lens"], t["new"], t["table"], t["free"], t["taken"],
                slot_mapping=o["slots"], positions=o["pos"], cu_tokens=o["cu"],
                lens_out=o["lens"], taken_out=o["taken"], page=page, status=t["status"])
    torch.cuda.synchronize()
    return dict(cu=o["cu"].tolist(), slots=o["slots"].tolist(), pos=o["pos"].tolist(),
                lens=o["lens"].tolist(), taken=int(o["taken"]), table=t["table"].tolist(),
                refused=int(t["status"]) == 3)


@pytest.mark.parametrize("R,n_hi,cap_more,page", [
    (1, 1, 0, 16), (1, 0, 3, 16), (3, 40, 7, 16), (17, 1, 0, 16), (64, 300, 100, 16),
    (513, 9, 5, 16), (4096, 3, 1, 16), (5, 50, 0, 7), (2, 9000, 0, 16)])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan(R, n_hi, cap_more, page, in_place):
    rng = random.Random(R * 31 + n_hi)
    lens = [rng.choice([0, 1, page - 1, page, page + 1, rng.randrange(400)]) for _ in range(R)]
    new = [rng.randrange(n_hi + 1) if n_hi > 1 else n_hi for _ in range(R)]
    width = max(-(-(a + b) // page) for a, b in zip(lens, new)) + 2
    ids = list(range(3 + R * width))
    rng.shuffle(ids)
    table = [[ids.pop() if c * page < a else -1 for c in range(width)] for a in lens]
    args = (lens, new, table, ids, 3, sum(new) + cap_more)
    assert run_plan(*args, page=page, in_place=in_place) == ref.plan(*args, page=page)


def test_plan_refuses_whole_requests():
    """A short free list, a short table row and a short token array each refuse the
    request they hit; requests behind it that need nothing are served."""
    table = [[1, -1, -1], [2, -1, -1], [3, -1, -1], [4, -1, -1]]
    # request 1 asks for two blocks where one is left; request 2 needs none
    args = ([16, 10, 3, 12], [1, 30, 5, 20], table, [9, 8], 0, 64)
    got = run_plan(*args)
    assert got == ref.plan(*args) and got["refused"] and got["lens"] == [17, 10, 8, 12]
    # request 0 is longer than its table row
    args = ([16, 10, 3, 12], [40, 1, 1, 5], table, [9, 8], 1, 64)
    got = run_plan(*args)
    assert got == ref.plan(*args) and got["refused"] and got["lens"] == [16, 11, 4, 17]
    # the token array ends inside request 2
    args = ([0, 0, 0, 0], [4, 4, 4, 0], table, [9, 8, 7, 6], 0, 10)
    got = run_plan(*args)
    assert got == ref.plan(*args) and got["refused"] and got["slots"][8:] == [-1, -1]
    # nothing free at all
    args = ([0, 1], [1, 1], [[-1], [5]], [], 0, 2)
    assert run_plan(*args) == ref.plan(*args)


# ---- head norms, rotation, cache write ------------------------------------------------
@pytest.mark.parametrize("T,n_kv,G,rot,neox,f32,weights", [
    (1, 8, 4, 128, True, False, True), (7, 2, 3, 64, True, True, True),
    (33, 1, 16, 128, False, False, True), (5, 4, 1, 20, True, False, True),
    (5, 4, 1, 20, False, True, True), (129, 2, 5, 96, True, False, False),
    (12, 2, 2, 2, False, False, True), (64, 8, 4, 16, True, True, True),
    (3, 2, 4, 0, True, False, True), (40, 3, 7, 100, False, True, False)])
def test_norm_rope(T, n_kv, G, rot, neox, f32, weights):
    """Rows of one projection (strided views), scattered slots, some without one.
    fp32 arithmetic: about ten roundings of 2^-24 of the pair's magnitudes plus
    rsqrt's two units, then one rounding to bf16."""
    from locks.attention import norm_rope_and_cache
    g = torch.Generator(device=DEV).manual_seed(T + rot)
    H, NB = n_kv * G, T // 16 + 3
    qkv = torch.randn(T, H + 2 * n_kv, 128, device=DEV, generator=g).to(BF16)
    q, k, v = qkv[:, :H], qkv[:, H:H + n_kv], qkv[:, H + n_kv:]
    kind = torch.float32 if f32 else BF16
    wq, wk = ((torch.randn(128, device=DEV, generator=g) + 1).to(kind) if weights else None
              for _ in range(2))
    table = torch.randn(50, max(rot, 2), device=DEV, generator=g).to(kind) if rot else None
    pos = torch.randint(0, 50, (T,), device=DEV, generator=g)
    slots = torch.randperm(NB * 16, device=DEV, generator=g)[:T]
    slots[T // 2::5] = -1
    cache = torch.randn(NB, 2, 16, n_kv, 128, device=DEV, generator=g).to(BF16)
    want_c, eps = cache.double(), 1e-5
    cs = table[pos] if rot else None
    want_q, want_k = (ref.norm_rope(x, w, eps, cs, rot, neox) for x, w in ((q, wq), (k, wk)))
    for t, s in enumerate(slots.tolist()):
        if s >= 0:
            want_c[s // 16, 0, s % 16], want_c[s // 16, 1, s % 16] = want_k[t], v[t].double()
    out = torch.empty(T, H, 128, device=DEV, dtype=BF16)
    got = norm_rope_and_cache(q, k, v, cache, slots, pos if rot else None, table,
                              q_weight=wq, k_weight=wk, eps=eps, q_out=out, neox=neox)
    assert got is out
    touched = torch.zeros(NB, 16, dtype=torch.bool, device=DEV)
    live = slots[slots >= 0]
    touched[live // 16, live % 16] = True
    assert torch.equal(cache[:, 0][~touched], want_c[:, 0][~touched].to(BF16))
    assert torch.equal(cache[:, 1], want_c[:, 1].to(BF16))
    for a, b in ((out, want_q), (cache[:, 0], want_c[:, 0])):
        big = b.abs().amax(-1, keepdim=True)
        assert bool(((a.double() - b).abs() <= ref.HALF_BF16 * b.abs() + 2.0 ** -19 * big).all())
    # in place, bit for bit the same
    norm_rope_and_cache(q, k, v, cache, slots, pos if rot else None, table, q_weight=wq,
                        k_weight=wk, eps=eps, neox=neox)
    assert torch.equal(q, out)


def test_norm_rope_odd_table_rows_and_outside_positions():
    """A table whose rows are not vector-aligned, positions outside it (clamped) and
    slots beyond the cache (not stored)."""
    from locks.attention import norm_rope_and_cache
    g = torch.Generator(device=DEV).manual_seed(4)
    T, n_kv = 6, 2
    q, k, v = (torch.randn(T, n_kv, 128, device=DEV, generator=g).to(BF16) for _ in range(3))
    table = torch.randn(9, 130, device=DEV, generator=g).to(BF16)[:, 1:129]
    pos = torch.tensor([0, -5, 8, 9, 2 ** 40, 3], device=DEV)
    slots = torch.tensor([0, 17, 48, 2 ** 40, -1, 47], device=DEV)
    cache = torch.zeros(3, 2, 16, n_kv, 128, device=DEV, dtype=BF16)
    out = norm_rope_and_cache(q, k, v, cache, slots, pos, table, q_out=torch.empty_like(q))
    want = ref.norm_rope(q, None, 0, table[pos.clamp(0, 8)], 128, True)
    big = want.abs().amax(-1, keepdim=True)
    assert bool(((out.double() - want).abs() <= ref.HALF_BF16 * want.abs() + 2.0 ** -19 * big).all())
    used = (cache != 0).flatten(3).any(-1)
    assert used[:, 0].nonzero().tolist() == used[:, 1].nonzero().tolist() == [[0, 0], [1, 1], [2, 15]]


def test_norm_rope_weight_on_one_side_only():
    """A query weight alone leaves the keys unnormalised, and the other way round."""
    from locks.attention import norm_rope_and_cache
    g = torch.Generator(device=DEV).manual_seed(8)
    q, k, v = (torch.randn(5, 2, 128, device=DEV, generator=g).to(BF16) for _ in range(3))
    w = torch.rand(128, device=DEV, generator=g)
    slots = torch.arange(5, device=DEV)
    for kind in (torch.float32, BF16):
        for wq, wk in ((w.to(kind), None), (None, w.to(kind))):
            cache = torch.zeros(3, 2, 16, 2, 128, device=DEV, dtype=BF16)
            out = norm_rope_and_cache(q, k, v, cache, slots, None, None, q_weight=wq, k_weight=wk,
                                      eps=0.0, q_out=torch.empty_like(q))
            for got, x, wt in ((out, q, wq), (cache[0, 0, :5], k, wk)):
                want = ref.norm_rope(x, wt, 0.0, None, 0, True)
                assert bool(((got.double() - want).abs() <= ref.HALF_BF16 * want.abs() + 1e-5).all())
                assert wt is not None or torch.equal(got, x)


# ---- paged inputs ---------------------------------------------------------------------
def paged(seed, lens, n_kv, *, planes_first=False, spare=3):
    """A cache and tables of exactly the pages the lengths need, scattered."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    R, W = len(lens), max(1, max(-(-max(x, 0) // 16) for x in lens))
    n = sum(-(-max(x, 0) // 16) for x in lens)
    NB = n + spare
    shape = (2, NB, 16, n_kv, 128) if planes_first else (NB, 2, 16, n_kv, 128)
    cache = torch.randn(shape, device=DEV, generator=g).to(BF16)
    ids = torch.randperm(NB, device=DEV, generator=g).to(I32)
    table = torch.zeros(R, W, dtype=I32, device=DEV)
    at = 0
    for r, x in enumerate(lens):
        m = -(-max(x, 0) // 16)
        table[r, :m] = ids[at:at + m]
        at += m
    k, v = (cache[0], cache[1]) if planes_first else (cache[:, 0], cache[:, 1])
    k.mul_(torch.where(torch.rand(n_kv, 128, device=DEV, generator=g) < 0.03, 8.0, 1.0).to(BF16))
    return g, cache, k, v, table


def check(out, lse, want, r=""):
    o, s, mean, size = want
    assert bool(((out.double() - o).abs() <= ref.out_tolerance(o, mean, size)).all()), \
        (r, float((out.double() - o).abs().max()))
    if lse is not None:
        empty = s == -math.inf
        assert torch.equal(lse == -math.inf, empty), r
        d = torch.where(empty, 0.0, lse.double() - s).abs()
        assert bool((d <= ref.lse_tolerance(s, size)).all()), (r, float(d.max()))


def want_window(q, k, v, row, length, n, window, sinks):
    end = min(max(length, 0), row.shape[0] * 16)
    pos = torch.arange(length - n, length, device=DEV)[:, None]
    key = torch.arange(end, device=DEV)[None]
    seen = (key <= pos) & ((pos - key < window) | (key < sinks))
    return ref.attend(q, ref.gather(k, row, end), ref.gather(v, row, end), seen, SCALE)


def run_window(q, cache, table, cu, lens, n_kv, G, window, sinks, max_q, *, out=None, lse=None,
               scratch=None):
    from locks.attention import window_paged_attention
    if out is None:
        out = torch.full_like(q, float("nan"))
    st = i32([0])
    window_paged_attention(q, cache, table, cu, lens, out, n_kv=n_kv, G=G, window=window,
                           sinks=sinks, scale=SCALE, max_q=max_q, lse=lse, scratch=scratch,
                           status=st)
    assert int(st) == 0
    return out


WINDOW_CASES = [
    # (n_kv, G, [(new, cached)], window, sinks)
    (8, 4, [(1, 1)], 100, 0),
    (8, 4, [(1, 1), (1, 16), (1, 17), (1, 15), (1, 33)], 16, 1),
    (2, 8, [(0, 0), (1, 40), (0, 5), (3, 90), (1, 0)], 20, 4),
    (2, 8, [(1, 40), (5, 90)], 0, 0),
    (2, 8, [(1, 40), (5, 90), (200, 200)], 0, 5),
    (4, 1, [(1, 700), (2, 64), (7, 7), (16, 300)], 1, 0),
    (1, 16, [(1, 5000), (1, 4097), (2, 129)], 1000, 3),
    (2, 16, [(1, 9000)], None, 0),
    (8, 1, [(300, 300)], None, 0),
    (2, 4, [(129, 700), (128, 128), (127, 1000), (64, 64), (1, 3)], 100, 20),
    (2, 3, [(43, 500), (86, 86), (200, 1000)], 130, 7),
    (1, 5, [(60, 2000), (26, 26), (1, 99)], 257, 128),
    (1, 7, [(19, 19), (150, 400)], 64, 200),
    (4, 2, [(257, 3000), (5, 6)], 2000, 16),
    (1, 12, [(600, 1500)], 333, 37),
    (2, 4, [(30, 20), (5, 2), (3, -4)], 50, 2),          # fewer cached than new
    (1, 4, [(1000, 1100)], 128, 0),
    (1, 8, [(40, 17000)], None, 0),
    (1, 1, [(130, 6000), (300, 300)], 5000, 1000),
    (1, 8, [(1, 40001), (2, 33000), (0, 7), (1, 3)], None, 0),   # few rows, very long
    (2, 16, [(1, 36000)], 34000, 50),
]


@pytest.mark.parametrize("case", range(len(WINDOW_CASES)))
def test_window(case):
    n_kv, G, reqs, window, sinks = WINDOW_CASES[case]
    lens = [l for _, l in reqs]
    g, cache, k, v, table = paged(case, lens, n_kv, planes_first=case % 2 == 1)
    w = 2 ** 31 - 1 if window is None else window
    cu = [0]
    for n, _ in reqs:
        cu.append(cu[-1] + n)
    T, H = cu[-1], n_kv * G
    # queries as a view of a wider projection, three rows behind the last sequence
    q = torch.randn(T + 3, H + 2, 128, device=DEV, generator=g).to(BF16)[:, 1:H + 1]
    # pages nobody sees: no table entry; slots past the end: not finite
    for r, (n, l) in enumerate(reqs):
        for pg in range(table.shape[1]):
            first = l - n - w + 1
            if pg * 16 >= l or (pg * 16 + 15 < first and pg * 16 >= sinks) or n == 0:
                table[r, pg] = (-1, 2 ** 30, -2 ** 31)[(r + pg) % 3]
            elif pg * 16 + 16 > l:
                k[table[r, pg], l - pg * 16:] = float("nan")
                v[table[r, pg], l - pg * 16:] = float("inf")
    used = torch.zeros(k.shape[0], dtype=torch.bool, device=DEV)
    used[table[(table >= 0) & (table < k.shape[0])].long()] = True
    k[~used], v[~used] = float("nan"), float("nan")
    for scratch in (None, torch.empty(2 ** 22, device=DEV)):
        out = torch.full((T + 3, H, 128), 7.0, device=DEV, dtype=BF16)
        lse = torch.full((T + 3, H), 7.0, device=DEV)
        run_window(q, cache, table, i32(cu), i32(lens), n_kv, G, window, sinks,
                   max(n for n, _ in reqs), out=out, lse=lse, scratch=scratch)
        assert bool((out[T:] == 7).all()) and bool((lse[T:] == 7).all())
        for r, (n, l) in enumerate(reqs):
            at = slice(cu[r], cu[r + 1])
            row = table[r].clamp(0, k.shape[0] - 1)
            kk, vv = k.nan_to_num(0, 0, 0), v.nan_to_num(0, 0, 0)
            if n:
                check(out[at], lse[at], want_window(q[at], kk, vv, row, l, n, w, sinks), r)


def test_window_short_table_and_small_bound():
    """Lengths beyond the table's last column end with it."""
    n_kv, G = 2, 4
    g, cache, k, v, table = paged(5, [64, 64], n_kv)
    lens, cu = [500, 70], [0, 1, 3]
    q = torch.randn(3, 8, 128, device=DEV, generator=g).to(BF16)
    out = run_window(q, cache, table, i32(cu), i32(lens), n_kv, G, None, 0, 2)
    for r in range(2):
        at = slice(cu[r], cu[r + 1])
        check(out[at], None, want_window(q[at], k, v, table[r], lens[r], cu[r + 1] - cu[r],
                                         2 ** 31 - 1, 0))


BEYOND_BOUND_CASES = [
    # (n_kv, G, [(new, cached)], max_q): requests with more query tokens than max_q says
    (2, 4, [(5, 200)], 1),                                  # few pairs, eight-row blocks
    (2, 4, [(41, 300), (1, 20), (2, 90)], 2),
    (1, 12, [(50, 90), (1, 64)], 1),                        # sixteen-row blocks
    (2, 4, [(3, 60 + r) for r in range(45)] + [(30, 100)], 2),      # many pairs
    (1, 8, [(3, 34000), (1, 33000)], 1),                    # few rows, very long
    (2, 8, [(300, 310), (1, 40), (700, 2000), (2, 2)], 20),         # tiles, in parts with scratch
    (8, 4, [(33, 100)] * 40 + [(400, 900)], 6),
]


@pytest.mark.parametrize("case", range(len(BEYOND_BOUND_CASES)))
def test_window_requests_with_more_queries_than_the_bound(case):
    """The bound steers how the work is cut, not what is computed: a call captured for
    fewer tokens meets longer requests."""
    n_kv, G, reqs, max_q = BEYOND_BOUND_CASES[case]
    lens = [l for _, l in reqs]
    g, cache, k, v, table = paged(70 + case, lens, n_kv)
    cu = [0]
    for n, _ in reqs:
        cu.append(cu[-1] + n)
    T, H = cu[-1], n_kv * G
    q = torch.randn(T + 2, H, 128, device=DEV, generator=g).to(BF16)
    for scratch in (None, torch.full((2 ** 23,), float("nan"), device=DEV)):
        out = torch.full((T + 2, H, 128), 7.0, device=DEV, dtype=BF16)
        lse = torch.full((T + 2, H), 7.0, device=DEV)
        run_window(q, cache, table, i32(cu), i32(lens), n_kv, G, None, 0, max_q, out=out, lse=lse,
                   scratch=scratch)
        assert bool((out[T:] == 7).all()) and bool((lse[T:] == 7).all())
        for r, (n, l) in enumerate(reqs):
            at = slice(cu[r], cu[r + 1])
            check(out[at], lse[at], want_window(q[at], k, v, table[r], l, n, 2 ** 31 - 1, 0), r)


@pytest.mark.parametrize("G", [4, 3])
def test_window_tiles_that_end_at_every_offset_of_a_page(G):
    """More tiles than SMs, so that a CTA takes several in a row, each with a last page
    that is cut off at another token; what lies behind is not finite."""
    n_kv, n = 4, 34
    lens = [200 + 17 * r for r in range(96)]
    g, cache, k, v, table = paged(60 + G, lens, n_kv)
    for r, l in enumerate(lens):
        if l % 16:
            k[table[r, l // 16], l % 16:] = float("nan")
            v[table[r, l // 16], l % 16:] = float("inf")
    q = torch.randn(n * len(lens), n_kv * G, 128, device=DEV, generator=g).to(BF16)
    cu = i32([n * r for r in range(len(lens) + 1)])
    lse = torch.full(q.shape[:2], 7.0, device=DEV)
    out = run_window(q, cache, table, cu, i32(lens), n_kv, G, 150, 5, n, lse=lse)
    kk, vv = k.nan_to_num(0, 0, 0), v.nan_to_num(0, 0, 0)
    for r, l in enumerate(lens):
        at = slice(n * r, n * r + n)
        check(out[at], lse[at], want_window(q[at], kk, vv, table[r], l, n, 150, 5), r)


@pytest.mark.parametrize("n,G", [(1, 4), (60, 8)])
def test_window_counts_beyond_32_bits(n, G):
    """More first tokens, a wider window or a larger bound than 32 bits hold: all of them."""
    g, cache, k, v, table = paged(33, [300], 2)
    q = torch.randn(n, 2 * G, 128, device=DEV, generator=g).to(BF16)
    want = run_window(q, cache, table, i32([0, n]), i32([300]), 2, G, None, 0, n)
    for window, sinks, max_q in ((10, 2 ** 32, n), (2 ** 33, 0, n), (None, 0, 2 ** 32)):
        got = run_window(q, cache, table, i32([0, n]), i32([300]), 2, G, window, sinks, max_q)
        # (another bound may cut the work another way)
        check(got, None, want_window(q, k, v, table[0], 300, n, 2 ** 31 - 1, 0))
        assert max_q != n or torch.equal(got, want)


def test_status_of_another_type_is_refused():
    from locks.attention import (append_plan, attention_scratch_floats, shared_prefix_paged_decode,
                                 window_paged_attention)
    g, cache, k, v, table = paged(34, [40], 2)
    q = torch.randn(1, 8, 128, device=DEV, generator=g).to(BF16)
    lens, cu = i32([40]), i32([0, 1])
    wide = torch.zeros(1, dtype=I64, device=DEV)
    for st in (wide.clone(), torch.zeros(1, dtype=torch.bool, device=DEV)):
        with pytest.raises(AssertionError, match="status"):
            window_paged_attention(q, cache, table, cu, lens, torch.empty_like(q), n_kv=2, G=4,
                                   window=None, scale=SCALE, max_q=1, status=st)
        with pytest.raises(AssertionError, match="status"):
            shared_prefix_paged_decode(q, cache, table, lens, cu, i32([16]), torch.empty_like(q), n_kv=2,
                                       G=4, scale=SCALE, status=st,
                                       scratch=torch.empty(attention_scratch_floats(1, 8), device=DEV))
        with pytest.raises(AssertionError, match="status"):
            append_plan(lens, i32([1]), table, i32([1]), i32([0]), slot_mapping=wide, positions=wide.clone(),
                        cu_tokens=cu, lens_out=lens, taken_out=i32([0]), status=st)
        assert int(st) == 0


def test_tables_much_wider_than_the_sequences():
    """Tables as wide as the longest sequence allowed, entries behind the own pages that
    name nothing, and scratch for many parts: most of them are empty."""
    n_kv, G, reqs, W = 2, 8, [(1, 300), (40, 500), (1, 16), (2, 90)], 9000
    lens = [l for _, l in reqs]
    g, cache, k, v, table = paged(51, lens, n_kv)
    wide = torch.full((4, W), -1, dtype=I32, device=DEV)
    for r, l in enumerate(lens):
        wide[r, :-(-l // 16)] = table[r, :-(-l // 16)]
    scratch = torch.full((2 ** 23,), float("nan"), device=DEV)
    cu = [0, 1, 41, 42, 44]
    q = torch.randn(44, n_kv * G, 128, device=DEV, generator=g).to(BF16)
    for rows in (slice(0, 4), slice(2, 4)):             # with tiles; few rows in parts
        sub, at0 = lens[rows], cu[rows.start]
        bounds = [c - at0 for c in cu[rows.start:]]
        n_q = [n for n, _ in reqs[rows]]
        lse = torch.full((bounds[-1], n_kv * G), 7.0, device=DEV)
        out = run_window(q[at0:], cache, wide[rows], i32(bounds), i32(sub), n_kv, G, None, 0, max(n_q),
                         lse=lse, scratch=scratch)
        for r, l in enumerate(sub):
            at = slice(bounds[r], bounds[r + 1])
            check(out[at], lse[at], want_window(q[at0:][at], k, v, wide[rows][r, :-(-l // 16)], l, n_q[r],
                                                2 ** 31 - 1, 0), r)
    g, cache, table, lens = prefix_paged(9, [(100, [101, 160, 113]), (33, [40])], n_kv)
    wide = torch.full((4, W), -1, dtype=I32, device=DEV)
    for r, l in enumerate(lens):
        wide[r, :-(-l // 16)] = table[r, :-(-l // 16)]
    lse = torch.full((4, n_kv * G), 7.0, device=DEV)
    out = run_prefix(q[:4], cache, wide, lens, [0, 3, 4], [100, 33], n_kv, G, lse=lse, floats=2 ** 22)
    for r, l in enumerate(lens):
        check(out[r:r + 1], lse[r:r + 1], want_window(q[r:r + 1], cache[:, 0], cache[:, 1], table[r], l, 1,
                                                      2 ** 31 - 1, 0), r)


def test_window_many_requests_few_of_them_long():
    """Several hundred requests, most with one token, prompts between them."""
    n_kv, G, R = 1, 8, 700
    rng = random.Random(5)
    n_q = [1] * R
    for r in (3, 31, 32, 500, 699):
        n_q[r] = rng.choice([17, 64, 129])
    lens = [n + rng.randrange(60) for n in n_q]
    g, cache, k, v, table = paged(11, lens, n_kv)
    cu = [0]
    for n in n_q:
        cu.append(cu[-1] + n)
    q = torch.randn(cu[-1], G, 128, device=DEV, generator=g).to(BF16)
    out = run_window(q, cache, table, i32(cu), i32(lens), n_kv, G, 40, 3, max(n_q))
    for r in (0, 3, 4, 31, 32, 33, 499, 500, 501, 698, 699):
        at = slice(cu[r], cu[r + 1])
        check(out[at], None, want_window(q[at], k, v, table[r], lens[r], n_q[r], 40, 3), r)
    assert bool(out.isfinite().all())


def test_window_head_major_cache_strided_table_and_no_programmatic_launch():
    """Heads outside tokens in storage, a table that is a view, G that does not divide
    128, and the launches without their programmatic edge: the same numbers."""
    from locks import _cabi
    n_kv, G, reqs = 3, 6, [(1, 500), (90, 300), (2, 33)]
    g, cache, k, v, table = paged(12, [l for _, l in reqs], n_kv)
    other = cache.transpose(2, 3).contiguous().transpose(2, 3)
    wide = torch.full((3, table.shape[1] + 5), -7, dtype=I32, device=DEV)
    wide[:, 2:-3] = table
    q = torch.randn(93, 18, 128, device=DEV, generator=g).to(BF16)
    cu, lens = i32([0, 1, 91, 93]), i32([l for _, l in reqs])
    a = run_window(q, cache, table, cu, lens, n_kv, G, 100, 9, 90)
    old = _cabi.lib().locks_set_pdl(0)
    try:
        b = run_window(q, other, wide[:, 2:-3], cu, lens, n_kv, G, 100, 9, 90)
        torch.cuda.synchronize()
    finally:
        _cabi.lib().locks_set_pdl(old)
    assert torch.equal(a, b)
    check(a[1:91], None, want_window(q[1:91], k, v, table[1], 300, 90, 100, 9))


def test_block_ids_outside_the_cache_touch_nothing():
    """Table entries of seen pages that name no block: read as some block of the cache,
    never outside it; other requests are not affected."""
    n_kv, G, reqs = 2, 8, [(1, 300), (60, 200), (1, 90), (40, 77)]
    lens = [l for _, l in reqs]
    g, cache, k, v, table = paged(31, lens, n_kv)
    cu = [0, 1, 61, 62, 102]
    table[0, ::2], table[1, 1::3] = -5, 2 ** 31 - 1
    q = torch.randn(102, 16, 128, device=DEV, generator=g).to(BF16)
    out = run_window(q, cache, table, i32(cu), i32(lens), n_kv, G, None, 0, 60)
    assert bool(out.isfinite().all())
    for r in (2, 3):
        at = slice(cu[r], cu[r + 1])
        check(out[at], None, want_window(q[at], k, v, table[r], lens[r], reqs[r][0], 2 ** 31 - 1, 0), r)
    one = run_prefix(q[:4], cache, table, lens, [0, 2, 4], [64, 48], n_kv, G)
    assert bool(one.isfinite().all())


def test_offsets_beyond_31_bits():
    """Blocks whose element offsets pass 2^31: attention of both kinds, and the write."""
    from locks.attention import norm_rope_and_cache
    n_kv, G, NB = 8, 2, 66000
    cache = torch.zeros(NB, 2, 16, n_kv, 128, device=DEV, dtype=BF16)
    g = torch.Generator(device=DEV).manual_seed(3)
    far = torch.arange(NB - 20, NB, device=DEV)
    cache[far] = torch.randn(20, 2, 16, n_kv, 128, device=DEV, generator=g).to(BF16)
    table = far.to(I32).reshape(2, 10)
    q = torch.randn(40, 16, 128, device=DEV, generator=g).to(BF16)
    cu, lens = [0, 1, 40], [160, 150]
    out = run_window(q, cache, table, i32(cu), i32(lens), n_kv, G, 70, 5, 39)
    for r in range(2):
        at = slice(cu[r], cu[r + 1])
        check(out[at], None, want_window(q[at], cache[:, 0], cache[:, 1], table[r], lens[r],
                                         cu[r + 1] - cu[r], 70, 5))
    two = run_prefix(q[:2], cache, table[:1].expand(2, -1), [160, 133], [0, 2], [128], n_kv, G)
    for r, l in enumerate((160, 133)):
        check(two[r:r + 1], None, want_window(q[r:r + 1], cache[:, 0], cache[:, 1], table[0], l, 1,
                                              2 ** 31 - 1, 0))
    kv = torch.randn(1, 2 * n_kv, 128, device=DEV, generator=g).to(BF16)
    slot = torch.tensor([NB * 16 - 1], device=DEV)
    norm_rope_and_cache(q[:1], kv[:, :n_kv], kv[:, n_kv:], cache, slot, None, None)
    assert torch.equal(cache[-1, 0, 15], kv[0, :n_kv]) and torch.equal(cache[-1, 1, 15], kv[0, n_kv:])


def test_empty_batches():
    from locks.attention import norm_rope_and_cache
    g, cache, k, v, table = paged(2, [20], 2)
    none, q = i32([]), torch.zeros(0, 8, 128, device=DEV, dtype=BF16)
    run_window(q, cache, table[:0], i32([0]), none, 2, 4, 10, 0, 0)
    run_window(q, cache, table, i32([0, 0]), i32([20]), 2, 4, 10, 0, 0)
    run_prefix(q, cache, table[:0], [], [0], [], 2, 4, floats=16)
    norm_rope_and_cache(q, q[:, :2], q[:, :2], cache, torch.zeros(0, dtype=I64, device=DEV), None, None)
    got = run_plan([], [], [[]], [4], 1, 3)
    assert got["slots"] == [-1] * 3 and got["taken"] == 1 and got["cu"] == [0]


NOT_FINITE_CASES = [
    # (n_kv, G, [(new, cached)], window, sinks): one for each way through the kernels
    (2, 4, [(1, 300), (2, 40)], None, 0),                       # few rows, clusters
    (1, 12, [(3, 77)], 20, 3),
    (2, 4, [(1, 90 + r) for r in range(60)], None, 0),          # many pairs
    (1, 8, [(1, 34000)], None, 0),                              # cut into parts with scratch
    (2, 4, [(30, 200), (100, 700)], None, 0),                   # tiles of shared and of own rows
    (2, 3, [(80, 300), (1, 9)], 64, 5),
    (1, 8, [(40, 9000)], None, 0),                              # tiles, parts with scratch
    (1, 4, [(120, 120)], 1, 0),                                 # one key to a row, every column
    (1, 4, [(20, 60)], 0, 0),                                   # no key: nothing to be wrong
]


def spoil(q, g):
    """NaN and infinities in single channels of scattered rows."""
    T, H, _ = q.shape
    at = torch.randperm(T * H, device=DEV, generator=g)[:max(3, T * H // 7)]
    for i, bad in enumerate((float("nan"), float("inf"), -float("inf"))):
        rows = at[i::3]
        q[rows // H, rows % H, (rows * 13 + 5 * i) % 128] = bad


def check_not_finite(q, out, lse, k, v, seen, r=""):
    """A seen score of NaN or +inf makes its row NaN; the other rows are what they are."""
    G = q.shape[1] // k.shape[1]
    x = torch.einsum("nhd,jhd->nhj", q.double(), k.double().repeat_interleave(G, 1)) * SCALE
    lost = ((x.isnan() | (x == math.inf)) & seen[:, None]).any(-1)
    assert bool(out[lost].isnan().all()) and bool(lse[lost].isnan().all()), r
    clean = q.isfinite().all(-1)
    some = seen.any(-1)
    assert bool((lost | clean | ~some[:, None] | (x.masked_fill(~seen[:, None], -math.inf) ==
                                                  -math.inf).all(-1)).all())
    none = ~lost & ~clean
    assert bool((out[none] == 0).all()) and bool((lse[none] == -math.inf).all()), r
    want = ref.attend(torch.where(clean[..., None], q, 0), k, v, seen, SCALE)
    check(out[clean], lse[clean], [t[clean] for t in want], r)


@pytest.mark.parametrize("case", range(len(NOT_FINITE_CASES)))
def test_window_queries_that_are_not_finite(case):
    n_kv, G, reqs, window, sinks = NOT_FINITE_CASES[case]
    lens = [l for _, l in reqs]
    g, cache, k, v, table = paged(90 + case, lens, n_kv)
    w = 2 ** 31 - 1 if window is None else window
    cu = [0]
    for n, _ in reqs:
        cu.append(cu[-1] + n)
    q = torch.randn(cu[-1], n_kv * G, 128, device=DEV, generator=g).to(BF16)
    spoil(q, g)
    for scratch in (None, torch.empty(2 ** 23, device=DEV)):
        lse = torch.full(q.shape[:2], 7.0, device=DEV)
        out = torch.full_like(q, 7.0)
        run_window(q, cache, table, i32(cu), i32(lens), n_kv, G, window, sinks,
                   max(n for n, _ in reqs), out=out, lse=lse, scratch=scratch)
        for r, (n, l) in enumerate(reqs):
            at = slice(cu[r], cu[r + 1])
            pos, key = torch.arange(l - n, l, device=DEV)[:, None], torch.arange(l, device=DEV)[None]
            seen = (key <= pos) & ((pos - key < w) | (key < sinks))
            check_not_finite(q[at], out[at], lse[at], ref.gather(k, table[r], l),
                             ref.gather(v, table[r], l), seen, r)


def test_bounds_beyond_the_queries_are_cut_off():
    """cu_q that runs past q (fewer rows than it says): the rows that exist are right,
    nothing behind them is touched."""
    n_kv, G = 2, 4
    g, cache, k, v, table = paged(21, [90, 50], n_kv)
    q = torch.randn(64, 8, 128, device=DEV, generator=g).to(BF16)
    out = torch.full((64, 8, 128), 7.0, device=DEV, dtype=BF16)
    run_window(q[:50], cache, table, i32([0, 40, 80]), i32([90, 50]), n_kv, G, None, 0, 40,
               out=out[:50])
    assert bool((out[50:] == 7).all())
    check(out[:40], None, want_window(q[:40], k, v, table[0], 90, 40, 2 ** 31 - 1, 0))
    want = want_window(q[40:64], k, v, table[1], 50 - 16, 24, 2 ** 31 - 1, 0)
    check(out[40:50], None, [x[:10] for x in want])


def test_window_repeats_bit_for_bit_on_another_stream():
    n_kv, G, reqs = 2, 8, [(1, 900), (70, 400), (3, 3000), (1, 2)]
    lens = [l for _, l in reqs]
    g, cache, k, v, table = paged(6, lens, n_kv)
    cu = i32([0, 1, 71, 74, 75])
    q = torch.randn(75, 16, 128, device=DEV, generator=g).to(BF16)
    scratch = torch.empty(2 ** 20, device=DEV)
    a = run_window(q, cache, table, cu, i32(lens), n_kv, G, 300, 4, 70, scratch=scratch)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = run_window(q, cache, table, cu, i32(lens), n_kv, G, 300, 4, 70, scratch=scratch)
    torch.cuda.synchronize()
    assert torch.equal(a, b)


def test_calls_on_two_streams_at_once_and_two_graphs():
    """Calls that overlap, each with a workspace of its own: what one after the other
    gives, eagerly and from two graphs replayed side by side."""
    n_kv, G, reqs = 2, 8, [(1, 700), (90, 400), (3, 2500)]
    lens = [l for _, l in reqs]
    cu = i32([0, 1, 91, 94])
    streams = [torch.cuda.Stream() for _ in range(2)]
    calls, want = [], []
    for k in range(2):
        g, cache, _, _, table = paged(40 + k, lens, n_kv)
        q = torch.randn(94, 16, 128, device=DEV, generator=g).to(BF16)
        out, scratch = torch.empty_like(q), torch.empty(2 ** 20, device=DEV)
        args = (q, cache, table, cu, i32(lens), n_kv, G, 200 + 300 * k, 4, 90)
        calls.append((args, out, scratch))
        want.append(run_window(*args, scratch=scratch).clone())
    torch.cuda.synchronize()

    def launch(k):
        from locks.attention import window_paged_attention
        (q, cache, table, cu_, ln, n, g_, w, s, mq), out, scratch = calls[k]
        window_paged_attention(q, cache, table, cu_, ln, out, n_kv=n, G=g_, window=w, sinks=s,
                               scale=SCALE, max_q=mq, scratch=scratch)

    for _ in range(20):
        for k in range(2):
            calls[k][1].zero_()
        torch.cuda.synchronize()
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                launch(k)
        torch.cuda.synchronize()
        assert all(torch.equal(calls[k][1], want[k]) for k in range(2))
    graphs = []
    for k in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[k]):
            for _ in range(3):
                launch(k)
    for _ in range(10):
        for k in range(2):
            calls[k][1].zero_()
        torch.cuda.synchronize()
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                graphs[k].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(calls[k][1], want[k]) for k in range(2))


# ---- shared prefix ----------------------------------------------------------------------
def prefix_paged(seed, groups, n_kv, spare=3):
    """groups: [(prefix, [cached lengths])]; whole prefix pages shared, the page a
    prefix ends in copied."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    lens = [l for _, ls in groups for l in ls]
    W = max(1, max(-(-max(l, 0) // 16) for l in lens + [p for p, _ in groups]))
    table = torch.zeros(len(lens), W, dtype=torch.int64)
    n, r, copies = 0, 0, []
    for pre, ls in groups:
        whole = pre // 16
        first = n
        n += whole
        r0 = r
        for l in ls:
            table[r, :whole] = torch.arange(first, first + whole)
            m = max(-(-l // 16) - whole, 0)
            table[r, whole:whole + m] = torch.arange(n, n + m)
            if m and pre % 16:
                copies.append((n, pre % 16, r0, whole))
            n += m
            r += 1
    ids = torch.randperm(n + spare, device=DEV, generator=g)
    cache = torch.randn(n + spare, 2, 16, n_kv, 128, device=DEV, generator=g).to(BF16)
    table = ids[table.to(DEV)].to(I32)
    for b, m, r0, whole in copies:
        cache[ids[b], :, :m] = cache[table[r0, whole].long(), :, :m]
    return g, cache, table, lens


def run_prefix(q, cache, table, lens, cu, pre, n_kv, G, *, floats=None, out=None, lse=None):
    from locks.attention import attention_scratch_floats, shared_prefix_paged_decode
    if out is None:
        out = torch.full_like(q, float("nan"))
    need = attention_scratch_floats(q.shape[0], q.shape[1])
    scratch = torch.full((floats or need,), float("nan"), device=DEV)
    st = i32([0])
    shared_prefix_paged_decode(q, cache, table, i32(lens), i32(cu), i32(pre), out, n_kv=n_kv,
                               G=G, scale=SCALE, scratch=scratch, lse=lse, status=st)
    assert int(st) == 0
    return out


PREFIX_CASES = [
    # (n_kv, G, [(prefix, [lengths])])
    (2, 4, [(0, [5, 1, 40])]),
    (2, 4, [(5, [6, 40, 5])]),
    (8, 4, [(16, [17, 16, 300])]),
    (2, 8, [(100, [101, 116, 112, 113, 500]), (17, [40]), (64, [64, 65])]),
    (1, 16, [(1000, [1000 + 7 * i for i in range(9)]), (2050, [2051] * 3)]),
    (4, 1, [(130, [131 + i for i in range(130)])]),
    (2, 5, [(128, [129 + 3 * i for i in range(60)]), (900, [950] * 27)]),
    (1, 3, [(5000, [5003])]),
    (2, 16, [(256, [300] * 33)]),
    (1, 8, [(9000, [9001 + 40 * i for i in range(20)])]),
    (2, 4, [(96, [40, 0, 97, 96, -3, 15])]),              # some shorter than the prefix
    (1, 12, [(333, [340, 400]), (20, [21]), (0, [3, 4])]),
]


@pytest.mark.parametrize("case", range(len(PREFIX_CASES)))
@pytest.mark.parametrize("more", [2, 7, 64])
def test_prefix(case, more):
    n_kv, G, groups = PREFIX_CASES[case]
    g, cache, table, lens = prefix_paged(case, groups, n_kv)
    R, H = len(lens), n_kv * G
    cu = [0]
    for _, ls in groups:
        cu.append(cu[-1] + len(ls))
    q = torch.randn(R, H, 128, device=DEV, generator=g).to(BF16)
    lse = torch.full((R, H), 7.0, device=DEV)
    out = run_prefix(q, cache, table, lens, cu, [p for p, _ in groups], n_kv, G, lse=lse,
                     floats=more * R * H * 130)
    for r, l in enumerate(lens):
        want = want_window(q[r:r + 1], cache[:, 0], cache[:, 1], table[r], l, 1, 2 ** 31 - 1, 0)
        check(out[r:r + 1], lse[r:r + 1], want, r)


@pytest.mark.parametrize("case", [3, 5, 7, 9, 10])
def test_prefix_queries_that_are_not_finite(case):
    n_kv, G, groups = PREFIX_CASES[case]
    g, cache, table, lens = prefix_paged(case, groups, n_kv)
    R, H = len(lens), n_kv * G
    cu = [0]
    for _, ls in groups:
        cu.append(cu[-1] + len(ls))
    q = torch.randn(R, H, 128, device=DEV, generator=g).to(BF16)
    spoil(q, g)
    for more in (2, 64):
        lse = torch.full((R, H), 7.0, device=DEV)
        out = run_prefix(q, cache, table, lens, cu, [p for p, _ in groups], n_kv, G, lse=lse,
                         floats=more * R * H * 130)
        for r, l in enumerate(max(x, 0) for x in lens):
            check_not_finite(q[r:r + 1], out[r:r + 1], lse[r:r + 1], ref.gather(cache[:, 0], table[r], l),
                             ref.gather(cache[:, 1], table[r], l),
                             torch.ones(1, l, dtype=torch.bool, device=DEV), r)


def test_prefix_rows_outside_groups_and_empty_groups():
    """Groups may be empty; rows before the first and behind the last are left alone."""
    n_kv, G = 2, 4
    g, cache, table, lens = prefix_paged(3, [(0, [9]), (40, [50, 60]), (0, [7])], n_kv)
    q = torch.randn(4, 8, 128, device=DEV, generator=g).to(BF16)
    out = torch.full_like(q, 7.0)
    lse = torch.full((4, 8), 7.0, device=DEV)
    run_prefix(q, cache, table, lens, [1, 1, 3, 3], [30, 40, 10], n_kv, G, out=out, lse=lse)
    assert bool((out[[0, 3]] == 7).all()) and bool((lse[[0, 3]] == 7).all())
    for r in (1, 2):
        check(out[r:r + 1], lse[r:r + 1],
              want_window(q[r:r + 1], cache[:, 0], cache[:, 1], table[r], lens[r], 1, 2 ** 31 - 1, 0))


def test_prefix_unseen_slots_may_hold_anything():
    """Slots behind a request's last token and blocks of nobody: not finite."""
    n_kv, G, groups = 2, 8, [(70, [75, 81, 100]), (33, [34, 48])]
    g, cache, table, lens = prefix_paged(8, groups, n_kv)
    q = torch.randn(5, 16, 128, device=DEV, generator=g).to(BF16)
    clean = cache.clone()
    used = torch.zeros(cache.shape[0], 16, dtype=torch.bool, device=DEV)
    for r, l in enumerate(lens):
        j = torch.arange(l, device=DEV)
        used[table[r].long()[j // 16], j % 16] = True
    cache.permute(0, 2, 1, 3, 4)[~used] = float("nan")
    a = run_prefix(q, cache, table, lens, [0, 3, 5], [70, 33], n_kv, G)
    b = run_prefix(q, clean, table, lens, [0, 3, 5], [70, 33], n_kv, G)
    assert torch.equal(a, b) and bool(a.isfinite().all())


# ---- the step ------------------------------------------------------------------------------
def test_step_together_and_captured():
    """Prompts in, then decode steps: plan, norm + rotation + write, attention; the
    same sequence again from a captured graph.  The cache, the lengths and the
    outputs follow a plain loop that keeps each request's keys in a list."""
    from locks.attention import (append_plan, norm_rope_and_cache, shared_prefix_paged_decode,
                                 window_paged_attention)
    R, n_kv, G, W, cap = 3, 2, 4, 8, 96
    H = n_kv * G
    g = torch.Generator(device=DEV).manual_seed(1)
    cache = torch.full((30, 2, 16, n_kv, 128), float("nan"), device=DEV, dtype=BF16)
    table = torch.full((R, W), -1, dtype=I32, device=DEV)
    free = torch.randperm(30, device=DEV, generator=g).to(I32)
    lens, taken = i32([0] * R), i32([0])
    slots, pos = (torch.empty(cap, dtype=I64, device=DEV) for _ in range(2))
    cu, new, status = i32([0] * (R + 1)), i32([0] * R), i32([0])
    wq, wk = (torch.rand(128, device=DEV, generator=g) + 0.5 for _ in range(2))
    ang = torch.rand(200, 64, device=DEV, generator=g) * 6
    cs = torch.cat([ang.cos(), ang.sin()], 1)
    qkv = torch.zeros(cap, H + 2 * n_kv, 128, device=DEV, dtype=BF16)
    q, k, v = qkv[:, :H], qkv[:, H:H + n_kv], qkv[:, H + n_kv:]
    qr, out, out2 = (torch.zeros(cap, H, 128, device=DEV, dtype=BF16) for _ in range(3))
    scratch = torch.empty(2 ** 18, device=DEV)
    groups, pre = i32([0, R]), i32([0])

    def step(max_q):
        append_plan(lens, new, table, free, taken, slot_mapping=slots, positions=pos,
                    cu_tokens=cu, lens_out=lens, taken_out=taken, status=status)
        norm_rope_and_cache(q, k, v, cache, slots, pos, cs, q_weight=wq, k_weight=wk, q_out=qr)
        window_paged_attention(qr, cache, table, cu, lens, out, n_kv=n_kv, G=G, window=20,
                               sinks=3, scale=SCALE, max_q=max_q, scratch=scratch, status=status)
        if max_q == 1:
            shared_prefix_paged_decode(qr[:R], cache, table, lens, groups, pre, out2[:R],
                                       n_kv=n_kv, G=G, scale=SCALE, scratch=scratch,
                                       status=status)

    keys = [torch.zeros(0, n_kv, 128, device=DEV, dtype=torch.float64) for _ in range(R)]
    vals = list(keys)

    def expect(n):
        t0 = 0
        for r in range(R):
            L = keys[r].shape[0]
            at = slice(t0, t0 + n[r])
            t0 += n[r]
            tab = cs[L:L + n[r]]
            kk = ref.norm_rope(k[at], wk, 1e-6, tab, 128, True).to(BF16).double()
            keys[r], vals[r] = torch.cat([keys[r], kk]), torch.cat([vals[r], v[at].double()])
            end = L + n[r]
            assert int(lens[r]) == end
            # (the stored key may be one step off where the fp32 and the fp64 result
            # round apart)
            got = ref.gather(cache[:, 0], table[r], end).double()
            assert bool(((got - keys[r]).abs() <= 2 * ref.HALF_BF16 * keys[r].abs() + 1e-6).all())
            assert torch.equal(ref.gather(cache[:, 1], table[r], end).double(), vals[r])
            qq = ref.norm_rope(q[at], wq, 1e-6, tab, 128, True)
            assert bool(((qr[at].double() - qq).abs() <= ref.HALF_BF16 * qq.abs() + 1e-5).all())
            check(out[at], None, want_window(qr[at], cache[:, 0], cache[:, 1], table[r], end,
                                             n[r], 20, 3), r)
            if max(n) == 1:
                check(out2[r:r + 1], None, want_window(qr[r:r + 1], cache[:, 0], cache[:, 1],
                                                       table[r], end, 1, 2 ** 31 - 1, 0), r)

    def fill(n):
        new.copy_(torch.tensor(n, dtype=I32))
        qkv.copy_(torch.randn(qkv.shape, device=DEV, generator=g))

    for n in ([40, 17, 1], [1, 1, 1], [0, 16, 15]):
        fill(n)
        step(max(n))
        torch.cuda.synchronize()
        expect(n)
    graph = torch.cuda.CUDAGraph()
    saved = [t.clone() for t in (lens, taken, table, cache)]
    fill([1, 1, 1])
    with torch.cuda.graph(graph):
        step(1)
    for t, s in zip((lens, taken, table, cache), saved):
        t.copy_(s)
    for _ in range(20):                                   # across page borders
        fill([1, 1, 1])
        graph.replay()
        torch.cuda.synchronize()
        expect([1, 1, 1])
    assert int(status) == 0


@pytest.mark.parametrize("R", [1, 4])
def test_norm_in_front_of_the_sparse_path_with_short_requests(R):
    """Requests inside their recent window give the scorer nothing to do; the decode
    behind it must still see the queries and the cache rows the head norm stores.  Two
    layers over one set of selection buffers, eager and captured, the same bits as
    without programmatic launches."""
    from locks import _cabi
    from locks.attention import norm_rope_and_cache, sparse_paged_decode_fused
    from locks.config import LocksConfig
    from locks.hotpath import HotPath
    from locks.selection.rki4_score import rki4_score_state
    L, n_kv, G, T = 2, 2, 4, 6000
    H, lens = n_kv * G, [20, 33, 7, 48][:R]
    g = torch.Generator(device=DEV).manual_seed(17)
    base = [torch.randn(-(-T // 16) + 12, 2, 16, n_kv, 128, device=DEV, generator=g).to(BF16)
            for _ in range(L)]
    caches = [c.clone() for c in base]
    table = torch.arange(1, 1 + 3 * R, device=DEV, dtype=I32).reshape(R, 3)
    sl = i32(lens)
    cfg = LocksConfig(budget_pages=2, sink_pages=1, window_pages=8)
    hp = HotPath(caches, table, sl, n_kv=n_kv, G=G, scale=SCALE, cfg=cfg)
    hp.derive()
    assert bool((hp.st.n_sel_hi[:R] <= 0).all())
    # a long norm launch whose last tokens are the requests' own
    qkv = torch.randn(L, T, H + 2 * n_kv, 128, device=DEV, generator=g).to(BF16)
    slots = torch.arange(T, device=DEV) + 13 * 16
    slots[T - R:] = torch.tensor([int(table[r, (n - 1) // 16]) * 16 + (n - 1) % 16
                                  for r, n in enumerate(lens)], device=DEV)
    slots[T - R - 400:T - R] = -1
    w = torch.rand(128, device=DEV, generator=g) + 0.5
    qr, out = (torch.zeros(L, T, H, 128, device=DEV, dtype=BF16) for _ in range(2))

    def step():
        for l in range(L):
            norm_rope_and_cache(qkv[l, :, :H], qkv[l, :, H:H + n_kv], qkv[l, :, H + n_kv:],
                                caches[l], slots, None, None, q_weight=w, k_weight=w, q_out=qr[l])
            q = qr[l, T - R:]
            rki4_score_state(hp.st, l, q, table, sl, R, SCALE)
            sparse_paged_decode_fused(q, caches[l], table, sl, hp.st, out[l, :R], hp.vsources[l])

    def fresh(run):
        qr.fill_(3.0)
        out.fill_(float("nan"))
        for c, b in zip(caches, base):
            c.copy_(b)
        torch.cuda.synchronize()
        run()
        torch.cuda.synchronize()
        return out[:, :R].clone()

    old = _cabi.lib().locks_set_pdl(0)
    try:
        want = fresh(step)
    finally:
        _cabi.lib().locks_set_pdl(old)
    for l in range(L):
        for r, n in enumerate(lens):
            o, _, mean, _ = want_window(qr[l, T - R + r:T - R + r + 1], caches[l][:, 0], caches[l][:, 1],
                                        table[r], n, 1, 2 ** 31 - 1, 0)
            assert bool(((want[l, r:r + 1].double() - o).abs() <= 2e-2 + 1e-2 * mean).all())
    for _ in range(10):
        assert torch.equal(fresh(step), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(10):
        assert torch.equal(fresh(graph.replay), want)
