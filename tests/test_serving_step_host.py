"""Refusals of the serving step's operators: every one is made before a launch, so
they are tested without a GPU."""
from __future__ import annotations

import ctypes

import pytest
import torch

from locks import _cabi
from locks._build import build_library

P = ctypes.c_void_p
A = P(1 << 20)            # an aligned address that nothing reads: the calls are refused


@pytest.fixture(scope="module", autouse=True)
def _library():
    build_library()


def rc(name, args):
    return getattr(_cabi.lib(), name)(*args), _cabi.lib().locks_last_error().decode()


def with_(args, **change):
    names, values = zip(*args)
    return [change.get(n, v) for n, v in zip(names, values)]


PLAN = [("seq_lens", A), ("n_new", A), ("table", A), ("bt_stride", 8), ("width", 8), ("free", A),
        ("n_free", 4), ("taken", A), ("slots", A), ("pos", A), ("cu", A), ("lens_out", A),
        ("taken_out", A), ("n_req", 2), ("cap", 16), ("page", 16), ("status", None), ("stream", None)]
NORM = [("q", A), ("q_tok", 512), ("q_head", 128), ("k", A), ("k_tok", 256), ("k_head", 128), ("v", A),
        ("v_tok", 256), ("v_head", 128), ("q_out", A), ("o_tok", 512), ("o_head", 128), ("kc", A),
        ("vc", A), ("cb", 8192), ("ct", 256), ("ch", 128), ("slot", A), ("pos", A), ("cs", A),
        ("cs_row", 128), ("n_pos", 9), ("rot", 128), ("neox", 1), ("t32", 0), ("wq", A), ("wk", A),
        ("w32", 0), ("eps", 1e-6), ("n_tok", 2), ("H", 4), ("n_kv", 2), ("d", 128), ("page", 16),
        ("NB", 4), ("stream", None)]
WINDOW = [("q", A), ("q_tok", 512), ("q_head", 128), ("k", A), ("v", A), ("sb", 8192), ("st", 256),
          ("sh", 128), ("table", A), ("bt_stride", 8), ("width", 8), ("NB", 4), ("cu", A), ("lens", A),
          ("out", A), ("o_tok", 512), ("o_head", 128), ("lse", None), ("lse_tok", 0), ("scratch", None),
          ("floats", 0), ("n_tok", 2), ("n_req", 2), ("max_q", 1), ("n_kv", 2), ("G", 2), ("d", 128),
          ("page", 16), ("window", 8), ("sinks", 0), ("scale", 0.1), ("status", None), ("stream", None)]
PREFIX = [("q", A), ("q_tok", 512), ("q_head", 128), ("k", A), ("v", A), ("sb", 8192), ("st", 256),
          ("sh", 128), ("table", A), ("bt_stride", 8), ("width", 8), ("NB", 4), ("lens", A), ("cu", A),
          ("pre", A), ("out", A), ("o_tok", 512), ("o_head", 128), ("lse", None), ("lse_tok", 0),
          ("scratch", A), ("floats", 1 << 20), ("n_req", 2), ("n_groups", 1), ("n_kv", 2), ("G", 2),
          ("d", 128), ("page", 16), ("scale", 0.1), ("status", None), ("stream", None)]
ODD = P((1 << 20) + 8)


@pytest.mark.parametrize("change,code,word", [
    (dict(seq_lens=None), -1, "null"), (dict(free=None), -1, "null"), (dict(slots=None), -1, "null"),
    (dict(taken_out=None), -1, "null"), (dict(n_req=0), -1, "size"), (dict(bt_stride=7), -1, "size"),
    (dict(page=0), -1, "size"), (dict(page=1 << 29), -1, "size"), (dict(cap=-1), -1, "size"), (dict(n_req=4097), -4, "4096")])
def test_plan_refusals(change, code, word):
    got, msg = rc("locks_append_plan", with_(PLAN, **change))
    assert got == code and word in msg


@pytest.mark.parametrize("change,code,word", [
    (dict(q=None), -1, "null"), (dict(slot=None), -1, "null"), (dict(d=64), -2, "head_dim"),
    (dict(page=32), -2, "page"), (dict(q=ODD), -1, "aligned"), (dict(k_tok=252), -1, "aligned"),
    (dict(cb=8188), -1, "aligned"), (dict(rot=130), -1, "rot_dim"), (dict(rot=7), -1, "rot_dim"),
    (dict(pos=None), -1, "rotation"), (dict(cs_row=64), -1, "rotation"), (dict(wq=ODD), -1, "weights"),
    (dict(n_kv=0), -1, "size"), (dict(n_tok=-1), -1, "size"), (dict(n_tok=0), 0, "")])
def test_norm_refusals(change, code, word):
    got, msg = rc("locks_norm_rope_write", with_(NORM, **change))
    assert got == code and word in msg


SHARED = [(dict(q=None), -1, "null"), (dict(lens=None), -1, "null"), (dict(cu=None), -1, "null"),
          (dict(d=64), -2, "head_dim"), (dict(page=8), -2, "page"), (dict(G=17), -2, "G <= 16"),
          (dict(G=0), -2, "G <= 16"), (dict(st=252), -1, "aligned"), (dict(q=ODD), -1, "aligned"),
          (dict(out=ODD), -1, "aligned"), (dict(scratch=ODD), -1, "aligned"), (dict(n_kv=0), -1, "size"),
          (dict(sh=136), -2, "multiple of 64"), (dict(sb=0), -1, "stride"), (dict(scale=0.0), -1, "positive"),
          (dict(scale=float("nan")), -1, "positive"), (dict(width=0), -1, "size"), (dict(n_req=65536), -1, "size"), (dict(n_req=0), 0, "")]


@pytest.mark.parametrize("change,code,word", SHARED + [
    (dict(window=-1), -1, "size"), (dict(sinks=-1), -1, "size"), (dict(max_q=-1), -1, "size"),
    (dict(max_q=0), 0, ""), (dict(n_tok=0), 0, "")])
def test_window_refusals(change, code, word):
    got, msg = rc("locks_window_attention", with_(WINDOW, **change))
    assert got == code and word in msg


@pytest.mark.parametrize("change,code,word", SHARED + [
    (dict(scratch=None), -1, "null"), (dict(pre=None), -1, "null"), (dict(floats=2079), -4, "2080"),
    (dict(n_groups=-1), -1, "size"), (dict(n_groups=0), 0, "")])
def test_prefix_refusals(change, code, word):
    got, msg = rc("locks_shared_prefix_decode", with_(PREFIX, **change))
    assert got == code and word in msg


def test_wrappers_refuse_host_tensors():
    from locks.attention import (append_plan, norm_rope_and_cache, shared_prefix_paged_decode,
                                 window_paged_attention)
    i, b = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 4, 128, dtype=torch.bfloat16)
    cache, cu = torch.zeros(3, 2, 16, 2, 128, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32)
    table, wide = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        append_plan(i, i, table, i, i[:1], slot_mapping=wide, positions=wide, cu_tokens=cu,
                    lens_out=i, taken_out=i[:1])
    with pytest.raises(RuntimeError, match="no CPU path"):
        norm_rope_and_cache(b, b[:, :2], b[:, :2], cache, wide, None, None)
    with pytest.raises(RuntimeError, match="no CPU path"):
        window_paged_attention(b, cache, table, cu, i, b, n_kv=2, G=2, window=4, scale=1.0, max_q=1)
    with pytest.raises(RuntimeError, match="no CPU path"):
        shared_prefix_paged_decode(b, cache, table, i, cu[:2], i[:1], b, n_kv=2, G=2, scale=1.0,
                                   scratch=torch.zeros(2048))
