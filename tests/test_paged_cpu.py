"""Refusals of the batched-decode entry points: argument checks that run on
the host, before any CUDA call."""

import ctypes as C

import pytest
import torch

from streamlx_b200 import _lib as L
from streamlx_b200 import ops

PTR = 1 << 20       # a 16-byte aligned address no check follows


def kv(**kw):
    f = dict(base=PTR, k_scale=None, v_scale=None, n_pages=8, page_size=16,
             n_kv=2, head_dim=128, dtype=L.KV_BF16)
    f.update(kw)
    return L.slx_kv_pages(**f)


def attn(pages=None, **kw):
    a = dict(q=PTR, q_stride=16 * 128, T=3, n_q=16, table=PTR, n_req=3,
             max_pages=4, req=None, pos=PTR, scale=0.1, out=PTR, ws=PTR,
             ws_bytes=1 << 30)
    a.update(kw)
    p = kv() if pages is None else pages
    return L.lib().slx_paged_attn_decode(
        a["q"], a["q_stride"], a["T"], a["n_q"], C.byref(p) if p else None,
        a["table"], a["n_req"], a["max_pages"], a["req"], a["pos"],
        a["scale"], a["out"], a["ws"], a["ws_bytes"], None, None)


def append(pages=None, **kw):
    a = dict(qkv=PTR, stride=20 * 128, T=3, n_q=16, qn=PTR, kn=PTR,
             inv=PTR, pos=PTR, slot=PTR, out=PTR)
    a.update(kw)
    p = kv() if pages is None else pages
    return L.lib().slx_paged_append(
        a["qkv"], a["stride"], a["T"], a["n_q"], a["qn"], a["kn"], 1e-6,
        a["inv"], a["pos"], a["slot"], C.byref(p) if p else None, a["out"],
        None, None)


@pytest.fixture(autouse=True)
def no_error_left():
    yield
    assert attn(T=0) == 0       # a call that passes clears the message


BAD_PAGES = [
    (dict(base=None), -1), (dict(base=PTR + 8), -1), (dict(dtype=2), -2),
    (dict(head_dim=96), -2), (dict(head_dim=256), -2), (dict(page_size=8), -2),
    (dict(page_size=48), -2), (dict(page_size=512), -2), (dict(n_pages=0), -1),
    (dict(n_pages=1 << 28), -1), (dict(n_kv=0), -1),
    (dict(dtype=L.KV_E4M3), -1), (dict(k_scale=PTR), -1)]


@pytest.mark.parametrize("fields,code", BAD_PAGES)
def test_bad_pages(fields, code):
    for call in (attn, append):
        assert call(kv(**fields)) == code
        assert L.lib().slx_last_error_string() != b""


@pytest.mark.parametrize("kw", [
    dict(T=-1), dict(n_q=15), dict(n_q=0), dict(n_q=34), dict(n_req=0),
    dict(n_req=2), dict(max_pages=0), dict(max_pages=1 << 28),
    dict(max_pages=(1 << 26) + 1), dict(q=None),
    dict(q=PTR + 8), dict(q_stride=16 * 128 - 8), dict(q_stride=16 * 128 + 4),
    dict(table=None), dict(pos=None), dict(out=None), dict(out=PTR + 2)])
def test_bad_attention(kw):
    assert attn(**kw) == -1


def test_no_rows_is_no_launch():
    assert attn(T=0, q=None, out=None) == 0
    assert append(T=0, qkv=None) == 0


@pytest.mark.parametrize("kw", [
    dict(T=-1), dict(n_q=3), dict(n_q=0), dict(n_q=65534), dict(qkv=None),
    dict(qkv=PTR + 2), dict(stride=20 * 128 - 8), dict(stride=20 * 128 + 2),
    dict(qn=None), dict(kn=PTR + 4), dict(inv=None), dict(pos=None),
    dict(slot=None), dict(out=None), dict(out=PTR + 8)])
def test_bad_append(kw):
    assert append(**kw) == -1


@pytest.mark.parametrize("kw,code", [
    (dict(n_req=0), -2), (dict(n_req=8193), -2), (dict(page=8), -2),
    (dict(page=24), -2), (dict(max_pages=0), -1), (dict(n_pages=0), -1),
    (dict(max_pages=1 << 28), -1), (dict(n_pages=1 << 28), -1),
    (dict(n_rows=-1), -1), (dict(rows=None), -1), (dict(table=None), -1),
    (dict(free=None), -1), (dict(n_new=None), -1)])
def test_bad_plan(kw, code):
    a = dict(n_new=PTR, n_req=4, table=PTR, max_pages=4, page=16, free=PTR,
             n_pages=9, rows=PTR, n_rows=8)
    a.update(kw)
    assert L.lib().slx_paged_plan(
        a["n_new"], PTR, PTR, a["n_req"], a["table"], a["max_pages"],
        a["page"], a["free"], a["n_pages"], PTR, PTR, a["rows"], a["rows"],
        a["rows"], a["n_rows"], PTR, None, None) == code


@pytest.mark.parametrize("rules,kw", [
    ({}, dict(V=0)), ({}, dict(T=-1)), ({}, dict(logits=None)),
    ({}, dict(logits=PTR + 1)), ({}, dict(logits=PTR + 2, f32=1)),
    ({}, dict(out=None, pick=None)),
    (dict(history=PTR, history_stride=8), {}),
    (dict(history=PTR, n_history=PTR, history_stride=262144), {}),
    (dict(history=PTR, n_history=PTR, history_stride=-1), {}),
    (dict(repetition=PTR), {}), (dict(presence=PTR), {}),
    (dict(bias_ids=PTR, bias_values=PTR, n_bias=4), {}),
    (dict(bias_start=PTR), {}),
    (dict(bias_ids=PTR, bias_values=PTR, bias_start=PTR, n_bias=-1), {}),
    (dict(mask=PTR, mask_stride=3), {})])
def test_bad_logits(rules, kw):
    a = dict(logits=PTR, f32=0, T=2, V=100, out=PTR, pick=PTR)
    a.update(kw)
    r = L.slx_logit_rules(**rules)
    assert L.lib().slx_logits_process(a["logits"], a["f32"], a["T"], a["V"],
                                      C.byref(r), a["out"], a["pick"], None,
                                      None) == -1


def test_workspace_bytes():
    f = L.paged_attn_workspace_bytes
    assert f(4, 24, 4, 96) == 0 and f(4, 25, 4, 128) == 0
    assert f(4, 68, 4, 128) == 0 and f(-1, 24, 4, 128) == 0


def test_ops_want_cuda_tensors():
    i = torch.zeros(4, dtype=torch.int32)
    pages = torch.zeros(2, 2, 1, 16, 64, dtype=torch.bfloat16)
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ops.paged_plan(i, i, i.reshape(4, 1), i, i[:1], 16, 4)
    with pytest.raises(ValueError):
        ops.paged_attention(q, pages, i.reshape(4, 1), i)
    with pytest.raises(ValueError):
        ops.paged_append(q.reshape(4, -1), pages, i, i, 0, q, q, 1e-6, i)
    with pytest.raises(ValueError):
        ops.process_logits(torch.zeros(2, 10))
