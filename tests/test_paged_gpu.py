"""Batched decode over a paged KV cache against plain 64-bit restatements
(tests/paged_cases.py): the step's plan, the append and the attention."""

import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from streamlx_b200 import _lib as L
from streamlx_b200 import ops
from tests import paged_cases as P

pytestmark = pytest.mark.gpu

BF, E4 = torch.bfloat16, torch.float8_e4m3fn
EPS = 1e-6


def dev_cache(*args, **kw):
    pages, sc, table = P.make_cache(*args, **kw)
    return (pages, sc, table), (pages.cuda(), None if sc is None else sc.cuda(),
                                table.cuda())


def queries(T, nq, hd, seed=1, std=1.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, nq, hd, generator=g) * std).to(BF)


def run_attention(q, dev, req, pos, scale=None, **kw):
    pages, sc, table = dev
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = ops.paged_attention(
        q.cuda(), pages, table, torch.tensor(pos, dtype=torch.int32).cuda(),
        req=None if req is None else torch.tensor(req, dtype=torch.int32).cuda(),
        scale=scale, kv_scale=sc, status=st, **kw)
    torch.cuda.synchronize()
    return out.cpu(), int(st.item())


def check_attention(q, host, dev, req, pos, scale=None, **kw):
    page, hd = host[0].shape[3], host[0].shape[4]
    out, st = run_attention(q, dev, req, pos, scale, **kw)
    assert st == 0
    want, bound = P.attention(q, host[0], host[1], host[2],
                              req or range(len(pos)), pos, page,
                              hd ** -0.5 if scale is None else scale)
    err = (out.double() - want).abs()
    assert torch.isfinite(out).all()
    assert (err <= bound).all(), float((err / bound.clamp(min=1e-30)).max())
    return out


# ------------------------------------------------------------- attention --

HEADS = [(24, 4), (16, 2), (1, 1), (8, 8), (32, 2), (9, 3), (12, 1)]


@pytest.mark.parametrize("dtype", [BF, E4])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nq,nkv", HEADS)
def test_attention_ragged(nq, nkv, hd, dtype):
    """Lengths around page and tile ends, an idle row, NaN in every place of
    the cache that no row holds, -1 in the table behind the last page."""
    lens = [1, 0, 15, 16, 17, 33, 64, 100, 129, 255]
    host, dev = dev_cache(lens, nkv, hd, 16, dtype, seed=nq + hd)
    q = queries(len(lens), nq, hd)
    out = check_attention(q, host, dev, None, [n - 1 for n in lens])
    assert (out[1] == 0).all()


@pytest.mark.parametrize("dtype", [BF, E4])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_attention_pages(page, dtype):
    lens = [page - 1, page, page + 1, 3 * page + 5, 700]
    host, dev = dev_cache(lens, 2, 128, page, dtype, seed=page)
    check_attention(queries(len(lens), 16, 128), host, dev, None,
                    [n - 1 for n in lens])


@pytest.mark.parametrize("nq,nkv,hd,dtype,lens", [
    (16, 2, 128, BF, [20000]), (24, 4, 128, E4, [9001, 3, 0, 1]),
    (8, 1, 64, BF, [1, 12345, 2]), (4, 4, 64, E4, [8192])])
def test_attention_long(nq, nkv, hd, dtype, lens):
    """The cache's length split over many CTAs and joined."""
    host, dev = dev_cache(lens, nkv, hd, 32, dtype, seed=3)
    check_attention(queries(len(lens), nq, hd), host, dev, None,
                    [n - 1 for n in lens])


@pytest.mark.parametrize("dtype", [BF, E4])
def test_attention_many_rows(dtype):
    """More rows than CTAs of one wave, short and long ones mixed."""
    g = np.random.default_rng(5)
    lens = [int(n) for n in g.integers(0, 60, 600)]
    lens[17], lens[599] = 3000, 900
    host, dev = dev_cache(lens, 2, 64, 16, dtype, seed=9)
    check_attention(queries(len(lens), 4, 64), host, dev, None,
                    [n - 1 for n in lens])


@pytest.mark.parametrize("dtype", [BF, E4])
@pytest.mark.parametrize("nq,nkv,hd", [(24, 4, 128), (8, 8, 64), (4, 2, 128),
                                       (9, 3, 64), (12, 1, 64), (1, 1, 128)])
def test_attention_prompt_rows(nq, nkv, hd, dtype):
    """Several rows of one request (each its own causal length), requests in
    any order, padding rows, the same row twice."""
    lens = [70, 5, 300]
    host, dev = dev_cache(lens, nkv, hd, 16, dtype, seed=4)
    req = [2] * 20 + [0] * 9 + [-1] + [1] + [0] + [2, 2] + [0, 0, 0, 2]
    pos = [280 + i for i in range(20)] + [61 + i for i in range(9)] + \
        [-1] + [4] + [0] + [31, 31] + [50, -1, 3, 299]
    out = check_attention(queries(len(req), nq, hd), host, dev, req, pos)
    assert (out[29] == 0).all() and (out[35] == 0).all()


@pytest.mark.parametrize("dtype", [BF, E4])
@pytest.mark.parametrize("nq,nkv,hd", [(8, 8, 64), (4, 2, 128), (12, 4, 128),
                                       (9, 1, 64)])
def test_attention_prompt_rows_hide_later_values(nq, nkv, hd, dtype):
    """Infinite and NaN values of later tokens of a request do not reach the
    rows before them, and do reach the rows that attend them."""
    lens = [60, 200]
    host, dev = dev_cache(lens, nkv, hd, 16, dtype, seed=14)
    pages = host[0].float()
    for i, n, bad in ((0, 43, float("nan")), (1, 190, float("nan")),
                      (1, 196, float("nan") if dtype == E4 else float("inf"))):
        pages[int(host[2][i, n // 16]), 1, :, n % 16] = bad
    pages = pages.to(dtype)
    dev = (pages.cuda(), dev[1], dev[2])
    req = [0] * 16 + [1] * 24
    pos = list(range(35, 51)) + list(range(176, 200))
    q = queries(40, nq, hd)
    out, st = run_attention(q, dev, req, pos)
    clean = [r for r in range(40) if pos[r] < (43 if req[r] == 0 else 190)]
    rest = [r for r in range(40) if r not in clean]
    assert st == 0 and torch.isnan(out[rest]).all()
    want, bound = P.attention(q[clean], pages, host[1], host[2],
                              [req[r] for r in clean],
                              [pos[r] for r in clean], 16, hd ** -0.5)
    assert ((out[clean].double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [BF, E4])
@pytest.mark.parametrize("nq,nkv,hd", [(8, 8, 64), (4, 2, 128), (9, 3, 64)])
def test_attention_rows_of_requests_in_turn(nq, nkv, hd, dtype):
    """Rows of two requests alternating, the later ones longer: rows that
    follow a row of another request are not the first one's group."""
    lens = [300, 280]
    host, dev = dev_cache(lens, nkv, hd, 16, dtype, seed=16)
    req = [0, 1] * 8 + [0, 0, 1, 0, 0, 0, 1, 1]
    pos = [int(p) for p in np.linspace(3, 270, 24)]
    check_attention(queries(24, nq, hd), host, dev, req, pos)


@pytest.mark.parametrize("dtype", [BF, E4])
def test_attention_long_prompt_rows(dtype):
    """A chunk of rows behind a long prefix: groups split over CTAs."""
    lens = [6000, 333]
    host, dev = dev_cache(lens, 2, 64, 32, dtype, seed=15)
    req = [0] * 45 + [1] * 6
    pos = list(range(5955, 6000)) + list(range(327, 333))
    check_attention(queries(51, 4, 64), host, dev, req, pos)


@pytest.mark.parametrize("dtype", [BF, E4])
@pytest.mark.parametrize("nq,nkv,hd,T", [
    (8, 8, 64, 460), (24, 4, 128, 160), (9, 3, 64, 410), (16, 2, 128, 240),
    (12, 4, 128, 300), (32, 2, 64, 140)])
def test_attention_many_prompt_rows(nq, nkv, hd, T, dtype):
    """Chunks long enough for the wider tile: ragged, some of a row, padding
    and idle rows between them, values of later tokens that are not finite."""
    g = np.random.default_rng(T)
    lens = [400, 37, 290, 64]
    host, dev = dev_cache(lens, nkv, hd, 16, dtype, seed=T)
    pages = host[0].float()
    for i, n in ((0, 190), (2, 120)):
        pages[int(host[2][i, n // 16]), 1, :, n % 16] = \
            float("inf") if dtype == BF and i else float("nan")
    pages = pages.to(dtype)
    req, pos = [], []
    while len(req) < T:
        i = int(g.integers(-1, 4))
        n = min(T - len(req), int(g.choice([1, 3, 16, 29, 70])))
        if i < 0:
            req += [-1] * min(n, 3)
            pos += [-1] * min(n, 3)
            continue
        n = min(n, lens[i])
        at = int(g.integers(0, lens[i] - n + 1))
        req += [i] * n
        pos += range(at, at + n)
    last = {0: 190, 1: 37, 2: 120, 3: 64}
    clean = [r for r in range(T) if req[r] < 0 or pos[r] < last[req[r]]]
    rest = [r for r in range(T) if req[r] >= 0 and pos[r] >= last[req[r]]]
    assert len(rest) > 0
    q = queries(T, nq, hd)
    out, st = run_attention(q, (pages.cuda(), dev[1], dev[2]), req, pos)
    assert st == 0 and not torch.isfinite(out[rest]).any()
    want, bound = P.attention(q[clean], pages, host[1], host[2],
                              [req[r] for r in clean],
                              [pos[r] for r in clean], 16, hd ** -0.5)
    assert ((out[clean].double() - want).abs() <= bound).all()


def chunk_rows(lens, first):
    """(req, pos): every request's rows from its token first[i] on."""
    req = [i for i, (n, f) in enumerate(zip(lens, first)) for _ in range(f, n)]
    return req, [p for n, f in zip(lens, first) for p in range(f, n)]


@pytest.mark.parametrize("dtype", [BF, E4])
@pytest.mark.parametrize("nq,nkv,hd,page,lens,first", [
    (24, 4, 128, 16, [200, 90, 64], [0, 26, 1]),      # from a request's start
    (16, 2, 128, 64, [130, 65], [65, 0]),
    (32, 2, 64, 32, [100, 129], [60, 100]),           # 16 heads a kv head
    (9, 3, 64, 256, [300, 500], [200, 400]),
    (13, 1, 128, 16, [150], [30]),                    # columns left over
    (8, 8, 64, 128, [700, 90], [500, 0]),
    (1, 1, 128, 16, [1100], [20])])                   # a row a column
def test_attention_chunks(nq, nkv, hd, page, lens, first, dtype):
    """Chunks of rows on the wide tiles: heads, pages, tails of every size."""
    host, dev = dev_cache(lens, nkv, hd, page, dtype, seed=nq)
    req, pos = chunk_rows(lens, first)
    assert len(req) * nq >= 1024
    check_attention(queries(len(req), nq, hd), host, dev, req, pos)


@pytest.mark.parametrize("dtype", [BF, E4])
def test_attention_chunk_behind_long_prefix(dtype):
    """Few blocks of rows: their keys split over CTAs, some parts with none
    that the first rows attend."""
    lens, first = [9000, 700], [8950, 600]
    host, dev = dev_cache(lens, 2, 128, 64, dtype, seed=21)
    req, pos = chunk_rows(lens, first)
    pos[3], pos[20] = 5, 1000
    check_attention(queries(len(req), 12, 128), host, dev, req, pos)


@pytest.mark.parametrize("scale", [0.0, 40.0, -1.0])
@pytest.mark.parametrize("dtype", [BF, E4])
def test_attention_chunk_scores(scale, dtype):
    """Maxima that keep growing (sums are scaled), and hardly grow."""
    lens, first = [520, 130], [440, 60]
    pages, sc, table = P.make_cache(lens, 2, 64, 16, dtype, seed=22)
    x = pages.float()
    for i, n in enumerate(lens):          # keys grow along the request
        for p in range(n):
            x[int(table[i, p // 16]), 0, :, p % 16] *= p / n
    pages = x.to(dtype)
    host, dev = (pages, sc, table), (pages.cuda(),
                                     None if sc is None else sc.cuda(),
                                     table.cuda())
    req, pos = chunk_rows(lens, first)
    check_attention(queries(len(req), 16, 64), host, dev, req, pos, scale=scale)


@pytest.mark.parametrize("dtype", [BF, E4])
def test_attention_chunk_bad_indices(dtype):
    """Pages, requests and positions out of range in chunks: the status, zeros
    read or written, the other rows untouched."""
    lens, first = [200, 150], [100, 60]
    host, dev = dev_cache(lens, 2, 128, 16, dtype, seed=23)
    pages, sc, table = dev
    req, pos = chunk_rows(lens, first)
    q = queries(len(req), 16, 128)
    good = check_attention(q, host, dev, req, pos)
    one = [r for r in range(len(req)) if req[r] == 1]
    zero = [r for r in range(len(req)) if req[r] == 0]
    for bad in (-1, pages.shape[0], 2 ** 31 - 1):
        t = table.clone()
        t[1, 2] = bad
        out, st = run_attention(q, (pages, sc, t), req, pos)
        assert st == L.SLX_ERR_OUT_OF_RANGE
        assert torch.equal(out[zero], good[zero])
        clear = host[0].float()
        clear[int(host[2][1, 2])] = 0
        want, bound = P.attention(q[one], clear.to(dtype), host[1], host[2],
                                  [1] * len(one), [pos[r] for r in one], 16,
                                  128 ** -0.5)
        assert ((out[one].double() - want).abs() <= bound).all()
    for r, (i, p) in ((5, (2, 50)), (60, (-1, 50)), (120, (1, 16 * 99)),
                      (121, (0, 2 ** 31 - 1)), (7, (0, -1))):
        rq, ps = list(req), list(pos)
        rq[r], ps[r] = i, p
        out, st = run_attention(q, dev, rq, ps)
        rest = [k for k in range(len(req)) if k != r]
        assert st == (0 if p == -1 else L.SLX_ERR_OUT_OF_RANGE)
        assert (out[r] == 0).all() and torch.equal(out[rest], good[rest])


@pytest.mark.parametrize("dtype", [BF, E4])
def test_attention_chunk_infinite_and_nan_keys(dtype):
    """A NaN key makes the rows that attend it NaN and no other; infinite keys
    (bf16) follow the formula."""
    lens, first = [150, 140], [70, 60]
    host, dev = dev_cache(lens, 1, 64, 16, dtype, seed=24)
    pages = dev[0]
    pages[int(host[2][0, 100 // 16]), 0, 0, 100 % 16] = float("nan")
    q = torch.ones(160, 16, 64, dtype=BF)
    req, pos = chunk_rows(lens, first)
    clean = [r for r in range(160) if req[r] == 1 or pos[r] < 100]
    rest = [r for r in range(160) if r not in clean]
    if dtype == BF:                        # weight 0 for every row behind it
        pages[int(host[2][1, 5]), 0, 0, 3] = float("-inf")
    out, st = run_attention(q, dev, req, pos)
    assert st == 0 and torch.isnan(out[rest]).all()
    want, _ = P.attention(q[clean], pages.cpu(), host[1], host[2],
                          [req[r] for r in clean], [pos[r] for r in clean], 16,
                          64 ** -0.5)
    err = (out[clean].double() - want).abs()
    assert (err <= 2.0 ** -7 * want.abs() + 1e-3).all()


def test_attention_chunk_strides_streams_graphs():
    """Strided queries, the same bits in every call, calls on two streams and
    in two graphs at once."""
    lens, first = [1000, 300], [900, 230]
    host, dev = dev_cache(lens, 2, 128, 16, BF, seed=25)
    pages, _, table = dev
    req, pos = (torch.tensor(v, dtype=torch.int32).cuda()
                for v in chunk_rows(lens, first))
    T = len(req)
    wide = torch.randn(T, 20 * 128, generator=torch.Generator().manual_seed(2))
    q = wide.to(BF).cuda()[:, 256:256 + 16 * 128].unflatten(1, (16, 128))
    want = ops.paged_attention(q, pages, table, pos, req=req)
    check_attention(q.cpu(), host, dev, req.tolist(), pos.tolist())
    ws = ops.paged_workspace(T, 16, 2, 128, "cuda")
    for _ in range(10):
        got = ops.paged_attention(q.contiguous(), pages, table, pos, req=req,
                                  workspace=ws)
        assert torch.equal(got, want)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs, graphs = [], []
    for s in streams:
        with torch.cuda.stream(s):
            for _ in range(10):
                outs.append(ops.paged_attention(q, pages, table, pos, req=req))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    for _ in streams:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            a = ops.paged_attention(q, pages, table, pos, req=req)
            b = ops.paged_attention(a, pages, table, pos, req=req)
        graphs.append((g, a, b))
    two = ops.paged_attention(want, pages, table, pos, req=req)
    torch.cuda.synchronize()
    for s, (g, _, _) in zip(streams, graphs):
        with torch.cuda.stream(s):
            for _ in range(5):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, want) and torch.equal(b, two)
               for _, a, b in graphs)


@pytest.mark.parametrize("dtype", [BF, E4])
@pytest.mark.parametrize("nq,nkv,hd", [(24, 4, 128), (8, 4, 64), (4, 1, 128)])
def test_attention_short_chunks(nq, nkv, hd, dtype):
    """Requests of a few rows each: two column tiles of the kernel for single
    tokens, more rows than one of its column tiles holds."""
    g = np.random.default_rng(nq)
    lens = [int(n) for n in g.integers(20, 300, 60)]
    each = 4 if nq == 24 else 8
    host, dev = dev_cache(lens, nkv, hd, 16, dtype, seed=26)
    req, pos = chunk_rows(lens, [n - each for n in lens])
    req[10], pos[10] = -1, -1
    out = check_attention(queries(len(req), nq, hd), host, dev, req, pos)
    assert (out[10] == 0).all()


def test_attention_strided_queries():
    """q as the head part of wider rows, and a row stride beyond them."""
    lens = [40, 7, 90]
    host, dev = dev_cache(lens, 2, 128, 16, BF, seed=6)
    wide = torch.randn(3, 24 * 128 + 64).to(BF).cuda()
    q = wide[:, 128:128 + 16 * 128].unflatten(1, (16, 128))
    pages, sc, table = dev
    pos = torch.tensor([n - 1 for n in lens], dtype=torch.int32).cuda()
    a = ops.paged_attention(q, pages, table, pos)
    b = ops.paged_attention(q.contiguous(), pages, table, pos)
    assert torch.equal(a, b)


@pytest.mark.parametrize("scale", [0.0, 40.0, -1.0])
def test_attention_extreme_scores(scale):
    """Equal scores, scores far apart (one key takes all), a negative scale."""
    lens = [500, 3, 64]
    host, dev = dev_cache(lens, 2, 128, 16, BF, seed=7)
    check_attention(queries(3, 16, 128), host, dev, None,
                    [n - 1 for n in lens], scale=scale)


def test_attention_infinite_and_nan_keys():
    """What the rows do hold follows the formula: an infinite score takes a
    row's weight away or makes it NaN, and touches no other row."""
    lens = [30, 200, 31]
    host, dev = dev_cache(lens, 1, 64, 16, BF, seed=8)
    pages, _, table = dev
    q = torch.ones(3, 2, 64, dtype=BF)
    page0, page2 = int(host[2][0, 1]), int(host[2][2, 0])
    pages[page0, 0, 0, 3] = float("-inf")         # request 0, key 19: weight 0
    pages[page2, 0, 0, 5] = float("nan")          # request 2: NaN
    out, st = run_attention(q, dev, None, [29, 199, 30])
    assert st == 0 and torch.isnan(out[2]).all()
    h = host[0].clone()
    h[page0, 0, 0, 3] = float("-inf")
    want, _ = P.attention(q, h, None, host[2], [0, 1, 2], [29, 199, -1], 16,
                          64 ** -0.5)
    err = (out[:2].double() - want[:2]).abs()
    assert (err <= 2.0 ** -7 * want[:2].abs() + 1e-3).all()
    # every key of a row at -inf: nothing to divide by, NaN as the formula
    pages[int(host[2][0, 0]), 0] = float("-inf")
    pages[page0, 0] = float("-inf")
    out, st = run_attention(q, dev, None, [29, 199, -1])
    assert torch.isnan(out[0]).all() and torch.isfinite(out[1:]).all()


@pytest.mark.parametrize("dtype,hd", [(BF, 128), (E4, 128), (E4, 64)])
def test_attention_bad_indices(dtype, hd):
    """A page, request or position out of range sets the status, is not
    followed, and leaves the other rows right."""
    lens = [40, 50, 60]
    host, dev = dev_cache(lens, 2, hd, 16, dtype, seed=10)
    pages, sc, table = dev
    q = queries(3, 16, hd)
    good = check_attention(q, host, dev, None, [39, 49, 59])
    for bad in (-1, pages.shape[0], 2 ** 31 - 1):
        for col in range(4):
            t = table.clone()
            t[1, col] = bad
            out, st = run_attention(q, (pages, sc, t), None, [39, 49, 59])
            assert st == L.SLX_ERR_OUT_OF_RANGE
            assert torch.equal(out[0], good[0])
            assert torch.equal(out[2], good[2])
            # the page's keys and values read as zeros
            zero = host[0].float()
            zero[int(host[2][1, col])] = 0
            want, bound = P.attention(q[1:2], zero.to(dtype), host[1],
                                      host[2], [1], [49], 16, hd ** -0.5)
            assert ((out[1:2].double() - want).abs() <= bound).all()
    cap = table.shape[1] * 16
    for req, pos in (([0, 3, 2], [39, 49, 59]), ([0, -1, 2], [39, 49, 59]),
                     ([0, 1, 2], [39, cap, 59]),
                     ([0, 1, 2], [39, 2 ** 31 - 1, 59])):
        out, st = run_attention(q, dev, req, pos)
        assert st == L.SLX_ERR_OUT_OF_RANGE
        assert torch.equal(out[0], good[0]) and torch.equal(out[2], good[2])
        assert (out[1] == 0).all()


def test_attention_same_bits_again():
    """Repeated calls on one workspace give the same bits: the joins do not
    depend on which CTA comes last."""
    lens = [5000, 40, 0, 2500, 1]
    host, dev = dev_cache(lens, 2, 128, 16, BF, seed=11)
    q, pos = queries(5, 16, 128), [n - 1 for n in lens]
    ws = ops.paged_workspace(5, 16, 2, 128, "cuda")
    first, _ = run_attention(q, dev, None, pos, workspace=ws)
    for _ in range(20):
        out, st = run_attention(q, dev, None, pos, workspace=ws)
        assert st == 0 and torch.equal(out, first)


def test_attention_streams_and_graphs():
    """Calls on two streams at once, and two captured graphs replayed side by
    side with changed lengths, each as the call alone."""
    lens = [3000, 77, 1500]
    host, dev = dev_cache(lens, 2, 128, 16, BF, seed=12)
    pages, sc, table = dev
    q = [queries(3, 16, 128, seed=s).cuda() for s in (1, 2)]
    pos = [torch.tensor(p, dtype=torch.int32).cuda()
           for p in ([2999, 76, 1499], [1200, -1, 900])]
    want = [[ops.paged_attention(q[i], pages, table, pos[j]).clone()
             for j in range(2)] for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        outs = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs.append(ops.paged_attention(q[i], pages, table, pos[i]))
        torch.cuda.synchronize()
        assert all(torch.equal(outs[i], want[i][i]) for i in range(2))
    graphs, outs, live = [], [], [p.clone() for p in pos]
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.paged_attention(q[i], pages, table, live[i]))
        graphs.append(g)
    for j in ((0, 1), (1, 0), (1, 1)):
        for i in range(2):
            live[i].copy_(pos[j[i]])
        torch.cuda.synchronize()
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                for _ in range(5):
                    graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(outs[i], want[i][j[i]]) for i in range(2))


def test_attention_far_pages():
    """Pages whose element offsets pass 2^32."""
    n_kv, hd, page = 8, 128, 64
    per = 2 * n_kv * page * hd
    n_pages = 2 ** 32 // per + 40
    pages = torch.empty(n_pages, 2, n_kv, page, hd, dtype=E4, device="cuda")
    sc = torch.full((2, n_kv), 0.02, device="cuda")
    ids = [n_pages - 1, 3, n_pages - 7, 2 ** 31 // per + 1]
    lens = [250, 100]
    table = torch.full((2, 5), -1, dtype=torch.int32)
    table[0, :4] = torch.tensor(ids)
    table[1, :2] = torch.tensor([n_pages - 9, 11])
    used = [i for i in table.reshape(-1).tolist() if i >= 0]
    g = torch.Generator().manual_seed(0)
    small = (torch.randn(len(used), 2, n_kv, page, hd, generator=g) * 50).to(E4)
    for j, i in enumerate(used):
        pages[i].copy_(small[j])
    near = torch.full_like(table, -1)
    near[0, :4] = torch.arange(4)
    near[1, :2] = torch.arange(4, 6)
    q = queries(2, 32, hd)
    out, st = run_attention(q, (pages, sc, table.cuda()), None, [249, 99])
    want, bound = P.attention(q, small, sc.cpu(), near, [0, 1], [249, 99],
                              page, hd ** -0.5)
    assert st == 0 and ((out.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("T", [1, 33, 2000])
@pytest.mark.parametrize("dtype", [BF, E4])
def test_attention_all_rows_idle(T, dtype):
    host, dev = dev_cache([5], 2, 64, 16, dtype, seed=17)
    out, st = run_attention(queries(T, 4, 64), dev, [0] * T, [-1] * T)
    assert st == 0 and (out == 0).all()
    pos = [-1] * T
    pos[T // 2] = 4
    check_attention(queries(T, 4, 64), host, dev, [0] * T, pos)


def test_attention_many_kv_heads():
    """More kv heads than a CTA has threads."""
    lens = [70, 0, 33]
    host, dev = dev_cache(lens, 200, 64, 16, BF, seed=18)
    check_attention(queries(3, 200, 64), host, dev, None,
                    [n - 1 for n in lens])


def test_chained_launches():
    """The step's kernels under programmatic dependent launch, eagerly and in
    a graph, give the same bits as without."""
    def step(state):
        n_new, ln, table, free, nf, qkv, pages, qn, kn, inv, logits = state
        p = ops.paged_plan(n_new, ln, table, free, nf, 16, 40)
        q = ops.paged_append(qkv, pages, p.slot, p.pos, 8, qn, kn, EPS, inv)
        o = ops.paged_attention(q, pages, table, p.pos, req=p.req)
        pick = ops.process_logits(logits)
        return [*p, q, o, pick, pages, table]

    def fresh():
        g = torch.Generator(device="cuda").manual_seed(5)
        i32 = dict(dtype=torch.int32, device="cuda")

        def rn(*shape):
            return torch.randn(*shape, generator=g, device="cuda").to(BF)
        return (torch.tensor([20, 1, 0, 9], **i32),
                torch.tensor([0, 31, 5, 0], **i32),
                torch.tensor([[-1] * 6, [0, 1] + [-1] * 4, [2] + [-1] * 5,
                              [-1] * 6], **i32),
                torch.arange(3, 43, **i32) % 40, torch.tensor([37], **i32),
                rn(40, 12 * 64), rn(40, 2, 2, 16, 64), rn(64), rn(64),
                torch.rand(32, generator=g, device="cuda"), rn(40, 5000))

    want = [t.clone() for t in step(fresh())]
    prev = L.set_pdl(True)
    try:
        s1, s2 = fresh(), fresh()
        torch.cuda.synchronize()
        a = step(s1)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            b = step(s2)
        graph.replay()
        torch.cuda.synchronize()
    finally:
        L.set_pdl(prev)
    for got in (a, b):
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    ops.check_status(torch.device("cuda", torch.cuda.current_device()))


def test_first_calls_in_a_capture():
    """In a new process, the first call of every operator inside a capture."""
    code = """
import sys, torch
sys.path.insert(0, %r)
from streamlx_b200 import ops
i32 = dict(dtype=torch.int32, device='cuda')
bf = dict(dtype=torch.bfloat16, device='cuda')
n_new, ln = torch.ones(3, **i32), torch.zeros(3, **i32)
table = torch.full((3, 4), -1, **i32)
free, nf = torch.arange(9, **i32), torch.tensor([9], **i32)
qkv, w = torch.randn(3, 8 * 64, device='cuda').bfloat16(), torch.ones(64, **bf)
pages = torch.zeros(9, 2, 2, 16, 64, **bf)
p8 = torch.zeros(9, 2, 2, 16, 64, device='cuda').to(torch.float8_e4m3fn)
sc, inv = torch.ones(2, 2, device='cuda'), torch.ones(32, device='cuda')
logits = torch.randn(3, 999, device='cuda')
torch.cuda.synchronize()

def step():
    p = ops.paged_plan(n_new, ln, table, free, nf, 16, 3)
    out = []
    for pg, s in ((pages, None), (p8, sc)):
        q = ops.paged_append(qkv, pg, p.slot, p.pos, 4, w, w, 1e-6, inv,
                             kv_scale=s)
        out.append(ops.paged_attention(q, pg, table, p.pos, req=p.req,
                                       kv_scale=s))
    return out + [ops.process_logits(logits), p.slot]

g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    a = step()
g.replay()
b = step()
torch.cuda.synchronize()
assert all(torch.equal(x, y) for x, y in zip(a, b))
print('same')
""" % os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


def test_attention_no_rows_and_grid_limit():
    """No rows; more rows than a grid's second dimension takes."""
    lens = [20, 33]
    host, dev = dev_cache(lens, 1, 64, 16, BF, seed=13)
    pages, sc, table = dev
    q = queries(0, 2, 64)
    assert ops.paged_attention(q.cuda(), pages, table, torch.empty(
        0, dtype=torch.int32, device="cuda")).shape == (0, 2, 64)
    T = 70001
    few = queries(2, 2, 64)
    req = torch.arange(T, dtype=torch.int32).cuda() % 2
    pos = torch.where(req == 0, 19, 32).to(torch.int32)
    out = ops.paged_attention(few.cuda()[req.long()].contiguous(), pages,
                              table, pos, req=req)
    want = run_attention(few, dev, None, [19, 32])[0].cuda()
    assert torch.equal(out, want[req.long()])


# ---------------------------------------------------------------- append --

def append_case(T, nq, nkv, hd, page, dtype, pos, seed=0, std=2.0):
    g = torch.Generator().manual_seed(seed)
    n_pages = T // page + 4
    pages = (torch.randn(n_pages, 2, nkv, page, hd, generator=g)).to(dtype)
    sc = None if dtype == BF else torch.rand(2, nkv, generator=g) * .02 + .01
    slot = torch.randperm(n_pages * page, generator=g)[:T].to(torch.int32)
    qkv = (torch.randn(T, (nq + 2 * nkv) * hd, generator=g) * std).to(BF)
    qn, kn = ((1 + .2 * torch.randn(hd, generator=g)).to(BF) for _ in "qk")
    inv = (1e6 ** (-torch.arange(hd // 2, dtype=torch.float64) / (hd // 2))
           ).float()
    return dict(qkv=qkv, pages=pages, sc=sc, slot=slot,
                pos=torch.tensor(pos, dtype=torch.int32), qn=qn, kn=kn,
                inv=inv)


def run_append(c, nq, **kw):
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    pages = c["pages"].cuda()
    q = ops.paged_append(
        c["qkv"].cuda() if "dev_qkv" not in c else c["dev_qkv"], pages,
        c["slot"].cuda(), c["pos"].cuda(), nq, c["qn"].cuda(), c["kn"].cuda(),
        EPS, c["inv"].cuda(),
        kv_scale=None if c["sc"] is None else c["sc"].cuda(), status=st, **kw)
    return q.cpu(), pages.cpu(), int(st.item())


def check_append(c, nq, nkv, hd, page):
    """q and keys: the 64-bit value rounded once (bf16 2^-8 relative, e4m3
    2^-4 or half a subnormal step 2^-10), and 2^-18 of the rotated pair's
    length for the fp32 arithmetic before it (norm, sine and cosine, two
    products: under 32 steps of 2^-24).  Values: copied, or rounded once."""
    q, pages, st = run_append(c, nq)
    assert st == 0
    T = c["qkv"].shape[0]
    x = c["qkv"].double().reshape(T, nq + 2 * nkv, hd)
    y = torch.cat([P.rope(x[:, :nq], c["qn"], c["pos"], c["inv"], EPS),
                   P.rope(x[:, nq:nq + nkv], c["kn"], c["pos"], c["inv"], EPS),
                   x[:, nq + nkv:]], 1)
    pair = (y[..., :hd // 2] ** 2 + y[..., hd // 2:] ** 2).sqrt().repeat(1, 1, 2)
    slack = 2.0 ** -18 * pair
    on = (c["slot"] >= 0) & (c["pos"] >= 0)
    err = (q.double() - y[:, :nq]).abs()
    assert (err <= 2.0 ** -8 * y[:, :nq].abs() + slack[:, :nq])[on].all()
    assert (q[~on] == 0).all()
    want = c["pages"].float().clone()
    to = c["slot"][on].long()
    got = pages.float()[to // page, :, :, to % page]     # [T, 2, nkv, hd]
    kv = torch.stack([y[:, nq:nq + nkv], y[:, nq + nkv:]], 1)[on]
    sl = torch.stack([slack[:, nq:nq + nkv], 0 * slack[:, nq + nkv:]], 1)[on]
    if c["sc"] is None:
        tol = 2.0 ** -8 * kv.abs() + sl
        assert torch.equal(got[:, 1].double(), kv[:, 1])
    else:
        s = c["sc"].double()[None, :, :, None]
        kv, sl = (kv / s).clamp(-448, 448), sl / s
        # the quotient's own rounding, 2^-23, stands before the e4m3 one
        tol = (2.0 ** -4 * kv.abs()).clamp(min=2.0 ** -10) + \
            2 * sl + 2.0 ** -23 * kv.abs()
    assert ((got.double() - kv).abs() <= tol).all()
    # every other place of the pages is as it was, bit for bit
    want[to // page, :, :, to % page] = got
    assert torch.equal(pages.float(), want)
    return q, pages


@pytest.mark.parametrize("dtype", [BF, E4])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nq,nkv", HEADS)
def test_append(nq, nkv, hd, dtype):
    pos = [0, 1, 17, 131071, 5, 1 << 20, 2 ** 31 - 1]
    c = append_case(len(pos), nq, nkv, hd, 16, dtype, pos, seed=nq)
    check_append(c, nq, nkv, hd, 16)


@pytest.mark.parametrize("T", [1, 2, 333, 5000])
def test_append_rows(T):
    pos = [(i * 7919) % 100000 for i in range(T)]
    c = append_case(T, 16, 2, 128, 64, E4, pos, seed=T)
    check_append(c, 16, 2, 128, 64)


def test_append_padding_and_bad_slots():
    """Rows without a slot or position: zero queries, no page touched; a slot
    out of range sets the status and is not written."""
    c = append_case(6, 8, 2, 128, 16, BF, [3, -1, 5, 9, -1, 7], seed=2)
    c["slot"][3] = -1
    check_append(c, 8, 2, 128, 16)
    c["slot"][5] = c["pages"].shape[0] * 16
    q, pages, st = run_append(c, 8)
    assert st == L.SLX_ERR_OUT_OF_RANGE and (q[5] == 0).all()
    ok = dict(c, slot=c["slot"].clone())
    ok["slot"][5] = -1
    q2, pages2, st = run_append(ok, 8)
    assert st == 0 and torch.equal(q, q2) and torch.equal(pages, pages2)


def test_append_saturates_and_zero_rows():
    """E4m3 values beyond 448 scales saturate, all-zero heads stay zero, NaN
    stays NaN."""
    c = append_case(4, 2, 1, 64, 16, E4, [1, 2, 3, 4], seed=3)
    c["qkv"][0] = 0
    c["qkv"][1, 3 * 64:] = 3e38
    c["qkv"][2, 3 * 64:] = -1e30
    c["qkv"][3, 3 * 64 + 5] = float("nan")
    q, pages, st = run_append(c, 2)
    at = [(int(s) // 16, int(s) % 16) for s in c["slot"]]
    f = pages.float()
    assert st == 0 and (q[0] == 0).all()
    assert (f[at[0][0], :, 0, at[0][1]] == 0).all()
    assert (f[at[1][0], 1, 0, at[1][1]] == 448).all()
    assert (f[at[2][0], 1, 0, at[2][1]] == -448).all()
    v = f[at[3][0], 1, 0, at[3][1]]
    assert torch.isnan(v[5]) and torch.isfinite(v[:5]).all()


def test_append_strided_rows():
    c = append_case(5, 8, 2, 64, 16, BF, [4, 5, 6, 7, 8], seed=4)
    q, pages, _ = run_append(c, 8)
    wide = torch.zeros(5, 12 * 64 + 72, dtype=BF, device="cuda")
    wide[:, :12 * 64] = c["qkv"].cuda()
    q2, pages2, st = run_append(dict(c, dev_qkv=wide[:, :12 * 64]), 8)
    assert st == 0 and torch.equal(q, q2) and torch.equal(pages, pages2)


# ------------------------------------------------------------------ plan --

class DevicePlan:
    """Plan state on the device beside its restatement on the host."""

    def __init__(self, n_req, page, n_pages, max_pages, seed=0):
        self.page, self.ref = page, P.Plan(page, n_pages, max_pages)
        g = np.random.default_rng(seed)
        self.lengths = [0] * n_req
        self.table = [[-1] * max_pages for _ in range(n_req)]
        self.free = [int(i) for i in g.permutation(n_pages)]
        self.n_free = n_pages
        i32 = dict(dtype=torch.int32, device="cuda")
        self.d_len = torch.tensor(self.lengths, **i32)
        self.d_table = torch.tensor(self.table, **i32)
        self.d_free = torch.tensor(self.free, **i32)
        self.d_n = torch.tensor([self.n_free], **i32)
        self.status = torch.zeros(1, **i32)

    def step(self, n_new, n_rows, alias=True):
        code, rows, start, self.lengths, self.table, self.free, self.n_free = \
            self.ref.step(n_new, self.lengths, self.table, self.free,
                          self.n_free, n_rows)
        p = ops.paged_plan(
            torch.tensor(n_new, dtype=torch.int32).cuda(), self.d_len,
            self.d_table, self.d_free, self.d_n, self.page, n_rows,
            lengths_out=self.d_len if alias else None,
            n_free_out=self.d_n if alias else None, status=self.status)
        self.d_len, self.d_n = p.lengths, p.n_free
        assert int(self.status.item()) == code
        self.status.zero_()
        got = list(zip(p.req.tolist(), p.pos.tolist(), p.slot.tolist()))
        assert got == rows
        assert p.start.tolist() == start
        self.check()
        return code, p

    def check(self):
        assert self.d_len.tolist() == self.lengths
        assert self.d_table.tolist() == self.table
        assert self.d_free.tolist() == self.free
        assert self.d_n.tolist() == [self.n_free]


@pytest.mark.parametrize("n_req,page,alias", [(1, 16, True), (7, 16, False),
                                              (65, 32, True), (513, 16, True),
                                              (8192, 64, True)])
def test_plan_runs(n_req, page, alias):
    """Random steps: prompts in chunks, single tokens, idle and finished
    requests, compared after every step."""
    max_pages = 9
    d = DevicePlan(n_req, page, n_req * max_pages // 2 + 5, max_pages)
    g = np.random.default_rng(n_req)
    for step in range(12):
        n_new = []
        for ln in d.lengths:
            room = max_pages * page - ln
            n_new.append(int(g.choice([0, min(1, room), min(1, room),
                                       int(g.integers(0, min(room, 40) + 1)),
                                       -1])))
        d.step(n_new, sum(max(n, 0) for n in n_new) + int(g.integers(0, 70)),
               alias)


def test_plan_large_chunks():
    """Rows and pages that take several turns of the launch."""
    d = DevicePlan(40, 16, 20000, 600, seed=3)
    d.step([9000, 0, 1, 4097] + [16 * i for i in range(36)], 30000)
    d.step([-1, 5, -1, 1] + [3] * 36, 200)


def test_plan_refusals_change_nothing():
    d = DevicePlan(3, 16, 5, 4)
    assert d.step([20, 10, 0], 64)[0] == 0
    assert d.step([10, 10, 10], 29)[0] == L.SLX_ERR_PAGES     # rows
    assert d.step([1, 40, 16], 64)[0] == L.SLX_ERR_PAGES      # pages
    assert d.step([1, 55, 0], 64)[0] == L.SLX_ERR_OUT_OF_RANGE  # over the table
    assert d.step([-2, 0, 0], 64)[0] == L.SLX_ERR_OUT_OF_RANGE
    assert d.step([2 ** 31 - 1, 0, 0], 64)[0] == L.SLX_ERR_OUT_OF_RANGE
    assert d.step([2 ** 31 - 1] * 3, 64)[0] == L.SLX_ERR_OUT_OF_RANGE
    # the pages of a finished request serve the same step
    assert d.step([-1, 22, 32], 64)[0] == 0
    d.d_n.fill_(6)
    d.n_free = 6
    assert d.step([0, 0, 0], 64)[0] == L.SLX_ERR_OUT_OF_RANGE
    d.d_n.fill_(0)
    d.n_free = 0
    d.d_len[1] = -5
    d.lengths[1] = -5
    assert d.step([0, 0, 0], 64)[0] == L.SLX_ERR_OUT_OF_RANGE


def test_plan_bad_page_in_table():
    """A page out of range in the table or on the stack: status, and the row
    gets no slot."""
    d = DevicePlan(2, 16, 4, 2)
    d.step([3, 3], 8)
    d.d_table[0, 0] = 99
    p = ops.paged_plan(torch.tensor([1, 1], dtype=torch.int32).cuda(), d.d_len,
                       d.d_table, d.d_free, d.d_n, 16, 4, status=d.status)
    assert int(d.status.item()) == L.SLX_ERR_OUT_OF_RANGE
    assert p.slot.tolist()[0] == -1 and p.slot.tolist()[1] >= 0


def test_plan_no_rows_and_repeats():
    d = DevicePlan(2, 16, 8, 4)
    d.step([0, 0], 0)
    d.step([17, 1], 20)
    args = (torch.tensor([30, -1], dtype=torch.int32).cuda(), d.d_len,
            d.d_table, d.d_free, d.d_n, 16, 40)
    a = [t.clone() for t in ops.paged_plan(*args)]
    table, free = d.d_table.clone(), d.d_free.clone()
    b = ops.paged_plan(*args)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert torch.equal(table, d.d_table) and torch.equal(free, d.d_free)


# -------------------------------------------------------------- together --

@pytest.mark.parametrize("dtype", [BF, E4])
def test_steps_together(dtype):
    """Plan, append and attention of several steps as a server runs them:
    chunks of prompts, single tokens, a finished request whose pages another
    one takes over; each step's attention against the 64-bit attention over
    everything the request was given."""
    nq, nkv, hd, page = 8, 2, 64, 16
    d = DevicePlan(4, page, 12, 6)
    pages = torch.full((12, 2, nkv, page, hd), float("nan")).to(dtype).cuda()
    sc = None if dtype == BF else torch.full((2, nkv), 0.02, device="cuda")
    g = torch.Generator().manual_seed(1)
    qn, kn = ((1 + .2 * torch.randn(hd, generator=g)).to(BF).cuda() for _ in "qk")
    inv = (1e6 ** (-torch.arange(hd // 2, dtype=torch.float64) / (hd // 2))
           ).float().cuda()
    for n_new in ([20, 0, 3, 0], [1, 33, 1, 0], [-1, 1, 1, 5], [16, 1, 1, 1],
                  [1, 1, -1, 60], [1, 1, 1, 1]):
        code, p = d.step(n_new, 80)
        assert code == 0
        qkv = (torch.randn(80, (nq + 2 * nkv) * hd, generator=g) * 2).to(BF)
        q = ops.paged_append(qkv.cuda(), pages, p.slot, p.pos, nq, qn, kn, EPS,
                             inv, kv_scale=sc)
        out = ops.paged_attention(q, pages, d.d_table, p.pos, req=p.req,
                                  kv_scale=sc).cpu()
        want, bound = P.attention(
            q.cpu(), pages.cpu(), None if sc is None else sc.cpu(),
            d.d_table.cpu(), p.req.tolist(), p.pos.tolist(), page, hd ** -0.5)
        assert torch.isfinite(out).all()
        assert ((out.double() - want).abs() <= bound).all()
        n = sum(max(k, 0) for k in n_new)
        # the keys that were appended are the ones the slots name
        k = P.rope(qkv.reshape(80, -1, hd)[:n, nq:nq + nkv], kn.cpu(),
                   p.pos.cpu()[:n], inv.cpu(), EPS)
        s = p.slot.cpu()[:n].long()
        got = pages.float().cpu()[s // page, 0, :, s % page].double()
        if sc is not None:
            got = got * 0.02
        assert ((got - k).abs() <= 2.0 ** (-8 if dtype == BF else -4)
                * k.abs() + 1e-3).all()
    ops.check_status(torch.device("cuda", torch.cuda.current_device()))


@pytest.mark.parametrize("seed", [0, 1])
def test_attention_chunks_as_single_rows(seed):
    """Random chunks against the same rows as requests of one row each (the
    other kernel), and the same bits twice."""
    g = np.random.default_rng(seed)
    for _ in range(25):
        G, nkv = int(g.integers(1, 17)), int(g.choice([1, 2, 3, 8]))
        hd, page = int(g.choice([64, 128])), int(g.choice([16, 32, 64, 256]))
        dtype = BF if g.random() < 0.5 else E4
        lens = [int(n) for n in g.integers(1, int(g.choice([80, 700, 2500])),
                                           int(g.integers(1, 6)))]
        host, dev = dev_cache(lens, nkv, hd, page, dtype, seed=seed)
        req, pos = [], []
        while len(req) < g.choice([60, 200, 600]):
            i = int(g.integers(0, len(lens)))
            n = min(lens[i], int(g.choice([1, 5, 20, 64, 128, 300])))
            at = int(g.integers(0, lens[i] - n + 1))
            req += [i] * n + [-1] * 2
            pos += list(range(at, at + n)) + [-1] * 2
        q = queries(len(req), G * nkv, hd)
        out, st = run_attention(q, dev, req, pos)
        assert st == 0 and torch.equal(out, run_attention(q, dev, req, pos)[0])
        rows = torch.tensor(req).clamp(min=0)
        one, st = run_attention(q, (dev[0], dev[1],
                                    dev[2][rows.cuda()].contiguous()), None,
                                pos)
        # both within their bound of the formula: half a bf16 step each, and
        # what the weights' two parts and fp32 sums leave of the row's size
        lim = 2.0 ** -7 * one.abs() + 1e-3 * one.abs().amax(-1, keepdim=True)
        assert st == 0 and ((out - one).abs() <= lim + 1e-4).all()


# -------------------------------------------------- small weights, e4m3 --

def sink_cache(n, n_kv, hd, dtype):
    """One request whose first key is far above the others, which are zero,
    and has a value of zero: all of the result is what the others weigh."""
    scale = torch.tensor([[1.0] * n_kv, [0.02] * n_kv])
    pages, sc, table = P.make_cache([n], n_kv, hd, 64, dtype, seed=41,
                                    scale=scale)
    x = pages.float()
    x[:, 0] = torch.where(torch.isnan(x[:, 0]), x[:, 0], 0.0)
    at = int(table[0, 0])
    x[at, 0, :, 0], x[at, 1, :, 0] = 8.0, 0.0
    pages = x.to(dtype)
    return (pages, sc, table), (pages.cuda(), None if sc is None else sc.cuda(),
                                table.cuda())


@pytest.mark.parametrize("dtype", [BF, E4])
@pytest.mark.parametrize("bits", [16.6, 24.6, 27.3, 30.4])
@pytest.mark.parametrize("nq,nkv,hd,n,rows", [
    (16, 2, 128, 400, 1), (16, 2, 128, 20000, 1), (24, 4, 64, 3000, 3),
    (16, 2, 128, 4000, 80),                 # the kernel for chunks, in parts
    (8, 8, 64, 2600, 2432)])                # and in one
def test_attention_small_weights(nq, nkv, hd, n, rows, bits, dtype):
    """Thousands of keys whose weights are 2^-bits of the first one's.

    The bound is the formula's, and for e4m3 pages half of the weights' fp16
    step, 2^-24 of 2^15, for every key: 2^-40 sum |v| (the greatest weight is
    at most 1)."""
    host, dev = sink_cache(n, nkv, hd, dtype)
    q = torch.ones(rows, nq, hd, dtype=BF)
    scale = bits * float(np.log(2.0)) / (8 * hd)
    pos = list(range(n - rows, n))
    out, st = run_attention(q, dev, [0] * rows, pos, scale)
    assert st == 0 and torch.isfinite(out).all()
    some = sorted({0, rows - 1, *range(0, rows, max(1, rows // 40))})
    want, bound = P.attention(q[some], host[0], host[1], host[2],
                              [0] * len(some), [pos[r] for r in some], 64,
                              scale)
    if dtype == E4:
        V = P.dense(host[0], host[1], host[2], 0, n, 64)[1]     # [kv, n, hd]
        step = 2.0 ** -40 * V.abs().sum(1)
        bound = bound + step.repeat_interleave(nq // nkv, 0)
    err = (out[some].double() - want).abs()
    assert (err <= bound).all(), float((err / bound).max())


# ------------------------------------- chunks beside single tokens --

def graph_us(call, n=10):
    """Time of one of n calls in a graph, the least of some replays."""
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for _ in range(n):
            call()
    a, b = (torch.cuda.Event(enable_timing=True) for _ in "ab")
    best = float("inf")
    for _ in range(10):
        a.record()
        g.replay()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b) * 1000 / n)
    return best


def attention_us(lens, rows, nq, nkv, hd, dtype, idle=0):
    """Of the last rows[i] tokens of every request, then `idle` padding rows
    (the pages' content is of no matter here)."""
    need = [P.pages_for(n, 64) for n in lens]
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = torch.arange(at, at + n)
        at += n
    pages = torch.zeros(at, 2, nkv, 64, hd, device="cuda").to(dtype)
    sc = torch.ones(2, nkv, device="cuda") if dtype == E4 else None
    req, pos = chunk_rows(lens, [n - r for n, r in zip(lens, rows)])
    req, pos = (torch.tensor(v + [-1] * idle, dtype=torch.int32).cuda()
                for v in (req, pos))
    q = torch.ones(len(req), nq, hd, dtype=BF, device="cuda")
    table = table.cuda()
    return graph_us(lambda: ops.paged_attention(q, pages, table, pos, req=req,
                                                kv_scale=sc))


@pytest.mark.parametrize("dtype", [BF, E4])
def test_mixed_rows_cost_their_parts(dtype):
    """A prompt chunk beside decoding requests, and a call that is padding for
    the most part, against the parts by themselves (the least of ten replays):
    the chunk's blocks hold 48 of 128 columns at least, so it may take 128 / 48
    of its time; 25 us for up to four launches more."""
    heads = (24, 4, 128, dtype)
    decode = attention_us([4000] * 63, [1] * 63, *heads)
    chunk = attention_us([4000], [512], *heads)
    mixed = attention_us([4000] * 64, [1] * 30 + [512] + [1] * 33, *heads)
    assert mixed <= decode + 128 / 48 * chunk + 25, (mixed, decode, chunk)
    heads = (16, 2, 128, dtype)
    decode = attention_us([30000] * 7, [1] * 7, *heads)
    chunk = attention_us([2000], [64], *heads)
    mixed = attention_us([2000] + [30000] * 7, [64] + [1] * 7, *heads)
    assert mixed <= decode + 128 / 48 * chunk + 25, (mixed, decode, chunk)
    few = attention_us([30000] * 3, [1] * 3, *heads)
    padded = attention_us([30000] * 3 + [1], [1] * 3 + [0], *heads, idle=61)
    assert padded <= few + 25, (padded, few)


@pytest.mark.parametrize("dtype", [BF, E4])
@pytest.mark.parametrize("nq,nkv,hd", [(24, 4, 128), (8, 8, 64), (32, 2, 64),
                                       (16, 2, 128), (13, 1, 128), (2, 1, 64)])
def test_attention_runs_of_every_length(nq, nkv, hd, dtype):
    """Chunks of 1 to 70 rows beside each other, in an order that puts their
    ends at any place of the blocks, idle rows between and inside them."""
    g = np.random.default_rng(nq + hd)
    each = [int(n) for n in g.permutation([*range(1, 40), 47, 48, 49, 63, 64,
                                           65, 70] + [1] * 12)]
    lens = [n + int(g.integers(0, 150)) for n in each]
    req, pos = [], []
    for i, (n, r) in enumerate(zip(lens, each)):
        req += [i] * r + [-1] * int(g.integers(0, 2))
        pos += list(range(n - r, n)) + [-1] * (len(req) - len(pos) - r)
    for r in g.integers(0, len(req), 5):
        pos[r] = -1
    host, dev = dev_cache(lens, nkv, hd, 16, dtype, seed=nq)
    out = check_attention(queries(len(req), nq, hd), host, dev, req, pos)
    assert all((out[r] == 0).all() for r in range(len(req)) if pos[r] < 0)


def graph_launches(call):
    """Kernels of one captured call."""
    g = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(g):
        call()
    n = ctypes.c_size_t()
    assert ctypes.CDLL("libcuda.so.1").cuGraphGetNodes(
        ctypes.c_void_p(g.raw_cuda_graph()), None, ctypes.byref(n)) == 0
    return n.value


def test_launches_are_counted():
    """LAUNCHES moves on by the kernels that a call launches: none without
    rows; one to four for attention."""
    pages = torch.zeros(200, 2, 2, 16, 64, dtype=BF, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    w, inv = torch.ones(64, dtype=BF, device="cuda"), torch.ones(32, device="cuda")
    table = torch.arange(200, **i32)

    def attention(T, n_req):
        q = torch.zeros(T, 16, 64, dtype=BF, device="cuda")
        pos = torch.arange(T, **i32) % (T // n_req or 1)
        req = torch.arange(T, **i32) // (T // n_req or 1)
        t = table.view(n_req, -1)
        return lambda: ops.paged_attention(q, pages, t, pos, req=req)

    def append(T):
        qkv = torch.zeros(T, 20 * 64, dtype=BF, device="cuda")
        at = torch.arange(T, **i32)
        return lambda: ops.paged_append(qkv, pages, at, at, 16, w, w, EPS, inv)

    def logits(T):
        x = torch.zeros(T, 99, device="cuda")
        return lambda: ops.process_logits(x)

    def plan(n_rows):
        a = [torch.zeros(4, **i32), torch.zeros(4, **i32), table.view(4, -1),
             table.clone(), torch.tensor([7], **i32)]
        return lambda: ops.paged_plan(*a, 16, n_rows)

    seen = set()
    for name, call, most in (
            ("no rows", attention(0, 1), 0), ("single", attention(4, 4), 2),
            ("a chunk", attention(300, 1), 2),
            ("a chunk in one part", attention(3200, 1), 2),
            ("chunks", attention(300, 4), 4), ("append", append(5), 1),
            ("no append", append(0), 0), ("logits", logits(3), 1),
            ("no logits", logits(0), 0), ("plan", plan(4), 1),
            ("large plan", plan(5000), 1)):
        call()
        before = L.LAUNCHES[0]
        call()
        n = L.LAUNCHES[0] - before
        assert n == graph_launches(call) <= most, name
        seen.add(n)
    assert seen >= {0, 1, 2, 4}


def as_single_rows(q, dev, req, pos):
    """The same rows as requests of one row each (the kernel for them)."""
    rows = torch.tensor(req).clamp(0, dev[2].shape[0] - 1).cuda()
    return run_attention(q, (dev[0], dev[1], dev[2][rows].contiguous()), None,
                         pos)[0]


def close_rows(out, one):
    """Both within their bound of the formula: half a bf16 step each, and what
    the weights' two parts and fp32 sums leave of the row's size."""
    lim = 2.0 ** -7 * one.abs() + 1e-3 * one.abs().amax(-1, keepdim=True)
    return ((out.float() - one.float()).abs() <= lim + 1e-4).all()


@pytest.mark.parametrize("dtype", [BF, E4])
def test_attention_more_blocks_than_flags(dtype):
    """Thousands of short requests, some with one row: more blocks of rows than
    the two kernels have flags for."""
    g = np.random.default_rng(5)
    each = [int(n) for n in g.choice([1, 3, 5, 8], 1300)]
    lens = [n + int(g.integers(0, 40)) for n in each]
    host, dev = dev_cache(lens, 1, 64, 16, dtype, seed=31)
    req, pos = chunk_rows(lens, [n - r for n, r in zip(lens, each)])
    rows = len(req) // len(lens)
    assert rows * 16 >= 48 and -(-len(req) // min(rows, 8)) > 1024
    q = queries(len(req), 16, 64)
    out, st = run_attention(q, dev, req, pos)
    assert st == 0 and close_rows(out, as_single_rows(q, dev, req, pos))


@pytest.mark.parametrize("pdl", [False, True])
@pytest.mark.parametrize("dtype", [BF, E4])
def test_attention_mixed_calls_again(dtype, pdl):
    """Calls of chunks beside single tokens that share a workspace, one behind
    the other, eagerly and in a graph: the same bits every time, with and
    without dependent launches."""
    lens = [900, 40, 3000, 700, 1, 2000]
    each = [120, 1, 64, 1, 1, 2]
    host, dev = dev_cache(lens, 2, 128, 16, dtype, seed=32)
    pages, sc, table = dev
    plans = []
    for back in (0, 1):                     # two calls of other rows
        req, pos = chunk_rows(lens, [n - r for n, r in zip(lens, each)])
        pos = [p if i % 7 or not back else -1 for i, p in enumerate(pos)]
        q = queries(len(req), 16, 128, seed=back)
        want = check_attention(q, host, dev, req, pos)
        plans.append((q.cuda(), torch.tensor(req, dtype=torch.int32).cuda(),
                      torch.tensor(pos, dtype=torch.int32).cuda(),
                      want.cuda()))
    ws = ops.paged_workspace(len(req), 16, 2, 128, "cuda")

    def calls():
        return [ops.paged_attention(q, pages, table, p, req=r, kv_scale=sc,
                                    workspace=ws) for q, r, p, _ in plans * 4]

    prev = L.set_pdl(pdl)
    try:
        eager = calls()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            captured = calls()
        for _ in range(5):
            g.replay()
        torch.cuda.synchronize()
    finally:
        L.set_pdl(prev)
    for outs in (eager, captured):
        assert all(torch.equal(o, p[3]) for o, p in zip(outs, plans * 4))
    ops.check_status(torch.device("cuda", torch.cuda.current_device()))


@pytest.mark.parametrize("dtype", [BF, E4])
def test_attention_of_a_long_document(dtype):
    """131071 keys, one row, held to what the kernel's sums can lose: a warp of
    its 4 x 444 adds five or six units of 16 or 32 keys, four warps and some 222
    CTAs' parts are joined, so fewer than 512 additions stand behind a sum (the
    bound for any order has one for every key)."""
    n, scale = 131071, 128 ** -0.5
    host, dev = dev_cache([n], 2, 128, 64, dtype, seed=51, tail="zero")
    q = queries(1, 16, 128)
    out, st = run_attention(q, dev, None, [n - 1])
    want, any_order = P.attention(q, *host, [0], [n - 1], 64, scale)
    K, V = P.dense(*host, 0, n, 64)
    p = torch.softmax(torch.einsum("kgd,kld->kgl", q[0].double().reshape(
        2, 8, 128), K) * scale, -1)
    A = torch.einsum("kgl,kld->kgd", p, V.abs()).reshape(1, 16, 128)
    bound = any_order - 2 * (n - 512) * 2.0 ** -23 * A
    err = (out.double() - want).abs()
    assert st == 0 and (bound > 0).all()
    assert (err <= bound).all(), float((err / bound).max())
