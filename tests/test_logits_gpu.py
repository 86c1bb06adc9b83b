"""Logit processing and the greedy pick against a plain 64-bit restatement
(tests/paged_cases.py)."""

import pytest
import torch

from streamlx_b200 import _lib as L
from streamlx_b200 import ops
from tests import paged_cases as P

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
INF = float("inf")


def case(T, V, dtype, hist, n_bias, masked, seed=0):
    g = torch.Generator().manual_seed(seed)
    c = dict(x=(torch.randn(T, V, generator=g) * 2.5).to(dtype), history=None,
             n_prompt=None, n_history=None, rep=None, freq=None, pres=None,
             bias=None, mask=None)
    if hist:
        # few distinct ids, so that many repeat; some outside the vocabulary
        ids = torch.randint(0, max(2, min(V, hist // 2)), (T, hist), generator=g)
        out = torch.rand(T, hist, generator=g) < 0.05
        ids = torch.where(out, torch.tensor([-1, V, 2 ** 31 - 1, -2 ** 31])[
            torch.randint(0, 4, (T, hist), generator=g)], ids)
        c["history"] = ids.to(torch.int32)
        c["n_history"] = torch.randint(0, hist + 1, (T,), generator=g).to(torch.int32)
        c["n_prompt"] = (c["n_history"] * torch.rand(T, generator=g)).to(torch.int32)
        c["rep"] = 0.8 + 0.6 * torch.rand(T, generator=g)
        c["freq"] = torch.rand(T, generator=g) - 0.2
        c["pres"] = torch.rand(T, generator=g) - 0.2
    if n_bias:
        n = torch.randint(0, n_bias + 1, (T,), generator=g)
        start = torch.zeros(T + 1, dtype=torch.int32)
        start[1:] = n.cumsum(0)
        total = max(1, int(start[-1]))
        # ids twice, and ids outside the vocabulary
        ids = torch.randint(-2, min(V, n_bias) + 2, (total,), generator=g)
        c["bias"] = (ids.to(torch.int32), torch.randn(total, generator=g) * 3,
                     start)
    if masked:
        words = (V + 31) // 32
        m = torch.randint(-2 ** 31, 2 ** 31, (T, words + 1), generator=g)
        m &= torch.randint(-2 ** 31, 2 ** 31, (T, words + 1), generator=g)
        c["mask"] = m.to(torch.int32)
    return c


def run(c, out=None, **kw):
    d = {k: tuple(t.cuda() for t in v) if isinstance(v, tuple) else
         None if v is None else v.cuda() for k, v in c.items()}
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    if out == "inplace":
        out = d["x"]
    elif out == "new":
        out = torch.empty_like(d["x"])
    pick = ops.process_logits(
        d["x"], d["history"], d["n_prompt"], d["n_history"],
        repetition=d["rep"], frequency=d["freq"], presence=d["pres"],
        bias=d["bias"], mask=d["mask"], out=out, status=st, **kw)
    torch.cuda.synchronize()
    return (None if pick is None else pick.tolist(),
            None if out is None else out.cpu(), int(st.item()))


def check(c, out="new"):
    want, picks = P.logits(c["x"], c["history"], c["n_prompt"],
                           c["n_history"], c["rep"], c["freq"], c["pres"],
                           c["bias"], c["mask"])
    got, y, st = run(c, out)
    assert st == 0
    assert got == picks
    if y is not None:
        # one rounding of a value computed in 64 bits; the fp64 value itself
        # passes through fp32 on the way to bf16 (2^-24)
        half = torch.finfo(c["x"].dtype).eps / 2
        fin = torch.isfinite(want)
        assert torch.equal(torch.isfinite(y), fin)
        assert torch.equal(y[~fin].double(), want[~fin])
        err = (y.double() - want)[fin].abs()
        assert (err <= (half + 2.0 ** -23) * want[fin].abs()).all()
    return got, y


@pytest.mark.parametrize("out", [None, "new", "inplace"])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,V", [(1, 1), (3, 31), (2, 33), (5, 1000),
                                 (2, 4099), (3, 151936)])
def test_rules(T, V, dtype, out):
    check(case(T, V, dtype, 40, 20, True, seed=V), out)


@pytest.mark.parametrize("hist,n_bias,masked", [
    (0, 0, False), (50, 0, False), (0, 30, False), (0, 0, True),
    (3000, 0, True), (1, 1, False)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_each_rule(hist, n_bias, masked, dtype):
    check(case(4, 2000, dtype, hist, n_bias, masked, seed=hist + n_bias))


@pytest.mark.parametrize("V", [196608, 196609, 300001])
def test_vocabulary_beyond_one_pass(V):
    c = case(2, V, BF, 200, 10, False, seed=1)
    c["history"][:, ::3] = V - 1 - c["history"][:, ::3].clamp(0, 1000)
    check(c)
    c["x"][1, V - 1] = 99.0
    assert check(c, None)[0][1] == V - 1 or int(c["n_history"][1]) > 0


def test_rows_of_a_batch_are_their_own():
    """Each row as if it were alone."""
    c = case(7, 5000, BF, 60, 9, True, seed=2)
    got, y, _ = run(c, "new")
    for b in range(7):
        one = {k: None if v is None else v[b:b + 1] for k, v in c.items()
               if k != "bias"}
        ids, vals, start = c["bias"]
        lo, hi = int(start[b]), int(start[b + 1])
        one["bias"] = (ids[lo:hi].contiguous(), vals[lo:hi].contiguous(),
                       torch.tensor([0, hi - lo], dtype=torch.int32))
        p, z, _ = run(one, "new")
        assert p == got[b:b + 1] and torch.equal(z[0], y[b])


def test_ties_take_the_lowest_id():
    x = torch.zeros(3, 40000, dtype=BF)
    x[0, [7, 39999]] = 1.0
    x[1, [39998, 20000, 25000]] = 1.0
    mask = torch.full((3, 1250), -1, dtype=torch.int32)
    mask[2, 0] = 0
    c = dict(case(3, 40000, BF, 0, 0, False), x=x, mask=mask)
    assert check(c, None)[0] == [7, 20000, 32]


def test_neighbouring_values():
    """Two penalised ids whose fp32 quotients are equal, and one 64-bit value
    above the other; the pick goes by the 64-bit one."""
    x = torch.full((1, 64), -5.0, dtype=BF)
    x[0, 10], x[0, 40] = 5.0, 5.5          # 5.5 / fp32(1.1) < 5 in 64 bits
    c = dict(case(1, 64, BF, 0, 0, False), x=x,
             history=torch.tensor([[40]], dtype=torch.int32),
             n_history=torch.tensor([1], dtype=torch.int32),
             rep=torch.tensor([1.1]))
    got = check(c)[0]
    assert got == [10]
    x[0, 10], x[0, 40] = 5.5, 5.0
    c["history"] = torch.tensor([[10]], dtype=torch.int32)
    assert check(c)[0] == [40]


def test_nothing_allowed_and_only_infinities():
    c = case(4, 300, BF, 0, 0, True, seed=3)
    c["mask"][0] = 0
    c["x"][1] = -INF
    c["x"][2, 17] = INF
    c["mask"][2, 0] |= 1 << 17
    c["x"][3, :200] = INF
    c["mask"][3, :6] = 0
    c["mask"][3, 6] = 0x7fffff00
    c["x"][3, 200] = 3.0
    got, y = check(c)
    assert got[0] == -1 and (y[0] == -INF).all()
    # row 3: the infinities stand in masked places
    assert got[2] == 17 and got[3] >= 200


def test_nan_logits():
    """A NaN is not picked over a number, counts as -inf among others, and
    passes through; one in a masked place becomes -inf."""
    c = case(3, 500, F32, 0, 0, True, seed=4)
    c["x"][0, 100:200] = float("nan")
    c["x"][1] = float("nan")
    got, y, st = run(c, "new")
    want, picks = P.logits(c["x"], None, None, None, None, None, None, None,
                           c["mask"])
    assert st == 0 and got == picks
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    assert torch.equal(y == -INF, want == -INF)


def test_counts_out_of_range():
    """Counts outside their arrays set the status and are clipped."""
    c = case(3, 100, BF, 20, 0, False, seed=5)
    for name, bad in (("n_history", 21), ("n_history", -1),
                      ("n_history", 2 ** 31 - 1), ("n_prompt", -3),
                      ("n_prompt", 21)):
        d = dict(c, n_history=c["n_history"].clone(),
                 n_prompt=c["n_prompt"].clone())
        d[name][1] = bad
        d[name][0], d[name][2] = c[name][0], c[name][2]
        got, y, st = run(d, "new")
        assert st == L.SLX_ERR_OUT_OF_RANGE, name
        n = max(0, min(20, int(d["n_history"][1])))
        d["n_history"][1] = n
        d["n_prompt"][1] = max(0, min(n, int(d["n_prompt"][1])))
        check(d)
    c = case(2, 100, BF, 0, 10, False, seed=6)
    ids, vals, start = c["bias"]
    for bad in ([0, 4, ids.numel() + 1], [-1, 4, 5], [3, 2, 4]):
        c["bias"] = (ids, vals, torch.tensor(bad, dtype=torch.int32))
        assert run(c, "new")[2] == L.SLX_ERR_OUT_OF_RANGE


def test_bias_entries_limit():
    """8191 entries of a row count; one more sets the status."""
    n = 8191
    ids = torch.arange(n).to(torch.int32) % 4000
    vals = torch.linspace(-1, 1, n)
    c = dict(case(1, 6000, F32, 0, 0, False, seed=7),
             bias=(ids, vals, torch.tensor([0, n], dtype=torch.int32)))
    check(c)
    c["bias"] = (torch.cat([ids, ids[:1]]), torch.cat([vals, vals[:1]]),
                 torch.tensor([0, n + 1], dtype=torch.int32))
    assert run(c, "new")[2] == L.SLX_ERR_OUT_OF_RANGE


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [999, 4104])
def test_rows_at_any_alignment(V, dtype):
    """Logits, output and history whose rows start anywhere."""
    c = case(5, V, dtype, 37, 11, True, seed=V)
    base, _, _ = run(c, "new")
    for a, b in ((0, 0), (1, 1), (1, 0), (0, 3), (5, 2)):
        def put(t, off):
            buf = torch.empty(t.numel() + off, dtype=t.dtype, device="cuda")
            v = buf[off:].view(t.shape)
            v.copy_(t)
            return v
        x, h = put(c["x"], a), put(c["history"], a + b)
        out = put(torch.zeros_like(c["x"]), b)
        pick = ops.process_logits(
            x, h, c["n_prompt"].cuda(), c["n_history"].cuda(),
            repetition=c["rep"].cuda(), frequency=c["freq"].cuda(),
            presence=c["pres"].cuda(), bias=tuple(t.cuda() for t in c["bias"]),
            mask=c["mask"].cuda(), out=out)
        want, picks = P.logits(c["x"], c["history"], c["n_prompt"],
                               c["n_history"], c["rep"], c["freq"], c["pres"],
                               c["bias"], c["mask"])
        assert pick.tolist() == picks == base
        fin = torch.isfinite(want)
        y = out.cpu().double()
        assert torch.equal(torch.isfinite(y), fin)
        half = torch.finfo(dtype).eps / 2 + 2.0 ** -23
        assert ((y - want)[fin].abs() <= half * want[fin].abs()).all()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_most_ids_touched(dtype):
    """A history that names most of the vocabulary: more ids than a pass
    lists."""
    V, n = 151936, 131072
    g = torch.Generator().manual_seed(10)
    ids = torch.randperm(V, generator=g)[:n].to(torch.int32)[None]
    x = (torch.randn(1, V, generator=g) * 2.5).to(dtype)
    rep, freq = torch.tensor([1.3]), torch.tensor([0.25])
    c = dict(case(1, V, dtype, 0, 0, False), x=x, history=ids,
             n_prompt=torch.tensor([n // 2], dtype=torch.int32),
             n_history=torch.tensor([n], dtype=torch.int32), rep=rep,
             freq=freq)
    got, y, st = run(c, "new")
    want = x[0].double()
    at = ids[0].long()
    v = want[at]
    want[at] = torch.where(v > 0, v / rep.double(), v * rep.double())
    want[at[n // 2:]] -= freq.double()
    assert st == 0 and got == [int(want.argmax())]
    half = torch.finfo(dtype).eps / 2 + 2.0 ** -23
    assert ((y[0].double() - want).abs() <= half * want.abs()).all()


def test_one_id_all_along():
    """The longest history, every entry the same id."""
    n = 262143
    x = torch.zeros(1, 100, dtype=F32)
    c = dict(case(1, 100, F32, 0, 0, False), x=x,
             history=torch.full((1, n), 7, dtype=torch.int32),
             n_history=torch.tensor([n], dtype=torch.int32),
             freq=torch.tensor([0.5]), pres=torch.tensor([1.0]),
             bias=(torch.tensor([7, 7], dtype=torch.int32),
                   torch.tensor([9.0, 2.5]),
                   torch.tensor([0, 2], dtype=torch.int32)))
    got, y, st = run(c, "new")
    assert st == 0 and got == [0]
    assert float(y[0, 7]) == -0.5 * n - 1.0 + 2.5


def test_without_pick_and_empty():
    c = case(2, 500, BF, 30, 5, True, seed=8)
    _, y, _ = run(c, "new")
    p, z, _ = run(c, "new", pick=False)
    assert p is None and torch.equal(y, z)
    x = torch.empty(0, 500, dtype=BF, device="cuda")
    assert ops.process_logits(x).shape == (0,)


def test_streams_and_graph():
    c = case(5, 151936, BF, 500, 50, True, seed=9)
    got, y, _ = run(c, "new")
    d = {k: tuple(t.cuda() for t in v) if isinstance(v, tuple) else
         None if v is None else v.cuda() for k, v in c.items()}

    def call():
        out = torch.empty_like(d["x"])
        return ops.process_logits(
            d["x"], d["history"], d["n_prompt"], d["n_history"],
            repetition=d["rep"], frequency=d["freq"], presence=d["pres"],
            bias=d["bias"], mask=d["mask"], out=out), out

    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append(call())
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs.append(call())
    g.replay()
    torch.cuda.synchronize()
    for p, o in outs:
        assert p.tolist() == got and torch.equal(o.cpu(), y)
