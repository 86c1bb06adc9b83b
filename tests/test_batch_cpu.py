"""Bookkeeping of the batched decoder that needs no GPU: what it takes, what it
refuses, and what it hands to the kernels' front ends."""

from types import SimpleNamespace

import pytest
import torch

from streamlx_b200 import batch, ops
from streamlx_b200.batch import BatchDecoder, LogitRules

VOCAB = 50


def decoder(**kw):
    """A decoder over a model of which only the sizes are looked at."""
    cfg = SimpleNamespace(has_trunk=True, head_dim=64, heads=4, kv_heads=2,
                          layers=2, vocab=VOCAB)
    layers = [SimpleNamespace(k_norm=torch.ones(64)) for _ in range(2)]
    model = SimpleNamespace(cfg=cfg, ep=None, device=torch.device("cpu"),
                            layers=layers)
    args = dict(max_requests=3, max_tokens=64, page_size=16)
    args.update(kw)
    return BatchDecoder(model, **args)


def test_history_of_penalised_requests_alone(monkeypatch):
    """The history that goes to the kernel is as wide as the longest request
    with penalties, and other requests' rows of it count for nothing: the
    longest of all may be longer than penalties reach."""
    monkeypatch.setattr(batch, "MAX_HISTORY", 30)
    dec = decoder()
    dec.submit(list(range(40)), 5)                       # longer than that
    dec.submit([1, 2, 3], 5, LogitRules(presence=1.0))
    dec.submit([4, 5], 5, LogitRules(bias={3: 1.0}))
    dec._admit()
    dec.slots[1].out = [7, 8]
    seen = {}

    def process(logits, **kw):
        seen.update(kw)
        return torch.tensor([10, 11, 12], dtype=torch.int32)

    monkeypatch.setattr(ops, "process_logits", process)
    dec.logits = torch.zeros(3, VOCAB)
    assert dec._pick((0, 1, 2), {}) == {0: 10, 1: 11, 2: 12}
    assert seen["history"].shape == (3, 5)
    assert seen["n_history"].tolist() == [0, 5, 0]
    assert seen["n_prompt"].tolist() == [0, 3, 0]
    # the picked tokens stand at their own places all the same
    assert dec.history[0, 40] == 10 and dec.history[1, 5] == 11
    assert dec.history[2, 2] == 12


def idle(dec):
    return (not dec.busy and dec._reserved == 0 and
            all(r is None for r in dec.slots))


def test_refused_generate_leaves_nothing_queued():
    dec = decoder()
    for prompts, rules in (([[1], [VOCAB]], None), ([[1], [2] * 64], None),
                           ([[1], []], None), ([[1], [2]], [None])):
        with pytest.raises(ValueError):
            dec.generate(prompts, 2, rules)
        assert idle(dec)
    with pytest.raises(ValueError):
        dec.generate([[1], [2]], 2, [None, LogitRules(bias={VOCAB: 1.0})])
    assert idle(dec)


def test_failed_generate_takes_its_requests_back():
    """A step that raises before it changed anything (a mask that raises):
    generate's requests go, running and waiting ones, and nobody else's are
    touched."""
    dec = decoder(max_requests=2)
    steps = []

    def step():
        dec._admit()
        steps.append([r.rid for r in dec.slots if r is not None])
        for r in dec.slots:
            r.fed = len(r.prompt)
        if len(steps) == 2:
            raise KeyError("no such state")
        return {r.rid: 1 for r in dec.slots}

    dec.step = step
    with pytest.raises(KeyError):
        dec.generate([[1], [2], [3]], 4)
    assert steps == [[0, 1], [0, 1]] and idle(dec)
    assert dec._gone == {0, 1}          # their pages go back with the next step
    rid = dec.submit([1], 2)
    with pytest.raises(RuntimeError):
        dec.generate([[1]], 2)          # not beside submitted ones
    assert [r.rid for r in dec._queue] == [rid]


@pytest.mark.parametrize("kw", [
    dict(max_requests=8193), dict(n_pages=0), dict(n_pages=1 << 27),
    dict(max_tokens=(1 << 30) + 1), dict(cache_dtype=torch.float16),
    dict(kv_scale=[torch.ones(2, 2)] * 2),              # bf16 pages have none
    *[dict(cache_dtype=torch.float8_e4m3fn, kv_scale=s) for s in (
        [torch.ones(2, 2)], torch.ones(2, 2), [torch.ones(2, 3)] * 2,
        [torch.ones(2, 2).double()] * 2, [torch.ones(2, 4)[:, ::2]] * 2,
        [None] * 2)]])
def test_caches_that_no_step_could_use(kw):
    """Refused with the decoder, not by the first step, which would lose the
    requests; nothing is allocated before."""
    with pytest.raises(ValueError):
        decoder(**kw)


def test_e4m3_caches():
    two = [torch.ones(2, 2)] * 2
    dec = decoder(cache_dtype=torch.float8_e4m3fn, kv_scale=two)
    assert dec.cache.kv_scale == two
    one = torch.full((2, 2, 2), 0.5)                    # a layer each
    dec = decoder(cache_dtype=torch.float8_e4m3fn, kv_scale=one)
    assert [s.tolist() for s in dec.cache.kv_scale] == one.tolist()
    dec = decoder(cache_dtype=torch.float8_e4m3fn)
    for s in dec.cache.kv_scale:
        assert s[0].tolist() == pytest.approx([8 / 448] * 2)
        assert s[1].tolist() == [1, 1]


def test_rows_of_a_step(monkeypatch):
    """Prompt chunks are cut where a step would have more rows than it can;
    every running request keeps its own."""
    monkeypatch.setattr(batch, "MAX_ROWS", 12, raising=False)
    dec = decoder(max_requests=4)
    for n in (7, 9, 1, 9):
        dec.submit([1] * n, 5)
    dec._admit()
    assert dec._rows_of_slots() == [7, 3, 1, 1]
    dec.slots[0].fed = 7                    # decodes
    assert dec._rows_of_slots() == [1, 9, 1, 1]
    dec.slots[2] = None
    assert dec._rows_of_slots() == [1, 9, 0, 2]
    dec._gone.add(2)
    dec.chunk = 4
    assert dec._rows_of_slots() == [1, 4, -1, 4]


def test_keys_without_a_weight():
    """A key norm of zeros has keys of zero: any scale but 0 holds them."""
    cfg_layers = decoder().model.layers
    cfg_layers[1].k_norm = torch.zeros(64)
    dec = decoder()
    scale = dec._key_scale(cfg_layers[1])
    assert (scale > 0).all() and torch.isfinite(scale).all()


@pytest.mark.parametrize("rules", [
    LogitRules(repetition=1e-50), LogitRules(bias={1.5: 1.0}),
    LogitRules(bias={"1": 1.0})])
def test_rules_as_the_kernel_has_them(rules):
    """A repetition that is 0 in 32 bits, ids that are not whole numbers."""
    dec = decoder()
    with pytest.raises(ValueError):
        dec.submit([1, 2], 3, rules)
    assert idle(dec)
