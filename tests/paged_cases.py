"""Plain 64-bit restatements of the batched-decode operators for their tests
(host side: torch float64 / Python integers)."""

from __future__ import annotations

import torch


def pages_for(n: int, page: int) -> int:
    return (n + page - 1) // page


def make_cache(lens, n_kv, hd, page, dtype, seed=0, spare=3, tail="nan",
               std=1.0, scale=None):
    """(pages, kv_scale, table) on the CPU: each request's tokens in randomly
    placed pages; everything no request holds is NaN (tail='nan')."""
    g = torch.Generator().manual_seed(seed)
    need = [pages_for(n, page) for n in lens]
    n_pages = sum(need) + spare
    perm = torch.randperm(n_pages, generator=g)
    cols = max(max(need), 1) + 1
    table = torch.full((len(lens), cols), -1, dtype=torch.int32)
    x = torch.randn(n_pages, 2, n_kv, page, hd, generator=g) * std
    keep = torch.zeros(n_pages, page, dtype=torch.bool)
    at = 0
    for i, n in enumerate(lens):
        for c in range(need[i]):
            p = int(perm[at])
            at += 1
            table[i, c] = p
            keep[p, :min(page, n - c * page)] = True
    if tail == "nan":
        x = torch.where(keep[:, None, None, :, None], x, float("nan"))
    kv_scale = None
    if dtype == torch.float8_e4m3fn:
        kv_scale = torch.rand(2, n_kv, generator=g) * 0.02 + 0.01 \
            if scale is None else scale
        x = (x / kv_scale[None, :, :, None, None]).clamp(-448, 448)
    return x.to(dtype), kv_scale, table


def dense(pages, kv_scale, table, i, n, page):
    """Request i's first n keys and values, float64 [2, n_kv, n, hd]."""
    ids = table[i, :pages_for(n, page)].long()
    x = pages.float()[ids].double()
    if kv_scale is not None:
        x = x * kv_scale.double()[None, :, :, None, None]
    x = x.permute(1, 2, 0, 3, 4)
    return x.reshape(2, x.shape[1], -1, x.shape[4])[:, :, :n]


def attention(q, pages, kv_scale, table, req, pos, page, scale):
    """(out, bound) in float64: softmax attention of each row over positions
    0..pos, and how far a bf16 result computed in fp32 may be from it.

    With A = sum p |v|: a score's error is at most hd steps of 2^-23 of
    scale * sum |q k| (fp32 sums of exact products), and 2^-22 |s| from the
    scaling and the exponential's argument; p is off by that relatively, and
    by 2^-15 from its own rounding to two 8-bit parts and the exponential; the
    sums over n keys add n 2^-23; numerator and denominator both count.  The
    output is rounded once: 2^-8 |out|."""
    T, nq, hd = q.shape
    kv = pages.shape[2]
    G = nq // kv
    out = torch.zeros(T, nq, hd, dtype=torch.float64)
    bound = torch.zeros_like(out)
    for t in range(T):
        n = int(pos[t]) + 1
        if n <= 0:
            continue
        K, V = dense(pages, kv_scale, table, int(req[t]), n, page)
        qt = q[t].double().reshape(kv, G, hd)
        s = torch.einsum("kgd,kld->kgl", qt, K) * scale
        mag = torch.einsum("kgd,kld->kgl", qt.abs(), K.abs()) * abs(scale)
        p = torch.softmax(s, -1)
        o = torch.einsum("kgl,kld->kgd", p, V)
        A = torch.einsum("kgl,kld->kgd", p, V.abs())
        ds = hd * 2.0 ** -23 * mag.amax(-1) + 2.0 ** -22 * s.abs().amax(-1)
        rel = 2 * (2.0 ** -15 + ds + n * 2.0 ** -23)
        out[t] = o.reshape(nq, hd)
        bound[t] = (2.0 ** -8 * o.abs() + rel[..., None] * A).reshape(nq, hd)
    return out, bound


def rope(x, w, pos, inv_freq, eps):
    """RMSNorm over the last dim, then rotate-half RoPE, float64 [T, h, hd]."""
    x = x.double()
    x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w.double()
    a = pos.double()[:, None, None] * inv_freq.double()
    u, v = x.chunk(2, -1)
    return torch.cat([u * a.cos() - v * a.sin(), u * a.sin() + v * a.cos()], -1)


class Plan:
    """Request by request: the step's plan on plain lists."""

    def __init__(self, page, n_pages, max_pages):
        self.page, self.n_pages, self.max_pages = page, n_pages, max_pages

    def step(self, n_new, lengths, table, free_list, n_free, n_rows):
        """Returns (code, rows, start, lengths, table, free_list, n_free)."""
        P = self.page
        cap = self.max_pages * P
        pad = [(-1, -1, -1)] * n_rows
        same = (pad, [0] * (len(n_new) + 1), list(lengths),
                [list(r) for r in table], list(free_list), n_free)
        for n, ln in zip(n_new, lengths):
            if n < -1 or ln < 0 or ln + max(n, 0) > cap:
                return (-4, *same)
        back = sum(pages_for(ln, P) for n, ln in zip(n_new, lengths) if n < 0)
        get = sum(pages_for(ln + n, P) - pages_for(ln, P)
                  for n, ln in zip(n_new, lengths) if n >= 0)
        if n_free < 0 or n_free + back > self.n_pages:
            return (-4, *same)
        if sum(max(n, 0) for n in n_new) > n_rows or get > n_free + back:
            return (-10, *same)
        table = [list(r) for r in table]
        stack, top = list(free_list), n_free
        lengths = list(lengths)
        for i, n in enumerate(n_new):
            if n < 0:
                for c in range(pages_for(lengths[i], P)):
                    stack[top] = table[i][c]
                    top += 1
                lengths[i] = 0
        rows, start = [], [0]
        for i, n in enumerate(n_new):
            for j in range(max(n, 0)):
                p = lengths[i] + j
                if p % P == 0:
                    top -= 1
                    table[i][p // P] = stack[top]
                rows.append((i, p, table[i][p // P] * P + p % P))
            lengths[i] += max(n, 0)
            start.append(len(rows))
        rows += [(-1, -1, -1)] * (n_rows - len(rows))
        return 0, rows, start, lengths, table, stack, top


def logits(x, history, n_prompt, n_history, rep, freq, pres, bias, mask):
    """Processed logits (float64) and picks, row by row."""
    x = x.double().clone()
    T, V = x.shape
    picks = []
    for b in range(T):
        n = int(n_history[b]) if history is not None else 0
        p = int(n_prompt[b]) if n_prompt is not None else 0
        ids = history[b, :n].tolist() if n else []
        ids = [(i, j >= p) for j, i in enumerate(ids) if 0 <= i < V]
        for i in {i for i, _ in ids}:
            v = float(x[b, i])
            if rep is not None:
                r = float(rep[b])
                v = v / r if v > 0 else v * r
            c = sum(1 for j, said in ids if j == i and said)
            if c:
                if freq is not None:
                    v = v - float(freq[b]) * c
                if pres is not None:
                    v = v - float(pres[b])
            x[b, i] = v
        if bias is not None:
            b_ids, vals, start = bias
            last = {int(b_ids[j]): float(vals[j])
                    for j in range(int(start[b]), int(start[b + 1]))}
            for i, v in last.items():
                if 0 <= i < V:
                    x[b, i] += v
        ok = torch.ones(V, dtype=torch.bool)
        if mask is not None:
            t = torch.arange(V)
            ok = ((mask[b].long()[t // 32] >> (t % 32)) & 1).bool()
            x[b, ~ok] = -float("inf")
        y = torch.where(torch.isnan(x[b]), -float("inf"), x[b])
        at = torch.nonzero(ok & (y == y[ok].max()))[:, 0] if ok.any() else []
        picks.append(int(at[0]) if len(at) else -1)
    return x, picks
