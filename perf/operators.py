"""The operators of a batched decode step over a paged key-value cache, as
cases that can be timed: the step's plan (block tables, slot maps), the q/k
norm + RoPE + append to the pages, the attention of the new tokens over the
pages, and the processing of the logits with the greedy pick.

``own`` selects between the plain torch form of an operator (float32, or
float64 where float32 loses what matters) and this package's kernels."""

import itertools
import math
import random

import torch

own = False

VOCAB = 151936          # vocabulary of the decoder presets
EPS = 1e-6
THETA = 1_000_000.0
CACHE = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}


# ------------------------------------------------------------------ cases --

def listed():
    return [
        # one user's chat, early in the conversation: latency
        dict(name="attn 1x1k bf16", op="attn", rows=1, chunk=1, lo=1021, hi=1021, n_q=24, n_kv=4, hd=128, page=16, cache="bf16"),
        # one user's long document: the split over the cache's length
        dict(name="attn 1x128k bf16", op="attn", rows=1, chunk=1, lo=131071, hi=131071, n_q=16, n_kv=2, hd=128, page=64, cache="bf16"),
        # a server's mixed batch, some places of the batch idle
        dict(name="attn 64 ragged bf16", op="attn", rows=64, chunk=1, lo=0, hi=4096, n_q=24, n_kv=4, hd=128, page=16, cache="bf16"),
        # a full server: all of the cache read once, bandwidth
        dict(name="attn 256x6k bf16", op="attn", rows=256, chunk=1, lo=4099, hi=8192, n_q=24, n_kv=4, hd=128, page=32, cache="bf16"),
        # the same cache in 8 bits
        dict(name="attn 128 ragged e4m3", op="attn", rows=128, chunk=1, lo=1000, hi=16384, n_q=16, n_kv=2, hd=128, page=64, cache="e4m3"),
        # prompt chunks of several requests in one step, one kv head per q head
        dict(name="attn chunks hd64 e4m3", op="attn", rows=320, chunk=64, lo=200, hi=1500, n_q=8, n_kv=8, hd=64, page=16, cache="e4m3"),
        # one decode step's rows, one per request
        dict(name="append 64 bf16", op="append", rows=64, chunk=1, lo=1, hi=8192, n_q=24, n_kv=4, hd=128, page=16, cache="bf16"),
        # a step of prompt chunks into an 8-bit cache, far positions among them
        dict(name="append 4096 e4m3", op="append", rows=4096, chunk=512, lo=600, hi=131072, n_q=16, n_kv=2, hd=128, page=64, cache="e4m3"),
        # decode: every request one token, some of them at a page's end
        dict(name="plan 64 decode", op="plan", requests=64, page=16, most=512, new=1, fresh=0.0, gone=0.0),
        # requests come and go, prompts are fed in chunks beside decoding ones
        dict(name="plan 512 mixed", op="plan", requests=512, page=32, most=256, new=512, fresh=0.15, gone=0.1),
        # greedy pick of one request under a grammar
        dict(name="logits 1 greedy", op="logits", rows=1, vocab=VOCAB, hist=1000, bias=0, mask=True, write=False, kind="bf16"),
        # a batch's logits made ready for a sampler, every option in use
        dict(name="logits 128 all", op="logits", rows=128, vocab=VOCAB, hist=8000, bias=300, mask=True, write=True, kind="bf16"),
    ]


def log_size(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "append", "plan", "logits"])
    if op in ("attn", "append"):
        n_q, n_kv = rng.choice([(24, 4), (16, 2), (4, 2), (8, 8), (32, 2), (20, 4), (9, 3), (12, 1), (1, 1)])
        c = dict(op=op, n_q=n_q, n_kv=n_kv, hd=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128]), cache=rng.choice(["bf16", "e4m3"]))
        if op == "append":
            chunk = rng.choice([1, 1, log_size(rng, 2, 1000)])
            rows = log_size(rng, 1, 4096 // chunk) * chunk
            lo = log_size(rng, chunk, 50000)
            return dict(c, rows=rows, chunk=chunk, lo=lo, hi=log_size(rng, lo, 131072))
        chunk = rng.choice([1, 1, 1, log_size(rng, 2, 100)])
        requests = log_size(rng, 1, 256)
        # the cache holds at most 128k tokens x 8 heads, or 256 x 4k of them
        hi = log_size(rng, chunk, max(chunk, min(131072, 262144 * 4 // (requests * n_kv * chunk))))
        lo = rng.choice([chunk, log_size(rng, chunk, hi), hi])
        return dict(c, rows=requests * chunk, chunk=chunk, lo=0 if chunk == 1 and lo == 1 else lo, hi=hi)
    if op == "plan":
        requests = log_size(rng, 1, 1024)
        page = rng.choice([16, 32, 64, 128])
        new = rng.choice([1, log_size(rng, 2, 1000)])
        return dict(op=op, requests=requests, page=page, most=log_size(rng, 1200 // page + 2, 1024), new=new,
                    fresh=round(rng.uniform(0, 0.5), 3), gone=round(rng.uniform(0, 0.3), 3))
    return dict(op=op, rows=log_size(rng, 1, 128), vocab=rng.choice([VOCAB, log_size(rng, 33, VOCAB)]), hist=rng.choice([0, log_size(rng, 1, 16000)]),
                bias=rng.choice([0, log_size(rng, 1, 300)]), mask=rng.random() < 0.6, write=rng.random() < 0.6, kind=rng.choice(["bf16", "f32"]))


# ------------------------------------------------- the shape of a case --

def lengths_of(c):
    """Tokens of each request after the step: fixed by the case."""
    r = random.Random(c["lo"] * 31 + c["hi"])
    n = c["rows"] // c["chunk"]
    return [r.randint(c["lo"], c["hi"]) for _ in range(n)]


def plan_of(c):
    """(tokens held, new tokens or -1) of each request: fixed by the case."""
    r = random.Random(c["requests"] * 7 + c["most"])
    held, new = [], []
    room = c["most"] * c["page"]
    for _ in range(c["requests"]):
        x = r.random()
        if x < c["gone"]:                       # finished: its pages go back
            held.append(r.randint(1, room))
            new.append(-1)
        elif x < c["gone"] + c["fresh"]:        # a new request's first chunk
            held.append(0)
            new.append(r.randint(1, min(room, c["new"])))
        elif r.random() < 0.05:                 # an idle place
            held.append(0)
            new.append(0)
        else:
            held.append(r.randint(1, room - 1))
            new.append(1)
    return held, new


def pages_for(n, page):
    return (n + page - 1) // page


def work(c):
    if c["op"] == "attn":
        e = 2 if c["cache"] == "bf16" else 1
        lens = lengths_of(c)
        keys = sum(sum(max(0, n - j) for j in range(c["chunk"])) for n in lens)
        held = sum(lens)
        row = c["n_kv"] * c["hd"]
        return {"bytes": 2 * e * held * row + 4 * c["rows"] * c["n_q"] * c["hd"] + 4 * c["rows"] + 4 * sum(pages_for(n, c["page"]) for n in lens),
                "flops": 4 * keys * c["n_q"] * c["hd"]}
    if c["op"] == "append":
        e = 2 if c["cache"] == "bf16" else 1
        q, kv = c["n_q"] * c["hd"], 2 * c["n_kv"] * c["hd"]
        return {"bytes": c["rows"] * (2 * (q + kv) + 2 * q + e * kv + 8), "flops": c["rows"] * 10 * (q + kv // 2)}
    if c["op"] == "plan":
        held, new = plan_of(c)
        rows = sum(max(0, n) for n in new)
        back = sum(pages_for(h, c["page"]) for h, n in zip(held, new) if n < 0)
        out = sum(pages_for(h + n, c["page"]) - pages_for(h, c["page"]) for h, n in zip(held, new) if n >= 0)
        return {"bytes": 4 * (4 * c["requests"] + 2 * back + 2 * out + 3 * rows), "flops": 0}
    e = 2 if c["kind"] == "bf16" else 4
    per = c["vocab"] * e * (2 if c["write"] else 1) + 4 * c["hist"] + 8 * c["bias"] + (c["vocab"] // 8 if c["mask"] else 0)
    return {"bytes": c["rows"] * per, "flops": c["rows"] * c["vocab"]}


# ----------------------------------------------------------------- prepare --

def randn(g, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.bfloat16) * std).to(dtype)


def make_pages(g, c, n_pages):
    shape = (n_pages, 2, c["n_kv"], c["page"], c["hd"])
    if c["cache"] == "bf16":
        return randn(g, *shape), None
    # 8-bit pages hold value / scale, the scale set so that 448 is far out
    scale = torch.rand(2, c["n_kv"], generator=g, device="cuda") * 0.02 + 0.01
    return randn(g, *shape, std=60.0, dtype=torch.float8_e4m3fn), scale


def make_table(g, lens, page, spare):
    """Pages of the requests in random places: (table, number of pages)."""
    need = [pages_for(n, page) for n in lens]
    total = sum(need) + spare
    perm = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    cols = max(max(need), 1)
    first = torch.tensor([0, *itertools.accumulate(need)][:-1], device="cuda")
    n = torch.tensor(need, device="cuda")
    col = torch.arange(cols, device="cuda")[None, :]
    at = (first[:, None] + col).clamp(max=total - 1)
    return torch.where(col < n[:, None], perm[at], -1).to(torch.int32), total


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=c)
    if c["op"] in ("attn", "append"):
        lens = lengths_of(c)
        n = torch.tensor(lens, device="cuda")
        back = torch.arange(c["chunk"], device="cuda") - c["chunk"]
        s["pos"] = (n[:, None] + back[None, :]).reshape(-1).to(torch.int32)
        s["req"] = torch.arange(len(lens), device="cuda", dtype=torch.int32).repeat_interleave(c["chunk"])
        # an append reaches the pages of its chunk alone
        before = [0 if c["op"] == "attn" else (m - c["chunk"]) // c["page"] * c["page"] for m in lens]
        s["table"], n_pages = make_table(g, [m - b for m, b in zip(lens, before)], c["page"], 8)
        s["pages"], s["kv_scale"] = make_pages(g, c, n_pages)
        if c["op"] == "attn":
            # normalised and rotated queries
            s["q"] = randn(g, c["rows"], c["n_q"], c["hd"], std=1.5)
            s["scale"] = 1.0 / math.sqrt(c["hd"])
        else:
            s["qkv"] = randn(g, c["rows"], (c["n_q"] + 2 * c["n_kv"]) * c["hd"], std=2.0)
            s["q_norm"] = (1 + 0.2 * torch.randn(c["hd"], generator=g, device="cuda")).to(torch.bfloat16)
            s["k_norm"] = (1 + 0.2 * torch.randn(c["hd"], generator=g, device="cuda")).to(torch.bfloat16)
            half = c["hd"] // 2
            s["inv_freq"] = (THETA ** (-torch.arange(half, dtype=torch.float64) / half)).to("cuda", torch.float32)
            p = s["pos"].long() - torch.tensor(before, device="cuda")[s["req"].long()]
            s["slot"] = (s["table"][s["req"].long(), p // c["page"]].long() * c["page"] + p % c["page"]).to(torch.int32)
    elif c["op"] == "plan":
        held, new = plan_of(c)
        rel = sum(pages_for(h, c["page"]) for h in held)
        get = sum(pages_for(h + max(n, 0), c["page"]) - pages_for(h, c["page"]) for h, n in zip(held, new))
        table, n_pages = make_table(g, held, c["page"], get + 16)
        s["n_pages"] = n_pages
        s["table"] = torch.full((c["requests"], c["most"]), -1, dtype=torch.int32, device="cuda")
        s["table"][:, :table.shape[1]] = table
        used = torch.zeros(n_pages, dtype=torch.bool, device="cuda")
        used[table[table >= 0].long()] = True
        spare = torch.arange(n_pages, device="cuda", dtype=torch.int32)[~used]
        spare = spare[torch.randperm(spare.numel(), generator=g, device="cuda")]
        s["free_list"] = torch.full((n_pages,), -1, dtype=torch.int32, device="cuda")
        s["free_list"][:spare.numel()] = spare
        s["n_free"] = torch.tensor([n_pages - rel], dtype=torch.int32, device="cuda")
        s["lengths"] = torch.tensor(held, dtype=torch.int32, device="cuda")
        s["n_new"] = torch.tensor(new, dtype=torch.int32, device="cuda")
        s["n_rows"] = max(1, (sum(max(n, 0) for n in new) + 63) // 64 * 64)
    else:
        B, V, L = c["rows"], c["vocab"], c["hist"]
        x = torch.randn(B, V, generator=g, device="cuda") * 2.5
        s["logits"] = x.to(torch.bfloat16 if c["kind"] == "bf16" else torch.float32)
        # text repeats itself: a few ids often, many once; half of it prompt
        u = torch.rand(B, max(L, 1), generator=g, device="cuda", dtype=torch.float64)
        s["history"] = (V ** u).long().clamp(max=V).sub(1).to(torch.int32)
        s["n_hist"] = torch.randint(L // 4, L + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        s["n_prompt"] = (s["n_hist"].double() * torch.rand(B, generator=g, device="cuda", dtype=torch.float64)).to(torch.int32)
        s["repetition"] = 1.0 + 0.3 * torch.rand(B, generator=g, device="cuda")
        s["frequency"] = 0.5 * torch.rand(B, generator=g, device="cuda")
        s["presence"] = 0.5 * torch.rand(B, generator=g, device="cuda")
        s["bias"] = None
        if c["bias"]:
            n = torch.randint(0, c["bias"] + 1, (B,), generator=g, device="cuda")
            start = torch.zeros(B + 1, dtype=torch.int32, device="cuda")
            start[1:] = n.cumsum(0)
            ids = torch.randint(0, V, (B * c["bias"],), generator=g, device="cuda", dtype=torch.int32)
            vals = torch.randn(B * c["bias"], generator=g, device="cuda") * 3
            s["bias"] = (ids, vals, start)
        s["mask"] = None
        if c["mask"]:
            # a grammar allows little: one id in 64 here, and the row's own last word
            words = (V + 31) // 32
            m = torch.ones(B, words, dtype=torch.int32, device="cuda")
            for _ in range(6):
                m &= torch.randint(-2 ** 31, 2 ** 31, (B, words), generator=g, device="cuda").to(torch.int32)
            s["mask"] = m | (torch.randint(-2 ** 31, 2 ** 31, (B, words), generator=g, device="cuda").to(torch.int32) &
                             torch.where(torch.rand(B, words, generator=g, device="cuda") < 0.03, -1, 0).to(torch.int32))
        s["out"] = torch.empty_like(s["logits"]) if c["write"] else None
    return s


# --------------------------------------------------------------------- run --

def run(s):
    return {"attn": run_attn, "append": run_append, "plan": run_plan, "logits": run_logits}[s["case"]["op"]](s)


def run_attn(s):
    if own:
        from streamlx_b200 import ops
        return ops.paged_attention(s["q"], s["pages"], s["table"], s["pos"], req=s["req"], scale=s["scale"], kv_scale=s["kv_scale"])
    pages, table, pos, q = s["pages"], s["table"], s["pos"], s["q"]
    ps, kv = pages.shape[3], pages.shape[2]
    T, nq, hd = q.shape
    at = torch.arange(table.shape[1] * ps, device=q.device)
    # each request's keys and values in order, in 32 bits, [R, L, kv, hd]
    page = table.clamp(min=0)[:, at // ps].long()
    if pages.dtype == torch.float8_e4m3fn:
        raw = pages.view(torch.uint8)
        K = raw[page, 0, :, at % ps].view(torch.float8_e4m3fn).float() * s["kv_scale"][0][:, None]
        V = raw[page, 1, :, at % ps].view(torch.float8_e4m3fn).float() * s["kv_scale"][1][:, None]
    else:
        K, V = pages[page, 0, :, at % ps].float(), pages[page, 1, :, at % ps].float()
    R, c = table.shape[0], T // table.shape[0]
    # the rows of one request stand together
    qr = q.float().reshape(R, c, kv, nq // kv, hd).permute(0, 2, 1, 3, 4).reshape(R, kv, c * (nq // kv), hd)
    x = (qr @ K.permute(0, 2, 3, 1)).reshape(R, kv, c, nq // kv, -1) * s["scale"]
    x = torch.where(at <= pos.reshape(R, 1, c, 1, 1), x, -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    held = at <= pos.reshape(R, c).amax(1)[:, None]
    V = torch.where(held[:, :, None, None], V, 0.0)
    o = p.reshape(R, kv, c * (nq // kv), -1) @ V.permute(0, 2, 1, 3)
    return o.reshape(R, kv, c, nq // kv, hd).permute(0, 2, 1, 3, 4).reshape(T, nq, hd).to(torch.bfloat16)


def rotated(x, w, ang):
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    a, b = x.chunk(2, -1)
    return torch.cat([a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()], -1)


def run_append(s):
    c, pages = s["case"], s["pages"]
    if own:
        from streamlx_b200 import ops
        q = ops.paged_append(s["qkv"], pages, s["slot"], s["pos"], c["n_q"], s["q_norm"], s["k_norm"], EPS, s["inv_freq"], kv_scale=s["kv_scale"])
        return {"q": q, "pages": pages}
    n_q, n_kv, hd, ps = c["n_q"], c["n_kv"], c["hd"], c["page"]
    q, k, v = s["qkv"].float().split([n_q * hd, n_kv * hd, n_kv * hd], -1)
    # far positions: the angle in 64 bits, within one turn
    ang = torch.remainder(s["pos"].double()[:, None] * s["inv_freq"].double(), 2 * math.pi).float()[:, None]
    on = (s["slot"] >= 0)[:, None, None]
    q = torch.where(on, rotated(q.reshape(-1, n_q, hd), s["q_norm"].float(), ang), 0.0).to(torch.bfloat16)
    k = rotated(k.reshape(-1, n_kv, hd), s["k_norm"].float(), ang)
    v = v.reshape(-1, n_kv, hd)
    put, to = s["slot"].long(), pages
    if pages.dtype == torch.float8_e4m3fn:
        k = (k / s["kv_scale"][0][:, None]).clamp(-448, 448)
        v = (v / s["kv_scale"][1][:, None]).clamp(-448, 448)
        k, v, to = k.to(pages.dtype).view(torch.uint8), v.to(pages.dtype).view(torch.uint8), pages.view(torch.uint8)
    # a row without a slot writes back what is there
    page, row = put.clamp(min=0) // ps, put.clamp(min=0) % ps
    to[page, 0, :, row] = torch.where(on, k.to(to.dtype), to[page, 0, :, row])
    to[page, 1, :, row] = torch.where(on, v.to(to.dtype), to[page, 1, :, row])
    return {"q": q, "pages": pages}


def run_plan(s):
    c = s["case"]
    if own:
        from streamlx_b200 import ops
        p = ops.paged_plan(s["n_new"], s["lengths"], s["table"], s["free_list"], s["n_free"], c["page"], s["n_rows"])
        return {"req": p.req, "pos": p.pos, "slot": p.slot, "start": p.start, "lengths": p.lengths, "n_free": p.n_free,
                "table": s["table"], "free_list": s["free_list"]}
    ps, held, table = c["page"], s["lengths"].long(), s["table"]
    gone, new = s["n_new"] < 0, s["n_new"].clamp(min=0).long()
    had, need = (held + ps - 1) // ps, (held + new + ps - 1) // ps
    back, get = torch.where(gone, had, 0), torch.where(gone, 0, need - had)
    col = torch.arange(table.shape[1], device=table.device)[None, :]
    n_free = s["n_free"].long()
    # released pages go on top of the stack, in the requests' order
    dest = torch.where(col < back[:, None], n_free + (back.cumsum(0) - back)[:, None] + col, s["n_pages"])
    stack = torch.cat([s["free_list"], s["free_list"][:1]]).scatter(0, dest.reshape(-1), table.reshape(-1))[:-1]
    s["free_list"].copy_(stack)
    top = n_free + back.sum()
    take = (top - 1 - (get.cumsum(0) - get)[:, None] - (col - had[:, None])).clamp(0, s["n_pages"] - 1)
    table.copy_(torch.where((col >= had[:, None]) & (col < (had + get)[:, None]), stack[take], table))
    start = torch.cat([new.new_zeros(1), new.cumsum(0)])
    r = torch.arange(s["n_rows"], device=table.device)
    on = r < start[-1]
    req = torch.searchsorted(start[1:], r, right=True).clamp(max=c["requests"] - 1)
    pos = torch.where(on, held[req] + r - start[req], 0)
    slot = table[req, pos // ps].long() * ps + pos % ps
    i32 = torch.int32
    return {"req": torch.where(on, req, -1).to(i32), "pos": torch.where(on, pos, -1).to(i32), "slot": torch.where(on, slot, -1).to(i32), "start": start.to(i32),
            "lengths": torch.where(gone, 0, held + new).to(i32), "n_free": (top - get.sum()).to(i32), "table": table, "free_list": s["free_list"]}


def run_logits(s):
    if own:
        from streamlx_b200 import ops
        pick = ops.process_logits(s["logits"], s["history"], s["n_prompt"], s["n_hist"], repetition=s["repetition"], frequency=s["frequency"],
                                  presence=s["presence"], bias=s["bias"], mask=s["mask"], out=s["out"])
        return {"pick": pick} if s["out"] is None else {"pick": pick, "logits": s["out"]}
    x = s["logits"].double()          # picks go by values next to each other
    B, V = x.shape
    h, dev = s["history"].long(), x.device
    at = torch.arange(h.shape[1], device=dev)[None, :]
    row = torch.arange(B, device=dev)[:, None]
    held = (at < s["n_hist"][:, None]).double()
    said = held * (at >= s["n_prompt"][:, None])
    seen = torch.zeros(B, V, device=dev, dtype=torch.float64).scatter_add(1, h, held) > 0
    count = torch.zeros(B, V, device=dev, dtype=torch.float64).scatter_add(1, h, said)
    rep = s["repetition"].double()[:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"].double()[:, None] * count
    x = torch.where(count > 0, x - s["presence"].double()[:, None], x)
    if s["bias"] is not None:
        ids, vals, start = s["bias"]
        i = torch.arange(ids.numel(), device=dev)
        of = torch.searchsorted(start[1:].long(), i, right=True)
        # an id that a row lists twice takes its last entry
        last = torch.full((B + 1, V), -1, device=dev, dtype=torch.int64).reshape(-1).scatter_reduce(0, of * V + ids.long(), i, "amax").reshape(B + 1, V)[:B]
        x = torch.where(last >= 0, x + vals.double()[last.clamp(min=0)], x)
    ok = torch.ones(B, V, device=dev, dtype=torch.bool)
    if s["mask"] is not None:
        t = torch.arange(V, device=dev)
        ok = (s["mask"][:, t // 32] >> (t % 32).to(torch.int32)) & 1 != 0
        x = torch.where(ok, x, -math.inf)
    best = ok & (x == x.amax(-1, keepdim=True))
    pick = torch.where(best, torch.arange(V, device=dev), V).amin(-1)
    pick = torch.where(pick < V, pick, -1).to(torch.int32)
    if s["out"] is None:
        return {"pick": pick}
    s["out"].copy_(x)
    return {"pick": pick, "logits": s["out"]}


# ------------------------------------------------------------------- exact --

def exact(c, seed):
    """The definitions in 64 bits, request by request."""
    if c["op"] == "plan":
        return None                   # whole numbers only
    s = prepare(c, seed)
    if c["op"] == "attn":
        return exact_attn(c, s)
    if c["op"] == "append":
        return exact_append(c, s)
    return exact_logits(c, s)


def exact_attn(c, s):
    G, ps = c["n_q"] // c["n_kv"], c["page"]
    out = torch.zeros(c["rows"], c["n_q"], c["hd"], dtype=torch.float64, device="cuda")
    for i, n in enumerate(lengths_of(c)):
        if n == 0:
            continue
        ids = s["table"][i, :pages_for(n, ps)].long()
        kv = s["pages"][ids] if c["cache"] == "bf16" else s["pages"].view(torch.uint8)[ids].view(torch.float8_e4m3fn)
        kv = kv.double()
        if s["kv_scale"] is not None:
            kv = kv * s["kv_scale"].double()[None, :, :, None, None]
        kv = kv.permute(1, 2, 0, 3, 4).reshape(2, c["n_kv"], -1, c["hd"])[:, :, :n]
        for j in range(c["chunk"]):
            r = i * c["chunk"] + j
            m = n - c["chunk"] + j + 1
            q = s["q"][r].double().reshape(c["n_kv"], G, c["hd"])
            w = torch.softmax(torch.einsum("kgd,kld->kgl", q, kv[0, :, :m]) * s["scale"], -1)
            out[r] = torch.einsum("kgl,kld->kgd", w, kv[1, :, :m]).reshape(c["n_q"], c["hd"])
    return out


def exact_append(c, s):
    n_q, n_kv, hd, ps = c["n_q"], c["n_kv"], c["hd"], c["page"]
    x = s["qkv"].double().reshape(c["rows"], n_q + 2 * n_kv, hd)
    a = s["pos"].double()[:, None] * s["inv_freq"].double()[None, :]
    turn = torch.polar(torch.ones_like(a), a)[:, None, :]

    def spun(v, w):
        v = v / torch.sqrt(v.pow(2).sum(-1, keepdim=True) / hd + EPS) * w.double()
        z = torch.complex(v[..., :hd // 2], v[..., hd // 2:]) * turn
        return torch.cat([z.real, z.imag], -1)

    on = s["slot"] >= 0
    q = spun(x[:, :n_q], s["q_norm"])
    q[~on] = 0
    kv = torch.stack([spun(x[:, n_q:n_q + n_kv], s["k_norm"]), x[:, n_q + n_kv:]], 1)
    if s["kv_scale"] is not None:
        # what the 8-bit cache holds is part of the definition
        kv = (kv / s["kv_scale"].double()[None, :, :, None]).clamp(-448, 448).float().to(torch.float8_e4m3fn).double()
    pages = s["pages"].double()
    to = s["slot"][on].long()
    pages[to // ps, :, :, to % ps] = kv[on]
    return {"q": q, "pages": pages}


def exact_logits(c, s):
    if s["out"] is None:
        return None                   # the pick alone: a whole number
    x = s["logits"].double()
    for b in range(c["rows"]):
        p, n = int(s["n_prompt"][b]), int(s["n_hist"][b])
        ids = s["history"][b, :n].long()
        every = ids.unique()
        rep = s["repetition"][b].double()
        v = x[b, every]
        x[b, every] = torch.where(v > 0, v / rep, v * rep)
        said, times = ids[p:].unique(return_counts=True)
        x[b, said] -= s["frequency"][b].double() * times + s["presence"][b].double()
        if s["bias"] is not None:
            ids, vals, start = s["bias"]
            lo, hi = int(start[b]), int(start[b + 1])
            last = dict(zip(ids[lo:hi].tolist(), vals[lo:hi].tolist()))
            if last:
                x[b, list(last)] += torch.tensor(list(last.values()), dtype=torch.float64, device="cuda")
        if s["mask"] is not None:
            bits = (s["mask"][b][:, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
            x[b, bits.reshape(-1)[:c["vocab"]] == 0] = -math.inf
    return {"pick": None, "logits": x}
