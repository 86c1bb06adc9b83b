"""Several requests decoded together over a paged KV cache.

``BatchDecoder`` drives a ``SynthDecoder`` (model.py) with rows of many
requests per step: the plan of the step (``ops.paged_plan``: pages, block
tables, slots), per layer the q/k norm + RoPE + append to the pages and the
attention over them, the pool-backed experts on all rows (the reference's
SwitchGLU wrapper takes any number of rows, streamlx/integrate.py:234-298), and
the logits' penalties, biases and grammar masks with the greedy pick.  Prompts
are fed in chunks beside the requests that already decode.  The reference
decodes one request at a time (examples/generate.py:67-89).
"""

from __future__ import annotations

from collections import deque
from dataclasses import dataclass, field

import numpy as np
import torch

from . import _lib as L
from . import ops


MAX_BIAS = 8191         # biased ids of a request
MAX_HISTORY = 262143    # tokens of a request with penalties
MAX_ROWS = 65535        # of a step: what the embedding and the router take
MAX_REQUESTS = 8192     # places of a cache
MAX_TOKENS = 1 << 30    # of a request; of a cache's pages: below 2^31


@dataclass
class LogitRules:
    """What one request's logits go through before the pick."""
    repetition: float = 1.0
    frequency: float = 0.0
    presence: float = 0.0
    bias: dict = field(default_factory=dict)    # id -> added logit
    # grammar: called with the request's output ids, returns uint32 words
    # (bit i of word w allows id 32 w + i) or None for "anything"
    mask: object = None

    @property
    def penalises(self) -> bool:
        return bool(self.repetition != 1 or self.frequency or self.presence)

    def check(self, vocab: int, tokens: int) -> None:
        """Raise ValueError unless a request of ``tokens`` tokens can have
        these rules."""
        if not np.float32(self.repetition) > 0:     # (what the kernel has)
            raise ValueError(f"repetition {self.repetition}: must be positive")
        if self.frequency != self.frequency or self.presence != self.presence:
            raise ValueError("frequency and presence must be numbers")
        if self.penalises and tokens > MAX_HISTORY:
            raise ValueError(f"{tokens} tokens: penalties reach "
                             f"{MAX_HISTORY} at most")
        if len(self.bias) > MAX_BIAS:
            raise ValueError(f"{len(self.bias)} biases: {MAX_BIAS} at most")
        for i, v in self.bias.items():
            if not isinstance(i, (int, np.integer)) or \
                    not 0 <= i < vocab or v != v:
                raise ValueError(f"bias {v} of id {i} (vocabulary {vocab})")


class PagedKVCache:
    """KV pages of every layer and the state of their requests, on the GPU.
    E4m3 pages hold value / scale; ``kv_scale`` [2, kv_heads] per layer."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, *,
                 n_pages: int, page_size: int, max_requests: int,
                 max_tokens: int, dtype=torch.bfloat16, kv_scale=None,
                 device=None):
        if page_size not in ops.PAGE_SIZES:
            raise ValueError(f"page_size {page_size}: one of {ops.PAGE_SIZES}")
        if not 1 <= max_requests <= MAX_REQUESTS or \
                not 1 <= max_tokens <= MAX_TOKENS or n_pages < 1 or \
                n_pages * page_size > 0x7fffffff:
            raise ValueError(f"{max_requests} requests of {max_tokens} tokens "
                             f"on {n_pages} pages of {page_size}: 1 to "
                             f"{MAX_REQUESTS} requests, 1 to {MAX_TOKENS} "
                             "tokens, pages for fewer than 2^31")
        if dtype == torch.float8_e4m3fn:
            kv_scale = [] if kv_scale is None else list(kv_scale)
            if len(kv_scale) != layers or not all(
                    isinstance(s, torch.Tensor) and s.is_contiguous() and
                    s.dtype == torch.float32 and s.shape == (2, kv_heads)
                    for s in kv_scale):
                raise ValueError("an e4m3 cache needs kv_scale, contiguous "
                                 f"float32 [2, {kv_heads}] for each of "
                                 f"{layers} layers")
            kv_scale = [s.to(device) for s in kv_scale]
        elif dtype != torch.bfloat16:
            raise ValueError(f"cache dtype {dtype}: bfloat16 or float8_e4m3fn")
        elif kv_scale is not None:
            raise ValueError("a bfloat16 cache takes no kv_scale")
        self.page_size, self.n_pages = page_size, n_pages
        self.pages = [torch.zeros(n_pages, 2, kv_heads, page_size, head_dim,
                                  dtype=dtype, device=device)
                      for _ in range(layers)]
        self.kv_scale = kv_scale or [None] * layers
        i32 = dict(dtype=torch.int32, device=device)
        cols = self.pages_for(max_tokens)
        self.table = torch.full((max_requests, cols), -1, **i32)
        self.lengths = torch.zeros(max_requests, **i32)
        # popped from the end: page 0 first
        self.free_list = torch.arange(n_pages - 1, -1, -1, **i32)
        self.n_free = torch.full((1,), n_pages, **i32)

    def pages_for(self, tokens: int) -> int:
        return (tokens + self.page_size - 1) // self.page_size

    def plan(self, n_new: torch.Tensor, n_rows: int, status) -> ops.PagedPlan:
        """Rows of a step; the cache's lengths and free pages move on."""
        return ops.paged_plan(n_new, self.lengths, self.table, self.free_list,
                              self.n_free, self.page_size, n_rows,
                              lengths_out=self.lengths, n_free_out=self.n_free,
                              status=status)


class _Request:
    def __init__(self, rid, prompt, max_new, rules, eos):
        self.rid, self.prompt, self.max_new = rid, prompt, max_new
        self.rules, self.eos = rules, eos
        self.fed = 0                # tokens in the cache
        self.out: list[int] = []


class BatchDecoder:
    """Decodes up to ``max_requests`` requests of a decoder together.

    ``submit`` queues a request, ``step`` runs one step and returns the tokens
    it picked, ``generate`` runs a list of prompts to their ends.  A request
    is admitted when the pages of its prompt and ``max_new`` tokens are free,
    so a running one never runs out.  The pools' bookkeeping is the eager
    path's (one host sync on the routed ids per layer); single-request decode
    through the step graph stays ``SynthDecoder.step``, and so does its
    temporal-reuse routing override (``repeat_p``), which does not apply here.

    A mask that raises, or whose words do not fit, leaves the requests as they
    were.  When a step fails later than that (a device error, an interrupt)
    its requests are lost: further steps raise, build a new decoder."""

    def __init__(self, model, max_requests: int = 8, max_tokens: int = 1024,
                 n_pages: int | None = None, page_size: int = 64,
                 cache_dtype=torch.bfloat16, kv_scale=None,
                 prompt_chunk: int = 64):
        cfg = model.cfg
        if not cfg.has_trunk:
            raise ValueError("batched decode needs a decoder with attention")
        if model.ep is not None:
            raise ValueError("batched decode runs on one GPU: the experts of "
                             "this model are sharded")
        if max_requests < 1 or max_tokens < 1 or prompt_chunk < 1:
            raise ValueError("max_requests, max_tokens and prompt_chunk must "
                             "be positive")
        if page_size not in ops.PAGE_SIZES:
            raise ValueError(f"page_size {page_size}: one of {ops.PAGE_SIZES}")
        if cfg.head_dim not in (64, 128) or cfg.heads > 16 * cfg.kv_heads:
            raise ValueError(f"batched decode needs heads of 64 or 128 and at "
                             f"most 16 of them a kv head, not {cfg.head_dim} "
                             f"and {cfg.heads}/{cfg.kv_heads}")
        self.model, self.cfg, self.device = model, cfg, model.device
        self.max_tokens, self.chunk = max_tokens, prompt_chunk
        if n_pages is None:
            n_pages = max_requests * ((max_tokens + page_size - 1) // page_size)
        if cache_dtype == torch.float8_e4m3fn and kv_scale is None:
            kv_scale = [self._key_scale(la) for la in model.layers]
        self.cache = PagedKVCache(
            cfg.layers, cfg.kv_heads, cfg.head_dim, n_pages=n_pages,
            page_size=page_size, max_requests=max_requests,
            max_tokens=max_tokens, dtype=cache_dtype, kv_scale=kv_scale,
            device=self.device)
        self.slots: list[_Request | None] = [None] * max_requests
        self._gone: set[int] = set()    # slots whose pages go back next step
        self._queue: deque = deque()
        self._next_id = 0
        self._reserved = 0              # pages promised to running requests
        self._failed = False            # a step did not come to its end
        i32 = dict(dtype=torch.int32, device=self.device)
        self.status = torch.zeros(1, **i32)
        self.history = torch.zeros(max_requests, max_tokens, **i32)
        self.last = torch.zeros(max_requests, **i32)    # last picked tokens
        self.logits: torch.Tensor | None = None     # of the last step's picks
        self.logits_of: list[int] = []              # their request ids

    def _key_scale(self, layer) -> torch.Tensor:
        """A key leaves the RMSNorm with at most sqrt(head_dim) times the
        largest norm weight, so this scale keeps it within e4m3's 448;
        values keep scale 1."""
        kv, hd = self.cfg.kv_heads, self.cfg.head_dim
        s = torch.ones(2, kv, device=self.device)
        most = layer.k_norm.float().abs().max() * hd ** 0.5 / 448
        s[0] = torch.where(most > 0, most, 1.0)     # (keys of zero)
        return s

    # ------------------------------------------------------------ requests --

    def submit(self, prompt, max_new: int, rules: LogitRules | None = None,
               eos: int | None = None) -> int:
        """Queue a request; returns its id."""
        prompt = [int(t) for t in prompt]
        if not prompt or max_new < 1:
            raise ValueError("a request needs a prompt and max_new >= 1")
        if any(not 0 <= t < self.cfg.vocab for t in prompt):
            raise ValueError("prompt token outside the vocabulary")
        total = len(prompt) + max_new
        if total > self.max_tokens or \
                self.cache.pages_for(total) > self.cache.n_pages:
            raise ValueError(f"{total} tokens do not fit the cache "
                             f"({self.max_tokens} a request, "
                             f"{self.cache.n_pages} pages)")
        if rules is not None:
            rules.check(self.cfg.vocab, total)
        r = _Request(self._next_id, prompt, max_new, rules, eos)
        self._next_id += 1
        self._queue.append(r)
        return r.rid

    def _pages(self, r: _Request) -> int:
        return self.cache.pages_for(len(r.prompt) + r.max_new)

    def _admit(self) -> None:
        for s, r in enumerate(self.slots):
            if not self._queue:
                return
            if r is not None or s in self._gone:
                continue
            new = self._queue[0]
            if self._reserved + self._pages(new) > self.cache.n_pages:
                return
            self._queue.popleft()
            self._reserved += self._pages(new)
            self.slots[s] = new
            self.history[s, :len(new.prompt)] = torch.tensor(
                new.prompt, dtype=torch.int32, device=self.device)

    @property
    def busy(self) -> bool:
        return bool(self._queue) or any(r is not None for r in self.slots)

    # ---------------------------------------------------------------- step --

    @torch.no_grad()
    def step(self) -> dict[int, int]:
        """One step of every running request: its next prompt chunk, or its
        last token.  Returns {request id: picked token} of the requests past
        their prompts; a request whose mask allows nothing ends with -1."""
        if self._failed:
            raise RuntimeError("an earlier step of this decoder failed and "
                               "its requests are lost: build a new one")
        with torch.cuda.device(self.device):
            self._admit()
            counts = self._rows_of_slots()
            masks = self._masks(counts)
            self._failed = True
            got = self._step(counts, masks)
            self._failed = False
        return got

    def _rows_of_slots(self) -> list[int]:
        """Rows of each slot's request in the next step (-1: its pages go
        back); chunks of later slots are cut where they pass MAX_ROWS."""
        n = []
        spare = MAX_ROWS - sum(r is not None for r in self.slots)
        for s, r in enumerate(self.slots):
            if r is None:
                n.append(-1 if s in self._gone else 0)
            else:
                more = min(len(r.prompt) - r.fed, self.chunk) - 1
                n.append(1 + max(0, min(more, spare)))
                spare -= n[-1] - 1
        return n

    def _masks(self, counts) -> dict:
        """{slot: mask words} of the requests that the step picks for."""
        words, out = (self.cfg.vocab + 31) // 32, {}
        for s, (r, n) in enumerate(zip(self.slots, counts)):
            if r is None or r.fed + n < len(r.prompt):
                continue
            if r.rules is None or r.rules.mask is None:
                continue
            w = r.rules.mask(list(r.out))
            if w is not None:
                w = np.asarray(w, dtype=np.uint32)
                if w.ndim != 1 or len(w) < words:
                    raise ValueError(f"request {r.rid}: mask of shape "
                                     f"{w.shape}, {words} words wanted")
                out[s] = w[:words]
        return out

    def _step(self, n_new, masks) -> dict[int, int]:
        self.model.flush()
        ids, from_last, picking = [], [], []
        for s, r in enumerate(self.slots):
            if r is None:
                continue
            n = n_new[s]
            if r.fed < len(r.prompt):
                ids += r.prompt[r.fed:r.fed + n]
            else:
                from_last.append((len(ids), s))
                ids.append(0)
            r.fed += n
            if r.fed >= len(r.prompt):
                picking.append((s, len(ids) - 1))   # slot, its last row
        dev = self.device
        rows = len(ids)
        plan = self.cache.plan(torch.tensor(n_new, dtype=torch.int32).to(dev),
                               rows, self.status)
        self._gone.clear()
        if rows == 0:
            self._check()
            return {}
        tok = torch.tensor(ids, dtype=torch.int32).to(dev)
        if from_last:
            at, slot = (torch.tensor(v, device=dev) for v in zip(*from_last))
            tok[at] = self.last[slot]
        used = max(s for s, n in enumerate(n_new) if n > 0) + 1
        x = self._forward(tok, plan, used)
        if not picking:
            self._check()
            return {}
        slots, last = zip(*picking)
        self.logits_of = [self.slots[s].rid for s in slots]
        x = x[torch.tensor(last, device=dev)].contiguous()
        self.logits = torch.empty(len(slots), self.cfg.vocab,
                                  dtype=torch.bfloat16, device=dev)
        L.qlinear(self.model.w_lm, self.cfg.vocab, self.cfg.hidden,
                  self.cfg.trunk_bits, x, self.logits, self.status)
        return self._pick(slots, masks)

    def _forward(self, tok, plan, n_slots: int) -> torch.Tensor:
        """Hidden rows (after the final norm) of the step's tokens, which
        belong to the first ``n_slots`` slots."""
        m, cfg, dev, st = self.model, self.cfg, self.device, self.status
        T, H, hd, bits = tok.shape[0], cfg.hidden, cfg.head_dim, cfg.trunk_bits
        bf = dict(dtype=torch.bfloat16, device=dev)
        h, x = torch.empty(T, H, **bf), torch.empty(T, H, **bf)
        L.dequant_rows(m.embed, H, bits, tok, T, cfg.vocab, h, st)
        qkv = torch.empty(T, (cfg.heads + 2 * cfg.kv_heads) * hd, **bf)
        att = torch.empty(T, cfg.heads, hd, **bf)
        o = torch.empty(T, H, **bf)
        work = ops.paged_workspace(T, cfg.heads, cfg.kv_heads, hd, dev)
        ids = torch.empty(T, cfg.top_k, dtype=torch.int32, device=dev)
        scores = torch.empty(T, cfg.top_k, dtype=torch.float32, device=dev)
        scratch = torch.zeros(L.router_scratch_bytes(T, cfg.n_experts),
                              dtype=torch.uint8, device=dev)
        # (the attention goes by the rows that a request of its table has)
        table = self.cache.table[:n_slots]
        delta = None
        for i, la in enumerate(m.layers):
            pages, scale = self.cache.pages[i], self.cache.kv_scale[i]
            L.add_rmsnorm(h, delta, la.w_in, cfg.rms_eps, x)
            L.qlinear(la.w_qkv, la.n_qkv, H, bits, x, qkv, st)
            q = ops.paged_append(qkv, pages, plan.slot, plan.pos, cfg.heads,
                                 la.q_norm, la.k_norm, cfg.rms_eps,
                                 m.inv_freq, kv_scale=scale, status=st)
            ops.paged_attention(q, pages, table, plan.pos,
                                req=plan.req, kv_scale=scale, out=att,
                                workspace=work, status=st)
            L.qlinear(la.w_o, H, cfg.heads * hd, bits, att, o, st, T=T)
            L.add_rmsnorm(h, o, la.post_attention_layernorm, cfg.rms_eps, x)
            blk = la.mlp
            L.router_topk(x, blk.w_gate, blk.bias, cfg.top_k,
                          cfg.norm_topk_prob, ids, scores, scratch, st)
            delta = blk.switch_mlp.fused(x[None], scores[None], ids[None])[0]
        L.add_rmsnorm(h, delta, m.norm, cfg.rms_eps, x)
        return x

    def _pick(self, slots, masks) -> dict[int, int]:
        """Rules, greedy pick and the requests' state after it."""
        dev, V = self.device, self.cfg.vocab
        reqs = [self.slots[s] for s in slots]
        rules = [r.rules or LogitRules() for r in reqs]
        at = torch.tensor(slots, device=dev)
        n_hist = [len(r.prompt) + len(r.out) for r in reqs]
        kw = {}
        if any(u.penalises for u in rules):
            kw = {name: torch.tensor([getattr(u, name) for u in rules],
                                     dtype=torch.float32).to(dev)
                  for name in ("repetition", "frequency", "presence")}
            # (no history of the others: they may be longer than MAX_HISTORY)
            said = [u.penalises for u in rules]
            n = [h if p else 0 for h, p in zip(n_hist, said)]
            kw["history"] = self.history[at, :max(n)].contiguous()
            kw["n_prompt"] = torch.tensor(
                [len(r.prompt) if p else 0 for r, p in zip(reqs, said)],
                dtype=torch.int32).to(dev)
            kw["n_history"] = torch.tensor(n, dtype=torch.int32).to(dev)
        if any(u.bias for u in rules):
            b = [list(u.bias.items()) for u in rules]
            start = np.cumsum([0] + [len(e) for e in b]).astype(np.int32)
            ids, vals = zip(*[e for row in b for e in row])
            kw["bias"] = (torch.tensor(ids, dtype=torch.int32).to(dev),
                          torch.tensor(vals, dtype=torch.float32).to(dev),
                          torch.from_numpy(start).to(dev))
        if masks:
            m = np.full((len(reqs), (V + 31) // 32), 0xFFFFFFFF,
                        dtype=np.uint32)
            for i, s in enumerate(slots):
                if s in masks:
                    m[i] = masks[s]
            kw["mask"] = torch.from_numpy(m.view(np.int32)).to(dev)
        pick = ops.process_logits(self.logits, status=self.status, **kw)
        self.last[at] = pick
        # the picked token's place: its request's history goes on with it
        hist = torch.tensor(n_hist, device=dev).clamp(max=self.max_tokens - 1)
        self.history[at, hist] = pick
        got = pick.tolist()
        self._check()
        for s, r, t in zip(slots, reqs, got):
            r.out.append(t)
            if t < 0 or t == r.eos or len(r.out) >= r.max_new:
                self._end(s)
        return {r.rid: t for r, t in zip(reqs, got)}

    def _check(self) -> None:
        ops.check_status(self.device)
        code = int(self.status.item())
        if code != 0:
            self.status.zero_()
            raise L.SlxError("device", code, "batched decode step device error")

    # ------------------------------------------------------------ generate --

    def generate(self, prompts, max_new: int, rules=None,
                 eos: int | None = None) -> list[list[int]]:
        """Every prompt to its end; ``rules``: one LogitRules, or one per
        prompt.  A mask that allows nothing ends a request without a token.
        Not while submitted requests run: their tokens come from ``step``.
        When it raises (a prompt that is refused, a mask that raises) none of
        its requests stays."""
        if self.busy:
            raise RuntimeError("generate: submitted requests are running, "
                               "their tokens come from step")
        if not isinstance(rules, (list, tuple)):
            rules = [rules] * len(prompts)
        if len(rules) != len(prompts):
            raise ValueError("one LogitRules per prompt")
        ids: list[int] = []
        try:
            for p, r in zip(prompts, rules):
                ids.append(self.submit(p, max_new, r, eos))
            out: dict = {i: [] for i in ids}
            while self.busy:
                for rid, t in self.step().items():
                    if t >= 0:
                        out[rid].append(t)
        except BaseException:
            self._withdraw(set(ids))
            raise
        self.release()
        return [out[i] for i in ids]

    def _withdraw(self, ids: set[int]) -> None:
        """Drop requests; the running ones' pages go back with the next step."""
        self._queue = deque(r for r in self._queue if r.rid not in ids)
        for s, r in enumerate(self.slots):
            if r is not None and r.rid in ids:
                self._end(s)

    def _end(self, s: int) -> None:
        self._reserved -= self._pages(self.slots[s])
        self.slots[s] = None
        self._gone.add(s)

    def release(self) -> None:
        """Hand the finished requests' pages back now (a step does, too)."""
        if self._gone:
            n = [-1 if s in self._gone else 0 for s in range(len(self.slots))]
            with torch.cuda.device(self.device):
                self.cache.plan(torch.tensor(n, dtype=torch.int32).to(
                    self.device), 0, self.status)
            self._gone.clear()
