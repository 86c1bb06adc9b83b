"""Kernel-calling helpers around the pools (device side of the wrapper)."""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib as L

_scratch: dict = {}

# When a list, every switchglu launch pair appends (start, end) CUDA events
# recorded around it on the current stream (the bench's roofline timing).
TIMING: list | None = None


def _status(device) -> torch.Tensor:
    key = ("status", device)
    t = _scratch.get(key)
    if t is None:
        t = torch.zeros(1, dtype=torch.int32, device=device)
        _scratch[key] = t
    return t


def scratch(nbytes: int, device, tag: str = "glu") -> torch.Tensor:
    """Grow-only device scratch shared by calls on one device."""
    key = (tag, device)
    t = _scratch.get(key)
    if t is None or t.numel() < nbytes:
        # zeroed: the switchglu scratch ends with grid-barrier words
        t = torch.zeros(max(nbytes, 1 << 16), dtype=torch.uint8, device=device)
        _scratch[key] = t
    return t


def check_status(device) -> None:
    """Raise if a kernel recorded a device-side error (synchronises)."""
    st = _status(device)
    v = int(st.item())
    if v != 0:
        st.zero_()
        raise L.SlxError("device", v, "device-side error status")


def as_bf16_2d(x: torch.Tensor) -> torch.Tensor:
    x = x.reshape(-1, x.shape[-1])
    if x.dtype != torch.bfloat16:
        x = x.to(torch.bfloat16)
    return x.contiguous()


def as_ids_2d(ids, k: int, device) -> torch.Tensor:
    if not isinstance(ids, torch.Tensor):
        ids = torch.as_tensor(ids)
    ids = ids.reshape(-1, k)
    if ids.dtype != torch.int32 or ids.device != device:
        ids = ids.to(device=device, dtype=torch.int32)
    return ids.contiguous()


def switchglu(bank, x2d: torch.Tensor, ids2d: torch.Tensor, k: int, *,
              scores: torch.Tensor | None = None, table: torch.Tensor | None = None,
              shared=None, out: torch.Tensor | None = None,
              inter: int, shared_inter: int = 0,
              scratch_buf: torch.Tensor | None = None,
              status: torch.Tensor | None = None) -> torch.Tensor:
    """One fused SwitchGLU launch pair.  scores None -> [T, k, H] per-expert
    unweighted outputs; else [T, H] combined (+ shared expert).
    ``scratch_buf`` / ``status`` override the per-device shared ones (a
    captured graph needs buffers that never move)."""
    T, H = x2d.shape
    dev = x2d.device
    if out is None:
        shape = (T, H) if scores is not None else (T, k, H)
        out = torch.empty(shape, dtype=torch.bfloat16, device=dev)
    sI = shared_inter if (scores is not None and shared is not None) else 0
    need = L.switchglu_scratch_bytes(T, k, inter, sI)
    if scratch_buf is not None:
        if scratch_buf.numel() * scratch_buf.element_size() < need:
            raise ValueError("switchglu: scratch_buf too small")
        sc = scratch_buf
    else:
        sc = scratch(need, dev)
    ev = None
    if TIMING is not None:
        ev = (torch.cuda.Event(enable_timing=True),
              torch.cuda.Event(enable_timing=True))
        ev[0].record()
    L.switchglu(bank, x2d, ids2d, out, sc,
                _status(dev) if status is None else status, scores=scores,
                slot_table=table, shared=shared if sI else None)
    if ev is not None:
        ev[1].record()
        TIMING.append((ev[0], ev[1], T, k, inter, sI))
    return out


def switch_forward_ids(pool, x, expert_ids) -> torch.Tensor:
    """streamlx/pool.py:299-304 on the pool: per-expert outputs [1,1,k,H]."""
    k = len(expert_ids)
    x2d = as_bf16_2d(x)
    pool.sync_device()
    ids = as_ids_2d(list(expert_ids), k, x2d.device)
    y = switchglu(pool.store.bank, x2d, ids, k, table=pool.store.table_dev,
                  inter=pool.inter)
    return y.reshape(1, 1, k, -1)


PREFILL_BLOCK = 128   # pairs per block (the kernel's MMA N)
# pairs per call from which the pool path uses the grouped tensor-core
# prefill instead of the per-token GEMV kernels
PREFILL_MIN_PAIRS = 64


def prefill_supported(hidden: int, inter: int, bits: int) -> bool:
    return bits == 2 and hidden % 512 == 0 and inter % 512 == 0 and \
        hidden <= 4096 and inter <= 4096


def prefill_blocks(slots, counts) -> "np.ndarray":
    """Blocks {slot, first pair, pairs, 0} of pairs grouped by expert:
    segment i (``counts[i]`` consecutive pairs of slot ``slots[i]``) is split
    into runs of at most PREFILL_BLOCK pairs."""
    import numpy as np
    rows = []
    p = 0
    for s, n in zip(slots, counts):
        n = int(n)
        for o in range(0, n, PREFILL_BLOCK):
            rows.append((int(s), p + o, min(PREFILL_BLOCK, n - o), 0))
        p += n
    return np.asarray(rows, dtype=np.int32).reshape(-1, 4)


def prefill_grouped(bank, x2d: torch.Tensor, pair_row, slots, counts, *,
                    out: torch.Tensor | None = None, out_row=None,
                    n_out: int | None = None) -> torch.Tensor:
    """Expert-major prefill on the tensor cores: pairs grouped by expert
    (``pair_row[p]`` = x row of pair p; segment i = ``counts[i]`` pairs of
    slot ``slots[i]``).  Returns per-pair unweighted outputs [P, H] (rows
    ``out_row[p]`` when given)."""
    import numpy as np
    dev = x2d.device
    H = x2d.shape[1]
    blocks = prefill_blocks(slots, counts)
    P = int(np.sum(counts)) if len(counts) else 0
    if out is None:
        out = torch.empty(n_out if n_out is not None else P, H,
                          dtype=torch.bfloat16, device=dev)
    if blocks.shape[0] == 0:
        return out
    pr = torch.as_tensor(np.asarray(pair_row, dtype=np.int32), device=dev)
    bl = torch.as_tensor(blocks, device=dev)
    orow = None if out_row is None else torch.as_tensor(
        np.asarray(out_row, dtype=np.int32), device=dev)
    need = L.prefill_scratch_bytes(blocks.shape[0], H, bank.inter, bank.bits)
    if need == 0:
        raise L.SlxError("slx_prefill_scratch_bytes", -2, "unsupported shape")
    sc = scratch(need, dev, tag="prefill")
    st = _status_word(dev, "prefill")
    L.prefill_grouped(bank, x2d, pr, bl, out, sc, st, out_row=orow)
    code = int(st.item())           # one sync per prefill call
    if code == 0:
        return out
    st.zero_()
    if code != L.SLX_ERR_RANGE:
        raise L.SlxError("slx_prefill_grouped", code, "device-side error")
    # an operand outside the tensor-core kernel's exact fp16 range: the
    # call runs on the GEMV kernels instead (fp32 scale/bias arithmetic)
    seg = np.repeat(np.asarray(slots, dtype=np.int32),
                    np.asarray(counts, dtype=np.int64))
    rows = torch.as_tensor(np.asarray(pair_row, dtype=np.int64), device=dev)
    xs = x2d[rows].contiguous()
    sid = torch.as_tensor(seg, device=dev).reshape(-1, 1)
    y = switchglu(bank, xs, sid, 1, inter=bank.inter,
                  status=st).reshape(-1, H)
    code = int(st.item())
    if code != 0:
        st.zero_()
        raise L.SlxError("prefill (GEMV path)", code,
                         "an activation is outside the fp16 range (|x| >= "
                         "65504) of the expert kernels")
    dst = torch.as_tensor(np.asarray(out_row if out_row is not None
                                     else np.arange(P), dtype=np.int64),
                          device=dev)
    out[dst] = y
    return out


def _status_word(device, tag: str) -> torch.Tensor:
    key = ("status", tag, device)
    t = _scratch.get(key)
    if t is None:
        t = torch.zeros(1, dtype=torch.int32, device=device)
        _scratch[key] = t
    return t


# ------------------------------------------------------- batched decode --
#
# One step of a batch of requests over a paged KV cache: paged_plan (pages
# and rows) -> per layer paged_append and paged_attention -> process_logits.
# Every call runs on the current stream of its tensors' device, allocates
# only what it returns, and does not synchronise; conditions found on the
# device go to the status word (check_status).

PAGE_SIZES = (16, 32, 64, 128, 256)


class PagedPlan(NamedTuple):
    """One step's rows and the state after it (int32, on the device)."""
    req: torch.Tensor       # [n_rows] request of each row, -1: padding
    pos: torch.Tensor       # [n_rows] its position in the request
    slot: torch.Tensor      # [n_rows] page * page_size + offset
    start: torch.Tensor     # [n_req + 1] first row of each request
    lengths: torch.Tensor   # [n_req] tokens held after the step
    n_free: torch.Tensor    # [1] free pages after it


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _ints(t, n: int, device, name: str) -> None:
    if (t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != n or
            t.device != device or not t.is_contiguous()):
        raise ValueError(f"{name}: contiguous int32 [{n}] on {device} wanted, "
                         f"got {t.dtype} {list(t.shape)} on {t.device}")


def _floats(t, n: int, device, name: str) -> None:
    if (t.dtype != torch.float32 or t.dim() != 1 or t.shape[0] != n or
            t.device != device or not t.is_contiguous()):
        raise ValueError(f"{name}: contiguous float32 [{n}] on {device} "
                         f"wanted, got {t.dtype} {list(t.shape)} on {t.device}")


def _raw_stream(device) -> int:
    """Current stream of a device, as the C ABI takes it."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def _call_status(device) -> torch.Tensor:
    """The device's status word; inside a capture that comes before its
    first use, one of the graph's own (the shared word must not be born in a
    graph's memory, where every replay would clear it)."""
    t = _scratch.get(("status", device))
    if t is not None:
        return t
    if torch.cuda.is_current_stream_capturing():
        return torch.zeros(1, dtype=torch.int32, device=device)
    return _status(device)


def _pages_of(pages: torch.Tensor, kv_scale, name: str) -> "L.slx_kv_pages":
    _need(pages.is_cuda and pages.dim() == 5 and pages.shape[1] == 2 and
          pages.is_contiguous(),
          f"{name}: pages must be contiguous [n_pages, 2, n_kv, page_size, "
          "head_dim] on a CUDA device")
    if pages.dtype == torch.bfloat16:
        _need(kv_scale is None, f"{name}: bf16 pages take no kv_scale")
    elif pages.dtype == torch.float8_e4m3fn:
        n_kv = pages.shape[2]
        _need(kv_scale is not None and kv_scale.dtype == torch.float32 and
              list(kv_scale.shape) == [2, n_kv] and
              kv_scale.device == pages.device and kv_scale.is_contiguous(),
              f"{name}: e4m3 pages need kv_scale, float32 [2, {n_kv}] (keys, "
              "values) on their device")
    else:
        raise ValueError(f"{name}: pages are bfloat16 or float8_e4m3fn, got "
                         f"{pages.dtype}")
    return L.kv_pages(pages, kv_scale)


def paged_plan(n_new: torch.Tensor, lengths: torch.Tensor,
               table: torch.Tensor, free_list: torch.Tensor,
               n_free: torch.Tensor, page_size: int, n_rows: int, *,
               lengths_out: torch.Tensor | None = None,
               n_free_out: torch.Tensor | None = None,
               status: torch.Tensor | None = None) -> PagedPlan:
    """Block tables and slot maps of one step, on the GPU
    (``slx_paged_plan``): request i gets ``n_new[i]`` new rows (-1: it is
    finished and its pages go back to the free stack) and the pages they
    need.  ``table`` [n_req, max_pages] and ``free_list`` [n_pages] are
    updated; ``lengths_out`` / ``n_free_out`` may be ``lengths`` /
    ``n_free`` themselves.  When pages or rows do not suffice nothing
    changes, every row is padding and the status word says SLX_ERR_PAGES."""
    dev = table.device
    _need(table.is_cuda and table.dim() == 2 and table.dtype == torch.int32
          and table.is_contiguous(),
          "paged_plan: table must be contiguous int32 [n_req, max_pages] on a "
          "CUDA device")
    if dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return paged_plan(n_new, lengths, table, free_list, n_free,
                              page_size, n_rows, lengths_out=lengths_out,
                              n_free_out=n_free_out, status=status)
    R = table.shape[0]
    _need(page_size in PAGE_SIZES, f"paged_plan: page_size {page_size}")
    _need(n_rows >= 0, f"paged_plan: n_rows {n_rows}")
    _ints(n_new, R, dev, "paged_plan: n_new")
    _ints(lengths, R, dev, "paged_plan: lengths")
    _ints(free_list, free_list.numel(), dev, "paged_plan: free_list")
    _ints(n_free, 1, dev, "paged_plan: n_free")
    rows = torch.empty(3, n_rows, dtype=torch.int32, device=dev)
    start = torch.empty(R + 1, dtype=torch.int32, device=dev)
    if lengths_out is None:
        lengths_out = torch.empty_like(lengths)
    else:
        _ints(lengths_out, R, dev, "paged_plan: lengths_out")
    if n_free_out is None:
        n_free_out = torch.empty_like(n_free)
    else:
        _ints(n_free_out, 1, dev, "paged_plan: n_free_out")
    req, pos, slot = rows.unbind(0)
    L.paged_plan(n_new, lengths, lengths_out, table, page_size, free_list,
                 n_free, n_free_out, req, pos, slot, start,
                 _call_status(dev) if status is None else status,
                 _raw_stream(dev))
    return PagedPlan(req, pos, slot, start, lengths_out, n_free_out)


def paged_append(qkv: torch.Tensor, pages: torch.Tensor, slot: torch.Tensor,
                 pos: torch.Tensor, n_q: int, q_norm: torch.Tensor,
                 k_norm: torch.Tensor, eps: float, inv_freq: torch.Tensor, *,
                 kv_scale: torch.Tensor | None = None,
                 q_out: torch.Tensor | None = None,
                 status: torch.Tensor | None = None) -> torch.Tensor:
    """q/k RMSNorm, RoPE and append to the pages (``slx_paged_append``):
    qkv [T, (n_q + 2 n_kv) * head_dim] bf16 (rows may be strided); returns
    the rotated queries [T, n_q, head_dim].  Rows with slot or pos < 0 give
    zero queries and write no page."""
    dev = pages.device
    kv = _pages_of(pages, kv_scale, "paged_append")
    if dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return paged_append(qkv, pages, slot, pos, n_q, q_norm, k_norm,
                                eps, inv_freq, kv_scale=kv_scale, q_out=q_out,
                                status=status)
    T, hd = qkv.shape[0], pages.shape[4]
    _need(qkv.dtype == torch.bfloat16 and qkv.dim() == 2 and
          qkv.device == dev and
          qkv.shape[1] == (n_q + 2 * pages.shape[2]) * hd and
          qkv.stride(1) == 1,
          "paged_append: qkv must be bfloat16 [T, (n_q + 2 n_kv) * head_dim] "
          "on the pages' device")
    _ints(slot, T, dev, "paged_append: slot")
    _ints(pos, T, dev, "paged_append: pos")
    for w, name in ((q_norm, "q_norm"), (k_norm, "k_norm")):
        _need(w.dtype == torch.bfloat16 and w.numel() == hd and
              w.device == dev and w.is_contiguous(),
              f"paged_append: {name} must be bfloat16 [{hd}]")
    _floats(inv_freq, hd // 2, dev, "paged_append: inv_freq")
    if q_out is None:
        q_out = torch.empty(T, n_q, hd, dtype=torch.bfloat16, device=dev)
    else:
        _need(q_out.dtype == torch.bfloat16 and q_out.device == dev and
              q_out.numel() == T * n_q * hd and q_out.is_contiguous(),
              "paged_append: q_out must be contiguous bfloat16 [T, n_q, "
              "head_dim]")
    L.paged_append(qkv, kv, slot, pos, n_q, q_norm, k_norm, eps, inv_freq,
                   q_out, _call_status(dev) if status is None else status,
                   _raw_stream(dev))
    return q_out


def paged_workspace(rows: int, n_q: int, n_kv: int, head_dim: int,
                    device) -> torch.Tensor:
    """Workspace of paged_attention for up to ``rows`` rows, for callers
    that must not allocate per call.  Its content does not matter; calls that
    may overlap (streams, graphs) need one each."""
    n = L.paged_attn_workspace_bytes(rows, n_q, n_kv, head_dim)
    return torch.empty(max(n, 16), dtype=torch.uint8, device=device)


def paged_attention(q: torch.Tensor, pages: torch.Tensor,
                    table: torch.Tensor, pos: torch.Tensor, *,
                    req: torch.Tensor | None = None,
                    scale: float | None = None,
                    kv_scale: torch.Tensor | None = None,
                    out: torch.Tensor | None = None,
                    workspace: torch.Tensor | None = None,
                    status: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of new tokens over a paged cache
    (``slx_paged_attn_decode``): row t of q [T, n_q, head_dim] (rows may be
    strided) attends positions 0..pos[t] of request req[t] (default: t);
    pos[t] < 0 gives zeros.  Returns [T, n_q, head_dim] bf16."""
    dev = pages.device
    kv = _pages_of(pages, kv_scale, "paged_attention")
    if dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return paged_attention(q, pages, table, pos, req=req, scale=scale,
                                   kv_scale=kv_scale, out=out,
                                   workspace=workspace, status=status)
    hd = pages.shape[4]
    _need(q.dim() == 3 and q.dtype == torch.bfloat16 and q.device == dev and
          q.shape[2] == hd and q.stride(2) == 1 and
          (q.stride(1) == hd or q.shape[1] == 1),
          "paged_attention: q must be bfloat16 [T, n_q, head_dim] with "
          "adjacent heads, on the pages' device")
    T, n_q = q.shape[0], q.shape[1]
    _need(table.dim() == 2 and table.dtype == torch.int32 and
          table.device == dev and table.is_contiguous(),
          "paged_attention: table must be contiguous int32 [n_req, max_pages]")
    _ints(pos, T, dev, "paged_attention: pos")
    if req is not None:
        _ints(req, T, dev, "paged_attention: req")
    if scale is None:
        scale = hd ** -0.5
    if out is None:
        out = torch.empty(T, n_q, hd, dtype=torch.bfloat16, device=dev)
    else:
        _need(out.dtype == torch.bfloat16 and out.device == dev and
              out.numel() == T * n_q * hd and out.is_contiguous(),
              "paged_attention: out must be contiguous bfloat16 [T, n_q, "
              "head_dim]")
    if workspace is None:
        # the call's own: calls on other streams or in graphs share nothing
        workspace = paged_workspace(T, n_q, pages.shape[2], hd, dev)
    else:
        _need(workspace.dtype == torch.uint8 and workspace.dim() == 1 and
              workspace.device == dev and workspace.is_contiguous(),
              "paged_attention: workspace must come from paged_workspace on "
              "the pages' device")
    L.paged_attn_decode(q, q.stride(0) if T > 1 else n_q * hd, n_q, kv, table,
                        req, pos, scale, out, workspace,
                        _call_status(dev) if status is None else status,
                        _raw_stream(dev))
    return out


def process_logits(logits: torch.Tensor, history: torch.Tensor | None = None,
                   n_prompt: torch.Tensor | None = None,
                   n_history: torch.Tensor | None = None, *,
                   repetition: torch.Tensor | None = None,
                   frequency: torch.Tensor | None = None,
                   presence: torch.Tensor | None = None,
                   bias: tuple | None = None,
                   mask: torch.Tensor | None = None,
                   out: torch.Tensor | None = None, pick=None,
                   status: torch.Tensor | None = None):
    """Penalties, biases and grammar mask on logits [T, V] (bf16 or fp32) and
    the greedy pick, in one launch (``slx_logits_process``).

    ``history`` int32 [T, max]: each row's prompt and output ids, of which
    the first ``n_history[t]`` count and the first ``n_prompt[t]`` are prompt;
    ``repetition`` / ``frequency`` / ``presence`` float32 [T]; ``bias``
    (ids, values, start): row t adds values[i] to ids[i] for i in
    start[t]..start[t + 1] (an id listed twice takes its last entry);
    ``mask`` int32 [T, >= ceil(V / 32)]: bit i of word w allows id 32 w + i.
    ``out`` (logits itself, or another tensor) receives the processed logits;
    None computes the pick alone.  Returns the picks (int32 [T], -1 where the
    mask allows nothing), written to ``pick`` if that is a tensor; None with
    ``pick=False``."""
    dev = logits.device
    _need(logits.is_cuda and logits.dim() == 2 and logits.is_contiguous() and
          logits.dtype in (torch.bfloat16, torch.float32),
          "process_logits: logits must be contiguous bfloat16 or float32 "
          "[T, V] on a CUDA device")
    if dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return process_logits(logits, history, n_prompt, n_history,
                                  repetition=repetition, frequency=frequency,
                                  presence=presence, bias=bias, mask=mask,
                                  out=out, pick=pick, status=status)
    T, V = logits.shape
    _need(pick is not False or out is not None,
          "process_logits: neither out nor pick wanted")
    r = L.slx_logit_rules()
    if history is not None:
        _need(history.dtype == torch.int32 and history.dim() == 2 and
              history.shape[0] == T and history.device == dev and
              history.is_contiguous() and n_history is not None,
              "process_logits: history must be contiguous int32 [T, max] "
              "with n_history")
        _ints(n_history, T, dev, "process_logits: n_history")
        if history.shape[1] > 0:
            r.history = history.data_ptr()
            r.history_stride = history.shape[1]
            r.n_history = n_history.data_ptr()
            if n_prompt is not None:
                _ints(n_prompt, T, dev, "process_logits: n_prompt")
                r.n_prompt = n_prompt.data_ptr()
            if repetition is not None:
                _floats(repetition, T, dev, "process_logits: repetition")
                r.repetition = repetition.data_ptr()
            if frequency is not None:
                _floats(frequency, T, dev, "process_logits: frequency")
                r.frequency = frequency.data_ptr()
            if presence is not None:
                _floats(presence, T, dev, "process_logits: presence")
                r.presence = presence.data_ptr()
    else:
        _need(repetition is None and frequency is None and presence is None
              and n_prompt is None and n_history is None,
              "process_logits: penalties need a history")
    if bias is not None:
        ids, vals, start = bias
        n = ids.numel()
        _ints(ids, n, dev, "process_logits: bias ids")
        _floats(vals, n, dev, "process_logits: bias values")
        _ints(start, T + 1, dev, "process_logits: bias start")
        if n > 0:
            r.bias_ids = ids.data_ptr()
            r.bias_values = vals.data_ptr()
            r.bias_start = start.data_ptr()
            r.n_bias = n
    if mask is not None:
        _need(mask.dtype == torch.int32 and mask.dim() == 2 and
              mask.shape[0] == T and mask.shape[1] >= (V + 31) // 32 and
              mask.device == dev and mask.is_contiguous(),
              "process_logits: mask must be contiguous int32 [T, >= "
              "ceil(V / 32)]")
        r.mask = mask.data_ptr()
        r.mask_stride = mask.shape[1]
    if out is not None:
        _need(out.dtype == logits.dtype and out.shape == logits.shape and
              out.device == dev and out.is_contiguous(),
              "process_logits: out must match logits")
    if pick is None:
        pick = torch.empty(T, dtype=torch.int32, device=dev)
    elif pick is False:
        pick = None
    else:
        _ints(pick, T, dev, "process_logits: pick")
    L.logits_process(logits, r, out, pick,
                     _call_status(dev) if status is None else status,
                     _raw_stream(dev))
    return pick
