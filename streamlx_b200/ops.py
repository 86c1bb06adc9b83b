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


_I32, _F32 = torch.int32, torch.float32
_BF16, _E4M3 = torch.bfloat16, torch.float8_e4m3fn
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_cur_device = getattr(torch._C, "_cuda_getDevice", None)


_status_words: dict = {}    # device index -> the word _status() keeps
_ws_bytes: dict = {}        # (n_q, n_kv, head_dim) -> bytes, T > 0


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _vec(t, n: int, dtype, idx: int, name: str) -> int:
    """Address of a contiguous vector [n] of a type on device idx."""
    if (t.dtype is not dtype or t.dim() != 1 or t.shape[0] != n or
            t.get_device() != idx or not t.is_contiguous()):
        raise ValueError(f"{name}: contiguous {dtype} [{n}] on cuda:{idx} "
                         f"wanted, got {t.dtype} {list(t.shape)} on {t.device}")
    return t.data_ptr()


def _call_status(status, idx: int) -> int:
    """Address of the call's status word: the given one, else the device's.
    A capture that comes before the device's first call has none unless it is
    given one (a word born in a graph's memory would be cleared by every
    replay): its device errors are not reported."""
    if status is not None:
        return _vec(status, 1, _I32, idx, "status")
    t = _status_words.get(idx)
    if t is None:
        if torch.cuda.is_current_stream_capturing():
            return 0
        t = _status_words[idx] = _status(torch.device("cuda", idx))
    return t.data_ptr()


def _pages_of(pages: torch.Tensor, kv_scale, name: str):
    """(slx_kv_pages as bytes, n_kv, head_dim) of a layer's pages."""
    shape = pages.shape
    if (len(shape) != 5 or shape[1] != 2 or not pages.is_cuda or
            not pages.is_contiguous()):
        raise ValueError(f"{name}: pages must be contiguous [n_pages, 2, n_kv, "
                         "page_size, head_dim] on a CUDA device")
    n, _, n_kv, ps, hd = shape
    if pages.dtype is _BF16:
        _need(kv_scale is None, f"{name}: bf16 pages take no kv_scale")
        return L.kv_pages(pages.data_ptr(), 0, n, n_kv, ps, hd), n_kv, hd
    if pages.dtype is not _E4M3:
        raise ValueError(f"{name}: pages are bfloat16 or float8_e4m3fn, got "
                         f"{pages.dtype}")
    if (kv_scale is None or kv_scale.dtype is not _F32 or
            kv_scale.shape != (2, n_kv) or not kv_scale.is_contiguous() or
            kv_scale.get_device() != pages.get_device()):
        raise ValueError(f"{name}: e4m3 pages need kv_scale, float32 [2, {n_kv}]"
                         " (keys, values) on their device")
    return (L.kv_pages(pages.data_ptr(), kv_scale.data_ptr(), n, n_kv, ps, hd),
            n_kv, hd)


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
    if (not table.is_cuda or table.dim() != 2 or table.dtype is not _I32 or
            not table.is_contiguous()):
        raise ValueError("paged_plan: table must be contiguous int32 [n_req, "
                         "max_pages] on a CUDA device")
    idx = table.get_device()
    if idx != _cur_device():
        with torch.cuda.device(idx):
            return paged_plan(n_new, lengths, table, free_list, n_free,
                              page_size, n_rows, lengths_out=lengths_out,
                              n_free_out=n_free_out, status=status)
    R, max_pages = table.shape
    n_pages = free_list.numel()
    _need(n_rows >= 0, f"paged_plan: n_rows {n_rows}")
    # rows (request, position, slot), their starts and the state after the
    # step, one allocation
    buf = torch.empty(3 * n_rows + 2 * R + 2, dtype=_I32, device=table.device)
    # (unsafe: integers, no autograd to track the parts for; 0.6 us less)
    req, pos, slot, start, ln, nf = torch.unsafe_split_with_sizes(
        buf, (n_rows, n_rows, n_rows, R + 1, R, 1))
    if lengths_out is None:
        lengths_out = ln
    if n_free_out is None:
        n_free_out = nf
    L.paged_plan(_vec(n_new, R, _I32, idx, "paged_plan: n_new"),
                 _vec(lengths, R, _I32, idx, "paged_plan: lengths"),
                 _vec(lengths_out, R, _I32, idx, "paged_plan: lengths_out"),
                 R, table.data_ptr(), max_pages, page_size,
                 _vec(free_list, n_pages, _I32, idx, "paged_plan: free_list"),
                 n_pages, _vec(n_free, 1, _I32, idx, "paged_plan: n_free"),
                 _vec(n_free_out, 1, _I32, idx, "paged_plan: n_free_out"),
                 buf.data_ptr(), n_rows, start.data_ptr(),
                 _call_status(status, idx), _raw_stream(idx))
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
    kv, n_kv, hd = _pages_of(pages, kv_scale, "paged_append")
    idx = pages.get_device()
    if idx != _cur_device():
        with torch.cuda.device(idx):
            return paged_append(qkv, pages, slot, pos, n_q, q_norm, k_norm,
                                eps, inv_freq, kv_scale=kv_scale, q_out=q_out,
                                status=status)
    if (qkv.dtype is not _BF16 or qkv.dim() != 2 or qkv.get_device() != idx or
            qkv.shape[1] != (n_q + 2 * n_kv) * hd or qkv.stride(1) != 1):
        raise ValueError("paged_append: qkv must be bfloat16 [T, (n_q + 2 n_kv)"
                         " * head_dim] on the pages' device")
    T = qkv.shape[0]
    if q_out is None:
        q_out = qkv.new_empty((T, n_q, hd))
    elif (q_out.dtype is not _BF16 or q_out.get_device() != idx or
          q_out.numel() != T * n_q * hd or not q_out.is_contiguous()):
        raise ValueError("paged_append: q_out must be contiguous bfloat16 [T, "
                         "n_q, head_dim]")
    L.paged_append(qkv.data_ptr(), qkv.stride(0) if T > 1 else qkv.shape[1], T,
                   n_q, _vec(q_norm, hd, _BF16, idx, "paged_append: q_norm"),
                   _vec(k_norm, hd, _BF16, idx, "paged_append: k_norm"), eps,
                   _vec(inv_freq, hd // 2, _F32, idx,
                        "paged_append: inv_freq"),
                   _vec(pos, T, _I32, idx, "paged_append: pos"),
                   _vec(slot, T, _I32, idx, "paged_append: slot"), kv,
                   q_out.data_ptr(), _call_status(status, idx),
                   _raw_stream(idx))
    return q_out


def paged_workspace(rows: int, n_q: int, n_kv: int, head_dim: int,
                    device) -> torch.Tensor:
    """Workspace of paged_attention for any number of rows up to ``rows``,
    for callers that must not allocate per call: the parts of the largest
    launch, about 10 MB with heads of 64 and 20 MB with heads of 128, however
    few the rows.  Its content does not matter; calls that may overlap
    (streams, graphs) need one each."""
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
    kv, n_kv, hd = _pages_of(pages, kv_scale, "paged_attention")
    idx = pages.get_device()
    if idx != _cur_device():
        with torch.cuda.device(idx):
            return paged_attention(q, pages, table, pos, req=req, scale=scale,
                                   kv_scale=kv_scale, out=out,
                                   workspace=workspace, status=status)
    shape, stride = q.shape, q.stride()
    if (len(shape) != 3 or q.dtype is not _BF16 or q.get_device() != idx or
            shape[2] != hd or stride[2] != 1 or
            (stride[1] != hd and shape[1] != 1)):
        raise ValueError("paged_attention: q must be bfloat16 [T, n_q, "
                         "head_dim] with adjacent heads, on the pages' device")
    T, n_q, _ = shape
    if (table.dim() != 2 or table.dtype is not _I32 or
            table.get_device() != idx or not table.is_contiguous()):
        raise ValueError("paged_attention: table must be contiguous int32 "
                         "[n_req, max_pages]")
    n_req, max_pages = table.shape
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(shape)
    elif (out.dtype is not _BF16 or out.get_device() != idx or
          out.numel() != T * n_q * hd or not out.is_contiguous()):
        raise ValueError("paged_attention: out must be contiguous bfloat16 [T, "
                         "n_q, head_dim]")
    if workspace is None:
        # the call's own: calls on other streams or in graphs share nothing
        need = _ws_bytes.get((n_q, n_kv, hd))
        if need is None:
            need = max(L.paged_attn_workspace_bytes(1, n_q, n_kv, hd), 16)
            _ws_bytes[n_q, n_kv, hd] = need
        workspace = q.new_empty(need, dtype=torch.uint8)
    elif (workspace.dtype is not torch.uint8 or workspace.dim() != 1 or
          workspace.get_device() != idx or not workspace.is_contiguous()):
        raise ValueError("paged_attention: workspace must come from "
                         "paged_workspace on the pages' device")
    L.paged_attn_decode(
        q.data_ptr(), stride[0] if T > 1 else n_q * hd, T, n_q, kv,
        table.data_ptr(), n_req, max_pages,
        None if req is None else _vec(req, T, _I32, idx,
                                      "paged_attention: req"),
        _vec(pos, T, _I32, idx, "paged_attention: pos"),
        hd ** -0.5 if scale is None else scale, out.data_ptr(),
        workspace.data_ptr(), workspace.shape[0], _call_status(status, idx),
        _raw_stream(idx))
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
    if (not logits.is_cuda or logits.dim() != 2 or
            not logits.is_contiguous() or
            logits.dtype not in (_BF16, _F32)):
        raise ValueError("process_logits: logits must be contiguous bfloat16 "
                         "or float32 [T, V] on a CUDA device")
    idx = logits.get_device()
    if idx != _cur_device():
        with torch.cuda.device(idx):
            return process_logits(logits, history, n_prompt, n_history,
                                  repetition=repetition, frequency=frequency,
                                  presence=presence, bias=bias, mask=mask,
                                  out=out, pick=pick, status=status)
    T, V = logits.shape
    _need(pick is not False or out is not None,
          "process_logits: neither out nor pick wanted")

    def vec(t, n, dtype, name):
        return 0 if t is None else _vec(t, n, dtype, idx,
                                        "process_logits: " + name)

    hist = stride = n_h = n_p = rep = freq = pres = 0
    if history is not None:
        if (history.dtype is not _I32 or history.dim() != 2 or
                history.shape[0] != T or history.get_device() != idx or
                not history.is_contiguous() or n_history is None):
            raise ValueError("process_logits: history must be contiguous int32 "
                             "[T, max] with n_history")
        n_h = vec(n_history, T, _I32, "n_history")
        n_p = vec(n_prompt, T, _I32, "n_prompt")
        rep = vec(repetition, T, _F32, "repetition")
        freq = vec(frequency, T, _F32, "frequency")
        pres = vec(presence, T, _F32, "presence")
        stride = history.shape[1]
        if stride > 0:
            hist = history.data_ptr()
        else:                       # nothing to count
            n_h = n_p = rep = freq = pres = 0
    else:
        _need(repetition is None and frequency is None and presence is None
              and n_prompt is None and n_history is None,
              "process_logits: penalties need a history")
    b_ids = b_vals = b_start = n_bias = 0
    if bias is not None:
        ids, vals, start = bias
        n_bias = ids.numel()
        b_ids = vec(ids, n_bias, _I32, "bias ids")
        b_vals = vec(vals, n_bias, _F32, "bias values")
        b_start = vec(start, T + 1, _I32, "bias start")
        if n_bias == 0:
            b_ids = b_vals = b_start = 0
    m = m_stride = 0
    if mask is not None:
        if (mask.dtype is not _I32 or mask.dim() != 2 or mask.shape[0] != T or
                mask.shape[1] * 32 < V or mask.get_device() != idx or
                not mask.is_contiguous()):
            raise ValueError("process_logits: mask must be contiguous int32 "
                             "[T, >= ceil(V / 32)]")
        m, m_stride = mask.data_ptr(), mask.shape[1]
    if out is not None and (out.dtype is not logits.dtype or
                            out.shape != logits.shape or
                            out.get_device() != idx or
                            not out.is_contiguous()):
        raise ValueError("process_logits: out must match logits")
    if pick is None:
        pick = logits.new_empty(T, dtype=_I32)
    elif pick is False:
        pick = None
    L.logits_process(
        logits.data_ptr(), logits.dtype is _F32, T, V,
        L.logit_rules(hist, n_p, n_h, rep, freq, pres, b_ids, b_vals, b_start,
                      m, stride, n_bias, m_stride),
        None if out is None else out.data_ptr(), vec(pick, T, _I32, "pick"),
        _call_status(status, idx), _raw_stream(idx))
    return pick
