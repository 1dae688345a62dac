"""Prompts in chunks over a raw paged K/V cache: the host side of ``launch_khq_paged_plan``, ``launch_khq_paged_prestep_*`` and
``launch_khq_paged_attn_*`` (include/khq_b200.h has the rules that all three keep).

The reference takes a prompt in chunks of up to 256 rows into one dense cache per layer (``main.mojo:1651-1734``).  Here the
raw K and V of all requests of a server share a pool of pages until a prompt is complete.  A step is

    plan.build(ctx_lens, new_lens, block_table, free_list, free_count)       # once, for all layers
    paged_prestep(plan, q, k, v, q_w, k_w, q, k_cache, v_cache, u_cache)     # per layer
    paged_attention(plan, q, k_cache, v_cache, block_table, out, scale, gate=gate)

with ragged ``q`` (tokens, H_q, d), ``k`` and ``v`` (tokens, H_kv, d), request by request in the order of the lengths, and
caches (n_pages, page_size, H_kv, d), fp16 or bf16.  Lengths, tables and slots stay on the device; nothing here waits for it or
allocates, so a step can be captured into a CUDA graph at its largest size and replayed with other lengths.

When a prompt is complete, ``KhqRuntime.khq_adopt_pages`` or ``BatchEngine.load_pages`` compresses its pages (fp16, K un-rotated from ``u_cache``)
and the sequence goes on in code words.
"""
from __future__ import annotations

import struct
from typing import Optional

import torch

from . import lib as _lib
from .lib import check

# the structs of include/khq_b200.h, field by field ("@": native alignment)
_PLAN_ARGS = struct.Struct("@12PNq9i0q")
_PRESTEP_ARGS = struct.Struct("@11P17q7i2f0q")
_ATTN_ARGS = struct.Struct("@9P2N12qq10if0q")
_TYPES = {torch.float16: "fp16", torch.bfloat16: "bf16"}


# A step's host time is mostly the look at its tensors (some 0.1 us per property): each is asked for what it is checked by once.


def _launch(fn, name: str, packed: bytes, device: int) -> None:
    if _current_device() != device:
        with torch.cuda.device(device):
            rc = fn(packed, _current_stream(device))
    else:
        rc = fn(packed, _current_stream(device))
    if rc != 0:
        check(name, rc)


def _current_device() -> int:
    return torch._C._cuda_getDevice()


def _current_stream(device: int) -> int:
    return torch._C._cuda_getCurrentRawStream(device)


def _refuse(t, name: str, want, dtype, device: int):
    if t.get_device() != device or t.dtype is not dtype or len(t.shape) != len(want) or any(w is not None and w != s for w, s in zip(want, t.shape)):
        shape = ", ".join("any" if w is None else str(w) for w in want)
        raise ValueError(f"{name}: wants ({shape}) {dtype} on cuda:{device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    raise ValueError(f"{name}: the last dimension has to be contiguous, strides {t.stride()}")


def _ints(t: torch.Tensor, name: str, numel: Optional[int], device: int, dtype=torch.int32) -> int:
    if t.dtype is not dtype or t.get_device() != device or not t.is_contiguous() or (numel is not None and t.numel() != numel):
        raise ValueError(f"{name}: wants contiguous {dtype} on cuda:{device}" + (f" with {numel} entries" if numel is not None else "")
                         + f", got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _rows(t: torch.Tensor, name: str, heads: int, d: int, tokens: int, dtype, device: int):
    """(tokens, heads, d) with any strides over tokens and heads."""
    st = t.stride()
    if t.shape != (tokens, heads, d) or st[2] != 1 or t.dtype is not dtype or t.get_device() != device:
        _refuse(t, name, (tokens, heads, d), dtype, device)
    return t.data_ptr(), st[0], st[1]


def _cache(t: torch.Tensor, name: str, shape, dtype, device: int):
    """(n_pages, page_size, heads, d) with any strides over the first three."""
    st = t.stride()
    if t.shape != shape or st[3] != 1 or t.dtype is not dtype or t.get_device() != device:
        _refuse(t, name, shape, dtype, device)
    return t.data_ptr(), st[0], st[1], st[2]


def _pages_of(t: torch.Tensor, page_size: int, heads: int, d: int):
    """The shape that a cache with as many pages as this one has."""
    return (t.shape[0] if t.dim() == 4 else None, page_size, heads, d)


class PagedPlan:
    """A step's ragged batch: who has how many new tokens, where they go, and what the attention runs from.

    Built for up to ``max_requests`` requests, ``max_tokens`` new tokens together and ``max_new`` of one request (default:
    ``max_tokens``).  ``max_new`` also says which attention kernel serves the step, so a plan of decode steps is given its 1.
    After ``build`` (device tensors, rewritten by the next one): ``cu_new`` (requests + 1), ``kv_lens`` (requests),
    ``positions`` and ``slots`` (max_tokens; -1 behind the last token), ``info`` (tokens, pages taken, pages given back, pages missing,
    tokens dropped, pages free, 0, 0).

    The attention's scratch memory belongs to the plan, so its calls belong on one stream; ``new_workspace`` makes scratch for another."""

    def __init__(self, max_requests: int, max_tokens: int, page_size: int, H_q: int, H_kv: int, d: int, max_new: Optional[int] = None, device="cuda"):
        self.lib = _lib.load()
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError(f"PagedPlan: a CUDA device, got {device}")
        self.device = device.index if device.index is not None else torch.cuda.current_device()
        self.max_requests, self.max_tokens, self.page_size = int(max_requests), int(max_tokens), int(page_size)
        self.H_q, self.H_kv, self.d = int(H_q), int(H_kv), int(d)
        self.max_new = min(int(max_new), self.max_tokens) if max_new is not None else self.max_tokens
        with torch.cuda.device(self.device):
            n = int(self.lib.khq_b200_paged_schedule_bytes(self.max_requests, self.max_tokens, self.max_new, self.H_q, self.H_kv, self.d))
            w = int(self.lib.khq_b200_paged_workspace_bytes(self.max_new, self.H_q, self.H_kv, self.d))
        if n == 0 or w == 0 or self.page_size not in (16, 32, 64, 128):
            raise ValueError(f"PagedPlan: max_requests={max_requests} max_tokens={max_tokens} max_new={max_new} page_size={page_size} H_q={H_q} H_kv={H_kv} d={d} "
                             "is not supported (page_size 16, 32, 64 or 128; d 128 or 256; H_q a multiple of H_kv)")
        empty = lambda count, dt: torch.empty(count, dtype=dt, device=torch.device("cuda", self.device))
        self._cu_new, self._kv_lens = empty(self.max_requests + 1, torch.int32), empty(self.max_requests, torch.int32)
        self.positions, self.slots = empty(self.max_tokens, torch.int32), empty(self.max_tokens, torch.int64)
        self.info = torch.zeros(8, dtype=torch.int32, device=self.positions.device)
        self.schedule, self._workspace_bytes = empty(n, torch.uint8), w
        self.workspace = self.new_workspace()
        self._scratch, self._schedule_bytes = (self.workspace.data_ptr(), w), n
        self.requests = self.max_pages = 0  # of the last build
        self._fns = {dt: (getattr(self.lib, "launch_khq_paged_prestep_" + t), getattr(self.lib, "launch_khq_paged_attn_" + t)) for dt, t in _TYPES.items()}
        self._own = (self._cu_new.data_ptr(), self._kv_lens.data_ptr(), self.positions.data_ptr(), self.slots.data_ptr(), self.info.data_ptr(),
                     self.schedule.data_ptr())

    def new_workspace(self) -> torch.Tensor:
        """Scratch memory for ``paged_attention`` calls that may run beside those with the plan's own."""
        return torch.empty(self._workspace_bytes, dtype=torch.uint8, device=self.positions.device)

    @property
    def cu_new(self) -> torch.Tensor:
        return self._cu_new[:self.requests + 1]

    @property
    def kv_lens(self) -> torch.Tensor:
        return self._kv_lens[:self.requests]

    def build(self, ctx_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor, free_list: Optional[torch.Tensor] = None,
              free_count: Optional[torch.Tensor] = None, free_count_out: Optional[torch.Tensor] = None) -> "PagedPlan":
        """``ctx_lens`` / ``new_lens`` (requests) int32: tokens in the cache and tokens to come, -1: the request has ended.
        ``block_table`` (requests, max_pages) int32.  With ``free_list`` (n_pages) and ``free_count`` (1) int32 the pages of the new
        tokens are taken from it and entered in the table, and those of ended requests go back; ``free_count`` is brought up
        to date, or left as it is and the new count written to ``free_count_out``.  Without, the table has all pages already."""
        dev, n = self.device, ctx_lens.numel()
        if not 0 < n <= self.max_requests:
            raise ValueError(f"PagedPlan.build: {n} requests, built for 1 to {self.max_requests}")
        ctx, new = _ints(ctx_lens, "ctx_lens", n, dev), _ints(new_lens, "new_lens", n, dev)
        st, shape = block_table.stride(), block_table.shape
        if len(shape) != 2 or shape[0] != n or shape[1] < 1 or st[1] != 1 or block_table.dtype is not torch.int32 or block_table.get_device() != dev:
            _refuse(block_table, "block_table", (n, None), torch.int32, dev)
        fl = fc = fo = n_pages = 0
        if free_list is not None:
            if free_count is None:
                raise ValueError("PagedPlan.build: free_list without free_count")
            n_pages = free_list.numel()
            fl, fc = _ints(free_list, "free_list", None, dev), _ints(free_count, "free_count", 1, dev)
            fo = fc if free_count_out is None else _ints(free_count_out, "free_count_out", 1, dev)
        elif free_count is not None or free_count_out is not None:
            raise ValueError("PagedPlan.build: free_count without free_list")
        max_pages = shape[1]
        packed = _PLAN_ARGS.pack(ctx, new, block_table.data_ptr(), fl, fc, fo, *self._own, self._schedule_bytes, st[0] if n > 1 else max_pages, n, max_pages,
                                 n_pages, self.page_size, self.max_tokens, self.max_new, self.H_q, self.H_kv, self.d)
        _launch(self.lib.launch_khq_paged_plan, "launch_khq_paged_plan", packed, dev)
        self.requests, self.max_pages = n, max_pages
        return self


def paged_prestep(plan: PagedPlan, q, k, v, q_norm_w, k_norm_w, q_out, k_cache, v_cache, u_cache=None, rotary_dim: int = 64,
                  rope_theta: float = 1e7, rms_eps: float = 1e-6) -> None:
    """Head RMS norms of ``q`` and ``k`` (weights fp32 (d) or None), rotation of the first ``rotary_dim`` dims at the plan's positions; ``q``
    to ``q_out`` (which may be ``q``), rotated ``k``, ``v`` and, with ``u_cache``, un-rotated ``k`` to the plan's slots.  The
    counterpart of ``CudaOps.prestep`` for ragged rows and pages."""
    dev, H_q, H_kv, d, P, dt = plan.device, plan.H_q, plan.H_kv, plan.d, plan.page_size, q.dtype
    fns = plan._fns.get(dt)
    if fns is None:
        raise TypeError(f"paged_prestep: fp16 or bf16, got {dt}")
    T = q.shape[0]
    if not 0 < T <= plan.max_tokens:
        raise ValueError(f"paged_prestep: {T} rows, the plan is for 1 to {plan.max_tokens}")
    if plan.requests == 0:
        raise ValueError("paged_prestep: the plan has not been built")
    cache = _pages_of(k_cache, P, H_kv, d)
    packed = _PRESTEP_ARGS.pack(*_prestep_pointers(plan, q, k, v, q_norm_w, k_norm_w, q_out, k_cache, v_cache, u_cache, T, cache, dt, dev), T, cache[0], P,
                                H_q, H_kv, d, rotary_dim, rope_theta, rms_eps)
    _launch(fns[0], "launch_khq_paged_prestep_" + _TYPES[dt], packed, dev)


def _prestep_pointers(plan, q, k, v, q_norm_w, k_norm_w, q_out, k_cache, v_cache, u_cache, T, cache, dt, dev):
    H_q, H_kv, d = plan.H_q, plan.H_kv, plan.d
    qp, q0, q1 = _rows(q, "q", H_q, d, T, dt, dev)
    kp, k0, k1 = _rows(k, "k", H_kv, d, T, dt, dev)
    vp, v0, v1 = _rows(v, "v", H_kv, d, T, dt, dev)
    op, o0, o1 = _rows(q_out, "q_out", H_q, d, T, dt, dev)
    kc, kc0, kc1, kc2 = _cache(k_cache, "k_cache", cache, dt, dev)
    vc, vc0, vc1, vc2 = _cache(v_cache, "v_cache", cache, dt, dev)
    uc, uc0, uc1, uc2 = _cache(u_cache, "u_cache", cache, dt, dev) if u_cache is not None else (0, 0, 0, 0)
    qw = _ints(q_norm_w, "q_norm_w", d, dev, torch.float32) if q_norm_w is not None else 0
    kw = _ints(k_norm_w, "k_norm_w", d, dev, torch.float32) if k_norm_w is not None else 0
    return (qp, kp, vp, qw, kw, op, kc, vc, uc, plan._own[2], plan._own[3], q0, q1, k0, k1, v0, v1, o0, o1, kc0, kc1, kc2, vc0, vc1, vc2, uc0, uc1, uc2)


def paged_attention(plan: PagedPlan, q, k_cache, v_cache, block_table, out, scale: float, gate=None, lse=None, workspace=None) -> None:
    """Every row of ``q`` attends its request's positions up to its own, this step's tokens included (their K and V are in the cache: the
    pre-step has run).  ``out`` (tokens, H_q, d); ``gate`` (tokens, H_q, d): logits of the output gate, as in
    ``CudaOps.gqa_prefill``; ``lse`` (tokens, H_q) fp32: log of the sum of exponentials.  ``q`` and ``gate`` may be the two halves of an
    interleaved projection."""
    dev, H_q, H_kv, d, P, dt = plan.device, plan.H_q, plan.H_kv, plan.d, plan.page_size, q.dtype
    fns = plan._fns.get(dt)
    if fns is None:
        raise TypeError(f"paged_attention: fp16 or bf16, got {dt}")
    T, B, M = q.shape[0], plan.requests, plan.max_pages
    if not 0 < T <= plan.max_tokens:
        raise ValueError(f"paged_attention: {T} rows, the plan is for 1 to {plan.max_tokens}")
    if B == 0:
        raise ValueError("paged_attention: the plan has not been built")
    qp, q0, q1 = _rows(q, "q", H_q, d, T, dt, dev)
    op, o0, o1 = _rows(out, "out", H_q, d, T, dt, dev)
    gp, g0, g1 = _rows(gate, "gate", H_q, d, T, dt, dev) if gate is not None else (0, 0, 0)
    cache = _pages_of(k_cache, P, H_kv, d)
    kc, kc0, kc1, kc2 = _cache(k_cache, "k_cache", cache, dt, dev)
    vc, vc0, vc1, vc2 = _cache(v_cache, "v_cache", cache, dt, dev)
    st = block_table.stride()
    if block_table.shape != (B, M) or st[1] != 1 or block_table.dtype is not torch.int32 or block_table.get_device() != dev:
        _refuse(block_table, "block_table (the plan's)", (B, M), torch.int32, dev)
    lp = _ints(lse, "lse", T * H_q, dev, torch.float32) if lse is not None else 0
    if workspace is None:
        ws, n_ws = plan._scratch
    else:
        ws, n_ws = _ints(workspace, "workspace", None, dev, torch.uint8), workspace.numel()
    packed = _ATTN_ARGS.pack(qp, gp, kc, vc, block_table.data_ptr(), plan._own[5], op, lp, ws, plan._schedule_bytes, n_ws, q0, q1, g0, g1, o0, o1,
                             kc0, kc1, kc2, vc0, vc1, vc2, st[0] if B > 1 else M, T, plan.max_tokens, plan.max_new, B, M, cache[0], P, H_q, H_kv, d, scale)
    _launch(fns[1], "launch_khq_paged_attn_" + _TYPES[dt], packed, dev)


# ---- a finished prompt: from pages to code words --------------------------------------------------------------------------------
def prompt_pages(block_row: torch.Tensor, tokens: int, k_cache, v_cache, u_cache, H_kv: int, d: int) -> torch.Tensor:
    """The pages of a prompt's ``tokens`` tokens as an int64 tensor, checked: fp16 caches of one shape with token-major pages (a page is a run of
    page_size * H_kv contiguous rows), ``u_cache`` and ``v_cache`` with the same distance between pages, page numbers inside the
    cache.  Waits for the device (the page numbers)."""
    shape = k_cache.shape
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache), ("u_cache", u_cache)):
        if c.shape != shape or c.dim() != 4 or c.shape[2:] != (H_kv, d) or c.dtype is not torch.float16 or c.device != block_row.device:
            raise ValueError(f"{name}: wants fp16 (n_pages, page_size, {H_kv}, {d}) on {block_row.device}, got {tuple(c.shape)} {c.dtype} on {c.device}")
        if c.stride()[1:] != (H_kv * d, d, 1) or c.data_ptr() & 15 or c.stride(0) & 7:
            raise ValueError(f"{name}: wants token-major pages on 16 bytes, strides {c.stride()}")
    if u_cache.stride(0) != v_cache.stride(0):
        raise ValueError(f"u_cache and v_cache: pages {u_cache.stride(0)} and {v_cache.stride(0)} apart")
    page_size = shape[1]
    if page_size not in (16, 32, 64, 128):
        raise ValueError(f"page_size {page_size}: 16, 32, 64 or 128")
    n = -(-int(tokens) // page_size)
    if block_row.dim() != 1 or block_row.dtype is not torch.int32 or block_row.numel() < n:
        raise ValueError(f"block_row: wants int32 with {n} pages or more for {tokens} tokens, got {tuple(block_row.shape)} {block_row.dtype}")
    pages = block_row[:n].long()
    if n and bool(((pages < 0) | (pages >= shape[0])).any()):
        raise ValueError("block_row: a page that is not in the cache")
    return pages


def page_runs(pages: torch.Tensor, tokens: int, u_cache, row0: int = 0) -> torch.Tensor:
    """The first ``tokens`` tokens (whole pages) of a prompt as runs for ``CudaOps.compress_runs``: K un-rotated, V at the byte distance of the caches."""
    _, page_size, H_kv, _ = u_cache.shape
    n = tokens // page_size
    at = u_cache.data_ptr() + pages[:n] * (u_cache.stride(0) * 2)
    return torch.stack((at, row0 + torch.arange(n, device=pages.device) * (page_size * H_kv)), 1)


def page_rows(pages: torch.Tensor, first: int, last: int, cache: torch.Tensor) -> torch.Tensor:
    """Rows ``first`` to ``last`` of a prompt from its pages, (last - first, H_kv * d)."""
    t = torch.arange(first, last, device=pages.device)
    return cache[pages[t // cache.shape[1]], t % cache.shape[1]].reshape(last - first, -1)
