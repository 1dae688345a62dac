"""Prompts in chunks over a raw paged K/V cache: the host side of ``launch_khq_paged_plan``, ``launch_khq_paged_prestep_*`` and
``launch_khq_paged_attn_*`` (include/khq_b200.h has the rules that all three keep).

The reference takes a prompt in chunks of up to 256 rows into one dense cache per layer (``main.mojo:1651-1734``).  Here the
raw K and V of all requests of a server share a pool of pages until a prompt is complete.  A step is

    plan.build(ctx_lens, new_lens, block_table, free_list, free_count)       # once, for all layers
    paged_prestep(plan, q, k, v, q_w, k_w, q, k_cache, v_cache, u_cache)     # per layer
    paged_attention(plan, q, k_cache, v_cache, block_table, out, scale, gate=gate)

with ragged ``q`` (tokens, H_q, d), ``k`` and ``v`` (tokens, H_kv, d), request by request in the order of the lengths, and
caches (n_pages, page_size, H_kv, d), fp16 or bf16.  Lengths, tables and slots stay on the device; nothing here waits for it or
allocates, so a step can be captured into a CUDA graph at its largest size and replayed with other lengths.  Where the host waits for a step's results anyway,
``plan.check()`` raises if a wait inside the attention's kernels has run out (they never hang).

When a prompt is complete, ``KhqRuntime.khq_adopt_pages`` or ``BatchEngine.load_pages`` compresses its pages (fp16, K un-rotated from ``u_cache``)
and the sequence goes on in code words; its later tokens go through the framework's other pre-step, whose angles are fp32 (``include/khq_b200.h`` has the
difference).  bf16 pages have no such way out: they, and single tokens over raw pages, are for callers who do not compress.
"""
from __future__ import annotations

import ctypes
import importlib.util
from typing import Optional

import torch

from . import build, lib as _lib
from .lib import KhqLaunchError, KhqLibraryError, check

_TYPES = {torch.float16: "fp16", torch.bfloat16: "bf16"}
_NO_FIT = -1000  # of the extension: a tensor is not what the plan asks for


class _PlanInfo(ctypes.Structure):
    """``PlanInfo`` of csrc/khq_paged_host.cpp."""

    _fields_ = [(n, ctypes.c_int64) for n in ("device", "H_q", "H_kv", "d", "page_size", "max_requests", "max_tokens", "max_new", "requests", "max_pages")] + [
        (n, ctypes.c_void_p) for n in ("cu_new", "kv_lens", "positions", "slots", "info", "schedule", "workspace")] + [
        (n, ctypes.c_int64) for n in ("schedule_bytes", "workspace_bytes")] + [
        (n, ctypes.c_void_p) for n in ("launch_plan", "launch_prestep_fp16", "launch_prestep_bf16", "launch_attn_fp16", "launch_attn_bf16")]


_host = None


def _load_host():
    """The extension that looks at a call's tensors and launches (csrc/khq_paged_host.cpp)."""
    global _host
    if _host is None:
        path = build.host_path()
        try:
            spec = importlib.util.spec_from_file_location("_khq_paged_host", path)
            host = importlib.util.module_from_spec(spec)
        except ImportError as e:
            raise KhqLibraryError(f"the paged operators' extension cannot be loaded ({e}): build it for this torch and Python with "
                                  "`python -m bonsai_mojo_1bit_optimization_t4_cuda_b200.build`") from e
        if host.info_bytes() != ctypes.sizeof(_PlanInfo):
            raise KhqLibraryError("the paged operators' extension is stale: build it anew")
        _host = host
    return _host


# ---- waits that ran out ------------------------------------------------------------------------------------------------------
def _read_status(device) -> int:
    with torch.cuda.device(device):
        torch.cuda.current_stream().synchronize()
        return int(_lib.load().khq_b200_paged_status())


def check_status(device=None) -> None:
    """Raises ``KhqLaunchError`` if a wait inside a ``paged_attention`` on ``device`` (None: the current one) has run out since the last look: the
    kernels then go on without data, and outputs since that look are not to be trusted.  Waits for the current stream, so it belongs where the host
    waits anyway, and not into a capture.  The word is the GPU's, shared by all plans on it, and is cleared."""
    st = _read_status(device)
    if st != 0:
        raise KhqLaunchError("paged_attention: outputs since the last look are not to be trusted, khq_b200_paged_status", st)


# ---- what does not fit, in words (a call comes here only when the extension has refused it) ------------------------------------------------
def _look(t, name: str, want, dtype, device: int, contiguous: bool = False) -> None:
    """``want``: the shape, None for any size."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: a tensor, got {type(t).__name__}")
    shape = tuple(t.shape)
    if t.get_device() != device or t.dtype is not dtype or len(shape) != len(want) or any(w is not None and w != s for w, s in zip(want, shape)):
        text = ", ".join("any" if w is None else str(w) for w in want)
        raise ValueError(f"{name}: wants ({text}) {dtype} on cuda:{device}, got {shape} {t.dtype} on {t.device}")
    if t.stride(-1) != 1 or (contiguous and not t.is_contiguous()):
        raise ValueError(f"{name}: {'has to be contiguous' if contiguous else 'the last dimension has to be contiguous'}, strides {t.stride()}")


def _look_flat(t, name: str, numel: Optional[int], dtype, device: int) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: a tensor, got {type(t).__name__}")
    if t.dtype is not dtype or t.get_device() != device or not t.is_contiguous() or (numel is not None and t.numel() != numel):
        raise ValueError(f"{name}: wants contiguous {dtype} on cuda:{device}" + (f" with {numel} entries" if numel is not None else "")
                         + f", got {t.dtype} {tuple(t.shape)} on {t.device}")


def _look_step(plan: "PagedPlan", what: str, q) -> int:
    if not isinstance(q, torch.Tensor):
        raise TypeError(f"{what}: q: a tensor, got {type(q).__name__}")
    if q.dtype not in _TYPES:
        raise TypeError(f"{what}: fp16 or bf16, got {q.dtype}")
    T = q.shape[0] if q.dim() else 0
    if not 0 < T <= plan.max_tokens:
        raise ValueError(f"{what}: {T} rows, the plan is for 1 to {plan.max_tokens}")
    if plan.requests == 0:
        raise ValueError(f"{what}: the plan has not been built")
    return T


def _look_caches(plan: "PagedPlan", dtype, **caches) -> None:
    pages = None
    for name, c in caches.items():
        if c is not None:
            _look(c, name, (pages, plan.page_size, plan.H_kv, plan.d), dtype, plan.device)
            pages = c.shape[0]


class PagedPlan:
    """A step's ragged batch: who has how many new tokens, where they go, and what the attention runs from.

    Built for up to ``max_requests`` requests, ``max_tokens`` new tokens together and ``max_new`` of one request (default:
    ``max_tokens``).  ``max_new`` also says which attention kernel serves the step, so a plan of decode steps is given its 1.
    After ``build`` (device tensors, rewritten by the next one): ``cu_new`` (requests + 1), ``kv_lens`` (requests),
    ``positions`` and ``slots`` (max_tokens; -1 behind the last token), ``info`` (tokens, pages taken, pages given back, pages missing,
    tokens dropped, pages free, 0, 0; the pages' words are 0 without a free list).

    The attention's scratch memory belongs to the plan, so its calls belong on one stream; ``new_workspace`` makes scratch for another.
    The plan's tensors are, like any, the stream's that is current when it is made: a plan that others use is kept until they are done."""

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
        self.info = empty(8, torch.int32)  # (filled here, a build on another stream could be overtaken by it)
        self.schedule, self._workspace_bytes = empty(n, torch.uint8), w
        self.workspace = self.new_workspace()
        fn = lambda name: ctypes.cast(getattr(self.lib, name), ctypes.c_void_p).value
        self._info = _PlanInfo(
            self.device, self.H_q, self.H_kv, self.d, self.page_size, self.max_requests, self.max_tokens, self.max_new, 0, 0, self._cu_new.data_ptr(),
            self._kv_lens.data_ptr(), self.positions.data_ptr(), self.slots.data_ptr(), self.info.data_ptr(), self.schedule.data_ptr(),
            self.workspace.data_ptr(), n, w, fn("launch_khq_paged_plan"), fn("launch_khq_paged_prestep_fp16"), fn("launch_khq_paged_prestep_bf16"),
            fn("launch_khq_paged_attn_fp16"), fn("launch_khq_paged_attn_bf16"))
        self._at = ctypes.addressof(self._info)
        host = _load_host()
        self._build, self._prestep, self._attention = host.build, host.prestep, host.attention

    @property
    def requests(self) -> int:
        """Of the last build (0: none yet)."""
        return self._info.requests

    @property
    def max_pages(self) -> int:
        return self._info.max_pages

    def new_workspace(self) -> torch.Tensor:
        """Scratch memory for ``paged_attention`` calls that may run beside those with the plan's own."""
        return torch.empty(self._workspace_bytes, dtype=torch.uint8, device=self.positions.device)

    @property
    def cu_new(self) -> torch.Tensor:
        return self._cu_new[:self.requests + 1]

    @property
    def kv_lens(self) -> torch.Tensor:
        return self._kv_lens[:self.requests]

    def check(self) -> None:
        """``check_status`` of the plan's GPU."""
        check_status(self.device)

    def build(self, ctx_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor, free_list: Optional[torch.Tensor] = None,
              free_count: Optional[torch.Tensor] = None, free_count_out: Optional[torch.Tensor] = None) -> "PagedPlan":
        """``ctx_lens`` / ``new_lens`` (requests) int32: tokens in the cache and tokens to come, -1: the request has ended.
        ``block_table`` (requests, max_pages) int32.  With ``free_list`` (n_pages) and ``free_count`` (1) int32 the pages of the new
        tokens are taken from it and entered in the table, and those of ended requests go back; ``free_count`` is brought up
        to date, or left as it is and the new count written to ``free_count_out``.  Without, the table has all pages already.

        Tokens beyond a request's table row, ``max_new`` or ``max_tokens`` are dropped, not moved elsewhere: ``info[4]`` counts them and
        ``cu_new`` has the rows that are left."""
        rc = self._build(self._at, ctx_lens, new_lens, block_table, free_list, free_count, free_count_out)
        if rc != 0:
            if rc == _NO_FIT:
                self._look_at_build(ctx_lens, new_lens, block_table, free_list, free_count, free_count_out)
            check("launch_khq_paged_plan", rc)
        return self

    def _look_at_build(self, ctx_lens, new_lens, block_table, free_list, free_count, free_count_out) -> None:
        if not isinstance(ctx_lens, torch.Tensor):
            raise TypeError(f"ctx_lens: a tensor, got {type(ctx_lens).__name__}")
        dev, n = self.device, ctx_lens.numel()
        if not 0 < n <= self.max_requests:
            raise ValueError(f"PagedPlan.build: {n} requests, built for 1 to {self.max_requests}")
        _look_flat(ctx_lens, "ctx_lens", n, torch.int32, dev)
        _look_flat(new_lens, "new_lens", n, torch.int32, dev)
        _look(block_table, "block_table", (n, None), torch.int32, dev)
        if block_table.shape[1] == 0:
            raise ValueError("block_table: has no columns")
        if free_list is None:
            if free_count is not None or free_count_out is not None:
                raise ValueError("PagedPlan.build: free_count without free_list")
            return
        if free_count is None:
            raise ValueError("PagedPlan.build: free_list without free_count")
        _look_flat(free_list, "free_list", None, torch.int32, dev)
        _look_flat(free_count, "free_count", 1, torch.int32, dev)
        if free_count_out is not None:
            _look_flat(free_count_out, "free_count_out", 1, torch.int32, dev)


def paged_prestep(plan: PagedPlan, q, k, v, q_norm_w, k_norm_w, q_out, k_cache, v_cache, u_cache=None, rotary_dim: int = 64,
                  rope_theta: float = 1e7, rms_eps: float = 1e-6) -> None:
    """Head RMS norms of ``q`` and ``k`` (weights fp32 (d) or None), rotation of the first ``rotary_dim`` dims at the plan's positions; ``q``
    to ``q_out`` (which may be ``q``), rotated ``k``, ``v`` and, with ``u_cache``, un-rotated ``k`` to the plan's slots.  The
    counterpart of ``CudaOps.prestep`` for ragged rows and pages."""
    rc = plan._prestep(plan._at, q, k, v, q_norm_w, k_norm_w, q_out, k_cache, v_cache, u_cache, rotary_dim, rope_theta, rms_eps)
    if rc != 0:
        if rc == _NO_FIT:
            T, dt, dev = _look_step(plan, "paged_prestep", q), q.dtype, plan.device
            for name, t, heads in (("q", q, plan.H_q), ("k", k, plan.H_kv), ("v", v, plan.H_kv), ("q_out", q_out, plan.H_q)):
                _look(t, name, (T, heads, plan.d), dt, dev)
            _look_caches(plan, dt, k_cache=k_cache, v_cache=v_cache, u_cache=u_cache)
            for name, w in (("q_norm_w", q_norm_w), ("k_norm_w", k_norm_w)):
                if w is not None:
                    _look_flat(w, name, plan.d, torch.float32, dev)
        check("launch_khq_paged_prestep_" + _TYPES[q.dtype], rc)


def paged_attention(plan: PagedPlan, q, k_cache, v_cache, block_table, out, scale: float, gate=None, lse=None, workspace=None) -> None:
    """Every row of ``q`` attends its request's positions up to its own, this step's tokens included (their K and V are in the cache: the
    pre-step has run).  ``out`` (tokens, H_q, d); ``gate`` (tokens, H_q, d): logits of the output gate, as in
    ``CudaOps.gqa_prefill``; ``lse`` (tokens, H_q) fp32: log of the sum of exponentials.  ``q`` and ``gate`` may be the two halves of an
    interleaved projection."""
    rc = plan._attention(plan._at, q, k_cache, v_cache, block_table, out, scale, gate, lse, workspace)
    if rc != 0:
        if rc == _NO_FIT:
            T, dt, dev = _look_step(plan, "paged_attention", q), q.dtype, plan.device
            for name, t in (("q", q), ("out", out), ("gate", gate)):
                if t is not None:
                    _look(t, name, (T, plan.H_q, plan.d), dt, dev)
            _look_caches(plan, dt, k_cache=k_cache, v_cache=v_cache)
            _look(block_table, "block_table (the plan's)", (plan.requests, plan.max_pages), torch.int32, dev)
            if lse is not None:
                _look_flat(lse, "lse", T * plan.H_q, torch.float32, dev)
            if workspace is not None:
                _look_flat(workspace, "workspace", None, torch.uint8, dev)
        check("launch_khq_paged_attn_" + _TYPES[q.dtype], rc)


# ---- a finished prompt: from pages to code words --------------------------------------------------------------------------------
def prompt_pages(block_row: torch.Tensor, tokens: int, k_cache, v_cache, u_cache, H_kv: int, d: int, device: Optional[torch.device] = None) -> torch.Tensor:
    """The pages of a prompt's ``tokens`` tokens as an int64 tensor, checked: fp16 caches of one shape with token-major pages (a page is a run of
    page_size * H_kv contiguous rows), ``u_cache`` and ``v_cache`` with the same distance between pages, page numbers inside the
    cache, all on ``device`` (of the state that takes them; None: any GPU).  Waits for the device (the page numbers), and raises if a wait of the attention
    that the prompt went through may have run out (``check_status``)."""
    if block_row.device.type != "cuda" or (device is not None and block_row.device != device):
        raise ValueError(f"block_row: wants a tensor on {device or 'a CUDA device'}, got {block_row.device}")
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
    check_status(pages.device)
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
