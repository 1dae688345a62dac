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
from .lib import KhqLaunchError, check

# the structs of include/khq_b200.h, field by field ("@": native alignment)
_PLAN_ARGS = struct.Struct("@12PNq8i0q")
_PRESTEP_ARGS = struct.Struct("@11P17q7i2f0q")
_ATTN_ARGS = struct.Struct("@9P2N12qq10if0q")
_TYPES = {torch.float16: "fp16", torch.bfloat16: "bf16"}


def _launch(fn, name: str, packed: bytes, device: int) -> None:
    if torch.cuda.current_device() != device:
        with torch.cuda.device(device):
            rc = fn(packed, _lib.current_stream())
    else:
        rc = fn(packed, _lib.current_stream())
    if rc != 0:
        check(name, rc)


def _want(cond: bool, text: str) -> None:
    if not cond:
        raise ValueError(text)


def _ints(t: torch.Tensor, name: str, numel: Optional[int], device: int, dtype=torch.int32) -> int:
    if t.dtype is not dtype or t.get_device() != device or not t.is_contiguous() or (numel is not None and t.numel() != numel):
        raise ValueError(f"{name}: wants contiguous {dtype} on cuda:{device}" + (f" with {numel} entries" if numel is not None else "")
                         + f", got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _rows(t: torch.Tensor, name: str, heads: int, d: int, tokens: Optional[int], dtype, device: int):
    """(tokens, heads, d) with any strides over tokens and heads."""
    if t.dim() != 3 or t.shape[1] != heads or t.shape[2] != d or (tokens is not None and t.shape[0] != tokens) or t.dtype is not dtype or t.get_device() != device:
        raise ValueError(f"{name}: wants ({tokens if tokens is not None else 'tokens'}, {heads}, {d}) {dtype} on cuda:{device}, got {tuple(t.shape)} "
                         f"{t.dtype} on {t.device}")
    st = t.stride()
    if st[2] != 1:
        raise ValueError(f"{name}: the last dimension has to be contiguous, strides {st}")
    return t.data_ptr(), st[0], st[1]


def _cache(t: torch.Tensor, name: str, heads: int, d: int, page_size: int, pages: Optional[int], dtype, device: int):
    """(n_pages, page_size, heads, d) with any strides over the first three."""
    if (t.dim() != 4 or t.shape[1] != page_size or t.shape[2] != heads or t.shape[3] != d or (pages is not None and t.shape[0] != pages) or t.dtype is not dtype
            or t.get_device() != device):
        raise ValueError(f"{name}: wants ({pages if pages is not None else 'n_pages'}, {page_size}, {heads}, {d}) {dtype} on cuda:{device}, got "
                         f"{tuple(t.shape)} {t.dtype} on {t.device}")
    st = t.stride()
    if st[3] != 1:
        raise ValueError(f"{name}: the last dimension has to be contiguous, strides {st}")
    return t.data_ptr(), st[0], st[1], st[2]


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
        _want(device.type == "cuda", "PagedPlan: a CUDA device")
        self.device = device.index if device.index is not None else torch.cuda.current_device()
        self.max_requests, self.max_tokens, self.page_size = int(max_requests), int(max_tokens), int(page_size)
        self.H_q, self.H_kv, self.d = int(H_q), int(H_kv), int(d)
        self.max_new = min(int(max_new), self.max_tokens) if max_new is not None else self.max_tokens
        with torch.cuda.device(self.device):
            n = int(self.lib.khq_b200_paged_schedule_bytes(self.max_requests, self.max_tokens, self.max_new, self.H_q, self.H_kv))
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
        self.requests = self.max_pages = 0  # of the last build
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
        if (block_table.dim() != 2 or block_table.shape[0] != n or block_table.dtype is not torch.int32 or block_table.get_device() != dev
                or block_table.shape[1] < 1 or block_table.stride(1) != 1):
            raise ValueError(f"block_table: wants ({n}, max_pages) int32 on cuda:{dev} with contiguous rows, got {tuple(block_table.shape)} {block_table.dtype} "
                             f"on {block_table.device}")
        fl = fc = fo = n_pages = 0
        if free_list is not None:
            if free_count is None:
                raise ValueError("PagedPlan.build: free_list without free_count")
            n_pages = free_list.numel()
            fl, fc = _ints(free_list, "free_list", None, dev), _ints(free_count, "free_count", 1, dev)
            fo = fc if free_count_out is None else _ints(free_count_out, "free_count_out", 1, dev)
        elif free_count is not None or free_count_out is not None:
            raise ValueError("PagedPlan.build: free_count without free_list")
        max_pages = block_table.shape[1]
        cu, kv, pos, slots, info, sched = self._own
        packed = _PLAN_ARGS.pack(ctx, new, block_table.data_ptr(), fl, fc, fo, cu, kv, pos, slots, info, sched, self.schedule.numel(),
                                 block_table.stride(0) if n > 1 else max_pages, n, max_pages, n_pages, self.page_size, self.max_tokens, self.max_new,
                                 self.H_q, self.H_kv)
        _launch(self.lib.launch_khq_paged_plan, "launch_khq_paged_plan", packed, dev)
        self.requests, self.max_pages = n, max_pages
        return self


def paged_prestep(plan: PagedPlan, q, k, v, q_norm_w, k_norm_w, q_out, k_cache, v_cache, u_cache=None, rotary_dim: int = 64,
                  rope_theta: float = 1e7, rms_eps: float = 1e-6) -> None:
    """Head RMS norms of ``q`` and ``k`` (weights fp32 (d) or None), rotation of the first ``rotary_dim`` dims at the plan's positions; ``q``
    to ``q_out`` (which may be ``q``), rotated ``k``, ``v`` and, with ``u_cache``, un-rotated ``k`` to the plan's slots.  The
    counterpart of ``CudaOps.prestep`` for ragged rows and pages."""
    dev, H_q, H_kv, d, dt = plan.device, plan.H_q, plan.H_kv, plan.d, q.dtype
    if dt not in _TYPES:
        raise TypeError(f"paged_prestep: fp16 or bf16, got {dt}")
    T = q.shape[0]
    if not 0 < T <= plan.max_tokens:
        raise ValueError(f"paged_prestep: {T} rows, the plan is for 1 to {plan.max_tokens}")
    if plan.requests == 0:
        raise ValueError("paged_prestep: the plan has not been built")
    qp, q0, q1 = _rows(q, "q", H_q, d, T, dt, dev)
    kp, k0, k1 = _rows(k, "k", H_kv, d, T, dt, dev)
    vp, v0, v1 = _rows(v, "v", H_kv, d, T, dt, dev)
    op, o0, o1 = _rows(q_out, "q_out", H_q, d, T, dt, dev)
    P = plan.page_size
    kc, kc0, kc1, kc2 = _cache(k_cache, "k_cache", H_kv, d, P, None, dt, dev)
    n_pages = k_cache.shape[0]
    vc, vc0, vc1, vc2 = _cache(v_cache, "v_cache", H_kv, d, P, n_pages, dt, dev)
    uc, uc0, uc1, uc2 = _cache(u_cache, "u_cache", H_kv, d, P, n_pages, dt, dev) if u_cache is not None else (0, 0, 0, 0)
    qw = _ints(q_norm_w, "q_norm_w", d, dev, torch.float32) if q_norm_w is not None else 0
    kw = _ints(k_norm_w, "k_norm_w", d, dev, torch.float32) if k_norm_w is not None else 0
    packed = _PRESTEP_ARGS.pack(qp, kp, vp, qw, kw, op, kc, vc, uc, plan._own[2], plan._own[3], q0, q1, k0, k1, v0, v1, o0, o1, kc0, kc1, kc2,
                                vc0, vc1, vc2, uc0, uc1, uc2, T, n_pages, P, H_q, H_kv, d, int(rotary_dim), float(rope_theta), float(rms_eps))
    name = "launch_khq_paged_prestep_" + _TYPES[dt]
    _launch(getattr(plan.lib, name), name, packed, dev)


def paged_attention(plan: PagedPlan, q, k_cache, v_cache, block_table, out, scale: float, gate=None, lse=None, workspace=None) -> None:
    """Every row of ``q`` attends its request's positions up to its own, this step's tokens included (their K and V are in the cache: the
    pre-step has run).  ``out`` (tokens, H_q, d); ``gate`` (tokens, H_q, d): logits of the output gate, as in
    ``CudaOps.gqa_prefill``; ``lse`` (tokens, H_q) fp32: log of the sum of exponentials.  ``q`` and ``gate`` may be the two halves of an
    interleaved projection."""
    dev, H_q, H_kv, d, dt = plan.device, plan.H_q, plan.H_kv, plan.d, q.dtype
    if dt not in _TYPES:
        raise TypeError(f"paged_attention: fp16 or bf16, got {dt}")
    T = q.shape[0]
    if not 0 < T <= plan.max_tokens:
        raise ValueError(f"paged_attention: {T} rows, the plan is for 1 to {plan.max_tokens}")
    if plan.requests == 0:
        raise ValueError("paged_attention: the plan has not been built")
    qp, q0, q1 = _rows(q, "q", H_q, d, T, dt, dev)
    op, o0, o1 = _rows(out, "out", H_q, d, T, dt, dev)
    gp, g0, g1 = _rows(gate, "gate", H_q, d, T, dt, dev) if gate is not None else (0, 0, 0)
    P = plan.page_size
    kc, kc0, kc1, kc2 = _cache(k_cache, "k_cache", H_kv, d, P, None, dt, dev)
    n_pages = k_cache.shape[0]
    vc, vc0, vc1, vc2 = _cache(v_cache, "v_cache", H_kv, d, P, n_pages, dt, dev)
    if (block_table.dim() != 2 or block_table.shape[0] != plan.requests or block_table.shape[1] != plan.max_pages or block_table.dtype is not torch.int32
            or block_table.get_device() != dev or block_table.stride(1) != 1):
        raise ValueError(f"block_table: wants the plan's ({plan.requests}, {plan.max_pages}) int32 on cuda:{dev}, got {tuple(block_table.shape)} "
                         f"{block_table.dtype} on {block_table.device}")
    lp = _ints(lse, "lse", T * H_q, dev, torch.float32) if lse is not None else 0
    if workspace is None:
        workspace = plan.workspace
    ws = _ints(workspace, "workspace", None, dev, torch.uint8)
    packed = _ATTN_ARGS.pack(qp, gp, kc, vc, block_table.data_ptr(), plan._own[5], op, lp, ws, plan.schedule.numel(),
                             workspace.numel(), q0, q1, g0, g1, o0, o1, kc0, kc1, kc2, vc0, vc1, vc2,
                             block_table.stride(0) if plan.requests > 1 else plan.max_pages, T, plan.max_tokens, plan.max_new, plan.requests, plan.max_pages,
                             n_pages, P, H_q, H_kv, d, float(scale))
    name = "launch_khq_paged_attn_" + _TYPES[dt]
    _launch(getattr(plan.lib, name), name, packed, dev)
