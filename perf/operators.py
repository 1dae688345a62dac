"""A raw paged K/V cache for prompts that arrive in chunks: the plan of a step, the pre-step that fills the cache, and the
attention that reads it, as cases that can be timed and compared.

Kinds of case:

* ``plan``     one step's block tables, slots and positions from the lengths of the requests, pages taken from and given back
               to the free list (``paged.PagedPlan.build``).
* ``prestep``  head norms of q and k, partial rotation, and K, V and the un-rotated K into their slots (``paged.paged_prestep``).
* ``attention``  causal attention of each request's new tokens over everything it has in the cache, with the sigmoid gate
               (``paged.paged_attention``).

``own`` false: elementary torch operations in 32 bits (positions' angles in 64); true: the framework's kernels.  A pass leaves
the state as it found it, apart from the slots, table entries and outputs that every pass writes alike.
"""
import math
import random

import torch

own = False

GATED = 2      # a head's row in the projection: query, then gate logits
THETA = 1e7
EPS = 1e-6
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    model = dict(H_q=24, H_kv=4, d=256)
    return [
        # a full server's decode step: 256 sequences of 4k to 32k tokens, one new token each
        dict(name="plan_decode", kind="plan", page=128, requests=256, ctx_lo=4096, ctx_hi=32768, new_lo=1, new_hi=1, decodes=0, finished=0,
             lens=11, **model),
        # prompts in chunks of up to 256 tokens between sequences that decode, some of which have ended
        dict(name="plan_chunks", kind="plan", page=64, requests=16, ctx_lo=1, ctx_hi=6000, new_lo=100, new_hi=256, decodes=32, finished=5,
             lens=12, **model),
        # the largest step: thousands of ragged requests on small pages
        dict(name="plan_large", kind="plan", page=16, requests=2048, ctx_lo=1, ctx_hi=4000, new_lo=1, new_hi=128, decodes=1024, finished=100,
             lens=13, **model),
        # the token of a single sequence: latency
        dict(name="prestep_token", kind="prestep", dtype="fp16", page=128, requests=1, ctx_lo=4000, ctx_hi=4000, new_lo=1, new_hi=1, decodes=0,
             rotary=64, weights=True, unroped=True, lens=21, **model),
        # one token of each of 256 sequences far into their contexts
        dict(name="prestep_decode", kind="prestep", dtype="bf16", page=64, requests=256, ctx_lo=4096, ctx_hi=262144, new_lo=1, new_hi=1,
             decodes=0, rotary=64, weights=True, unroped=True, lens=22, **model),
        # chunks of four prompts, 8192 tokens together, K kept un-rotated too for the compression that follows
        dict(name="prestep_prompts", kind="prestep", dtype="fp16", page=128, requests=4, ctx_lo=1, ctx_hi=8192, new_lo=2048, new_hi=2048,
             decodes=0, rotary=64, weights=True, unroped=True, lens=23, **model),
        # the token of a single sequence, some thousand tokens in: latency
        dict(name="attention_token", kind="attention", dtype="fp16", page=128, requests=1, ctx_lo=4001, ctx_hi=4001, new_lo=1, new_hi=1,
             decodes=0, gate=True, lse=False, lens=31, **model),
        # a server with load: one token of each of 64 sequences of 4k to 32k tokens
        dict(name="attention_serve", kind="attention", dtype="fp16", page=128, requests=64, ctx_lo=4096, ctx_hi=32768, new_lo=1, new_hi=1,
             decodes=0, gate=True, lse=False, lens=32, **model),
        # five guessed tokens of each of 16 sequences checked at once, small heads, small pages
        dict(name="attention_guesses", kind="attention", dtype="bf16", page=16, requests=16, ctx_lo=500, ctx_hi=9000, new_lo=5, new_hi=5,
             decodes=0, gate=False, lse=True, lens=33, H_q=20, H_kv=4, d=128),
        # chunks of two prompts in one step with 40 sequences that decode
        dict(name="attention_mixed", kind="attention", dtype="bf16", page=64, requests=2, ctx_lo=300, ctx_hi=9000, new_lo=500, new_hi=1003,
             decodes=40, gate=True, lse=True, lens=34, **model),
        # a chunk of 2048 tokens of one long prompt
        dict(name="attention_chunk", kind="attention", dtype="bf16", page=128, requests=1, ctx_lo=24576, ctx_hi=24576, new_lo=2048, new_hi=2048,
             decodes=0, gate=True, lse=False, lens=35, **model),
        # four whole prompts of 8192 tokens
        dict(name="attention_prompts", kind="attention", dtype="fp16", page=128, requests=4, ctx_lo=0, ctx_hi=0, new_lo=8192, new_hi=8192,
             decodes=0, gate=True, lse=False, lens=36, **model),
    ]


def _log_int(rng, lo, hi):
    if lo >= hi:
        return lo
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(max(lo, 1)), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["plan", "prestep", "attention", "attention"])
    page = rng.choice([16, 32, 64, 128])
    H_q, H_kv, d = rng.choice([(24, 4, 256), (24, 4, 256), (20, 4, 256), (16, 16, 128), (32, 8, 128), (8, 1, 256), (20, 4, 128)])
    case = dict(kind=kind, page=page, H_q=H_q, H_kv=H_kv, d=d, lens=rng.randrange(1 << 30))
    if kind == "plan":
        decode = rng.random() < 0.4
        case.update(requests=_log_int(rng, 1, 2048), ctx_lo=0, ctx_hi=_log_int(rng, 1, 32768 * page // 128), new_lo=1,
                    new_hi=1 if decode else _log_int(rng, 2, 128), decodes=0 if decode else _log_int(rng, 1, 1024),
                    finished=_log_int(rng, 1, 100) - 1)
        return case
    case.update(dtype=rng.choice(["fp16", "bf16"]))
    if kind == "prestep":
        tokens = _log_int(rng, 1, 8192)
        requests = _log_int(rng, 1, tokens)
        case.update(requests=requests, ctx_lo=0, ctx_hi=_log_int(rng, 1, 262144), new_lo=max(1, tokens // requests // 2), new_hi=tokens // requests,
                    decodes=0, rotary=rng.choice([64, 64, 32, d]), weights=rng.random() < 0.8, unroped=rng.random() < 0.7)
        return case
    case.update(gate=rng.random() < 0.7, lse=rng.random() < 0.5)
    shape = rng.choice(["decode", "decode", "guesses", "mixed", "chunk", "prompts"])
    if shape == "decode":
        requests = _log_int(rng, 1, 64)
        hi = _log_int(rng, 16, 65536 if requests < 8 else 16384)
        case.update(requests=requests, ctx_lo=max(1, hi // 8), ctx_hi=hi, new_lo=1, new_hi=1, decodes=0)
    elif shape == "guesses":
        hi = _log_int(rng, 16, 16384)
        case.update(requests=_log_int(rng, 1, 48), ctx_lo=max(1, hi // 8), ctx_hi=hi, new_lo=2, new_hi=rng.randint(2, 40), decodes=0)
    elif shape == "mixed":
        case.update(requests=rng.randint(1, 4), ctx_lo=1, ctx_hi=_log_int(rng, 16, 16384), new_lo=33, new_hi=_log_int(rng, 64, 1500),
                    decodes=_log_int(rng, 1, 64))
    elif shape == "chunk":
        case.update(requests=1, ctx_lo=0, ctx_hi=_log_int(rng, 1, 32768), new_lo=200, new_hi=_log_int(rng, 256, 2500), decodes=0)
    else:
        hi = _log_int(rng, 100, 6000)
        case.update(requests=rng.randint(1, 6), ctx_lo=0, ctx_hi=0, new_lo=hi // 3, new_hi=hi, decodes=0)
    return case


# ---- lengths, tables ----------------------------------------------------------------------------------------------------------
def _lens(case):
    """(ctx, new) of every request; new == -1: the request has ended and gives its pages back."""
    rng = random.Random(case["lens"])
    rows = []
    for _ in range(case["requests"]):
        ctx = 0 if case["ctx_lo"] == 0 and rng.random() < 0.3 else _log_int(rng, case["ctx_lo"], case["ctx_hi"])
        rows.append((ctx, rng.randint(case["new_lo"], case["new_hi"])))
    for _ in range(case["decodes"]):
        rows.append((_log_int(rng, max(1, case["ctx_lo"]), max(1, case["ctx_hi"])), 1))
    for _ in range(case.get("finished", 0)):
        rows.append((_log_int(rng, 1, max(1, case["ctx_hi"])), -1))
    rng.shuffle(rows)
    return [c for c, _ in rows], [n for _, n in rows]


def _pages(n, page):
    return -(-n // page)


def _tables(ctx, new, page, gen, held_only):
    """A block table over a pool of shuffled pages, and the free list behind it; `held_only`: the pages of the new tokens are
    still to be taken."""
    counts = [_pages(c if held_only else c + max(n, 0), page) for c, n in zip(ctx, new)]
    after = [_pages(c + max(n, 0), page) for c, n in zip(ctx, new)]
    pool = sum(max(a, b) for a, b in zip(counts, after)) + 8
    order = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
    width = max(1, max(after + counts))
    n = torch.tensor(counts, device="cuda")
    at = torch.cumsum(n, 0) - n
    col = torch.arange(width, device="cuda")
    mine = col[None, :] < n[:, None]
    table = torch.where(mine, order[(at[:, None] + col[None, :]).clamp(max=pool - 1)], torch.full((), -1, dtype=torch.int32, device="cuda"))
    used = sum(counts)
    free = torch.cat([order[used:], torch.full((used,), -1, dtype=torch.int32, device="cuda")])
    return table.contiguous(), pool, free, torch.tensor([pool - used], dtype=torch.int32, device="cuda")


def _make_plan(case, s):
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.paged import PagedPlan

    return PagedPlan(len(s["ctx"]), s["tokens"], case["page"], case["H_q"], case["H_kv"], case["d"],
                     max_new=max(1, max(s["new"])))


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    ctx, new = _lens(case)
    s = dict(case=case, ctx=ctx, new=new, tokens=max(1, sum(max(n, 0) for n in new)))
    s["d_ctx"] = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    s["d_new"] = torch.tensor(new, dtype=torch.int32, device="cuda")
    plan = case["kind"] == "plan"
    s["table"], s["pool"], s["free"], s["count"] = _tables(ctx, new, case["page"], gen, held_only=plan)
    if plan:
        return s
    dt, T, H_q, H_kv, d = DTYPES[case["dtype"]], s["tokens"], case["H_q"], case["H_kv"], case["d"]
    rand = lambda *shape: torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)
    flat = [(c + i, b) for b, (c, n) in enumerate(zip(ctx, new)) for i in range(max(n, 0))]
    s["positions"] = torch.tensor([p for p, _ in flat], dtype=torch.int32, device="cuda")
    row = torch.tensor([b for _, b in flat], device="cuda")
    at = s["positions"].long()
    s["slots"] = s["table"][row, at // case["page"]].long() * case["page"] + at % case["page"]
    if case["kind"] == "prestep":
        # projections of a hidden state: log-normal channel scales with a few large channels
        scale = torch.exp(0.5 * rand(H_q + H_kv, d))
        scale[:, torch.randperm(d, generator=gen, device="cuda")[:4]] *= 8.0
        q = rand(T, H_q, GATED * d)
        q[..., :d] *= scale[:H_q]
        s["q_gate"] = q.to(dt)
        s["k"] = (rand(T, H_kv, d) * scale[H_q:]).to(dt)
        s["v"] = rand(T, H_kv, d).to(dt)
        s["q_w"] = 1.0 + 0.2 * rand(d) if case["weights"] else None
        s["k_w"] = 1.0 + 0.2 * rand(d) if case["weights"] else None
        s["q_out"] = torch.zeros(T, H_q, d, dtype=dt, device="cuda")
        # pages of the new tokens only: the pool of a server is larger, what a pass touches is this
        used, back = torch.unique(s["slots"] // case["page"], return_inverse=True)
        s["slots"] = back * case["page"] + s["slots"] % case["page"]
        remap = torch.full((s["pool"],), -1, dtype=torch.int32, device="cuda")
        remap[used] = torch.arange(len(used), dtype=torch.int32, device="cuda")
        s["table"] = torch.where(s["table"] >= 0, remap[s["table"].clamp(min=0).long()], s["table"])
        s["pool"] = len(used)
        for name in ("k_cache", "v_cache") + (("u_cache",) if case["unroped"] else ()):
            s[name] = torch.zeros(s["pool"], case["page"], H_kv, d, dtype=dt, device="cuda")
        return s
    # queries and keys behind their head norms: unit scale; the queries sharpened so that a row has keys that stand out
    s["q_gate"] = rand(T, H_q, GATED * d)
    s["q_gate"][..., :d] *= 2.0
    s["q_gate"] = s["q_gate"].to(dt)
    for name in ("k_cache", "v_cache"):
        s[name] = torch.empty(s["pool"], case["page"], H_kv, d, dtype=dt, device="cuda")
        for p in range(0, s["pool"], 4096):
            part = s[name][p:p + 4096]
            part.copy_(rand(*part.shape))
    s["out"] = torch.zeros(T, H_q, d, dtype=dt, device="cuda")
    s["lse"] = torch.zeros(T, H_q, dtype=torch.float32, device="cuda") if case["lse"] else None
    s["scale"] = d ** -0.5
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        s["plan"] = _make_plan(case, s)
        if case["kind"] == "plan":
            s["count_out"] = torch.zeros_like(s["count"])
        else:  # the step's plan stands before its layers run; the pages of the new tokens are in the table
            s["plan"].build(s["d_ctx"], s["d_new"], s["table"])
    return s


def run(s):
    case = s["case"]
    return {"plan": _plan, "prestep": _prestep, "attention": _attention}[case["kind"]](case, s)


# ---- the plan of a step ---------------------------------------------------------------------------------------------------------
def _plan(case, s):
    if own:
        p = s["plan"].build(s["d_ctx"], s["d_new"], s["table"], s["free"], s["count"], s["count_out"])
        return [p.cu_new, p.kv_lens, p.positions, p.slots, s["table"], s["free"], s["count_out"]]
    page, T = case["page"], s["tokens"]
    ctx, new, table, free = s["d_ctx"].long(), s["d_new"].long(), s["table"], s["free"]
    n = new.clamp(min=0)
    cu = torch.cat([n.new_zeros(1), torch.cumsum(n, 0)])
    kv = torch.where(new >= 0, ctx + n, torch.zeros_like(ctx))
    held, after = (ctx + page - 1) // page, (kv + page - 1) // page
    # pages of ended requests go behind the free ones, and pages are taken from the end
    col = torch.arange(table.shape[1], device=table.device)[None, :]
    back = (new < 0)[:, None] & (col < held[:, None])
    n_back = torch.where(new < 0, held, torch.zeros_like(held))
    at = s["count"].long() + torch.cumsum(n_back, 0)[:, None] - n_back[:, None] + col
    stack = torch.cat([free, free.new_zeros(1)])
    stack.scatter_(0, torch.where(back, at, torch.full_like(at, len(free))).reshape(-1), table.reshape(-1))
    free.copy_(stack[:-1])
    top = s["count"].long() + n_back.sum()
    need = torch.where(new >= 0, after - held, torch.zeros_like(held))
    nth = torch.cumsum(need, 0)[:, None] - need[:, None] + col - held[:, None]
    mine = (new >= 0)[:, None] & (col >= held[:, None]) & (col < after[:, None])
    page_of = torch.where(nth < top, stack[(top - 1 - nth).clamp(min=0, max=len(free))], stack.new_full((), -1))
    table.copy_(torch.where(mine, page_of, table))
    t = torch.arange(T, device=table.device)
    row = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp(max=len(ctx) - 1)
    pos = ctx[row] + t - cu[row]
    pages = table[row, (pos // page).clamp(max=table.shape[1] - 1)].long()
    live = t < cu[-1]
    slots = torch.where(live & (pages >= 0), pages * page + pos % page, torch.full_like(pos, -1))
    pos = torch.where(live, pos, torch.full_like(pos, -1))
    count = (top - need.sum()).clamp(min=0)
    i32 = torch.int32
    return [cu.to(i32), kv.to(i32), pos.to(i32), slots, table, free, count.to(i32)]


# ---- norms, rotation, cache rows --------------------------------------------------------------------------------------------------
def _prestep(case, s):
    d, rot = case["d"], case["rotary"]
    if own:
        from bonsai_mojo_1bit_optimization_t4_cuda_b200.paged import paged_prestep

        paged_prestep(s["plan"], s["q_gate"][..., :d], s["k"], s["v"], s["q_w"], s["k_w"], s["q_out"], s["k_cache"], s["v_cache"],
                      s.get("u_cache"), rotary_dim=rot, rope_theta=THETA, rms_eps=EPS)
    else:
        half = rot // 2
        freq = THETA ** (-torch.arange(half, device="cuda", dtype=torch.float64) * 2.0 / rot)
        angle = s["positions"].double()[:, None, None] * freq
        cos, sin = angle.cos().float(), angle.sin().float()

        def norm(x, w):
            x = x.float()
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
            return x if w is None else x * w

        def turn(x):
            a, b = x[..., :half], x[..., half:rot]
            return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., rot:]], -1)

        dt = s["q_out"].dtype
        s["q_out"].copy_(turn(norm(s["q_gate"][..., :d], s["q_w"])).to(dt))
        k = norm(s["k"], s["k_w"])
        rows = lambda c: c.view(-1, c.shape[2], d)
        rows(s["k_cache"])[s["slots"]] = turn(k).to(dt)
        rows(s["v_cache"])[s["slots"]] = s["v"]
        if "u_cache" in s:
            rows(s["u_cache"])[s["slots"]] = k.to(dt)
    return [s["q_out"], s["k_cache"], s["v_cache"]] + ([s["u_cache"]] if "u_cache" in s else [])


# ---- attention ------------------------------------------------------------------------------------------------------------------------
def _attention(case, s):
    d = case["d"]
    if own:
        from bonsai_mojo_1bit_optimization_t4_cuda_b200.paged import paged_attention

        paged_attention(s["plan"], s["q_gate"][..., :d], s["k_cache"], s["v_cache"], s["table"], s["out"], s["scale"],
                        gate=s["q_gate"][..., d:] if case["gate"] else None, lse=s["lse"])
    else:
        H_q, H_kv, page, t0 = case["H_q"], case["H_kv"], case["page"], 0
        rep = H_q // H_kv
        for b, (c, n) in enumerate(zip(s["ctx"], s["new"])):
            kv = c + n
            pages = s["table"][b, :_pages(kv, page)].long()
            k = s["k_cache"][pages].reshape(-1, H_kv, d)[:kv].float().permute(1, 2, 0)
            v = s["v_cache"][pages].reshape(-1, H_kv, d)[:kv].float().permute(1, 0, 2)
            step = max(1, min(n, (1 << 28) // (kv * H_q)))
            for i in range(0, n, step):
                m = min(step, n - i)
                rows = slice(t0 + i, t0 + i + m)
                q = s["q_gate"][rows, :, :d].float().reshape(m, H_kv, rep, d).permute(1, 0, 2, 3).reshape(H_kv, m * rep, d)
                x = torch.matmul(q, k).view(H_kv, m, rep, kv) * s["scale"]
                at = c + i + torch.arange(m, device="cuda")
                x.masked_fill_((torch.arange(kv, device="cuda")[None, :] > at[:, None])[None, :, None, :], float("-inf"))
                top = x.amax(-1, keepdim=True)
                p = torch.exp(x - top)
                z = p.sum(-1, keepdim=True)
                o = torch.matmul(p.view(H_kv, m * rep, kv), v).view(H_kv, m, rep, d) / z
                o = o.permute(1, 0, 2, 3).reshape(m, H_q, d)
                if case["gate"]:
                    o = o / (1.0 + torch.exp(-s["q_gate"][rows, :, d:].float()))
                s["out"][rows] = o.to(s["out"].dtype)
                if case["lse"]:
                    s["lse"][rows] = (top + torch.log(z)).squeeze(-1).permute(1, 0, 2).reshape(m, H_q)
            t0 += n
    return [s["out"]] + ([s["lse"]] if case["lse"] else [])


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------------------
def work(case):
    ctx, new = _lens(case)
    T = sum(max(n, 0) for n in new)
    H_q, H_kv, d, page = case["H_q"], case["H_kv"], case["d"], case["page"]
    if case["kind"] == "plan":
        moved = sum(_pages(c, page) if n < 0 else _pages(c + n, page) - _pages(c, page) for c, n in zip(ctx, new))
        return {"bytes": 8 * len(ctx) + 8 * len(ctx) + 12 * T + 8 * moved, "flops": 0}
    if case["kind"] == "prestep":
        moved = T * d * 2 * (2 * H_q + 4 * H_kv + (H_kv if case["unroped"] else 0)) + 12 * T
        return {"bytes": moved, "flops": T * (H_q + H_kv) * (4 * d + 3 * case["rotary"])}
    kv = sum(c + n for c, n in zip(ctx, new))
    pairs = sum(n * c + n * (n + 1) // 2 for c, n in zip(ctx, new))
    moved = kv * H_kv * d * 4 + T * H_q * d * 2 * (3 if case["gate"] else 2) + (T * H_q * 4 if case["lse"] else 0)
    return {"bytes": moved, "flops": pairs * H_q * d * 4}


# ---- the definitions, in 64 bits ----------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    d, page = case["d"], case["page"]
    f64 = torch.float64
    if case["kind"] == "plan":
        return None  # whole numbers: the outputs have to be equal
    if case["kind"] == "prestep":
        rot, pos = case["rotary"], s["positions"].to(f64)
        i = torch.arange(rot // 2, device="cuda", dtype=f64)
        z = torch.polar(torch.ones(len(pos), 1, rot // 2, device="cuda", dtype=f64),
                        pos[:, None, None] * torch.exp(-i * (2.0 / rot) * math.log(THETA)))
        outs = []
        for x, w in ((s["q_gate"][..., :d].to(f64), s["q_w"]), (s["k"].to(f64), s["k_w"])):
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
            if w is not None:
                x = x * w.to(f64)
            y = torch.complex(x[..., :rot // 2].contiguous(), x[..., rot // 2:rot].contiguous()) * z
            outs.append((x, torch.cat([y.real, y.imag, x[..., rot:]], -1)))
        res = [outs[0][1]]
        for value in (outs[1][1], s["v"].to(f64)) + ((outs[1][0],) if "u_cache" in s else ()):
            cache = torch.zeros(s["pool"] * page, case["H_kv"], d, device="cuda", dtype=f64)
            cache.index_copy_(0, s["slots"], value)
            res.append(cache.view(s["pool"], page, case["H_kv"], d))
        return res
    H_q, H_kv = case["H_q"], case["H_kv"]
    rep, t0 = H_q // H_kv, 0
    out = torch.zeros(s["tokens"], H_q, d, device="cuda", dtype=f64)
    lse = torch.zeros(s["tokens"], H_q, device="cuda", dtype=f64)
    for b, (c, n) in enumerate(zip(s["ctx"], s["new"])):
        pages = s["table"][b, :_pages(c + n, page)].long()
        for h in range(H_kv):
            k = s["k_cache"][pages, :, h].reshape(-1, d)
            v = s["v_cache"][pages, :, h].reshape(-1, d)
            for i in range(0, n, 512):
                m = min(512, n - i)
                end = c + i + m  # keys that any of these rows attends
                q = s["q_gate"][t0 + i:t0 + i + m, h * rep:(h + 1) * rep, :d].to(f64)
                x = torch.einsum("mrd,kd->mrk", q, k[:end].to(f64)) * s["scale"]
                hidden = torch.ones(m, end, dtype=torch.bool, device="cuda").triu(diagonal=c + i + 1)
                x = x.masked_fill(hidden[:, None, :], -math.inf)
                total = torch.logsumexp(x, -1)
                lse[t0 + i:t0 + i + m, h * rep:(h + 1) * rep] = total
                out[t0 + i:t0 + i + m, h * rep:(h + 1) * rep] = torch.einsum("mrk,kd->mrd", torch.exp(x - total[..., None]), v[:end].to(f64))
        t0 += n
    if case["gate"]:
        out = out * torch.sigmoid(s["q_gate"][..., d:].to(f64))
    return [out] + ([lse] if case["lse"] else [])
