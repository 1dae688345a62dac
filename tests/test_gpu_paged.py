"""The paged operators against plain 64-bit forms, at the sizes and masks where they can go wrong."""
import math
import random

import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(autouse=True)
def _clean(cuda_ops):
    yield
    assert cuda_ops.lib.khq_b200_paged_status() == 0


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def make_table(ctx, new, page, gen, spare=3, width=None):
    counts = [-(-(c + max(n, 0)) // page) for c, n in zip(ctx, new)]
    pool = sum(counts) + spare
    order = torch.randperm(pool, generator=gen).tolist()
    width = width or max(1, max(counts))
    table = [[order.pop() for _ in range(c)] + [-1] * (width - c) for c in counts]
    return table, pool


def built(ctx, new, table, page, H_q, H_kv, d, max_tokens=None, max_new=None, requests=None):
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.paged import PagedPlan

    T = sum(max(n, 0) for n in new)
    plan = PagedPlan(requests or len(ctx), max_tokens or max(T, 1), page, H_q, H_kv, d, max_new=max_new or max(1, max(new)))
    return plan.build(i32(ctx), i32(new), table)


# ---- plan -------------------------------------------------------------------------------------------------------------------------
def check_plan(ctx, new, page, max_tokens, max_new, pool, free_share=1.0, seed=0, alias=True):
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.paged import PagedPlan

    rng = random.Random(seed)
    held = [-(-max(c, 0) // page) for c in ctx]
    width = max(1, max(-(-(max(c, 0) + max(n, 0)) // page) for c, n in zip(ctx, new)))
    order = list(range(pool))
    rng.shuffle(order)
    table = [[order.pop() for _ in range(h)] + [-1] * (width - h) for h in held]
    count = int(len(order) * free_share)
    free = order[:count] + [-7] * (pool - count)
    d_table, d_free, d_count = i32(table), i32(free), i32([count])
    plan = PagedPlan(len(ctx), max_tokens, page, 24, 4, 256, max_new=max_new)
    out = None if alias else torch.full((1,), -5, dtype=torch.int32, device="cuda")
    plan.build(i32(ctx), i32(new), d_table, d_free, d_count, out)
    want = ref.plan(ctx, new, table, page, max_tokens, max_new, free, count)
    assert plan.cu_new.tolist() == want["cu"]
    assert plan.kv_lens.tolist() == want["kv"]
    assert plan.positions.tolist() == want["positions"]
    assert plan.slots.tolist() == want["slots"]
    assert d_table.tolist() == table
    assert d_free.tolist() == free
    assert (d_count if alias else out).tolist() == [want["count"]]
    if not alias:
        assert d_count.tolist() == [count]
    assert plan.info[:5].tolist() == want["info"] and plan.info[5].item() == want["count"]


@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("requests,ctx_hi,new_hi,ended", [(1, 0, 1, 0), (1, 300, 5, 0), (7, 130, 40, 2), (300, 700, 1, 20), (1500, 90, 30, 300)])
def test_plan(cuda_ops, page, requests, ctx_hi, new_hi, ended):
    rng = random.Random(page * 1000 + requests)
    ctx = [rng.randint(0, ctx_hi) for _ in range(requests)]
    new = [rng.randint(0, new_hi) for _ in range(requests)]
    for b in rng.sample(range(requests), min(ended, requests)):
        new[b] = -1
    pool = sum(-(-(c + max(n, 0)) // page) for c, n in zip(ctx, new)) + 5
    check_plan(ctx, new, page, sum(max(n, 0) for n in new) + 3, max(1, new_hi), pool, alias=requests % 2 == 0)


def test_plan_pages_run_out(cuda_ops):
    ctx, new = [10, 33, 5, 16, 0], [40, 60, -1, 1, 100]
    check_plan(ctx, new, 16, 300, 100, 12, seed=3)


def test_plan_row_that_ran_out_ends(cuda_ops):
    """Its pages go back, the ones that it never got do not."""
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.paged import PagedPlan

    table, free, count = i32([[-1] * 6, [-1] * 6]), i32([0, 1, 2, 3, 4]), i32([5])
    t, f = table.tolist(), free.tolist()
    plan, c, lens = PagedPlan(2, 96, 16, 24, 4, 256), 5, [0, 0]
    for new in ([20, 70], [-1, 0], [0, -1], [40, 40]):
        plan.build(i32(lens), i32(new), table, free, count)
        want = ref.plan(lens, new, t, 16, 96, 96, f, c)
        c = want["count"]
        assert table.tolist() == t and free.tolist() == f and count.item() == c and plan.slots.tolist() == want["slots"]
        assert plan.info[:5].tolist() == want["info"]
        lens = [0 if n < 0 else x + n for x, n in zip(lens, new)]
    assert c == 0 and sorted(x for row in t for x in row[:3]) == [-1, 0, 1, 2, 3, 4]  # every page is in use once


def test_plan_drops_what_does_not_fit(cuda_ops):
    check_plan([3, 50, 7], [30, 20, 9], 16, 41, 25, 20, seed=4)


def test_plan_nothing_to_do(cuda_ops):
    check_plan([3, 0], [0, 0], 16, 4, 4, 9)
    check_plan([40, 17], [-1, -1], 16, 4, 4, 9)


def test_plan_with_pages_held(cuda_ops):
    gen = torch.Generator().manual_seed(1)
    ctx, new = [5, 100, 0], [20, 1, 7]
    table, pool = make_table(ctx, new, 32, gen)
    plan = built(ctx, new, i32(table), 32, 24, 4, 256, max_tokens=40)
    want = ref.plan(ctx, new, table, 32, 40, 20)
    assert plan.slots.tolist() == want["slots"] and plan.positions.tolist() == want["positions"] and plan.kv_lens.tolist() == want["kv"]


def test_plan_table_rows_apart(cuda_ops):
    """A table whose rows are a part of wider ones."""
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.paged import PagedPlan

    wide = torch.full((3, 20), -9, dtype=torch.int32, device="cuda")
    table = wide[:, 4:10]
    plan = PagedPlan(3, 64, 16, 24, 4, 256)
    plan.build(i32([0, 0, 0]), i32([20, 0, 33]), table, i32(range(9)), i32([9]))
    assert table[0, :2].tolist() == [8, 7] and table[2, :3].tolist() == [6, 5, 4]
    assert (wide[:, :4] == -9).all() and (wide[:, 10:] == -9).all() and (table[1] == -9).all()


# ---- pre-step -----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("H_q,H_kv,d,page,rotary,weights,unroped,ctx,new", [
    (24, 4, 256, 128, 64, True, True, [4000], [1]),
    (24, 4, 256, 16, 64, True, True, [0, 17, 250000, 31], [5, 0, 3, 40]),
    (5, 1, 128, 32, 128, False, False, [3, 90], [31, 2]),
    (9, 3, 128, 64, 32, True, True, [63, 1], [1, 64]),
    (8, 8, 256, 64, 256, True, False, [100, 5], [7, 1]),
    (6, 2, 256, 16, 0, True, True, [9], [12]),
])
def test_prestep(cuda_ops, dtype, H_q, H_kv, d, page, rotary, weights, unroped, ctx, new):
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.paged import paged_prestep

    gen = torch.Generator(device="cuda").manual_seed(5)
    dt, T = DT[dtype], sum(new)
    width = max(-(-(c + n) // page) for c, n in zip(ctx, new))
    table = [[-1] * width for _ in ctx]
    free = list(range(sum(-(-(c + n) // page) - c // page for c, n in zip(ctx, new)) + 2))
    pool = len(free)
    for b, (c, n) in enumerate(zip(ctx, new)):  # pages of the new tokens only
        for col in range(c // page, -(-(c + n) // page)):
            table[b][col] = free.pop()
    cap = T + 3
    plan = built(ctx, new, i32(table), page, H_q, H_kv, d, max_tokens=cap)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    q_gate = (3 * rand(cap, H_q, 2 * d)).to(dt)
    kv = (2 * rand(cap, 2, H_kv, d)).to(dt)
    k, v = kv[:, 0], kv[:, 1]
    qw, kw = (1 + 0.3 * rand(d), 1 + 0.3 * rand(d)) if weights else (None, None)
    fill = lambda *s: torch.full(s, 7.0, dtype=dt, device="cuda")
    both = fill(pool, 2, page, H_kv, d)  # K and V of a page side by side
    kc, vc = both[:, 0], both[:, 1]
    uc = fill(H_kv, pool, page, d).permute(1, 2, 0, 3) if unroped else None  # heads outermost
    q_out = fill(cap, H_q, d)
    paged_prestep(plan, q_gate[..., :d], k, v, qw, kw, q_out, kc, vc, uc, rotary_dim=rotary)
    want = ref.plan(ctx, new, table, page, cap, max(new))
    pos, slots = torch.tensor(want["positions"][:T], device="cuda"), torch.tensor(want["slots"][:T], device="cuda")
    half = torch.finfo(dt).eps / 2

    def near(got, value, base):
        # one rounding; fp32 arithmetic: sums of up to 256 squares and a rotation by an angle good to 2^-22, together below 2^-18 of the pair's size;
        # fp16 below its normal range is off by half of 2^-24
        bound = half * value.abs() + 2.0 ** -18 * base + (2.0 ** -25 if dt is torch.float16 else 0.0)
        assert ((got.double() - value).abs() <= bound).all()

    size = lambda x: x.abs().amax(-1, keepdim=True).expand_as(x)
    qn, qr = ref.prestep(q_gate[:T, :, :d], qw, pos, rotary, 1e7, 1e-6)
    kn, kr = ref.prestep(k[:T], kw, pos, rotary, 1e7, 1e-6)
    near(q_out[:T], qr, size(qn))
    assert (q_out[T:] == 7.0).all()
    for cache, value in ((kc, kr), (vc, v[:T].double())) + (((uc, kn),) if unroped else ()):
        rows = cache.reshape(pool * page, H_kv, d)
        near(rows[slots], value, size(kn) if cache is not vc else torch.zeros_like(value))
        rest = torch.ones(pool * page, dtype=torch.bool, device="cuda")
        rest[slots] = False
        assert (rows[rest] == 7.0).all()


def test_prestep_in_place_and_without_pages(cuda_ops):
    """q normed where it stands; tokens for which no page was left keep their queries and touch no cache row."""
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.paged import PagedPlan, paged_prestep

    torch.manual_seed(0)
    plan = PagedPlan(2, 40, 16, 6, 1, 256)
    table = torch.full((2, 3), -1, dtype=torch.int32, device="cuda")
    plan.build(i32([0, 0]), i32([20, 20]), table, i32([0, 1, 2]), i32([3]))
    assert plan.info.tolist()[:6] == [40, 3, 0, 1, 0, 0]
    q_gate = torch.randn(40, 6, 512, device="cuda").half()
    before = q_gate.clone()
    k, v = torch.randn(40, 1, 256, device="cuda").half(), torch.randn(40, 1, 256, device="cuda").half()
    kc, vc = torch.zeros(3, 16, 1, 256, dtype=torch.float16, device="cuda"), torch.zeros(3, 16, 1, 256, dtype=torch.float16, device="cuda")
    paged_prestep(plan, q_gate[..., :256], k, v, None, None, q_gate[..., :256], kc, vc)
    assert torch.equal(q_gate[..., 256:], before[..., 256:])
    pos = torch.tensor(list(range(20)) * 2, device="cuda")
    _, want = ref.prestep(before[..., :256], None, pos, 64, 1e7, 1e-6)
    assert ((q_gate[..., :256].double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -16).all()
    assert plan.slots[36:].tolist() == [-1] * 4
    assert (vc.reshape(48, 256)[torch.tensor([s for s in plan.slots.tolist() if s >= 0], device="cuda")] == torch.cat([v[:36, 0]])).all()


# ---- attention -----------------------------------------------------------------------------------------------------------------------------
def attend(dtype, H_q, H_kv, d, page, ctx, new, gated=True, seed=0, poison=True, holes=(), layout="tokens", extra=2, scale=None, sharp=2.0, max_new=None,
           shared=0):
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.paged import paged_attention

    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, T = DT[dtype], sum(max(n, 0) for n in new)
    table, pool = make_table(ctx, new, page, torch.Generator().manual_seed(seed))
    for row in table[1:]:  # the same pages at the front of every request
        row[:shared] = table[0][:shared]
    cap = T + extra
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    q_gate = rand(cap, H_q, 2 * d)
    q_gate[..., :d] *= sharp
    q_gate = q_gate.to(dt)
    if layout == "tokens":
        kc, vc = rand(pool, page, H_kv, d).to(dt), rand(pool, page, H_kv, d).to(dt)
    elif layout == "heads":
        kc, vc = (rand(pool, H_kv, page, d).to(dt).permute(0, 2, 1, 3) for _ in range(2))
    else:
        both = rand(pool, 2, page, H_kv, d).to(dt)
        kc, vc = both[:, 0], both[:, 1]
    clean_k, clean_v = kc.clone(), vc.clone()
    if poison:  # cache rows that no token stands in
        used = torch.zeros(pool, page, dtype=torch.bool)
        for b, (c, n) in enumerate(zip(ctx, new)):
            for t in range(c + max(n, 0)):
                used[table[b][t // page], t % page] = True
        used = used.cuda()
        kc[~used] = float("nan")
        vc[~used] = float("inf")
        vc[~used] *= torch.tensor([1.0, -1.0], device="cuda").repeat(d // 2).to(dt)
    for b, col, value in holes:
        table[b][col] = value
    d_table = i32(table)
    plan = built(ctx, new, d_table, page, H_q, H_kv, d, max_tokens=cap, max_new=max_new)
    out = torch.full((cap, H_q, d), 7.0, dtype=dt, device="cuda")
    lse = torch.full((cap, H_q), 7.0, dtype=torch.float32, device="cuda")
    scale = d ** -0.5 if scale is None else scale
    gate = q_gate[..., d:] if gated else None
    paged_attention(plan, q_gate[..., :d], kc, vc, d_table, out, scale, gate=gate, lse=lse)
    want, want_lse, tol, lse_tol = ref.attention(q_gate[:T, :, :d], clean_k, clean_v, table, ctx, new, scale, gate[:T] if gated else None)
    err = (out[:T].double() - want).abs()
    assert torch.isfinite(out[:T].float()).all()
    assert (err <= tol).all(), f"worst {(err / tol).max().item():.3g} of the bound at {torch.nonzero(err > tol)[0].tolist()}"
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse[:T]), empty)
    assert ((lse[:T].double() - want_lse).masked_fill(empty, 0.0).abs() <= lse_tol).all()
    assert (out[T:] == 7.0).all() and (lse[T:] == 7.0).all()
    return out[:T], plan


DECODES = [
    ([0], [1]), ([15], [1]), ([63], [1]), ([64], [1]), ([4001], [1]), ([0, 5, 63, 64, 65, 700, 1, 127], [1] * 8),
    ([3000, 10, 0, 511], [1, 0, 1, 1]), ([20000], [1]), ([7, 200, 90], [-1, 1, 1]),
]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("ctx,new", DECODES)
def test_attention_one_token(cuda_ops, dtype, ctx, new):
    attend(dtype, 24, 4, 256, 128, ctx, new)


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("H_q,H_kv,d", [(24, 4, 256), (8, 1, 256), (16, 16, 128), (20, 4, 128), (16, 1, 128), (3, 3, 256)])
@pytest.mark.parametrize("layout", ["tokens", "heads", "both"])
def test_attention_heads_and_pages(cuda_ops, page, H_q, H_kv, d, layout):
    attend("bf16", H_q, H_kv, d, page, [300, 0, 77, 1200], [1, 1, 1, 1], layout=layout, gated=H_q != 20, seed=page)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("ctx,new", [([0], [2]), ([100], [2]), ([61, 0, 500], [2, 2, 1]), ([0, 64], [7, 70]), ([0], [300]), ([130, 900], [129, 43]),
                                     ([0, 0, 5], [1, 200, 33]), ([2000], [257])])
@pytest.mark.parametrize("H_q,H_kv,d,page", [(24, 4, 256, 64), (20, 4, 128, 16), (8, 8, 128, 32)])
def test_attention_chunks(cuda_ops, dtype, ctx, new, H_q, H_kv, d, page):
    attend(dtype, H_q, H_kv, d, page, ctx, new, seed=len(ctx) + sum(new))


@pytest.mark.parametrize("H_q,H_kv,d,page", [(32, 1, 128, 16), (128, 1, 128, 64), (48, 1, 256, 128), (100, 1, 256, 32), (34, 2, 128, 128)])
@pytest.mark.parametrize("ctx,new", [([0, 200, 5], [1, 1, 1]), ([64, 0, 700], [9, 130, 2])])
def test_attention_many_heads_of_a_kv_head(cuda_ops, H_q, H_kv, d, page, ctx, new):
    attend("fp16", H_q, H_kv, d, page, ctx, new, seed=H_q)


@pytest.mark.parametrize("H_q,H_kv,d,page", [(24, 4, 256, 64), (20, 4, 128, 16)])
def test_attention_chunks_between_decodes(cuda_ops, H_q, H_kv, d, page):
    """Both kernels in one call, either of them with little, much or nothing to do."""
    rng = random.Random(3)
    for ctx, new in (([500, 20, 3000, 0, 77], [1, 300, 1, 90, 2]), ([0, 64, 65], [1, 1, 200]), ([4000, 4000], [17, 1]), ([300] * 5, [2, 1, 2, 1, 1]),
                     ([rng.randint(0, 900) for _ in range(120)], [rng.choice([0, 1, 1, 1, 2, 40]) for _ in range(120)])):
        attend("bf16", H_q, H_kv, d, page, ctx, new, max_new=300, seed=len(ctx))


@pytest.mark.parametrize("H_q,H_kv,d", [(24, 4, 256), (20, 4, 128)])
def test_attention_few_and_many_rows_in_turn(cuda_ops, H_q, H_kv, d):
    """Tiles with one, some and all of their rows in use, one after the other in the same CTAs."""
    rng = random.Random(7)
    rows = [(rng.randint(0, 600), rng.choice([4, 5, 7, 9, 12, 16, 21, 22, 30, 43, 70])) for _ in range(300)]
    attend("fp16", H_q, H_kv, d, 32, [c for c, _ in rows], [n for _, n in rows], seed=21)


def test_attention_long_contexts_shared(cuda_ops):
    """Few requests over long contexts: every segment is shared by many CTAs."""
    attend("fp16", 24, 4, 256, 128, [40000], [30], seed=1)
    attend("bf16", 8, 1, 256, 16, [30011], [1], seed=2)
    attend("fp16", 4, 1, 128, 16, [60000, 3], [50, 1], seed=3)


def test_attention_many_requests(cuda_ops):
    rng = random.Random(8)
    ctx = [rng.choice([0, 1, 15, 16, 17, 100, 400]) for _ in range(400)]
    attend("fp16", 24, 4, 256, 16, ctx, [1] * 400, seed=9)
    attend("bf16", 20, 4, 128, 32, ctx, [rng.choice([0, 1, 1, 3]) for _ in range(400)], seed=10)


@pytest.mark.parametrize("new", [[1, 1, 1], [50, 1, 90]])
def test_attention_missing_pages(cuda_ops, new):
    """Pages that could not be had, or with numbers outside the cache: not attended; a row without any gets 0 and -inf."""
    ctx = [100, 20, 300]
    big = 1 << 30
    holes = [(0, 1, -1), (0, 3, big), (2, 0, -5), (2, 2, 2147483647)] + [(1, c, -1) for c in range(-(-(20 + new[1]) // 32))]
    attend("fp16", 24, 4, 256, 32, ctx, new, holes=holes, poison=False)


@pytest.mark.parametrize("new", [[1, 1, 1], [30, 1, 100]])
def test_attention_shared_pages(cuda_ops, new):
    attend("bf16", 24, 4, 256, 32, [200, 130, 300], new, shared=4)


@pytest.mark.parametrize("new", [1, 40])
def test_attention_large_scores(cuda_ops, new):
    """Scores of some hundreds: the maximum moves by more than the weights' range, again and again."""
    attend("bf16", 24, 4, 256, 64, [700], [new], sharp=60.0)


def test_attention_captured_and_replayed(cuda_ops):
    """One graph at the step's largest size, replayed with other lengths: plan, pre-step and attention together."""
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.paged import PagedPlan, paged_attention, paged_prestep

    H_q, H_kv, d, page, B, T, pool = 24, 4, 256, 32, 5, 64, 120
    gen = torch.Generator(device="cuda").manual_seed(2)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda").half()
    q, k, v = torch.zeros(T, H_q, d, dtype=torch.float16, device="cuda"), rand(T, H_kv, d), rand(T, H_kv, d)
    kc, vc = torch.zeros(pool, page, H_kv, d, dtype=torch.float16, device="cuda"), torch.zeros(pool, page, H_kv, d, dtype=torch.float16, device="cuda")
    out = torch.zeros(T, H_q, d, dtype=torch.float16, device="cuda")
    table = torch.full((B, 24), -1, dtype=torch.int32, device="cuda")
    free, count = torch.arange(pool, dtype=torch.int32, device="cuda"), i32([pool])
    ctx, new = i32([0] * B), i32([0] * B)
    plan = PagedPlan(B, T, page, H_q, H_kv, d)

    def step():
        plan.build(ctx, new, table, free, count)
        paged_prestep(plan, q, k, v, None, None, q, kc, vc)
        paged_attention(plan, q, kc, vc, table, out, d ** -0.5)

    step()  # nothing new: changes nothing
    assert count.item() == pool and (kc == 0).all() and (out == 0).all()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    lens, rng = [0] * B, random.Random(4)
    for turn in range(12):
        n = [rng.choice([0, 1, 1, 7, 30]) for _ in range(B)]
        while sum(n) > T:
            n[n.index(max(n))] = 1
        if turn == 7:
            n[2] = -1
        ctx.copy_(i32(lens))
        new.copy_(i32(n))
        for x in (q, k, v):
            x.copy_(rand(*x.shape))
        out.fill_(7.0)
        g.replay()
        rows = sum(max(m, 0) for m in n)
        want, _, tol, _ = ref.attention(q[:rows], kc, vc, table.tolist(), lens, n, d ** -0.5)
        assert ((out[:rows].double() - want).abs() <= tol).all() and (out[rows:] == 7.0).all()
        lens = [0 if m < 0 else c + m for c, m in zip(lens, n)]
        assert count.item() == pool - sum(-(-c // page) for c in lens)


def test_attention_chunked_is_the_whole_prompt(cuda_ops):
    """A prompt in chunks of odd sizes: the attention that the whole prompt at once gets from gqa_prefill."""
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.paged import PagedPlan, paged_attention

    torch.manual_seed(3)
    T, page, pool = 700, 64, 16
    q_gate = torch.randn(T, 24, 512, device="cuda").half()
    k, v = torch.randn(T, 4, 256, device="cuda").half(), torch.randn(T, 4, 256, device="cuda").half()
    whole, parts = torch.empty(T, 24, 256, dtype=torch.float16, device="cuda"), torch.empty(T, 24, 256, dtype=torch.float16, device="cuda")
    cuda_ops.gqa_prefill(q_gate, k, v, whole, 1, T, 24, 4, 256, 1 / 16)
    kc, vc = torch.zeros(pool, page, 4, 256, dtype=torch.float16, device="cuda"), torch.zeros(pool, page, 4, 256, dtype=torch.float16, device="cuda")
    table = torch.full((1, 11), -1, dtype=torch.int32, device="cuda")
    free, count = torch.arange(pool, dtype=torch.int32, device="cuda"), i32([pool])
    plan, at = PagedPlan(1, 333, page, 24, 4, 256), 0
    for n in (1, 200, 333, 2, 164):
        plan.build(i32([at]), i32([n]), table, free, count)
        kc.view(-1, 4, 256)[plan.slots[:n]], vc.view(-1, 4, 256)[plan.slots[:n]] = k[at:at + n], v[at:at + n]
        paged_attention(plan, q_gate[at:at + n, :, :256], kc, vc, table, parts[at:at + n], 1 / 16, gate=q_gate[at:at + n, :, 256:])
        at += n
    assert at == T
    # two kernels, each within its rounding of the weights and of the output: 4 half steps of values below 2
    assert (parts.float() - whole.float()).abs().max().item() <= 4 * 2.0 ** -11 * 2


def test_attention_beyond_32_bits(cuda_ops):
    """Pages whose first value lies more than 2^32 values into the cache."""
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.paged import PagedPlan, paged_attention, paged_prestep

    H_q, H_kv, d, page, pool = 16, 16, 256, 128, 8300
    kc = torch.empty(pool, page, H_kv, d, dtype=torch.bfloat16, device="cuda")
    vc = torch.empty_like(kc)
    assert kc.numel() > 1 << 32
    torch.manual_seed(0)
    for new in (1, 70):
        table, free, count = torch.full((2, 3), -1, dtype=torch.int32, device="cuda"), i32([0, 1, pool - 1, 5, pool - 2]), i32([5])
        plan = PagedPlan(2, 400, page, H_q, H_kv, d)
        lens = [0, 0]
        for n in ([200, 100], [new, new]):
            plan.build(i32(lens), i32(n), table, free, count)
            T = sum(n)
            q, k, v = (torch.randn(T, h, d, device="cuda").bfloat16() for h in (H_q, H_kv, H_kv))
            paged_prestep(plan, q, k, v, None, None, q, kc, vc)
            out = torch.empty_like(q)
            paged_attention(plan, q, kc, vc, table, out, d ** -0.5)
            want, _, tol, _ = ref.attention(q, kc, vc, table.tolist(), lens, n, d ** -0.5)
            assert ((out.double() - want).abs() <= tol).all()
            lens = [a + b for a, b in zip(lens, n)]
        assert pool - 2 in table.tolist()[0] + table.tolist()[1]


def test_attention_two_calls_at_once(cuda_ops):
    """One plan, two layers on two streams, each with scratch memory of its own; and the same call again."""
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.paged import paged_attention

    torch.manual_seed(1)
    ctx, new = [5000, 300, 40, 7000], [1, 130, 1, 30]
    table, pool = make_table(ctx, new, 64, torch.Generator().manual_seed(3))
    T, d_table = sum(new), i32(table)
    plan = built(ctx, new, d_table, 64, 24, 4, 256)
    layers = []
    for _ in range(2):
        q = torch.randn(T, 24, 256, device="cuda").half()
        layers.append((q, *(torch.randn(pool, 64, 4, 256, device="cuda").half() for _ in range(2))))
    single = []
    for q, kc, vc in layers:
        out = torch.empty_like(q)
        paged_attention(plan, q, kc, vc, d_table, out, 1 / 16)
        single.append(out)
    scratch, streams = [None, plan.new_workspace()], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        outs = []
        for (q, kc, vc), ws, s in zip(layers, scratch, streams):
            with torch.cuda.stream(s):
                out = torch.empty_like(q)
                paged_attention(plan, q, kc, vc, d_table, out, 1 / 16, workspace=ws)
                outs.append(out)
        torch.cuda.synchronize()
        for a, b in zip(outs, single):
            assert torch.equal(a, b)


@pytest.mark.parametrize("H_q,H_kv,d,ctx,new", [(17, 1, 128, [2295], [333]), (128, 1, 128, [2549, 2159], [306, 273]), (20, 4, 128, [900, 0, 70], [5, 300, 40]),
                                               (24, 4, 256, [900, 0, 70], [5, 300, 40])])
def test_attention_is_the_same_every_time(cuda_ops, H_q, H_kv, d, ctx, new):
    """Segments of all lengths, shared and whole: bit for bit the same output in every run, whatever else the GPU's clocks do."""
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.paged import paged_attention

    torch.manual_seed(5)
    table, pool = make_table(ctx, new, 64, torch.Generator().manual_seed(5))
    T, d_table = sum(new), i32(table)
    plan = built(ctx, new, d_table, 64, H_q, H_kv, d)
    q = (2 * torch.randn(T, H_q, d, device="cuda")).bfloat16()
    kc, vc = (torch.randn(pool, 64, H_kv, d, device="cuda").bfloat16() for _ in range(2))
    outs = torch.empty(150, T, H_q, d, dtype=torch.bfloat16, device="cuda")
    for i in range(len(outs)):
        paged_attention(plan, q, kc, vc, d_table, outs[i], d ** -0.5)
    want, _, tol, _ = ref.attention(q, kc, vc, table, ctx, new, d ** -0.5)
    assert ((outs[0].double() - want).abs() <= tol).all()
    assert all(torch.equal(o, outs[0]) for o in outs[1:])


def test_attention_on_another_stream(cuda_ops):
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        attend("fp16", 24, 4, 256, 64, [500, 3], [1, 1])
    torch.cuda.current_stream().wait_stream(s)


def test_refusals(cuda_ops):
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.lib import KhqLaunchError
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.paged import PagedPlan, paged_attention, paged_prestep

    for bad in (dict(page_size=48), dict(page_size=256), dict(d=64), dict(H_q=25), dict(max_tokens=0)):
        args = dict(max_requests=4, max_tokens=64, page_size=16, H_q=24, H_kv=4, d=256)
        args.update(bad)
        with pytest.raises(ValueError):
            PagedPlan(**args)
    plan = PagedPlan(2, 8, 16, 24, 4, 256)
    half = lambda *s: torch.zeros(*s, dtype=torch.float16, device="cuda")
    q, k, kc, table = half(4, 24, 256), half(4, 4, 256), half(3, 16, 4, 256), i32([[0, 1], [2, -1]])
    with pytest.raises(ValueError, match="not been built"):
        paged_attention(plan, q, kc, kc, table, q, 0.1)
    plan.build(i32([3, 0]), i32([2, 2]), table)
    for call in (
        lambda: plan.build(i32([3]), i32([2, 2]), table),
        lambda: plan.build(i32([1, 1, 1]), i32([1, 1, 1]), i32([[0]] * 3)),
        lambda: plan.build(i32([3, 0]).long(), i32([2, 2]), table),
        lambda: plan.build(i32([3, 0]), i32([2, 2]), table.cpu()),
        lambda: plan.build(i32([3, 0]), i32([2, 2]), table, i32([5])),
        lambda: plan.build(i32([3, 0]), i32([2, 2]), table.t()),
        lambda: paged_attention(plan, q.transpose(0, 1), kc, kc, table, q, 0.1),
        lambda: paged_attention(plan, half(9, 24, 256), kc, kc, table, half(9, 24, 256), 0.1),
        lambda: paged_attention(plan, q, kc.bfloat16(), kc, table, q, 0.1),
        lambda: paged_attention(plan, q, kc[:, :8], kc, table, q, 0.1),
        lambda: paged_attention(plan, q, kc, kc[:2], table, q, 0.1),
        lambda: paged_attention(plan, q, kc, kc, table[:, :1], q, 0.1),
        lambda: paged_attention(plan, q, kc, kc, table, q, 0.1, lse=half(4, 24)),
        lambda: paged_prestep(plan, q, k[:3], k, None, None, q, kc, kc),
        lambda: paged_prestep(plan, q, k, k, half(256), None, q, kc, kc),
    ):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        paged_attention(plan, q.float(), kc, kc, table, q, 0.1)
    for call in (
        lambda: paged_attention(plan, q, kc, kc, table, q, 0.0),
        lambda: paged_attention(plan, q, kc, kc, table, q, -1.0),
        lambda: paged_attention(plan, q, kc, kc, table, q, float("nan")),
        lambda: paged_attention(plan, q, kc, kc, table, q, 0.1, workspace=plan.workspace[:256]),
        lambda: paged_attention(plan, q, kc, kc, table, half(4 * 24 * 256 + 1)[1:].view(4, 24, 256), 0.1),
        lambda: paged_attention(plan, half(4, 24, 260)[..., :256], kc, kc, table, q, 0.1),
        lambda: paged_prestep(plan, q, k, k, None, None, q, kc, kc, rotary_dim=24),
        lambda: paged_prestep(plan, q, k, k, None, None, q, kc, kc, rotary_dim=272),
        lambda: paged_prestep(plan, q, k, k, None, None, q, kc, kc, rope_theta=0.0),
        lambda: paged_prestep(plan, q, k, k, None, None, q, kc, kc, rms_eps=-1.0),
    ):
        with pytest.raises(KhqLaunchError):
            call()
