"""The paged operators where a pool runs out, a row ends, or a value is not a number."""
import random

import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean(cuda_ops):
    yield
    assert cuda_ops.lib.khq_b200_paged_status() == 0


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Pool:
    """Steps of a plan on lists: what a request that ended had of the pool goes back, whatever its row has between the pages."""

    def __init__(self, requests, width, page, n_pages):
        self.page, self.n_pages = page, n_pages
        self.table, self.lens = [[-1] * width for _ in range(requests)], [0] * requests
        self.free = list(range(n_pages))

    def step(self, new):
        back = [p for row, c, n in zip(self.table, self.lens, new) if n < 0 for p in row[:-(-c // self.page)] if 0 <= p < self.n_pages]
        self.free += back
        taken = missing = 0
        for b, n in enumerate(new):
            for col in range(-(-self.lens[b] // self.page), -(-(self.lens[b] + n) // self.page) if n >= 0 else 0):
                self.table[b][col] = self.free.pop() if self.free else -1
                taken, missing = taken + (self.table[b][col] >= 0), missing + (self.table[b][col] < 0)
        self.slots = [self.table[b][at // self.page] * self.page + at % self.page if self.table[b][at // self.page] >= 0 else -1
                      for b, n in enumerate(new) for at in range(self.lens[b], self.lens[b] + max(n, 0))]
        self.lens = [0 if n < 0 else c + n for c, n in zip(self.lens, new)]
        return taken, len(back), missing

    def check(self):
        held = [p for row, c in zip(self.table, self.lens) for p in row[:-(-c // self.page)] if p >= 0]
        assert sorted(held + self.free) == list(range(self.n_pages))  # every page exactly once


def run_steps(requests, width, page, n_pages, steps, max_new):
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.paged import PagedPlan

    pool = Pool(requests, width, page, n_pages)
    table, free, count = i32(pool.table), i32(pool.free), i32([n_pages])
    plan = PagedPlan(requests, requests * max_new, page, 24, 4, 256, max_new=max_new)
    for new in steps(pool):
        lens = list(pool.lens)
        plan.build(i32(lens), i32(new), table, free, count)
        taken, back, missing = pool.step(new)
        pool.check()
        assert table.tolist() == pool.table
        assert count.item() == len(pool.free) and free.tolist()[:len(pool.free)] == pool.free
        assert plan.slots.tolist()[:len(pool.slots)] == pool.slots
        assert plan.info.tolist()[:6] == [len(pool.slots), taken, back, missing, 0, len(pool.free)]
    return pool


def test_plan_row_with_a_hole_ends(cuda_ops):
    """A request whose pages ran out takes more of them later: its row is page, none, page.  It ends, and another one takes its pages."""
    pool = run_steps(2, 4, 16, 3, lambda _: [[20, 30], [-1, 10], [0, -1], [32, 0]], 64)
    assert min(pool.table[0][:2]) >= 0 and len(pool.free) == 1
    run_steps(2, 5, 16, 3, lambda _: [[16, 48], [-1, 0], [0, 16], [0, -1], [48, 0]], 64)


def test_plan_row_with_holes_at_its_end(cuda_ops):
    """page, none, page, none."""
    run_steps(3, 8, 16, 3, lambda _: [[16, 16, 32], [-1, 0, 16], [0, 0, 16], [0, 0, -1], [32, 0, 0]], 64)


@pytest.mark.parametrize("requests,n_pages,page,longest", [(5, 9, 16, 60), (40, 60, 32, 300), (1100, 900, 16, 40), (6, 700, 16, 5000)])
def test_plan_pool_that_runs_out_again_and_again(cuda_ops, requests, n_pages, page, longest):
    """Rows with holes of every kind, of up to some hundred pages, ending and starting anew."""
    rng = random.Random(requests)
    width = 4 * -(-longest // page) + 2

    def steps(pool):
        for _ in range(40):
            new = [rng.choice([0, 0, 1, 1, rng.randint(1, longest), rng.randint(1, longest)]) for _ in range(requests)]
            new = [-1 if c > 0 and (c + n > width * page or rng.random() < 0.15) else n for c, n in zip(pool.lens, new)]
            yield new

    run_steps(requests, width, page, n_pages, steps, longest)


def test_plan_gives_back_pages_of_the_pool_only(cuda_ops):
    """Numbers that the pool does not have, and more pages than it has room for."""
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.paged import PagedPlan

    plan = PagedPlan(2, 8, 16, 24, 4, 256)
    free, count = i32([4, 2, 9, 9, 9]), i32([2])
    plan.build(i32([64, 0]), i32([-1, 0]), i32([[1, 5, 1 << 30, 3], [-1] * 4]), free, count)
    assert free.tolist()[:4] == [4, 2, 1, 3] and count.item() == 4 and plan.info.tolist()[:6] == [0, 0, 2, 0, 0, 4]
    plan.build(i32([64, 0]), i32([-1, 0]), i32([[1, 3, 1, 3], [-1] * 4]), free, count)  # pages that are free already
    assert count.item() == 5 and plan.info[5].item() == 5


def test_plan_lanes_with_more_to_move_than_others(cuda_ops):
    """More pages than the plan's threads, by five: the last rounds of its loops are of a part of a warp."""
    run_steps(3, 8300, 16, 8200, lambda _: [[16 * 8192 + 65, 0, 0], [-1, 1, 0], [0, 16 * 8192 + 65, 17]], 16 * 8192 + 65)


@pytest.mark.parametrize("d,H_q,H_kv", [(256, 24, 4), (128, 20, 4)])
@pytest.mark.parametrize("page", [16, 128])
def test_attention_stale_rows_stay_out_every_time(cuda_ops, d, H_q, H_kv, page):
    """NaN behind every request's last token, in both halves of the head dims: overwritten by either CTA of a pair before the products."""
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.paged import PagedPlan, paged_attention

    torch.manual_seed(page)
    ctx, new = [0, 3, 100, 250, 511, 640], [129, 30, 27, 64, 130, 21]
    counts = [-(-(c + n) // page) for c, n in zip(ctx, new)]
    table = [list(range(sum(counts[:b]), sum(counts[:b + 1]))) + [-1] * (max(counts) - counts[b]) for b in range(len(ctx))]
    T = sum(new)
    plan = PagedPlan(len(ctx), T, page, H_q, H_kv, d).build(i32(ctx), i32(new), i32(table))
    q = torch.randn(T, H_q, d, device="cuda").half()
    kc, vc = (torch.randn(sum(counts), page, H_kv, d, device="cuda").half() for _ in range(2))
    for b, (c, n) in enumerate(zip(ctx, new)):
        if (c + n) % page:
            kc[table[b][counts[b] - 1], (c + n) % page:], vc[table[b][counts[b] - 1], (c + n) % page:] = float("nan"), float("nan")
    outs = torch.empty(40, T, H_q, d, dtype=torch.float16, device="cuda")
    for o in outs:
        paged_attention(plan, q, kc, vc, i32(table), o, d ** -0.5)
    want, _, tol, _ = ref.attention(q, torch.nan_to_num(kc), torch.nan_to_num(vc), table, ctx, new, d ** -0.5)
    assert ((outs[0].double() - want).abs() <= tol).all()
    assert all(torch.equal(o, outs[0]) for o in outs[1:])


@pytest.mark.parametrize("pool", [False, True])
def test_plan_drops_what_the_row_has_no_room_for(cuda_ops, pool):
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.paged import PagedPlan

    plan = PagedPlan(4, 64, 16, 24, 4, 256)
    table = i32([[0, 1], [2, 3], [4, 5], [6, -1 if pool else 7]])
    args = (i32([7, 8, 9] + [-1] * 7), i32([3])) if pool else ()
    plan.build(i32([30, 32, 40, 5]), i32([5, 3, 2, 20]), table, *args)
    assert plan.cu_new.tolist() == [0, 2, 2, 2, 22]
    assert plan.kv_lens.tolist() == [32, 32, 32, 25]
    last = 9 if pool else 7
    assert table.tolist() == [[0, 1], [2, 3], [4, 5], [6, last]]
    assert plan.positions.tolist() == [30, 31] + list(range(5, 25)) + [-1] * 42
    assert plan.slots.tolist() == [30, 31] + list(range(6 * 16 + 5, 7 * 16)) + list(range(last * 16, last * 16 + 9)) + [-1] * 42
    assert plan.info.tolist()[:5] == [22, int(pool), 0, 0, 8]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H_q,H_kv,d,ctx,new", [(24, 4, 256, [100, 7, 300], [1, 1, 1]), (24, 4, 256, [20000, 9], [1, 2]), (20, 4, 128, [40, 9000], [2, 1]),
                                               (24, 4, 256, [300, 20, 3000], [40, 1, 30]), (20, 4, 128, [5000], [90])])
def test_attention_rows_that_are_not_numbers(cuda_ops, dtype, H_q, H_kv, d, ctx, new):
    """A query of NaNs: NaN in that row's output and lse, nowhere else.  The same for a key of NaNs in the rows that attend it."""
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.paged import PagedPlan, paged_attention

    torch.manual_seed(len(ctx))
    page, T = 64, sum(new)
    counts = [-(-(c + n) // page) for c, n in zip(ctx, new)]
    table = [list(range(sum(counts[:b]), sum(counts[:b + 1]))) + [-1] * (max(counts) - counts[b]) for b in range(len(ctx))]
    pool = sum(counts)
    plan = PagedPlan(len(ctx), T, page, H_q, H_kv, d, max_new=max(new)).build(i32(ctx), i32(new), i32(table))
    q = torch.randn(T, H_q, d, device="cuda").to(dtype)
    kc, vc = (torch.randn(pool, page, H_kv, d, device="cuda").to(dtype) for _ in range(2))
    rows = sorted({0, T // 2, T - 1})
    bad_q = q.clone()
    for t in rows:
        bad_q[t, (5 * t) % H_q] = float("nan")
    want, want_lse, tol, lse_tol = ref.attention(q, kc, vc, table, ctx, new, d ** -0.5)

    def check(queries, keys, bad):
        out, lse = torch.full_like(q, 7.0), torch.full((T, H_q), 7.0, device="cuda")
        paged_attention(plan, queries, keys, vc, i32(table), out, d ** -0.5, lse=lse)
        assert torch.isnan(out[bad]).all() and torch.isnan(lse[bad]).all()
        assert ((out.double() - want).abs() <= tol)[~bad].all() and ((lse.double() - want_lse).abs() <= lse_tol)[~bad].all()

    bad = torch.zeros(T, H_q, dtype=torch.bool, device="cuda")
    for t in rows:
        bad[t, (5 * t) % H_q] = True
    check(bad_q, kc, bad)
    # the first request's keys of the last kv head, from its first new token's page on: its rows of that head
    first = ctx[0] // page
    bad_k = kc.clone()
    for col in range(first, counts[0]):
        bad_k[table[0][col], :, H_kv - 1] = float("nan")
    bad = torch.zeros_like(bad)
    bad[:new[0], (H_kv - 1) * (H_q // H_kv):] = True
    check(q, bad_k, bad)


def test_plan_counts_dropped_rows_up_to_the_largest_int(cuda_ops):
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.paged import PagedPlan

    plan = PagedPlan(4096, 8, 16, 24, 4, 256)
    lens, table = i32([0] * 4096), torch.zeros(4096, 4, dtype=torch.int32, device="cuda")
    for new, dropped in ((1 << 20, 2 ** 31 - 1), (2 ** 31 - 1, 2 ** 31 - 1), (1000, 4096 * 1000 - 8)):
        plan.build(lens, i32([new] * 4096), table)
        assert plan.info.tolist()[:5] == [8, 0, 0, 0, dropped]
    plan.build(lens, i32([2 ** 31 - 1] + [0] * 4095), table)
    assert plan.info[4].item() == 2 ** 31 - 1 - 8


def test_plan_without_a_pool_has_no_free_pages(cuda_ops):
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.paged import PagedPlan

    plan = PagedPlan(1, 8, 16, 24, 4, 256)
    table = i32([[-1, -1]])
    plan.info.fill_(77)
    plan.build(i32([0]), i32([8]), table, i32([0, 1, 2]), i32([3]))
    assert plan.info.tolist() == [8, 1, 0, 0, 0, 2, 0, 0]
    plan.info.fill_(77)
    plan.build(i32([0]), i32([8]), table)
    assert plan.info.tolist() == [8, 0, 0, 0, 0, 0, 0, 0]


def test_plan_built_at_once_on_another_stream(cuda_ops):
    """The plan is made while the current stream is busy and built on an idle one: nothing of the first may come in behind."""
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.paged import PagedPlan

    lens, new, table = i32([5, 0]), i32([3, 20]), i32([[0, -1], [1, 2]])
    PagedPlan(2, 32, 16, 24, 4, 256).build(lens, new, table)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(20_000_000)  # some 10 ms
    plan = PagedPlan(2, 32, 16, 24, 4, 256)
    with torch.cuda.stream(side):
        plan.build(lens, new, table)
    torch.cuda.synchronize()
    assert plan.info.tolist() == [23, 0, 0, 0, 0, 0, 0, 0] and plan.cu_new.tolist() == [0, 3, 23]


def test_pages_behind_a_wait_that_ran_out_are_not_compressed(cuda_ops, monkeypatch):
    import numpy as np

    import cases
    from bonsai_mojo_1bit_optimization_t4_cuda_b200 import paged
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.engine import BatchEngine
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.lib import KhqLaunchError
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.runtime import KhqRuntime

    paged.check_status()  # clean, on this GPU
    rng = np.random.default_rng(0)
    k, v = cases.synth.make_kv(rng, 128, cases.synth.channel_scales(rng), cases.synth.channel_scales(rng))
    tables = cases.synth.make_tables(rng, 3, k.reshape(-1, 256), v.reshape(-1, 256), vq_scale=1.0 / 16.0)
    rt = KhqRuntime(cuda_ops)
    assert rt.khq_activate([tables], max_seq=512)
    rt.khq_init_layer(3, 24, 4, 256)
    eng = BatchEngine([tables], [128], [128])
    kc, vc, uc = (torch.ones(3, 128, 4, 256, dtype=torch.float16, device="cuda") for _ in range(3))
    word = [1]
    monkeypatch.setattr(paged, "_read_status", lambda device: word[0])
    with pytest.raises(KhqLaunchError):
        rt.khq_adopt_pages(3, kc, vc, uc, i32([0, 1, 2]), 300)
    with pytest.raises(KhqLaunchError):
        eng.load_pages(0, 0, kc, vc, uc, i32([0, 1]))
    assert rt.layers[3].write_pos == 0 and (eng.ring_k[0] == 0).all() and (eng.pay[0]["k_mask"] == 0).all()
    word[0] = 0
    assert rt.khq_adopt_pages(3, kc, vc, uc, i32([0, 1, 2]), 300)
    eng.load_pages(0, 0, kc, vc, uc, i32([0, 1]))
