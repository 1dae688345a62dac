"""Prompts in chunks end to end: plan, pre-step and attention chunk by chunk for two prompts of different lengths, then their pages
become the compressed state of a runtime and of a batch engine, and decoding goes on."""
import numpy as np
import pytest

import cases
from cases import D, H_KV, H_Q, SCALE

pytestmark = pytest.mark.gpu
STATE = (("kmask", 16), ("kpay", 40), ("knorm", 1), ("krn", 1), ("vpay", 104), ("vnorm", 1), ("vrn", 1), ("vsm", 4))


@pytest.mark.parametrize("page,T,chunk", [(128, (700, 301), 256), (16, (384, 40), 100), (64, (257, 513), 333)])
def test_chunked_prompts_become_compressed_state(cuda_ops, page, T, chunk):
    import torch

    from bonsai_mojo_1bit_optimization_t4_cuda_b200.engine import BatchEngine
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.paged import PagedPlan, paged_attention, paged_prestep
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.runtime import KhqRuntime

    B = len(T)
    rng = np.random.default_rng(sum(T))
    sk, sv = cases.synth.channel_scales(rng), cases.synth.channel_scales(rng)
    sample_k, sample_v = cases.synth.make_kv(rng, 128, sk, sv)
    table = cases.synth.make_tables(rng, 3, sample_k.reshape(-1, D), sample_v.reshape(-1, D), vq_scale=1.0 / 16.0)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
    qg = [dev(rng.standard_normal((t, H_Q, 2 * D)).astype(np.float16)) for t in T]
    k = [dev((rng.standard_normal((t, H_KV, D)) * sk).astype(np.float16)) for t in T]
    v = [dev((rng.standard_normal((t, H_KV, D)) * sv).astype(np.float16)) for t in T]
    qw, kw = (dev((1 + 0.1 * rng.standard_normal(D)).astype(np.float32)) for _ in range(2))

    # ---- chunks through the pages: queries normed in place, K rotated, K un-rotated and V side by side in one pool --------------
    pool = sum(-(-t // page) for t in T) + 3
    kc = torch.zeros(pool, page, H_KV, D, dtype=torch.float16, device="cuda")
    uv = torch.zeros(pool, 2, page, H_KV, D, dtype=torch.float16, device="cuda")
    uc, vc = uv[:, 0], uv[:, 1]
    blocks = torch.full((B, max(-(-t // page) for t in T)), -1, dtype=torch.int32, device="cuda")
    free, count = torch.arange(pool - 1, -1, -1, dtype=torch.int32, device="cuda"), torch.tensor([pool], dtype=torch.int32, device="cuda")
    plan = PagedPlan(B, B * chunk, page, H_Q, H_KV, D, max_new=chunk)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    done, outs, qs = [0] * B, [[] for _ in T], [[] for _ in T]
    while any(d < t for d, t in zip(done, T)):
        n = [min(chunk, t - d) for d, t in zip(done, T)]
        plan.build(i32(done), i32(n), blocks, free, count)
        part = lambda xs: torch.cat([x[d:d + m] for x, d, m in zip(xs, done, n)])
        q = part(qg)
        out = torch.empty(sum(n), H_Q, D, dtype=torch.float16, device="cuda")
        paged_prestep(plan, q[..., :D], part(k), part(v), qw, kw, q[..., :D], kc, vc, uc)
        paged_attention(plan, q[..., :D], kc, vc, blocks, out, SCALE, gate=q[..., D:])
        at = 0
        for b in range(B):
            outs[b].append(out[at:at + n[b]])
            qs[b].append(q[at:at + n[b]])
            at += n[b]
        done = [d + m for d, m in zip(done, n)]
    assert cuda_ops.lib.khq_b200_paged_status() == 0
    assert count.item() == pool - sum(-(-t // page) for t in T)

    boundary = []
    states = []
    for b in range(B):
        rows = torch.tensor([int(blocks[b, t // page]) * page + t % page for t in range(T[b])], device="cuda")
        take = lambda c: c.reshape(-1, H_KV, D)[rows].contiguous()
        kr, ku, vv = take(kc), take(uc), take(vc)
        assert torch.equal(vv, v[b])
        # the same prompt at once
        whole, adopted = KhqRuntime(cuda_ops), KhqRuntime(cuda_ops)
        for rt in (whole, adopted):
            assert rt.khq_activate([table], max_seq=1024)
            rt.khq_init_layer(3, H_Q, H_KV, D)
        out = torch.empty(T[b], H_Q, D, dtype=torch.float16, device="cuda")
        assert whole.khq_prefill(3, torch.cat(qs[b]), ku, kr, vv, out, SCALE)
        # both kernels round weights and outputs to 16 bits: half a step (2^-11) each of outputs up to the largest |v|
        assert (torch.cat(outs[b]).float() - out.float()).abs().max().item() <= 4 * 2.0 ** -11 * vv.abs().max().item()
        assert adopted.khq_adopt_pages(3, kc, vc, uc, blocks[b], T[b])
        La, Lw = adopted.layers[3], whole.layers[3]
        assert (La.boundary, La.write_pos) == (Lw.boundary, Lw.write_pos)
        assert [(e.boundary, e.write_pos) for e in adopted.events] == [(e.boundary, e.write_pos) for e in whole.events]
        for key, w in STATE:
            n = La.boundary * H_KV * w
            assert torch.equal(La.t[key][:n].view(torch.uint8), Lw.t[key][:n].view(torch.uint8)), key
        live = [t % 256 for t in range(La.boundary, T[b])]
        for ring in ("ring_k", "ring_v", "ring_u"):
            assert torch.equal(La.t[ring].view(256, -1)[live], Lw.t[ring].view(256, -1)[live]), ring
        assert not adopted.khq_adopt_pages(3, kc, vc, uc, blocks[b], T[b])  # not a fresh layer any more
        boundary.append(La.boundary)
        states.append(Lw)

    # ---- the same pages into a batch engine ------------------------------------------------------------------------------
    eng = BatchEngine([table], boundary, [t - c for t, c in zip(T, boundary)], grow_tokens=256)
    for b in range(B):
        eng.load_pages(0, b, kc, vc, uc, blocks[b])
        names = dict(kmask="k_mask", kpay="k_payload", knorm="k_norms", krn="k_r_norms", vpay="v_payload", vnorm="v_norms", vrn="v_r_norms", vsm="v_shared_meta")
        for key, w in STATE:
            r0, n = int(eng.row_off[b]) * w, boundary[b] * H_KV * w
            assert torch.equal(eng.pay[0][names[key]][r0:r0 + n].view(torch.uint8), states[b].t[key][:n].view(torch.uint8)), key
        live = [t % 256 for t in range(boundary[b], T[b])]
        for ring, have in (("ring_k", eng.ring_k), ("ring_v", eng.ring_v), ("ring_u", eng.ring_u)):
            assert torch.equal(have[0][b][live], states[b].t[ring].view(256, -1)[live]), ring
    eng.h_q.copy_(torch.from_numpy(rng.standard_normal(eng.h_q.shape).astype(np.float16)))
    eng.h_k.copy_(torch.from_numpy(rng.standard_normal(eng.h_k.shape).astype(np.float16)))
    eng.h_v.copy_(torch.from_numpy(rng.standard_normal(eng.h_v.shape).astype(np.float16)))
    out = eng.decode_step()
    torch.cuda.synchronize()
    assert torch.isfinite(out.float()).all()


def test_adopting_refuses_what_it_cannot_read(cuda_ops):
    import torch

    from bonsai_mojo_1bit_optimization_t4_cuda_b200.runtime import KhqRuntime

    rng = np.random.default_rng(0)
    sample_k, sample_v = cases.synth.make_kv(rng, 128, cases.synth.channel_scales(rng), cases.synth.channel_scales(rng))
    table = cases.synth.make_tables(rng, 3, sample_k.reshape(-1, D), sample_v.reshape(-1, D), vq_scale=1.0 / 16.0)
    rt = KhqRuntime(cuda_ops)
    assert not rt.khq_adopt_pages(3, None, None, None, None, 5)  # not active
    assert rt.khq_activate([table], max_seq=512)
    rt.khq_init_layer(3, H_Q, H_KV, D)
    cache = lambda *s, dt=torch.float16: torch.zeros(*s, dtype=dt, device="cuda")
    kc, vc, uc = (cache(4, 128, H_KV, D) for _ in range(3))
    row = torch.tensor([0, 1, -1, 7], dtype=torch.int32, device="cuda")
    heads_first = cache(4, H_KV, 128, D).permute(0, 2, 1, 3)
    for args in ((kc, vc, uc, row, 300), (kc, vc, uc, row[:2], 300), (kc, vc, uc, row.long(), 100), (kc, vc, uc, row, 0), (kc.bfloat16(), vc, uc, row, 100),
                 (kc, vc[:3], uc, row, 100), (heads_first, heads_first, heads_first, row, 100), (kc, cache(4, 2, 128, H_KV, D)[:, 0], uc, row, 100)):
        with pytest.raises(ValueError):
            rt.khq_adopt_pages(3, *args)
    assert rt.layers[3].write_pos == 0
    assert rt.khq_adopt_pages(3, kc, vc, uc, row, 256)
