"""The paged operators' refusals and sizes through the C ABI: nothing here reaches a launch."""
import ctypes
import struct

import pytest

from bonsai_mojo_1bit_optimization_t4_cuda_b200 import lib as _lib

P = 4096  # an aligned address that is never used
# the argument structs of include/khq_b200.h, field by field
PLAN_ARGS, PRESTEP_ARGS, ATTN_ARGS = struct.Struct("@12PNq9i0q"), struct.Struct("@11P17q7i2f0q"), struct.Struct("@9P2N12qq10if0q")


@pytest.fixture(scope="module")
def lib():
    from bonsai_mojo_1bit_optimization_t4_cuda_b200 import build

    build.build()
    return _lib.load()


PLAN = [("ctx_lens", P), ("new_lens", P), ("block_table", P), ("free_list", P), ("free_count", P), ("free_count_out", P), ("cu_new", P), ("kv_lens", P),
        ("positions", P), ("slots", P), ("info", P), ("schedule", P), ("schedule_bytes", 1 << 40), ("table_stride", 9), ("requests", 3), ("max_pages", 9),
        ("n_pages", 40), ("page_size", 16), ("max_tokens", 64), ("max_new", 64), ("H_q", 24), ("H_kv", 4), ("d", 256)]
PRESTEP = ([(n, P) for n in ("q", "k", "v", "q_norm_w", "k_norm_w", "q_out", "k_cache", "v_cache", "u_cache", "positions", "slots")]
           + [(n, 256) for n in ("q0", "q1", "k0", "k1", "v0", "v1", "o0", "o1", "kc0", "kc1", "kc2", "vc0", "vc1", "vc2", "uc0", "uc1", "uc2")]
           + [("tokens", 5), ("n_pages", 4), ("page_size", 16), ("H_q", 24), ("H_kv", 4), ("d", 256), ("rotary_dim", 64), ("rope_theta", 1e7), ("rms_eps", 1e-6)])
ATTN = ([(n, P) for n in ("q", "gate", "k_cache", "v_cache", "block_table", "schedule", "out", "lse", "workspace")]
        + [("schedule_bytes", 1 << 40), ("workspace_bytes", 1 << 40)]
        + [(n, 256) for n in ("q0", "q1", "g0", "g1", "o0", "o1", "kc0", "kc1", "kc2", "vc0", "vc1", "vc2")]
        + [("table_stride", 9), ("tokens", 5), ("max_tokens", 64), ("max_new", 64), ("requests", 3), ("max_pages", 9), ("n_pages", 40), ("page_size", 16),
           ("H_q", 24), ("H_kv", 4), ("d", 256), ("scale", 0.1)])


def call(fn, layout, fields, **change):
    values = dict(fields)
    assert set(change) <= set(values)
    values.update(change)
    return fn(layout.pack(*values.values()), None)


def test_layouts_are_the_structs(tmp_path):
    import subprocess
    from pathlib import Path

    src = tmp_path / "sizes.c"
    src.write_text('#include "khq_b200.h"\n#include <stdio.h>\nint main(void) { printf("%zu %zu %zu", sizeof(khq_paged_plan_args), '
                   'sizeof(khq_paged_prestep_args), sizeof(khq_paged_attn_args)); return 0; }\n')
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-I", str(Path(__file__).resolve().parent.parent / "include"), str(src), "-o", str(exe)], check=True)
    want = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert [PLAN_ARGS.size, PRESTEP_ARGS.size, ATTN_ARGS.size] == want


@pytest.mark.parametrize("change,code", [
    (dict(requests=0), -100), (dict(max_tokens=0), -100), (dict(max_new=-1), -100), (dict(max_pages=0), -100), (dict(ctx_lens=0), -100),
    (dict(slots=0), -100), (dict(schedule=0), -100), (dict(free_count=0), -100), (dict(free_count_out=0), -100), (dict(n_pages=0), -100),
    (dict(free_list=0), -100), (dict(page_size=17), -103), (dict(page_size=0), -103), (dict(H_q=25), -103), (dict(d=64), -103), (dict(requests=16385), -103),
    (dict(max_tokens=(1 << 20) + 1), -103), (dict(table_stride=8), -103), (dict(max_pages=1 << 27, table_stride=1 << 27), -103),
    (dict(ctx_lens=P + 2), -104), (dict(slots=P + 4), -104), (dict(schedule=P + 8), -104), (dict(schedule_bytes=64), -105),
])
def test_plan_refusals(lib, change, code):
    assert call(lib.launch_khq_paged_plan, PLAN_ARGS, PLAN, **change) == code


@pytest.mark.parametrize("change,code", [
    (dict(tokens=0), -100), (dict(q=0), -100), (dict(v_cache=0), -100), (dict(slots=0), -100), (dict(n_pages=0), -100), (dict(rope_theta=0.0), -100),
    (dict(rope_theta=float("nan")), -100), (dict(rms_eps=-1e-6), -100), (dict(d=64), -103), (dict(rotary_dim=20), -103), (dict(rotary_dim=-16), -103),
    (dict(rotary_dim=272), -103), (dict(page_size=8), -103), (dict(k=P + 8), -104), (dict(u_cache=P + 2), -104), (dict(q_norm_w=P + 4), -104),
    (dict(q1=252), -104), (dict(vc2=4), -104), (dict(uc0=1), -104), (dict(slots=P + 4), -104),
])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_prestep_refusals(lib, dtype, change, code):
    assert call(getattr(lib, "launch_khq_paged_prestep_" + dtype), PRESTEP_ARGS, PRESTEP, **change) == code


@pytest.mark.parametrize("change,code", [
    (dict(tokens=0), -100), (dict(q=0), -100), (dict(out=0), -100), (dict(workspace=0), -100), (dict(schedule=0), -100), (dict(scale=0.0), -100),
    (dict(scale=-0.1), -100), (dict(scale=float("nan")), -100), (dict(scale=float("inf")), -100), (dict(max_new=0), -100), (dict(d=192), -103),
    (dict(H_q=26), -103), (dict(page_size=24), -103), (dict(table_stride=8), -103), (dict(q=P + 8), -104), (dict(gate=P + 8), -104), (dict(lse=P + 2), -104),
    (dict(workspace=P + 128), -104), (dict(o1=4), -104), (dict(kc1=12), -104), (dict(vc0=-256), -104), (dict(schedule_bytes=100), -105),
    (dict(workspace_bytes=1000), -105),
])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_attention_refusals(lib, dtype, change, code):
    assert call(getattr(lib, "launch_khq_paged_attn_" + dtype), ATTN_ARGS, ATTN, **change) == code


def test_extension_knows_the_plan(lib):
    from bonsai_mojo_1bit_optimization_t4_cuda_b200 import paged

    assert paged._load_host().info_bytes() == ctypes.sizeof(paged._PlanInfo)


def test_extension_refuses_what_is_no_tensor_of_the_plan(lib):
    """Host tensors and other objects: refused before anything is launched."""
    import torch

    from bonsai_mojo_1bit_optimization_t4_cuda_b200 import paged

    host = paged._load_host()
    info = paged._PlanInfo(0, 24, 4, 256, 16, 4, 64, 64, 2, 3)
    at = ctypes.addressof(info)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    half = lambda *s: torch.zeros(*s, dtype=torch.float16)
    q, k, c, table = half(5, 24, 256), half(5, 4, 256), half(9, 16, 4, 256), i32(2, 3)
    assert host.build(at, i32(2), i32(2), table, None, None, None) == -1000
    assert host.build(at, 7, i32(2), table, None, None, None) == -1000
    assert host.prestep(at, q, k, k, None, None, q, c, c, None, 64, 1e7, 1e-6) == -1000
    assert host.attention(at, q, c, c, table, q, 0.1, None, None, None) == -1000
    assert host.attention(at, q.float(), c, c, table, q, 0.1, None, None, None) == -1000
    for call in (lambda: host.build(at, 1), lambda: host.attention(at)):
        with pytest.raises(TypeError):
            call()


def test_null_arguments(lib):
    for name in ("launch_khq_paged_plan", "launch_khq_paged_prestep_fp16", "launch_khq_paged_prestep_bf16", "launch_khq_paged_attn_fp16",
                 "launch_khq_paged_attn_bf16"):
        assert getattr(lib, name)(None, None) == -100


def test_sizes(lib):
    assert lib.khq_b200_paged_schedule_bytes(0, 8, 8, 24, 4, 256) == 0
    assert lib.khq_b200_paged_schedule_bytes(2, 8, 8, 24, 5, 256) == 0
    assert lib.khq_b200_paged_workspace_bytes(1, 24, 4, 64) == 0
    for requests, tokens, new in ((1, 1, 1), (3, 4096, 2048), (16384, 1 << 20, 1 << 20)):
        n = lib.khq_b200_paged_schedule_bytes(requests, tokens, new, 24, 4, 256)
        assert n > 16 * requests
        w = lib.khq_b200_paged_workspace_bytes(new, 24, 4, 256)
        assert w > 0 and w % 256 == 0
