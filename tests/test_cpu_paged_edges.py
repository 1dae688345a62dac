"""The paged operators' host side: what is refused before anything reaches the GPU."""
import pytest
import torch

from bonsai_mojo_1bit_optimization_t4_cuda_b200 import paged


def test_prompt_pages_on_the_host_are_refused():
    """Their addresses would go to kernels."""
    cache = torch.zeros(4, 16, 4, 256, dtype=torch.float16)
    row = torch.tensor([0, 1, 2, 3], dtype=torch.int32)
    for device in (None, torch.device("cuda", 0)):
        with pytest.raises(ValueError, match="CUDA|cuda:0"):
            paged.prompt_pages(row, 40, cache, cache, cache, 4, 256, *([device] if device else []))


def test_adopting_pages_on_the_host_is_refused():
    """Through the runtime, before any launch."""
    import numpy as np

    import cases
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.runtime import KhqRuntime

    class Ops:
        def compress_runs(self, *args):
            raise AssertionError("host addresses given to a kernel")

    rng = np.random.default_rng(0)
    k, v = cases.synth.make_kv(rng, 128, cases.synth.channel_scales(rng), cases.synth.channel_scales(rng))
    table = cases.synth.make_tables(rng, 3, k.reshape(-1, 256), v.reshape(-1, 256))
    rt = KhqRuntime(Ops(), device="cpu")
    assert rt.khq_activate([table], max_seq=1024)
    rt.khq_init_layer(3, 24, 4, 256)
    cache = torch.zeros(5, 128, 4, 256, dtype=torch.float16)
    with pytest.raises(ValueError):
        rt.khq_adopt_pages(3, cache, cache, cache, torch.arange(5, dtype=torch.int32), 640)
    assert rt.layers[3].write_pos == 0


@pytest.mark.parametrize("word", [1, 2, -1])
def test_a_wait_that_ran_out_is_reported(monkeypatch, word):
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.lib import KhqLaunchError

    seen = []
    monkeypatch.setattr(paged, "_read_status", lambda device: seen.append(device) or word)
    plan = object.__new__(paged.PagedPlan)
    plan.device = 3
    with pytest.raises(KhqLaunchError, match="not to be trusted") as e:
        plan.check()
    assert e.value.code == word and seen == [3]
    monkeypatch.setattr(paged, "_read_status", lambda device: 0)
    plan.check()
    paged.check_status()


def test_the_library_is_built_without_torch(monkeypatch, tmp_path, capsys):
    """One source stands for all: what matters is that nvcc runs and that the extension's absence ends nothing."""
    import sys

    from bonsai_mojo_1bit_optimization_t4_cuda_b200 import build

    monkeypatch.setattr(build, "LIB_PATH", tmp_path / build.LIB_NAME)
    monkeypatch.setattr(build, "SOURCES", ["khq_calib.cu"])
    monkeypatch.setattr(build, "host_path", lambda: tmp_path / "host.so")
    monkeypatch.setitem(sys.modules, "torch", None)  # an import of it raises
    assert build.build() == build.LIB_PATH
    assert (tmp_path / build.LIB_NAME).exists() and not (tmp_path / "host.so").exists()
    assert "extension was not built" in capsys.readouterr().err
    with pytest.raises(ImportError):
        build.build_host()


def test_an_extension_for_another_torch_or_python_is_not_taken(monkeypatch):
    from importlib import metadata

    from bonsai_mojo_1bit_optimization_t4_cuda_b200 import build
    from bonsai_mojo_1bit_optimization_t4_cuda_b200.lib import KhqLibraryError

    build.build_host()
    assert not build.needs_host_build()
    monkeypatch.setattr(metadata, "version", lambda name: "1.0.0")
    assert build.needs_host_build()
    monkeypatch.setattr(paged, "_host", None)
    with pytest.raises(KhqLibraryError, match="build it"):
        paged._load_host()


def test_refusals_say_what_does_not_fit():
    plan = object.__new__(paged.PagedPlan)
    plan.device, plan.max_requests, plan.max_tokens = -1, 4, 8  # -1: where host tensors are
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    for args, error, text in (
        ((i32(2), i32(2), i32(2, 0), None, None, None), ValueError, "block_table"),
        ((i32(2), i32(3), i32(2, 1), None, None, None), ValueError, "new_lens"),
        ((i32(2), i32(2), i32(2, 1), None, i32(1), None), ValueError, "free_count without"),
        ((i32(2), i32(2), i32(2, 1), None, None, i32(1)), ValueError, "free_count without"),
        ((i32(2), i32(2), i32(2, 1), i32(5), None, None), ValueError, "free_list without"),
        ((i32(2), i32(2), i32(2, 1), i32(5), i32(2), None), ValueError, "free_count"),
        (([0, 0], i32(2), i32(2, 1), None, None, None), TypeError, "ctx_lens"),
        ((i32(2), [0, 0], i32(2, 1), None, None, None), TypeError, "new_lens"),
    ):
        with pytest.raises(error, match=text):
            plan._look_at_build(*args)
    plan._look_at_build(i32(2), i32(2), i32(2, 1), None, None, None)  # nothing to say
    plan._prestep = plan._attention = lambda *args: paged._NO_FIT
    plan._at = 0
    with pytest.raises(TypeError, match="q"):
        paged.paged_prestep(plan, 7, None, None, None, None, None, None, None)
    with pytest.raises(TypeError, match="q"):
        paged.paged_attention(plan, None, None, None, None, None, 0.1)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_a_scale_that_overflows_is_refused(dtype):
    """2.5e38 is finite, its product with log2 e is not."""
    from test_cpu_paged import ATTN, ATTN_ARGS, call

    from bonsai_mojo_1bit_optimization_t4_cuda_b200 import build, lib

    build.build()
    assert call(getattr(lib.load(), "launch_khq_paged_attn_" + dtype), ATTN_ARGS, ATTN, scale=2.5e38, schedule_bytes=100) == -100
    assert call(getattr(lib.load(), "launch_khq_paged_attn_" + dtype), ATTN_ARGS, ATTN, scale=2e38, schedule_bytes=100) == -105  # the next look
