"""How the norms' gradients are launched: no worker waits for another to leave."""
import json
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROWS = 20000
FORMS = [(D, dtype, bias, gated) for D in (64, 250, 256, 384, 512, 1000, 1024, 1536, 1999, 2048, 2050, 4096, 8192) for dtype in ("bfloat16", "float32") for bias in (False, True)
         for gated in (False, True)]


def profile_all(path):
    """Every form's gradients once, under one profiler: run in a process of its own, which leaves the tests' process without one."""
    import torch
    from torch.profiler import ProfilerActivity, profile
    import __graft_entry__ as entry
    lib = entry.load_package()

    def calls():
        for D, dtype, bias, gated in FORMS:
            draw = lambda *s: torch.zeros(*s, device="cuda", dtype=getattr(torch, dtype))
            p, x = torch.ones(D, device="cuda"), draw(ROWS, D)
            kw = dict(post="layer", pre="rms", post_weight=p, pre_weight=p, **(dict(post_bias=p, pre_bias=p) if bias else {}), **(dict(gate=draw(1, D), gate_rows=ROWS) if gated else {}))
            lib.norm_residual_backward(x, x, x, x, **kw)
        torch.cuda.synchronize()

    calls()
    with profile(activities=[ProfilerActivity.CUDA]) as prof:
        calls()
    prof.export_chrome_trace(path)


@pytest.fixture(scope="module")
def launches(tmp_path_factory):
    path, here = str(tmp_path_factory.mktemp("launches") / "trace.json"), os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([os.path.dirname(here), here]))
    r = subprocess.run([sys.executable, "-c", f"import test_gpu_residual_launches as t; t.profile_all({path!r})"], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    with open(path) as f:
        kernels = sorted((e for e in json.load(f)["traceEvents"] if e.get("cat") == "kernel" and "norm_backward_kernel" in e["name"]), key=lambda e: e["ts"])
    assert len(kernels) == len(FORMS)
    return {form: k["args"] for form, k in zip(FORMS, kernels)}


@pytest.mark.parametrize("D, dtype, bias, gated", FORMS)
def test_all_workers_of_the_norm_gradients_are_resident_at_once(launches, D, dtype, bias, gated):
    """A worker takes consecutive rows; a second wave of them would take as long as the first however few they are. The launch's registers and shared memory say how many CTAs a
    multiprocessor holds: 65,536 registers, 228 KB of which each CTA costs 1 KB more than it asks for, 2,048 threads."""
    import torch
    a = launches[D, dtype, bias, gated]
    threads = a["block"][0]
    resident = min(65536 // (a["registers per thread"] * threads), 228 * 1024 // (a["shared memory"] + 1024), 2048 // threads)
    assert a["grid"][0] <= torch.cuda.get_device_properties(0).multi_processor_count * resident, a
