"""How the norms' gradients are launched: no worker waits for another to leave."""
import json

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 250, 256, 384, 512, 1000, 1024, 1536, 1999, 2048, 2050, 4096, 8192])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bias, gated", [(False, False), (True, False), (False, True), (True, True)])
def test_all_workers_of_the_norm_gradients_are_resident_at_once(lib, tmp_path, D, dtype, bias, gated):
    """A worker takes consecutive rows; a second wave of them would take as long as the first however few they are. The launch's registers and shared memory say how many CTAs a
    multiprocessor holds: 65,536 registers, 228 KB of which each CTA costs 1 KB more than it asks for, 2,048 threads."""
    from torch.profiler import ProfilerActivity, profile
    R = 20000
    draw = lambda *s: torch.zeros(*s, device="cuda", dtype=dtype)
    p = torch.ones(D, device="cuda")
    kw = dict(post="layer", pre="rms", post_weight=p, pre_weight=p, **(dict(post_bias=p, pre_bias=p) if bias else {}), **(dict(gate=draw(1, D), gate_rows=R) if gated else {}))
    operands = [draw(R, D) for _ in range(4)]
    lib.norm_residual_backward(*operands, **kw)
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as prof:
        lib.norm_residual_backward(*operands, **kw)
        torch.cuda.synchronize()
    prof.export_chrome_trace(str(tmp_path / "trace.json"))
    with open(tmp_path / "trace.json") as f:
        launches = [e["args"] for e in json.load(f)["traceEvents"] if e.get("cat") == "kernel" and "norm_backward_kernel" in e["name"]]
    assert len(launches) == 1
    a = launches[0]
    threads = a["block"][0]
    resident = min(65536 // (a["registers per thread"] * threads), 228 * 1024 // (a["shared memory"] + 1024), 2048 // threads)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    print(D, dtype, bias, gated, a["grid"], threads, a["registers per thread"], a["shared memory"], resident)
    assert a["grid"][0] <= sms * resident
