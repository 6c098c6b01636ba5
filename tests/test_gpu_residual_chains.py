"""The residual operators directly behind the kernels that write what they read: a chain of calls, on a stream and captured, gives the bits of the same calls made one by one with the device
idle in between."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


class Chain:
    """Norms and a layer whose parameters lie in one arena, stepped by Adam between any two calls that read them; nothing else runs between an optimizer step and its reader."""

    def __init__(self, lib, R, D, dtype, post, pre, bias, gate_rows, offset, meet):
        g = torch.Generator(device="cuda").manual_seed(R + D)
        self.lib, self.meet, self.kinds, self.gate_rows = lib, meet, (post, pre), gate_rows
        names = ["post_weight", "pre_weight"] + (["post_bias", "pre_bias"] if bias else [])
        n = offset + (len(names) + 1) * D
        self.params, self.grads, self.m, self.v = (torch.zeros(n, device="cuda") for _ in range(4))
        self.state = torch.zeros(4, device="cuda", dtype=torch.int32)
        lib.check(lib.lib().b200rl_adam_reset(self.state.data_ptr(), None))
        self.params.copy_(torch.randn(n, device="cuda", generator=g))
        part = lambda t, i: t[offset + i * D:offset + (i + 1) * D]
        self.p = {k: part(self.params, i) for i, k in enumerate(names)}
        self.g = {"d_" + k: part(self.grads, i) for i, k in enumerate(names)}
        self.bias = part(self.params, len(names))
        self.grads[offset + len(names) * D:] = 0.3
        draw = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)
        self.branch, self.residual, self.d_out, self.d_normed = (draw(R, D) for _ in range(4))
        self.gate = draw(-(-R // gate_rows), D) if gate_rows else None
        self.out, self.normed, self.d_branch, self.d_residual = (torch.empty_like(self.branch) for _ in range(4))
        self.W, self.x, self.few = draw(D, 40).to(BF16), draw(100, 40).to(BF16), draw(5, 40).to(BF16)
        self.y, self.y_few = torch.empty(100, D, device="cuda", dtype=BF16), torch.empty(5, D, device="cuda", dtype=BF16)
        self.counter = torch.zeros(1, device="cuda", dtype=torch.int64)
        self.hyper = lib.AdamHyper(alpha=0.05)

    def adam(self):
        L = self.lib
        L.check(L.lib().b200rl_adam_step(self.params.data_ptr(), self.grads.data_ptr(), self.m.data_ptr(), self.v.data_ptr(), self.params.numel(), self.hyper, self.state.data_ptr(),
                                         C.c_void_p(torch.cuda.current_stream().cuda_stream)))
        self.meet()

    def norms(self):
        post, pre = self.kinds
        return dict(post=post, pre=pre, gate=self.gate, gate_rows=self.gate_rows or 1, scale=0.7, **self.p)

    def update(self):
        L, meet = self.lib, self.meet
        L.norm_residual_forward(self.branch, self.residual, out=self.out, normed=self.normed, **self.norms())
        meet()
        self.adam()
        L.norm_residual_backward(self.branch, self.out, self.d_out, self.d_normed, d_branch=self.d_branch, d_residual=self.d_residual, **self.norms(), **self.g)
        meet()
        self.adam()
        L.dense_residual_forward(self.W, self.x, "gelu", bias=self.bias, y=self.y)
        meet()
        self.adam()
        L.dense_residual_forward(self.W, self.few, "gelu", bias=self.bias, y=self.y_few)
        meet()
        L.counter_advance(self.counter)
        meet()
        L.dropout(self.d_residual, 0.25, 9, call_counter=self.counter, y=self.d_out)
        meet()
        self.adam()

    def tensors(self):
        return [self.params, self.grads, self.m, self.v, self.state, self.counter, self.out, self.normed, self.d_branch, self.d_residual, self.d_out, self.y, self.y_few]


@pytest.mark.parametrize("R, D, dtype, post, pre, bias, gate_rows, offset", [(3, 256, BF16, "rms", "rms", False, 3, 0), (200, 2048, BF16, "layer", "rms", True, 7, 0),
                                                                           (500, 4096, BF16, "rms", "layer", False, 0, 0), (64, 777, torch.float32, "layer", "layer", True, 1, 3),
                                                                           (130, 100, torch.float16, "rms", "rms", False, 4, 1)])
def test_norms_layers_and_dropout_directly_behind_what_writes_their_operands(lib, R, D, dtype, post, pre, bias, gate_rows, offset):
    results = []
    for how in ("one by one", "stream", "graph"):
        chain = Chain(lib, R, D, dtype, post, pre, bias, gate_rows, offset, torch.cuda.synchronize if how == "one by one" else lambda: None)
        torch.cuda.synchronize()
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            if how == "graph":
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream):
                    chain.update()
            for _ in range(20):
                graph.replay() if how == "graph" else chain.update()
        torch.cuda.synchronize()
        results.append([t.clone() for t in chain.tensors()])
    assert all(torch.isfinite(t.float()).all() for t in results[0])
    for got in results[1:]:
        for a, b in zip(got, results[0]):
            assert torch.equal(a, b)
