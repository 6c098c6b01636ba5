"""What the operators of residual networks refuse, on machines without a GPU too: through the C entry points by status, through the package by B200RLError; and the
definitions that the GPU tests compare with, against known answers."""
import ctypes as C

import pytest
import torch

from residual_reference import philox_halves, norm64, act64, slope64

ADDRESS = 1 << 20                   # an address that a call which refuses its arguments never touches


def test_dense_entry_points_refuse(lib):
    L = lib.lib()
    p = ADDRESS

    def forward(type=1, W=p, ldw=8, bias=None, x=p, ldx=8, residual=None, ldr=0, pre=None, ldpre=0, y=p, ldy=8, batch=4, I=8, O=8, act=0, ws=None, n=0):
        return L.b200rl_dense_residual_forward(type, W, ldw, bias, x, ldx, residual, ldr, 1.0, pre, ldpre, y, ldy, batch, I, O, act, ws, n, None)

    assert forward(type=0) == 2 and forward(type=3) == 2 and forward(act=7) == 2 and forward(act=-1) == 2
    assert forward(batch=-1) == 1 and forward(I=0) == 1 and forward(O=0) == 1
    assert forward(W=None) == 1 and forward(x=None) == 1 and forward(y=None) == 1
    assert forward(ldw=7) == 1 and forward(ldx=7) == 1 and forward(ldy=7) == 1 and forward(residual=p, ldr=7) == 1 and forward(pre=p, ldpre=7) == 1
    assert forward(x=p + 1) == 1 and forward(y=p + 1) == 1 and forward(bias=p + 2) == 1
    assert forward(batch=0, W=None, x=None, y=None) == 0                          # nothing to do

    def backward_input(type=1, W=p, ldw=8, d=p, ldd=8, add=None, lda=0, pre=None, ldp=0, act=0, out=p, ldi=8, batch=4, I=8, O=8):
        return L.b200rl_dense_residual_backward_input(type, W, ldw, d, ldd, add, lda, pre, ldp, act, out, ldi, batch, I, O, None, 0, None)

    assert backward_input(type=0) == 2 and backward_input(act=9) == 2 and backward_input(act=1) == 1          # the slope needs the pre-activations
    assert backward_input(W=None) == 1 and backward_input(d=None) == 1 and backward_input(out=None) == 1 and backward_input(ldd=3) == 1 and backward_input(ldi=3) == 1
    assert backward_input(add=p, lda=7) == 1 and backward_input(pre=p, ldp=7, act=1) == 1 and backward_input(I=0) == 1 and backward_input(batch=-3) == 1
    assert backward_input(batch=0) == 0

    def backward_weights(type=1, x=p, ldx=8, d=p, ldd=8, dW=p, db=p, batch=4, I=8, O=8):
        return L.b200rl_dense_residual_backward_weights(type, x, ldx, d, ldd, dW, db, 0, batch, I, O, None, 0, None)

    assert backward_weights(type=0) == 2 and backward_weights(x=None) == 1 and backward_weights(d=None) == 1 and backward_weights(dW=p + 2) == 1 and backward_weights(db=p + 1) == 1
    assert backward_weights(ldx=7) == 1 and backward_weights(ldd=7) == 1 and backward_weights(batch=-1) == 1 and backward_weights(O=0) == 1
    assert backward_weights(dW=None, db=None) == 0

    def backward_activation(type=1, pre=p, d=p, out=p, ld=8, act=1, rows=4, cols=8):
        return L.b200rl_dense_residual_backward_activation(type, pre, ld, d, ld, 1.0, out, ld, rows, cols, act, None)

    assert backward_activation(type=0) == 2 and backward_activation(act=7) == 2 and backward_activation(pre=None) == 1 and backward_activation(d=None) == 1
    assert backward_activation(out=None) == 1 and backward_activation(ld=7) == 1 and backward_activation(cols=0) == 1 and backward_activation(rows=0) == 0


def test_workspaces_are_asked_for_and_checked(lib):
    """Rows that start on 16-byte boundaries need none; rows that do not are copied, and a call without the room for it is refused."""
    L, p = lib.lib(), ADDRESS
    size = L.b200rl_dense_residual_forward_workspace_bytes
    assert size(p, 64, p, 64, 500, 64, 64) == 0 and size(p, 65, p, 65, 20, 64, 64) == 0
    n = size(p, 65, p, 64, 500, 64, 64)
    assert n >= 64 * 64 * 2 and size(p, 64, p + 2, 64, 500, 64, 64) >= 500 * 64 * 2 and size(p, 65, p, 65, 0, 64, 64) == 0

    def forward(ws, n):
        return L.b200rl_dense_residual_forward(1, p, 65, None, p, 64, None, 0, 1.0, None, 0, p, 64, 500, 64, 64, 0, ws, n, None)

    assert forward(None, 0) == 1 and forward(p, n - 1) == 1 and forward(p + 8, n) == 1
    size = L.b200rl_dense_residual_backward_weights_workspace_bytes
    assert size(p, 4096, p, 4096, p, 4096, 4096, 4096) == 0 and size(p, 64, p, 64, None, 100000, 64, 64) == 0
    n = size(p, 64, p, 64, p, 100000, 64, 64)
    assert n > 0
    assert L.b200rl_dense_residual_backward_weights(1, p, 64, p, 64, p, None, 0, 100000, 64, 64, p, n - 256, None) == 1
    assert L.b200rl_dense_residual_backward_input_workspace_bytes(p, 63, p, 64, 100, 63, 64) >= 64 * 64 * 2
    # sizes that no memory holds are refused, not computed with
    top = 2 ** 31 - 1
    assert L.b200rl_dense_residual_forward(1, p, top, None, p, top, None, 0, 1.0, None, 0, p, top, top, top, top, 0, p, 1 << 62, None) == 2


def test_norm_entry_points_refuse(lib):
    L = lib.lib()
    p = ADDRESS

    def forward(type=0, post=1, branch=p, ldb=8, gate=None, ldg=8, gate_rows=1, residual=p, ldr=8, out=p, ldo=8, pre=2, normed=p, ldn=8, rows=4, dim=8, epsilon=1e-5, post_weight=None):
        return L.b200rl_norm_residual_forward(type, post, post_weight, None, branch, ldb, gate, ldg, gate_rows, 1.0, residual, ldr, out, ldo, pre, None, None, normed, ldn, rows, dim,
                                              epsilon, None)

    assert forward(type=5) == 2 and forward(post=3) == 2 and forward(pre=-1) == 2 and forward(dim=8193, ldb=9000, ldr=9000, ldo=9000, ldn=9000) == 2
    assert forward(rows=-1) == 1 and forward(dim=0) == 1 and forward(epsilon=-1.0) == 1 and forward(epsilon=float("nan")) == 1
    assert forward(normed=None) == 1 and forward(pre=0) == 1 and forward(branch=None, post=0, residual=None) == 1 and forward(branch=None) == 1
    assert forward(gate=p, gate_rows=0) == 1 and forward(gate=p, ldg=7) == 1 and forward(gate=p, branch=None, post=0) == 1 and forward(out=None, pre=0, normed=None) == 1
    assert forward(ldb=7) == 1 and forward(ldr=7) == 1 and forward(ldo=7) == 1 and forward(ldn=7) == 1 and forward(branch=p + 2) == 1
    assert forward(rows=0, normed=None) == 0

    def backward(type=0, post=1, branch=p, ldb=8, gate=None, gate_rows=1, out=p, pre=2, d_out=p, d_normed=p, d_branch=p, d_residual=p, d_gate=None, dpw=None, dnw=None, rows=4, dim=8,
                 epsilon=1e-5, scratch=p, n=1 << 20, ld=8):
        return L.b200rl_norm_residual_backward(type, post, None, None, branch, ldb, gate, ld, gate_rows, 1.0, out, ld, pre, None, d_out, ld, d_normed, ld, d_branch, ld, d_residual, ld,
                                               d_gate, ld, dpw, None, dnw, None, 0, rows, dim, epsilon, scratch, n, None)

    assert backward(type=-1) == 2 and backward(post=4) == 2 and backward(dim=8193) == 2 and backward(rows=-1) == 1 and backward(epsilon=-1e-3) == 1
    assert backward(d_normed=None) == 1 and backward(pre=0) == 1 and backward(out=None) == 1 and backward(branch=None) == 1 and backward(ldb=3) == 1 and backward(ld=3) == 1
    assert backward(d_gate=p) == 1 and backward(gate=p, gate_rows=0) == 1 and backward(post=0, dpw=p) == 1 and backward(pre=0, d_normed=None, dnw=p) == 1
    assert backward(scratch=None) == 1 and backward(scratch=p + 8) == 1 and backward(n=16) == 1
    assert backward(rows=0) == 0
    assert L.b200rl_norm_residual_backward_scratch_bytes(0, 8) == 0 and L.b200rl_norm_residual_backward_scratch_bytes(100, 8) > 0


def test_dropout_refuses(lib):
    L = lib.lib()
    p = ADDRESS

    def dropout(type=0, x=p, ldx=8, residual=None, ldr=8, y=p, ldy=8, rows=4, cols=8, prob=0.5, stream=0, counter=None):
        return L.b200rl_dropout(type, x, ldx, residual, ldr, y, ldy, rows, cols, prob, 1, stream, 0, counter, None)

    assert dropout(type=3) == 2 and dropout(x=None) == 1 and dropout(y=None) == 1 and dropout(ldx=7) == 1 and dropout(ldy=7) == 1 and dropout(residual=p, ldr=7) == 1
    assert dropout(prob=-0.1) == 1 and dropout(prob=1.1) == 1 and dropout(prob=float("nan")) == 1 and dropout(stream=65536) == 1 and dropout(cols=0) == 1 and dropout(rows=-1) == 1
    assert dropout(x=p + 2) == 1 and dropout(counter=p + 4) == 1 and dropout(rows=0) == 0


@pytest.mark.parametrize("break_it, what", [
    (dict(W=torch.zeros(4, 9)), "W is a"), (dict(x=torch.zeros(3, 8, dtype=torch.float64)), "no kernel"), (dict(x=torch.zeros(3, 8)), "no kernel"), (dict(x=torch.zeros(3)), "matrix"),
    (dict(bias=torch.zeros(5)), "bias"), (dict(bias=torch.zeros(4, dtype=torch.bfloat16)), "bias"), (dict(residual=torch.zeros(3, 5)), "residual"), (dict(act="softplus"), "activation"),
    (dict(x=torch.zeros(8, 3, dtype=torch.bfloat16).t()), "follow one another"), (dict(x=torch.zeros(1, 8, dtype=torch.bfloat16).expand(3, 8)), "overlap"),
    (dict(y=torch.zeros(3, 3, dtype=torch.bfloat16)), "y is a"), (dict(), "CUDA tensors"),
])
def test_dense_wrapper_refuses(lib, break_it, what):
    half = torch.bfloat16
    args = dict(W=torch.zeros(4, 8, dtype=half), x=torch.zeros(3, 8, dtype=half), act="relu", bias=torch.zeros(4), residual=torch.zeros(3, 4, dtype=half))
    args.update(break_it)
    with pytest.raises(lib.B200RLError, match=what):
        lib.dense_residual_forward(**args)


@pytest.mark.parametrize("break_it, what", [
    (dict(W=torch.zeros(5, 8, dtype=torch.float16)), "W is a"), (dict(x=torch.zeros(2, 8, dtype=torch.float16)), "x is a"), (dict(act_in="relu"), "pre-activations"),
    (dict(add=torch.zeros(3, 8)), "add"), (dict(d_W=torch.zeros(4, 8, dtype=torch.float16)), "d_W"), (dict(d_bias=torch.zeros(3)), "d_bias"), (dict(), "CUDA tensors"),
])
def test_dense_backward_wrapper_refuses(lib, break_it, what):
    half = torch.float16
    args = dict(W=torch.zeros(4, 8, dtype=half), x=torch.zeros(3, 8, dtype=half), d_pre=torch.zeros(3, 4, dtype=half))
    args.update(break_it)
    with pytest.raises(lib.B200RLError, match=what):
        lib.dense_residual_backward(**args)


@pytest.mark.parametrize("break_it, what", [
    (dict(branch=None, residual=None), "neither"), (dict(post="batch"), "norm"), (dict(branch=None), "not there"), (dict(post="none"), "not there"), (dict(gate=torch.zeros(2, 8)), "gate"),
    (dict(gate=torch.zeros(3, 8), gate_rows=0), "gate row"), (dict(post_weight=torch.zeros(7)), "post_weight"), (dict(residual=torch.zeros(3, 8, dtype=torch.float16)), "residual"),
    (dict(branch=torch.zeros(3, 8200), residual=None, post_weight=None), "8192"), (dict(), "CUDA tensors"),
])
def test_norm_wrapper_refuses(lib, break_it, what):
    args = dict(branch=torch.zeros(3, 8), residual=torch.zeros(3, 8), post="rms", post_weight=torch.ones(8), pre="layer")
    args.update(break_it)
    with pytest.raises(lib.B200RLError, match=what):
        lib.norm_residual_forward(**args)


@pytest.mark.parametrize("break_it, what", [
    (dict(d_out=None, d_normed=None), "neither"), (dict(d_normed=None), "go with"), (dict(out=None), "go with"), (dict(pre="none"), "go with"), (dict(d_gate=torch.zeros(3, 8)), "not there"),
    (dict(post="none"), "not there"), (dict(d_pre_weight=torch.zeros(8)), "not there"), (dict(d_post_weight=torch.zeros(3)), "d_post_weight"), (dict(), "CUDA tensors"),
])
def test_norm_backward_wrapper_refuses(lib, break_it, what):
    args = dict(branch=torch.zeros(3, 8), out=torch.zeros(3, 8), d_out=torch.zeros(3, 8), d_normed=torch.zeros(3, 8), post="rms", post_weight=torch.ones(8), pre="layer")
    args.update(break_it)
    with pytest.raises(lib.B200RLError, match=what):
        lib.norm_residual_backward(**args)


def test_dropout_wrapper_refuses(lib):
    x = torch.zeros(3, 8)
    for args in (dict(p=-0.5), dict(p=1.5), dict(p=0.5, stream_id=-1), dict(p=0.5, stream_id=65536), dict(p=0.5, residual=torch.zeros(2, 8)), dict(p=0.5, call_counter=torch.zeros(1)),
                 dict(p=0.5)):
        with pytest.raises(lib.B200RLError):
            lib.dropout(x, seed=1, **args)
    with pytest.raises(lib.B200RLError, match="no kernel"):
        lib.dropout(torch.zeros(3, 8, dtype=torch.int32), 0.5, 1)


def test_references_against_known_answers():
    """The 64-bit definitions: Philox against the published known-answer vector's generator (the package's host code draws from the same), norms against torch's, slopes
    against differences."""
    # blocks of different counters differ and every half is 16 bits; the same call draws the same bits
    h = philox_halves(4096, 7, 0, 3)
    assert h.min() >= 0 and h.max() < 65536 and len(set(h.tolist())) > 3500 and (philox_halves(4096, 7, 0, 3) == h).all()
    assert (philox_halves(64, 7, 1, 3) != h[:64]).any() and (philox_halves(64, 7, 0, 4) != h[:64]).any() and (philox_halves(64, 8, 0, 3) != h[:64]).any()
    x = torch.randn(5, 33, dtype=torch.float64, generator=torch.Generator().manual_seed(0)) + 0.3
    w, b = torch.rand(33, dtype=torch.float64), torch.rand(33, dtype=torch.float64)
    assert torch.allclose(norm64("layer", x, w, b, 1e-5), torch.nn.functional.layer_norm(x, (33,), w, b, 1e-5))
    assert torch.allclose(norm64("rms", x, w, None, 1e-5), torch.nn.functional.rms_norm(x, (33,), w, 1e-5))
    for name in ("identity", "relu", "tanh", "sigmoid", "gelu", "silu"):
        d = (act64(name, x + 1e-6) - act64(name, x - 1e-6)) / 2e-6
        assert torch.allclose(slope64(name, x), d, atol=1e-8), name
