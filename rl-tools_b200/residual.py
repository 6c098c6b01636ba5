"""The operators of residual networks in 16-bit types, on torch CUDA tensors: dense layers whose epilogue carries bias, activation and residual,
the norms around a block with its gate and residual scale, and dropout whose mask is drawn from a counter.

Matrices are 2-D tensors of one type (bfloat16 or float16; the norms and dropout take float32 too) whose rows may be views into wider tables; biases, norm weights
and every parameter gradient are float32, so that they can be slices of the arenas that b200rl_adam_step steps. A gradient that is passed in is
accumulated onto, one that is not is made. What is passed has to lie on the current device; calls run on its current stream. Arguments that no kernel
takes raise B200RLError. The calls take no part in autograd: operands that require gradients are taken as they are, results carry none, and writing into a tensor that was passed
does not raise its version; the gradients are the calls below. One block, forward and backward (x the residual stream, n = pre(x) from the block before):

    h_pre, h = dense_residual_forward(W1, n, "gelu", bias=b1, want_pre=True)
    _, f     = dense_residual_forward(W2, h, "identity", bias=b2)
    f_kept   = dropout(f, p, seed, call_index=step)
    out, n2  = norm_residual_forward(f_kept, x, post="rms", post_weight=w_post, gate=gate, gate_rows=rows, pre="rms", pre_weight=w_pre)

    g        = norm_residual_backward(f_kept, out, d_out, d_n2, post="rms", ...)
    d_f      = dropout(g["d_branch"], p, seed, call_index=step)
    dW2, db2, d_h_pre = dense_residual_backward(W2, h, d_f, pre_in=h_pre, act_in="gelu")
    dW1, db1, d_n     = dense_residual_backward(W1, n, d_h_pre)
"""
from . import ACT, B200RLError, check, lib

RESIDUAL_ACT = {**ACT, "gelu": 5, "silu": 6}
NORM = {"none": 0, "layer": 1, "rms": 2}
_ENTRIES = ("dense_residual_forward_workspace_bytes", "dense_residual_forward", "dense_residual_backward_activation", "dense_residual_backward_input_workspace_bytes",
            "dense_residual_backward_input", "dense_residual_backward_weights_workspace_bytes", "dense_residual_backward_weights", "norm_residual_forward",
            "norm_residual_backward_scratch_bytes", "norm_residual_backward", "dropout")
_module = None


def _tensors():
    """The compiled checks and calls (csrc/tensors.cpp), bound to the library's entry points. Raises if it has not been built: there is no fallback path."""
    global _module
    if _module is None:
        import ctypes
        import torch  # noqa: F401  (its libraries have to be loaded first)
        try:
            from . import _tensors as module
        except ImportError as e:
            raise B200RLError(f"the operators on torch tensors are not built: run rl_tools_b200.build() ({e})") from None
        L = lib()
        module.bind(*(ctypes.cast(getattr(L, "b200rl_" + name), ctypes.c_void_p).value for name in _ENTRIES))
        _module = module
    return _module


def _failed(call, e):
    """A refusal of the arguments, or the status of a C entry point, as the package's error."""
    if isinstance(e, _module.Status):
        check(e.args[0], "b200rl_" + call)
    raise B200RLError(str(e)) from None


def dense_residual_forward(W, x, act, bias=None, residual=None, scale=1.0, want_pre=False, y=None, pre=None):
    """y = residual + scale act(x W^T + bias); returns (pre or None, y). pre (kept when want_pre or given) holds the pre-activations for the backward pass.
    y may be the residual itself."""
    T = _module or _tensors()
    try:
        return T.dense_residual_forward(W, x, RESIDUAL_ACT.get(act, act), bias, residual, scale, bool(want_pre), y, pre)
    except (T.Refusal, T.Status) as e:
        _failed("dense_residual_forward", e)


def dense_residual_backward_activation(pre, d_y, act, scale=1.0, d_pre=None):
    """d_pre = scale act'(pre) d_y (pre may be None for the identity); d_pre may be d_y or pre itself."""
    T = _module or _tensors()
    try:
        return T.dense_residual_backward_activation(pre, d_y, RESIDUAL_ACT.get(act, act), scale, d_pre)
    except (T.Refusal, T.Status) as e:
        _failed("dense_residual_backward_activation", e)


def dense_residual_backward(W, x, d_pre, d_W=None, d_bias=None, add=None, pre_in=None, act_in="identity", d_in=None, want_d_in=True, want_grads=True):
    """The gradients of a layer with the pre-activation gradient d_pre: returns (d_W, d_bias, d_in) with d_W += d_pre^T x and d_bias += column sums of d_pre (float32),
    d_in = act_in'(pre_in) (d_pre W + add). want_grads=False leaves out the first two, want_d_in=False the last. d_in may be add or pre_in itself."""
    T = _module or _tensors()
    try:
        return T.dense_residual_backward(W, x, d_pre, d_W, d_bias, add, pre_in, RESIDUAL_ACT.get(act_in, act_in), d_in, bool(want_d_in), bool(want_grads))
    except (T.Refusal, T.Status) as e:
        _failed("dense_residual_backward", e)


def norm_residual_forward(branch, residual, post="none", post_weight=None, post_bias=None, gate=None, gate_rows=1, scale=1.0, pre="none", pre_weight=None, pre_bias=None,
                          epsilon=1e-5, out=None, normed=None):
    """out = residual + scale gate post(branch), normed = pre(out); returns (out, normed or None). post, pre: "none", "layer" or "rms", each with its weight and bias. gate
    [ceil(rows / gate_rows), dim]: row r takes gate row r // gate_rows (a batch without rows takes any gate). branch or residual may be None; out may be the residual itself."""
    T = _module or _tensors()
    try:
        return T.norm_residual_forward(branch, residual, NORM.get(post, post), post_weight, post_bias, gate, gate_rows, scale, NORM.get(pre, pre), pre_weight, pre_bias, epsilon, out,
                                       normed)
    except (T.Refusal, T.Status) as e:
        _failed("norm_residual_forward", e)


def norm_residual_backward(branch, out, d_out=None, d_normed=None, post="none", post_weight=None, post_bias=None, gate=None, gate_rows=1, scale=1.0, pre="none",
                           pre_weight=None, pre_bias=None, epsilon=1e-5, d_branch=None, d_residual=None, d_gate=None, d_post_weight=None, d_post_bias=None,
                           d_pre_weight=None, d_pre_bias=None):
    """The gradients of norm_residual_forward from those of out and normed (each may be None), as a dict: d_branch, d_residual, d_gate, d_post_weight, d_post_bias,
    d_pre_weight and d_pre_bias (None where there is nothing to derive). `out` is the sum that the forward pass returned."""
    T = _module or _tensors()
    try:
        return T.norm_residual_backward(branch, out, d_out, d_normed, NORM.get(post, post), post_weight, post_bias, gate, gate_rows, scale, NORM.get(pre, pre), pre_weight, pre_bias,
                                        epsilon, d_branch, d_residual, d_gate, d_post_weight, d_post_bias, d_pre_weight, d_pre_bias)
    except (T.Refusal, T.Status) as e:
        _failed("norm_residual_backward", e)


def dropout(x, p, seed, stream_id=0, call_index=0, call_counter=None, residual=None, y=None):
    """y = residual + (kept ? x / P(kept) : 0): element e of x is dropped with probability p (to 1 / 65536) by the generator's bits for (seed, stream_id, call, e), call =
    call_index + call_counter[0]. The backward pass is the same call on the gradient. y may be x or the residual itself."""
    T = _module or _tensors()
    try:
        return T.dropout(x, p, seed, stream_id, call_index, call_counter, residual, y)
    except (T.Refusal, T.Status) as e:
        _failed("dropout", e)
