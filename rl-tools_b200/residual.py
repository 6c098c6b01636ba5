"""The operators of residual networks in 16-bit types, on torch CUDA tensors: dense layers whose epilogue carries bias, activation and residual,
the norms around a block with its gate and residual scale, and dropout whose mask is drawn from a counter.

Matrices are 2-D tensors of one type (bfloat16 or float16; the norms and dropout take float32 too) whose rows may be views into wider tables; biases, norm weights
and every parameter gradient are float32, so that they can be slices of the arenas that b200rl_adam_step steps. A gradient that is passed in is
accumulated onto, one that is not is made. What is passed has to lie on the current device; calls run on its current stream. Arguments that no kernel
takes raise B200RLError. One block, forward and backward (x the residual stream, n = pre(x) from the block before):

    h_pre, h = dense_residual_forward(W1, n, "gelu", bias=b1, want_pre=True)
    _, f     = dense_residual_forward(W2, h, "identity", bias=b2)
    f_kept   = dropout(f, p, seed, call_index=step)
    out, n2  = norm_residual_forward(f_kept, x, post="rms", post_weight=w_post, gate=gate, gate_rows=rows, pre="rms", pre_weight=w_pre)

    g        = norm_residual_backward(f_kept, out, d_out, d_n2, post="rms", ...)
    d_f      = dropout(g["d_branch"], p, seed, call_index=step)
    dW2, db2, d_h_pre = dense_residual_backward(W2, h, d_f, pre_in=h_pre, act_in="gelu")
    dW1, db1, d_n     = dense_residual_backward(W1, n, d_h_pre)
"""
from . import B200RLError, ACT, lib, check, _stream

RESIDUAL_ACT = {**ACT, "gelu": 5, "silu": 6}
NORM = {"none": 0, "layer": 1, "rms": 2}
NORM_MAX_DIM = 8192
_TYPES = None


def _types():
    global _TYPES
    if _TYPES is None:
        import torch
        _TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
    return _TYPES


def _refuse(what):
    raise B200RLError(what)


def _device():
    from torch import _C
    return _C._cuda_getDevice()


class _Operands:
    """The operands of one call: each is checked against the type, the shape and the current device and gives its address and pitch."""

    def __init__(self, call, first, types):
        self.call, self.dtype = call, first.dtype
        self.type = _types().get(first.dtype, -1)
        if self.type not in types:
            _refuse(f"{call}: no kernel for matrices of {first.dtype}")
        self.tensors = []

    def matrix(self, name, t, rows, cols):
        if t is None:
            return None, 0
        shape, stride = t.shape, t.stride()
        if t.dtype != self.dtype or len(shape) != 2 or shape[0] != rows or shape[1] != cols:
            _refuse(f"{self.call}: {name} is a {tuple(shape)} {t.dtype}, not a [{rows}, {cols}] {self.dtype}")
        if cols > 1 and stride[1] != 1:
            _refuse(f"{self.call}: the elements of {name}'s rows do not follow one another")
        if rows > 1 and stride[0] < cols:
            _refuse(f"{self.call}: the rows of {name} overlap")
        self.tensors.append(t)
        return t.data_ptr(), stride[0] if rows > 1 else cols

    def vector(self, name, t, n):
        if t is None:
            return None
        import torch
        if t.dtype != torch.float32 or t.dim() != 1 or t.shape[0] != n or (n > 1 and t.stride(0) != 1):
            _refuse(f"{self.call}: {name} is not {n} float32 values in a row")
        self.tensors.append(t)
        return t.data_ptr()

    def here(self):
        """All on the current device (looked at last: shapes and types are refused on machines without one too)."""
        device = None
        for t in self.tensors:
            if not t.is_cuda:
                _refuse(f"{self.call}: takes CUDA tensors, got one on {t.device}")
            device = _device() if device is None else device
            if t.device.index != device:
                _refuse(f"{self.call}: a tensor lies on {t.device}, the current device is cuda:{device}")


def _activation(call, act):
    a = RESIDUAL_ACT.get(act, act)
    if not isinstance(a, int) or not 0 <= a <= 6:
        _refuse(f"{call}: no activation {act!r}")
    return a


def _norm(call, kind):
    if kind not in NORM:
        _refuse(f"{call}: no norm {kind!r}")
    return NORM[kind]


def _is_matrix(call, name, t):
    if t.dim() != 2:
        _refuse(f"{call}: {name} has to be a matrix")
    return t.shape


def _workspace(n, device):
    if n == 0:
        return None, None
    import torch
    t = torch.empty(n, device=device, dtype=torch.uint8)
    return t, t.data_ptr()


def dense_residual_forward(W, x, act, bias=None, residual=None, scale=1.0, want_pre=False, y=None, pre=None):
    """y = residual + scale act(x W^T + bias); returns (pre or None, y). pre (kept when want_pre or given) holds the pre-activations for the backward pass.
    y may be the residual itself."""
    call = "dense_residual_forward"
    B, I = _is_matrix(call, "x", x)
    O = _is_matrix(call, "W", W)[0]
    if I < 1 or O < 1:
        _refuse(f"{call}: a layer has at least one input and one output")
    o, a = _Operands(call, x, (1, 2)), _activation(call, act)
    px, ldx = o.matrix("x", x, B, I)
    pw, ldw = o.matrix("W", W, O, I)
    pr, ldr = o.matrix("residual", residual, B, O)
    pb = o.vector("bias", bias, O)
    y = x.new_empty((B, O)) if y is None else y
    py, ldy = o.matrix("y", y, B, O)
    pre = x.new_empty((B, O)) if pre is None and want_pre else pre
    pp, ldp = o.matrix("pre", pre, B, O)
    o.here()
    L = lib()
    n = L.b200rl_dense_residual_forward_workspace_bytes(pw, ldw, px, ldx, B, I, O)
    ws, pws = _workspace(n, x.device)
    check(L.b200rl_dense_residual_forward(o.type, pw, ldw, pb, px, ldx, pr, ldr, scale, pp, ldp, py, ldy, B, I, O, a, pws, n, _stream()), call)
    return pre, y


def dense_residual_backward_activation(pre, d_y, act, scale=1.0, d_pre=None):
    """d_pre = scale act'(pre) d_y (pre may be None for the identity); d_pre may be d_y or pre itself."""
    call = "dense_residual_backward_activation"
    B, O = _is_matrix(call, "d_y", d_y)
    o, a = _Operands(call, d_y, (1, 2)), _activation(call, act)
    if O < 1 or (pre is None and a != 0):
        _refuse(f"{call}: the slope of {act!r} needs the pre-activations, and rows at least one element")
    pd, ldd = o.matrix("d_y", d_y, B, O)
    pp, ldp = o.matrix("pre", pre, B, O)
    d_pre = d_y.new_empty((B, O)) if d_pre is None else d_pre
    po, ldo = o.matrix("d_pre", d_pre, B, O)
    o.here()
    check(lib().b200rl_dense_residual_backward_activation(o.type, pp, ldp, pd, ldd, scale, po, ldo, B, O, a, _stream()), call)
    return d_pre


def dense_residual_backward(W, x, d_pre, d_W=None, d_bias=None, add=None, pre_in=None, act_in="identity", d_in=None, want_d_in=True, want_grads=True):
    """The gradients of a layer with the pre-activation gradient d_pre: returns (d_W, d_bias, d_in) with d_W += d_pre^T x and d_bias += column sums of d_pre (float32),
    d_in = act_in'(pre_in) (d_pre W + add). want_grads=False leaves out the first two, want_d_in=False the last. d_in may be add or pre_in itself."""
    call = "dense_residual_backward"
    B, O = _is_matrix(call, "d_pre", d_pre)
    I = _is_matrix(call, "W", W)[1]
    if I < 1 or O < 1:
        _refuse(f"{call}: a layer has at least one input and one output")
    o, a = _Operands(call, d_pre, (1, 2)), _activation(call, act_in)
    pd, ldd = o.matrix("d_pre", d_pre, B, O)
    pw, ldw = o.matrix("W", W, O, I)
    px, ldx = o.matrix("x", x, B, I) if want_grads else (None, 0)
    if want_grads:
        import torch
        given = [t for t in (d_W, d_bias) if t is not None]
        made = torch.zeros if given else torch.empty
        d_W = made((O, I), device=d_pre.device, dtype=torch.float32) if d_W is None else d_W
        d_bias = made((O,), device=d_pre.device, dtype=torch.float32) if d_bias is None else d_bias
        if d_W.dtype != torch.float32 or d_W.shape != (O, I) or not d_W.is_contiguous():
            _refuse(f"{call}: d_W is not a dense [{O}, {I}] float32 matrix")
        o.tensors.append(d_W)
        pgb = o.vector("d_bias", d_bias, O)
    if want_d_in:
        if a != 0 and pre_in is None:
            _refuse(f"{call}: the slope of {act_in!r} needs the pre-activations")
        pa, lda = o.matrix("add", add, B, I)
        pp, ldp = o.matrix("pre_in", pre_in, B, I)
        d_in = d_pre.new_empty((B, I)) if d_in is None else d_in
        pi, ldi = o.matrix("d_in", d_in, B, I)
    o.here()
    L = lib()
    # the weights first: d_in may overwrite what it reads, never x or d_pre
    if want_grads:
        n = L.b200rl_dense_residual_backward_weights_workspace_bytes(px, ldx, pd, ldd, d_W.data_ptr(), B, I, O)
        ws, pws = _workspace(n, d_pre.device)
        check(L.b200rl_dense_residual_backward_weights(o.type, px, ldx, pd, ldd, d_W.data_ptr(), pgb, len(given) > 0, B, I, O, pws, n, _stream()), call)
    if want_d_in:
        n = L.b200rl_dense_residual_backward_input_workspace_bytes(pw, ldw, pd, ldd, B, I, O)
        ws, pws = _workspace(n, d_pre.device)
        check(L.b200rl_dense_residual_backward_input(o.type, pw, ldw, pd, ldd, pa, lda, pp, ldp, a, pi, ldi, B, I, O, pws, n, _stream()), call)
    return (d_W, d_bias) + (d_in,) if want_grads else (None, None, d_in if want_d_in else None)


def _gates(call, gate, gate_rows, rows):
    if gate is not None and gate_rows < 1:
        _refuse(f"{call}: a gate row serves at least one row")
    return -(-rows // gate_rows) if gate is not None else 0


def norm_residual_forward(branch, residual, post="none", post_weight=None, post_bias=None, gate=None, gate_rows=1, scale=1.0, pre="none", pre_weight=None, pre_bias=None,
                          epsilon=1e-5, out=None, normed=None):
    """out = residual + scale gate post(branch), normed = pre(out); returns (out, normed or None). post, pre: "none", "layer" or "rms", each with its weight and bias. gate
    [ceil(rows / gate_rows), dim]: row r takes gate row r // gate_rows. branch or residual may be None; out may be the residual itself."""
    call = "norm_residual_forward"
    first = branch if branch is not None else residual
    if first is None:
        _refuse(f"{call}: neither branch nor residual")
    R, D = _is_matrix(call, "branch" if branch is not None else "residual", first)
    o, kp, kn = _Operands(call, first, (0, 1, 2)), _norm(call, post), _norm(call, pre)
    if not 1 <= D <= NORM_MAX_DIM:
        _refuse(f"{call}: rows have 1 to {NORM_MAX_DIM} elements, not {D}")
    if branch is None and (kp or gate is not None):
        _refuse(f"{call}: a norm or a gate of a branch that is not there")
    if (not kp and (post_weight is not None or post_bias is not None)) or (not kn and (pre_weight is not None or pre_bias is not None or normed is not None)):
        _refuse(f"{call}: a weight, bias or output of a norm that is not there")
    pb, ldb = o.matrix("branch", branch, R, D)
    pr, ldr = o.matrix("residual", residual, R, D)
    pg, ldg = o.matrix("gate", gate, _gates(call, gate, gate_rows, R), D)
    w = [o.vector(n, t, D) for n, t in (("post_weight", post_weight), ("post_bias", post_bias), ("pre_weight", pre_weight), ("pre_bias", pre_bias))]
    out = first.new_empty((R, D)) if out is None else out
    po, ldo = o.matrix("out", out, R, D)
    if kn:
        normed = first.new_empty((R, D)) if normed is None else normed
    pn, ldn = o.matrix("normed", normed, R, D)
    o.here()
    if R:
        check(lib().b200rl_norm_residual_forward(o.type, kp, w[0], w[1], pb, ldb, pg, ldg, gate_rows, scale, pr, ldr, po, ldo, kn, w[2], w[3], pn, ldn, R, D, epsilon, _stream()), call)
    return out, normed


def norm_residual_backward(branch, out, d_out=None, d_normed=None, post="none", post_weight=None, post_bias=None, gate=None, gate_rows=1, scale=1.0, pre="none",
                           pre_weight=None, pre_bias=None, epsilon=1e-5, d_branch=None, d_residual=None, d_gate=None, d_post_weight=None, d_post_bias=None,
                           d_pre_weight=None, d_pre_bias=None):
    """The gradients of norm_residual_forward from those of out and normed (each may be None), as a dict: d_branch, d_residual, d_gate, d_post_weight, d_post_bias,
    d_pre_weight and d_pre_bias (None where there is nothing to derive). `out` is the sum that the forward pass returned."""
    call = "norm_residual_backward"
    first = d_normed if d_normed is not None else d_out
    if first is None:
        _refuse(f"{call}: neither d_out nor d_normed")
    R, D = _is_matrix(call, "d_out" if d_normed is None else "d_normed", first)
    o, kp, kn = _Operands(call, first, (0, 1, 2)), _norm(call, post), _norm(call, pre)
    if not 1 <= D <= NORM_MAX_DIM:
        _refuse(f"{call}: rows have 1 to {NORM_MAX_DIM} elements, not {D}")
    if branch is None and (kp or gate is not None):
        _refuse(f"{call}: a norm or a gate of a branch that is not there")
    if bool(kn) != (d_normed is not None) or (kn and out is None):
        _refuse(f"{call}: d_normed and out go with the norm behind the sum")
    if (not kp and (post_weight is not None or post_bias is not None)) or (not kn and (pre_weight is not None or pre_bias is not None)):
        _refuse(f"{call}: a weight or bias of a norm that is not there")
    pb, ldb = o.matrix("branch", branch, R, D)
    po, ldo = o.matrix("out", out, R, D)
    pdo, lddo = o.matrix("d_out", d_out, R, D)
    pdn, lddn = o.matrix("d_normed", d_normed, R, D)
    G = _gates(call, gate, gate_rows, R)
    pg, ldg = o.matrix("gate", gate, G, D)
    w = [o.vector(n, t, D) for n, t in (("post_weight", post_weight), ("post_bias", post_bias), ("pre_weight", pre_weight))]
    if (branch is None and d_branch is not None) or (gate is None and d_gate is not None):
        _refuse(f"{call}: the gradient of an operand that is not there")
    if branch is not None:
        d_branch = first.new_empty((R, D)) if d_branch is None else d_branch
    d_residual = first.new_empty((R, D)) if d_residual is None else d_residual
    if gate is not None:
        d_gate = first.new_empty((G, D)) if d_gate is None else d_gate
    pdb, lddb = o.matrix("d_branch", d_branch, R, D)
    pdr, lddr = o.matrix("d_residual", d_residual, R, D)
    pdg, lddg = o.matrix("d_gate", d_gate, G, D)
    # parameter gradients: those of the parameters that are there; accumulated onto when given
    import torch
    params = [("d_post_weight", post_weight, d_post_weight), ("d_post_bias", post_bias, d_post_bias), ("d_pre_weight", pre_weight, d_pre_weight), ("d_pre_bias", pre_bias, d_pre_bias)]
    given = [g for _, _, g in params if g is not None]
    made = torch.zeros if given else torch.empty
    grads = {}
    for name, t, g in params:
        if t is None and g is not None:
            _refuse(f"{call}: {name} of a parameter that is not there")
        grads[name] = made((D,), device=first.device, dtype=torch.float32) if t is not None and g is None else g
    pgrads = [o.vector(name, grads[name], D) for name, _, _ in params]
    o.vector("pre_bias", pre_bias, D)
    o.here()
    L = lib()
    n = L.b200rl_norm_residual_backward_scratch_bytes(R, D)
    ws, pws = _workspace(n, first.device)
    check(L.b200rl_norm_residual_backward(o.type, kp, w[0], w[1], pb, ldb, pg, ldg, gate_rows, scale, po, ldo, kn, w[2], pdo, lddo, pdn, lddn, pdb, lddb, pdr, lddr, pdg, lddg,
                                          *pgrads, len(given) > 0, R, D, epsilon, pws, n, _stream()), call)
    return dict(d_branch=d_branch, d_residual=d_residual, d_gate=d_gate, **grads)


def dropout(x, p, seed, stream_id=0, call_index=0, call_counter=None, residual=None, y=None):
    """y = residual + (kept ? x / P(kept) : 0): element e of x is dropped with probability p (to 1 / 65536) by the generator's bits for (seed, stream_id, call, e), call =
    call_index + call_counter[0]. The backward pass is the same call on the gradient. y may be x or the residual itself."""
    call = "dropout"
    R, D = _is_matrix(call, "x", x)
    o = _Operands(call, x, (0, 1, 2))
    if D < 1 or not 0.0 <= p <= 1.0 or not 0 <= stream_id < 65536:
        _refuse(f"{call}: rows of at least one element, 0 <= p <= 1, 0 <= stream_id < 65536")
    px, ldx = o.matrix("x", x, R, D)
    pr, ldr = o.matrix("residual", residual, R, D)
    y = x.new_empty((R, D)) if y is None else y
    py, ldy = o.matrix("y", y, R, D)
    pc = None
    if call_counter is not None:
        import torch
        if call_counter.dtype != torch.int64 or call_counter.numel() != 1:
            _refuse(f"{call}: call_counter is one int64 value")
        o.tensors.append(call_counter)
        pc = call_counter.data_ptr()
    o.here()
    check(lib().b200rl_dropout(o.type, px, ldx, pr, ldr, py, ldy, R, D, p, seed & 0xFFFFFFFFFFFFFFFF, stream_id, call_index & 0xFFFFFFFFFFFFFFFF, pc, _stream()), call)
    return y
