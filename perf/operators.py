"""The operators of residual networks in 16-bit types as measurable cases: dense layers whose epilogue carries bias, activation and residual,
the norms around a block fused with its gate and residual scale, and dropout whose mask is drawn from a counter and never stored.

    listed()            the cases: the smallest calls, the ordinary ones and the largest of each operator
    draw(rng)           one more case of the same ranges
    prepare(case, seed) what the program holds before the call: inputs, weights and incoming gradients
    run(state)          one pass: in plain torch operations, or (own = True) through the framework's entry points
    exact(case, seed)   what run returns for these inputs, from the definition in 64 bits
    work(case)          bytes and floating-point operations that the pass cannot do without

The kinds:
    dense           y = residual + scale act(x W^T + bias), the pre-activations kept on request
    dense_backward  d_in = act'(pre_in) (d_pre W + add), d_W = d_pre^T x, d_bias = column sums of d_pre
    norm            out = residual + scale gate post(branch), normed = pre(out), post and pre layer or root-mean-square norms
    norm_backward   the gradients of branch, residual, gate and of both norms' weights and biases
    dropout         y = residual + keep x / P(keep), keep drawn from Philox blocks numbered by the element
"""
import importlib
import math

import numpy as np
import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
EPSILON = 1e-5


def listed():
    return [
        # one token of a serving loop through the widening layer of a block: the smallest product, bound by reading the weights
        dict(name="dense_token_1", kind="dense", type="bfloat16", batch=1, input=1024, output=4096, act="silu", bias=True, residual=False, scale=1.0, keep_pre=False, pad=0),
        # a training forward pass of sizes that fit no tile and rows that start at odd addresses
        dict(name="dense_ragged_1003", kind="dense", type="float16", batch=1003, input=777, output=1001, act="tanh", bias=True, residual=True, scale=0.5, keep_pre=True, pad=0),
        # the training forward pass of a block's widening layer
        dict(name="dense_block_4096", kind="dense", type="bfloat16", batch=4096, input=1024, output=4096, act="gelu", bias=True, residual=False, scale=1.0, keep_pre=True, pad=0),
        # a wide layer over a long batch, added onto the residual stream: the largest product
        dict(name="dense_large_16384", kind="dense", type="bfloat16", batch=16384, input=4096, output=4096, act="identity", bias=True, residual=True, scale=0.5, keep_pre=False, pad=0),
        # the backward pass of a 256-wide layer at the batch size of the off-policy algorithms: latency counts
        dict(name="dense_backward_256", kind="dense_backward", type="float16", batch=256, input=256, output=256, act="relu", add=False, pad=0),
        # the backward pass of a block's narrowing layer, on through the activation in front of it
        dict(name="dense_backward_block_4096", kind="dense_backward", type="bfloat16", batch=4096, input=4096, output=1024, act="gelu", add=False, pad=0),
        # one token between two blocks of a serving loop
        dict(name="norm_token_1", kind="norm", type="bfloat16", rows=1, dim=4096, post="rms", pre="rms", gate_rows=1, bias=False, scale=1.0),
        # the same over a long batch with a learned gate per channel: memory bound
        dict(name="norm_large_16384", kind="norm", type="bfloat16", rows=16384, dim=4096, post="rms", pre="rms", gate_rows=16384, bias=False, scale=0.5),
        # the backward pass in 32 bits, odd sizes, a gate per group of 17 rows that the last group does not fill
        dict(name="norm_backward_1003", kind="norm_backward", type="float32", rows=1003, dim=777, post="layer", pre="layer", gate_rows=17, bias=True, scale=1.0),
        # the backward pass over a long batch
        dict(name="norm_backward_16384", kind="norm_backward", type="bfloat16", rows=16384, dim=4096, post="rms", pre="rms", gate_rows=16384, bias=False, scale=0.5),
        # dropout of odd sizes: blocks of random numbers straddle rows
        dict(name="dropout_1003", kind="dropout", type="float32", rows=1003, dim=777, p=0.5, residual=False),
        # dropout of a branch on its way onto the residual stream of a long batch
        dict(name="dropout_16384", kind="dropout", type="bfloat16", rows=16384, dim=4096, p=0.1, residual=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    n = _log_int(rng, lo, hi)
    return n if rng.random() < 0.5 else min(hi, max(lo, (n + 31) // 64 * 64)) or lo


def draw(rng):
    kind = rng.choice(["dense", "dense", "dense_backward", "dense_backward", "norm", "norm_backward", "dropout"])
    if kind in ("dense", "dense_backward"):
        c = dict(kind=kind, type=rng.choice(["bfloat16", "float16"]), batch=_size(rng, 1, 16384), input=_size(rng, 16, 4096), output=_size(rng, 16, 4096),
                 act=rng.choice(["identity", "relu", "tanh", "sigmoid", "gelu", "silu"]), pad=rng.choice([0, 0, 8, 24, 5]))
        if kind == "dense":
            c.update(bias=rng.random() < 0.7, residual=rng.random() < 0.5, scale=rng.choice([1.0, 0.5, 0.1]), keep_pre=rng.random() < 0.5)
        else:
            c.update(add=rng.random() < 0.5)
            if c["batch"] * c["input"] * c["output"] > 8192 * 4096 * 4096:
                c["batch"] = 8192 * 4096 * 4096 // (c["input"] * c["output"])
        return c
    if kind == "dropout":
        dim = _size(rng, 1, 8192)
        return dict(kind=kind, type=rng.choice(["bfloat16", "float16", "float32"]), rows=_size(rng, 1, min(16384, 2 ** 25 // dim)), dim=dim,
                    p=rng.choice([0.1, 0.2, 0.5, 0.75]), residual=rng.random() < 0.5)
    dim = _size(rng, 16, 8192)
    rows = _size(rng, 1, min(16384, 2 ** 25 // dim))
    norms = rng.choice([("rms", "rms"), ("layer", "layer"), ("none", "rms"), ("rms", "none"), ("none", "layer")])
    return dict(kind=kind, type=rng.choice(["bfloat16", "float16", "float32"]), rows=rows, dim=dim, post=norms[0], pre=norms[1],
                gate_rows=rng.choice([0, 1, rows, _log_int(rng, 1, rows)]), bias=rng.random() < 0.5, scale=rng.choice([1.0, 0.5]))


# ---- inputs ------------------------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    c, kind, t = dict(case), case["kind"], TYPES[case["type"]]
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, dtype=t, mean=0.0):
        return (torch.randn(*shape, device="cuda", generator=g) * std + mean).to(dtype)

    def matrix(rows, cols, std=1.0):
        # rows of a wider table where the case has a pad
        return normal(rows, cols + c.get("pad", 0), std=std)[:, :cols]

    if kind == "dense":
        B, I, O = c["batch"], c["input"], c["output"]
        return dict(case=c, W=matrix(O, I, 1 / math.sqrt(I)), x=matrix(B, I), bias=normal(O, std=0.1, dtype=torch.float32) if c["bias"] else None,
                    residual=matrix(B, O) if c["residual"] else None)
    if kind == "dense_backward":
        B, I, O = c["batch"], c["input"], c["output"]
        return dict(case=c, W=matrix(O, I, 1 / math.sqrt(I)), x=matrix(B, I), d_pre=matrix(B, O, 0.25), add=matrix(B, I, 0.25) if c["add"] else None,
                    pre_in=matrix(B, I) if c["act"] != "identity" else None)
    R, D = c["rows"], c["dim"]
    if kind == "dropout":
        return dict(case=c, x=normal(R, D), residual=normal(R, D) if c["residual"] else None, seed=seed, call=seed % 1000)
    params = {}
    for side in ("post", "pre"):
        has = c[side] != "none"
        params[side + "_weight"] = normal(D, std=0.1, dtype=torch.float32, mean=1.0) if has else None
        params[side + "_bias"] = normal(D, std=0.1, dtype=torch.float32) if has and c["bias"] else None
    gate = normal(-(-R // c["gate_rows"]), D, std=0.3, mean=0.7) if c["gate_rows"] else None
    s = dict(case=c, branch=normal(R, D, std=0.8, mean=0.1), residual=normal(R, D, std=1.5, mean=-0.1), gate=gate, **params)
    if kind == "norm_backward":
        s.update(d_out=normal(R, D, std=0.1), d_normed=normal(R, D, std=0.1) if c["pre"] != "none" else None)
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------------------------------------
def _act(name, v):
    if name == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if name == "tanh":
        return torch.tanh(v)
    if name == "sigmoid":
        return 1 / (1 + torch.exp(-v))
    if name == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if name == "silu":
        return v / (1 + torch.exp(-v))
    return v


def _d_act(name, v):
    if name == "relu":
        return (v > 0).to(v.dtype)
    if name == "tanh":
        return 1 - torch.tanh(v) ** 2
    if name == "sigmoid":
        e = 1 / (1 + torch.exp(-v))
        return e * (1 - e)
    if name == "gelu":
        return 0.5 * (1 + torch.erf(v * math.sqrt(0.5))) + v * torch.exp(-0.5 * v * v) / math.sqrt(2 * math.pi)
    if name == "silu":
        e = 1 / (1 + torch.exp(-v))
        return e * (1 + v * (1 - e))
    return torch.ones_like(v)


def _plain_dense(s, c, t):
    pre = s["x"].float() @ s["W"].float().t()
    if s["bias"] is not None:
        pre = pre + s["bias"]
    y = c["scale"] * _act(c["act"], pre)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return dict(y=y.to(t), pre=pre.to(t) if c["keep_pre"] else None)


def _plain_dense_backward(s, c, t):
    d_pre = s["d_pre"].float()
    d_in = d_pre @ s["W"].float()
    if s["add"] is not None:
        d_in = d_in + s["add"].float()
    if s["pre_in"] is not None:
        d_in = d_in * _d_act(c["act"], s["pre_in"].float())
    return dict(d_in=d_in.to(t), d_W=d_pre.t() @ s["x"].float(), d_bias=d_pre.sum(0))


def _normalised(kind, v):
    """The normalised rows and the factor that scaled them."""
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((v * v).mean(1, keepdim=True) + EPSILON)
    return v * rstd, rstd


def _affine(v, weight, bias):
    if weight is not None:
        v = v * weight
    return v if bias is None else v + bias


def _gate_rows(s, c):
    return s["gate"].float().repeat_interleave(c["gate_rows"], 0)[:c["rows"]]


def _plain_norm(s, c, t):
    u = s["branch"].float()
    if c["post"] != "none":
        u = _affine(_normalised(c["post"], u)[0], s["post_weight"], s["post_bias"])
    if s["gate"] is not None:
        u = u * _gate_rows(s, c)
    out = s["residual"].float() + c["scale"] * u
    normed = _affine(_normalised(c["pre"], out)[0], s["pre_weight"], s["pre_bias"]) if c["pre"] != "none" else None
    return dict(out=out.to(t), normed=None if normed is None else normed.to(t))


def _through_norm(kind, q, normalised, rstd):
    """The gradient in front of a norm, from the one behind it (already times the weight)."""
    inner = q - normalised * (q * normalised).mean(1, keepdim=True)
    if kind == "layer":
        inner = inner - q.mean(1, keepdim=True)
    return inner * rstd


def _plain_norm_backward(s, c, t):
    # the point of the gradient: `residual` stands for the sum that the forward pass left
    d = s["d_out"].float()
    r = dict(d_post_weight=None, d_post_bias=None, d_pre_weight=None, d_pre_bias=None, d_gate=None)
    if c["pre"] != "none":
        hat, rstd = _normalised(c["pre"], s["residual"].float())
        d_normed = s["d_normed"].float()
        r["d_pre_weight"] = (d_normed * hat).sum(0)
        r["d_pre_bias"] = d_normed.sum(0) if s["pre_bias"] is not None else None
        d = d + _through_norm(c["pre"], d_normed * s["pre_weight"], hat, rstd)
    r["d_residual"] = d.to(t)
    v, u = c["scale"] * d, s["branch"].float()
    if c["post"] != "none":
        hat, rstd = _normalised(c["post"], u)
        u = _affine(hat, s["post_weight"], s["post_bias"])
    if s["gate"] is not None:
        n = s["gate"].shape[0] * c["gate_rows"]
        both = torch.nn.functional.pad(v * u, (0, 0, 0, n - c["rows"]))
        r["d_gate"] = both.view(s["gate"].shape[0], c["gate_rows"], c["dim"]).sum(1).to(t)
        v = v * _gate_rows(s, c)
    if c["post"] != "none":
        r["d_post_weight"] = (v * hat).sum(0)
        r["d_post_bias"] = v.sum(0) if s["post_bias"] is not None else None
        v = _through_norm(c["post"], v * s["post_weight"], hat, rstd)
    r["d_branch"] = v.to(t)
    return r


def _threshold(p):
    return int(math.floor(p * 65536 + 0.5))


def _plain_philox(n_blocks, call, seed):
    """The four words of each Philox-4x32-10 block (block low, call low, call high, 2^31 + block high 2^16), as 32-bit values in int64."""
    i = torch.arange(n_blocks, device="cuda", dtype=torch.int64)
    low = 0xFFFFFFFF
    c0, c3 = i & low, (i >> 32 << 16) + (1 << 31)
    c1, c2 = torch.full_like(i, call & low), torch.full_like(i, call >> 32)
    k0, k1 = seed & low, seed >> 32 & low

    def product(constant, v):
        # the halves of a 32 x 32 bit product, 16 bits of the factor at a time
        a, b = constant * (v & 0xFFFF), constant * (v >> 16)
        lower = a + ((b & 0xFFFF) << 16)
        return (b >> 16) + (lower >> 32), lower & low

    for _ in range(10):
        h0, l0 = product(0xD2511F53, c0)
        h1, l1 = product(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], 1)


def _plain_dropout(s, c, t):
    n, T = c["rows"] * c["dim"], _threshold(c["p"])
    words = _plain_philox((n + 7) // 8, s["call"], s["seed"])
    draws = torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[:n].view(c["rows"], c["dim"])
    y = torch.where(draws >= T, s["x"].float() * (65536 / (65536 - T)), torch.zeros((), device="cuda"))
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return dict(y=y.to(t))


_PLAIN = {"dense": _plain_dense, "dense_backward": _plain_dense_backward, "norm": _plain_norm, "norm_backward": _plain_norm_backward, "dropout": _plain_dropout}


# ---- one pass ----------------------------------------------------------------------------------------------------------------------------------
def run(state):
    s, c = state, state["case"]
    if not own:
        return _PLAIN[c["kind"]](s, c, TYPES[c["type"]])
    pkg = importlib.import_module("rl-tools_b200")
    if c["kind"] == "dense":
        pre, y = pkg.dense_residual_forward(s["W"], s["x"], c["act"], bias=s["bias"], residual=s["residual"], scale=c["scale"], want_pre=c["keep_pre"])
        return dict(y=y, pre=pre)
    if c["kind"] == "dense_backward":
        d_W, d_bias, d_in = pkg.dense_residual_backward(s["W"], s["x"], s["d_pre"], add=s["add"], pre_in=s["pre_in"], act_in=c["act"])
        return dict(d_in=d_in, d_W=d_W, d_bias=d_bias)
    if c["kind"] == "norm":
        out, normed = pkg.norm_residual_forward(s["branch"], s["residual"], post=c["post"], post_weight=s["post_weight"], post_bias=s["post_bias"], gate=s["gate"],
                                                gate_rows=c["gate_rows"], scale=c["scale"], pre=c["pre"], pre_weight=s["pre_weight"], pre_bias=s["pre_bias"], epsilon=EPSILON)
        return dict(out=out, normed=normed)
    if c["kind"] == "norm_backward":
        return pkg.norm_residual_backward(s["branch"], s["residual"], s["d_out"], s["d_normed"], post=c["post"], post_weight=s["post_weight"], post_bias=s["post_bias"],
                                          gate=s["gate"], gate_rows=c["gate_rows"], scale=c["scale"], pre=c["pre"], pre_weight=s["pre_weight"], pre_bias=s["pre_bias"],
                                          epsilon=EPSILON)
    return dict(y=pkg.dropout(s["x"], c["p"], s["seed"], call_index=s["call"], residual=s["residual"]))


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------------------------------
def _act64(name, v):
    """(value, slope) of the activation, the slope by the chain of its parts."""
    one = torch.ones_like(v)
    if name == "relu":
        return v.clamp(min=0), (v > 0).double()
    if name == "tanh":
        return torch.tanh(v), 1 / torch.cosh(v) ** 2
    if name in ("sigmoid", "silu"):
        s = torch.special.expit(v)
        slope = s * torch.special.expit(-v)
        return (s, slope) if name == "sigmoid" else (v * s, s + v * slope)
    if name == "gelu":
        cdf = 0.5 * torch.special.erfc(-v / 2 ** 0.5)
        return v * cdf, cdf + v * torch.exp(-v * v / 2) / (2 * math.pi) ** 0.5
    return v, one


def _norm64(kind, v):
    centred = v - v.mean(1, keepdim=True) if kind == "layer" else v
    power = centred.pow(2).sum(1, keepdim=True) / v.shape[1] + EPSILON
    return centred / power.sqrt(), power


def _slope64(kind, d_hat, hat, power):
    """The norm's Jacobian, applied to d_hat: the part along the row (and, for the layer norm, along the constant row) is taken out."""
    n = hat.shape[1]
    along = hat * (torch.einsum("rd,rd->r", d_hat, hat) / n)[:, None]
    mean = torch.einsum("rd->r", d_hat)[:, None] / n if kind == "layer" else 0
    return (d_hat - mean - along) / power.sqrt()


def exact(case, seed):
    c, kind = case, case["kind"]
    s = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in prepare(case, seed).items()}
    if kind == "dense":
        pre = torch.einsum("bi,oi->bo", s["x"], s["W"])
        pre = pre if s["bias"] is None else pre + s["bias"][None]
        y = _act64(c["act"], pre)[0] * c["scale"] + (0 if s["residual"] is None else s["residual"])
        return dict(y=y, pre=pre if c["keep_pre"] else None)
    if kind == "dense_backward":
        d_x = torch.einsum("bo,oi->bi", s["d_pre"], s["W"]) + (0 if s["add"] is None else s["add"])
        slope = 1 if s["pre_in"] is None else _act64(c["act"], s["pre_in"])[1]
        return dict(d_in=d_x * slope, d_W=torch.einsum("bo,bi->oi", s["d_pre"], s["x"]), d_bias=torch.einsum("bo->o", s["d_pre"]))
    if kind == "dropout":
        return _exact_dropout(c, s)
    ones = torch.ones(c["rows"], c["dim"], device="cuda", dtype=torch.float64)
    group = torch.arange(c["rows"], device="cuda") // max(1, c["gate_rows"])
    gate = ones if s["gate"] is None else s["gate"][group]
    post_w, post_b = (0 * ones[0] + (f if s[k] is None else s[k]) for k, f in (("post_weight", 1), ("post_bias", 0)))
    pre_w, pre_b = (0 * ones[0] + (f if s[k] is None else s[k]) for k, f in (("pre_weight", 1), ("pre_bias", 0)))
    hat, power = (s["branch"], None) if c["post"] == "none" else _norm64(c["post"], s["branch"])
    u = hat * post_w + post_b
    if kind == "norm":
        out = s["residual"] + c["scale"] * gate * u
        return dict(out=out, normed=None if c["pre"] == "none" else _norm64(c["pre"], out)[0] * pre_w + pre_b)
    d, r = s["d_out"], dict(d_pre_weight=None, d_pre_bias=None, d_post_weight=None, d_post_bias=None, d_gate=None)
    if c["pre"] != "none":
        out_hat, out_power = _norm64(c["pre"], s["residual"])
        d = d + _slope64(c["pre"], s["d_normed"] * pre_w, out_hat, out_power)
        r["d_pre_weight"] = torch.einsum("rd,rd->d", s["d_normed"], out_hat)
        r["d_pre_bias"] = None if s["pre_bias"] is None else torch.einsum("rd->d", s["d_normed"])
    r["d_residual"] = d
    d_u = c["scale"] * d * gate
    if s["gate"] is not None:
        r["d_gate"] = torch.zeros_like(s["gate"]).index_add_(0, group, c["scale"] * d * u)
    if c["post"] != "none":
        r["d_post_weight"] = torch.einsum("rd,rd->d", d_u, hat)
        r["d_post_bias"] = None if s["post_bias"] is None else torch.einsum("rd->d", d_u)
        d_u = _slope64(c["post"], d_u * post_w, hat, power)
    r["d_branch"] = d_u
    return r


def _exact_dropout(c, s):
    n, m = c["rows"] * c["dim"], np.uint64(0xFFFFFFFF)
    block = np.arange((n + 7) // 8, dtype=np.uint64)
    w = [block & m, np.full_like(block, s["call"] & 0xFFFFFFFF), np.full_like(block, s["call"] >> 32), np.uint64(0x80000000) + ((block >> np.uint64(32)) << np.uint64(16))]
    key = [s["seed"] & 0xFFFFFFFF, s["seed"] >> 32 & 0xFFFFFFFF]
    for _ in range(10):
        a, b = w[0] * np.uint64(0xD2511F53), w[2] * np.uint64(0xCD9E8D57)          # 64-bit products of 32-bit words
        w = [(b >> np.uint64(32)) ^ w[1] ^ np.uint64(key[0]), b & m, (a >> np.uint64(32)) ^ w[3] ^ np.uint64(key[1]), a & m]
        key = [key[0] + 0x9E3779B9 & 0xFFFFFFFF, key[1] + 0xBB67AE85 & 0xFFFFFFFF]
    halves = np.stack(w, 1).astype("<u4").view("<u2").reshape(-1)[:n].reshape(c["rows"], c["dim"])
    dropped = int(math.floor(c["p"] * 65536 + 0.5))
    keep = torch.from_numpy((halves.astype(np.int32) >= dropped)).cuda()
    y = torch.where(keep, s["x"] / (1 - dropped / 65536), torch.zeros_like(s["x"]))
    return dict(y=y if s["residual"] is None else y + s["residual"])


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------------------------------
def work(case):
    c, b = case, torch.finfo(TYPES[case["type"]]).bits // 8
    if c["kind"] == "dense":
        B, I, O = c["batch"], c["input"], c["output"]
        return dict(bytes=b * (O * I + B * I + B * O * (1 + c["residual"] + c["keep_pre"])) + 4 * O * c["bias"], flops=2 * B * I * O)
    if c["kind"] == "dense_backward":
        B, I, O = c["batch"], c["input"], c["output"]
        return dict(bytes=b * (O * I + B * O + B * I * (2 + c["add"] + (c["act"] != "identity"))) + 4 * (O * I + O), flops=4 * B * I * O)
    n = c["rows"] * c["dim"]
    if c["kind"] == "dropout":
        return dict(bytes=b * n * (2 + c["residual"]), flops=2 * n)
    has_pre, norms = c["pre"] != "none", (c["pre"] != "none") + (c["post"] != "none")
    gate = 0 if not c["gate_rows"] else -(-c["rows"] // c["gate_rows"]) * c["dim"]
    params = 4 * c["dim"] * norms * (1 + c["bias"])
    if c["kind"] == "norm":
        return dict(bytes=b * (n * (3 + has_pre) + gate) + params, flops=n * (3 + 5 * norms))
    # the forward sum is read for the norm behind it alone
    return dict(bytes=b * (n * (4 + 2 * has_pre) + 2 * gate) + 2 * params, flops=n * (4 + 12 * norms))
