"""The operators of residual networks against their 64-bit definitions: sizes that fit no tile, rows at odd addresses, views into wider tables, every type, in-place
forms, captured graphs and other streams. The bounds count roundings (residual_reference.py)."""
import math

import pytest
import torch

from residual_reference import (U32, half_step, smallest, act64, slope64, product_error, activation_error, norm_residual64, norm64, dropout64, assert_within)

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def table(rows, cols, dtype, g, pad=0, offset=0, std=1.0, mean=0.0):
    """A [rows, cols] view into a table with `pad` more columns, starting `offset` columns in; the table is returned too, to see that its other columns stay."""
    t = (torch.randn(rows, cols + pad, device="cuda", generator=g) * std + mean).to(dtype)
    return t[:, offset:offset + cols], t


def blank(rows, cols, dtype, pad=0, offset=0, fill=7.0):
    t = torch.full((rows, cols + pad), fill, device="cuda", dtype=dtype)
    return t[:, offset:offset + cols], t


def untouched(t, cols, offset, fill=7.0):
    other = torch.cat([t[:, :offset], t[:, offset + cols:]], 1)
    return bool((other == fill).all())


def seeded(n):
    return torch.Generator(device="cuda").manual_seed(n)


# sizes: one token, a few, tiles and their neighbours, odd depths, depths of one element; the largest are small enough for a 64-bit product in milliseconds
DENSE_SIZES = [(1, 1, 1), (1, 64, 256), (1, 1024, 777), (2, 17, 5), (5, 250, 131), (8, 512, 512), (16, 4096, 33), (31, 77, 129), (33, 264, 136), (64, 256, 1024), (65, 128, 64),
               (127, 63, 255), (128, 64, 256), (129, 65, 257), (200, 1000, 320), (256, 256, 256), (300, 40, 1111), (513, 640, 384), (1003, 777, 1001), (2048, 512, 768), (4100, 72, 40),
               (16400, 72, 300), (5003, 200, 1000), (1100, 2050, 2100), (128, 4096, 96), (33, 4000, 520), (100, 1030, 1000), (260, 2000, 250)]


def dense_inputs(B, I, O, dtype, pad, offset, seed):
    g = seeded(seed)
    x, _ = table(B, I, dtype, g, pad, offset)
    W, _ = table(O, I, dtype, g, pad, offset, std=1 / math.sqrt(I))
    return g, x, W


@pytest.mark.parametrize("act", ["identity", "relu", "tanh", "fast_tanh", "sigmoid", "gelu", "silu"])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_dense_forward_activations(lib, dtype, act):
    check_forward(lib, 150, 200, 170, dtype, act, 0, 0, True, True, 0.5, True, 1)
    check_forward(lib, 3, 200, 170, dtype, act, 0, 0, True, True, 0.5, True, 1)


@pytest.mark.parametrize("size", DENSE_SIZES)
@pytest.mark.parametrize("layout", [(0, 0), (8, 0), (24, 8), (5, 3)])
def test_dense_forward_sizes(lib, size, layout):
    B, I, O = size
    dtype = BF16 if (B + I + O) % 2 else F16
    check_forward(lib, B, I, O, dtype, "gelu", *layout, bias=True, residual=True, scale=0.5, keep=True, seed=B)
    check_forward(lib, B, I, O, dtype, "identity", *layout, bias=False, residual=False, scale=1.0, keep=False, seed=B + 1)


def check_forward(lib, B, I, O, dtype, act, pad, offset, bias, residual, scale, keep, seed):
    g, x, W = dense_inputs(B, I, O, dtype, pad, offset, seed)
    b = torch.randn(O, device="cuda", generator=g) if bias else None
    r = table(B, O, dtype, g, pad, offset)[0] if residual else None
    y, y_table = blank(B, O, dtype, pad, offset)
    pre, pre_table = blank(B, O, dtype, pad, offset) if keep else (None, None)
    lib.dense_residual_forward(W, x, act, bias=b, residual=r, scale=scale, y=y, pre=pre)
    want_pre = x.double() @ W.double().t() + (0 if b is None else b.double())
    err = product_error(x.double(), W.double()) + 2 * U32 * (1 + want_pre.abs())
    want = scale * act64(act, want_pre) + (0 if r is None else r.double())
    # the steepest slope is 1.13; one more rounding each for the scale and the sum
    err_y = abs(scale) * (1.13 * err + activation_error(want_pre)) + 4 * U32 * (want.abs() + (0 if r is None else r.double().abs()))
    assert_within(y, want, err_y + half_step(dtype) * (want.abs() + err_y) + smallest(dtype), "y")
    assert untouched(y_table, O, offset)
    if keep:
        assert_within(pre, want_pre, err + half_step(dtype) * (want_pre.abs() + err) + smallest(dtype), "pre")
        assert untouched(pre_table, O, offset)


@pytest.mark.parametrize("size", DENSE_SIZES)
@pytest.mark.parametrize("layout", [(0, 0), (24, 8), (5, 3)])
def test_dense_backward_sizes(lib, size, layout):
    B, I, O = size
    dtype = F16 if (B + I + O) % 2 else BF16
    check_backward(lib, B, I, O, dtype, "gelu", *layout, add=True, seed=B)
    check_backward(lib, B, I, O, dtype, "identity", *layout, add=False, seed=B + 1)


@pytest.mark.parametrize("act", ["relu", "tanh", "fast_tanh", "sigmoid", "gelu", "silu"])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_dense_backward_activations(lib, dtype, act):
    check_backward(lib, 140, 170, 200, dtype, act, 0, 0, True, 3)
    check_backward(lib, 2, 170, 200, dtype, act, 0, 0, True, 3)


def check_backward(lib, B, I, O, dtype, act, pad, offset, add, seed):
    g, x, W = dense_inputs(B, I, O, dtype, pad, offset, seed)
    d_pre = table(B, O, dtype, g, pad, offset, std=0.25)[0]
    a = table(B, I, dtype, g, pad, offset)[0] if add else None
    pre = table(B, I, dtype, g, pad, offset)[0] if act != "identity" else None
    d_in, d_in_table = blank(B, I, dtype, pad, offset)
    d_W, d_b, d_in = lib.dense_residual_backward(W, x, d_pre, add=a, pre_in=pre, act_in=act, d_in=d_in)
    X, D, w = x.double(), d_pre.double(), W.double()
    inner = D @ w + (0 if a is None else a.double())
    err = product_error(D, w.t()) + 2 * U32 * inner.abs()
    slope = 1.0 if pre is None else slope64(act, pre.double())
    want = inner * slope
    err_in = 1.13 * err + (0 if pre is None else activation_error(pre.double()) * (1 + pre.double().abs()) * (inner.abs() + err)) + 2 * U32 * want.abs()
    assert_within(d_in, want, err_in + half_step(dtype) * (want.abs() + err_in) + smallest(dtype), "d_in")
    assert untouched(d_in_table, I, offset)
    assert_within(d_W, D.t() @ X, product_error(D.t().contiguous(), X.t().contiguous()) + 1e-30, "d_W")
    assert_within(d_b, D.sum(0), (B + 2) * U32 * D.abs().sum(0) + 1e-30, "d_bias")


def test_dense_backward_parts_and_accumulation(lib):
    g, x, W = dense_inputs(300, 130, 70, BF16, 0, 0, 5)
    d_pre = table(300, 70, BF16, g, std=0.25)[0]
    d_W, d_b, d_in = lib.dense_residual_backward(W, x, d_pre)
    again_W, again_b, again_in = lib.dense_residual_backward(W, x, d_pre)
    assert torch.equal(d_W, again_W) and torch.equal(d_b, again_b) and torch.equal(d_in, again_in)          # a fixed order
    assert torch.equal(lib.dense_residual_backward(W, x, d_pre, want_grads=False)[2], d_in)
    only = lib.dense_residual_backward(W, x, d_pre, want_d_in=False)
    assert torch.equal(only[0], d_W) and torch.equal(only[1], d_b) and only[2] is None
    base_W, base_b = torch.randn(70, 130, device="cuda", generator=g), torch.randn(70, device="cuda", generator=g)
    sum_W, sum_b = base_W.clone(), base_b.clone()
    lib.dense_residual_backward(W, x, d_pre, d_W=sum_W, d_bias=sum_b, want_d_in=False)
    assert torch.equal(sum_W, base_W + d_W) and torch.equal(sum_b, base_b + d_b)


def test_dense_gradient_of_an_empty_batch(lib):
    W = torch.randn(6, 10, device="cuda").to(BF16)
    x, d_pre = W.new_empty(0, 10), W.new_empty(0, 6)
    pre, y = lib.dense_residual_forward(W, x, "relu", want_pre=True)
    assert y.shape == (0, 6) and pre.shape == (0, 6)
    d_W, d_b, d_in = lib.dense_residual_backward(W, x, d_pre)
    assert d_in.shape == (0, 10) and not d_W.any() and not d_b.any()
    d_W.fill_(2.0)
    d_b.fill_(3.0)
    lib.dense_residual_backward(W, x, d_pre, d_W=d_W, d_bias=d_b)
    assert (d_W == 2).all() and (d_b == 3).all()


def test_dense_weight_gradient_of_a_long_batch_keeps_fp32(lib):
    """40,000 rows whose products all have one sign: an accumulator that truncates would fall behind by (40,000 / 16) 2^-24 of the sum. The error stays below what 512 rows in
    one accumulator (32 truncating additions of 16 products, and the products within each) and about 80 fp32 additions of the pieces explain."""
    B, I, O = 40000, 96, 72
    g = seeded(11)
    x, d_pre = (torch.rand(B, n, device="cuda", generator=g).to(BF16) for n in (I, O))
    d_W, d_b, _ = lib.dense_residual_backward(x.new_zeros(O, I), x, d_pre, want_d_in=False)
    want = d_pre.double().t() @ x.double()
    assert_within(d_W, want, (2 * 40 + 80) * U32 * want, "d_W")


@pytest.mark.parametrize("batch", [4, 260])
def test_dense_in_place_forms(lib, batch):
    g, x, W = dense_inputs(batch, 96, 80, BF16, 0, 0, 6)
    r = table(batch, 80, BF16, g)[0]
    _, y = lib.dense_residual_forward(W, x, "silu", residual=r, scale=0.5)
    kept = r.clone()
    lib.dense_residual_forward(W, x, "silu", residual=kept, scale=0.5, y=kept)
    assert torch.equal(kept, y)
    d_pre, a, pre = table(batch, 80, BF16, g)[0], table(batch, 96, BF16, g)[0], table(batch, 96, BF16, g)[0]
    want = lib.dense_residual_backward(W, x, d_pre, add=a, pre_in=pre, act_in="tanh", want_grads=False)[2]
    for over in (a.clone(), pre.clone()):
        args = dict(add=a, pre_in=pre)
        args["add" if torch.equal(over, a) else "pre_in"] = over
        lib.dense_residual_backward(W, x, d_pre, act_in="tanh", want_grads=False, d_in=over, **args)
        assert torch.equal(over, want)
    d = lib.dense_residual_backward_activation(pre, a, "gelu", scale=0.5)
    for over in (a.clone(), pre.clone()):
        args = dict(pre=pre, d_y=a)
        args["d_y" if torch.equal(over, a) else "pre"] = over
        assert torch.equal(lib.dense_residual_backward_activation(act="gelu", scale=0.5, d_pre=over, **args), d)


@pytest.mark.parametrize("act", ["identity", "relu", "tanh", "fast_tanh", "sigmoid", "gelu", "silu"])
@pytest.mark.parametrize("shape, layout", [((1, 1), (0, 0)), ((37, 129), (0, 0)), ((64, 256), (8, 8)), ((33, 40), (3, 1))])
def test_dense_backward_activation(lib, act, shape, layout):
    g = seeded(7)
    for dtype in (BF16, F16):
        pre, d = table(*shape, dtype, g, *layout)[0], table(*shape, dtype, g, *layout)[0]
        out, out_table = blank(*shape, dtype, *layout)
        lib.dense_residual_backward_activation(pre, d, act, scale=0.25, d_pre=out)
        want = 0.25 * slope64(act, pre.double()) * d.double()
        err = 0.25 * d.double().abs() * activation_error(pre.double()) * (1 + pre.double().abs())
        assert_within(out, want, err + half_step(dtype) * (want.abs() + err) + smallest(dtype), "d_pre")
        assert untouched(out_table, shape[1], layout[1])


def test_dense_values_that_are_not_finite_stay_in_their_row(lib):
    """An infinity or NaN in one row of x, or behind the views' rows, reaches that row of y alone."""
    for B in (9, 140):
        g = seeded(8)
        wide = torch.full((B, 72 + 16), float("nan"), device="cuda", dtype=BF16)
        wide[:, 8:80] = torch.randn(B, 72, device="cuda", generator=g).to(BF16)
        x, W = wide[:, 8:80], torch.randn(50, 72, device="cuda", generator=g).to(BF16)
        clean = lib.dense_residual_forward(W, x, "identity")[1].clone()
        assert torch.isfinite(clean).all()
        wide[3, 10], wide[5, 20] = float("inf"), float("nan")
        y = lib.dense_residual_forward(W, x, "identity")[1]
        rows = [i for i in range(B) if i not in (3, 5)]
        assert torch.equal(y[rows], clean[rows]) and not torch.isfinite(y[3]).any() and torch.isnan(y[5]).all()


@pytest.mark.parametrize("layout", [(16, 8), (5, 3)])
@pytest.mark.parametrize("B", [9, 140])
def test_dense_backward_reads_only_its_views(lib, B, layout):
    """NaN behind and in front of every operand's rows, and in the rows behind the last, reach nothing."""
    g, (pad, offset), I, O = seeded(9), layout, 72, 50

    def island(rows, cols, std=1.0):
        t = torch.full((rows + 3, cols + pad), float("nan"), device="cuda", dtype=BF16)
        t[:rows, offset:offset + cols] = (torch.randn(rows, cols, device="cuda", generator=g) * std).to(BF16)
        return t[:rows, offset:offset + cols]

    W, x, d, a, p = island(O, I), island(B, I), island(B, O), island(B, I), island(B, I)
    got = lib.dense_residual_backward(W, x, d, add=a, pre_in=p, act_in="silu")
    want = lib.dense_residual_backward(*(t.contiguous() for t in (W, x, d)), add=a.contiguous(), pre_in=p.contiguous(), act_in="silu")
    for u, v in zip(got, want):
        assert torch.isfinite(u).all() and torch.equal(u, v)
    pre, y = lib.dense_residual_forward(W, x, "silu", residual=island(B, O), want_pre=True)
    assert torch.isfinite(y).all() and torch.isfinite(pre).all()


def test_dense_weight_gradients_at_any_address_and_alone(lib):
    """Slices of a parameter arena at odd offsets; through the C entry point one gradient without the other."""
    B, I, O = 700, 90, 77
    g, x, _ = dense_inputs(B, I, O, BF16, 0, 0, 12)
    d = table(B, O, BF16, g, std=0.25)[0]
    W = x.new_zeros(O, I)
    d_W, d_b, _ = lib.dense_residual_backward(W, x, d, want_d_in=False)
    arena = torch.full((O * I + O + 8,), 5.0, device="cuda")
    a_W, a_b = arena[3:3 + O * I].view(O, I), arena[3 + O * I:3 + O * I + O]
    a_W.zero_()
    a_b.zero_()
    lib.dense_residual_backward(W, x, d, d_W=a_W, d_bias=a_b, want_d_in=False)
    assert torch.equal(a_W, d_W) and torch.equal(a_b, d_b) and (arena[:3] == 5).all() and (arena[3 + O * I + O:] == 5).all()
    L, st = lib.lib(), torch.cuda.current_stream().cuda_stream
    n = L.b200rl_dense_residual_backward_weights_workspace_bytes(x.data_ptr(), I, d.data_ptr(), O, a_W.data_ptr(), B, I, O)
    ws = torch.empty(max(n, 16), device="cuda", dtype=torch.uint8)
    only_W, only_b = torch.empty_like(d_W), torch.ones_like(d_b)
    assert L.b200rl_dense_residual_backward_weights(1, x.data_ptr(), I, d.data_ptr(), O, only_W.data_ptr(), None, 0, B, I, O, ws.data_ptr(), n, st) == 0
    assert L.b200rl_dense_residual_backward_weights(1, None, 0, d.data_ptr(), O, None, only_b.data_ptr(), 1, B, I, O, None, 0, st) == 0
    assert torch.equal(only_W, d_W)
    want = d.double().sum(0)
    assert_within(only_b, 1 + want, (B + 3) * U32 * (1 + d.double().abs().sum(0)), "d_bias")


def test_offsets_beyond_32_bits(lib):
    """Rows 40,000 elements apart: the last ones lie more than 2^31 elements behind the first."""
    R, ld, I, O = 66000, 40000, 64, 40
    assert R * ld > 2 ** 31
    big = torch.empty(R, ld, device="cuda", dtype=BF16)
    x, y, r = big[:, :I], big[:, 1000:1000 + O], big[:, 2000:2000 + O]
    g = seeded(13)
    x.copy_(torch.randn(R, I, device="cuda", generator=g))
    r.copy_(torch.randn(R, O, device="cuda", generator=g))
    W = torch.randn(O, I, device="cuda", generator=g).to(BF16)
    lib.dense_residual_forward(W, x, "relu", residual=r, y=y)
    assert torch.equal(y, lib.dense_residual_forward(W, x.contiguous(), "relu", residual=r.contiguous())[1])
    d_W, d_b, d_in = lib.dense_residual_backward(W, x, r, add=x, d_in=big[:, 3000:3000 + I])
    want = lib.dense_residual_backward(W, x.contiguous(), r.contiguous(), add=x.contiguous())
    assert all(torch.equal(a, b) for a, b in zip((d_W, d_b, d_in), want))
    out, normed = lib.norm_residual_forward(y, r, post="rms", pre="layer", out=big[:, 4000:4000 + O], normed=big[:, 5000:5000 + O])
    want = lib.norm_residual_forward(y.contiguous(), r.contiguous(), post="rms", pre="layer")
    assert torch.equal(out, want[0]) and torch.equal(normed, want[1])
    got = lib.norm_residual_backward(y, out, r, normed, post="rms", pre="layer")
    want = lib.norm_residual_backward(y.contiguous(), out.contiguous(), r.contiguous(), normed.contiguous(), post="rms", pre="layer")
    assert torch.equal(got["d_branch"], want["d_branch"]) and torch.equal(got["d_residual"], want["d_residual"])
    assert torch.equal(lib.dropout(x, 0.3, 5, y=big[:, 6000:6000 + I]), lib.dropout(x.contiguous(), 0.3, 5))


def test_calls_on_two_streams_at_once(lib):
    """Nothing is shared between calls: products that split k and share workspaces' sizes run on two streams and give what each gives alone."""
    jobs = []
    for n, (B, I, O) in enumerate([(3000, 70, 66), (2900, 66, 70)]):
        g, x, W = dense_inputs(B, I, O, BF16, 0, 0, n)
        d = table(B, O, BF16, g, std=0.25)[0]
        jobs.append((W, x, d, [t.clone() for t in lib.dense_residual_backward(W, x, d)]))
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream() for _ in jobs], [[], []]
    for _ in range(20):
        for s, (W, x, d, _), out in zip(streams, jobs, results):
            with torch.cuda.stream(s):
                out.append(lib.dense_residual_backward(W, x, d))
    torch.cuda.synchronize()
    for (_, _, _, want), out in zip(jobs, results):
        assert all(torch.equal(a, b) for got in out for a, b in zip(got, want))


FIRST_CALL = """
import sys
sys.path.insert(0, {root!r})
import __graft_entry__ as entry
lib = entry.load_package()
import torch
T = torch.bfloat16
x, W, d = torch.ones(300, 64, device="cuda", dtype=T), torch.ones(48, 64, device="cuda", dtype=T), torch.ones(300, 48, device="cuda", dtype=T)
w = torch.ones(64, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = lib.dense_residual_forward(W, x, "identity")[1]
    one = lib.dense_residual_forward(W, x[:1], "identity")[1]
    d_W, d_b, d_in = lib.dense_residual_backward(W, x, d)
    out, normed = lib.norm_residual_forward(x, x, post="rms", post_weight=w, pre="layer", pre_weight=w)
    g = lib.norm_residual_backward(x, out, x, normed, post="rms", post_weight=w, pre="layer", pre_weight=w)
    drop = lib.dropout(x, 0.5, 1)
graph.replay()
torch.cuda.synchronize()
assert (y == 64).all() and (one == 64).all() and (d_W == 300).all() and (d_b == 300).all() and (d_in == 48).all()
assert torch.isfinite(g["d_branch"]).all() and ((drop == 0) | (drop == 2)).all()
print("captured first")
"""


def test_the_first_call_of_a_process_may_be_captured(lib):
    import subprocess
    import sys
    from conftest import ROOT
    done = subprocess.run([sys.executable, "-c", FIRST_CALL.format(root=ROOT)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured first" in done.stdout, done.stdout + done.stderr


# ---- norms -------------------------------------------------------------------------------------------------------------------------------------
NORM_SIZES = [(1, 1), (1, 4096), (3, 5), (7, 64), (50, 257), (33, 512), (130, 777), (64, 1024), (20, 2048), (9, 2049), (300, 100), (5, 4097), (4, 8192), (700, 33), (2500, 16), (5003, 40), (2000, 600)]


def norm_inputs(R, D, dtype, post, pre, gate_rows, bias, layout, seed):
    g = seeded(seed)
    p = lambda has, mean: torch.randn(D, device="cuda", generator=g) * 0.2 + mean if has else None
    s = dict(branch=table(R, D, dtype, g, *layout, std=0.8, mean=0.2)[0], residual=table(R, D, dtype, g, *layout, std=1.5, mean=-0.3)[0], post=post, pre=pre, gate_rows=gate_rows, scale=0.5,
             gate=table(-(-R // gate_rows), D, dtype, g, *layout, std=0.3, mean=0.7)[0] if gate_rows else None,
             post_weight=p(post != "none", 1.0), post_bias=p(bias and post != "none", 0.0), pre_weight=p(pre != "none", 1.0), pre_bias=p(bias and pre != "none", 0.0), epsilon=1e-5)
    return g, s


def doubled(s):
    return {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in s.items()}


def hat_error(kind, v, epsilon, err_v=0.0):
    """How far fp32 statistics (sums of at most 64 additions in a row) leave a normalised row, and its values: (hat, rstd, bound)."""
    if kind == "none":
        return v, None, err_v + 0 * v
    mean = v.mean(1, keepdim=True) if kind == "layer" else 0 * v[:, :1]
    c = v - mean
    rstd = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + epsilon)
    hat = c * rstd
    err_in = err_v + 0 * v
    # the mean is off by 64 roundings of the mean magnitude and by the inputs' own errors, the standard deviation by 64 roundings of itself
    shift = 64 * U32 * v.abs().mean(1, keepdim=True) + err_in.mean(1, keepdim=True) if kind == "layer" else 0
    bound = rstd * (err_in + shift) + hat.abs() * (80 * U32 + rstd * ((err_in + shift) ** 2).mean(1, keepdim=True).sqrt()) + 4 * U32
    return hat, rstd, bound


@pytest.mark.parametrize("size", NORM_SIZES)
@pytest.mark.parametrize("kinds", [("rms", "rms"), ("layer", "layer"), ("none", "layer"), ("rms", "none")])
def test_norm_forward(lib, size, kinds):
    R, D = size
    for n, (dtype, layout, gate_rows) in enumerate([(BF16, (0, 0), 1), (F16, (24, 8), 0), (F32, (5, 3), 7), (F32, (0, 0), R), (BF16, (5, 3), 3)]):
        g, s = norm_inputs(R, D, dtype, *kinds, gate_rows, n % 2 == 0, layout, R + n)
        out, out_table = blank(R, D, dtype, *layout)
        normed, normed_table = blank(R, D, dtype, *layout) if kinds[1] != "none" else (None, None)
        lib.norm_residual_forward(**s, out=out, normed=normed)
        q = doubled(s)
        want, want_normed = norm_residual64(**q)
        _, _, err = hat_error(kinds[0], q["branch"], s["epsilon"])
        u = norm64(kinds[0], q["branch"], q["post_weight"], q["post_bias"], s["epsilon"])
        err = err * (1 if q["post_weight"] is None else q["post_weight"].abs()) + 4 * U32 * (1 + u.abs())
        gate = 1 if q["gate"] is None else q["gate"][torch.arange(R, device="cuda") // gate_rows].abs()
        err = 0.5 * err * gate + 4 * U32 * (want.abs() + u.abs() * gate)
        assert_within(out, want, err + half_step(dtype) * (want.abs() + err) + smallest(dtype), f"out {dtype} {layout}")
        assert untouched(out_table, D, layout[1])
        if normed is not None:
            _, _, e = hat_error(kinds[1], want, s["epsilon"], err)
            e = e * q["pre_weight"].abs() + 4 * U32 * (1 + want_normed.abs())
            assert_within(normed, want_normed, e + half_step(dtype) * (want_normed.abs() + e) + smallest(dtype), f"normed {dtype} {layout}")
            assert untouched(normed_table, D, layout[1])


def gradients64(s, d_out, d_normed):
    """By automatic differentiation in 64 bits; `residual` of s stands for the sum that the norm behind it saw."""
    q = doubled(s)
    leaves = {k: q[k].detach().clone().requires_grad_(True) for k in ("branch", "residual", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias") if q[k] is not None}
    out = leaves["residual"]
    d = torch.zeros_like(out) if d_out is None else d_out.double()
    r = {}
    if s["pre"] != "none":
        keys = [k for k in ("pre_weight", "pre_bias") if k in leaves]
        normed = norm64(s["pre"], out, leaves.get("pre_weight"), leaves.get("pre_bias"), s["epsilon"])
        grads = torch.autograd.grad(normed, [out] + [leaves[k] for k in keys], d_normed.double())
        d = d + grads[0]
        r.update({"d_" + k: v for k, v in zip(keys, grads[1:])})
    r["d_residual"] = d
    if "branch" in leaves:
        keys = [k for k in ("branch", "gate", "post_weight", "post_bias") if k in leaves]
        u = norm64(s["post"], leaves["branch"], leaves.get("post_weight"), leaves.get("post_bias"), s["epsilon"])
        if "gate" in leaves:
            u = u * leaves["gate"][torch.arange(u.shape[0], device="cuda") // s["gate_rows"]]
        r.update({"d_" + k: v for k, v in zip(keys, torch.autograd.grad(s["scale"] * u, [leaves[k] for k in keys], d))})
    return r


def gradient_errors(s, d_out, d_normed):
    """Bounds on the fp32 errors of d_residual, d_branch, d_gate and the parameter gradients, from those of the normalised rows."""
    q = doubled(s)
    R = q["residual"].shape[0]
    d, e = (0 * q["residual"], 0 * q["residual"]) if d_out is None else (d_out.double(), 0 * q["residual"])
    r = {}

    def through(kind, g, err_g, weight, x):
        hat, rstd, err_hat = hat_error(kind, x, s["epsilon"])
        w = 1 if weight is None else weight.abs()
        a, ea = g.abs() * w, err_g * w + 2 * U32 * g.abs() * w
        m, em = a.mean(1, keepdim=True), ea.mean(1, keepdim=True)
        along = (a * hat.abs()).mean(1, keepdim=True)
        e_along = (a * err_hat + ea * hat.abs()).mean(1, keepdim=True) + 64 * U32 * along
        rel = (err_hat.abs() / (1 + hat.abs())).amax(1, keepdim=True) + 80 * U32
        err = rstd * (ea + (em + 64 * U32 * m) * (kind == "layer") + hat.abs() * e_along + err_hat * along) + rel * rstd * (a + m * (kind == "layer") + hat.abs() * along)
        return err, (g.abs() * err_hat + err_g * (hat.abs() + err_hat), g.abs() * hat.abs()), (hat, err_hat)

    def column(err, magnitude):
        return err.sum(0) + (R + 4) * U32 * magnitude.sum(0) + 1e-30

    if s["pre"] != "none":
        g = d_normed.double()
        err, product, _ = through(s["pre"], g, 0 * g, q["pre_weight"], q["residual"])
        r["d_pre_weight"], r["d_pre_bias"] = column(*product), column(0 * g, g.abs())
        e = e + err
    want = gradients64(s, d_out, d_normed)
    d = want["d_residual"]
    e = e + 2 * U32 * d.abs()
    r["d_residual"] = e
    if s["branch"] is not None:
        gate = 1 if q["gate"] is None else q["gate"][torch.arange(R, device="cuda") // s["gate_rows"]].abs()
        v, ev = abs(s["scale"]) * d.abs(), abs(s["scale"]) * e + U32 * d.abs()
        u = norm64(s["post"], q["branch"], q["post_weight"], q["post_bias"], s["epsilon"])
        eu = hat_error(s["post"], q["branch"], s["epsilon"])[2] * (1 if q["post_weight"] is None else q["post_weight"].abs()) + 4 * U32 * (1 + u.abs())
        if q["gate"] is not None:
            n = q["gate"].shape[0]
            index = torch.arange(R, device="cuda") // s["gate_rows"]
            total = lambda t: torch.zeros(n, t.shape[1], device="cuda", dtype=torch.float64).index_add_(0, index, t)
            r["d_gate"] = total(v * eu + ev * (u.abs() + eu)) + (min(R, s["gate_rows"]) + 4) * U32 * total(v * u.abs()) + 1e-30
        g, eg = v * gate, ev * gate + U32 * v * gate
        if s["post"] == "none":
            r["d_branch"] = eg
        else:
            r["d_branch"], product, _ = through(s["post"], g, eg, q["post_weight"], q["branch"])
            r["d_post_weight"], r["d_post_bias"] = column(*product), column(eg, g)
    return want, r


@pytest.mark.parametrize("size", NORM_SIZES)
@pytest.mark.parametrize("kinds", [("rms", "rms"), ("layer", "layer"), ("none", "layer"), ("rms", "none")])
def test_norm_backward(lib, size, kinds):
    R, D = size
    for n, (dtype, layout, gate_rows) in enumerate([(BF16, (0, 0), 1), (F16, (24, 8), 0), (F32, (5, 3), 7), (F32, (0, 0), R), (BF16, (5, 3), 3), (F16, (0, 0), max(1, R // 2))]):
        g, s = norm_inputs(R, D, dtype, *kinds, gate_rows, n % 2 == 0, layout, R + n)
        d_out = table(R, D, dtype, g, *layout, std=0.1)[0] if n != 1 or kinds[1] == "none" else None
        d_normed = table(R, D, dtype, g, *layout, std=0.1)[0] if kinds[1] != "none" else None
        outs = {k: blank(R, D, dtype, *layout) for k in ("d_branch", "d_residual")}
        if gate_rows:
            outs["d_gate"] = blank(-(-R // gate_rows), D, dtype, *layout)
        a = {k: v for k, v in s.items() if k != "residual"}
        got = lib.norm_residual_backward(out=s["residual"], d_out=d_out, d_normed=d_normed, **a, **{k: v[0] for k, v in outs.items()})
        want, bounds = gradient_errors(s, d_out, d_normed)
        for k, v in got.items():
            if v is None:
                assert k not in want, k
                continue
            rounded = half_step(dtype) * (want[k].abs() + bounds[k]) + smallest(dtype) if v.dtype != F32 else U32 * want[k].abs()
            assert_within(v, want[k], bounds[k] + rounded, f"{k} {dtype} {layout} gate_rows {gate_rows}")
        for k, (_, t) in outs.items():
            assert untouched(t, D, layout[1]), k


def test_norm_gradient_against_differences(lib):
    """The directional derivative of sum(d_out out + d_normed normed) along random directions of every input, by central differences of the 64-bit definition: the sum taken
    at the point that the backward pass is given (fp32: the rounding of `out` is 2^-24)."""
    R, D = 40, 96
    g, s = norm_inputs(R, D, F32, "layer", "rms", 3, True, (0, 0), 3)
    out, normed = lib.norm_residual_forward(**s)
    d_out, d_normed = (torch.randn(R, D, device="cuda", generator=g) for _ in range(2))
    a = {k: v for k, v in s.items() if k != "residual"}
    got = lib.norm_residual_backward(out=out, d_out=d_out, d_normed=d_normed, **a)
    q = doubled(s)

    def value(p):
        o, n = norm_residual64(**p)
        return (o * d_out.double()).sum() + (n * d_normed.double()).sum()

    for name in ("branch", "residual", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias"):
        direction = torch.randn(q[name].shape, device="cuda", dtype=torch.float64, generator=g)
        h = 1e-5
        slope = (value({**q, name: q[name] + h * direction}) - value({**q, name: q[name] - h * direction})) / (2 * h)
        along = (got["d_" + name].double() * direction).sum()
        scale = (got["d_" + name].double() * direction).abs().sum()
        # each gradient element is good to about 1e-5 of itself, the difference quotient to 1e-16 / h and h^2
        assert abs(float(along - slope)) <= 2e-5 * float(scale) + 1e-6, name


def test_norm_parts_and_in_place_forms(lib):
    R, D = 70, 200
    g, s = norm_inputs(R, D, BF16, "rms", "layer", 5, True, (0, 0), 4)
    out, normed = lib.norm_residual_forward(**s)
    stream = s["residual"].clone()
    o, n = lib.norm_residual_forward(**{**s, "residual": stream}, out=stream)
    assert o is stream and torch.equal(stream, out) and torch.equal(n, normed)
    # the first norm of a network, a block's end without a norm behind it, a branch without a stream
    only = lib.norm_residual_forward(None, out, pre="layer", pre_weight=s["pre_weight"], pre_bias=s["pre_bias"])
    assert torch.equal(only[0], out)
    end = lib.norm_residual_forward(**{**s, "pre": "none", "pre_weight": None, "pre_bias": None})
    assert torch.equal(end[0], out) and end[1] is None
    bare = lib.norm_residual_forward(**{**s, "residual": torch.zeros_like(out)})
    assert torch.equal(lib.norm_residual_forward(**{**s, "residual": None})[0], bare[0])
    d_out, d_normed = (torch.randn(R, D, device="cuda", generator=g).to(BF16) for _ in range(2))
    a = {k: v for k, v in s.items() if k != "residual"}
    full = lib.norm_residual_backward(out=out, d_out=d_out, d_normed=d_normed, **a)
    again = lib.norm_residual_backward(out=out, d_out=d_out, d_normed=d_normed, **a)
    assert all(torch.equal(full[k], again[k]) for k in full)
    over = d_out.clone()
    assert torch.equal(lib.norm_residual_backward(out=out, d_out=over, d_normed=d_normed, d_residual=over, **a)["d_residual"], full["d_residual"])
    base = {k: torch.randn(D, device="cuda", generator=g) for k in ("d_post_weight", "d_post_bias", "d_pre_weight", "d_pre_bias")}
    got = lib.norm_residual_backward(out=out, d_out=d_out, d_normed=d_normed, **a, **{k: v.clone() for k, v in base.items()})
    assert all(torch.equal(got[k], base[k] + full[k]) for k in base)
    stem = lib.norm_residual_backward(None, out, d_out, d_normed, pre="layer", pre_weight=s["pre_weight"], pre_bias=s["pre_bias"])
    assert torch.equal(stem["d_residual"], full["d_residual"]) and torch.equal(stem["d_pre_weight"], full["d_pre_weight"]) and stem["d_branch"] is None
    empty = lib.norm_residual_backward(out=out[:0], d_out=d_out[:0], d_normed=d_normed[:0], **{**a, "branch": s["branch"][:0], "gate": s["gate"][:0]})
    assert empty["d_branch"].shape == (0, D) and not empty["d_post_weight"].any() and not empty["d_pre_bias"].any()


def test_norm_rows_keep_apart(lib):
    """Rows that are constant, zero, huge or not finite: each row's result is what it is alone, and a variance of 0 leaves no NaN."""
    D = 96
    x = torch.randn(8, D, device="cuda")
    clean = lib.norm_residual_forward(None, x, pre="layer")[1].clone()
    x2 = x.clone()
    x2[1], x2[2], x2[3], x2[4, 5], x2[5, 6] = 0.0, 3.25, 1e18, float("nan"), float("inf")
    out, normed = lib.norm_residual_forward(None, x2, pre="layer")
    assert torch.equal(normed[[0, 6, 7]], clean[[0, 6, 7]]) and not normed[1].any() and not normed[2].any() and not normed[3].any() and torch.isnan(normed[4]).all()
    assert torch.isnan(normed[5]).any()


# ---- dropout -----------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("shape, layout", [((1, 1), (0, 0)), ((3, 5), (0, 0)), ((17, 24), (0, 0)), ((17, 24), (16, 8)), ((9, 130), (3, 1)), ((40, 1), (0, 0)), ((13, 4096), (0, 0)), ((700, 12), (4, 4))])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
def test_dropout(lib, shape, layout, p):
    for n, dtype in enumerate((F32, BF16, F16)):
        g = seeded(n)
        x, r = table(*shape, dtype, g, *layout)[0], table(*shape, dtype, g, *layout)[0]
        for residual in (None, r):
            y, y_table = blank(*shape, dtype, *layout)
            seed, call = 0x1234567890ABCDEF, (1 << 33) + 5
            lib.dropout(x, p, seed, stream_id=9, call_index=call, residual=residual, y=y)
            want, keep = dropout64(x.double(), p, seed, 9, call, None if residual is None else residual.double())
            err = 3 * U32 * (want.abs() + x.double().abs() * 2 + r.double().abs())
            assert_within(y, want, err + half_step(dtype) * want.abs() + smallest(dtype), f"y {dtype}")
            assert untouched(y_table, shape[1], layout[1])
            if residual is None:
                assert torch.equal(y.double() != 0, keep & (x != 0))


def test_dropout_drops_whatever_is_there(lib):
    x = torch.ones(64, 256, device="cuda")
    keep = lib.dropout(x, 0.5, 3) != 0
    bad = torch.where(keep, x, torch.full_like(x, float("nan")))
    bad[::2] = torch.where(keep[::2], x[::2], torch.full_like(x[::2], float("inf")))
    assert torch.equal(lib.dropout(bad, 0.5, 3), lib.dropout(x, 0.5, 3))
    assert not lib.dropout(torch.full_like(x, float("nan")), 1.0, 3).any()
    assert abs(float(keep.double().mean()) - 0.5) < 5 * 0.5 / math.sqrt(keep.numel())


def test_dropout_in_place_counter_and_graph(lib):
    """In place, with the call taken from the device: a captured call draws another mask with every replay, and the gradient's call the same one."""
    x, r = (torch.randn(33, 200, device="cuda") for _ in range(2))
    want = lib.dropout(x, 0.25, 5, call_index=7, residual=r)
    a = x.clone()
    assert torch.equal(lib.dropout(a, 0.25, 5, call_index=7, residual=r, y=a), want)
    b = r.clone()
    assert torch.equal(lib.dropout(x, 0.25, 5, call_index=7, residual=b, y=b), want)
    counter = torch.full((1,), 3, device="cuda", dtype=torch.int64)
    assert torch.equal(lib.dropout(x, 0.25, 5, call_index=4, call_counter=counter, residual=r), want)
    y, d = torch.empty_like(x), torch.empty_like(x)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        lib.dropout(x, 0.25, 5, call_counter=counter, y=y)
        lib.dropout(torch.ones_like(x), 0.25, 5, call_counter=counter, y=d)
        lib.counter_advance(counter)
    for call in (3, 4, 5):
        graph.replay()
        assert torch.equal(y, lib.dropout(x, 0.25, 5, call_index=call)) and torch.equal(y != 0, d != 0)


# ---- together ----------------------------------------------------------------------------------------------------------------------------------
class Block:
    """A residual block as a user writes it: pre norm -> widening layer -> narrowing layer -> dropout -> post norm, gate, residual."""

    def __init__(self, lib, D, H, dtype, seed=0):
        self.lib, self.D, self.H, self.dtype = lib, D, H, dtype
        g = seeded(seed)
        n = {"W1": (H, D), "b1": (H,), "W2": (D, H), "b2": (D,), "w_pre": (D,), "w_post": (D,)}
        sizes = [math.prod(s) for s in n.values()]
        self.params, self.grads, self.m, self.v = (torch.zeros(sum(sizes), device="cuda") for _ in range(4))
        self.state = torch.zeros(4, device="cuda", dtype=torch.int32)
        self.p, self.g, at = {}, {}, 0
        for (k, shape), size in zip(n.items(), sizes):
            self.p[k], self.g[k] = self.params[at:at + size].view(shape), self.grads[at:at + size].view(shape)
            at += size
            self.p[k].copy_(torch.ones(shape, device="cuda") if k.startswith("w_") else torch.randn(shape, device="cuda", generator=g) / math.sqrt(shape[-1]))
        self.gate = torch.full((1, D), 0.5, device="cuda", dtype=dtype)
        self.W1, self.W2 = torch.empty(H, D, device="cuda", dtype=dtype), torch.empty(D, H, device="cuda", dtype=dtype)

    def step(self, x, d_out, counter, rate=0.1):
        """Forward and backward; the parameter gradients land in the arena."""
        L, p, g, R = self.lib, self.p, self.g, x.shape[0]
        self.W1.copy_(p["W1"])
        self.W2.copy_(p["W2"])
        self.grads.zero_()
        _, n = L.norm_residual_forward(None, x, pre="rms", pre_weight=p["w_pre"])
        h_pre, h = L.dense_residual_forward(self.W1, n, "gelu", bias=p["b1"], want_pre=True)
        _, f = L.dense_residual_forward(self.W2, h, "identity", bias=p["b2"])
        kept = L.dropout(f, rate, 17, call_counter=counter)
        out, _ = L.norm_residual_forward(kept, x, post="layer", post_weight=p["w_post"], gate=self.gate, gate_rows=R, scale=0.7)
        b = L.norm_residual_backward(kept, None, d_out, post="layer", post_weight=p["w_post"], gate=self.gate, gate_rows=R, scale=0.7, d_post_weight=g["w_post"])
        d_f = L.dropout(b["d_branch"], rate, 17, call_counter=counter)
        _, _, d_h = L.dense_residual_backward(self.W2, h, d_f, d_W=g["W2"], d_bias=g["b2"], pre_in=h_pre, act_in="gelu")
        _, _, d_n = L.dense_residual_backward(self.W1, n, d_h, d_W=g["W1"], d_bias=g["b1"])
        s = L.norm_residual_backward(None, x, b["d_residual"], d_n, pre="rms", pre_weight=p["w_pre"], d_pre_weight=g["w_pre"])
        return out, s["d_residual"]

    def reference(self, x, d_out, call, rate=0.1):
        q = {k: (self.W1 if k == "W1" else self.W2 if k == "W2" else v).detach().double().requires_grad_(True) for k, v in self.p.items()}
        X = x.double().requires_grad_(True)
        n = norm64("rms", X, q["w_pre"], None, 1e-5)
        f = act64("gelu", n @ q["W1"].t() + q["b1"]) @ q["W2"].t() + q["b2"]
        kept = dropout64(f, rate, 17, 0, call)[0]
        out = X + 0.7 * self.gate.double() * norm64("layer", kept, q["w_post"], None, 1e-5)
        grads = torch.autograd.grad(out, [X] + list(q.values()), d_out.double())
        return out.detach(), grads[0], dict(zip(q, grads[1:]))

    def optimize(self):
        import ctypes as C
        L = self.lib
        L.check(L.lib().b200rl_adam_step(self.params.data_ptr(), self.grads.data_ptr(), self.m.data_ptr(), self.v.data_ptr(), self.params.numel(), L.AdamHyper(), self.state.data_ptr(),
                                         C.c_void_p(torch.cuda.current_stream().cuda_stream)))


def relative(a, b):
    return float((a.double() - b).norm() / b.norm())


@pytest.mark.parametrize("R, D, H, dtype", [(1, 64, 128, BF16), (37, 72, 200, F16), (256, 256, 512, BF16), (515, 130, 390, BF16)])
def test_a_block_forward_and_backward(lib, R, D, H, dtype):
    """The operators one after another as a residual block: every intermediate is rounded to 16 bits, about ten on the longest way, each by at most half a step."""
    block = Block(lib, D, H, dtype)
    g = seeded(1)
    x, d_out = (torch.randn(R, D, device="cuda", generator=g).to(dtype) for _ in range(2))
    counter = torch.full((1,), 11, device="cuda", dtype=torch.int64)
    out, d_x = block.step(x, d_out, counter)
    want, want_d_x, want_grads = block.reference(x, d_out, 11)
    limit = 10 * half_step(dtype) * 2          # the norms' gradients subtract rows' means: twice the share of the roundings
    assert relative(out, want) < limit and relative(d_x, want_d_x) < limit
    for k, v in want_grads.items():
        assert relative(block.g[k], v) < limit, k


def test_a_captured_training_step(lib):
    """A block's whole step with its optimizer as one CUDA graph: replays equal eager calls bit for bit, on another stream than the tensors were made on."""
    results = []
    for captured in (False, True):
        block = Block(lib, 128, 256, BF16)
        g = seeded(2)
        x, d_out = (torch.randn(200, 128, device="cuda", generator=g).to(BF16) for _ in range(2))
        counter = torch.zeros(1, device="cuda", dtype=torch.int64)
        lib.check(lib.lib().b200rl_adam_reset(block.state.data_ptr(), None))
        torch.cuda.synchronize()

        def whole():
            out, d_x = block.step(x, d_out, counter)
            block.optimize()
            lib.counter_advance(counter)
            return out, d_x

        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            if captured:
                graph = torch.cuda.CUDAGraph()
                stream.synchronize()
                with torch.cuda.graph(graph, stream=stream):
                    out, d_x = whole()
                for _ in range(3):
                    graph.replay()
            else:
                for _ in range(3):
                    out, d_x = whole()
        torch.cuda.synchronize()
        results.append((block.params.clone(), out.clone(), d_x.clone()))
    for a, b in zip(*results):
        assert torch.equal(a, b)
