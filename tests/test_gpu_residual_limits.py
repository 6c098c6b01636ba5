"""The residual operators where an absolute bound or an ordinary size sees nothing: activations in their tails, relative to their values; long batches with a remainder, by bounds that a few
lost rows exceed; the largest sizes that an entry point takes."""
import math

import pytest
import torch

from residual_reference import U32, half_step, smallest, act64, assert_within

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def every_value(dtype):
    """All finite numbers of a 16-bit type."""
    v = torch.arange(65536, device="cuda", dtype=torch.int32).to(torch.int16).view(dtype)
    return v[torch.isfinite(v)]


def gelu_error(x):
    """Relative error of Phi(-|x|) = P(t) exp(-x^2 / 2), and of the density: 1.2e-5 by the fit of P; its argument t (six roundings), that of P's six additions and products through t^6 (36
    and 12); the exponential's argument e = x^2 / 2 (a rounding of it is |e| roundings of the result) and the exponential itself, within 2 + 1.2 |e| units of 2^-23."""
    e = (x * x / 2).clamp(max=100)
    return 1.2e-5 + 60 * U32 + e * U32 + (2 + 1.2 * e) * 2 * U32


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("few_rows", [True, False])
def test_gelu_of_every_value_relative_to_its_result(lib, dtype, few_rows):
    v = every_value(dtype)
    one = torch.ones(1, 1, device="cuda", dtype=dtype)
    y = lib.dense_residual_forward(v[:, None], one, "gelu")[1][0] if few_rows else lib.dense_residual_forward(one, v[:, None], "gelu")[1][:, 0]
    x = v.double()
    want = act64("gelu", x)
    # below 2^-126 the exponential may be 0; above the type's largest number nothing is rounded to infinity, since |gelu(x)| <= |x|
    bound = (half_step(dtype) + 2 * gelu_error(x)) * want.abs() + smallest(dtype) + 2.0 ** -126 * (1 + x.abs()).clamp(max=100)
    assert_within(y, want, bound, f"gelu {dtype}")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("layout", ["rows of one element", "one row"])
def test_slope_of_gelu_of_every_value_relative_to_its_terms(lib, dtype, layout):
    v = every_value(dtype)
    pre = v[:, None].contiguous() if layout == "rows of one element" else v[:v.numel() // 8 * 8].view(1, -1)
    d = lib.dense_residual_backward_activation(pre, torch.ones_like(pre), "gelu")
    x = pre.double()
    phi, along = 0.5 * torch.erfc(-x / math.sqrt(2)), x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    along = torch.where(x.abs() > 50, 0 * along, along)
    terms = 0.5 * torch.erfc(x.abs() / math.sqrt(2)) + along.abs()
    want = phi + along
    bound = half_step(dtype) * want.abs() + 2 * gelu_error(x) * terms + 4 * U32 * (phi + along.abs()) + smallest(dtype) + 2.0 ** -126 * (1 + x.abs()).clamp(max=100)
    assert_within(d, want, bound, f"slope {dtype}")


@pytest.mark.parametrize("layout", [(0, 0), (5, 3)])
@pytest.mark.parametrize("B, I, O", [(40017, 96, 72), (16400, 72, 300), (4096 + 37, 520, 40), (1000, 30, 50), (577, 200, 260)])
def test_gradients_of_long_batches_lose_no_row(lib, B, I, O, layout):
    """Products of one sign, so that a row is a share 1 / B of every sum. A piece of 512 rows is 32 truncating additions of 16 products (and those within each: 40 steps of 2^-23 in all); the
    pieces, and the shares of the batch that several CTAs take, are added with a rounding each. A column sum is at most B / 64 additions a thread, 8 between threads and those of the shares."""
    g = torch.Generator(device="cuda").manual_seed(B)
    draw = lambda n: (torch.rand(B, n + layout[0], device="cuda", generator=g) + 0.5).to(BF16)[:, layout[1]:layout[1] + n]
    x, d = draw(I), draw(O)
    d_W, d_b, _ = lib.dense_residual_backward(x.new_zeros(O, I), x, d, want_d_in=False)
    want, want_b = d.double().t() @ x.double(), d.double().sum(0)
    pieces, blocks = -(-B // 512), -(-B // 64)
    bound, bound_b = (2 * 40 + 2 * pieces) * U32, (blocks + 8 + pieces) * U32
    assert 16 * 0.25 / (B * 2.25) > bound and 16 * 0.5 / (B * 1.5) > bound_b               # the smallest share of 16 rows shows
    assert_within(d_W, want, bound * want, "d_W")
    assert_within(d_b, want_b, bound_b * want_b, "d_bias")


@pytest.mark.parametrize("B, I, O", [(4096, 256, 200), (5003, 200, 1000), (40017, 96, 72)])
def test_weight_gradients_have_the_error_of_fp32_sums(lib, B, I, O):
    """Of products of both signs: a piece's truncations lose half a step of 2^-23 each in the mean, 40 of them of sums no larger than the piece's; what rounds is less. A single accumulator
    for 4,096 rows would lose eight times that."""
    g = torch.Generator(device="cuda").manual_seed(B + 1)
    x, d = (torch.randn(B, n, device="cuda", generator=g).to(BF16) for n in (I, O))
    d_W = lib.dense_residual_backward(x.new_zeros(O, I), x, d, want_d_in=False)[0]
    want = d.double().t() @ x.double()
    assert float((d_W.double() - want).norm() / want.norm()) < (40 + 8) * U32


def test_bias_gradient_alone_of_the_most_rows_there_can_be(lib):
    """2^31 - 1 rows, the largest batch of the entry point: a row index of 32 bits would pass its range behind the last one."""
    B = 2 ** 31 - 1
    d = torch.zeros(B, 1, device="cuda", dtype=BF16)
    rows = torch.tensor([0, 31, 32, B // 2, B - 34, B - 32, B - 1], device="cuda")
    d[rows] = 1.0
    out = torch.full((1,), 3.0, device="cuda")
    L, st = lib.lib(), torch.cuda.current_stream().cuda_stream
    assert L.b200rl_dense_residual_backward_weights(1, None, 0, d.data_ptr(), 1, None, out.data_ptr(), 1, B, 1, 1, None, 0, st) == 0
    assert out.item() == 3 + rows.numel()


@pytest.mark.parametrize("act", ["relu", "tanh", "fast_tanh", "sigmoid", "gelu", "silu"])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_an_activation_is_a_function_of_its_element_alone(lib, dtype, act):
    """Whatever stands beside a value, in its row or in the rows before and behind it, and whichever kernel takes it, the result has the same bits: a row of a batch is what it is alone."""
    v = every_value(dtype)
    v = v[:v.numel() // 8 * 8]
    n, one = v.numel(), torch.ones(1, 1, device="cuda", dtype=dtype)
    y = lib.dense_residual_forward(v[:, None], one, act)[1][0]                                # a few rows: element by element
    slope = lib.dense_residual_backward_activation(v[:, None].contiguous(), torch.ones(n, 1, device="cuda", dtype=dtype), act)[:, 0]
    assert torch.equal(lib.dense_residual_backward_activation(v[None], torch.ones(1, n, device="cuda", dtype=dtype), act)[0].nan_to_num(7.0), slope.nan_to_num(7.0))
    same = lambda a, b, what: torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) or pytest.fail(f"{what}: {int((a.nan_to_num(7.0) != b.nan_to_num(7.0)).sum())} of {n} values differ")
    g = torch.Generator(device="cuda").manual_seed(1)
    for _ in range(3):
        p = torch.randperm(n, device="cuda", generator=g)
        w = v[p]
        # rows of one element (2-byte accesses) and of 64 (16-byte accesses)
        same(lib.dense_residual_forward(one, w[:, None], act)[1][:, 0], y[p], "forward, rows of one")
        eye = torch.eye(64, device="cuda", dtype=dtype)
        finite = torch.where(w.abs() < 1e30, w, torch.zeros_like(w)) if dtype == BF16 else w  # a product with 0 would spread what overflows
        wide, keep = finite[:n // 64 * 64].view(-1, 64), (finite == w)[:n // 64 * 64]
        same(torch.where(keep, lib.dense_residual_forward(eye, wide, act)[1].reshape(-1), y[p][:keep.numel()]), y[p][:keep.numel()], "forward, rows of 64")
        same(lib.dense_residual_backward(one, None, torch.ones(n, 1, device="cuda", dtype=dtype), pre_in=w[:, None].contiguous(), act_in=act, want_grads=False)[2][:, 0], slope[p], "slope, rows of one")
        same(lib.dense_residual_backward(torch.ones(1, n, device="cuda", dtype=dtype), None, one, pre_in=w[None], act_in=act, want_grads=False)[2][0], slope[p], "slope, one row")
