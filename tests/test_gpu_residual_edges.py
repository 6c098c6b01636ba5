"""Calls of the residual operators at the edges of what their documentation allows: batches without rows, outputs that no memory holds."""
import pytest
import torch

BF16 = torch.bfloat16


def empty_batch(device):
    x = torch.zeros(0, 24, device=device, dtype=BF16)
    return x, dict(post="rms", post_weight=torch.ones(24, device=device), gate=torch.ones(1, 24, device=device, dtype=BF16), gate_rows=x.shape[0])


def test_a_batch_without_rows_is_taken_with_its_gate_per_channel(lib):
    """Through the checks of the arguments, which end with the device's."""
    x, norms = empty_batch("cpu")
    with pytest.raises(lib.B200RLError, match="CUDA tensors"):
        lib.norm_residual_forward(x, x, **norms)
    with pytest.raises(lib.B200RLError, match="CUDA tensors"):
        lib.norm_residual_backward(x, None, d_out=x, **norms)
    with pytest.raises(lib.B200RLError, match="gate is a"):
        lib.norm_residual_forward(x, x, **{**norms, "gate": torch.ones(1, 23, dtype=BF16)})


@pytest.mark.gpu
def test_gradients_of_a_batch_without_rows(lib):
    x, norms = empty_batch("cuda")
    out, normed = lib.norm_residual_forward(x, x, **norms, pre="layer")
    assert out.shape == normed.shape == (0, 24)
    g = lib.norm_residual_backward(x, out, d_out=x, d_normed=x, **norms, pre="layer")
    assert g["d_branch"].shape == g["d_residual"].shape == (0, 24) and g["d_gate"].shape == (1, 24) and not g["d_gate"].any() and not g["d_post_weight"].any()
    given, weight = torch.full((1, 24), 5.0, device="cuda", dtype=BF16), torch.full((24,), 5.0, device="cuda")
    lib.norm_residual_backward(x, out, d_out=x, d_normed=x, **norms, pre="layer", d_gate=given, d_post_weight=weight)
    assert not given.any() and (weight == 5).all()                  # a gate's gradient is overwritten, a parameter's accumulated onto


@pytest.mark.gpu
def test_outputs_that_no_memory_holds_raise_what_torch_raises(lib):
    """320 GB of outputs from operands of 0.8 MB: refused by the allocator, as the error that programs catch to take a smaller batch."""
    x = torch.zeros(400000, 1, device="cuda", dtype=BF16)
    with pytest.raises(torch.OutOfMemoryError):
        lib.dense_residual_forward(x, x, "identity")
    assert lib.dense_residual_forward(x[:5], x[:40], "identity")[1].shape == (40, 5)
