"""Properties of the residual operators' sources that no run can show: which loads the compiler may move, and in front of what."""
import os
import re

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, "rl-tools_b200", "csrc")
SOURCES = ["residual.cuh", "product.cuh", "product_tc.cu", "product_rows.cu", "dense_residual.cu", "norm_residual.cu", "dropout.cu"]


def code(name):
    """A source without its comments."""
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)


@pytest.mark.parametrize("name", SOURCES)
def test_no_load_may_pass_the_wait_for_the_kernel_before(name):
    """These kernels start while the kernel before them may still write what they read (an optimizer step and the norm behind it). Their wait holds ordinary loads; a read-only load
    may be moved in front of it."""
    assert not re.findall(r"__ldg\b|__restrict__|ld\.global\.nc|ldu\b", code(name))


def test_no_register_of_a_tensor_memory_load_is_named_before_its_wait():
    """What tcgen05.ld writes is there behind tcgen05.wait::ld alone. With both in one statement no copy, spill or loop variable of the registers can lie between them."""
    assert not re.findall(r"tmem_ld_32x32|tmem_wait_ld|tcgen05\.ld", code("product_tc.cu"))


def test_every_function_of_these_sources_is_called():
    text = {name: code(name) for name in SOURCES + ["tcgen05.cuh"]}
    everything = "\n".join(text.values())
    defined = {m for name in SOURCES for m in re.findall(r"__device__ __forceinline__ [\w:<> ,]+?[ &*](\w+)\(", text[name])}
    assert len(defined) > 40
    assert [f for f in sorted(defined) if len(re.findall(rf"\b{f}\b", everything)) < 2] == []
