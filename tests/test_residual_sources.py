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


def test_the_norms_are_built_for_the_row_shapes_of_their_types_alone(lib):
    """The threads of a row and the elements of a thread: 16-bit rows take up to 16 elements a thread, fp32 rows 8."""
    import subprocess
    names = subprocess.run(["nm", "-C", lib.LIB_PATH], capture_output=True, text=True, check=True).stdout
    built = {}
    for kernel, of, threads, elements in re.findall(r"b200rl::norm_(forward|backward)_kernel<([\w ]+), \d+, (\d+), (\d+)", names):
        built.setdefault((kernel, of), set()).add((int(threads), int(elements)))
    narrow, wide = {(32, 8), (32, 16), (128, 8), (128, 16), (256, 16), (512, 16)}, {(32, 8), (128, 8), (256, 8), (512, 8), (1024, 8)}
    assert built == {(kernel, of): wide if of == "float" else narrow for kernel in ("forward", "backward") for of in ("float", "__half", "__nv_bfloat16")}
