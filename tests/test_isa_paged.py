"""What sgpu_paged.hip relies on in its own compiled code: no packed fp32 arithmetic, its matrix products and transposing LDS
reads as written, kernel arguments by scalar loads."""
import os
import re

import pytest

from test_isa_prologue import argument_vector_loads, kernels

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def code():
    if not os.path.exists(os.path.join(ROOT, "switch-l4t-gpu_amd", "build", "sgpu_paged.co")):
        pytest.skip("code objects not built (make)")
    return kernels("sgpu_paged")


def test_no_packed_fp32(code):
    assert not [(k, t) for k, ts in code.items() for t in ts if re.match(r"v_pk_(add|mul|fma)_f32", t)]


def test_no_vector_loads_of_kernel_arguments(code):
    bad = {k: v for k, v in ((k, argument_vector_loads(t)) for k, t in code.items()) if v}
    assert not bad, bad


def test_attention_uses_the_matrix_cores(code):
    shapes = {"r16": "16x16x32", "r32": "32x32x16", "r64": "32x32x16", "r128": "32x32x16"}
    seen = 0
    for name, text in code.items():
        m = re.match(r"sgpu_tree_(r\d+)_", name)
        if m:
            products = {x.group(1) for x in (re.match(r"v_mfma_f32_(\w+)_f16", t) for t in text) if x}
            assert products == {shapes[m.group(1)]} and any(t.startswith("ds_read_b64_tr_b16") for t in text), name
            seen += 1
    assert seen == 24
