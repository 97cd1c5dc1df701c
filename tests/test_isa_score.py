"""What sgpu_score.hip relies on in its own compiled code: the loads that go straight into LDS are written as asm
that sets m0 just before, which holds only while nothing else lives there; and no packed fp32 arithmetic."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CO = os.path.join(ROOT, "switch-l4t-gpu_amd", "build", "sgpu_score.co")
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


@pytest.fixture(scope="module")
def lines():
    if not os.path.exists(OBJDUMP):
        pytest.skip("llvm-objdump not installed")
    if not os.path.exists(CO):
        pytest.skip("code objects not built (make)")
    text = subprocess.run([OBJDUMP, "-d", "--mcpu=gfx950", CO], capture_output=True, text=True, check=True).stdout
    return [t for t in (l.split("//")[0].strip() for l in text.splitlines()) if t]


def test_m0_is_set_right_before_each_load_into_lds(lines):
    loads = 0
    for i, t in enumerate(lines):
        if re.search(r"buffer_load_dwordx4\b.*\blds\b", t):
            assert re.match(r"s_mov_b32 m0, ", lines[i - 2]) and lines[i - 1] == "s_nop 0", lines[i - 2:i + 1]
            loads += 1
        elif re.search(r"\bm0\b", t):
            assert re.match(r"s_mov_b32 m0, ", t) and re.search(r"\blds\b", lines[i + 2]), lines[i:i + 3]
        assert not re.match(r"(v_movrel|s_set_gpr_idx|s_sendmsg|ds_gws)", t), t
    assert loads > 0


def test_no_packed_fp32(lines):
    assert not [t for t in lines if re.match(r"v_pk_(add|mul|fma)_f32", t)]


def test_no_vector_loads_of_kernel_arguments(lines):
    from test_isa_prologue import argument_vector_loads, kernels

    bad = {k: v for k, v in ((k, argument_vector_loads(t)) for k, t in kernels("sgpu_score").items()) if v}
    assert not bad, bad
