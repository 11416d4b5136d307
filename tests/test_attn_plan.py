"""What every block of the attention takes (streamoe_amd/csrc/attn_plan.h), run on
the host against the definition: all waves of a block have the same parts in
whatever order they run, the parts of all blocks are every group's units once,
and the join looks for them in the blocks that had them."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("plan") / "attn_plan_check")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wno-unknown-pragmas", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-o", exe,
                    os.path.join(HERE, "native", "attn_plan_check.cpp")], check=True)
    return exe


@pytest.mark.parametrize("seed", range(3))
def test_every_unit_has_one_block_and_waves_agree(program, seed):
    r = subprocess.run([program, str(seed)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


def test_a_unit_s_block_and_a_block_s_units_agree(program):
    """Totals up to the most that a call can have, past 32 bits."""
    r = subprocess.run([program, "blocks"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
