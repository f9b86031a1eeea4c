"""What the transformer block's nodes of the C++ host layer keep between passes (tests/cpp/test_block_states.cpp)."""
import os
import subprocess

import pytest

CPP = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")


def build():
    from oracle import oracle as orc
    orc.build_cpu_path()
    res = subprocess.run(["make", "-C", CPP, "test_block_states"], capture_output=True, text=True)
    assert res.returncode == 0, res.stdout + res.stderr


def test_block_states_compile_with_a_host_compiler():
    build()


@pytest.mark.gpu
def test_block_states_on_gpu():
    build()
    res = subprocess.run([os.path.join(CPP, "test_block_states")], capture_output=True, text=True, timeout=300)
    print(res.stdout, res.stderr)
    assert res.returncode == 0, res.stdout + res.stderr
