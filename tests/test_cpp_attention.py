"""The attention operators of the C++ interface: the compiled program
tests/cpp/test_attention_cpp (tests/cpp/Makefile). On the CPU its argument
errors; on a GPU the operators against their definitions in double."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BINARY = os.path.join(ROOT, "tests", "cpp", "_build", "test_attention_cpp")


def _run(args, timeout):
    p = subprocess.run([BINARY, *args], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=timeout)
    print(p.stdout, flush=True)
    assert p.returncode == 0 and "all passed" in p.stdout, p.stdout[-2000:]


def test_errors_on_the_host():
    if not os.path.exists(BINARY):
        import oracle as orc
        from t2h import _build

        if not os.path.exists(_build.LIB_PATH):
            _build.build()
        orc.build()
        subprocess.run(["make", "-C", os.path.join(ROOT, "tests", "cpp")], check=True, stdout=subprocess.PIPE,
                       stderr=subprocess.STDOUT)
    _run(["--host"], 60)


@pytest.mark.gpu
def test_operators(dev):
    if not os.path.exists(BINARY):
        pytest.fail(f"{BINARY} is not built: run __graft_entry__.build() (make -C tests/cpp)")
    _run([], 100)
