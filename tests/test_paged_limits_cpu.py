"""The paged cache's calls at the ends of what they take, as far as the CPU can check them."""
import ctypes
import os
import random
import subprocess

import pytest

import test_paged_cpu as base

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("paged") / "paged_limits_check.so")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-fsanitize=undefined", "-fno-sanitize-recover",
                    "-I", os.path.join(ROOT, "qwen3-27b-thor-runner_b200", "csrc"), "-o", out,
                    os.path.join(ROOT, "tests", "cpp", "paged_limits_check.cpp")], check=True)
    return ctypes.CDLL(out)


def test_what_is_cut_off_is_noticed(lib):
    """Rows outside [0, tokens] and lengths behind the table, by the definition: for 10 rows and a table of 32 positions."""
    rng = random.Random(5)
    wild = [-2147483648, -5, 0, 3, 9, 10, 11, 500, 2147483647]
    seen = [0, 0]
    for _ in range(2000):
        cu, kv = sorted(rng.choice(wild) for _ in range(4)), [rng.choice(wild + [31, 32, 33]) for _ in range(3)]
        if rng.random() < 0.2:
            rng.shuffle(cu)
        c, b = base.arrays(kv, [[0, 1]] * 3, cu=cu, tokens=10, page_size=16)
        for s in range(3):
            rows_out = cu[s] < 0 or cu[s + 1] > 10 or cu[s + 1] < cu[s]
            want = rows_out or (cu[s + 1] > cu[s] and kv[s] > 32)
            assert lib.paged_cut_off(ctypes.byref(c), ctypes.byref(b), s) == want, (cu, kv, s)
            seen[want] += 1
    assert min(seen) > 200
    c, b = base.arrays([32, 33, 0, -1], [[0, 1]] * 4, page_size=16)            # a token a sequence
    assert [lib.paged_cut_off(ctypes.byref(c), ctypes.byref(b), s) for s in range(4)] == [0, 1, 0, 0]
