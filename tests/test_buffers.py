"""Sets of device buffers where an allocation fails: nothing made is lost, and nothing missing is taken for made (an
allocator of the host's that fails at a chosen call)."""
import os
import re
import subprocess

import pytest

from conftest import ROOT


@pytest.fixture(scope="module")
def attempts(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("buffers") / "buffers_check")
    subprocess.run(["g++", "-std=c++17", f"-I{ROOT}/laicompute_b200/csrc",
                    os.path.join(ROOT, "tests", "host", "buffers_check.cpp"), "-o", exe], check=True)

    def ask(n, fail_at):
        out = subprocess.run([exe], input=f"{n} {fail_at}\n", text=True, capture_output=True, check=True).stdout
        return [tuple(map(int, x.split(":"))) for x in out.split()]
    return ask


@pytest.mark.parametrize("n", [1, 2, 3])
def test_a_failed_set_is_completed_by_the_next_call(attempts, n):
    for fail_at in range(n):
        assert attempts(n, fail_at) == [(2, fail_at, fail_at), (0, n - fail_at, n)]
    assert attempts(n, 99) == [(0, n, n)]


def test_the_engine_makes_its_late_buffers_as_sets():
    """The buffers of a first verification and of a first prompt pass: no pointer is tested for the others."""
    src = open(os.path.join(ROOT, "laicompute_b200", "csrc", "engine.cu")).read()
    assert not re.search(r"cudaMalloc\(&(?:d->)?(?:vf_|pf_)", src)
    assert not re.search(r"if \(!?(?:d->)?(?:vf|pf)_(?!ready)\w+\) (?:return LAIC_OK|\{)", src)


def test_a_growing_buffer_that_fails_is_known_to_be_gone(tmp_path):
    """(error, moved, present, capacity) of each request: after a failure the smaller request allocates again."""
    exe = str(tmp_path / "regrow_check")
    subprocess.run(["g++", "-std=c++17", f"-I{ROOT}/laicompute_b200/csrc",
                    os.path.join(ROOT, "tests", "host", "regrow_check.cpp"), "-o", exe], check=True)

    def ask(fail_at, *needs):
        out = subprocess.run([exe], input=" ".join(map(str, (fail_at, *needs))) + "\n", text=True, capture_output=True,
                             check=True).stdout
        return [tuple(map(int, x.split(":"))) for x in out.split()]
    assert ask(9, 10, 5, 10, 20) == [(0, 1, 1, 10), (0, 0, 1, 10), (0, 0, 1, 10), (0, 1, 1, 20)]
    assert ask(1, 10, 20, 5, 5) == [(0, 1, 1, 10), (2, 1, 0, 0), (0, 1, 1, 5), (0, 0, 1, 5)]
    assert ask(0, 10, 0, 10) == [(2, 1, 0, 0), (0, 0, 0, 0), (0, 1, 1, 10)]


def test_the_engine_grows_its_scratch_that_way():
    src = open(os.path.join(ROOT, "laicompute_b200", "csrc", "engine.cu")).read()
    assert not re.search(r"cudaMalloc\(&(?:sc\.(?!err)|attn_ws)", src) and src.count("laic::regrow(") == 2
