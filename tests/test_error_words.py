"""An engine's two error words: a refused index of the paged cache is never reported as a device wait, nor a wait as
an index, whichever values they share."""
import os
import re
import subprocess

import pytest

from conftest import ROOT

WAITS = {1: "bulk copy", 2: "partial-sum slot", 3: "grid barrier", 4: "peer never published", 5: "dependency counter"}
BITS = {1: "sequence index", 2: "position or length", 4: "page id", 8: "group rows", 16: "a device wait timed out"}


@pytest.fixture(scope="module")
def report(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("errors") / "errors_check")
    subprocess.run(["g++", "-std=c++17", f"-I{ROOT}/laicompute_b200/csrc",
                    os.path.join(ROOT, "tests", "host", "errors_check.cpp"), "-o", exe], check=True)

    def ask(pairs):
        return subprocess.run([exe], input="\n".join(f"{a} {b}" for a, b in pairs), text=True, capture_output=True,
                              check=True).stdout.split("\n")
    return ask


def test_every_pair_is_reported_in_its_own_words(report):
    pairs = [(w, b) for w in range(6) for b in range(32)]
    for (w, b), text in zip(pairs, report(pairs)):
        assert all((t in text) == (w == k) for k, t in WAITS.items()), (w, b, text)
        assert all((t in text) == bool(b & k) for k, t in BITS.items()), (w, b, text)
        assert (text == "") == (w == 0 and b == 0)


def test_the_paged_cache_has_a_word_of_its_own():
    """The engine's pages never take the matvec kernels' word, which holds codes."""
    src = open(os.path.join(ROOT, "laicompute_b200", "csrc", "engine.cu")).read()
    made = re.findall(r"return laic_kv_pages\{(.*?)\};", src)
    assert made and all(m.endswith("d_err + 1") for m in made) and "mvs.err" not in " ".join(made)
