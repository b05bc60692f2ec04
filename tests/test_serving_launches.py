"""How the serving operators launch: early behind their predecessor or not, as asked, and counted (recorded by
stand-ins for the runtime, no GPU); and the paged engine, which passes its flag on and reports the count."""
import os
import re
import subprocess

import numpy as np
import pytest

from conftest import ROOT, golden_model


@pytest.fixture(scope="module")
def launches(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("launch") / "launch_check")
    subprocess.run(["nvcc", "-std=c++17", "-O0", "-gencode", "arch=compute_100a,code=compute_100a", f"-I{ROOT}/include",
                    f"-I{ROOT}/laicompute_b200/csrc", os.path.join(ROOT, "tests", "host", "launch_check.cu"), "-o", exe],
                   check=True, capture_output=True)

    def ask(lines):
        out = subprocess.run([exe], input="\n".join(lines) + "\n", text=True, capture_output=True, check=True).stdout
        return [tuple(map(int, x.split())) for x in out.splitlines()]
    return ask


# rows heads max_len groups max_group_rows max_shared max_private, and the kernels they take
ATTENTION = [("2 8 100 0 0 0 -1", 1), ("2 8 5000 0 0 0 -1", 2), ("4 8 3000 1 4 2000 900", 3), ("4 8 3000 1 4 2000 200", 2),
             ("40 8 3000 1 40 2000 900", 3), ("40 8 2000 1 40 2000 0", 1)]


def test_launches_follow_the_flag_and_are_counted(launches):
    ops = [("append", 1), ("probs", 1), ("verify", 1)] + [("attention " + a, n) for a, n in ATTENTION]
    got = launches([f"{op} {pdl}" for op, _ in ops for pdl in (1, 0)])
    assert got == [(n,) + (pdl,) * n for _, n in ops for pdl in (1, 0)]


def test_the_engine_passes_its_flag_to_every_operator():
    src = open(os.path.join(ROOT, "laicompute_b200", "csrc", "engine.cu")).read()
    calls = re.findall(r"laic::(?:kv_append|kv_attention|logits_probs|verify_drafts)\((.*)\)\) return rc;", src)
    assert len(calls) == 6 and all(re.search(r"\{(?:pdl, &nl|use_pdl)\}$", c) for c in calls), calls


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [True, False])
def test_paged_engine_without_early_launches(graphs):
    """The same tokens, logits and verified tokens with the flag either way."""
    from laicompute_b200.engine import Engine
    path = golden_model("tiny_q8")
    prompt = np.random.default_rng(1).integers(0, 300, size=80).astype(np.uint32)
    got = []
    for pdl in (True, False):
        e = Engine(path, max_seqs=3, paged=True, pdl=pdl, graphs=graphs)
        e.prefill_batch(prompt, 0)
        e.fork(0, 1)
        e.prefill_batch(prompt[:9], 2)
        tok, out = np.array([5, 6, 7], np.uint32), []
        for _ in range(5):
            tok, lg = e.step(tok, want_logits=True)
            out.append(lg)
        ids, cnt = e.verify(np.stack([tok, tok, tok], axis=1), [2, 0, 1])
        got.append((np.stack(out), ids, cnt))
        e.close()
    (la, ia, ca), (lb, ib, cb) = got
    assert (np.abs(la - lb).max(axis=-1) / np.abs(lb).max(axis=-1)).max() <= 1e-4
    assert np.array_equal(ia, ib) and np.array_equal(ca, cb)


@pytest.mark.gpu
def test_paged_engine_counts_its_launches(tmp_path):
    """launches_per_step: the contiguous engine's, the rows' kernel, and per layer an append, the preparation of the
    o-projection's activations (the contiguous attention of this small model writes them itself) and as many attention
    kernels as the lengths take, in the place of the contiguous engine's one."""
    from laicompute_b200 import gguf, synth
    from laicompute_b200.engine import Engine
    a = synth.tiny_arch(gguf.Q8_0, gguf.F16, name="count", hidden=256, layers=2, heads=4, kv_heads=2, ffn=256, vocab=512,
                        ctx=2048)
    path = synth.write_model(os.path.join(str(tmp_path), "count.gguf"), a, seed=5)
    rng = np.random.default_rng(0)
    for n, forked, kernels in ((20, False, 1), (1200, False, 2), (100, True, 2), (20, True, 1)):
        counts = []
        for paged in (False, True):
            e = Engine(path, max_seqs=2, paged=paged, speculate=False)
            prompts = rng.integers(0, 512, size=(2, n)).astype(np.uint32)
            e.prefill_batch(prompts[0], 0)
            if paged and forked:
                e.fork(0, 1)
            else:
                e.prefill_batch(prompts[1], 1)
            e.step([1, 2])
            counts.append(e.stats().launches_per_step)
            e.close()
        assert counts[1] - counts[0] == 1 + 2 * (1 + 1 + kernels - 1), (n, forked, counts)
