"""Memory that the library clears or fills on the host's behalf is ready before its own streams use it, also
while the legacy default stream is busy with a caller's work (for which those streams do not wait)."""
import numpy as np
import pytest

from conftest import golden_model

pytestmark = pytest.mark.gpu

BUSY = 200_000_000  # SM clocks, 0.1 s or more: longer than any call here takes


def _legacy_busy():
    import torch
    torch.cuda._sleep(BUSY)  # (torch's default stream is the legacy one)


@pytest.mark.parametrize("ggml", ["F16", "Q8_0", "Q4_0"])
def test_matrix_made_while_the_legacy_stream_is_busy(ggml):
    import torch
    from laicompute_b200 import gguf, synth
    from laicompute_b200.engine import Matrix
    t, n, k = getattr(gguf, ggml), 272, 512
    w = (np.random.default_rng(3).standard_normal(n * k, dtype=np.float32) * np.float32(0.02)).astype(np.float32)
    raw = np.frombuffer(synth.encode(w, t), dtype=np.uint8)
    x = torch.randn(2, k, device="cuda")
    want, got = torch.zeros(2, n, device="cuda"), torch.zeros(2, n, device="cuda")
    torch.cuda.synchronize()
    Matrix(t, k, n, raw).matvec(x.data_ptr(), want.data_ptr(), 2)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    _legacy_busy()
    m = Matrix(t, k, n, raw)
    _legacy_busy()
    m.matvec(x.data_ptr(), got.data_ptr(), 2, stream=s.cuda_stream)  # (the first call makes its working memory)
    torch.cuda.synchronize()
    assert want.abs().max() > 0 and torch.equal(got, want)


@pytest.mark.parametrize("paged", [False, True])
def test_engine_and_slots_while_the_legacy_stream_is_busy(paged):
    """A new engine, and a slot reset and used at once: positions and history start from nothing."""
    import torch
    from laicompute_b200.engine import Engine, sample_params
    torch.zeros(1, device="cuda")
    path, sp = golden_model("tiny_q8"), sample_params(repeat_penalty=1.5)
    first, second = np.array([5, 77, 131, 250, 19], np.uint32), np.array([9, 30, 2], np.uint32)

    def run(e, prompt):
        e.reset_slot(0)
        e.prefill_batch(prompt, 0)
        tok, out = [int(prompt[-1])], []
        for _ in range(6):
            tok, lg = e.step(tok, params=sp, want_logits=True)
            out.append(lg)
        return np.stack(out)
    quiet = Engine(path, paged=paged)
    want = run(quiet, first), run(quiet, second)
    _legacy_busy()
    e = Engine(path, paged=paged)
    got = []
    for prompt in (first, second):
        torch.cuda.synchronize()
        _legacy_busy()
        got.append(run(e, prompt))
    torch.cuda.synchronize()
    for a, b in zip(want, got):  # (as the engine's other tests allow between two runs)
        assert (np.abs(a - b).max(axis=-1) / np.abs(a).max(axis=-1)).max() <= 1e-4
