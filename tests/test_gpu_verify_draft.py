"""laic_dev_verify with the probabilities of a draft model: the decisions follow the 64-bit rule, and the
probabilities are read behind the stream that writes them."""
import os

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

V = 512


def _model(tmp_path):
    from laicompute_b200 import gguf, synth
    a = synth.tiny_arch(gguf.Q8_0, gguf.F16, name="draft", hidden=256, layers=2, heads=4, kv_heads=2, ffn=256, vocab=V,
                        ctx=256)
    return synth.write_model(os.path.join(str(tmp_path), "draft.gguf"), a, seed=5)


def _uniforms(seed, m):
    from test_gpu_paged_engine import _Mt64
    g = _Mt64(seed)
    return [(g() >> 40) * 2.0 ** -24 for _ in range(m + 1)]


def _soft(x):
    e = np.exp(x - x.max(axis=-1, keepdims=True))
    return e / e.sum(axis=-1, keepdims=True)


@pytest.mark.parametrize("nseq,m,stream", [(3, 5, "legacy"), (8, 7, "own"), (1, 63, "own"), (64, 0, "legacy")])
def test_verify_with_draft_probabilities(tmp_path, nseq, m, stream):
    """Ragged drafts drawn from a noisy copy of the target's rows, up to 64 rows a step. The buffer holds other
    probabilities until the writing stream, which is busy, gets to the right ones."""
    import torch
    from laicompute_b200.engine import Engine, sample_params
    path = _model(tmp_path)
    rng = np.random.default_rng(nseq)
    prompts = rng.integers(0, V, size=(nseq, 20)).astype(np.uint32)
    e = Engine(path, max_seqs=nseq, paged=True)
    side = torch.cuda.Stream()
    drawn = refused = 0  # decisions that no error of the logits could have turned
    for rnd in range(6):
        T = (0.1, 0.15, 0.2)[rnd % 3]
        nd = rng.integers(0, m + 1, size=nseq)
        nd[0] = m

        def fresh():
            for s in range(nseq):
                e.reset_slot(s)
                e.prefill_batch(prompts[s, :-1], s)
        fresh()
        # the target's rows after each drafted prefix; the drafted tokens drawn from the draft's rows
        toks, rows, q = [prompts[:, -1].copy()], [], np.zeros((nseq, m, V), np.float32)
        for j in range(m + 1):
            _, lg = e.step(toks[-1], want_logits=True)
            rows.append(lg.astype(np.float64))
            if j < m:
                q[:, j] = _soft(rows[j] / np.float32(T) + 0.7 * rng.standard_normal((nseq, V)))
                c = np.cumsum(q[:, j].astype(np.float64), axis=1)
                u = rng.random((nseq, 1)) * c[:, -1:]
                toks.append(np.minimum((c <= u).sum(axis=1), V - 1).astype(np.uint32))
        fresh()
        right = torch.from_numpy(q).cuda()
        buf = torch.zeros(max(1, q.size), device="cuda")  # (nothing drafted could be drawn from these)
        torch.cuda.synchronize()
        with torch.cuda.stream(side if stream == "own" else torch.cuda.default_stream()):
            torch.cuda._sleep(100_000_000)  # 50 ms: longer than the step
            buf[:q.size].copy_(right.flatten())
            at = torch.cuda.current_stream().cuda_stream
        seeds = [int(x) for x in rng.integers(1, 1 << 30, size=nseq)]
        ids, cnt = e.verify(np.stack(toks, axis=1), nd, params=[sample_params(temperature=T, seed=x) for x in seeds],
                            draft_probs=buf.data_ptr(), stream=at)
        for i in range(nseq):
            u = _uniforms(seeds[i], m)
            p = [_soft(r[i] / np.float32(T)) for r in rows]
            # logits to 1e-4 of their maximum: weights to twice that over T, sums of them and their ratios to twice
            # that again; so far the borders may have moved
            eps = 4e-4 * max(np.abs(r[i]).max() for r in rows) / T
            acc = int(cnt[i]) - 1
            assert 0 <= acc <= nd[i] and ids[i, :acc].tolist() == [int(t[i]) for t in toks[1:acc + 1]], (rnd, i)
            for j in range(acc):
                x = int(toks[j + 1][i])
                assert u[j] * float(q[i, j, x]) < p[j][x] + eps, (rnd, i, j)
            if acc < nd[i]:
                x = int(toks[acc + 1][i])
                margin = u[acc] * float(q[i, acc, x]) - p[acc][x]
                assert margin > -eps, (rnd, i)
                refused += margin > eps  # (the buffer's first contents would have been accepted)
            w = np.maximum(p[acc] - q[i, acc].astype(np.float64), 0) if acc < nd[i] else p[acc]
            c = np.cumsum(w) / w.sum()
            off, t = 2 * eps / w.sum(), int(ids[i, acc])
            assert c[t] + off > u[m] and (t == 0 or c[t - 1] - off <= u[m]), (rnd, i)
            drawn += np.abs(c - u[m]).min() > off  # (one token alone was right)
            assert e.slot_pos(i) == 19 + acc + 1
    e.close()
    assert drawn >= 1 and (refused >= 1 or m == 0), (drawn, refused)


def test_wait_stream_refusals():
    import torch
    from conftest import golden_model
    from laicompute_b200._native import LAIC_E_INVALID, LaicError
    from laicompute_b200.engine import Engine
    e = Engine(golden_model("tiny_q8"))
    e.wait_stream(0)
    x = torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, capture_error_mode="thread_local"):
        x += 1
        with pytest.raises(LaicError) as ex:
            e.wait_stream(torch.cuda.current_stream().cuda_stream)
    assert ex.value.code == LAIC_E_INVALID and "captured" in str(ex.value)
    g.replay()
    torch.cuda.synchronize()
    assert torch.all(x == 1)
    ids, _ = e.step([3])
    assert 0 <= int(ids[0]) < e.vocab
