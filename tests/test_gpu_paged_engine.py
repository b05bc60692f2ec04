"""Engines with the KV cache in pages: the same tokens and logits as the contiguous cache, forked slots that
share their prompt's pages, and verification steps over drafted tokens."""
import os

import numpy as np
import pytest

from conftest import golden_model

pytestmark = pytest.mark.gpu


def _engine(path, **kw):
    from laicompute_b200.engine import Engine
    return Engine(path, **kw)


def _model(tmp_path, name, **kw):
    from laicompute_b200 import gguf, synth
    a = synth.tiny_arch(gguf.Q8_0, gguf.F16, name=name, **kw)
    return a, synth.write_model(os.path.join(str(tmp_path), name + ".gguf"), a, seed=5)


def _close(a, b):
    """Both caches are FP16 and both attentions FP32-accurate; the engine's tests allow 1e-4 between such runs."""
    err = np.abs(a - b).max(axis=-1) / np.abs(b).max(axis=-1)
    assert err.max() <= 1e-4, err


@pytest.mark.parametrize("name", ["tiny_f16", "tiny_q8", "tiny_q4"])
@pytest.mark.parametrize("batched", [False, True])
def test_paged_equals_contiguous(name, batched):
    path = golden_model(name)
    rng = np.random.default_rng(1)
    e, p = _engine(path), _engine(path, paged=True)
    prompt = rng.integers(0, e.vocab, size=70).astype(np.uint32)
    a = e.generate(prompt, 20, want_logits=True, batched_prefill=batched)
    b = p.generate(prompt, 20, want_logits=True, batched_prefill=batched)
    assert np.array_equal(a[0], b[0])
    _close(b[1], a[1])
    assert p.slot_pos(0) == e.slot_pos(0)


@pytest.mark.parametrize("nseq,hidden,heads,kv_heads", [(1, 512, 4, 1), (5, 256, 4, 2), (24, 256, 8, 8), (40, 512, 4, 2)])
def test_paged_batches(tmp_path, nseq, hidden, heads, kv_heads):
    """Head dims 32 to 128, ragged prompts, batches on every projection kernel; the chained decode loop."""
    a, path = _model(tmp_path, f"paged{nseq}", hidden=hidden, layers=2, heads=heads, kv_heads=kv_heads, ffn=256, vocab=512,
                     ctx=512)
    rng = np.random.default_rng(nseq)
    lens = rng.integers(1, 300, size=nseq)
    prompts = [rng.integers(0, 512, size=n).astype(np.uint32) for n in lens]
    got = []
    for paged in (False, True):
        e = _engine(path, max_seqs=nseq, paged=paged)
        for s, p in enumerate(prompts):
            e.prefill_batch(p, s)
        tok = np.arange(nseq, dtype=np.uint32)
        steps = []
        for _ in range(3):
            tok, lg = e.step(tok, want_logits=True)
            steps.append((tok.copy(), lg))
        ids, _ = e.decode(tok, steps=70)  # crosses page ends
        got.append((steps, ids))
        e.close()
    for (ta, la), (tb, lb) in zip(got[0][0], got[1][0]):
        assert np.array_equal(ta, tb)
        _close(lb, la)
    assert np.array_equal(got[0][1], got[1][1])


def test_forked_slots(tmp_path):
    """Slots forked from one prompt at a page's end and inside a page, among slots of their own; each equals the
    same tokens run alone; a reset slot and its source go on undisturbed."""
    a, path = _model(tmp_path, "fork", hidden=512, layers=2, heads=8, kv_heads=2, ffn=256, vocab=512, ctx=1024)
    rng = np.random.default_rng(3)
    for plen in (128, 301, 40):
        prompt = rng.integers(0, 512, size=plen).astype(np.uint32)
        other = rng.integers(0, 512, size=55).astype(np.uint32)
        e = _engine(path, max_seqs=6, paged=True)
        e.prefill_batch(prompt, 0)
        for s in (2, 3, 5):
            e.fork(0, s)
            assert e.slot_pos(s) == plen
        e.prefill_batch(other, 1)
        e.prefill_batch(other[:7], 4)
        order = [0, 2, 3, 5, 1, 4]
        feed = rng.integers(0, 512, size=(6, 6)).astype(np.uint32)
        logits = []
        for t in range(6):
            _, lg = e.step(feed[t], order, want_logits=True)
            logits.append(lg)
        for i, slot in enumerate(order):
            r = _engine(path)
            r.prefill_batch({1: other, 4: other[:7]}.get(slot, prompt), 0)
            for t in range(6):
                _, lg = r.step([feed[t, i]], want_logits=True)
                _close(logits[t][i:i + 1], lg)
            r.close()
        e.reset_slot(2)   # shared pages stay with the others
        e.fork(3, 2)      # and a fork of a fork
        e.reset_slot(0)
        e.prefill_batch(other, 0)
        _, lg = e.step([9, 9, 9], [2, 3, 0], want_logits=True)
        _close(lg[:1], lg[1:2])
        r = _engine(path)
        r.prefill_batch(other, 0)
        _, ref = r.step([9], want_logits=True)
        _close(lg[2:], ref)
        r.close()
        e.close()


def test_verify_greedy(tmp_path):
    """Drafts that are right, wrong at some token, absent; the tokens and positions are those of plain steps."""
    a, path = _model(tmp_path, "verify", hidden=256, layers=2, heads=4, kv_heads=2, ffn=256, vocab=512, ctx=512)
    rng = np.random.default_rng(7)
    nseq, steps, m = 4, 30, 5
    prompts = rng.integers(0, 512, size=(nseq, 90)).astype(np.uint32)
    e = _engine(path, max_seqs=nseq)
    for s in range(nseq):
        e.prefill_batch(prompts[s, :-1], s)
    tok, want = prompts[:, -1].copy(), []
    for _ in range(steps + m + 1):
        tok, _ = e.step(tok)
        want.append(tok.copy())
    want = np.stack(want, axis=1)
    p = _engine(path, max_seqs=nseq, paged=True)
    for s in range(nseq):
        p.prefill_batch(prompts[s, :-1], s)
    tok, have = prompts[:, -1].copy(), [[] for _ in range(nseq)]
    while min(map(len, have)) < steps:
        t = np.zeros((nseq, m + 1), dtype=np.uint32)
        nd = rng.integers(0, m + 1, size=nseq)
        right = []
        for i in range(nseq):
            k = len(have[i])
            t[i, 0] = tok[i]
            draft = want[i, k:k + nd[i]].copy() if k + m < want.shape[1] else np.zeros(0, np.uint32)
            nd[i] = len(draft)
            bad = int(rng.integers(0, m + 3))
            if bad < nd[i]:
                draft[bad] = (draft[bad] + 1) % 512
            right.append(min(bad, nd[i]))
            t[i, 1:1 + nd[i]] = draft
        ids, cnt = p.verify(t, nd)
        for i in range(nseq):
            assert cnt[i] == right[i] + 1
            assert np.all(ids[i, cnt[i]:] == 0xFFFFFFFF)
            have[i] += ids[i, :cnt[i]].tolist()
            tok[i] = ids[i, cnt[i] - 1]
            assert p.slot_pos(i) == 89 + len(have[i])
    for i in range(nseq):
        assert have[i][:steps] == want[i, :steps].tolist()


def test_verify_leaves_the_history_as_steps_do():
    """The repeat penalty after verified tokens equals that after plain steps (refused drafts are forgotten)."""
    from laicompute_b200.engine import sample_params
    path = golden_model("tiny_q8")
    prompt = np.array([3, 50, 120, 7], dtype=np.uint32)
    e, p = _engine(path, paged=True), _engine(path, paged=True)
    e.prefill_batch(prompt[:-1])
    p.prefill_batch(prompt[:-1])
    t1, _ = e.step([prompt[-1]])
    t2, _ = e.step(t1)
    ids, cnt = p.verify([[prompt[-1], t1[0], (t2[0] + 1) % e.vocab, 11]], [3])
    assert cnt[0] == 2 and ids[0, 1] == t2[0]
    sp = sample_params(repeat_penalty=1.7)
    _, la = e.step(t2, params=sp, want_logits=True)
    a, b = t2, ids[0, 1:2]
    outs = []
    for eng, tok in ((e, a), (p, b)):
        if eng is p:
            tok, _ = eng.step(tok, params=sp)
        else:
            tok = np.array([int(la[0].argmax())], dtype=np.uint32)
            eng.reset_slot(0)
            eng.prefill_batch(np.concatenate([prompt, t1]))
            tok, _ = eng.step(t2, params=sp)
        seq = []
        for _ in range(12):
            tok, _ = eng.step(tok, params=sp)
            seq.append(int(tok[0]))
        outs.append(seq)
    assert outs[0] == outs[1]


class _Mt64:
    """std::mt19937_64 (its published recurrence)."""

    def __init__(self, seed):
        M = (1 << 64) - 1
        self.s, self.i = [seed & M], 312
        for i in range(1, 312):
            x = self.s[-1] ^ (self.s[-1] >> 62)
            self.s.append((6364136223846793005 * x + i) & M)

    def __call__(self):
        if self.i == 312:
            for i in range(312):
                x = (self.s[i] & 0xFFFFFFFF80000000) | (self.s[(i + 1) % 312] & 0x7FFFFFFF)
                self.s[i] = self.s[(i + 156) % 312] ^ (x >> 1) ^ (0xB5026F5AA96619E9 if x & 1 else 0)
            self.i = 0
        x = self.s[self.i]
        self.i += 1
        x ^= (x >> 29) & 0x5555555555555555
        x ^= (x << 17) & 0x71D67FFFEDA60000
        x ^= (x << 37) & 0xFFF7EEE000000000
        return x ^ (x >> 43)


def test_verify_sampled_follows_its_rule(tmp_path):
    """temperature > 0: the decisions and the drawn token from the target's logits and the seed's numbers."""
    from laicompute_b200.engine import sample_params
    a, path = _model(tmp_path, "vsample", hidden=256, layers=2, heads=4, kv_heads=2, ffn=256, vocab=512, ctx=256)
    rng = np.random.default_rng(2)
    prompt = rng.integers(0, 512, size=20).astype(np.uint32)
    m, checked, refused = 3, 0, 0
    for T, seed in [(t, s) for t in (0.05, 0.15, 0.4) for s in range(1, 21)]:
        e = _engine(path, paged=True)
        e.prefill_batch(prompt[:-1])
        toks, rows = [int(prompt[-1])], []
        for j in range(m + 1):  # the target's logits after each drafted prefix (greedy drafts)
            _, lg = e.step([toks[-1]], want_logits=True)
            rows.append(lg[0].astype(np.float64))
            toks.append(int(lg[0].argmax()))
        e.reset_slot(0)
        e.prefill_batch(prompt[:-1])
        ids, cnt = e.verify([toks[:m + 1]], [m], params=sample_params(temperature=T, seed=seed))
        g = _Mt64(seed)
        u = [(g() >> 40) * 2.0 ** -24 for _ in range(m + 1)]
        ps = [np.exp((r - r.max()) / np.float32(T)) for r in rows]
        ps = [q / q.sum() for q in ps]
        j = 0
        # logits to 1e-4 of their maximum: weights to 2e-4 max / T, sums of them and their ratios to twice that;
        # a decision closer to its border is left out
        near, eps = False, 4e-4 * max(np.abs(r).max() for r in rows) / T
        while j < m and not near:
            p = ps[j][toks[j + 1]]
            near = abs(p - u[j]) < eps
            if not u[j] < p:
                break
            j += 1
        w = ps[j].copy()
        if j < m:
            w[toks[j + 1]] = 0
        c = np.cumsum(w) / w.sum()
        near = near or np.abs(c - u[m]).min() < eps
        e.close()
        if near:
            continue
        checked += 1
        refused += j < m
        assert cnt[0] == j + 1 and ids[0, :j].tolist() == toks[1:j + 1]
        assert ids[0, j] == int(np.searchsorted(c, u[m], side="right")), seed
    assert checked >= 20 and refused >= 1, (checked, refused)


def test_paged_refusals(tmp_path):
    from laicompute_b200._native import LAIC_E_CONTEXT, LAIC_E_INVALID, LAIC_E_UNSUPPORTED, LaicError
    from laicompute_b200.engine import sample_params
    path = golden_model("tiny_q8")

    def refused(code, text, f):
        with pytest.raises(LaicError) as ex:
            f()
        assert ex.value.code == code and text in str(ex.value), str(ex.value)
    e = _engine(path, max_seqs=2)
    refused(LAIC_E_UNSUPPORTED, "paged cache", lambda: e.fork(0, 1))
    refused(LAIC_E_UNSUPPORTED, "paged cache", lambda: e.verify([[1, 2]], [1]))
    refused(LAIC_E_UNSUPPORTED, "FP16 KV", lambda: _engine(path, paged=True, kv_f32=True))
    p = _engine(path, max_seqs=2, paged=True, kv_capacity=70)
    refused(LAIC_E_INVALID, "slot out of range", lambda: p.fork(0, 2))
    refused(LAIC_E_UNSUPPORTED, "contiguous", lambda: p.fill_kv(0, 5))
    refused(LAIC_E_INVALID, "listed twice", lambda: p.verify([[1, 2], [1, 2]], [1, 1], slots=[1, 1]))
    refused(LAIC_E_INVALID, "n_draft", lambda: p.verify([[1, 2]], [2]))
    refused(LAIC_E_INVALID, "embedding", lambda: p.verify([[1, 10 ** 6]], [1]))
    refused(LAIC_E_UNSUPPORTED, "at most 64", lambda: p.verify(np.zeros((2, 33)), [1, 1]))
    refused(LAIC_E_UNSUPPORTED, "whole vocabulary",
            lambda: p.verify([[1, 2]], [1], params=sample_params(temperature=1.0, top_k=5)))
    refused(LAIC_E_UNSUPPORTED, "repeat penalty", lambda: p.verify([[1, 2]], [1], params=sample_params(repeat_penalty=2.0)))
    p.prefill_batch(np.arange(68))
    refused(LAIC_E_CONTEXT, "context length", lambda: p.verify([[1, 2, 3]], [2]))
    ids, cnt = p.verify([[1, 2, 3]], [1])
    assert cnt[0] in (1, 2)
    p.verify([[1, 2]], [0], slots=[1])  # an empty slot, no drafts
    assert p.slot_pos(1) == 1
