"""Attention over the pages where what a row does see is not finite: scores that are NaN or infinite."""
import pytest
import torch

from serving_util import F16, F32, TORCH, Cache, attend, close, reference

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


def _q(rows, heads, d, dtype, seed):
    return (torch.randn(rows, heads * d, generator=torch.Generator().manual_seed(seed)) * 1.5).to(TORCH[dtype]).cuda()


def _put(cache, what, seqs, pos, value, dim=slice(None)):
    """k or v of a position of these sequences, in the pages and in the reference's copies."""
    for s in seqs:
        getattr(cache, what)[cache.rows[s][pos // cache.page], :, pos % cache.page, dim] = value
        getattr(cache, "seq_" + what)[s][pos, :, dim] = value


def _shape(kind, heads, hkv, d, seed=1):
    """(cache, lens, seqs, groups): rows of their own (one CTA; split), a narrow group, a wide one."""
    if kind in ("whole", "split"):
        n = {"whole": 90, "split": 1500}[kind]
        return Cache([n] * 3, hkv, d, 16, seed=seed), [n] * 3, None, None
    rows = {"narrow": 3, "wide": 24}[kind]
    n = 300
    cache = Cache([n + 5] * rows, hkv, d, 32, seed=seed, shared=[(list(range(rows)), n)])
    return cache, [n + 5] * rows, None, ([0, rows], [n])


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("heads,hkv,d", [(8, 2, 64), (4, 2, 32), (8, 1, 128)])
@pytest.mark.parametrize("kind", ["whole", "split", "narrow", "wide"])
def test_nan_scores_reach_their_rows_alone(kind, heads, hkv, d, dtype):
    """A query head that is NaN, or infinite: every score is NaN or infinite, and so the head's output is NaN; the
    other heads and rows are right."""
    cache, lens, seqs, groups = _shape(kind, heads, hkv, d)
    q = _q(len(lens), heads, d, dtype, seed=3)
    ref, tol = reference(cache, q[:3], lens[:3])
    q[0, 2 * d + 5] = NAN           # row 0, head 2
    q[2, 0] = INF                   # row 2, head 0: scores of both signs
    out = attend(cache, q, lens, groups=groups)
    cache.pages().check()
    bad = torch.zeros(len(lens), heads, d, dtype=torch.bool)
    bad[0, 2] = bad[2, 0] = True
    bad = bad.flatten(1)
    assert torch.isnan(out.cpu()[bad]).all()
    good = ~bad[:3]
    close(out[:3][good.cuda()], ref[good], tol[good])
    assert torch.isfinite(out.cpu()[~bad]).all()


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("n", [1, 17])
def test_a_row_that_sees_only_nan_keys(n, dtype):
    cache = Cache([n, 40], 1, 64, 16, seed=2)
    q = _q(2, 4, 64, dtype, seed=1)
    ref, tol = reference(cache, q, [n, 40])
    for t in range(n):
        _put(cache, "k", [0], t, NAN, 3)
    out = attend(cache, q, [n, 40])
    assert torch.isnan(out[0]).all()
    close(out[1:], ref[1:], tol[1:])
