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


def _close_nonfinite(out, ref, tol):
    """Finite elements within their bound; the others are the definition's infinities and NaN."""
    out = out.double().cpu()
    odd = ~torch.isfinite(ref)
    assert odd.any()
    same = (out[odd] == ref[odd]) | (torch.isnan(out[odd]) & torch.isnan(ref[odd]))
    assert same.all(), (out[odd][~same][:8], ref[odd][~same][:8])
    close(out[~odd], ref[~odd], tol[~odd])


@pytest.mark.parametrize("scale", [0.0, 2.0])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("heads,hkv,d", [(8, 2, 64), (4, 2, 32), (8, 1, 128), (6, 1, 64)])
@pytest.mark.parametrize("kind", ["whole", "split", "narrow", "wide"])
def test_seen_values_that_are_not_finite(kind, heads, hkv, d, dtype, scale):
    """Infinities and NaN in values that every row sees, in the first and last tiles and in the row's own positions,
    of each sign and both, at weights down to e^-200 of the sum (beyond binary32 and binary16)."""
    cache, lens, seqs, groups = _shape(kind, heads, hkv, d, seed=4)
    n, all_ = lens[0], range(len(lens))
    for pos, dim, value in ((3, 1, INF), (n - 40, 2, -INF), (50, 3, INF), (60, 3, -INF), (70, 4, NAN), (n - 30, 5, INF),
                            (n - 29, 5, INF), (0, 6, -INF)):
        _put(cache, "v", all_, pos, value, dim)
    _put(cache, "v", [1], n - 1, INF, 7)   # (one row alone)
    q = _q(len(lens), heads, d, dtype, seed=6)
    out = attend(cache, q, lens, groups=groups, scale=scale)
    cache.pages().check()
    ref, tol = reference(cache, q[:3], lens[:3], scale=scale)
    _close_nonfinite(out[:3], ref, tol)


@pytest.mark.parametrize("scale", [0.0, 2.0])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("heads,hkv,d,rows,start", [(4, 2, 64, 30, 150), (32, 8, 128, 12, 150), (2, 2, 32, 9, 150),
                                                    (8, 1, 128, 40, 300), (4, 1, 64, 80, 490)])
def test_values_that_some_rows_see(heads, hkv, d, rows, start, dtype, scale):
    """Causal rows: infinite values seen by all, by the last rows only, and by none but the last."""
    total = start + rows
    cache = Cache([total], hkv, d, 16, seed=2)
    lens = [start + j + 1 for j in range(rows)]
    for pos, dim, value in ((5, 0, INF), (start - 1, 1, -INF), (total - 4, 2, INF), (total - 3, 2, -INF), (total - 5, 3, NAN),
                            (total - 1, 4, INF), (start + 1, 5, -INF)):
        _put(cache, "v", [0], pos, value, dim)
    q = _q(rows, heads, d, dtype, seed=4)
    out = attend(cache, q, lens, seqs=[0] * rows, groups=([0, rows], [total]), scale=scale)
    cache.pages().check()
    at = sorted({0, 1, 2, rows // 2, rows - 6, rows - 5, rows - 4, rows - 3, rows - 2, rows - 1})
    ref, tol = reference(cache, q[at], [lens[r] for r in at], [0] * len(at), scale=scale)
    _close_nonfinite(out[at], ref, tol)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("heads,hkv,d", [(8, 2, 64), (4, 2, 32), (8, 1, 128)])
@pytest.mark.parametrize("kind", ["whole", "split", "narrow", "wide"])
def test_scores_of_minus_infinity(kind, heads, hkv, d, dtype):
    """Infinite keys whose scores are -inf at the head of the positions, with all other scores far below zero: they
    weigh nothing. Where every score is -inf, zeros."""
    cache, lens, seqs, groups = _shape(kind, heads, hkv, d, seed=7)
    n = lens[0]
    q = _q(len(lens), heads, d, dtype, seed=8).view(len(lens), heads, d)
    # q[0] k[0] = -inf with both parts of the split q of one sign, q[1] k[1] = -500 / scale
    q[:, :, 0], q[:, :, 1] = (1.0 + 2.0 ** -13 if dtype == F32 else 1.0), 1.0
    q = q.flatten(1).contiguous()

    class Rest:  # the positions behind the infinite keys
        head_dim, kv_heads = d, hkv
    for s in range(len(lens)):
        for t in range(n):
            _put(cache, "k", [s], t, -1000.0, 1)
    for first in (64, 70, 200 if n > 200 else 80):
        for t in range(first):
            _put(cache, "k", range(len(lens)), t, -INF, 0)
        Rest.seq_k = [k[first:] for k in cache.seq_k]
        Rest.seq_v = [v[first:] for v in cache.seq_v]
        out = attend(cache, q, lens, groups=groups, scale=0.5)
        cache.pages().check()
        ref, tol = reference(Rest, q[:3], [m - first for m in lens[:3]], scale=0.5)
        close(out[:3], ref, tol)
    for t in range(n):
        _put(cache, "k", range(len(lens)), t, -INF, 0)
    out = attend(cache, q, lens, groups=groups, scale=0.5)
    assert not out.any()
    if groups:  # and where a group's rows see the shared positions alone
        out = attend(cache, q, [groups[1][0]] * len(lens), groups=groups, scale=0.5)
        assert not out.any()
