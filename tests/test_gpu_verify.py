"""Probabilities of logits rows and the verification of drafted tokens on the GPU against 64-bit forms."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

NONE = -1  # LAIC_NO_TOKEN as int32


# ------------------------------------------------------------------------------------------------
# probabilities
# ------------------------------------------------------------------------------------------------

def _probs(x, temp, ld=None, ldp=None, in_place=False):
    from laicompute_b200.serving import logits_probs
    rows, v = x.shape
    ld, ldp = ld or v, ldp or v
    src = torch.full((rows, ld), 123.0)
    src[:, :v] = x
    src = src.cuda()
    dst = src if in_place else torch.full((rows, ldp), -3.0, device="cuda")
    t = torch.tensor(temp, dtype=torch.float32, device="cuda")
    logits_probs(rows, v, src.data_ptr(), t.data_ptr(), dst.data_ptr(), ld_logits=ld, ld_probs=ld if in_place else ldp)
    torch.cuda.synchronize()
    if not in_place and ldp > v:
        assert torch.all(dst[:, v:] == -3.0)
    return dst[:, :v].cpu()


def _check_probs(p, x, temp):
    """Relative error of p = 2^E / S, E = (x - max) log2(e) / T: the exponent is one fused product and sum with a
    factor rounded once, |E| (2^-24 + 2^-24) absolute, ln 2 times that relative in 2^E (twice: S has it too, at most
    that of its terms); the exponential 2^-22 (twice), the products with the slice's scale and 1 / S 2^-22; the sum of
    v terms in at most v / 256 + 40 FP32 steps."""
    v = x.shape[1]
    rel = 2.0 ** -20 + (v / 256 + 40) * 2.0 ** -24
    for r, t in enumerate(temp):
        if t <= 0:
            want = torch.zeros(v, dtype=torch.float64)
            want[int(np.argmax(x[r].numpy()))] = 1.0
            assert torch.equal(p[r].double(), want)
        else:
            e = (x[r].double() - x[r].double().max()) / np.float64(np.float32(t))
            want = torch.softmax(e, dim=0)
            err = (p[r].double() - want).abs()
            tol = rel + e.abs() * 1.4427 * 2 * 2.0 ** -23 * 0.6932
            assert bool((err <= tol * want + 2.0 ** -126).all()), float((err / (want + 1e-300)).max())


@pytest.mark.parametrize("v", [1, 2, 3, 31, 320, 1000, 4097, 49152, 128256, 262147])
def test_probs(v):
    g = torch.Generator().manual_seed(v)
    x = torch.randn(5, v, generator=g) * 4
    temp = [1.0, 0.3, 0.0, 7.5, -1.0]
    _check_probs(_probs(x, temp), x, temp)


@pytest.mark.parametrize("ld,ldp,in_place", [(1001, 1003, False), (1004, 1000, False), (1001, 0, True), (1000, 0, True)])
def test_probs_strides_and_in_place(ld, ldp, in_place):
    g = torch.Generator().manual_seed(ld)
    x = torch.randn(7, 1000, generator=g) * 3
    temp = [1.0, 0.0, 0.5, 2.0, 0.0, 1.0, 0.7]
    _check_probs(_probs(x, temp, ld=ld, ldp=ldp, in_place=in_place), x, temp)


@pytest.mark.parametrize("v", [40, 1000, 40000, 140000])
def test_probs_extreme_temperatures(v):
    """From the smallest binary32 numbers to the largest and infinity, ordinary logits and huge ones."""
    inf = float("inf")
    x = torch.randn(8, v, generator=torch.Generator().manual_seed(v)) * 3
    x[:, 7] = 20.0                                    # one clear first
    x[1] = 0.0                                        # a constant row
    x[5] *= 1e37
    temp = [1e-45, 1e-45, 1e-30, inf, 3e38, 3e38, 1e-39, inf]
    x[7, 3] = -inf
    p = _probs(x, temp)
    uniform = torch.full((v,), 1 / v, dtype=torch.float64)
    _check_probs(p[2:3], x[2:3], [1e-30])
    _check_probs(p[5:6], x[5:6], [3e38])
    rel = 2.0 ** -20 + (v / 256 + 40) * 2.0 ** -24    # of the sum and the products, as in _check_probs
    one = torch.zeros(v, dtype=torch.float64)
    one[7] = 1.0
    assert torch.equal(p[0].double(), one) and torch.equal(p[6].double(), one)
    for r in (1, 3, 4):                               # (row 4: exponents below 1e-36)
        assert float((p[r].double() / uniform - 1).abs().max()) <= rel
    assert p[7, 3] == 0
    rest = torch.cat([p[7, :3], p[7, 4:]]).double() * (v - 1)
    assert float((rest - 1).abs().max()) <= rel


def test_probs_ties_masks_and_infinities():
    inf, nan = float("inf"), float("nan")
    lowest = torch.finfo(torch.float32).min
    x = torch.zeros(8, 700)
    x[0, [3, 500]] = 2.0                      # greedy tie: the first
    x[1] = -inf                               # nothing allowed
    x[2] = -inf
    x[2, 77] = -5.0                           # one allowed
    x[3, :] = lowest                          # all of the lowest value: uniform
    x[4, [10, 600]] = inf                     # share the row
    x[5, 5] = nan                             # a NaN cannot be chosen
    x[6] = nan
    x[7] = lowest
    x[7, 9] = 1.0
    p = _probs(x, [0.0, 1.0, 1.0, 0.5, 1.0, 1.0, 1.0, 0.8])
    assert p[0, 3] == 1 and p[0].sum() == 1
    assert not p[1].any() and p[2, 77] == 1 and p[2].sum() == 1
    assert torch.allclose(p[3], torch.full((700,), 1 / 700), rtol=1e-5)
    assert p[4, 10] == 0.5 and p[4, 600] == 0.5 and p[4].sum() == 1
    assert p[5, 5] == 0 and torch.allclose(p[5, 6], torch.tensor(1 / 699), rtol=1e-5)
    assert not p[6].any() and p[7, 9] == 1 and p[7].sum() == 1
    g = _probs(x, [0.0] * 8)
    assert not g[1].any() and g[2, 77] == 1 and g[3, 0] == 1 and g[4, 10] == 1 and g[5, 0] == 1 and not g[6].any()


# ------------------------------------------------------------------------------------------------
# verification
# ------------------------------------------------------------------------------------------------

def _verify_ref(target, draft, ids, n, au, su):
    """Plain Python doubles; target [S][M+1][V], draft [S][M][V] or None."""
    S, M = ids.shape
    V = target.shape[2]
    out = np.full((S, M + 1), NONE, np.int64)
    cnt = np.zeros(S, np.int64)
    clean = lambda a: np.where(a > 0, a, 0).astype(np.float64)  # noqa: E731
    for s in range(S):
        if n[s] < 0:
            out[s], cnt[s] = -9, -9
            continue
        m, j = min(n[s], M), 0
        while j < m:
            x = int(ids[s, j]) & 0xFFFFFFFF
            if x >= V:
                break
            p = float(clean(target[s, j])[x])
            q = float(clean(draft[s, j])[x]) if draft is not None else 1.0
            if not float(au[s, j]) * q < p:
                break
            out[s, j] = x
            j += 1
        w = clean(target[s, j])
        if j < m:
            x = int(ids[s, j]) & 0xFFFFFFFF
            if draft is not None:
                r = np.maximum(w - clean(draft[s, j]), 0)
            else:
                r = w.copy()
                if x < V:
                    r[x] = 0
            if r.sum() > 0:
                w = r
        cum = np.cumsum(w)
        t = float(su[s]) * cum[-1]
        over = np.nonzero(cum > t)[0]
        pos = np.nonzero(w > 0)[0]
        out[s, j] = over[0] if len(over) else pos[-1] if len(pos) else 0
        cnt[s] = j + 1
    return out, cnt


def _verify(target, draft, ids, n, au, su, ldt=0, ldd=0, stream=0):
    from laicompute_b200.serving import verify_drafts
    S, M = ids.shape
    V = target.shape[2]

    def rows(a, ld):
        a = torch.as_tensor(a, dtype=torch.float32).reshape(-1, V)
        if ld:
            wide = torch.full((a.shape[0], ld), 50.0)
            wide[:, :V] = a
            a = wide
        return a.contiguous().cuda()
    dev = [rows(target, ldt), rows(draft, ldd) if draft is not None else None,
           torch.as_tensor(ids.astype(np.uint32).view(np.int32)).cuda(), torch.as_tensor(n, dtype=torch.int32).cuda(),
           torch.as_tensor(au, dtype=torch.float32).cuda(), torch.as_tensor(su, dtype=torch.float32).cuda()]
    out = torch.full((S, M + 1), -9, dtype=torch.int32, device="cuda")
    cnt = torch.full((S,), -9, dtype=torch.int32, device="cuda")
    ptr = lambda t: t.data_ptr() if t is not None and t.numel() else 4096  # noqa: E731
    torch.cuda.synchronize()
    verify_drafts(S, M, V, ptr(dev[0]), ptr(dev[1]) if draft is not None else 0, ptr(dev[2]), ptr(dev[3]), ptr(dev[4]),
                  ptr(dev[5]), out.data_ptr(), cnt.data_ptr(), ld_target=ldt, ld_draft=ldd, stream=stream)
    torch.cuda.synchronize()
    return out.cpu().numpy().astype(np.int64), cnt.cpu().numpy().astype(np.int64)


def _case(S, M, V, seed, sharp=2.0, same=False):
    rng = np.random.default_rng(seed)

    def soft(a):
        e = np.exp(a - a.max(axis=-1, keepdims=True))
        return (e / e.sum(axis=-1, keepdims=True)).astype(np.float32)
    base = rng.standard_normal((S, M + 1, V)) * sharp
    target = soft(base)
    draft = target[:, :M].copy() if same else soft(base[:, :M] + 0.7 * rng.standard_normal((S, M, V)))
    ids = np.zeros((S, M), np.int64)
    for s in range(S):
        for j in range(M):
            c = np.cumsum(draft[s, j].astype(np.float64))
            ids[s, j] = min(V - 1, np.searchsorted(c, rng.random() * c[-1], side="right"))
    return target, draft, ids, rng.random((S, M)).astype(np.float32), rng.random(S).astype(np.float32)


@pytest.mark.parametrize("S,M,V", [(1, 1, 1), (3, 2, 2), (5, 4, 7), (9, 3, 31), (4, 7, 320), (33, 5, 1000),
                                   (2, 64, 50), (3, 33, 129), (8, 4, 49152), (2, 2, 128257)])
@pytest.mark.parametrize("point", [False, True])
def test_verify(S, M, V, point):
    target, draft, ids, au, su = _case(S, M, V, seed=S * 100 + M)
    n = np.random.default_rng(V).integers(-1, M + 2, size=S)
    n[0] = M
    d = None if point else draft
    got, ref = _verify(target, d, ids, n, au, su), _verify_ref(target, d, ids, n, au, su)
    assert np.array_equal(got[1], ref[1]) and np.array_equal(got[0], ref[0])


def test_verify_equal_models_accept_everything():
    target, draft, ids, au, su = _case(6, 5, 400, seed=1, same=True)
    got = _verify(target, draft, ids, np.full(6, 5), au, su)
    assert np.all(got[1] == 6) and np.array_equal(got[0][:, :5], ids)


def test_verify_without_drafts_draws_from_the_target():
    target, _, _, _, su = _case(7, 0, 900, seed=2)
    ids, au = np.zeros((7, 0), np.int64), np.zeros((7, 0), np.float32)
    got, ref = _verify(target, None, ids, np.zeros(7, int), au, su), _verify_ref(target, None, ids, np.zeros(7, int), au, su)
    assert np.array_equal(got[0], ref[0]) and np.all(got[1] == 1)


def test_verify_borders():
    """Numbers at the borders, zero and unusable probabilities, ids outside the vocabulary."""
    V, M = 10, 2
    rows = np.zeros((9, M + 1, V), np.float32)
    drows = np.zeros((9, M, V), np.float32)
    ids = np.zeros((9, M), np.int64)
    au, su = np.zeros((9, M), np.float32), np.zeros(9, np.float32)
    rows[:, :, 3], rows[:, :, 6] = 0.5, 0.5
    drows[:, :, 3], drows[:, :, 6] = 0.5, 0.5
    ids[:] = 3
    au[0] = 0.99999994                       # u q < p with equal p and q: accepted below one
    ids[1] = 5                               # p = q = 0: 0 < 0 is refused; the rest max(p - q, 0) is zero: p itself
    su[1] = 0.5                              # cumulative sums 0.5, 1: the lowest above 0.5 is the second
    ids[2], drows[2, :, 4] = 4, 1.0          # drafted where p is zero
    drows[2, :, 3] = 0.25
    su[3], ids[3, 1] = 1.0, 7                # a number of one: the last possible token
    ids[4] = 4000000000                      # outside the vocabulary
    rows[5] = 0                              # no probability anywhere: token 0
    rows[6, :, 1], rows[6, :, 2], drows[6, :, 3] = np.nan, -4.0, np.nan
    au[7] = 1.0                              # u q < p fails at equality: refused, and p - q leaves nothing
    su[8] = np.nextafter(np.float32(0.5), np.float32(0))
    n = np.full(9, M)
    for d in (drows, None):
        got, ref = _verify(rows, d, ids, n, au, su), _verify_ref(rows, d, ids, n, au, su)
        assert np.array_equal(got[1], ref[1]), (got[1], ref[1])
        assert np.array_equal(got[0], ref[0]), (got[0], ref[0])


@pytest.mark.parametrize("ldt,ldd", [(1001, 1003), (1008, 1000), (1000, 1001)])
def test_verify_strides_and_stream(ldt, ldd):
    target, draft, ids, au, su = _case(5, 3, 1000, seed=9)
    n = np.array([3, 2, 0, 3, 1])
    s = torch.cuda.Stream()
    got = _verify(target, draft, ids, n, au, su, ldt=ldt, ldd=ldd, stream=s.cuda_stream)
    ref = _verify_ref(target, draft, ids, n, au, su)
    assert np.array_equal(got[0], ref[0]) and np.array_equal(got[1], ref[1])


def test_verified_tokens_follow_the_target():
    """20,000 sequences of one drafted token: the first given token is distributed as the target's row
    whatever the draft's. Each of 6 counts is binomial; 5 standard deviations bound it (p < 1e-5 in all)."""
    V, S = 6, 20000
    p = np.array([0.4, 0.05, 0.25, 0.1, 0.2, 0.0], np.float32)
    q = np.array([0.1, 0.5, 0.2, 0.05, 0.05, 0.1], np.float32)
    rng = np.random.default_rng(11)
    ids = rng.choice(V, size=(S, 1), p=q.astype(np.float64) / q.astype(np.float64).sum())
    target = np.broadcast_to(p, (S, 2, V)).copy()
    draft = np.broadcast_to(q, (S, 1, V)).copy()
    got = _verify(target, draft, ids, np.ones(S, int), rng.random((S, 1)).astype(np.float32),
                  rng.random(S).astype(np.float32))
    counts = np.bincount(got[0][:, 0], minlength=V)
    for v in range(V):
        assert abs(counts[v] - S * p[v]) <= 5 * math.sqrt(S * p[v] * (1 - p[v])) + 1e-9, counts


def test_probs_then_verify_captured():
    """The two together in one graph, replayed over new logits."""
    from laicompute_b200.serving import logits_probs, verify_drafts
    S, M, V = 4, 3, 2000
    g = torch.Generator().manual_seed(0)
    logits = torch.zeros(S * (M + 1), V, device="cuda")
    temp = torch.full((S * (M + 1),), 0.8, device="cuda")
    probs = torch.zeros_like(logits)
    ids = torch.randint(0, V, (S, M), generator=g).int().cuda()
    n = torch.full((S,), M, dtype=torch.int32, device="cuda")
    au, su = torch.rand(S, M, generator=g).cuda(), torch.rand(S, generator=g).cuda()
    out = torch.zeros(S, M + 1, dtype=torch.int32, device="cuda")
    cnt = torch.zeros(S, dtype=torch.int32, device="cuda")

    def call(stream):
        logits_probs(S * (M + 1), V, logits.data_ptr(), temp.data_ptr(), probs.data_ptr(), stream=stream)
        verify_drafts(S, M, V, probs.data_ptr(), 0, ids.data_ptr(), n.data_ptr(), au.data_ptr(), su.data_ptr(),
                      out.data_ptr(), cnt.data_ptr(), stream=stream)
    call(0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(torch.cuda.current_stream().cuda_stream)
    for seed in range(3):
        x = torch.randn(S * (M + 1), V, generator=torch.Generator().manual_seed(seed)) * 3
        x[torch.arange(0, S * (M + 1), M + 1), ids[:, 0].cpu().long()] = 12.0  # the first draft is likely
        logits.copy_(x)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        ref = _verify_ref(probs.cpu().numpy().reshape(S, M + 1, V), None, ids.cpu().numpy(), n.cpu().numpy(),
                          au.cpu().numpy(), su.cpu().numpy())
        assert np.array_equal(out.cpu().numpy(), ref[0]) and np.array_equal(cnt.cpu().numpy(), ref[1])
