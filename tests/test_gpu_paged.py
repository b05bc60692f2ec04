"""The KV cache in pages on the GPU: append with the position rotation (exact), and attention with shared
prefixes against the definition in 64 bits, at the sizes and masks where they can go wrong."""
import math
import random

import numpy as np
import pytest
import torch

from serving_util import F16, F32, TORCH, Cache, attend, close, ints, reference

pytestmark = pytest.mark.gpu

LAYOUTS = [(9, 3, 64), (32, 8, 128), (4, 2, 32), (8, 1, 128), (3, 3, 64), (10, 2, 128), (7, 1, 32)]


# ------------------------------------------------------------------------------------------------
# append
# ------------------------------------------------------------------------------------------------

def _rope(positions, dim, seed=0):
    g = torch.Generator().manual_seed(seed)
    a = torch.randn(positions, dim // 2, generator=g) * 3
    return torch.stack([torch.cos(a), torch.sin(a)], dim=-1).float().contiguous()


def _rotate_np(x, cs, pairs):
    """Adjacent pairs in FP32, unfused (the reference's arithmetic)."""
    y = x.astype(np.float32).copy()
    a, b = y[..., 0:2 * pairs:2].copy(), y[..., 1:2 * pairs:2].copy()
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    y[..., 0:2 * pairs:2] = a * c - b * s
    y[..., 1:2 * pairs:2] = a * s + b * c
    return y


def _append(heads, hkv, d, page, rows, in_type, q_type, rope_dim, seed, pad=0, aligned=True, padding=True):
    rng = random.Random(seed)
    nseq, per_seq = 3, 5
    num_pages = nseq * per_seq + 1
    places = [(s, t) for s in range(nseq) for t in range(per_seq * page)]
    rng.shuffle(places)
    places = places[:rows]
    pos = [t for _, t in places]
    if padding and rows > 2:
        pos[1] = -1
    ids = list(range(num_pages))
    rng.shuffle(ids)
    table = np.array(ids[:nseq * per_seq]).reshape(nseq, per_seq)
    g = torch.Generator().manual_seed(seed)
    w = [heads * d, hkv * d, hkv * d]
    ld = sum(w) + pad
    x = torch.randn(rows * ld + 1, generator=g).to(TORCH[in_type])
    off = 0 if aligned else 1
    xs = x[off:off + rows * ld].view(rows, ld).float().numpy()
    cs = _rope(per_seq * page, rope_dim) if rope_dim else torch.zeros(1, 1, 2)
    xd, csd = x.cuda(), cs.cuda()
    qout = torch.full((rows * (w[0] + pad) + 1,), 5.0, dtype=TORCH[q_type], device="cuda")
    k = torch.full((num_pages, hkv, page, d), 9.0, dtype=torch.float16, device="cuda")
    v = torch.full_like(k, 11.0)
    err = ints([0])
    from laicompute_b200.serving import KvPages
    pages = KvPages(k.data_ptr(), v.data_ptr(), num_pages, hkv, page, d, err=err.data_ptr())
    plan = pages.append_plan(rows, heads, nseq, per_seq, in_type=in_type, q_type=q_type, ldq=ld, ldk=ld, ldv=ld,
                             ldqo=w[0] + pad, rope_dim=rope_dim, rope_positions=per_seq * page if rope_dim else 0)
    e, eq = xd.element_size(), qout.element_size()
    base = xd.data_ptr() + off * e
    post, seqt, tabt = ints(pos), ints([s for s, _ in places]), ints(table.tolist())
    plan(base, base + w[0] * e, base + (w[0] + w[1]) * e, qout.data_ptr() + off * eq, post.data_ptr(), tabt.data_ptr(),
         csd.data_ptr() if rope_dim else 0, seq=seqt.data_ptr())
    pages.check()
    live = [i for i in range(rows) if pos[i] >= 0]
    csr = cs.numpy()[[max(p, 0) for p in pos]] if rope_dim else np.zeros((rows, 0, 2), np.float32)
    rot = _rotate_np(xs[:, :w[0] + w[1]].reshape(rows, heads + hkv, d), csr, rope_dim // 2)
    nt = np.float32 if q_type == F32 else np.float16
    want_q = np.full((rows, w[0] + pad), 5.0, nt)
    want_q[live, :w[0]] = rot[live, :heads].reshape(len(live), -1).astype(nt)
    wk, wv = np.full(k.shape, 9.0, np.float16), np.full(k.shape, 11.0, np.float16)
    for i in live:
        s, t = places[i]
        wk[table[s, t // page], :, t % page] = rot[i, heads:].astype(np.float16)
        wv[table[s, t // page], :, t % page] = xs[i, w[0] + w[1]:sum(w)].reshape(hkv, d).astype(np.float16)
    got_q = qout[off:off + rows * (w[0] + pad)].view(rows, -1).cpu().numpy()
    assert np.array_equal(got_q, want_q)
    assert np.array_equal(k.cpu().numpy(), wk) and np.array_equal(v.cpu().numpy(), wv)


@pytest.mark.parametrize("heads,hkv,d", LAYOUTS)
@pytest.mark.parametrize("in_type,q_type", [(F32, F32), (F32, F16), (F16, F32), (F16, F16)])
def test_append_exact(heads, hkv, d, in_type, q_type):
    """Rotation, rounding and place of every element, bit for bit; padding rows and everything else untouched."""
    _append(heads, hkv, d, 16, 23, in_type, q_type, d, seed=heads * d + in_type)


@pytest.mark.parametrize("rope_dim", [0, 2, 6, 32, 62])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_append_partial_rotation_and_pages(rope_dim, page):
    _append(6, 2, 64, page, 40, F32, F32, rope_dim, seed=page + rope_dim)


@pytest.mark.parametrize("in_type", [F32, F16])
@pytest.mark.parametrize("pad,aligned", [(8, True), (1, True), (3, False), (0, False)])
def test_append_strides_and_alignment(pad, aligned, in_type):
    _append(5, 1, 32, 32, 9, in_type, in_type, 32, seed=pad, pad=pad, aligned=aligned)


@pytest.mark.parametrize("rows", [1, 2, 200])
def test_append_row_counts(rows):
    _append(32, 8, 128, 128, rows, F32, F32, 128, seed=rows)


def test_append_in_place_and_without_queries():
    """q rotated in place; heads = 0 writes only the pages."""
    from laicompute_b200.serving import KvPages
    hkv, d, page = 2, 64, 16
    g = torch.Generator().manual_seed(3)
    x = torch.randn(4, 4 * d + 2 * hkv * d, generator=g)
    cs = _rope(32, d)
    want = _rotate_np(x[:, :6 * d].view(4, 6, d).numpy(), cs.numpy()[[5, 6, 7, 30]], d // 2)
    for heads in (4, 0):
        xd, csd = x.cuda(), cs.cuda()
        k = torch.zeros(3, hkv, page, d, dtype=torch.float16, device="cuda")
        v = torch.zeros_like(k)
        err = ints([0])
        pages = KvPages(k.data_ptr(), v.data_ptr(), 3, hkv, page, d, err=err.data_ptr())
        ld = x.shape[1]
        plan = pages.append_plan(4, heads, 1, 2, ldq=ld, ldk=ld, ldv=ld, ldqo=ld, rope_dim=d, rope_positions=32)
        b = xd.data_ptr()
        pos, seq, table = ints([5, 6, 7, 30]), ints([0] * 4), ints([[2, 0]])
        plan(b if heads else 0, b + 4 * 4 * d, b + 4 * 6 * d, b if heads else 0, pos.data_ptr(), table.data_ptr(),
             csd.data_ptr(), seq=seq.data_ptr())
        pages.check()
        got = xd.cpu().numpy()
        assert np.array_equal(got[:, :4 * d], want[:, :4].reshape(4, -1) if heads else x[:, :4 * d].numpy())
        assert np.array_equal(got[:, 4 * d:], x[:, 4 * d:].numpy())
        assert np.array_equal(k[2, :, 5].cpu().numpy(), want[0, 4:].astype(np.float16))
        assert np.array_equal(k[0, :, 14].cpu().numpy(), want[3, 4:].astype(np.float16))


def test_append_bad_indices_are_left_out():
    """Rows with a bad position, sequence or page are skipped and reported; the others are written."""
    from laicompute_b200._native import LAIC_E_INVALID, LaicError
    from laicompute_b200.serving import KvPages
    hkv, d, page = 1, 32, 16
    x = torch.randn(6, 3 * d).cuda()
    k = torch.zeros(2, hkv, page, d, dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    qo = torch.zeros(6, d, device="cuda")
    err = ints([0])
    pages = KvPages(k.data_ptr(), v.data_ptr(), 2, hkv, page, d, err=err.data_ptr())
    plan = pages.append_plan(6, 1, 2, 2, ldq=3 * d, ldk=3 * d, ldv=3 * d)
    pos, seq, table = ints([0, 32, 1, 0, 17, 2]), ints([0, 0, 2, 1, 0, 0]), ints([[1, 2], [-1, 0]])
    b = x.data_ptr()
    plan(b, b + 4 * d, b + 8 * d, qo.data_ptr(), pos.data_ptr(), table.data_ptr(), seq=seq.data_ptr())
    with pytest.raises(LaicError) as ex:
        pages.check()
    assert ex.value.code == LAIC_E_INVALID
    assert all(w in str(ex.value) for w in ("sequence index", "position", "page id"))
    pages.check()  # cleared
    live = [0, 5]
    assert torch.equal(qo[live], x[live, :d]) and not qo[[1, 2, 3, 4]].any()
    want = torch.zeros_like(k)
    want[1, 0, 0], want[1, 0, 2] = x[0, d:2 * d].half(), x[5, d:2 * d].half()
    assert torch.equal(k, want)


# ------------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------------

def _q(rows, heads, d, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, heads * d, generator=g) * 1.5).to(TORCH[dtype]).cuda()


@pytest.mark.parametrize("heads,hkv,d", LAYOUTS)
@pytest.mark.parametrize("dtype", [F32, F16])
def test_attention_lengths(heads, hkv, d, dtype):
    """Lengths around the tiles' and pages' ends, none at all, padding; NaN in every place no row sees."""
    lens = [1, 0, 2, 15, 16, 17, 63, -1, 64, 65, 127, 129, 200]
    cache = Cache([max(n, 0) for n in lens], hkv, d, 16, seed=d)
    q = _q(len(lens), heads, d, dtype, seed=heads)
    out = attend(cache, q, lens)
    cache.pages().check()
    ref, tol = reference(cache, q, lens)
    live = [i for i, n in enumerate(lens) if n >= 0]
    close(out[live], ref[live], tol[live])
    assert not out[1].any() and torch.all(out[7] == 7.0)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_attention_pages_and_splits(page, dtype):
    """Long and short rows together: several items per row, joined; rows in any order of sequences."""
    lens = [1500, 3, 777, 64, 1024, 511]
    cache = Cache(lens, 2, 64, page, seed=page, room=3)
    seqs = [4, 0, 2, 5, 3, 1]
    rl = [lens[s] for s in seqs]
    q = _q(6, 8, 64, dtype, seed=5)
    out = attend(cache, q, rl, seqs)
    ref, tol = reference(cache, q, rl, seqs)
    close(out, ref, tol)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_attention_strides(dtype):
    """Rows of q and out inside wider rows, at odd offsets."""
    cache = Cache([40, 90], 2, 64, 16, seed=1)
    wide = torch.randn(2, 4 * 64 + 7).to(TORCH[dtype]).cuda()
    q = wide[:, 3:3 + 256]
    buf = torch.full((2, 256 + 5), 7.0, dtype=TORCH[dtype], device="cuda")
    out = buf[:, 1:257]
    attend(cache, q, [40, 90], out=out)
    ref, tol = reference(cache, q, [40, 90])
    close(out, ref, tol)
    assert torch.all(buf[:, 0] == 7.0) and torch.all(buf[:, 257:] == 7.0)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("heads,hkv,d,nrows", [(32, 8, 128, 3), (9, 3, 64, 7), (4, 2, 32, 20), (8, 1, 128, 33),
                                               (8, 8, 64, 5)])
@pytest.mark.parametrize("shared,page", [(1, 16), (100, 16), (64, 64), (700, 32)])
def test_attention_shared_prefix(heads, hkv, d, nrows, shared, page, dtype):
    """Two groups with their own prefixes (whole pages shared, a partly filled one copied) and rows of none."""
    rng = random.Random(shared + nrows)
    n1 = nrows // 2 + 1
    a, b = list(range(n1)), list(range(n1, nrows))
    sb = shared // 2 + 1
    lens = [shared + rng.randint(0, 90) for _ in a] + [sb + rng.randint(0, 150) for _ in b] + [33, 200]
    groups = ([0, n1, nrows] if b else [0, n1], [shared, sb] if b else [shared])
    cache = Cache(lens, hkv, d, page, seed=shared, shared=[(a, shared)] + ([(b, sb)] if b else []))
    q = _q(len(lens), heads, d, dtype, seed=nrows)
    out = attend(cache, q, lens, groups=groups)
    cache.pages().check()
    ref, tol = reference(cache, q, lens)
    close(out, ref, tol)
    plain = attend(cache, q, lens)  # the same rows without groups
    close(plain, ref, tol)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("heads,hkv,d,nrows,shared,page", [
    (8, 2, 128, 12, 256, 16), (8, 2, 128, 12, 300, 64), (8, 2, 64, 40, 700, 16), (8, 1, 128, 33, 1111, 256),
    (9, 3, 64, 90, 520, 32), (2, 2, 64, 130, 640, 128), (8, 1, 64, 70, 2500, 64), (4, 1, 128, 65, 2048, 32)])
def test_attention_wide_groups(heads, hkv, d, nrows, shared, page, dtype):
    """Groups of many columns behind long prefixes (whole tiles of theirs go to the tensor-memory kernel), one
    or two column pairs, partly filled ones, and rows that see less, nothing, or are padding."""
    rng = random.Random(shared)
    lens = [shared + rng.randint(0, 70) for _ in range(nrows)] + [shared // 2 + 20] * (nrows // 2 + 3) + [17]
    groups = ([0, nrows, nrows + nrows // 2 + 3], [shared, shared // 2])
    cache = Cache(lens, hkv, d, page, seed=shared, shared=[(list(range(nrows)), shared),
                                                           (list(range(nrows, len(lens) - 1)), shared // 2)])
    q = _q(len(lens), heads, d, dtype, seed=nrows)
    rows = list(range(0, len(lens), 5)) + [nrows - 1, nrows, len(lens) - 2, len(lens) - 1]  # checked in 64 bits
    out = attend(cache, q, lens, groups=groups)
    cache.pages().check()
    ref, tol = reference(cache, q[rows], [lens[r] for r in rows], rows)
    close(out[rows], ref, tol)
    plain = attend(cache, q, lens)
    assert (out.double() - plain.double()).abs().max() <= 2 * tol.max()
    short = list(lens)
    short[1], short[2], short[nrows - 1], short[nrows] = shared - 3, 0, -1, 5
    out = attend(cache, q, short, groups=groups)
    cache.pages().check()
    rows = [r for r in rows + [1, nrows] if short[r] > 0]
    ref, tol = reference(cache, q[rows], [short[r] for r in rows], rows)
    close(out[rows], ref, tol)
    assert not out[2].any() and torch.all(out[nrows - 1] == 7.0)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("heads,hkv,d,start,nrows,page", [(8, 2, 128, 400, 150, 64), (9, 3, 64, 900, 100, 16),
                                                          (8, 1, 64, 0, 400, 128), (8, 2, 128, 2000, 16, 32)])
def test_attention_prompt_rows(heads, hkv, d, start, nrows, page, dtype):
    """A prompt's rows behind cached ones: whole tiles seen by all rows of a column pair, causal edges beyond."""
    total = start + nrows
    cache = Cache([total], hkv, d, page, seed=nrows)
    lens = [start + j + 1 for j in range(nrows)]
    q = _q(nrows, heads, d, dtype, seed=start + 2)
    buf = torch.zeros(nrows, heads * d + 3, dtype=q.dtype, device="cuda")  # rows that are not 16-byte aligned
    buf[:, 1:heads * d + 1] = q
    rows = sorted({0, 1, nrows // 3, nrows // 2, nrows - 2, nrows - 1})
    ref, tol = reference(cache, q[rows], [lens[r] for r in rows], [0] * len(rows))
    for x in (q, buf[:, 1:heads * d + 1]):
        out = attend(cache, x, lens, seqs=[0] * nrows, groups=([0, nrows], [total]))
        cache.pages().check()
        close(out[rows], ref, tol)


@pytest.mark.parametrize("scale", [0.05, 1e-30, 3.0])
def test_attention_wide_group_scales(scale):
    """Small, vanishing and large scales (maxima that outgrow their reference again and again)."""
    cache = Cache([1000] * 20, 1, 64, 64, seed=4, shared=[(list(range(20)), 1000)])
    q = _q(20, 4, 64, F32, seed=3)
    out = attend(cache, q, [1000] * 20, groups=([0, 20], [1000]), scale=scale)
    rows = [0, 7, 19]
    ref, tol = reference(cache, q[rows], [1000] * 3, rows, scale=scale)
    close(out[rows], ref, tol)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_attention_rows_shorter_than_their_prefix(dtype):
    """Rows that see less than the shared positions, nothing, or are padding."""
    lens = [300, 10, 0, 150, -1, 129, 1]
    cache = Cache([300] * 7, 2, 64, 16, seed=8, shared=[(list(range(7)), 300)])
    q = _q(7, 8, 64, dtype, seed=9)
    out = attend(cache, q, lens, groups=([0, 7], [300]))
    ref, tol = reference(cache, q, lens)
    live = [i for i, n in enumerate(lens) if n >= 0]
    close(out[live], ref[live], tol[live])
    assert not out[2].any() and torch.all(out[4] == 7.0)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("heads,hkv,d", [(32, 8, 128), (9, 3, 64), (4, 2, 32)])
@pytest.mark.parametrize("start,rows", [(0, 1), (0, 70), (200, 37), (1000, 5)])
def test_attention_causal_rows(heads, hkv, d, start, rows, dtype):
    """A prompt's rows (or drafted tokens): one sequence, lengths one apart, one group."""
    total = start + rows
    cache = Cache([total], hkv, d, 32, seed=rows)
    lens = [start + j + 1 for j in range(rows)]
    q = _q(rows, heads, d, dtype, seed=start + 1)
    out = attend(cache, q, lens, seqs=[0] * rows, groups=([0, rows], [total]))
    cache.pages().check()
    ref, tol = reference(cache, q, lens, [0] * rows)
    close(out, ref, tol)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("heads,hkv,d,rows,start", [(4, 2, 64, 30, 150), (32, 8, 128, 12, 150), (2, 2, 32, 9, 150),
                                                    (8, 1, 128, 40, 150), (8, 1, 128, 40, 300), (4, 1, 64, 80, 490)])
def test_masked_infinities_stay_out(heads, hkv, d, rows, start, dtype):
    """Keys and values of a later row that are infinite or NaN reach only the rows that see them."""
    total = start + rows
    cache = Cache([total], hkv, d, 16, seed=2)
    lens = [start + j + 1 for j in range(rows)]
    q = _q(rows, heads, d, dtype, seed=4)
    bad = total - 4  # position seen by the last four rows only
    p, off = cache.rows[0][bad // 16], bad % 16
    cache.k[p, :, off, 0] = float("nan")
    cache.v[p, :, off, 1] = float("inf")
    cache.v[p, :, off, 2] = float("nan")
    out = attend(cache, q, lens, seqs=[0] * rows, groups=([0, rows], [total]))
    ref, tol = reference(cache, q, lens, [0] * rows)  # (the reference's own copy is finite)
    n = rows - 4
    close(out[:n], ref[:n], tol[:n])
    assert torch.isnan(out[n:]).all()


def test_attention_extreme_queries():
    """Query magnitudes outside binary16's range, zero rows, scores far apart, a given scale."""
    cache = Cache([200] * 5, 1, 64, 16, seed=6)
    q = _q(5, 4, 64, F32, seed=7)
    q[0] *= 1e6
    q[1] *= 1e-9
    q[2] = 0
    q[3] *= 40
    for scale in (0.0, 1e-6, 0.7):
        out = attend(cache, q, [200] * 5, scale=scale)
        ref, tol = reference(cache, q, [200] * 5, scale=scale)
        if scale != 1e-6:  # row 0's scores are beyond FP32's resolution of their differences
            out, ref, tol = out[1:], ref[1:], tol[1:]
        close(out, ref, tol)


def test_attention_bad_indices():
    """Bad pages, sequences, lengths and groups are reported; rows that name none are right."""
    from laicompute_b200._native import LaicError
    cache = Cache([50, 50, 50], 1, 32, 16, seed=3)
    q = _q(3, 2, 32, F32, seed=1)
    ref, tol = reference(cache, q, [50] * 3)
    good = cache.table.clone()
    for value, text in ((-1, "page id"), (10 ** 6, "page id"), (cache.num_pages, "page id")):
        cache.table = good.clone()
        cache.table[1, 2] = value
        out = attend(cache, q, [50] * 3)
        with pytest.raises(LaicError) as ex:
            cache.pages().check()
        assert text in str(ex.value)
        close(out[[0, 2]], ref[[0, 2]], tol[[0, 2]])
    cache.table = good
    out = attend(cache, q, [50] * 3, seqs=[0, 3, 2])
    with pytest.raises(LaicError) as ex:
        cache.pages().check()
    assert "sequence index" in str(ex.value)
    close(out[[0, 2]], ref[[0, 2]], tol[[0, 2]])
    out = attend(cache, q, [50, 64, 50], bounds=dict(max_len=50))  # a length above its bound is cut to it
    with pytest.raises(LaicError) as ex:
        cache.pages().check()
    assert "beyond" in str(ex.value)
    close(out, ref, tol)
    for starts in ([0, 4], [2, 1], [-1, 2]):
        out = attend(cache, q, [50] * 3, groups=(starts, [16]), bounds=dict(max_group_rows=3, max_private=50))
        with pytest.raises(LaicError) as ex:
            cache.pages().check()
        assert "group rows" in str(ex.value)
        close(out, ref, tol)  # the refused group shares nothing
    cache.pages().check()


def test_attention_captured_and_on_two_streams():
    """A captured call replays over new lengths and queries; two calls at once with their own workspaces."""
    cache = Cache([700, 900, 40], 2, 64, 16, seed=12)
    pages = cache.pages()
    plan = pages.attention_plan(3, 8, 3, cache.per_seq, 900)
    q, out = _q(3, 8, 64, F32, 1), torch.zeros(3, 512, device="cuda")
    lens = ints([5, 6, 7])
    ws = [torch.empty(plan.workspace_bytes, dtype=torch.uint8, device="cuda") for _ in range(2)]
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    plan(q.data_ptr(), out.data_ptr(), lens.data_ptr(), cache.table.data_ptr(), workspace=ws[0].data_ptr())  # warm up
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        plan(q.data_ptr(), out.data_ptr(), lens.data_ptr(), cache.table.data_ptr(), workspace=ws[0].data_ptr(),
             stream=torch.cuda.current_stream().cuda_stream)
    for seed, ln in ((2, [700, 900, 40]), (3, [1, 0, 33]), (4, [512, 513, 40])):
        q.copy_(_q(3, 8, 64, F32, seed))
        lens.copy_(ints(ln))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        ref, tol = reference(cache, q, ln)
        close(out, ref, tol)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    qs = [_q(3, 8, 64, F32, 20 + i) for i in range(2)]
    outs = [torch.zeros(3, 512, device="cuda") for _ in range(2)]
    lens.copy_(ints([700, 900, 40]))
    torch.cuda.synchronize()
    for _ in range(5):
        for i in range(2):
            plan(qs[i].data_ptr(), outs[i].data_ptr(), lens.data_ptr(), cache.table.data_ptr(),
                 workspace=ws[i].data_ptr(), stream=streams[i].cuda_stream)
    torch.cuda.synchronize()
    for i in range(2):
        ref, tol = reference(cache, qs[i], [700, 900, 40])
        close(outs[i], ref, tol)


@pytest.mark.parametrize("shared", [0, 600])
def test_offsets_beyond_32_bits(shared):
    """A pool of more than 2^31 elements per side: append and both attentions at its last pages."""
    from laicompute_b200.serving import KvPages
    hkv, d, page, heads, n = 8, 128, 64, 32, 12
    num_pages = (1 << 31) // (hkv * page * d) + 40
    small = Cache([640] * n, hkv, d, page, seed=3, shared=[(list(range(n)), shared)] if shared else None)
    k = torch.empty(num_pages, hkv, page, d, dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    base = num_pages - small.num_pages
    k[base:], v[base:] = small.k, small.v
    table = torch.where(small.table >= 0, small.table + base, small.table)
    assert table.dtype == torch.int32
    pages = KvPages(k.data_ptr(), v.data_ptr(), num_pages, hkv, page, d, err=small.err.data_ptr())
    # the last position of every row is appended again, at a place past 2^31 elements
    new = torch.randn(n, 2 * hkv * d).half()
    ld = 2 * hkv * d
    x, pos = new.cuda(), ints([639] * n)
    plan = pages.append_plan(n, 0, n, table.shape[1], in_type=F16, q_type=F16, ldk=ld, ldv=ld)
    plan(0, x.data_ptr(), x.data_ptr() + 2 * hkv * d, 0, pos.data_ptr(), table.data_ptr())
    for i in range(n):
        small.seq_k[i][639] = new[i, :hkv * d].view(hkv, d)
        small.seq_v[i][639] = new[i, hkv * d:].view(hkv, d)
    q = _q(n, heads, d, F32, seed=8)
    big = Cache.__new__(Cache)
    big.__dict__.update(small.__dict__)
    big.k, big.v, big.table, big.num_pages = k, v, table, num_pages
    lens = [640] * n
    out = attend(big, q, lens, groups=([0, n], [shared]) if shared else None)
    big.pages().check()
    rows = [0, 5, n - 1]
    ref, tol = reference(small, q[rows], [640] * 3, rows)
    close(out[rows], ref, tol)


def test_attention_is_repeatable():
    """The same call gives the same bits (no order of arrival enters a sum)."""
    cache = Cache([1200] * 6, 2, 128, 16, seed=1, shared=[(list(range(6)), 1000)])
    q = _q(6, 8, 128, F32, seed=2)
    a = attend(cache, q, [1200] * 6, groups=([0, 6], [1000]))
    for _ in range(3):
        assert torch.equal(a, attend(cache, q, [1200] * 6, groups=([0, 6], [1000])))


@pytest.mark.parametrize("dtype", [F32, F16])
def test_rows_of_no_group(dtype):
    """Rows before, between and behind the groups, with and without positions of their own; groups without rows."""
    cache = Cache([400] * 30, 1, 64, 32, seed=9, shared=[(list(range(2, 22)), 400)])
    lens = [0, -1] + [400] * 20 + [0, -1] + [0] * 6
    q = _q(30, 4, 64, dtype, seed=6)
    out = attend(cache, q, lens, groups=([2, 2, 22, 22], [64, 400, 10]), bounds=dict(max_private=0))
    cache.pages().check()
    rows = [2, 11, 21]
    ref, tol = reference(cache, q[rows], [400] * 3, rows)
    close(out[rows], ref, tol)
    assert not out[[0, 22, 24, 29]].any() and torch.all(out[[1, 23]] == 7.0)
    lens = [37, 5] + [400] * 20 + [1, 0, 399] + [12] * 5
    out = attend(cache, q, lens, groups=([2, 2, 22, 22], [64, 400, 10]))
    cache.pages().check()
    rows = list(range(0, 30, 3)) + [1, 22, 23, 24]
    ref, tol = reference(cache, q[rows], [lens[r] for r in rows], rows)
    close(out[rows], ref, tol)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("heads,hkv,d", [(8, 2, 64), (8, 2, 128), (7, 1, 128), (10, 2, 64)])
@pytest.mark.parametrize("cols", [20, 28, 40, 124, 128, 132, 256, 260])
def test_widths_around_the_tiles(cols, heads, hkv, d, dtype):
    """Widths at the kernels' thresholds and tiles' ends, causal (no private positions) and with private ones."""
    n = max(1, cols // (heads // hkv))
    cache = Cache([330] * n, hkv, d, 32, seed=cols, shared=[(list(range(n)), 300)])
    q = _q(n, heads, d, dtype, seed=cols)
    rows = sorted({0, n // 3, n // 2, n - 1})
    for lens in ([300 - (n - 1 - r) for r in range(n)], [301 + (r * 7) % 29 for r in range(n)]):
        out = attend(cache, q, lens, groups=([0, n], [300]))
        cache.pages().check()
        ref, tol = reference(cache, q[rows], [lens[r] for r in rows], rows)
        close(out[rows], ref, tol)


@pytest.mark.parametrize("n,length", [(3, 448), (3, 449), (3, 1024), (60, 448), (60, 1024), (60, 1025)])
def test_private_ranges_around_the_split(n, length):
    """Few and many rows whose ranges end at and behind what one CTA takes, ragged."""
    lens = [max(1, length - (37 * r) % length) for r in range(n)]
    cache = Cache(lens, 8, 64, 64, seed=n)
    q = _q(n, 16, 64, F32, seed=length)
    out = attend(cache, q, lens)
    cache.pages().check()
    rows = sorted({0, 1, n // 2, n - 1})
    ref, tol = reference(cache, q[rows], [lens[r] for r in rows], rows)
    close(out[rows], ref, tol)


def test_long_bounds_and_many_groups():
    """A bound far above the lengths (its splits are empty), and a group per pair of rows."""
    n = 40
    lens = [70 + 13 * i for i in range(n)]
    cache = Cache(lens, 2, 64, 16, seed=2, shared=[([2 * i, 2 * i + 1], 64) for i in range(n // 2)], room=4000)
    q = _q(n, 8, 64, F32, seed=4)
    ref, tol = reference(cache, q, lens)
    groups = (list(range(0, n + 1, 2)), [64] * (n // 2))
    for kw in (dict(max_len=60000, max_private=60000, max_shared=60000), dict(max_len=60000, max_private=2000)):
        out = attend(cache, q, lens, groups=groups, bounds=kw)
        cache.pages().check()
        close(out, ref, tol)
    out = attend(cache, q, lens, bounds=dict(max_len=60000))
    close(out, ref, tol)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_wide_group_captured_on_two_streams(dtype):
    """Wide groups and private positions: a captured call replays over other lengths, groups and queries, with
    padding rows and one sequence named by several rows; then calls at once, each with its own workspace."""
    n, heads, hkv, d = 36, 8, 2, 64
    cache = Cache([900 + 3 * i for i in range(n)], hkv, d, 32, seed=4, shared=[(list(range(n)), 850)])
    pages = cache.pages()
    kw = dict(type=dtype, groups=2, max_group_rows=32, max_shared=850, max_private=400)
    plan = pages.attention_plan(n, heads, n, cache.per_seq, 1024, **kw)
    ws = [torch.full((plan.workspace_bytes,), 255, dtype=torch.uint8, device="cuda") for _ in range(2)]
    q, out = _q(n, heads, d, dtype, 1), torch.full((n, heads * d), 7.0, dtype=TORCH[dtype], device="cuda")
    lens, seq = ints([0] * n), ints([0] * n)
    starts, shared = ints([0, 0, 0]), ints([0, 0])

    def call(k, stream, qk, ok):
        plan(qk.data_ptr(), ok.data_ptr(), lens.data_ptr(), cache.table.data_ptr(), workspace=ws[k].data_ptr(),
             seq=seq.data_ptr(), group_rows=starts.data_ptr(), group_len=shared.data_ptr(), stream=stream)
    call(0, 0, q, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(0, torch.cuda.current_stream().cuda_stream, q, out)
    cases = [([0, 20, 36], [850, 700], [900 + 3 * i for i in range(n)], list(range(n))),
             ([4, 4, 34], [850, 850], [30, -1, 0, 250] + [860] * 30 + [399, 1], [5] * n),
             ([0, 32, 36], [64, 850], [450] * 31 + [-1] + [851, 850, 849, 0], [0, 0, 1, 2] * 9)]
    for seed, (gr, gl, ln, sq) in enumerate(cases):
        q.copy_(_q(n, heads, d, dtype, seed + 2))
        for t, x in ((lens, ln), (seq, sq), (starts, gr), (shared, gl)):
            t.copy_(ints(x))
        out.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        pages.check()
        rows = [r for r in range(0, n, 3) if ln[r] >= 0] + [35]
        ref, tol = reference(cache, q[rows], [ln[r] for r in rows], [sq[r] for r in rows])
        close(out[rows], ref, tol)
        assert all(torch.all(out[r] == 7.0) for r in range(n) if ln[r] < 0)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    qs = [_q(n, heads, d, dtype, 30 + i) for i in range(2)]
    outs = [torch.zeros_like(out) for _ in range(2)]
    alone = []
    for i in range(2):
        call(i, 0, qs[i], outs[i])
        torch.cuda.synchronize()
        alone.append(outs[i].clone())
        outs[i].zero_()
    torch.cuda.synchronize()
    for _ in range(5):
        for i in range(2):
            call(i, streams[i].cuda_stream, qs[i], outs[i])
    torch.cuda.synchronize()
    assert torch.equal(outs[0], alone[0]) and torch.equal(outs[1], alone[1])


FIRST_CALL = """
import torch
from laicompute_b200.serving import KvPages, logits_probs, verify_drafts
d, page, n = 64, 32, 64
k, v = (torch.randn(40, 1, page, d, device="cuda").half() for _ in range(2))
err, table = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.arange(40, dtype=torch.int32, device="cuda")[None].contiguous()
pages = KvPages(k.data_ptr(), v.data_ptr(), 40, 1, page, d, err=err.data_ptr())
q, out = torch.randn(n, d, device="cuda"), torch.zeros(n, d, device="cuda")
ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
lens, seq, gr, gl, one = ints([1280] * n), ints([0] * n), ints([0, n]), ints([1280]), ints([1])
x, t, pr = torch.randn(3, 20000, device="cuda"), torch.ones(3, device="cuda"), torch.zeros(3, 20000, device="cuda")
u, ids, cnt = torch.full((2,), 0.5, device="cuda"), ints([5, 6]), ints([0])
oid = ints([0, 0, 0])
new = torch.randn(1, d, device="cuda")
app = pages.append_plan(1, 0, 1, 40)
plan = pages.attention_plan(n, 1, 1, 40, 1280, groups=1, max_group_rows=n, max_shared=1280, max_private=0)
ws = torch.zeros(max(16, plan.workspace_bytes), dtype=torch.uint8, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    st = torch.cuda.current_stream().cuda_stream
    app(0, new.data_ptr(), new.data_ptr(), 0, one.data_ptr(), table.data_ptr(), stream=st)
    plan(q.data_ptr(), out.data_ptr(), lens.data_ptr(), table.data_ptr(), workspace=ws.data_ptr(), seq=seq.data_ptr(),
         group_rows=gr.data_ptr(), group_len=gl.data_ptr(), stream=st)
    logits_probs(3, 20000, x.data_ptr(), t.data_ptr(), pr.data_ptr(), stream=st)
    verify_drafts(1, 2, 20000, pr.data_ptr(), 0, ids.data_ptr(), gr.data_ptr(), u.data_ptr(), u.data_ptr(),
                  oid.data_ptr(), cnt.data_ptr(), stream=st)
graph.replay()
torch.cuda.synchronize()
pages.check()
ref = torch.nn.functional.scaled_dot_product_attention(q[None, None].double(), k.view(1, 1, 1280, d).double(), v.view(1, 1, 1280, d).double())
# as in reference(): scores to 35 * 1.2e-6 + 2e-6, weights to twice that and 2e-5, values to 0.8 on average
assert float((out - ref[0, 0]).abs().max()) < 1e-4
assert float((pr.double() - torch.softmax(x.double(), 1)).abs().max()) < 1e-6
assert int(cnt[0]) == 1
print("captured")
"""


def test_first_call_is_captured():
    """A process whose first call of each operator is made under stream capture."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALL], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


# ------------------------------------------------------------------------------------------------
# append and attention together, as a decode loop uses them
# ------------------------------------------------------------------------------------------------

def test_decode_loop_over_a_forked_cache():
    """A prompt of one sequence, forked to four by sharing its whole pages and copying the last: each then
    appends its own tokens and attends through the group; against plain attention over what was appended."""
    from laicompute_b200.serving import KvPages
    heads, hkv, d, page, prompt, steps, n = 8, 2, 64, 16, 37, 6, 4
    rng = torch.Generator().manual_seed(5)
    per_seq, num_pages = 4, 24
    k = torch.full((num_pages, hkv, page, d), float("nan"), dtype=torch.float16, device="cuda")
    v = torch.full_like(k, float("nan"))
    err = ints([0])
    pages = KvPages(k.data_ptr(), v.data_ptr(), num_pages, hkv, page, d, err=err.data_ptr())
    cs = _rope(64, d)
    csd = cs.cuda()
    w = (heads + 2 * hkv) * d

    def append(x, pos, seq, table):
        q = torch.empty(len(pos), heads * d, device="cuda")
        plan = pages.append_plan(len(pos), heads, table.shape[0], per_seq, ldq=w, ldk=w, ldv=w, rope_dim=d,
                                 rope_positions=64)
        b = x.data_ptr()
        keep = ints(pos), ints(seq)
        plan(b, b + 4 * heads * d, b + 4 * (heads + hkv) * d, q.data_ptr(), keep[0].data_ptr(), table.data_ptr(),
             csd.data_ptr(), seq=keep[1].data_ptr())
        append.keep = keep
        return q

    class Seen:  # what reference() reads
        head_dim, kv_heads = d, hkv
        seq_k, seq_v = [], []

    def rotated(x, pos):
        r = _rotate_np(x.numpy()[:, :(heads + hkv) * d].reshape(len(pos), heads + hkv, d), cs.numpy()[pos], d // 2)
        return torch.from_numpy(r[:, heads:]).half(), x[:, (heads + hkv) * d:].view(-1, hkv, d).half()

    x = torch.randn(prompt, w, generator=rng)
    table = ints([[3, 9, 1, 20]])
    q = append(x.cuda(), list(range(prompt)), [0] * prompt, table)
    kk, vv = rotated(x, list(range(prompt)))
    Seen.seq_k, Seen.seq_v = [kk], [vv]
    lens = [j + 1 for j in range(prompt)]

    def run(q, lens, seqs, table, starts, shared, max_private):
        out = torch.zeros_like(q)
        plan = pages.attention_plan(len(lens), heads, table.shape[0], per_seq, max(lens), groups=1,
                                    max_group_rows=len(lens), max_shared=shared, max_private=max_private)
        ws = torch.empty(max(16, plan.workspace_bytes), dtype=torch.uint8, device="cuda")
        keep = ints(lens), ints(seqs), ints(starts), ints([shared])
        plan(q.data_ptr(), out.data_ptr(), keep[0].data_ptr(), table.data_ptr(), workspace=ws.data_ptr(),
             seq=keep[1].data_ptr(), group_rows=keep[2].data_ptr(), group_len=keep[3].data_ptr())
        torch.cuda.synchronize()
        return out

    out = run(q, lens, [0] * prompt, table, [0, prompt], prompt, 0)
    ref, tol = reference(Seen, q, lens, [0] * prompt)
    close(out, ref, tol)
    rows = [[3, 9, 1, 20]] + [[3, 9, 4 + i, 12 + i] for i in range(1, n)]
    for i in range(1, n):  # the partly filled page is copied
        k[rows[i][2]], v[rows[i][2]] = k[1], v[1]
    table = ints(rows)
    Seen.seq_k, Seen.seq_v = [kk.clone() for _ in range(n)], [vv.clone() for _ in range(n)]
    for step in range(steps):
        pos = prompt + step
        x = torch.randn(n, w, generator=rng)
        q = append(x.cuda(), [pos] * n, list(range(n)), table)
        a, b = rotated(x, [pos] * n)
        for i in range(n):
            Seen.seq_k[i] = torch.cat([Seen.seq_k[i], a[i:i + 1]])
            Seen.seq_v[i] = torch.cat([Seen.seq_v[i], b[i:i + 1]])
        out = run(q, [pos + 1] * n, list(range(n)), table, [0, n], prompt, step + 1)
        ref, tol = reference(Seen, q, [pos + 1] * n)
        close(out, ref, tol)
    pages.check()
