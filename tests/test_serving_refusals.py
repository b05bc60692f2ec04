"""What the serving operators refuse, without a GPU: arguments on the host (before any launch), and the
index rules the kernels apply to device arrays (the same functions, compiled for the host)."""
import os
import subprocess

import pytest

from conftest import ROOT

BAD_SEQ, BAD_POS, BAD_PAGE, BAD_GROUP = 1, 2, 4, 8
PTR = 4096  # any non-null, 16-byte aligned value: every call here ends before it is used


def _pages(**kw):
    from laicompute_b200.serving import KvPages
    a = dict(k=PTR, v=PTR, num_pages=4, kv_heads=2, page_size=16, head_dim=64, err=PTR)
    a.update(kw)
    return KvPages(**a)


def _refused(code, text, f):
    from laicompute_b200._native import LaicError
    with pytest.raises(LaicError) as ex:
        f()
    assert ex.value.code == code and text in str(ex.value), str(ex.value)


INVALID, UNSUPPORTED = -1, -5


@pytest.mark.parametrize("kw,code,text", [
    (dict(head_dim=48), UNSUPPORTED, "head_dim"), (dict(page_size=24), UNSUPPORTED, "page_size"),
    (dict(page_size=8), UNSUPPORTED, "page_size"), (dict(page_size=512), UNSUPPORTED, "page_size"),
    (dict(kv_heads=0), INVALID, "kv_heads"), (dict(num_pages=0), INVALID, "num_pages"),
    (dict(k=0), INVALID, "null"), (dict(err=0), INVALID, "null"), (dict(v=PTR + 8), INVALID, "aligned")])
def test_pages_refused(kw, code, text):
    pages = _pages(**kw)
    _refused(code, text, lambda: pages.append_plan(1, 4, 1, 2)(PTR, PTR, PTR, PTR, PTR, PTR))

    def attend():
        pages.attention_plan(1, 4, 1, 2, 32)(PTR, PTR, PTR, PTR)
    _refused(code, text, attend)


@pytest.mark.parametrize("kw,code,text", [
    (dict(rows=-1), INVALID, "rows"), (dict(in_type=2), UNSUPPORTED, "F32 or F16"), (dict(q_type=30), UNSUPPORTED, "F32"),
    (dict(rope_dim=3), INVALID, "RoPE"), (dict(rope_dim=66), INVALID, "RoPE"), (dict(rope_dim=-2), INVALID, "RoPE"),
    (dict(rope_dim=64), INVALID, "table"), (dict(nseq=0), INVALID, "nseq"), (dict(pages_per_seq=0), INVALID, "nseq"),
    (dict(rows=3), INVALID, "seq_dev"), (dict(rows=2, nseq=2, ldk=127), INVALID, "strides"),
    (dict(rows=2, nseq=2, ldqo=255), INVALID, "strides"), (dict(pages_per_seq=1 << 28), INVALID, "too long")])
def test_append_refused(kw, code, text):
    a = dict(rows=1, heads=4, nseq=1, pages_per_seq=2)
    a.update(kw)
    plan = _pages().append_plan(**a)
    _refused(code, text, lambda: plan(PTR, PTR, PTR, PTR + 16, PTR, PTR))


def test_append_null_and_in_place_refused():
    plan = _pages().append_plan(1, 4, 1, 2)
    for i in (0, 1, 2, 3, 4, 5):
        ptrs = [PTR, PTR + 16, PTR + 32, PTR + 48, PTR + 64, PTR + 80]
        ptrs[i] = 0
        _refused(INVALID, "null", lambda: plan(*ptrs))
    other = _pages().append_plan(1, 4, 1, 2, in_type=0, q_type=1)  # FP32 rotated in place into binary16
    _refused(INVALID, "in place", lambda: other(PTR, PTR + 16, PTR + 32, PTR, PTR, PTR))
    assert _pages().append_plan(0, 4, 1, 2)(0, 0, 0, 0, 0, 0) is None  # no rows: nothing to do


@pytest.mark.parametrize("kw,code,text", [
    (dict(heads=5), INVALID, "multiple"), (dict(heads=0), INVALID, "multiple"), (dict(heads=18), UNSUPPORTED, "at most 8"),
    (dict(type=8), UNSUPPORTED, "F32 or F16"), (dict(max_len=33), INVALID, "must not exceed"),
    (dict(max_len=-1), INVALID, "negative"), (dict(max_private=-2), INVALID, "negative"),
    (dict(groups=1), INVALID, "max_group_rows"), (dict(groups=1, max_group_rows=2), INVALID, "max_group_rows"),
    (dict(groups=1, max_group_rows=1, max_shared=33), INVALID, "must not exceed"), (dict(rows=-1), INVALID, "rows"),
    (dict(scale=-0.5), INVALID, "scale"), (dict(scale=float("nan")), INVALID, "scale")])
def test_attention_bounds_refused(kw, code, text):
    a = dict(rows=1, heads=4, nseq=1, pages_per_seq=2, max_len=32)
    a.update(kw)
    _refused(code, text, lambda: _pages().attention_plan(**a))


def test_attention_pointers_and_workspace_refused():
    plan = _pages(num_pages=100).attention_plan(1, 4, 1, 100, 1600)
    assert plan.workspace_bytes > 0  # several items per row
    _refused(INVALID, "bytes of workspace", lambda: plan(PTR, PTR, PTR, PTR))
    _refused(INVALID, "16-byte aligned", lambda: plan(PTR, PTR, PTR, PTR, workspace=PTR + 4))
    plan.args.workspace_bytes -= 1
    _refused(INVALID, "bytes of workspace", lambda: plan(PTR, PTR, PTR, PTR, workspace=PTR))
    one = _pages().attention_plan(1, 4, 1, 2, 32)
    assert one.workspace_bytes == 0
    for i in range(4):
        ptrs = [PTR] * 4
        ptrs[i] = 0
        _refused(INVALID, "null", lambda: one(*ptrs))
    grouped = _pages().attention_plan(2, 4, 2, 2, 32, groups=1, max_group_rows=2, max_shared=16)
    _refused(INVALID, "null", lambda: grouped(PTR, PTR, PTR, PTR, workspace=PTR))
    _refused(INVALID, "seq_dev", lambda: _pages().attention_plan(3, 4, 1, 2, 32)(PTR, PTR, PTR, PTR))
    narrow = _pages().attention_plan(2, 4, 2, 2, 32, ldo=255)
    _refused(INVALID, "strides", lambda: narrow(PTR, PTR, PTR, PTR))


def test_probs_and_verify_refused():
    from laicompute_b200.serving import logits_probs, verify_drafts
    _refused(INVALID, "vocab", lambda: logits_probs(1, 0, PTR, PTR, PTR))
    _refused(INVALID, "null", lambda: logits_probs(1, 10, PTR, 0, PTR))
    _refused(INVALID, "strides", lambda: logits_probs(2, 10, PTR, PTR, PTR + 16, ld_probs=9))
    _refused(INVALID, "in place", lambda: logits_probs(2, 10, PTR, PTR, PTR, ld_logits=10, ld_probs=12))
    logits_probs(0, 10, 0, 0, 0)
    ok = [PTR] * 8
    _refused(UNSUPPORTED, "at most 64", lambda: verify_drafts(1, 65, 10, *ok))
    _refused(INVALID, "max_draft", lambda: verify_drafts(1, -1, 10, *ok))
    _refused(INVALID, "vocab", lambda: verify_drafts(1, 2, 0, *ok))
    _refused(INVALID, "strides", lambda: verify_drafts(1, 2, 10, *ok, ld_target=9))
    _refused(INVALID, "strides", lambda: verify_drafts(1, 2, 10, *ok, ld_draft=9))
    for i in (0, 2, 3, 4, 5, 6, 7):  # 1: the draft's probabilities may be absent
        ptrs = list(ok)
        ptrs[i] = 0
        _refused(INVALID, "null", lambda: verify_drafts(1, 2, 10, *ptrs))
    verify_drafts(0, 2, 10, *([0] * 8))


@pytest.fixture(scope="module")
def host_rules(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("paged") / "paged_check")
    subprocess.run(["nvcc", "-std=c++17", "-O1", "-gencode", "arch=compute_100a,code=sm_100a", f"-I{ROOT}/include",
                    f"-I{ROOT}/laicompute_b200/csrc", os.path.join(ROOT, "tests", "host", "paged_check.cu"), "-o", exe],
                   check=True, capture_output=True)

    def ask(*lines):
        out = subprocess.run([exe], input="\n".join(" ".join(map(str, q)) for q in lines) + "\n", text=True,
                             capture_output=True, check=True).stdout
        return [tuple(map(int, x.split())) for x in out.splitlines()]
    return ask


def test_place_rules(host_rules):
    table = [3, -1, 7, 0, 2, 1]  # two sequences of three pages, five pages in the pool

    def place(seq, pos, positions=1 << 30):
        return ("place", seq, pos, 2, 3, 4, 5, positions, *table)
    got = host_rules(place(0, 0), place(0, 15), place(0, 16), place(0, 32), place(0, 47), place(0, 48), place(1, 0),
                     place(1, 47), place(2, 0), place(-1, 0), place(0, -1), place(1, 20, 20), place(1, 20, 21),
                     place(1, 2147483647))
    assert got == [(3, 0), (3, 0), (-1, BAD_PAGE), (-1, BAD_PAGE), (-1, BAD_PAGE), (-1, BAD_POS), (0, 0), (1, 0),
                   (-1, BAD_SEQ), (-1, BAD_SEQ), (-1, BAD_POS), (-1, BAD_POS), (2, 0), (-1, BAD_POS)]


def test_row_rules(host_rules):
    def row(r, n, shared=0, seq=None, max_len=40, nseq=2):
        return ("row", r, 2, nseq, 3, 4, max_len, shared, int(seq is not None), *n, *(seq or ()))
    got = host_rules(row(0, (5, 9)), row(1, (5, 9)), row(0, (0, 0)), row(0, (-7, 0)), row(0, (41, 0)),
                     row(0, (100, 0), max_len=100), row(0, (5, 5), shared=3), row(0, (2, 5), shared=3),
                     row(0, (5, 5), seq=(1, 0)), row(0, (5, 5), seq=(2, 0)), row(1, (5, 5), seq=(0, -1), shared=4),
                     row(1, (5, 5), nseq=1))
    assert got == [(5, 0, 0, 0), (9, 0, 1, 0), (0, 0, 0, 0), (-1, 0, -1, 0), (40, 0, 0, BAD_POS), (48, 0, 0, BAD_POS),
                   (5, 3, 0, 0), (2, 2, 0, 0), (5, 0, 1, 0), (0, 0, -1, BAD_SEQ), (0, 0, -1, BAD_SEQ),
                   (0, 0, -1, BAD_SEQ)]


def test_group_rules(host_rules):
    def group(g, start, ln, rows=6, nseq=6, max_rows=4, max_shared=30):
        return ("group", g, rows, len(ln), nseq, 3, 4, max_rows, max_shared, *start, *ln)
    got = host_rules(group(0, (0, 4, 6), (10, 20)), group(1, (0, 4, 6), (10, 20)), group(0, (0, 5, 6), (10, 20)),
                     group(0, (3, 2, 6), (10, 20)), group(1, (0, 4, 7), (10, 20)), group(0, (-1, 2, 6), (10, 20)),
                     group(0, (0, 4, 6), (31, 20)), group(0, (0, 4, 6), (-3, 20)), group(0, (2, 2, 6), (9, 20)))
    assert got == [(1, 0, 4, 10, 0), (1, 4, 6, 20, 0), (0, 0, 5, 0, BAD_GROUP), (0, 3, 2, 0, BAD_GROUP),
                   (0, 4, 7, 0, BAD_GROUP), (0, -1, 2, 0, BAD_GROUP), (1, 0, 4, 30, BAD_POS), (1, 0, 4, 0, 0),
                   (1, 2, 2, 0, 0)]
