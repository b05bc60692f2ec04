"""Far bounds of an attention call (no GPU): what would leave the kernels' 32-bit positions is refused."""
import pytest

from test_serving_refusals import UNSUPPORTED, _pages, _refused

MOST = 1073000000


@pytest.mark.parametrize("page", [16, 64, 256])
def test_far_bounds_are_refused_or_planned(page):
    per_seq = (2 ** 31 - 1) // page
    far = per_seq * page
    pages = _pages(page_size=page, kv_heads=1)
    grouped = dict(groups=1, max_group_rows=1)
    for kw in (dict(max_len=far), dict(max_len=MOST + 1), dict(max_len=100, max_shared=far, **grouped),
               dict(max_len=far, max_shared=64, max_private=10, **grouped)):
        _refused(UNSUPPORTED, "1,073,000,000", lambda: pages.attention_plan(1, 1, 1, per_seq, **kw))
    for kw in (dict(max_len=MOST), dict(max_len=MOST, max_shared=MOST, **grouped), dict(max_len=MOST, max_shared=64, **grouped)):
        plan = pages.attention_plan(1, 1, 1, per_seq, **kw)
        # a partial of 64 + 2 floats for every split of each bound: neither negative nor wrapped
        most = 2 * (MOST // 128 + 1) * 66 * 4
        assert 0 < plan.workspace_bytes <= most


def test_positions_of_far_bounds_stay_within_an_int():
    """The largest start of a private split, as the kernel adds it up, and its end."""
    i32 = lambda x: (x + 2 ** 31) % 2 ** 32 - 2 ** 31  # noqa: E731
    for split in (128, 1024, 2048 * 8):
        last = (MOST + split - 1) // split - 1
        for shared in (0, 1, MOST):
            assert i32(shared + last * split) >= 0 and i32(shared + MOST) >= 0
        assert i32(MOST + split) >= 0 and i32(MOST + split - 1) >= 0


@pytest.mark.parametrize("rows,heads", [(1 << 29, 8), (1 << 28, 8), ((1 << 28) + 1, 8), ((1 << 31) - 1, 2)])
def test_too_many_rows_are_refused(rows, heads):
    """More (row, head) pairs than an int holds, with a group of them all (whose columns wrapped to zero)."""
    for kw in (dict(groups=1, max_group_rows=rows, max_shared=16), dict(groups=1, max_group_rows=rows, max_shared=16, max_private=0),
               {}):
        _refused(UNSUPPORTED, "too many", lambda: _pages(kv_heads=1).attention_plan(rows, heads, rows, 2, 32, **kw))


def test_the_most_rows_that_are_planned():
    rows = ((1 << 31) - 1) // 8
    plan = _pages(kv_heads=1).attention_plan(rows, 8, rows, 2, 32, groups=1, max_group_rows=rows, max_shared=16, max_private=0)
    assert plan.workspace_bytes == rows * 8 * (64 * 4 + 8)  # one shared item per row and head


@pytest.mark.parametrize("vocab", [(1 << 30) + 1, (1 << 31) - 1])
def test_vocabularies_that_leave_an_int_are_refused(vocab):
    """A row's loops step past its end: near 2^31 they would have wrapped to addresses before it."""
    from laicompute_b200.serving import logits_probs, verify_drafts
    _refused(UNSUPPORTED, "2^30", lambda: logits_probs(1, vocab, 4096, 4096, 4096))
    _refused(UNSUPPORTED, "2^30", lambda: verify_drafts(1, 2, vocab, *[4096] * 8))
    logits_probs(0, 1 << 30, 0, 0, 0)
    verify_drafts(0, 2, 1 << 30, *[0] * 8)
