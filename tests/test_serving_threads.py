"""One plan called by several threads at once: every call hands the library its own pointers (no GPU: the C entry
is a stand-in that reads the arguments it is given while the other thread is inside its own call)."""
import threading

import pytest

PTR = 4096


def _plans():
    from laicompute_b200.serving import KvPages
    pages = KvPages(PTR, PTR, 4, 2, 16, 64, err=PTR)
    return {"append": (pages.append_plan(1, 4, 1, 2), ("q_dev", "k_dev", "v_dev", "q_out_dev", "pos_dev", "page_table_dev",
                                                       "rope_dev", "seq_dev")),
            "attention": (pages.attention_plan(1, 4, 1, 2, 32),
                          ("q_dev", "out_dev", "len_dev", "page_table_dev", "workspace_dev", "seq_dev", "group_rows_dev",
                           "group_len_dev"))}


@pytest.mark.parametrize("kind", ["append", "attention"])
def test_calls_at_once_keep_their_pointers(kind):
    plan, fields = _plans()[kind]
    inside, seen = threading.Barrier(2, timeout=30), {}

    def entry(desc, args, stream):
        inside.wait()  # both threads have filled their arguments
        seen[stream] = [getattr(args._obj, f) for f in fields]
        inside.wait()
        return 0
    plan._call = entry
    mine = {i: [PTR * (10 * i + k + 1) for k in range(len(fields))] for i in (1, 2)}
    threads = [threading.Thread(target=lambda i=i: plan(*mine[i], stream=i)) for i in (1, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert seen == mine


@pytest.mark.parametrize("kind", ["append", "attention"])
def test_a_call_takes_the_plan_as_it_stands(kind):
    """The shape in plan.args is the call's, also after a change; a call leaves no pointer behind."""
    plan, fields = _plans()[kind]
    got = []
    plan._call = lambda desc, args, stream: got.append((args._obj.rows, args._obj.heads)) or 0
    plan(*[PTR] * len(fields))
    plan.args.rows = 3
    plan(*[PTR] * len(fields))
    assert got == [(1, 4), (3, 4)] and not any(getattr(plan.args, f) for f in fields)
