"""Groups whose first rows are padding or see nothing: which row of the page table they are read through, on the host, and the
outputs on the GPU."""
import os
import subprocess

import pytest

from conftest import ROOT

BAD_SEQ = 1


def test_the_first_row_that_sees_something_leads(tmp_path):
    exe = str(tmp_path / "group_check")
    subprocess.run(["nvcc", "-std=c++17", "-O1", "-gencode", "arch=compute_100a,code=sm_100a", f"-I{ROOT}/include",
                    f"-I{ROOT}/laicompute_b200/csrc", os.path.join(ROOT, "tests", "host", "group_check.cu"), "-o", exe],
                   check=True, capture_output=True)
    cases = [((0, 3), 4, (5, 5, 5, 5), None, (0, 0)), ((1, 3), 4, (5, 5, 5, 5), (3, 2, 1, 0), (2, 0)),
             ((0, 3), 4, (-1, -1, 5, 5), (-1, 99, 2, 0), (2, 0)), ((0, 3), 4, (-1, 0, 5, 5), (-1, 3, 2, 0), (2, 0)), ((0, 2), 4, (0, 0, 5, 5), (1, 3, 2, 0), (0, 0)),
             ((0, 2), 4, (-1, -3, 5, 5), (-1, 99, 2, 0), (0, 0)), ((0, 3), 2, (-1, 5, 5, 5), (0, 2, 1, 1), (0, BAD_SEQ)),
             ((1, 4), 4, (5, -1, -1, 7), None, (3, 0)), ((0, 1), 4, (3, 3, 3, 3), (-1, 0, 0, 0), (0, BAD_SEQ))]
    lines = [" ".join(map(str, (*r, 4, nseq, int(seq is not None), *ln, *(seq or ())))) for r, nseq, ln, seq, _ in cases]
    out = subprocess.run([exe], input="\n".join(lines) + "\n", text=True, capture_output=True, check=True).stdout
    assert [tuple(map(int, x.split())) for x in out.splitlines()] == [c[-1] for c in cases]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("heads,hkv,d,nrows", [(8, 2, 64, 4), (4, 2, 32, 12), (8, 2, 128, 12), (8, 1, 64, 20)])
def test_padding_rows_lead_a_group(heads, hkv, d, nrows, dtype):
    """One, or all but one, of a group's rows are padding at its head and name no sequence of the table; narrow
    groups and wide ones, with and without positions of their own."""
    import torch

    from serving_util import TORCH, Cache, attend, close, reference
    shared = 300
    cache = Cache([400] + [shared + 20] * nrows + [50], hkv, d, 32, seed=nrows, shared=[(list(range(1, nrows + 1)), shared)])
    q = (torch.randn(nrows + 1, heads * d, generator=torch.Generator().manual_seed(2)) * 1.5).to(TORCH[dtype]).cuda()
    for pads, extra in ((1, 20), (1, 0), (nrows - 1, 20), (nrows, 0)):
        lens = [-1] * pads + [shared + extra] * (nrows - pads) + [50]
        seqs = [-1] * pads + list(range(pads + 1, nrows + 1)) + [nrows + 1]
        out = attend(cache, q, lens, seqs=seqs, groups=([0, nrows], [shared]))
        cache.pages().check()
        rows = sorted({pads, nrows - 1, nrows}) if pads < nrows else [nrows]
        ref, tol = reference(cache, q[rows], [lens[r] for r in rows], [seqs[r] for r in rows])
        close(out[rows], ref, tol)
        assert torch.all(out[:pads] == 7.0)
        # the same rows seeing nothing, of a sequence that holds nothing
        table = cache.table.clone()
        cache.table[0] = -1
        out = attend(cache, q, [0] * pads + lens[pads:], seqs=[0] * pads + seqs[pads:], groups=([0, nrows], [shared]))
        cache.pages().check()
        close(out[rows], ref, tol)
        assert not out[:pads].any()
        cache.table = table
