"""Builders and 64-bit reference forms for the serving operators' tests."""
import math
import random

import torch

F32, F16 = 0, 1
TORCH = {F32: torch.float32, F16: torch.float16}
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11}  # half a unit in the last place, relative


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Cache:
    """Sequences of given lengths in shuffled pages of one pool; every place no sequence owns holds NaN."""

    def __init__(self, lens, kv_heads, head_dim, page, seed=0, shared=None, spare=2, room=0):
        """shared: list of (sequences, positions): those sequences name the same whole pages for their first
        positions (and equal copies of the partly filled one). room: unused page table entries per row."""
        g = torch.Generator().manual_seed(seed)
        rng = random.Random(seed)
        need = [(n + page - 1) // page for n in lens]
        first = {}
        for seqs, n in shared or ():
            for s in seqs:
                first[s] = (seqs[0], n)
        rows, used = [], 0
        for s, k in enumerate(need):
            lead, n = first.get(s, (s, 0))
            row = list(rows[lead][:min(n // page, k)]) if lead != s else []
            while len(row) < k:
                row.append(used)
                used += 1
            rows.append(row)
        self.num_pages = used + spare
        ids = list(range(self.num_pages))
        rng.shuffle(ids)
        self.rows = [[ids[p] for p in r] for r in rows]
        self.per_seq = max(1, max(len(r) for r in rows)) + room
        self.lens, self.page, self.kv_heads, self.head_dim = list(lens), page, kv_heads, head_dim
        shape = (self.num_pages, kv_heads, page, head_dim)
        self.k = torch.full(shape, float("nan"), dtype=torch.float16)
        self.v = torch.full(shape, float("nan"), dtype=torch.float16)
        self.seq_k, self.seq_v = [], []
        for s, n in enumerate(lens):
            kk = torch.randn(n, kv_heads, head_dim, generator=g).half()
            vv = torch.randn(n, kv_heads, head_dim, generator=g).half()
            lead, m = first.get(s, (s, 0))
            if lead != s:
                m = min(m, n)
                kk[:m], vv[:m] = self.seq_k[lead][:m], self.seq_v[lead][:m]
            self.seq_k.append(kk)
            self.seq_v.append(vv)
            for t0 in range(0, n, page):
                t1 = min(n, t0 + page)
                p = self.rows[s][t0 // page]
                self.k[p, :, :t1 - t0] = kk[t0:t1].transpose(0, 1)
                self.v[p, :, :t1 - t0] = vv[t0:t1].transpose(0, 1)
        self.k, self.v = self.k.cuda(), self.v.cuda()
        self.err = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.table = ints([r + [-1] * (self.per_seq - len(r)) for r in self.rows])

    def pages(self):
        from laicompute_b200.serving import KvPages
        return KvPages(self.k.data_ptr(), self.v.data_ptr(), self.num_pages, self.kv_heads, self.page, self.head_dim,
                       err=self.err.data_ptr())


def attend(cache, q, lens, seqs=None, groups=None, out=None, ldq=None, ldo=None, scale=0.0, bounds=None, stream=0,
           workspace=None):
    """One laic_kv_attention call. q [rows][heads * dim] (or a view with row stride ldq); groups: (starts, lens)."""
    rows = len(lens)
    t = F32 if q.dtype == torch.float32 else F16
    heads = q.shape[1] // cache.head_dim
    if out is None:
        out = torch.full((rows, q.shape[1]), 7.0, dtype=q.dtype, device="cuda")
    kw = dict(type=t, ldq=ldq or q.stride(0), ldo=ldo or out.stride(0), scale=scale)
    ptrs = {}
    keep = [ints(lens), ints(seqs) if seqs is not None else None]
    if groups:
        starts, shared = groups
        member = {r: g for g in range(len(shared)) for r in range(starts[g], starts[g + 1])}
        private = max([max(0, n - (shared[member[r]] if r in member else 0)) for r, n in enumerate(lens)] + [0])
        kw.update(groups=len(shared), max_group_rows=max(max(b - a for a, b in zip(starts, starts[1:])), 1),
                  max_shared=max(shared), max_private=private)
        keep += [ints(starts), ints(shared)]
        ptrs = dict(group_rows=keep[2].data_ptr(), group_len=keep[3].data_ptr())
    kw.update(bounds or {})
    max_len = kw.pop("max_len", max(max(lens), 0))
    plan = cache.pages().attention_plan(rows, heads, cache.table.shape[0], cache.per_seq, max_len, **kw)
    if workspace is None:
        workspace = torch.full((max(16, plan.workspace_bytes),), 255, dtype=torch.uint8, device="cuda")  # NaNs
    plan(q.data_ptr(), out.data_ptr(), keep[0].data_ptr(), cache.table.data_ptr(), workspace=workspace.data_ptr(),
         seq=keep[1].data_ptr() if keep[1] is not None else 0, stream=stream, **ptrs)
    attend.keep = (keep, workspace, plan)
    return out


def reference(cache, q, lens, seqs=None, scale=0.0):
    """The definition in 64 bits, and per element the error bound of the kernels' arithmetic."""
    d, hkv = cache.head_dim, cache.kv_heads
    heads = q.shape[1] // d
    G = heads // hkv
    sc = scale or 1.0 / math.sqrt(d)
    qd = q.double().cpu().view(len(lens), heads, d)
    out = torch.zeros(len(lens), heads, d, dtype=torch.float64)
    tol = torch.zeros(len(lens), heads, d, dtype=torch.float64)
    asc = abs(sc)
    hs = HALF_STEP[F32 if q.dtype == torch.float32 else F16]
    for r, n in enumerate(lens):
        if n <= 0:
            continue
        s = seqs[r] if seqs is not None else r
        for h in range(heads):
            k = cache.seq_k[s][:n, h // G].double()
            v = cache.seq_v[s][:n, h // G].double()
            x = (k @ qd[r, h]) * sc
            p = torch.softmax(x, dim=0)
            out[r, h] = p @ v
            # Score error: q to 2^-22 of its row's maximum; the FP32 sum of d products in d / 16 steps of
            # the tensor cores, which may truncate (2^-23 of the magnitudes each), taken as d / 8 roundings;
            # the scaling to base 2, the difference to the maximum and 2^x of it, 2^-22 relative each.
            mag = (k.abs().sum(dim=1) * qd[r, h].abs().max()).max().item() * asc
            ds = mag * (2.0 ** -22 + (d / 8) * 2.0 ** -23) + 3 * x.abs().max().item() * 2.0 ** -23
            # Weights relative to their sum: the score error twice (numerator and sum), the exponential, the
            # hi + lo split, and sums of n / 16 steps plus the joins of 4 warps and up to 64 items.
            dw = 2 * ds + 2.0 ** -21 + (n / 16 + 72) * 2.0 ** -23
            if q.dtype == torch.float16:
                dw += 2.0 ** -11  # binary16 weights
            tol[r, h] = dw * (p[:, None] * v.abs()).sum(dim=0) + hs * out[r, h].abs() + 2.0 ** -25
    return out.flatten(1), tol.flatten(1)


def close(out, ref, tol):
    err = (out.double().cpu() - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (int(bad.sum()), float((err / tol).max()), bad.nonzero()[:4].tolist())
