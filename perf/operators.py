"""The serving operators on real work: the paged KV append with rotation, attention over the pages
(shared prefixes read once), probabilities of logits rows and the verification of drafted tokens.

``run`` computes them with elementary torch operations (``own`` false) or with the framework's kernels
(``own`` true); ``exact`` gives the same outputs from the definitions in 64 bits. Shapes are those of the
135M, 1B and 8B decoders this repository is benchmarked on, or generic.
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16}


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------

def listed():
    return [
        # one decode step of 64 sequences of the 135M shape: the smallest append
        dict(name="append_step_135m", op="append", heads=9, kv_heads=3, head_dim=64, page=16, in_type="f32",
             q_type="f32", seqs=64, rows_each=1, ctx_lo=1, ctx_hi=1900, shape=11),
        # four long prompts of odd lengths entered at once on the 8B shape, binary16 activations: the largest append
        dict(name="append_prompts_8b", op="append", heads=32, kv_heads=8, head_dim=128, page=64, in_type="f16",
             q_type="f16", seqs=4, rows_each=2047, ctx_lo=1, ctx_hi=700, shape=12),
        # one sequence of the 135M shape a hundred tokens in: launch latency
        dict(name="attn_one_135m", op="attention", mode="batch", heads=9, kv_heads=3, head_dim=64, page=16, type="f32",
             seqs=1, len_lo=101, len_hi=101, shape=21),
        # a decode step of 64 unrelated sequences of the 8B shape with ragged contexts: HBM
        dict(name="attn_step_8b", op="attention", mode="batch", heads=32, kv_heads=8, head_dim=128, page=64, type="f32",
             seqs=64, len_lo=1024, len_hi=8192, shape=22),
        # 64 chats behind one 4,101-token system prompt, up to 512 tokens of their own each
        dict(name="attn_prefix_8b", op="attention", mode="prefix", heads=32, kv_heads=8, head_dim=128, page=64,
             type="f32", seqs=64, groups=1, shared=4101, len_lo=1, len_hi=512, shape=23),
        # 64 samples of few-shot prompts: three shared prefixes of 8,000 tokens, binary16 activations
        dict(name="attn_prefixes_8b_f16", op="attention", mode="prefix", heads=32, kv_heads=8, head_dim=128, page=16,
             type="f16", seqs=64, groups=3, shared=8000, len_lo=1, len_hi=300, shape=24),
        # four drafted tokens and the one before them for 8 sequences of the 1B shape: five rows share a context
        dict(name="attn_draft_1b", op="attention", mode="draft", heads=32, kv_heads=8, head_dim=64, page=32, type="f32",
             seqs=8, drafted=4, len_lo=500, len_hi=8000, shape=25),
        # one prefill pass: 512 prompt tokens of the 8B shape behind 1,537 cached ones, causal
        dict(name="attn_prompt_8b", op="attention", mode="prompt", heads=32, kv_heads=8, head_dim=128, page=64,
             type="f16", seqs=1, rows_each=512, len_lo=1537, len_hi=1537, shape=26),
        # the logits of five rows of one 135M sequence (four drafted tokens and the one before)
        dict(name="probs_one_135m", op="probs", rows=5, vocab=49152, greedy=0.0, shape=31),
        # the logits of a verified batch of the 8B vocabulary, a quarter of the rows greedy
        dict(name="probs_batch_8b", op="probs", rows=320, vocab=128256, greedy=0.25, shape=32),
        # one sequence, four tokens drafted without probabilities (looked up in the prompt)
        dict(name="verify_one_135m", op="verify", seqs=1, drafted=4, vocab=49152, draft="point", ragged=False, shape=41),
        # 64 sequences with up to seven tokens of a small draft model
        dict(name="verify_batch_8b", op="verify", seqs=64, drafted=7, vocab=128256, draft="probs", ragged=True,
             shape=42),
    ]


HEADS = [(9, 3, 64), (32, 8, 64), (32, 8, 128), (4, 2, 32), (8, 1, 128), (6, 6, 64), (10, 2, 128)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "attention", "probs", "verify"])
    h, hkv, d = rng.choice(HEADS)
    shape = rng.randrange(1 << 30)
    page = rng.choice([16, 32, 64, 128, 256])
    if op == "append":
        seqs = _log(rng, 1, 64)
        each = _log(rng, 1, max(2, 8000 // seqs))
        return dict(op=op, heads=h, kv_heads=hkv, head_dim=d, page=page, in_type=rng.choice(["f32", "f16"]),
                    q_type=rng.choice(["f32", "f16"]), seqs=seqs, rows_each=each, ctx_lo=1, ctx_hi=_log(rng, 2, 3000),
                    shape=shape)
    if op == "attention":
        mode = rng.choice(["batch", "prefix", "draft", "prompt"])
        c = dict(op=op, mode=mode, heads=h, kv_heads=hkv, head_dim=d, page=page, type=rng.choice(["f32", "f16"]),
                 shape=shape)
        if mode == "batch":
            hi = _log(rng, 1, 8000)
            c.update(seqs=_log(rng, 1, min(64, 220000 // hi)), len_lo=max(1, hi // rng.choice([1, 4, 50])), len_hi=hi)
        elif mode == "prefix":
            seqs = _log(rng, 2, 64)
            c.update(seqs=seqs, groups=rng.randint(1, min(4, seqs)), shared=_log(rng, 1, 8000), len_lo=1,
                     len_hi=_log(rng, 2, 600))
        elif mode == "draft":
            c.update(seqs=_log(rng, 1, 12), drafted=rng.randint(1, 7), len_lo=1, len_hi=_log(rng, 2, 8000))
        else:
            ctx = _log(rng, 1, 1600)
            c.update(seqs=1, rows_each=_log(rng, 2, 512), len_lo=ctx, len_hi=ctx)
        return c
    vocab = rng.choice([49152, 128256, _log(rng, 50, 128000)])
    if op == "probs":
        return dict(op=op, rows=_log(rng, 1, 300), vocab=vocab, greedy=rng.choice([0.0, 0.3, 1.0]), shape=shape)
    return dict(op=op, seqs=_log(rng, 1, 64), drafted=rng.randint(1, 7), vocab=vocab,
                draft=rng.choice(["point", "probs"]), ragged=rng.random() < 0.5, shape=shape)


# ------------------------------------------------------------------------------------------------
# shapes that follow from a case: sequence lengths, rows, groups
# ------------------------------------------------------------------------------------------------

def _plan(case):
    """Per sequence its cached positions; per row its sequence and length; the groups."""
    rng = random.Random(case["shape"])
    if case["op"] == "append":
        start = [_log(rng, case["ctx_lo"], case["ctx_hi"]) for _ in range(case["seqs"])]
        n = case["rows_each"]
        return dict(total=[s + n for s in start], seq=[i for i in range(case["seqs"]) for _ in range(n)],
                    pos=[s + j for s in start for j in range(n)])
    own_len = [_log(rng, case["len_lo"], case["len_hi"]) for _ in range(case["seqs"])]
    mode, n = case["mode"], case["seqs"]
    if mode == "batch":
        return dict(total=own_len, seq=list(range(n)), lens=own_len, groups=None, prefix=[0] * n)
    if mode == "prefix":
        shared = case["shared"]
        cuts = sorted(rng.sample(range(1, n), case["groups"] - 1)) if case["groups"] > 1 else []
        starts = [0] + cuts + [n]
        total = [shared + m for m in own_len]
        return dict(total=total, seq=list(range(n)), lens=total, groups=(starts, [shared] * case["groups"]),
                    prefix=[shared] * n)
    rows = case["drafted"] + 1 if mode == "draft" else case["rows_each"]
    total = [m + rows for m in own_len]
    return dict(total=total, seq=[i for i in range(n) for _ in range(rows)],
                lens=[m + j + 1 for m in own_len for j in range(rows)],
                groups=([i * rows for i in range(n + 1)], total), prefix=[0] * n)


def _pages(case, plan):
    """Page table (shared prefixes name the same whole pages, everything else its own) and the pool's size."""
    rng = random.Random(case["shape"] + 1)
    ps = case["page"]
    per_seq = max((t + ps - 1) // ps for t in plan["total"])
    table, used = [], 0
    group_of = {}
    if plan.get("groups") and case["mode"] == "prefix":
        starts = plan["groups"][0]
        for g in range(len(starts) - 1):
            for i in range(starts[g], starts[g + 1]):
                group_of[i] = starts[g]
    copies = []  # (from page, to page): the shared prefix's last, partly filled page
    for i, t in enumerate(plan["total"]):
        need = (t + ps - 1) // ps
        first = group_of.get(i, i)
        whole = case["shared"] // ps if first != i else 0
        row = table[first][:whole] if first != i else []
        while len(row) < need:
            row.append(used)
            used += 1
        if first != i and case["shared"] % ps:
            copies.append((table[first][whole], row[whole]))
        table.append(row)
    ids = list(range(used + 2))
    rng.shuffle(ids)
    table = [[ids[p] for p in row] + [-1] * (per_seq - len(row)) for row in table]
    return table, used + 2, per_seq, [(ids[a], ids[b]) for a, b in copies]


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------

def _rope_table(positions, rope_dim):
    ang = torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * (
        500000.0 ** (-torch.arange(0, rope_dim, 2, dtype=torch.float64, device=DEV) / rope_dim))[None, :]
    return torch.stack([torch.cos(ang), torch.sin(ang)], dim=-1).float().contiguous()


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _inputs(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 1000003 + case["shape"])

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)

    op = case["op"]
    st = dict(case=case)
    if op in ("append", "attention"):
        h, hkv, d, ps = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
        plan = _plan(case)
        table, num_pages, per_seq, copies = _pages(case, plan)
        st.update(plan=plan, table=_ints(table), num_pages=num_pages, per_seq=per_seq, seq=_ints(plan["seq"]),
                  err=torch.zeros(1, dtype=torch.int32, device=DEV))
        rows = len(plan["seq"])
        shape = (num_pages, hkv, ps, d)
        if op == "append":
            t = TYPES[case["in_type"]]
            # the fused projection's rows: q, k and v side by side
            st["qkv"] = randn(rows, (h + 2 * hkv) * d).to(t)
            st["q_out"] = torch.zeros(rows, h * d, dtype=TYPES[case["q_type"]], device=DEV)
            st["k"] = torch.zeros(shape, dtype=torch.float16, device=DEV)
            st["v"] = torch.zeros(shape, dtype=torch.float16, device=DEV)
            st["pos"] = _ints(plan["pos"])
            st["rope"] = _rope_table(max(plan["total"]), d)
        else:
            st["k"] = randn(*shape, dtype=torch.float16)
            st["v"] = randn(*shape, dtype=torch.float16)
            for a, b in copies:
                st["k"][b] = st["k"][a]
                st["v"][b] = st["v"][a]
            st["q"] = (randn(rows, h * d) * 1.5).to(TYPES[case["type"]])
            st["out"] = torch.zeros(rows, h * d, dtype=TYPES[case["type"]], device=DEV)
            st["lens"] = _ints(plan["lens"])
            if plan["groups"]:
                st["group_rows"], st["group_len"] = _ints(plan["groups"][0]), _ints(plan["groups"][1])
        return st
    rng = random.Random(case["shape"])
    v = case["vocab"]
    if op == "probs":
        st["logits"] = randn(case["rows"], v) * 3.0
        temp = [0.0 if rng.random() < case["greedy"] else rng.uniform(0.5, 1.3) for _ in range(case["rows"])]
        st["temperature"] = torch.tensor(temp, dtype=torch.float32, device=DEV)
        st["probs"] = torch.zeros(case["rows"], v, device=DEV)
        return st
    n, m = case["seqs"], case["drafted"]
    base = randn(n * (m + 1), v) * 2.5
    st["target"] = torch.softmax(base, dim=-1)
    drafted = base.view(n, m + 1, v)[:, :m].reshape(n * m, v) + 0.7 * randn(n * m, v)
    dp = torch.softmax(drafted, dim=-1)
    del drafted, base
    st["ids"] = torch.multinomial(dp, 1, generator=g).to(torch.int32).view(n, m).contiguous()
    if case["draft"] == "probs":
        st["draft"] = dp
    else:  # a lookup drafts what the text repeats: mostly the target's favourites
        st["draft"] = None
        top = st["target"].view(n, m + 1, v)[:, :m].argmax(dim=-1).to(torch.int32)
        keep = torch.rand(n, m, generator=g, device=DEV) < 0.9
        st["ids"] = torch.where(keep, top, st["ids"]).contiguous()
    st["n_draft"] = _ints([rng.randint(0, m) if case["ragged"] else m for _ in range(n)])
    st["accept_u"] = torch.rand(n, m, generator=g, device=DEV)
    st["sample_u"] = torch.rand(n, generator=g, device=DEV)
    st["out_ids"] = torch.zeros(n, m + 1, dtype=torch.int32, device=DEV)
    st["out_n"] = torch.zeros(n, dtype=torch.int32, device=DEV)
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    if not own or case["op"] in ("probs", "verify"):
        return st
    from laicompute_b200 import gguf
    from laicompute_b200.serving import KvPages
    code = {"f32": gguf.F32, "f16": gguf.F16}
    h, hkv, d = case["heads"], case["kv_heads"], case["head_dim"]
    st["pages"] = KvPages(st["k"].data_ptr(), st["v"].data_ptr(), st["num_pages"], hkv, case["page"], d,
                          err=st["err"].data_ptr())
    rows, nseq = len(st["plan"]["seq"]), case["seqs"]
    if case["op"] == "append":
        ld = (h + 2 * hkv) * d
        st["call"] = st["pages"].append_plan(rows, h, nseq, st["per_seq"], in_type=code[case["in_type"]],
                                             q_type=code[case["q_type"]], ldq=ld, ldk=ld, ldv=ld, rope_dim=d,
                                             rope_positions=st["rope"].shape[0])
    else:
        groups = st["plan"]["groups"]
        kw = {}
        if groups:
            starts, shared = groups
            private = [n - s for g, s in enumerate(shared) for n in st["plan"]["lens"][starts[g]:starts[g + 1]]]
            kw = dict(groups=len(shared), max_group_rows=max(b - a for a, b in zip(starts, starts[1:])),
                      max_shared=max(shared), max_private=max(0, max(private)))
        st["call"] = st["pages"].attention_plan(rows, h, nseq, st["per_seq"], max(st["plan"]["lens"]),
                                                type=code[case["type"]], **kw)
        st["workspace"] = torch.empty(max(16, st["call"].workspace_bytes), dtype=torch.uint8, device=DEV)
    return st


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------

def run(st):
    op = st["case"]["op"]
    if own:
        return _OWN[op](st)
    return _PLAIN[op](st)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_append(st):
    c = st["case"]
    q = st["qkv"].data_ptr()
    hq, kv, b = c["heads"] * c["head_dim"], c["kv_heads"] * c["head_dim"], st["qkv"].element_size()
    st["call"](q, q + hq * b, q + (hq + kv) * b, st["q_out"].data_ptr(), st["pos"].data_ptr(), st["table"].data_ptr(),
               st["rope"].data_ptr(), seq=st["seq"].data_ptr(), stream=_stream())
    return {"q": st["q_out"], "k": st["k"], "v": st["v"]}


def _own_attention(st):
    kw = {}
    if st["plan"]["groups"]:
        kw = dict(group_rows=st["group_rows"].data_ptr(), group_len=st["group_len"].data_ptr())
    st["call"](st["q"].data_ptr(), st["out"].data_ptr(), st["lens"].data_ptr(), st["table"].data_ptr(),
               workspace=st["workspace"].data_ptr(), seq=st["seq"].data_ptr(), stream=_stream(), **kw)
    return st["out"]


def _own_probs(st):
    from laicompute_b200.serving import logits_probs
    c = st["case"]
    logits_probs(c["rows"], c["vocab"], st["logits"].data_ptr(), st["temperature"].data_ptr(), st["probs"].data_ptr(),
                 stream=_stream())
    return st["probs"]


def _own_verify(st):
    from laicompute_b200.serving import verify_drafts
    c = st["case"]
    verify_drafts(c["seqs"], c["drafted"], c["vocab"], st["target"].data_ptr(),
                  st["draft"].data_ptr() if st["draft"] is not None else 0, st["ids"].data_ptr(),
                  st["n_draft"].data_ptr(), st["accept_u"].data_ptr(), st["sample_u"].data_ptr(),
                  st["out_ids"].data_ptr(), st["out_n"].data_ptr(), stream=_stream())
    return {"ids": st["out_ids"], "n": st["out_n"]}


def _rotate(x, cs):
    """Adjacent pairs of [rows][heads][d] by the (cos, sin) of [rows][d/2][2]."""
    x0, x1 = x[..., 0::2], x[..., 1::2]
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    return torch.stack([x0 * c - x1 * s, x1 * c + x0 * s], dim=-1).flatten(-2)


def _plain_append(st):
    c = st["case"]
    h, hkv, d, ps = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    x = st["qkv"].float().view(-1, h + 2 * hkv, d)
    cs = st["rope"][st["pos"].long()]
    st["q_out"].copy_(_rotate(x[:, :h], cs).flatten(1))
    page = st["table"][st["seq"].long(), (st["pos"] // ps).long()].long()
    off = (st["pos"] % ps).long()
    st["k"][page, :, off] = _rotate(x[:, h:h + hkv], cs).half()
    st["v"][page, :, off] = x[:, h + hkv:].half()
    return {"q": st["q_out"], "k": st["k"], "v": st["v"]}


def _plain_attention(st):
    c, plan = st["case"], st["plan"]
    h, hkv, d, ps = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    q = st["q"].float().view(-1, hkv, h // hkv, d)
    rows = len(plan["seq"]) // c["seqs"]  # consecutive rows of one sequence
    for i, total in enumerate(plan["total"]):
        used = st["table"][i, :(total + ps - 1) // ps].long()
        k = st["k"][used].float().transpose(0, 1).reshape(hkv, -1, d)
        v = st["v"][used].float().transpose(0, 1).reshape(hkv, -1, d)
        qi = q[i * rows:(i + 1) * rows].transpose(0, 1).reshape(hkv, -1, d)
        s = torch.matmul(qi, k.transpose(1, 2)) / math.sqrt(d)
        s = s.view(hkv, rows, h // hkv, -1)
        seen = torch.arange(s.shape[-1], device=DEV)[None, :] < st["lens"][i * rows:(i + 1) * rows, None]
        s = s.masked_fill(~seen[None, :, None, :], float("-inf"))
        p = torch.exp(s - s.amax(dim=-1, keepdim=True))
        p = (p / p.sum(dim=-1, keepdim=True)).view(hkv, -1, s.shape[-1])
        o = torch.matmul(p, v).view(hkv, rows, h // hkv, d).transpose(0, 1)
        st["out"][i * rows:(i + 1) * rows] = o.reshape(rows, h * d).to(st["out"].dtype)
    return st["out"]


def _plain_probs(st):
    x, t = st["logits"], st["temperature"][:, None]
    m = x.amax(dim=-1, keepdim=True)
    e = torch.exp((x - m) / torch.where(t > 0, t, torch.ones_like(t)))
    soft = e / e.sum(dim=-1, keepdim=True)
    hot = torch.zeros_like(x).scatter_(1, x.argmax(dim=-1, keepdim=True), 1.0)
    st["probs"].copy_(torch.where(t > 0, soft, hot))
    return st["probs"]


def _plain_verify(st):
    c = st["case"]
    n, m, v = c["seqs"], c["drafted"], c["vocab"]
    target = st["target"].view(n, m + 1, v)
    ids = st["ids"].long()
    p = target[:, :m].gather(2, ids[:, :, None])[:, :, 0]
    if st["draft"] is not None:
        q = st["draft"].view(n, m, v).gather(2, ids[:, :, None])[:, :, 0]
    else:
        q = torch.ones_like(p)
    j = torch.arange(m, device=DEV)[None, :]
    ok = (st["accept_u"].double() * q.double() < p.double()) & (j < st["n_draft"][:, None])
    acc = torch.cumprod(ok.int(), dim=1).sum(dim=1)  # tokens accepted
    seqs = torch.arange(n, device=DEV)
    r = target[seqs, acc].double()
    refused = acc < st["n_draft"]
    at = acc.clamp(max=m - 1)
    if st["draft"] is not None:
        minus = st["draft"].view(n, m, v)[seqs, at].double()
    else:
        minus = torch.zeros_like(r).scatter_(1, ids[seqs, at][:, None], r.gather(1, ids[seqs, at][:, None]))
    left = torch.where(refused[:, None], (r - minus).clamp(min=0), r)
    left = torch.where(left.sum(dim=1, keepdim=True) > 0, left, r)
    cum = torch.cumsum(left, dim=1)
    t = st["sample_u"].double()[:, None] * cum[:, -1:]
    tok = (cum <= t).sum(dim=1).clamp(max=v - 1).to(torch.int32)
    jj = torch.arange(m + 1, device=DEV)[None, :]
    drafted = torch.cat([st["ids"], st["ids"][:, :1]], dim=1)
    out = torch.where(jj < acc[:, None], drafted, torch.full_like(drafted, -1))
    st["out_ids"].copy_(torch.where(jj == acc[:, None], tok[:, None], out))
    st["out_n"].copy_(acc + 1)
    return {"ids": st["out_ids"], "n": st["out_n"]}


_OWN = {"append": _own_append, "attention": _own_attention, "probs": _own_probs, "verify": _own_verify}
_PLAIN = {"append": _plain_append, "attention": _plain_attention, "probs": _plain_probs, "verify": _plain_verify}


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------

def work(case):
    if case["op"] in ("append", "attention"):
        h, hkv, d = case["heads"], case["kv_heads"], case["head_dim"]
        plan = _plan(case)
        rows = len(plan["seq"])
    if case["op"] == "append":
        bi, bq = (4 if case["in_type"] == "f32" else 2), (4 if case["q_type"] == "f32" else 2)
        return {"bytes": rows * ((h + 2 * hkv) * d * bi + h * d * bq + 2 * hkv * d * 2 + 12)
                + len(set(plan["pos"])) * d * 4, "flops": rows * (h + hkv) * d * 3}
    if case["op"] == "attention":
        b = 4 if case["type"] == "f32" else 2
        if case["mode"] == "prefix":
            distinct = sum(t - case["shared"] for t in plan["total"]) + case["groups"] * case["shared"]
        else:
            distinct = sum(plan["total"])
        return {"bytes": distinct * hkv * d * 4 + 2 * rows * h * d * b, "flops": 4 * h * d * sum(plan["lens"])}
    if case["op"] == "probs":
        return {"bytes": 8 * case["rows"] * case["vocab"], "flops": 4 * case["rows"] * case["vocab"]}
    rows = 2 if case["draft"] == "probs" else 1  # the target's row and, mostly, the draft's
    return {"bytes": 4 * rows * case["seqs"] * case["vocab"], "flops": 3 * case["seqs"] * case["vocab"]}


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------

def exact(case, seed):
    st = _inputs(case, seed)
    op = case["op"]
    if op == "append":
        h, hkv, d, ps = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
        x = st["qkv"].double().view(-1, h + 2 * hkv, d // 2, 2)
        turn = torch.view_as_complex(st["rope"].double())[st["pos"].long()][:, None, :]
        rot = torch.view_as_real(torch.view_as_complex(x[:, :h + hkv].contiguous()) * turn).flatten(-2)
        k, v = st["k"].double(), st["v"].double()
        flat = st["table"].long()[st["seq"].long(), torch.div(st["pos"], ps, rounding_mode="floor").long()] * ps \
            + (st["pos"] % ps).long()
        kt, vt = k.transpose(1, 2).reshape(-1, hkv, d), v.transpose(1, 2).reshape(-1, hkv, d)
        kt[flat] = rot[:, h:]
        vt[flat] = x[:, h + hkv:].flatten(-2)
        back = lambda z: z.view(-1, ps, hkv, d).transpose(1, 2).contiguous()
        return {"q": rot[:, :h].flatten(1), "k": back(kt), "v": back(vt)}
    if op == "attention":
        h, hkv, d, ps = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
        plan, g = st["plan"], h // hkv
        out = torch.zeros(len(plan["seq"]), h, d, dtype=torch.float64, device=DEV)
        by_seq = {}
        for r, s in enumerate(plan["seq"]):
            by_seq.setdefault(s, []).append(r)
        for s, rs in by_seq.items():
            n = max(plan["lens"][r] for r in rs)
            at = torch.arange(n, device=DEV)
            page = st["table"][s].long()[at // ps]
            q = st["q"][rs].double().view(len(rs), h, d)
            lens = torch.tensor([plan["lens"][r] for r in rs], device=DEV)
            for kh in range(hkv):
                k, v = st["k"][page, kh, at % ps].double(), st["v"][page, kh, at % ps].double()
                sc = torch.einsum("rgd,td->rgt", q[:, kh * g:(kh + 1) * g], k) * d ** -0.5
                sc = torch.where(at[None, None, :] < lens[:, None, None], sc, torch.full_like(sc, -math.inf))
                out[rs, kh * g:(kh + 1) * g] = torch.einsum("rgt,td->rgd", torch.softmax(sc, dim=-1), v)
        return out.flatten(1)
    if op == "probs":
        out = torch.zeros(st["logits"].shape, dtype=torch.float64, device=DEV)
        for r, t in enumerate(st["temperature"].double().tolist()):
            row = st["logits"][r].double()
            if t > 0:
                out[r] = torch.softmax(row / t, dim=0)
            else:
                out[r, int((row == row.max()).nonzero()[0, 0])] = 1.0
        return out
    n, m, v = case["seqs"], case["drafted"], case["vocab"]
    ids_out = torch.full((n, m + 1), -1, dtype=torch.int32)
    n_out = torch.zeros(n, dtype=torch.int32)
    ids, nd = st["ids"].tolist(), st["n_draft"].tolist()
    au, su = st["accept_u"].double().tolist(), st["sample_u"].double().tolist()
    for i in range(n):
        j = 0
        while j < nd[i]:
            x = ids[i][j]
            p = float(st["target"][i * (m + 1) + j, x])
            q = float(st["draft"][i * m + j, x]) if st["draft"] is not None else 1.0
            if not au[i][j] * q < p:
                break
            ids_out[i, j] = x
            j += 1
        w = st["target"][i * (m + 1) + j].double()
        if j < nd[i]:
            if st["draft"] is not None:
                w2 = torch.clamp(w - st["draft"][i * m + j].double(), min=0)
            else:
                w2 = w.clone()
                w2[ids[i][j]] = 0
            w = w2 if float(w2.sum()) > 0 else w
        cum = torch.cumsum(w, 0)
        tok = int(torch.searchsorted(cum, su[i] * cum[-1], right=True))
        ids_out[i, j] = min(tok, v - 1)
        n_out[i] = j + 1
    return {"ids": ids_out.to(DEV), "n": n_out.to(DEV)}
