"""Serving operators on device pointers: a KV cache in pages (append with the position rotation,
attention that reads shared prefixes for all their rows together), probabilities of logits rows and
the verification of drafted tokens (``laic_kv_*``, ``laic_logits_probs``, ``laic_verify_drafts`` of
include/laic_b200.h).

As in ``engine.Matrix``, pointers are plain integers (``tensor.data_ptr()``) and ``stream`` a
``cudaStream_t``; calls return when their kernels are queued. A plan holds a call's shape, so that a
loop passes only its pointers; threads may call one plan at once, each with outputs and a workspace of its own.
"""
from __future__ import annotations

import ctypes

from . import gguf
from ._native import KvAppendArgs, KvAttentionArgs, KvPagesDesc, VerifyArgs, check, lib


class KvPages:
    """One layer's KV cache in pages: ``k``, ``v`` [num_pages][kv_heads][page_size][head_dim] binary16,
    ``err`` a zeroed int32 the kernels record refused indices in (the caller owns all three)."""

    def __init__(self, k: int, v: int, num_pages: int, kv_heads: int, page_size: int, head_dim: int, err: int,
                 device: int = 0) -> None:
        self.desc = KvPagesDesc(device=device, kv_heads=kv_heads, head_dim=head_dim, page_size=page_size,
                                num_pages=num_pages, k_dev=k, v_dev=v, err_dev=err)

    def append_plan(self, rows: int, heads: int, nseq: int, pages_per_seq: int, **kw) -> "AppendPlan":
        return AppendPlan(self, rows, heads, nseq, pages_per_seq, **kw)

    def attention_plan(self, rows: int, heads: int, nseq: int, pages_per_seq: int, max_len: int,
                       **kw) -> "AttentionPlan":
        return AttentionPlan(self, rows, heads, nseq, pages_per_seq, max_len, **kw)

    def check(self, stream: int = 0) -> None:
        """Synchronise `stream` and raise if a kernel refused an index since the last check."""
        check(lib().laic_kv_check(ctypes.byref(self.desc), stream))


class AppendPlan:
    """``plan(q, k, v, q_out, pos, table, rope, seq, stream)``: rotate `rows` tokens' q and k, write q to
    q_out and k, v into the pages. Row strides (elements) default to packed rows."""

    def __init__(self, pages: KvPages, rows: int, heads: int, nseq: int, pages_per_seq: int, *,
                 in_type: int = gguf.F32, q_type: int = gguf.F32, ldq: int = 0, ldk: int = 0, ldv: int = 0, ldqo: int = 0,
                 rope_dim: int = 0, rope_positions: int = 0) -> None:
        d = pages.desc
        kvw = d.kv_heads * d.head_dim
        self.pages = pages
        self.args = KvAppendArgs(rows=rows, heads=heads, in_type=in_type, q_type=q_type, rope_dim=rope_dim,
                                 rope_positions=rope_positions, nseq=nseq, pages_per_seq=pages_per_seq,
                                 ldq=ldq or heads * d.head_dim, ldk=ldk or kvw, ldv=ldv or kvw,
                                 ldqo=ldqo or heads * d.head_dim)
        self._call = lib().laic_kv_append
        self._desc = ctypes.byref(d)

    def __call__(self, q: int, k: int, v: int, q_out: int, pos: int, table: int, rope: int = 0, seq: int = 0,
                 stream: int = 0) -> None:
        a = KvAppendArgs.from_buffer_copy(self.args)  # this call's own: another thread may be in one of its own
        a.q_dev, a.k_dev, a.v_dev, a.q_out_dev = q, k, v, q_out
        a.pos_dev, a.page_table_dev, a.rope_dev, a.seq_dev = pos, table, rope, seq
        rc = self._call(self._desc, ctypes.byref(a), stream)
        if rc:
            check(rc)


class AttentionPlan:
    """``plan(q, out, lens, table, workspace, seq, group_rows, group_len, stream)``: attention of `rows`
    query rows over the pages. `max_len` and the ``max_*`` values bound what the device arrays hold;
    `max_private` = -1 stands for `max_len`. `workspace_bytes` of device memory (16-byte aligned)
    belong to the call while it runs."""

    def __init__(self, pages: KvPages, rows: int, heads: int, nseq: int, pages_per_seq: int, max_len: int, *,
                 type: int = gguf.F32, ldq: int = 0, ldo: int = 0, groups: int = 0, max_group_rows: int = 0,
                 max_shared: int = 0, max_private: int = -1, scale: float = 0.0) -> None:
        w = heads * pages.desc.head_dim
        self.pages = pages
        self.args = KvAttentionArgs(rows=rows, heads=heads, type=type, nseq=nseq, pages_per_seq=pages_per_seq,
                                    max_len=max_len, groups=groups, max_group_rows=max_group_rows, max_shared=max_shared,
                                    max_private=max_private, scale=scale, ldq=ldq or w, ldo=ldo or w)
        self._call = lib().laic_kv_attention
        self._desc = ctypes.byref(pages.desc)
        n = ctypes.c_uint64()
        check(lib().laic_kv_attention_workspace(self._desc, ctypes.byref(self.args), ctypes.byref(n)))
        self.workspace_bytes = self.args.workspace_bytes = int(n.value)

    def __call__(self, q: int, out: int, lens: int, table: int, workspace: int = 0, seq: int = 0, group_rows: int = 0,
                 group_len: int = 0, stream: int = 0) -> None:
        a = KvAttentionArgs.from_buffer_copy(self.args)  # this call's own: another thread may be in one of its own
        a.q_dev, a.out_dev, a.len_dev, a.page_table_dev, a.workspace_dev = q, out, lens, table, workspace
        a.seq_dev, a.group_rows_dev, a.group_len_dev = seq, group_rows, group_len
        rc = self._call(self._desc, ctypes.byref(a), stream)
        if rc:
            check(rc)


def logits_probs(rows: int, vocab: int, logits: int, temperature: int, probs: int, ld_logits: int = 0,
                 ld_probs: int = 0, device: int = 0, stream: int = 0) -> None:
    """probs[r] = softmax(logits[r] / temperature[r]); one for the first maximum where temperature <= 0."""
    check(lib().laic_logits_probs(device, rows, vocab, logits, ld_logits or vocab, temperature, probs,
                                  ld_probs or vocab, stream))


def verify_drafts(nseq: int, max_draft: int, vocab: int, target: int, draft: int, draft_ids: int, n_draft: int,
                  accept_u: int, sample_u: int, out_ids: int, out_n: int, ld_target: int = 0, ld_draft: int = 0,
                  device: int = 0, stream: int = 0) -> None:
    """Accept or refuse each sequence's drafted tokens and draw the next one (laic_verify_drafts);
    draft = 0: tokens drafted with certainty."""
    a = VerifyArgs(nseq, max_draft, vocab, ld_target or vocab, ld_draft or vocab, target, draft, draft_ids, n_draft,
                   accept_u, sample_u, out_ids, out_n)
    check(lib().laic_verify_drafts(device, ctypes.byref(a), stream))
