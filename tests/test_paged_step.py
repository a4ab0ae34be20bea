"""Refusals of the paged serving step's operators. Each check returns before any CUDA call, so this runs without a GPU;
the pointers are never dereferenced."""

import ctypes

import pytest

from rosylnalive_b200 import native as N
from rosylnalive_b200 import ops as O

A = 0x10000  # a 16-byte aligned address


def plan(**kw):
    d = dict(slots=A, new_len=A, seq_len=A, page_table=A, free_list=A, free_count=A, cu_seqlens=A, kv_len=A, tok_pos=A,
             slot_map=A, seq_len_out=A, free_count_out=A, requests=3, max_seqs=4, pages_per_seq=5, kv_pages=6,
             max_tokens=7)
    return "lrm_op_page_plan", O.PagePlanDesc(**{**d, **kw})


def release(**kw):
    d = dict(slots=A, keep_len=A, seq_len=A, page_table=A, free_list=A, free_count=A, seq_len_out=A, free_count_out=A,
             requests=3, max_seqs=4, pages_per_seq=5, kv_pages=6)
    return "lrm_op_page_release", O.PageReleaseDesc(**{**d, **kw})


def append(**kw):
    d = dict(qkv=A, q_norm=A, k_norm=A, cos=A, sin=A, tok_pos=A, slot_map=A, q_out=A, pool=A, ld_qkv=32 * 128,
             ld_q=16 * 128, tokens=5, q_heads=16, kv_heads=8, head_dim=128, rope_rows=9, kv_pages=6, eps=1e-6)
    return "lrm_op_qkv_append", O.QkvAppendDesc(**{**d, **kw})


def attn(**kw):
    d = dict(q=A, pool=A, page_table=A, slots=A, cu_seqlens=A, kv_len=A, out=A, workspace=A, ld_q=16 * 128,
             ld_out=16 * 128, workspace_bytes=1 << 40, requests=3, tokens=5, q_heads=16, kv_heads=8, head_dim=128, max_seqs=4, pages_per_seq=5,
             kv_pages=6, scale=0.1)
    return "lrm_op_paged_attention", O.PagedAttnDesc(**{**d, **kw})


BIG = (1 << 31) - 1
INF, NAN = float("inf"), float("nan")
REFUSED = [
    *[plan(**{f: v}) for f, _ in O.PagePlanDesc._fields_[:12] for v in (0, A + 2)],
    *[plan(**{f: v}) for f in ("requests", "max_seqs", "pages_per_seq", "kv_pages", "max_tokens") for v in (0, -1, BIG)],
    plan(requests=65536), plan(max_seqs=(1 << 17) + 1), plan(pages_per_seq=(1 << 20) + 1), plan(max_tokens=(1 << 24) + 1),
    *[release(**{f: v}) for f, _ in O.PageReleaseDesc._fields_[:8] for v in (0, A + 1)],
    *[release(**{f: v}) for f in ("requests", "max_seqs", "pages_per_seq", "kv_pages") for v in (0, -1, BIG)],
    *[append(**{f: v}) for f in ("qkv", "slot_map", "q_out", "pool", "tok_pos") for v in (0, A + 2)],
    *[append(**{f: v}) for f in ("qkv", "q_norm", "k_norm", "cos", "sin", "q_out", "pool") for v in (A + 8,)],
    append(q_norm=0), append(k_norm=0), append(cos=0), append(sin=0), append(rope_rows=0), append(rope_rows=-1),
    *[append(**{f: v}) for f in ("tokens", "q_heads", "kv_heads", "kv_pages") for v in (0, -1, BIG)],
    append(head_dim=64), append(ld_qkv=32 * 128 - 8), append(ld_qkv=32 * 128 + 4), append(ld_q=16 * 128 - 8),
    append(ld_q=16 * 128 + 1), append(ld_qkv=1 << 40), append(eps=-1.0), append(eps=INF), append(eps=NAN),
    *[attn(**{f: v}) for f in ("q", "pool", "out", "workspace") for v in (0, A + 8)],
    *[attn(**{f: v}) for f in ("page_table", "slots", "cu_seqlens", "kv_len") for v in (0, A + 2)],
    *[attn(**{f: v}) for f in ("requests", "tokens", "q_heads", "kv_heads", "max_seqs", "pages_per_seq", "kv_pages")
      for v in (0, -1, BIG)],
    attn(q_heads=15), attn(q_heads=129, kv_heads=1, ld_q=129 * 128, ld_out=129 * 128), attn(head_dim=64),
    attn(kv_pages=1 << 26, kv_heads=16), attn(ld_q=16 * 128 - 8), attn(ld_q=16 * 128 + 4), attn(ld_out=0),
    attn(ld_out=1 << 40), attn(workspace_bytes=0), attn(workspace_bytes=-1), attn(workspace_bytes=1000), attn(scale=0.0), attn(scale=-1.0), attn(scale=INF), attn(scale=NAN), attn(scale=3e38),
]


@pytest.mark.parametrize("k", range(len(REFUSED)))
def test_refused(k):
    name, desc = REFUSED[k]
    assert getattr(N.lib(), name)(None, ctypes.byref(desc)) == N.LRM_ERR_ARGUMENT
    assert N.last_error()


@pytest.mark.parametrize("name", ["lrm_op_page_plan", "lrm_op_page_release", "lrm_op_qkv_append", "lrm_op_paged_attention"])
def test_a_null_descriptor_is_refused(name):
    assert getattr(N.lib(), name)(None, None) == N.LRM_ERR_ARGUMENT


@pytest.mark.parametrize("sizes", [(0, 16, 8), (-1, 16, 8), ((1 << 24) + 1, 16, 8), (4, 15, 8), (4, 0, 8), (4, 16, 0),
                                   (4, 129, 1)])
def test_no_workspace_for_impossible_sizes(sizes):
    assert O.paged_attention_workspace(*sizes) == 0


def test_the_wrappers_check_types_shapes_and_devices():
    import torch

    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    b = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    ok_plan = [i(2), i(2), i(3), i(3, 4), i(5), i(1), i(3), i(2), i(7), i(7)]
    ok_release = [i(2), i(2), i(3), i(3, 4), i(5), i(1)]
    pool = b(3, 2, 2, 16, 128)
    ok_append = [b(5, 8 * 128), b(128), b(128), 1e-6, torch.zeros(9, 64), torch.zeros(9, 64), i(5), i(5), b(5, 4, 128), pool]
    ok_attn = [b(5, 4, 128), pool, i(3, 4), i(2), i(3), i(2), b(5, 4, 128), torch.zeros(1 << 20, dtype=torch.uint8), 0.1]

    def refused(fn, args, at=None, value=None, match=None):
        args = list(args)
        if at is not None:
            args[at] = value
        with pytest.raises(ValueError, match=match):
            fn(*args)

    for fn, args in ((O.page_plan, ok_plan), (O.page_release, ok_release), (O.qkv_append, ok_append),
                     (O.paged_attention, ok_attn)):
        refused(fn, args, match="one CUDA device")  # all on the CPU: the last check before the launch
    for at in range(10):
        refused(O.page_plan, ok_plan, at, ok_plan[at].long(), "int32")
        refused(O.page_plan, ok_plan, at, i(11), "page_plan")
    refused(O.page_plan, ok_plan, 3, i(4, 3).t(), "contiguous")
    for at in range(6):
        refused(O.page_release, ok_release, at, ok_release[at].float(), "int32")
    refused(O.page_release, ok_release, 1, i(3), "keep_len")
    refused(O.qkv_append, ok_append, 0, b(5, 8 * 128 + 8), "columns")
    refused(O.qkv_append, ok_append, 0, b(8 * 128, 5).t(), "strided")
    refused(O.qkv_append, ok_append, 0, torch.zeros(5, 8 * 128), "bfloat16")
    refused(O.qkv_append, ok_append, 1, None, "both gains")
    refused(O.qkv_append, ok_append, 2, torch.zeros(128), "q_norm")
    refused(O.qkv_append, ok_append, 4, None, "cos")
    refused(O.qkv_append, ok_append, 5, torch.zeros(8, 64), "shape")
    refused(O.qkv_append, ok_append, 6, None, "tok_pos")
    refused(O.qkv_append, ok_append, 7, i(4), "slot_map")
    refused(O.qkv_append, ok_append, 8, b(4, 5, 128).transpose(0, 1), "strided")
    refused(O.qkv_append, ok_append, 9, pool.float(), "pool")
    refused(O.paged_attention, ok_attn, 0, torch.zeros(5, 4, 128), "bfloat16")
    refused(O.paged_attention, ok_attn, 0, b(4, 5, 128).transpose(0, 1), "strided")
    refused(O.paged_attention, ok_attn, 1, b(3, 2, 2, 16, 64), "pool")
    refused(O.paged_attention, ok_attn, 4, i(4), "cu_seqlens")
    refused(O.paged_attention, ok_attn, 6, b(4, 4, 128), "out")


def test_the_packed_descriptors_are_the_structures():
    for packed, desc in ((O._PLAN, plan()[1]), (O._RELEASE, release()[1]), (O._APPEND, append()[1]), (O._ATTN, attn()[1])):
        values = [getattr(desc, name) for name, _ in desc._fields_]
        assert packed.pack(*values) == bytes(desc)[:packed.size]
