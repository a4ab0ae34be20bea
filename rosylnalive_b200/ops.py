"""Python access to liblrmcuda.so's fast-path operators (include/lrm_cuda.h, "fast-path operators").

Arguments are torch CUDA tensors (used only as device memory and streams); every call goes through the C ABI.
"""

from __future__ import annotations

import ctypes
import struct

from . import native as N

P, I32, U32, U64, I64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_uint32, ctypes.c_uint64, ctypes.c_int64

GEMM_F32, GEMM_RESID, GEMM_SWIGLU, GEMM_PARTIAL, GEMM_BF16 = range(5)


class GemmDesc(ctypes.Structure):
    _fields_ = [("m", I32), ("n", I32), ("k", I32), ("a", U64), ("b", U64), ("epilogue", I32), ("bn", I32),
                ("splits", I32), ("out", U64), ("ldo", I32), ("resid", U64), ("ldr", I32), ("split_stride", U64),
                ("cta_pair", I32)]


class PrefillAttnDesc(ctypes.Structure):
    _fields_ = [("q", U64), ("k", U64), ("v", U64), ("out", U64), ("cu_seqlens", U64), ("nseq", I32),
                ("max_len", I32), ("q_heads", I32), ("kv_heads", I32), ("head_dim", I32), ("total_tokens", I32),
                ("scale", ctypes.c_float)]


class DecodeAttnDesc(ctypes.Structure):
    _fields_ = [("q", U64), ("pool", U64), ("page_table", U64), ("seq_len", U64), ("slots", U64), ("out", U64),
                ("workspace", U64), ("batch", I32), ("q_heads", I32), ("kv_heads", I32), ("head_dim", I32),
                ("pages_per_seq", I32), ("pages_per_split", I32), ("scale", ctypes.c_float)]


class DecodeGemmDesc(ctypes.Structure):
    _fields_ = [("m", I32), ("n", I32), ("k", I32), ("w", U64), ("b", U64), ("epilogue", I32), ("splits", I32),
                ("ss", U64), ("nss", I32), ("hidden", I32), ("ss_stride", U64), ("eps", ctypes.c_float),
                ("x", U64), ("gain", U64), ("u", U64), ("ss_out", U64), ("act", U64), ("ld_act", I32)]


class PagePlanDesc(ctypes.Structure):
    _fields_ = [("slots", U64), ("new_len", U64), ("seq_len", U64), ("page_table", U64), ("free_list", U64),
                ("free_count", U64), ("cu_seqlens", U64), ("kv_len", U64), ("tok_pos", U64), ("slot_map", U64),
                ("seq_len_out", U64), ("free_count_out", U64), ("requests", I32), ("max_seqs", I32),
                ("pages_per_seq", I32), ("kv_pages", I32), ("max_tokens", I32)]


class PageReleaseDesc(ctypes.Structure):
    _fields_ = [("slots", U64), ("keep_len", U64), ("seq_len", U64), ("page_table", U64), ("free_list", U64),
                ("free_count", U64), ("seq_len_out", U64), ("free_count_out", U64), ("requests", I32),
                ("max_seqs", I32), ("pages_per_seq", I32), ("kv_pages", I32)]


class QkvAppendDesc(ctypes.Structure):
    _fields_ = [("qkv", U64), ("q_norm", U64), ("k_norm", U64), ("cos", U64), ("sin", U64), ("tok_pos", U64),
                ("slot_map", U64), ("q_out", U64), ("pool", U64), ("ld_qkv", I64), ("ld_q", I64), ("tokens", I32),
                ("q_heads", I32), ("kv_heads", I32), ("head_dim", I32), ("rope_rows", I32), ("kv_pages", I32),
                ("eps", ctypes.c_float)]


class PagedAttnDesc(ctypes.Structure):
    _fields_ = [("q", U64), ("pool", U64), ("page_table", U64), ("slots", U64), ("cu_seqlens", U64), ("kv_len", U64),
                ("out", U64), ("workspace", U64), ("ld_q", I64), ("ld_out", I64), ("workspace_bytes", I64),
                ("requests", I32), ("tokens", I32), ("q_heads", I32), ("kv_heads", I32), ("head_dim", I32),
                ("max_seqs", I32), ("pages_per_seq", I32), ("kv_pages", I32), ("scale", ctypes.c_float)]


DEC_SWIGLU, DEC_RESID = 1, 2

N.extra_signatures({
    "lrm_op_set_device": [I32],
    "lrm_op_error_word": [ctypes.POINTER(U32), I32],
    "lrm_op_gemm_bf16": [P, ctypes.POINTER(GemmDesc)],
    "lrm_op_prefill_attention": [P, ctypes.POINTER(PrefillAttnDesc)],
    "lrm_op_decode_attention_workspace": [I32, I32, I32, I32],
    "lrm_op_decode_attention": [P, ctypes.POINTER(DecodeAttnDesc)],
    "lrm_op_decode_attention_static": [P, ctypes.POINTER(DecodeAttnDesc)],
    "lrm_op_wait_probe": [P, U32, U32],
    "lrm_op_argmax_rows": [P, P, I32, I32, P],
    "lrm_op_decode_gemm": [P, ctypes.POINTER(DecodeGemmDesc)],
    "lrm_op_page_plan": [P, P],  # the descriptors of these four also as packed bytes
    "lrm_op_page_release": [P, P],
    "lrm_op_qkv_append": [P, P],
    "lrm_op_paged_attention_workspace": [I32, I32, I32],
    "lrm_op_paged_attention": [P, P],
}, {"lrm_op_decode_attention_workspace": U64, "lrm_op_paged_attention_workspace": U64})

# Scratch built into liblrmcuda.so for lrm_op_decode_attention_static (LRM_DECODE_ATTN_STATIC_SCRATCH_BYTES).
DECODE_ATTN_STATIC_SCRATCH_BYTES = 16 << 20


def _stream(stream):
    import torch

    s = stream if stream is not None else torch.cuda.current_stream()
    return ctypes.c_void_p(s.cuda_stream)


def set_device(index: int):
    N.check(N.lib().lrm_op_set_device(index), None, "set_device")


def error_word(clear: bool = True) -> int:
    v = ctypes.c_uint32()
    N.check(N.lib().lrm_op_error_word(ctypes.byref(v), 1 if clear else 0), None, "error_word")
    return v.value


def argmax_rows(logits, out, stream=None):
    """out[r] (uint32 as int32 storage) = the lowest index of the maximum of logits[r] (fp32 [rows, vocab] on the
    device), or 0xFFFFFFFF for a row holding a NaN: the engine's greedy pick."""
    N.check(N.lib().lrm_op_argmax_rows(_stream(stream), ctypes.c_void_p(logits.data_ptr()), logits.shape[0],
                                       logits.shape[1], ctypes.c_void_p(out.data_ptr())), None, "argmax_rows")


def wait_probe(polls: int, code: int, stream=None):
    """Launches a kernel whose bounded wait cannot complete: after `polls` polls it records `code` in the error word
    and returns (the path every kernel takes when a wait runs out)."""
    N.check(N.lib().lrm_op_wait_probe(_stream(stream), polls, code), None, "wait_probe")


def gemm(a, b, out, epilogue=GEMM_F32, resid=None, splits=1, bn=0, ldo=None, split_stride=0, cta_pair=0,
         stream=None):
    """out = epilogue(a @ b.T); a bf16 [m, k], b bf16 [n, k] (torch CUDA tensors). cta_pair: 0 chooses, 1 one CTA
    per 128-row tile, 2 two-SM clusters sharing 256 x 256 tiles (bn 256)."""
    m, k = a.shape
    n, k2 = b.shape
    assert k == k2
    d = GemmDesc(m, n, k, a.data_ptr(), b.data_ptr(), epilogue, bn, splits, out.data_ptr(),
                 ldo if ldo is not None else (m if epilogue == GEMM_PARTIAL else out.shape[-1]),
                 resid.data_ptr() if resid is not None else 0, resid.shape[-1] if resid is not None else 0,
                 split_stride, cta_pair)
    N.check(N.lib().lrm_op_gemm_bf16(_stream(stream), ctypes.byref(d)), None, "gemm")


def decode_gemm_resid(w, b, x, gain=None, u=None, ss_out=None, splits=0, stream=None):
    """x [n, m] fp32 += b @ w.T (w bf16 [m, k], b bf16 [n, k]); with gain also u [n, m] = bf16(gain * x) and
    ss_out [m / 128, n] = the sums of x^2 over 128-column groups. K split over a cluster of `splits` CTAs."""
    m, k = w.shape
    n = b.shape[0]
    d = DecodeGemmDesc(m, n, k, w.data_ptr(), b.data_ptr(), DEC_RESID, splits, 0, 0, 0,
                       ss_out.shape[1] if ss_out is not None else 0, 0.0, x.data_ptr(),
                       gain.data_ptr() if gain is not None else 0, u.data_ptr() if u is not None else 0,
                       ss_out.data_ptr() if ss_out is not None else 0, 0, 0)
    N.check(N.lib().lrm_op_decode_gemm(_stream(stream), ctypes.byref(d)), None, "decode_gemm")


def decode_gemm_swiglu(w, b, ss, hidden, eps, act, splits=0, stream=None):
    """act [n, m / 2] bf16 = silu(r g) * (r u) of y = b @ w.T (gate and up rows of w interleaved in blocks of 64),
    r[t] = 1 / sqrt(sum_g ss[g, t] / hidden + eps)."""
    m, k = w.shape
    n = b.shape[0]
    d = DecodeGemmDesc(m, n, k, w.data_ptr(), b.data_ptr(), DEC_SWIGLU, splits, ss.data_ptr(), ss.shape[0], hidden,
                       ss.shape[1], eps, 0, 0, 0, 0, act.data_ptr(), act.shape[1])
    N.check(N.lib().lrm_op_decode_gemm(_stream(stream), ctypes.byref(d)), None, "decode_gemm")


def prefill_attention(q, k, v, out, cu_seqlens, max_len, scale, stream=None):
    """Causal GQA attention of packed sequences: q [T, qh, 128], k/v [T, kvh, 128], cu_seqlens int32 [nseq + 1]."""
    d = PrefillAttnDesc(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), cu_seqlens.data_ptr(),
                        cu_seqlens.numel() - 1, max_len, q.shape[1], k.shape[1], q.shape[2], q.shape[0], scale)
    N.check(N.lib().lrm_op_prefill_attention(_stream(stream), ctypes.byref(d)), None, "prefill_attention")


def decode_attention_workspace(batch, kv_heads, pages_per_seq, pages_per_split) -> int:
    return int(N.lib().lrm_op_decode_attention_workspace(batch, kv_heads, pages_per_seq, pages_per_split))


def decode_attention(q, pool, page_table, seq_len, slots, out, workspace, pages_per_split, scale, stream=None):
    """Paged decode attention: q [B, qh, 128], pool [pages, kvh, 2, 16, 128], page_table int32 [seqs, pages_per_seq],
    seq_len int32 [seqs], slots int32 [B]."""
    d = DecodeAttnDesc(q.data_ptr(), pool.data_ptr(), page_table.data_ptr(), seq_len.data_ptr(), slots.data_ptr(),
                       out.data_ptr(), workspace.data_ptr(), q.shape[0], q.shape[1], pool.shape[1], q.shape[2],
                       page_table.shape[1], pages_per_split, scale)
    N.check(N.lib().lrm_op_decode_attention(_stream(stream), ctypes.byref(d)), None, "decode_attention")


def decode_attention_static(q, pool, page_table, seq_len, slots, out, pages_per_split, scale, stream=None):
    """decode_attention for callers that cannot allocate device memory: the split scratch is the 16 MiB array built
    into liblrmcuda.so (DECODE_ATTN_STATIC_SCRATCH_BYTES); the caller passes only inputs and the output. Calls that
    overlap on the GPU share that array and race; the first call on a device should come before any stream capture."""
    d = DecodeAttnDesc(q.data_ptr(), pool.data_ptr(), page_table.data_ptr(), seq_len.data_ptr(), slots.data_ptr(),
                       out.data_ptr(), 0, q.shape[0], q.shape[1], pool.shape[1], q.shape[2], page_table.shape[1],
                       pages_per_split, scale)
    N.check(N.lib().lrm_op_decode_attention_static(_stream(stream), ctypes.byref(d)), None,
            "decode_attention_static")


# ---- a paged serving step on the device (include/lrm_cuda.h, same heading) -----------------------------------------
#
# plan -> append -> attention -> release, with lengths, page table and free pages kept on the device and no copy to or
# from the host. These take tensors of any CUDA device (all of a call on one) and launch on `stream`, or on that
# device's current stream. What only the device knows (slots, lengths, page ids) is checked there: error_word(). Arrays
# without elements are refused (ValueError), as by the operators above: a step has one request and one row at least, which
# may be padding (slot -1, slot_map -1).

# A call is a few microseconds on the device, so the checks are kept to a few as well: one loop over its tensors, and the
# descriptor packed in one go (the layouts of PagePlanDesc and its like above).

_PLAN, _RELEASE = struct.Struct("12Q5i"), struct.Struct("8Q4i")
_APPEND, _ATTN = struct.Struct("9Q2q6if"), struct.Struct("8Q3q8if")
assert [x.size for x in (_PLAN, _RELEASE, _APPEND, _ATTN)] == [
    _LAST.offset + _LAST.size for _LAST in (PagePlanDesc.max_tokens, PageReleaseDesc.kv_pages, QkvAppendDesc.eps,
                                            PagedAttnDesc.scale)]
_torch = None


def _t():
    global _torch
    if _torch is None:
        import torch

        _torch = torch
    return _torch


def _int32(call, names, tensors, dev):
    """Checks that the tensors are contiguous int32 tensors of device `dev`."""
    i32 = _t().int32
    for t in tensors:
        if t.dtype is not i32 or t.get_device() != dev or not t.is_contiguous():
            if t.dtype is i32 and t.is_contiguous():
                raise ValueError(f"{call}: all tensors must be on one CUDA device")
            name = names.split()[next(i for i, x in enumerate(tensors) if x is t)]
            raise ValueError(f"{call}: {name} must be a contiguous int32 tensor")


def _pool(call, pool):
    if pool.dtype is not _t().bfloat16 or pool.dim() != 5 or pool.shape[2:] != (2, 16, 128) or not pool.is_contiguous():
        raise ValueError(f"{call}: pool must be contiguous bfloat16 [pages, kv_heads, 2, 16, 128]")


def _rows_of_heads(t, shape):
    """The row stride of [T, heads, 128] when only its rows are strided, else None."""
    rows, heads, last = t.stride()
    if last != 1 or (heads != 128 and shape[1] != 1):
        return None
    return rows if shape[0] > 1 else shape[1] * 128


def _launch(call, fn, desc, dev, stream):
    if dev < 0:
        raise ValueError(f"{call}: all tensors must be on one CUDA device")
    torch = _t()
    if dev == torch._C._cuda_getDevice():
        s = torch._C._cuda_getCurrentRawStream(dev) if stream is None else stream.cuda_stream
        status = fn(s, desc)
    else:
        with torch.cuda.device(dev):
            s = torch.cuda.current_stream(dev) if stream is None else stream
            status = fn(s.cuda_stream, desc)
    if status:
        N.check(status, None, call)


def page_plan(slots, new_len, seq_len, page_table, free_list, free_count, cu_seqlens, kv_len, tok_pos, slot_map,
              seq_len_out=None, free_count_out=None, stream=None):
    """Takes pages for each request's new tokens and writes the step's cu_seqlens [requests + 1], kv_len [requests],
    tok_pos and slot_map [max_tokens]; int32 tensors throughout. slots [requests] (-1: padding) with new_len tokens
    each; seq_len [max_seqs], page_table [max_seqs, pages_per_seq], free_list [kv_pages] and free_count [1] are the
    cache's state, updated in place unless seq_len_out / free_count_out are given. All or nothing: a step that breaks a
    rule (error_word 0x5001 .. 0x5004) takes no page and becomes a step of no tokens, and seq_len_out / free_count_out
    get the old lengths of its slots and the old count."""
    if seq_len_out is None:
        seq_len_out = seq_len
    if free_count_out is None:
        free_count_out = free_count
    dev = slots.get_device()
    _int32("page_plan", "slots new_len seq_len page_table free_list free_count cu_seqlens kv_len tok_pos slot_map "
           "seq_len_out free_count_out",
           (slots, new_len, seq_len, page_table, free_list, free_count, cu_seqlens, kv_len, tok_pos, slot_map,
            seq_len_out, free_count_out), dev)
    n, seqs, tokens, table = slots.numel(), seq_len.numel(), tok_pos.numel(), page_table.shape
    if len(table) != 2 or table[0] != seqs or seq_len_out.numel() != seqs:
        raise ValueError("page_plan: page_table must be [max_seqs, pages_per_seq] and seq_len, seq_len_out [max_seqs]")
    if (new_len.numel() != n or kv_len.numel() != n or cu_seqlens.numel() != n + 1 or slot_map.numel() != tokens
            or free_count.numel() != 1 or free_count_out.numel() != 1):
        raise ValueError("page_plan: new_len and kv_len are [requests], cu_seqlens [requests + 1], tok_pos and slot_map "
                         "one size, free_count and free_count_out one element")
    _launch("page_plan", N.lib().lrm_op_page_plan, _PLAN.pack(
        slots.data_ptr(), new_len.data_ptr(), seq_len.data_ptr(), page_table.data_ptr(), free_list.data_ptr(),
        free_count.data_ptr(), cu_seqlens.data_ptr(), kv_len.data_ptr(), tok_pos.data_ptr(), slot_map.data_ptr(),
        seq_len_out.data_ptr(), free_count_out.data_ptr(), n, seqs, table[1], free_list.numel(), tokens), dev, stream)


def page_release(slots, keep_len, seq_len, page_table, free_list, free_count, seq_len_out=None, free_count_out=None,
                 stream=None):
    """Cuts slots [requests] (-1: padding) back to their first keep_len tokens (0 frees a slot) and puts the pages
    behind them back on top of the free list. State and outputs as in page_plan. All or nothing: a call that breaks a
    rule (error_word 0x5011, 0x5012, 0x5014) changes no length, page or count; seq_len_out / free_count_out get the old
    ones, as in page_plan."""
    if seq_len_out is None:
        seq_len_out = seq_len
    if free_count_out is None:
        free_count_out = free_count
    dev = slots.get_device()
    _int32("page_release", "slots keep_len seq_len page_table free_list free_count seq_len_out free_count_out",
           (slots, keep_len, seq_len, page_table, free_list, free_count, seq_len_out, free_count_out), dev)
    n, seqs, table = slots.numel(), seq_len.numel(), page_table.shape
    if len(table) != 2 or table[0] != seqs or seq_len_out.numel() != seqs:
        raise ValueError("page_release: page_table must be [max_seqs, pages_per_seq] and seq_len, seq_len_out [max_seqs]")
    if keep_len.numel() != n or free_count.numel() != 1 or free_count_out.numel() != 1:
        raise ValueError("page_release: keep_len is [requests], free_count and free_count_out one element")
    _launch("page_release", N.lib().lrm_op_page_release, _RELEASE.pack(
        slots.data_ptr(), keep_len.data_ptr(), seq_len.data_ptr(), page_table.data_ptr(), free_list.data_ptr(),
        free_count.data_ptr(), seq_len_out.data_ptr(), free_count_out.data_ptr(), n, seqs, table[1],
        free_list.numel()), dev, stream)


def qkv_append(qkv, q_norm, k_norm, eps, cos, sin, tok_pos, slot_map, q_out, pool, stream=None):
    """QK-RMSNorm, RoPE and the paged append of one fused projection qkv [T, (q_heads + 2 kv_heads) * 128] (bfloat16,
    rows may be strided): q to q_out [T, q_heads, 128] (rows may be strided; may be a view of qkv's q columns), k and v
    to pool [pages, kv_heads, 2, 16, 128] at slot_map [T] (int32 page * 16 + offset; -1 skips the row). q_norm, k_norm:
    bfloat16 [128], or both None for no norm. cos, sin: float32 [rows, 64] read at tok_pos [T], or all three None for
    no rotation."""
    torch = _t()
    bf16, dev = torch.bfloat16, qkv.get_device()
    _pool("qkv_append", pool)
    shape, q_shape, pool_shape = qkv.shape, q_out.shape, pool.shape
    if (qkv.dtype is not bf16 or q_out.dtype is not bf16 or len(shape) != 2 or len(q_shape) != 3 or q_shape[2] != 128
            or q_shape[0] != shape[0]):
        raise ValueError("qkv_append: qkv must be bfloat16 [T, columns] and q_out bfloat16 [T, q_heads, 128]")
    tokens, q_heads, kv_heads = shape[0], q_shape[1], pool_shape[1]
    if shape[1] != (q_heads + 2 * kv_heads) * 128:
        raise ValueError("qkv_append: qkv has (q_heads + 2 kv_heads) * 128 columns")
    ld_q, (ld_qkv, inner) = _rows_of_heads(q_out, q_shape), qkv.stride()
    if inner != 1 or ld_q is None:
        raise ValueError("qkv_append: only the rows of qkv and q_out may be strided")
    _int32("qkv_append", "slot_map", (slot_map,), dev)
    if slot_map.numel() != tokens:
        raise ValueError("qkv_append: slot_map is [T]")
    gains = table = (0, 0)
    at = rope_rows = 0
    if q_norm is not None or k_norm is not None:
        if q_norm is None or k_norm is None:
            raise ValueError("qkv_append: give both gains or none")
        for g in (q_norm, k_norm):
            if g.dtype is not bf16 or g.numel() != 128 or not g.is_contiguous():
                raise ValueError("qkv_append: q_norm and k_norm are contiguous bfloat16 [128]")
            if g.get_device() != dev:
                raise ValueError("qkv_append: all tensors must be on one CUDA device")
        gains = q_norm.data_ptr(), k_norm.data_ptr()
    if cos is not None or sin is not None:
        if cos is None or sin is None or tok_pos is None:
            raise ValueError("qkv_append: give cos, sin and tok_pos, or none of them")
        _int32("qkv_append", "tok_pos", (tok_pos,), dev)
        rope = cos.shape
        for c in (cos, sin):
            if c.dtype is not torch.float32 or c.dim() != 2 or c.shape[1] != 64 or not c.is_contiguous():
                raise ValueError("qkv_append: cos and sin are contiguous float32 [rows, 64]")
            if c.get_device() != dev:
                raise ValueError("qkv_append: all tensors must be on one CUDA device")
        if rope != sin.shape or tok_pos.numel() != tokens:
            raise ValueError("qkv_append: cos and sin have one shape and tok_pos is [T]")
        table, at, rope_rows = (cos.data_ptr(), sin.data_ptr()), tok_pos.data_ptr(), rope[0]
    if q_out.get_device() != dev or pool.get_device() != dev:
        raise ValueError("qkv_append: all tensors must be on one CUDA device")
    _launch("qkv_append", N.lib().lrm_op_qkv_append, _APPEND.pack(
        qkv.data_ptr(), *gains, *table, at, slot_map.data_ptr(), q_out.data_ptr(), pool.data_ptr(),
        ld_qkv if tokens > 1 else shape[1], ld_q, tokens, q_heads, kv_heads, 128, rope_rows, pool_shape[0], eps), dev,
        stream)


def paged_attention_workspace(tokens, q_heads, kv_heads) -> int:
    """Bytes of workspace for paged_attention calls of up to `tokens` rows, on the current device; 0 for sizes that no
    call has."""
    return int(N.lib().lrm_op_paged_attention_workspace(tokens, q_heads, kv_heads))


def paged_attention(q, pool, page_table, slots, cu_seqlens, kv_len, out, workspace, scale, stream=None):
    """Causal GQA attention of new tokens over the paged cache: rows cu_seqlens[i] .. cu_seqlens[i + 1] - 1 of q
    [T, q_heads, 128] (bfloat16, rows may be strided, as may out's) are the last tokens of the kv_len[i] keys of slot
    slots[i], read through page_table [max_seqs, pages_per_seq] from pool [pages, kv_heads, 2, 16, 128]. Rows of no
    request are left as they were. workspace: paged_attention_workspace(T, ...) bytes, any contents."""
    bf16, dev = _t().bfloat16, q.get_device()
    _pool("paged_attention", pool)
    shape, pool_shape, table = q.shape, pool.shape, page_table.shape
    if q.dtype is not bf16 or out.dtype is not bf16 or len(shape) != 3 or shape[2] != 128 or out.shape != shape:
        raise ValueError("paged_attention: q and out must be bfloat16 [T, q_heads, 128]")
    ld_q, ld_out = _rows_of_heads(q, shape), _rows_of_heads(out, shape)
    if ld_q is None or ld_out is None:
        raise ValueError("paged_attention: only the rows of q and out may be strided")
    _int32("paged_attention", "page_table slots cu_seqlens kv_len", (page_table, slots, cu_seqlens, kv_len), dev)
    (tokens, q_heads, _), kv_heads, n = shape, pool_shape[1], slots.numel()
    if len(table) != 2 or kv_len.numel() != n or cu_seqlens.numel() != n + 1:
        raise ValueError("paged_attention: page_table is [max_seqs, pages_per_seq], kv_len [requests], cu_seqlens "
                         "[requests + 1]")
    if out.get_device() != dev or pool.get_device() != dev or workspace.get_device() != dev:
        raise ValueError("paged_attention: all tensors must be on one CUDA device")
    if not workspace.is_contiguous():
        raise ValueError("paged_attention: the workspace must be contiguous")
    _launch("paged_attention", N.lib().lrm_op_paged_attention, _ATTN.pack(
        q.data_ptr(), pool.data_ptr(), page_table.data_ptr(), slots.data_ptr(), cu_seqlens.data_ptr(),
        kv_len.data_ptr(), out.data_ptr(), workspace.data_ptr(), ld_q, ld_out, workspace.nbytes, n, tokens, q_heads,
        kv_heads, 128, table[0], table[1], pool_shape[0], scale), dev, stream)
