"""Cases of the operators of a paged serving step: page plan, q/k/v append, paged attention and page release.

Layout (that of the decode attention and of the engine's cache): pool bf16 [pages][kv_heads][2 (K, V)][16][128],
page_table int32 [slots][pages_per_seq], lengths int32 by slot. ``run`` computes an operator in elementary torch
operations, or through ``rosylnalive_b200.ops`` when ``own`` is true.
"""

import math

import numpy as np
import torch

own = False

PAGE, HD = 16, 128
DEV = "cuda"


# ---- cases ----------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one decode step of 64 sequences with about 4096 cached tokens: a page is taken now and then
        dict(name="plan-decode-64", op="plan", requests=64, chunks=0, new_lo=1, new_hi=1, past_lo=4000, past_hi=4352,
             idle=0, spare=0, lens=1),
        # a full server's step: decodes, prefill chunks of odd lengths, fresh sequences, idle rows and a padded batch
        dict(name="plan-mixed-2000", op="plan", requests=2000, chunks=600, new_lo=3, new_hi=259, past_lo=0,
             past_hi=6000, idle=48, spare=1234, lens=2),
        # the same decode step's q/k/v rows: latency counts
        dict(name="append-decode-64", op="append", requests=64, chunks=0, new_lo=1, new_hi=1, past_lo=4000,
             past_hi=4352, idle=0, spare=0, q_heads=16, kv_heads=8, extra=0, lens=3),
        # a prefill of 16 prompts of 2048 tokens
        dict(name="append-prefill-16x2048", op="append", requests=16, chunks=16, new_lo=2048, new_hi=2048, past_lo=0,
             past_hi=0, idle=0, spare=0, q_heads=16, kv_heads=8, extra=0, lens=4),
        # one interactive sequence, one new token: latency counts
        dict(name="attn-decode-1", op="attn", requests=1, chunks=0, new_lo=1, new_hi=1, past_lo=900, past_hi=900,
             idle=0, spare=0, q_heads=16, kv_heads=8, extra=0, lens=6),
        # batched decode: 64 sequences with 4096 and more cached tokens
        dict(name="attn-decode-64x4096", op="attn", requests=64, chunks=0, new_lo=1, new_hi=1, past_lo=4096,
             past_hi=4352, idle=0, spare=0, q_heads=16, kv_heads=8, extra=0, lens=7),
        # drafted tokens verified in one step, five to a sequence, lengths far apart, four query heads a KV head
        dict(name="attn-verify-32x5", op="attn", requests=32, chunks=32, new_lo=5, new_hi=5, past_lo=100, past_hi=6000,
             idle=0, spare=3, q_heads=32, kv_heads=8, extra=0, lens=8),
        # a prefill chunk of one long prompt: many keys, few rows
        dict(name="attn-chunk-1000-on-120k", op="attn", requests=1, chunks=1, new_lo=1000, new_hi=1000, past_lo=120001,
             past_hi=120001, idle=0, spare=0, q_heads=16, kv_heads=8, extra=0, lens=9),
        # prefill chunks among decode rows, as a server batches them; q is a view of the fused q/k/v rows
        dict(name="attn-mixed-8x511-56", op="attn", requests=64, chunks=8, new_lo=511, new_hi=511, past_lo=0,
             past_hi=3000, idle=0, spare=17, q_heads=16, kv_heads=8, extra=2048, lens=10),
        # a prefill of 16 prompts of 2048 tokens
        dict(name="attn-prefill-16x2048", op="attn", requests=16, chunks=16, new_lo=2048, new_hi=2048, past_lo=0,
             past_hi=0, idle=0, spare=0, q_heads=16, kv_heads=8, extra=0, lens=11),
        # a few sequences that end, or lose the tokens of a refused draft
        dict(name="release-40", op="release", requests=40, chunks=0, new_lo=1, new_hi=1, past_lo=1, past_hi=4352,
             idle=0, spare=0, lens=5),
        # a full server's sequences that end, and others cut back to a kept prefix
        dict(name="release-1500", op="release", requests=1500, chunks=0, new_lo=1, new_hi=1, past_lo=1, past_hi=6000,
             idle=20, spare=0, lens=12),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


GROUPS = ((16, 8), (8, 8), (32, 8), (40, 8), (64, 8), (32, 4), (64, 4), (2, 1), (6, 2))


def draw(rng):
    op = rng.choice(("plan", "append", "append", "attn", "attn", "attn", "attn", "release"))
    lens = rng.randrange(1 << 30)
    if op in ("plan", "release"):
        requests = _log_int(rng, 1, 2000)
        return dict(op=op, requests=requests, chunks=rng.randint(0, requests) if op == "plan" else 0, new_lo=2,
                    new_hi=rng.randint(2, 259), past_lo=0 if op == "plan" else 1, past_hi=_log_int(rng, 20, 6000),
                    idle=rng.randint(0, 20), spare=rng.randint(0, 999) if op == "plan" else 0, lens=lens)
    q_heads, kv_heads = rng.choice(GROUPS)
    requests = _log_int(rng, 1, 64)
    case = dict(op=op, requests=requests, chunks=rng.randint(0, requests), new_lo=2, new_hi=_log_int(rng, 2, 2048),
                past_lo=rng.choice((0, 10, 300)), past_hi=_log_int(rng, 300, 8000 if requests > 3 else 60000),
                idle=rng.randint(0, 2), spare=rng.choice((0, 1, 50)), q_heads=q_heads, kv_heads=kv_heads,
                extra=rng.choice((0, 8, 256)), lens=lens)
    while not _affordable(case):
        case["new_hi"] = max(2, case["new_hi"] * 3 // 4)
        case["past_hi"] = max(case["past_lo"], case["past_hi"] * 3 // 4)
        case["requests"] = max(1, case["requests"] * 7 // 8)
        case["chunks"] = min(case["chunks"], case["requests"])
    return case


def _affordable(case):
    """Whether a drawn case costs no more than the largest listed one of its kind."""
    w = work(case)
    if case["op"] == "append":
        return w["bytes"] <= 4e8
    new, past = _lengths(case)
    padded = len(new) * int(max(new)) * int(max(new + past)) * case["q_heads"]
    gathered = len(new) * int(max(new + past)) * case["kv_heads"]
    return w["bytes"] <= 1.1e9 and w["flops"] <= 9e11 and padded <= 1.8e9 and gathered <= 5e6


def _lengths(case):
    """New and cached tokens of each request: `chunks` of new_lo .. new_hi, the rest single tokens, in mixed order."""
    r = np.random.RandomState(case["lens"])

    def spread(lo, hi, n):  # log-uniform whole numbers, 0 among them when lo is 0
        return np.floor(np.exp(r.uniform(math.log(lo + 1), math.log(hi + 2), n)) - 1).astype(np.int64).clip(lo, hi)

    n = case["requests"]
    new = np.ones(n, np.int64)
    new[: case["chunks"]] = spread(case["new_lo"], case["new_hi"], case["chunks"])
    new = new[r.permutation(n)]
    past = spread(case["past_lo"], case["past_hi"], n)
    return new, past


def work(case):
    new, past = _lengths(case)
    kv, tokens = new + past, int(new.sum())
    held, need = -(-past // PAGE), -(-kv // PAGE)
    rows = case["requests"] + case["idle"]
    if case["op"] == "plan":
        touched = int((need - past // PAGE).sum())
        return {"bytes": 12 * rows + 4 * (rows + 1) + 8 * rows + 8 * int((need - held).sum())
                + 4 * touched + 8 * (tokens + case["spare"]), "flops": 0}
    if case["op"] == "release":
        kept = _kept(case, past)
        return {"bytes": 16 * rows + 8 * int((held - -(-kept // PAGE)).sum()), "flops": 0}
    qh, kvh = case["q_heads"], case["kv_heads"]
    if case["op"] == "append":
        heads = qh + 2 * kvh
        positions = min(tokens, int(kv.max()))
        return {"bytes": tokens * (2 * heads * HD * 2 + 8) + positions * HD * 4, "flops": 10 * tokens * heads * HD}
    pairs = int((new * past + new * (new + 1) // 2).sum())
    return {"bytes": int(kv.sum()) * kvh * HD * 4 + 2 * tokens * qh * HD * 2 + 4 * int(need.sum()),
            "flops": 4 * pairs * qh * HD}


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _kept(case, past):
    """Tokens a release keeps: none for two sequences in three, a prefix of the others."""
    r = np.random.RandomState(case["lens"] ^ 0x5EED)
    kept = np.floor(r.uniform(0, 1, len(past)) * (past + 1)).astype(np.int64)
    kept[r.uniform(0, 1, len(past)) < 0.67] = 0
    return kept


def _i32(x):
    return torch.as_tensor(np.ascontiguousarray(x), dtype=torch.int32).to(DEV)


def prepare(case, seed):
    """The device state of a server before the call: lengths, page table, free pages, and the call's rows."""
    r = np.random.RandomState((seed * 7919 + 11) % (1 << 31))
    g = torch.Generator(device=DEV).manual_seed(seed)
    op = case["op"]
    new, past = _lengths(case)
    n, rows = case["requests"], case["requests"] + case["idle"]
    kv = new + past
    cached = past if op in ("plan", "release") else kv  # tokens whose pages are held already
    held = -(-cached // PAGE)
    slots_total = n + 3
    per_seq = int((-(-kv // PAGE)).max()) + 2
    slot_of = r.permutation(slots_total)[:n]
    need = int((-(-kv // PAGE)).sum())
    pages = need + need // 16 + 2  # a few more than needed; the last one stays unused
    order = r.permutation(pages - 1)
    table = np.zeros((slots_total, per_seq), np.int32)
    owner = np.repeat(np.arange(n), held)
    first = np.cumsum(held) - held
    table[slot_of[owner], np.arange(int(held.sum())) - first[owner]] = order[: int(held.sum())]
    place = np.sort(r.permutation(rows)[:n])  # where the live requests stand among the padded rows
    slots, new_rows, kv_rows = np.full(rows, -1), np.zeros(rows, np.int64), np.zeros(rows, np.int64)
    slots[place], new_rows[place], kv_rows[place] = slot_of, new, kv
    tokens = int(new.sum())
    cap = tokens + case["spare"]
    s = dict(case=case, op=op, slots=_i32(slots), table=_i32(table))
    if op in ("plan", "release"):
        seq_len = np.zeros(slots_total, np.int64)
        seq_len[slot_of] = past
        spare_pages = order[int(held.sum()):]
        free = np.zeros(pages, np.int32)
        free[: len(spare_pages)] = spare_pages
        s.update(seq_len=_i32(seq_len), free=_i32(free), count=_i32([len(spare_pages)]))
        s.update(seq_len_out=s["seq_len"].clone(), count_out=torch.zeros_like(s["count"]))
        if op == "release":
            keep = np.zeros(rows, np.int64)
            keep[place] = _kept(case, past)
            s.update(keep=_i32(keep))
            return s
        s.update(new=_i32(new_rows), cu=torch.empty(rows + 1, dtype=torch.int32, device=DEV),
                 kv_len=torch.empty(rows, dtype=torch.int32, device=DEV),
                 tok_pos=torch.empty(cap, dtype=torch.int32, device=DEV),
                 slot_map=torch.empty(cap, dtype=torch.int32, device=DEV))
        return s
    qh, kvh = case["q_heads"], case["kv_heads"]
    cu = np.concatenate([[0], np.cumsum(new_rows)])

    def bf16(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.bfloat16).mul_(scale)

    s.update(pool=bf16(pages, kvh, 2, PAGE, HD))
    if op == "append":
        req = np.repeat(np.arange(rows), new_rows)
        pos = kv_rows[req] - new_rows[req] + np.arange(tokens) - cu[req]
        slot_map = np.full(cap, -1)
        slot_map[:tokens] = table[slots[req], pos // PAGE].astype(np.int64) * PAGE + pos % PAGE
        tok_pos = np.zeros(cap, np.int64)
        tok_pos[:tokens] = pos
        positions = int(kv.max())
        inv = torch.exp(torch.arange(64, device=DEV, dtype=torch.float64) * (-math.log(1e6) / 64))
        angle = torch.arange(positions, device=DEV, dtype=torch.float64)[:, None] * inv
        s.update(qkv=bf16(cap, (qh + 2 * kvh) * HD + case["extra"])[:, : (qh + 2 * kvh) * HD], eps=1e-6,
                 q_norm=bf16(HD, scale=0.02) + 1, k_norm=bf16(HD, scale=0.02) + 1, cos=angle.cos().float(),
                 sin=angle.sin().float(), tok_pos=_i32(tok_pos), slot_map=_i32(slot_map),
                 q_out=torch.zeros(cap, qh, HD, dtype=torch.bfloat16, device=DEV))
        return s
    q = bf16(cap, qh * HD + case["extra"], scale=2.0)[:, : qh * HD].unflatten(1, (qh, HD))
    s.update(q=q, cu=_i32(cu), kv_len=_i32(kv_rows), scale=HD ** -0.5, max_new=int(new.max()), max_kv=int(kv.max()),
             out=torch.zeros(cap, qh, HD, dtype=torch.bfloat16, device=DEV))
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------

def run(s):
    if own:
        return _own(s)
    return {"plan": _plan, "append": _append, "attn": _attn, "release": _release}[s["op"]](s)


def _own(s):
    from rosylnalive_b200 import ops

    op = s["op"]
    if op == "plan":
        ops.page_plan(s["slots"], s["new"], s["seq_len"], s["table"], s["free"], s["count"], s["cu"], s["kv_len"],
                      s["tok_pos"], s["slot_map"], seq_len_out=s["seq_len_out"], free_count_out=s["count_out"])
        return {k: s[k] for k in ("table", "cu", "kv_len", "tok_pos", "slot_map", "seq_len_out", "count_out")}
    if op == "release":
        ops.page_release(s["slots"], s["keep"], s["seq_len"], s["table"], s["free"], s["count"],
                         seq_len_out=s["seq_len_out"], free_count_out=s["count_out"])
        return {k: s[k] for k in ("free", "seq_len_out", "count_out")}
    if op == "append":
        ops.qkv_append(s["qkv"], s["q_norm"], s["k_norm"], s["eps"], s["cos"], s["sin"], s["tok_pos"], s["slot_map"],
                       s["q_out"], s["pool"])
        return {"q_out": s["q_out"], "pool": s["pool"]}
    if "workspace" not in s:  # kept by the program, for all its calls in a row
        size = ops.paged_attention_workspace(s["q"].shape[0], s["q"].shape[1], s["pool"].shape[1])
        s["workspace"] = torch.empty(size, dtype=torch.uint8, device=DEV)
    ops.paged_attention(s["q"], s["pool"], s["table"], s["slots"], s["cu"], s["kv_len"], s["out"], s["workspace"],
                        s["scale"])
    return {"out": s["out"]}


def _exclusive(x):
    return torch.cumsum(x, 0) - x


def _plan(s):
    live = s["slots"] >= 0
    slot = s["slots"].clamp(min=0).long()
    new = torch.where(live, s["new"], 0).long()
    past = torch.where(live, s["seq_len"][slot], 0).long()
    kv = new + past
    held = (past + PAGE - 1) // PAGE
    count = (kv + PAGE - 1) // PAGE - held
    offset, start = _exclusive(count), _exclusive(new)
    # the pages taken, from the top of the free list; places past the last one go to a column that is cut off again
    j = torch.arange(s["free"].numel(), device=DEV)
    req = torch.searchsorted(offset + count, j, right=True)
    taken = req < slot.numel()
    req = req.clamp(max=slot.numel() - 1)
    width = s["table"].shape[1]
    wide = torch.cat([s["table"], s["table"][:, :1]], 1)
    at = slot[req] * (width + 1) + torch.where(taken, held[req] + j - offset[req], width)
    page = s["free"][(s["count"].long() - 1 - j).clamp(min=0)]
    wide.view(-1).scatter_(0, at, page)
    s["table"].copy_(wide[:, :width])
    s["cu"][0] = 0
    s["cu"][1:] = (start + new).int()
    s["kv_len"].copy_(kv)
    t = torch.arange(s["tok_pos"].numel(), device=DEV)
    req = torch.searchsorted(start + new, t, right=True)
    real = req < slot.numel()
    req = req.clamp(max=slot.numel() - 1)
    pos = torch.where(real, past[req] + t - start[req], 0)
    place = s["table"][slot[req], pos // PAGE].long() * PAGE + pos % PAGE
    s["tok_pos"].copy_(pos)
    s["slot_map"].copy_(torch.where(real, place, -1))
    lens = torch.cat([s["seq_len"], s["seq_len"][:1]])
    s["seq_len_out"].copy_(lens.scatter_(0, torch.where(live, slot, lens.numel() - 1), kv.int())[:-1])
    s["count_out"].copy_(s["count"] - count.sum())
    return {k: s[k] for k in ("table", "cu", "kv_len", "tok_pos", "slot_map", "seq_len_out", "count_out")}


def _release(s):
    live = s["slots"] >= 0
    slot = s["slots"].clamp(min=0).long()
    past = torch.where(live, s["seq_len"][slot], 0).long()
    keep = torch.where(live, s["keep"], 0).long()
    first = (keep + PAGE - 1) // PAGE
    count = (past + PAGE - 1) // PAGE - first
    offset = _exclusive(count)
    j = torch.arange(s["free"].numel(), device=DEV)
    req = torch.searchsorted(offset + count, j, right=True)
    given = req < slot.numel()
    req = req.clamp(max=slot.numel() - 1)
    column = torch.where(given, first[req] + j - offset[req], 0)
    page = s["table"][slot[req], column]
    wide = torch.cat([s["free"], s["free"][:1]])
    end = s["free"].numel()
    wide.scatter_(0, torch.where(given, s["count"].long() + j, end).clamp(max=end), page)
    s["free"].copy_(wide[:-1])
    lens = torch.cat([s["seq_len"], s["seq_len"][:1]])
    s["seq_len_out"].copy_(lens.scatter_(0, torch.where(live, slot, lens.numel() - 1), keep.int())[:-1])
    s["count_out"].copy_(s["count"] + count.sum())
    return {k: s[k] for k in ("free", "seq_len_out", "count_out")}


def _rotated(x, gain, s, cos, sin):
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + s["eps"]) * gain.float()
    a, b = y[..., :64], y[..., 64:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _append(s):
    qh, kvh = s["case"]["q_heads"], s["case"]["kv_heads"]
    rows = s["qkv"].float().unflatten(1, (qh + 2 * kvh, HD))
    real = s["slot_map"] >= 0
    cos, sin = (t[s["tok_pos"].long()][:, None] for t in (s["cos"], s["sin"]))
    q = _rotated(rows[:, :qh], s["q_norm"], s, cos, sin).bfloat16()
    k = _rotated(rows[:, qh : qh + kvh], s["k_norm"], s, cos, sin).bfloat16()
    v = rows[:, qh + kvh :].bfloat16()
    s["q_out"].copy_(torch.where(real[:, None, None], q, s["q_out"]))
    # rows of the padding write the unused last page's own first values back
    pool = s["pool"]
    page = torch.where(real, s["slot_map"] // PAGE, pool.shape[0] - 1).long()
    off = torch.where(real, s["slot_map"] % PAGE, 0).long()
    kv = torch.where(real[:, None, None, None], torch.stack([k, v], 2), pool[-1, None, :, :, 0])
    pool[page, :, :, off] = kv
    return {"q_out": s["q_out"], "pool": pool}


def _attn(s):
    q, pool, cu = s["q"], s["pool"], s["cu"].long()
    qh, kvh = q.shape[1], pool.shape[1]
    group, most, wide = qh // kvh, s["max_new"], -(-s["max_kv"] // PAGE)
    new, kv = cu[1:] - cu[:-1], s["kv_len"].long()
    held = pool[s["table"][s["slots"].clamp(min=0).long(), :wide].long()]  # [R, pages, kvh, 2, 16, 128]
    k, v = (held[:, :, :, c].transpose(1, 2).flatten(2, 3).float() for c in (0, 1))  # [R, kvh, keys, 128]
    i = torch.arange(most, device=DEV)
    at = (cu[:-1, None] + i).clamp(max=q.shape[0] - 1)
    rows = q[at].float().unflatten(2, (kvh, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [R, kvh, most * group, 128]
    p = torch.matmul(rows, k.transpose(2, 3)).mul_(s["scale"])
    last = (kv - new)[:, None] + i  # the last key that a row sees
    seen = torch.arange(k.shape[2], device=DEV) <= last[:, :, None]
    p = p.unflatten(2, (most, group)).masked_fill_(~seen[:, None, :, None], -math.inf).flatten(2, 3)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    o = o.unflatten(2, (most, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [R, most, qh, 128]
    t = torch.arange(q.shape[0], device=DEV)
    req = torch.searchsorted(cu[1:], t, right=True)
    real = req < new.numel()
    req = req.clamp(max=new.numel() - 1)
    o = o[req, (t - cu[req]).clamp(max=most - 1)].bfloat16()
    s["out"].copy_(torch.where(real[:, None, None], o, s["out"]))
    return {"out": s["out"]}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def exact(case, seed):
    """The computed outputs from the operators' definitions, one request (append: all rows of one head) at a time."""
    if case["op"] in ("plan", "release"):
        return None  # whole numbers
    s = prepare(case, seed)
    qh, kvh = case["q_heads"], case["kv_heads"]
    pool = s["pool"].double()
    if case["op"] == "append":
        out = s["q_out"].double()
        live = torch.nonzero(s["slot_map"] >= 0)[:, 0]
        where = s["slot_map"][live].long()
        cos, sin = s["cos"].double()[s["tok_pos"][live].long()], s["sin"].double()[s["tok_pos"][live].long()]
        for h in range(qh + 2 * kvh):
            x = s["qkv"][live, h * HD : (h + 1) * HD].double()
            if h < qh + kvh:
                norm = torch.sqrt((x * x).sum(1) / HD + s["eps"])
                x = x / norm[:, None] * s["q_norm" if h < qh else "k_norm"].double()
                lo, hi = x[:, :64].clone(), x[:, 64:].clone()
                x = torch.hstack([lo * cos - hi * sin, hi * cos + lo * sin])
            if h < qh:
                out[live, h] = x
            else:
                pool[where // PAGE, (h - qh) % kvh, (h - qh) // kvh, where % PAGE] = x
        return {"q_out": out, "pool": pool}
    out = s["out"].double()
    cu, kv, slots = s["cu"].tolist(), s["kv_len"].tolist(), s["slots"].tolist()
    for i, slot in enumerate(slots):
        n = cu[i + 1] - cu[i]
        if n == 0:
            continue
        pages = s["table"][slot, : -(-kv[i] // PAGE)].long()
        key, value = (pool[pages, :, c].permute(1, 0, 2, 3).reshape(kvh, -1, HD)[:, : kv[i]] for c in (0, 1))
        for a in range(0, n, 128):
            b = min(n, a + 128)
            q = s["q"][cu[i] + a : cu[i] + b].double()  # [rows, qh, 128]
            hidden = torch.arange(kv[i], device=DEV)[None, :] > torch.arange(kv[i] - n + a, kv[i] - n + b, device=DEV)[:, None]
            for h in range(qh):
                score = (q[:, h] @ key[h // (qh // kvh)].T) * s["scale"]
                weight = torch.softmax(score.masked_fill(hidden, -math.inf), 1)
                out[cu[i] + a : cu[i] + b, h] = weight @ value[h // (qh // kvh)]
    return {"out": out}
