"""The paged serving step's operators (ops.page_plan, qkv_append, paged_attention, page_release) on the GPU, against
plain implementations: Python lists for the bookkeeping, 64 bits for the numbers.

Tolerances, from the arithmetic:
  append     y = x gain / sqrt(mean x^2 + eps) and the rotation in fp32 (a sum of 128 squares in 8 + 4 steps, a square
             root, a division, two products: under 32 roundings of 2^-24), then one rounding to bf16 (2^-8):
             2^-8 |ref| + 2^-19 (|y_d cos| + |y_d+64 sin|). v is copied: equal bits.
  attention  scores are fp32 sums of 128 products: off by ds <= 130 * 2^-24 * scale * sum |q_d k_d|, so a weight is off
             by 2 ds + 2^-20 (its exponential included); weights are rounded to bf16 before the product with v (2^-8);
             sums over n keys are fp32 (at most n / 16 + 300 additions, 2^-23 each). All act on sum p |v| / sum p = A,
             twice (numerator and denominator) but for the rounding of the weights. Then one rounding to bf16:
             2^-8 |ref| + (2^-8 + 2 (2 ds + 2^-20 + (n / 16 + 300) 2^-23)) A.
"""

import numpy as np
import pytest

from tests.conftest import cuda_available

pytestmark = pytest.mark.gpu

if cuda_available():
    import torch

    from rosylnalive_b200 import ops

HD, PAGE = 128, 16
SCALE = HD ** -0.5


@pytest.fixture(autouse=True)
def _device():
    ops.set_device(0)
    yield
    torch.cuda.synchronize()
    assert ops.error_word() == 0


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def pages(n):
    return (n + PAGE - 1) // PAGE


# ---- plan and release: a model of the server in Python lists ---------------------------------------------------------

class Server:
    def __init__(self, max_seqs, pages_per_seq, kv_pages, seed=0):
        r = np.random.default_rng(seed)
        self.len = [0] * max_seqs
        self.own = [[] for _ in range(max_seqs)]
        self.free = [int(x) for x in r.permutation(kv_pages)]
        self.P, self.F = pages_per_seq, kv_pages
        self.seq_len = i32(self.len)
        self.table = i32(r.integers(0, kv_pages, (max_seqs, pages_per_seq)))
        self.stale = self.table.cpu().numpy().copy()
        self.free_list, self.count = i32(self.free), i32([kv_pages])

    def plan(self, slots, new):
        cu, kv, pos, smap = [0], [], [], []
        for s, n in zip(slots, new):
            n = 0 if s == -1 else n
            cu.append(cu[-1] + n)
            if s == -1:
                kv.append(0)
                continue
            while len(self.own[s]) < pages(self.len[s] + n):
                self.stale[s, len(self.own[s])] = self.free[-1]
                self.own[s].append(self.free.pop())
            for p in range(self.len[s], self.len[s] + n):
                pos.append(p)
                smap.append(self.own[s][p // PAGE] * PAGE + p % PAGE)
            self.len[s] += n
            kv.append(self.len[s])
        return cu, kv, pos, smap

    def release(self, slots, keep):
        for s, k in zip(slots, keep):
            if s == -1:
                continue
            self.free += self.own[s][pages(k):]
            self.own[s] = self.own[s][:pages(k)]
            self.len[s] = k

    def same_state(self):
        assert self.seq_len.tolist() == self.len
        assert int(self.count) == len(self.free)
        assert self.free_list[: len(self.free)].tolist() == self.free
        assert np.array_equal(self.table.cpu().numpy(), self.stale)  # new entries written, all others left


def step_buffers(requests, max_tokens):
    f = lambda n: torch.full((n,), -77, dtype=torch.int32, device="cuda")  # noqa: E731
    return f(requests + 1), f(requests), f(max_tokens), f(max_tokens)


def gpu_plan(sv, slots, new, max_tokens, **kw):
    bufs = step_buffers(len(slots), max_tokens)
    ops.page_plan(i32(slots), i32(new), sv.seq_len, sv.table, sv.free_list, sv.count, *bufs, **kw)
    torch.cuda.synchronize()
    return [b.tolist() for b in bufs]


def check_plan(sv, slots, new, max_tokens):
    got = gpu_plan(sv, slots, new, max_tokens)
    cu, kv, pos, smap = sv.plan(slots, new)
    pad = max_tokens - len(pos)
    assert got[0] == cu and got[1] == kv
    assert got[2] == pos + [0] * pad
    assert got[3] == smap + [-1] * pad
    sv.same_state()


def gpu_release(sv, slots, keep, **kw):
    ops.page_release(i32(slots), i32(keep), sv.seq_len, sv.table, sv.free_list, sv.count, **kw)
    torch.cuda.synchronize()


@pytest.mark.parametrize("requests,max_seqs,cap", [(1, 1, 40), (5, 9, 90), (64, 70, 300), (1023, 1030, 100),
                                                   (1024, 2000, 60), (1025, 1100, 100), (2600, 4000, 50)])
def test_plan_and_release_follow_the_lists(requests, max_seqs, cap):
    r = np.random.default_rng(requests)
    P = pages(cap)
    sv = Server(max_seqs, P, max_seqs * P, seed=requests)
    for step in range(6):
        slots = r.permutation(max_seqs)[:requests]
        slots = np.where(r.uniform(size=requests) < 0.1, -1, slots)  # a padded batch
        room = np.array([0 if s == -1 else cap - sv.len[s] for s in slots])
        new = np.minimum(r.choice([0, 1, 1, 2, 15, 16, 17, 33], requests), room)
        new[slots == -1] = -9  # not read
        total = int(new[slots != -1].sum())
        check_plan(sv, slots.tolist(), new.tolist(), max(1, total + int(r.choice([0, 1, 700, 5000]))))
        slots = r.permutation(max_seqs)[:requests]
        slots = np.where(r.uniform(size=requests) < 0.1, -1, slots)
        keep = [0 if s == -1 else int(r.integers(0, sv.len[s] + 1)) if r.uniform() < 0.5 else (0, sv.len[s])[step % 2]
                for s in slots]
        gpu_release(sv, slots.tolist(), keep)
        sv.release(slots.tolist(), keep)
        sv.same_state()


def test_plan_and_release_of_more_requests_than_one_pass_of_the_cluster():
    max_seqs, requests, P = 20000, 9001, 3
    sv = Server(max_seqs, P, max_seqs * P, seed=5)
    r = np.random.default_rng(5)
    for step in range(2):
        slots = r.permutation(max_seqs)[:requests]
        slots = np.where(r.uniform(size=requests) < 0.1, -1, slots)
        new = np.array([0 if s == -1 else min(int(r.integers(0, 25)), 48 - sv.len[s]) for s in slots])
        check_plan(sv, slots.tolist(), new.tolist(), int(new.sum()) + 3)
        slots = r.permutation(max_seqs)[:requests]
        keep = [int(r.integers(0, sv.len[s] + 1)) for s in slots]
        gpu_release(sv, slots.tolist(), keep)
        sv.release(slots.tolist(), keep)
        sv.same_state()


@pytest.mark.parametrize("shift", [0, 1, 2, 3])
def test_a_large_plan_writes_rows_at_any_alignment(shift):
    # Above 5120 rows the outputs are written 16 bytes at a time where they can be.
    requests, max_seqs, P = 300, 300, 12
    sv = Server(max_seqs, P, max_seqs * P, seed=shift)
    slots = np.random.default_rng(9).permutation(max_seqs).tolist()
    new = np.random.default_rng(8).integers(0, 60, requests).tolist()
    max_tokens = 12000
    big = [torch.full((max_tokens + 4,), -77, dtype=torch.int32, device="cuda") for _ in range(2)]
    pos, smap = [b[shift: shift + max_tokens] for b in big]
    cu, kv = step_buffers(requests, 1)[:2]
    ops.page_plan(i32(slots), i32(new), sv.seq_len, sv.table, sv.free_list, sv.count, cu, kv, pos, smap)
    want = sv.plan(slots, new)
    pad = max_tokens - len(want[2])
    assert cu.tolist() == want[0] and kv.tolist() == want[1]
    assert pos.tolist() == want[2] + [0] * pad and smap.tolist() == want[3] + [-1] * pad
    for b in big:
        assert b[:shift].tolist() == [-77] * shift and b[shift + max_tokens:].tolist() == [-77] * (4 - shift)
    sv.same_state()


def test_plan_takes_the_very_last_page_and_fills_a_row():
    sv = Server(2, 3, 4, seed=3)
    check_plan(sv, [1, 0], [48, 16], 64)
    assert int(sv.count) == 0
    check_plan(sv, [0, 1], [0, 0], 1)  # no tokens at all


def test_plan_writes_beside_the_state_when_asked():
    sv = Server(4, 5, 20, seed=4)
    check_plan(sv, [2, 0], [20, 7], 30)
    before, count = sv.seq_len.clone(), sv.count.clone()
    lens, left = torch.full_like(sv.seq_len, -5), torch.full_like(sv.count, -5)
    for _ in range(2):  # the same call again gives the same step
        got = gpu_plan(sv, [0, -1, 3], [10, 0, 4], 14, seq_len_out=lens, free_count_out=left)
        assert got[0] == [0, 10, 10, 14] and got[1] == [17, 0, 4]
        assert lens.tolist() == [17, -5, -5, 4]  # only the call's slots are written
        assert int(left) == int(count) - 2
        assert torch.equal(sv.seq_len, before) and torch.equal(sv.count, count)
    lens.fill_(-5), left.fill_(-5)
    tail = sv.free_list.clone()
    gpu_release(sv, [2], [3], seq_len_out=lens, free_count_out=left)
    assert lens.tolist() == [-5, -5, 3, -5] and int(left) == int(count) + 1
    assert torch.equal(sv.seq_len, before) and torch.equal(sv.count, count)
    tail[int(count)] = sv.table[2, 1]
    assert torch.equal(sv.free_list, tail)


BAD_PLANS = {
    "slot past the end": ([0, 4], [1, 1], 8, 0x5001), "slot below -1": ([0, -2], [1, 1], 8, 0x5001),
    "slot twice": ([1, 0, 1], [1, 1, 0], 8, 0x5001), "negative tokens": ([0, 1], [1, -1], 8, 0x5001),
    "past the row": ([0, 1], [1, 49], 99, 0x5001), "huge": ([0, 1], [2**31 - 1, 2**31 - 1], 8, 0x5001),
    "pages": ([0, 1, 2], [48, 48, 1], 99, 0x5002), "tokens": ([0, 1], [4, 5], 8, 0x5003),
}


@pytest.mark.parametrize("name", BAD_PLANS)
@pytest.mark.parametrize("pad", [0, 1500])
def test_a_plan_that_breaks_a_rule_takes_nothing(name, pad):
    slots, new, max_tokens, code = BAD_PLANS[name]
    sv = Server(4, 3, 6, seed=6)
    slots, new = slots + [-1] * pad, new + [0] * pad
    got = gpu_plan(sv, slots, new, max_tokens)
    assert ops.error_word() == code
    assert got == [[0] * (len(slots) + 1), [0] * len(slots), [0] * max_tokens, [-1] * max_tokens]
    sv.same_state()
    lens = torch.full_like(sv.seq_len, -5)
    gpu_plan(sv, slots, new, max_tokens, seq_len_out=lens, free_count_out=torch.zeros_like(sv.count))
    assert ops.error_word() == code
    want = [0 if s in slots else -5 for s in range(4)]
    assert lens.tolist() == want


@pytest.mark.parametrize("what", ["count above", "count below", "id above", "id below", "old length"])
def test_a_plan_on_a_broken_state_takes_nothing(what):
    sv = Server(4, 3, 6, seed=7)
    if what.startswith("count"):
        sv.count.fill_(7 if what == "count above" else -1)
    elif what.startswith("id"):
        sv.free_list[4] = 6 if what == "id above" else -1
    else:
        sv.seq_len[1] = 49
    before = sv.table.clone(), sv.seq_len.clone(), sv.count.clone()
    got = gpu_plan(sv, [0, 1], [20, 10 if what != "old length" else 0], 40)
    assert ops.error_word() == (0x5001 if what == "old length" else 0x5004)
    assert got == [[0, 0, 0], [0, 0], [0] * 40, [-1] * 40]
    assert all(torch.equal(x, y) for x, y in zip(before, (sv.table, sv.seq_len, sv.count)))


def test_a_held_page_outside_the_pool_is_not_mapped():
    sv = Server(2, 3, 6, seed=8)
    check_plan(sv, [0], [5], 5)
    sv.table[0, 0] = 6
    got = gpu_plan(sv, [0], [12], 12)
    assert ops.error_word() == 0x5005
    assert got[2] == list(range(5, 17)) and got[3][:11] == [-1] * 11 and got[3][11] >= 0


BAD_RELEASES = {"slot past the end": ([0, 4], [1, 1], 0x5011), "slot below -1": ([0, -2], [1, 1], 0x5011),
                "slot twice": ([1, 1], [0, 0], 0x5011), "keep above": ([0, 1], [0, 31], 0x5011),
                "keep below": ([0, 1], [0, -1], 0x5011)}


@pytest.mark.parametrize("name", list(BAD_RELEASES) + ["count", "page", "page, many requests"])
def test_a_release_that_breaks_a_rule_changes_nothing(name):
    sv = Server(4, 3, 9, seed=9)
    check_plan(sv, [0, 1], [40, 30], 70)
    slots, keep, code = BAD_RELEASES.get(name, ([0, 1], [0, 0], 0x5014))
    if name == "count":
        sv.count.fill_(7)
        code = 0x5012
    elif name.startswith("page"):
        sv.table[1, 1] = 9
    if name.endswith("many requests"):
        slots, keep = [-1] * 1300 + slots, [0] * 1300 + keep
    before = [x.clone() for x in (sv.table, sv.seq_len, sv.count, sv.free_list)]
    gpu_release(sv, slots, keep)
    assert ops.error_word() == code
    assert all(torch.equal(x, y) for x, y in zip(before, (sv.table, sv.seq_len, sv.count, sv.free_list)))


# ---- append ----------------------------------------------------------------------------------------------------------

def append_reference(qkv, gains, eps, cos, sin, pos, qh, kvh):
    """(rows [T, heads, 128] in 64 bits, their tolerance)."""
    x = qkv.double().cpu().unflatten(1, (qh + 2 * kvh, HD))
    y = x.clone()
    if gains:
        r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
        y[:, :qh] = x[:, :qh] * r[:, :qh] * gains[0].double().cpu()
        y[:, qh:qh + kvh] = x[:, qh:qh + kvh] * r[:, qh:qh + kvh] * gains[1].double().cpu()
    a, b = y[:, :qh + kvh, :64].clone(), y[:, :qh + kvh, 64:].clone()
    size = y.abs()
    if cos is not None:
        c, s = (t.double().cpu()[pos][:, None] for t in (cos, sin))
        y[:, :qh + kvh] = torch.cat([a * c - b * s, b * c + a * s], -1)
        size[:, :qh + kvh] = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()], -1)
    tol = 2.0 ** -8 * y.abs() + 2.0 ** -19 * size
    tol[:, qh + kvh:] = 0
    return y, tol


@pytest.mark.parametrize("qh,kvh,T,extra", [(16, 8, 1, 0), (16, 8, 64, 0), (40, 8, 37, 8), (1, 1, 5, 128), (7, 1, 130, 0),
                                            (64, 4, 19, 1024), (2, 2, 3, 0)])
@pytest.mark.parametrize("norm,rope", [(True, True), (False, True), (True, False), (False, False)])
def test_append(qh, kvh, T, extra, norm, rope):
    g = torch.Generator(device="cuda").manual_seed(qh * 1000 + T)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    cols = (qh + 2 * kvh) * HD
    wide = rnd(T, cols + extra) * 3
    qkv = wide[:, :cols]
    gains = [1 + 0.3 * rnd(HD), 1 + 0.3 * rnd(HD)] if norm else None
    ang = torch.rand(200, 64, generator=g, device="cuda") * 6
    cos, sin = (ang.cos(), ang.sin()) if rope else (None, None)
    F = T // PAGE + 3
    r = np.random.default_rng(T)
    places = r.permutation(F * PAGE)[:T]
    places[r.uniform(size=T) < 0.2] = -1
    pos = r.integers(0, 200, T)
    pos[0] = 199
    pool = rnd(F, kvh, 2, PAGE, HD)
    out = rnd(T, qh * HD + extra)[:, :qh * HD].unflatten(1, (qh, HD))
    ref_pool, ref_out = pool.clone(), out.clone()
    y, tol = append_reference(qkv, gains, 1e-6, cos, sin, pos, qh, kvh)
    kept = wide.clone()
    ops.qkv_append(qkv, *(gains or (None, None)), 1e-6, cos, sin, i32(pos) if rope else None, i32(places), out, pool)
    torch.cuda.synchronize()
    assert torch.equal(wide, kept)
    got = ref_out.double().cpu()
    for t in range(T):
        if places[t] >= 0:
            pg, off = places[t] // PAGE, places[t] % PAGE
            for c, h0 in ((0, qh), (1, qh + kvh)):
                d = (pool[pg, :, c, off].double().cpu() - y[t, h0:h0 + kvh]).abs()
                assert (d <= tol[t, h0:h0 + kvh]).all(), (t, c, float((d - tol[t, h0:h0 + kvh]).max()))
                ref_pool[pg, :, c, off] = pool[pg, :, c, off]
            d = (out[t].double().cpu() - y[t, :qh]).abs()
            assert (d <= tol[t, :qh]).all(), (t, float((d - tol[t, :qh]).max()))
            got[t] = out[t].double().cpu()
    assert torch.equal(pool, ref_pool) and torch.equal(out.double().cpu(), got)  # all else left as it was


def test_append_in_place_equals_append_beside():
    g = torch.Generator(device="cuda").manual_seed(1)
    qkv = torch.randn(50, 32 * HD, generator=g, device="cuda", dtype=torch.bfloat16)
    gain = 1 + 0.1 * torch.randn(HD, generator=g, device="cuda", dtype=torch.bfloat16)
    ang = torch.rand(60, 64, generator=g, device="cuda")
    pos, place = i32(np.arange(50)), i32(np.arange(50))
    pools = [torch.zeros(4, 8, 2, PAGE, HD, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    out = torch.zeros(50, 16, HD, device="cuda", dtype=torch.bfloat16)
    ops.qkv_append(qkv, gain, gain, 1e-6, ang.cos(), ang.sin(), pos, place, out, pools[0])
    view = qkv[:, :16 * HD].unflatten(1, (16, HD))
    ops.qkv_append(qkv, gain, gain, 1e-6, ang.cos(), ang.sin(), pos, place, view, pools[1])
    assert torch.equal(out, view) and torch.equal(pools[0], pools[1])


@pytest.mark.parametrize("bad", ["place above", "place below", "position above", "position below"])
def test_append_skips_a_row_outside_its_arrays(bad):
    qkv = torch.ones(3, 4 * HD, device="cuda", dtype=torch.bfloat16)
    pool = torch.zeros(2, 1, 2, PAGE, HD, device="cuda", dtype=torch.bfloat16)
    out = torch.zeros(3, 2, HD, device="cuda", dtype=torch.bfloat16)
    place, pos = [3, 4, 5], [0, 1, 2]
    if bad.startswith("place"):
        place[1] = 32 if bad == "place above" else -2
    else:
        pos[1] = 3 if bad == "position above" else -1
    table = torch.ones(3, 64, device="cuda")
    ops.qkv_append(qkv, None, None, 0.0, table, table, i32(pos), i32(place), out, pool)
    torch.cuda.synchronize()
    assert ops.error_word() == 0x6001
    assert float(out[1].abs().sum()) == 0 and float(pool[0, 0, :, 4].abs().sum()) == 0
    assert (pool[0, 0, 1, [3, 5]] == 1).all() and (out[0, 0, 64:] == 2).all()


def test_append_where_the_pool_passes_32_bits():
    # 600,000 pages of one head: elements past 2^31, bytes past 2^32
    pool = torch.zeros(600_000, 1, 2, PAGE, HD, device="cuda", dtype=torch.bfloat16)
    qkv = torch.arange(1, 3 * HD + 1, device="cuda", dtype=torch.float32).to(torch.bfloat16)[None].contiguous()
    out = torch.zeros(1, 1, HD, device="cuda", dtype=torch.bfloat16)
    ops.qkv_append(qkv, None, None, 0.0, None, None, None, i32([600_000 * PAGE - 1]), out, pool)
    assert torch.equal(pool[-1, 0, 0, 15], qkv[0, HD:2 * HD]) and torch.equal(pool[-1, 0, 1, 15], qkv[0, 2 * HD:])
    assert int((pool != 0).sum()) == 2 * HD


# ---- attention -------------------------------------------------------------------------------------------------------

class Cache:
    """Requests (new, kv) over a shuffled pool; unowned pages and the ends of last pages hold `stale`."""

    def __init__(self, reqs, qh, kvh, seed=0, stale=float("nan"), pad_q=0, pad_out=0, spare=0, gap=0, extra_pages=0, qscale=2.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = np.random.default_rng(seed)
        rnd = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=torch.bfloat16)  # noqa: E731
        self.reqs, self.qh, self.kvh = reqs, qh, kvh
        n = len(reqs)
        need = [pages(kv) for _, kv in reqs]
        P, F = max(max(need), 1) + 1, sum(need) + 3 + extra_pages
        order = r.permutation(F)
        table = r.integers(0, F, (n + 2, P))
        slot = r.permutation(n + 2)[:n]
        self.pool = torch.full((F, kvh, 2, PAGE, HD), stale, device="cuda", dtype=torch.bfloat16)
        self.k, self.v, at = [], [], 0
        for i, (_, kv) in enumerate(reqs):
            ids = order[at:at + need[i]]
            at += need[i]
            table[slot[i], :need[i]] = ids
            self.k.append(rnd(kv, kvh, HD))
            self.v.append(rnd(kv, kvh, HD))
            if kv:
                p = torch.arange(kv, device="cuda")
                pg = torch.tensor(ids, device="cuda")[p // PAGE]
                self.pool[pg, :, 0, p % PAGE] = self.k[i]
                self.pool[pg, :, 1, p % PAGE] = self.v[i]
        self.T = sum(a for a, _ in reqs) + gap + spare
        self.cu_host = np.concatenate([[0], np.cumsum([a for a, _ in reqs])]) + gap
        self.q = (rnd(self.T, qh * HD + pad_q) * qscale)[:, :qh * HD].unflatten(1, (qh, HD))
        self.out = rnd(self.T, qh * HD + pad_out)[:, :qh * HD].unflatten(1, (qh, HD))
        self.table, self.slots, self.cu = i32(table), i32(slot), i32(self.cu_host)
        self.kv_len = i32([kv for _, kv in reqs])
        self.ws = torch.full((ops.paged_attention_workspace(self.T, qh, kvh),), 0xFF, dtype=torch.uint8, device="cuda")

    def args(self):
        return (self.q, self.pool, self.table, self.slots, self.cu, self.kv_len, self.out, self.ws, SCALE)

    def run(self, **kw):
        ops.paged_attention(*self.args(), **kw)
        torch.cuda.synchronize()
        return self.out

    def reference(self, i):
        """Request i's rows in 64 bits and their tolerance. Values that are not finite reach only the rows that see
        their key; such a row's tolerance is infinite where the result is not finite."""
        n, kv = self.reqs[i]
        g = self.qh // self.kvh
        q = self.q[self.cu_host[i]:self.cu_host[i] + n].double().unflatten(1, (self.kvh, g))
        k, v = self.k[i].double(), self.v[i].double()
        hidden = torch.arange(kv, device="cuda")[None] > torch.arange(kv - n, kv, device="cuda")[:, None]
        ref, tol = torch.empty(n, self.kvh, g, HD, dtype=torch.float64, device="cuda"), None
        tol = torch.empty_like(ref)
        for h in range(self.kvh):
            s = torch.einsum("ngd,kd->ngk", q[:, h], k[:, h]) * SCALE
            s = s.masked_fill(hidden[:, None], -torch.inf)
            p = torch.softmax(s, -1)
            seen = p > 0
            fin = torch.nan_to_num(v[:, h], 0, 0, 0)
            ref[:, h] = torch.einsum("ngk,kd->ngd", torch.nan_to_num(p), fin)
            bad = ~torch.isfinite(v[:, h])
            if bad.any():
                for key in torch.nonzero(bad.any(1))[:, 0].tolist():
                    rows = ~hidden[:, key]
                    ref[rows, h] += torch.where(bad[key], v[key, h], 0.0)
            ds = 130 * 2.0 ** -24 * SCALE * torch.einsum("ngd,kd->ngk", q[:, h].abs(), k[:, h].abs())
            ds = torch.where(seen, ds, 0).amax(-1)
            A = torch.einsum("ngk,kd->ngd", torch.nan_to_num(p), fin.abs())
            tol[:, h] = 2.0 ** -8 * ref[:, h].abs() + (2.0 ** -8 + 2 * (
                2 * ds + 2.0 ** -20 + (kv / 16 + 300) * 2.0 ** -23))[..., None] * A
        return ref.flatten(1, 2), tol.flatten(1, 2)

    def check(self, out, before, only=None):
        seen = torch.zeros(self.T, dtype=torch.bool, device="cuda")
        for i, (n, kv) in enumerate(self.reqs):
            a = int(self.cu_host[i])
            if n == 0 or (only is not None and i not in only):
                continue
            seen[a:a + n] = True
            ref, tol = self.reference(i)
            got = out[a:a + n].double()
            fine = torch.isfinite(ref)
            assert torch.equal(torch.isnan(got), torch.isnan(ref)), (i, "NaN")
            inf = torch.isinf(ref)
            assert torch.equal(got[inf], ref[inf]), (i, "infinities")
            over = ((got - ref).abs() - tol)[fine]
            assert over.numel() == 0 or float(over.max()) <= 0, (i, n, kv, float(over.max()))
        assert torch.equal(out[~seen], before[~seen])  # rows of no request are left as they were


MIXES = {
    "one key": [(1, 1)],
    "single token": [(1, 900)],
    "edges of tiles and pages": [(1, 15), (1, 16), (1, 17), (1, 127), (1, 128), (1, 129), (1, 255), (1, 257)],
    "fresh chunks": [(1, 1), (2, 2), (63, 63), (64, 64), (65, 65), (127, 127), (128, 128), (129, 129), (300, 300)],
    "chunks on a cache": [(5, 400), (17, 129), (64, 1000), (65, 192), (100, 611), (200, 513)],
    "idle and mixed": [(0, 0), (1, 77), (0, 50), (130, 640), (1, 3000), (0, 0), (3, 3), (1, 1)],
    "one long, few rows": [(3, 20000)],
    "long chunk": [(700, 5000)],
    "many short": [(1, 1 + 7 * i % 300) for i in range(200)],
    "many long": [(1, 2500 + 37 * i) for i in range(40)],
    "all kinds in turn": [x for i in range(6) for x in ((1, 700 + i), (150, 900), (20, 400 + i), (3, 30), (40, 45), (1, 2))],
}


@pytest.mark.parametrize("heads", [(16, 8), (4, 4), (8, 2), (5, 1), (16, 1), (40, 8), (3, 3)])
@pytest.mark.parametrize("mix", MIXES)
def test_attention(mix, heads):
    c = Cache(MIXES[mix], *heads, seed=len(mix), pad_q=64, pad_out=8, spare=5, gap=2)
    before = c.out.clone()
    c.check(c.run(), before)


def test_attention_of_more_requests_than_a_block_has_threads():
    # 900 requests: a thread counts several of them, some without tokens.
    r = np.random.default_rng(3)
    new = r.choice([0, 1, 1, 1, 2, 30], 900)
    c = Cache([(int(n), int(n + p)) for n, p in zip(new, r.integers(0, 120, 900))], 6, 2, seed=13, spare=2)
    before = c.out.clone()
    c.check(c.run(), before)


@pytest.mark.parametrize("heads", [(64, 1), (100, 1), (128, 1), (33, 1), (256, 2)])
def test_attention_of_wide_groups(heads):
    c = Cache([(1, 200), (3, 130), (0, 0), (9, 9)], *heads, seed=2)
    before = c.out.clone()
    c.check(c.run(), before)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("heads", [(16, 8), (4, 4), (10, 1)])
def test_values_that_are_not_finite_reach_only_the_rows_that_see_them(value, what, heads):
    # Tokens 40, 100, 199 (and 300 of the second request) hold them: rows before must not change at all.
    c = Cache([(200, 200), (150, 400), (1, 90)], *heads, seed=5, stale=value)
    clean = c.run().clone()
    own = c.table.cpu().numpy()
    slots = c.slots.tolist()
    kv_of = (c.k, c.v)[what == "v"]
    first = {}
    for i, keys in ((0, (40, 100, 199)), (1, (300, 390))):
        first[i] = min(keys)
        for key in keys:
            pg = int(own[slots[i], key // PAGE])
            dims = slice(0, HD, 7) if what == "v" else slice(3, 4)
            c.pool[pg, :, int(what == "v"), key % PAGE, dims] = value
            kv_of[i][key, :, dims] = value
    before = c.out.clone()
    got = c.run().clone()
    if what == "v":
        c.check(got, before)
    for i, (n, kv) in enumerate(c.reqs):
        a = int(c.cu_host[i])
        sees = n if i not in first else max(0, first[i] - (kv - n))  # rows before the first such key
        assert torch.equal(got[a:a + sees], clean[a:a + sees]), i
        if i in first and value != value:
            assert torch.isnan(got[a + sees:a + n].float()).any()


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("heads", [(16, 8), (6, 2), (40, 8)])
def test_values_that_are_not_finite_in_many_short_requests(value, heads):
    # Short requests follow one another closely in a CTA, so that the values of one are looked at while the results of the
    # one before are still read out; all of them hold a value that only their later rows see.
    r = np.random.default_rng(1)
    new = r.choice([2, 3, 5, 17, 40, 70], 160).tolist()
    c = Cache([(n, n + int(p)) for n, p in zip(new, r.choice([0, 1, 20, 90], 160))], *heads, seed=31)
    own, slots = c.table.cpu().numpy(), c.slots.tolist()
    for i, (n, kv) in enumerate(c.reqs):
        key = kv - 1 - (n - 1) // 2
        c.pool[int(own[slots[i], key // PAGE]), :, 1, key % PAGE, i % 16::16] = value
        c.v[i][key, :, i % 16::16] = value
    before = c.out.clone()
    c.check(c.run(), before)


def test_keys_of_minus_infinity_weigh_nothing():
    # q = 1 in dim 0 and k = -inf there: scores of -inf at the first 140 keys, more than a whole tile of them
    c = Cache([(1, 300), (20, 300)], 4, 2, seed=6)
    c.q.zero_()
    c.q[..., 0] = 1
    for i in range(2):
        c.k[i][:140, :, 0] = float("-inf")
        p = torch.arange(300, device="cuda")
        pg = c.table[c.slots[i].long(), p // PAGE].long()
        c.pool[pg, :, 0, p % PAGE] = c.k[i]
    before = c.out.clone()
    got = c.run()
    assert torch.isfinite(got.float()).all()
    for i in range(2):
        n, kv = c.reqs[i]
        for h in range(2):
            s = c.k[i][:, h, 0].double() * SCALE
            for row in range(n):
                p = torch.softmax(s[: kv - n + row + 1], 0)
                ref = p @ c.v[i][: kv - n + row + 1, h].double()
                A = p @ c.v[i][: kv - n + row + 1, h].double().abs()
                d = (got[int(c.cu_host[i]) + row, 2 * h].double() - ref).abs()
                assert (d <= 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -12) * A).all()
    del before


def test_scores_far_apart():
    # keys in rising order of score over a long range: every tile moves the maximum, by far more than fp32's 2^127
    c = Cache([(1, 2000), (64, 1500)], 8, 2, seed=7)
    for i in range(2):
        n = c.reqs[i][1]
        ramp = torch.linspace(-300, 300, n, device="cuda")
        c.k[i][:] = 0
        c.k[i][:, :, 0] = ramp[:, None].to(torch.bfloat16)
        p = torch.arange(n, device="cuda")
        pg = c.table[c.slots[i].long(), p // PAGE].long()
        c.pool[pg, :, 0, p % PAGE] = c.k[i]
    c.q.zero_()
    c.q[..., 0] = 12
    before = c.out.clone()
    c.check(c.run(), before)
    c.q[..., 0] = -12
    c.check(c.run(), before)


BAD_REQUESTS = {"slot above": ("slots", 1, 5), "slot below": ("slots", 1, -1), "kv below the rows": ("kv_len", 1, 29),
                "kv past the row": ("kv_len", 1, 10_000), "kv negative": ("kv_len", 1, -4)}


@pytest.mark.parametrize("name", BAD_REQUESTS)
def test_a_request_outside_its_arrays_is_not_computed(name):
    c = Cache([(4, 100), (30, 200), (2, 50)], 16, 8, seed=8)
    field, i, value = BAD_REQUESTS[name]
    getattr(c, field)[i] = value
    before = c.out.clone()
    out = c.run()
    assert ops.error_word() == 0x4001
    c.check(out, before, only=(0, 2))


@pytest.mark.parametrize("cu", [[0, 4, 40, 36], [-3, 4, 34, 36], [0, 4, 34, 99]])
def test_rows_outside_the_tokens_are_not_touched(cu):
    c = Cache([(4, 100), (30, 200), (2, 50)], 16, 8, seed=9)
    c.cu.copy_(i32(cu))
    before = c.out.clone()
    out = c.run()
    assert ops.error_word() == 0x4001
    good = [i for i in range(3) if cu[i] == c.cu_host[i] and cu[i + 1] == c.cu_host[i + 1]]
    for i in good:
        ref, tol = c.reference(i)
        a, n = int(c.cu_host[i]), c.reqs[i][0]
        if all(not (cu[j] <= a < cu[j + 1]) for j in range(3) if j != i):
            assert ((out[a:a + n].double() - ref).abs() <= tol).all()
    del before


@pytest.mark.parametrize("value", [-1, 1 << 20, -(1 << 31)])
def test_a_page_outside_the_pool_is_not_read(value):
    c = Cache([(4, 100), (30, 200)], 16, 8, seed=10)
    c.table[c.slots[1].long(), 3] = value
    c.k[1][48:64] = 0
    c.v[1][48:64] = 0
    before = c.out.clone()
    out = c.run()
    assert ops.error_word() == 0x4002
    c.check(out, before)  # its keys count as zeros


def test_attention_twice_is_the_same_and_pages_may_be_shared():
    c = Cache([(1, 5000), (33, 800), (7, 7)], 16, 8, seed=11)
    # request 2's row now starts with request 1's first pages: a shared prefix
    first = c.run().clone()
    c.ws.fill_(0)
    assert torch.equal(c.run(), first)
    c.ws.fill_(0xFF)
    assert torch.equal(c.run(), first)


def test_attention_where_the_pool_passes_32_bits():
    c = Cache([(2, 1000), (40, 500)], 2, 1, seed=12, stale=0.0, extra_pages=600_000)
    c.check(c.run(), c.out.clone())


def test_attention_on_another_stream_and_in_a_graph():
    c = Cache([(1, 5000), (33, 800), (7, 7)], 16, 8, seed=13)
    want = c.run().clone()
    c.out.zero_()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    ops.paged_attention(*c.args(), stream=s)
    s.synchronize()
    assert torch.equal(c.out, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.paged_attention(*c.args())
    c.out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(c.out, want)


def test_two_calls_at_once_with_a_workspace_each():
    a, b = Cache([(1, 9000)], 16, 8, seed=14), Cache([(90, 3000)], 16, 8, seed=15)
    want = a.run().clone(), b.run().clone()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(20):
        ops.paged_attention(*a.args(), stream=s)
        ops.paged_attention(*b.args(), stream=t)
    torch.cuda.synchronize()
    assert torch.equal(a.out, want[0]) and torch.equal(b.out, want[1])


# ---- all of them together --------------------------------------------------------------------------------------------

class Step:
    """A server of max_seqs slots: one layer's weights are skipped, the projection's rows are the inputs."""

    QH, KVH = 16, 8

    def __init__(self, max_seqs, P, F, requests, max_tokens, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.sv = Server(max_seqs, P, F, seed)
        self.slots, self.new, self.keep = i32([-1] * requests), i32([0] * requests), i32([0] * requests)
        self.bufs = step_buffers(requests, max_tokens)
        self.qkv = torch.zeros(max_tokens, 32 * HD, device="cuda", dtype=torch.bfloat16)
        self.gain = 1 + 0.1 * torch.randn(HD, generator=g, device="cuda", dtype=torch.bfloat16)
        ang = torch.arange(P * PAGE, device="cuda")[:, None] * torch.exp(-torch.arange(64, device="cuda") / 9.0)
        self.cos, self.sin = ang.cos(), ang.sin()
        self.q = torch.zeros(max_tokens, self.QH, HD, device="cuda", dtype=torch.bfloat16)
        self.out = torch.zeros_like(self.q)
        self.pool = torch.full((F, self.KVH, 2, PAGE, HD), float("nan"), device="cuda", dtype=torch.bfloat16)
        self.ws = torch.empty(ops.paged_attention_workspace(max_tokens, self.QH, self.KVH), dtype=torch.uint8, device="cuda")
        self.k, self.v = [None] * max_seqs, [None] * max_seqs

    def launch(self):
        sv = self.sv
        cu, kv_len, tok_pos, slot_map = self.bufs
        ops.page_plan(self.slots, self.new, sv.seq_len, sv.table, sv.free_list, sv.count, *self.bufs)
        ops.qkv_append(self.qkv, self.gain, self.gain, 1e-6, self.cos, self.sin, tok_pos, slot_map, self.q, self.pool)
        ops.paged_attention(self.q, self.pool, sv.table, self.slots, cu, kv_len, self.out, self.ws, SCALE)
        ops.page_release(self.slots, self.keep, sv.seq_len, sv.table, sv.free_list, sv.count)

    def model(self, slots, new, keep, qkv):
        """The same step on the lists and in 64 bits: the rows of out and their tolerance."""
        cu, kv, pos, _ = self.sv.plan(slots, new)
        y, _ = append_reference(qkv[:cu[-1]], [self.gain, self.gain], 1e-6, self.cos, self.sin, pos, self.QH, self.KVH)
        y = y.cuda()
        refs = []
        for i, s in enumerate(slots):
            n = cu[i + 1] - cu[i]
            if s == -1 or n == 0:
                continue
            old = 0 if self.k[s] is None else self.k[s].shape[0]
            rows = y[cu[i]:cu[i + 1]]
            new_k, new_v = rows[:, self.QH:self.QH + self.KVH], rows[:, self.QH + self.KVH:]
            self.k[s] = new_k if not old else torch.cat([self.k[s], new_k])
            self.v[s] = new_v if not old else torch.cat([self.v[s], new_v])
            total = old + n
            q = rows[:, :self.QH].unflatten(1, (self.KVH, 2))
            sc = torch.einsum("nhgd,khd->nhgk", q, self.k[s]) * SCALE
            hidden = torch.arange(total, device="cuda")[None] > torch.arange(old, total, device="cuda")[:, None]
            p = torch.softmax(sc.masked_fill(hidden[:, None, None], -torch.inf), -1)
            ref = torch.einsum("nhgk,khd->nhgd", p, self.v[s])
            A = torch.einsum("nhgk,khd->nhgd", p, self.v[s].abs())
            # q and k are rounded to bf16 on the way (2^-8 each): a score is off by 2 * 2^-8 * sum |q_d k_d| * scale
            ds = torch.where(p > 0, torch.einsum("nhgd,khd->nhgk", q.abs(), self.k[s].abs()), 0.0).amax(-1)
            ds = ds * SCALE * (2.0 ** -7 + 2.0 ** -16) + 130 * 2.0 ** -24 * SCALE * ds
            tol = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2 * (2 * ds + 2.0 ** -20 + (total / 16 + 300) * 2.0 ** -23))[..., None] * A
            refs.append((cu[i], n, ref.flatten(1, 2), tol.flatten(1, 2)))
        self.sv.release(slots, keep)
        for s, k in zip(slots, keep):
            if s != -1 and self.k[s] is not None:
                self.k[s], self.v[s] = self.k[s][:k], self.v[s][:k]
        return refs


@pytest.mark.parametrize("graph", [False, True])
def test_steps_of_a_server(graph):
    # Ten steps with sequences that start, grow by chunks and single tokens, lose drafted tokens and end. As a graph, the
    # step is captured once and replayed with other requests in its buffers.
    max_seqs, requests, max_tokens, P = 9, 7, 260, 14
    st = Step(max_seqs, P, 60, requests, max_tokens, seed=20)
    r = np.random.default_rng(20)
    g = None
    if graph:
        st.launch()  # an empty step (every request is padding) before the capture
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            st.launch()
    for step in range(10):
        slots = r.permutation(max_seqs)[:requests]
        slots = np.where(r.uniform(size=requests) < 0.2, -1, slots)
        new, keep, left, pages_left = [], [], max_tokens, len(st.sv.free)
        for s in slots:
            old = 0 if s == -1 else st.sv.len[s]
            n = 0 if s == -1 else int(min(r.choice([1, 1, 3, 16, 60, 90]), P * PAGE - old, left, max(0, pages_left - 1) * PAGE))
            left -= n
            pages_left -= pages(old + n) - pages(old)
            new.append(n)
            keep.append(0 if s == -1 else int(r.choice([old + n, old + n, old + n, old + n // 2, 0])))
        qkv = torch.randn(max_tokens, 32 * HD, device="cuda", generator=torch.Generator(device="cuda").manual_seed(step)).bfloat16()
        st.qkv.copy_(qkv)
        st.slots.copy_(i32(slots)), st.new.copy_(i32(new)), st.keep.copy_(i32(keep))
        st.out.fill_(7)
        if g is None:
            st.launch()
        else:
            g.replay()
        torch.cuda.synchronize()
        assert ops.error_word() == 0, step
        refs = st.model(slots.tolist(), new, keep, qkv)
        for a, n, ref, tol in refs:
            got = st.out[a:a + n].double()
            assert torch.isfinite(got).all() and ((got - ref).abs() <= tol).all(), (step, a, n)
        assert (st.out[sum(new):] == 7).all()
        assert st.sv.seq_len.tolist() == st.sv.len and int(st.sv.count) == len(st.sv.free)
        assert st.sv.free_list[: len(st.sv.free)].tolist() == st.sv.free


def test_a_step_without_pages_does_nothing():
    st = Step(4, 8, 3, 2, 100, seed=21)
    st.slots.copy_(i32([0, 1])), st.new.copy_(i32([40, 30])), st.keep.copy_(i32([0, 0]))
    st.qkv.fill_(1)
    st.launch()
    torch.cuda.synchronize()
    assert ops.error_word() == 0x5002
    assert int(st.sv.count) == 3 and st.sv.seq_len.tolist() == [0] * 4
    assert (st.out == 0).all() and (st.q == 0).all() and torch.isnan(st.pool.float()).all()


def test_attention_equals_the_contiguous_prefill_and_the_decode_operator():
    # beside their siblings on shapes that all of them take: within the two operators' roundings of each other
    c = Cache([(150, 150), (64, 64)], 16, 8, seed=22, stale=0.0)
    k, v = torch.cat(c.k), torch.cat(c.v)
    out = torch.zeros_like(c.out).contiguous()
    ops.prefill_attention(c.q.contiguous(), k, v, out, c.cu, 150, SCALE)
    got = c.run()
    for i in range(2):
        _, tol = c.reference(i)
        a, n = int(c.cu_host[i]), c.reqs[i][0]
        assert ((got[a:a + n].double() - out[a:a + n].double()).abs() <= 2 * tol).all()
    d = Cache([(1, 700), (1, 33)], 16, 8, seed=23, stale=0.0)
    lens = torch.zeros(4, dtype=torch.int32, device="cuda")
    lens[d.slots.long()] = d.kv_len
    ws = torch.empty(ops.decode_attention_workspace(2, 8, d.table.shape[1], 4) // 4, device="cuda")
    out = torch.zeros(2, 16, HD, device="cuda", dtype=torch.bfloat16)
    ops.decode_attention(d.q.contiguous(), d.pool, d.table, lens, d.slots, out, ws, 4, SCALE)
    got = d.run()
    for i in range(2):
        _, tol = d.reference(i)
        assert ((got[i].double() - out[i].double()).abs() <= 2 * tol).all()
