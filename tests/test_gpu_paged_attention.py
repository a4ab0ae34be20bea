"""Paged attention on the GPU beside tests/test_gpu_paged_step.py: the precision of items of few rows, values that are not
finite in keys that every row sees, pages that requests share, and rows that a refused request leaves alone.

Tolerance of items of up to 32 rows: that of tests/test_gpu_paged_step.py with weights that keep 16 bits. The first bf16 has
p's first 8 significant bits, cut off (the rest is below 2^-7 p), and the second the rest, rounded (2^-8 of it): 2^-15 A in
the place of 2^-8 A.
"""

import numpy as np
import pytest

from tests.conftest import cuda_available

pytestmark = pytest.mark.gpu

if cuda_available():
    import torch

    from rosylnalive_b200 import ops
    from tests.test_gpu_paged_step import HD, PAGE, SCALE, Cache, i32


@pytest.fixture(autouse=True)
def _device():
    ops.set_device(0)
    yield
    torch.cuda.synchronize()
    assert ops.error_word() == 0


@pytest.mark.parametrize("heads,reqs", [((16, 8), [(1, 900)]), ((16, 8), [(1, 4000 + i) for i in range(30)]),
                                        ((32, 8), [(5, 100 + 300 * i) for i in range(12)]), ((4, 4), [(32, 700), (9, 20)]),
                                        ((32, 1), [(1, 2500), (1, 1), (1, 129)]), ((12, 2), [(4, 3000), (5, 64), (1, 7)]),
                                        ((8, 8), [(17, 1300), (8, 8), (16, 333)])])
def test_items_of_few_rows_keep_16_bits_of_the_weights(heads, reqs):
    c = Cache(reqs, *heads, seed=41)
    out = c.run()
    for i, (n, kv) in enumerate(reqs):
        ref, tol = c.reference(i)
        # less the rounding of the weights: A is what the tolerance adds beside the output's rounding
        q = c.q[c.cu_host[i]:c.cu_host[i] + n].double().unflatten(1, (c.kvh, c.qh // c.kvh))
        s = torch.einsum("nhgd,khd->nhgk", q, c.k[i].double()) * SCALE
        hidden = torch.arange(kv, device="cuda")[None] > torch.arange(kv - n, kv, device="cuda")[:, None]
        p = torch.softmax(s.masked_fill(hidden[:, None, None], -torch.inf), -1)
        A = torch.einsum("nhgk,khd->nhgd", p, c.v[i].double().abs()).flatten(1, 2)
        tol = tol - (2.0 ** -8 - 2.0 ** -15) * A
        d = (out[c.cu_host[i]:c.cu_host[i] + n].double() - ref).abs()
        assert (d <= tol).all(), (i, float((d - tol).max()))


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("heads", [(16, 8), (4, 4), (10, 1)])
def test_values_that_are_not_finite_in_keys_that_every_row_sees(value, heads):
    # An infinite v of a key with a weight above 0 gives that infinity; each key has dims of its own, so none meets another.
    c = Cache([(1, 700), (1, 90), (4, 300), (40, 500), (130, 400)], *heads, seed=42)
    own, slots = c.table.cpu().numpy(), c.slots.tolist()
    for i, (n, kv) in enumerate(c.reqs):
        for e, key in enumerate((0, 17, (kv - n) // 2, kv - n - 1 if n < kv else 0)):
            dims = slice(e, HD, 8)
            c.pool[int(own[slots[i], key // PAGE]), :, 1, key % PAGE, dims] = value
            c.v[i][key, :, dims] = value
    before = c.out.clone()
    c.check(c.run(), before)


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), 3e38])
@pytest.mark.parametrize("heads", [(16, 8), (4, 4), (10, 1)])
def test_weights_of_one_bit_times_large_values(value, heads):
    # q = 0: all weights are equal and p is 1, whose second bf16 has nothing left to hold. q_0 k_0 = -83: p is about 2^-120.
    c = Cache([(1, 1), (1, 2), (3, 90), (1, 300), (40, 500), (1, 64)], *heads, seed=47)
    c.q.zero_()
    c.q[-1, :, 0] = 1
    own, slots = c.table.cpu().numpy(), c.slots.tolist()
    for i, (n, kv) in enumerate(c.reqs):
        key = 0
        pg = int(own[slots[i], key // PAGE])
        c.pool[pg, :, 1, key % PAGE, 1::4] = value
        c.v[i][key, :, 1::4] = value
    c.k[5][0, :, 0] = -83 / SCALE
    c.k[5][1:, :, 0] = 0
    for key in range(64):
        c.pool[int(own[slots[5], key // PAGE]), :, 0, key % PAGE, 0] = c.k[5][key, :, 0]
    before = c.out.clone()
    c.check(c.run(), before)


def by_slot(c, i):
    return int(c.slots[i])


@pytest.mark.parametrize("heads", [(16, 8), (4, 4), (16, 1)])
def test_pages_that_requests_share(heads):
    # Four requests whose rows of the page table start with the same pages, and one in a row that another one has too.
    c = Cache([(1, 5000), (33, 800), (7, 450), (150, 700), (1, 333), (3, 800)], *heads, seed=43)
    for i, shared in ((2, 27), (3, 30), (4, 20)):  # whole pages of request 1's prefix, their own keys behind
        c.table[by_slot(c, i), :shared] = c.table[by_slot(c, 1), :shared].clone()
        c.k[i][:shared * PAGE] = c.k[1][:shared * PAGE]
        c.v[i][:shared * PAGE] = c.v[1][:shared * PAGE]
    c.slots[5] = c.slots[1]  # the same slot in two requests: its last 33 and its last 3 tokens
    c.k[5], c.v[5] = c.k[1], c.v[1]
    before = c.out.clone()
    c.check(c.run(), before)


@pytest.mark.parametrize("cu", [[0, 4, 40, 36], [-3, 4, 34, 36], [0, 4, 34, 99], [0, 4, 3, 36], [0, 37, 34, 36],
                                [2**31 - 1, 4, 34, 36], [0, 4, -(2**31), 36]])
@pytest.mark.parametrize("heads", [(16, 8), (4, 4), (16, 1)])
def test_rows_of_refused_requests_stay(cu, heads):
    c = Cache([(4, 100), (30, 200), (2, 50)], *heads, seed=44)
    c.cu.copy_(i32(cu))
    before = c.out.clone()
    out = c.run()
    assert ops.error_word() == 0x4001
    # The requests that are sound with the rows that they have now. (In [0, 4, 3, 36] two of them have row 3, which holds the
    # result of either; no other row is in doubt.)
    sound = [i for i in range(3) if cu[i] >= 0 and 0 < cu[i + 1] - cu[i] <= c.reqs[i][1] and cu[i + 1] <= c.T]
    owners = torch.zeros(c.T, dtype=torch.int32, device="cuda")
    for i in sound:
        owners[cu[i]:cu[i + 1]] += 1
    for i in sound:
        c.reqs[i], c.cu_host[i] = (cu[i + 1] - cu[i], c.reqs[i][1]), cu[i]
        ref, tol = c.reference(i)
        alone = owners[cu[i]:cu[i + 1]] == 1
        assert ((out[cu[i]:cu[i + 1]].double() - ref).abs() <= tol)[alone].all(), i
    stay = owners == 0
    assert torch.equal(out[stay], before[stay])


@pytest.mark.parametrize("name,field,i,value", [("slot", "slots", 1, 7), ("slot", "slots", 1, -2), ("keys", "kv_len", 1, 29),
                                                ("keys", "kv_len", 1, 10_000), ("keys", "kv_len", 1, -4),
                                                ("first", "slots", 0, 5), ("last", "kv_len", 2, 0)])
@pytest.mark.parametrize("heads", [(16, 8), (16, 1)])
def test_rows_of_a_request_outside_its_arrays_stay(name, field, i, value, heads):
    c = Cache([(4, 100), (30, 200), (2, 50)], *heads, seed=45, spare=3, gap=1)
    getattr(c, field)[i] = value
    before = c.out.clone()
    out = c.run()
    assert ops.error_word() == 0x4001
    c.check(out, before, only=[j for j in range(3) if j != i])  # and all other rows, its own among them, as they were


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("heads", [(16, 8), (4, 4), (10, 1)])
def test_keys_that_are_not_finite_act_on_every_row_that_sees_them(value, heads):
    # A score of +inf or NaN makes its row NaN and one of -inf weighs nothing; which of them a row gets goes by the sign of
    # its q in that dim. Keys of the request itself (some rows see them) and of its past (all rows do).
    c = Cache([(200, 200), (150, 400), (1, 90), (5, 700), (1, 1500)], *heads, seed=46)
    own, slots = c.table.cpu().numpy(), c.slots.tolist()
    for i, keys in ((0, (40, 199)), (1, (30, 300)), (2, (89,)), (3, (697, 100)), (4, (3,))):
        for key in keys:
            c.pool[int(own[slots[i], key // PAGE]), :, 0, key % PAGE, 3] = value
            c.k[i][key, :, 3] = value
    before = c.out.clone()
    got = c.run()
    nans = 0
    for i, (n, kv) in enumerate(c.reqs):
        a = int(c.cu_host[i])
        q = c.q[a:a + n].double().unflatten(1, (c.kvh, c.qh // c.kvh))
        k, v = c.k[i].double(), c.v[i].double()
        # elementwise: a product of matrices need not keep 0 * inf apart
        s = (q[:, :, :, 3:4] * k[:, :, 3].T[None, :, None]) + torch.einsum(
            "nhgd,khd->nhgk", torch.cat([q[..., :3], q[..., 4:]], -1), torch.cat([k[..., :3], k[..., 4:]], -1))
        s = s * SCALE
        hidden = torch.arange(kv, device="cuda")[None] > torch.arange(kv - n, kv, device="cuda")[:, None]
        s = s.masked_fill(hidden[:, None, None], -torch.inf)
        p = torch.softmax(s, -1)
        bad = torch.isnan(p).any(-1)
        ref = torch.einsum("nhgk,khd->nhgd", torch.nan_to_num(p), v)
        A = torch.einsum("nhgk,khd->nhgd", torch.nan_to_num(p), v.abs())
        ds = 130 * 2.0 ** -24 * SCALE * torch.einsum("nhgd,khd->nhgk", q.abs(), torch.nan_to_num(k, 0, 0, 0).abs())
        ds = torch.where(p > 0, ds, 0).amax(-1)
        tol = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2 * (2 * ds + 2.0 ** -20 + (kv / 16 + 300) * 2.0 ** -23))[..., None] * A
        out = got[a:a + n].double().unflatten(1, (c.kvh, c.qh // c.kvh))
        assert torch.equal(torch.isnan(out).all(-1), bad) and torch.equal(torch.isnan(out).any(-1), bad), i
        assert ((out - ref).abs() <= tol)[~bad].all(), i
        nans += int(bad.sum())
    assert nans > 0
    del before
