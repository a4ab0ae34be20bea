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
    from tests.test_gpu_paged_step import HD, PAGE, SCALE, Cache


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
