"""The q/k/v append of more rows than a call has blocks, so that blocks copy rows ahead and go on from one to the next."""

import numpy as np
import pytest

from tests.conftest import cuda_available

pytestmark = pytest.mark.gpu

if cuda_available():
    import torch

    from rosylnalive_b200 import ops
    from tests.test_gpu_paged_step import HD, PAGE, append_reference, i32


@pytest.fixture(autouse=True)
def _device():
    ops.set_device(0)
    yield
    torch.cuda.synchronize()
    assert ops.error_word() == 0


@pytest.mark.parametrize("qh,kvh,T", [(16, 8, 2500), (40, 8, 1201), (2, 1, 4000), (64, 16, 700)])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("rope", [False, True])
def test_append_of_more_rows_than_blocks(qh, kvh, T, in_place, rope):
    # Tolerance of tests/test_gpu_paged_step.py. Rows without a place, and rows outside their arrays, among the others.
    g = torch.Generator(device="cuda").manual_seed(T)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    heads = qh + 2 * kvh
    qkv = (rnd(T, heads * HD + 64) * 3)[:, :heads * HD]
    gains = [1 + 0.3 * rnd(HD), 1 + 0.3 * rnd(HD)]
    ang = torch.rand(500, 64, generator=g, device="cuda") * 6
    cos, sin = ang.cos(), ang.sin()
    r = np.random.default_rng(T)
    F = T // PAGE + 3
    places, pos = r.permutation(F * PAGE)[:T], r.integers(0, 500, T)
    places[r.uniform(size=T) < 0.3] = -1
    places[T // 3: T // 3 + 700] = -1  # a block's rows in a row
    places[T - 1], places[5] = F * PAGE, -7
    out = qkv[:, :qh * HD].unflatten(1, (qh, HD)) if in_place else rnd(T, qh, HD)
    pool = rnd(F, kvh, 2, PAGE, HD)
    y, tol = append_reference(qkv, gains, 1e-6, cos if rope else None, sin if rope else None, pos, qh, kvh)
    before, ref_pool = out.clone(), pool.clone()
    ops.qkv_append(qkv, *gains, 1e-6, cos if rope else None, sin if rope else None, i32(pos) if rope else None, i32(places),
                   out, pool)
    torch.cuda.synchronize()
    assert ops.error_word() == 0x6001
    live = np.nonzero((places >= 0) & (places < F * PAGE))[0]
    d = (out.double().cpu()[live] - y[live, :qh]).abs()
    assert (d <= tol[live, :qh]).all(), float((d - tol[live, :qh]).max())
    pg, off = torch.tensor(places[live] // PAGE), torch.tensor(places[live] % PAGE)
    for c, h0 in ((0, qh), (1, qh + kvh)):
        d = (pool.cpu()[pg, :, c, off].double() - y[live, h0:h0 + kvh]).abs()
        assert (d <= tol[live, h0:h0 + kvh]).all(), (c, float((d - tol[live, h0:h0 + kvh]).max()))
    dead = np.setdiff1d(np.arange(T), live)
    assert torch.equal(out.cpu()[dead], before.cpu()[dead])
    pool[pg.cuda(), :, :, off.cuda()] = ref_pool[pg.cuda(), :, :, off.cuda()]
    assert torch.equal(pool, ref_pool)
