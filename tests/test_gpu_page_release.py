"""Releases that can be of many pages, on the GPU: a cluster of CTAs does them, whatever the number of requests."""

import numpy as np
import pytest

from tests.conftest import cuda_available

pytestmark = pytest.mark.gpu

if cuda_available():
    import torch

    from rosylnalive_b200 import ops
    from tests.test_gpu_paged_step import PAGE, Server, check_plan, gpu_release


@pytest.fixture(autouse=True)
def _device():
    ops.set_device(0)
    yield
    torch.cuda.synchronize()
    assert ops.error_word() == 0


@pytest.mark.parametrize("requests,per_seq,pool", [(1, 9000, 9000), (2, 4097, 8500), (3, 5000, 20000), (7, 1300, 9000),
                                                   (9, 1000, 8500), (40, 300, 12000), (500, 17, 8500), (768, 11, 8448)])
def test_a_release_of_few_requests_that_hold_many_pages(requests, per_seq, pool):
    r = np.random.default_rng(requests)
    sv = Server(requests + 2, per_seq, pool, seed=requests)
    for step in range(4):
        slots = r.permutation(requests + 2)[:requests]
        slots = np.where(r.uniform(size=requests) < 0.1, -1, slots)
        left = len(sv.free)
        new = []
        for s in slots:  # uneven: some requests take nearly all that is left
            pages = 0 if s == -1 else int(min(per_seq - len(sv.own[s]), left * r.choice([0, 0.01, 0.9]), 4000))
            left -= pages
            new.append(max(0, pages * PAGE - int(r.integers(0, 15))) if pages else 0)
        check_plan(sv, slots.tolist(), new, max(1, sum(new)))
        slots = r.permutation(requests + 2)[:requests]
        keep = [int(r.integers(0, sv.len[s] + 1)) if r.uniform() < 0.5 else (0, sv.len[s])[step % 2] for s in slots]
        gpu_release(sv, slots.tolist(), keep)
        sv.release(slots.tolist(), keep)
        sv.same_state()
