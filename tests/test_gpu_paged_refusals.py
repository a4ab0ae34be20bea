"""What the paged serving step's operators leave alone when a call breaks a rule, on the GPU."""

import numpy as np
import pytest

from tests.conftest import cuda_available

pytestmark = pytest.mark.gpu

if cuda_available():
    import torch

    from rosylnalive_b200 import ops
    from tests.test_gpu_paged_step import BAD_RELEASES, Server, check_plan, gpu_plan, gpu_release, i32


@pytest.fixture(autouse=True)
def _device():
    ops.set_device(0)
    yield
    torch.cuda.synchronize()
    assert ops.error_word() == 0


def broken_release(name, pad):
    """A server, a release that it refuses (padded, so that above 768 requests a cluster does it) and the code."""
    sv = Server(4, 3, 9, seed=9)
    check_plan(sv, [0, 1], [40, 30], 70)
    slots, keep, code = BAD_RELEASES.get(name, ([0, 1], [0, 0], 0x5014 if name == "page" else 0x5012))
    if name == "count above":
        sv.count.fill_(7)
    elif name == "count below":
        sv.count.fill_(-1)
    elif name == "page":
        sv.table[1, 1] = 9
    r = np.random.default_rng(1)
    at = np.sort(r.permutation(pad + len(slots))[:len(slots)])  # somewhere among the padding, so in parts of several CTAs
    all_slots, all_keep = np.full(pad + len(slots), -1), np.zeros(pad + len(slots), int)
    all_slots[at], all_keep[at] = slots, keep
    return sv, all_slots.tolist(), all_keep.tolist(), code


NAMES = ["slot past the end", "slot below -1", "slot twice", "keep above", "keep below", "count above", "count below", "page"]


@pytest.mark.parametrize("pad", [0, 900, 9000])
@pytest.mark.parametrize("name", NAMES)
def test_a_refused_release_gives_separate_outputs_the_old_state(name, pad):
    sv, slots, keep, code = broken_release(name, pad)
    before = [x.clone() for x in (sv.table, sv.seq_len, sv.count, sv.free_list)]
    lens, left = torch.full_like(sv.seq_len, -5), torch.full_like(sv.count, -5)
    gpu_release(sv, slots, keep, seq_len_out=lens, free_count_out=left)
    assert ops.error_word() == code
    assert all(torch.equal(x, y) for x, y in zip(before, (sv.table, sv.seq_len, sv.count, sv.free_list)))
    assert lens.tolist() == [sv.len[s] if s in slots else -5 for s in range(4)]
    assert torch.equal(left, sv.count)
    gpu_release(sv, slots, keep)  # in place
    assert ops.error_word() == code
    assert all(torch.equal(x, y) for x, y in zip(before, (sv.table, sv.seq_len, sv.count, sv.free_list)))


@pytest.mark.parametrize("pad", [0, 1500])
def test_a_refused_plan_gives_separate_outputs_the_old_state(pad):
    sv = Server(5, 3, 8, seed=10)
    check_plan(sv, [0, 3], [40, 10], 70)
    before = [x.clone() for x in (sv.table, sv.seq_len, sv.count, sv.free_list)]
    lens, left = torch.full_like(sv.seq_len, -5), torch.full_like(sv.count, -5)
    slots, new = [3, 1, 0] + [-1] * pad, [30, 48, 1] + [0] * pad
    got = gpu_plan(sv, slots, new, 100, seq_len_out=lens, free_count_out=left)
    assert ops.error_word() == 0x5002
    assert got == [[0] * (len(slots) + 1), [0] * len(slots), [0] * 100, [-1] * 100]
    assert all(torch.equal(x, y) for x, y in zip(before, (sv.table, sv.seq_len, sv.count, sv.free_list)))
    assert lens.tolist() == [40, 0, -5, 10, -5] and torch.equal(left, sv.count)


def test_state_kept_in_two_buffers_goes_through_refused_calls():
    # Lengths and counts that swap places with every call, as a caller who keeps the step before has them.
    sv = Server(3, 4, 10, seed=11)
    lens, counts = [sv.seq_len, sv.seq_len.clone()], [sv.count, sv.count.clone()]
    bufs = [torch.zeros(n, dtype=torch.int32, device="cuda") for n in (4, 3, 64, 64)]
    slots, turn = i32([0, 1, 2]), 0

    def call(op, amounts, code):
        nonlocal turn
        a, b = turn & 1, 1 - (turn & 1)
        turn += 1
        args = (slots, i32(amounts), lens[a], sv.table, sv.free_list, counts[a], *(bufs if op is ops.page_plan else ()))
        op(*args, seq_len_out=lens[b], free_count_out=counts[b])
        torch.cuda.synchronize()
        assert ops.error_word() == code
        if not code:
            (sv.plan if op is ops.page_plan else sv.release)([0, 1, 2], amounts)
        assert lens[b].tolist() == sv.len and int(counts[b]) == len(sv.free)
        assert sv.free_list[: len(sv.free)].tolist() == sv.free

    call(ops.page_plan, [20, 30, 5], 0)
    call(ops.page_plan, [44, 34, 59], 0x5002)
    call(ops.page_release, [20, 31, 0], 0x5011)
    call(ops.page_release, [3, 30, 0], 0)
    call(ops.page_plan, [1, 1, 65], 0x5001)
    call(ops.page_plan, [14, 0, 40], 0)
