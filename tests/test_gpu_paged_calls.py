"""The paged serving step's operators on the GPU as programs call them: from several threads, in a process's first capture,
in graphs that share a workspace, and with arrays that have no elements."""

import subprocess
import sys
import threading

import numpy as np
import pytest

from tests.conftest import ROOT, cuda_available

pytestmark = pytest.mark.gpu

if cuda_available():
    import torch

    from rosylnalive_b200 import ops
    from tests.test_gpu_paged_step import SCALE, Cache, Server, Step, check_plan, gpu_release, i32


@pytest.fixture(autouse=True)
def _device():
    ops.set_device(0)
    yield
    torch.cuda.synchronize()
    assert ops.error_word() == 0


def test_calls_from_several_threads():
    caches = [Cache(reqs, 16, 8, seed=50 + i) for i, reqs in enumerate((
        [(1, 3000), (1, 50)], [(90, 1200), (5, 40)], [(5, 700)] * 9, [(300, 300), (1, 1)]))]
    want = [c.run().clone() for c in caches]
    servers = [Server(6, 5, 30, seed=60 + i) for i in range(len(caches))]
    torch.cuda.synchronize()
    failures = []

    def work(i):
        try:
            ops.set_device(0)
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for step in range(25):
                    caches[i].out.zero_()
                    ops.paged_attention(*caches[i].args())
                    s.synchronize()
                    assert torch.equal(caches[i].out, want[i]), step
                    check_plan(servers[i], [i, 5, -1], [20 + i, step % 3, 0], 40)
                    gpu_release(servers[i], [5, i], [0, 0])
                    servers[i].release([5, i], [0, 0])
                    servers[i].same_state()
                    with pytest.raises(ValueError):  # messages are a thread's own
                        ops.paged_attention(*caches[i].args()[:-1], -1.0)
        except BaseException as e:  # noqa: BLE001
            failures.append((i, e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(caches))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures


FIRST_CAPTURE = """
import torch
from rosylnalive_b200 import ops
i = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
bf = dict(device="cuda", dtype=torch.bfloat16)
slots, new, lens, table = i(0, 1), i(3, 4), i(0, 0), torch.zeros(2, 4, dtype=torch.int32, device="cuda")
free, count, cu, kv, pos, place = i(*range(8)), i(8), i(0, 0, 0), i(0, 0), i(*[0] * 7), i(*[0] * 7)
qkv, pool, q, out = torch.ones(7, 4 * 128, **bf), torch.zeros(8, 1, 2, 16, 128, **bf), *(torch.zeros(7, 2, 128, **bf),) * 2
angles, ws = torch.ones(64, 64, device="cuda"), torch.empty(1 << 23, dtype=torch.uint8, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    ops.page_plan(slots, new, lens, table, free, count, cu, kv, pos, place)
    ops.qkv_append(qkv, None, None, 0.0, angles, angles, pos, place, q, pool)
    ops.paged_attention(q, pool, table, slots, cu, kv, out, ws, 0.1)
    ops.page_release(slots, new, lens, table, free, count)
g.replay()
torch.cuda.synchronize()
assert ops.error_word() == 0 and lens.tolist() == [3, 4] and count.tolist() == [6]
assert (out == 1).all()  # every v is 1
"""


def test_the_first_calls_of_a_process_may_be_captured():
    r = subprocess.run([sys.executable, "-c", FIRST_CAPTURE], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_two_graphs_share_a_workspace_when_they_run_in_turn():
    a, b = Cache([(1, 9000), (40, 800)], 16, 8, seed=70), Cache([(90, 3000), (3, 70)], 16, 8, seed=71)
    want = a.run().clone(), b.run().clone()
    ws = a.ws if a.ws.numel() > b.ws.numel() else b.ws
    graphs = []
    for c in (a, b):
        c.ws = ws
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.paged_attention(*c.args())
        graphs.append(g)
    for _ in range(5):
        a.out.zero_(), b.out.zero_()
        graphs[0].replay(), graphs[1].replay(), graphs[0].replay()
        torch.cuda.synchronize()
        assert torch.equal(a.out, want[0]) and torch.equal(b.out, want[1])


def test_arrays_without_elements_are_refused():
    e, f = i32([]), torch.zeros(0, dtype=torch.bfloat16, device="cuda")
    st = Step(4, 8, 20, 2, 50, seed=72)
    sv, one = st.sv, i32([0])
    state = (sv.seq_len, sv.table, sv.free_list, sv.count)
    for call in (lambda: ops.page_plan(e, e, *state, i32([0]), e, i32([0]), i32([0])),
                 lambda: ops.page_plan(one, one, *state, i32([0, 0]), one, e, e),
                 lambda: ops.page_release(e, e, *state),
                 lambda: ops.qkv_append(f.view(0, 32 * 128), None, None, 0.0, None, None, None, e, f.view(0, 16, 128), st.pool),
                 lambda: ops.paged_attention(f.view(0, 16, 128), st.pool, sv.table, one, i32([0, 0]), one, f.view(0, 16, 128),
                                             st.ws, SCALE),
                 lambda: ops.paged_attention(st.q, st.pool, sv.table, e, i32([0]), e, st.out, st.ws, SCALE)):
        with pytest.raises(ValueError):
            call()
    sv.same_state()
    # a step of padding alone is a step
    check_plan(sv, [-1], [0], 1)
    cu, kv = i32([0, 0]), i32([0])
    before = st.out[:1].clone()
    ops.qkv_append(st.qkv[:1], None, None, 0.0, None, None, None, i32([-1]), st.q[:1], st.pool)
    ops.paged_attention(st.q[:1], st.pool, sv.table, i32([-1]), cu, kv, st.out[:1], st.ws, SCALE)
    gpu_release(sv, [-1], [0])
    sv.same_state()
    assert torch.equal(st.out[:1], before) and np.isnan(st.pool.float().cpu().numpy()).all()
