"""The paged attention's schedule on the CPU: paged_sched.h, which the kernel uses, built with the host compiler."""

import ctypes
import os
import random
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def sched(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    if not cxx:
        pytest.skip("no host C++ compiler")
    lib = str(tmp_path_factory.mktemp("sched") / "sched.so")
    subprocess.run([cxx, "-O2", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-o", lib,
                    os.path.join(HERE, "paged_sched_check.cpp")], check=True)
    return ctypes.CDLL(lib)


# ---- the cut of a call's work ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("group", [1, 2, 3, 5, 8, 16, 31, 32, 33, 64, 65, 128])
def test_items_of_a_request(sched, group):
    sched.check_items.argtypes = [ctypes.c_uint64] + [ctypes.c_int] * 3
    rng = random.Random(group)
    span = 2 * (128 // group)
    most = 1 << 24  # tokens of a call, and keys of a request
    new = [1, 2, span - 1, span, span + 1, 3 * span, 5 * span + 1, most - 1, most] + [rng.randint(1, 5000) for _ in range(40)]
    for n in new:
        if n < 1:
            continue
        for kv in {n, min(most, n + 1), min(most, n + rng.randint(0, 300)), min(most, n + rng.randint(0, 1 << 23)), most}:
            assert sched.check_items(n * 31 + kv, group, n, kv) == 0, (n, kv)


@pytest.mark.parametrize("most", [1, 2, 16, 148, 200])
def test_every_tile_of_a_call_is_computed_once_and_merged_once(sched, most):
    sched.check_call.argtypes = [ctypes.c_uint64, ctypes.c_int]
    for seed in range(400):
        assert sched.check_call(seed * 1000 + most, most) == 0, seed


# ---- the ring of K and V tiles ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("wide", [0, 1])
def test_the_ring_order_is_the_order_of_use(sched, wide):
    lead = sched.lead_of(wide)
    for nt in range(1, 60):
        order = [None] * (2 * nt)
        for t in range(nt):
            for what, x in (("K", sched.place_of_k(t, lead)), ("V", sched.place_of_v(t, nt, lead))):
                assert order[x] is None
                order[x] = (what, t)
        use = []
        for step in range(nt + 2):
            if step < nt:
                use.append(("K", step))
            if 0 <= step - (lead - 1) < nt:
                use.append(("V", step - (lead - 1)))
        # a step's V is used behind its K, and of a wide item P V comes a step earlier
        assert order == use, (nt, order, use)


class Barrier:
    """An mbarrier: a wait for a parity passes when the phase under way has the other one."""

    def __init__(self):
        self.done = 0

    def passes(self, parity):
        return (self.done & 1) != parity


class Cta:
    """The roles of a CTA that fill, use and free the ring, as generators that yield what they wait for. MMAs complete when
    they are issued; a copy lands when the memory's turn comes. Every wait that passes is checked to be the phase meant."""

    ITEMS = 4

    def __init__(self, lib, items, rng):
        self.lib, self.items, self.rng = lib, items, rng  # items: (tiles, wide, dirty tile, whether a key is marked)
        self.R = lib.ring_stages()
        self.full, self.empty = ([Barrier() for _ in range(self.R)] for _ in range(2))
        self.flying, self.issued = set(), {}  # ring items on their way; the last one of each stage
        self.picked = {r: -1 for r in ("K", "V", "issuer", "softmax")}
        self.s_full, self.p_full, self.o_done, self.s_free = [0, 0], [0, 0], [0, 0], [0, 0]
        self.o_free, self.q_empty, self.cleaned = 0, 0, 0
        self.MARKS = lib.marks()
        self.mark, self.read, self.ahead = [0] * self.MARKS, [0, 0], 0  # read: items whose mark has been read, a slot
        self.ended = False
        self.waits, self.last, self.most = 0, [0, 0], 0  # the issuer's waits, and the most from a slot's commit to its next

    def commit(self, s):
        self.most = max(self.most, self.waits - self.last[s])
        self.last[s] = self.waits

    def item(self, role, k):
        """Until the scheduler has handed out item k: four items on from one that all have taken."""
        while k >= self.ITEMS and min(self.picked.values()) < k - self.ITEMS:
            yield
        self.picked[role] = k

    def wait(self, bar, parity, phase):
        while not bar.passes(parity):
            yield
        assert bar.done == phase, "a wait passed on another phase"

    def producer(self, v):
        ring = 0
        for k, (nt, wide, dirty, marked) in enumerate(self.items):
            yield from self.item("V" if v else "K", k)
            lead = self.lib.lead_of(wide)
            while not v and self.q_empty < k:
                yield

            def clean(j):
                x = ring + self.lib.place_of_v(j, nt, lead)
                yield from self.wait(self.full[x % self.R], self.lib.parity_of(x), x // self.R + 1)
                if marked and j == nt - 1:
                    self.mark[k % self.MARKS] = k + 1
                    self.ahead = max(self.ahead, k - min(self.read))
                self.cleaned += 1

            for t in range(nt):
                x = ring + (self.lib.place_of_v(t, nt, lead) if v else self.lib.place_of_k(t, lead))
                yield from self.wait(self.empty[x % self.R], self.lib.parity_of(x) ^ 1, x // self.R)
                assert x - self.R not in self.flying
                self.issued[x % self.R] = x
                self.flying.add(x)
                yield
                if v and t > dirty:
                    yield from clean(t - 1)
            if v and dirty < nt:
                yield from clean(nt - 1)
            ring += 2 * nt

    def memory(self):
        while True:
            if self.flying:
                x = self.rng.choice(sorted(self.flying))
                self.flying.remove(x)
                self.full[x % self.R].done += 1
            yield

    def issuer(self):
        x, cleaned, before = 0, 0, [0, 0]
        for k, (nt, wide, dirty, marked) in enumerate(self.items):
            yield from self.item("issuer", k)
            self.waits += 2  # the item and its q

            def tile():
                nonlocal x
                self.waits += 1
                yield from self.wait(self.full[x % self.R], self.lib.parity_of(x), x // self.R + 1)
                x += 1
                return (x - 1) % self.R

            def product(s, n):
                self.waits += 1
                while self.p_full[s] < before[s] + n + 1:
                    yield
                self.o_done[s] += 1
                self.commit(s)

            def score(s, n):
                self.waits += 1
                while self.s_free[s] < before[s] + n:
                    yield
                self.s_full[s] += 1
                self.commit(s)

            vt = None
            for t in range(nt + 2):
                if wide:
                    if t < nt:
                        kt = yield from tile()
                        yield from score(0, t)
                    if t >= 2:
                        yield from product(1, t - 2)
                        self.empty[vt].done += 1
                    if t < nt:
                        yield from score(1, t)
                        self.empty[kt].done += 1
                        self.q_empty += t == nt - 1
                    if 1 <= t <= nt:
                        vt = yield from tile()
                        self.waits += (t == 1) + (t > dirty)
                        while t == 1 and self.o_free < 2 * k:
                            yield
                        while t > dirty and self.cleaned < cleaned + t - dirty:
                            yield
                        yield from product(0, t - 1)
                else:
                    s = t & 1
                    if t < nt:
                        kt = yield from tile()
                        yield from score(s, t >> 1)
                        self.empty[kt].done += 1
                        self.q_empty += t == nt - 1
                    if t >= 2:
                        vt = yield from tile()
                        self.waits += (t == 2) + (t - 2 >= dirty)
                        while t == 2 and self.o_free < 2 * k:
                            yield
                        while t - 2 >= dirty and self.cleaned < cleaned + t - 1 - dirty:
                            yield
                        yield from product(s, (t - 2) >> 1)
                        self.empty[vt].done += 1
            count = 2 * nt if wide else nt
            before[0] += (count + 1) // 2
            before[1] += count // 2
            cleaned += max(0, nt - dirty)
        self.ended = True

    def softmax(self, s):
        steps, done = 0, [0, 0]
        for k, (nt, wide, dirty, marked) in enumerate(self.items):
            yield from self.item("softmax", k)
            for _ in range(nt if wide else (nt + 1 - s) // 2):
                while self.s_full[s] < steps + 1 or self.o_done[s] < steps:
                    yield
                self.s_free[s] += 1
                yield
                self.p_full[s] += 1
                steps += 1
            done[0] += nt if wide else (nt + 1) // 2
            done[1] += nt if wide else nt // 2
            while self.o_done[s] < done[s] or (not wide and self.o_done[1 - s] < done[1 - s]):
                yield
            yield
            assert (self.mark[k % self.MARKS] == k + 1) == bool(marked), "a mark was lost"
            self.read[s] = k + 1
            self.o_free += 1

    def run(self, steps=None):
        """Takes roles in turn, some of them rarely, until all are through or for so many steps; then how many were taken."""
        roles = [self.producer(0), self.producer(1), self.issuer(), self.softmax(0), self.softmax(1), self.memory()]
        weight = [self.rng.choice((1, 1, 8, 40)) for _ in roles]
        left, n, live = roles[:-1], 0, dict(zip(map(id, roles), weight))
        bound = 4000 * (10 + sum(x[0] for x in self.items)) if steps is None else steps
        while left and n < bound:
            n += 1
            role = self.rng.choices(left + roles[-1:], [live[id(r)] for r in left + roles[-1:]])[0]
            try:
                next(role)
            except StopIteration:
                left.remove(role)
        assert steps is not None or not left, "the roles wait for one another"
        return n


def some_items(rng, n):
    out = []
    for _ in range(n):
        nt = rng.choice((1, 1, 1, 2, 3, rng.randint(1, 9)))
        dirty = rng.randint(0, nt)
        out.append((nt, rng.randint(0, 1), dirty, int(dirty < nt and rng.random() < 0.7)))
    return out


def test_the_roles_get_through_and_lose_no_mark(sched):
    for seed in range(150):
        rng = random.Random(seed)
        cta = Cta(sched, some_items(rng, rng.randint(1, 14)), rng)
        cta.run()
        assert cta.ended and not cta.flying


def test_the_cleaning_runs_as_far_ahead_as_there_are_marks(sched):
    # Items of one tile whose epilogues are slow: the mark of the item farthest ahead takes the last place that is free.
    most = 0
    for seed in range(300):
        rng = random.Random(3000 + seed)
        cta = Cta(sched, [(1, 0, 0, 1)] * 12, rng)
        cta.run()
        most = max(most, cta.ahead)
    assert most == sched.marks() - 1


def test_what_is_waited_for_after_giving_up_is_what_is_in_flight(sched):
    # All roles stop somewhere. Then each stage's last copy is waited for, and no other: the wait passes at once for a copy
    # that has landed, and only then, and behind all of the waits nothing is on its way.
    in_flight = 0
    for seed in range(400):
        rng = random.Random(1000 + seed)
        items = some_items(rng, rng.randint(1, 12))
        whole = Cta(sched, items, random.Random(seed)).run()
        cta = Cta(sched, items, random.Random(seed))
        cta.run(rng.randint(1, whole))
        if cta.ended:
            assert not cta.flying
            continue
        in_flight += bool(cta.flying)
        for st, x in cta.issued.items():
            assert x % cta.R == st and cta.full[st].passes(sched.parity_of(x)) == (x not in cta.flying)
        for x in list(cta.flying):
            assert cta.issued[x % cta.R] == x
            cta.full[x % cta.R].done += 1
        for st, x in cta.issued.items():
            assert cta.full[st].passes(sched.parity_of(x))
    assert in_flight > 50


def test_the_issuer_commits_or_gives_up_before_a_wait_of_the_softmax_ends(sched):
    # The softmax's warps wait for a slot's next commit; an issuer that never waits longer than its limit has made it, or has
    # returned, by the time theirs ends. (Items of one tile leave slot 1 out, so whole runs of them stand between its commits,
    # but then slot 1's warps wait for slot 0's.)
    for seed in range(60):
        rng = random.Random(2000 + seed)
        items = [(max(2, nt), wide, dirty, marked) for nt, wide, dirty, marked in some_items(rng, 12)]
        cta = Cta(sched, items, rng)
        cta.run()
        assert cta.most <= sched.issuer_waits()
    assert sched.polls(1) > sched.issuer_waits() * sched.polls(0)
