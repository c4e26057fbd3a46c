"""The give-up logic of the kernels' bounded waits and of the window attention's items, built for the host from the kernels' own headers.

The warps of a block of the tensor-memory kernel are generators here, which yield what they wait for; barriers are counts of completed
phases, waited for by parity as on the device. A wait gives up when nothing else can run, or at random.
"""
import ctypes as C
import os
import random
import shutil
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MS = 1000 * 1000


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    out = str(tmp_path_factory.mktemp("protocol") / "libprotocol.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I" + os.path.join(ROOT, "cubert_b200", "csrc", "kernels"),
                    os.path.join(ROOT, "tests", "window_protocol_host.cpp"), "-o", out], check=True)
    return C.CDLL(out)


def over_at(host, readings):
    a = np.array(readings, dtype=np.uint64)
    return host.wait_over_at(a.ctypes.data_as(C.c_void_p), len(a))


def test_a_wait_ends_after_its_time(host):
    every = 50 * 1000                                            # 64 polls
    readings = [10 ** 18 + every * i for i in range(10000)]
    assert over_at(host, readings) == 200 * MS // every + 2      # the first reading past 0.2 s


@pytest.mark.parametrize("away", [250 * MS, 10 ** 12])
@pytest.mark.parametrize("at", [1, 100, 3990])
def test_time_off_the_sm_does_not_end_a_wait(host, at, away):
    """A block that comes back after the deadline has had no chance to look: it goes on for what is left of its 0.2 s,
    less a millisecond."""
    every = 50 * 1000
    readings = [10 ** 18 + every * i + (away if i >= at else 0) for i in range(10000)]
    # a gap of 20 readings' time: 19 readings fewer, or the first one back where less than that was left
    assert over_at(host, readings) == max(200 * MS // every + 2 - 19, at + 1)


def test_every_wait_ends(host):
    """However often a block is taken off, 201 gaps are enough."""
    assert over_at(host, [10 ** 18 + 10 ** 10 * i for i in range(1000)]) == 202


class Barrier:
    def __init__(self, need):
        self.need, self.here, self.phases = need, 0, 0

    def arrive(self):
        self.here += 1
        if self.here == self.need:
            self.here, self.phases = 0, self.phases + 1


class Block:
    """One block of the kernel: a warp that takes items and loads, one per tile that multiplies, four per tile for the softmax."""
    STAGES, QUERIES, SLOTS = 2, 2, 8

    def __init__(self, host, rng, tiles, items, lost=None, giving_up=0.0, no_more_after=None):
        self.host, self.rng, self.tiles, self.queue, self.giving_up, self.no_more_after = host, rng, tiles, list(items), giving_up, no_more_after
        self.rows_by_tma = tiles == 2
        one = lambda n, need: [Barrier(need) for _ in range(n)]
        self.qfull, self.qempty = one(2, 1), one(2, tiles + (4 * tiles if self.rows_by_tma else 0))
        self.kfull, self.kempty, self.vfull, self.vempty = one(2, 1), one(2, tiles), one(2, 1), one(2, tiles)
        self.sfull, self.sfree, self.pfull, self.ofull = one(tiles, 2), one(tiles, 4), one(tiles, 4), one(tiles, 1)
        self.takes, self.answers, self.stop = Barrier(1), {}, False
        self.slots = [None] * self.SLOTS
        self.turns = C.create_string_buffer(host.turns_size())
        host.turns_reset(self.turns)
        self.begun, self.rows = [], set()                        # items begun or taken over; (item, tile, warp) written
        self.lost, self.events = lost, 0                         # the number of the completion that never comes

    def complete(self, barrier):
        """An asynchronous completion: a copy's bytes, a product's commit, a taken block's answer."""
        self.events += 1
        if self.events != self.lost:
            barrier.arrive()

    def add(self, turn, item):
        self.host.turns_add(self.turns, turn, item)
        self.begun.append(item)

    def loader(self):
        item, step, turn, ok, asked = self.queue.pop(0), 0, 0, True, True
        while item >= 0 and ok:
            self.add(turn, item)
            qb = turn % 2
            if turn >= 2:
                ok = yield self.qempty[qb], turn // 2 - 1
            if ok:
                self.complete(self.qfull[qb])
            n = self.rng.choice([0, 0, 1, 1, 2, 3, 6])
            for s in range(n + 1):
                if not ok:
                    break
                end = s == n
                flags = 0 if end else self.rng.randrange(1, 1 << self.tiles)
                if end:
                    asked = not self.stop
                    if asked:
                        taken = self.queue.pop(0) if self.queue else -1
                        self.answers[turn & 1] = taken
                        self.complete(self.takes)
                st = step % 2
                if step >= 2:
                    ok = yield self.kempty[st], step // 2 - 1
                self.slots[step % self.SLOTS] = (step, item, 0 if end else 1, flags)
                if ok:
                    self.complete(self.kfull[st])
                if ok and step >= 2:
                    ok = yield self.vempty[st], step // 2 - 1
                if ok:
                    self.complete(self.vfull[st])
                step += ok
            if ok and asked:
                ok = yield self.takes, turn
            item = self.answers[turn & 1] if ok and asked else -1
            turn += 1
        if ok:
            st = step % 2
            if step >= 2:
                ok = yield self.kempty[st], step // 2 - 1
            if ok:
                self.slots[step % self.SLOTS] = (step, -1, -1, 0)
                self.complete(self.kfull[st])
        if not ok and turn > 0:
            if (yield self.takes, turn - 1) and self.answers[(turn - 1) & 1] >= 0:
                self.add(turn, self.answers[(turn - 1) & 1])

    def step_of(self, step):
        got = self.slots[step % self.SLOTS]
        assert got[0] == step, "a descriptor was overwritten before its step"
        return got[1:]

    def multiplier(self, t):
        step, turn, ok, new_item = 0, 0, True, True
        while ok:
            st, before = step % 2, (step + 1) % 2
            ok = yield self.kfull[st], step // 2
            if not ok:
                break
            _, columns, flags = self.step_of(step)
            if new_item and columns >= 0:
                ok = yield self.qfull[turn % 2], turn // 2
                new_item = False
            if step > 0 and ok:
                ok = yield self.sfree[t], step - 1
            if ok:
                self.complete(self.sfull[t])
                self.sfull[t].arrive()
                if columns >= 0:
                    self.complete(self.kempty[st])
                if columns == 0:
                    self.complete(self.qempty[turn % 2])
            if columns < 0:
                break
            if step > 0:
                if ok:
                    ok = yield self.vfull[before], (step - 1) // 2
                if ok:
                    ok = yield self.pfull[t], step - 1
                if ok:
                    self.complete(self.ofull[t])
                    self.complete(self.vempty[before])
            if columns == 0:
                new_item, turn = True, turn + 1
            step += 1

    def softmax(self, t, w):
        step, turn = 0, 0
        while True:
            ok = yield self.sfull[t], step
            if not ok:
                return self.host.turns_gave_up(self.turns, turn)
            item, columns, _ = self.step_of(step)
            if columns < 0:
                return
            waited = True
            while ok:
                if not waited:
                    ok = yield self.sfull[t], step
                waited = False
                if not ok:
                    break
                _, columns, flags = self.step_of(step)
                if flags >> t & 1:
                    if step > 0:
                        ok = yield self.ofull[t], step - 1
                    self.sfree[t].arrive()
                else:
                    if step > 0:
                        ok = yield self.ofull[t], step - 1
                    if not ok or columns == 0:
                        break
                    self.sfree[t].arrive()
                if ok:
                    self.pfull[t].arrive()
                step += 1
            if not ok:
                return self.host.turns_gave_up(self.turns, turn)
            self.sfree[t].arrive()
            self.pfull[t].arrive()
            self.rows.add((item, t, w))
            if self.rows_by_tma:
                self.qempty[turn % 2].arrive()
            if turn == self.no_more_after:
                self.stop = True                                 # a row to compute again
            step, turn = step + 1, turn + 1

    def run(self):
        """Every warp to its end; the number of waits that gave up."""
        warps = [self.loader()] + [self.multiplier(t) for t in range(self.tiles)] + [self.softmax(t, w) for t in range(self.tiles) for w in range(4)]
        waits, gave_up = {}, 0
        for g in warps:
            waits[g] = next(g)
        while waits:
            ready = [g for g, (bar, phase) in waits.items() if bar.phases % 2 != phase % 2]
            clean = self.lost is None and self.giving_up == 0
            assert not clean or all(waits[g][0].phases == waits[g][1] + 1 for g in ready), "a parity of another phase"
            late = [g for g in waits if g not in ready]
            fails = late and (not ready or self.rng.random() < self.giving_up)
            g = self.rng.choice(late if fails else ready)
            gave_up += bool(fails)
            try:
                waits[g] = g.send(not fails)
            except StopIteration:
                del waits[g]
        return gave_up

    def check(self, gave_up):
        first, known = self.host.turns_first_bad(self.turns), self.host.turns_known(self.turns)
        again = [self.host.turns_item(self.turns, turn) for turn in range(first, known)]
        whole = lambda item: all((item, t, w) in self.rows for t in range(self.tiles) for w in range(4))
        missing = [item for item in self.begun if not whole(item)]
        assert set(missing) <= set(again), (missing, again)
        assert len(again) <= 4 and again == self.begun[len(self.begun) - len(again):]
        assert gave_up or (first == 0x7fffffff and not missing)
        assert not missing or first != 0x7fffffff                # it is counted


@pytest.mark.parametrize("tiles", [1, 2])
def test_without_a_give_up_every_item_is_written_once(host, tiles):
    for seed in range(150):
        rng = random.Random(seed)
        n = rng.choice([1, 2, 3, 5, 9])
        block = Block(host, rng, tiles, range(n), no_more_after=rng.choice([None, None, 0, 2]))
        assert block.run() == 0
        block.check(0)
        if block.no_more_after is None:
            assert block.begun == list(range(n))
        else:                                                    # rows to compute again: no item is asked for far behind them
            assert len(block.begun) <= block.no_more_after + 5


@pytest.mark.parametrize("tiles", [1, 2])
def test_every_row_left_without_a_result_is_found(host, tiles):
    """A completion that never comes, anywhere in a run: all warps end, and the items with missing rows are the ones written over."""
    for seed in range(600):
        rng = random.Random(seed)
        n = rng.choice([1, 2, 3, 5, 9])
        block = Block(host, rng, tiles, range(n), lost=rng.randrange(1, 12 * n * tiles + 6))
        block.check(block.run())


@pytest.mark.parametrize("tiles", [1, 2])
def test_every_row_is_found_when_single_waits_give_up(host, tiles):
    """A warp whose wait gives up too early, while the others go on."""
    for seed in range(600):
        rng = random.Random(seed)
        block = Block(host, rng, tiles, range(rng.choice([1, 2, 3, 5, 9])), giving_up=rng.choice([0.002, 0.01, 0.05]))
        block.check(block.run())
