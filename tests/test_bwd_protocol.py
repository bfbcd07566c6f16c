"""A model of the attention-gradient kernel's synchronisation protocol, run on the CPU.

attn_bwd.cuh runs, per CTA, a producer, a waiter, an MMA issuer, four softmax warpgroups (two
in this model) and an epilogue warpgroup over the flat sequence of its items' tiles, in two variants (dK/dV and
dQ).  As for the forward kernel, each role's schedule is restated as a generator and run
under random interleavings with asynchronous copies and an in-order tensor pipe; the model
checks that every schedule ends, that no named barrier keeps arrivals, and that no buffer
(X1, X2, the Y1 and Y2 slots, the statistics slots, T1, T2, dS, the accumulators) is read
before it is written or overwritten before it is read.  Planted mistakes must be caught.

The abort is modelled too: from a random step on every mbarrier wait whose phase has not
completed gives up, as after a watchdog expiry, while the others go on; the roles then keep
their barrier rounds as the kernel does.  Every schedule still has to end with no arrivals
left, and no buffer may have two copies in flight.
"""

from __future__ import annotations

import random

import pytest

from test_pipeline_protocol import Model

Y2 = 2
GROUPS = 2  # the softmax warps, as two warpgroups of four


class BwdModel(Model):
    def __init__(self, items, dq, rnd, fault=None, abort_after=None):
        super().__init__(items, rnd, fault)
        self.dq = dq
        self.y1 = 4 if dq else 3
        self.abort_after, self.aborted = abort_after, False
        threads = {3: 64, 10: 160, 11: 160, 12: 160, 13: 160}
        for k in (0, 3):
            threads |= {4 + k: 320 if dq else 288, 5 + k: 320, 6 + k: 288 if dq else 320}
        self.nb = {k: [v, 0, 0] for k, v in threads.items()}
        self.buf = {}
        self.progress = {}
        # (item, first, last) of every tile
        self.tiles = [(i, j == 0, j == n - 1) for i, n in enumerate(items) for j in range(n)]
        self.busy = [i for i, n in enumerate(items) if n]

    # ---- primitives
    def wait(self, name, k):
        """Yields whether the phase completed: after an abort a wait that has not gives up."""
        ready = super().wait(name, k)
        return lambda: "done" if ready() else "gave up" if self.aborted else False

    def landed(self, name, k):
        """The waiter's wait.  After an abort it no longer matters what it answers: copies that
        were never made leave its phases behind."""
        ready = super().wait(name, k)
        return lambda: self.aborted or ready()

    def sync4(self, bar_id):
        """Four warps of a warpgroup sync (a blocking arrival of all of them)."""
        b = self.nb[bar_id]
        gen = b[2]
        self.arrive(bar_id, warps=4)
        return lambda: b[2] > gen

    def fail(self, text):
        if not self.aborted:  # after an abort the data is invalid anyway
            self.errors.append(text)

    def load(self, name, full, tag):
        old = self.buf.get(name)
        if old is not None and old[0] == "in flight":  # an abort does not excuse this
            self.errors.append(f"{name}: a second copy ({tag}) while {old} is in flight")
        self.buf[name] = ("in flight", tag)

        def land():
            self.buf[name] = (tag,)
            self.complete(full)
        self.copies.append(land)

    def expect(self, who, name, tag):
        if self.buf.get(name) not in (tag, (tag,)):
            self.fail(f"{who}: {name} holds {self.buf.get(name)}, wanted {tag}")

    def t_full(self, which, u):
        """Tile u's T1 or T2 commit."""
        return self.wait(f"T{which}_FULL{u % 2}", u // 2)

    # ---- named barriers with two ids
    def tile_bar(self, base, n):
        return base + 3 * (n % 2 if self.fault != f"one_barrier_{base}" else 0)

    def acc(self, which, item):
        return (10 if which == 1 else 12) + (item % 2 if self.fault != "one_acc_barrier" else 0)

    def x1(self, item):
        return 12 + (item % 2 if self.fault != "one_x1_barrier" else 0)

    # ---- loads
    def reuse(self, fault, *wait):
        """The wait before a buffer is loaded again; false after an abort."""
        ok = True
        if self.fault != fault:
            ok = (yield wait[0]) == "done"
        return ok and not self.aborted

    def producer(self):
        items = 0
        for n, (item, first, last) in enumerate(self.tiles):
            s1, s2 = n % self.y1, n % Y2
            if n >= self.y1:
                done = self.wait(f"Y1_EMPTY{s1}", n // self.y1 - 1) if self.dq else self.t_full(2, n - 2)
                if not (yield from self.reuse("no_y1_wait", done)):
                    return
            self.load(f"Y1_{s1}", f"Y1_FULL{s1}", n)
            if first and not self.dq:
                if items > 0 and not (yield from self.reuse("no_x1_wait", self.t_full(1, n - 1))):
                    return
                self.load("X1", "X1_FULL", item)
            if n >= Y2:
                done = self.t_full(2, n - 2) if self.dq else self.wait(f"Y2_EMPTY{s2}", n // Y2 - 1)
                if not (yield from self.reuse("no_y2_wait", done)):
                    return
            self.load(f"Y2_{s2}", f"Y2_FULL{s2}", n)
            if first:
                if items > 0 and not (yield from self.reuse("no_x2_wait", self.t_full(2, n - 1))):
                    return
                self.load("X2", "X2_FULL", item)
                items += 1
            if not self.dq:
                if n >= 2 and not (yield from self.reuse("no_stat_wait", self.t_full(2, n - 1))):
                    return
                self.load(f"STAT_{n % 2}", f"STAT{n % 2}", n)

    def loaded(self, which):
        """The waiter's wait for the operands of T1 / T2 of the next tile in turn."""
        n = self.seen[which]
        self.seen[which] += 1
        if n >= len(self.tiles):
            return
        item, first, last = self.tiles[n]
        if first and not (self.dq and which == 1):
            yield self.landed(f"X{which}_FULL", self.busy.index(item))
        slots = self.y1 if which == 1 else Y2
        yield self.landed(f"Y{which}_FULL{n % slots}", n // slots)

    def waiter(self):
        self.seen = {1: 0, 2: 0}
        if not self.tiles:
            return
        for which in (1, 2):
            yield from self.loaded(which)
            yield self.sync(3)
        for n in range(len(self.tiles)):
            for which, bar in ((1, 4), (2, 5)) if self.dq else ((1, 5), (2, 6)):
                if self.fault != "no_load_wait":
                    yield from self.loaded(which)
                yield self.sync(self.tile_bar(bar, n))

    # ---- tensor work
    def op(self, fn):
        self.pipe.append(("op", fn))

    def commit(self, name):
        self.pipe.append(("commit", name))

    def issue_t(self, which, n):
        item = self.tiles[n][0]
        slot = n % (self.y1 if which == 1 else Y2)

        def run():
            self.expect(f"T{which}({n})", f"X{which}", item)
            self.expect(f"T{which}({n})", f"Y{which}_{slot}", n)
            old = self.buf.get(f"T{which}")
            if old is not None and old[0] != "used":
                self.fail(f"T{which}({n}) overwrote {old}")
            self.buf[f"T{which}"] = ("raw", n, 0)
        self.op(run)
        self.commit(f"T{which}_FULL{n % 2}")
        if self.dq and which == 1 and self.tiles[n][2]:
            self.commit("X1_DONE")

    def issue_acc(self, which, n, src, half):
        item, first, last = self.tiles[n]
        y = f"Y{which}_{n % (self.y1 if which == 1 else Y2)}"

        def run():
            got = self.buf.get(src)
            if got is None or got[:2] != ("done", n) or got[2] <= half:
                self.fail(f"acc{which}({n}, {half}): {src} holds {got}")
            self.expect(f"acc{which}({n})", y, n)
            acc = self.buf.get(f"A{which}")
            if half == 1:
                if acc != ("sum", item, n, 0):
                    self.fail(f"acc{which}({n}) second half after {acc}")
            elif first:
                if acc is not None and acc[0] != "read":
                    self.fail(f"acc{which}({n}) overwrote {acc}")
            elif acc != ("sum", item, n - 1, 1):
                self.fail(f"acc{which}({n}) added to {acc}")
            self.buf[f"A{which}"] = ("sum", item, n, half)
            if half == 1:
                self.buf[src] = ("used",)
        self.op(run)
        if self.dq and half == 1:
            self.commit(f"Y1_EMPTY{n % self.y1}")
        if which == 2 and half == 1:
            self.commit(f"Y2_EMPTY{n % Y2}")
        if last and half == 1:
            self.commit(f"ACC{which}")

    def mma(self):
        total = len(self.tiles)
        items = 0
        if total:
            yield self.sync(3)
            if self.dq:
                yield self.sync(self.x1(0))
            self.issue_t(1, 0)
            yield self.sync(3)
            self.issue_t(2, 0)
        for n in range(total):
            first = self.tiles[n][1]
            more = n + 1 < total
            acc_wait = first and items > 0 and self.fault != "no_acc_wait"
            if self.dq:
                yield self.sync(self.tile_bar(4, n))
                if more and self.tiles[n + 1][1]:
                    yield self.sync(self.x1(items + first))
                if more:
                    self.issue_t(1, n + 1)
                if self.fault != "no_t2_read":
                    yield self.sync(self.tile_bar(5, n))
                if more:
                    self.issue_t(2, n + 1)
                if self.fault == "no_t2_read":
                    yield self.sync(self.tile_bar(5, n))
                if acc_wait:
                    yield self.sync(self.acc(1, items - 1))
                yield self.sync(self.tile_bar(6, n))
                for half in (0, 1):
                    self.issue_acc(1, n, "DS", half)
            else:
                if acc_wait:
                    yield self.sync(self.acc(2, items - 1))
                yield self.sync(self.tile_bar(4, n))
                self.issue_acc(2, n, "T1", 0)
                yield self.sync(self.tile_bar(5, n))
                self.issue_acc(2, n, "T1", 1)
                if more:
                    self.issue_t(1, n + 1)
                if acc_wait:
                    yield self.sync(self.acc(1, items - 1))
                yield self.sync(self.tile_bar(6, n))
                for half in (0, 1):
                    self.issue_acc(1, n, "T2", half)
                if more:
                    self.issue_t(2, n + 1)
            items += first
        if items:
            if not self.dq:
                yield self.sync(self.acc(2, items - 1))
            yield self.sync(self.acc(1, items - 1))

    # ---- softmax
    def read(self, name, n):
        """One warpgroup has its part of T1 or T2 in registers (dQ)."""
        old = self.buf.get(name)
        if old is None or old[:2] != ("raw", n):
            self.fail(f"softmax read {name} = {old} for tile {n}")
            return
        self.buf[name] = ("used",) if old[2] + 1 == GROUPS else ("raw", n, old[2] + 1)

    def put(self, name, n, halves):
        """One warpgroup has written its part of P or dS; `halves` of it are published."""
        old = self.buf.get(name)
        in_place = not self.dq
        if in_place and (old is None or old[:2] not in (("raw", n), ("done", n))):
            self.fail(f"softmax wrote {name} of tile {n} over {old}")
            return
        if not in_place and old is not None and old != ("used",) and old[:2] != ("done", n):
            self.fail(f"dS of tile {n} overwrote {old}")
            return
        seen = self.progress.setdefault((name, n), [])
        seen.append(halves)
        complete = max((k for k in (1, 2) if sum(h >= k for h in seen) >= GROUPS), default=0)
        self.buf[name] = ("done", n, complete)

    def rounds(self, n, start):
        if self.dq:
            for bar in (4, 5, 6)[start:]:
                yield self.sync4(self.tile_bar(bar, n))
        else:
            for bar in (4, 5, 6) if start < 1 else (6,):
                yield self.sync4(self.tile_bar(bar, n))

    def softmax(self, group):
        dead = False
        for n in range(len(self.tiles)):
            if dead:
                yield from self.rounds(n, 0)
                continue
            dead = (yield self.t_full(1, n)) != "done"
            if not self.dq and not dead:
                dead = (yield self.wait(f"STAT{n % 2}", n // 2)) != "done"
            if dead:
                yield from self.rounds(n, 0)
                continue
            if self.dq:
                self.read("T1", n)
                yield lambda: True
                self.arrive(self.tile_bar(4, n), warps=4)
            else:
                self.expect(f"P({n})", f"STAT_{n % 2}", n)
                for half in (0, 1):
                    self.put("T1", n, half + 1)
                    yield lambda: True
                    self.arrive(self.tile_bar(4 + half, n), warps=4)
            if self.fault != "no_t2_wait":
                dead = (yield self.t_full(2, n)) != "done"
            if dead:
                yield from self.rounds(n, 1)
                continue
            if self.dq:
                self.read("T2", n)
                yield lambda: True
                self.arrive(self.tile_bar(5, n), warps=4)
                if n > 0 and self.fault != "no_ds_wait":
                    dead = (yield self.wait(f"Y1_EMPTY{(n - 1) % self.y1}", (n - 1) // self.y1)) != "done"
                if dead:
                    yield from self.rounds(n, 2)
                    continue
                self.put("DS", n, 2)
            else:
                self.expect(f"dS({n})", f"STAT_{n % 2}", n)
                self.put("T2", n, 2)
            yield lambda: True
            self.arrive(self.tile_bar(6, n), warps=4)

    # ---- epilogue
    def epilogue(self):
        x_signals = acc_signals = 0
        tiles = 0
        if self.dq and self.busy:
            self.buf["X1"] = self.busy[0]
            yield lambda: True
            self.arrive(self.x1(0), warps=4)
            x_signals += 1
        ok = True
        for k, item in enumerate(self.busy):
            tiles += self.seq[item]
            if self.dq and k + 1 < len(self.busy):
                if self.fault != "no_x1_wait":
                    ok = (yield self.wait("X1_DONE", k)) == "done"
                if not ok:
                    break
                self.buf["X1"] = self.busy[k + 1]
                yield lambda: True
                self.arrive(self.x1(k + 1), warps=4)
                x_signals += 1
            for which in ([1] if self.dq else [2, 1]):
                ok = (yield self.wait(f"ACC{which}", k)) == "done"
                if not ok:
                    break
                self.expect(f"epilogue of item {item}", f"A{which}", ("sum", item, tiles - 1, 1))
                self.buf[f"A{which}"] = ("read",)
                yield lambda: True
                self.arrive(self.acc(which, k), warps=4)
                acc_signals += 1
            if not ok:
                break
        if ok:
            return
        seen = {"x": 0, "acc": 0}

        def x_round():
            seen["x"] += 1
            if seen["x"] > x_signals:
                yield self.sync4(self.x1(seen["x"] - 1))

        def acc_round(k):
            for which in ([1] if self.dq else [2, 1]):
                seen["acc"] += 1
                if seen["acc"] > acc_signals:
                    yield self.sync4(self.acc(which, k))

        if self.dq:
            yield from x_round()
        for k, item in enumerate(self.busy):
            more, n = k + 1 < len(self.busy), self.seq[item]
            if self.dq and more and n == 1 and self.fault != "x_round_order":
                yield from x_round()
            if k > 0:
                yield from acc_round(k - 1)
            if self.dq and more and (n > 1 or self.fault == "x_round_order"):
                yield from x_round()
            if not more:
                yield from acc_round(k)

    def run(self):
        roles = [self.producer(), self.waiter(), self.mma(), self.epilogue()]
        roles += [self.softmax(g) for g in range(GROUPS)]
        ready = [None] * len(roles)
        done = [False] * len(roles)
        steps = 0
        while not self.errors:
            steps += 1
            if self.abort_after is not None and steps > self.abort_after:
                self.aborted = True
            answer = [True if ready[r] is None else not done[r] and ready[r]() for r in range(len(roles))]
            runnable = [r for r in range(len(roles)) if not done[r] and answer[r]]
            n_async = len(self.copies) + (1 if self.pipe else 0)
            if not runnable and not n_async:
                break
            pick = self.rnd.randrange(len(runnable) + n_async)
            if pick < len(runnable):
                r = runnable[pick]
                try:
                    ready[r] = roles[r].send(None if ready[r] is None else answer[r])
                except StopIteration:
                    done[r], ready[r] = True, None
            elif pick < len(runnable) + len(self.copies):
                self.copies.pop(self.rnd.randrange(len(self.copies)))()
            else:
                kind, x = self.pipe.pop(0)
                x() if kind == "op" else self.complete(x)
        if not self.errors and not all(done):
            self.errors.append(f"deadlock: roles {[r for r in range(len(roles)) if not done[r]]} never finish")
        if not self.errors and any(b[1] for b in self.nb.values()):
            self.errors.append("named barriers left with arrivals")


def errors_of(items, dq, seed, fault=None, abort_after=None):
    model = BwdModel(items, dq, random.Random(seed), fault, abort_after)
    model.run()
    return model.errors


@pytest.mark.parametrize("dq", [False, True])
@pytest.mark.parametrize("items", [[1], [2], [3], [1, 1, 1, 1], [5, 0, 2, 1, 4], [0, 0, 1], [0], [7, 6], [32, 1, 9]])
def test_protocol_holds_under_random_interleavings(items, dq):
    for seed in range(25):
        assert errors_of(items, dq, seed) == []


@pytest.mark.parametrize("dq", [False, True])
def test_protocol_random_item_sequences(dq):
    rnd = random.Random(2)
    for trial in range(150):
        items = [rnd.choice([0, 1, 1, 2, 3, 5, 8]) for _ in range(rnd.randint(1, 6))]
        assert errors_of(items, dq, trial) == [], items


@pytest.mark.parametrize("dq", [False, True])
def test_every_role_ends_after_an_abort(dq):
    rnd = random.Random(3)
    for trial in range(1500):
        items = [rnd.choice([0, 1, 1, 2, 3, 5]) for _ in range(rnd.randint(1, 6))]
        assert errors_of(items, dq, trial, abort_after=rnd.randint(0, 300)) == [], items


@pytest.mark.parametrize("fault,dqs", [
    # Where two waits of the producer follow from each other only one of them can be missed.
    ("no_y1_wait", (True,)), ("no_y2_wait", (True, False)), ("no_x1_wait", (False, True)),
    ("no_x2_wait", (False, True)), ("no_stat_wait", (False,)), ("no_acc_wait", (False, True)),
    ("no_t2_wait", (False, True)), ("no_t2_read", (True,)),
    ("no_ds_wait", (True,)), ("no_load_wait", (False, True)),
])
def test_planted_mistakes_are_caught(fault, dqs):
    for dq in dqs:
        found = [errors_of(items, dq, seed, fault) for items in ([4, 4, 3], [1, 1, 2], [5, 5]) for seed in range(25)]
        assert any(found), (fault, dq)


@pytest.mark.parametrize("fault,dqs", [("x_round_order", (True,)), ("one_barrier_4", (False, True)),
                                       ("one_barrier_5", (True,)), ("one_barrier_6", (False,)),
                                       ("one_acc_barrier", (True,)), ("one_x1_barrier", (True,))])
def test_mistakes_that_only_an_abort_shows_are_caught(fault, dqs):
    for dq in dqs:
        rnd = random.Random(4)
        assert any(errors_of(items, dq, trial, fault, rnd.randint(0, 300))
                   for trial in range(3000) for items in ([1, 1, 1, 1, 2], [5], [2, 1, 3])), (fault, dq)
