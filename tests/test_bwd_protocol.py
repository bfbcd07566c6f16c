"""A model of the attention-gradient kernel's synchronisation protocol, run on the CPU.

attn_bwd.cuh runs, per CTA, a producer, a waiter, an MMA issuer, eight softmax warps and an
epilogue warpgroup over the flat sequence of its items' tiles.  As for the forward kernel,
each role's schedule is restated as a generator and run under random interleavings with
asynchronous copies and an in-order tensor pipe; the model checks that every schedule ends,
that no named barrier keeps arrivals, and that no buffer (X1, X2, the Y1 and Y2 slots, the
statistics slots, T1, T2, the accumulators) is read before it is written or overwritten
before it is read.  Planted mistakes must be caught.
"""

from __future__ import annotations

import random

import pytest

from test_pipeline_protocol import Model

Y1, Y2 = 3, 2
GROUPS = 2  # the softmax warps, as two warpgroups of four


class BwdModel(Model):
    def __init__(self, items, dq, rnd, fault=None):
        super().__init__(items, rnd, fault)
        self.dq = dq
        self.nb = {3: [64, 0, 0], 4: [288, 0, 0], 5: [288, 0, 0], 6: [160, 0, 0], 7: [160, 0, 0]}
        self.buf = {}
        # (item, first, last) of every tile
        self.tiles = [(i, j == 0, j == n - 1) for i, n in enumerate(items) for j in range(n)]
        self.busy = [i for i, n in enumerate(items) if n]

    def load(self, name, full, tag):
        self.buf[name] = ("in flight", tag)

        def land():
            self.buf[name] = tag
            self.complete(full)
        self.copies.append(land)

    def expect(self, who, name, tag):
        if self.buf.get(name) != tag:
            self.errors.append(f"{who}: {name} holds {self.buf.get(name)}, wanted {tag}")

    def producer(self):
        items = 0
        for n, (item, first, last) in enumerate(self.tiles):
            s1, s2 = n % Y1, n % Y2
            if n >= Y1:
                if self.fault != "no_y1_wait":
                    yield self.wait(f"Y1_EMPTY{s1}", n // Y1 - 1)
                yield self.wait(f"Y1_FULL{s1}", n // Y1 - 1)
            self.load(f"Y1_{s1}", f"Y1_FULL{s1}", n)
            if first and items > 0:
                if self.fault != "no_x1_wait":
                    yield self.wait("X1_EMPTY", items - 1)
                yield self.wait("X1_FULL", items - 1)
            if first:
                self.load("X1", "X1_FULL", item)
            if n >= Y2:
                yield self.wait(f"Y2_EMPTY{s2}", n // Y2 - 1)
                yield self.wait(f"Y2_FULL{s2}", n // Y2 - 1)
            self.load(f"Y2_{s2}", f"Y2_FULL{s2}", n)
            if first:
                if items > 0:
                    yield self.wait("X2_EMPTY", items - 1)
                    yield self.wait("X2_FULL", items - 1)
                self.load("X2", "X2_FULL", item)
                items += 1
            if not self.dq:
                u = n - 2
                if u >= 0:
                    if self.fault != "no_stat_wait":
                        yield self.wait(f"Y1_EMPTY{u % Y1}", u // Y1)
                    yield self.wait(f"STAT{u % 2}", u // 2)
                self.load(f"STAT_{n % 2}", f"STAT{n % 2}", n)

    def waiter(self):
        items = 0
        for n, (item, first, last) in enumerate(self.tiles):
            if first:
                yield self.wait("X1_FULL", items)
            yield self.wait(f"Y1_FULL{n % Y1}", n // Y1)
            yield self.sync(3)
            if first:
                yield self.wait("X2_FULL", items)
                items += 1
            yield self.wait(f"Y2_FULL{n % Y2}", n // Y2)
            yield self.sync(3)

    # ---- tensor work
    def t1_name(self, n):
        return f"T1_{n % 2}" if self.dq else "T1_0"

    def op(self, fn):
        self.pipe.append(("op", fn))

    def commit(self, name):
        self.pipe.append(("commit", name))

    def issue_t1(self, n):
        item, first, last = self.tiles[n]

        def run():
            self.expect(f"T1({n})", "X1", item)
            self.expect(f"T1({n})", f"Y1_{n % Y1}", n)
            old = self.buf.get(self.t1_name(n))
            if old is not None and old[0] != "used":
                self.errors.append(f"T1({n}) overwrote {old}")
            self.buf[self.t1_name(n)] = ("s", n, 0)
        self.op(run)
        self.commit(f"T1_FULL{n % 2 if self.dq else 0}")
        if last and self.fault != "no_x1_commit":
            self.commit("X1_EMPTY")

    def issue_t2(self, n):
        item, first, last = self.tiles[n]

        def run():
            self.expect(f"T2({n})", "X2", item)
            self.expect(f"T2({n})", f"Y2_{n % Y2}", n)
            old = self.buf.get("T2")
            if old is not None and old[0] != "used":
                self.errors.append(f"T2({n}) overwrote {old}")
            self.buf["T2"] = ("dp", n, 0)
        self.op(run)
        self.commit("T2_FULL")
        if self.dq:
            self.commit(f"Y2_EMPTY{n % Y2}")
        if last:
            self.commit("X2_EMPTY")

    def issue_acc(self, which, n, src, want, y):
        item, first, last = self.tiles[n]

        def run():
            self.expect(f"acc{which}({n})", src, want)
            self.expect(f"acc{which}({n})", y, n)
            acc = self.buf.get(f"A{which}")
            if first:
                if acc is not None and acc[0] != "read":
                    self.errors.append(f"acc{which}({n}) overwrote {acc}")
            elif acc != ("sum", item, n - 1):
                self.errors.append(f"acc{which}({n}) added to {acc}")
            self.buf[f"A{which}"] = ("sum", item, n)
            self.buf[src] = ("used",)
        self.op(run)
        self.commit(f"Y{1 if which == 1 else 2}_EMPTY{n % (Y1 if which == 1 else Y2)}")
        if last:
            self.commit(f"ACC{which}")

    def mma(self):
        total = len(self.tiles)
        items = 0
        if self.dq:
            for k in range(min(2, total)):
                yield self.sync(3)
                self.issue_t1(k)
                if k == 0:
                    yield self.sync(3)
                    self.issue_t2(0)
            for n in range(total):
                first = self.tiles[n][1]
                yield self.sync(5)
                if n + 1 < total:
                    yield self.sync(3)
                    self.issue_t2(n + 1)
                if first and items > 0 and self.fault != "no_acc_wait":
                    yield self.sync(6)
                self.issue_acc(1, n, self.t1_name(n), ("ds", n), f"Y1_{n % Y1}")
                if n + 2 < total:
                    yield self.sync(3)
                    self.issue_t1(n + 2)
                items += first
            if items:
                yield self.sync(6)
            return
        if total:
            yield self.sync(3)
            self.issue_t1(0)
            yield self.sync(3)
            self.issue_t2(0)
        for n in range(total):
            first = self.tiles[n][1]
            if first and items > 0 and self.fault != "no_acc_wait":
                yield self.sync(7)
            yield self.sync(4)
            self.issue_acc(2, n, "T1_0", ("p", n), f"Y2_{n % Y2}")
            if n + 1 < total:
                yield self.sync(3)
                self.issue_t1(n + 1)
            if first and items > 0 and self.fault != "no_acc_wait":
                yield self.sync(6)
            yield self.sync(5)
            self.issue_acc(1, n, "T2", ("ds", n), f"Y1_{n % Y1}")
            if n + 1 < total:
                yield self.sync(3)
                self.issue_t2(n + 1)
            items += first
        if items:
            yield self.sync(7)
            yield self.sync(6)

    def part(self, name, kind, n, done):
        """One warpgroup has turned its half of `name` into `done`."""
        old = self.buf.get(name)
        if old is None or old[:2] != (kind, n):
            self.errors.append(f"softmax read {name} = {old}, wanted {(kind, n)}")
            return
        halves = old[2] + 1
        self.buf[name] = (done, n) if halves == GROUPS else (kind, n, halves)

    def softmax(self, group):
        for n in range(len(self.tiles)):
            t1 = self.t1_name(n)
            yield self.wait(f"T1_FULL{n % 2 if self.dq else 0}", n // 2 if self.dq else n)
            if not self.dq:
                yield self.wait(f"STAT{n % 2}", n // 2)
                self.expect(f"P({n})", f"STAT_{n % 2}", n)
                self.part(t1, "s", n, "p")
                yield lambda: True
                self.arrive(4, warps=4)
            if self.fault != "no_t2_wait":
                yield self.wait("T2_FULL", n)
            if self.dq:
                if self.buf.get("T2", (None,))[:2] != ("dp", n):
                    self.errors.append(f"dS({n}) read T2 = {self.buf.get('T2')}")
                else:
                    halves = self.buf["T2"][2] + 1
                    self.buf["T2"] = ("used",) if halves == GROUPS else ("dp", n, halves)
                self.part(t1, "s", n, "ds")
            else:
                self.expect(f"dS({n})", f"STAT_{n % 2}", n)
                self.part("T2", "dp", n, "ds")
            yield lambda: True
            self.arrive(5, warps=4)

    def epilogue(self):
        for k, item in enumerate(self.busy):
            for which in ([1] if self.dq else [2, 1]):
                yield self.wait(f"ACC{which}", k)
                last = max(n for n, t in enumerate(self.tiles) if t[0] == item)
                self.expect(f"epilogue of item {item}", f"A{which}", ("sum", item, last))
                self.buf[f"A{which}"] = ("read",)
                yield lambda: True
                self.arrive(5 + which, warps=4)

    def run(self):
        roles = [self.producer(), self.waiter(), self.mma(), self.epilogue()]
        roles += [self.softmax(g) for g in range(GROUPS)]
        ready = [None] * len(roles)
        done = [False] * len(roles)
        while not self.errors:
            runnable = [r for r in range(len(roles)) if not done[r] and (ready[r] is None or ready[r]())]
            n_async = len(self.copies) + (1 if self.pipe else 0)
            if not runnable and not n_async:
                break
            pick = self.rnd.randrange(len(runnable) + n_async)
            if pick < len(runnable):
                r = runnable[pick]
                try:
                    ready[r] = next(roles[r])
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


def errors_of(items, dq, seed, fault=None):
    model = BwdModel(items, dq, random.Random(seed), fault)
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


@pytest.mark.parametrize("fault,dqs", [
    # dK/dV: the wait for the previous tile's statistics slot already implies the Y1 wait.
    ("no_y1_wait", (True,)),
    ("no_x1_wait", (False, True)), ("no_x1_commit", (False, True)),
    ("no_stat_wait", (False,)), ("no_acc_wait", (False, True)), ("no_t2_wait", (False, True)),
])
def test_planted_mistakes_are_caught(fault, dqs):
    for dq in dqs:
        assert any(errors_of([4, 4, 3], dq, seed, fault) for seed in range(25)), (fault, dq)
