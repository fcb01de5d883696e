"""The barriers of the tensor-memory attention as a model on the host: its warps as processes in any order, with the
waits, phases and stages of the kernel.  A wait knows a phase by its parity alone, so none may be two phases behind, and
nothing that is read may have been written over."""
import random

import pytest

OP, SCALES, NANS = 2, 16, 4


class Barrier:
    def __init__(self, need):
        self.need, self.got, self.done = need, 0, 0

    def arrive(self):
        self.got += 1
        if self.got == self.need:
            self.got, self.done = 0, self.done + 1


class Wrong(Exception):
    pass


class Kernel:
    """One CTA on a list of groups (steps, narrow).  `ready`: "both", as in the kernel, narrow groups have a barrier of their own
    that both softmax warpgroups arrive at; "own", that stream 0's alone does; "one", none, stream 0's barrier counts
    all groups, and the other stream looks at it in narrow ones."""

    def __init__(self, groups, stages, ready):
        self.groups, self.RS, self.one_ready, self.both_ready = groups, stages, ready == "one", ready == "both"
        bars = lambda n, need: [Barrier(need) for _ in range(n)]
        self.rfull, self.rempty = [bars(stages, 1) for _ in "kv"], [bars(stages, 1) for _ in "kv"]
        self.full, self.empty = [bars(OP, 1) for _ in "kv"], [bars(OP, 2) for _ in "kv"]
        self.sfull, self.pready = [bars(2, 1) for _ in range(2)], [bars(2, 1) for _ in range(2)]
        self.pvdone, self.ofull, self.qready, self.nready = bars(2, 1), bars(2, 1), bars(2, 1), Barrier(2 if self.both_ready else 1)
        self.stage, self.tile = [[None] * OP, [None] * OP], [None, None]  # step in a stage of keys, of values; group in a query operand
        self.scale, self.parts, self.nans, self.factor = [None] * SCALES, [None] * SCALES, [None] * NANS, None
        self.queue = [[], []]  # products and commits of the two issuing warps, done in order
        self.join = [0, 0]

    def walk(self):
        steps = narrows = wides = 0
        for g, (n, narrow) in enumerate(self.groups):
            yield g, n, narrow, steps, narrows, wides
            steps, narrows, wides = steps + n, narrows + narrow, wides + (not narrow)

    def ready(self, q, g, narrow, narrows, wides):  # what says that the queries of stream q's tile are there
        if self.one_ready:
            return (self.qready[0], g) if narrow or q == 0 else (self.qready[1], wides)
        return (self.nready, narrows) if narrow else (self.qready[q], wides)

    @staticmethod
    def need(what, want):
        if what != want:
            raise Wrong(f"{what} where {want} belongs")

    def own_steps(self, q, n, narrow, steps):
        return range((steps ^ q) & 1 if narrow else 0, n, 2 if narrow else 1)

    def copies(self, v):
        for g, n, narrow, steps, *_ in self.walk():
            for s in range(steps, steps + n):
                if s >= self.RS:
                    yield self.rempty[v][s % self.RS], s // self.RS - 1
                (self.parts if v else self.scale)[s % SCALES] = s
                yield
                self.rfull[v][s % self.RS].arrive()

    def widen(self, v):
        for g, n, narrow, steps, *_ in self.walk():
            if v:
                self.nans[g % NANS] = g
            for s in range(steps, steps + n):
                yield self.rfull[v][s % self.RS], s // self.RS
                if v:
                    self.need(self.parts[s % SCALES], s)
                if s >= OP:
                    yield self.empty[v][s % OP], s // OP - 1
                self.stage[v][s % OP] = s
                yield
                self.full[v][s % OP].arrive()
                self.rempty[v][s % self.RS].arrive()

    def products(self, q):
        turns = 0
        for g, n, narrow, steps, narrows, wides in self.walk():
            yield self.ready(q, g, narrow, narrows, wides)
            own = list(self.own_steps(q, n, narrow, steps))

            def score(j):
                s, turn = steps + own[j], turns + j
                yield self.full[0][s % OP], s // OP
                tile = 0 if narrow else q
                self.queue[q].append(lambda: (self.need(self.stage[0][s % OP], s), self.need(self.tile[tile], g)))
                self.queue[q] += [self.sfull[q][turn & 1].arrive, self.empty[0][s % OP].arrive]
                if narrow:
                    self.empty[0][s % OP].arrive()

            for j in range(min(2, len(own))):
                yield from score(j)
            for j, i in enumerate(own):
                s, turn = steps + i, turns + j
                yield self.full[1][s % OP], s // OP
                yield self.pready[q][turn & 1], turn >> 1
                self.queue[q].append(lambda s=s: self.need(self.stage[1][s % OP], s))
                self.queue[q] += [self.pvdone[q].arrive, self.empty[1][s % OP].arrive]
                if narrow:
                    self.empty[1][s % OP].arrive()
                if j + 2 < len(own):
                    yield from score(j + 2)
            turns += len(own)
            self.queue[q].append(self.ofull[q].arrive)
            yield

    def both(self, q):  # the two warpgroups' own barrier
        self.join[q] += 1
        yield lambda at=self.join[q]: self.join[1 - q] >= at

    def softmax(self, q, rng):
        turns = 0
        for g, n, narrow, steps, narrows, wides in self.walk():
            if not narrow or q == 0:
                self.tile[q] = g
                if narrow:
                    self.factor = g
                yield
                (self.nready if narrow and not self.one_ready else self.qready[q]).arrive()
            else:
                if self.both_ready:
                    self.nready.arrive()
                yield self.ready(0, g, narrow, narrows, wides)
                self.need(self.factor, g)
            own = self.own_steps(q, n, narrow, steps)
            for j, i in enumerate(own):
                yield self.sfull[q][turns & 1], turns >> 1
                self.need(self.scale[(steps + i) % SCALES], steps + i)
                if j and rng.random() < 0.5:
                    yield self.pvdone[q], turns - 1
                yield
                self.pready[q][turns & 1].arrive()
                turns += 1
            yield self.ofull[q], g
            if narrow:
                if q == 1:
                    yield self.ofull[0], g
                    self.tile = [None, None]  # its sums lie there
                yield from self.both(q)
            if not narrow or q == 0:
                yield
                self.need(self.nans[g % NANS], g)
            if narrow:
                yield from self.both(q)

    def engine(self, q):
        while True:
            yield lambda: bool(self.queue[q])
            self.queue[q].pop(0)()
            yield

    def run(self, seed):
        rng = random.Random(seed)
        agents = [self.copies(0), self.copies(1), self.widen(0), self.widen(1), self.products(0), self.products(1), self.softmax(0, rng),
                  self.softmax(1, rng), self.engine(0), self.engine(1)]
        work, waits, alive = 8, [None] * 10, [True] * 10
        slow = [rng.random() < 0.3 for _ in agents]  # a warp may be slow for a while

        def held(a):
            if waits[a] is None:
                return False
            if callable(waits[a]):
                return not waits[a]()
            bar, phase = waits[a]
            return (bar.done & 1) == (phase & 1)  # the phase of this parity is the one under way: not yet

        while any(alive[:work]):
            if rng.random() < 0.05:
                slow[rng.randrange(10)] ^= True
            free = [a for a in range(10) if alive[a] and not held(a)]
            if not free:
                raise Wrong("stuck")
            fast = [a for a in free if not slow[a]]
            a = rng.choice(fast if fast and rng.random() < 0.98 else free)
            if isinstance(waits[a], tuple):
                self.need(waits[a][0].done, waits[a][1] + 1)
            try:
                waits[a] = next(agents[a])
            except StopIteration:
                alive[a] = False


SEQUENCES = {  # (steps, narrow)
    "a prompt of 200 tokens of 4 queries, three heads": [(4, True), (3, False), (2, False), (1, False)] * 3,
    "90 tokens beside 150, heads in turn": [(2, True), (1, False)] * 5 + [(3, True), (2, False)] * 5,
    "whole groups of one step before half ones": [(1, False), (1, False), (4, True)] * 5,
    "whole alone": [(2, False), (1, False), (5, False)] * 4,
    "half alone": [(1, True), (2, True), (5, True)] * 4,
    "single steps": [(1, True), (1, False)] * 8,
}


def runs(name, stages, ready, seeds):
    """How many of the runs in random orders go wrong, of the named groups and of random ones."""
    rng, wrong = random.Random(7), 0
    for seed in range(seeds):
        for groups in (SEQUENCES[name], [(rng.choice([1, 1, 2, 3, 9]), {"whole alone": False, "half alone": True}.get(name, rng.random() < 0.5)) for _ in range(12)]):
            try:
                Kernel(groups, stages, ready).run(seed)
            except Wrong:
                wrong += 1
    return wrong


@pytest.mark.parametrize("stages", [4, 8])
@pytest.mark.parametrize("name", SEQUENCES)
def test_no_wait_takes_another_phase(name, stages):
    assert runs(name, stages, "both", 60) == 0


def test_the_model_finds_phases_taken_for_others():
    """One barrier for the queries of stream 0 in wide and narrow groups: the other stream, which skips its phases in wide
    groups, takes an older phase for a narrow group's.  One of their own for narrow groups that stream 0's softmax alone
    arrives at: where a narrow group of one step has none for the other stream, that stream's products end it before its
    softmax has seen the end of the group before, and it waits for a phase that is past."""
    mixed = [n for n in SEQUENCES if not n.endswith("alone")]
    assert sum(runs(n, 4, "one", 40) for n in mixed) > 0 and sum(runs(n, 8, "own", 40) for n in mixed) > 0
    assert runs("whole alone", 4, "one", 40) == 0
