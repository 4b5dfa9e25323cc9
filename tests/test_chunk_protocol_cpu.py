"""The barrier protocol of the tensor-core chunk attention (paged_chunk_tc5.cuh) as a model on the CPU: a producer, two MMA warps and two
softmax groups that take turns in a random order, with loads that land in any order.

A wait on an mbarrier names the parity of a phase, so it is right only while the barrier is in that phase or just behind it: one
phase too early it passes at once, one too late it never does.  The model counts phases and stops at either; it also checks that a
product finds its own tile in its stage.  What it states is the kernel's order of arrivals and waits, step by step."""
import random

import pytest


class Fault(Exception):
    pass


class Bar:
    """An mbarrier that counts its phases."""

    def __init__(self, name, count=1):
        self.name, self.count, self.pending, self.done = name, count, count, 0

    def arrive(self, n=1):
        for _ in range(n):
            self.pending -= 1
            if self.pending == 0:
                self.pending, self.done = self.count, self.done + 1

    def passes(self, phase):
        """Would the hardware's parity wait for `phase` pass?  Faults when its answer is not the truth."""
        parity = (self.done - 1) % 2 == phase % 2
        if parity and self.done <= phase:
            raise Fault(f"{self.name}: a wait for phase {phase} passes although only {self.done} are complete")
        if self.done > phase + 1:
            raise Fault(f"{self.name}: a wait for phase {phase} was overtaken, {self.done} are complete")
        return parity


class Order:
    """Places of the tiles in the ring (TcOrder)."""

    def __init__(self, p0, n, split):
        self.p0, self.n, self.ahead = p0, n, min(2 if split else 1, n)

    def k(self, t):
        return self.p0 + t if t < self.ahead else self.p0 + 2 * t - self.ahead + 1

    def v(self, t):
        return self.p0 + self.ahead + 2 * t if t < self.n - self.ahead else self.p0 + self.n + t


class Model:
    def __init__(self, items, stages, seed, full_barriers=2, idle_slot_answers=True, item_slots=4):
        self.items, self.stages, self.rng = items, stages, random.Random(seed)
        self.full_barriers, self.idle_slot_answers, self.slots = full_barriers, idle_slot_answers, item_slots
        self.full = [[Bar(f"full[{r}][{i}]") for i in range(stages)] for r in range(full_barriers)]
        self.empty = [Bar(f"empty[{i}]", 2) for i in range(stages)]
        pair = lambda name: [Bar(f"{name}[{s}]") for s in range(2)]
        self.s_full, self.p_full, self.o_full, self.q_full = pair("s_full"), pair("p_full"), pair("o_full"), pair("q_full")
        self.meet_all = Bar("meet_all", 2)
        self.item_full = [Bar(f"item_full[{i}]") for i in range(item_slots)]
        self.item_empty = [Bar(f"item_empty[{i}]", 4) for i in range(item_slots)]
        self.content = [None] * stages          # ring place of the tile that a stage holds
        self.flying = []                        # loads that have not landed
        self.commits = [[], []]                 # arrivals that wait for a slot's products, in order

    def full_wait(self, at):
        stage, turn = at % self.stages, at // self.stages
        return self.full[turn % self.full_barriers][stage], turn // self.full_barriers

    def producer(self):
        pos = 0
        for i, (n, split) in enumerate(self.items):
            slot = i % self.slots
            if i >= self.slots:
                yield self.item_empty[slot], i // self.slots - 1
            self.item_full[slot].arrive()
            order = Order(pos, n, split)
            at = sorted([order.k(t) for t in range(n)] + [order.v(t) for t in range(n)])
            assert at == list(range(pos, pos + 2 * n))
            for a in at:
                if a >= self.stages:
                    yield self.empty[a % self.stages], a // self.stages - 1
                self.flying.append(a)
                yield None
            pos += 2 * n

    def land(self, a):
        self.content[a % self.stages] = a
        self.full_wait(a)[0].arrive()

    def mma(self, s):
        pos = products = 0
        for i, (n, split) in enumerate(self.items):
            slot = i % self.slots
            yield self.item_full[slot], i // self.slots
            self.item_empty[slot].arrive()
            order = Order(pos, n, split)
            pos += 2 * n
            yield self.q_full[s], i
            if split:
                yield self.q_full[s ^ 1], i
            tiles = range(s if split else 0, n, 2 if split else 1)
            if not tiles and self.idle_slot_answers:
                self.commits[s].append([(self.o_full[s], 1)])
            for t in tiles:
                for a, bars in ((order.k(t), [(self.s_full[s], 1)]), (order.v(t), [(self.o_full[s], 1)] if t == tiles[-1] else [])):
                    yield self.full_wait(a)
                    if a == order.v(t):
                        yield self.p_full[s], products
                    if self.content[a % self.stages] != a:
                        raise Fault(f"slot {s} multiplies place {a}, its stage holds {self.content[a % self.stages]}")
                    self.commits[s].append(bars + [(self.empty[a % self.stages], 2 if split else 1)])
                products += 1

    def group(self, g):
        tiles_done = finished = met = 0
        was_split = True
        for i, (n, split) in enumerate(self.items):
            slot = i % self.slots
            yield self.item_full[slot], i // self.slots
            if split and not was_split:
                self.meet_all.arrive()
                yield self.meet_all, met
                met += 1
            was_split = split
            self.q_full[g].arrive()
            yield None
            mine = range(g if split else 0, n, 2 if split else 1)
            for _ in mine:
                yield self.s_full[g], tiles_done
                tiles_done += 1
                self.p_full[g].arrive()
            if mine or self.idle_slot_answers:
                yield self.o_full[g], finished
                finished += 1
            if split:
                for _ in range(2):
                    self.meet_all.arrive()
                    yield self.meet_all, met
                    met += 1
            self.item_empty[slot].arrive()

    def run(self):
        agents = {name: [gen, None] for name, gen in (("producer", self.producer()), ("mma 0", self.mma(0)), ("mma 1", self.mma(1)),
                                                      ("group 0", self.group(0)), ("group 1", self.group(1)))}
        # some parts of the machine are slow in this run: the schedules that a fair draw hardly ever makes
        weight = {who: self.rng.choice([1, 1, 8, 64]) for who in [*agents, "land", 0, 1]}
        idle = 0
        while agents:
            moves = list(agents) + ["land"] * bool(self.flying) + [s for s in (0, 1) if self.commits[s]]
            who = self.rng.choices(moves, [weight[m] for m in moves])[0]
            idle += 1
            if idle > 20000:
                raise Fault(f"nothing moves: {sorted(map(str, agents))}")
            if who == "land":
                self.land(self.flying.pop(self.rng.randrange(len(self.flying))))
            elif who in (0, 1):
                for bar, n in self.commits[who].pop(0):
                    bar.arrive(n)
            else:
                gen, waits = agents[who]
                if waits is not None and not waits[0].passes(waits[1]):
                    continue
                try:
                    agents[who][1] = next(gen)
                except StopIteration:
                    del agents[who]
            idle = 0


def batches(seed, split_only):
    rng = random.Random(seed)
    return [(rng.choice([1, 1, 1, 2, 3, 4, 7]), split_only or rng.random() < 0.6) for _ in range(rng.randint(3, 12))]


def faults(stages, **kw):
    found = []
    for seed in range(120):
        try:
            Model(batches(seed, True), stages, seed, **kw).run()
        except Fault as f:
            found.append(str(f))
    return found


@pytest.mark.parametrize("stages", [4, 5, 8])
def test_the_model_sees_a_slot_that_nobody_waits_for(stages):
    """Without an answer from a slot that has no tile, its MMA warp is overtaken at the queries' barrier."""
    found = faults(stages, idle_slot_answers=False)
    assert any("q_full" in f for f in found), found[:5]


@pytest.mark.parametrize("stages", [4, 5, 8])
def test_a_slot_without_tiles_is_waited_for(stages):
    assert not [f for f in faults(stages) if "q_full" in f]


# ring stages: heads of 128 with f32 / bf16 activations, heads of 64; f32 activations share every item between the slots
@pytest.mark.parametrize("stages,split_only", [(4, True), (5, False), (5, True), (8, False), (8, True)])
def test_no_wait_is_early_or_overtaken(stages, split_only):
    for seed in range(200):
        Model(batches(seed, split_only), stages, seed).run()


def test_the_model_sees_a_stage_asked_for_before_the_tile_ahead_has_landed():
    """With one `full` barrier a stage, a slot's wait passes while the other slot's tile before it is still on its way."""
    found = faults(4, full_barriers=1) + faults(5, full_barriers=1)
    assert found and all("full[0]" in f and "passes" in f for f in found)


def unwinding(fail_at, fail_where, items):
    """The producer's requests for blocks that have not started, up to a wait that runs out (`fail_where` of round `fail_at`) or the
    answer "none" after `items` blocks.  Returns (requests made, phases waited for in full, phase of the last wait or None)."""
    asked = answered = 0
    waited, ok, index = [], True, 0
    while ok:
        if asked > answered:
            if (fail_at, fail_where) == (asked, "answer"):
                ok = False
                break
            waited.append(answered)
            answered += 1
            index += 1
            if index >= items:
                break
        asked += 1
        if asked - 1 == fail_at and fail_where == "deal":
            ok = False
            break
        if asked - 1 == fail_at and fail_where == "fetch":
            ok = False
    last = answered if asked > answered else None
    return asked, waited, last


@pytest.mark.parametrize("where", ["answer", "deal", "fetch", None])
def test_a_block_that_gives_up_waits_for_the_answer_on_its_way(where):
    """However the producer ends, every request's phase is waited for once and in order; only the answer "none" leaves nothing open."""
    for fail_at in range(6):
        asked, waited, last = unwinding(fail_at, where, 5)
        assert waited + ([last] if last is not None else []) == list(range(asked))
        assert (last is None) == (where is None or asked == 5 and len(waited) == 5)
