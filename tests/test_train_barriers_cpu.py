"""CPU: how the warps of the training attention kernels wait for each other, as a model. A block's roles run as generators in random order; a barrier counts its
arrivals as the kernels initialise it. No order may leave all of them waiting, nobody may arrive at a barrier more often than a phase takes, and whoever waits for a
phase may be at most one behind: a parity cannot tell more apart. Copies and products are events that have happened once they are issued (their
completion can only be later, which the random order covers).

The model's numbers of stages, slots and groups are read from the sources."""
import os
import random
import re
from collections import defaultdict

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tensor-ffn_b200", "csrc")


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return f.read()


def constant(text, name, width):
    """of `NAME = HD == 64 ? a : b` or `NAME = a`"""
    m = re.search(r"\b%s = (?:HD == 64 \? (\d+) : )?(\d+)[,;]" % name, text)
    assert m, name
    return int(m.group(1) if m.group(1) and width == 64 else m.group(2))


SLOTS = constant(source("train_attn.cuh"), "kUnitSlots", 64)


class Block:
    def __init__(self, seed):
        self.rng, self.phase, self.arrived, self.need = random.Random(seed), defaultdict(int), defaultdict(int), {}

    def arrive(self, b, n=1):
        for _ in range(n):
            self.arrived[b] += 1
            if self.arrived[b] == self.need[b]:
                self.arrived[b] = 0
                self.phase[b] += 1

    def over(self, b, k):
        """a wait for the k-th phase"""
        def ready():
            assert k <= self.phase[b] <= k + 1, ("a parity cannot tell these apart", b, k, self.phase[b])
            return self.phase[b] > k
        return ready

    def run(self, roles):
        waits, alive = [None] * len(roles), set(range(len(roles)))
        while alive:
            ready = [a for a in alive if waits[a] is None or waits[a]()]
            if not ready:
                return False
            a = self.rng.choice(ready)
            try:
                waits[a] = next(roles[a])
            except StopIteration:
                alive.discard(a)
        return all(n == 0 for b, n in self.arrived.items())


def forward(groups, part, units, own, seed):
    """units: (tiles, units of the groups) of a block's steps; own: each group has a unit to itself"""
    x = Block(seed)
    W, arrive = x.over, x.arrive
    for i in range(part * groups):
        x.need["k full", i] = x.need["v full", i] = 1
        x.need["k empty", i] = x.need["v empty", i] = groups if own else 1
    for g in range(groups):
        for b in ("q full", "s full", "o full"):
            x.need[b, g] = 1
        for b in ("s free", "p full", "o free"):
            x.need[b, g] = 4  # warps
        x.need["q empty", g] = 1 if own else groups
    for i in range(2):
        x.need["joined", i] = 4 * groups
    for i in range(SLOTS):
        x.need["unit", i], x.need["unit taken", i] = 1, groups + 4 * groups
    steps = units + [(-1, 0)]

    def loader():
        filled, begun = [0] * groups, [0] * groups
        for u, (tiles, n) in enumerate(steps):
            if u >= SLOTS:
                yield W(("unit taken", u % SLOTS), u // SLOTS - 1)
            arrive(("unit", u % SLOTS))
            if tiles < 0:
                return
            for g in range(n if own else 1):
                if tiles > 0:
                    if begun[g]:
                        yield W(("q empty", g), begun[g] - 1)
                    arrive(("q full", g))
                    begun[g] += 1
            for t in range(tiles):
                to = 0 if own else t % groups
                stage, turn = to * (0 if own else part) + filled[to] % part, filled[to] // part
                filled[to] += 1
                for operand in "kv":
                    if turn:
                        yield W((operand + " empty", stage), turn - 1)
                    arrive((operand + " full", stage))

    def products(g):
        step, begin, queries, ring = (1, 0, g, 0) if own else (groups, g, 0, g * part)
        ks = vs = turns = seen = results = 0
        ahead = False

        def keys():
            return W(("k full", ring + ks % part), ks // part)

        def scores(last):
            nonlocal ks
            arrive(("s full", g))
            arrive(("k empty", ring + ks % part))
            ks += 1
            if last:
                arrive(("q empty", queries))
        for u, (tiles, n) in enumerate(steps):
            yield W(("unit", u % SLOTS), u // SLOTS)
            arrive(("unit taken", u % SLOTS))
            if tiles < 0:
                return
            if own and g >= n:
                for _ in range(tiles):
                    yield keys()
                    arrive(("k empty", ring + ks % part))
                    ks += 1
                    yield W(("v full", ring + vs % part), vs // part)
                    arrive(("v empty", ring + vs % part))
                    vs += 1
                continue
            if begin < tiles and not ahead:
                yield W(("q full", queries), seen)
                yield keys()
                scores(begin + step >= tiles)
            ahead = False
            if 0 < tiles <= begin:
                yield W(("q full", queries), seen)
                arrive(("q empty", queries))
            seen += tiles > 0
            for t in range(begin, tiles, step):
                if t + step < tiles:
                    yield keys()
                    yield W(("s free", g), turns)
                    scores(t + 2 * step >= tiles)
                elif u + 1 < len(steps) and W(("unit", (u + 1) % SLOTS), (u + 1) // SLOTS)():  # a look, not a wait
                    more, n_more = steps[u + 1]
                    if begin < more and (not own or g < n_more) and W(("q full", queries), seen)() and keys()():
                        yield W(("s free", g), turns)
                        scores(begin + step >= more)
                        ahead = True
                yield W(("v full", ring + vs % part), vs // part)
                if t == begin and results:
                    yield W(("o free", g), results - 1)
                yield W(("p full", g), turns)
                arrive(("o full", g))
                arrive(("v empty", ring + vs % part))
                vs += 1
                turns += 1
            results += begin < tiles

    def softmax(g):
        step, begin = (1, 0) if own else (groups, g)
        turns = shared = 0
        for u, (tiles, n) in enumerate(steps):
            yield W(("unit", u % SLOTS), u // SLOTS)
            arrive(("unit taken", u % SLOTS))
            if tiles < 0:
                return
            if own and g >= n:
                continue
            for t in range(begin, tiles, step):
                yield W(("s full", g), turns)
                arrive(("s free", g))
                if t > begin:
                    yield W(("o full", g), turns - 1)
                arrive(("p full", g))
                turns += 1
            if begin < tiles:
                yield W(("o full", g), turns - 1)
            if not own:
                for i in range(2):
                    arrive(("joined", i))
                    yield W(("joined", i), shared)
                shared += 1
            if begin < tiles:
                arrive(("o free", g))
    return x.run([loader()] + [products(g) for g in range(groups)] + [softmax(g) for g in range(groups) for _ in range(4)])


def backward(groups, stages, buffers, units, sums, seed):
    """units: tiles of a block's units; sums: the groups' row sums go to the results (dQ)"""
    x = Block(seed)
    W, arrive = x.over, x.arrive
    for i in range(stages):
        x.need["full", i] = x.need["empty", i] = 1
    for i in range(buffers):
        x.need["a full", i], x.need["a empty", i] = 1, groups
    for g in range(groups):
        for b in ("s full", "dp full", "p added", "ds added"):
            x.need[b, g] = 1
        x.need["p full", g] = x.need["ds full", g] = 4  # warps
    x.need["done"], x.need["free"] = 1, 4
    for i in range(2):
        x.need["sum full", i], x.need["sum empty", i] = 4 * groups, 4
    for i in range(SLOTS):
        x.need["unit", i], x.need["unit taken", i] = 1, groups + 4 * groups + 4
    steps = units + [-1]

    def take(u):
        yield W(("unit", u % SLOTS), u // SLOTS)
        arrive(("unit taken", u % SLOTS))

    def loader():
        item = n = 0
        for u, tiles in enumerate(steps):
            if u >= SLOTS:
                yield W(("unit taken", u % SLOTS), u // SLOTS - 1)
            arrive(("unit", u % SLOTS))
            if tiles > 0:
                if item >= buffers:
                    yield W(("a empty", item % buffers), item // buffers - 1)
                arrive(("a full", item % buffers))
                item += 1
            for _ in range(tiles):
                if n >= stages:
                    yield W(("empty", n % stages), n // stages - 1)
                arrive(("full", n % stages))
                n += 1

    def products(g):
        before = (g - 1) % groups
        s = dict(index=0, item=-1, seen=-1, t=g, n=g, more=True, tiles=0, have=False)

        def standing():
            if s["seen"] != s["item"]:
                yield W(("a full", s["item"] % buffers), s["item"] // buffers)
            s["seen"] = s["item"]

        def find(most):
            s["have"] = False
            while s["more"] and s["t"] >= s["tiles"]:
                if most == 0:
                    return
                most -= 1
                if s["tiles"] > 0:
                    yield from standing()
                    arrive(("a empty", s["item"] % buffers))
                s["t"] -= s["tiles"]
                yield from take(s["index"])
                s["more"] = steps[s["index"]] >= 0
                s["tiles"] = max(steps[s["index"]], 0)
                s["index"] += 1
                s["item"] += s["tiles"] > 0
            s["have"] = s["more"]

        def scores():
            yield from standing()
            yield W(("full", s["n"] % stages), s["n"] // stages)
            arrive(("s full", g))
        mine, early = 0, False
        while True:
            if not s["have"] and s["more"]:
                yield from find(1 << 30)
            if not s["have"]:
                return
            if not early:
                yield from scores()
            arrive(("dp full", g))
            n, unit = s["n"], s["item"]
            first, last, follows = s["t"] == 0, s["t"] == s["tiles"] - 1, g > 0 or mine > 0
            turns = mine if g > 0 else mine - 1
            s["t"] += groups
            s["n"] += groups
            yield W(("p full", g), mine)
            if follows:
                yield W(("p added", before), turns)
            if first and unit > 0:
                yield W("free", unit - 1)
            arrive(("p added", g))
            yield from find(1)
            early = s["have"] and (s["seen"] == s["item"] or W(("a full", s["item"] % buffers), s["item"] // buffers)()) and W(("full", s["n"] % stages), s["n"] // stages)()
            if early:
                yield from scores()
            yield W(("ds full", g), mine)
            if follows:
                yield W(("ds added", before), turns)
            arrive(("ds added", g))
            arrive(("empty", n % stages))
            if last:
                arrive("done")
            mine += 1

    def weights(g):
        turn = item = mine = 0
        for u, tiles in enumerate(steps):
            yield from take(u)
            if tiles < 0:
                return
            for _ in range((g - turn) % groups, tiles, groups):
                yield W(("s full", g), mine)
                arrive(("p full", g))
                yield W(("dp full", g), mine)
                arrive(("ds full", g))
                mine += 1
            turn = (turn + tiles) % groups
            if sums and tiles > 0:
                if item >= 2:
                    yield W(("sum empty", item & 1), item // 2 - 1)
                arrive(("sum full", item & 1))
            item += tiles > 0

    def results():
        item = 0
        for u, tiles in enumerate(steps):
            yield from take(u)
            if tiles < 0:
                return
            if tiles == 0:
                continue
            yield W("done", item)
            if sums:
                yield W(("sum full", item & 1), item // 2)
                arrive(("sum empty", item & 1))
            arrive("free")
            item += 1
    return x.run([loader()] + [products(g) for g in range(groups)] + [weights(g) for g in range(groups) for _ in range(4)] + [results() for _ in range(4)])


@pytest.mark.parametrize("own", [True, False])
@pytest.mark.parametrize("width", [64, 128])
def test_forward(width, own):
    """units without tiles, fewer tiles than groups, groups without a unit, the next unit's scores ahead"""
    text, r = source("train_attn.cu"), random.Random(width + own)
    groups, part = constant(text, "GROUPS", width), constant(text, "OWN_STAGES" if own else "PART", width)
    for seed in range(150):
        units = [(r.choice([0, 1, 1, 2, 3, 5, 8, 17]), r.choice([groups, groups, r.randint(1, groups)])) for _ in range(r.randint(1, 12))]
        assert forward(groups, part, units, own, seed), units


@pytest.mark.parametrize("sums", [True, False])
@pytest.mark.parametrize("width", [64, 128])
def test_backward(width, sums):
    text, r = source("train_attn_bwd.cu"), random.Random(width + sums)
    groups, stages, buffers = (constant(text, n, width) for n in ("GROUPS", "STAGES", "UNITS"))
    for seed in range(120):
        units = [r.choice([0, 1, 1, 2, 3, 5, 8, 17]) for _ in range(r.randint(1, 12))]
        assert backward(groups, stages, buffers, units, sums, seed), units


def test_the_model_sees_a_ring_without_an_owner():
    """one ring shared by groups that take turns: whoever waits for a stage has not seen its last phase"""
    def shared(part):
        x = Block(3)
        for i in range(part):
            x.need["full", i] = x.need["empty", i] = 1

        def loader():
            for t in range(40):
                if t >= part:
                    yield x.over(("empty", t % part), t // part - 1)
                x.arrive(("full", t % part))

        def reader(g):
            phase = 0  # of this reader's own: it takes every second tile, but a stage comes to it every third time
            for t in range(g, 40, 2):
                yield x.over(("full", t % part), phase // part)
                x.arrive(("empty", t % part))
                phase += 1
        return x.run([loader(), reader(0), reader(1)])
    try:
        assert not shared(3)
    except AssertionError as e:
        assert "parity" in str(e)


@pytest.mark.parametrize("name", ["train_attn.cu", "train_attn_bwd.cu"])
def test_waits_have_a_limit(name):
    """between the roles there are barriers in shared memory, whose waits run out, and no others: a warp whose wait has run out may have left. A
    block ends behind a barrier that all of its threads reach, and only once what it has issued has landed"""
    text = re.sub(r"//[^\n]*", "", source(name) + source("train_attn.cuh"))
    kernel = text[text.index("__global__ void __launch_bounds__"):]
    kernel = kernel[:kernel.index("tmem_dealloc")]
    assert "bar.sync" not in text and "bar.arrive" not in text and "barrier.sync" not in text and "named_barrier" not in text and "cooperative_groups" not in text
    assert kernel.count("__syncthreads()") == 1  # barriers are initialised
    assert kernel.count("__syncthreads_or(!ok)") == 1 and kernel.rindex("__syncthreads_or(!ok)") > kernel.rindex("wait")
