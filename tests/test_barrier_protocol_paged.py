"""CPU: barrier model (tests/barrier_model.py) of attention over a paged cache, dadgpt_b200/csrc/paged_attention_sm100.cu.
An item is a pair of query tiles with the key tiles that each of them sees, ("pair", a, b), or one tile whose keys the groups
share, ("one", n), taking its steps in turn. The key tiles are of one step and two parts (head size 128) or of two steps, the last
of which may be left out (head size 64; there a turn may be a tile's two steps, which is what CTAs of a cluster do). A softmax
group is two agents, each with its rows. The request for another block is a load whose answer names the item. The turns that the
groups' exponentials take bound nobody's progress and are not part of it."""
import random

import pytest

from tests.barrier_model import Aborted, Model, survives

HALVES = (0, 1)


KINDS = {"d128": (1, 2, 1), "d64": (2, 1, 1), "d64_tiles": (2, 1, 2)}   # steps of a key tile, parts of a step, steps of a turn


class Paged(Model):
    SLOTS, RING = 5, 4
    need = {"slot_empty": 2, "item_free": 7, "p_full": 2, "joined": 4, "parted": 6, "freed": 4}

    def __init__(self, items, kind, rng, abort=False):
        super().__init__(rng, abort)
        self.items = items
        self.per_tile, self.parts, self.turn = KINDS[kind]
        # of the last tile only a half is seen
        self.half = [[self.per_tile == 2 and rng.random() < 0.5 for _ in HALVES] for _ in items]

    # what Share says
    def single(self, i):
        return self.items[i][0] == "one"

    def n_kv(self, i):
        return self.items[i][-1]

    def n(self, i, x):
        return self.items[i][1] if self.single(i) else self.items[i][1 + x]

    def at(self, i, x, k):
        return (k // self.turn * 2 + x) * self.turn + k % self.turn if self.single(i) else k

    def steps(self, i, x):
        every = self.per_tile * self.n(i, x) - self.half[i][0 if self.single(i) else x]
        return sum(u // self.turn % 2 == x for u in range(every)) if self.single(i) else every

    def every(self, i):   # whether each step is its group's only one of the tile
        return self.single(i) and self.turn < self.per_tile

    def slot(self, tile, m):
        return (2 * tile + m) % self.SLOTS, (2 * tile + m) // self.SLOTS

    def items_of(self, own=lambda i: ()):
        for i in range(len(self.items) + 1):
            yield ("wait", f"item_ready[{i % self.RING}]", i // self.RING)
            yield ("read", ("item", i % self.RING), i)
            if i == len(self.items):
                return
            yield from own(i)
            yield ("arrive", f"item_free[{i % self.RING}]")

    def scheduler(self):
        at = 0
        for i in range(len(self.items) + 1):
            if i >= self.RING:
                yield ("wait", f"item_free[{i % self.RING}]", i // self.RING - 1)
            yield ("write", ("item", i % self.RING), i)
            yield ("arrive", f"item_ready[{i % self.RING}]")
            if i == len(self.items):
                return
            for j in range(self.n_kv(i)):
                if j + 1 == self.n_kv(i):
                    yield ("tma", "stolen", [("answer", i + 1)])
                for _ in range(2):
                    s, use = at % self.SLOTS, at // self.SLOTS
                    if use > 0:
                        yield ("wait", f"slot_empty[{s}]", use - 1)
                    yield ("tma", f"slot_full[{s}]", [(("kv", s), at)])
                    at += 1
            yield ("wait", "stolen", i)
            yield ("read", "answer", i + 1)

    def q_producer(self):
        n = [0, 0]

        def own(i):
            for x in HALVES:
                if self.steps(i, x):
                    if n[x] > 0:
                        yield ("wait", f"q_empty[{x}]", n[x] - 1)
                    yield ("tma", f"q_full[{x}]", [(("q", x), i)])
                    n[x] += 1
        yield from self.items_of(own)

    def issuer(self, x):
        g = u = joins = gone = 0

        def wait_slot(tile, m):
            return ("wait", "slot_full[%d]" % self.slot(tile, m)[0], self.slot(tile, m)[1])

        def skip(tile):
            for m in range(2):
                yield wait_slot(tile, m)
                yield ("arrive", "slot_empty[%d]" % self.slot(tile, m)[0])

        def held(tile, m):
            return ("kv", self.slot(tile, m)[0]), 2 * tile + m

        def own(i):
            nonlocal g, u, joins, gone
            steps = self.steps(i, x)

            def tile_of(k):
                return self.at(i, x, k) // self.per_tile

            def first_of(k):
                return self.every(i) or k % self.per_tile == 0

            def last_of(k):
                return self.every(i) or k % self.per_tile == self.per_tile - 1 or k + 1 == steps

            def scores(k):
                at = tile_of(k)
                if first_of(k):
                    yield wait_slot(gone + at, 0)
                yield ("mma", [(("q", x), i), held(gone + at, 0)],
                       [(("s", x, c, a), ("s", i, k)) for c in range(self.parts) for a in HALVES])
                if last_of(k):
                    yield ("commit", "slot_empty[%d]" % self.slot(gone + at, 0)[0])
                if k + 1 == steps:
                    yield ("commit", f"q_empty[{x}]")
                yield ("commit", f"s_full[{x}]")
                if self.single(i) and last_of(k) and at + 1 < (self.n_kv(i) if k + 1 == steps else tile_of(k + 1)):
                    yield from skip(gone + at + 1)

            if self.single(i) and (tile_of(0) if steps else self.n_kv(i)) > 0:
                yield from skip(gone)
            if steps:
                yield ("wait", f"q_full[{x}]", u)
                u += 1
                yield from scores(0)
            for k in range(steps):
                tile = gone + tile_of(k)
                if first_of(k):
                    yield wait_slot(tile, 1)
                for c in range(self.parts):
                    yield ("wait", f"p_full[{x}{c}]", g)
                    zeroed = [(("zero", x, a), tile) for a in HALVES] if tile == gone + self.n_kv(i) - 1 else []
                    so_far = [(("o", x), (i, k, c))] if k or c else []
                    yield ("mma", [(("s", x, c, a), ("p", i, k)) for a in HALVES] + [held(tile, 1)] + zeroed + so_far,
                           [(("o", x), (i, k, c + 1) if c + 1 < self.parts else (i, k + 1, 0))])
                if last_of(k):
                    yield ("commit", "slot_empty[%d]" % self.slot(tile, 1)[0])
                if k + 1 == steps:
                    yield ("commit", f"o_done[{x}]")
                else:
                    yield from scores(k + 1)
                g += 1
            if not self.single(i):
                for j in range(self.n(i, x), self.n_kv(i)):
                    yield from skip(gone + j)
            else:
                yield ("arrive", "parted")
                yield ("wait", "parted", joins)
                joins += 1
            gone += self.n_kv(i)
        yield from self.items_of(own)

    def softmax(self, x, a):
        g = u = joins = gone = 0
        shared = False

        def own(i):
            nonlocal g, u, joins, gone, shared
            steps = self.steps(i, x)

            if shared:
                yield ("wait", "freed", joins - 1)
                shared = False
            for k in range(steps):
                yield ("wait", f"s_full[{x}]", g)
                for c in range(self.parts):
                    yield ("read", ("s", x, c, a), ("s", i, k))
                if k > 0 and self.rng.random() < 0.3:   # the rescale
                    yield ("read", ("o", x), (i, k, 0))
                    yield ("write", ("o", x), (i, k, 0))
                tile = gone + self.at(i, x, k) // self.per_tile
                if (self.every(i) or k % self.per_tile == 0) and tile == gone + self.n_kv(i) - 1:   # V behind the sequence's end
                    s, use = self.slot(tile, 1)
                    yield ("wait", f"slot_full[{s}]", use)
                    yield ("read", ("kv", s), 2 * tile + 1)
                    yield ("write", ("zero", x, a), tile)
                for c in range(self.parts):
                    yield ("write", ("s", x, c, a), ("p", i, k))
                    yield ("arrive", f"p_full[{x}{c}]")
                g += 1
            if steps:
                yield ("wait", f"o_done[{x}]", u)
                u += 1
            if self.single(i):
                yield ("write", ("s", x, 0, a), ("stats", i))
                yield ("arrive", "joined")
                yield ("wait", "joined", joins)
                yield ("read", ("s", 1 - x, 0, a), ("stats", i))
                yield ("arrive", "parted")
            for y in HALVES if self.single(i) else (x,):
                if self.steps(i, y):
                    yield ("read", ("o", y), (i, self.steps(i, y), 0))
            if self.single(i):
                yield ("arrive", "freed")
                joins += 1
                shared = True
            gone += self.n_kv(i)
        yield from self.items_of(own)

    def loading(self, body, mine):
        """As Model.producing, with the loads of one of the two producers."""
        try:
            yield from body
        except Aborted:
            pass
        for bar, n in sorted(self.loads.items()):
            if bar.split("[")[0] in mine:
                yield ("settle", bar, n - 1)

    def agents(self):
        return {"scheduler": self.loading(self.scheduler(), ("slot_full", "stolen")),
                "q producer": self.loading(self.q_producer(), ("q_full",)),
                **{f"issuer{x}": self.issuing(self.issuer(x), f"settled[{x}]") for x in HALVES},
                **{f"softmax{x}{a}": self.softmax(x, a) for x in HALVES for a in HALVES}}


# pairs whose second tile sees no more, one or two more tiles; tiles shared by the groups, of one key tile and of several; in turn
WORK = ([("pair", 1, 1)], [("pair", 5, 6), ("pair", 3, 3), ("pair", 1, 3)], [("one", 1)] * 12, [("one", 2), ("one", 7), ("one", 4)],
        [("one", 3), ("pair", 2, 3), ("one", 1), ("one", 1), ("pair", 1, 2), ("one", 5)], [("pair", 1, 2), ("one", 1)] * 6,
        [("pair", 1, 1)] * 9)


@pytest.mark.parametrize("abort", [False, True], ids=["runs", "gives_up"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("items", WORK)
def test_every_schedule(items, kind, abort):
    assert survives(lambda s: Paged(items, kind, random.Random(s), abort), range(60)) is None


@pytest.mark.parametrize("role,gone", [("scheduler", "slot_empty"), ("scheduler", "stolen"),
                                       ("q_producer", "q_empty"), ("issuer", "q_full"), ("issuer", "p_full"), ("issuer", "slot_full"),
                                       ("issuer", "parted"), ("softmax", "s_full"), ("softmax", "o_done"), ("softmax", "joined"),
                                       ("softmax", "freed"), ("softmax", "slot_full")])
def test_the_model_misses_no_wait_that_is_left_out(role, gone):
    class Faulty(Paged):
        pass

    def faulty(self, *args):
        for op in getattr(Paged, role)(self, *args):
            if not (op[0] == "wait" and op[1].split("[")[0] == gone):
                yield op
    setattr(Faulty, role, faulty)
    assert any(survives(lambda s: Faulty(items, kind, random.Random(s)), range(200)) for kind in KINDS for items in WORK)
