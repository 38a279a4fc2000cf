"""CPU: barrier model (tests/barrier_model.py) of the decode kernel over lists of tiles, dadgpt_b200/csrc/decode_window.cu: the
producer with its ring of tiles, whose stages have a second arrival (of the copies of an 8-bit tile's scales), and of items, and
two of the consumer warps, with the barriers behind which a full tail becomes a block and, in a cluster, those that it meets at."""
import random

import pytest

from tests.barrier_model import Aborted, Model, survives

WARPS = (0, 1)


class DecodeWindow(Model):
    """Items are (number of tiles, whether the token completes a block); an item may have no tile (its only row comes with the
    token). `agreed`: the warps agree on `ok` ahead of the barriers that an item in order has and others do not; without it
    they agree behind the item only."""
    STAGES, RING = 3, 2
    need = {"full": 2, "empty": 2, "item_free": 2}

    def __init__(self, items, rng, cluster=False, agreed=True, abort=False):
        super().__init__(rng, abort)
        self.items, self.cluster, self.agreed = items, cluster, agreed

    def meet(self, name):
        """A barrier of the cluster, here of this CTA's warps."""
        if self.cluster:
            yield ("sync", name, len(WARPS) + 1)

    def producer(self):
        g = 0
        for n, (tiles, _) in enumerate(self.items):
            for _ in range(tiles):
                s, lap = g % self.STAGES, g // self.STAGES
                if lap > 0:
                    yield ("wait", f"empty[{s}]", lap - 1)
                yield ("tma", f"full[{s}]", [(("rows", s), g)])
                yield ("tma", f"full[{s}]", [(("scales", s), g)])
                g += 1
            if n >= self.RING:
                yield ("wait", f"item_free[{n % self.RING}]", n // self.RING - 1)
            yield ("write", ("item", n % self.RING), n + 1)
            yield ("arrive", f"item_ready[{n % self.RING}]")

    def settled(self):
        """As Model.producing, with two loads to a completion; then the cluster's barriers."""
        try:
            yield from self.producer()
        except Aborted:
            pass
        for bar, n in sorted(self.loads.items()):
            yield ("settle", bar, n // 2 - 1)
        yield from self.meet("handed over")

    def consumer(self, w):
        ok, g, n, have = True, 0, 0, True
        while have:
            tiles, completes = self.items[n]
            for _ in range(tiles):
                if ok:
                    try:
                        yield ("wait", f"full[{g % self.STAGES}]", g // self.STAGES)
                        yield ("read", ("rows", g % self.STAGES), g)
                        yield ("read", ("scales", g % self.STAGES), g)
                        yield ("arrive", f"empty[{g % self.STAGES}]")
                    except Aborted:
                        ok = False
                g += 1
            have = False
            if ok and not self.cluster:
                try:
                    yield ("wait", f"item_ready[{n % self.RING}]", n // self.RING)
                    yield ("read", ("item", n % self.RING), n + 1)
                    yield ("arrive", f"item_free[{n % self.RING}]")
                    have = n + 1 < len(self.items)
                except Aborted:
                    ok = False
            yield ("write", ("acc", w), n)
            if self.agreed:
                ok = not (yield ("any", "merge", 2, not ok))
            else:
                yield ("sync", "merge", 2)
            for v in WARPS:
                yield ("read", ("acc", v), n)
            if completes and ok:
                for side in range(2):
                    yield ("sync", "block", 2)   # what was in the four words is read
                    yield ("write", ("most", w), (n, side))
                    yield ("sync", "block", 2)
                    for v in WARPS:
                        yield ("read", ("most", v), (n, side))
            if not self.cluster:
                if self.agreed:
                    yield ("sync", "block", 2)   # (the same barrier)
                    have = have and ok
                elif (yield ("any", "merged", 2, not ok)):
                    have = False
            n += 1
        yield from self.meet("handed over")

    def agents(self):
        return {"producer": self.settled(), **{f"consumer{w}": self.consumer(w) for w in WARPS}}


ITEMS = [[(9, True), (3, False), (0, True), (1, True)], [(0, True)] * 4, [(1, False), (1, True), (1, True), (1, False)],
         [(5, True)], [(2, True), (7, True), (2, False)]]


@pytest.mark.parametrize("abort", [False, True], ids=["runs", "gives_up"])
@pytest.mark.parametrize("cluster", [False, True], ids=["", "cluster"])
def test_every_schedule_ends(cluster, abort):
    for items in ITEMS:
        items = items[:1] if cluster else items   # (a CTA of a cluster has one)
        assert survives(lambda s: DecodeWindow(items, random.Random(s), cluster, abort=abort), range(150)) is None, items


@pytest.mark.parametrize("cluster", [False, True], ids=["", "cluster"])
def test_warps_have_to_agree_ahead_of_the_block(cluster):
    items = [(9, True)] if cluster else [(2, True)] * 4
    found = survives(lambda s: DecodeWindow(items, random.Random(s), cluster, agreed=False, abort=True), range(1000))
    assert found is not None and "stuck" in found[1]
