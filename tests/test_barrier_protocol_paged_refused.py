"""CPU: barrier model of how attention over a paged cache learns that a page is outside the pool
(dadgpt_b200/csrc/paged_attention_sm100.cu). The producer looks at a key tile's pages when it fetches them and notes in the item's
entry what it found: in one flag for the tiles that both query tiles of a pair see (or the groups of a single tile share), in
another for those that only the second sees. A softmax group may look at a flag only when every tile that the flag speaks for has
been looked at. Here a flag's cell holds how many of them have."""
import random

import pytest

from tests.barrier_model import survives
from tests.test_barrier_protocol_paged import KINDS, WORK, Paged

BOTH, SECOND = 0, 1


class Refused(Paged):
    def tiles(self, i, which):
        """How many tiles of item i the flag speaks for."""
        first = self.n_kv(i) if self.single(i) else self.n(i, 0)
        return first if which == BOTH else self.n_kv(i) - first

    def scheduler(self):
        i = loads = None
        for op in super().scheduler():
            if op[0] == "tma" and op[1].startswith("slot_full"):
                if loads % 2 == 0:   # K and V of a tile: its pages are looked at once, ahead of both
                    j = loads // 2
                    which = BOTH if j < self.tiles(i, BOTH) else SECOND
                    yield ("write", ("flag", i % self.RING, which), (i, j + 1 - (self.tiles(i, BOTH) if which else 0)))
                loads += 1
            yield op
            if op[0] == "write" and op[1][0] == "item":
                i, loads = op[2], 0
                for which in (BOTH, SECOND):
                    yield ("write", ("flag", i % self.RING, which), (i, 0))

    def look(self, i, x):
        """What group x reads: the second query tile sees the tiles of both flags."""
        for which in (BOTH, SECOND) if x or self.single(i) else (BOTH,):
            yield ("read", ("flag", i % self.RING, which), (i, self.tiles(i, which)))

    def when(self, i, op):
        """Whether the group looks behind this operation of item i: its own results, or the results of both groups."""
        return op[0] == "wait" and op[1].split("[")[0] == ("joined" if self.single(i) else "o_done")

    def softmax(self, x, a):
        i = None
        for op in super().softmax(x, a):
            yield op
            if op[0] == "read" and op[1][0] == "item":
                i = op[2]
            elif i is not None and self.when(i, op):
                yield from self.look(i, x)


@pytest.mark.parametrize("abort", [False, True], ids=["runs", "gives_up"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("items", WORK)
def test_flags_are_read_behind_every_look(items, kind, abort):
    assert survives(lambda s: Refused(items, kind, random.Random(s), abort), range(60)) is None


def fails(model):
    return any(survives(lambda s: model(items, kind, random.Random(s)), range(200)) for kind in KINDS for items in WORK)


def test_looking_ahead_of_the_other_group_is_too_early():
    """A group without steps of a shared tile waits for nothing ahead of `joined`."""
    class Early(Refused):
        def softmax(self, x, a):
            i = seen = None
            for op in Paged.softmax(self, x, a):
                if i is not None and not seen and op[0] in ("write", "arrive") and op[1] in (("s", x, 0, a), "joined") \
                        and self.single(i) and (op[1] == "joined" or op[2] == ("stats", i)):
                    seen = True   # (as the results are handed over)
                    yield from self.look(i, x)
                yield op
                if op[0] == "read" and op[1][0] == "item":
                    i, seen = op[2], False
                elif i is not None and not self.single(i) and self.when(i, op):
                    yield from self.look(i, x)
    assert fails(Early)


def test_one_flag_for_a_pair_is_too_early_for_its_first_tile():
    class One(Refused):
        def look(self, i, x):
            yield from Refused.look(self, i, 1)
    assert fails(One)
