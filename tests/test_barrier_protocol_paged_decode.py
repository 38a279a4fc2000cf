"""CPU: barrier model (tests/barrier_model.py) of a CTA of a decode step over a paged cache, dadgpt_b200/csrc/paged_decode.cu: one
producer warp, four or eight consumer warps with their rows of every tile, and results that go where the ring was."""
import random

import pytest

from tests.barrier_model import Aborted, Model, survives


class Decode(Model):
    def __init__(self, stages, warps, tiles, rng, abort=False):
        super().__init__(rng, abort)
        self.stages, self.warps, self.tiles = stages, warps, tiles
        self.need = {"empty": warps}

    def loads_of(self):
        for j in range(self.tiles):
            s = j % self.stages
            if j >= self.stages:
                yield ("wait", f"empty[{s}]", j // self.stages - 1)
            yield ("tma", f"full[{s}]", [(("tile", s, w), j) for w in range(self.warps)])

    def producer(self):
        yield from self.producing(self.loads_of())
        yield ("sync", "all", self.warps + 1)

    def reads(self, w):
        for j in range(self.tiles):
            s = j % self.stages
            yield ("wait", f"full[{s}]", j // self.stages)
            yield ("read", ("tile", s, w), j)
            if j + 1 == self.tiles:   # V of rows that are not there
                yield ("write", ("tile", s, w), j)
                yield ("read", ("tile", s, w), j)
            yield ("arrive", f"empty[{s}]")

    def consumer(self, w):
        yield ("sync", "consumers", self.warps)   # the rotation's table, then the queries
        yield ("sync", "consumers", self.warps)
        try:
            yield from self.reads(w)
        except Aborted:
            pass
        yield ("sync", "all", self.warps + 1)
        for s in range(self.stages):
            yield ("write", ("tile", s, w), "sums")
        yield ("sync", "joined", self.warps)
        for s in range(self.stages):
            yield ("read", ("tile", s, (w + 1) % self.warps), "sums")

    def agents(self):
        return {"producer": self.producer(), **{f"consumer{w}": self.consumer(w) for w in range(self.warps)}}


SHAPES = [(3, 4), (2, 4), (6, 8), (3, 8)]   # stages and warps: head size 64, 128, and of CTAs with an SM to themselves


@pytest.mark.parametrize("abort", [False, True], ids=["runs", "gives_up"])
@pytest.mark.parametrize("stages,warps", SHAPES)
@pytest.mark.parametrize("tiles", [0, 1, 2, 3, 7, 20])
def test_every_schedule(stages, warps, tiles, abort):
    assert survives(lambda s: Decode(stages, warps, tiles, random.Random(s), abort), range(40)) is None


@pytest.mark.parametrize("role,gone", [("loads_of", "empty"), ("reads", "full")])
def test_the_model_misses_no_wait_that_is_left_out(role, gone):
    class Faulty(Decode):
        pass

    def faulty(self, *args):
        for op in getattr(Decode, role)(self, *args):
            if not (op[0] == "wait" and op[1].split("[")[0] == gone):
                yield op
    setattr(Faulty, role, faulty)
    assert all(survives(lambda s: Faulty(stages, warps, 20, random.Random(s)), range(100)) for stages, warps in SHAPES)
