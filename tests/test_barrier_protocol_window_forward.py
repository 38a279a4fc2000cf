"""CPU: barrier model (tests/barrier_model.py) of the windowed forward, dadgpt_b200/csrc/flash_window_fwd_sm100.cu, with
one score buffer (head size 64) and with two (128). A CTA has one item of n key tiles; a softmax warp is an agent with
its rows, which may see nothing of a tile."""
import random

import pytest

from tests.barrier_model import Model, survives

WARPS = range(4)


class Forward(Model):
    STAGES = 2
    need = {"p_full": len(WARPS)}

    def __init__(self, n, bufs, rng, abort=False):
        super().__init__(rng, abort)
        self.n, self.bufs = n, bufs

    def load(self, kind, j):
        return ("tma", f"{kind}_full[{j % self.STAGES}]", [((kind, j % self.STAGES), j)])

    def producer(self):
        yield ("tma", "q_full", [(("q", a), "Q") for a in WARPS])
        yield self.load("k", 0)   # (what the thread asks for ahead of the CTA's set-up)
        yield self.load("v", 0)
        for j in range(1, self.n):
            for kind in "kv":
                if j >= self.STAGES:
                    yield ("wait", f"{kind}_empty[{j % self.STAGES}]", j // self.STAGES - 1)
                yield self.load(kind, j)

    def product(self, i):   # O += P V
        s, b = i % self.STAGES, i % self.bufs
        yield ("wait", f"v_full[{s}]", i // self.STAGES)
        yield ("wait", f"p_full[{b}]", i // self.bufs)
        so_far = [(("o", a), i - 1) for a in WARPS] if i else []
        yield ("mma", [(("s", b, a), ("p", i)) for a in WARPS] + [(("v", s), i)] + so_far, [(("o", a), i) for a in WARPS])
        yield ("commit", f"v_empty[{s}]")
        yield ("commit", f"o_done[{i % 2}]")

    def issuer(self):
        yield ("wait", "q_full", 0)
        for j in range(self.n):
            s, b = j % self.STAGES, j % self.bufs
            if self.bufs == 1 and j:
                yield from self.product(j - 1)
            yield ("wait", f"k_full[{s}]", j // self.STAGES)
            yield ("mma", [(("q", a), "Q") for a in WARPS] + [(("k", s), j)], [(("s", b, a), ("s", j)) for a in WARPS])
            yield ("commit", f"k_empty[{s}]")
            yield ("commit", f"s_full[{b}]")
            if self.bufs == 2 and j:
                yield from self.product(j - 1)
        yield from self.product(self.n - 1)

    def softmax(self, a):
        for j in range(self.n):
            b = j % self.bufs
            yield ("wait", f"s_full[{b}]", j // self.bufs)
            if self.rng.random() < 0.7:   # rows that see something of the tile
                yield ("read", ("s", b, a), ("s", j))
                if j and self.rng.random() < 0.3:   # the rescale
                    yield ("wait", f"o_done[{(j - 1) % 2}]", (j - 1) // 2)
                    yield ("read", ("o", a), j - 1)
                    yield ("write", ("o", a), j - 1)
                yield ("read", ("s", b, a), ("s", j))   # (half of them a second time)
            yield ("write", ("s", b, a), ("p", j))
            yield ("arrive", f"p_full[{b}]")
        yield ("wait", f"o_done[{(self.n - 1) % 2}]", (self.n - 1) // 2)
        yield ("read", ("o", a), self.n - 1)
        yield ("write", ("q", a), "out")
        yield ("bulk", [(("q", a), "out")])
        yield ("bulk_wait", 0)

    def agents(self):
        return {"producer": self.producing(self.producer()), "issuer": self.issuing(self.issuer()),
                **{f"softmax{a}": self.softmax(a) for a in WARPS}}


TILES = (1, 2, 3, 4, 5, 9, 40)


@pytest.mark.parametrize("abort", [False, True], ids=["runs", "gives_up"])
@pytest.mark.parametrize("bufs", [1, 2])
@pytest.mark.parametrize("n", TILES)
def test_every_schedule(n, bufs, abort):
    assert survives(lambda s: Forward(n, bufs, random.Random(s), abort), range(120)) is None


@pytest.mark.parametrize("bufs", [1, 2])
@pytest.mark.parametrize("role,gone", [("producer", "k_empty"), ("producer", "v_empty"), ("issuer", "q_full"),
                                       ("issuer", "k_full"), ("issuer", "v_full"), ("issuer", "p_full"),
                                       ("softmax", "s_full"), ("softmax", "o_done")])
def test_the_model_misses_no_wait_that_is_left_out(role, gone, bufs):
    class Faulty(Forward):
        pass

    def faulty(self, *args):
        for op in getattr(Forward, role)(self, *args):
            if not (op[0] == "wait" and op[1].split("[")[0] == gone):
                yield op
    setattr(Faulty, role, faulty)
    assert any(survives(lambda s: Faulty(n, bufs, random.Random(s)), range(200)) for n in TILES)
