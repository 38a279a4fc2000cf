"""CPU: the order in which paged attention takes its items, as the kernel finds it (find_item of paged_attention_sm100.cu): every
item once, those with the most keys first."""
import random


def _find(x, ahead, count, tokens):
    """The x-th item of up to 32 sequences: (sequence, index), and its weight in units, by the kernel's arithmetic."""
    n = len(count)
    mine = [(c + tokens - 1) // tokens for c in count]
    keys = [a + c for a, c in zip(ahead, count)]
    most = max(2 * k if m else 0 for k, m in zip(keys, mine))
    assert most < 2 ** 32
    unit = max(1, most.bit_length() - 6)
    assert most < 64 << unit
    whole = [max(m - 1, 0) for m in mine]
    last = [(k if c - (m - 1) * tokens <= tokens // 2 else 2 * k) >> unit if m else -1 for k, c, m in zip(keys, count, mine)]

    def start(i, units):
        need = (units << (unit - 1)) - ahead[i] + tokens - 1
        assert abs(need) < 2 ** 31
        quotient = abs(need) // tokens * (1 if need >= 0 else -1)   # (as C divides; a shift would go below: both are clamped)
        return min(max(quotient - 1, 0), whole[i])

    def reach(i, units):
        return whole[i] - start(i, units) + (last[i] >= units)

    low, step = 0, 32
    while step:
        if sum(reach(i, low + step) for i in range(n)) > x:
            low += step
        step >>= 1
    rest = x - sum(whole[i] - start(i, low + 1) + (last[i] > low) for i in range(n))
    for i in range(n):
        here, with_last = start(i, low + 1), last[i] == low
        have = here - start(i, low) + with_last
        if rest < have:
            return (i, mine[i] - 1 if with_last and rest == 0 else here - 1 - rest + with_last), low, unit
        rest -= have
    raise AssertionError("no item")


def test_every_item_once_and_the_longest_first():
    rng = random.Random(4)
    for _ in range(300):
        n, tokens = rng.randint(1, 32), rng.choice([2, 8, 50, 64, 84, 256])
        ahead = [rng.choice([0, rng.randint(0, 300), rng.randint(0, 20000)]) for _ in range(n)]
        count = [rng.choice([0, 1, tokens // 2, tokens, tokens + 1, rng.randint(0, 3000)]) for _ in range(n)]
        want = {(b, i) for b, c in enumerate(count) for i in range(-(-c // tokens))}
        got = [_find(x, ahead, count, tokens) for x in range(len(want))]
        assert {g for g, _, _ in got} == want
        weights = [w for _, w, _ in got]
        assert weights == sorted(weights, reverse=True)
        for (b, i), w, unit in got:
            keys = ahead[b] + min(count[b], (i + 1) * tokens)
            whole = i + 1 < -(-count[b] // tokens) or count[b] - i * tokens > tokens // 2
            assert (2 * keys if whole else keys) >> unit == w


def test_longest_sequences():
    """Lengths up to the largest that the calls take."""
    most = 2 ** 30
    assert _find(0, [most - 5], [5], 64)[0] == (0, 0)
    assert sorted(_find(x, [most - 300, 0], [300, 300], 256)[0] for x in range(4)) == [(0, 0), (0, 1), (1, 0), (1, 1)]
