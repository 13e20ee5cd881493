"""CPU model of how ``ops/csrc/cache_q8_sm100.cu`` divides attention over an 8-bit cache: the sequence of
places (``ENTRY`` per head and sequence, then its 32-key units) is cut into equal runs, one per CTA; a
CTA's warps take tiles of their heads from it and write partial results; the merge finds them again by
arithmetic alone. Checked for random ragged batches: every unit of every head is taken exactly once, a
warp's partials have distinct numbers within the workspace, and the merge counts exactly those written."""

import random

import pytest

WARPS, ENTRY = 8, 2


class Runs:
    def __init__(self, total, most):
        self.n = min(most, total)
        self.base = total // self.n if self.n else 0
        self.rem = total - self.base * self.n

    def begin(self, r):
        return r * self.base + min(r, self.rem)

    def owner(self, i):
        longer = self.rem * (self.base + 1)
        return i // (self.base + 1) if i < longer else self.rem + (i - longer) // self.base


def side_by_side(u):
    return next(h for h in (8, 4, 2, 1) if u % h == 0)


def taken(lens, heads_groups, ut, sms):
    """{(b, head group): {unit: times}}, {(b, head group): [(run, key warp)]}, the highest partial number."""
    units = [-(-n // 32) for n in lens]
    cost = [n + ENTRY if n else 0 for n in units]
    heads = side_by_side(heads_groups)
    keys, per = WARPS // heads, heads_groups // heads
    runs = Runs(sum(cost) * per, sms)
    got, partials, seen = {}, {}, set()
    for run in range(runs.n):
        first, count = runs.begin(run), runs.begin(run + 1) - runs.begin(run)
        for warp in range(WARPS):
            my_head, my_key, turn = warp % heads, warp // heads, 0
            # locate
            i, b = first, 0
            while i >= cost[b] * per:
                i -= cost[b] * per
                b += 1
            n = cost[b]
            j, i = divmod(i, n)
            left = count - (min(n, i + count) - i)
            start, end = max(0, i - ENTRY), min(n, i + count) - ENTRY
            t = start + my_key * ut
            while True:
                done = False
                while t >= end:
                    if left == 0:
                        done = True
                        break
                    turn += max(0, -(-(end - start) // ut))
                    j += 1
                    if j == per:
                        j, b = 0, b + 1
                    while cost[b] == 0:
                        b += 1
                    n = min(cost[b], left)
                    left -= n
                    start, end = 0, n - ENTRY
                    t = (my_key - turn) % keys * ut
                if done:
                    break
                hg = j * heads + my_head
                for u in range(t, min(t + ut, end)):
                    d = got.setdefault((b, hg), {})
                    d[u] = d.get(u, 0) + 1
                key = (run, (my_key - turn) % keys)
                if key not in partials.setdefault((b, hg), []):
                    partials[b, hg].append(key)
                    number = (b * per + j + run) * WARPS + key[1] * heads + my_head
                    assert number not in seen
                    seen.add(number)
                t += keys * ut
    assert not seen or max(seen) < (len(lens) * per + sms) * WARPS
    return got, partials


def merged(lens, heads_groups, ut, sms, b, hg):
    units = [-(-n // 32) for n in lens]
    cost = [n + ENTRY if n else 0 for n in units]
    heads = side_by_side(heads_groups)
    keys, per = WARPS // heads, heads_groups // heads
    runs = Runs(sum(cost) * per, sms)
    f, n = sum(cost[:b]) * per + hg // heads * cost[b], cost[b]
    r0, out = runs.owner(f), []
    for i in range((runs.owner(f + n - 1) + 1 - r0) * keys):
        run = r0 + i // keys
        lo, hi = max(f, runs.begin(run)) - f, min(f + n, runs.begin(run + 1)) - f
        if max(0, lo - ENTRY) + i % keys * ut < hi - ENTRY:
            out.append((run, i % keys))
    return out


@pytest.mark.parametrize("seed", range(40))
def test_runs(seed):
    rng = random.Random(seed)
    B, hgs, ut, sms = rng.randint(1, 9), rng.choice([1, 2, 3, 4, 5, 8, 12, 16]), rng.choice([1, 2]), rng.choice([3, 13, 148])
    lens = [rng.choice([0, 1, 31, 32, 33, 64, rng.randint(1, 700), rng.randint(1, 3000)]) for _ in range(B)]
    got, partials = taken(lens, hgs, ut, sms)
    for b, n in enumerate(lens):
        for hg in range(hgs):
            units = -(-n // 32)
            assert got.get((b, hg), {}) == {u: 1 for u in range(units)}
            if units:
                assert merged(lens, hgs, ut, sms, b, hg) == sorted(partials[b, hg])


def test_constants_are_the_kernel_s():
    import os
    import re

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = open(os.path.join(root, "flextensor_b200", "ops", "csrc", "cache_q8_sm100.cu")).read()
    value = lambda name: int(re.search(rf"constexpr int {name} = (\d+);", text).group(1))  # noqa: E731
    assert (value("WARPS"), value("ENTRY"), value("UNIT")) == (WARPS, ENTRY, 32)
    assert re.search(r"units_of_tile\(int column_tiles\) \{ return column_tiles == 1 \? 2 : 1; \}", text)  # ut of test_runs


def scratch_bytes(B, Sq, Hq, Hk, sms):
    """What one launch may write: a partial result (128 dims, reference, sum) for each row of every warp of
    every piece, whose numbers stay below steps of heads + runs."""
    rows = Sq * (Hq // Hk)
    tiles = 2 if rows > 8 else 1
    units = Hk * -(-rows // (8 * tiles))
    return (B * units // side_by_side(units) + sms) * WARPS * 8 * tiles * 130 * 4


def test_launches_of_many_queries_stay_within_the_workspace():
    from flextensor_b200.ops import native

    if not native.available():
        pytest.skip("native extension not built")
    rng = random.Random(7)
    cases = [(64, 8024, 1, 1), (16, 1000, 64, 8), (32, 2048, 64, 8), (1, 1, 8, 1), (1, 100000, 7, 7), (256, 3, 96, 3)]
    for _ in range(300):
        Hk = rng.choice([1, 2, 3, 5, 7, 8])
        cases.append((rng.choice([1, 3, 16, 64, 200]), int(2 ** rng.uniform(0, 14)), Hk * rng.choice([1, 2, 5, 6, 8, 16]), Hk))
    split = 0
    for B, Sq, Hq, Hk in cases:
        for sms in (148, 132):
            queries, held = native.lib().decode_attention_q8_plan(B, Sq, Hq, Hk, sms)
            assert sum(queries) == Sq and min(queries) >= 1
            assert held == max(scratch_bytes(B, n, Hq, Hk, sms) for n in queries)
            assert held <= 256 << 20 or held == scratch_bytes(B, 1, Hq, Hk, sms)
            if scratch_bytes(B, Sq, Hq, Hk, sms) <= 256 << 20:
                assert queries == [Sq]
            split += len(queries) > 1
    assert split > 50
