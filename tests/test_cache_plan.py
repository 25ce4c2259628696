"""How the narrow tiles of ncmb_cache_attention and ncmb_block_attention deal units to CTAs (csrc/cache_mma.cuh, "how the chunks of all units are dealt"),
the same arithmetic on the CPU: every chunk of every unit is somebody's, partial results do not meet, and who joins finds them all."""
import random

import pytest

WARPS = START = 4


def span_of(chunks):
    return (chunks + WARPS - 1) // WARPS * WARPS + START


def run(chunks_of, units_an_item, ctas):
    """Deals the units out and checks; the most places that a CTA has, and the mean."""
    size = [span_of(n) * units_an_item for n in chunks_of]
    total = sum(size)
    per = ((total + ctas - 1) // ctas + WARPS - 1) // WARPS * WARPS
    parts, sums, contexts = {}, set(), set()
    for c in range(ctas):
        at, end = min(c * per, total), min(total, (c + 1) * per)
        item = item_at = 0
        while at < end and not item_at <= at < item_at + size[item]:
            item_at += size[item]
            item += 1
        while at < end:
            n = chunks_of[item]
            span = span_of(n)
            sub = (at - item_at) // span
            begin = item_at + sub * span
            take = min(begin + span, end) - at
            first, stop = max(0, at - begin - START), min(n, at + take - begin - START)
            unit = item * units_an_item + sub
            if stop > first:
                parts.setdefault(unit, []).append((c, first, stop, begin, n))
                assert c + unit not in sums                      # slots of maxima and sums: units + ctas
                sums.add(c + unit)
                if (first, stop) != (0, n):
                    assert 2 * c + (first == 0) not in contexts  # slots of contexts: 2 ctas
                    contexts.add(2 * c + (first == 0))
            at += take
            if at == item_at + size[item]:
                item_at, item = at, item + 1
    assert len(parts) == len(chunks_of) * units_an_item and max(sums) < ctas + len(parts)
    for p in parts.values():
        begin, n = p[0][3], p[0][4]
        c0 = (begin + START) // per
        assert [x[0] for x in p] == list(range(c0, (begin + span_of(n) - 1) // per + 1))
        assert [x[1] for x in p] == [0] + [x[2] for x in p[:-1]] and p[-1][2] == n
        assert all((x[1] == 0) == (x[0] == c0) for x in p)
        assert n > WARPS or len(p) == 1                          # what one round does is not cut
    return per, total / ctas


@pytest.mark.parametrize("seed", range(300))
def test_random_rows(seed):
    rng = random.Random(seed)
    chunks = [rng.choice([1, 1, 2, 3, rng.randint(1, 12), rng.randint(1, 400)]) for _ in range(rng.randint(1, 30))]
    run(chunks, rng.choice([1, 2, 3, 8, 24]), rng.choice([1, 2, 5, 296, 444, rng.randint(1, 500)]))


def test_a_row_of_few_chunks_does_not_go_to_one_cta():
    """8 kv heads of 24 tokens of a row that has just been opened, beside long rows: 192 units of one chunk each."""
    per, mean = run([128] * 24 + [1] * 24 + [100] * 48, 8, 444)
    assert per <= 1.02 * mean + WARPS
    assert per // span_of(1) <= 30                               # 192 / 30: seven CTAs at least
