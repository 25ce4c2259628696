"""How ncmb_rope and ncmb_paged_append share tokens, heads and angles among a CTA's threads (csrc/rope.cuh, "RopeShare"), and what a launch of ncmb_rope
asks for: the same arithmetic on the CPU."""
import os
import random
import re

import pytest

import helpers

THREADS = 256
LAUNCH = 48 * 1024                      # shared memory that a launch may have without an attribute, static arrays included


def source(name):
    return open(os.path.join(helpers.ROOT, "saphira-cncm_b200", "csrc", name)).read()


def cdiv(a, b):
    return -(-a // b)


def rope_vec(halves, dims, es):
    v = 16 // es
    while halves and dims // 2 % v:
        v >>= 1
    return v


def rope_items(halves, dims, hd, v):
    return dims // 2 // v + cdiv(hd - dims, 2 * v) if halves else cdiv(hd, 2 * v)


def rope_launch(halves, dims, hd, n_head, tokens, es, sms=148, in_place=False):
    """(tokens a CTA, bytes of dynamic shared memory, whether by k_rope_any) of a call of ncmb_rope"""
    hd = (dims + 7) & ~7 if in_place else hd
    v = 16 // es
    other = rope_vec(halves, dims, es) < v
    items = cdiv(hd, v) if other else rope_items(halves, dims, hd, v)
    held = (8 if other else 4) * (THREADS // items)
    heads = min(n_head, held) if other else n_head
    angles, staged, spare = ((dims // 2 + 7) & ~7) * 8, heads * items * 16 if other else 0, 16 if other else 0
    per = max(1, min(16 if other else 32, held // heads, (LAUNCH - 32 * 20 - spare) // (angles + staged), tokens // (4 * sms)))
    return per, per * (angles + staged) + spare, other


def append_per(halves, dims, hd, heads, tokens, es, sms=148):
    """tokens a CTA of a call of ncmb_paged_append; dims 0: no rotation; heads: query heads and twice the kv heads"""
    v = rope_vec(halves and dims > 0, dims, es)
    items = rope_items(halves and dims > 0, dims, hd, v)
    return max(1, min(32, (4 if v * es == 16 else 20) * THREADS // (heads * items), tokens // (4 * sms)))


def test_the_sources_say_the_same():
    rope, share, append = source("rope.cu"), source("rope.cuh"), source("paged_cache.cu")
    assert "RO_THREADS = 256, RO_TOKENS = 32, RO_BATCH = 4" in rope and "RO_SMEM = 48 * 1024 - RO_TOKENS * (8 + 8 + 4)" in rope
    assert "(RO_SMEM - spare) / (angles + staged), a.tokens / (4 * ctx().sm_count)" in rope and "smem = (size_t)a.per * (angles + staged) + spare" in rope
    assert len(re.findall(r"__shared__ int64_t xo\[RO_TOKENS\], yo\[RO_TOKENS\];\s+__shared__ int place\[RO_TOKENS\];", rope)) == 2
    assert "(uint32_t)cdiv(65536, d)" in share and "return (dims / 2 + 7) & ~7" in share
    assert "PA_THREADS = 256, PA_TOKENS = 32" in append and "rounds = V * sizeof(QE) == 16 ? 4 : 20" in append
    assert "{PA_TOKENS, rounds * PA_THREADS / per_token, a.tokens / (4 * ctx().sm_count)}" in append


@pytest.mark.parametrize("es", [2, 4])
@pytest.mark.parametrize("halves", [True, False])
def test_launches_ask_for_no_more_than_they_may_have(es, halves):
    """Any head and rotated dims, any number of heads, so many tokens that a CTA has as many as it takes."""
    for hd in range(8, 257, 8):
        for dims in range(2, hd + 1, 2):
            for heads in list(range(1, 40)) + [64, 65, 300]:
                for in_place in (False, True):
                    per, smem, _ = rope_launch(halves, dims, hd, heads, 10 ** 6, es, in_place=in_place)
                    assert per >= 1 and smem + 32 * 20 <= LAUNCH, (hd, dims, heads, per, smem)
    # the calls that asked for too much
    assert not halves or rope_launch(True, 250, 256, 4 if es == 2 else 2, 9472, es) == ((15, 15 * (1024 + 2048) + 16, True))


def walk(tid, items, heads, per):
    """(token, head, item) that a thread comes to, by additions and by multiplications that stand for divisions"""
    step, by = THREADS // items, lambda d: cdiv(65536, d)
    p = tid * by(items) >> 16
    u = tid - p * items
    tok = (p * (by(heads) if heads <= 256 else 0) >> 16) if p < step else 1 << 20
    h = p - tok * heads if p < step else 0
    while tok < per:
        yield tok, h, u
        tok += step // heads
        h += step % heads
        if h >= heads:
            h -= heads
            tok += 1


def angles(tid, pairs, per):
    t = tid * cdiv(65536, pairs) >> 16
    i = tid - t * pairs
    while t < per:
        yield t, i
        t += THREADS // pairs
        i += THREADS % pairs
        if i >= pairs:
            i -= pairs
            t += 1


def test_every_vector_and_every_angle_is_somebody_s_once():
    rng = random.Random(1)
    for _ in range(300):
        items, heads, per = rng.randint(1, 128), rng.choice([1, 2, 3, rng.randint(1, 60), rng.randint(200, 300)]), rng.randint(1, 32)
        seen = [x for tid in range(THREADS) for x in walk(tid, items, heads, per)]
        assert len(seen) == len(set(seen)) == per * heads * items and max(x[1] for x in seen) < heads and max(x[2] for x in seen) < items
    for pairs in range(1, 129):
        for per in (1, 2, 7, 32):
            seen = [x for tid in range(THREADS) for x in angles(tid, pairs, per)]
            assert len(seen) == len(set(seen)) == per * pairs and max(x[1] for x in seen) < pairs
