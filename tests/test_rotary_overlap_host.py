"""Which destinations the rotary launch takes: all whose values lie apart from one another and from every source, whatever their strides, and no
others.  Addresses are counted one by one here.  (inv_freq is misaligned throughout, so that a layout that is taken ends in that refusal.)"""
import ctypes as C
import random

import pytest

import __graft_entry__ as entry
from quartet_b200 import _lib

TAKEN, REFUSED = -3, -4


@pytest.fixture(scope="module")
def lib():
    entry.build()
    return _lib.load()


def call(lib, batch, tokens, d, segs, f32=True):
    """segs: (src element, src strides, dst element, dst strides, heads)"""
    base, eb, n = 1 << 20, 4 if f32 else 2, len(segs)
    arr = lambda v: (C.c_void_p * n)(*[base + eb * x for x in v])  # noqa: E731
    strides = [x for s in segs for x in (*s[1], *s[3])]
    return lib.quartet_rotary(n, arr([s[0] for s in segs]), arr([s[2] for s in segs]), (C.c_int64 * (6 * n))(*strides), (C.c_int32 * n)(*[s[4] for s in segs]),
                              (C.c_int32 * n)(*[1] * n), 1 if f32 else 0, batch, tokens, d, 2, 1, None, 1, 0, 0, 0, C.c_void_p(base + 4), 1.0, 0, None)


def cells(at, st, batch, tokens, heads, d):
    return [at + b * st[0] + t * st[1] + h * st[2] + k for b in range(batch) for t in range(tokens) for h in range(heads) for k in range(d)]


def expected(batch, tokens, d, segs):
    src = [cells(s[0], s[1], batch, tokens, s[4], d) for s in segs]
    dst = [cells(s[2], s[3], batch, tokens, s[4], d) for s in segs]
    for g, x in enumerate(dst):
        if len(set(x)) != len(x):
            return REFUSED
        for h in range(len(segs)):
            if h != g and set(x) & set(dst[h]):
                return REFUSED
            if not (h == g and x == src[g]) and set(x) & set(src[h]):
                return REFUSED
    return TAKEN


def nested(rng, extents):
    """Strides of a buffer that holds the axes in some order, with gaps."""
    step, st = 1, [0] * 4
    for i in [3] + rng.sample(range(3), 3):
        st[i] = step
        step *= extents[i] + rng.choice([0, 0, 1, 3])
    return st[:3], step


@pytest.mark.parametrize("seed", range(400))
def test_every_layout_is_judged_by_its_addresses(lib, seed):
    rng = random.Random(seed)
    batch, tokens, d = rng.choice([1, 2, 3]), rng.choice([1, 2, 4]), rng.choice([2, 3, 4])
    segs = []
    for _ in range(rng.choice([1, 2, 3])):
        heads = rng.choice([1, 2, 3])
        seg = []
        for _ in "sd":
            kind = rng.random()
            if kind < 0.7:
                st, size = nested(rng, (batch, tokens, heads, d))
            else:
                st, size = [rng.choice([-7, -2, 0, 1, 2, 3, 4, 5, 8, 12, 13, 24]) for _ in range(3)], 40
            seg += [500 + rng.choice([0, 0, 1, 2, d, size // 2, size, 2 * size, 300]), st]
        if rng.random() < 0.3:
            seg[2:] = seg[:2]                                  # in place
        segs.append((*seg, heads))
    assert call(lib, batch, tokens, d, segs) == expected(batch, tokens, d, segs)


def test_the_layouts_in_use_are_taken(lib):
    """Heads split from a packed projection, joined into one, turned in place, in long batches."""
    for b, t, hq, hk, d in ((64, 512, 5, 5, 128), (3, 1021, 8, 2, 64), (1, 1, 1, 1, 2), (2, 32768, 32, 8, 128), (1 << 15, 1, 4, 1, 64)):
        w, far = (hq + 2 * hk) * d, 1 << 40
        packed, at, q = (t * w, w, d), 0, []
        for h in (hq, hk, hk):
            q.append((at, h))
            at += h * d
        for major in (True, False):
            out = lambda h: (h * t * d, d, t * d) if major else (t * h * d, h * d, d)  # noqa: E731
            split = [(o, packed, far * (i + 1), out(h), h) for i, (o, h) in enumerate(q)]
            join = [(far * (i + 1), out(h), o, packed, h) for i, (o, h) in enumerate(q)]
            for f32 in (True, False):
                assert call(lib, b, t, d, split, f32) == TAKEN and call(lib, b, t, d, join, f32) == TAKEN
        assert call(lib, b, t, d, [(o, packed, o, packed, h) for o, h in q]) == TAKEN
        if hq > 1:
            assert call(lib, b, t, d, [(q[0][0], packed, q[0][0] + d, packed, hq)]) == REFUSED
            assert call(lib, b, t, d, [(far, packed, 0, (t * w, w, 0), hq)]) == REFUSED
    assert b"one address" in lib.quartet_last_error_string()
