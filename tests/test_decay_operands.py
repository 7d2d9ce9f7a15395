"""CPU tests of what the decaying-attention calls take of operands that lie in one array.  Heads of 129 and more
channels are refused last of all, as unsupported, so that nothing is launched here."""
import ctypes as C

import numpy as np

import fufft_amd as ff

INV, UNSUP = ff.ERR_INVALID, ff.ERR_UNSUPPORTED
P = [0x100000000 * (i + 1) for i in range(12)]          # addresses that are checked and never read
WIDE = 129


def by(s):
    return C.byref(ff._Strides(*s))


def strides(dim, tokens, heads):
    return (tokens * heads * dim, heads * dim, dim)


def forward(batch=1, tokens=2, heads=3, dk=WIDE, dv=WIDE, q=P[0], out=P[3], sq=None, so=None, decay=P[4], state=None, new=None, lens=None,
            work=None, splits=0):
    sk, sv = strides(dk, tokens, heads), strides(dv, tokens, heads)
    return ff.lib.fufft_decay_attention(q, by(sq or sk), P[1], by(sk), P[2], by(sv), 0, decay, out, by(so or sv), state, new, lens, 1.0,
                                        batch, tokens, heads, dk, dv, work, splits, None)


def test_only_the_state_may_be_the_new_state():
    """new_state may be state; nothing else may be there, whatever its address."""
    S = P[6]
    assert forward(state=S, new=S) == UNSUP
    assert forward(state=S, new=S, work=P[7], splits=2, lens=P[8]) == UNSUP
    for bad in (dict(work=S, splits=1), dict(work=S, splits=4), dict(lens=S), dict(decay=S), dict(lens=S, work=S, splits=1)):
        assert forward(state=S, new=S, **bad) == INV, bad
        assert forward(new=S, **bad) == INV, bad
    for bad in (dict(work=S, splits=1), dict(work=S, splits=2)):        # work is written
        assert forward(state=S, **bad) == INV, bad
        assert forward(state=S, new=P[7], **bad) == INV, bad
    assert forward(state=S, lens=S, decay=S) == UNSUP                   # inputs may share what they like
    assert forward(state=S, new=S + 4) == INV and forward(state=S, new=S - 4) == INV


def places(batch, tokens, heads, s, dim, off=0):
    at = off + s[0] * np.arange(batch)[:, None, None, None] + s[1] * np.arange(tokens)[:, None, None] + s[2] * np.arange(heads)[:, None]
    return (at + np.arange(dim)).ravel()


def shared(batch, tokens, heads, dk, dv, sq, so, at):
    """(whether q and out `at` elements behind it share an element, whether out's own are distinct)"""
    q, o = places(batch, tokens, heads, sq, dk), places(batch, tokens, heads, so, dv, at)
    return bool(np.intersect1d(q, o).size), len(np.unique(o)) == len(o)


def test_parts_longer_than_the_step_between_them():
    """Tokens 803 apart whose heads are 647 apart, in an array of tokens 647 and heads 803 apart: parts of one
    reach over the other's second next."""
    sq, so, at = (0, 803, 647), (0, 647, 803), 478
    assert shared(1, 2, 3, 131, 131, sq, so, at) == (True, True)
    assert forward(dk=131, dv=131, sq=sq, so=so, out=P[0] + 4 * at) == INV


def test_apart_with_axes_in_any_order():
    """What a call takes of an input and an output in one array, against the sets of their elements: strides in any order, the
    same for both arrays, swapped, or near each other."""
    rng = np.random.default_rng(11)
    taken = apart = 0
    for _ in range(12000):
        batch, tokens, heads = (int(n) for n in rng.integers(1, 5, 3))
        dk, dv = (int(n) for n in rng.integers(129, 133, 2))
        sq = [int(n) for n in rng.integers(0, 1000, 3)]
        if rng.random() < 0.4:                      # rows of parts, one inside the other
            inner = int(rng.integers(129, 300))
            middle = inner * 4 + int(rng.integers(0, 200))
            sq = [middle * 4 + int(rng.integers(0, 300)), middle, inner]
        so = list(sq)
        if rng.random() < 0.5:
            so = [so[i] for i in rng.permutation(3)]
        elif rng.random() < 0.5:
            so[int(rng.integers(0, 3))] += int(rng.integers(1, 200))
        if rng.random() < 0.3:
            sq = [sq[i] for i in rng.permutation(3)]
        at = int(rng.integers(-2500, 2500))
        status = forward(batch, tokens, heads, dk, dv, sq=tuple(sq), so=tuple(so), out=P[0] + 4 * at)
        assert status in (INV, UNSUP)
        both, distinct = shared(batch, tokens, heads, dk, dv, sq, so, at)
        assert status == INV or (distinct and not both), (batch, tokens, heads, dk, dv, sq, so, at)
        taken, apart = taken + (status == UNSUP), apart + (distinct and not both)
    assert apart > 1000 and taken > 0.5 * apart, (taken, apart)
