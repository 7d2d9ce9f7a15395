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
