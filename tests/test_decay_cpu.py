"""CPU tests of the decaying-attention calls: what the C ABI and the Python binding refuse
before anything is launched, and the 64-bit form that the GPU tests compare with."""
import ctypes as C

import numpy as np
import pytest
import torch

import fufft_amd as ff
import layer_reference as R

INV, ALIGN, OK, UNSUP = ff.ERR_INVALID, ff.ERR_ALIGN, ff.OK, ff.ERR_UNSUPPORTED
P = [0x100000000 * (i + 1) for i in range(16)]          # addresses that are checked and never read
BATCH, TOKENS, HEADS, DK, DV = 2, 6, 3, 8, 16
STATE = 4 * BATCH * HEADS * DK * DV


def strides(dim, tokens=TOKENS, heads=HEADS):
    return (tokens * heads * dim, heads * dim, dim)


def by(s):
    return None if s is None else C.byref(ff._Strides(*s))


SK, SV = strides(DK), strides(DV)


def forward(q=P[0], sq=SK, k=P[1], sk=SK, v=P[2], sv=SV, type=0, decay=P[3], out=P[4], so=SV, state=P[5], new=P[6], lens=P[7],
            batch=BATCH, tokens=TOKENS, heads=HEADS, dk=DK, dv=DV, work=P[8], splits=4):
    return ff.lib.fufft_decay_attention(q, by(sq), k, by(sk), v, by(sv), type, decay, out, by(so), state, new, lens, 1.0, batch,
                                        tokens, heads, dk, dv, work, splits, None)


def test_forward_refusals():
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(decay=None), dict(sq=None), dict(so=None), dict(type=3),
                dict(batch=-1), dict(tokens=-1), dict(heads=-1), dict(dk=0), dict(dv=0), dict(dk=-1), dict(splits=-1), dict(work=None),
                dict(sq=(-1, 24, 8)), dict(so=(TOKENS * 48, 48, 0)), dict(so=(0, 48, 16)), dict(so=(TOKENS * 48, 48, 15)),
                dict(so=(TOKENS * 48, 40, 16)), dict(batch=1 << 40, tokens=1 << 40), dict(splits=1 << 40, batch=1 << 20),
                # outputs over inputs
                dict(out=P[2]), dict(out=P[0] + 8), dict(out=P[3] - 64), dict(out=P[5] - 64), dict(out=P[8] + 4), dict(new=P[0]), dict(new=P[3]),
                dict(new=P[5] + 4), dict(new=P[7]), dict(new=P[8]), dict(work=P[1]), dict(work=P[5]), dict(work=P[3])):
        assert forward(**bad) == INV, bad
    for bad in (dict(q=P[0] + 2), dict(k=P[1] + 1, type=1), dict(out=P[4] + 1), dict(decay=P[3] + 2), dict(state=P[5] + 1), dict(new=P[6] + 2),
                dict(lens=P[7] + 2), dict(work=P[8] + 1)):
        assert forward(**bad) == ALIGN, bad
    assert forward(dk=129, sq=strides(129), sk=strides(129)) == UNSUP
    assert forward(dv=129, sv=strides(129), so=strides(129)) == UNSUP
    for nothing in (dict(batch=0), dict(heads=0), dict(batch=0, q=None, sq=None)):
        assert forward(**nothing) == OK


def test_gradient_refusals():
    row = HEADS * (2 * DK + DV)         # dq, dk and dv of a token side by side

    def call(do=P[0], sdo=SV, q=P[1], k=P[2], v=P[3], sk=SK, sv=SV, type=0, decay=P[4], dq=P[5], dk_=P[6], dv_=P[7], sq2=SK, sk2=SK, sv2=SV,
             state=P[8], dnew=P[9], ds=P[10], lens=P[11], batch=BATCH, tokens=TOKENS, heads=HEADS, dk=DK, dv=DV, work=P[12], splits=4):
        return ff.lib.fufft_decay_attention_grad(do, by(sdo), q, by(sk), k, by(sk), v, by(sv), type, decay, dq, by(sq2), dk_, by(sk2), dv_, by(sv2),
                                                 state, dnew, ds, lens, 1.0, batch, tokens, heads, dk, dv, work, splits, None)
    for bad in (dict(do=None), dict(q=None), dict(dq=None), dict(dk_=None), dict(dv_=None), dict(decay=None), dict(type=9), dict(dk=0),
                dict(splits=-2), dict(work=None), dict(dq=P[1]), dict(dk_=P[5]), dict(dk_=P[5] + 4), dict(dv_=P[0]), dict(dv_=P[6] + 8), dict(ds=P[9]), dict(ds=P[8]),
                dict(ds=P[5] + 16), dict(work=P[7] - 4 * 8), dict(work=P[8]), dict(sq2=(144, 24, 0)),
                # parts of one row, where one reaches into the next
                dict(dq=P[5], dk_=P[5] + 4 * (HEADS * DK - 1), sq2=(TOKENS * row, row, DK), sk2=(TOKENS * row, row, DK))):
        assert call(**bad) == INV, bad
    for bad in (dict(dq=P[5] + 2), dict(ds=P[10] + 1), dict(work=P[12] + 2), dict(dnew=P[9] + 2)):
        assert call(**bad) == ALIGN, bad
    assert call(dk=200, dv=200, sdo=strides(200), sk=strides(200), sv=strides(200), sq2=strides(200), sk2=strides(200), sv2=strides(200)) == UNSUP
    # ... and where they do not: only the width, refused later, keeps it from a launch
    wide = HEADS * 3 * 130
    side = (TOKENS * wide, wide, 130)
    s = strides(130)
    kw = dict(dk=130, dv=130, sdo=s, sk=s, sv=s, sq2=side, sk2=side, sv2=side)
    assert call(dq=P[5], dk_=P[5] + 4 * HEADS * 130, dv_=P[5] + 8 * HEADS * 130, **kw) == UNSUP
    assert call(dq=P[5], dk_=P[5] + 8 * HEADS * 130, dv_=P[5] + 4 * HEADS * 130, **kw) == UNSUP
    assert call(dq=P[5], dk_=P[5] + 4 * HEADS * 130, dv_=P[5] + 8 * HEADS * 130 + 4, **kw) == INV      # wraps into the next token's dq
    # heads of two widths side by side, and one element into each other
    row = HEADS * (2 * 130 + 30)
    kw = dict(dk=130, dv=30, sdo=strides(30), sk=s, sv=strides(30), sq2=(TOKENS * row, row, 130), sk2=(TOKENS * row, row, 130),
              sv2=(TOKENS * row, row, 30))
    assert call(dq=P[5], dk_=P[5] + 4 * HEADS * 130, dv_=P[5] + 8 * HEADS * 130, **kw) == UNSUP
    assert call(dq=P[5], dk_=P[5] + 4 * HEADS * 130, dv_=P[5] + 8 * HEADS * 130 - 4, **kw) == INV
    assert call(dq=P[5], dk_=P[5] + 4 * HEADS * 130, dv_=P[5] + 8 * HEADS * 130 + 4, **kw) == INV
    # a step that is no whole part of the other's row
    assert call(dq=P[5], dk_=P[5] + 4 * HEADS * 130, dv_=P[5] + 8 * HEADS * 130, **{**kw, "sv2": (TOKENS * row, row - 1, 30)}) == INV
    assert call(batch=0) == OK


def test_apart_by_brute_force():
    """What a call takes of an input and an output in one array, against the sets of their elements.  (Heads of 129
    and more, which are refused last of all, so that nothing is launched.)"""
    rng = np.random.default_rng(7)
    taken = apart = 0
    for _ in range(1500):
        heads, tokens = int(rng.integers(1, 4)), int(rng.integers(1, 4))
        dk, dv = int(rng.integers(129, 132)), int(rng.integers(129, 132))
        sk = (0, int(rng.integers(0, 900)), dk + int(rng.integers(0, 150)))
        sv = (0, sk[1] if rng.random() < 0.8 else int(rng.integers(0, 900)), sk[2] if rng.random() < 0.5 else dv + int(rng.integers(0, 150)))
        at = int(rng.integers(0, 900))

        def places(s, d, off):
            return [off + t * s[1] + h * s[2] + i for t in range(tokens) for h in range(heads) for i in range(d)]
        q, o = places(sk, dk, 0), places(sv, dv, at)
        status = forward(sq=sk, sk=strides(dk, tokens, heads), sv=strides(dv, tokens, heads), so=sv, out=P[0] + 4 * at, batch=1, tokens=tokens,
                         heads=heads, dk=dk, dv=dv, splits=0, work=None)
        assert status in (INV, UNSUP)
        fine = len(set(o)) == len(o) and not set(q) & set(o)
        assert fine or status == INV, (heads, tokens, dk, dv, sk, sv, at)
        taken, apart = taken + (status == UNSUP), apart + fine
    assert apart > 200 and taken > 0.7 * apart, (taken, apart)


def test_step_refusals():
    def call(q=P[0], k=P[1], v=P[2], sk=(24, 0, 8), sv=(48, 0, 16), type=0, decay=P[3], out=P[4], so=(48, 0, 16), state=P[5], count=4, slots=P[6],
             batch=BATCH, heads=HEADS, dk=DK, dv=DV):
        return ff.lib.fufft_decay_attention_step(q, by(sk), k, by(sk), v, by(sv), type, decay, out, by(so), state, count, slots, 1.0, batch, heads, dk,
                                                 dv, None)
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(state=None), dict(decay=None), dict(type=4), dict(count=-1),
                dict(slots=None, count=1), dict(dk=0), dict(dv=-1), dict(out=P[2]), dict(out=P[5] + 64), dict(state=P[0]), dict(state=P[6]), dict(state=P[3]),
                dict(so=(48, 0, 8)), dict(so=(0, 0, 16)), dict(sk=None)):
        assert call(**bad) == INV, bad
    for bad in (dict(q=P[0] + 2), dict(out=P[4] + 2), dict(state=P[5] + 2), dict(slots=P[6] + 4), dict(decay=P[3] + 1)):
        assert call(**bad) == ALIGN, bad
    assert call(dk=129, sk=(3 * 129, 0, 129)) == UNSUP
    assert call(batch=0) == OK and call(heads=0) == OK


def test_binding_refusals():
    q = torch.zeros(2, 6, 3, 8)
    v = torch.zeros(2, 6, 3, 16)
    g = torch.zeros(3)
    s = torch.zeros(2, 3, 8, 16)
    f, d, st = ff.decay_attention, ff.decay_attention_grad, ff.decay_attention_step
    q1, v1 = q[:, 0].contiguous(), v[:, 0].contiguous()
    bad = [
        (TypeError, "q: expected a torch tensor", lambda: f(np.zeros((2, 6, 3, 8)), q, v, g, v)),
        (ValueError, "q: dtype", lambda: f(q.double(), q, v, g, v)),
        (ValueError, "k: dtype", lambda: f(q, q.half(), v, g, v)),
        (ValueError, "q: expected", lambda: f(q[0], q, v, g, v)),
        (ValueError, "k: expected", lambda: f(q, q[:, :5], v, g, v)),
        (ValueError, "v: expected", lambda: f(q, q, v[:1], g, v)),
        (ValueError, "out: expected", lambda: f(q, q, v, g, q)),
        (ValueError, "head are not contiguous", lambda: f(q.transpose(1, 3).contiguous().transpose(1, 3), q, v, g, v)),
        (ValueError, "log_decay: holds", lambda: f(q, q, v, g[:2], v)),
        (ValueError, "state: expected", lambda: f(q, q, v, g, v, state=s.transpose(2, 3).contiguous())),
        (ValueError, "state: tensor is not contiguous", lambda: f(q, q, v, g, v, state=torch.zeros(2, 3, 16, 8).transpose(2, 3))),
        (ValueError, "new_state: dtype", lambda: f(q, q, v, g, v, new_state=s.half())),
        (ValueError, "lens: holds", lambda: f(q, q, v, g, v, lens=torch.zeros(1, dtype=torch.int32))),
        (ValueError, "lens: dtype", lambda: f(q, q, v, g, v, lens=torch.zeros(2, dtype=torch.int64))),
        (ValueError, "work: dtype", lambda: f(q, q, v, g, v, work=torch.zeros(2, 768).half())),
        (ValueError, "not in GPU memory", lambda: f(q, q, v, g, v)),
        (ValueError, "dout: expected", lambda: d(q, q, q, v, g, q, q, v)),
        (ValueError, "dq: expected", lambda: d(v, q, q, v, g, v, q, v)),
        (ValueError, "dstate: holds", lambda: d(v, q, q, v, g, q, q, v, dstate=s[:1])),
        (ValueError, "not in GPU memory", lambda: d(v, q, q, v, g, q, q, v)),
        (ValueError, "q: expected", lambda: st(q, q1, v1, g, s, v1)),
        (ValueError, "state: expected", lambda: st(q1, q1, v1, g, s[:, :2], v1)),
        (ValueError, "state: 1 states", lambda: st(q1, q1, v1, g, s[:1], v1)),
        (ValueError, "slots: dtype", lambda: st(q1, q1, v1, g, s, v1, slots=torch.zeros(2, dtype=torch.int32))),
        (ValueError, "not in GPU memory", lambda: st(q1, q1, v1, g, s, v1)),
    ]
    for error, text, call in bad:
        with pytest.raises(error, match=text):
            call()


def test_reference():
    """The 64-bit recurrence against the sum that it stands for, forwards and from the back."""
    rng = np.random.default_rng(1)
    q, k, v, s = rng.standard_normal((9, 4)), rng.standard_normal((9, 4)), rng.standard_normal((9, 5)), rng.standard_normal((4, 5))
    g = -0.3
    out, new, mags, _ = R.mixed(q, k, v, g, s)
    for t in range(9):
        want = np.exp(g * (t + 1)) * q[t] @ s + sum(np.exp(g * (t - i)) * (q[t] @ k[i]) * v[i] for i in range(t + 1))
        assert np.allclose(out[t], want, rtol=1e-12) and np.all(mags[t] >= np.abs(want) - 1e-9)
    assert np.allclose(new, np.exp(9 * g) * s + sum(np.exp(g * (8 - i)) * np.outer(k[i], v[i]) for i in range(9)), rtol=1e-12)
    out, new, _, _ = R.mixed(q, k, v, g, s, late=1)
    assert np.allclose(out[2], np.exp(2 * g) * q[2] @ s + sum(np.exp(g * (2 - i)) * (q[2] @ k[i]) * v[i] for i in range(3)), rtol=1e-12)
    assert np.allclose(new, np.exp(9 * g) * s + sum(np.exp(g * (9 - i)) * np.outer(k[i], v[i]) for i in range(9)), rtol=1e-12)
    out, new, _, _ = R.mixed(q, k, v, float("-inf"), s)
    assert np.allclose(out, (q * k).sum(1)[:, None] * v) and np.allclose(new, np.outer(k[8], v[8]))
