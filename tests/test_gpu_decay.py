"""GPU tests of fufft_decay_attention, _grad and _step against the 64-bit recurrence of
tests/layer_reference.py, with the bounds derived there."""
import numpy as np
import pytest

import layer_reference as R

pytestmark = pytest.mark.gpu

DECAYS = [0.0, -0.003, -0.1, -1.0, -20.0, float("-inf")]


def decays(heads, first=0):
    return np.array([DECAYS[(first + h) % len(DECAYS)] for h in range(heads)], dtype=np.float32)


def inputs(rng, dev, kind, batch, tokens, heads, *dims):
    out = []
    for d in dims:
        out += R.typed(rng.standard_normal((batch, tokens, heads, d)), kind, dev)
    return out


def to_dev(x, dev):
    import torch
    return None if x is None else torch.from_numpy(np.ascontiguousarray(x)).to(dev)


def states(rng, dev, *shape):
    x = rng.standard_normal(shape).astype(np.float32)
    return to_dev(x, dev), x.astype(np.float64)


def check_rows(got, want, err, lens, fill):
    """got within its bounds up to each length, and as it was behind it."""
    for b in range(got.shape[0]):
        n = got.shape[1] if lens is None else min(max(int(lens[b]), 0), got.shape[1])
        assert R.inside(got[b, :n], want[b, :n], err[b, :n])
        assert bool((got[b, n:] == fill).all())


SHAPES = [(1, 1), (8, 8), (16, 40), (33, 7), (64, 64), (72, 40), (128, 128), (128, 20), (100, 128), (65, 65), (64, 128)]


@pytest.mark.parametrize("dk,dv", SHAPES)
@pytest.mark.parametrize("kind", R.TYPES)
def test_attention(dev, rng, dk, dv, kind):
    import torch
    import fufft_amd as ff
    for tokens in (1, 2, 63, 64, 65, 300):
        batch, heads = 2, 3
        print(f"case decay_attention {tokens}x{dk}x{dv} {kind}", flush=True)
        q, q64, k, k64, v, v64 = inputs(rng, dev, kind, batch, tokens, heads, dk, dk, dv)
        g = decays(heads, tokens)
        state, s64 = states(rng, dev, batch, heads, dk, dv)
        scale = dk ** -0.5
        for st, st64, lens in ((None, None, None), (state, s64, None), (state, s64, np.array([tokens // 2, tokens], dtype=np.int32))):
            want, err, new, nerr = R.attention(q64, k64, v64, g, st64, lens, scale, kind)
            got_new = torch.empty(batch, heads, dk, dv, device=dev)
            out = torch.full_like(v, 5.0)
            ff.decay_attention(q, k, v, to_dev(g, dev), out, state=st, new_state=got_new, lens=to_dev(lens, dev), scale=scale)
            check_rows(out, want, err, lens, 5.0)
            assert R.inside(got_new, new, nerr)


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("splits", [0, 1, 2, 3, 7, 40])
def test_segments(dev, rng, kind, splits):
    """Tokens cut into segments: lengths that end in any of them, and states in the places of the results."""
    import torch
    import fufft_amd as ff
    batch, tokens, heads, dk, dv = 5, 1500, 2, 48, 72
    lens = np.array([1500, 0, 700, 1, 64 * 17], dtype=np.int32)
    q, q64, k, k64, v, v64 = inputs(rng, dev, kind, batch, tokens, heads, dk, dk, dv)
    g = np.array([-0.002, -0.7], dtype=np.float32)
    state, s64 = states(rng, dev, batch, heads, dk, dv)
    print(f"case decay segments {kind} {splits}", flush=True)
    work = None if splits == 0 else torch.full((splits, batch, heads, dk, dv), float("nan"), device=dev)
    want, err, new, nerr = R.attention(q64, k64, v64, g, s64, lens, 0.25, kind)
    out = torch.full_like(v, 5.0)
    ff.decay_attention(q, k, v, to_dev(g, dev), out, state=state, new_state=state, lens=to_dev(lens, dev), work=work, scale=0.25)
    check_rows(out, want, err, lens, 5.0)
    assert R.inside(state, new, nerr)
    # lengths outside 0 .. tokens are taken as its ends
    lens2 = np.array([1501, -3, 700, 1, 2 ** 31 - 1], dtype=np.int32)
    want, err, new, nerr = R.attention(q64, k64, v64, g, None, lens2, 0.25, kind)
    out.fill_(5.0)
    ff.decay_attention(q, k, v, to_dev(g, dev), out, new_state=state, lens=to_dev(lens2, dev), work=work, scale=0.25)
    check_rows(out, want, err, lens2, 5.0)
    assert R.inside(state, new, nerr)


def test_strides(dev, rng):
    """q, k and v as parts of one array, heads first, keys shared by all heads, odd starts."""
    import torch
    import fufft_amd as ff
    batch, tokens, heads, dk, dv = 2, 150, 4, 40, 40
    g = decays(heads, 1)
    for kind in R.TYPES:
        print(f"case decay strides {kind}", flush=True)
        packed, p64 = R.typed(rng.standard_normal((batch, tokens, 3, heads, dk)), kind, dev)
        want, err, _, _ = R.attention(p64[:, :, 0], p64[:, :, 1], p64[:, :, 2], g, None, None, 1.0, kind)
        out = torch.full((batch, heads, tokens, dv + 3), 5.0, dtype=packed.dtype, device=dev)
        view = out.transpose(1, 2)[..., 1:dv + 1]
        ff.decay_attention(packed[:, :, 0], packed[:, :, 1], packed[:, :, 2], to_dev(g, dev), view)
        assert R.inside(view, want, err)
        assert bool((out[..., 0] == 5).all()) and bool((out[..., dv + 1:] == 5).all())
        one, o64 = R.typed(rng.standard_normal((batch, tokens, 1, dk)), kind, dev)
        want, err, _, _ = R.attention(p64[:, :, 0], np.broadcast_to(o64, p64[:, :, 0].shape), p64[:, :, 2], g, None, None, 1.0, kind)
        ff.decay_attention(packed[:, :, 0], one.expand(batch, tokens, heads, dk), packed[:, :, 2], to_dev(g, dev), view)
        assert R.inside(view, want, err)


@pytest.mark.parametrize("dk,dv", [(1, 1), (16, 40), (33, 7), (64, 64), (128, 128), (128, 20), (100, 128)])
@pytest.mark.parametrize("kind", R.TYPES)
def test_grad(dev, rng, dk, dv, kind):
    import torch
    import fufft_amd as ff
    for tokens, splits in ((1, 0), (64, 0), (130, 0), (700, 3)):
        batch, heads = 2, 2
        print(f"case decay_grad {tokens}x{dk}x{dv} {kind}", flush=True)
        q, q64, k, k64, v, v64, do, do64 = inputs(rng, dev, kind, batch, tokens, heads, dk, dk, dv, dv)
        g = decays(heads, tokens + 1)
        state, s64 = states(rng, dev, batch, heads, dk, dv)
        dnew, dn64 = states(rng, dev, batch, heads, dk, dv)
        work = torch.full((splits, 3, batch, heads, dk, dv), float("nan"), device=dev) if splits else None
        for st, st64, dn, dn_64, lens in ((None, None, None, None, None), (state, s64, dnew, dn64, np.array([tokens, tokens // 3], dtype=np.int32)),
                                          (None, None, dnew, dn64, None)):
            wants = R.attention_grad(do64, q64, k64, v64, g, st64, dn_64, lens, 0.3, kind)
            gq, gk, gv = torch.full_like(q, 5.0), torch.full_like(k, 5.0), torch.full_like(v, 5.0)
            ds = torch.empty_like(state)
            ff.decay_attention_grad(do, q, k, v, to_dev(g, dev), gq, gk, gv, state=st, dnew_state=dn, dstate=ds, lens=to_dev(lens, dev),
                                    work=work, scale=0.3)
            for got, (want, err) in zip((gq, gk, gv), wants):
                check_rows(got, want, err, lens, 5.0)
            assert R.inside(ds, *wants[3])


def test_grad_packed_and_differences(dev, rng):
    """Gradients into parts of one array; against central differences of the recurrence."""
    import torch
    import fufft_amd as ff
    batch, tokens, heads, d = 1, 70, 2, 24
    q, q64, k, k64, v, v64, do, do64 = inputs(rng, dev, "f32", batch, tokens, heads, d, d, d, d)
    g = np.array([-0.05, -0.4], dtype=np.float32)
    state, s64 = states(rng, dev, batch, heads, d, d)
    dnew, dn64 = states(rng, dev, batch, heads, d, d)
    grads = torch.empty(batch, tokens, 3, heads, d, device=dev)
    ds = torch.empty_like(state)
    ff.decay_attention_grad(do, q, k, v, to_dev(g, dev), grads[:, :, 0], grads[:, :, 1], grads[:, :, 2], state=state, dnew_state=dnew,
                            dstate=ds, scale=0.5)

    def loss(q, k, v, s):
        o, _, n, _ = R.attention(q, k, v, g, s, None, 0.5, "f32")
        return (o * do64).sum() + (n * dn64).sum()
    base = [q64, k64, v64, s64]
    got = [grads[:, :, 0], grads[:, :, 1], grads[:, :, 2], ds]
    step = 2.0 ** -10
    # the sum is quadratic at most in each input alone, so central differences are exact but for 64-bit rounding
    for which, at in ((0, (0, 3, 1, 5)), (0, (0, 69, 0, 23)), (1, (0, 0, 0, 0)), (1, (0, 65, 1, 7)), (2, (0, 33, 0, 1)), (2, (0, 69, 1, 2)),
                      (3, (0, 1, 4, 9)), (3, (0, 0, 0, 23))):
        lo, hi = [x.copy() for x in base], [x.copy() for x in base]
        lo[which][at] -= step
        hi[which][at] += step
        diff = (loss(*hi) - loss(*lo)) / (2 * step)
        assert abs(diff - float(got[which][at])) < 1e-4 * max(1.0, abs(diff)), (which, at)


@pytest.mark.parametrize("kind", R.TYPES)
def test_later_tokens_do_not_matter(dev, rng, kind):
    """Infinities and NaN in keys, values and queries of a token leave every earlier token's result as it
    was, and so do those behind a length."""
    import torch
    import fufft_amd as ff
    batch, tokens, heads, dk, dv = 1, 200, 2, 32, 48
    g = to_dev(np.array([-0.01, 0.0], dtype=np.float32), dev)
    q, _, k, _, v, _ = inputs(rng, dev, kind, batch, tokens, heads, dk, dk, dv)
    clean = torch.empty_like(v)
    ff.decay_attention(q, k, v, g, clean)
    for at in (0, 5, 63, 64, 100, 199):
        for bad in (float("nan"), float("inf")):
            for which in range(3):
                x = [q.clone(), k.clone(), v.clone()]
                x[which][0, at, 1, 3] = bad
                out = torch.empty_like(v)
                ff.decay_attention(*x, g, out)
                assert torch.equal(out[:, :at], clean[:, :at]) and torch.equal(out[:, :, 0], clean[:, :, 0]), (at, bad, which)
                if which == 0:
                    assert not out[0, at, 1].isfinite().any() and torch.equal(out[:, at + 1:], clean[:, at + 1:])
                if which == 1:
                    assert not out[0, at:, 1].isfinite().any()
                if which == 2:
                    assert not out[0, at:, 1, 3].isfinite().any()
                    assert torch.equal(out[..., :3], clean[..., :3]) and torch.equal(out[..., 4:], clean[..., 4:])
    n = to_dev(np.array([130], dtype=np.int32), dev)
    x = [t.clone() for t in (q, k, v)]
    for t in x:
        t[:, 130:] = float("nan")
    out, new = torch.zeros_like(v), torch.empty(batch, heads, dk, dv, device=dev)
    ff.decay_attention(*x, g, out, lens=n)
    assert torch.equal(out[:, :130], clean[:, :130]) and not out[:, 130:].any()
    ff.decay_attention(q, k, v, g, clean, new_state=new)
    ff.decay_attention(*x, g, out, new_state=new, lens=n)
    assert torch.equal(out[:, :130], clean[:, :130]) and not out[:, 130:].any() and bool(new.isfinite().all())


@pytest.mark.parametrize("dk,dv", [(1, 1), (8, 4), (33, 7), (64, 64), (128, 128), (128, 33), (100, 127)])
@pytest.mark.parametrize("kind", R.TYPES)
def test_step(dev, rng, dk, dv, kind):
    import torch
    import fufft_amd as ff
    batch, heads = 5, 3
    print(f"case decay_step {dk}x{dv} {kind}", flush=True)
    q, q64, k, k64, v, v64 = inputs(rng, dev, kind, batch, 1, heads, dk, dk, dv)
    g = decays(heads, dk)
    for slots in (None, [3, -1, 0, 7, 6], [2, 9, 2, 0, 2]):
        state, s64 = states(rng, dev, 8, heads, dk, dv)
        out = torch.empty(batch, heads, dv, dtype=q.dtype, device=dev)
        di = None if slots is None else torch.tensor(slots, device=dev)
        want, err, new = np.zeros((batch, heads, dv)), np.zeros((batch, heads, dv)), s64.copy()
        nerr, seen = np.zeros_like(s64), set()
        for b in range(batch):
            at = b if slots is None else slots[b]
            if not 0 <= at < 8 or at in seen:
                continue
            seen.add(at)
            for h in range(heads):
                o, s, mo, ms = R.mixed(q64[b, :, h], k64[b, :, h], v64[b, :, h], g[h], s64[at, h])
                want[b, h], err[b, h], new[at, h] = 0.5 * o[0], 0.5 * mo[0] * (dk + 10) * R.EPS24, s
                nerr[at, h] = ms * 6 * R.EPS24          # the power, its product, the key's and the sum
        ff.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], to_dev(g, dev), state, out, slots=di, scale=0.5)
        assert R.inside(out, want, err)
        assert R.inside(state, new, nerr)
        untouched = [i for i in range(8) if i not in seen]
        assert np.array_equal(state[untouched].double().cpu().numpy(), s64[untouched])


@pytest.mark.parametrize("kind", R.TYPES)
def test_prompt_then_tokens(dev, rng, kind):
    """A prompt, then tokens one by one from its state: as the whole text at once."""
    import torch
    import fufft_amd as ff
    batch, tokens, heads, dk, dv = 3, 100, 2, 64, 48
    q, q64, k, k64, v, v64 = inputs(rng, dev, kind, batch, tokens, heads, dk, dk, dv)
    g = np.array([-0.02, -0.3], dtype=np.float32)
    dg = to_dev(g, dev)
    want, err, new, nerr = R.attention(q64, k64, v64, g, None, None, 0.125, kind)
    state, out = torch.empty(batch, heads, dk, dv, device=dev), torch.empty_like(v)
    lens = torch.tensor([90, 64, 91], dtype=torch.int32, device=dev)
    ff.decay_attention(q, k, v, dg, out, new_state=state, lens=lens, scale=0.125)
    for i in range(36):
        at = (lens.long() + i).clamp_max(tokens - 1)
        slots = torch.where(lens.long() + i < tokens, torch.arange(batch, device=dev), -1)
        pick = [x[torch.arange(batch, device=dev), at].contiguous() for x in (q, k, v)]
        o = torch.empty_like(pick[2])
        ff.decay_attention_step(*pick, dg, state, o, slots=slots, scale=0.125)
        for b in range(batch):
            if int(slots[b]) >= 0:
                out[b, int(at[b])] = o[b]
    # the step meets a state that the chunks left within nerr, and adds its own few roundings
    assert R.inside(out, want, err + 40 * R.EPS24 * np.abs(want) + 2.0 ** -16 * err.max())
    assert R.inside(state, new, nerr + 50 * R.EPS24 * np.abs(new) + 4 * nerr)


def test_empty(dev):
    import torch
    import fufft_amd as ff
    g = torch.zeros(3, device=dev)
    s = torch.randn(2, 3, 8, 8, device=dev)
    new = torch.empty_like(s)
    x = torch.empty(2, 0, 3, 8, device=dev)
    ff.decay_attention(x, x, x, g, torch.empty_like(x), state=s, new_state=new)
    assert torch.equal(new, s)
    ff.decay_attention(x, x, x, g, torch.empty_like(x), new_state=new)
    assert not new.any()
    ds = torch.empty_like(s)
    ff.decay_attention_grad(x, x, x, x, g, torch.empty_like(x), torch.empty_like(x), torch.empty_like(x), dnew_state=s, dstate=ds)
    assert torch.equal(ds, s)
    y = torch.empty(0, 4, 3, 8, device=dev)
    ff.decay_attention(y, y, y, g, torch.empty_like(y))
    z = torch.empty(0, 3, 8, device=dev)
    ff.decay_attention_step(z, z, z, g, s, torch.empty_like(z))
