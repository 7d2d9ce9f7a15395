"""GPU tests of the norm, 8-bit and decaying-attention calls where one kernel gives way to the next, where tokens
are split with and without a state to return, and where operands pass 4 GiB.  References and bounds in
tests/layer_reference.py."""
import numpy as np
import pytest

import layer_reference as R

pytestmark = pytest.mark.gpu


def integers(dev, rows, k):
    import torch
    import fufft_amd as ff
    c = torch.zeros(rows, ff.i8_padded(k), dtype=torch.int8, device=dev)
    c[:, :k] = torch.randint(-127, 128, (rows, k), device=dev)
    return c, torch.rand(rows, device=dev) + 0.5


# rows of a: 1, 2, 4 and 8 of the four-byte products; to 16 and beyond by columns; K in parts of 1 KiB and of its wavefronts
@pytest.mark.parametrize("m", [1, 2, 3, 4, 6, 8, 9, 16, 17, 32, 33])
@pytest.mark.parametrize("n,k", [(1, 1023), (7, 1024), (4097, 1025), (8193, 300), (258, 8200), (63, 20000)])
def test_products_of_few_rows(dev, m, n, k):
    import torch
    import fufft_amd as ff
    print(f"case i8_matmul {m}x{n}x{k}", flush=True)
    a, sa = integers(dev, m, k)
    b, sb = integers(dev, n, k)
    out = torch.full((m, n + 3), 7.0, device=dev)
    ff.i8_matmul(a, sa, b, sb, out[:, :n], k)
    want, err = R.matmul(a.cpu().numpy(), sa.cpu().numpy(), b.cpu().numpy(), sb.cpu().numpy(), None, k)
    assert R.inside(out[:, :n], want, err)
    assert bool((out[:, n:] == 7).all())


def test_products_beyond_4gib(dev):
    """Rows of b, and results, that lie beyond 4 GiB: the sums are exact, so parts of them agree bit for bit."""
    import torch
    import fufft_amd as ff
    n, k = 140000, 32768
    b = torch.randint(-127, 128, (n, k), dtype=torch.int8, device=dev)
    sb = torch.rand(n, device=dev)
    for m in (1, 12, 20, 200):
        a, sa = integers(dev, m, k)
        out, tail = torch.empty(m, n, device=dev), torch.empty(m, 1000, device=dev)
        ff.i8_matmul(a, sa, b, sb, out, k)
        ff.i8_matmul(a, sa, b[-1000:], sb[-1000:], tail, k)
        assert torch.equal(out[:, -1000:], tail)
    del b, out
    m, n, k = 40000, 60000, 64
    a, sa = integers(dev, m, k)
    b, sb = integers(dev, n, k)
    out, tail = torch.empty(m, n, dtype=torch.bfloat16, device=dev), torch.empty(100, n, dtype=torch.bfloat16, device=dev)
    ff.i8_matmul(a, sa, b, sb, out, k)
    ff.i8_matmul(a[-100:], sa[-100:], b, sb, tail, k)
    assert torch.equal(out[-100:], tail)


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128), (40, 100), (128, 64)])
@pytest.mark.parametrize("splits", [1, 2, 5, 64])
def test_split_tokens(dev, rng, kind, dk, dv, splits):
    """Tokens split among workgroups, lengths at and around the parts' ends: results with and without the state behind
    them, and the gradients."""
    import torch
    import fufft_amd as ff
    batch, tokens, heads = 6, 643, 1
    lens = np.array([643, 0, 1, 128, 129, 320], dtype=np.int32)
    print(f"case decay split {kind} {dk}x{dv} {splits}", flush=True)
    ts, x64 = [], []
    for d in (dk, dk, dv, dv):
        t, x = R.typed(rng.standard_normal((batch, tokens, heads, d)), kind, dev)
        ts.append(t)
        x64.append(x)
    q, k, v, do = ts
    g = np.array([-0.01], dtype=np.float32)
    gd, ld = torch.from_numpy(g).to(dev), torch.from_numpy(lens).to(dev)
    states = [rng.standard_normal((batch, heads, dk, dv)).astype(np.float32) for _ in range(2)]
    state, dnew = (torch.from_numpy(s).to(dev) for s in states)
    s64, d64 = (s.astype(np.float64) for s in states)
    work = torch.full((splits * 3, batch, heads, dk, dv), float("nan"), device=dev)

    def rows(got, want, err):
        for b in range(batch):
            assert R.inside(got[b, :lens[b]], want[b, :lens[b]], err[b, :lens[b]])
            assert bool((got[b, lens[b]:] == 5).all())
    want, err, new, nerr = R.attention(x64[0], x64[1], x64[2], g, s64, lens, 0.2, kind)
    for behind in (None, torch.empty_like(state)):
        out = torch.full_like(v, 5.0)
        ff.decay_attention(q, k, v, gd, out, state=state, new_state=behind, lens=ld, work=work[:splits], scale=0.2)
        rows(out, want, err)
        if behind is not None:
            assert R.inside(behind, new, nerr)
    wants = R.attention_grad(x64[3], x64[0], x64[1], x64[2], g, s64, d64, lens, 0.2, kind)
    for ds in (None, torch.empty_like(state)):
        got = [torch.full_like(x, 5.0) for x in (q, k, v)]
        work.fill_(float("nan"))
        ff.decay_attention_grad(do, q, k, v, gd, *got, state=state, dnew_state=dnew, dstate=ds, lens=ld, work=work, scale=0.2)
        for x, (want, err) in zip(got, wants):
            rows(x, want, err)
        if ds is not None:
            assert R.inside(ds, *wants[3])


def test_split_tokens_beyond_4gib(dev):
    import torch
    import fufft_amd as ff
    t, h, d = 600, 2, 24
    big = torch.empty((1 << 32) // 2 + (1 << 20), dtype=torch.bfloat16, device=dev)
    far = big.as_strided((1, t, h, d), (0, (1 << 31) // t // 8 * 8, d, 1))
    far.copy_(torch.randn(1, t, h, d, device=dev))
    near, g = far.contiguous(), torch.tensor([-0.1, 0.0], device=dev)
    work, state = torch.empty(5 * 3, 1, h, d, d, device=dev), [torch.empty(1, h, d, d, device=dev) for _ in range(4)]
    outs = []
    for x, s in ((far, state[:2]), (near, state[2:])):
        o = [torch.empty_like(near) for _ in range(4)]
        ff.decay_attention(x, x, x, g, o[0], new_state=s[0], work=work)
        ff.decay_attention_grad(x, x, x, x, g, *o[1:], dstate=s[1], work=work)
        outs.append(o)
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert torch.equal(state[0], state[2]) and torch.equal(state[1], state[3])


def test_widths_between_kernels(dev, rng):
    """Norms and 8-bit rows of one element more and less than a kernel holds, and no row at all."""
    import torch
    import fufft_amd as ff
    for k in (31, 33, 127, 129, 511, 513, 1023, 1025, 2047, 2049, 4095, 4097, 8191, 8193, 16383, 16385, 32767, 32769, 65536):
        print(f"case widths {k}", flush=True)
        x, x64 = R.typed(rng.standard_normal((5, k)), "bf16", dev)
        w = rng.standard_normal(k).astype(np.float32)
        wd = torch.from_numpy(w).to(dev)
        out = torch.empty(5, k, dtype=torch.bfloat16, device=dev)
        codes, scales = ff.i8_empty(5, k)
        ff.rms_norm(x, wd, out, codes=codes, scales=scales)
        want, share = R.norm(x64, w.astype(np.float64), 1e-6)
        assert R.inside(out, want, np.abs(want) * share)
        assert not bool(codes[:, k:].any())
        # a code stands for y to within half a step of its scale
        back = codes[:, :k].double().cpu().numpy() * scales.double().cpu().numpy()[:, None]
        top = np.abs(want).max(1, keepdims=True)
        assert (np.abs(back - want) <= top / 254 * 1.0001 + np.abs(want) * 2 * share).all()
