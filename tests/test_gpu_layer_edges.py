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


def recurrence(q, k, v, g, lens, state=None, late=0):
    """mixed of tests/layer_reference.py for all sequences and heads at once, in fp64 tensors: (out, state behind, their magnitudes)."""
    import torch
    batch, tokens, heads, dk = q.shape
    a = torch.exp(g)[:, None, None]
    s = torch.zeros(batch, heads, dk, v.shape[3], dtype=torch.float64, device=q.device) if state is None else state.clone()
    m = s.abs()
    out, mags = torch.zeros_like(v), torch.zeros_like(v)
    for t in range(tokens):
        there = (lens > t)[:, None, None, None]
        f = torch.ones_like(a) if late and t == 0 else a
        kv = k[:, t, :, :, None] * v[:, t, :, None, :]
        s, m = torch.where(there, f * s + kv, s), torch.where(there, f * m + kv.abs(), m)
        out[:, t], mags[:, t] = (q[:, t, :, :, None] * s).sum(2), (q[:, t, :, :, None].abs() * m).sum(2)
    if late:
        some = (lens > 0)[:, None, None, None]
        s, m = torch.where(some, a * s, s), torch.where(some, a * m, m)
    return out, s, mags, m


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("dk,dv", [(16, 24), (5, 9)])
def test_long_split(dev, kind, dk, dv):
    """Segments of two parts of several chunks each: 32 sequences and heads, lengths at and around the parts' ends."""
    import torch
    import fufft_amd as ff
    tokens, heads = 8192, 2
    lens = torch.tensor([8192, 0, 1, 511, 512, 513, 1024, 1025, 2047, 2048, 2049, 4096, 4097, 6144, 8128, 8191], device=dev)
    batch = len(lens)
    print(f"case decay long split {kind} {dk}x{dv}", flush=True)
    gen = torch.Generator(device=dev).manual_seed(7)
    q, k, v, do = (torch.randn(batch, tokens, heads, d, device=dev, generator=gen).to(R.torch_type(kind)) for d in (dk, dk, dv, dv))
    state, dnew = (torch.randn(batch, heads, dk, dv, device=dev, generator=gen) for _ in range(2))
    g = torch.tensor([-0.001, -0.3], device=dev)
    work = torch.full((16 * 3, batch, heads, dk, dv), float("nan"), device=dev)
    ld, scale = lens.int(), 0.25
    x = [t.double() for t in (q, k, v, do)]
    # a share for each head, of the longest sequence
    share = lambda dim, carried=False: torch.tensor([R.mixed_share(kind, tokens, dim, float(h), carried) for h in g], dtype=torch.float64, device=dev)[:, None]
    at = torch.arange(tokens, device=dev)
    inside_len = (at[None, :] < lens[:, None])

    def near(got, want, err):
        # half a step of the type, and of its smallest number
        eps = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[kind]
        off = (got.double() - want).abs() - err - (want.abs() + err) * eps - 2.0 ** -25
        assert bool((off[inside_len] <= 0).all()) and bool((got[~inside_len] == 5).all())

    def carried(got, want, mags):
        assert bool(((got.double() - want).abs() <= mags * share(0, True)[:, None] + want.abs() * 2.0 ** -24).all())
    want, new, mags, nm = recurrence(x[0], x[1], x[2], g.double(), lens, state.double())
    for behind in (None, torch.empty_like(state)):
        out = torch.full_like(v, 5.0)
        work.fill_(float("nan"))
        ff.decay_attention(q, k, v, g, out, state=state, new_state=behind, lens=ld, work=work[:16], scale=scale)
        near(out, scale * want, scale * mags * share(dk))
        if behind is not None:
            carried(behind, new, nm)
    # the gradients, from the last token back
    back = (lens[:, None] - 1 - at[None, :]).clamp(0)[:, :, None, None]
    turned = [t.gather(1, back.expand_as(t)) for t in x]
    wq, _, mq, _ = recurrence(x[3], x[2], x[1], g.double(), lens, state.double().transpose(2, 3))
    wk, _, mk, _ = recurrence(turned[2], scale * turned[3], turned[0], g.double(), lens, dnew.double().transpose(2, 3), 1)
    wv, ws, mv, ms = recurrence(turned[1], scale * turned[0], turned[3], g.double(), lens, dnew.double(), 1)
    wk, mk, wv, mv = (t.gather(1, back.expand_as(t)) for t in (wk, mk, wv, mv))
    got, ds = [torch.full_like(t, 5.0) for t in (q, k, v)], torch.empty_like(state)
    work.fill_(float("nan"))
    ff.decay_attention_grad(do, q, k, v, g, *got, state=state, dnew_state=dnew, dstate=ds, lens=ld, work=work, scale=scale)
    near(got[0], scale * wq, scale * mq * share(dv))
    near(got[1], wk, mk * share(dv))
    near(got[2], wv, mv * share(dk))
    carried(ds, ws, ms)


def test_split_in_graphs(dev):
    """Split calls captured into two graphs, each with a workspace of its own, replayed in turn and at once over changed inputs."""
    import torch
    import fufft_amd as ff
    batch, tokens, heads, d = 2, 2500, 3, 40
    g = torch.tensor([-0.05, 0.0, -2.0], device=dev)
    lens = torch.tensor([2500, 1300], dtype=torch.int32, device=dev)

    class One:
        def __init__(self):
            self.x = [torch.empty(batch, tokens, heads, d, dtype=torch.bfloat16, device=dev) for _ in range(4)]
            self.out = [torch.zeros_like(self.x[0]) for _ in range(4)]
            self.state = torch.zeros(batch, heads, d, d, device=dev)
            self.work = torch.empty(6, 3, batch, heads, d, d, device=dev)

        def fill(self, seed):
            gen = torch.Generator(device=dev).manual_seed(seed)
            for t in self.x:
                t.copy_(torch.randn(t.shape, device=dev, generator=gen))
            self.state.fill_(0.5)

        def run(self):
            q, k, v, do = self.x
            ff.decay_attention(q, k, v, g, self.out[0], state=self.state, new_state=self.state, lens=lens, work=self.work)
            ff.decay_attention_grad(do, q, k, v, g, *self.out[1:], dstate=None, lens=lens, work=self.work)
    ones, graphs = [One(), One()], []
    side = torch.cuda.Stream()
    for o in ones:
        o.fill(0)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            o.run()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            o.run()
    for seed in (1, 2, 3):
        for i, o in enumerate(ones):
            o.fill(2 * seed + i)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in ones]
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for i, o in enumerate(ones):
            want = One()
            want.fill(2 * seed + i)
            want.run()
            torch.cuda.synchronize()
            assert torch.equal(o.state, want.state) and all(torch.equal(a, b) for a, b in zip(o.out, want.out))
