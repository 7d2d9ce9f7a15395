"""GPU tests of the norm, 8-bit and decaying-attention calls together, as a model's block uses them:
without the native binding, in captured graphs, on other streams, and prompt against token by token."""
import numpy as np
import pytest

import layer_reference as R

pytestmark = pytest.mark.gpu

WIDTH, HEADS, DK, DV = 192, 3, 40, 56


class Block:
    """h += attention(norm(h) Wi) Wo with 8-bit products: norm to 8 bits, one projection to q, k and v, the attention, its
    result in 8 bits again, the projection back, and the norm that takes its sum with the residual."""

    def __init__(self, torch, ff, dev, kind):
        g = torch.Generator(device=dev).manual_seed(5)
        self.torch, self.ff, self.dev, self.type = torch, ff, dev, R.torch_type(kind)
        self.inner = HEADS * (2 * DK + DV)
        wi = torch.randn(self.inner, WIDTH, device=dev, generator=g) / WIDTH ** 0.5
        wo = torch.randn(WIDTH, HEADS * DV, device=dev, generator=g) / (HEADS * DV) ** 0.5
        self.wi, self.wo = ff.i8_empty(self.inner, WIDTH), ff.i8_empty(WIDTH, HEADS * DV)
        ff.i8_quantize(wi, *self.wi)
        ff.i8_quantize(wo, *self.wo)
        self.weight = 1 + torch.randn(WIDTH, device=dev, generator=g) / 8
        self.decay = torch.tensor([-0.01, -0.1, -0.5], device=dev)

    def empty(self, *shape, dtype=None):
        return self.torch.empty(*shape, dtype=dtype or self.type, device=self.dev)

    def split(self, qkv):
        at = [HEADS * DK, HEADS * DK, HEADS * DV]
        return [x.unflatten(-1, (HEADS, -1)) for x in qkv.split(at, dim=-1)]

    def project(self, x, residual):
        """(q, k, v) of rows x, residual (fp32) updated."""
        ff, rows = self.ff, x.shape[0]
        q = ff.i8_empty(rows, WIDTH)
        ff.rms_norm(x, self.weight, codes=q[0], scales=q[1], residual=residual, total=residual)
        qkv = self.empty(rows, self.inner)
        ff.i8_matmul(*q, *self.wi, qkv, WIDTH)
        return qkv

    def back(self, mixed):
        ff, rows = self.ff, mixed.shape[0]
        q = ff.i8_empty(rows, HEADS * DV)
        ff.i8_quantize(mixed, *q)
        out = self.empty(rows, WIDTH)
        ff.i8_matmul(*q, *self.wo, out, HEADS * DV)
        return out

    def prompt(self, x, state, lens, work=None):
        batch, tokens, _ = x.shape
        residual = self.torch.zeros(batch * tokens, WIDTH, device=self.dev)
        qkv = self.project(x.reshape(-1, WIDTH), residual).view(batch, tokens, -1)
        mixed = self.torch.zeros(batch, tokens, HEADS, DV, dtype=self.type, device=self.dev)
        self.ff.decay_attention(*self.split(qkv), self.decay, mixed, new_state=state, lens=lens, work=work, scale=DK ** -0.5)
        return self.back(mixed.view(batch * tokens, -1)).view(batch, tokens, -1)

    def token(self, x, state, slots=None):
        residual = self.torch.zeros(x.shape[0], WIDTH, device=self.dev)
        qkv = self.project(x, residual)
        mixed = self.empty(x.shape[0], HEADS, DV)
        self.ff.decay_attention_step(*self.split(qkv), self.decay, state, mixed, slots=slots, scale=DK ** -0.5)
        return self.back(mixed.view(x.shape[0], -1))

    def gradients(self, x, dy, work):
        """Of the norm and of the attention on what it made, as a training pass calls them."""
        batch, tokens, _ = x.shape
        rows = x.reshape(-1, WIDTH)
        normed = self.torch.empty_like(rows)
        self.ff.rms_norm(rows, self.weight, normed)
        h = self.torch.cat((normed, normed, normed), dim=1)[:, :self.inner].contiguous().view(batch, tokens, -1)
        q, k, v = self.split(h)
        grads = self.torch.empty_like(h)
        self.ff.decay_attention_grad(dy, q, k, v, self.decay, *self.split(grads), work=work, scale=0.2)
        dn = grads.view(-1, self.inner)[:, :WIDTH]
        dx, dw = self.torch.empty_like(rows), self.torch.empty(WIDTH, device=self.dev)
        self.ff.rms_norm_grad(dn, rows, self.weight, dx, dw, self.torch.empty(16, WIDTH, device=self.dev))
        return dx, dw, grads


def inputs(torch, dev, kind, batch=3, tokens=300, seed=1):
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randn(batch, tokens, WIDTH, device=dev, generator=g).to(R.torch_type(kind))


def every_call(torch, ff, dev, kind):
    b = Block(torch, ff, dev, kind)
    x = inputs(torch, dev, kind)
    lens = torch.tensor([300, 20, 0], dtype=torch.int32, device=dev)
    state = torch.empty(3, HEADS, DK, DV, device=dev)
    out = b.prompt(x, state, lens, work=torch.empty(5, 3, HEADS, DK, DV, device=dev))
    kept = state.clone()
    one = b.token(x[:, 5], state, slots=torch.tensor([2, 0, -1], device=dev))
    dy = inputs(torch, dev, kind, seed=2)[..., :HEADS * DV].reshape(3, 300, HEADS, DV)
    grads = b.gradients(x, dy, torch.empty(4, 3, 3, HEADS, DK, DV, device=dev))
    codes, scales = ff.i8_empty(900, WIDTH)
    ff.i8_quantize(x.view(900, WIDTH), codes, scales)
    read = torch.empty(900, WIDTH, device=dev)
    ff.i8_dequantize(codes, scales, read)
    torch.cuda.synchronize()
    return [out, kept, one, state, *grads, read]


@pytest.mark.parametrize("kind", R.TYPES)
def test_same_without_the_binding(dev, monkeypatch, kind):
    """Through ctypes the same kernels, bit for bit."""
    import torch
    import fufft_amd as ff
    assert ff._binding is not None
    want = every_call(torch, ff, dev, kind)
    monkeypatch.setattr(ff, "_binding", None)
    for got, ref in zip(every_call(torch, ff, dev, kind), want):
        assert torch.equal(got, ref)


@pytest.mark.parametrize("kind", R.TYPES)
def test_prompt_is_its_tokens(dev, kind):
    """The block over a prompt, and over its tokens one by one: the same within the roundings between them."""
    import torch
    import fufft_amd as ff
    b = Block(torch, ff, dev, kind)
    x = inputs(torch, dev, kind, batch=2, tokens=90)
    state, steps = torch.empty(2, HEADS, DK, DV, device=dev), torch.zeros(2, HEADS, DK, DV, device=dev)
    whole = b.prompt(x, state, None).double()
    one = torch.stack([b.token(x[:, t], steps) for t in range(90)], dim=1).double()
    # A value that both ways round to 8 bits apart is off by one of 254 steps of its row's largest; the attention's bf16
    # operands by 2^-7 of it in sum; the result is a sum of 168 such values.  2 % of the norm holds both.
    assert float((whole - one).norm() / whole.norm()) < 0.02
    assert float((state - steps).norm() / steps.norm()) < 1e-4


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_graphs(dev, kind):
    """A captured prompt, token and training pass, replayed over changed inputs with eager work between, as the
    eager calls give them."""
    import torch
    import fufft_amd as ff
    b = Block(torch, ff, dev, kind)
    x = inputs(torch, dev, kind)
    lens = torch.tensor([300, 20, 100], dtype=torch.int32, device=dev)
    state, slots = torch.zeros(3, HEADS, DK, DV, device=dev), torch.tensor([2, 0, 1], device=dev)
    work, work3 = torch.empty(5, 3, HEADS, DK, DV, device=dev), torch.empty(4, 3, 3, HEADS, DK, DV, device=dev)
    dy = inputs(torch, dev, kind, seed=2)[..., :HEADS * DV].reshape(3, 300, HEADS, DV).contiguous()

    def all_of(x, state):
        out = b.prompt(x, state, lens, work)
        one = b.token(x[:, 5], state, slots)
        return [out, one, *b.gradients(x, dy, work3)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        all_of(x, state)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = all_of(x, state)
    for seed in (3, 4, 5):
        x.copy_(inputs(torch, dev, kind, seed=seed))
        graph.replay()
        torch.cuda.synchronize()
        got, s = [t.clone() for t in captured], state.clone()
        other = torch.empty_like(state)
        want = all_of(x.clone(), other)
        torch.cuda.synchronize()
        assert torch.equal(s, other)
        for g, w in zip(got, want):
            assert torch.equal(g, w)


def test_streams(dev):
    """Two blocks at once, each on a stream of its own with its own workspace, given as argument or current."""
    import torch
    import fufft_amd as ff
    b = Block(torch, ff, dev, "bf16")
    xs = [inputs(torch, dev, "bf16", seed=s) for s in (7, 8)]
    states = [torch.empty(3, HEADS, DK, DV, device=dev) for _ in xs]
    want = [b.prompt(x, s, None) for x, s in zip(xs, states)]
    kept = [s.clone() for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(3):
        got = []
        for x, s, st in zip(xs, states, streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append(b.prompt(x, s, None, torch.empty(5, 3, HEADS, DK, DV, device=dev)))
        torch.cuda.synchronize()
        for g, w, s, k in zip(got, want, states, kept):
            # with a workspace the tokens are split, so sums are in another order: within bf16's own step
            assert float((g.double() - w.double()).norm() / w.double().norm()) < 0.01
            assert float((s - k).norm() / k.norm()) < 1e-5
    x = torch.randn(64, 96, device=dev)
    out, here = torch.empty_like(x), torch.empty_like(x)
    ff.rms_norm(x, None, here)
    streams[0].wait_stream(torch.cuda.current_stream())
    ff.rms_norm(x, None, out, stream=streams[0])
    torch.cuda.synchronize()
    assert torch.equal(out, here)


def test_beyond_4gib(dev):
    """Rows of an array, states of a pool and tokens of a text that lie beyond 4 GiB."""
    import torch
    import fufft_amd as ff
    rows, k = 3, 520
    big = torch.empty((1 << 32) // 2 + (1 << 20), dtype=torch.bfloat16, device=dev)     # 4 GiB and some
    ld = (1 << 30) + 64
    x = big.as_strided((rows, k), (ld, 1))
    x.copy_(torch.randn(rows, k, device=dev))
    want, out = torch.empty(rows, k, dtype=torch.bfloat16, device=dev), torch.empty(rows, k, dtype=torch.bfloat16, device=dev)
    ff.rms_norm(x.contiguous(), None, want)
    ff.rms_norm(x, None, out)
    assert torch.equal(out, want)
    codes, scales = ff.i8_empty(rows, k)
    c2, s2 = ff.i8_empty(rows, k)
    ff.i8_quantize(x, codes, scales)
    ff.i8_quantize(x.contiguous(), c2, s2)
    assert torch.equal(codes, c2) and torch.equal(scales, s2)
    # a text whose tokens are far apart, forwards and back
    t, h, d = 70, 1, 16
    step = (1 << 31) // t // 8 * 8
    q = big.as_strided((1, t, h, d), (0, step, d, 1))
    q.copy_(torch.randn(1, t, h, d, device=dev))
    near, g = q.contiguous(), torch.tensor([-0.1], device=dev)
    o1, o2 = torch.empty_like(near), torch.empty_like(near)
    ff.decay_attention(q, near, q, g, o1)
    ff.decay_attention(near, near, near, g, o2)
    assert torch.equal(o1, o2)
    a, b = [torch.empty_like(near) for _ in range(3)], [torch.empty_like(near) for _ in range(3)]
    ff.decay_attention_grad(q, q, near, q, g, *a)
    ff.decay_attention_grad(near, near, near, near, g, *b)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    del big, x, q
    pool = torch.empty(2100, 32, 128, 128, device=dev)                    # 4.2 GiB of states
    for slot in (0, 2047, 2099):
        pool[slot].normal_()
    slots = torch.tensor([2099, 2047, 0], device=dev)
    small = pool[slots].contiguous()
    qkv = [torch.randn(3, 32, 128, device=dev) for _ in range(3)]
    g = -torch.rand(32, device=dev)
    o1, o2 = torch.empty(3, 32, 128, device=dev), torch.empty(3, 32, 128, device=dev)
    ff.decay_attention_step(*qkv, g, pool, o1, slots=slots)
    ff.decay_attention_step(*qkv, g, small, o2)
    assert torch.equal(o1, o2) and torch.equal(pool[slots], small)


def test_many_sequences(dev):
    """More sequences and heads than a grid's first axis has of workgroups at once, and than 65535."""
    import torch
    import fufft_amd as ff
    batch, heads, d = 40000, 2, 8
    q, k, v = (torch.randn(batch, 3, heads, d, device=dev) for _ in range(3))
    g = torch.tensor([-0.2, 0.0], device=dev)
    out, new = torch.empty_like(v), torch.empty(batch, heads, d, d, device=dev)
    ff.decay_attention(q, k, v, g, out, new_state=new)
    state, one = torch.zeros_like(new), torch.empty(batch, heads, d, device=dev)
    for t in range(3):
        ff.decay_attention_step(q[:, t], k[:, t], v[:, t], g, state, one)
        # sums of 8 products in other orders
        assert float((one - out[:, t]).abs().max()) < 200 * R.EPS24 * float(out.abs().max())
    assert float((state - new).abs().max()) < 100 * R.EPS24 * float(new.abs().max())
