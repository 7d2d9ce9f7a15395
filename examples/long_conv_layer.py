"""A gated long-convolution layer on this library's calls: its projections in
microscaled 4-bit blocks, its causal convolution by FFT over whole texts and from a
paged cache token by token.

    v, g = split(x Wi^T)      y[t] = g[t] * sum_j taps[j] v[t - j]      out = y Wo^T

`prompt` runs whole texts (two at a time: the two-for-one convolution takes two real
signals a filter), `step` one more token of each, `gradients` the training pass.

    python examples/long_conv_layer.py
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import fufft_amd as ff  # noqa: E402

DEV = "cuda"


class Projection:
    """y = x w^T with w in blocks along its rows (forward) and columns (its input's gradient)."""

    def __init__(self, w: torch.Tensor):
        self.n, self.k = w.shape
        self.rows, self.columns = ff.mx4_empty(self.n, self.k), ff.mx4_empty(self.k, self.n)
        ff.mx4_quantize(w, *self.rows, *self.columns)

    def __call__(self, x):
        """Many rows: x made 4-bit too."""
        q, y = ff.mx4_empty(*x.shape), torch.empty(x.shape[0], self.n, device=DEV)
        ff.mx4_quantize(x, *q)
        ff.mx4_matmul(*q, *self.rows, y, self.k)
        return y

    def tokens(self, x):
        """A few rows: x as it is."""
        y = torch.empty(x.shape[0], self.n, device=DEV)
        ff.mx4_linear(x, *self.rows, y)
        return y

    def gradients(self, x, dy):
        """(dx, dw); dy is rounded at random, so that what it loses averages out."""
        m = x.shape[0]
        rand = torch.randint(0, 256, dy.shape, dtype=torch.uint8, device=DEV)
        qx, qd, qd_t = ff.mx4_empty(self.k, m), ff.mx4_empty(m, self.n), ff.mx4_empty(self.n, m)
        ff.mx4_quantize(x, None, None, *qx)
        ff.mx4_quantize(dy, *qd, *qd_t, rand=rand)
        dx, dw = torch.empty(m, self.k, device=DEV), torch.empty(self.n, self.k, device=DEV)
        ff.mx4_matmul(*qd, *self.columns, dx, self.n)
        ff.mx4_matmul(*qd_t, *qx, dw, m)
        return dx, dw


class LongConvLayer:
    TEXTS = 2           # the two real signals of a two-for-one convolution

    def __init__(self, width: int, channels: int, longest: int, page: int = 64):
        self.channels, self.longest = channels, longest
        self.n = max(256, 2 << (longest - 1).bit_length())           # transform: a text and its zero padding
        self.inp = Projection(torch.randn(2 * channels, width, device=DEV) / math.sqrt(width))
        self.out = Projection(torch.randn(width, channels, device=DEV) / math.sqrt(channels))
        j = torch.arange(longest, device=DEV)[:, None]
        rate = torch.exp(torch.rand(channels, device=DEV) * -4) / 4
        self.taps = torch.randn(longest, channels, device=DEV) * torch.exp(-j * rate)
        # a filter a channel, and its conjugate's for the gradient (correlation)
        spec = torch.fft.fft(self.taps.t(), n=self.n).contiguous()
        self.filt, self.filt_conj = torch.empty_like(spec), torch.empty_like(spec)
        ff.plan_filter_device(spec, self.filt, self.n, count=channels, kind=ff.FILTER_SPECTRUM)
        ff.plan_filter_device(spec.conj().resolve_conj().contiguous(), self.filt_conj, self.n, count=channels,
                              kind=ff.FILTER_SPECTRUM)
        # the cache: every text's pages in a table, written as tokens come
        pages = -(-longest // page)
        self.page = page
        self.table = torch.arange(self.TEXTS * pages, dtype=torch.int32, device=DEV).view(self.TEXTS, pages)
        codes, scales = ff.mx4_empty(self.TEXTS * pages * page, channels)
        self.cache = codes.view(self.TEXTS * pages, page, -1), scales.view(self.TEXTS * pages, page, -1)
        self.lens = torch.zeros(self.TEXTS, dtype=torch.int32, device=DEV)
        self.work = torch.empty(64, self.TEXTS, channels, device=DEV)

    def _slots(self, t):
        """Slots of tokens t (texts, any count) of each text."""
        return (self.table.long().gather(1, t // self.page) * self.page + t % self.page).reshape(-1)

    def _convolve(self, signals, filt):
        """The texts' signals (texts, channels, n) with a filter a channel."""
        u = torch.empty_like(signals)
        ff.conv_r2(signals[0], signals[1], filt, u[0], u[1], self.n, self.channels, filt_stride=self.n)
        return u

    def prompt(self, x):
        """x (texts, length, width): the layer's outputs, the cache holding the texts."""
        texts, length, width = x.shape
        v, g = self.inp(x.reshape(texts * length, width)).split(self.channels, dim=1)
        self.lens.fill_(length)
        t = torch.arange(length, device=DEV).expand(texts, length)
        ff.mx4_cache_write(v, self._slots(t), *self.cache)
        signals = torch.empty(texts, self.channels, self.n, device=DEV)
        ff.mx4_cache_read(*self.cache, self.table, self.lens, signals, order="channels")
        self.convolved = self._convolve(signals, self.filt)[:, :, :length].transpose(1, 2)
        y = (self.convolved * g.reshape(texts, length, -1)).reshape(texts * length, -1)
        return self.out(y).view(texts, length, -1)

    def step(self, x):
        """x (texts, width): one more token of each text."""
        v, g = self.inp.tokens(x).split(self.channels, dim=1)
        ff.mx4_cache_write(v, self._slots(self.lens.long()[:, None]), *self.cache)
        self.lens += 1
        return self.out.tokens(self.last() * g)

    def last(self):
        """The convolution at the last token of each text, from the cache."""
        y = torch.empty(self.TEXTS, self.channels, device=DEV)
        ff.mx4_cache_conv(*self.cache, self.table, self.lens, self.taps, y, work=self.work)
        return y

    def gradients(self, x, dout):
        """(dx, dWi, dWo) for texts x and the gradient dout of the layer's outputs."""
        texts, length, width = x.shape
        rows = x.reshape(texts * length, width)
        v, g = self.inp(rows).view(texts, length, -1).split(self.channels, dim=2)
        signals = torch.zeros(texts, self.channels, self.n, device=DEV)
        signals[:, :, :length] = v.transpose(1, 2)
        c = self._convolve(signals, self.filt)[:, :, :length].transpose(1, 2)
        dy, dwo = self.out.gradients((c * g).reshape(texts * length, -1), dout.reshape(texts * length, -1))
        dy = dy.view(texts, length, -1)
        signals.zero_()
        signals[:, :, :length] = (dy * g).transpose(1, 2)
        dv = self._convolve(signals, self.filt_conj)[:, :, :length].transpose(1, 2)
        dx, dwi = self.inp.gradients(rows, torch.cat((dv, dy * c), dim=2).reshape(texts * length, -1))
        return dx.view_as(x), dwi, dwo


def main():
    torch.manual_seed(0)
    ff.init(0)
    layer = LongConvLayer(width=512, channels=768, longest=1500)
    x = torch.randn(2, 1001, 512, device=DEV)
    out = layer.prompt(x)
    rel = float((layer.last() - layer.convolved[:, -1]).norm() / layer.convolved[:, -1].norm())
    print(f"prompt of {x.shape[1]} tokens: {tuple(out.shape)}; the step form at its last token is {rel:.1e} from the FFT's")
    for _ in range(3):
        token = layer.step(torch.randn(2, 512, device=DEV))
    print(f"three more tokens: {tuple(token.shape)}, lengths {layer.lens.tolist()}")
    dx, dwi, dwo = layer.gradients(x, torch.randn_like(out))
    print(f"gradients: {tuple(dx.shape)}, {tuple(dwi.shape)}, {tuple(dwo.shape)}")


if __name__ == "__main__":
    main()
