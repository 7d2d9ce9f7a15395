"""CPU tests of the norm and 8-bit calls: what the C ABI and the Python binding refuse before
anything is launched, and the 64-bit form that the GPU tests compare with."""
import numpy as np
import pytest
import torch

import fufft_amd as ff
import layer_reference as R

INV, ALIGN, OK, UNSUP = ff.ERR_INVALID, ff.ERR_ALIGN, ff.OK, ff.ERR_UNSUPPORTED
P = [0x10000000 * (i + 1) for i in range(12)]          # addresses that are checked and never read


def test_padded():
    assert [ff.i8_padded(k) for k in (0, 1, 128, 129)] == [0, 128, 128, 256]
    assert [ff.lib.fufft_i8_padded(k) for k in (0, 1, 128, 129, -1)] == [0, 128, 128, 256, INV]
    codes, scales = ff.i8_empty(3, 130, device="cpu")
    assert codes.shape == (3, 256) and codes.dtype == torch.int8 and scales.shape == (3,)


def test_quantize_refusals():
    def call(x=P[0], type=0, ld=256, rows=4, k=200, c=P[1], s=P[2]):
        return ff.lib.fufft_i8_quantize(x, type, ld, rows, k, c, s, None)
    for bad in (dict(type=3), dict(ld=199), dict(rows=-1), dict(k=-1), dict(k=1 << 62), dict(x=None), dict(c=None),
                dict(s=None), dict(c=P[0]), dict(s=P[1] + 1020), dict(s=P[0] + 4 * (3 * 256 + 196))):
        assert call(**bad) == INV, bad
    for bad in (dict(c=P[1] + 8), dict(s=P[2] + 2), dict(x=P[0] + 2), dict(x=P[0] + 1, type=1)):
        assert call(**bad) == ALIGN, bad
    assert call(rows=0) == OK and call(k=0) == OK

    def back(c=P[0], s=P[1], o=P[2], type=0, ld=200, rows=4, k=200):
        return ff.lib.fufft_i8_dequantize(c, s, o, type, ld, rows, k, None)
    for bad in (dict(c=None), dict(s=None), dict(o=None), dict(type=7), dict(ld=100), dict(rows=-2), dict(o=P[0] + 16),
                dict(o=P[1] - 8)):
        assert back(**bad) == INV, bad
    for bad in (dict(c=P[0] + 1), dict(s=P[1] + 1), dict(o=P[2] + 1)):
        assert back(**bad) == ALIGN, bad
    assert back(rows=0) == OK


def test_matmul_refusals():
    def call(a=P[0], sa=P[1], b=P[2], sb=P[3], bias=P[4], o=P[5], type=0, ld=8, m=4, n=8, k=64):
        return ff.lib.fufft_i8_matmul(a, sa, b, sb, bias, o, type, ld, m, n, k, None)
    for bad in (dict(a=None), dict(sa=None), dict(b=None), dict(sb=None), dict(o=None), dict(type=3), dict(ld=7),
                dict(m=-1), dict(n=-1), dict(k=-1), dict(m=1 << 40, k=1 << 40), dict(o=P[0]), dict(o=P[4] + 4),
                dict(o=P[3] - 32), dict(o=P[1] + 12)):
        assert call(**bad) == INV, bad
    for bad in (dict(a=P[0] + 8), dict(b=P[2] + 8), dict(sa=P[1] + 1), dict(sb=P[3] + 2), dict(bias=P[4] + 2),
                dict(o=P[5] + 2)):
        assert call(**bad) == ALIGN, bad
    assert call(k=131072) == UNSUP and call(k=1 << 20) == UNSUP
    assert call(m=0) == OK and call(n=0) == OK


def norm(x=P[0], type=1, ldx=200, res=P[1], ldr=200, total=P[2], ldt=200, st=0, w=P[3], eps=1e-6, o=P[4], ldo=200, c=P[5],
         s=P[6], rows=4, k=200):
    return ff.lib.fufft_rms_norm(x, type, ldx, res, ldr, total, ldt, st, w, eps, o, ldo, c, s, rows, k, None)


def test_norm_refusals():
    for bad in (dict(x=None), dict(type=5), dict(st=2), dict(type=0, st=1), dict(ldx=199), dict(ldr=1), dict(ldt=199),
                dict(ldo=0), dict(eps=-1.0), dict(eps=float("inf")), dict(eps=float("nan")), dict(rows=-1), dict(k=-1),
                dict(o=None, c=None, s=None), dict(c=None), dict(s=None), dict(o=None, s=None),
                dict(o=P[0] + 4), dict(o=P[0], ldx=400, ldo=200), dict(o=P[1]), dict(o=P[2]), dict(total=P[0]),
                dict(total=P[1] + 4), dict(total=P[1], ldt=300), dict(total=P[3] - 4 * 700), dict(c=P[0]), dict(s=P[4]),
                dict(c=P[3]), dict(s=P[5] + 64)):
        assert norm(**bad) == INV, bad
    for bad in (dict(x=P[0] + 1), dict(res=P[1] + 2), dict(total=P[2] + 2), dict(w=P[3] + 1), dict(o=P[4] + 1),
                dict(c=P[5] + 4), dict(s=P[6] + 2)):
        assert norm(**bad) == ALIGN, bad
    assert norm(rows=0) == OK and norm(k=0) == OK


def test_norm_grad_refusals():
    def call(dy=P[0], type=1, ldy=200, h=P[1], ldh=200, dt=P[2], ldt=200, st=0, w=P[3], eps=1e-6, dx=P[4], xt=0, ldx=200,
             dw=P[5], work=P[6], splits=8, rows=4, k=200):
        return ff.lib.fufft_rms_norm_grad(dy, type, ldy, h, ldh, dt, ldt, st, w, eps, dx, xt, ldx, dw, work, splits, rows, k,
                                          None)
    for bad in (dict(dy=None), dict(h=None), dict(dx=None), dict(type=5), dict(st=2), dict(xt=2), dict(type=0, st=0, xt=1),
                dict(ldy=1), dict(ldh=1), dict(ldt=1), dict(ldx=1), dict(eps=-1.0), dict(splits=0), dict(splits=-1),
                dict(work=None), dict(rows=-1), dict(k=-1), dict(dx=P[1]), dict(dx=P[0]), dict(dx=P[2] + 4),
                dict(dx=P[2], ldx=300), dict(dw=P[0]), dict(dw=P[3]), dict(dw=P[6] + 400), dict(work=P[4]),
                dict(work=P[1])):
        assert call(**bad) == INV, bad
    for bad in (dict(dy=P[0] + 1), dict(h=P[1] + 2), dict(dt=P[2] + 1), dict(dx=P[4] + 2), dict(w=P[3] + 2), dict(dw=P[5] + 1),
                dict(work=P[6] + 2)):
        assert call(**bad) == ALIGN, bad
    assert call(k=0) == OK and call(rows=0, dw=None) == OK


def test_binding_refusals():
    x = torch.zeros(4, 200)
    c, s = ff.i8_empty(4, 200, device="cpu")
    out = torch.zeros(4, 6)
    bad = [
        (TypeError, "x: expected a torch tensor", lambda: ff.i8_quantize(np.zeros((4, 200), np.float32), c, s)),
        (ValueError, "x: dtype", lambda: ff.i8_quantize(x.double(), c, s)),
        (ValueError, "row are not contiguous", lambda: ff.i8_quantize(x.t(), c, s)),
        (ValueError, "codes: dtype", lambda: ff.i8_quantize(x, c.byte(), s)),
        (ValueError, "codes: holds", lambda: ff.i8_quantize(x, c[:3], s)),
        (ValueError, "codes: has rows of 200 bytes", lambda: ff.i8_quantize(x, torch.zeros(6, 200, dtype=torch.int8), s)),
        (ValueError, "scales: holds", lambda: ff.i8_quantize(x, c, s[:3])),
        (ValueError, "not in GPU memory", lambda: ff.i8_quantize(x, c, s)),
        (ValueError, "not in GPU memory", lambda: ff.i8_dequantize(c, s, x)),
        (ValueError, "a: holds", lambda: ff.i8_matmul(c, s, *ff.i8_empty(6, 200, device="cpu"), torch.zeros(5, 6), 200)),
        (ValueError, "b: has rows of 256", lambda: ff.i8_matmul(*ff.i8_empty(4, 300, device="cpu"), *ff.i8_empty(12, 200, device="cpu"), out, 300)),
        (ValueError, "bias: holds", lambda: ff.i8_matmul(c, s, *ff.i8_empty(6, 200, device="cpu"), out, 200, bias=torch.zeros(5))),
        (ValueError, "not in GPU memory", lambda: ff.i8_matmul(c, s, *ff.i8_empty(6, 200, device="cpu"), out, 200)),
        (ValueError, "neither", lambda: ff.rms_norm(x, None)),
        (ValueError, "weight: holds", lambda: ff.rms_norm(x, torch.zeros(199), x)),
        (ValueError, "weight: dtype", lambda: ff.rms_norm(x, torch.zeros(200).half(), x)),
        (ValueError, "residual: is 4 x 100", lambda: ff.rms_norm(x, None, x, residual=torch.zeros(4, 100))),
        (ValueError, "residual: dtype", lambda: ff.rms_norm(x, None, x, residual=x.half())),
        (ValueError, "total: dtype", lambda: ff.rms_norm(x.half(), None, x.half(), residual=x.half(), total=x)),
        (ValueError, "out: dtype", lambda: ff.rms_norm(x.half(), None, x)),
        (TypeError, "scales", lambda: ff.rms_norm(x, None, codes=c)),
        (ValueError, "not in GPU memory", lambda: ff.rms_norm(x, None, x)),
        (ValueError, "work: dweight needs", lambda: ff.rms_norm_grad(x, x, None, x, torch.zeros(200))),
        (ValueError, "dtotal: dtype", lambda: ff.rms_norm_grad(x.half(), x, None, x, dtotal=x.half())),
        (ValueError, "dx: dtype", lambda: ff.rms_norm_grad(x.half(), x.half(), None, x)),
        (TypeError, "dx: expected", lambda: ff.rms_norm_grad(x, x, None, None)),
        (TypeError, "h: expected", lambda: ff.rms_norm_grad(x, None, None, x)),
        (ValueError, "not in GPU memory", lambda: ff.rms_norm_grad(x, x, None, x)),
    ]
    for error, text, call in bad:
        with pytest.raises(error, match=text):
            call()


def test_reference():
    """The 64-bit form's own corners: ties to even, the largest magnitude at 127, a row's end."""
    codes, scales = R.quantize([[1.0, 0.5, -0.5, 0.25, 0.0], [0.0] * 5, [np.inf, 1, 2, 3, 4]])
    assert codes[0, :5].tolist() == [127, 64, -64, 32, 0] and not codes[1:].any() and not codes[:, 5:].any()
    assert scales[0] == np.float32(1) / np.float32(127) and scales[1] == 0 and np.isnan(scales[2])
    v, _ = R.matmul(codes[:1], scales[:1], codes[:1], scales[:1], None, 5)
    assert abs(v[0, 0] - (127 ** 2 + 2 * 64 ** 2 + 32 ** 2) / 127 ** 2) < 1e-6
