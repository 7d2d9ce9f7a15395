"""CPU tests of the microscaled 4-bit calls: what the C ABI and the Python binding refuse
before anything is launched, and the 64-bit form that the GPU tests compare with."""
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

import fufft_amd as ff
import mx4_reference as R

INV, ALIGN, OK = ff.ERR_INVALID, ff.ERR_ALIGN, ff.OK
P = [0x10000000 * (i + 1) for i in range(12)]          # addresses that are checked and never read


def u8(*shape):
    return torch.zeros(*shape, dtype=torch.uint8)


def test_padded():
    assert [ff.mx4_padded(k) for k in (0, 1, 127, 128, 129)] == [0, 128, 128, 128, 256]
    assert [ff.lib.fufft_mx4_padded(k) for k in (0, 1, 127, 128, 129, -1)] == [0, 128, 128, 128, 256, INV]
    codes, scales = ff.mx4_empty(3, 130, device="cpu")
    assert codes.shape == (3, 128) and scales.shape == (3, 8)


def quantize(x=P[0], type=0, ld=256, rows=4, k=200, rule=0, rand=None, c=P[1], s=P[2], ct=None, st=None):
    return ff.lib.fufft_mx4_quantize(x, type, ld, rows, k, rule, rand, c, s, ct, st, None)


def test_quantize_refusals():
    for bad in (dict(type=3), dict(type=-1), dict(ld=199), dict(rows=-1), dict(k=-1), dict(k=1 << 62), dict(rule=2),
                dict(x=None), dict(c=None), dict(s=None), dict(c=None, s=None), dict(ct=P[3]), dict(st=P[3]),
                dict(c=P[0]), dict(s=P[0] + 4 * (3 * 256 + 196)), dict(s=P[1] + 16), dict(ct=P[1], st=P[4]),
                dict(ct=P[3], st=P[2]), dict(rand=P[1], type=1)):
        assert quantize(**bad) == INV, bad
    for bad in (dict(c=P[1] + 8), dict(s=P[2] + 2), dict(x=P[0] + 2), dict(x=P[0] + 1, type=1),
                dict(ct=P[3] + 4, st=P[4]), dict(ct=P[3], st=P[4] + 1)):
        assert quantize(**bad) == ALIGN, bad
    assert quantize(rows=0) == OK and quantize(k=0) == OK and quantize(x=None, rows=0, c=None, s=None) == OK


def test_dequantize_refusals():
    def call(c=P[0], s=P[1], o=P[2], type=0, ld=200, rows=4, k=200):
        return ff.lib.fufft_mx4_dequantize(c, s, o, type, ld, rows, k, None)
    for bad in (dict(c=None), dict(s=None), dict(o=None), dict(type=7), dict(ld=100), dict(rows=-2), dict(o=P[0] + 16)):
        assert call(**bad) == INV, bad
    for bad in (dict(c=P[0] + 1), dict(s=P[1] + 1), dict(o=P[2] + 1)):
        assert call(**bad) == ALIGN, bad
    assert call(rows=0) == OK


def test_matmul_refusals():
    def call(a=P[0], sa=P[1], b=P[2], sb=P[3], bias=P[4], o=P[5], type=0, ld=8, m=4, n=8, k=64):
        return ff.lib.fufft_mx4_matmul(a, sa, b, sb, bias, o, type, ld, m, n, k, None)
    for bad in (dict(a=None), dict(sa=None), dict(b=None), dict(sb=None), dict(o=None), dict(type=3), dict(ld=7),
                dict(m=-1), dict(n=-1), dict(k=-1), dict(m=1 << 40, k=1 << 40), dict(o=P[0]), dict(o=P[4] + 4),
                dict(o=P[3] - 32)):
        assert call(**bad) == INV, bad
    for bad in (dict(a=P[0] + 8), dict(b=P[2] + 8), dict(sa=P[1] + 1), dict(sb=P[3] + 2), dict(bias=P[4] + 2),
                dict(o=P[5] + 2)):
        assert call(**bad) == ALIGN, bad
    assert call(m=0) == OK and call(n=0) == OK


def test_linear_refusals():
    def call(x=P[0], xt=1, ldx=64, w=P[1], sw=P[2], bias=None, o=P[3], type=0, ld=8, m=4, n=8, k=64):
        return ff.lib.fufft_mx4_linear(x, xt, ldx, w, sw, bias, o, type, ld, m, n, k, None)
    for bad in (dict(x=None), dict(xt=3), dict(ldx=63), dict(w=None), dict(sw=None), dict(o=None), dict(type=-1),
                dict(ld=7), dict(m=-1), dict(o=P[0] + 4), dict(o=P[1])):
        assert call(**bad) == INV, bad
    for bad in (dict(x=P[0] + 1), dict(w=P[1] + 4), dict(sw=P[2] + 2), dict(o=P[3] + 1)):
        assert call(**bad) == ALIGN, bad
    assert call(m=0) == OK and call(n=0) == OK


def test_cache_refusals():
    def write(x=P[0], type=0, ld=64, slots=P[1], rows=4, ch=64, c=P[2], s=P[3], count=32):
        return ff.lib.fufft_mx4_cache_write(x, type, ld, slots, rows, ch, c, s, count, None)
    for bad in (dict(x=None), dict(slots=None), dict(c=None), dict(s=None), dict(type=3), dict(ld=63), dict(rows=-1),
                dict(count=-1), dict(c=P[0]), dict(s=P[2] + 64), dict(c=P[1] - 16)):
        assert write(**bad) == INV, bad
    for bad in (dict(x=P[0] + 2), dict(slots=P[1] + 4), dict(c=P[2] + 8), dict(s=P[3] + 1)):
        assert write(**bad) == ALIGN, bad
    assert write(rows=0) == OK and write(count=0) == OK

    def read(c=P[0], s=P[1], pages=8, page=16, ch=64, t=P[2], w=4, l=P[3], b=2, n=50, o=P[4], type=0, order=0):
        return ff.lib.fufft_mx4_cache_read(c, s, pages, page, ch, t, w, l, b, n, o, type, order, None)
    for bad in (dict(c=None), dict(s=None), dict(t=None), dict(l=None), dict(o=None), dict(page=0), dict(page=12),
                dict(page=1 << 17), dict(pages=-1), dict(w=-1), dict(b=-1), dict(n=-1), dict(type=3), dict(order=2),
                dict(o=P[0]), dict(o=P[2] + 4), dict(o=P[3] + 4)):
        assert read(**bad) == INV, bad
    for bad in (dict(c=P[0] + 4), dict(s=P[1] + 2), dict(t=P[2] + 2), dict(l=P[3] + 1), dict(o=P[4] + 2)):
        assert read(**bad) == ALIGN, bad
    assert read(b=0) == OK and read(n=0) == OK and read(ch=0) == OK

    def conv(c=P[0], s=P[1], pages=8, page=16, ch=64, t=P[2], w=4, l=P[3], b=2, h=P[4], ht=0, n=50, o=P[5], type=0,
             work=P[6], splits=3):
        return ff.lib.fufft_mx4_cache_conv(c, s, pages, page, ch, t, w, l, b, h, ht, n, o, type, work, splits, None)
    for bad in (dict(c=None), dict(s=None), dict(t=None), dict(l=None), dict(h=None), dict(o=None), dict(page=3),
                dict(ht=4), dict(type=3), dict(n=-1), dict(splits=-1), dict(work=None), dict(type=1, splits=0, work=None),
                dict(o=P[4]), dict(o=P[6]), dict(work=P[0]), dict(work=P[4] + 4)):
        assert conv(**bad) == INV, bad
    for bad in (dict(c=P[0] + 4), dict(h=P[4] + 1), dict(o=P[5] + 1), dict(work=P[6] + 2)):
        assert conv(**bad) == ALIGN, bad
    assert conv(b=0) == OK and conv(ch=0) == OK


def test_binding_refusals():
    x = torch.zeros(4, 200)
    c, s = ff.mx4_empty(4, 200, device="cpu")
    with pytest.raises(TypeError, match="x: expected a torch tensor"):
        ff.mx4_quantize(np.zeros((4, 200), np.float32), c, s)
    with pytest.raises(ValueError, match="x: dtype"):
        ff.mx4_quantize(x.double(), c, s)
    with pytest.raises(ValueError, match="matrix"):
        ff.mx4_quantize(x[0], c, s)
    with pytest.raises(ValueError, match="row are not contiguous"):
        ff.mx4_quantize(x.t(), c, s)
    with pytest.raises(ValueError, match="rows overlap"):
        ff.mx4_quantize(torch.zeros(200).expand(4, 200), c, s)
    with pytest.raises(ValueError, match="neither"):
        ff.mx4_quantize(x)
    with pytest.raises(ValueError, match="codes: holds"):
        ff.mx4_quantize(x, c[:3], s)
    with pytest.raises(ValueError, match="codes_scales: holds"):
        ff.mx4_quantize(x, c, s[:3])
    with pytest.raises(TypeError, match="codes_scales"):
        ff.mx4_quantize(x, c)
    with pytest.raises(ValueError, match="codes_t: holds"):
        ff.mx4_quantize(x, None, None, u8(199, 64), u8(200, 4))
    with pytest.raises(ValueError, match="rand: holds"):
        ff.mx4_quantize(x, c, s, rand=u8(799))
    with pytest.raises(ValueError, match="not in GPU memory"):
        ff.mx4_quantize(x, c, s)
    with pytest.raises(ValueError, match="not in GPU memory"):
        ff.mx4_dequantize(c, s, x)
    with pytest.raises(ValueError, match="b: holds"):
        ff.mx4_matmul(c, s, c, s, torch.zeros(4, 5), 200)
    with pytest.raises(ValueError, match="bias: holds"):
        ff.mx4_matmul(c, s, c, s, torch.zeros(4, 4), 200, bias=torch.zeros(3))
    with pytest.raises(ValueError, match="out: 3 rows"):
        ff.mx4_linear(x, c, s, torch.zeros(3, 4))
    with pytest.raises(ValueError, match="w: holds"):
        ff.mx4_linear(x, c, s, torch.zeros(4, 5))
    cc, cs = u8(6, 16, 128), u8(6, 16, 8)
    table, lens, out = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(2, 48, 200)
    with pytest.raises(ValueError, match="codes: expected"):
        ff.mx4_cache_write(x, torch.zeros(4, dtype=torch.int64), cc[:, :, :64].contiguous(), cs)
    with pytest.raises(ValueError, match="slots: dtype"):
        ff.mx4_cache_write(x, torch.zeros(4, dtype=torch.int32), cc, cs)
    with pytest.raises(ValueError, match="slots: holds"):
        ff.mx4_cache_write(x, torch.zeros(3, dtype=torch.int64), cc, cs)
    with pytest.raises(ValueError, match="power of two"):
        ff.mx4_cache_write(x, torch.zeros(4, dtype=torch.int64), cc[:, :12].contiguous(), cs[:, :12].contiguous())
    with pytest.raises(ValueError, match="order must be"):
        ff.mx4_cache_read(cc, cs, table, lens, out, order="rows")
    with pytest.raises(ValueError, match="pages and lens"):
        ff.mx4_cache_read(cc, cs, table, lens[:1], out)
    with pytest.raises(ValueError, match="pages: dtype"):
        ff.mx4_cache_read(cc, cs, table.long(), lens, out)
    with pytest.raises(ValueError, match="2 sequences"):
        ff.mx4_cache_read(cc, cs, table, lens, out[:1])
    with pytest.raises(ValueError, match="not contiguous"):
        ff.mx4_cache_read(cc, cs, table, lens, out[:, ::2])
    taps = torch.zeros(48, 200)
    with pytest.raises(ValueError, match="channels"):
        ff.mx4_cache_conv(cc, cs, table, lens, taps, torch.zeros(2, 100))
    with pytest.raises(ValueError, match="workspace"):
        ff.mx4_cache_conv(cc, cs, table, lens, taps, torch.zeros(2, 200, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="taps and out"):
        ff.mx4_cache_conv(cc, cs, table, lens, torch.zeros(48, 400)[:, :200], torch.zeros(2, 200))
    with pytest.raises(ValueError, match="work: dtype"):
        ff.mx4_cache_conv(cc, cs, table, lens, taps, torch.zeros(2, 200), work=torch.zeros(4, 2, 200).half())
    with pytest.raises(ValueError, match="rule must be"):
        ff.mx4_quantize(x, c, s, rule="nearest")


@pytest.mark.parametrize("rule", ["fit", "floor"])
def test_reference_definition(rule):
    """The 64-bit form itself: scales by search over every power, codes by search over the grid."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((8, 64)) * 10.0 ** rng.uniform(-20, 20, (8, 1))
    x[0, :32] = 0
    codes, scales = R.quantize(x, rule)
    back = R.values(codes, scales, 64)
    for r in range(8):
        for b in range(2):
            v = x[r, 32 * b:32 * b + 32]
            top = np.abs(v).max()
            powers = 2.0 ** (np.arange(255) - 127.0)
            if top == 0:
                assert scales[r, b] == 0
                continue
            p = powers[scales[r, b]]
            if rule == "fit":
                assert scales[r, b] == np.argmax(top <= 6 * powers)
            else:
                assert 4 * p <= top < 8 * p
            for i in range(32):
                near = min(R.GRID, key=lambda g: abs(abs(v[i]) - g * p)) * p
                assert abs(abs(back[r, 32 * b + i]) - near) == 0 or \
                    abs(abs(abs(v[i]) - near) - abs(abs(v[i]) - abs(back[r, 32 * b + i]))) < 1e-12 * p


def test_cpp_header(tmp_path):
    """The 4-bit part of include/fufft/fufft.hpp: built with g++ and run without a GPU."""
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    root = Path(__file__).resolve().parent.parent
    exe, lib = tmp_path / "mx4_hpp_check", root / "fufft_amd"
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", f"-I{root / 'include'}",
                    str(root / "tests" / "cpp" / "mx4_hpp_check.cpp"), f"-L{lib}", "-lfufft_amd", f"-Wl,-rpath,{lib}",
                    "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], timeout=60).returncode == 0
