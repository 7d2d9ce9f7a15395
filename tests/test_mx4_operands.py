"""CPU tests of the 4-bit calls' operands in blocks: a pair whose rows have another length than the
call's, made for other sizes, is refused, as its rows would be read at the wrong places; a flat
array is rows of the call's length."""
import pytest
import torch

import fufft_amd as ff


def wrong_operands(dev):
    """(call, what it names) for every operand in blocks, and the random bytes, with rows of another
    length but bytes enough."""
    e = lambda rows, k: ff.mx4_empty(rows, k, device=dev)                   # noqa: E731
    f = lambda *shape: torch.zeros(*shape, device=dev)                      # noqa: E731
    u8 = lambda *shape: torch.zeros(*shape, dtype=torch.uint8, device=dev)  # noqa: E731
    x, (c, s), (wide_c, wide_s) = f(6, 256), e(6, 256), e(6, 512)
    t, wide_t = e(256, 6), e(256, 200)
    for name, call in (
            # a weight of 512 values a row to rows of 256
            ("w", lambda: ff.mx4_linear(x, wide_c, s, f(6, 6))),
            ("w_scales", lambda: ff.mx4_linear(x, c, wide_s, f(6, 6))),
            # a product over fewer values than the operands have
            ("a", lambda: ff.mx4_matmul(wide_c, wide_s, wide_c, wide_s, f(6, 6), 256)),
            ("a_scales", lambda: ff.mx4_matmul(c, wide_s, c, s, f(6, 6), 256)),
            ("b", lambda: ff.mx4_matmul(c, s, wide_c, s, f(6, 6), 256)),
            ("b_scales", lambda: ff.mx4_matmul(c, s, c, wide_s, f(6, 6), 256)),
            # values read back into a narrower matrix
            ("codes", lambda: ff.mx4_dequantize(wide_c, wide_s, f(6, 100))),
            ("codes_scales", lambda: ff.mx4_dequantize(c, wide_s, f(6, 256))),
            # quantising
            ("codes", lambda: ff.mx4_quantize(x, wide_c, s)),
            ("codes_scales", lambda: ff.mx4_quantize(x, c, wide_s)),
            ("codes", lambda: ff.mx4_quantize(x, c.view(3, 256), s)),
            ("codes_t", lambda: ff.mx4_quantize(x, None, None, wide_t[0], t[1])),
            ("codes_t_scales", lambda: ff.mx4_quantize(x, c, s, t[0], wide_t[1])),
            ("rand", lambda: ff.mx4_quantize(x, c, s, rand=u8(6, 264))),
            ("rand", lambda: ff.mx4_quantize(x, c, s, rand=u8(256, 6)))):
        yield name, call


def test_rows_of_another_length_are_refused():
    for name, call in wrong_operands("cpu"):
        with pytest.raises(ValueError, match=f"^{name}: has rows of"):
            call()


def test_flat_arrays_and_nothing_pass():
    """Up to the check of the device, the last one."""
    x, (c, s) = torch.zeros(6, 256), ff.mx4_empty(6, 256, device="cpu")
    more = torch.zeros(10, 128, dtype=torch.uint8), torch.zeros(10, 8, dtype=torch.uint8)       # rows to spare
    none = ff.mx4_empty(6, 512, device="cpu")
    for call in (lambda: ff.mx4_quantize(x, c.view(-1), s.view(-1)),
                 lambda: ff.mx4_quantize(x, *more),
                 lambda: ff.mx4_quantize(x, c, s, rand=torch.zeros(6 * 256 + 5, dtype=torch.uint8)),
                 lambda: ff.mx4_dequantize(torch.zeros(5000, dtype=torch.uint8), s.view(-1), x),
                 lambda: ff.mx4_matmul(c.view(2, 3, 128), s.view(2, 3, 8), *more, torch.zeros(6, 10), 256),
                 lambda: ff.mx4_matmul(*none, *none, torch.zeros(6, 6), 0)):                   # nothing of them is read
        with pytest.raises(ValueError, match="not in GPU memory"):
            call()
