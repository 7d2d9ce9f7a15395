"""GPU tests of norms and 8-bit rows whose results take 16 MiB and more, which are stored past the L2: bit for
bit what the same rows give in parts of less, between columns that stay as they were."""
import pytest

import layer_reference as R

pytestmark = pytest.mark.gpu

MIB16 = 1 << 24


def odd_rows(rows, k, dtype, dev, extra=3):
    """rows x k with an odd leading dimension for odd k, from the second row's place and one element on; and all of it."""
    import torch
    ld = k + extra + (k + extra + 1) % 2
    flat = torch.full(((rows + 2) * ld,), 7.0, dtype=dtype, device=dev)
    return flat, flat[ld + 1:].as_strided((rows, k), (ld, 1))


def gaps_kept(flat, view):
    import torch
    keep = torch.ones_like(flat, dtype=torch.bool)
    keep.as_strided(view.shape, view.stride(), view.storage_offset()).fill_(False)
    return bool((flat[keep] == 7).all())


# a kernel's width each, odd ones; the codes alone pass 16 MiB from the second on
SIZES = [(450000, 20), (150000, 101), (33000, 511), (17000, 1001), (8200, 2047), (4200, 4101), (2200, 8001), (1100, 16101), (520, 32701), (430, 40001)]


@pytest.mark.parametrize("rows,k", SIZES)
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_past_the_l2(dev, rows, k, kind):
    import torch
    import fufft_amd as ff
    print(f"case past L2 {rows}x{k} {kind}", flush=True)
    t = R.torch_type(kind)
    _, x = odd_rows(rows, k, t, dev)
    x.copy_(torch.randn(rows, k, device=dev))
    x[::7, 1] = float("nan")
    w = torch.randn(k, device=dev)
    part = min(rows, (MIB16 - 1) // (R.padded(k) + 2 * k))
    assert rows > part and rows * k * 2 >= MIB16 and (k < 101 or rows * R.padded(k) >= MIB16)

    def same(small, rows_of):
        """rows_of(i, j): rows i .. j - 1 of the results of all; small(i, j): what these rows give by themselves"""
        for i in range(0, rows, part):
            j = min(rows, i + part)
            for a, b in zip(rows_of(i, j), small(i, j)):
                assert torch.equal(torch.nan_to_num(a, nan=99.0), torch.nan_to_num(b, nan=99.0)), (i, j)

    flat, out = odd_rows(rows, k, t, dev)
    codes, scales = ff.i8_empty(rows, k)

    def in_parts(i, j):
        o, (c, s) = torch.empty(j - i, k, dtype=t, device=dev), ff.i8_empty(j - i, k)
        ff.rms_norm(x[i:j], w, o, codes=c, scales=s)
        return o, c, s
    for with_out, with_codes in ((True, False), (False, True), (True, True)):
        flat.fill_(7.0), codes.fill_(99), scales.fill_(99.0)
        ff.rms_norm(x, w, out if with_out else None, codes=codes if with_codes else None, scales=scales if with_codes else None)
        pick = [p for p, there in zip(range(3), (with_out, with_codes, with_codes)) if there]
        same(lambda i, j: [in_parts(i, j)[p] for p in pick], lambda i, j: [(out, codes, scales)[p][i:j] for p in pick])
        assert gaps_kept(flat, out)
    # to 8 bits and back
    codes.fill_(99)
    ff.i8_quantize(x, codes, scales)

    def quantized(i, j):
        c, s = ff.i8_empty(j - i, k)
        ff.i8_quantize(x[i:j], c, s)
        return c, s
    same(quantized, lambda i, j: (codes[i:j], scales[i:j]))
    flat.fill_(7.0)
    ff.i8_dequantize(codes, scales, out)

    def back(i, j):
        o = torch.empty(j - i, k, dtype=t, device=dev)
        ff.i8_dequantize(codes[i:j], scales[i:j], o)
        return (o,)
    same(back, lambda i, j: (out[i:j],))
    assert gaps_kept(flat, out)
