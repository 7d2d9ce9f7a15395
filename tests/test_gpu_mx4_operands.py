"""GPU tests of the 4-bit calls' operands in blocks, through the native binding: rows of another
length are refused, flat arrays give the same as rows."""
import pytest

import mx4_reference as R
from test_gpu_mx4 import random_blocks, to_dev
from test_mx4_operands import wrong_operands

pytestmark = pytest.mark.gpu


def test_rows_of_another_length_are_refused(dev):
    for name, call in wrong_operands(dev):
        with pytest.raises(ValueError, match=f"^{name}: has rows of"):
            call()


def test_flat_arrays_and_rows_to_spare(dev, rng):
    import torch
    import fufft_amd as ff
    m, n, k = 5, 40, 200
    x = torch.randn(m, k, device=dev)
    w = to_dev(dev, *random_blocks(rng, n, k))
    flat = [t.reshape(-1) for t in w]
    more = [torch.cat((t, t[:3])) for t in w]
    want = torch.empty(m, n, device=dev)
    ff.mx4_linear(x, *w, want)
    for other in (flat, more):
        out = torch.empty(m, n, device=dev)
        ff.mx4_linear(x, *other, out)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    kp = R.padded(k)
    q, f = ff.mx4_empty(m, k), (torch.empty(m * kp // 2, dtype=torch.uint8, device=dev),
                                torch.empty(m * kp // 32, dtype=torch.uint8, device=dev))
    ff.mx4_quantize(x, *q)
    ff.mx4_quantize(x, *f)
    torch.cuda.synchronize()
    assert torch.equal(q[0].view(-1), f[0]) and torch.equal(q[1].view(-1), f[1])
