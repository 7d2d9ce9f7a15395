"""GPU test: mx4_linear reads its rows from some columns of an array and writes others of it."""
import pytest

from test_gpu_mx4 import TYPES, random_blocks, to_dev, torch_type

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,k", [(1, 40, 200), (3, 40, 200), (40, 33, 130)])
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("first", ["x", "out"])
def test_linear_within_one_array(dev, rng, m, n, k, kind, first):
    import torch
    import fufft_amd as ff
    w = to_dev(dev, *random_blocks(rng, n, k))
    both = torch.randn(m, n + k + 1, device=dev).to(torch_type(kind))
    x, out = (both[:, :k], both[:, k + 1:]) if first == "x" else (both[:, n + 1:], both[:, :n])
    gap = both[:, k].clone() if first == "x" else both[:, n].clone()
    before, want = x.clone(), torch.empty(m, n, dtype=both.dtype, device=dev)
    ff.mx4_linear(before, *w, want)
    ff.mx4_linear(x, *w, out)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(x, before)
    assert torch.equal(both[:, k] if first == "x" else both[:, n], gap)
    with pytest.raises(ff.FufftError):                  # a column that both have
        ff.mx4_linear(x, *w, both[:, k - 1:k - 1 + n] if first == "x" else both[:, 2:2 + n])
