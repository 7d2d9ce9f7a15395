"""GPU tests of 8-bit products whose scales are far apart: the result lies in the type's range where a sum
times one scale alone does not."""
import numpy as np
import pytest

import layer_reference as R

pytestmark = pytest.mark.gpu

# (scales of a, scales of b): their products, times sums of some 10^6, stay within fp32 and bf16
FAR = [(1e33, 1e-33), (1e-33, 1e33), (8e30, 1e-5), (3e38, 1e-44), (1e-40, 1e30), (2.0 ** 64, 2.0 ** -100), (1e-3, 1e-3)]


# a kernel each for few tokens, few rows, tiles of 64, 128 and 256
@pytest.mark.parametrize("m,n,k", [(1, 50, 700), (4, 50, 700), (8, 90, 1030), (16, 130, 520), (300, 150, 200), (2100, 2100, 128), (4000, 4090, 128)])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_scales_far_apart(dev, rng, m, n, k, kind):
    import torch
    import fufft_amd as ff
    print(f"case i8_matmul scales {m}x{n}x{k} {kind}", flush=True)
    a, b = (np.zeros((r, R.padded(k)), dtype=np.int8) for r in (m, n))
    a[:, :k], b[:, :k] = rng.integers(-127, 128, (m, k)), rng.integers(-127, 128, (n, k))
    da, db = torch.from_numpy(a).to(dev), torch.from_numpy(b).to(dev)
    sums = (da.double() @ db.double().t().contiguous()).cpu().numpy()           # exact below 2^53
    far = FAR[:2] if m * n > 1 << 20 else FAR
    for large, small in far:
        sa = (rng.uniform(0.5, 1, m) * large).astype(np.float32)
        sb = (rng.uniform(0.5, 1, n) * small).astype(np.float32)
        sa[::3] *= -1
        sa[1::7] = 1.0                          # ordinary rows among them
        sa[2::7] = 0.0
        for bias in (None, rng.standard_normal(n).astype(np.float32)):
            out = torch.empty(m, n, dtype=R.torch_type(kind), device=dev)
            ff.i8_matmul(da, torch.from_numpy(sa).to(dev), db, torch.from_numpy(sb).to(dev), out, k,
                         bias=None if bias is None else torch.from_numpy(bias).to(dev))
            v = sums * sa.astype(np.float64)[:, None] * sb.astype(np.float64)
            want = v if bias is None else v + bias
            # four fp32 roundings, and below the normal numbers half their step
            err = R.EPS24 * (3.001 * np.abs(v) + 1.001 * np.abs(want))
            ok = np.abs(want) < 3e38
            got = torch.where(torch.from_numpy(ok).to(dev), out, torch.zeros_like(out))
            assert R.inside(got, np.where(ok, want, 0), np.where(ok, err, 0)), (large, small)
            # beyond the range: infinities of the sign
            assert bool((out.double().cpu().numpy()[np.abs(want) > 3.5e38] == np.sign(want[np.abs(want) > 3.5e38]) * np.inf).all())
