"""GPU tests of how near the decaying-attention calls come to the 64-bit recurrence over a whole head
(tests/decay_accuracy.py): results and gradients, tokens split and not, with and without the states."""
import numpy as np
import pytest

import decay_accuracy as A
import layer_reference as R

pytestmark = pytest.mark.gpu

DECAYS = np.array([0.0, -0.001, -0.02, -0.5], dtype=np.float32)


def near(got, want, kind, what):
    got = got.double().cpu().numpy()
    for b in range(want.shape[0]):
        for h in range(want.shape[2]):
            far = A.excess(got[b, :, h], want[b, :, h], kind)
            assert far < A.MARGIN, (what, b, h, far)


@pytest.mark.parametrize("tokens,dk,dv", [(70, 128, 128), (643, 64, 64), (300, 40, 100), (4100, 128, 128), (2500, 33, 65)])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_accuracy(dev, rng, tokens, dk, dv, kind):
    import torch
    import fufft_amd as ff
    print(f"case decay accuracy {tokens} {dk}x{dv} {kind}", flush=True)
    batch, heads = 1, len(DECAYS)
    ts, x64 = zip(*(R.typed(rng.standard_normal((batch, tokens, heads, d)), kind, dev) for d in (dk, dk, dv, dv)))
    q, k, v, do = ts
    g = torch.from_numpy(DECAYS).to(dev)
    state, dnew = (rng.standard_normal((batch, heads, dk, dv)).astype(np.float32) for _ in range(2))
    want = R.attention(x64[0], x64[1], x64[2], DECAYS, state, None, 0.125, kind)[0]
    grads = R.attention_grad(x64[3], x64[0], x64[1], x64[2], DECAYS, state, dnew, None, 0.125, kind)
    state, dnew = torch.from_numpy(state).to(dev), torch.from_numpy(dnew).to(dev)
    for splits in (0, 5, 64):
        work = torch.full((3 * splits, batch, heads, dk, dv), float("nan"), device=dev) if splits else None
        part = None if work is None else work[:splits]
        for behind in (None, torch.empty_like(state)):
            out = torch.empty_like(v)
            ff.decay_attention(q, k, v, g, out, state=state, new_state=behind, work=part, scale=0.125)
            near(out, want, kind, ("out", splits, behind is not None))
            got = [torch.empty_like(x) for x in (q, k, v)]
            ff.decay_attention_grad(do, q, k, v, g, *got, state=state, dnew_state=dnew, dstate=behind, work=work, scale=0.125)
            for x, (w, _), name in zip(got, grads, ("dq", "dk", "dv")):
                near(x, w, kind, (name, splits, behind is not None))
