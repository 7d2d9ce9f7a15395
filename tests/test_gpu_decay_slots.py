"""GPU tests of decay_attention_step with many sequences: slots in any order, places without a sequence, and the
same slot twice, hundreds of places apart."""
import numpy as np
import pytest

import layer_reference as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch,heads,dk,dv", [(300, 3, 16, 12), (1000, 2, 8, 32), (700, 1, 33, 7), (777, 2, 64, 64)])
@pytest.mark.parametrize("kind", R.TYPES)
def test_many_slots(dev, rng, batch, heads, dk, dv, kind):
    import torch
    import fufft_amd as ff
    print(f"case decay_step slots {batch} {heads} {dk}x{dv} {kind}", flush=True)
    count = batch + 40
    slots = rng.permutation(count)[:batch]
    slots[5::50] = -1
    slots[7::90] = count + rng.integers(0, 3, len(slots[7::90])) * (1 << 33)
    for first, second in ((0, 256), (1, 257), (2, 299), (3, 258), (3, 280), (20, 21), (batch - 2, batch - 1), (4, batch - 3), (255, 256)):
        slots[second] = slots[first]
    seen, wins = set(), np.zeros(batch, dtype=bool)
    for b, at in enumerate(slots):
        wins[b] = 0 <= at < count and at not in seen
        seen.add(int(at))
    q, q64 = R.typed(rng.standard_normal((batch, heads, dk)), kind, dev)
    k, k64 = R.typed(rng.standard_normal((batch, heads, dk)), kind, dev)
    v, v64 = R.typed(rng.standard_normal((batch, heads, dv)), kind, dev)
    g = rng.uniform(-2, 0, heads).astype(np.float32)
    s0 = rng.standard_normal((count, heads, dk, dv)).astype(np.float32)
    state, out = torch.from_numpy(s0).to(dev), torch.full_like(v, 5.0)
    ff.decay_attention_step(q, k, v, torch.from_numpy(g).to(dev), state, out, slots=torch.from_numpy(slots.astype(np.int64)).to(dev), scale=0.5)
    got = state.double().cpu().numpy()
    a = np.exp(g.astype(np.float64))[:, None, None]
    for b in np.flatnonzero(wins):
        old = s0[slots[b]].astype(np.float64)
        kv = k64[b][:, :, None] * v64[b][:, None, :]
        new, mag = a * old + kv, a * np.abs(old) + np.abs(kv)
        assert np.all(np.abs(got[slots[b]] - new) <= 6 * R.EPS24 * mag + 2.0 ** -126), b     # the power, its product, the key's and the sum
        want, terms = (q64[b][:, :, None] * new).sum(1), (np.abs(q64[b])[:, :, None] * mag).sum(1)
        assert R.inside(out[b], 0.5 * want, 0.5 * terms * (dk + 10) * R.EPS24), b
    assert not out[torch.from_numpy(~wins).to(dev)].any()
    untouched = np.setdiff1d(np.arange(count), slots[wins])
    assert np.array_equal(got[untouched], s0[untouched].astype(np.float64))
