"""CPU tests of the measure in tests/decay_accuracy.py: what the calls promise passes it, and what keeps fewer
bits does not."""
import numpy as np
import pytest

import decay_accuracy as A
import layer_reference as R


@pytest.mark.parametrize("log_decay", [0.0, -0.001, -0.02])
def test_fewer_bits_are_seen(log_decay):
    rng = np.random.default_rng(3)
    tokens, dk, dv = 1500, 64, 48
    q, k, v = (A.rounded(rng.standard_normal((tokens, d)), "bf16") for d in (dk, dk, dv))
    want = R.mixed(q, k, v, log_decay)[0]
    assert A.excess(A.rounded(want, "bf16"), want, "bf16") == 1.0
    promised = A.excess(A.rounded(A.emulated(q, k, v, log_decay), "bf16"), want, "bf16")
    assert promised < 1.01, promised
    assert A.excess(A.rounded(want * 1.005, "bf16"), want, "bf16") > A.MARGIN
    fewer = [dict(state=1), dict(state=1, scores=1), dict(carried=1)]
    if log_decay < 0:                       # else a weighted key is the key, which bf16 holds
        fewer += [dict(keys=1), dict(carried=1, keys=1)]
    if log_decay < -0.01:                   # elsewhere scores of the same chunk are a small part
        fewer.append(dict(scores=1))
    for less in fewer:
        seen = A.excess(A.rounded(A.emulated(q, k, v, log_decay, **less), "bf16"), want, "bf16")
        assert seen > A.MARGIN, (less, seen)
    # fp16's results have three bits more, and are held to as many more
    q, k, v = (A.rounded(rng.standard_normal((tokens, d)), "f16") for d in (dk, dk, dv))
    want = R.mixed(q, k, v, log_decay)[0]
    assert A.excess(A.rounded(A.emulated(q, k, v, log_decay), "f16"), want, "f16") < 1.05
    assert A.excess(A.rounded(A.emulated(q, k, v, log_decay, state=1), "f16"), want, "f16") > 2
