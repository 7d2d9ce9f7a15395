"""How near the decaying-attention calls come to the 64-bit recurrence over a whole head, and what
keeps fewer bits than they promise.  CPU only.

Element by element a bound has to allow for all terms of a sum being off the same way (layer_reference.py),
which for a slowly decaying head is a large part of the result itself.  Over a head the terms' own
roundings, 2^-17 of each and independent, all but vanish, and what is left is the rounding of
the result to its type.  So the distance to the 64-bit result, over a head, may be MARGIN times that of
the 64-bit result rounded to the type: with an error before the rounding of x of the rounding's own size the
distance is sqrt(1 + x^2) times it, so that 1.1 allows x = 0.45, and the some hundreds of
independent roundings and more that a head has here move it by 2 % (0.9 / sqrt(n) of the square).  One rounding to bf16 of the state or
of the scores of a bf16 call has x near 0.7 where that part makes half of the results, 1 where it makes them all."""
import numpy as np

import layer_reference as R

MARGIN = 1.1


def rounded(x, kind):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x)).to(R.torch_type(kind)).double().numpy()


def excess(got, want, kind):
    """||got - want|| over a head in units of ||want rounded - want||."""
    return np.linalg.norm(np.asarray(got) - want) / np.linalg.norm(rounded(want, kind) - want)


def parts(x, n):
    """x in 64 bits as the sum of n bf16 parts."""
    total, left = np.zeros_like(x), x
    for _ in range(n):
        p = rounded(left, "bf16")
        total, left = total + p, left - p
    return total


def emulated(q, k, v, log_decay, state=2, scores=2, keys=2, carried=None):
    """One head in chunks of 64 tokens, in 64 bits but for what is held in that many bf16 parts: the
    state that q meets, weighted scores, weighted keys, and the state carried from chunk to chunk."""
    a = np.exp(np.float64(log_decay))
    tokens, dk = q.shape
    s, out = np.zeros((dk, v.shape[1])), np.zeros((tokens, v.shape[1]))
    for t0 in range(0, tokens, 64):
        Q, K, V = q[t0:t0 + 64], k[t0:t0 + 64], v[t0:t0 + 64]
        n = len(Q)
        i = np.arange(n)
        weights = np.where(i[:, None] >= i, a ** np.maximum(i[:, None] - i, 0), 0.0)
        out[t0:t0 + n] = a ** (i + 1)[:, None] * (Q @ parts(s, state)) + parts((Q @ K.T) * weights, scores) @ V
        s = a ** n * s + parts(K * (a ** (n - 1 - i))[:, None], keys).T @ V
        if carried:
            s = parts(s, carried)
    return out
