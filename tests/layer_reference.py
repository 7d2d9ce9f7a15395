"""Plain 64-bit forms of the norm, 8-bit and decaying-attention calls, from their definitions,
and the bounds that fp32 arithmetic with one rounding at the end can keep.  CPU only."""
import numpy as np

EPS24 = 2.0 ** -24          # half a step of fp32, relative
TYPES = ("f32", "bf16", "f16")


def torch_type(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def typed(x, name, dev):
    """x rounded to the type: the tensor on the GPU, and its values in 64 bits."""
    import torch
    t = torch.from_numpy(np.ascontiguousarray(x)).to(torch_type(name))
    return t.to(dev), t.double().numpy()


def with_stride(t, extra=5, offset=3):
    """The same matrix as rows of a wider one, its first element `offset` elements in."""
    import torch
    rows, k = t.shape
    wide = torch.full((rows * (k + extra) + offset,), float("nan"), dtype=t.dtype, device=t.device)
    v = wide[offset:].view(rows, k + extra)[:, :k]
    v.copy_(t)
    return v


def padded(k):
    return -(-k // 128) * 128


def inside(got, want, err):
    """Whether every element of the tensor `got` is one that a value within err of `want` gives
    when it is rounded to got's type (rounding keeps the order, so the ends tell)."""
    import torch
    err = err + 2.0 ** -126         # products below the smallest normal number may be anything that small
    lo, hi = (torch.from_numpy(np.asarray(want + d, dtype=np.float64)).to(got.dtype).double().numpy() for d in (-err, err))
    got = got.double().cpu().numpy()
    return bool(np.all((got >= lo) & (got <= hi)))


# ---- 8-bit rows ----------------------------------------------------------------------

def quantize(x):
    """(codes with padding, scales fp32) of the rows of x.  127 x / top is exact enough in 64 bits: x and
    top have 24 bits, so what is not half-way between integers is at least 2^-33 from it."""
    x = np.asarray(x, dtype=np.float64)
    rows, k = x.shape
    codes = np.zeros((rows, padded(k)), dtype=np.int8)
    scales = np.zeros(rows, dtype=np.float32)
    for r in range(rows):
        top = np.max(np.abs(x[r])) if k else 0.0
        if not np.isfinite(top):
            scales[r] = np.nan
        elif top > 0:
            scales[r] = np.float32(top) / np.float32(127)
            codes[r, :k] = np.rint(127 * x[r] / top).astype(np.int8)
    return codes, scales


def matmul(a, sa, b, sb, bias, k):
    """(value, bound of fp32's error): the integer sum exact, made fp32, times each scale, plus the
    bias: four roundings, three of them of the product."""
    s = a.astype(np.int64)[:, :k] @ b.astype(np.int64)[:, :k].T
    v = s * sa.astype(np.float64)[:, None] * sb.astype(np.float64)
    out = v if bias is None else v + bias
    return out, EPS24 * (3.001 * np.abs(v) + 1.001 * np.abs(out))


# ---- norms -----------------------------------------------------------------------------

# Roundings that the sum of a row's squares goes through at most: a lane adds up to 64 of them one
# after the other, a wavefront's lanes 6 times, 16 wavefronts; and one for the square.  All terms are
# positive, so the relative error of the sum is at most that many half steps, of its root half
# of it; mean, eps, root and reciprocal add four, h itself one.
CHAIN = 64 + 6 + 16 + 1
ROOT = CHAIN / 2 + 5


def norm(h, weight, eps):
    """(y, bound of fp32's relative error before the rounding to the type)."""
    h = np.asarray(h, dtype=np.float64)
    y = h / np.sqrt((h * h).mean(1, keepdims=True) + eps)
    return (y if weight is None else y * weight), (ROOT + 4) * EPS24


def norm_grad(dy, h, weight, dtotal, eps):
    """(dx, its bound, dweight, the sum of the magnitudes of its terms)."""
    dy, h = np.asarray(dy, dtype=np.float64), np.asarray(h, dtype=np.float64)
    k = h.shape[1]
    r = 1 / np.sqrt((h * h).mean(1, keepdims=True) + eps)
    n = h * r
    g = dy if weight is None else dy * weight
    dx = r * (g - n * (g * n).mean(1, keepdims=True))
    # the mean: its terms are off by ROOT + 3 roundings, their sum by CHAIN; then n, r, and the products
    err = EPS24 * ((ROOT + 6) * np.abs(r * g) + (CHAIN + 3 * ROOT + 12) * np.abs(r * n) * np.abs(g * n).sum(1, keepdims=True) / k)
    if dtotal is not None:
        dx = dx + dtotal
        err = err + EPS24 * np.abs(dx)
    terms = dy * n
    return dx, err, terms.sum(0), np.abs(terms).sum(0)


# ---- decaying attention --------------------------------------------------------------------

def mixed(q, k, v, log_decay, state=None, late=0):
    """One head, token by token: (out without a scale, state behind, and the same of the magnitudes of
    all terms).  late: the state given meets its first token undecayed, the one returned is decayed
    once more."""
    a = np.exp(np.float64(log_decay))
    tokens, dk = q.shape
    dv = v.shape[1]
    s = np.zeros((dk, dv)) if state is None else np.array(state, dtype=np.float64)
    m = np.abs(s)
    out, mags = np.zeros((tokens, dv)), np.zeros((tokens, dv))
    for t in range(tokens):
        if not (late and t == 0):
            s, m = (a * s, a * m) if a > 0 else (np.zeros_like(s), np.zeros_like(m))
        s = s + np.outer(k[t], v[t])
        m = m + np.outer(np.abs(k[t]), np.abs(v[t]))
        out[t], mags[t] = q[t] @ s, np.abs(q[t]) @ m
    if late and tokens:
        s, m = a * s, a * m
    return out, s, mags, m


def mixed_share(kind, tokens, dim, log_decay, carried=False):
    """The share of the magnitudes that the call's arithmetic may be off by, before the result's own rounding.
    fp32's part: sums of dim and of 64 terms a chunk, up to five products a term, the chunk's decay; powers whose exponent
    is off by its own rounding, 2^-23 of |log_decay| tokens.
    bf16: weighted scores are rounded once, at 2^-8, and so is the state that q meets; two bf16 parts of weighted keys leave 2^-16.
    fp16: two bf16 parts of a weight, of the state and of weighted keys each leave 2^-16, and a product of second parts that is left
    out 2^-16, so 2^-15 in the state and as much again where q meets it.
    A state that is returned (carried): three bf16 parts of weighted keys leave 2^-24, and the products of fp16's parts that
    are left out (second of values with third of keys) 2^-24 too."""
    chunks = tokens // 64 + 1
    decay = 0.0 if not np.isfinite(log_decay) else abs(log_decay)
    chain = dim + 64 + (64 * 5 + 4) * chunks + 12 + 4 * decay * (tokens + 1)
    if carried:
        return (chain + 3) * EPS24
    return chain * EPS24 + {"f32": 0.0, "bf16": 1.02 * 2.0 ** -8, "f16": 1.05 * 2.0 ** -14}[kind]


def attention(q, k, v, log_decay, state, lens, scale, kind):
    """(out, its bound, new state, its bound) of (batch, tokens, heads, dim) arrays; rows from lens on are zero."""
    batch, tokens, heads, dk = q.shape
    dv = v.shape[3]
    out, err = np.zeros((batch, tokens, heads, dv)), np.zeros((batch, tokens, heads, dv))
    new, nerr = np.zeros((batch, heads, dk, dv)), np.zeros((batch, heads, dk, dv))
    for b in range(batch):
        n = tokens if lens is None else min(max(int(lens[b]), 0), tokens)
        for h in range(heads):
            o, s, mo, ms = mixed(q[b, :n, h], k[b, :n, h], v[b, :n, h], log_decay[h], None if state is None else state[b, h])
            out[b, :n, h], new[b, h] = scale * o, s
            err[b, :n, h] = abs(scale) * mo * mixed_share(kind, n, dk, log_decay[h])
            nerr[b, h] = ms * mixed_share(kind, n, 0, log_decay[h], carried=True)
    return out, err, new, nerr


def attention_grad(do, q, k, v, log_decay, state, dnew, lens, scale, kind):
    """((dq, bound), (dk, bound), (dv, bound), (dstate, bound)), from the recurrence of D[t] = q[t] do[t]^T + a D[t + 1]."""
    batch, tokens, heads, dk = q.shape
    dv = v.shape[3]
    got = [(np.zeros(x.shape), np.zeros(x.shape)) for x in (q, k, v)] + [(np.zeros((batch, heads, dk, dv)), np.zeros((batch, heads, dk, dv)))]
    for b in range(batch):
        n = tokens if lens is None else min(max(int(lens[b]), 0), tokens)
        for h in range(heads):
            g = log_decay[h]
            Q, K, V, D = q[b, :n, h], k[b, :n, h], v[b, :n, h], do[b, :n, h]
            st = None if state is None else state[b, h].T
            dn = None if dnew is None else dnew[b, h]
            o, _, m, _ = mixed(D, V, K, g, st)
            got[0][0][b, :n, h], got[0][1][b, :n, h] = scale * o, abs(scale) * m * mixed_share(kind, n, dv, g)
            o, _, m, _ = mixed(V[::-1], scale * D[::-1], Q[::-1], g, None if dn is None else dn.T, 1)
            got[1][0][b, :n, h], got[1][1][b, :n, h] = o[::-1], m[::-1] * mixed_share(kind, n, dv, g)
            o, s, m, ms = mixed(K[::-1], scale * Q[::-1], D[::-1], g, dn, 1)
            got[2][0][b, :n, h], got[2][1][b, :n, h] = o[::-1], m[::-1] * mixed_share(kind, n, dk, g)
            got[3][0][b, h], got[3][1][b, h] = s, ms * mixed_share(kind, n, 0, g, carried=True)
    return got
