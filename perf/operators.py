"""The work that a long-convolution model gives the microscaled 4-bit calls: its layers'
matrix products in training and in serving, and the cache of signals that generation
convolves token by token.

The format ("mx4"): blocks of 32 consecutive values share one power of two 2^(s - 127),
s a byte; a value is that power times a 4-bit number of the set 0, .5, 1, 1.5, 2, 3, 4, 6
with a sign.  Rows are padded with zero blocks to a multiple of 128 values; two values
to a byte, the earlier one in the low half.  What a call holds in 4 bits is returned here
as the values it stands for (bfloat16, which holds them exactly).
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BLOCK = 32
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # The smallest call: a few rows of a narrow layer, an odd length, made 4-bit and read
        # back (weights of a small adapter).  Launch and call overhead.
        {"name": "codec_5x1000_f32", "op": "codec", "rows": 5, "k": 1000, "dtype": "f32", "rule": "fit",
         "columns": False, "random": False},
        # A training step's activations: both directions at once (the forward product contracts
        # over channels, the weight's gradient over tokens), rounded by given random bytes.
        {"name": "codec_8192x4096_bf16", "op": "codec", "rows": 8192, "k": 4096, "dtype": "bf16", "rule": "floor",
         "columns": True, "random": True},
        # A small batch of users in one serving step: activations made 4-bit in the call,
        # weights 4-bit since loading.
        {"name": "project_48x4096x4096_bf16", "op": "project", "m": 48, "n": 4096, "k": 4096, "dtype": "bf16",
         "bias": True},
        # A prompt of odd length through a layer of odd widths, results in fp32.
        {"name": "project_1001x2000x1504_f32", "op": "project", "m": 1001, "n": 2000, "k": 1504, "dtype": "f32",
         "bias": True},
        # The largest: the wide projection of a training step, forward and both gradients.
        {"name": "train_8192x8192x4096_bf16", "op": "train", "m": 8192, "n": 8192, "k": 4096, "dtype": "bf16"},
        # A short ragged training batch through a narrow layer, fp16.
        {"name": "train_777x520x1304_f16", "op": "train", "m": 777, "n": 520, "k": 1304, "dtype": "f16"},
        # One token of one user: the activations as they are, the weights' bytes are the time.
        {"name": "linear_1x8192x8192_bf16", "op": "linear", "m": 1, "n": 8192, "k": 8192, "dtype": "bf16",
         "out": "bf16", "bias": False},
        # A few users' tokens through an odd layer, fp16 in and fp32 out.
        {"name": "linear_13x5000x2056_f16", "op": "linear", "m": 13, "n": 5000, "k": 2056, "dtype": "f16",
         "out": "f32", "bias": True},
        # Generation: one new token for each of a few users appended to the cache, and their short
        # histories read back.
        {"name": "cache_5x70x200_bf16", "op": "cache", "batch": 5, "length": 70, "channels": 200, "page": 16,
         "dtype": "bf16", "new": 1, "order": "tokens"},
        # A prompt's end written, and whole histories read back as the zero-padded signals, one
        # a channel, that the FFT convolution takes.
        {"name": "cache_4x8192x2048_f32", "op": "cache", "batch": 4, "length": 8192, "channels": 2048, "page": 64,
         "dtype": "f32", "new": 2048, "order": "channels"},
        # One user far into a long text: a single sequence, so the work is split over its taps.
        {"name": "step_1x65536x1024_bf16", "op": "step", "batch": 1, "length": 65536, "channels": 1024, "page": 64,
         "taps": 65536, "dtype": "bf16"},
        # A full batch with ragged histories, one of them empty.
        {"name": "step_24x8000x4096_f32", "op": "step", "batch": 24, "length": 8000, "channels": 4096, "page": 16,
         "taps": 8000, "dtype": "f32"},
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the same operators: sizes spread over the range, odd ones as often as
    even ones, none dearer than the largest listed case of its operator."""
    op = rng.choice(("codec", "project", "project", "train", "linear", "linear", "cache", "step", "step"))
    dtype = rng.choice(("f32", "bf16", "bf16", "f16"))
    if op == "codec":
        k = _spread(rng, 32, 8192)
        return {"op": op, "rows": _spread(rng, 1, (1 << 25) // k), "k": k, "dtype": dtype,
                "rule": rng.choice(("fit", "floor")), "columns": rng.random() < 0.5, "random": rng.random() < 0.5}
    if op in ("project", "train"):
        m, n, k = _spread(rng, 1 if op == "project" else 64, 8192), _spread(rng, 64, 8192), _spread(rng, 64, 8192)
        if rng.random() < 0.5:                  # half of them with a layer's usual widths
            n, k = (n + 127) // 128 * 128, (k + 127) // 128 * 128
        if op == "train" and m * n * k > 1 << 38:
            m = (1 << 38) // (n * k)
        case = {"op": op, "m": m, "n": n, "k": k, "dtype": dtype}
        return {**case, "bias": rng.random() < 0.5} if op == "project" else case
    if op == "linear":
        return {"op": op, "m": _spread(rng, 1, 64), "n": _spread(rng, 100, 16384), "k": _spread(rng, 100, 16384),
                "dtype": dtype, "out": rng.choice((dtype, "f32")), "bias": rng.random() < 0.5}
    channels = _spread(rng, 40, 4096)
    case = {"op": op, "channels": channels, "page": 1 << rng.randint(4, 7), "dtype": dtype}
    if op == "cache":
        length = _spread(rng, 1, 8192)
        batch = _spread(rng, 1, max(1, min(64, (1 << 26) // (length * channels))))
        return {**case, "batch": batch, "length": length, "new": rng.randint(1, length),
                "order": rng.choice(("tokens", "channels"))}
    length = _spread(rng, 1, 65536)
    batch = _spread(rng, 1, max(1, min(64, (3 << 28) // (length * channels))))
    return {**case, "batch": batch, "length": length, "taps": rng.choice((length, _spread(rng, 1, 65536)))}


# ---- inputs --------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 7919 + 29)
    return g


def _activations(g, rows, k, dtype):
    """Rows of Gaussian values, one channel in 64 of them 20 times as large."""
    loud = torch.where(torch.rand(k, device=DEV, generator=g) < 1 / 64, 20.0, 1.0)
    return (torch.randn(rows, k, device=DEV, generator=g) * loud).to(dtype)


def _weights(g, n, k):
    """Trained weights, as 4-bit blocks: made once, when a program loads them."""
    return _quantize(torch.randn(n, k, device=DEV, generator=g) / math.sqrt(k))


def _inputs(case, seed):
    """The inputs of a case from the seed alone."""
    g, op, dtype = _gen(seed), case["op"], DTYPES[case["dtype"]]
    if op == "codec":
        rows, k = case["rows"], case["k"]
        s = {"x": _activations(g, rows, k, dtype), "rand": None}
        if case["random"]:
            s["rand"] = torch.randint(0, 256, (rows, k), device=DEV, generator=g, dtype=torch.uint8)
        return s
    if op == "train":
        m, n, k = case["m"], case["n"], case["k"]
        return {"x": _activations(g, m, k, dtype),
                "w": (torch.randn(n, k, device=DEV, generator=g) / math.sqrt(k)).to(dtype),
                "dy": (torch.randn(m, n, device=DEV, generator=g) * 2.0 ** -8).to(dtype),
                "rand": torch.randint(0, 256, (m, n), device=DEV, generator=g, dtype=torch.uint8)}
    if op in ("project", "linear"):
        m, n, k = case["m"], case["n"], case["k"]
        codes, scales = _weights(g, n, k)
        return {"x": _activations(g, m, k, dtype), "codes": codes, "scales": scales,
                "bias": torch.randn(n, device=DEV, generator=g) if case["bias"] else None}
    # a cache: each sequence's pages anywhere among the pages, lengths from the whole length
    # down, the second one empty (where there are three or more)
    batch, length, channels, page = case["batch"], case["length"], case["channels"], case["page"]
    most = -(-length // page)
    lens = (length * (1 - 0.6 * torch.rand(batch, device=DEV, generator=g))).ceil().to(torch.int32)
    lens[0] = length
    if batch > 2:
        lens[1] = 0
    pages = torch.randperm(batch * most, device=DEV, generator=g).to(torch.int32).view(batch, most)
    codes, scales = _quantize(_activations(g, batch * most * page, channels, torch.float16))
    s = {"pages": pages, "lens": lens, "codes": codes.view(batch * most, page, -1),
         "scales": scales.view(batch * most, page, -1)}
    if op == "cache":
        # the last `new` tokens of every sequence, packed; a token that a sequence lacks has no slot
        t = lens.long()[:, None] - 1 - torch.arange(case["new"], device=DEV)
        slots = pages.long().gather(1, t.clamp_min(0) // page) * page + t.clamp_min(0) % page
        s["slots"] = torch.where(t >= 0, slots, -1).reshape(-1)
        s["x"] = _activations(g, batch * case["new"], channels, dtype)
    else:
        # a decaying filter a channel, tap-major
        rate = torch.exp(torch.rand(channels, device=DEV, generator=g) * -6) / 16
        decay = torch.exp(-torch.arange(case["taps"], device=DEV)[:, None] * rate)
        s["taps"] = (torch.randn(case["taps"], channels, device=DEV, generator=g) * decay).to(dtype)
    return s


def prepare(case, seed):
    case = dict(case)
    s = _inputs(case, seed)
    s["case"] = case
    op = case["op"]
    if op == "codec":
        rows, k = case["rows"], case["k"]
        s["q"] = _blocks_for(rows, k)
        s["back"] = torch.empty(rows, k, dtype=torch.bfloat16, device=DEV)
        if case["columns"]:
            s["qt"] = _blocks_for(k, rows)
            s["back_t"] = torch.empty(k, rows, dtype=torch.bfloat16, device=DEV)
    elif op == "project":
        s["q"] = _blocks_for(case["m"], case["k"])
        s["out"] = torch.empty(case["m"], case["n"], dtype=DTYPES[case["dtype"]], device=DEV)
    elif op == "train":
        m, n, k, dtype = case["m"], case["n"], case["k"], DTYPES[case["dtype"]]
        for name, a, b in (("qx", m, k), ("qw", n, k), ("qdy", m, n)):
            s[name], s[name + "_t"] = _blocks_for(a, b), _blocks_for(b, a)
        s["y"] = torch.empty(m, n, dtype=dtype, device=DEV)
        s["dx"] = torch.empty(m, k, dtype=dtype, device=DEV)
        s["dw"] = torch.empty(n, k, dtype=torch.float32, device=DEV)
    elif op == "linear":
        s["out"] = torch.empty(case["m"], case["n"], dtype=DTYPES[case["out"]], device=DEV)
    elif op == "cache":
        shape = (case["length"], case["channels"])
        s["out"] = torch.empty(case["batch"], *(shape if case["order"] == "tokens" else shape[::-1]),
                               dtype=DTYPES[case["dtype"]], device=DEV)
    else:
        s["out"] = torch.empty(case["batch"], case["channels"], dtype=torch.float32, device=DEV)
        s["work"] = torch.empty(64, case["batch"], case["channels"], dtype=torch.float32, device=DEV)
    return s


def _blocks_for(rows, k):
    kp = _padded(k)
    return (torch.empty(rows, kp // 2, dtype=torch.uint8, device=DEV),
            torch.empty(rows, kp // BLOCK, dtype=torch.uint8, device=DEV))


# ---- the plain form --------------------------------------------------------------------

def _padded(k):
    return (k + 127) // 128 * 128


def _levels(x, rule, rand):
    """x's rows, padded, as blocks: (4-bit codes, scale bytes)."""
    rows, k = x.shape
    v = torch.nn.functional.pad(x.float(), (0, _padded(k) - k)).view(rows, -1, BLOCK)
    mant, ex = torch.frexp(v.abs().amax(-1))            # absmax = mant * 2^ex, .5 <= mant < 1
    e = ex - 3
    if rule == "fit":                                   # the smallest e with absmax <= 6 * 2^e
        e = e + (mant > 0.75)
    e = torch.where(mant == 0, torch.full_like(e, -127), e.clamp_min(-127))
    a = torch.ldexp(v.abs(), -e[..., None])
    step = 0.5 * (1 + (a >= 2) + 2 * (a >= 4))
    a = a / step
    if rand is None:
        a = torch.round(a)
    else:
        r = torch.nn.functional.pad(rand, (0, _padded(k) - k)).view(rows, -1, BLOCK).float()
        low = torch.floor(a)
        a = low + (a - low >= 1 - (r + 0.5) / 256)
    a = (a * step).clamp_max(6)
    code = 2 * a * (a <= 2) + (a + 2) * ((a > 2) & (a <= 4)) + 7 * (a > 4)
    return code.to(torch.uint8) + 8 * torch.signbit(v).to(torch.uint8), (e + 127).to(torch.uint8)


def _quantize(x, rule="fit", rand=None):
    code, scale = _levels(x, rule, rand)
    code = code.view(x.shape[0], -1, 2)
    return code[..., 0] + 16 * code[..., 1], scale


def _values(codes, scales, k):
    """The values that rows of blocks stand for, in fp32."""
    half = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0.0, -.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    q = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    v = half[q.int()].view(*scales.shape, BLOCK) * torch.exp2(scales.float() - 127)[..., None]
    return v.flatten(-2)[..., :k]


def _history(s):
    """(batch, length, channels) of the cache in fp32, zero at and beyond each length."""
    c = s["case"]
    t = torch.arange(c["length"], device=DEV)
    at = s["pages"].long()[:, t // c["page"]] * c["page"] + t % c["page"]
    v = _values(s["codes"].flatten(0, 1)[at], s["scales"].flatten(0, 1)[at], c["channels"])
    return v * (t < s["lens"][:, None])[..., None]


def _plain(s):
    c = s["case"]
    op = c["op"]
    if op == "codec":
        back = _values(*_quantize(s["x"], c["rule"], s["rand"]), c["k"]).bfloat16()
        if not c["columns"]:
            return back
        rand = None if s["rand"] is None else s["rand"].t()
        return back, _values(*_quantize(s["x"].t(), c["rule"], rand), c["rows"]).bfloat16()
    if op == "project":
        y = _values(*_quantize(s["x"]), c["k"]) @ _values(s["codes"], s["scales"], c["k"]).t()
        return (y if s["bias"] is None else y + s["bias"]).to(DTYPES[c["dtype"]])
    if op == "train":
        x, w, dy, r, (m, n, k) = s["x"], s["w"], s["dy"], s["rand"], (c["m"], c["n"], c["k"])
        y = _values(*_quantize(x), k) @ _values(*_quantize(w), k).t()
        dx = _values(*_quantize(dy, "fit", r), n) @ _values(*_quantize(w.t()), n).t()
        dw = _values(*_quantize(dy.t(), "fit", r.t()), m) @ _values(*_quantize(x.t()), m).t()
        return y.to(x.dtype), dx.to(x.dtype), dw
    if op == "linear":
        y = s["x"].float() @ _values(s["codes"], s["scales"], c["k"]).t()
        return (y if s["bias"] is None else y + s["bias"]).to(DTYPES[c["out"]])
    if op == "cache":
        codes, scales = _quantize(s["x"])
        there = s["slots"] >= 0
        s["codes"].flatten(0, 1)[s["slots"][there]] = codes[there]
        s["scales"].flatten(0, 1)[s["slots"][there]] = scales[there]
        v = _history(s).to(DTYPES[c["dtype"]])
        return v if c["order"] == "tokens" else v.transpose(1, 2).contiguous()
    # tap j meets the token j before the last: the history reversed, its last token first
    j = torch.arange(min(c["taps"], c["length"]), device=DEV)
    t = s["lens"].long()[:, None] - 1 - j
    at = s["pages"].long().gather(1, t.clamp_min(0) // c["page"]) * c["page"] + t.clamp_min(0) % c["page"]
    v = _values(s["codes"].flatten(0, 1)[at], s["scales"].flatten(0, 1)[at], c["channels"])
    v.mul_((t >= 0)[..., None])
    return v.mul_(s["taps"][:j.numel()].float()).sum(1)


# ---- one pass ----------------------------------------------------------------------------

def run(s):
    if not own:
        return _plain(s)
    import fufft_amd as ff
    c = s["case"]
    op = c["op"]
    if op == "codec":
        if not c["columns"]:
            ff.mx4_quantize(s["x"], *s["q"], rand=s["rand"], rule=c["rule"])
            ff.mx4_dequantize(*s["q"], s["back"])
            return s["back"]
        ff.mx4_quantize(s["x"], *s["q"], *s["qt"], rand=s["rand"], rule=c["rule"])
        ff.mx4_dequantize(*s["q"], s["back"])
        ff.mx4_dequantize(*s["qt"], s["back_t"])
        return s["back"], s["back_t"]
    if op == "project":
        ff.mx4_quantize(s["x"], *s["q"])
        ff.mx4_matmul(*s["q"], s["codes"], s["scales"], s["out"], c["k"], bias=s["bias"])
        return s["out"]
    if op == "train":
        ff.mx4_quantize(s["x"], *s["qx"], *s["qx_t"])
        ff.mx4_quantize(s["w"], *s["qw"], *s["qw_t"])
        ff.mx4_quantize(s["dy"], *s["qdy"], *s["qdy_t"], rand=s["rand"])
        ff.mx4_matmul(*s["qx"], *s["qw"], s["y"], c["k"])
        ff.mx4_matmul(*s["qdy"], *s["qw_t"], s["dx"], c["n"])
        ff.mx4_matmul(*s["qdy_t"], *s["qx_t"], s["dw"], c["m"])
        return s["y"], s["dx"], s["dw"]
    if op == "linear":
        ff.mx4_linear(s["x"], s["codes"], s["scales"], s["out"], bias=s["bias"])
    elif op == "cache":
        ff.mx4_cache_write(s["x"], s["slots"], s["codes"], s["scales"])
        ff.mx4_cache_read(s["codes"], s["scales"], s["pages"], s["lens"], s["out"], order=c["order"])
    else:
        ff.mx4_cache_conv(s["codes"], s["scales"], s["pages"], s["lens"], s["taps"], s["out"], work=s["work"])
    return s["out"]


# ---- what a pass cannot do without ---------------------------------------------------------

def work(case):
    """Bytes: every input read once, every output written once, 17 bytes to a block of 32 values
    that is kept in 4 bits.  Operations: two for each product and its sum; one a value made
    4-bit or read back."""
    op, size = case["op"], 2 if case["dtype"] != "f32" else 4
    if op == "codec":
        pts, ways = case["rows"] * case["k"], 2 if case["columns"] else 1
        return {"bytes": pts * (size + (1 if case["random"] else 0) + ways * 2), "flops": 2 * ways * pts}
    if op in ("project", "train", "linear"):
        m, n, k = case["m"], case["n"], case["k"]
        if op == "train":
            return {"bytes": size * (2 * m * k + n * k + 2 * m * n) + m * n + 4 * n * k, "flops": 6 * m * n * k}
        out = 4 if case.get("out", case["dtype"]) == "f32" else 2
        return {"bytes": size * m * k + n * k * 17 // 32 + out * m * n + (4 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    # lengths are uniform between 0.4 and 1 of the longest; the first is that, the second empty
    batch, length, channels = case["batch"], case["length"], case["channels"]
    tokens = length * (1 + max(0, batch - 2) * 0.7) if batch > 2 else length * (1 + (batch - 1) * 0.7)
    if op == "cache":
        return {"bytes": int(batch * channels * case["new"] * size + tokens * channels * 17 / 32
                             + batch * length * channels * size), "flops": int(tokens * channels)}
    met = min(length, case["taps"]) / length * tokens
    return {"bytes": int(met * channels * 17 / 32 + min(length, case["taps"]) * channels * size
                         + 4 * batch * channels), "flops": int(2 * met * channels)}


# ---- the same in 64 bits ---------------------------------------------------------------------

_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _rounded(x, rule="fit", rand=None):
    """Rows of x after the 4-bit rounding, in 64 bits, from its definition: the power of two
    from the block's largest magnitude, then the neighbours on the grid."""
    rows, k = x.shape
    pad = -k % BLOCK
    v = torch.nn.functional.pad(x.double(), (0, pad)).view(rows, -1, BLOCK)
    top = v.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(top.clamp_min(2.0 ** -200))) - 3
    limit = 6.0 if rule == "fit" else 8.0               # floor: top < 8 * 2^e, so that top / 2^e is in [4, 8)
    for _ in range(4):
        over = top > limit * torch.exp2(e) if rule == "fit" else top >= limit * torch.exp2(e)
        e = e + over
    p = torch.exp2(e.clamp_min(-127))
    grid = torch.tensor(_GRID, dtype=torch.float64, device=x.device)
    mag = (v.abs() / p).clamp_max(6.0)
    above = torch.searchsorted(grid, mag).clamp_max(7)  # the first grid value >= mag
    hi = grid[above]
    below = torch.where(hi > mag, above - 1, above)
    lo = grid[below]
    if rand is None:
        up = (hi - mag < mag - lo) | ((hi - mag == mag - lo) & (above % 2 == 0))
    else:
        share = torch.where(hi > lo, (mag - lo) / (hi - lo).clamp_min(0.5), torch.zeros_like(mag))
        r = torch.nn.functional.pad(rand.double(), (0, pad)).view(rows, -1, BLOCK)
        up = share + (r + 0.5) / 256 >= 1
    q = torch.where(up, hi, lo) * p
    return torch.where(v < 0, -q, q).view(rows, -1)[:, :k]


def _decoded(codes, scales):
    """Blocks to 64-bit values by the code's fields: one sign, two exponent and one mantissa bit."""
    q = torch.stack((codes.long() % 16, codes.long() // 16), dim=-1).reshape(len(codes), 2 * codes.shape[-1])
    ex, man = (q // 2) % 4, (q % 2).double()
    mag = torch.where(ex == 0, man / 2, (1 + man / 2) * torch.exp2((ex - 1).double()))
    p = torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, dim=-1)
    return torch.where(q >= 8, -mag, mag) * p


def exact(case, seed):
    s, op = _inputs(case, seed), case["op"]
    if op == "codec":
        out = _rounded(s["x"], case["rule"], s["rand"])
        if not case["columns"]:
            return out
        rt = None if s["rand"] is None else s["rand"].t().contiguous()
        return out, _rounded(s["x"].t().contiguous(), case["rule"], rt)
    if op == "train":
        x, w, dy, r = s["x"], s["w"], s["dy"], s["rand"]
        turned = lambda a: a.t().contiguous()  # noqa: E731
        return (torch.matmul(_rounded(x), turned(_rounded(w))),
                torch.matmul(_rounded(dy, rand=r), turned(_rounded(turned(w)))),
                torch.matmul(_rounded(turned(dy), rand=turned(r)), turned(_rounded(turned(x)))))
    if op in ("project", "linear"):
        x = _rounded(s["x"]) if op == "project" else s["x"].double()
        y = torch.matmul(x, _decoded(s["codes"], s["scales"])[:, :case["k"]].t().contiguous())
        return y if s["bias"] is None else y + s["bias"].double()
    batch, length, channels, page = case["batch"], case["length"], case["channels"], case["page"]
    codes, scales = s["codes"].view(-1, s["codes"].shape[-1]), s["scales"].view(-1, s["scales"].shape[-1])
    if op == "cache":
        full = _decoded(codes, scales)[:, :channels]
        for i in (s["slots"] >= 0).nonzero().view(-1).split(1 << 14):
            full[s["slots"][i]] = _rounded(s["x"][i])
        out = torch.zeros(batch, length, channels, dtype=torch.float64, device=DEV)
        for b in range(batch):
            t = torch.arange(int(s["lens"][b]), device=DEV)
            out[b, :t.numel()] = full[s["pages"][b].long()[t // page] * page + t % page]
        return out if case["order"] == "tokens" else out.transpose(1, 2).contiguous()
    out = torch.zeros(batch, channels, dtype=torch.float64, device=DEV)
    for b in range(batch):
        n = int(s["lens"][b])
        for t in torch.arange(max(0, n - case["taps"]), n, device=DEV).split(4096):
            at = s["pages"][b].long()[t // page] * page + t % page
            h = s["taps"][n - 1 - t].double()
            out[b] += (h * _decoded(codes[at], scales[at])[:, :channels]).sum(0)
    return out
