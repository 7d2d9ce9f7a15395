"""The work of the calls around a sequence mixer: the norm before a layer with the residual's
sum and its result in 8 bits, 8-bit products, and linear attention whose state decays by a
constant of each head, over whole texts, in training and token by token.

8-bit rows ("i8"): a row of k values is k signed bytes (padded with zeros to a multiple of
128) and one fp32 scale, its largest magnitude over 127; a byte stands for itself times the
scale.  What a call holds in 8 bits is returned here as the values it stands for, in bfloat16.

Decaying linear attention, a head:  S[t] = a S[t - 1] + k[t] v[t]^T,  out[t] = scale q[t]^T S[t],
a = exp(log_decay).  States are (key dim, value dim) in fp32.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6
CHUNK = 64


def listed():
    return [
        # The smallest: a few tokens through the norm before a projection, an odd width.
        {"name": "norm_5x1000_f32", "op": "norm", "rows": 5, "k": 1000, "dtype": "f32", "residual": None, "codes": False},
        # A prompt's tokens: the residual stream in fp32 takes the layer's result, and the norm of
        # the sum goes on in 8 bits.
        {"name": "norm_8192x4096_bf16_i8", "op": "norm", "rows": 8192, "k": 4096, "dtype": "bf16", "residual": "f32",
         "codes": True},
        # A short training batch of odd width, fp16.
        {"name": "norm_grad_777x520_f16", "op": "norm_grad", "rows": 777, "k": 520, "dtype": "f16", "residual": None,
         "through": False},
        # A training step: gradients of the norm, with what comes along the residual.
        {"name": "norm_grad_8192x4096_bf16", "op": "norm_grad", "rows": 8192, "k": 4096, "dtype": "bf16",
         "residual": None, "through": True},
        # One token of one user through a wide layer: the weights' bytes are the time.
        {"name": "project_1x8192x8192_bf16", "op": "project", "m": 1, "n": 8192, "k": 8192, "dtype": "bf16",
         "out": "bf16", "bias": False},
        # A prompt through a wide layer: the matrix cores are the time.
        {"name": "project_8192x8192x4096_bf16", "op": "project", "m": 8192, "n": 8192, "k": 4096, "dtype": "bf16",
         "out": "bf16", "bias": True},
        # One long text: few heads, so the work has to be split along it.
        {"name": "mix_1x65536x16_128x128_bf16", "op": "mix", "batch": 1, "tokens": 65536, "heads": 16, "dk": 128,
         "dv": 128, "dtype": "bf16", "state": False, "ragged": False},
        # A padded batch of texts that go on from earlier states, odd sizes, fp32.
        {"name": "mix_3x777x6_72x40_f32", "op": "mix", "batch": 3, "tokens": 777, "heads": 6, "dk": 72, "dv": 40,
         "dtype": "f32", "state": True, "ragged": True},
        # A training step: all gradients of a batch of texts.
        {"name": "mix_grad_4x4096x16_128x128_bf16", "op": "mix_grad", "batch": 4, "tokens": 4096, "heads": 16, "dk": 128,
         "dv": 128, "dtype": "bf16", "state": False, "ragged": False},
        # A short ragged batch in fp16, states and their gradients among it.
        {"name": "mix_grad_2x500x5_64x64_f16", "op": "mix_grad", "batch": 2, "tokens": 500, "heads": 5, "dk": 64,
         "dv": 64, "dtype": "f16", "state": True, "ragged": True},
        # Generation for one user.
        {"name": "step_1x16_128x128_bf16", "op": "step", "batch": 1, "heads": 16, "dk": 128, "dv": 128, "dtype": "bf16"},
        # Generation for a full batch: every state is read and written once.
        {"name": "step_128x32_128x128_bf16", "op": "step", "batch": 128, "heads": 32, "dk": 128, "dv": 128,
         "dtype": "bf16"},
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _dim(rng):
    """A head's width: mostly the usual ones, odd ones among them."""
    return rng.choice((32, 64, 64, 96, 128, 128, 128, rng.randint(1, 16) * 8, rng.randint(1, 128)))


def draw(rng):
    """One more case of the same operators: sizes spread over the range, odd ones as often as
    even ones, none dearer than the largest listed case of its operator."""
    op = rng.choice(("norm", "norm_grad", "project", "project", "mix", "mix", "mix_grad", "step"))
    dtype = rng.choice(("f32", "bf16", "bf16", "f16"))
    if op in ("norm", "norm_grad"):
        k = _spread(rng, 16, 16384)
        if rng.random() < 0.5:                  # half of them with a layer's usual widths
            k = (k + 127) // 128 * 128
        residual = rng.choice((None, dtype, "f32"))
        most = 1 << (24 if "f32" in (dtype, residual) and (op == "norm_grad" or dtype == residual) else 25)
        case = {"op": op, "rows": _spread(rng, 1, most // k), "k": k, "dtype": dtype, "residual": residual}
        return {**case, "codes": rng.random() < 0.5} if op == "norm" else {**case, "through": rng.random() < 0.5}
    if op == "project":
        n, k = _spread(rng, 64, 16384), _spread(rng, 64, 16384)
        if rng.random() < 0.5:
            n, k = (n + 127) // 128 * 128, (k + 127) // 128 * 128
        m = _spread(rng, 1, max(1, min(8192, (1 << 38) // (n * k))))
        return {"op": op, "m": m, "n": n, "k": k, "dtype": dtype, "out": rng.choice((dtype, "f32")),
                "bias": rng.random() < 0.5}
    dk, dv, heads = _dim(rng), _dim(rng), _spread(rng, 1, 32)
    case = {"op": op, "heads": heads, "dk": dk, "dv": dv, "dtype": dtype}
    if op == "step":
        return {**case, "batch": _spread(rng, 1, max(1, min(256, (1 << 26) // (heads * dk * dv))))}
    most = 1 << (20 if op == "mix" else 18) - (dtype == "f32")      # tokens of all heads and texts
    tokens = _spread(rng, 1, min(65536 if op == "mix" else 8192, most // heads))
    batch = _spread(rng, 1, max(1, min(32, most // (heads * tokens))))
    return {**case, "tokens": tokens, "batch": batch, "state": rng.random() < 0.5, "ragged": rng.random() < 0.5}


# ---- inputs --------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 6661 + 17)
    return g


def _activations(g, rows, k, dtype):
    """Rows of Gaussian values, one channel in 64 of them 20 times as large."""
    loud = torch.where(torch.rand(k, device=DEV, generator=g) < 1 / 64, 20.0, 1.0)
    return (torch.randn(rows, k, device=DEV, generator=g) * loud).to(dtype)


def _inputs(case, seed):
    """The inputs of a case from the seed alone."""
    g, op, dtype = _gen(seed), case["op"], DTYPES[case["dtype"]]
    randn = lambda *shape: torch.randn(*shape, device=DEV, generator=g)  # noqa: E731
    if op in ("norm", "norm_grad"):
        rows, k = case["rows"], case["k"]
        s = {"weight": 1 + randn(k) / 8}
        sum_type = dtype if case["residual"] is None else DTYPES[case["residual"]]
        if op == "norm":
            s["x"] = _activations(g, rows, k, dtype)
            s["residual"] = None if case["residual"] is None else (2 * randn(rows, k)).to(sum_type)
        else:
            s["x"] = _activations(g, rows, k, sum_type)         # the sum that the norm was taken of
            s["dy"] = (randn(rows, k) / 256).to(dtype)
            s["dsum"] = (randn(rows, k) / 256).to(sum_type) if case["through"] else None
        return s
    if op == "project":
        s = {"x": _activations(g, case["m"], case["k"], dtype)}
        s["codes"], s["scales"] = _quantize(randn(case["n"], case["k"]) / math.sqrt(case["k"]))   # trained weights
        s["bias"] = randn(case["n"]) if case["bias"] else None
        return s
    batch, heads, dk, dv = case["batch"], case["heads"], case["dk"], case["dv"]
    # memories from 4 tokens to 1024, a head each
    s = {"decay": -torch.exp2(-2 - 8 * torch.arange(heads, device=DEV) / max(1, heads - 1))}
    if op == "step":
        s["q"], s["v"] = randn(batch, heads, dk).to(dtype), randn(batch, heads, dv).to(dtype)
        s["k"] = (randn(batch, heads, dk) / math.sqrt(dk)).to(dtype)
        pool = batch + batch // 8 + 1                           # states of texts that wait among them
        s["state"] = randn(pool, heads, dk, dv)
        s["slots"] = torch.randperm(pool, device=DEV, generator=g)[:batch].contiguous()
        return s
    tokens = case["tokens"]
    s["q"], s["v"] = randn(batch, tokens, heads, dk).to(dtype), randn(batch, tokens, heads, dv).to(dtype)
    s["k"] = (randn(batch, tokens, heads, dk) / math.sqrt(dk)).to(dtype)
    s["state"] = randn(batch, heads, dk, dv) if case["state"] else None
    s["lens"] = None
    if case["ragged"]:
        s["lens"] = (tokens * (1 - 0.6 * torch.rand(batch, device=DEV, generator=g))).ceil().to(torch.int32)
        s["lens"][0] = tokens
    if op == "mix_grad":
        s["do"] = (randn(batch, tokens, heads, dv) / 16).to(dtype)
        s["dnew"] = randn(batch, heads, dk, dv) / 16 if case["state"] else None
    return s


def prepare(case, seed):
    case = dict(case)
    s = _inputs(case, seed)
    s["case"] = case
    op, dtype = case["op"], DTYPES[case["dtype"]]
    if op in ("norm", "norm_grad"):
        rows, k = case["rows"], case["k"]
    if op == "norm":
        s["total"] = None if s["residual"] is None else torch.empty_like(s["residual"])
        if case["codes"]:
            s["q"] = _rows_for(rows, k)
            s["back"] = torch.empty(rows, k, dtype=torch.bfloat16, device=DEV)
        else:
            s["out"] = torch.empty(rows, k, dtype=dtype, device=DEV)
    elif op == "norm_grad":
        s["dx"], s["dw"] = torch.empty(rows, k, dtype=dtype, device=DEV), torch.empty(k, device=DEV)
        s["work"] = torch.empty(512, k, device=DEV)
    elif op == "project":
        s["q"] = _rows_for(case["m"], case["k"])
        s["out"] = torch.empty(case["m"], case["n"], dtype=DTYPES[case["out"]], device=DEV)
    elif op == "step":
        s["out"] = torch.empty_like(s["v"])
    else:
        # tokens behind a text's last stay as they are, so they are zeros from the start
        batch, heads, dk, dv = case["batch"], case["heads"], case["dk"], case["dv"]
        s["work"] = torch.empty(max(1, min(64, 1024 // (batch * heads))) * batch * heads * dk * dv
                                * (3 if op == "mix_grad" else 1), device=DEV)
        s["new"] = torch.empty(batch, heads, dk, dv, device=DEV)
        if op == "mix":
            s["out"] = torch.zeros_like(s["v"])
        else:
            s["dq"], s["dk"], s["dv"] = torch.zeros_like(s["q"]), torch.zeros_like(s["k"]), torch.zeros_like(s["v"])
    return s


def _rows_for(rows, k):
    return torch.empty(rows, (k + 127) // 128 * 128, dtype=torch.int8, device=DEV), torch.empty(rows, device=DEV)


# ---- the plain form --------------------------------------------------------------------

def _quantize(y):
    """y's rows in 8 bits: (padded bytes, scales)."""
    y = y.float()
    top = y.abs().amax(1)
    # in 64 bits, as half of the largest magnitude is half-way between two bytes
    code = torch.round(y.double() * 127 / torch.where(top > 0, top, torch.ones_like(top)).double()[:, None])
    return torch.nn.functional.pad(code, (0, -y.shape[1] % 128)).to(torch.int8), top / 127


def _norm(s):
    c = s["case"]
    h = s["x"].float() if s["residual"] is None else s["x"].float() + s["residual"].float()
    y = h * torch.rsqrt(h.square().mean(1, keepdim=True) + EPS) * s["weight"]
    out = ()
    if s["residual"] is not None:
        out = (h.to(s["residual"].dtype),)
    if not c["codes"]:
        return out + (y.to(s["x"].dtype),)
    code, scale = _quantize(y)
    return out + ((code[:, :c["k"]].float() * scale[:, None]).bfloat16(), scale)


def _norm_grad(s):
    x, dy = s["x"].float(), s["dy"].float()
    r = torch.rsqrt(x.square().mean(1, keepdim=True) + EPS)
    n = x * r
    wdy = dy * s["weight"]
    dx = r * (wdy - n * (wdy * n).mean(1, keepdim=True))
    if s["dsum"] is not None:
        dx = dx + s["dsum"].float()
    return dx.to(s["dy"].dtype), (dy * n).sum(0)


def _project(s):
    code, scale = _quantize(s["x"])
    y = code.float() @ s["codes"].float().t() * scale[:, None] * s["scales"]
    return (y if s["bias"] is None else y + s["bias"]).to(DTYPES[s["case"]["out"]])


def _powers(decay, n):
    """exp(decay n) for every head and the numbers n."""
    return torch.exp(decay.double().view(-1, *[1] * n.dim()) * n.double()).float()


def _mixed(q, k, v, decay, state, lens, late):
    """(out, new state) of q, k, v (batch, heads, tokens, dim), zeros from lens on: products
    within chunks of 64 tokens, and of the state before each chunk.  late: 0, or 1 where the state
    given meets its first token undecayed, and the one returned is decayed once more."""
    batch, heads, tokens, dk = q.shape
    dv, n = v.shape[-1], -(-tokens // CHUNK)
    t = torch.arange(tokens, device=DEV)
    left = lens.long()[:, None] - 1 - t + late
    w = torch.exp(decay.double()[None, :, None] * left[:, None].clamp_min(0)).float() * (left >= late)[:, None]
    new = (k * w[..., None]).transpose(2, 3) @ v
    q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, n * CHUNK - tokens)).view(batch, heads, n, CHUNK, -1) for x in (q, k, v))
    i = torch.arange(CHUNK, device=DEV)
    far = i[:, None] - i
    out = (q @ k.transpose(3, 4) * (_powers(decay, far.clamp_min(0)) * (far >= 0))[:, None]) @ v
    local = (k * _powers(decay, CHUNK - 1 - i + late)[:, None, :, None]).transpose(3, 4) @ v
    far = torch.arange(n, device=DEV)[:, None] - 1 - torch.arange(n, device=DEV)
    before = (_powers(decay, CHUNK * far.clamp_min(0)) * (far >= 0)) @ local.flatten(3)
    if state is not None:
        before = before + _powers(decay, CHUNK * torch.arange(n, device=DEV))[..., None] * state.flatten(2)[:, :, None]
        new = new + torch.exp(decay.double()[:, None, None] * lens.double()[:, None, None, None]).float() * state
    out = out + (q * _powers(decay, i + 1 - late)[:, None, :, None]) @ before.view(batch, heads, n, dk, dv)
    return out.view(batch, heads, n * CHUNK, dv)[:, :, :tokens], new


def _mix(s):
    c = s["case"]
    lens = s["lens"] if s["lens"] is not None else torch.full((c["batch"],), c["tokens"], device=DEV)
    t = torch.arange(c["tokens"], device=DEV)
    there = (t < lens[:, None])[:, None, :, None]
    back = (lens.long()[:, None] - 1 - t).clamp_min(0)[:, None, :, None]
    heads_first = lambda x: x.transpose(1, 2).float() * there  # noqa: E731
    turned = lambda x: x.gather(2, back.expand(x.shape)) * there  # noqa: E731
    to = lambda x: x.transpose(1, 2).contiguous().to(DTYPES[c["dtype"]])  # noqa: E731
    q, k, v = (heads_first(s[n]) for n in ("q", "k", "v"))
    if c["op"] == "mix":
        out, new = _mixed(q, k, v, s["decay"], s["state"], lens, 0)
        return to(out * there / math.sqrt(c["dk"])), new
    # With S[t] = a S[t - 1] + k[t] v[t]^T, dq[t] = S[t] dout[t] is the same sum with v for keys and k for
    # values; D[t] = q[t] dout[t]^T + a D[t + 1] from the last token back gives dk[t] = D[t] v[t],
    # dv[t] = D[t]^T k[t] and the state's gradient a D[0].
    do, scale, late = heads_first(s["do"]), 1 / math.sqrt(c["dk"]), 1
    st, dnew = s["state"], s["dnew"]
    other = lambda x: None if x is None else x.transpose(2, 3).contiguous()  # noqa: E731
    dq, _ = _mixed(do, v, k, s["decay"], other(st), lens, 0)
    qt, kt, vt, dot = turned(q) * scale, turned(k), turned(v), turned(do)
    dk, _ = _mixed(vt, dot, qt, s["decay"], other(dnew), lens, late)
    dv, dstate = _mixed(kt, qt, dot, s["decay"], dnew, lens, late)
    grads = to(dq * there * scale), to(turned(dk)), to(turned(dv))
    return grads + (dstate,) if c["state"] else grads


def _step(s):
    c, at = s["case"], s["slots"]
    q, k, v = (s[n].float() for n in ("q", "k", "v"))
    state = s["state"][at] * torch.exp(s["decay"].double()).float()[:, None, None] + k[..., None] * v[..., None, :]
    s["state"][at] = state
    out = (q[..., None] * state).sum(2) / math.sqrt(c["dk"])
    return out.to(s["v"].dtype), s["state"]


# ---- one pass ----------------------------------------------------------------------------

def run(s):
    c = s["case"]
    op = c["op"]
    if not own:
        return {"norm": _norm, "norm_grad": _norm_grad, "project": _project, "mix": _mix, "mix_grad": _mix, "step": _step}[op](s)
    import fufft_amd as ff
    if op == "norm":
        out = () if s["total"] is None else (s["total"],)
        if not c["codes"]:
            ff.rms_norm(s["x"], s["weight"], s["out"], residual=s["residual"], total=s["total"], eps=EPS)
            return out + (s["out"],)
        ff.rms_norm(s["x"], s["weight"], codes=s["q"][0], scales=s["q"][1], residual=s["residual"], total=s["total"], eps=EPS)
        ff.i8_dequantize(*s["q"], s["back"])
        return out + (s["back"], s["q"][1])
    if op == "norm_grad":
        ff.rms_norm_grad(s["dy"], s["x"], s["weight"], s["dx"], s["dw"], s["work"], dtotal=s["dsum"], eps=EPS)
        return s["dx"], s["dw"]
    if op == "project":
        ff.i8_quantize(s["x"], *s["q"])
        ff.i8_matmul(*s["q"], s["codes"], s["scales"], s["out"], c["k"], bias=s["bias"])
        return s["out"]
    scale = 1 / math.sqrt(c["dk"])
    if op == "step":
        ff.decay_attention_step(s["q"], s["k"], s["v"], s["decay"], s["state"], s["out"], slots=s["slots"], scale=scale)
        return s["out"], s["state"]
    if op == "mix":
        ff.decay_attention(s["q"], s["k"], s["v"], s["decay"], s["out"], state=s["state"], new_state=s["new"],
                           lens=s["lens"], work=s["work"], scale=scale)
        return s["out"], s["new"]
    grads = s["dq"], s["dk"], s["dv"]
    dstate = s["new"] if c["state"] else None
    ff.decay_attention_grad(s["do"], s["q"], s["k"], s["v"], s["decay"], *grads, state=s["state"], dnew_state=s["dnew"],
                            dstate=dstate, lens=s["lens"], work=s["work"], scale=scale)
    return grads if dstate is None else grads + (dstate,)


# ---- what a pass cannot do without ---------------------------------------------------------

def work(case):
    """Bytes: every input read once, every output written once.  Operations: two for each product
    and its sum, the attention's as its recurrence makes them; a few for each value of a norm."""
    op, size = case["op"], 2 if case["dtype"] != "f32" else 4
    if op in ("norm", "norm_grad"):
        pts, k = case["rows"] * case["k"], case["k"]
        stream = size if case["residual"] is None else 4 if case["residual"] == "f32" else 2
        if op == "norm":
            # a byte a value written and read again where 8 bits are asked for, two for what they stand for
            sides = size + (4 if case["codes"] else size) + (0 if case["residual"] is None else 2 * stream)
            return {"bytes": pts * sides + 4 * k, "flops": 6 * pts}
        return {"bytes": pts * (2 * size + stream * (2 if case["through"] else 1)) + 8 * k, "flops": 12 * pts}
    if op == "project":
        m, n, k = case["m"], case["n"], case["k"]
        out = 4 if case["out"] == "f32" else 2
        return {"bytes": size * m * k + n * k + out * m * n + 4 * n * (2 if case["bias"] else 1), "flops": 2 * m * n * k}
    batch, heads, dk, dv = case["batch"], case["heads"], case["dk"], case["dv"]
    state = 4 * batch * heads * dk * dv
    if op == "step":
        return {"bytes": 2 * state + size * batch * heads * 2 * (dk + dv), "flops": 5 * batch * heads * dk * dv}
    # lengths are uniform between 0.4 and 1 of the longest; the first is that
    share = (1 + 0.7 * (batch - 1)) / batch if case["ragged"] else 1
    each = int(batch * case["tokens"] * heads * share)
    states = (2 if case["state"] else 1) * state
    if op == "mix":
        return {"bytes": each * size * 2 * (dk + dv) + states, "flops": 4 * each * dk * dv}
    return {"bytes": each * size * (4 * dk + 3 * dv) + (3 * state if case["state"] else 0), "flops": 10 * each * dk * dv}


# ---- the same in 64 bits ---------------------------------------------------------------------

def _rounded(y):
    """Rows of y as the multiples of a 127th of their largest magnitude that they are nearest to."""
    top = y.abs().max(dim=1, keepdim=True).values
    share = 127 * y / top.clamp_min(1e-300)
    return torch.round(share) * top / 127, top[:, 0] / 127


def exact(case, seed):
    s, op = _inputs(case, seed), case["op"]
    if op == "norm":
        h = s["x"].double()
        h = h if s["residual"] is None else h + s["residual"].double()
        y = s["weight"].double() * h / torch.sqrt((h * h).sum(1, keepdim=True) / case["k"] + EPS)
        out = [] if s["residual"] is None else [h]
        return out + (list(_rounded(y)) if case["codes"] else [y])
    if op == "norm_grad":
        # y_i = w_i x_i / r, r^2 = sum x^2 / k + eps:  dx_i = dy_i w_i / r - x_i sum_j (dy_j w_j x_j) / (k r^3)
        x, dy, w = s["x"].double(), s["dy"].double(), s["weight"].double()
        r = torch.sqrt((x * x).sum(1, keepdim=True) / case["k"] + EPS)
        dx = dy * w / r - x * (dy * w * x).sum(1, keepdim=True) / (case["k"] * r ** 3)
        if s["dsum"] is not None:
            dx = dx + s["dsum"].double()
        return dx, (dy * x / r).sum(0)
    if op == "project":
        x, _ = _rounded(s["x"].double())
        w = (s["codes"].double() * s["scales"].double()[:, None])[:, :case["k"]].t().contiguous()
        y = x @ w
        return y if s["bias"] is None else y + s["bias"].double()
    a = torch.exp(s["decay"].double())[:, None, None]
    scale = case["dk"] ** -0.5
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    if op == "step":
        state, at = s["state"].double(), s["slots"]
        new = a * state[at] + torch.einsum("bhi,bhj->bhij", k, v)
        state[at] = new
        return scale * torch.einsum("bhi,bhij->bhj", q, new), state
    # token by token, from the recurrence itself
    batch, tokens, heads, dk, dv = case["batch"], case["tokens"], case["heads"], case["dk"], case["dv"]
    lens = [tokens] * batch if s["lens"] is None else s["lens"].tolist()
    there = torch.tensor([[t < n for n in lens] for t in range(tokens)], dtype=torch.float64, device=DEV)[:, :, None, None]
    keep = torch.where(there[..., None] > 0, a, torch.ones_like(a)) if s["lens"] is not None else [a] * tokens
    cut = (lambda x: x * there.transpose(0, 1)) if s["lens"] is not None else (lambda x: x)
    first = lambda x, shape: torch.zeros(*shape, dtype=torch.float64, device=DEV) if x is None else x.double().clone()  # noqa: E731
    q, k, v = cut(q) * scale, cut(k), cut(v)
    state = first(s["state"], (batch, heads, dk, dv))
    out = torch.zeros(batch, tokens, heads, dv if op == "mix" else dk, dtype=torch.float64, device=DEV)
    do = None if op == "mix" else cut(s["do"].double())
    for t in range(tokens):
        state.mul_(keep[t]).addcmul_(k[:, t, :, :, None], v[:, t, :, None, :])
        if op == "mix":
            out[:, t] = (q[:, t, :, None] @ state)[:, :, 0]
        else:
            out[:, t] = (state @ do[:, t, :, :, None])[..., 0]
    if op == "mix":
        return out, state
    dkey, dval, d = torch.zeros_like(k), torch.zeros_like(v), first(s["dnew"], (batch, heads, dk, dv))
    for t in reversed(range(tokens)):
        d.addcmul_(q[:, t, :, :, None], do[:, t, :, None, :])
        dkey[:, t] = (d @ v[:, t, :, :, None])[..., 0]
        dval[:, t] = (k[:, t, :, None] @ d)[:, :, 0]
        d.mul_(keep[t])
    grads = cut(out) * scale, cut(dkey), cut(dval)
    return grads + (d,) if case["state"] else grads
