"""The operators on microscaled 4-bit numbers, as cases that can be timed and compared.

A matrix [n, k] in this form (MXFP4 of the OCP microscaling formats) holds, for every 32 neighbouring entries of a row, one
power of two 2^(s - 127) in a byte s (255: not a number) and 32 numbers of 4 bits, a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6.
A block's scale comes from its largest magnitude a: s - 127 = max(floor(log2 a) - 2, -127); its numbers are the entries divided by
the scale, rounded to the nearest of the sixteen (ties to the even code) and at most 6.  Both steps are exact but for that rounding.

  quantise   rows to codes and scales, and back to the values that they stand for
  linear     Q(x) W^T for rows x that the call quantises itself and a weight W that is kept in 4 bits
  gated      glu(Q(h) Wg^T, Q(h) Wu^T), the first half of a feed-forward
  up, down   the same two products of routed experts: the tokens' rows sorted by expert, the gated product with each expert's
             matrices; the rows back through each expert's second matrix and summed for every token with the router's weights

Weights come as a checkpoint holds them (codes [n, k / 2], two to a byte, the even entry in the low half; scales [n, k / 32]) and, laid
out once, with the scales in blocks of 128 rows by 4, the order in which the tensor cores read them: entry
[row / 128][block / 4][row % 32][row / 32 % 4][block % 4], an even number of blocks of 4 along k, zeros where there is no row.
"""
from __future__ import annotations

import math

import torch

own = False
DEVICE = "cuda:0"
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
GLU = {"swiglu": (0.0, 1.0, 0.0), "clamped": (7.0, 1.702, 1.0)}      # limit, alpha, shift: the forms of this package's models
MOST_FLOPS = 2.0 * 2048 * 2 * 12288 * 4096                           # of a drawn case: the largest listed one's


# ---------------------------------------------------------------- cases

def listed():
    """Widths of 4,096 with 12,288 features: the layers of the benchmark's main model; 1,024: those of its small one; experts: its
    models of width 2,048 (16 experts of 768 features, 4 to a token)."""
    return [
        # a decode step's rows in front of a product: 8 requests
        dict(name="quantise 8 x 4096", op="quantise", m=8, k=4096, dtype="bf16"),
        # a prompt's activations in front of the second product of a feed-forward, one row short of whole tiles
        dict(name="quantise 2047 x 12288", op="quantise", m=2047, k=12288, dtype="bf16"),
        # one request decodes: the attention's output projection
        dict(name="linear 1 x 4096 x 4096", op="linear", m=1, n=4096, k=4096, out="bf16"),
        # sixteen requests decode with the small model: queries, keys and values in float32 for the norms behind them
        dict(name="linear 16 x 4096 x 1024", op="linear", m=16, n=4096, k=1024, out="f32"),
        # a ragged portion of a prompt: no size a multiple of a tile
        dict(name="linear 300 x 1000 x 2080", op="linear", m=300, n=1000, k=2080, out="bf16"),
        # a whole prompt through the second product of a feed-forward
        dict(name="linear 2048 x 4096 x 12288", op="linear", m=2048, n=4096, k=12288, out="bf16"),
        # eight requests decode: gate and up
        dict(name="gated 8 x 12288 x 4096", op="gated", m=8, n=12288, k=4096, glu="swiglu"),
        # a whole prompt: gate and up
        dict(name="gated 2048 x 12288 x 4096", op="gated", m=2048, n=12288, k=4096, glu="swiglu"),
        # eight requests decode through 16 experts: few rows each, every matrix read
        dict(name="up 8 of 16 x 768 x 2048", op="up", m=8, n=768, k=2048, experts=16, top=4, glu="clamped", skew=0.0),
        # a portion of prompts, some experts far more liked than others
        dict(name="up 1000 of 16 x 768 x 2048", op="up", m=1000, n=768, k=2048, experts=16, top=4, glu="clamped", skew=1.0),
        # the way back of both
        dict(name="down 8 of 16 x 2048 x 768", op="down", m=8, n=2048, k=768, experts=16, top=4, skew=0.0),
        dict(name="down 1000 of 16 x 2048 x 768", op="down", m=1000, n=2048, k=768, experts=16, top=4, skew=1.0),
    ]


def draw(rng):
    """Another size of the same: 1 to 2,048 rows (spread over the logarithm), rows of 32 to 12,288 entries in whole blocks, any
    number of output columns; up to 64 experts of which a token uses up to 8."""
    def log(a, b):
        return min(b, max(a, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))
    op = rng.choice(("quantise", "linear", "linear", "gated", "up", "down"))
    m = log(1, 2048)
    if op == "quantise":
        return dict(op=op, m=m, k=32 * log(1, 384), dtype=rng.choice(("bf16", "f32")))
    if op in ("linear", "gated"):
        k, n = 32 * log(4, 384), log(24, 12288)
        n = min(n, int(MOST_FLOPS / ((2.0 if op == "linear" else 4.0) * m * k)))
        if op == "linear":
            return dict(op=op, m=m, n=n, k=k, out=rng.choice(("bf16", "f32")) if k <= 1024 else "bf16")
        return dict(op=op, m=m, n=n, k=k, glu=rng.choice(sorted(GLU)))
    experts, m = log(2, 64), log(1, 1000)
    top = rng.randint(1, min(8, experts))
    wide, feat = 32 * log(4, 64), 32 * log(2, 32)
    c = dict(op=op, m=m, n=feat if op == "up" else wide, k=wide if op == "up" else feat, experts=experts, top=top,
             skew=rng.choice((0.0, 1.0, 2.0)))
    return {**c, "glu": rng.choice(sorted(GLU))} if op == "up" else c


# ---------------------------------------------------------------- inputs

def _activations(shape, gen, dtype):
    """Rows as they reach a product: normal, some columns far larger than the others, an empty block here and there."""
    x = torch.randn(shape, generator=gen, device=DEVICE)
    gain = torch.exp(0.7 * torch.randn(shape[-1], generator=gen, device=DEVICE))
    x = x * gain
    quiet = torch.rand(shape[0], shape[-1] // 32, generator=gen, device=DEVICE) < 0.01
    x = torch.where(quiet.repeat_interleave(32, -1), torch.zeros_like(x), x)
    return x.to(torch.bfloat16 if dtype == "bf16" else torch.float32)


def _power(e):
    """2^e in float64, from its bits."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _pack(x):
    """codes uint8 [..., k / 2] and scales uint8 [..., k / 32] of float32 x [..., k], by comparison with the borders of the grid."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    exponent = (torch.frexp(top)[1] - 3).clamp(min=-127)              # frexp: top = f 2^e with f in [0.5, 1)
    exponent = torch.where(top > 0, exponent, torch.full_like(exponent, -127))
    v = (b.double() * _power(-exponent)).float()
    # the number of borders below |v|; one where the tie goes up counts from the number in front of it
    border = torch.tensor((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0), device=x.device)
    border[1::2] = torch.nextafter(border[1::2], border.new_zeros(()))
    code = torch.bucketize(v.abs(), border, out_int32=True)
    code = (code + torch.signbit(v) * 8).to(torch.uint8).reshape(x.shape)
    return code[..., 0::2] | (code[..., 1::2] << 4), (exponent.squeeze(-1) + 127).to(torch.uint8)


def _values(codes, scales):
    """What codes and scales stand for, in float32 (exact)."""
    grid = torch.tensor(GRID + tuple(-g for g in GRID), device=codes.device)
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    v = grid[code].reshape(*scales.shape, 32)
    return (v * _power(scales.to(torch.int32) - 127).float().unsqueeze(-1)).flatten(-2)


def _tiles(scales):
    """The scales in blocks of 128 rows by 4 (see the top)."""
    *lead, n, g = scales.shape
    rb, kb = -(-n // 128), 2 * -(-g // 8)
    t = scales.new_zeros(*lead, rb * 128, kb * 4)
    t[..., :n, :g] = scales
    t = t.view(*lead, rb, 4, 32, kb, 4)
    i = len(lead)
    return t.permute(*range(i), i, i + 3, i + 2, i + 1, i + 4).contiguous()


def _routing(case, gen):
    """For every token `top` different experts, the liked ones more often, and weights that sum to 1."""
    E, n = case["experts"], case["m"]
    liked = -case["skew"] * torch.log1p(torch.arange(E, device=DEVICE, dtype=torch.float32))
    noise = -torch.log(-torch.log(torch.rand(n, E, generator=gen, device=DEVICE).clamp(1e-6, 1 - 1e-6)))
    idx = (liked + noise).topk(case["top"], -1).indices.to(torch.int32).contiguous()
    weight = torch.softmax(torch.randn(n, case["top"], generator=gen, device=DEVICE), -1)
    return idx, weight


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    op, m, k = case["op"], case["m"], case["k"]
    s = {"case": case}
    if op == "quantise":
        s["x"] = _activations((m, k), gen, case["dtype"])
        return s
    n = case["n"]
    lead = {"linear": (), "gated": (2,), "up": (case.get("experts"), 2), "down": (case.get("experts"),)}[op]
    w = torch.randn(*lead, n, k, generator=gen, device=DEVICE) * k ** -0.5
    s["codes"], s["scales"] = _pack(w)
    s["tiles"] = _tiles(s["scales"])
    if op in ("up", "down"):
        s["idx"], s["weight"] = _routing(case, gen)
        # (expert by expert, tokens in order: where a token's row lies among the sorted ones)
        order = torch.sort(s["idx"].flatten().long(), stable=True).indices
        s["place"] = torch.empty_like(order).scatter_(0, order, torch.arange(order.numel(), device=DEVICE)).to(torch.int32)
        count = torch.bincount(s["idx"].flatten().long(), minlength=case["experts"])
        s["offsets"] = torch.cat((count.new_zeros(1), count.cumsum(0))).to(torch.int32)
    s["x"] = _activations((m * case["top"] if op == "down" else m, k), gen, "bf16")
    return s


# ---------------------------------------------------------------- one pass

def _glu(g, u, form):
    limit, alpha, shift = GLU[form]
    if limit:
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    return g / (1.0 + torch.exp(-alpha * g)) * (u + shift)


def _plain(s):
    case = s["case"]
    op = case["op"]
    x = _values(*_pack(s["x"].float()))
    if op == "quantise":
        return x.to(torch.bfloat16)
    w = _values(s["codes"], s["scales"])
    if op == "linear":
        return (x @ w.T).to(torch.bfloat16 if case["out"] == "bf16" else torch.float32)
    if op == "gated":
        return _glu(x @ w[0].T, x @ w[1].T, case["glu"]).to(torch.bfloat16)
    expert, place = s["idx"].flatten().long(), s["place"].long()
    if op == "up":
        token = torch.arange(case["m"], device=DEVICE).repeat_interleave(case["top"])
        every = _glu(torch.matmul(x, w[:, 0].mT), torch.matmul(x, w[:, 1].mT), case["glu"])      # [expert, token, n]
        rows = torch.empty(place.numel(), case["n"], device=DEVICE)
        rows[place] = every[expert, token]
        return rows.to(torch.bfloat16)
    # down: every expert's matrix over all sorted rows costs what a plain form may; each row keeps its own expert's
    own_expert = torch.empty_like(expert)
    own_expert[place] = expert
    every = torch.matmul(x, w.mT)                                                                # [expert, row, n]
    y = every[own_expert, torch.arange(place.numel(), device=DEVICE)]
    return (y[place].view(case["m"], case["top"], -1) * s["weight"].unsqueeze(-1)).sum(1)


def run(s):
    if not own:
        return _plain(s)
    from rllm_b200.csrc import ops
    case = s["case"]
    op, x = case["op"], s["x"]
    if op == "quantise":
        return ops.mx4_quantize(x).dequantize(torch.bfloat16)
    w = ops.Mx4Matrix(s["codes"], s["tiles"], settled=True)          # a loaded model's weight: nothing writes it any more
    if op == "linear":
        return ops.linear(x, w, out_dtype=torch.bfloat16 if case["out"] == "bf16" else torch.float32)
    if op == "gated":
        out = torch.empty(case["m"], case["n"], dtype=torch.bfloat16, device=x.device)
        return ops.gate_up_swiglu(x, w, out, glu=GLU[case["glu"]])
    if op == "up":
        offsets, place = ops.moe_sort(s["idx"], case["experts"])
        act = torch.empty(place.numel(), case["n"], dtype=torch.bfloat16, device=x.device)
        return ops.mx4_experts_up(x, w, offsets, place, act, glu=GLU[case["glu"]])
    y = torch.empty(x.shape[0], case["n"], dtype=torch.float32, device=x.device)
    ops.mx4_experts_down(x, w, s["offsets"], y)
    return ops.moe_combine(y, s["place"], s["weight"], torch.empty(case["m"], case["n"], dtype=torch.float32, device=x.device))


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    op, m, k = case["op"], case["m"], case["k"]
    if op == "quantise":            # the rows in, codes and scales out, and the values of them in 16 bits out
        return {"bytes": m * k * (2 if case["dtype"] == "bf16" else 4) + m * k * 17 // 32 + m * k * 2, "flops": 4.0 * m * k}
    n = case["n"]
    four = 17 / 32                  # bytes of an entry: half a byte and a scale for 32
    if op == "linear":
        return {"bytes": int(n * k * four) + m * k * 2 + m * n * (2 if case["out"] == "bf16" else 4), "flops": 2.0 * m * n * k}
    if op == "gated":
        return {"bytes": int(2 * n * k * four) + m * k * 2 + m * n * 2, "flops": 4.0 * m * n * k}
    pairs, E = m * case["top"], case["experts"]
    used = E * (1 - (1 - case["top"] / E) ** m)       # experts that some token uses, were all liked alike
    if op == "up":
        return {"bytes": int(used * 2 * n * k * four) + m * k * 2 + pairs * (n * 2 + 8), "flops": 4.0 * pairs * n * k}
    return {"bytes": int(used * n * k * four) + pairs * (k * 2 + 8) + m * n * 4, "flops": 2.0 * pairs * n * k}


# ---------------------------------------------------------------- the definition in 64 bits

def _rounded(x):
    """Q(x) in float64: a step of 0.5 below 2, of 1 below 4, of 2 above, nearest even, at most 6."""
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    # (whole numbers: the logarithm of a power of two may come out a little below itself)
    below = (top.view(torch.int64) >> 52) - 1023                      # floor(log2 top); -1023 for zero
    scale = ((below - 2).clamp(min=-127) + 1023 << 52).view(torch.float64)
    v = b / scale
    step = torch.where(v.abs() < 2, 0.5, torch.where(v.abs() < 4, 1.0, 2.0)).to(v.dtype)
    return ((v / step).round() * step).clamp(-6, 6).mul(scale).flatten(-2)


def _held(codes, scales):
    """The weight's values in float64, code by code."""
    def number(c):
        e, f = ((c >> 1) & 3).double(), (c & 1).double()
        mag = torch.where(e == 0, f / 2, torch.where(e == 1, 1.0, 2 * e - 2) * (1 + f / 2))
        return torch.where(c >= 8, -mag, mag)
    v = torch.stack((number(codes & 15), number(codes >> 4)), -1).flatten(-2)
    return v * (scales.long() + (1023 - 127) << 52).view(torch.float64).repeat_interleave(32, -1)


def exact(case, seed):
    s = prepare(case, seed)
    op, x = case["op"], _rounded(s["x"])
    if op == "quantise":
        return x

    def unit(g, u):
        limit, alpha, shift = GLU[case["glu"]]
        if limit > 0:
            g, u = torch.minimum(g, torch.full_like(g, limit)), torch.clamp(u, -limit, limit)
        return g * torch.sigmoid(alpha * g) * (u + shift)

    if op == "linear":
        return x @ _held(s["codes"], s["scales"]).T
    if op == "gated":
        return unit(*(x @ _held(c, z).T for c, z in zip(s["codes"], s["scales"])))
    idx, place = s["idx"].cpu(), s["place"].cpu().view(case["m"], case["top"])
    if op == "up":
        rows = torch.zeros(place.numel(), case["n"], dtype=torch.float64, device=DEVICE)
        for e in range(case["experts"]):
            t, j = (idx == e).nonzero(as_tuple=True)
            if t.numel():
                w = _held(s["codes"][e], s["scales"][e])
                h = x[t.to(DEVICE)]
                rows[place[t, j].long().to(DEVICE)] = unit(h @ w[0].T, h @ w[1].T)
        return rows
    out = torch.zeros(case["m"], case["n"], dtype=torch.float64, device=DEVICE)
    for e in range(case["experts"]):
        t, j = (idx == e).nonzero(as_tuple=True)
        if t.numel():
            y = x[place[t, j].long().to(DEVICE)] @ _held(s["codes"][e], s["scales"][e]).T
            out.index_add_(0, t.to(DEVICE), y * s["weight"].double()[t.to(DEVICE), j.to(DEVICE)].unsqueeze(-1))
    return out
