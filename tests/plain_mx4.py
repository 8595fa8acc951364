"""Microscaled 4-bit numbers and their products in float64, from the format's definition; nothing of the package."""
import torch

BLOCK = 32


def quantize(x):
    """(codes, scales, values) of x [..., k]: codes [..., k] 0..15, scales [..., k / 32] 0..255, values float64."""
    b = x.double().unflatten(-1, (-1, BLOCK))
    bad = ~torch.isfinite(b).all(-1, keepdim=True)
    top = torch.where(bad, torch.ones_like(b), b.abs()).amax(-1, keepdim=True)
    e = torch.frexp(top)[1].long() - 1                      # floor(log2 top)
    e = torch.where(top > 0, (e - 2).clamp(min=-127), torch.full_like(e, -127))
    v = torch.where(bad, torch.zeros_like(b), b) * power(-e)
    step = torch.where(v.abs() < 2, 0.5, torch.where(v.abs() < 4, 1.0, 2.0)).to(v.dtype)
    r = ((v / step).round() * step).clamp(-6, 6)            # torch.round: ties to even, which is the even code in each range
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    codes = torch.bucketize(r.abs(), grid) + 8 * torch.signbit(v).long()
    scales = torch.where(bad, torch.full_like(e, 255), e + 127).squeeze(-1)
    return codes.flatten(-2), scales, dequantize(codes.flatten(-2), scales)


def power(e):
    """2^e in float64, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def dequantize(codes, scales):
    """float64 values of codes [..., k] and scales [..., k / 32]; scale 255: NaN."""
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=codes.device)
    mag = grid[(codes & 7).long()]
    v = torch.where(codes >= 8, -mag, mag).unflatten(-1, (-1, BLOCK))
    s = torch.where(scales == 255, torch.full(scales.shape, float("nan"), dtype=torch.float64, device=codes.device),
                    power(scales.long() - 127))
    return (v * s.unsqueeze(-1)).flatten(-2)


def pack(codes):
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).to(torch.uint8)


def product(xq, wq):
    """(x . w^T, the sum of the magnitudes of its terms)."""
    return xq @ wq.mT, xq.abs() @ wq.abs().mT


def product_slack(size, k):
    """How far a float32 sum of k exact products may be from theirs.  An instruction adds 64 products to the accumulator: every
    addition rounds or cuts to 24 bits, at most 2^-23 of what it adds up, which is at most `size`, the sum of magnitudes; the
    64 products inside an instruction add up in a tree of six levels or one aligned sum, so 6 + 1 such steps for the first and one
    more for each of the others; partial sums of a K range split over up to eight blocks: seven more additions."""
    return (-(-k // 64) + 6 + 7) * 2.0 ** -23 * size


def glu(g, u, limit, alpha, shift):
    if limit > 0:
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    if alpha == 0:
        return g * torch.sigmoid(1.5957691216057308 * (g + 0.044715 * g ** 3)) * (u + shift)
    return g * torch.sigmoid(alpha * g) * (u + shift)


def gated(xq, wg, wu, form):
    """(glu, its slack) for the float32 path: both products' slack through the unit (its gate's factor rises by at most 1.13 for
    silu and the tanh form of gelu at alpha 1, likewise for other alphas: z sigmoid(alpha z) is z sigmoid(z) scaled in both directions;
    the clamps do not widen anything), and 2^-16 of the result for the exponential of the fast unit (2 ulp plus 2^-23 of an argument
    of at most 88, where it matters), the division and the products."""
    (g, sg), (u, su) = product(xq, wg), product(xq, wu)
    limit, alpha, shift = form
    out = glu(g, u, *form)
    dg, du = product_slack(sg, xq.shape[-1]), product_slack(su, xq.shape[-1])
    gate = glu(g, torch.ones_like(u) - shift, *((0.0,) + tuple(form[1:]))) if limit == 0 else glu(g.clamp(max=limit), torch.ones_like(u) - shift, 0.0, alpha, shift)
    uu = (u.clamp(-limit, limit) if limit > 0 else u) + shift
    return out, 1.13 * dg * (uu.abs() + du) + gate.abs() * du + 2.0 ** -16 * out.abs()


def near(got, want, slack, what=""):
    """got against float64 `want`: within `slack` and half a step of got's own type (2^-8 of the value in bfloat16, 2^-24 in float32)."""
    half = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}[got.dtype]
    g = got.double()
    assert torch.equal(torch.isnan(g), torch.isnan(want)), what + ": not the same places are NaN"
    tol = slack + half * (want.abs() + slack) + 1e-37
    bad = ~((g - want).abs() <= tol) & ~torch.isnan(want)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}, " \
        f"worst {float(((g - want).abs() / tol)[~torch.isnan(want)].max()):.3g} of the slack"
