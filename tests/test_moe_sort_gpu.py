"""Pairs that name no expert: `moe_sort` gives them no place, and what follows leaves them out."""
import pytest
import torch

import plain_mx4 as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

# few pairs, one block, a cluster of blocks, and more experts than those take
SIZES = [(1, 3, 2), (40, 16, 4), (250, 300, 1), (300, 16, 4), (512, 256, 4), (700, 7, 3), (2000, 64, 2), (1500, 300, 3), (9000, 128, 8)]


def ops():
    from rllm_b200.csrc import ops as o
    return o


def route(n, E, top, every):
    """idx with one pair in `every` (1: all of them) outside 0 .. E - 1."""
    g = torch.Generator().manual_seed(n + E)
    idx = torch.randint(0, E, (n, top), generator=g)
    none = torch.tensor([-1, E, E + 1, 2 ** 31 - 1, -2 ** 31])[torch.randint(0, 5, (n, top), generator=g)]
    out = torch.rand(n, top, generator=g) < (2.0 if every == 1 else 1.0 / every)
    return torch.where(out, none, idx).to(torch.int32).to(DEV)


def places(idx, E):
    """(offsets, place) by sorting."""
    e = idx.flatten().long()
    ok = ((e >= 0) & (e < E)).nonzero().flatten()
    order = ok[torch.sort(e[ok], stable=True).indices]
    place = torch.full_like(e, -1)
    place[order] = torch.arange(order.numel(), device=e.device)
    count = torch.bincount(e[ok], minlength=E)
    return torch.cat([count.new_zeros(1), count.cumsum(0)]), place


@pytest.mark.parametrize("every", [1, 3, 50])
@pytest.mark.parametrize("n,E,top", SIZES)
def test_sort(n, E, top, every):
    idx = route(n, E, top, every)
    junk = [torch.full((idx.numel(),), 77, dtype=torch.int32, device=DEV) for _ in range(4)]      # (what an allocation then finds)
    del junk
    offsets, place = ops().moe_sort(idx, E)
    want_offsets, want = places(idx, E)
    assert torch.equal(offsets.long(), want_offsets) and torch.equal(place.long(), want)


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.float32, 64), (torch.bfloat16, 33), (torch.float32, 33)])
@pytest.mark.parametrize("n,E,top", SIZES[1:7])
def test_rows_there_and_back(n, E, top, dtype, d):
    idx = route(n, E, top, 3)
    offsets, place = ops().moe_sort(idx, E)
    last = int(offsets[-1])
    g = torch.Generator().manual_seed(1)
    h = torch.randn(n, d, generator=g).to(dtype).to(DEV)
    weight = torch.rand(n, top, generator=g).to(DEV)
    rows = torch.full((n * top, d), 9.0, dtype=dtype, device=DEV)
    given = torch.full((n * top,), 9.0, device=DEV)
    ops().moe_gather_rows(h, place, rows, top, weight, given)
    ok = place >= 0
    src = torch.arange(n * top, device=DEV)[ok]
    assert torch.equal(rows[place[ok].long()], h[src // top]) and torch.equal(given[place[ok].long()], weight.flatten()[ok])
    assert bool((rows[last:] == 9.0).all()) and bool((given[last:] == 9.0).all())
    # pairs without a place add nothing, whatever their weight; the rows behind the last place are not read
    y = torch.randn(n * top, d, generator=g).to(DEV)
    y[last:] = float("nan")
    bad = weight.clone()
    bad.view(-1)[~ok] = float("nan")
    shared = torch.randn(n, d, generator=g).to(DEV)
    for wt, sh in ((bad, None), (bad, shared), (None, None)):
        out = ops().moe_combine(y, place, wt, torch.empty(n, d, device=DEV), sh, top_k=top)
        terms = torch.zeros(n * top, d, dtype=torch.float64, device=DEV)
        terms[ok] = y[place[ok].long()].double() * (1.0 if wt is None else weight.flatten()[ok].double()[:, None])
        terms = terms.view(n, top, d)
        want, size = terms.sum(1), terms.abs().sum(1)
        if sh is not None:
            want, size = want + sh.double(), size + sh.double().abs()
        # a product and an addition a term, each off by 2^-24 of at most the sum of magnitudes; one more addition for the shared row
        assert bool(((out.double() - want).abs() <= (2 * top + 1) * 2.0 ** -24 * size).all())


@pytest.mark.parametrize("n,E,top", [(9, 4, 2), (40, 16, 4), (200, 5, 3), (700, 7, 3)])
def test_products_of_4_bit_numbers(n, E, top):
    o, d, F = ops(), 256, 96
    idx = route(n, E, top, 3)
    offsets, place = o.moe_sort(idx, E)
    g = torch.Generator().manual_seed(2)
    h, weight = torch.randn(n, d, generator=g).bfloat16().to(DEV), torch.rand(n, top, generator=g).to(DEV)
    up, down = (torch.randn(*s, generator=g).to(DEV) * s[-1] ** -0.5 for s in ((E, 2, F, d), (E, d, F)))
    act = torch.full((n * top, F), 5.0, dtype=torch.bfloat16, device=DEV)
    o.mx4_experts_up(h, o.mx4_quantize(up), offsets, place, act)
    vu, vd, hq = plain.quantize(up)[2], plain.quantize(down)[2], plain.quantize(h)[2]
    last = int(offsets[-1])
    for e in range(E):
        t, j = (idx == e).nonzero(as_tuple=True)
        if t.numel():
            want, slack = plain.gated(hq[t], vu[e, 0], vu[e, 1], (0.0, 1.0, 0.0))
            plain.near(act[place.view(n, top)[t, j].long()], want, slack, f"expert {e}")
    act[last:] = 0.0
    y = torch.full((n * top, d), float("nan"), device=DEV)
    o.mx4_experts_down(act, o.mx4_quantize(down), offsets, y)
    out = o.moe_combine(y, place, weight, torch.empty(n, d, device=DEV))
    aq = plain.quantize(act)[2]
    want, size = torch.zeros(n, d, dtype=torch.float64, device=DEV), torch.zeros(n, d, dtype=torch.float64, device=DEV)
    for e in range(E):
        t, j = (idx == e).nonzero(as_tuple=True)
        if t.numel():
            p, s = plain.product(aq[place.view(n, top)[t, j].long()], vd[e])
            want.index_add_(0, t, p * weight.double()[t, j, None])
            size.index_add_(0, t, s * weight.double()[t, j, None])
    plain.near(out, want, plain.product_slack(size, F) + top * 2.0 ** -23 * size)
    o.check_device_errors(DEV)
