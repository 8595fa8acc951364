"""Microscaled 4-bit numbers on the GPU: rows to codes and scales and back, products, gated products, and those of routed experts,
against the definition in float64 (plain_mx4.py has the tolerances)."""
import pytest
import torch

import plain_mx4 as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SWIGLU, CLAMPED, GELU = (0.0, 1.0, 0.0), (7.0, 1.702, 1.0), (0.0, 0.0, 0.0)


def ops():
    from rllm_b200.csrc import ops as o
    return o


def rnd(*shape, seed, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def weight(*shape, seed):
    """(Mx4Matrix, values in float64)"""
    w = rnd(*shape, seed=seed) * shape[-1] ** -0.5
    codes, scales, values = plain.quantize(w)
    return ops().Mx4Matrix.from_blocks(plain.pack(codes), scales.to(torch.uint8)), values


@pytest.fixture(params=["by rule", "one SM a tile", "two SMs a tile"])
def many(request, monkeypatch):
    """The kernels that the sizes lead to; or those for many rows, whatever the sizes."""
    if request.param != "by rule":
        monkeypatch.setattr(ops(), "mx4_few_rows", lambda *a: None)
        monkeypatch.setattr(ops(), "mx4_pairs", lambda *a: request.param.startswith("two"))
    return request.param


# ---------------------------------------------------------------- rows to codes and back

def same(q, x):
    codes, scales, values = plain.quantize(x)
    assert torch.equal(q.codes.long(), plain.pack(codes).long())
    assert torch.equal(q.block_scales().long(), scales)
    again = ops().Mx4Matrix.from_blocks(q.codes, q.block_scales())
    assert torch.equal(again.scales, q.scales)                   # zeros behind the last row and the last block
    for dt in (torch.float32, torch.bfloat16):
        got = q.dequantize(dt).double()
        assert torch.equal(torch.isnan(got), torch.isnan(values))
        assert torch.equal(got.nan_to_num(), values.nan_to_num())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,k", [(1, 32), (1, 4096), (3, 96), (127, 288), (129, 256), (33, 2080), (300, 1024)])
def test_quantize(rows, k, dtype):
    x = rnd(rows, k, seed=rows + k, dtype=dtype) * torch.exp(rnd(rows, 1, seed=5)).to(dtype)
    same(ops().mx4_quantize(x), x)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_strides_and_addresses(dtype):
    base = rnd(40, 200, seed=3, dtype=dtype)
    for x in (base[:, :64], base[3:, 5:69], base[:, 1:193], base.view(-1)[1:7937].view(-1, 128)[:, :96]):
        same(ops().mx4_quantize(x), x)


@pytest.mark.parametrize("shape", [(3, 5, 64), (2, 128, 288), (2, 3, 256, 32), (4, 1, 96)])
def test_quantize_stacks(shape):
    x = rnd(*shape, seed=9)
    same(ops().mx4_quantize(x), x)


def test_quantize_borders():
    """Ties, the largest and smallest numbers, subnormal ones, empty blocks, infinities and NaN."""
    grid = torch.tensor([0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7.9])
    near = torch.cat([grid, -grid])
    blocks = [near * 2.0 ** e for e in (0, -1, 60, 124, -100, -127, -140, -148)]
    blocks += [torch.nextafter(near, torch.full_like(near, 9.0)), torch.nextafter(near, torch.full_like(near, -9.0))]
    blocks += [torch.zeros(32), -torch.zeros(32), torch.full((32,), 3.4e38), torch.full((32,), 2.0 ** -149)]
    for bad in (float("inf"), float("-inf"), float("nan")):
        b = near.clone()
        b[7] = bad
        blocks += [b, near]
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.cat(blocks).to(dtype).reshape(2, -1).to(DEV)
        same(ops().mx4_quantize(x), x)


def test_every_code_and_scale():
    codes = torch.arange(16, device=DEV).repeat(2)[None, None].expand(2, 256, 32).reshape(2, 256 * 32)
    scales = torch.arange(256, device=DEV)[None].expand(2, 256)
    q = ops().Mx4Matrix.from_blocks(plain.pack(codes), scales.to(torch.uint8).contiguous())
    want = plain.dequantize(codes, scales)
    got = q.dequantize(torch.float32).double()
    most = 3.4028234663852886e38                                  # 2^127 times 2 and more: infinite in 32 bits
    want = torch.where(want.abs() > most, want.sign() * float("inf"), want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))
    assert torch.equal(q.dequantize(torch.bfloat16).double().nan_to_num(7.0), want.nan_to_num(7.0))


# ---------------------------------------------------------------- products

SHAPES = [(1, 1, 32), (1, 128, 256), (2, 200, 64), (5, 130, 288), (8, 4096, 1024), (16, 257, 4096), (31, 96, 12288), (33, 1000, 2080),
          (64, 640, 512), (65, 129, 544), (128, 256, 256), (129, 300, 96), (257, 513, 1056), (300, 1000, 2080), (1030, 384, 320)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear(m, n, k, many):
    x = rnd(m, k, seed=1, dtype=torch.bfloat16)
    w, values = weight(n, k, seed=2)
    want, size = plain.product(plain.quantize(x)[2], values)
    slack = plain.product_slack(size, k)
    plain.near(ops().linear(x, w), want, slack, "bfloat16")
    plain.near(ops().linear(x, w, out_dtype=torch.float32), want, slack, "float32")
    c = rnd(m, n, seed=3)
    got = ops().linear(x, w, out=c.clone(), accumulate=True)
    # one more rounding, of the sum
    plain.near(got, want + c.double(), slack + 2.0 ** -24 * (want.abs() + c.double().abs()), "added")
    w.settled = True
    torch.cuda.synchronize()
    assert torch.equal(ops().linear(x, w, out=c.clone(), accumulate=True), got)
    ops().check_device_errors()


@pytest.mark.parametrize("m,n,k", [(3, 40, 96), (70, 300, 288), (140, 130, 512)])
def test_linear_strides_and_margins(m, n, k, many):
    """Rows of wider matrices in and out, at addresses that no 16 bytes divide; what lies beside the output stays."""
    w, values = weight(n, k, seed=2)
    for dtype in (torch.bfloat16, torch.float32):
        base = rnd(m, k + 13, seed=4, dtype=dtype)
        x = base[:, 5:5 + k]
        want, size = plain.product(plain.quantize(x)[2], values)
        for dt in (torch.bfloat16, torch.float32):
            out = torch.full((m + 2, n + 7), 123.0, dtype=dt, device=DEV)
            ops().linear(x, w, out=out[1:-1, 3:3 + n])
            plain.near(out[1:-1, 3:3 + n], want, plain.product_slack(size, k))
            out[1:-1, 3:3 + n] = 123.0
            assert bool((out == 123.0).all())


@pytest.mark.parametrize("m", [2, 100])
def test_linear_not_finite(m, many):
    """A row with a NaN or an infinity gives a row of NaN, a weight's block that is not a number a column; nothing else changes."""
    n, k = 150, 320
    x = rnd(m, k, seed=1, dtype=torch.bfloat16)
    x[1, 40] = float("inf")
    codes, scales, _ = plain.quantize(rnd(n, k, seed=2))
    scales[7, 3] = 255
    w = ops().Mx4Matrix.from_blocks(plain.pack(codes), scales.to(torch.uint8))
    want, size = plain.product(plain.quantize(x)[2], plain.dequantize(codes, scales))
    assert bool(torch.isnan(want[1]).all()) and bool(torch.isnan(want[:, 7]).all()) and not torch.isnan(want[0, 0])
    plain.near(ops().linear(x, w, out_dtype=torch.float32), want, plain.product_slack(size, k).nan_to_num())


@pytest.mark.parametrize("m", [3, 130])
def test_linear_scales_far_apart(m, many):
    """Scales from 2^-127 to 2^100: a block's power of two counts wherever it lies."""
    n, k = 140, 512
    g = torch.Generator().manual_seed(1)
    codes = torch.randint(0, 16, (n, k), generator=g).to(DEV)
    scales = torch.randint(0, 20, (n, k // 32), generator=g).to(DEV)
    w = ops().Mx4Matrix.from_blocks(plain.pack(codes), scales.to(torch.uint8))
    x = (rnd(m, k, seed=3) * 2.0 ** 100).to(torch.bfloat16)
    want, size = plain.product(plain.quantize(x)[2], plain.dequantize(codes, scales))
    plain.near(ops().linear(x, w, out_dtype=torch.float32), want, plain.product_slack(size, k))


@pytest.mark.parametrize("form", [None, CLAMPED, GELU])
@pytest.mark.parametrize("m,F,k", [(1, 1, 32), (1, 96, 256), (8, 1536, 1024), (16, 130, 288), (40, 200, 2080), (65, 257, 544), (300, 1000, 512)])
def test_gated(m, F, k, form, many):
    h = rnd(m, k, seed=1, dtype=torch.bfloat16)
    w, values = weight(2, F, k, seed=2)
    if form == CLAMPED:
        h, values, w = h * 4, values, w                       # values beyond the limit on both sides
    want, slack = plain.gated(plain.quantize(h)[2], values[0], values[1], form or SWIGLU)
    for dt in (torch.bfloat16, torch.float32):
        out = torch.full((m, F + 3), 5.0, dtype=dt, device=DEV)
        ops().gate_up_swiglu(h, w, out[:, :F], glu=form)
        plain.near(out[:, :F], want, slack, str(dt))
        assert bool((out[:, F:] == 5.0).all())
    ops().check_device_errors()


@pytest.mark.parametrize("m", [2, 100])
def test_gated_not_finite(m, many):
    """A row that is not a number stays one behind the clamps; so does a column whose gate or up row has a block that is not."""
    F, k = 96, 320
    h = rnd(m, k, seed=1, dtype=torch.bfloat16)
    h[1, 40] = float("nan")
    codes, scales, _ = plain.quantize(rnd(2, F, k, seed=2))
    scales[0, 7, 3] = scales[1, 9, 0] = 255
    w = ops().Mx4Matrix.from_blocks(plain.pack(codes), scales.to(torch.uint8))
    values = plain.dequantize(codes, scales)
    for form in (SWIGLU, CLAMPED):
        want, slack = plain.gated(plain.quantize(h)[2], values[0], values[1], form)
        assert bool(torch.isnan(want[1]).all()) and bool(torch.isnan(want[:, [7, 9]]).all()) and not torch.isnan(want[0, 0])
        out = torch.empty(m, F, device=DEV)
        plain.near(ops().gate_up_swiglu(h, w, out, glu=form), want, slack.nan_to_num())


# ---------------------------------------------------------------- routed experts

ROUTES = [(1, 1, 1, 0), (1, 4, 2, 0), (64, 4, 4, 2), (17, 40, 8, 1), (5, 7, 3, 1), (40, 16, 4, 2), (64, 3, 2, 0), (200, 16, 4, 1), (301, 5, 5, 0), (130, 64, 1, 1)]


def route(n, E, top, skew, seed):
    g = torch.Generator().manual_seed(seed)
    liked = -skew * torch.log1p(torch.arange(E).float())
    noise = -torch.log(-torch.log(torch.rand(n, E, generator=g).clamp(1e-6, 1 - 1e-6)))
    idx = (liked + noise).topk(top, -1).indices.to(torch.int32)
    return idx.to(DEV), torch.softmax(torch.randn(n, top, generator=g), -1).to(DEV)


@pytest.mark.parametrize("n,E,top,skew", ROUTES)
@pytest.mark.parametrize("d,F,form", [(256, 96, None), (288, 130, CLAMPED), (1024, 384, None)])
def test_experts_up(n, E, top, skew, d, F, form, many):
    idx, _ = route(n, E, top, skew, seed=n + E)
    h = rnd(n, d, seed=1, dtype=torch.bfloat16)
    w, values = weight(E, 2, F, d, seed=2)
    offsets, place = ops().moe_sort(idx, E)
    act = torch.full((n * top + 3, F), 5.0, dtype=torch.bfloat16, device=DEV)
    ops().mx4_experts_up(h, w, offsets, place, act[:n * top], glu=form)
    hq = plain.quantize(h)[2]
    for e in range(E):
        t, j = (idx == e).nonzero(as_tuple=True)
        if t.numel():
            want, slack = plain.gated(hq[t], values[e, 0], values[e, 1], form or SWIGLU)
            plain.near(act[place.view(n, top)[t, j].long()], want, slack, f"expert {e}")
    assert bool((act[n * top:] == 5.0).all())
    ops().check_device_errors()


@pytest.mark.parametrize("n,E,top,skew", ROUTES)
@pytest.mark.parametrize("F,d", [(96, 256), (160, 300), (384, 1024)])
def test_experts_down(n, E, top, skew, F, d, many):
    idx, wgt = route(n, E, top, skew, seed=n + E)
    offsets, place = ops().moe_sort(idx, E)
    act = rnd(n * top, F, seed=1, dtype=torch.bfloat16)
    w, values = weight(E, d, F, seed=2)
    y = torch.full((n * top + 3, d), 5.0, device=DEV)
    ops().mx4_experts_down(act, w, offsets, y[:n * top])
    assert bool((y[n * top:] == 5.0).all())
    aq, at = plain.quantize(act)[2], place.view(n, top).long()
    want, size = torch.zeros(n, d, dtype=torch.float64, device=DEV), torch.zeros(n, d, dtype=torch.float64, device=DEV)
    for e in range(E):
        t, j = (idx == e).nonzero(as_tuple=True)
        if t.numel():
            p, s = plain.product(aq[at[t, j]], values[e])
            plain.near(y[at[t, j]], p, plain.product_slack(s, F), f"expert {e}")
            want.index_add_(0, t, p * wgt.double()[t, j, None])
            size.index_add_(0, t, s * wgt.double()[t, j, None].abs())
    out = ops().moe_combine(y[:n * top], place, wgt, torch.empty(n, d, device=DEV))
    plain.near(out, want, plain.product_slack(size, F) + top * 2.0 ** -23 * size)
    ops().check_device_errors()


@pytest.mark.parametrize("n,E,top", [(1, 1, 1), (3, 256, 2), (700, 16, 4), (1000, 255, 8), (2000, 256, 1), (900, 300, 3), (5000, 2, 2),
                                     (64, 33, 4), (257, 256, 1), (256, 1, 8), (683, 128, 3), (8192, 128, 8), (65537, 7, 1), (33000, 256, 5)])
def test_sort_is_stable(n, E, top):
    """Pairs in the order of their experts, and within an expert in their own, with every number of experts a kernel takes."""
    idx = torch.randint(0, E, (n, top), generator=torch.Generator().manual_seed(n)).to(torch.int32).to(DEV)
    offsets, place = ops().moe_sort(idx, E)
    order = torch.sort(idx.flatten().long(), stable=True).indices
    want = torch.empty_like(order).scatter_(0, order, torch.arange(order.numel(), device=DEV))
    assert torch.equal(place.long(), want)
    count = torch.bincount(idx.flatten().long(), minlength=E)
    assert torch.equal(offsets.long(), torch.cat([count.new_zeros(1), count.cumsum(0)]))


# ---------------------------------------------------------------- as they are used

def test_products_in_a_graph_and_on_another_stream():
    """Two graphs captured from the same calls share nothing; replays see new inputs; another stream gives the same bits."""
    n, k, F = 260, 512, 192
    w, _ = weight(n, k, seed=1)
    g, _ = weight(2, F, k, seed=2)
    runs = []
    for m in (3, 70):
        x = torch.empty(m, k, dtype=torch.bfloat16, device=DEV)

        def go(x=x):
            act = torch.empty(x.shape[0], F, dtype=torch.bfloat16, device=DEV)
            return ops().linear(x, w, out_dtype=torch.float32), ops().gate_up_swiglu(x, g, act)
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            x.copy_(rnd(m, k, seed=9))
            go()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = go()
        runs.append((x, graph, out, go))
    for turn in (4, 5):
        for x, graph, out, go in runs:
            x.copy_(rnd(*x.shape, seed=turn))
        for x, graph, out, go in runs:
            graph.replay()
        torch.cuda.synchronize()
        for x, graph, out, go in runs:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                again = go()
            side.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, again))
    ops().check_device_errors()


def test_weights_quantized_right_before_their_product():
    """A product behind the kernel that makes its weight: nothing is read ahead of it."""
    k, n = 1024, 2048
    x = rnd(4, k, seed=1, dtype=torch.bfloat16)
    for seed in range(5):
        w = rnd(n, k, seed=10 + seed, dtype=torch.bfloat16)
        torch.cuda.synchronize()
        got = ops().linear(x, ops().mx4_quantize(w), out_dtype=torch.float32)
        want, size = plain.product(plain.quantize(x)[2], plain.quantize(w)[2])
        plain.near(got, want, plain.product_slack(size, k))


def test_feed_forward_chain():
    """The run of them as a layer makes it: gate and up, the second product added to the stream; then the experts' way there and back.
    Every step is held to the definition on what the step before left."""
    m, d, F, E, top = 37, 512, 416, 6, 2
    h, x = rnd(m, d, seed=1, dtype=torch.bfloat16), rnd(m, d, seed=2)
    wg, vg = weight(2, F, d, seed=3)
    wd, vd = weight(d, F, seed=4)
    act = torch.empty(m, F, dtype=torch.bfloat16, device=DEV)
    ops().gate_up_swiglu(h, wg, act)
    want, slack = plain.gated(plain.quantize(h)[2], vg[0], vg[1], SWIGLU)
    plain.near(act, want, slack)
    stream = ops().linear(act, wd, out=x.clone(), accumulate=True)
    want, size = plain.product(plain.quantize(act)[2], vd)
    plain.near(stream, want + x.double(), plain.product_slack(size, F) + 2.0 ** -24 * (want.abs() + x.double().abs()))
    idx, wgt = route(m, E, top, 0, seed=5)
    eg, ed = ops().mx4_quantize(rnd(E, 2, F, d, seed=6) * d ** -0.5), ops().mx4_quantize(rnd(E, d, F, seed=7) * F ** -0.5)
    offsets, place = ops().moe_sort(idx, E)
    act = ops().mx4_experts_up(h, eg, offsets, place, torch.empty(m * top, F, dtype=torch.bfloat16, device=DEV))
    y = ops().mx4_experts_down(act, ed, offsets, torch.empty(m * top, d, device=DEV))
    out = ops().moe_combine(y, place, wgt, torch.empty(m, d, device=DEV))
    # each pair as two single products
    for t in (0, m - 1):
        total = torch.zeros(d, dtype=torch.float64, device=DEV)
        bound = torch.zeros(d, dtype=torch.float64, device=DEV)
        for j in range(top):
            e, p = int(idx[t, j]), int(place[t * top + j])
            pv, ps = plain.product(plain.quantize(act[p:p + 1])[2], ed.dequantize().double()[e])
            total += pv[0] * wgt[t, j].double()
            bound += ps[0] * wgt[t, j].double()
        plain.near(out[t], total, plain.product_slack(bound, F) + top * 2.0 ** -23 * bound)
    ops().check_device_errors()


@pytest.mark.parametrize("m", [3, 70, 200])
def test_offsets_beyond_32_bits(m, many):
    """Rows in and out 2^25 and more entries apart, so that the last ones lie beyond 2^31 entries; what lies beside them stays."""
    n, k, apart = 136, 320, (1 << 31) // (m - 1) + 64
    apart -= apart % 8
    x = torch.empty((m - 1) * apart + k, dtype=torch.bfloat16, device=DEV).as_strided((m, k), (apart, 1))
    x.copy_(rnd(m, k, seed=1))
    w, values = weight(n, k, seed=2)
    out = torch.zeros((m - 1) * apart + n, device=DEV).as_strided((m, n), (apart, 1))
    want, size = plain.product(plain.quantize(x.contiguous())[2], values)
    plain.near(ops().linear(x, w, out=out), want, plain.product_slack(size, k))
    assert float(out[0].abs().sum()) == float(out.as_strided((apart,), (1,)).abs().sum())
    ops().linear(x, w, out=out, accumulate=True)
    plain.near(out, 2 * want, 2 * plain.product_slack(size, k))
    q = ops().mx4_quantize(x)
    assert torch.equal(q.dequantize().double(), plain.quantize(x.contiguous())[2])


@pytest.mark.parametrize("m", [1, 40, 129])
def test_weights_beyond_32_bits(m):
    """Codes of more than 2^32 bytes: the last columns come from the last rows."""
    n, k, tail = (1 << 20) + 200, 8256, 300
    codes = torch.zeros(n, k // 2, dtype=torch.uint8, device=DEV)
    scales = torch.full(ops().mx4_scale_shape(n, k), 127, dtype=torch.uint8, device=DEV)
    w = ops().Mx4Matrix(codes, scales)
    c = torch.randint(0, 16, (tail, k), generator=torch.Generator().manual_seed(1)).to(DEV)
    codes[-tail:] = plain.pack(c)
    x = rnd(m, k, seed=2, dtype=torch.bfloat16)
    values = plain.dequantize(c, torch.full((tail, k // 32), 127, device=DEV))
    want, size = plain.product(plain.quantize(x)[2], values)
    out = ops().linear(x, w, out_dtype=torch.float32)
    plain.near(out[:, -tail:], want, plain.product_slack(size, k))
    assert float(out[:, :-tail].abs().max()) == 0.0
    del out
    if m == 1:
        got = w.dequantize(torch.bfloat16)
        assert torch.equal(got[-tail:].double(), values) and not bool(got[:-tail].any())
        again = ops().mx4_quantize(got)                       # 17 GB in, rows beyond 2^32 entries
        assert torch.equal(again.dequantize(torch.bfloat16)[-tail:], got[-tail:])


def test_two_threads_at_once():
    """Products called from two threads, each on a stream of its own."""
    import threading
    w, values = weight(512, 768, seed=1)
    g, _ = weight(2, 320, 768, seed=2)
    xs = [rnd(m, 768, seed=m, dtype=torch.bfloat16) for m in (3, 90)]
    want = [(ops().linear(x, w), ops().gate_up_swiglu(x, g, torch.empty(x.shape[0], 320, dtype=torch.bfloat16, device=DEV))) for x in xs]
    torch.cuda.synchronize()
    wrong = []

    def go(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(200):
                a = ops().linear(xs[i], w)
                b = ops().gate_up_swiglu(xs[i], g, torch.empty(xs[i].shape[0], 320, dtype=torch.bfloat16, device=DEV))
                torch.cuda.current_stream().synchronize()
                if not (torch.equal(a, want[i][0]) and torch.equal(b, want[i][1])):
                    wrong.append(i)
    threads = [threading.Thread(target=go, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    ops().check_device_errors()


# ---------------------------------------------------------------- refusals

def test_refusals():
    o = ops()
    w, _ = weight(64, 128, seed=1)
    s, _ = weight(2, 64, 128, seed=1)
    x = rnd(4, 128, seed=1, dtype=torch.bfloat16)
    out = torch.empty(4, 64, device=DEV)
    bad = [
        lambda: o.mx4_quantize(rnd(3, 40, seed=1)),                              # not whole blocks
        lambda: o.mx4_quantize(rnd(3, 64, seed=1).half()),                       # a type that the kernels do not take
        lambda: o.mx4_quantize(rnd(64, 64, seed=1).t()),                         # entries of a row apart
        lambda: o.mx4_quantize(rnd(64, seed=1)),
        lambda: o.mx4_quantize(torch.randn(4, 64)),                              # on the host
        lambda: o.linear(rnd(4, 96, seed=1, dtype=torch.bfloat16), w),           # another length than the weight's
        lambda: o.linear(x.cpu(), w),
        lambda: o.linear(x, s),                                                  # a stack where one matrix is needed
        lambda: o.linear(x, w, out=torch.empty(5, 64, device=DEV)),
        lambda: o.linear(x, w, out=torch.empty(4, 65, device=DEV)),
        lambda: o.linear(x, w, out=torch.empty(64, 4, device=DEV).t()),
        lambda: o.linear(x, w, accumulate=True),
        lambda: o.linear(x, w, out=out.bfloat16(), accumulate=True),
        lambda: o.linear(x, w, out=out.half()),
        lambda: o.linear(x, w, out=torch.empty(1, 64, device=DEV).expand(4, 64)),   # rows on top of one another
        lambda: o.linear(x, w, out=out, accumulate=True, then_norm=(torch.ones(64, device=DEV), 1e-6)),
        lambda: o.gate_up_swiglu(x, w, out),
        lambda: o.gate_up_swiglu(x[:3], s, out),
        lambda: o.mx4_experts_down(x, w, torch.zeros(2, dtype=torch.int32, device=DEV), out),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(o.KernelError):
            call()
            pytest.fail(f"call {i} was not refused")
    e, _ = weight(3, 2, 64, 128, seed=1)
    idx = torch.tensor([[0, 2]] * 4, dtype=torch.int32, device=DEV)
    offsets, place = o.moe_sort(idx, 3)
    act = torch.empty(8, 64, dtype=torch.bfloat16, device=DEV)
    for args in ((x, e, offsets[:3], place, act), (x, e, offsets, place[:7], act), (x, e, offsets.long(), place, act),
                 (x, e, offsets, place, act[:7]), (x[:0], e, offsets, place, act), (x, s, offsets, place, act)):
        with pytest.raises(o.KernelError):
            o.mx4_experts_up(*args)
    # nothing to do
    assert o.linear(x[:0], w).shape == (0, 64)
    assert o.mx4_quantize(x[:0]).dequantize().shape == (0, 128)
    o.mx4_experts_up(x[:0], e, offsets, place[:0], act[:0])


def test_offsets_that_do_not_rise(many):
    """Offsets that are no offsets give rows without meaning, but no access outside the buffers."""
    o = ops()
    w, _ = weight(4, 2, 64, 128, seed=1)
    x = rnd(300, 128, seed=1, dtype=torch.bfloat16)
    place = torch.arange(300, dtype=torch.int32, device=DEV)
    act = torch.empty(302, 64, dtype=torch.bfloat16, device=DEV)
    act[300:] = 5.0
    for off in ([0, 300, 0, 300, 300], [0, 1000, -5, 2000, 300], [300, 200, 100, 50, 0], [7, 7, 7, 7, 7]):
        o.mx4_experts_up(x, w, torch.tensor(off, dtype=torch.int32, device=DEV), place, act[:300])
        bad = place.clone()
        bad[5], bad[9] = 100000, -1
        o.mx4_experts_up(x, w, torch.tensor([0, 100, 100, 250, 300], dtype=torch.int32, device=DEV), bad, act[:300])
    torch.cuda.synchronize()
    assert bool((act[300:] == 5.0).all())
    o.check_device_errors()


FEW = [(m, bn, n, k, s) for m, bn in ((1, 16), (2, 16), (7, 16), (16, 16), (1, 32), (17, 32), (32, 32), (40, 64), (64, 64), (90, 128), (128, 128),
                                      (300, 128), (70, 0)) for n, k in ((200, 2080), (128, 256), (1000, 8192)) for s in (1, 2, 4, 8)
       if s <= -(-k // 256) and (bn or s == 1)]


@pytest.mark.parametrize("m,bn,n,k,splits", FEW)
def test_few_rows_shared_k(m, bn, n, k, splits):
    """Every kernel for few rows with every way to share K; float32 rows; a ring that wraps.  bn 0: the kernel for many rows."""
    o = ops()
    few, few_gated = (bn, splits) if bn else False, (bn, min(splits, 4)) if 0 < bn < 128 else False
    w, values = weight(n, k, seed=1)
    g, gv = weight(2, n, k, seed=2)
    for dtype in (torch.bfloat16, torch.float32):
        x = rnd(m, k, seed=3, dtype=dtype)
        xq = plain.quantize(x)[2]
        want, size = plain.product(xq, values)
        slack = plain.product_slack(size, k)
        out = torch.full((m + 1, n + 2), 5.0, device=DEV)
        o._mx4_product(x, w, out[:m, :n], (), o.EPI_STORE, SWIGLU, "", few)
        plain.near(out[:m, :n], want, slack)
        c = rnd(m, n, seed=4)
        out[:m, :n] = c
        o._mx4_product(x, w, out[:m, :n], (), o.EPI_ACCUM, SWIGLU, "", few)
        plain.near(out[:m, :n], want + c.double(), slack + 2.0 ** -24 * (want.abs() + c.double().abs()))
        out[:m, :n] = 5.0
        assert bool((out == 5.0).all())
        act = torch.empty(m, n, dtype=torch.bfloat16, device=DEV)
        g.settled = True
        o._mx4_product(x, g, act, (2,), o.EPI_SWIGLU, CLAMPED, "", few_gated)
        plain.near(act, *plain.gated(xq, gv[0], gv[1], CLAMPED))
    o.check_device_errors()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m", [3, 40, 300])
def test_gated_far_below_zero(m, dtype, many):
    """Gates whose sigmoid has a denominator between 2^126 and 2^128: small results, not zeros.  The products are sums of a few small whole
    and half numbers, exact in any order; what may be off is e^88 by 2 + 1.173 * 88 ulp (of 2^-23), its argument with a factor by half a step of
    88, and six more roundings and the division's 2 ulp: 2^-15 of the result covers them, with the output's half step."""
    k, F = 64, 200
    for form, x, w in ((None, (6, 6, 4, 0), (6, 6, 4, 0)), (CLAMPED, (6, 4, 6, 0.5), (6, 3, 0.5, 1))):
        h = torch.zeros(m, k, dtype=torch.bfloat16, device=DEV)
        h[:, :4] = torch.tensor(x, dtype=torch.bfloat16)
        up = torch.zeros(F, k, device=DEV)
        up[:, :4] = torch.tensor(w, dtype=torch.float32)
        up[5:] *= 0.5                                             # (the others' gates are moderate)
        got = ops().gate_up_swiglu(h, ops().mx4_quantize(torch.stack([-up, up])), torch.empty(m, F, dtype=dtype, device=DEV), glu=form)
        y = (h.double() @ up.double().T)
        limit, alpha, shift = form or SWIGLU
        alpha = float(torch.tensor(alpha, dtype=torch.float32))
        gate, u = -y, y.clamp(max=limit) if limit else y
        want = gate / (1 + torch.exp(-alpha * gate)) * (u + shift)
        assert 87.4 < -alpha * float(gate[0, 0]) < 88.7
        half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
        assert bool(((got.double() - want).abs() <= (2.0 ** -15 + half) * want.abs()).all()), (got[0, 0], want[0, 0])


@pytest.mark.parametrize("m,bn,splits", [(8, 16, 8), (16, 16, 4), (13, 16, 1), (32, 32, 4), (33, 64, 4), (64, 64, 1), (128, 128, 4), (300, 128, 2), (300, 0, 1)])
def test_a_row_alone_and_among_others(m, bn, splits, monkeypatch):
    """With the same kernel and the same number of CTAs that share K a row's bits do not depend on the rows around it: the sizes decide the
    order of the sums, and which rows stand where does not."""
    o, n, k = ops(), 300, 4096
    x = rnd(m, k, seed=1, dtype=torch.bfloat16) * torch.exp(2 * rnd(1, k, seed=4)).to(torch.bfloat16)
    w, _ = weight(n, k, seed=2)
    g, _ = weight(2, n, k, seed=3)
    for pairs in (False, True) if not bn else (False,):          # (the gated product of 128 and more rows has no kernel for few)
        monkeypatch.setattr(o, "mx4_pairs", lambda *a: pairs)
        few, few_gated = (bn, splits) if bn else False, (bn, min(splits, 4)) if 0 < bn < 128 else False

        def both(rows):
            out, act = torch.empty(rows.shape[0], n, device=DEV), torch.empty(rows.shape[0], n, device=DEV)
            o._mx4_product(rows, w, out, (), o.EPI_STORE, SWIGLU, "", few)
            o._mx4_product(rows, g, act, (2,), o.EPI_SWIGLU, SWIGLU, "", few_gated)
            return out, act
        whole = both(x)
        for r in (0, m // 2, m - 1):
            assert all(torch.equal(a[0], b[r]) for a, b in zip(both(x[r:r + 1]), whole))
        turn = torch.arange(m - 1, -1, -1, device=DEV)
        assert all(torch.equal(a[turn], b) for a, b in zip(both(x[turn]), whole))
        assert all(torch.equal(a, b) for a, b in zip(both(x), whole))
    o.check_device_errors()


@pytest.mark.parametrize("n,top", [(4, 8), (16, 8), (64, 4)])
def test_many_experts_with_few_rows_each(n, top):
    """256 experts: few pairs through the kernel for few rows, more of them through the tiles for many, as the sizes lead."""
    E, d, F = 256, 1024, 96
    idx, _ = route(n, E, top, 0, seed=n)
    offsets, place = ops().moe_sort(idx, E)
    g = torch.Generator(device=DEV).manual_seed(1)
    used = idx.flatten().unique().tolist()
    w_up, w_down = (ops().mx4_quantize(torch.randn(s, generator=g, device=DEV) * s[-1] ** -0.5) for s in ((E, 2, F, d), (E, d, F)))
    h = rnd(n, d, seed=1, dtype=torch.bfloat16)
    act = ops().mx4_experts_up(h, w_up, offsets, place, torch.empty(n * top, F, dtype=torch.bfloat16, device=DEV))
    y = ops().mx4_experts_down(act, w_down, offsets, torch.empty(n * top, d, device=DEV))
    up, down = w_up.dequantize(), w_down.dequantize()
    hq, aq = plain.quantize(h)[2], plain.quantize(act)[2]
    for e in used:
        t, j = (idx == e).nonzero(as_tuple=True)
        at = place.view(n, top)[t, j].long()
        plain.near(act[at], *plain.gated(hq[t], up[e, 0].double(), up[e, 1].double(), SWIGLU), f"up {e}")
        want, size = plain.product(aq[at], down[e].double())
        plain.near(y[at], want, plain.product_slack(size, F), f"down {e}")
    ops().check_device_errors()
