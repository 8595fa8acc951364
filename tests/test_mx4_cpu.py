"""What of the microscaled 4-bit numbers needs no GPU: the layout of the scales, and what is refused."""
import pytest
import torch

import plain_mx4 as plain
from rllm_b200.csrc import ops


@pytest.mark.parametrize("lead,n,k", [((), 1, 32), ((), 130, 288), ((2,), 128, 256), ((3, 2), 5, 544)])
def test_scale_layout(lead, n, k):
    g = torch.Generator().manual_seed(1)
    codes = torch.randint(0, 256, (*lead, n, k // 2), generator=g).to(torch.uint8)
    scales = torch.randint(0, 256, (*lead, n, k // 32), generator=g).to(torch.uint8)
    m = ops.Mx4Matrix.from_blocks(codes, scales)
    assert m.shape == (*lead, n, k) and m.scales.shape == (*lead, *ops.mx4_scale_shape(n, k))
    assert torch.equal(m.block_scales(), scales)
    tiles, rows = m.scales.view(-1, *m.scales.shape[-5:]), scales.view(-1, n, k // 32)
    for i in range(rows.shape[0]):
        for r in range(0, n, 7):
            for b in range(k // 32):
                assert tiles[i, r // 128, b // 4, r % 32, r // 32 % 4, b % 4] == rows[i, r, b]
    assert int(m.scales.long().sum()) == int(scales.long().sum())          # zeros elsewhere


def test_refusals():
    codes = torch.zeros(4, 32, dtype=torch.uint8)
    scales = torch.zeros(ops.mx4_scale_shape(4, 64), dtype=torch.uint8)
    ops.Mx4Matrix(codes, scales)
    for c, s in ((codes.int(), scales), (codes, scales.float()), (codes[0], scales), (codes, scales[0]), (codes[:, :24], scales),
                 (torch.zeros(4, 20, dtype=torch.uint8), scales), (torch.zeros(4, 0, dtype=torch.uint8), scales),
                 (torch.zeros(129, 32, dtype=torch.uint8), scales), (torch.zeros(32, 4, dtype=torch.uint8).t(), scales)):
        with pytest.raises(ops.KernelError):
            ops.Mx4Matrix(c, s)
    m = ops.Mx4Matrix(codes, scales)
    for call in (lambda: m.dequantize(), lambda: ops.mx4_quantize(torch.zeros(4, 64)),
                 lambda: ops.linear(torch.zeros(4, 64, dtype=torch.bfloat16), m)):
        with pytest.raises(ops.KernelError):                             # there is no CPU path
            call()


def test_refusals_of_experts():
    """Sorted rows need their order: without it the products would take all rows for those of one matrix."""
    up = ops.mx4_scale_shape(4, 64)
    w_up = ops.Mx4Matrix(torch.zeros(3, 2, 4, 32, dtype=torch.uint8), torch.zeros(3, 2, *up, dtype=torch.uint8))
    w_down = ops.Mx4Matrix(torch.zeros(3, 4, 32, dtype=torch.uint8), torch.zeros(3, *up, dtype=torch.uint8))
    h, act = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(4, 4, dtype=torch.bfloat16)
    place = torch.arange(4, dtype=torch.int32)
    for call in (lambda: ops.mx4_experts_up(h, w_up, None, place, act), lambda: ops.mx4_experts_up(h, w_up, None, None, act),
                 lambda: ops.mx4_experts_down(torch.zeros(4, 64, dtype=torch.bfloat16), w_down, None, act)):
        with pytest.raises(ops.KernelError, match="offsets is missing"):
            call()


def test_refusal_of_unplaced_rows(monkeypatch):
    monkeypatch.setattr(ops, "_mx4_current", lambda *t: None)               # (as on a GPU)
    up = ops.mx4_scale_shape(4, 64)
    w = ops.Mx4Matrix(torch.zeros(3, 2, 4, 32, dtype=torch.uint8), torch.zeros(3, 2, *up, dtype=torch.uint8))
    act, offsets = torch.zeros(4, 4, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ops.KernelError, match="place is missing"):
        ops.mx4_experts_up(torch.zeros(2, 64, dtype=torch.bfloat16), w, offsets, None, act)


def test_plain_rounding():
    """The oracle itself: ties to the even code, at most 6, the scale of a block."""
    x = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9, -0.25, -0.75, -5.0, 4.0] + [0.0] * 20)
    _, scales, v = plain.quantize(x[None])
    assert scales.tolist() == [[127]]
    assert v[0, :12].tolist() == [0, 1, 1, 2, 2, 4, 4, 6, 0, -1, -4, 4]
    _, scales, v = plain.quantize((x * 2.0 ** -130)[None])
    assert scales.tolist() == [[0]] and v[0, 11] == 2.0 ** -128


def test_refusal_of_sizes_beyond_31_bits(monkeypatch):
    """The launchers take rows as 32-bit numbers: more of them would arrive as another number, or as none."""
    monkeypatch.setattr(ops, "_mx4_current", lambda *t: None)               # (as on a GPU)
    many = 1 << 31
    x = torch.zeros(1, 64, dtype=torch.bfloat16).expand(many, 64)
    w = ops.Mx4Matrix(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(ops.mx4_scale_shape(4, 64), dtype=torch.uint8))
    out = torch.empty(many, 4, device="meta")
    for call in (lambda: ops.mx4_quantize(x), lambda: ops.mx4_linear(x, w, out)):
        with pytest.raises(ops.KernelError, match="2147483648 rows"):
            call()
    for lead, n in (((), many), ((2,), many // 2), ((1 << 20, 2), 1 << 10)):
        codes = torch.empty(*lead, n, 32, dtype=torch.uint8, device="meta")
        scales = torch.empty(*lead, *ops.mx4_scale_shape(n, 64), dtype=torch.uint8, device="meta")
        with pytest.raises(ops.KernelError, match="2147483648 rows"):
            ops.Mx4Matrix(codes, scales)
    monkeypatch.setattr(ops, "_need_cuda", lambda *t: None)
    with pytest.raises(ops.KernelError, match="2147483648 pairs"):
        ops.moe_sort(torch.empty(many // 2, 2, dtype=torch.int32, device="meta"), 4)


def test_few_rows_of_many_experts():
    """The product of few rows keeps to as many CTAs as the SMs go through a few times."""
    for pairs, n, k, gated, experts, few in ((64, 2048, 512, False, 256, True), (128, 2048, 512, False, 256, False),
                                             (128, 512, 2048, True, 256, True), (64, 4096, 1536, False, 128, True),
                                             (128, 4096, 1536, False, 128, False), (32, 768, 2048, True, 16, True), (129, 768, 2048, True, 16, False)):
        got = ops.mx4_few_rows(pairs, n, k, gated, True, experts)
        assert (got is not None) == few, (pairs, n, k, gated, experts)
        if few:
            assert got[0] == 16 and -(-n // 128) * (2 if gated else 1) * min(experts, pairs) <= 14 * 148
