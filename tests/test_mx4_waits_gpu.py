"""The bounded waits of the products of 4-bit numbers: their limit can be set, a wait that runs out is reported, and the products
run on afterwards."""
import time

import pytest
import torch

import plain_mx4 as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def check_product(ops, m):
    g = torch.Generator().manual_seed(m)
    x, w = torch.randn(m, 512, generator=g).bfloat16().to(DEV), torch.randn(4200, 512, generator=g).to(DEV)
    got = ops.linear(x, ops.mx4_quantize(w), out_dtype=torch.float32)
    want, size = plain.product(plain.quantize(x)[2], plain.quantize(w)[2])
    plain.near(got, want, plain.product_slack(size, 512))
    ops.check_device_errors(DEV)


@pytest.mark.parametrize("library,code", [("mx4", 31), ("mx4_rows", 35)])
def test_a_bounded_wait_runs_out(library, code):
    from rllm_b200.csrc import ops
    ops.check_device_errors(DEV)
    ops.set_wait_cycles(100_000, [library])
    try:
        torch.cuda.synchronize()
        t0 = time.time()
        ops.wait_probe(library, code, DEV)
        torch.cuda.synchronize()
        assert time.time() - t0 < 0.5                  # far below the default limit of about a second
        with pytest.raises(ops.KernelError, match=f"bounded wait ran out .code {code}"):
            ops.check_device_errors(DEV)
        ops.check_device_errors(DEV)                   # cleared
    finally:
        ops.set_wait_cycles(0, [library])
    for m in (3, 1200):
        check_product(ops, m)


def test_the_limit_of_all_libraries():
    """The default: every library that has one."""
    from rllm_b200.csrc import ops
    ops.set_wait_cycles(1_000_000_000)
    ops.set_wait_cycles()
    for m in (3, 1200):
        check_product(ops, m)
