"""GPU tests of the 4-bit operators' bounded waits: when they begin, and what a caller learns of one that runs out.  No fault
is involved: fbmoe_test_expire_grid_wait shortens the limits (2 ms), and set to 1 it also makes waits for one arrival that
never comes."""
import os
import sys

import pytest
import torch

from conftest import REPO

sys.path.insert(0, os.path.join(REPO, "tests"))
from test_gpu_w4 import BF16, Case, check_linear, random_packed  # noqa: E402, F401

pytestmark = pytest.mark.gpu


@pytest.fixture
def expire(fbmoe_lib):
    lib = fbmoe_lib.load_library()

    def set_(mode):
        assert lib.fbmoe_test_expire_grid_wait(mode) == 0
    yield set_
    set_(0)


def long_call(fbmoe_lib):
    """A call of one CTA that lets its successor start at once and takes longer than the shortened limit, and a function
    that makes it."""
    K = 1 << 23
    x = torch.zeros((8, K), dtype=BF16, device="cuda")
    p = torch.zeros((1, K // 128, 1056), dtype=torch.uint8, device="cuda")
    return lambda: fbmoe_lib.linear_w4(x, p)


@pytest.mark.parametrize("T,N,K", [(16, 130, 12288), (64, 18432, 1024)])  # clusters, single CTAs
def test_waits_begin_when_the_predecessor_has_ended(fbmoe_lib, expire, T, N, K):
    p, v = random_packed(N, K, 64, 3)
    x = torch.randn((T, K), generator=torch.Generator().manual_seed(4)).to(BF16).cuda()
    before = long_call(fbmoe_lib)
    before()
    check_linear(fbmoe_lib.linear_w4(x, p, N), x, v, 64)
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    before()
    b.record()
    torch.cuda.synchronize()
    assert a.elapsed_time(b) > 4.0  # twice the limit
    expire(2)
    before()
    y = fbmoe_lib.linear_w4(x, p, N)
    torch.cuda.synchronize()
    check_linear(y, x, v, 64)
