"""GPU tests of calls that the 4-bit operators' documentation allows or forbids and that are easily made."""
import os
import sys

import pytest
import torch

from conftest import REPO

sys.path.insert(0, os.path.join(REPO, "tests"))
from test_gpu_w4 import BF16, F16, check_linear, random_packed  # noqa: E402

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ outputs that overlap
@pytest.mark.parametrize("T", [1, 7, 20])
def test_linear_refuses_an_output_over_its_input(fbmoe_lib, T):
    K = N = 1408
    p, v = random_packed(N, K, 64, 1)
    x = torch.randn((T, K), generator=torch.Generator().manual_seed(T)).to(BF16).cuda()
    for out in (x, x.view(-1)[:T * 704].view(T, 704)):
        with pytest.raises(RuntimeError, match="overlap"):
            fbmoe_lib.linear_w4(x, p if out.size(1) == N else p[:44].contiguous(), out=out)
    with pytest.raises(RuntimeError, match="overlap"):
        fbmoe_lib.linear_w4(x, p, out=p.view(-1)[:T * N * 2].view(BF16).view(T, N))
    # columns of one tensor, beside each other
    both = torch.zeros((T, K + N), dtype=BF16, device="cuda")
    both[:, :K] = x
    check_linear(fbmoe_lib.linear_w4(both[:, :K], p, out=both[:, K:]), x, v, 64)
    assert torch.equal(both[:, :K], x)
