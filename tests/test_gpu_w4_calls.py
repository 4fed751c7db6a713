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


# ------------------------------------------------------------------ one call after another
def test_weights_written_by_the_call_before(fbmoe_lib):
    """Weights quantised into the memory of others, then read at once: by the streaming and the plain kernel of few tokens,
    by the one of many, and by the layer."""
    g = torch.Generator(device="cuda").manual_seed(1)
    sets = [torch.randn((8448, 2048), generator=g, device="cuda").to(BF16) for _ in range(2)]
    x = torch.randn((16, 2048), generator=g, device="cuda").to(BF16)
    moe = [[torch.randn(shape, generator=g, device="cuda").to(BF16) for shape in ((8, 512, 512), (8, 512, 256))]
           for _ in range(2)]
    logits = torch.zeros((12, 256), device="cuda")
    logits[:, :8] = 5.0
    bias, h = torch.zeros(256, dtype=BF16, device="cuda"), torch.randn((12, 512), generator=g, device="cuda").to(BF16)
    buffers, want = {}, []

    def step(i, wait):
        def now(name, w):  # the library's packed tensor, always in the same memory
            p = fbmoe_lib.quantize_w4(w, 64)
            buffers.setdefault(name, torch.empty_like(p)).copy_(p)
            return buffers[name]
        out = []
        for T in (1, 8, 16):
            p = now("linear", sets[i])
            if wait:
                torch.cuda.synchronize()
            out.append(fbmoe_lib.linear_w4(x[:T], p))
        w1, w2 = now("w1", moe[i][0]), now("w2", moe[i][1])
        if wait:
            torch.cuda.synchronize()
        out.append(fbmoe_lib.forward_w4(logits, bias, h, w1, w2, 0, 2.5))
        # without the copy between: the quantiser is the kernel before
        out.append(fbmoe_lib.linear_w4(x[:8], fbmoe_lib.quantize_w4(sets[i], 64)))
        out.append(fbmoe_lib.forward_w4(logits, bias, h, fbmoe_lib.quantize_w4(moe[i][0], 64),
                                        fbmoe_lib.quantize_w4(moe[i][1], 64), 0, 2.5))
        return out

    for i in range(2):
        want.append(step(i, True))
        torch.cuda.synchronize()
    for r in range(20):
        for y, z in zip(step(r % 2, False), want[r % 2]):
            assert torch.equal(y, z)
