"""GPU tests of the 4-bit MoE layer on activations and intermediates whose magnitudes differ widely inside a token: an
output is as accurate as the fp32 sums behind it, whatever else stands beside its terms.

Tolerances.  The first product's sums are off by at most steps(H, G) * sum |w x| (test_gpu_w4.py), x being exact.  Through
h = silu(g) u (|silu'| < 1.1, |silu(g)| <= |g|) that reaches h, which is also rounded by expf, a division and two products
(2^-20 in all) and held as two bf16 numbers: the first is off by at most 2^-8 |h|, the second, which holds what the first
lost, by 2^-8 of that.  The second product's own sums follow, over two terms for each h; each output is a sum of up to 8
weighted pairs (16 * 2^-24) and is rounded once.  None of it depends on what is not multiplied: a column whose weights are
zero adds nothing to a bound."""
import os
import sys

import pytest
import torch

from conftest import REPO

sys.path.insert(0, os.path.join(REPO, "tests"))
import w4_oracle as W  # noqa: E402
from test_gpu_w4 import half_step, steps  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


class Layer:
    """A layer whose tokens hold, in every 128 columns, one value of magnitude `loud`, and whose intermediates hold, in
    every 32 columns, one that is `loud_h` times larger.  heard: whether the weights of those columns are drawn as the
    others or are zeros."""

    def __init__(self, lib, T, E, H, I, G1, G2, dtype, loud, loud_h, heard, seed):
        g = torch.Generator().manual_seed(seed)
        self.T, self.E, self.H, self.I, self.G1, self.G2 = T, E, H, I, G1, G2
        self.logits = torch.randn((T, 256), generator=g)
        self.logits[:, :E] += 5.0
        self.logits, self.bias = self.logits.cuda(), torch.zeros(256, dtype=BF16, device="cuda")
        x = torch.randn((T, H), generator=g)
        at = torch.arange(0, H, 128) + torch.randint(0, 128, (H // 128,), generator=g)
        x[:, at] = loud * (1 - 2 * torch.randint(0, 2, (T, H // 128), generator=g)).float()
        self.x = x.to(dtype).cuda()
        at_h = torch.arange(0, I, 32) + torch.randint(0, 32, (I // 32,), generator=g)
        self.w1, self.w2, self.v1, self.v2 = [], [], [], []
        for _ in range(E):
            q1 = torch.randint(-8, 8, (2 * I, H), generator=g)
            q2 = torch.randint(-8, 8, (H, I), generator=g)
            if not heard:
                q1[:, at], q2[:, at_h] = 0, 0
            s1 = ((torch.rand((2 * I, H // G1), generator=g) + 0.5) * H ** -0.5 / 5)
            s2 = ((torch.rand((H, I // G2), generator=g) + 0.5) * I ** -0.5 / 5)
            s1[at_h] *= loud_h  # of the linear half
            for q, s, G, w, v in ((q1, s1, G1, self.w1, self.v1), (q2, s2, G2, self.w2, self.v2)):
                p = W.pack(q, s.to(BF16), G)
                w.append(p)
                v.append(W.values(p, *q.shape, G).cuda())
        self.w1, self.w2 = torch.stack(self.w1).cuda(), torch.stack(self.w2).cuda()
        self.idx, self.w = lib.route(self.logits, self.bias, 2.5)

    def worst(self, y):
        """The largest error of an output of the layer, as a share of its bound."""
        assert y.dtype == self.x.dtype and tuple(y.shape) == (self.T, self.H)
        I, worst = self.I, 0.0
        for t in range(self.T):
            ref = torch.zeros(self.H, dtype=torch.float64, device="cuda")
            err = torch.zeros_like(ref)
            for e, w in zip(self.idx[t].tolist(), self.w[t].tolist()):
                if e >= self.E:
                    continue
                v1, v2, x = self.v1[e], self.v2[e], self.x[t].double()
                a, d = v1 @ x, steps(self.H, self.G1) * (v1.abs() @ x.abs())
                u, gate = a[:I], a[I:]
                silu = gate / (1 + torch.exp(-gate))
                h = silu * u
                dh = 1.1 * d[I:] * (u.abs() + d[:I]) + silu.abs() * d[:I] + 2.0 ** -20 * h.abs()
                dh = dh + 2.0 ** -16 * (h.abs() + dh)
                ref += w * (v2 @ h)
                err += abs(w) * (v2.abs() @ dh + (2 * steps(I, self.G2) + 2.0 ** -20) * (v2.abs() @ h.abs()))
            tol = half_step(ref, y.dtype) * (1 + 2.0 ** -8) + err
            worst = max(worst, ((y[t].double() - ref).abs() / tol).max().item())
        return worst


@pytest.mark.parametrize("heard", [True, False])
@pytest.mark.parametrize("dtype,loud,loud_h", [(BF16, 64.0, 1.0), (BF16, 1024.0, 1.0), (BF16, 2.0 ** 15, 1.0), (F16, 64.0, 1.0),
                                               (F16, 1024.0, 1.0), (F16, 2.0 ** 15, 1.0), (BF16, 1.0, 1024.0),
                                               (F16, 1.0, 64.0), (F16, 8.0, 1024.0)])
@pytest.mark.parametrize("T,E,H,I,G1,G2", [(1, 8, 512, 128, 128, 128), (3, 8, 256, 256, 64, 32), (20, 4, 384, 128, 32, 64)])
def test_loud_columns(fbmoe_lib, T, E, H, I, G1, G2, dtype, loud, loud_h, heard):
    if dtype == F16 and heard:
        loud = min(loud, 256.0)  # outputs in f16's range
    c = Layer(fbmoe_lib, T, E, H, I, G1, G2, dtype, loud, loud_h, heard, T + H)
    y = fbmoe_lib.forward_w4(c.logits, c.bias, c.x, c.w1, c.w2, 0, 2.5)
    assert c.worst(y) <= 1


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_one_loud_column_among_small_ones(fbmoe_lib, dtype):
    """2048 beside 127 values of about 0.05, at which no weight looks."""
    c = Layer(fbmoe_lib, 5, 8, 256, 128, 128, 64, dtype, 2048.0, 1.0, False, 3)
    c.x = torch.where(c.x.abs() < 2048, c.x * 0.05, c.x)
    y = fbmoe_lib.forward_w4(c.logits, c.bias, c.x, c.w1, c.w2, 0, 2.5)
    assert c.worst(y) <= 1


@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** -50, 2.0 ** 30])
def test_tokens_of_other_magnitudes(fbmoe_lib, scale):
    """Tokens that only bf16's range holds; h is a product of two values of their magnitude."""
    c = Layer(fbmoe_lib, 6, 8, 256, 128, 64, 64, BF16, 1.0, 1.0, True, 9)
    c.x = (c.x.double() * scale).to(BF16)
    y = fbmoe_lib.forward_w4(c.logits, c.bias, c.x, c.w1, c.w2, 0, 2.5)
    assert c.worst(y) <= 1
