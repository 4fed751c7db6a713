"""GPU tests of calls that the 4-bit operators' documentation allows or forbids and that are easily made."""
import os
import sys

import pytest
import torch

from conftest import REPO

sys.path.insert(0, os.path.join(REPO, "tests"))
import w4_oracle as W  # noqa: E402
from test_gpu_w4 import BF16, F16, F32, check_linear, random_packed  # noqa: E402
from test_gpu_w4_magnitudes import Layer  # noqa: E402

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


# ------------------------------------------------------------------ values that are not ordinary numbers
def test_given_scales_that_are_no_scales(fbmoe_lib):
    """Kept, with zeros: they read back as 0, or as NaN where the scale is infinite or NaN."""
    N, G = 16, 64
    w = torch.randn((N, 128), generator=torch.Generator().manual_seed(1)).cuda()
    s = torch.ones((N, 2), dtype=BF16)
    odd = [float("inf"), float("-inf"), float("nan"), 0.0, -0.0, -1.0, 2.0 ** -130, 2.0 ** -126]
    s[:len(odd), 0] = torch.tensor(odd).to(BF16)
    p = fbmoe_lib.quantize_w4(w, G, scale=s.cuda())
    q, s2 = W.unpack(p, N, 128, G)
    assert torch.equal(s2.view(torch.int16), s.view(torch.int16))
    assert not q[:7, :G].any() and (q[7, :G].abs() >= 7).all()  # the smallest normal scale is one
    back = fbmoe_lib.dequantize_w4(p, dtype=F32).cpu()
    assert back[:3, :G].isnan().all() and (back[3:7, :G] == 0).all()
    assert torch.equal(back[8:], W.values(p, N, 128, G)[8:].float())
    assert torch.equal(back[:, G:], W.values(p, N, 128, G)[:, G:].float())


class Local:
    """Local experts' matrices in 64 bits, as w4_oracle.moe takes them."""

    def __init__(self, packed, N, K, G):
        self.local, self.at = range(packed.shape[0]), lambda e: W.values(packed[e], N, K, G)

    def __call__(self, e):
        return self.at(e)


def bad_token_case(dtype):
    g = torch.Generator().manual_seed(4)
    T, E, H, I, G1, G2 = 12, 256, 256, 128, 32, 64
    logits, bias = torch.randn((T, 256), generator=g).cuda(), (torch.randn(256, generator=g) * 0.1).to(BF16).cuda()
    x = torch.randn((T, H), generator=g).to(dtype).cuda()
    w1, w2 = random_packed(2 * I, H, G1, 5, (E,))[0], random_packed(H, I, G2, 6, (E,))[0]
    return logits, bias, x, w1, w2, Local(w1, 2 * I, H, G1), Local(w2, H, I, G2), I


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_bad_activations_spoil_their_token(fbmoe_lib, dtype, value):
    """A NaN or an infinity among a token's activations: the formula gives it no finite output (an infinity times each of a
    row's weights, some of them zero), and the other tokens keep their bits."""
    logits, bias, x, w1, w2, v1, v2, I = bad_token_case(dtype)
    clean = fbmoe_lib.forward_w4(logits, bias, x, w1, w2, 0, 2.5)
    bad = x.clone()
    bad[5, 2] = value
    y = fbmoe_lib.forward_w4(logits, bias, bad, w1, w2, 0, 2.5)
    idx, w = fbmoe_lib.route(logits, bias, 2.5)
    ref, _ = W.moe(idx[5:6], w[5:6], bad[5:6], v1, v2, 0, I)
    assert not ref.isfinite().any() and not y[5].isfinite().any()
    keep = [t for t in range(12) if t != 5]
    assert torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_bad_logits(fbmoe_lib, dtype):
    """What routing gives for logits that are not numbers, carried through the layer: a NaN weight makes its token NaN, a
    token whose scores are all 0 gets weights of 0 / 1e-20 and zeros."""
    logits, bias, x, w1, w2, v1, v2, I = bad_token_case(dtype)
    logits[7] = float("nan")
    logits[9] = float("-inf")
    logits[2, :200] = float("-inf")
    logits[3, 17] = float("inf")
    y = fbmoe_lib.forward_w4(logits, bias, x, w1, w2, 0, 2.5)
    idx, w = fbmoe_lib.route(logits, bias, 2.5)
    assert w[7].isnan().all() and not w[9].any() and w[[2, 3]].isfinite().all()
    assert y[7].isnan().all() and not y[9].any()
    good = [t for t in range(12) if t != 7]
    c = Layer.__new__(Layer)
    c.T, c.E, c.H, c.I, c.G1, c.G2, c.x, c.idx, c.w = 11, 256, 256, I, 32, 64, x[good], idx[good], w[good]
    c.v1, c.v2 = [v1(e).cuda() for e in range(256)], [v2(e).cuda() for e in range(256)]
    assert c.worst(y[good]) <= 1
    for value in (float("nan"), float("-inf")):
        logits[:] = value
        y = fbmoe_lib.forward_w4(logits, bias, x, w1, w2, 0, 2.5)
        assert y.isnan().all() if value != value else not y.any()


def test_a_decoder_in_the_same_buffers(fbmoe_lib):
    """Projection, layer, projection, each reading what the one before wrote, call after call into the same memory with
    nothing between: every pass gives what it gives alone."""
    g = torch.Generator(device="cuda").manual_seed(2)
    H, I, T = 1024, 256, 24
    up, down = random_packed(H, 2048, 64, 1)[0], random_packed(2048, H, 32, 2)[0]
    w1, w2 = random_packed(2 * I, H, 128, 3, (8,))[0], random_packed(H, I, 64, 4, (8,))[0]
    inputs = [torch.randn((T, 2048), generator=g, device="cuda").to(BF16) for _ in range(5)]
    logits = torch.randn((T, 256), generator=g, device="cuda")
    logits[:, :8] += 4.0
    bias = torch.zeros(256, dtype=BF16, device="cuda")

    def run(x, t, h, y):
        fbmoe_lib.linear_w4(x[:t], up, out=h[:t])
        fbmoe_lib.forward_w4(logits[:t], bias, h[:t], w1, w2, 0, 2.5, out=h[:t])
        fbmoe_lib.linear_w4(h[:t], down, out=y[:t])

    want = {}
    for i, x in enumerate(inputs):
        for t in (1, 8, T):
            h, y = torch.empty((T, H), dtype=BF16, device="cuda"), torch.empty((T, 2048), dtype=BF16, device="cuda")
            run(x, t, h, y)
            torch.cuda.synchronize()
            want[i, t] = y[:t].clone()
    h, y = torch.empty((T, H), dtype=BF16, device="cuda"), torch.empty((T, 2048), dtype=BF16, device="cuda")
    got = []
    for r in range(60):
        i, t = r % 5, (1, 8, T)[r % 3]
        run(inputs[i], t, h, y)
        got.append((i, t, y[:t].clone()) if r % 2 else None)
    torch.cuda.synchronize()
    assert all(torch.equal(z, want[i, t]) for i, t, z in filter(None, got))
    x = inputs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(3):  # three layers of the same weights
            run(x, T, h, y)
            x.copy_(y)
    ref = inputs[1].clone()
    for _ in range(3):
        run(ref, T, h, y)
        torch.cuda.synchronize()
        ref = y.clone()
    for _ in range(4):
        x.copy_(inputs[1])
        graph.replay()
        assert torch.equal(x, ref)
