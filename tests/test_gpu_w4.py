"""GPU tests of the 4-bit weight operators against their 64-bit restatement (w4_oracle.py).

Tolerances.  A product sums K terms in fp32: inside a group the tensor core adds 16 columns at a time to its running sum
(at most 2 * G / 16 roundings or truncations, 2^-23 each), K / G scaled groups follow, then the partial sums of up to 16
warps.  So |error| <= (G / 8 + K / G + 20) * 2^-23 * sum |x w|, and half a step of the output type where it is rounded.
"""
import os
import sys

import pytest
import torch

from conftest import REPO

sys.path.insert(0, os.path.join(REPO, "tests"))
import w4_oracle as W  # noqa: E402

pytestmark = pytest.mark.gpu
ROUTING_AT = 1280  # bytes of the layer's counters, rounded up: where its workspace holds the chosen experts
BF16, F16, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def steps(K, G):
    return (G / 8 + K / G + 20) * 2.0 ** -23


def half_step(y, dtype):
    info = torch.finfo(dtype)
    return y.abs() * (info.eps / 2) + info.smallest_normal * info.eps  # subnormal results: their absolute step


def plane_error(x, block):
    """What is lost of x [.., K] as 16-bit integers: per `block` columns in units of s, the power of two that puts the
    largest magnitude m, times 1 + 2^-7, into [2^14, 2^15)."""
    b = x.double().view(*x.shape[:-1], -1, block)
    m = b.abs().amax(-1, keepdim=True) * (1 + 2.0 ** -7)
    s = torch.where(m > 0, 2.0 ** (torch.floor(torch.log2(m)) - 14), torch.ones_like(m))
    return (b - torch.round(b / s) * s).abs().view(x.shape)


def random_packed(N, K, G, seed, lead=(), q_range=(-8, 8)):
    """Packed random weights of about unit row norm, and their 64-bit values [lead.., N, K] on the GPU."""
    g = torch.Generator().manual_seed(seed)
    mats, vals = [], []
    for _ in range(lead[0] if lead else 1):
        q = torch.randint(*q_range, (N, K), generator=g)
        s = ((torch.rand((N, K // G), generator=g) + 0.5) * K ** -0.5 / 5).to(BF16)
        mats.append(W.pack(q, s, G))
        vals.append((q.double() * s.double().repeat_interleave(G, 1)).cuda())
    p, v = torch.stack(mats).cuda(), torch.stack(vals)
    return (p, v) if lead else (p[0], v[0])


# ------------------------------------------------------------------ quantise and read back
def hard_weights(N, K, seed):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn((N, K), generator=g) * torch.exp(torch.randn((N, 1), generator=g) * 2)
    w[0, :128] = 0.0                                     # a group of zeros
    w[-1, -128:] = torch.arange(-64, 64) / 64.0 * 7 * 0.5  # halves of a step: ties
    if N > 2:
        w[1, 5] = float("nan")
        w[2, K - 1] = float("-inf")
    if N > 4:
        w[3, :128] = torch.linspace(-1e-38, 1e-38, 128)   # scale below the smallest normal number
        w[4, 0] = 3.0e38
    return w


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("N,K,G", [(1, 128, 128), (16, 256, 32), (33, 384, 64), (200, 1408, 128), (5, 128, 32)])
def test_quantize_exact(fbmoe_lib, dtype, N, K, G):
    w = hard_weights(N, K, N + G).to(dtype)
    p = fbmoe_lib.quantize_w4(w.cuda(), G)
    q, s = W.unpack(p, N, K, G)
    q_ref, s_ref = W.quantize(w, G)
    assert torch.equal(s.isnan(), s_ref.isnan()) and torch.equal(s.nan_to_num(), s_ref.nan_to_num())
    assert torch.equal(q, q_ref)
    pad_q, pad_s = W.unpack(p, p.shape[0] * 16, K, G)
    assert not pad_q[N:].any() and not pad_s[N:].any()    # rows past N hold zeros


@pytest.mark.parametrize("N,K,G", [(128, 256, 64), (200, 128, 32), (384, 1024, 128)])
def test_quantize_block_scaled_fp8(fbmoe_lib, N, K, G):
    g = torch.Generator().manual_seed(K)
    w = torch.randn((3, N, K), generator=g).to(E4M3)
    bs = torch.rand((3, (N + 127) // 128, K // 128), generator=g) * 0.01
    p = fbmoe_lib.quantize_w4(w.cuda(), G, block_scale=bs.cuda())
    for e in range(3):
        v = w[e].float() * bs[e].repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)
        q, s = W.unpack(p[e], N, K, G)
        q_ref, s_ref = W.quantize(v, G)
        assert torch.equal(q, q_ref) and torch.equal(s, s_ref)


@pytest.mark.parametrize("G", [32, 64, 128])
def test_quantize_with_given_scales_repacks_exactly(fbmoe_lib, G):
    """Weights that are q * scale already, -8 among them, come back as they were; a scale that is zero or not finite
    gives zeros, and q is clamped."""
    g = torch.Generator().manual_seed(G)
    N, K = 40, 512
    q = torch.randint(-8, 8, (N, K), generator=g)
    s = torch.exp(torch.randn((N, K // G), generator=g) * 3).to(BF16)
    w = q.float() * s.float().repeat_interleave(G, 1)
    p = fbmoe_lib.quantize_w4(w.cuda(), G, scale=s.cuda())
    q2, s2 = W.unpack(p, N, K, G)
    assert torch.equal(q2, q) and torch.equal(s2, s)
    s[0, 0], s[1, 0], s[2, 0] = 0.0, float("inf"), s[2, 0] / 16
    p = fbmoe_lib.quantize_w4(w.cuda(), G, scale=s.cuda())
    q2, s2 = W.unpack(p, N, K, G)
    q_ref, s_ref = W.quantize(w, G, s)
    assert torch.equal(q2, q_ref) and torch.equal(s2, s_ref) and q2[2, :G].abs().max() in (7, 8)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("N,K,G,lead", [(1, 128, 32, ()), (16, 128, 128, (2,)), (45, 1408, 64, (3,)), (4096, 256, 32, ())])
def test_dequantize_exact(fbmoe_lib, dtype, N, K, G, lead):
    p, v = random_packed(N, K, G, N + K, lead)
    out = fbmoe_lib.dequantize_w4(p, N, dtype)
    assert out.dtype == dtype and tuple(out.shape) == lead + (N, K)
    assert torch.equal(out, v.to(dtype))                   # q * s is exact in fp32, then one rounding


def test_empty_stacks(fbmoe_lib):
    p = fbmoe_lib.quantize_w4(torch.empty((0, 20, 256), device="cuda"), 64)
    assert tuple(p.shape) == (0, 2, 2, 1088)
    assert tuple(fbmoe_lib.dequantize_w4(p, 20).shape) == (0, 20, 256)


def test_offsets_past_32_bits(fbmoe_lib):
    """More than 2^31 weights in one stack: its last matrix is the one quantised and read back alone."""
    E, N, K = 37, 7168, 8192
    g = torch.Generator(device="cuda").manual_seed(3)
    w = torch.empty((E, N, K), dtype=BF16, device="cuda")
    w[:-1].fill_(0.25)
    w[-1].copy_(torch.randn((N, K), generator=g, device="cuda"))
    p = fbmoe_lib.quantize_w4(w, 64)
    assert torch.equal(p[-1], fbmoe_lib.quantize_w4(w[-1].contiguous(), 64))
    last = w[-1].clone()
    del w
    out = fbmoe_lib.dequantize_w4(p)
    assert torch.equal(out[-1], fbmoe_lib.dequantize_w4(p[-1].contiguous()))
    assert (out[-1].float() - last.float()).abs().max() < 0.75 * last.abs().max() / 7


# ------------------------------------------------------------------ linear
def check_linear(y, x, v, G):
    K = v.shape[1]
    ref, size = x.double() @ v.t(), x.double().abs() @ v.abs().t()
    tol = half_step(ref, y.dtype) * (1 + 2.0 ** -8) + steps(K, G) * size
    worst = ((y.double() - ref).abs() / tol).max().item()
    assert worst <= 1, worst


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("T,N,K", [(1, 1, 128), (1, 512, 7168), (2, 17, 256), (7, 100, 1408), (8, 4096, 512), (9, 33, 128),
                                   (16, 2000, 2048), (17, 31, 640), (33, 257, 1024), (64, 640, 4096), (63, 16, 14336)])
def test_linear(fbmoe_lib, dtype, G, T, N, K):
    p, v = random_packed(N, K, G, T + N)
    x = torch.randn((T, K), generator=torch.Generator().manual_seed(K)).to(dtype).cuda()
    y = fbmoe_lib.linear_w4(x, p, N)
    assert y.dtype == dtype and tuple(y.shape) == (T, N)
    check_linear(y, x, v, G)
    assert torch.equal(y, fbmoe_lib.linear_w4(x, p, N))


def test_linear_every_token_count(fbmoe_lib):
    p, v = random_packed(250, 768, 128, 5)
    x = torch.randn((64, 768), generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    for T in range(0, 65):
        y = fbmoe_lib.linear_w4(x[:T], p, 250)
        assert tuple(y.shape) == (T, 250)
        if T:
            check_linear(y, x[:T], v, 128)


def test_linear_strides_and_out(fbmoe_lib):
    """Rows of a wider tensor in, columns of a wider tensor out; what lies between the rows is left as it was."""
    p, v = random_packed(50, 384, 64, 9)
    for T in (1, 6, 20, 64):
        big = torch.randn((T, 400), generator=torch.Generator().manual_seed(T)).to(F16).cuda()
        x = big[:, 8:392]
        out = torch.full((T, 61), 7.0, dtype=F16, device="cuda")
        y = fbmoe_lib.linear_w4(x, p, 50, out=out[:, 5:55])
        assert y.data_ptr() == out[:, 5:55].data_ptr()
        check_linear(y, x, v, 64)
        assert (out[:, :5] == 7).all() and (out[:, 55:] == 7).all()


def test_linear_bad_values_stay_in_their_row(fbmoe_lib):
    p, v = random_packed(70, 512, 32, 2)
    for T in (3, 12, 40):
        x = torch.randn((T, 512), generator=torch.Generator().manual_seed(4)).to(BF16).cuda()
        clean = fbmoe_lib.linear_w4(x, p, 70)
        bad = x.clone()
        bad[1, 7], bad[2, 100] = float("nan"), float("inf")
        y = fbmoe_lib.linear_w4(bad, p, 70)
        assert y[1].isnan().all() and not y[2].isfinite().any()
        keep = [t for t in range(T) if t not in (1, 2)]
        assert torch.equal(y[keep], clean[keep])
    q = p.clone()
    q[0, 0, 1024:1026] = torch.tensor([0xC0, 0x7F], dtype=torch.uint8)  # row 0's first scale: NaN
    y = fbmoe_lib.linear_w4(x, q, 70)
    assert y[:, 0].isnan().all() and torch.equal(y[:, 1:], clean[:, 1:])


def test_linear_large_values(fbmoe_lib):
    """bf16 activations up to 2^120: the group sums stay below fp32's largest number."""
    p, v = random_packed(64, 256, 128, 8)
    x = (torch.randn((5, 256), generator=torch.Generator().manual_seed(4)) * 2.0 ** 115).to(BF16).cuda()
    check_linear(fbmoe_lib.linear_w4(x, p), x, v, 128)


# More than 8 tokens with a K of 12288 or more, or with more than 8192 tiles to read: the kernel of 128 rows per CTA.
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("T,N,K", [(9, 1, 12288), (16, 17, 12416), (17, 130, 12288), (33, 257, 12544), (64, 640, 14336),
                                   (64, 33000, 128), (16, 18500, 1024), (20, 9000, 1152), (31, 2100, 4096)])
def test_linear_rows(fbmoe_lib, dtype, G, T, N, K):
    p, v = random_packed(N, K, G, T + N)
    x = torch.randn((T, K), generator=torch.Generator().manual_seed(K)).to(dtype).cuda()
    y = fbmoe_lib.linear_w4(x, p, N)
    check_linear(y, x, v, G)
    for _ in range(3):
        assert torch.equal(y, fbmoe_lib.linear_w4(x, p, N))


def test_linear_rows_every_token_count(fbmoe_lib):
    p, v = random_packed(130, 12288, 128, 5)
    x = torch.randn((64, 12288), generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    for T in range(7, 65):
        y = fbmoe_lib.linear_w4(x[:T], p, 130)
        assert tuple(y.shape) == (T, 130)
        check_linear(y, x[:T], v, 128)


@pytest.mark.parametrize("T,N,K", [(16, 8192, 2048), (16, 8193, 2048), (64, 2049, 2048), (64, 2048, 2048), (64, 16, 12160),
                                   (64, 16, 12288), (8, 16, 12288), (8, 8192, 2048), (8, 8193, 2048), (1, 20000, 1024), (1, 40000, 2048)])
def test_linear_on_both_sides_of_the_choice(fbmoe_lib, T, N, K):
    p, v = random_packed(N, K, 64, T + N)
    x = torch.randn((T, K), generator=torch.Generator().manual_seed(K)).to(BF16).cuda()
    check_linear(fbmoe_lib.linear_w4(x, p, N), x, v, 64)


def test_linear_rows_strides_and_bad_values(fbmoe_lib):
    """Rows of a wider tensor in, columns of a wider tensor out; a NaN or an infinity spoils its token's outputs only, a NaN
    scale its row's."""
    N, K = 150, 12288
    p, v = random_packed(N, K, 64, 9)
    for T in (9, 20, 64):
        big = torch.randn((T + 3, K + 16), generator=torch.Generator().manual_seed(T)).to(F16).cuda()
        big[T:], big[:, :8], big[:, -8:] = float("nan"), float("nan"), float("nan")  # what is not x
        x = big[:T, 8:-8]
        out = torch.full((T + 1, N + 11), 7.0, dtype=F16, device="cuda")
        y = fbmoe_lib.linear_w4(x, p, N, out=out[:T, 5:N + 5])
        check_linear(y, x, v, 64)
        assert (out[:, :5] == 7).all() and (out[:, N + 5:] == 7).all() and (out[T] == 7).all()
        bad = x.clone()
        bad[1, 7], bad[2, 12000] = float("nan"), float("inf")
        z = fbmoe_lib.linear_w4(bad, p, N)
        assert z[1].isnan().all() and not z[2].isfinite().any()
        keep = [t for t in range(T) if t not in (1, 2)]
        assert torch.equal(z[keep], y[keep])
    q = p.clone()
    q[0, 50, 1024:1026] = torch.tensor([0xC0, 0x7F], dtype=torch.uint8)  # row 0's scale in K position 50: NaN
    z = fbmoe_lib.linear_w4(x, q, N)
    assert z[:, 0].isnan().all() and torch.equal(z[:, 1:], y[:, 1:])


def test_linear_rows_on_two_streams(fbmoe_lib):
    """Clusters and single CTAs that take all of an SM's tensor memory, of two calls at once."""
    calls = []
    for T, N, K in ((64, 300, 12288), (33, 4096, 4096), (12, 19000, 1024)):
        p, _ = random_packed(N, K, 64, N)
        x = torch.randn((T, K), generator=torch.Generator().manual_seed(T)).to(BF16).cuda()
        calls.append((x, p, N, fbmoe_lib.linear_w4(x, p, N)))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    results = []
    for i in range(30):
        for j, s in enumerate(streams):
            x, p, N, ref = calls[(i + j) % 3]
            with torch.cuda.stream(s):
                results.append((fbmoe_lib.linear_w4(x, p, N), ref))
    torch.cuda.synchronize()
    assert all(torch.equal(y, ref) for y, ref in results)


def test_linear_rows_captured(fbmoe_lib):
    """Two layers, one reading the other's result, captured once and replayed over new inputs."""
    p1, _ = random_packed(12288, 1024, 128, 1)
    p2, _ = random_packed(512, 12288, 32, 2)
    x = torch.zeros((32, 1024), dtype=BF16, device="cuda")
    inputs = [torch.randn((32, 1024), generator=torch.Generator().manual_seed(i)).to(BF16).cuda() for i in range(3)]
    eager = [fbmoe_lib.linear_w4(fbmoe_lib.linear_w4(i, p1), p2) for i in inputs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fbmoe_lib.linear_w4(fbmoe_lib.linear_w4(x, p1), p2)
    for i, e in zip(inputs * 2, eager * 2):
        x.copy_(i)
        graph.replay()
        assert torch.equal(y, e)


def test_linear_offsets_past_32_bits(fbmoe_lib):
    """More than 2^32 packed bytes in one matrix: its last rows, and its first."""
    N, K, G = 1 << 20, 8192, 128
    g = torch.Generator(device="cuda").manual_seed(2)
    p = torch.randint(0, 256, (N // 16, K // 128, 1056), generator=g, device="cuda", dtype=torch.uint8)
    scales = ((torch.rand((N // 16, K // 128, 16), generator=g, device="cuda") + 0.5) * 0.01).to(BF16)
    p[..., 1024:] = scales.view(torch.uint8)
    for T in (1, 9, 64):
        x = torch.randn((T, K), generator=g, device="cuda").to(BF16)
        y = fbmoe_lib.linear_w4(x, p)
        for rows in (slice(0, 512), slice(N - 2000, N)):
            v = fbmoe_lib.dequantize_w4(p[rows.start // 16:rows.stop // 16].contiguous(), dtype=F32).double()
            check_linear(y[:, rows], x, v, G)


# ------------------------------------------------------------------ the MoE layer
class Case:
    def __init__(self, lib, T, E, offset, H, I, G1, G2, dtype, config, seed):
        g = torch.Generator().manual_seed(seed)
        self.T, self.E, self.offset, self.H, self.I, self.G1, self.G2 = T, E, offset, H, I, G1, G2
        logits = torch.randn((T, 256), generator=g)
        if config == "group":
            logits[:, offset // 32 * 32:offset // 32 * 32 + 32] += 5.0
        elif config == "away":
            logits[:, offset:offset + E] -= 50.0
        elif config == "zero":
            logits.zero_()
        elif config == "one":  # every token chooses the same eight experts
            logits = logits[:1].repeat(T, 1)
        self.logits, self.bias = logits.cuda(), (torch.randn(256, generator=g) * 0.1).to(BF16).cuda()
        self.x = torch.randn((T, H), generator=g).to(dtype).cuda()
        self.w1, self.v1 = random_packed(2 * I, H, G1, seed + 1, (E,))
        self.w2, self.v2 = random_packed(H, I, G2, seed + 2, (E,))
        self.idx, self.w = lib.route(self.logits, self.bias, 2.5)

    def args(self):
        return (self.logits, self.bias, self.x, self.w1, self.w2, self.offset, 2.5)

    def check(self, y):
        """The layer in 64 bits and its error bound.  d1 bounds the error of both halves of the first product: its sums,
        and x as 16-bit integers.  Through h = silu(g) u (|silu'| < 1.1, |silu(g)| <= |g|) it reaches h, which is also
        rounded by expf, a division and two products (2^-20 in all) and kept as a 16-bit integer: half a unit, and the
        unit is at most 2^-14 (1 + 2^-6) of the largest of 32.  The second product's own sums follow; each output is a
        sum of up to 8 weighted pairs (16 * 2^-24), rounded once.  The weights come from lib.route in fp32 as the
        kernel's do."""
        assert y.dtype == self.x.dtype and tuple(y.shape) == (self.T, self.H)
        lost = plane_error(self.x, 128)
        for t in range(self.T):
            ref = torch.zeros(self.H, dtype=torch.float64, device="cuda")
            err = torch.zeros_like(ref)
            for e, w in zip(self.idx[t].tolist(), self.w[t].tolist()):
                if not self.offset <= e < self.offset + self.E:
                    continue
                v1, v2, x = self.v1[e - self.offset], self.v2[e - self.offset], self.x[t].double()
                a, size = v1 @ x, v1.abs() @ x.abs()
                d1 = steps(self.H, self.G1) * size + v1.abs() @ lost[t]
                u, gate = a[:self.I], a[self.I:]
                silu = gate / (1 + torch.exp(-gate))
                h = silu * u
                dh = 1.1 * d1[self.I:] * (u.abs() + d1[:self.I]) + silu.abs() * d1[:self.I] + 2.0 ** -20 * h.abs()
                top = (h.abs() + dh).view(-1, 32).amax(-1).repeat_interleave(32)
                dh = dh + top * (2.0 ** -15 * (1 + 2.0 ** -6))
                ref += w * (v2 @ h)
                err += abs(w) * (v2.abs() @ dh + (2 * steps(self.I, self.G2) + 2.0 ** -20) * (v2.abs() @ h.abs()))
            tol = half_step(ref, y.dtype) * (1 + 2.0 ** -8) + err
            worst = ((y[t].double() - ref).abs() / tol.clamp_min(1e-300)).max().item()
            assert worst <= 1, (t, worst)


@pytest.mark.parametrize("T,E,offset,H,I,G1,G2,dtype,config", [
    (1, 8, 0, 128, 128, 128, 128, BF16, "group"),
    (1, 32, 96, 512, 256, 32, 64, F16, "group"),
    (2, 64, 0, 384, 128, 64, 32, BF16, "standard"),
    (5, 256, 0, 256, 128, 128, 32, BF16, "standard"),
    (8, 32, 224, 1408, 384, 32, 32, F16, "group"),
    (16, 32, 32, 256, 640, 64, 128, BF16, "group"),
    (17, 100, 77, 256, 256, 128, 64, F16, "standard"),
    (33, 16, 5, 384, 256, 64, 64, BF16, "group"),
    (64, 32, 0, 256, 384, 32, 128, BF16, "one"),
    (64, 256, 0, 128, 128, 128, 128, F16, "standard"),
    (64, 1, 40, 256, 128, 32, 32, BF16, "group"),
    (63, 32, 64, 640, 128, 128, 64, BF16, "zero"),
    (3, 8, 255, 256, 128, 64, 64, F16, "standard"),   # a shard that reaches past the last expert
])
def test_moe(fbmoe_lib, T, E, offset, H, I, G1, G2, dtype, config):
    import main
    c = Case(fbmoe_lib, T, E, offset, H, I, G1, G2, dtype, config, T + E + H)
    y = main.fused_moe_w4(*c.args())
    c.check(y)
    assert torch.equal(y, main.fused_moe_w4(*c.args()))


def test_moe_every_token_count(fbmoe_lib):
    c = Case(fbmoe_lib, 64, 32, 64, 256, 128, 64, 64, BF16, "group", 21)
    for T in range(0, 65):
        y = fbmoe_lib.forward_w4(c.logits[:T], c.bias, c.x[:T], c.w1, c.w2, c.offset, 2.5)
        assert tuple(y.shape) == (T, c.H)
        part = Case.__new__(Case)
        part.__dict__.update(c.__dict__, T=T)
        part.check(y)


def test_moe_without_local_experts_is_zero(fbmoe_lib):
    c = Case(fbmoe_lib, 9, 32, 224, 256, 128, 64, 64, BF16, "away", 3)
    assert not ((c.idx >= 224).any())
    out = torch.full((9, 256), 5.0, dtype=BF16, device="cuda")
    assert fbmoe_lib.forward_w4(*c.args(), out=out) is out and not out.any()


def test_moe_bad_token_stays_alone(fbmoe_lib):
    """NaN and infinity in one token's activations, and NaN in another's logits, leave the other tokens' bits alone."""
    c = Case(fbmoe_lib, 12, 256, 0, 256, 128, 32, 64, F16, "standard", 4)
    clean = fbmoe_lib.forward_w4(*c.args())
    x, logits = c.x.clone(), c.logits.clone()
    x[3, 17], x[5, 2], logits[7, 9] = float("nan"), float("-inf"), float("nan")
    y = fbmoe_lib.forward_w4(logits, c.bias, x, c.w1, c.w2, 0, 2.5)
    assert y[3].isnan().all()
    keep = [t for t in range(12) if t not in (3, 5, 7)]
    assert torch.equal(y[keep], clean[keep])
    logits[:] = float("nan")
    fbmoe_lib.forward_w4(logits, c.bias, x, c.w1, c.w2, 0, 2.5)
    logits[:] = float("-inf")
    fbmoe_lib.forward_w4(logits, c.bias, x, c.w1, c.w2, 0, 2.5)
    torch.cuda.synchronize()


def test_moe_full_geometry(fbmoe_lib):
    """The framework's own H and I, from its fp8 block-scaled weights: quantised, run, and checked against the layer on
    the weights read back."""
    import fbmoe_workloads
    import main
    f1, s1, f2, s2 = fbmoe_workloads.make_weights(8, 5, "cuda")
    w1, w2 = fbmoe_lib.quantize_w4(f1, 64, block_scale=s1), fbmoe_lib.quantize_w4(f2, 128, block_scale=s2)
    c = Case.__new__(Case)
    c.T, c.E, c.offset, c.H, c.I, c.G1, c.G2 = 20, 8, 64, 7168, 2048, 64, 128
    g = torch.Generator().manual_seed(6)
    c.logits = torch.randn((20, 256), generator=g).cuda()
    c.logits[:, 64:72] += 4.0
    c.bias = torch.zeros(256, dtype=BF16, device="cuda")
    c.x = torch.randn((20, 7168), generator=g).to(BF16).cuda()
    c.w1, c.w2 = w1, w2
    c.v1, c.v2 = fbmoe_lib.dequantize_w4(w1, dtype=F32).double(), fbmoe_lib.dequantize_w4(w2, dtype=F32).double()
    # the weights read back are within half a step (amax / 14, and the scale's own rounding) of the fp8 ones
    back = (f1.float() * s1.repeat_interleave(128, 1).repeat_interleave(128, 2))
    step = back.view(8, 4096, -1, 64).abs().amax(-1).double() / 7
    off = (c.v1 - back.double()).view(8, 4096, -1, 64).abs().amax(-1)
    assert (off <= step * (0.5 + 7 * 2.0 ** -8)).all()
    c.idx, c.w = fbmoe_lib.route(c.logits, c.bias, 2.5)
    c.check(main.fused_moe_w4(*c.args()))


# ------------------------------------------------------------------ streams, graphs, workspaces
def test_other_stream_and_graph(fbmoe_lib):
    c = Case(fbmoe_lib, 6, 64, 0, 512, 256, 64, 32, BF16, "standard", 8)
    p, _ = random_packed(96, 512, 128, 1)
    want, lin = fbmoe_lib.forward_w4(*c.args()), fbmoe_lib.linear_w4(c.x, p)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        a, b = fbmoe_lib.forward_w4(*c.args()), fbmoe_lib.linear_w4(c.x, p)
    s.synchronize()
    assert torch.equal(a, want) and torch.equal(b, lin)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = fbmoe_lib.forward_w4(*c.args()), fbmoe_lib.linear_w4(c.x, p)
        back = fbmoe_lib.dequantize_w4(fbmoe_lib.quantize_w4(c.x, 32), 6)
    x0 = c.x.clone()
    for _ in range(3):
        c.x.neg_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(b, fbmoe_lib.linear_w4(c.x, p)) and torch.equal(a, fbmoe_lib.forward_w4(*c.args()))
        assert torch.equal(back, fbmoe_lib.dequantize_w4(fbmoe_lib.quantize_w4(c.x, 32), 6))
    assert torch.equal(c.x, -x0)


def test_two_graphs_and_two_streams_at_once(fbmoe_lib):
    """Calls that overlap share nothing: two captured graphs replayed on two streams, many times."""
    cases = [Case(fbmoe_lib, 16, 32, 0, 1024, 512, 64, 64, BF16, "group", 30 + i) for i in range(2)]
    want = [fbmoe_lib.forward_w4(*c.args()) for c in cases]
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for c in cases:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append([fbmoe_lib.forward_w4(*c.args()) for _ in range(4)])
    torch.cuda.synchronize()
    for _ in range(25):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(y, w) for y in o)


@pytest.mark.parametrize("fill", [0x00, 0x7F, 0xFF])
def test_workspace_contents_do_not_matter(fbmoe_lib, fill):
    c = Case(fbmoe_lib, 7, 32, 64, 512, 256, 128, 64, BF16, "group", 12)
    lib = fbmoe_lib.load_library()
    want = fbmoe_lib.forward_w4(*c.args())
    n = lib.fbmoe_w4_workspace_size(7, 512, 256)
    ws = torch.full((n + 256,), fill, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(want)
    for _ in range(2):
        rc = lib.fbmoe_forward_w4(c.logits.data_ptr(), c.bias.data_ptr(), c.x.data_ptr(), 0, c.w1.data_ptr(), 128,
                                  c.w2.data_ptr(), 64, 7, 512, 256, 32, 64, 2.5, out.data_ptr(), ws.data_ptr(), n, None,
                                  torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert (ws[n:] == fill).all()


def test_expired_wait_is_reported(fbmoe_lib):
    """A down unit that waits for one arrival that never comes gives up, and the call says so."""
    lib = fbmoe_lib.load_library()
    c = Case(fbmoe_lib, 4, 32, 0, 256, 128, 64, 64, BF16, "group", 77)
    want = fbmoe_lib.forward_w4(*c.args(), sync_status=True)
    lib.fbmoe_test_expire_grid_wait(1)
    try:
        with pytest.raises(fbmoe_lib.DeviceStatusError) as e:
            fbmoe_lib.forward_w4(*c.args(), sync_status=True)
        assert e.value.word & 4
        fbmoe_lib.forward_w4(*c.args())
        with pytest.raises(fbmoe_lib.DeviceStatusError):
            fbmoe_lib.check_status()
    finally:
        lib.fbmoe_test_expire_grid_wait(0)
    torch.cuda.synchronize()
    assert torch.equal(fbmoe_lib.forward_w4(*c.args(), sync_status=True), want)


@pytest.mark.parametrize("kind", ["normal", "grid", "groups", "zero", "large", "nan", "inf"])
def test_moe_routes_as_route(fbmoe_lib, kind):
    """The layer's own routing, read back from its workspace, is fbmoe_route's bit for bit: ties at a group's or an
    expert's boundary, equal values inside, values that are not numbers."""
    lib = fbmoe_lib.load_library()
    g = torch.Generator().manual_seed(11)
    w1, w2 = random_packed(256, 128, 128, 1, (1,))[0], random_packed(128, 128, 128, 2, (1,))[0]
    x = torch.zeros((64, 128), dtype=BF16, device="cuda")
    for trial in range(30):
        logits, bias = torch.randn((64, 256), generator=g), torch.randn(256, generator=g) * 0.1
        if kind == "grid":
            logits, bias = (logits * 2).round() / 2, (bias * 8).round() / 8
        elif kind == "groups":   # equal groups, distinct experts in them
            logits, bias = logits[:, :32].repeat(1, 8), bias[:32].repeat(8)
        elif kind == "zero":
            logits, bias = logits * 0, bias * (trial % 2)
        elif kind == "large":
            logits = logits * 60
        elif kind == "nan":
            logits[torch.rand(logits.shape, generator=g) < 0.02] = float("nan")
        elif kind == "inf":
            logits[torch.rand(logits.shape, generator=g) < 0.02] = float("inf")
            logits[torch.rand(logits.shape, generator=g) < 0.02] = float("-inf")
        logits, bias = logits.cuda(), bias.to(BF16).cuda()
        idx, w = fbmoe_lib.route(logits, bias, 2.5)
        n = lib.fbmoe_w4_workspace_size(64, 128, 128)
        ws, out = torch.zeros(n, dtype=torch.uint8, device="cuda"), torch.empty_like(x)
        assert lib.fbmoe_forward_w4(logits.data_ptr(), bias.data_ptr(), x.data_ptr(), 0, w1.data_ptr(), 128, w2.data_ptr(),
                                    128, 64, 128, 128, 1, 0, 2.5, out.data_ptr(), ws.data_ptr(), n, None,
                                    torch.cuda.current_stream().cuda_stream) == 0
        at = ROUTING_AT
        got_idx = ws[at:at + 2048].view(torch.int32).view(64, 8)
        got_w = ws[at + 2048:at + 4096].view(torch.float32).view(64, 8)
        assert torch.equal(got_idx, idx) and torch.equal(got_w.view(torch.int32), w.view(torch.int32))


# ------------------------------------------------------------------ calls at once
def test_two_threads(fbmoe_lib):
    """Two host threads, a stream each: layers and linears of either, many times."""
    import threading
    c = [Case(fbmoe_lib, T, 16, 0, 512, 256, 64, 64, BF16, "group", T) for T in (5, 33)]
    p, _ = random_packed(300, 12288, 128, 4)
    x = torch.randn((20, 12288), generator=torch.Generator().manual_seed(3)).to(BF16).cuda()
    want, lin = [fbmoe_lib.forward_w4(*i.args()) for i in c], fbmoe_lib.linear_w4(x, p, 300)
    torch.cuda.synchronize()
    wrong = []

    def work(k):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(40):
                    y, z = fbmoe_lib.forward_w4(*c[k].args()), fbmoe_lib.linear_w4(x, p, 300)
                    s.synchronize()
                    if not (torch.equal(y, want[k]) and torch.equal(z, lin)):
                        wrong.append(k)
        except Exception as e:  # reported below: an exception in a thread would pass unseen
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_layer_in_place(fbmoe_lib):
    """The output may take the activations' place: they are read before the first output is written."""
    c = Case(fbmoe_lib, 17, 16, 0, 512, 256, 64, 64, F16, "group", 3)
    want = fbmoe_lib.forward_w4(*c.args())
    x = c.x.clone()
    args = list(c.args())
    args[2] = x
    y = fbmoe_lib.forward_w4(*args, out=x)
    assert y.data_ptr() == x.data_ptr() and torch.equal(y, want)


def test_beside_the_fp8_layer(fbmoe_lib, workloads):
    """The fp8 layer (decode and prefill, which also use tensor memory) on one stream, 4-bit calls on another."""
    w = workloads.make_weights(32, 77, "cuda")
    inputs = [workloads.as_args(workloads.make_inputs(T, seed=T, device="cuda", E_local=32, weights=w)) for T in (16, 300)]
    c = Case(fbmoe_lib, 33, 16, 0, 512, 256, 64, 64, BF16, "group", 8)
    p, _ = random_packed(4096, 4096, 64, 4)
    x = torch.randn((64, 4096), generator=torch.Generator().manual_seed(3)).to(BF16).cuda()
    fp8 = [fbmoe_lib.forward(*i) for i in inputs]
    want, lin = fbmoe_lib.forward_w4(*c.args()), fbmoe_lib.linear_w4(x, p)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(a):
        for i in inputs:
            fbmoe_lib.forward(*i)
    torch.cuda.synchronize()
    got = []
    for _ in range(15):
        with torch.cuda.stream(a):
            got += [(fbmoe_lib.forward(*i), r) for i, r in zip(inputs, fp8)]
        with torch.cuda.stream(b):
            got += [(fbmoe_lib.forward_w4(*c.args()), want), (fbmoe_lib.linear_w4(x, p), lin)]
    torch.cuda.synchronize()
    assert all(torch.equal(y, r) for y, r in got)
    fbmoe_lib.check_status()
