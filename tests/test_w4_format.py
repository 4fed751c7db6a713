"""CPU tests of the 4-bit weight operators: the oracle's restatement of the packed format, and the refusals of the
Python checks and of the C ABI (no kernel is launched)."""
import os
import sys

import pytest
import torch

from conftest import REPO

sys.path.insert(0, os.path.join(REPO, "tests"))
import w4_oracle as W  # noqa: E402


def packed(N=48, K=256, G=64, lead=()):
    return torch.zeros(lead + (-(-N // 16), K // 128, 1024 + 4096 // G), dtype=torch.uint8)


@pytest.mark.parametrize("N,K,G", [(16, 128, 128), (17, 256, 64), (48, 384, 32), (1, 128, 32)])
def test_oracle_pack_and_unpack_are_inverse(N, K, G):
    g = torch.Generator().manual_seed(N + K + G)
    q = torch.randint(-8, 8, (N, K), generator=g)
    s = (torch.rand((N, K // G), generator=g) + 0.5).to(torch.bfloat16)
    q2, s2 = W.unpack(W.pack(q, s, G), N, K, G)
    assert torch.equal(q2, q) and torch.equal(s2, s)


def test_oracle_word_layout_by_hand():
    """Row 9 (h 1, g 1), column 75 = 32 * 2 + 8 * 1 + 3 (j 2, t 1, element 3): word ((1 * 8 + 1) * 4 + 1) * 4 + 2, bits
    16 + 4 of the unrotated word, 23 of the rotated one."""
    q = torch.full((16, 128), -8)
    q[9, 75] = -5  # u = 3
    s = torch.ones((16, 1), dtype=torch.bfloat16)
    tile = W.pack(q, s, 128)[0, 0]
    words = tile[:1024].view(torch.int32)
    at = ((1 * 8 + 1) * 4 + 1) * 4 + 2
    assert words[at].item() == 3 << 23 and words.count_nonzero() == 1


def test_packed_bytes(fbmoe_lib):
    lib = fbmoe_lib.load_library()
    assert lib.fbmoe_w4_bytes(3, 17, 256, 64) == 3 * 2 * 2 * 1088
    for bad in ((-1, 16, 128, 64), (1, 0, 128, 64), (1, 16, 64, 64), (1, 16, 192, 64), (1, 16, 128, 16)):
        assert lib.fbmoe_w4_bytes(*bad) == 0


def test_quantize_and_dequantize_refuse(fbmoe_lib):
    L, w = fbmoe_lib, torch.zeros((16, 256), dtype=torch.bfloat16)
    f8 = torch.zeros((16, 256), dtype=torch.float8_e4m3fn)
    bs = torch.ones((1, 2))
    for args in ((w, 16), (w, 256), (w.t(),), (w[0],), (w[:, :200],), (w.double(),), (w.long(),), (w[:0],), (f8, 64),
                 (w, 64, None, bs), (f8, 64, None, bs[:, :1]), (f8, 64, None, bs.double()),
                 (w, 64, torch.ones((16, 4))), (w, 64, torch.ones((16, 2), dtype=torch.bfloat16))):
        with pytest.raises(RuntimeError):
            L.quantize_w4(*args)
    with pytest.raises(RuntimeError, match="CUDA"):
        L.quantize_w4(w, 64)
    p = packed()
    for args in ((p, 49), (p, 32), (p.int(),), (p[0],), (p[..., :1024],), (p, 48, torch.float8_e4m3fn),
                 (p, 48, torch.float64), (p.transpose(0, 1),)):
        with pytest.raises(RuntimeError):
            L.dequantize_w4(*args)
    with pytest.raises(RuntimeError, match="CUDA"):
        L.dequantize_w4(p)


def test_linear_refuses(fbmoe_lib):
    L, p = fbmoe_lib, packed()
    x = torch.zeros((4, 256), dtype=torch.bfloat16)
    wide = torch.zeros((4, 260), dtype=torch.bfloat16)
    for args in ((x.float(), p), (x[0], p), (x[:, :128], p), (wide[:, :256], p), (x.expand(1, 4, 256), p),
                 (x[:1].expand(4, 256), p), (x, p.unsqueeze(0)), (x, p, 49), (x, p, 32),
                 (torch.zeros((65, 256), dtype=torch.bfloat16), p), (torch.zeros((256, 4), dtype=torch.bfloat16).t(), p)):
        with pytest.raises(RuntimeError):
            L.linear_w4(*args)
    with pytest.raises(RuntimeError, match="CUDA"):
        L.linear_w4(x, p)


def test_moe_refuses(fbmoe_lib):
    import main
    w1, w2 = packed(512, 384, 64, (4,)), packed(384, 256, 64, (4,))
    x, lo = torch.zeros((2, 384), dtype=torch.bfloat16), torch.zeros((2, 256))
    b = torch.zeros(256, dtype=torch.bfloat16)
    good = [lo, b, x, w1, w2, 0, 2.5]
    with pytest.raises(RuntimeError, match="CUDA"):
        main.fused_moe_w4(*good)
    many = torch.zeros((65, 384), dtype=torch.bfloat16)
    for at, bad in ((0, lo[:1]), (0, lo.double()), (0, lo[:, :255]), (1, b.float()), (1, b[:255]), (2, x.float()),
                    (2, x[:, :256]), (2, x[0]), (3, w1[0]), (3, w1[:3]), (3, w1[:, :31]), (3, packed(512, 256, 64, (4,))),
                    (4, w2[:, :23]), (4, w2.int()), (5, -1), (5, 256), (3, w1.transpose(0, 1))):
        args = list(good)
        args[at] = bad
        with pytest.raises(RuntimeError):
            main.fused_moe_w4(*args)
    with pytest.raises(RuntimeError, match="64 tokens"):
        main.fused_moe_w4(torch.zeros((65, 256)), b, many, w1, w2, 0, 2.5)


def test_c_entry_points_refuse(fbmoe_lib):
    lib, nul, a16 = fbmoe_lib.load_library(), None, 4096
    q = lambda *a: lib.fbmoe_quantize_w4(*a, nul)  # noqa: E731
    assert q(nul, 0, nul, nul, 0, 16, 128, 64, nul) == 0              # nothing to do
    assert q(nul, 0, nul, nul, 1, 16, 128, 64, nul) == -3
    assert q(a16, 3, nul, nul, 1, 16, 128, 64, a16) == -3             # e4m3 without its block scales
    assert q(a16 + 8, 0, nul, nul, 1, 16, 128, 64, a16) == -4
    for bad in ((a16, 4, nul, nul, 1, 16, 128, 64, a16), (a16, -1, nul, nul, 1, 16, 128, 64, a16),
                (a16, 0, nul, nul, -1, 16, 128, 64, a16), (a16, 0, nul, nul, 1, 0, 128, 64, a16),
                (a16, 0, nul, nul, 1, 16, 100, 64, a16), (a16, 0, nul, nul, 1, 16, 128, 48, a16)):
        assert q(*bad) == -1
    d = lambda *a: lib.fbmoe_dequantize_w4(*a, nul)  # noqa: E731
    assert d(nul, 0, 16, 128, 64, 0, nul) == 0 and d(nul, 1, 16, 128, 64, 0, nul) == -3
    assert d(a16, 1, 16, 128, 64, 3, a16) == -1 and d(a16, 1, 16, 0, 64, 0, a16) == -1
    assert d(a16, 1, 16, 128, 64, 0, a16 + 4) == -4
    f = lambda *a: lib.fbmoe_linear_w4(*a, nul)  # noqa: E731
    assert f(nul, 128, 0, 0, nul, 16, 128, 64, nul, 16) == 0 and f(nul, 128, 0, 1, nul, 16, 128, 64, nul, 16) == -3
    for bad in ((a16, 128, 0, 65, a16, 16, 128, 64, a16, 16), (a16, 128, 0, -1, a16, 16, 128, 64, a16, 16),
                (a16, 120, 0, 1, a16, 16, 128, 64, a16, 16), (a16, 128, 0, 1, a16, 16, 128, 64, a16, 15),
                (a16, 128, 2, 1, a16, 16, 128, 64, a16, 16), (a16, 128, 0, 1, a16, 16, 128, 24, a16, 16)):
        assert f(*bad) == -1
    assert f(a16, 132, 0, 2, a16, 16, 128, 64, a16, 16) == -4 and f(a16 + 2, 128, 0, 1, a16, 16, 128, 64, a16, 16) == -4
    size = lib.fbmoe_w4_workspace_size
    assert size(65, 128, 128) == 0 and size(-1, 128, 128) == 0 and size(1, 100, 128) == 0 and size(1, 128, 0) == 0
    assert 0 < size(1, 128, 128) < size(64, 7168, 2048)

    def m(T=1, H=128, I=128, E=1, off=0, type_=0, g1=64, g2=64, p=a16, ws=4096, n=1 << 30, sink=nul):
        return lib.fbmoe_forward_w4(p, p, p, type_, p, g1, p, g2, T, H, I, E, off, 2.5, p, ws, n, sink, nul)

    assert m(T=0) == 0 and m(p=nul) == -3 and m(ws=nul) == -3 and m(p=a16 + 4) == -4 and m(ws=4096 + 16) == -4
    assert m(n=1) == -2 and m(sink=4097) == -4
    for bad in (dict(T=65), dict(T=-1), dict(H=64), dict(I=200), dict(E=0), dict(E=257), dict(off=-1), dict(off=256),
                dict(type_=2), dict(g1=16), dict(g2=256), dict(H=1 << 21)):
        assert m(**bad) == -1, bad


def test_sizes_past_32_bits_are_refused(fbmoe_lib):
    """N and K are 32-bit numbers in the C ABI: larger ones are refused, not cut to their low half.  (Shapes only: tensors
    without memory.)"""
    L, big = fbmoe_lib, 1 << 32
    meta = dict(device="meta")
    with pytest.raises(RuntimeError, match="2\\^31"):
        L.dequantize_w4(torch.empty((1, big // 128 + 1, 1056), dtype=torch.uint8, **meta), 1)  # K = 2^32 + 128
    with pytest.raises(RuntimeError, match="2\\^31"):
        L.dequantize_w4(torch.empty((big // 16 + 1, 1, 1056), dtype=torch.uint8, **meta))
    for shape in ((1, big + 128), (big + 1, 128), (1 << 31, 128)):
        with pytest.raises(RuntimeError, match="2\\^31"):
            L.quantize_w4(torch.empty(shape, dtype=torch.bfloat16, **meta))
    with pytest.raises(RuntimeError, match="2\\^31"):
        L.linear_w4(torch.empty((1, big + 128), dtype=torch.bfloat16, **meta),
                    torch.empty((1, big // 128 + 1, 1056), dtype=torch.uint8, **meta))
    with pytest.raises(RuntimeError, match="CUDA"):  # the largest of either
        L.dequantize_w4(torch.empty((1, (1 << 24) - 1, 1056), dtype=torch.uint8, **meta))
    with pytest.raises(RuntimeError, match="CUDA"):
        L.dequantize_w4(torch.empty((1 << 27, 1, 1056), dtype=torch.uint8, **meta), (1 << 31) - 1)


@pytest.mark.parametrize("rows,other", [(1, 1), (1, 4), (4, 4), (4, 9), (3, 1)])
def test_rows_that_share_memory_are_found(fbmoe_lib, rows, other):
    """Against the sets of elements, for two windows of one buffer at all offsets."""
    def elements(t):
        return {t.storage_offset() + r * t.stride(0) + c for r in range(t.size(0)) for c in range(t.size(1))}

    buf = torch.zeros(400, dtype=torch.float16)
    for wide, narrow in ((10, 10), (12, 5), (7, 3)):
        a = buf.as_strided((rows, narrow), (wide, 1), 100)
        for at in range(0, 260):
            for stride, width in ((wide, wide - narrow), (wide, 1), (8, 8)):
                b = buf.as_strided((other, max(width, 1)), (stride, 1), at)
                meet = bool(elements(a) & elements(b))
                found = fbmoe_lib._rows_meet(a, b)
                assert found or not meet
                if stride == wide or rows == other == 1:
                    # the same distance apart: exact, but for windows whose columns meet in rows past one another's last
                    columns = {i % wide for i in elements(a)} & {i % wide for i in elements(b)}
                    assert not found or meet or columns
