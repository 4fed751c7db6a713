"""The 4-bit weight operators restated in plain torch, in 64 bits where values are computed (test infrastructure)."""
import torch

MIN_NORMAL = 2.0 ** -126


def word_places(device="cpu"):
    """For row r and column k of a tile: the index of its word and the bits [4] of the word that hold u, low first."""
    r, k = torch.arange(16, device=device)[:, None], torch.arange(128, device=device)[None, :]
    word = ((r // 8 * 8 + r % 8) * 4 + k // 8 % 4) * 4 + k // 32
    first = 4 * (k % 8 // 2) + 16 * (k % 2) + 3
    return word, (first.expand(16, 128)[..., None] + torch.arange(4, device=device)) % 32


def pack(q, scale, G):
    """q [N, K] in -8..7 and bf16 scale [N, K / G] -> packed [ceil(N / 16), K / 128, tile]; the rows past N are zeros."""
    N, K = q.shape
    Nt, Kt = -(-N // 16), K // 128
    u = torch.full((Nt * 16, K), 8, dtype=torch.int64)
    u[:N] = q + 8
    s = torch.zeros((Nt * 16, K // G), dtype=torch.bfloat16)
    s[:N] = scale
    u = u.view(Nt, 16, Kt, 128).transpose(1, 2)
    word, bits = word_places()
    words = torch.zeros((Nt, Kt, 256), dtype=torch.int64)
    for i in range(4):
        at = ((u >> i) & 1) << bits[..., i]
        words.scatter_add_(2, word.reshape(1, 1, -1).expand(Nt, Kt, -1), at.reshape(Nt, Kt, -1))
    s = s.view(Nt, 2, 8, Kt, 128 // G).permute(0, 3, 4, 2, 1).contiguous()  # [group][g][h]
    low = torch.stack([(words >> (8 * b)) & 255 for b in range(4)], dim=-1).to(torch.uint8)
    return torch.cat([low.view(Nt, Kt, 1024), s.view(torch.uint8).view(Nt, Kt, -1)], dim=2)


def unpack(packed, N, K, G):
    """packed [Nt, Kt, tile] -> (q int64 [N, K], bf16 scale [N, K / G])."""
    packed = packed.cpu()
    Nt, Kt = packed.shape[0], packed.shape[1]
    word, bits = word_places()
    words = packed[..., :1024].contiguous().view(torch.int32).long() & 0xFFFFFFFF
    words = words.view(Nt, Kt, 256)[:, :, word]
    u = sum(((words >> bits[..., i]) & 1) << i for i in range(4))
    q = (u - 8).transpose(1, 2).reshape(Nt * 16, K)[:N]
    s = packed[..., 1024:].contiguous().view(torch.bfloat16).view(Nt, Kt, 128 // G, 8, 2)
    return q, s.permute(0, 4, 3, 1, 2).reshape(Nt * 16, K // G)[:N]


def values(packed, N, K, G):
    """The weights in 64 bits."""
    q, s = unpack(packed, N, K, G)
    return q.double() * s.double().repeat_interleave(G, 1)


def quantize(w, G, scale=None):
    """(q, bf16 scale) of fp32 values w [N, K] by the operator's rule."""
    g = w.float().view(w.shape[0], -1, G)
    finite = g.isfinite().all(-1)
    if scale is None:
        top = g.abs().amax(-1)
        s = (top / torch.full_like(top, 7.0)).to(torch.bfloat16)
        s = torch.where(s.float() < MIN_NORMAL, torch.zeros_like(s), s)
    else:
        s = scale
    s = torch.where(finite, s, torch.full_like(s, float("nan")))
    use = (s.float() >= MIN_NORMAL) & s.float().isfinite()
    q = torch.where(use[..., None], (g / s.float()[..., None]).round().clamp(-8, 7), torch.zeros_like(g))
    return q.long().view(w.shape), s


def moe(topk_idx, topk_w, x, w1, w2, offset, I):
    """The layer in 64 bits: w1[e], w2[e] give local expert e's matrices in 64 bits; also the sums of the absolute values
    of the products behind each output, the yardstick for rounding errors."""
    x = x.double().cpu()
    y = torch.zeros((x.shape[0], w2(0).shape[0]), dtype=torch.float64)
    size = torch.zeros_like(y)
    for t in range(x.shape[0]):
        for e, w in zip(topk_idx[t].tolist(), topk_w[t].double().tolist()):
            if e - offset not in w1.local:
                continue
            a = w1(e - offset) @ x[t]
            gate = a[I:]
            h = gate / (1 + torch.exp(-gate)) * a[:I]
            m = w2(e - offset)
            y[t] += w * (m @ h)
            size[t] += abs(w) * (m.abs() @ h.abs())
    return y, size
