"""Cases and plain forms of the 4-bit weight operators: quantising weights to 4 bits with group scales, reading them back,
products of a few tokens with such a matrix, and the whole mixture-of-experts layer for a few tokens on such weights.

The packed format ("W4"): a matrix [N, K] is cut into tiles of 16 rows by 128 columns, stored [ceil(N / 16), K / 128, tile].
A tile is 1024 bytes of 4-bit values u = q + 8 and 4096 / G bytes of bf16 scales, G the group size along K.  Its 256 words of
32 bits are ordered [h, g, t, j] (2, 8, 4, 4): word (h, g, t, j) holds row 8h + g, columns 32j + 8t .. + 7, and is
rotl32(sum over i < 4 of u[2i] << 4i | u[2i + 1] << (16 + 4i), 3).  Its scales are ordered [group, g, h].
"""
import math
import os
import sys

import torch

own = False

E_GLOBAL, TOP_K, N_GROUP, KEPT_GROUPS = 256, 8, 8, 4
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}
MIN_NORMAL = 2.0 ** -126


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one expert's gate-up matrix of the framework's own MoE, quantised from a 16-bit checkpoint and read back
        dict(name="quantize_w1_bf16_g128", op="quantize", E=1, N=4096, K=7168, G=128, src="bf16", out="bf16"),
        # the down matrices of an eight-expert shard, from the framework's fp8 block-scaled weights
        dict(name="quantize_w2_e4m3_g32", op="quantize", E=8, N=7168, K=2048, G=32, src="e4m3", out="f32"),
        # one expert's gate-up matrix read back for a library GEMM of a long prompt
        dict(name="dequantize_w1_bf16_g128", op="dequantize", E=1, N=4096, K=7168, G=128, out="bf16"),
        # a ragged stack read back to f16
        dict(name="dequantize_ragged_f16_g64", op="dequantize", E=5, N=2045, K=1408, G=64, out="f16"),
        # the smallest call: one token through a shared expert's down projection
        dict(name="linear_t1_shared_down", op="linear", T=1, N=7168, K=2048, G=128, dtype="bf16"),
        # one token through its gate-up projection, fine groups
        dict(name="linear_t1_shared_up_g32", op="linear", T=1, N=4096, K=7168, G=32, dtype="f16"),
        # a small batch through a vocabulary-sized head, an odd number of rows
        dict(name="linear_t13_head", op="linear", T=13, N=32001, K=7168, G=128, dtype="bf16"),
        # the largest batch the operator takes, through a wide projection
        dict(name="linear_t64_wide", op="linear", T=64, N=18432, K=7168, G=64, dtype="bf16"),
        # decoding one token with every expert on the device
        dict(name="moe_t1_all_experts", op="moe", T=1, E=256, offset=0, H=7168, I=2048, G=128, dtype="bf16", config="standard"),
        # a small batch on one shard of an eight-way expert-parallel layer, fine groups
        dict(name="moe_t8_shard_g32", op="moe", T=8, E=32, offset=96, H=7168, I=2048, G=32, dtype="f16", config="standard"),
        # the largest batch on a quarter of the experts
        dict(name="moe_t64_quarter", op="moe", T=64, E=64, offset=64, H=7168, I=2048, G=128, dtype="bf16", config="standard"),
        # a smaller model's experts, every token routed to one group: experts with many rows
        dict(name="moe_t33_small_hot_group", op="moe", T=33, E=256, offset=0, H=2048, I=768, G=64, dtype="bf16", config="group"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "dequantize", "linear", "linear", "moe", "moe"])
    G = rng.choice([32, 64, 128])
    if op in ("quantize", "dequantize"):
        src = rng.choice(["bf16", "f16", "f32", "e4m3"])
        N, K = _log(rng, 64, 8192), 128 * _log(rng, 1, 64)
        if op == "quantize" and src == "e4m3":
            N = 128 * max(1, N // 128)
        E = max(1, min(16, _log(rng, 1, 32), 100_000_000 // (N * K)))
        case = dict(op=op, E=E, N=N, K=K, G=G, out=rng.choice(["bf16", "f16", "f32"]))
        return dict(case, src=src) if op == "quantize" else case
    if op == "linear":
        T, K = _log(rng, 1, 64), 128 * _log(rng, 4, 112)
        N = min(_log(rng, 256, 32768), 130_000_000 // K)
        return dict(op=op, T=T, N=N, K=K, G=G, dtype=rng.choice(["bf16", "f16"]))
    T = _log(rng, 1, 64)
    if rng.random() < 0.5:
        H, I, E = 7168, 2048, rng.choice([32, 64])  # the framework's geometry, sharded
    else:
        H, I, E = 128 * _log(rng, 8, 40), 128 * _log(rng, 3, 16), rng.choice([32, 64, 128])
    offset = E * rng.randrange(256 // E)
    return dict(op=op, T=T, E=E, offset=offset, H=H, I=I, G=G, dtype=rng.choice(["bf16", "f16"]),
                config=rng.choice(["standard", "standard", "group"]))


# ------------------------------------------------------------------ inputs
def _packed(gen, rows, N, K, G, std):
    """Random packed weights [rows, ceil(N / 16), K / 128, tile] of about the given standard deviation: values of a normal
    distribution whose groups reach about +-7, scales that differ from group to group."""
    Nt, Kt = -(-N // 16), K // 128
    normal = torch.distributions.Normal(0.0, 2.6)
    edges = torch.arange(-7, 7, device="cuda").float() + 0.5
    cut = normal.cdf(edges)  # 14 borders between the values -7 .. 7
    pairs = torch.bucketize((torch.arange(256, device="cuda").float() + 0.5) / 256, cut) + 1  # u = q + 8 in 1 .. 15
    pairs = (pairs[:, None] | (pairs[None, :] << 4)).reshape(-1).to(torch.uint8)  # a byte for each 16-bit number
    tile = 1024 + 4096 // G
    out = torch.empty((rows, Nt, Kt, tile), dtype=torch.uint8, device="cuda")
    for r in range(rows):
        at = torch.randint(0, 65536, (Nt, Kt, 1024), generator=gen, device="cuda")
        w = pairs[at].view(torch.int32)
        out[r, :, :, :1024] = ((w << 3) | ((w >> 29) & 7)).view(torch.uint8)
        s = torch.randn((Nt, Kt, 2048 // G), generator=gen, device="cuda").mul_(0.15).exp_().mul_(std / 2.6)
        out[r, :, :, 1024:] = s.to(torch.bfloat16).view(torch.uint8)
    return out


def _tokens(gen, T, K, dtype):
    """Activations after a normalisation: unit normal, a few channels eight times larger."""
    x = torch.randn((T, K), generator=gen, device="cuda")
    big = torch.randint(0, K, (max(1, K // 512),), generator=gen, device="cuda")
    x[:, big] *= 8
    return x.to(DTYPES[dtype])


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    if c["op"] == "quantize":
        E, N, K = c["E"], c["N"], c["K"]
        w = torch.randn((E, N, K), generator=gen, device="cuda").mul_(K ** -0.5)
        w[:, :, ::97] *= 4  # a few wide columns
        if c["src"] != "e4m3":
            return dict(c, w=w.to(DTYPES[c["src"]]), block=None)
        blocks = w.view(E, N // 128, 128, K // 128, 128)
        block = blocks.abs().amax(dim=(2, 4)) / 448
        w = (blocks / block[:, :, None, :, None]).clamp(-448, 448).view(E, N, K).to(torch.float8_e4m3fn)
        return dict(c, w=w, block=block)
    if c["op"] == "dequantize":
        return dict(c, w=_packed(gen, c["E"], c["N"], c["K"], c["G"], c["K"] ** -0.5))
    if c["op"] == "linear":
        w = _packed(gen, 1, c["N"], c["K"], c["G"], c["K"] ** -0.5)[0]
        return dict(c, x=_tokens(gen, c["T"], c["K"], c["dtype"]), w=w)
    T, E, H, I = c["T"], c["E"], c["H"], c["I"]
    logits = torch.randn((T, E_GLOBAL), generator=gen, device="cuda")
    if c["config"] == "group":  # one group of 32 experts, the shard's first, draws most of every token's choice
        first = c["offset"] // 32 * 32
        logits[:, first:first + 32] += 5.0
    bias = (torch.randn((E_GLOBAL,), generator=gen, device="cuda") * 0.1).to(torch.bfloat16)
    return dict(c, x=_tokens(gen, T, H, c["dtype"]), logits=logits, bias=bias, scale=2.5,
                w1=_packed(gen, E, 2 * I, H, c["G"], H ** -0.5), w2=_packed(gen, E, H, I, c["G"], I ** -0.5))


# ------------------------------------------------------------------ plain forms
def _unpack(w, N, K, G):
    """W4 [..., Nt, Kt, tile] -> fp32 [..., N, K], exact (4 bits times 8)."""
    lead, Nt, Kt = w.shape[:-3], w.shape[-3], w.shape[-2]
    words = w[..., :1024].contiguous().view(torch.int32).view(*lead, Nt, Kt, 2, 8, 4, 4, 1)
    words = ((words >> 3) & 0x1FFFFFFF) | (words << 29)
    shift = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], dtype=torch.int32, device=w.device)
    q = ((words >> shift) & 15).to(torch.int8) - 8  # [..., Nt, Kt, h, g, t, j, element]
    n = len(lead)
    q = q.permute(*range(n), n, n + 2, n + 3, n + 1, n + 5, n + 4, n + 6).reshape(*lead, Nt * 16, K // G, G)
    s = w[..., 1024:].contiguous().view(torch.bfloat16).view(*lead, Nt, Kt, 128 // G, 8, 2)
    s = s.permute(*range(n), n, n + 4, n + 3, n + 1, n + 2).reshape(*lead, Nt * 16, K // G, 1)
    return (q.float() * s.float()).view(*lead, Nt * 16, K)[..., :N, :]


def _plain_quantize(w, block, G):
    w = w.float()
    if block is not None:
        w = w * block.repeat_interleave(128, 1).repeat_interleave(128, 2)
    g = w.view(*w.shape[:-1], w.shape[-1] // G, G)
    top = g.abs().amax(-1, keepdim=True)
    s = (top / torch.full_like(top, 7.0)).to(torch.bfloat16).float()  # a tensor: a number would be a product with 1/7
    s = torch.where(s < MIN_NORMAL, torch.zeros_like(s), s)
    q = torch.where(s > 0, (g / s).round().clamp(-8, 7), torch.zeros_like(g))
    return (q * s).view(w.shape)


def _scores(logits, bias):
    """Scores as the router defines them, in fp32 with a correctly rounded exponential; the chosen experts [T, 8]."""
    s = 1.0 / (1.0 + torch.exp(-logits.double()).float())
    b = s + bias.float()
    T = s.shape[0]
    two = b.view(T, N_GROUP, -1).sort(dim=-1, descending=True).values[..., :2]
    kept = (two[..., 0] + two[..., 1]).sort(dim=-1, descending=True, stable=True).indices[:, :KEPT_GROUPS]
    keep = torch.zeros((T, N_GROUP), dtype=torch.bool, device=s.device).scatter_(1, kept, True)
    b = torch.where(keep.repeat_interleave(E_GLOBAL // N_GROUP, 1), b, torch.full_like(b, torch.finfo(b.dtype).min))
    return s, b.sort(dim=-1, descending=True, stable=True).indices[:, :TOP_K]


def _plain_moe(s):
    T, E, H, I, G = s["T"], s["E"], s["H"], s["I"], s["G"]
    score, chosen = _scores(s["logits"], s["bias"])
    weight = score.gather(1, chosen)
    weight = weight / (weight.sum(1, keepdim=True) + 1e-20) * s["scale"]
    local = chosen - s["offset"]
    here = (local >= 0) & (local < E)
    weight, local = torch.where(here, weight, torch.zeros_like(weight)), local.clamp(0, E - 1)
    x = s["x"].float()
    if T * TOP_K < E:  # the experts of each (token, slot)
        w1, w2 = _unpack(s["w1"][local], 2 * I, H, G), _unpack(s["w2"][local], H, I, G)
        a = (w1 @ x[:, None, :, None]).squeeze(-1)
        h = a[..., I:] * torch.sigmoid(a[..., I:]) * a[..., :I]
        y = ((w2 @ h[..., None]).squeeze(-1) * weight[..., None]).sum(1)
    else:  # every token through every local expert
        dense = torch.zeros((T, E), device=x.device).scatter_add_(1, local, weight)
        a = x @ _unpack(s["w1"], 2 * I, H, G).transpose(1, 2)
        h = a[..., I:] * torch.sigmoid(a[..., I:]) * a[..., :I]
        y = ((h @ _unpack(s["w2"], H, I, G).transpose(1, 2)) * dense.t()[..., None]).sum(0)
    return y.to(s["x"].dtype)


# ------------------------------------------------------------------ one pass
_lib = None


def _framework():
    global _lib
    if _lib is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "flashinfer-bench-moe_b200"))
        import fbmoe_lib
        import main as solution

        _lib = (fbmoe_lib, solution)
    return _lib


def run(s):
    if own:
        lib, solution = _lib or _framework()
        if s["op"] == "quantize":
            packed = lib.quantize_w4(s["w"], s["G"], block_scale=s["block"])
            return lib.dequantize_w4(packed, s["N"], DTYPES[s["out"]])
        if s["op"] == "dequantize":
            return lib.dequantize_w4(s["w"], s["N"], DTYPES[s["out"]])
        if s["op"] == "linear":
            return lib.linear_w4(s["x"], s["w"], s["N"])
        return solution.fused_moe_w4(s["logits"], s["bias"], s["x"], s["w1"], s["w2"], s["offset"], s["scale"])
    if s["op"] == "quantize":
        return _plain_quantize(s["w"], s["block"], s["G"]).to(DTYPES[s["out"]])
    if s["op"] == "dequantize":
        return _unpack(s["w"], s["N"], s["K"], s["G"]).to(DTYPES[s["out"]])
    if s["op"] == "linear":
        return (s["x"].float() @ _unpack(s["w"], s["N"], s["K"], s["G"]).t()).to(s["x"].dtype)
    return _plain_moe(s)


def work(case):
    c = case
    size = {"bf16": 2, "f16": 2, "f32": 4, "e4m3": 1}
    per = 0.5 + 2.0 / c["G"]
    if c["op"] == "quantize":
        n = c["E"] * c["N"] * c["K"]
        return {"bytes": n * (size[c["src"]] + size[c["out"]]), "flops": 3 * n}
    if c["op"] == "dequantize":
        n = c["E"] * c["N"] * c["K"]
        return {"bytes": n * (per + size[c["out"]]), "flops": n}
    if c["op"] == "linear":
        T, N, K = c["T"], c["N"], c["K"]
        return {"bytes": N * K * per + 2 * T * (N + K), "flops": 2 * T * N * K}
    # a token chooses 8 of 256 experts alike, or (one hot group) nearly all 8 of that group's 32
    T, E, H, I = c["T"], c["E"], c["H"], c["I"]
    hot = c["config"] == "group"
    pool = min(E, 32) if hot else E
    share = TOP_K / 32 if hot else TOP_K / E_GLOBAL
    active, pairs = pool * (1 - (1 - share) ** T), T * pool * share
    return {"bytes": active * 3 * H * I * per + 4 * T * H + 4 * T * E_GLOBAL, "flops": 6 * H * I * pairs}


# ------------------------------------------------------------------ 64 bits
def _decoded(tiles, G):
    """[Nt, Kt, tile] -> fp64 [16 Nt, 128 Kt], one value at a time: for row n and column k, the word and the bits that hold it."""
    Nt, Kt, tile = tiles.shape
    r = torch.arange(16, device=tiles.device)[:, None]
    k = torch.arange(128, device=tiles.device)[None, :]
    e = k % 8
    word = ((r // 8 * 8 + r % 8) * 4 + k // 8 % 4) * 4 + k // 32
    bit = 3 + 4 * (e // 2) + 16 * (e % 2)  # of the word; the last one wraps round
    flat = tiles.reshape(Nt * Kt, tile)
    value = torch.zeros((Nt * Kt, 16, 128), dtype=torch.float64, device=tiles.device)
    for i in range(4):
        b = (bit + i) % 32
        value += ((flat[:, word * 4 + b // 8].int() >> (b % 8)) & 1).double() * 2 ** i
    at = 1024 + 2 * (k // G * 16 + r % 8 * 2 + r // 8)
    raw = (flat[:, at].int() | (flat[:, at + 1].int() << 8)) << 16
    value = (value - 8) * raw.view(torch.float32).double()
    return value.view(Nt, Kt, 16, 128).transpose(1, 2).reshape(Nt * 16, Kt * 128)


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "quantize":
        found = []
        for e in range(s["E"]):
            w = s["w"][e].double()
            if s["block"] is not None:  # the weight is the fp32 product
                w = (w * s["block"][e].double().repeat_interleave(128, 0).repeat_interleave(128, 1)).float().double()
            g = w.view(w.shape[0], -1, s["G"])
            step = (g.abs().amax(2, keepdim=True) / 7).float().to(torch.bfloat16).double()  # the scale is held in bf16
            step = step * (step >= MIN_NORMAL)
            q = (g / step).float().double().round().clamp(-8, 7)  # one fp32 division
            found.append((q * step).nan_to_num(0.0).view(w.shape))
        return torch.stack(found)
    if s["op"] == "dequantize":
        return torch.stack([_decoded(s["w"][e], s["G"])[:s["N"]] for e in range(s["E"])])
    if s["op"] == "linear":
        x = s["x"].double()
        return torch.cat([x @ _decoded(part, s["G"]).t() for part in s["w"].split(256)], 1)[:, :s["N"]]
    _, chosen = _scores(s["logits"], s["bias"])  # the choice is defined on fp32 scores
    score = torch.sigmoid(s["logits"].double()).gather(1, chosen)
    weight = score / (score.sum(1, keepdim=True) + 1e-20) * s["scale"]
    y = torch.zeros((s["T"], s["H"]), dtype=torch.float64, device="cuda")
    for e in torch.unique(chosen).tolist():
        if not 0 <= e - s["offset"] < s["E"]:
            continue
        t, slot = (chosen == e).nonzero(as_tuple=True)
        a = s["x"][t].double() @ _decoded(s["w1"][e - s["offset"]], s["G"]).t()
        gate = a[:, s["I"]:]
        h = gate / (1 + torch.exp(-gate)) * a[:, :s["I"]]
        y[t] += (h @ _decoded(s["w2"][e - s["offset"]], s["G"]).t()) * weight[t, slot][:, None]
    return y
