"""The operators of the 4-bit weight path and what they are measured on.

``run`` computes each operator in elementary torch operations (32-bit, rounded once at the end), or, where ``own`` is true, makes the
framework's call.  Both start from the same stored data, which ``prepare`` makes:

* weights w[n, k] = scale[n, k // G] * q[n, k], q in -8..7, G in {32, 64, 128}; the stored form pads the rows to a multiple of 16 and
  the columns to a multiple of 64 (128 if G is), with zeros.  ``packed`` uint8 [tiles of 16 rows, blocks of 64 columns, 32, 16]: of a tile's
  block, entry [4 g + t, 8 r + 4 c + b] holds row g + 8 r, its low four bits column 32 c + 8 t + b, its high ones column 32 c + 8 t + 4 + b.
  ``scales`` bfloat16 [tiles, groups, 16]: entry [2 g + r] is row g + 8 r; they have five significant bits, so that every weight is a
  bfloat16 number.
* rows in 8 bits x[t, k] = scale[t, k // G] * q[t, k]: ``q`` int8 [T, padded columns], ``scales`` float32 [T, groups].

Rows in 8 bits that an operator makes are compared as the numbers that they stand for, rounded to bfloat16.
"""
import math

import torch

own = False
DEV = "cuda:0"
EPS = 1e-6


def listed():
    return [
        # output projection of the 0.5B shape, one token: nothing but latency
        dict(name="o_896_t1", op="product8", M=1, N=896, K=896, G=32, bias=False, f32=True),
        # q|k|v of the 7B shape with its bias, one token
        dict(name="qkv_7b_t1", op="product8", M=1, N=4608, K=3584, G=128, bias=True, f32=False),
        # gate/up of the 7B shape, the batch that the benchmark decodes
        dict(name="gate_up_7b_t8", op="product8", M=8, N=37888, K=3584, G=128, bias=False, f32=False),
        # down of the 7B shape, a full batch: the longest sums
        dict(name="down_7b_t64", op="product8", M=64, N=3584, K=18944, G=64, bias=False, f32=True),
        # gate/up of the 14B shape on 16-bit rows
        dict(name="gate_up_14b_t16_bf16", op="product", M=16, N=27648, K=5120, G=128, bias=False, f32=False),
        # ragged in every direction: three tokens, odd rows, columns that end inside a group
        dict(name="odd_t3_bf16", op="product", M=3, N=1003, K=1100, G=32, bias=True, f32=True),
        # a prompt through the down product of the 7B shape
        dict(name="down_7b_t1999_bf16", op="product", M=1999, N=3584, K=18944, G=128, bias=False, f32=True),
        # the norm before a product, the K splits of the product before it still to be added: one token, a batch
        dict(name="norm_896_t1", op="norm", T=1, H=896, G=32, S=4),
        dict(name="norm_14b_t64", op="norm", T=64, H=5120, G=128, S=5),
        # ... and the rows of a prompt, after a 16-bit update
        dict(name="norm_7b_t2048", op="norm", T=2048, H=3584, G=128, S=0),
        # the gated unit between gate/up and down: one token of the 0.5B shape, a large batch of the 7B shape
        dict(name="glu_4864_t1", op="glu", T=1, H=4864, G=64, act="silu"),
        dict(name="glu_7b_t128", op="glu", T=128, H=18944, G=128, act="gelu_tanh"),
    ]


def draw(rng):
    span = lambda a, b: int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))  # noqa: E731
    op, G = rng.choice(["product8", "product8", "product", "norm", "glu"]), rng.choice([32, 64, 128])
    if op == "norm":
        H = rng.choice([64 * span(1, 128), span(64, 8192)])
        return dict(op=op, T=min(span(1, 4096), 8_000_000 // H), H=H, G=G, S=rng.choice([0, 1, 3, 4, 7, 12]))
    if op == "glu":
        H = rng.choice([64 * span(1, 300), span(64, 19000)])
        return dict(op=op, T=min(span(1, 2048), 4_000_000 // H + 1), H=H, G=G, act=rng.choice(["silu", "gelu_tanh", "relu"]))
    N, K = rng.choice([16 * span(4, 2400), span(64, 38000)]), rng.choice([128 * span(1, 148), span(64, 19000)])
    N = min(N, 140_000_000 // K)
    M = span(1, 128) if op == "product8" or rng.random() < 0.5 else min(span(1, 2000), 100_000_000_000 // (N * K) + 1)
    return dict(op=op, M=M, N=N, K=K, G=G, bias=rng.random() < 0.5, f32=rng.random() < 0.5)


def _padded(n, step):
    return (n + step - 1) // step * step


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    normal = lambda *shape: torch.randn(*shape, device=DEV, generator=g)  # noqa: E731
    G, s = case["G"], dict(case)
    if case["op"] == "norm":
        T, H = case["T"], case["H"]
        s["h"] = normal(T, H) * torch.exp(0.5 * normal(H))              # a few columns of the stream are much larger than the rest
        s["pending"] = 0.2 * normal(case["S"], T, H) if case["S"] else normal(T, H).to(torch.bfloat16)
        s["w"] = (1.0 + 0.2 * normal(H)).to(torch.bfloat16)
        return s
    if case["op"] == "glu":
        s["gu"] = (1.5 * normal(case["T"], 2 * case["H"])).to(torch.bfloat16)
        return s
    M, N, K = case["M"], case["N"], case["K"]
    Np, Kp = _padded(N, 16), _padded(K, max(G, 64))
    w = torch.zeros(Np, Kp, device=DEV)
    w[:N, :K] = normal(N, K) / math.sqrt(K)
    groups = w.view(Np, Kp // G, G)
    mantissa, exponent = torch.frexp(groups.abs().amax(-1) / 7.5)
    scale = torch.ldexp((mantissa * 32).round_() / 32, exponent).to(torch.bfloat16)
    q = (groups / scale.float().clamp_min(1e-30)[..., None]).round_().clamp_(-8, 7).to(torch.int8).view(Np, Kp)
    # row 16 tile + g + 8 r, column 64 block + 32 c + 8 t + 4 half + b
    q = q.view(Np // 16, 2, 8, Kp // 64, 2, 4, 2, 4).permute(0, 3, 2, 5, 1, 4, 7, 6)
    s["packed"] = ((q[..., 0] & 15) | (q[..., 1] << 4)).view(torch.uint8).reshape(Np // 16, Kp // 64, 32, 16).contiguous()
    s["scales"] = scale.view(Np // 16, 2, 8, Kp // G).permute(0, 3, 2, 1).reshape(Np // 16, Kp // G, 16).contiguous()
    s["b"] = normal(N).to(torch.bfloat16) if case["bias"] else None
    x = normal(M, K) * torch.exp(0.5 * normal(K))
    if case["op"] == "product":
        s["x"] = x.to(torch.bfloat16)
        return s
    xp = torch.zeros(M, Kp, device=DEV)
    xp[:, :K] = x
    a = xp.view(M, Kp // G, G).abs().amax(-1) / 127
    s["xs"] = a.contiguous()
    s["xq"] = (xp.view(M, Kp // G, G) / a.clamp_min(1e-30)[..., None]).round_().to(torch.int8).view(M, Kp)
    return s


def _weight(s):
    """The stored weights as float32 [N, K]."""
    N, K, G = s["N"], s["K"], s["G"]
    tiles, blocks = s["packed"].shape[:2]
    p = s["packed"].view(torch.int8).view(tiles, blocks, 8, 4, 2, 2, 4)
    q = torch.stack([((p & 15) ^ 8) - 8, p >> 4], dim=-1)               # both halves with their signs
    q = q.permute(0, 4, 2, 1, 5, 3, 7, 6).reshape(16 * tiles, 64 * blocks)
    scale = s["scales"].view(tiles, -1, 8, 2).permute(0, 3, 2, 1).reshape(16 * tiles, -1)
    return (q.float().view(16 * tiles, -1, G) * scale.float()[..., None]).view(16 * tiles, -1)[:N, :K]


def _to_8_bits_and_back(y, G):
    """Numbers in 64 bits to 8-bit groups of ``G`` along the rows, and the numbers that those stand for, in bfloat16."""
    T, H = y.shape
    p = torch.zeros(T, _padded(H, G), dtype=y.dtype, device=y.device)
    p[:, :H] = y
    p = p.view(T, -1, G)
    a = (p.abs().amax(-1, keepdim=True) / 127)
    q = torch.where(a > 0, p / a, 0.0).round()
    return (q * a.float()).view(T, -1)[:, :H].to(torch.bfloat16)


def _act(x, kind):
    if kind == "relu":
        return torch.where(x > 0, x, 0.0)
    if kind == "silu":
        return x / (1 + torch.exp(-x))
    u = 2 * 0.7978845608028654 * (x + 0.044715 * x * x * x)             # 0.5 (1 + tanh(u / 2)) = 1 / (1 + exp(-u))
    return x / (1 + torch.exp(-u))


def run(s):
    if own:
        return _run_own(s)
    if s["op"] == "norm":
        s["h"].add_(s["pending"].float() if s["pending"].dim() == 2 else s["pending"].sum(0))
        h = s["h"].double()                                             # (a number's 8 bits may hang on its last ones)
        y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS) * s["w"].double()
        return {"h": s["h"], "y": _to_8_bits_and_back(y, s["G"])}
    if s["op"] == "glu":
        gu = s["gu"].double()
        return _to_8_bits_and_back(_act(gu[:, 0::2], s["act"]) * gu[:, 1::2], s["G"])
    if s["op"] == "product":
        x = s["x"].float()
    else:
        x = (s["xq"].float().view(s["M"], -1, s["G"]) * s["xs"][..., None]).view(s["M"], -1)[:, :s["K"]]
    y = x @ _weight(s).T
    if s["b"] is not None:
        y += s["b"].float()
    return y if s["f32"] else y.to(torch.bfloat16)


def _run_own(s):
    from rocmforge_b200 import kernels
    if s["op"] == "norm":
        y = kernels.add_rmsnorm_q8(s["h"], s["w"], EPS, torch.bfloat16, s["G"], pending=s["pending"])
        return {"h": s["h"], "y": y.materialize()}
    if s["op"] == "glu":
        return kernels.swiglu_q8(s["gu"], s["G"], activation=s["act"]).materialize()
    w = kernels.W4Weight(s["packed"], s["scales"], s["N"], s["K"], s["G"])
    x = s["x"] if s["op"] == "product" else kernels.Q8Rows(s["xq"], s["xs"], s["K"], s["G"], torch.bfloat16)
    return kernels.gemm_w4(x, w, s["b"], out_f32=s["f32"])


def work(case):
    G = case["G"]
    if case["op"] == "norm":
        T, H = case["T"], case["H"]
        return {"bytes": T * H * (8 + (4 * case["S"] or 2) + 1 + 4 / G) + 2 * H, "flops": T * H * (8 + case["S"])}
    if case["op"] == "glu":
        return {"bytes": case["T"] * case["H"] * (4 + 1 + 4 / G), "flops": case["T"] * case["H"] * 12}
    M, N, K = case["M"], case["N"], case["K"]
    rows = M * K * (2 if case["op"] == "product" else 1 + 4 / G)
    return {"bytes": N * K * (0.5 + 2 / G) + rows + M * N * (4 if case["f32"] else 2) + (2 * N if case["bias"] else 0), "flops": 2 * M * N * K}


def exact(case, seed):
    """From the definitions, in 64 bits: a weight, a row's number and a group's scale each looked up by their place."""
    s = prepare(case, seed)
    G = case["G"]

    def through_8_bits(y):
        T, H = y.shape
        out = torch.empty_like(y)
        for lo in range(0, H, G):
            part = y[:, lo:lo + G]
            a = part.abs().max(dim=1, keepdim=True).values / 127.0
            out[:, lo:lo + G] = torch.where(a == 0, torch.zeros_like(part), torch.round(part / a) * a)
        return out

    if case["op"] == "norm":
        p = s["pending"].double()
        h = s["h"].double() + (p if p.dim() == 2 else p.sum(dim=0))
        ms = torch.linalg.vector_norm(h, dim=1, keepdim=True).square() / case["H"]
        return {"h": h, "y": through_8_bits(h * (ms + EPS).rsqrt() * s["w"].double()[None])}
    if case["op"] == "glu":
        gate, up = s["gu"].double().view(case["T"], -1, 2).unbind(-1)
        if case["act"] == "relu":
            a = gate.clamp_min(0)
        elif case["act"] == "silu":
            a = gate * torch.sigmoid(gate)
        else:
            a = 0.5 * gate * (1 + torch.tanh(math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3)))
        return through_8_bits(a * up)
    N, K = case["N"], case["K"]
    n = torch.arange(N, device=DEV)[:, None]
    scales = s["scales"].double()
    by_place = s["packed"].reshape(-1)
    y = torch.zeros(case["M"], N, dtype=torch.float64, device=DEV)
    for lo in range(0, K, 2048):
        k = torch.arange(lo, min(K, lo + 2048), device=DEV)[None]
        g, r, t, c = n % 8, n % 16 // 8, k % 32 // 8, k % 64 // 32
        at = ((n // 16 * s["packed"].shape[1] + k // 64) * 32 + 4 * g + t) * 16 + 8 * r + 4 * c + k % 4
        v = by_place[at].to(torch.int16) >> (4 * (k % 8 // 4)).to(torch.int16) & 15
        w = torch.where(v > 7, v - 16, v).double() * scales[n // 16, k // G, 2 * g + r]
        if case["op"] == "product":
            x = s["x"][:, lo:lo + 2048].double()
        else:
            x = s["xq"][:, k[0]].double() * s["xs"].double()[:, k[0] // G]
        y += x @ w.T
    return y if s["b"] is None else y + s["b"].double()
