"""Operators around the quantized MoE layers, with the cases on which they are timed and compared.

fp8:  y = Q(x) . W^T, the dense product in block-scaled e4m3 (``fp8.linear``).  W holds one e4m3 code per weight and one
      float32 scale per 128 x 128 block; Q rounds x to e4m3 with one float32 scale per row and 128 columns, or x comes as
      codes and scales already.  Dense projections and shared experts next to the block-FP8 expert layer.
ggml: out[i] = x[row i] . W_g^T for the rows of every group g, the product grouped by expert over GGUF Q4_K / Q6_K
      weights (``kogarashi.grouped_gemm``).  `up`: two matrices side by side (gate | up); `swiglu`: the rows of x hold
      gate | up and silu(gate) * up is what gets multiplied (the down product).

`run` computes the plain forms with elementary torch operations in float32; with `own` set it calls the library.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
Q4_K, Q6_K = 12, 14


def listed():
    return [
        # one token through a projection of a decode step: the weights are streamed once, latency counts
        dict(name="fp8 one token", op="fp8", m=1, n=4096, k=4096, x="bf16", out="bf16"),
        # a speculative window through a smaller projection, float32 activations
        dict(name="fp8 window", op="fp8", m=7, n=1536, k=2048, x="f32", out="f32"),
        # an odd batch, a last block of 16 columns, rows that are no multiple of a tile
        dict(name="fp8 odd", op="fp8", m=77, n=1000, k=1552, x="f16", out="f16"),
        # a batch of decode streams or a short prompt
        dict(name="fp8 batch", op="fp8", m=256, n=4096, k=2048, x="bf16", out="bf16"),
        # a prefill chunk through a projection of a layer
        dict(name="fp8 prefill", op="fp8", m=4096, n=4096, k=4096, x="bf16", out="bf16"),
        # the largest: a long prefill whose activations were quantized by the operator before
        dict(name="fp8 prefill codes", op="fp8", m=8192, n=8192, k=4096, x="codes", out="bf16"),
        # gate and up of one token's eight experts out of 128
        dict(name="ggml one token", op="ggml", ty=Q4_K, groups=128, tokens=1, topk=8, n=768, k=2048, up=True, swiglu=False,
             x="f32", out="f32", skew=0.0),
        # down of sixteen tokens: most experts that are hit have a single row
        dict(name="ggml sixteen tokens", op="ggml", ty=Q6_K, groups=256, tokens=16, topk=8, n=2048, k=1024, up=False, swiglu=True,
             x="f32", out="f32", skew=0.0),
        # a verify window or a short prompt over skewed experts
        dict(name="ggml window", op="ggml", ty=Q4_K, groups=256, tokens=256, topk=8, n=1024, k=2048, up=True, swiglu=False,
             x="bf16", out="bf16", skew=0.5),
        # an odd number of groups and of columns, some groups empty
        dict(name="ggml odd", op="ggml", ty=Q6_K, groups=37, tokens=45, topk=3, n=1000, k=768, up=False, swiglu=False,
             x="f16", out="f16", skew=1.0),
        # a prefill chunk: gate and up
        dict(name="ggml prefill gate up", op="ggml", ty=Q4_K, groups=128, tokens=4096, topk=8, n=768, k=2048, up=True, swiglu=False,
             x="bf16", out="bf16", skew=0.0),
        # the same chunk: SwiGLU and down in float32, as the layer's residual stream has it
        dict(name="ggml prefill down", op="ggml", ty=Q6_K, groups=128, tokens=4096, topk=8, n=2048, k=768, up=False, swiglu=True,
             x="f32", out="f32", skew=0.0),
    ]


def draw(rng):
    def span(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    while True:
        if rng.random() < 0.5:
            m, n, k = span(1, 8192), span(1, 8192), 16 * span(1, 512)
            c = dict(op="fp8", m=m, n=n, k=k, x=rng.choice(["f32", "bf16", "f16", "codes"]), out=rng.choice(["f32", "bf16", "f16"]))
            if m * n * k <= 8192 * 8192 * 4096:
                return c
        else:
            groups, tokens, topk = span(1, 256), span(1, 4096), rng.randint(1, 8)
            n, k = span(1, 4096), 256 * span(1, 16)
            x, out = rng.choice(["f32", "bf16", "f16"]), rng.choice(["f32", "bf16", "f16"])
            c = dict(op="ggml", ty=rng.choice([Q4_K, Q6_K]), groups=groups, tokens=tokens, topk=min(topk, groups), n=n, k=k,
                     up=rng.random() < 0.5, swiglu=False, x=x, out=out, skew=rng.choice([0.0, 0.5, 1.0]))
            if not c["up"]:
                c["swiglu"] = rng.random() < 0.5
            nn = n * (2 if c["up"] else 1)
            rows = tokens * c["topk"]
            most = min(tokens, 40 + rows * (1.5 if c["skew"] == 0 else 12) / groups)      # rows of the busiest group, about
            if groups * nn * k <= 1 << 29 and rows * nn * k <= 32768 * 1536 * 2048 and groups * most * (2 * k + nn) <= 1 << 30:
                return c


def work(case):
    if case["op"] == "fp8":
        m, n, k = case["m"], case["n"], case["k"]
        kb, nb = -(-k // 128), -(-n // 128)
        xb = m * k + m * kb * 4 if case["x"] == "codes" else m * k * TYPES[case["x"]].itemsize
        return {"bytes": xb + n * k + nb * kb * 4 + m * n * TYPES[case["out"]].itemsize, "flops": 2 * m * n * k}
    g, t, rows, k = case["groups"], case["tokens"], case["tokens"] * case["topk"], case["k"]
    n = case["n"] * (2 if case["up"] else 1)
    # expected number of groups that have rows (uniform popularity)
    active = g * (1 - (1 - case["topk"] / g) ** t)
    wbytes = active * n * (k // 256) * (144 if case["ty"] == Q4_K else 210)
    x_rows = rows if case["swiglu"] else t
    xbytes = x_rows * k * (2 if case["swiglu"] else 1) * TYPES[case["x"]].itemsize
    return {"bytes": wbytes + xbytes + rows * n * TYPES[case["out"]].itemsize, "flops": 2 * rows * n * k}


# ---- inputs --------------------------------------------------------------------------------------------------------


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def block_fp8(g, n, k):
    """N(0, 1/sqrt(k)) weights as e4m3 codes and one scale per 128 x 128 block."""
    nb, kb = -(-n // 128), -(-k // 128)
    w = torch.zeros(nb * 128, kb * 128, device="cuda")
    w[:n, :k] = torch.randn(n, k, generator=g, device="cuda") * k ** -0.5
    blocks = w.view(nb, 128, kb, 128)
    scale = blocks.abs().amax((1, 3)) / 448
    codes = (blocks / scale[:, None, :, None]).clamp(-448, 448).view(nb * 128, kb * 128)[:n, :k]
    return codes.to(torch.float8_e4m3fn).view(torch.uint8).contiguous(), scale.contiguous()


def q4k(w):
    """float32 [rows, k] -> Q4_K rows: per 256 columns d, dmin (f16), twelve bytes of 6-bit scales and mins, 128 bytes of nibbles."""
    rows, k = w.shape
    b = w.view(-1, 8, 32)
    low = (-b.amin(2)).clamp_min(0)                                   # m >= 0
    step = (b.amax(2) + low) / 15
    d = (step.amax(1, keepdim=True) / 63).half().float().clamp_min(6e-8)
    dm = (low.amax(1, keepdim=True) / 63).half().float().clamp_min(6e-8)
    sc, mi = (step / d).round().clamp(0, 63), (low / dm).round().clamp(0, 63)
    q = ((b + (dm * mi)[:, :, None]) / (d * sc).clamp_min(1e-12)[:, :, None]).round().clamp(0, 15).to(torch.uint8)
    sc, mi = sc.to(torch.uint8), mi.to(torch.uint8)
    head = torch.cat([d.half().view(torch.uint8), dm.half().view(torch.uint8)], 1)
    packed = torch.cat([sc[:, :4] | ((sc[:, 4:] >> 4) << 6), mi[:, :4] | ((mi[:, 4:] >> 4) << 6), (sc[:, 4:] & 15) | ((mi[:, 4:] & 15) << 4)], 1)
    nibbles = (q[:, 0::2] | (q[:, 1::2] << 4)).reshape(-1, 128)
    return torch.cat([head, packed, nibbles], 1).view(rows, -1)


def q6k(w):
    """float32 [rows, k] -> Q6_K rows in the device layout: per 256 columns ql 128 | qh 64 | int8 scales 16, then the f16
    block scales of the row padded to 16 bytes."""
    rows, k = w.shape
    b = w.view(-1, 16, 16)
    step = b.abs().amax(2) / 31
    d = (step.amax(1, keepdim=True) / 127).half().float().clamp_min(6e-8)
    sc = (step / d).round().clamp(1, 127)
    q = ((b / (d * sc)[:, :, None]).round().clamp(-32, 31) + 32).to(torch.uint8).view(-1, 2, 4, 32)     # [half][group of 32][l]
    ql = torch.stack([(q[:, :, 0] & 15) | ((q[:, :, 2] & 15) << 4), (q[:, :, 1] & 15) | ((q[:, :, 3] & 15) << 4)], 2).reshape(-1, 128)
    qh = ((q[:, :, 0] >> 4) | ((q[:, :, 1] >> 4) << 2) | ((q[:, :, 2] >> 4) << 4) | ((q[:, :, 3] >> 4) << 6)).reshape(-1, 64)
    body = torch.cat([ql, qh, sc.to(torch.int8).view(torch.uint8)], 1).view(rows, -1)
    tail = torch.zeros(rows, (2 * (k // 256) + 15) // 16 * 16, dtype=torch.uint8, device=w.device)
    tail[:, : 2 * (k // 256)] = d.half().view(rows, -1).view(torch.uint8)
    return torch.cat([body, tail], 1)


def experts(g, ty, groups, n, k):
    """groups x n rows of N(0, 0.02) weights, quantized a few groups at a time."""
    pack = q4k if ty == Q4_K else q6k
    at_once = max(1, (1 << 25) // (n * k))
    return torch.cat([pack(torch.randn(min(at_once, groups - i) * n, k, generator=g, device="cuda") * 0.02) for i in range(0, groups, at_once)])


def prepare(case, seed):
    g = generator(seed)
    s = dict(case=case)
    if case["op"] == "fp8":
        m, n, k = case["m"], case["n"], case["k"]
        s["w"], s["ws"] = block_fp8(g, n, k)
        x = torch.randn(m, k, generator=g, device="cuda")
        if case["x"] == "codes":
            codes, scale = quantize(x)
            s["x"], s["xs"] = codes.to(torch.float8_e4m3fn).view(torch.uint8).contiguous(), scale.contiguous()
        else:
            s["x"], s["xs"] = x.to(TYPES[case["x"]]), None
        return s
    groups, tokens, topk, n, k = case["groups"], case["tokens"], case["topk"], case["n"], case["k"]
    names = ("w", "wu") if case["up"] else ("w",)
    for name in names:
        s[name] = experts(g, case["ty"], groups, n, k)
    # routes: top-k of Gumbel noise over a popularity that falls as rank^-skew, then the rows sorted by expert
    noise = -torch.log(-torch.log(torch.rand(tokens, groups, generator=g, device="cuda").clamp(1e-9, 1 - 1e-7)))
    popularity = -case["skew"] * torch.log(1 + torch.randperm(groups, generator=g, device="cuda").float())
    ids = (noise + popularity).topk(topk, 1).indices.reshape(-1)
    order = ids.argsort(stable=True)
    counts = torch.bincount(ids, minlength=groups)
    s["ranges"] = torch.stack([counts, counts.cumsum(0) - counts], 1).to(torch.int32).contiguous()
    s["most"] = int(counts.max())
    rows = tokens * topk
    if case["swiglu"]:      # the products of gate and up, one row per route
        s["x"], s["assignments"] = (1.5 * torch.randn(rows, 2 * k, generator=g, device="cuda")).to(TYPES[case["x"]]), None
    else:                   # the tokens' rows, fetched through the routes
        s["x"], s["assignments"] = torch.randn(tokens, k, generator=g, device="cuda").to(TYPES[case["x"]]), order.to(torch.int32)
    return s


# ---- the operators ---------------------------------------------------------------------------------------------------


def quantize(x):
    """e4m3 values (as float32) [m, k] and scales [m, ceil(k/128)] of float rows: scale = absmax / 448 (1 for zeros),
    code = e4m3(x * (1 / scale)), every step rounded to float32."""
    m, k = x.shape
    kb = -(-k // 128)
    xf = torch.nn.functional.pad(x.float(), (0, kb * 128 - k)).view(m, kb, 128)
    top = xf.abs().amax(2)
    scale = torch.where(top == 0, torch.ones_like(top), top / torch.full_like(top, 448))
    codes = (xf * (1 / scale)[:, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn).float()
    return codes.view(m, kb * 128)[:, :k], scale


def decode_q4k(w, k):
    b = w.view(-1, 144)
    d, dm = b[:, 0:2].contiguous().view(torch.float16).float(), b[:, 2:4].contiguous().view(torch.float16).float()
    a, c, e = b[:, 4:8], b[:, 8:12], b[:, 12:16]
    sc = torch.cat([a & 63, (e & 15) | ((a >> 6) << 4)], 1).float()
    mi = torch.cat([c & 63, (e >> 4) | ((c >> 6) << 4)], 1).float()
    qs = b[:, 16:].view(-1, 4, 32)
    q = torch.stack([qs & 15, qs >> 4], 2).view(-1, 8, 32).float()
    return ((d * sc)[:, :, None] * q - (dm * mi)[:, :, None]).view(w.shape[0], k)


def decode_q6k(w, k):
    nb = k // 256
    b = w[:, : nb * 208].reshape(-1, 208)
    d = w[:, nb * 208: nb * 210].contiguous().view(torch.float16).reshape(-1, 1).float()
    ql, qh = b[:, :128].view(-1, 2, 2, 32), b[:, 128:192].view(-1, 2, 32)
    sc = b[:, 192:].view(torch.int8).float()
    low = torch.stack([ql[:, :, 0] & 15, ql[:, :, 1] & 15, ql[:, :, 0] >> 4, ql[:, :, 1] >> 4], 2)
    high = torch.stack([qh & 3, (qh >> 2) & 3, (qh >> 4) & 3, qh >> 6], 2)
    q = (low | (high << 4)).view(-1, 16, 16).float() - 32
    return ((d * sc)[:, :, None] * q).view(w.shape[0], k)


def run(s):
    case = s["case"]
    if own:
        import darask_inference_engine_b200 as D
        out = TYPES[case["out"]]
        if case["op"] == "fp8":
            return D.fp8.linear(s["x"], s["w"], s["ws"], x_scales=s["xs"], out_dtype=out)
        weight = [D.kogarashi.Weight(s[name], case["ty"], case["k"], case["n"], (case["k"], case["n"], case["groups"]))
                  for name in ("w", "wu") if name in s]
        return D.kogarashi.grouped_gemm(s["x"], s["ranges"], *weight, assignments=s["assignments"], topk=case["topk"],
                                        swiglu=case["swiglu"], out_dtype=out)
    if case["op"] == "fp8":
        m, n, k = case["m"], case["n"], case["k"]
        if s["xs"] is None:
            codes, scale = quantize(s["x"])
        else:
            codes, scale = s["x"].view(torch.float8_e4m3fn).float(), s["xs"]
        x = codes * scale.repeat_interleave(128, 1)[:, :k]
        w = s["w"].view(torch.float8_e4m3fn).float() * s["ws"].repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
        return (x @ w.T).to(TYPES[case["out"]])
    groups, n, k = case["groups"], case["n"], case["k"]
    decode = decode_q4k if case["ty"] == Q4_K else decode_q6k
    x = s["x"].float()
    if case["swiglu"]:
        gate, up = x[:, :k], x[:, k:]
        x = gate / (1 + torch.exp(-gate)) * up
    else:
        x = x[s["assignments"].long() // case["topk"]]
    # groups that have rows, their rows padded to the busiest group's number, one batched product, rows back in their order
    active = s["ranges"][:, 0].nonzero().view(-1)
    counts, first = s["ranges"][active, 0].long(), s["ranges"][active, 1].long()
    place = torch.arange(s["most"], device=x.device)
    valid = place[None, :] < counts[:, None]
    at = torch.where(valid, first[:, None] + place[None, :], torch.zeros_like(first)[:, None])
    padded = x[at.view(-1)].view(len(active), s["most"], k)
    w = decode(s["w"].view(groups, -1)[active].view(len(active) * n, -1), k).view(len(active), n, k)
    y = torch.bmm(padded, w.transpose(1, 2))
    if case["up"]:
        w = decode(s["wu"].view(groups, -1)[active].view(len(active) * n, -1), k).view(len(active), n, k)
        y = torch.cat([y, torch.bmm(padded, w.transpose(1, 2))], 2)
    return y[valid].to(TYPES[case["out"]])


# ---- the same from the definitions, in 64 bits -----------------------------------------------------------------------


def e4m3_nearest(v):
    """Nearest e4m3 value (ties to the even code) of float64 numbers of at most 448: three fraction bits, exponents from -6."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e - 1).clamp_min(-6) - 3)
    return torch.round(v / step) * step


def e4m3_table(device):
    code = torch.arange(256, device=device)
    e, f = ((code >> 3) & 15).double(), (code & 7).double()
    v = torch.where(e == 0, f * 2.0 ** -9, (8 + f) * 2.0 ** (e - 10))
    return torch.where(code >= 128, -v, v)


def gguf_weight(rows, ty, k):
    """float64 [r, k] of packed rows, element by element: the byte that holds column j, its shift, its scale."""
    j = torch.arange(k, device=rows.device)
    blk, i = j // 256, j % 256
    as_half = lambda at: (rows[:, at].int() | (rows[:, at + 1].int() << 8)).to(torch.int16).view(torch.float16).double()  # noqa: E731
    if ty == Q4_K:
        base, sub = blk * 144, i // 32
        q = (rows[:, base + 16 + i // 64 * 32 + i % 32].int() >> (4 * (sub % 2)).int()) & 15
        s0 = base + 4 + sub % 4
        high = rows[:, base + 12 + sub % 4].int()
        upper = sub >= 4
        sc = torch.where(upper, (high & 15) | ((rows[:, s0].int() >> 6) << 4), rows[:, s0].int() & 63)
        mi = torch.where(upper, (high >> 4) | ((rows[:, s0 + 4].int() >> 6) << 4), rows[:, s0 + 4].int() & 63)
        return as_half(base) * sc * q - as_half(base + 2) * mi
    base, half, part, l = blk * 208, i // 128, i % 128 // 32, i % 32
    low = (rows[:, base + half * 64 + part % 2 * 32 + l].int() >> (part // 2 * 4).int()) & 15
    high = (rows[:, base + 128 + half * 32 + l].int() >> (2 * part).int()) & 3
    sc = rows[:, base + 192 + i // 16].view(torch.int8).int()
    return as_half(k // 256 * 208 + 2 * blk) * (sc * ((low | (high << 4)) - 32))


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "fp8":
        k, n = case["k"], case["n"]
        block = torch.arange(k, device="cuda") // 128
        table = e4m3_table("cuda")
        if s["xs"] is None:
            x = s["x"].double()
            top = torch.stack([p.abs().amax(1) for p in x.split(128, 1)], 1)
            scale = (top / 448).float().double()                       # the rounding steps that Q is defined with
            scale[top == 0] = 1
            inv = (1 / scale).float().double()
            x = e4m3_nearest((x * inv[:, block]).float().double().clamp(-448, 448)) * scale[:, block]
        else:
            x = table[s["x"].long()] * s["xs"].double()[:, block]
        out = torch.empty(case["m"], n, dtype=torch.float64, device="cuda")
        for i in range(0, n, 128):
            out[:, i:i + 128] = x @ (table[s["w"][i:i + 128].long()] * s["ws"][i // 128].double()[block]).T
        return out
    k, n, names = case["k"], case["n"], ("w", "wu") if case["up"] else ("w",)
    out = torch.empty(case["tokens"] * case["topk"], n * len(names), dtype=torch.float64, device="cuda")
    for e, (count, first) in enumerate(s["ranges"].tolist()):
        if not count:
            continue
        if case["swiglu"]:
            x = s["x"][first:first + count].double()
            x = x[:, :k] * torch.sigmoid(x[:, :k]) * x[:, k:]
        else:
            x = s["x"].double()[s["assignments"][first:first + count].long() // case["topk"]]
        for p, name in enumerate(names):
            out[first:first + count, p * n:(p + 1) * n] = x @ gguf_weight(s[name][e * n:(e + 1) * n], case["ty"], k).T
    return out
