"""What is timed to judge the speed of the microscaled operators: weights in 4 bits, rows in 8 bits, the norm that makes
such rows, and the products of the two.

The format: numbers along the depth in blocks of 32 that share one power of two, kept as a byte s that stands for
2^(s - 127).  Rows are E4M3 (up to 448): the scale is the smallest power of two by which the block's largest number is no
more than 448.  Weights are E2M1 (0, 0.5, 1, 1.5, 2, 3, 4, 6): the scale is 2^(floor(log2(largest)) - 2), and what is over 6
by it becomes 6.  Both round to nearest, ties to the even code.  A depth is padded with zeros to whole groups of 128.

A case's ``op``:

* ``weight``: a weight ``[n, k]`` to 4 bits, ``gated``: the gate's rows above the up projection's;
* ``rows``: rows ``[t, k]`` to 8 bits;
* ``norm``: ``h = base + planes + bias`` (``planes`` sums of ``[t, k]`` that a product split over its depth has left), and the
  norm of h's rows in 8 bits: the root-mean-square norm, or (``layer``) the layer norm;
* ``linear``: rows in 8 bits times a weight in 4, ``out``: "store" (bfloat16, with a bias) or "add" (fp32, to another tensor);
* ``gated``: silu(x Wg^T) * (x Wu^T) of n features as rows in 8 bits.

What is held in 8 or 4 bits is returned as the values it stands for, in bfloat16, which has them all."""
import math

import torch

own = False

BLOCK, GROUP, EPS = 32, 128, 1e-6
#: (hidden, intermediate, rows of q, k and v) of the shapes that bench.py measures, Qwen2.5's 0.5B, 1.5B and 7B
SHAPES = ((896, 4864, 1152), (1536, 8960, 2048), (3584, 18944, 4608))


def case(name, op, **sizes):
    c = dict({"op": op}, **sizes)
    return dict(c, name=name) if name else c


def listed():
    return [
        # loading a model: the smallest model's down projection, and the gate and up projections of the largest
        case("weight_05b_down", "weight", n=896, k=4864, dtype="bfloat16", gated=False),
        case("weight_7b_gate_up", "weight", n=37888, k=3584, dtype="bfloat16", gated=True),
        # what attention leaves for its output projection: eight decoded tokens, and a prompt of an odd length
        case("rows_7b_8", "rows", t=8, k=3584, dtype="bfloat16"),
        case("rows_15b_1999", "rows", t=1999, k=1536, dtype="bfloat16"),
        # the norm before a sublayer: one decoded token of the smallest model, a batch of odd size, a prompt of the largest
        case("norm_05b_1", "norm", t=1, k=896, planes=4, bias=False, layer=False),
        case("norm_15b_37", "norm", t=37, k=1536, planes=2, bias=False, layer=False),
        case("norm_7b_2048", "norm", t=2048, k=3584, planes=1, bias=False, layer=False),
        # q, k and v of one decoded token; the down projection of a batch into the stream; q, k and v of a prompt
        case("linear_05b_qkv_1", "linear", t=1, n=1152, k=896, out="store"),
        case("linear_7b_down_8", "linear", t=8, n=3584, k=18944, out="add"),
        case("linear_7b_qkv_2048", "linear", t=2048, n=4608, k=3584, out="store"),
        # the gate and up projections of a few requests, and of a prompt: the largest case
        case("gated_15b_5", "gated", t=5, n=8960, k=1536),
        case("gated_7b_1999", "gated", t=1999, n=18944, k=3584),
    ]


def log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("weight", "rows", "norm", "linear", "linear", "linear", "gated", "gated"))
    hidden, inter, qkv = rng.choice(SHAPES)
    # two of three are a model's own sizes, the third any size
    odd = rng.random() < 0.33
    k, n = log_between(rng, 33, 4864), log_between(rng, 30, 8960)
    t = log_between(rng, 1, 1999)
    dtype = rng.choice(("bfloat16", "bfloat16", "float32"))
    if op == "weight":
        k, n = (k, n) if odd else rng.choice(((hidden, inter), (inter, hidden), (hidden, qkv), (hidden, hidden)))
        gated = rng.random() < 0.4
        return case(None, op, n=2 * n if gated else n, k=k, dtype=dtype, gated=gated)
    if op == "rows":
        return case(None, op, t=t, k=k if odd else rng.choice((hidden, hidden, inter)), dtype=dtype)
    if op == "norm":
        return case(None, op, t=t, k=k if odd else hidden, planes=rng.choice((0, 1, 2, 3, 4, 8)) if t <= 64 else rng.choice((0, 1, 2)), bias=rng.random() < 0.3, layer=rng.random() < 0.3)
    if op == "linear":
        n, k = (n, k) if odd else rng.choice(((qkv, hidden), (hidden, hidden), (hidden, inter)))
        return case(None, op, t=t, n=n, k=k, out=rng.choice(("store", "add")))
    n, k = (n, k) if odd else (inter, hidden)
    return case(None, op, t=t, n=n, k=k)


def padded(k):
    return -(-k // GROUP) * GROUP


def work(c):
    op, row = c["op"], lambda k: 33 / 32 * k  # bytes of a row in 8 bits
    if op == "weight":
        return {"bytes": c["n"] * c["k"] * ((2 if c["dtype"] == "bfloat16" else 4) + 2), "flops": 0}
    if op == "rows":
        return {"bytes": c["t"] * c["k"] * ((2 if c["dtype"] == "bfloat16" else 4) + 2), "flops": 0}
    if op == "norm":
        return {"bytes": c["t"] * c["k"] * (4 * (2 + c["planes"]) + 2) + 4 * c["k"], "flops": 0}
    rows = c["n"] * (2 if op == "gated" else 1)
    out = c["t"] * c["n"] * (2 if op == "gated" or c["out"] == "store" else 8)
    return {"bytes": int(rows * c["k"] * 17 / 32 + c["t"] * row(c["k"]) + out), "flops": 2 * c["t"] * rows * c["k"]}


# ---- what a case's seed decides -------------------------------------------------------------------------------------

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def random_rows(gen, t, k):
    """Rows as a decoder's are: mostly N(0, 1), every 97th channel 20 times as large, rows of different size."""
    x = torch.randn(t, k, generator=gen, device="cuda")
    x[:, ::97] *= 20.0
    return x * torch.exp(torch.randn(t, 1, generator=gen, device="cuda"))


def random_bytes(gen, shape, lo, hi):
    return torch.randint(lo, hi, shape, generator=gen, device="cuda", dtype=torch.int32).to(torch.uint8)


def weight_codes(gen, n, k):
    """A checkpoint's weight in 4 bits: two codes a byte, the first in the low half, and a scale for each 32, most of them about 2^-7."""
    kp = padded(k)
    codes = random_bytes(gen, (n, kp // 2), 0, 256)
    scales = (120 + 1.5 * torch.randn(n, kp // BLOCK, generator=gen, device="cuda")).round().clamp(112, 126).to(torch.uint8)
    codes[:, (k + 1) // 2 :] = 0  # zeros behind the depth
    if k % 2:
        codes[:, k // 2] &= 15
    return codes, scales


def prepare(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    op, k = c["op"], c["k"]
    s = {"case": c}
    if op == "weight":
        # a weight matrix, rows of different size, as training leaves them
        w = 0.02 * torch.randn(c["n"], k, generator=gen, device="cuda") * torch.exp(0.3 * torch.randn(c["n"], 1, generator=gen, device="cuda"))
        s["w"] = w.to(getattr(torch, c["dtype"]))
        return s
    if op == "rows":
        s["x"] = random_rows(gen, c["t"], k).to(getattr(torch, c["dtype"]))
        return s
    if op == "norm":
        s["base"] = random_rows(gen, c["t"], k)
        s["owed"] = torch.randn(c["planes"], c["t"], k, generator=gen, device="cuda") if c["planes"] else None
        s["weight"] = 1 + 0.1 * torch.randn(k, generator=gen, device="cuda")
        s["bias"] = 0.1 * torch.randn(k, generator=gen, device="cuda") if c["bias"] else None
        s["shift"] = 0.1 * torch.randn(k, generator=gen, device="cuda") if c["layer"] else None
        s["h"] = torch.empty_like(s["base"])
        return s
    kp, t, rows = padded(k), c["t"], c["n"] * (2 if op == "gated" else 1)
    # rows as the norm leaves them: a block's largest number is between 224 and 448, the others normal below it
    x = (120 * torch.randn(t, kp, generator=gen, device="cuda")).clamp(-448, 448)
    x[:, k:] = 0
    s["x_codes"] = x.to(torch.float8_e4m3fn).view(torch.uint8)
    s["x_scales"] = random_bytes(gen, (t, kp // BLOCK), 117, 121)
    s["w_codes"], s["w_scales"] = weight_codes(gen, rows, k)
    s["bias"] = torch.randn(c["n"], generator=gen, device="cuda") if c.get("out") == "store" else None
    s["add"] = torch.randn(t, c["n"], generator=gen, device="cuda") if c.get("out") == "add" else None
    if own:
        from alofa_b200 import mx

        # a program lays a weight out once and keeps it so; the rows are as the norm's kernel writes them
        s["w"] = mx.MxWeight.from_codes(s["w_codes"], s["w_scales"], k, gated=op == "gated")
        s["x"] = mx.MxRows(s["x_codes"], s["x_scales"], k)
    return s


# ---- the operators in their plain form ------------------------------------------------------------------------------


def blocks_of(x):
    """The last axis, padded to whole blocks, as [..., blocks, 32] in 32 bits."""
    k = x.shape[-1]
    x = torch.nn.functional.pad(x.float(), (0, -k % BLOCK))
    return x.reshape(*x.shape[:-1], -1, BLOCK)


def times_power(x, e):
    """x * 2^e, exact in 32 bits for the exponents met here: two factors, each a normal number."""
    half = torch.div(e, 2, rounding_mode="floor")
    return torch.ldexp(torch.ldexp(x, half), e - half)


def plain_values(x, weights):
    """What x's numbers become in 8 bits (``weights``: 4 bits) with a scale for each 32."""
    b = blocks_of(x)
    m, e = torch.frexp(b.abs().amax(-1, keepdim=True))  # largest = m 2^e, m in [1/2, 1)
    e = e.int()
    scale = (e - 3 if weights else e - 9 + (m > 0.875).int()).clamp(-127, 127)
    v = times_power(b, -scale)
    least, bits, most = (0, 1, 6.0) if weights else (-6, 3, 448.0)
    step = (torch.frexp(v.abs())[1].int() - 1).clamp(min=least) - bits  # the exponent of a unit in the last place
    v = times_power(torch.round(times_power(v, -step)), step).clamp(-most, most)
    return times_power(v, scale).flatten(-2)[..., : x.shape[-1]]


def plain_weight(codes, scales, k):
    """The numbers that a weight's codes and scales stand for."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    v = table[torch.stack((codes & 15, codes >> 4), -1).flatten(-2).int()]
    return (v.unflatten(-1, (-1, BLOCK)) * torch.exp2(scales.float() - 127).unsqueeze(-1)).flatten(-2)[:, :k]


def plain_rows(codes, scales, k):
    v = codes.view(torch.float8_e4m3fn).float()
    return (v.unflatten(-1, (-1, BLOCK)) * torch.exp2(scales.float() - 127).unsqueeze(-1)).flatten(-2)[:, :k]


def plain(s):
    c = s["case"]
    op, k = c["op"], c["k"]
    if op == "weight":
        return plain_values(s["w"], True).bfloat16()
    if op == "rows":
        return plain_values(s["x"], False).bfloat16()
    if op == "norm":
        h = s["base"]
        if s["owed"] is not None:
            h = h + s["owed"].sum(0)
        if s["bias"] is not None:
            h = h + s["bias"]
        d = h - h.mean(-1, keepdim=True) if c["layer"] else h
        y = d / torch.sqrt((d * d).mean(-1, keepdim=True) + EPS) * s["weight"]
        if c["layer"]:
            y = y + s["shift"]
        return {"h": h, "rows": plain_values(y, False).bfloat16()}
    y = plain_rows(s["x_codes"], s["x_scales"], k) @ plain_weight(s["w_codes"], s["w_scales"], k).T
    if op == "gated":
        g, u = y[:, : c["n"]], y[:, c["n"] :]
        return plain_values(g / (1 + torch.exp(-g)) * u, False).bfloat16()
    return (y + s["bias"]).bfloat16() if c["out"] == "store" else y + s["add"]


def run(s):
    if not own:
        return plain(s)
    from alofa_b200 import mx

    c = s["case"]
    op = c["op"]
    if op == "weight":
        return mx.pack_weight(s["w"], gated=c["gated"]).dequantize()
    if op == "rows":
        return mx.quantize_rows(s["x"]).dequantize()
    if op == "norm":
        rows = mx.norm_rows(s["h"], s["weight"], EPS, base=s["base"], owed=s["owed"], bias=s["bias"], shift=s["shift"])
        return {"h": s["h"], "rows": rows.dequantize()}
    if op == "gated":
        return mx.gated_linear(s["x"], s["w"]).dequantize()
    if c["out"] == "store":
        return mx.linear(s["x"], s["w"], bias=s["bias"])
    return mx.linear(s["x"], s["w"], add=s["add"])


# ---- the same from the definition, in 64 bits -----------------------------------------------------------------------


def representable(weights):
    """Every number from zero up that a code stands for, in the codes' order."""
    if weights:
        return torch.tensor(E2M1, dtype=torch.float64, device="cuda")
    low = [i / 512 for i in range(8)]  # below the smallest normal number, 2^-6
    return torch.tensor(low + [(8 + i) / 8 * 2.0 ** e for e in range(-6, 9) for i in range(8)][:-1], dtype=torch.float64, device="cuda")


def exact_values(x, weights):
    """The nearest representable numbers, found among all of them; a tie goes to the even code."""
    r, k = representable(weights), x.shape[-1]
    most = float(r[-1])
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for at in range(0, x.shape[0], 2048):  # pieces that fit
        part = x[at : at + 2048].double()
        b = torch.nn.functional.pad(part, (0, -k % BLOCK)).unflatten(-1, (-1, BLOCK))
        top = b.abs().amax(-1, keepdim=True)
        safe = torch.where(top > 0, top, torch.ones_like(top))
        if weights:
            e = torch.floor(torch.log2(safe)) - 2
        else:
            e = torch.ceil(torch.log2(safe / most))
        # a logarithm next to a whole number may have been rounded over it
        if weights:
            e = torch.where(torch.exp2(e + 3) <= safe, e + 1, e)
            e = torch.where(torch.exp2(e + 2) > safe, e - 1, e)
        else:
            e = torch.where(torch.exp2(e) * most < safe, e + 1, e)
            e = torch.where(torch.exp2(e - 1) * most >= safe, e - 1, e)
        scale = torch.exp2(e.clamp(-127, 127))
        v = b / scale
        size = v.abs().clamp(max=most)
        above = torch.searchsorted(r, size.contiguous()).clamp(max=r.numel() - 1)
        below = (above - 1).clamp(min=0)
        up, down = r[above] - size, size - r[below]
        code = torch.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
        got = torch.where(v < 0, -r[code], r[code]) * scale
        out[at : at + 2048] = got.flatten(-2)[:, :k]
    return out


def exact_product(x_codes, x_scales, w_codes, w_scales, k):
    r, q = representable(False), representable(True)
    power = lambda s: torch.exp2(s.double() - 127).repeat_interleave(BLOCK, -1)  # noqa: E731
    x = torch.where(x_codes >= 128, -r[(x_codes & 127).long()], r[(x_codes & 127).long()]) * power(x_scales)
    nibbles = torch.empty(w_codes.shape[0], 2 * w_codes.shape[1], dtype=torch.uint8, device=w_codes.device)
    nibbles[:, 0::2], nibbles[:, 1::2] = w_codes & 15, w_codes >> 4
    w = torch.where(nibbles >= 8, -q[(nibbles & 7).long()], q[(nibbles & 7).long()]) * power(w_scales)
    return x[:, :k] @ w[:, :k].T


def exact(c, seed):
    s = prepare(c, seed)
    op = c["op"]
    if op == "weight":
        return exact_values(s["w"], True)
    if op == "rows":
        return exact_values(s["x"], False)
    if op == "norm":
        h = s["base"].double()
        for z in range(c["planes"]):
            h = h + s["owed"][z].double()
        if c["bias"]:
            h = h + s["bias"].double()
        mean = h.sum(1, keepdim=True) / c["k"] if c["layer"] else 0.0
        y = (h - mean) * ((h - mean).square().sum(1, keepdim=True) / c["k"] + EPS).rsqrt() * s["weight"].double()
        return {"h": h, "rows": exact_values(y + s["shift"].double() if c["layer"] else y, False)}
    y = exact_product(s["x_codes"], s["x_scales"], s["w_codes"], s["w_scales"], c["k"])
    if op == "gated":
        g, u = y.split(c["n"], 1)
        return exact_values(g * torch.sigmoid(g) * u, False)
    return y + s["bias"].double() if c["out"] == "store" else y + s["add"].double()
