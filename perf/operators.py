"""The 4-bit and expert operators of blockfp8_b200, as cases to measure.

Three operators, each in its plain form (elementary torch operations in 32
bits) and as the framework's calls:

  quant   x -> MXFP4 (e2m1 codes, one power-of-two scale per 32 values along
          K) and back to the values that the codes stand for
  linear  x [M, K] bf16 @ W [N, K]^T with W in MXFP4 and x quantized to MXFP4
          as part of the call
  moe     a mixture-of-experts layer for a few tokens: router logits to the
          top k experts, gate and up projections, SiLU-and-mul, down
          projection, weighted sum; expert weights in block FP8 (e4m3, one
          fp32 scale per 128 x 128) or in MXFP4

`own` false: the plain forms; true: the framework's kernels.
"""

import math
import random

import torch

own = False

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # the magnitudes of e2m1
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


# ---- the cases --------------------------------------------------------------


def listed():
    return [
        # the activations of a decode batch of 16, quantized and read back: launch latency
        {"name": "quant decode batch", "op": "quant", "m": 16, "k": 4096, "dtype": "bfloat16"},
        # an odd batch with a K that ends inside a 128-wide scale tile, in 32 bits
        {"name": "quant ragged fp32", "op": "quant", "m": 777, "k": 4128, "dtype": "float32"},
        # quantizing a gate-up weight when a model is loaded
        {"name": "quant gate_up weight", "op": "quant", "m": 24576, "k": 4096, "dtype": "bfloat16"},
        # one token through the qkv projection
        {"name": "linear qkv 1 token", "op": "linear", "m": 1, "n": 6144, "k": 4096},
        # a decode batch through the down projection (long K)
        {"name": "linear down 24 tokens", "op": "linear", "m": 24, "n": 4096, "k": 12288},
        # a short prompt of odd length, N off the tile grid
        {"name": "linear ragged prompt", "op": "linear", "m": 509, "n": 6120, "k": 4128},
        # a long prompt through gate_up: the headline shape of the FP8 path
        {"name": "linear gate_up 8192", "op": "linear", "m": 8192, "n": 24576, "k": 4096},
        # one token through a small block-FP8 layer of many experts
        {"name": "moe fp8 1 token", "op": "moe", "fmt": "fp8", "t": 1, "e": 128, "top_k": 8, "h": 2048, "i": 768},
        # a decode batch through a wider block-FP8 layer
        {"name": "moe fp8 13 tokens", "op": "moe", "fmt": "fp8", "t": 13, "e": 64, "top_k": 6, "h": 4096, "i": 1408},
        # the largest batch of this form: every expert is read
        {"name": "moe fp8 64 tokens", "op": "moe", "fmt": "fp8", "t": 64, "e": 128, "top_k": 8, "h": 4096, "i": 1280},
        # one token through an MXFP4 layer whose H and I end inside a 128-wide block
        {"name": "moe mxfp4 1 token", "op": "moe", "fmt": "mxfp4", "t": 1, "e": 32, "top_k": 4, "h": 2880, "i": 2880},
        # a decode batch through an MXFP4 layer
        {"name": "moe mxfp4 40 tokens", "op": "moe", "fmt": "mxfp4", "t": 40, "e": 64, "top_k": 4, "h": 4096, "i": 2048},
    ]


def _log_uniform(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def draw(rng: random.Random):
    op = rng.choice(("quant", "linear", "linear", "moe", "moe"))
    if op == "quant":
        k = 32 * max(1, int(_log_uniform(rng, 1, 384)))
        m = int(_log_uniform(rng, 1, min(32768, (24576 * 4096) // k)))
        return {"op": op, "m": m, "k": k, "dtype": rng.choice(("bfloat16", "bfloat16", "float16", "float32"))}
    if op == "linear":
        while True:
            m, k = int(_log_uniform(rng, 1, 8192)), 32 * int(_log_uniform(rng, 8, 384))
            n = 8 * int(_log_uniform(rng, 32, 3200))
            if m * n * k <= 8192 * 24576 * 4096:
                return {"op": op, "m": m, "n": n, "k": k}
    while True:
        e = int(_log_uniform(rng, 4, 160))
        c = {"op": op, "fmt": rng.choice(("fp8", "mxfp4")), "t": int(_log_uniform(rng, 1, 64.99)), "e": e,
             "top_k": rng.randint(1, min(8, e)), "h": 32 * int(_log_uniform(rng, 16, 224)),
             "i": 32 * int(_log_uniform(rng, 8, 160))}
        if e * c["h"] * c["i"] <= 128 * 4096 * 1280:
            return c


def work(case):
    """Bytes (each input read once, each output written once) and operations of one pass."""
    if case["op"] == "quant":
        mk, size = case["m"] * case["k"], 4 if case["dtype"] == "float32" else 2
        return {"bytes": mk * (size + 2), "flops": 2 * mk}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": 2 * m * k + n * k // 2 + n * k // 32 + 2 * m * n, "flops": 2 * m * n * k}
    t, e, top_k, h, i = (case[x] for x in ("t", "e", "top_k", "h", "i"))
    used = e * (1 - (1 - top_k / e) ** t)  # experts that t tokens meet, on average
    per_weight = 1 if case["fmt"] == "fp8" else 0.5 + 1 / 32
    return {"bytes": int(used * 3 * h * i * per_weight) + 4 * t * h + 4 * t * e, "flops": 6 * t * top_k * h * i}


# ---- the inputs -------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(m, k, dtype, gen):
    """Hidden states: normal, with some channels an order of magnitude larger."""
    channel = torch.exp(0.5 * torch.randn(k, device="cuda", generator=gen))
    channel[torch.randint(0, k, (max(1, k // 256),), device="cuda", generator=gen)] *= 12.0
    return (torch.randn(m, k, device="cuda", generator=gen) * channel).to(dtype)


def _mxfp4_weights(rows, k, gen):
    """Normal weights as MXFP4: packed codes [rows, k / 2], scale bytes [rows, k / 32]."""
    packed, scales = [], []
    step = max(1, (1 << 28) // k)
    for r in range(0, rows, step):
        w = 0.02 * torch.randn(min(step, rows - r), k, device="cuda", generator=gen)
        code, e = _mxfp4_codes(w)
        packed.append(code[:, 0::2] | (code[:, 1::2] << 4))
        scales.append((e + 127).to(torch.uint8))
    return torch.cat(packed), torch.cat(scales)


def _tiled(scales):
    """Scale bytes [..., R, K / 32] in the operand layout [..., ceil(R / 128), ceil(K / 128), 32, 16]:
    row r of a 128-row tile at [r % 32], its four bytes of a 128-wide K block at 4 * (r / 32)."""
    *lead, rows, kb = scales.shape
    rt, kt = -(-rows // 128), -(-kb // 4)
    s = torch.nn.functional.pad(scales, (0, kt * 4 - kb, 0, rt * 128 - rows))
    s = s.reshape(*lead, rt, 4, 32, kt, 4)
    n = len(lead)
    return s.permute(*range(n), n, n + 3, n + 2, n + 1, n + 4).reshape(*lead, rt, kt, 32, 16).contiguous()


def prepare(case, seed):
    gen = _generator(seed)
    if case["op"] == "quant":
        return {"op": "quant", "x": _activations(case["m"], case["k"], DTYPES[case["dtype"]], gen)}
    if case["op"] == "linear":
        q, s = _mxfp4_weights(case["n"], case["k"], gen)
        return {"op": "linear", "x": _activations(case["m"], case["k"], torch.bfloat16, gen), "w": q, "w_scales": _tiled(s)}
    t, e, h, i = (case[x] for x in ("t", "e", "h", "i"))
    popular = 0.5 * torch.randn(e, device="cuda", generator=gen)
    state = {"op": "moe", "fmt": case["fmt"], "top_k": case["top_k"],
             "x": torch.randn(t, h, device="cuda", generator=gen).to(torch.bfloat16),
             "logits": torch.randn(t, e, device="cuda", generator=gen) + popular}
    for name, rows, k in (("w13", 2 * i, h), ("w2", h, i)):
        if case["fmt"] == "fp8":
            w = torch.empty(e, rows, k, dtype=torch.float8_e4m3fn, device="cuda")
            flat = w.view(-1)
            for at in range(0, flat.numel(), 1 << 28):
                part = flat[at:at + (1 << 28)]
                part.copy_((90.0 * torch.randn(part.numel(), device="cuda", generator=gen)).clamp_(-448, 448))
            sizes = (e, -(-rows // 128), -(-k // 128))
            state[name], state[name + "_scales"] = w, (0.5 + torch.rand(sizes, device="cuda", generator=gen)) * 2e-4
        else:
            q, s = _mxfp4_weights(e * rows, k, gen)
            state[name], state[name + "_scales"] = q.view(e, rows, k // 2), _tiled(s.view(e, rows, k // 32))
    return state


# ---- the plain forms --------------------------------------------------------


def _power(e):
    """2^e in 32 bits, from its bits (a computed power may be off by a unit, which moves values across a border)."""
    return torch.where(e > -127, (e + 127) << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _mxfp4_codes(x):
    """e2m1 codes (one a byte) and the scales' exponents of x [M, K] in 32 bits.  The exponent of a block of
    32 is that of its largest magnitude less 2, so that the largest lies in [4, 8); values round to the
    nearest of GRID, ties to the even code, and stop at 6."""
    blocks = x.view(x.shape[0], -1, 32)
    amax = blocks.abs().amax(dim=2)
    e = torch.where(amax > 0, torch.frexp(amax).exponent - 3, -127).clamp_(-127, 125)
    v = (blocks * _power(-e).unsqueeze(2)).abs_()
    code = (v > 0.25).to(torch.uint8)
    code += v >= 0.75
    code += v > 1.25
    code += v >= 1.75
    code += v > 2.5
    code += v >= 3.5
    code += v > 5.0
    return (code + 8 * (blocks < 0)).view(x.shape), e


def _mxfp4_values(code, e):
    """The values of codes (one a byte) [..., K] under exponents [..., K / 32], in 32 bits."""
    grid = torch.tensor(GRID + tuple(-v for v in GRID), device=code.device)
    v = grid[code.int()]
    return (v.view(*e.shape, 32) * _power(e).unsqueeze(-1)).view(code.shape)


def _unpack(packed):
    return torch.stack((packed & 15, packed >> 4), dim=-1).flatten(-2)


def _untiled(tiles, rows, kb):
    """The exponents [..., rows, kb] of scale bytes in the operand layout."""
    *lead, rt, kt, _, _ = tiles.shape
    n = len(lead)
    s = tiles.reshape(*lead, rt, kt, 32, 4, 4).permute(*range(n), n, n + 3, n + 2, n + 1, n + 4)
    return s.reshape(*lead, rt * 128, kt * 4)[..., :rows, :kb].int() - 127


def _mxfp4_weight(packed, tiles):
    return _mxfp4_values(_unpack(packed), _untiled(tiles, packed.shape[-2], packed.shape[-1] // 16))


def _fp8_weight(w, scales):
    *_, rows, k = w.shape
    s = scales.repeat_interleave(128, dim=-2)[..., :rows, :].repeat_interleave(128, dim=-1)[..., :k]
    return w.float() * s


def _moe(state):
    x, logits, top_k = state["x"].float(), state["logits"], state["top_k"]
    tokens, experts = logits.shape
    ids = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :top_k]
    weights = torch.softmax(logits.gather(1, ids), dim=1)  # softmax over all, renormalized over the chosen
    weight_of = _fp8_weight if state["fmt"] == "fp8" else _mxfp4_weight

    def expert_weights(name, which):
        w, s = state[name], state[name + "_scales"]
        if which is not None:
            w, s = w.view(torch.uint8)[which].view(w.dtype), s[which]
        return weight_of(w, s)

    if tokens * top_k <= experts:  # one product per pair of token and expert
        pairs = ids.flatten()
        gate, up = torch.bmm(expert_weights("w13", pairs), x.repeat_interleave(top_k, 0).unsqueeze(2)).chunk(2, dim=1)
        hidden = gate * torch.sigmoid(gate) * up
        z = torch.bmm(expert_weights("w2", pairs), hidden).view(tokens, top_k, -1)
        return (z * weights.unsqueeze(2)).sum(1).to(state["x"].dtype)
    # every expert on every token, and the weights of the experts that a token did not choose are zero
    share = torch.zeros(tokens, experts, device=x.device).scatter_(1, ids, weights)
    gate, up = torch.matmul(x, expert_weights("w13", None).transpose(1, 2)).chunk(2, dim=2)
    hidden = gate * torch.sigmoid(gate) * up
    z = torch.bmm(hidden, expert_weights("w2", None).transpose(1, 2))
    return (z * share.t().unsqueeze(2)).sum(0).to(state["x"].dtype)


def _hold_bytes(state):
    """MXFP4 codes come out of prepare()'s arithmetic in 64-bit integers.  A program holds its weights as the
    bytes that the calls take: they are narrowed once, at a state's first pass, and kept in the state."""
    for name in ("w", "w13", "w2"):
        if name in state and state[name].dtype == torch.int64:
            state[name] = state[name].to(torch.uint8)


def run(state):
    if own:
        import blockfp8_b200 as bf

        _hold_bytes(state)
        if state["op"] == "quant":
            return bf.dequantize_mxfp4(*bf.quantize_mxfp4(state["x"]))
        if state["op"] == "linear":
            return bf.linear_mxfp4(state["x"], state["w"], state["w_scales"])
        return bf.moe(state["x"], state["logits"], state["w13"], state["w13_scales"], state["w2"], state["w2_scales"],
                      top_k=state["top_k"])
    if state["op"] == "moe":
        return _moe(state)
    values = _mxfp4_values(*_mxfp4_codes(state["x"].float()))
    if state["op"] == "quant":
        return values.to(torch.bfloat16)
    return (values @ _mxfp4_weight(state["w"], state["w_scales"]).t()).to(torch.bfloat16)


# ---- the definitions, in 64 bits --------------------------------------------


def _nearest(v):
    """Values in units of their block's scale to e2m1: a step of 0.5 below 2, of 1 below 4, of 2 up to 6; torch.round
    takes ties to the even multiple, which is the even code on every one of the three pieces."""
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).to(v.dtype)
    return torch.sign(v) * (torch.round(a / step) * step).clamp(max=6.0)


def _rounded(x):
    """x [M, K] as MXFP4 holds it, from the definition: scale 2^(floor(log2 max) - 2)."""
    x = x.double().unflatten(1, (-1, 32))
    top = x.abs().amax(2, keepdim=True)
    # the exponent field of a double is floor(log2) + 1023, and a field with no fraction is the power itself
    field = top.clamp(min=2.0 ** -125).view(torch.int64) >> 52
    power = ((field - 2) << 52).view(torch.float64)
    return (_nearest(x / power) * power).flatten(1)


def _magnitude(code):
    """e2m1 from its fields: two bits of exponent (bias 1), one of mantissa."""
    e, m, sign = (code >> 1) & 3, code & 1, (code >> 3).double()
    return torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * torch.exp2(e.double() - 1)) * (1 - 2 * sign)


def _weight64(packed, tiles):
    """[rows, K] of one MXFP4 matrix, in 64 bits."""
    rows, k = packed.shape[0], 2 * packed.shape[1]
    v = torch.empty(rows, k, dtype=torch.float64, device=packed.device)
    v[:, 0::2], v[:, 1::2] = _magnitude(packed & 15), _magnitude(packed >> 4)
    r = torch.arange(rows, device=packed.device)[:, None]
    b = torch.arange(k // 32, device=packed.device)[None, :]
    byte = tiles[r // 128, b // 4, r % 32, 4 * ((r % 128) // 32) + b % 4]
    power = ((byte.long() - 127 + 1023) << 52).view(torch.float64)
    return v * power.repeat_interleave(32, 1)


def _block64(w, scales):
    rows, k = w.shape
    r, c = torch.arange(rows, device=w.device) // 128, torch.arange(k, device=w.device) // 128
    return w.double() * scales.double()[r][:, c]


def exact(case, seed):
    state = prepare(case, seed)
    if state["op"] == "quant":
        return _rounded(state["x"])
    if state["op"] == "linear":
        return _rounded(state["x"]) @ _weight64(state["w"], state["w_scales"]).t()
    x, logits, top_k = state["x"].double(), state["logits"].double(), state["top_k"]
    matrix = _block64 if state["fmt"] == "fp8" else _weight64
    order = torch.sort(-logits, dim=1, stable=True).indices[:, :top_k]
    p = torch.exp(logits - logits.amax(1, keepdim=True)).gather(1, order)
    p = p / p.sum(1, keepdim=True)
    y = torch.zeros_like(x)
    for e in order.unique().tolist():
        t, j = (order == e).nonzero(as_tuple=True)
        both = x[t] @ matrix(state["w13"][e], state["w13_scales"][e]).t()
        gate, up = both[:, : case["i"]], both[:, case["i"]:]
        z = (gate / (1 + torch.exp(-gate)) * up) @ matrix(state["w2"][e], state["w2_scales"][e]).t()
        y.index_add_(0, t, z * p[t, j].unsqueeze(1))
    return y
