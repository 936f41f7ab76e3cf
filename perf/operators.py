"""Operators of training in 8 bits, as measurable cases.

* ``norm``     - residual addition + RMSNorm with an 8-bit output (``fp8_ops.rmsnorm_quant``) and its backward
                 (``fp8_ops.rmsnorm_quant_bwd``);
* ``quantize`` - 8-bit codes with a power-of-two scale per block of 128 (``fp8_ops.quantize``, ``fp8_ops.quantize_both``);
* ``matmul``   - products of such codes (``fp8_ops.matmul``): forward, input gradient, weight gradient;
* ``adamw``    - one AdamW step over many tensors, states in 32 or 8 bits (``optim_ops.adamw_multi``).

Sizes are the ones of the Llama configurations, the tests and the benchmark of this repository, or generic.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32,
          "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
ITEM = {"bf16": 2, "fp16": 2, "fp32": 4}
BLOCK = 128        # values that share a scale in activations, gradients and weights
STATE_BLOCK = 256  # values that share a scale in an 8-bit optimizer state
EPS = 1e-5
LR, BETA1, BETA2, ADAM_EPS, DECAY, CLIP, GRAD_SCALE, HASH_SEED = 3e-4, 0.9, 0.95, 1e-8, 0.1, 1.0, 0.5, 11

# one decoder layer of Llama-3-8B: QKV, output, gate | up, down, two norms
LAYER_8B = "6144x4096,4096x4096,28672x4096,4096x14336,4096,4096"
# the two-layer model of the tests: embedding, head, final norm, and per layer four matrices and two norms
TINY = "4096x1024,4096x1024,1024," + ",".join(["1536x1024,1024x1024,4096x1024,1024x2048,1024,1024"] * 2)


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # evaluation of a handful of tokens: latency
        {"name": "norm_8x4096", "op": "norm", "back": False, "rows": 8, "width": 4096, "dtype": "bf16", "residual": True},
        # the norm before a layer's MLP, 16384 tokens of Llama-3-8B
        {"name": "norm_16k", "op": "norm", "back": False, "rows": 16384, "width": 4096, "dtype": "bf16", "residual": True},
        # its backward, an odd number of tokens and a width that no power of two divides
        {"name": "norm_back_odd", "op": "norm", "back": True, "rows": 5003, "width": 5120, "dtype": "bf16", "residual": True},
        # the gradient of gate | up, quantised along rows (input gradient) and along tokens (weight gradient)
        {"name": "quantize_grad_16k", "op": "quantize", "how": "both", "rows": 16384, "width": 28672, "dtype": "bf16", "code": "e4m3"},
        # a small model's weight
        {"name": "quantize_weight_tiny", "op": "quantize", "how": "blocks", "rows": 1536, "width": 1024, "dtype": "bf16", "code": "e4m3"},
        # QKV projection of a handful of tokens: bound by reading the weight
        {"name": "matmul_17_tokens", "op": "matmul", "how": "forward", "m": 17, "n": 6144, "k": 4096, "code": "e4m3", "out": "bf16"},
        # gate | up projection of 16384 tokens
        {"name": "matmul_forward_16k", "op": "matmul", "how": "forward", "m": 16384, "n": 28672, "k": 4096, "code": "e4m3", "out": "bf16"},
        # input gradient of the down projection, ragged number of tokens
        {"name": "matmul_dgrad_odd", "op": "matmul", "how": "dgrad", "m": 5003, "n": 14336, "k": 4096, "code": "e4m3", "out": "bf16"},
        # weight gradient of the QKV projection
        {"name": "matmul_wgrad_16k", "op": "matmul", "how": "wgrad", "m": 6144, "n": 4096, "k": 16384, "code": "e4m3", "out": "bf16"},
        # the test model's whole update: 15 tensors, many of them small
        {"name": "adamw_tiny_8", "op": "adamw", "bits": 8, "shapes": TINY, "dtype": "bf16", "clip": True},
        {"name": "adamw_layer_32", "op": "adamw", "bits": 32, "shapes": LAYER_8B, "dtype": "bf16", "clip": True},
        {"name": "adamw_layer_8", "op": "adamw", "bits": 8, "shapes": LAYER_8B, "dtype": "bf16", "clip": True},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["norm", "quantize", "matmul", "matmul", "adamw"])
    if op == "norm":
        width = _log(rng, 64, 8192)
        return {"op": op, "back": rng.random() < 0.5, "rows": _log(rng, 1, min(16384, 16384 * 4096 // width)), "width": width,
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "residual": rng.random() < 0.6}
    if op == "quantize":
        width = _log(rng, 64, 28672)
        return {"op": op, "how": rng.choice(["rows", "cols", "blocks", "both"]), "rows": _log(rng, 1, 16384), "width": width,
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "code": rng.choice(["e4m3", "e4m3", "e5m2"])}
    if op == "matmul":
        n, k = _log(rng, 64, 16384), _log(rng, 64, 16384)
        return {"op": op, "how": rng.choice(["forward", "dgrad", "wgrad"]), "m": _log(rng, 1, min(16384, 16384 * 28672 * 4096 // (n * k))),
                "n": n, "k": k, "code": rng.choice(["e4m3", "e4m3", "e5m2"]), "out": rng.choice(["bf16", "bf16", "fp16"])}
    left, sizes = _log(rng, 1000, 100_000_000), []
    for _ in range(rng.randint(1, 40)):
        sizes.append(_log(rng, 1, max(1, left)))
        left -= sizes[-1]
        if left < 1:
            break
    return {"op": op, "bits": rng.choice([8, 32]), "shapes": ",".join(map(str, sizes)), "dtype": rng.choice(["bf16", "bf16", "fp32"]),
            "clip": rng.random() < 0.6}


def _sizes(case):
    return [math.prod(int(d) for d in s.split("x")) for s in case["shapes"].split(",")]


# --------------------------------------------------------------------------- inputs
def _values(gen, rows, width, dtype, spread=1.0):
    """Activations or gradients: normal values, a few channels with larger ones, a few rows of zeros (padding)."""
    x = torch.randn(rows, width, device="cuda", generator=gen)
    x *= 1.0 + 20.0 * (torch.rand(width, device="cuda", generator=gen) < 0.01)
    if rows > 8:
        x *= torch.rand(rows, 1, device="cuda", generator=gen) > 0.02
    return (x * spread).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": dict(case)}
    op = case["op"]
    if op == "norm":
        dtype, rows, width = DTYPES[case["dtype"]], case["rows"], case["width"]
        state["x"] = _values(gen, rows, width, dtype)
        state["w"] = (1.0 + 0.1 * torch.randn(width, device="cuda", generator=gen)).to(dtype)
        if case["residual"]:
            state["residual"] = _values(gen, rows, width, dtype)
        if case["back"]:
            state["rstd"] = torch.rsqrt(state["x"].double().square().mean(-1) + EPS).float()
            state["dy"] = _values(gen, rows, width, dtype, 1e-2)
    elif op == "quantize":
        state["x"] = _values(gen, case["rows"], case["width"], DTYPES[case["dtype"]], 1e-2)
    elif op == "matmul":
        m, n, k, code = case["m"], case["n"], case["k"], DTYPES[case["code"]]
        how = case["how"]
        a = _values(gen, *((k, m) if how == "wgrad" else (m, k)), torch.float32)
        b = _values(gen, *((n, k) if how == "forward" else (k, n)), torch.float32, 2e-2)
        state["a"] = _quantize(a, (BLOCK, 1) if how == "wgrad" else (1, BLOCK), code)
        state["b"] = _quantize(b, (BLOCK, 1) if how == "wgrad" else (BLOCK, BLOCK), DTYPES["e4m3"])
    else:
        sizes = _sizes(case)
        n, dtype = sum(sizes), DTYPES[case["dtype"]]
        # each tensor begins at a multiple of 256 values of the flat storages, as a program that keeps flat buffers lays them out
        starts, at = [], 0
        for s in sizes:
            starts.append(at)
            at += -(-s // STATE_BLOCK) * STATE_BLOCK
        where = list(zip(starts, sizes))
        w = 0.02 * torch.randn(at, device="cuda", generator=gen)
        g = 2e-3 * torch.randn(at, device="cuda", generator=gen) * (1 + 10 * torch.rand(at, device="cuda", generator=gen) ** 8)
        m = 1e-3 * torch.randn(at, device="cuda", generator=gen)
        v = (1e-3 * torch.randn(at, device="cuda", generator=gen)).square() + 1e-8
        inside = torch.zeros(at, dtype=torch.bool, device="cuda")
        for s, c in where:
            inside[s:s + c] = True
        m, v, w, g = m * inside, v * inside, w * inside, g * inside
        flat = {"param": w.to(dtype), "grad": g.to(dtype)}
        if dtype != torch.float32:
            flat["master"] = flat["param"].float()
        if case["bits"] == 32:
            flat["m"], flat["v"] = m, v
        else:
            for key, t in (("m", m), ("v", v.sqrt())):
                codes, scales, _ = _quantize(t.view(-1, STATE_BLOCK), (1, STATE_BLOCK), torch.float8_e4m3fn)
                flat[key], flat[key + "_scale"] = codes.view(-1), scales.view(-1)
        state["flat"] = flat
        state["step"] = torch.full((1,), 100, dtype=torch.int64, device="cuda")
        part = lambda t, s, c: t[s // STATE_BLOCK:-(-(s + c) // STATE_BLOCK)] if t.dtype == torch.float8_e8m0fnu else t[s:s + c]  # noqa: E731
        state["lists"] = {key: [part(t, s, c) for s, c in where] for key, t in flat.items()}
    return state


# --------------------------------------------------------------------------- plain forms
def _scale_exponent(amax, largest):
    """The smallest k with amax <= largest * 2^k, for largest = 1.75 * 2^e, as an e8m0 exponent; NaN for an amax that is not finite."""
    mantissa, exponent = torch.frexp(amax)
    e = math.frexp(largest)[1]                               # largest = 0.875 * 2^e
    k = (exponent - e + (mantissa > 0.875)).clamp(-127, 127)
    k = torch.where(amax == 0, torch.full_like(k, -127), k)
    return torch.where(torch.isfinite(amax), k + 127, torch.full_like(k, 255))


def _quantize(x, block, code):
    """(codes, scales, block) of a 2-D tensor; the last blocks may be short."""
    rows, cols = x.shape
    br, bc = block
    nr, nc = -(-rows // br), -(-cols // bc)
    padded = torch.zeros(nr * br, nc * bc, device=x.device)
    padded[:rows, :cols] = x
    tiles = padded.view(nr, br, nc, bc)
    largest = torch.finfo(code).max
    e = _scale_exponent(tiles.abs().amax((1, 3)), largest)
    scales = e.to(torch.uint8).view(torch.float8_e8m0fnu)
    codes = (tiles / scales.float()[:, None, :, None]).clamp(-largest, largest).view(nr * br, nc * bc)[:rows, :cols].to(code)
    return codes, scales, block


def _dequantize(q, dtype=torch.float32):
    codes, scales, (br, bc) = q
    rows, cols = codes.shape
    s = scales.to(dtype).repeat_interleave(br, 0)[:rows].repeat_interleave(bc, 1)[:, :cols]
    return codes.to(dtype) * s


def _hash(x):
    """32-bit finaliser of MurmurHash3, on int64 tensors or ints that hold 32-bit words."""
    x = ((x ^ (x >> 16)) * 0x85EBCA6B) & 0xFFFFFFFF
    x = ((x ^ (x >> 13)) * 0xC2B2AE35) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _stochastic(x, floor, bits):
    """Codes and scales of a state: |x| / scale cut to e4m3 after 16 random bits were added behind its last place."""
    n = x.numel()
    blocks = torch.zeros(-(-n // STATE_BLOCK) * STATE_BLOCK, device=x.device)
    blocks[:n] = x
    blocks = blocks.view(-1, STATE_BLOCK)
    scales = _scale_exponent(blocks.abs().amax(1), 448.0).to(torch.uint8).view(torch.float8_e8m0fnu)
    # 2^-120 takes e4m3's smallest exponent to fp32's, so that the cut goes through its denormals too
    y = (blocks.abs() / scales.float()[:, None] * 2.0 ** -120).view(-1)[:n].contiguous()
    code = ((y.view(torch.int32).long() + (bits << 4)) >> 20).clamp(max=0x7E)
    if floor:
        code = torch.where(x > 0, code.clamp(min=1), code)
    code = code | ((x < 0).long() << 7)
    return code.to(torch.uint8).view(torch.float8_e4m3fn), scales


def _adamw_plain(state):
    case, lists = state["case"], state["lists"]
    state["step"] += 1
    t = state["step"].double()
    bc1, bc2 = (1 / (1 - BETA1 ** t)).float(), (1 / (1 - BETA2 ** t)).float()
    coef, norm = GRAD_SCALE, None
    if case["clip"]:
        norm = (state["flat"]["grad"].double() * GRAD_SCALE).square().sum().sqrt()
        coef = GRAD_SCALE * (CLIP / (norm + 1e-6)).clamp(max=1.0).float()
    key = _hash((HASH_SEED + state["step"] * 0x9E3779B1) & 0xFFFFFFFF)
    eight = case["bits"] == 8
    for i in range(len(lists["param"])):
        w = lists["master"][i] if "master" in lists else lists["param"][i]
        g = lists["grad"][i].float() * coef
        m, v = lists["m"][i], lists["v"][i]
        if eight:
            spread = lambda s, n: s.float().repeat_interleave(STATE_BLOCK)[:n]  # noqa: E731
            m32 = m.float() * spread(lists["m_scale"][i], m.numel())
            v32 = (v.float() * spread(lists["v_scale"][i], v.numel())).square()
        else:
            m32, v32 = m, v
        m32 = BETA1 * m32 + (1 - BETA1) * g
        v32 = BETA2 * v32 + (1 - BETA2) * g * g
        w -= LR * (m32 * bc1 / ((v32 * bc2).sqrt() + ADAM_EPS) + DECAY * w)
        if "master" in lists:
            lists["param"][i].copy_(w)
        if eight:
            at = torch.arange(g.numel(), device=g.device)
            r = _hash((at * 0x9E3779B1 + _hash((key + i * 0x85EBCA77) & 0xFFFFFFFF)) & 0xFFFFFFFF)
            codes, scales = _stochastic(m32, False, r & 0xFFFF)
            m.copy_(codes), lists["m_scale"][i].view(torch.uint8).copy_(scales.view(torch.uint8))
            codes, scales = _stochastic(v32.sqrt(), True, r >> 16)
            v.copy_(codes), lists["v_scale"][i].view(torch.uint8).copy_(scales.view(torch.uint8))
        else:
            m.copy_(m32), v.copy_(v32)
    return norm.float().view(1) if norm is not None else None


def _plain(state):
    case = state["case"]
    op = case["op"]
    if op == "norm" and not case["back"]:
        h = state["x"]
        if case["residual"]:
            h = (h.float() + state["residual"].float()).to(h.dtype)
        h32 = h.float()
        rstd = torch.rsqrt(h32.square().mean(-1) + EPS)
        codes, scales, _ = _quantize(h32 * rstd[:, None] * state["w"].float(), (1, BLOCK), DTYPES["e4m3"])
        return {"codes": codes, "scales": scales, "h": h, "rstd": rstd}
    if op == "norm":
        xh = state["x"].float() * state["rstd"][:, None]
        dy = state["dy"].float()
        g = dy * state["w"].float()
        dx = state["rstd"][:, None] * (g - xh * (g * xh).mean(-1, keepdim=True))
        if case["residual"]:
            dx = dx + state["residual"].float()
        return {"dx": dx.to(state["x"].dtype), "dw": (dy * xh).sum(0)}
    if op == "quantize":
        code = DTYPES[case["code"]]
        kinds = {"rows": [(1, BLOCK)], "cols": [(BLOCK, 1)], "blocks": [(BLOCK, BLOCK)], "both": [(1, BLOCK), (BLOCK, 1)]}
        got = [_quantize(state["x"].float(), block, code) for block in kinds[case["how"]]]
        return [t for codes, scales, _ in got for t in (codes, scales)]
    if op == "matmul":
        a, b = _dequantize(state["a"]), _dequantize(state["b"])
        product = (a.t() if case["how"] == "wgrad" else a) @ (b.t() if case["how"] == "forward" else b)
        return product.to(DTYPES[case["out"]])
    norm = _adamw_plain(state)
    return {**{k: v for k, v in state["flat"].items() if k != "grad"}, "step": state["step"], "norm": norm}


# --------------------------------------------------------------------------- the framework's calls
def _own(state):
    from dcp_b200.ops import fp8_ops, optim_ops

    case = state["case"]
    op = case["op"]
    if op == "norm" and not case["back"]:
        y, h, rstd = fp8_ops.rmsnorm_quant(state["x"], state["w"], EPS, state.get("residual"))
        return {"codes": y.codes, "scales": y.scales, "h": h, "rstd": rstd}
    if op == "norm":
        dx, dw = fp8_ops.rmsnorm_quant_bwd(state["x"], state["w"], state["rstd"], state["dy"], state.get("residual"))
        return {"dx": dx, "dw": dw}
    if op == "quantize":
        code = DTYPES[case["code"]]
        if case["how"] == "both":
            got = fp8_ops.quantize_both(state["x"], code)
        else:
            got = [fp8_ops.quantize(state["x"], {"rows": (1, BLOCK), "cols": (BLOCK, 1), "blocks": (BLOCK, BLOCK)}[case["how"]], code)]
        return [t for q in got for t in (q.codes, q.scales)]
    if op == "matmul":
        a, b = fp8_ops.BlockScaled(*state["a"]), fp8_ops.BlockScaled(*state["b"])
        return fp8_ops.matmul(a, b, trans_a=case["how"] == "wgrad", trans_b=case["how"] == "forward", out_dtype=DTYPES[case["out"]])
    lists = state["lists"]
    norm = optim_ops.adamw_multi(lists["param"], lists["grad"], lists.get("master"), lists["m"], lists["v"], state["step"], lr=LR,
                                 beta1=BETA1, beta2=BETA2, eps=ADAM_EPS, weight_decay=DECAY, grad_scale=GRAD_SCALE,
                                 clip=CLIP if case["clip"] else None, m_scales=lists.get("m_scale"), v_scales=lists.get("v_scale"),
                                 seed=HASH_SEED)
    return {**{k: v for k, v in state["flat"].items() if k != "grad"}, "step": state["step"], "norm": norm}


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "norm":
        rows, width, b = case["rows"], case["width"], ITEM[case["dtype"]]
        n = rows * width
        if case["back"]:
            return {"bytes": n * b * (3 + case["residual"]) + width * (b + 4) + 4 * rows, "flops": 10 * n}
        moved = 3 * b if case["residual"] else b     # the sum is written only where there is one
        return {"bytes": n * (moved + 1) + n // BLOCK + width * b + 4 * rows, "flops": 6 * n}
    if op == "quantize":
        n = case["rows"] * case["width"]
        kinds = 2 if case["how"] == "both" else 1
        return {"bytes": n * (ITEM[case["dtype"]] + kinds) + kinds * n // BLOCK, "flops": 3 * kinds * n}
    if op == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + 2 * m * n + (m * k + n * k) // BLOCK, "flops": 2 * m * n * k}
    n = sum(_sizes(case))
    states = 16 if case["bits"] == 32 else 4
    weights = (2 + 2 + 8) if case["dtype"] != "fp32" else (4 + 8)
    return {"bytes": n * (states + weights), "flops": 20 * n}


# --------------------------------------------------------------------------- in 64 bits
def _scale64(x, block, largest):
    """2^k per block as float64, by comparison with powers of two."""
    rows, cols = x.shape
    br, bc = block
    nr, nc = -(-rows // br), -(-cols // bc)
    full = torch.nn.functional.pad(x, (0, nc * bc - cols, 0, nr * br - rows))
    amax = full.abs().reshape(nr, br, nc, bc).amax(3).amax(1)
    k = torch.ceil(torch.log2(amax / largest))
    k = torch.where(largest * torch.exp2(k - 1) >= amax, k - 1, k)
    k = torch.where(largest * torch.exp2(k) < amax, k + 1, k).clamp(-127, 127)
    k = torch.where(amax > 0, k, torch.full_like(k, -127.0))
    return torch.exp2(k).repeat_interleave(br, 0)[:rows].repeat_interleave(bc, 1)[:, :cols]


def _nearest64(x, places, least):
    """To the nearest float of ``places`` mantissa bits whose smallest normal exponent is ``least``, ties to even."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** least)))
    e = torch.where(torch.exp2(e) > x.abs().clamp(min=2.0 ** least), e - 1, e)
    e = torch.where(torch.exp2(e + 1) <= x.abs(), e + 1, e)
    step = torch.exp2(e - places)
    return torch.round(x / step) * step


def exact(case, seed):
    """Codes of the norm and of the optimizer: what they round, the value over its block's scale, because a value may lie
    next to a border.  Scales: none, they are exact or one of two neighbours."""
    state = prepare(case, seed)
    op = case["op"]
    if op == "norm" and not case["back"]:
        h = state["x"].double()
        if case["residual"]:
            h = h + state["residual"].double()
        kept = h.to(state["x"].dtype).double()     # the sum as it is kept, which the norm is taken of
        rstd = (kept.pow(2).sum(-1) / case["width"] + EPS).pow(-0.5)
        y = kept * rstd.unsqueeze(1) * state["w"].double()
        return {"codes": y / _scale64(y, (1, BLOCK), 448.0), "scales": None, "h": h, "rstd": rstd}
    if op == "norm":
        x, r, dy, w = state["x"].double(), state["rstd"].double().unsqueeze(1), state["dy"].double(), state["w"].double()
        dot = torch.einsum("rc,rc,c->r", dy, x, w).unsqueeze(1)
        dx = r * dy * w - x * r.pow(3) * dot / case["width"]
        if case["residual"]:
            dx += state["residual"].double()
        return {"dx": dx, "dw": torch.einsum("rc,rc->c", dy, x * r)}
    if op == "quantize":
        x, out = state["x"].double(), []
        largest, places, least = (448.0, 3, -6) if case["code"] == "e4m3" else (57344.0, 2, -14)
        for block in {"rows": [(1, 128)], "cols": [(128, 1)], "blocks": [(128, 128)], "both": [(1, 128), (128, 1)]}[case["how"]]:
            out += [_nearest64(x / _scale64(x, block, largest), places, least), None]
        return out
    if op == "matmul":
        how = case["how"]
        big = [q[0].double() * torch.kron(q[1].double(), torch.ones(q[2], dtype=torch.float64, device="cuda"))[:q[0].shape[0], :q[0].shape[1]]
               for q in (state["a"], state["b"])]
        return torch.matmul(big[0].mT if how == "wgrad" else big[0], big[1].mT if how == "forward" else big[1])
    flat = state["flat"]
    t = int(state["step"]) + 1
    w = flat.get("master", flat["param"]).double()
    g = flat["grad"].double() * GRAD_SCALE
    norm = g.norm()
    if case["clip"]:
        g = g * min(1.0, CLIP / (float(norm) + 1e-6))
    m, v = flat["m"].double(), flat["v"].double()
    if case["bits"] == 8:
        m = (m.view(-1, STATE_BLOCK) * flat["m_scale"].double().unsqueeze(1)).view(-1)
        v = (v.view(-1, STATE_BLOCK) * flat["v_scale"].double().unsqueeze(1)).view(-1).pow(2)
    m = m + (1 - BETA1) * (g - m)
    v = v + (1 - BETA2) * (g * g - v)
    new = w * (1 - LR * DECAY) - LR * (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + ADAM_EPS)
    out = {"param": new, "master": new if "master" in flat else None, "m": m, "v": v, "step": None, "norm": norm.view(1) if case["clip"] else None}
    if case["bits"] == 8:
        for key, value in (("m", m), ("v", v.sqrt())):
            rows = value.view(-1, STATE_BLOCK)
            out[key] = (rows / _scale64(rows, (1, STATE_BLOCK), 448.0)).view(-1)
            out[key + "_scale"] = None
    return {k: x for k, x in out.items() if k in flat or k in ("step", "norm")}
