"""The operators of a serving step at few tokens and in 8-bit floating point, as cases to measure.

Three operators:

* ``moe``: the PACKED mixture-of-experts layer for at most 32 tokens (router, experts and combine, or the
  experts alone where the caller brings the routing);
* ``quantize``: values to e4m3 with one fp32 scale per 128 of a row, or per 128 x 128 block;
* ``linear``: the product of rows with an e4m3 weight with a scale per 128 x 128 block, from rows that are
  quantized on the way (``codes`` false) or are held in e4m3 already (``codes`` true).

Where ``own`` is false, ``run`` computes them in elementary torch operations in 32 bits.
"""

from __future__ import annotations

import math

import torch

own = False

E4M3_MAX = 448.0
BLOCK = 128
#: groups whose largest magnitude lies below this are scaled as if it were this (keeps scales normal in fp32)
AMAX_FLOOR = E4M3_MAX * 2.0 ** -60
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def _moe(T, E, H, I, k, bits, group, routed=False, absent=0.0, renormalize=False, name=None):
    c = {"op": "moe", "T": T, "E": E, "H": H, "I": I, "k": k, "bits": bits, "group": group, "routed": routed,
         "absent": absent, "renormalize": renormalize}
    return {"name": name, **c} if name else c


def _quantize(M, K, rows, dtype, name=None):
    c = {"op": "quantize", "M": M, "K": K, "rows": rows, "dtype": dtype}
    return {"name": name, **c} if name else c


def _linear(M, N, K, dtype, codes=False, bias=False, name=None):
    c = {"op": "linear", "M": M, "N": N, "K": K, "dtype": dtype, "codes": codes, "bias": bias}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one new token through a layer of the 64-expert model: what a user waits for at batch one
        _moe(1, 64, 2048, 1024, 8, 4, 128, name="moe one token int4"),
        # one block of 32 masked positions, the unit of a diffusion decoding step
        _moe(32, 64, 2048, 1024, 8, 4, 128, name="moe block of 32 int4"),
        # eight sequences, one token each, on INT8 experts with the routing made elsewhere
        _moe(8, 64, 2048, 1024, 8, 8, 128, routed=True, name="moe routed 8 int8"),
        # the small test model's layer on an odd number of tokens, renormalised weights
        _moe(5, 16, 1024, 512, 2, 4, 128, renormalize=True, name="moe small 5 int4"),
        # a rank of an expert-parallel group: most choices belong to other ranks; one scale per row, odd sizes
        _moe(19, 24, 1184, 352, 4, 8, -1, routed=True, absent=0.6, name="moe rank of a group int8"),
        # the activations of one block before a dense product, and those of a long prompt
        _quantize(32, 2048, 1, "bf16", name="quantize rows 32"),
        _quantize(8192, 4096, 1, "bf16", name="quantize rows 8192"),
        # a dense weight when a model is loaded; 1000 rows end inside a block
        _quantize(1000, 2048, 128, "fp32", name="quantize weight odd"),
        # one token through a square projection
        _linear(1, 2048, 2048, "bf16", name="linear one token"),
        # a batch of blocks through the dense comparator's shape
        _linear(256, 8192, 2048, "bf16", name="linear 256 rows"),
        # an odd product: rows, columns and depth that end inside tiles and blocks, with a bias
        _linear(45, 1000, 1360, "fp16", bias=True, name="linear odd"),
        # a long prompt whose rows were quantized once for several products
        _linear(8192, 8192, 2048, "bf16", codes=True, name="linear prompt codes"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["moe", "moe", "quantize", "linear", "linear"])
    if op == "moe":
        while True:
            E, H, I = _log(rng, 4, 128), 32 * _log(rng, 8, 128), 32 * _log(rng, 4, 64)
            if E * H * I <= 64 * 2048 * 1024:
                break
        bits, routed = rng.choice([4, 8]), rng.random() < 0.4
        group = 128 if H % 128 == 0 and I % 128 == 0 and rng.random() < 0.8 else -1
        return _moe(rng.randint(1, 32), E, H, I, min(E, rng.randint(1, 8)), bits, group, routed=routed,
                    absent=rng.choice([0.0, 0.5]) if routed else 0.0, renormalize=not routed and rng.random() < 0.5)
    if op == "quantize":
        K = _log(rng, 16, 8192)
        M = _log(rng, 1, min(65536, 8192 * 4096 // K // 2))
        return _quantize(M, K, rng.choice([1, 1, 128]), rng.choice(list(DTYPES)))
    while True:
        M, N, K = _log(rng, 1, 8192), _log(rng, 16, 8192), 16 * _log(rng, 2, 256)
        if M * N * K <= 8192 * 8192 * 2048:
            break
    return _linear(M, N, K, rng.choice(["bf16", "fp16"]), codes=rng.random() < 0.4, bias=rng.random() < 0.5)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _packed(g, E, rows, K, bits, group):
    """Packed codes and fp32 scales of N(0, 0.02) weights [E, rows, K], quantized symmetrically along K."""
    G = 1 if group == -1 else K // group
    w = torch.randn(E, rows, G, K // G, generator=g, device="cuda").mul_(0.02)
    s = w.abs().amax(-1, keepdim=True) / (7.0 if bits == 4 else 127.0)
    q = torch.round_(w.div_(s)).to(torch.int8).reshape(E, rows, K)
    if bits == 4:
        q = (q[..., 0::2] & 15) | (q[..., 1::2] << 4)
    return q.contiguous(), s.reshape(E, rows, G).contiguous()


def _codes(x, rows):
    """e4m3 codes (row pitch a multiple of 16 bytes) and scales of x, from the plain form."""
    code, scale = _plain_quantize(x, rows)
    M, K = code.shape
    held = torch.zeros(M, (K + 15) // 16 * 16, dtype=torch.float8_e4m3fn, device=x.device)[:, :K]
    held.copy_(code)
    return held, scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = case
    s = {"case": c}
    if c["op"] == "moe":
        T, E, H, I, k = c["T"], c["E"], c["H"], c["I"], c["k"]
        s["qw1"], s["sw1"] = _packed(g, E, 2 * I, H, c["bits"], c["group"])
        s["qw2"], s["sw2"] = _packed(g, E, H, I, c["bits"], c["group"])
        s["x"] = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
        if c["routed"]:  # distinct experts of a token, some of them on other ranks (-1)
            order = torch.rand(T, E, generator=g, device="cuda").argsort(-1)[:, :k].to(torch.int32)
            here = torch.rand(T, k, generator=g, device="cuda") >= c["absent"]
            s["ids"] = torch.where(here, order, -1).contiguous()
            s["weights"] = torch.rand(T, k, generator=g, device="cuda") / k
        else:
            s["gate"] = (torch.randn(E, H, generator=g, device="cuda") * 0.02).to(torch.bfloat16)
        if own:
            from llada_quant_b200.few_tokens import FewTokenMoE
            from llada_quant_b200.moe import PackedExperts
            packed = PackedExperts(s["qw1"], s["sw1"], s["qw2"], s["sw2"], c["bits"], c["group"])
            s["layer"] = FewTokenMoE(packed, s.get("gate"), k, renormalize=c["renormalize"])
        return s
    dtype = DTYPES[c["dtype"]]
    # activations have a few channels much larger than the rest
    x = torch.randn(c["M"], c["K"], generator=g, device="cuda")
    x = (x * torch.exp(0.7 * torch.randn(c["K"], generator=g, device="cuda"))).to(dtype)
    if c["op"] == "quantize":
        s["x"] = x
        if own:
            from llada_quant_b200.fp8 import quantize_fp8
            s["quantize"] = quantize_fp8
        return s
    w = torch.randn(c["N"], c["K"], generator=g, device="cuda") * 0.02
    s["w_codes"], s["w_scale"] = _codes(w, BLOCK)
    s["bias"] = (torch.randn(c["N"], generator=g, device="cuda") * 0.1).to(dtype) if c["bias"] else None
    s["out"] = dtype
    if c["codes"]:
        s["x_codes"], s["x_scale"] = _codes(x, 1)
    else:
        s["x"] = x
    if own:
        from llada_quant_b200.fp8 import Fp8Linear, Fp8Tensor
        s["linear"] = Fp8Linear.from_codes(Fp8Tensor(s["w_codes"], s["w_scale"], BLOCK), bias=s["bias"],
                                           compute_dtype=dtype)
        s["rows"] = Fp8Tensor(s["x_codes"], s["x_scale"], 1) if c["codes"] else s["x"]
    return s


# ---------------------------------------------------------------------------
# plain forms, 32 bits
# ---------------------------------------------------------------------------

def _weights(q, scale, bits):
    """Packed codes and scales as fp32 weights q * s."""
    if bits == 4:
        q = torch.stack([(q << 4) >> 4, q >> 4], dim=-1).flatten(-2)
    E, rows, K = q.shape
    G = scale.shape[-1]
    return (q.to(torch.float32).view(E, rows, G, K // G) * scale.unsqueeze(-1)).view(E, rows, K)


def _plain_moe(s):
    c = s["case"]
    E, I, k = c["E"], c["I"], c["k"]
    x = s["x"].float()
    if c["routed"]:
        ids, weights = s["ids"], s["weights"]
    else:
        # whole numbers hang on which logit is larger: 64 bits
        logits = s["x"].double() @ s["gate"].double().t()
        z = torch.exp(logits - logits.amax(-1, keepdim=True))
        order = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :k]
        p = (z / z.sum(-1, keepdim=True)).gather(1, order)
        weights = (p / p.sum(-1, keepdim=True) if c["renormalize"] else p).float()
        ids = order.to(torch.int32)
    here = (ids >= 0) & (ids < E)
    share = torch.zeros(x.shape[0], E, device=x.device)
    share.scatter_add_(1, torch.where(here, ids, 0).long(), torch.where(here, weights, 0.0))
    gu = torch.matmul(x.unsqueeze(0), _weights(s["qw1"], s["sw1"], c["bits"]).transpose(1, 2))
    gate, up = gu[..., :I], gu[..., I:]
    h = gate / (1 + torch.exp(-gate)) * up
    y = torch.matmul(h, _weights(s["qw2"], s["sw2"], c["bits"]).transpose(1, 2))
    out = (y * share.t().unsqueeze(-1)).sum(0).to(torch.bfloat16)
    return {"out": out} if c["routed"] else {"out": out, "weights": weights, "ids": ids}


def _plain_quantize(x, rows):
    M, K = x.shape
    R, G = -(-M // rows), -(-K // BLOCK)
    v = torch.zeros(R * rows, G * BLOCK, device=x.device)
    v[:M, :K] = x
    v = v.view(R, rows, G, BLOCK)
    amax = v.abs().amax((1, 3), keepdim=True).clamp(min=AMAX_FLOOR)
    # x * 448 / amax, with 448 = 0.4375 * 2^10 so that no product leaves fp32's range
    code = ((v * 0.4375) / (amax * 2.0 ** -10)).view(R * rows, G * BLOCK)[:M, :K].to(torch.float8_e4m3fn)
    return code, (amax / torch.full_like(amax, E4M3_MAX)).view(R, G)


def _spread(codes, scale, rows):
    """e4m3 codes times their scales, fp32."""
    M, K = codes.shape
    wide = scale.repeat_interleave(rows, 0)[:M].repeat_interleave(BLOCK, 1)[:, :K]
    return codes.float() * wide


def _plain_linear(s):
    codes, scale = (s["x_codes"], s["x_scale"]) if s["case"]["codes"] else _plain_quantize(s["x"], 1)
    y = _spread(codes, scale, 1) @ _spread(s["w_codes"], s["w_scale"], BLOCK).t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["out"])


def run(state):
    s, op = state, state["case"]["op"]
    if op == "moe":
        if not own:
            return _plain_moe(s)
        if s["case"]["routed"]:
            return {"out": s["layer"].routed(s["x"], s["weights"], s["ids"])}
        out, weights, ids = s["layer"](s["x"])
        return {"out": out, "weights": weights, "ids": ids}
    if op == "quantize":
        if own:
            q = s["quantize"](s["x"], s["case"]["rows"])
            return {"values": q.codes, "scale": q.scale}
        code, scale = _plain_quantize(s["x"], s["case"]["rows"])
        return {"values": code, "scale": scale}
    return {"out": s["linear"](s["rows"]) if own else _plain_linear(s)}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    c = case
    if c["op"] == "moe":
        T, E, H, I, k = c["T"], c["E"], c["H"], c["I"], c["k"]
        chosen = k * (1.0 - c["absent"])
        hit = E * (1.0 - (1.0 - chosen / E) ** T)  # experts that some token chose
        G1, G2 = (1, 1) if c["group"] == -1 else (H // c["group"], I // c["group"])
        bytes_ = hit * (3 * I * H * c["bits"] / 8 + 4 * (2 * I * G1 + H * G2)) + 4 * T * H
        bytes_ += 8 * T * k + (0 if c["routed"] else 2 * E * H)
        return {"bytes": bytes_, "flops": 6.0 * T * chosen * H * I + (0 if c["routed"] else 2.0 * T * E * H)}
    M, K = c["M"], c["K"]
    G = -(-K // BLOCK)
    size = 4 if c["dtype"] == "fp32" else 2
    if c["op"] == "quantize":
        return {"bytes": M * K * (size + 1) + 4 * -(-M // c["rows"]) * G, "flops": 4.0 * M * K}
    N = c["N"]
    rows = M * K + 4 * M * G if c["codes"] else M * K * size
    return {"bytes": rows + N * K + 4 * -(-N // BLOCK) * G + 2 * M * N + (2 * N if c["bias"] else 0),
            "flops": 2.0 * M * N * K}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _wide(q, scale, bits):
    """One expert's weights in fp64 from its bytes."""
    if bits == 4:
        byte = q.to(torch.int32) & 255
        w = torch.empty(q.shape[0], 2 * q.shape[1], dtype=torch.float64, device=q.device)
        for half in (0, 1):
            n = (byte // 16 ** half) % 16
            w[:, half::2] = (n - 16 * (n >= 8)).double()
    else:
        w = q.double()
    return w * torch.kron(scale.double(), torch.ones(1, w.shape[1] // scale.shape[1], dtype=torch.float64,
                                                     device=q.device))


def _exact_moe(s):
    c = s["case"]
    x = s["x"].double()
    found = {}
    if c["routed"]:
        ids, weights = s["ids"].long(), s["weights"].double()
    else:
        p = torch.softmax(torch.einsum("th,eh->te", x, s["gate"].double()), -1)
        weights, ids = torch.topk(p, c["k"], dim=-1)
        if c["renormalize"]:
            weights = weights / weights.sum(-1, keepdim=True)
        found = {"weights": weights, "ids": ids.to(torch.int32)}
    out = torch.zeros_like(x)
    for e in range(c["E"]):
        w1 = _wide(s["qw1"][e], s["sw1"][e], c["bits"])
        w2 = _wide(s["qw2"][e], s["sw2"][e], c["bits"])
        a, b = (x @ w1.t()).chunk(2, dim=1)
        part = (a * torch.sigmoid(a) * b) @ w2.t()
        out += part * (weights * (ids == e)).sum(1, keepdim=True)
    return {"out": out, **found}


def _exact_quantize(x, rows):
    """Nearest e4m3 to x * 448 / amax of the block, and amax / 448, in fp64; the last step to the 3-bit
    significand is done on the value itself: spacing 2^(e - 3), at least 2^-9."""
    M, K = x.shape
    x = x.double()
    amax = torch.nn.functional.max_pool2d(
        torch.nn.functional.pad(x.abs(), (0, -K % BLOCK, 0, -M % rows))[None], (rows, BLOCK))[0].clamp(min=AMAX_FLOOR)
    v = x * 448.0 / torch.kron(amax, torch.ones(rows, BLOCK, dtype=torch.float64, device=x.device))[:M, :K]
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step, amax / 448.0


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "moe":
        return _exact_moe(s)
    if case["op"] == "quantize":
        values, scale = _exact_quantize(s["x"], case["rows"])
        return {"values": values, "scale": scale}
    v, a = (s["x_codes"].double(), s["x_scale"].double()) if case["codes"] else _exact_quantize(s["x"], 1)
    w, b = s["w_codes"].double(), s["w_scale"].double()
    y = torch.zeros(case["M"], case["N"], dtype=torch.float64, device=v.device)
    for g in range(a.shape[1]):  # block of 128 after block of 128 along the depth
        at = slice(BLOCK * g, min(BLOCK * (g + 1), case["K"]))
        y += (v[:, at] @ w[:, at].t()) * a[:, g:g + 1] * b[:, g].repeat_interleave(BLOCK)[:case["N"]]
    return {"out": y if s["bias"] is None else y + s["bias"].double()}
