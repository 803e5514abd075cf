"""The PACKED layer for at most 32 tokens against its definition in 64 bits, and its refusals.

Error bound of an output, element by element, from the arithmetic (u = 2^-23 covers a rounded or a truncated
fp32 step).  A sum of products runs through at most D fp32 steps: 16 inside an MMA, one per MMA of a 128-group
(8, or 16 where h comes in two parts), two per group (scale, sum), one per partial that meets it.  With
A = sum |W| |x| (and B for the up rows):

    da <= D1 u A,   D1 = 32 + 2 G1
    dh <= w (1.1 |b| da + |silu(a)| db) + 2^-16 |h| + 16 u |h|     (|silu'| <= 1.1; h = hi + lo, each half a
                                                                   bf16 step of 2^-8; exp, quotient, products)
    dv <= sum |W2| dh + D2 u sum |W2| |h|,   D2 = 64 + 2 G2 (experts of the token)
    |out - v| <= dv + 2^-8 (|v| + dv)                              (one rounding to bf16)
"""

from __future__ import annotations

import pytest
import torch

from llada_quant_b200 import _lib

U = 2.0 ** -23


# ---------------------------------------------------------------------------
# 64-bit definition
# ---------------------------------------------------------------------------

def dense64(q, s, bits):
    """One expert's weights q * s in fp64 from its packed rows."""
    q = q.to(torch.int64)
    if bits == 4:
        lo, hi = ((q & 15) ^ 8) - 8, q >> 4
        q = torch.stack([lo, hi], -1).reshape(q.shape[0], -1)
    return q.double() * s.double().repeat_interleave(q.shape[1] // s.shape[1], 1)


def experts64(x, packed, weights, ids):
    """(v, bound): the layer's value and the bound on the kernel's distance from it, both [T, H] fp64."""
    x, weights, ids = x.double(), weights.double(), ids.long()
    qw1, sw1, qw2, sw2, bits = packed
    E, inter = qw1.shape[0], qw1.shape[1] // 2
    v, dv = torch.zeros_like(x), torch.zeros_like(x)
    used = ((ids >= 0) & (ids < E)).sum(1, keepdim=True).clamp(min=1)
    D1, D2 = 32 + 2 * -(-x.shape[1] // 128), 64 + 2 * -(-inter // 128) * used
    for e in range(E):
        w = (weights * (ids == e)).sum(1, keepdim=True)
        toks = (ids == e).any(1)
        if not toks.any():
            continue
        w, xe = w[toks], x[toks]
        W1, W2 = dense64(qw1[e], sw1[e], bits), dense64(qw2[e], sw2[e], bits)
        a, b = xe @ W1[:inter].t(), xe @ W1[inter:].t()
        A, B = xe.abs() @ W1[:inter].abs().t(), xe.abs() @ W1[inter:].abs().t()
        silu = a * torch.sigmoid(a)
        h = silu * b * w
        dh = w.abs() * (1.1 * b.abs() * D1 * U * A + silu.abs() * D1 * U * B) + (2.0 ** -16 + 16 * U) * h.abs()
        v[toks] += h @ W2.t()
        dv[toks] += dh @ W2.abs().t() + D2[toks] * U * (h.abs() @ W2.abs().t())
    return v, dv + 2.0 ** -8 * (v.abs() + dv)


def logits64(x, gate, bias):
    z = x.double() @ gate.double().t()
    # 16 inside an MMA, two MMAs per 32 of a warp's eighth of H, 8 partials, the bias
    dz = (25 + 2 * -(-x.shape[1] // 256)) * U * (x.double().abs() @ gate.double().abs().t())
    if bias is not None:
        z, dz = z + bias.double(), dz + U * bias.double().abs().nan_to_num(0.0, 0.0, 0.0)
    return z, dz


def make_layer(T, E, H, I, k, bits, group, seed=0, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    out = []
    for rows, K in ((2 * I, H), (H, I)):
        G = K // group if group > 0 and K % group == 0 else 1
        w = torch.randn(E, rows, G, K // G, generator=g, device=device) * 0.02
        s = w.abs().amax(-1, keepdim=True) / (7.0 if bits == 4 else 127.0)
        q = torch.round(w / s).to(torch.int8).reshape(E, rows, K)
        if bits == 4:
            q = (q[..., 0::2] & 15) | (q[..., 1::2] << 4)
        out += [q.contiguous(), s.reshape(E, rows, G).contiguous()]
    x = torch.randn(T, H, generator=g, device=device).to(torch.bfloat16)
    gate = (torch.randn(E, H, generator=g, device=device) * 0.02).to(torch.bfloat16)
    ids = torch.rand(T, E, generator=g, device=device).argsort(-1)[:, :k].to(torch.int32).contiguous()
    weights = torch.rand(T, k, generator=g, device=device) / k
    return (*out, bits), x, gate, weights, ids


def packed_of(layer, group):
    from llada_quant_b200.moe import PackedExperts
    return PackedExperts(*layer[:4], layer[4], group)


def check(out, x, layer, weights, ids):
    v, bound = experts64(x, layer, weights, ids)
    assert out.shape == x.shape and out.dtype == torch.bfloat16
    off = (out.double() - v).abs()
    assert bool((off <= bound).all()), (off - bound).max().item()


def check_routing(x, gate, bias, k, renormalize, logits, weights, ids):
    """The k largest z in order, up to the logits' own error; the weights of that choice."""
    z, dz = logits64(x, gate, bias)
    both_inf = torch.isinf(z) & (logits.double() == z)
    assert bool((((logits.double() - z).abs() <= dz) | both_inf).all())
    zc, dzc = z.gather(1, ids.long()), dz.gather(1, ids.long())
    assert all(len(set(r)) == k for r in ids.tolist())
    if k > 1:
        assert bool((zc[:, 1:] <= zc[:, :-1] + dzc[:, 1:] + dzc[:, :-1]).all())
    rest = z.scatter(1, ids.long(), -torch.inf)
    assert bool((rest <= (zc[:, -1:] + dzc[:, -1:] + dz)).all())
    p = torch.softmax(z, -1).gather(1, ids.long())
    p = p / p.sum(-1, keepdim=True) if renormalize else p
    # exp of z - max: both ends' errors and the subtraction; exp, the sum over up to 256 and the quotients: 64 steps
    rel = torch.expm1(2 * (dz.amax(1, keepdim=True) + dzc) + U * (z.amax(1, keepdim=True) - zc).nan_to_num(posinf=0)) + 64 * U
    assert bool(((weights.double() - p).abs() <= (2 if renormalize else 1) * rel * p).all())


SHAPES = [
    # T, E, H, I, k, bits, group
    (1, 64, 2048, 1024, 8, 4, 128),
    (32, 64, 2048, 1024, 8, 4, 128),
    (7, 16, 1024, 512, 2, 8, 128),
    (9, 4, 256, 256, 4, 4, 128),       # every expert holds every token: two column tiles
    (32, 3, 384, 128, 2, 8, 128),
    (32, 1, 128, 128, 1, 4, 128),      # one expert, 32 tokens
    (1, 1, 32, 32, 1, 8, -1),          # the smallest layer
    (5, 5, 32, 32, 3, 4, -1),
    (19, 24, 1184, 352, 4, 8, -1),     # nothing a multiple of 128
    (13, 40, 1056, 224, 3, 4, -1),
    (3, 256, 128, 128, 32, 4, 128),    # the most experts and choices
    (17, 65, 160, 96, 9, 8, -1),
    (4, 8, 512, 1024, 2, 4, 256),      # scales wider than a step
    (6, 8, 1024, 160, 2, 8, 128),      # w1 in groups, w2 with one scale per row
    (2, 6, 4224, 2080, 2, 4, -1),      # long rows
]


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,H,I,k,bits,group", SHAPES)
def test_layer_with_its_router(T, E, H, I, k, bits, group):
    from llada_quant_b200.few_tokens import FewTokenMoE
    layer, x, gate, _, _ = make_layer(T, E, H, I, k, bits, group, seed=T + E)
    renorm = T % 2 == 0
    out, weights, ids, logits = FewTokenMoE(packed_of(layer, group), gate, k, renormalize=renorm).with_logits(x)
    torch.cuda.synchronize()
    check_routing(x, gate, None, k, renorm, logits, weights, ids)
    check(out, x, layer, weights, ids)


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,H,I,k,bits,group", SHAPES)
def test_experts_with_given_routing(T, E, H, I, k, bits, group):
    """Some choices lie on other ranks; one token has none left."""
    from llada_quant_b200.few_tokens import FewTokenMoE
    layer, x, _, weights, ids = make_layer(T, E, H, I, k, bits, group, seed=7 * T + E)
    ids[torch.rand(T, k, device="cuda", generator=torch.Generator("cuda").manual_seed(1)) < 0.3] = -1
    ids[T // 2] = E
    out = FewTokenMoE(packed_of(layer, group), None, k).routed(x, weights, ids)
    torch.cuda.synchronize()
    check(out, x, layer, weights, ids)
    assert bool((out[T // 2] == 0).all())


@pytest.mark.gpu
def test_nothing_chosen_anywhere_gives_zeros():
    from llada_quant_b200.few_tokens import FewTokenMoE
    layer, x, _, weights, ids = make_layer(4, 8, 256, 128, 2, 4, 128)
    out = FewTokenMoE(packed_of(layer, 128), None, 2).routed(x, weights, torch.full_like(ids, -5))
    assert bool((out == 0).all())


@pytest.mark.gpu
def test_same_expert_twice_counts_both_weights():
    from llada_quant_b200.few_tokens import FewTokenMoE
    layer, x, _, weights, ids = make_layer(11, 8, 256, 256, 3, 4, 128)
    ids[:, 2] = ids[:, 0]
    out = FewTokenMoE(packed_of(layer, 128), None, 3).routed(x, weights, ids)
    check(out, x, layer, weights, ids)
    wide = torch.tensor([[2 ** 32 + 1, -2 ** 40, 2]] * 11, device="cuda")  # int64 ids are not wrapped into range
    out = FewTokenMoE(packed_of(layer, 128), None, 3).routed(x, weights, wide)
    check(out, x, layer, weights, wide)


@pytest.mark.gpu
def test_equal_logits_go_to_the_lower_expert_and_bias_bars_experts():
    from llada_quant_b200.few_tokens import FewTokenMoE
    layer, x, gate, _, _ = make_layer(6, 16, 256, 128, 4, 8, 128)
    gate[:] = gate[0]
    _, weights, ids = FewTokenMoE(packed_of(layer, 128), gate, 4)(x)
    assert ids.tolist() == [[0, 1, 2, 3]] * 6 and bool(((weights - 1 / 16).abs() <= 8 * U).all())
    bias = torch.zeros(16, device="cuda")
    bias[[0, 2, 3]] = -torch.inf
    _, weights, ids = FewTokenMoE(packed_of(layer, 128), gate, 4, bias=bias)(x)
    assert ids.tolist() == [[1, 4, 5, 6]] * 6 and bool(((weights - 1 / 13).abs() <= 8 * U).all())
    bias[4:] = -torch.inf  # one expert is left: the barred ones follow with weight 0
    out, weights, ids = FewTokenMoE(packed_of(layer, 128), gate, 4, bias=bias)(x)
    assert ids.tolist() == [[1, 0, 2, 3]] * 6 and weights.tolist() == [[1.0, 0.0, 0.0, 0.0]] * 6
    check(out, x, layer, weights, ids)
    bias[:] = -torch.inf  # none is left: NaN, as softmax
    out, weights, ids = FewTokenMoE(packed_of(layer, 128), gate, 4, bias=bias)(x)
    assert bool(weights.isnan().all()) and bool(out.isnan().all()) and ids.tolist() == [[0, 1, 2, 3]] * 6


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_bad_token_spoils_its_own_row_alone(bad):
    from llada_quant_b200.few_tokens import FewTokenMoE
    layer, x, gate, _, _ = make_layer(10, 8, 256, 256, 3, 4, 128)
    moe = FewTokenMoE(packed_of(layer, 128), gate, 3)
    _, cw, ci = moe(x)
    x[4, 17] = bad
    out, w, ids = moe(x)
    rest = [t for t in range(10) if t != 4]
    assert torch.equal(w[rest], cw[rest]) and torch.equal(ids[rest], ci[rest])
    check(out[rest], x[rest], layer, w[rest], ids[rest])
    assert bool(out[4].isnan().any()) and bool(((ids >= 0) & (ids < 8)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 7])  # h's two parts in one plane, or in two
@pytest.mark.parametrize("bits", [4, 8])
def test_an_infinite_h_stays_infinite(T, bits):
    """h beyond fp32: with positive weights its sum is infinite, not a NaN."""
    from llada_quant_b200.few_tokens import FewTokenMoE
    q1 = torch.full((2, 64, 32 if bits == 8 else 16), 1 if bits == 8 else 0x11, dtype=torch.int8, device="cuda")
    q2 = torch.full((2, 32, 32 if bits == 8 else 16), 1 if bits == 8 else 0x11, dtype=torch.int8, device="cuda")
    layer = (q1, torch.ones(2, 64, 1, device="cuda"), q2, torch.ones(2, 32, 1, device="cuda"), bits)
    moe = FewTokenMoE(packed_of(layer, -1), torch.zeros(2, 32, dtype=torch.bfloat16, device="cuda"), 1)
    x = torch.full((T, 32), 1.0, dtype=torch.bfloat16, device="cuda")
    x[1] = 1e30
    ids = torch.zeros(T, 1, dtype=torch.int32, device="cuda")
    out = moe.routed(x, torch.ones(T, 1, device="cuda"), ids)
    assert bool((out[1] == float("inf")).all()) and bool((out[0] == out[2]).all()) and bool(out[0].isfinite().all())


@pytest.mark.gpu
def test_every_code_of_both_formats():
    """One-hot rows read single weights: every byte value through w1's up rows with a constant gate."""
    from llada_quant_b200.few_tokens import FewTokenMoE
    for bits in (4, 8):
        layer, x, _, weights, ids = make_layer(32, 2, 256, 128, 1, bits, 128)
        g = torch.Generator("cuda").manual_seed(5)
        for i in (0, 2):
            layer[i].copy_(torch.randint(-128, 128, layer[i].shape, generator=g, device="cuda", dtype=torch.int8))
        out = FewTokenMoE(packed_of(layer, 128), None, 1).routed(x, weights, ids)
        check(out, x, layer, weights, ids)


@pytest.mark.gpu
def test_moe_layer_and_fused_moe_reach_it():
    from llada_quant_b200 import ops
    from llada_quant_b200.few_tokens import FewTokenMoE
    from llada_quant_b200.fused_moe import fused_moe, moe_layer
    from llada_quant_b200.router_capture import RouterCapture
    from llada_quant_b200.routing_stats import RoutingRecorder
    layer, x, gate, _, _ = make_layer(12, 16, 1024, 512, 2, 4, 128)
    packed = packed_of(layer, 128)
    want, w, ids = FewTokenMoE(packed, gate, 2)(x)
    rec, cap = RoutingRecorder(16, "cuda"), RouterCapture()
    got = moe_layer(x, gate, packed, 2, impl="few", recorder=rec, capture=cap, name="l0")
    assert torch.equal(got, want)
    assert torch.equal(cap.topk_ids["l0"], ids.cpu().long()) and cap.gates["l0"].shape == (12, 16)
    assert rec.stats().counts == torch.bincount(ids.reshape(-1).long(), minlength=16).tolist()
    assert torch.equal(fused_moe(x.view(3, 4, 1024), packed, None, None, ids, topk_weights=w, impl="few").view(12, 1024), want)
    # the layer for many tokens, on the same routing: W and h rounded to bf16 there (rel-L2 bar of its own tests)
    many = ops.fused_moe_packed(x, packed.qw1, packed.sw1, packed.qw2, packed.sw2, w, ids, 4, _lib.LLQ_GEMM_AUTO)
    assert ((many.double() - want.double()).norm() / want.double().norm()).item() <= 1e-2


@pytest.mark.gpu
@pytest.mark.parametrize("T,bits,E", [(1, 8, 40), (32, 8, 40), (32, 4, 3)])
def test_the_longest_rows_and_offsets_beyond_32_bits(T, bits, E):
    """H = I = 8192; with 40 INT8 experts w1 has 5.4 GB, and the tokens choose the last experts."""
    from llada_quant_b200.few_tokens import FewTokenMoE
    H = I = 8192
    per = 2 if bits == 4 else 1
    g = torch.Generator("cuda").manual_seed(T + bits)
    q1 = torch.randint(-128, 128, (E, 2 * I, H // per), generator=g, device="cuda", dtype=torch.int8)
    q2 = torch.randint(-128, 128, (E, H, I // per), generator=g, device="cuda", dtype=torch.int8)
    s1 = torch.rand(E, 2 * I, H // 128, generator=g, device="cuda") * 1e-4
    s2 = torch.rand(E, H, I // 128, generator=g, device="cuda") * 1e-4
    layer = (q1, s1, q2, s2, bits)
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    ids = (E - 1 - torch.arange(2, device="cuda", dtype=torch.int32)).repeat(T, 1)
    ids[T // 2:, 1] = E
    weights = torch.rand(T, 2, generator=g, device="cuda")
    gate = (torch.randn(E, H, generator=g, device="cuda") * 0.02).to(torch.bfloat16)
    bias = torch.full((E,), -torch.inf, device="cuda")
    bias[E - 2:] = 0
    moe = FewTokenMoE(packed_of(layer, 128), gate, 2, bias)
    check(moe.routed(x, weights, ids), x, layer, weights, ids)
    out, w, ids = moe(x)
    assert bool((ids >= E - 2).all())
    check(out, x, layer, w, ids)


@pytest.mark.gpu
def test_copied_router_operands_live_until_the_call():
    """gate_w and bias that have to be copied: the copies' memory is not given to the call's own tensors."""
    from llada_quant_b200.fused_moe import moe_layer
    layer, x, gate, _, _ = make_layer(9, 16, 512, 256, 4, 4, 128)
    p = packed_of(layer, 128)
    bias = (torch.arange(16, device="cuda") / 8).to(torch.bfloat16)  # exact in bf16
    wide = torch.zeros(16, 1031, dtype=torch.bfloat16, device="cuda")
    wide[:, 3:515] = gate
    flat = torch.zeros(16 * 512 + 3, dtype=torch.bfloat16, device="cuda")
    flat[3:] = gate.reshape(-1)
    want = moe_layer(x, gate, p, 4, bias.float(), impl="few")
    torch.cuda.synchronize()
    for g in (gate, gate.t().contiguous().t(), wide[:, 3:515], flat[3:].view(16, 512)):
        for _ in range(3):
            assert torch.equal(moe_layer(x, g, p, 4, bias, impl="few"), want)
    with pytest.raises(RuntimeError, match="no backward pass"):
        moe_layer(x, gate.clone().requires_grad_(), p, 4, impl="few")


@pytest.mark.gpu
def test_captured_replayed_and_on_two_streams_at_once():
    from llada_quant_b200.few_tokens import FewTokenMoE
    layer, x, gate, _, _ = make_layer(9, 16, 512, 256, 4, 4, 128)
    moe = FewTokenMoE(packed_of(layer, 128), gate, 4)
    xs = [x, x.flip(0).contiguous(), (x * 0.5).contiguous(), x.roll(1, 1).contiguous()]
    want = [moe(v) for v in xs]
    torch.cuda.synchronize()
    graphs, outs, ins = [], [], [torch.empty_like(x) for _ in range(2)]
    for v in ins:  # two graphs alive together
        v.copy_(x)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(moe(v))
        graphs.append(g)
    for a, b in ((0, 1), (2, 3), (3, 0)):
        ins[0].copy_(xs[a])
        ins[1].copy_(xs[b])
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        eager = moe(xs[a])  # and a call beside them
        torch.cuda.synchronize()
        for got, i in ((outs[0], a), (outs[1], b), (eager, a)):
            assert all(torch.equal(p, q) for p, q in zip(got, want[i]))


@pytest.mark.gpu
def test_slices_strides_no_tokens_and_repeatability():
    from llada_quant_b200.few_tokens import FewTokenMoE
    layer, x, gate, _, _ = make_layer(8, 16, 512, 256, 4, 8, 128)
    moe = FewTokenMoE(packed_of(layer, 128), gate, 4)
    want = moe(x)
    wide = torch.zeros(8, 1024, dtype=torch.bfloat16, device="cuda")
    wide[:, 3:515] = x
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(moe(wide[:, 3:515]), want))
    off = torch.zeros(8 * 512 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(8, 512)
    off.copy_(x)
    assert torch.equal(moe(off)[0], want[0])
    out, w, ids = moe(x[:0])
    assert out.shape == (0, 512) and w.shape == (0, 4) and ids.shape == (0, 4)
    # a token's row does not depend on the others
    for t in (0, 5):
        one = moe(x[t:t + 1])
        assert torch.equal(one[2][0], want[2][t])


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------

def _c_layer(**kw):
    f = dict(gate_w=None, bias=None, qw1=16, sw1=16, qw2=16, sw2=16, E=8, H=256, I=128, k=2, bits=4, group_size=128,
             renormalize=0)
    f.update(kw)
    return _lib.FewLayer(*(f[n] for n, _ in _lib.FewLayer._fields_))


@pytest.mark.parametrize("kw,T,code,text", [
    (dict(k=9), 4, _lib.LLQ_EINVAL, b"bad shape"),
    (dict(k=0), 4, _lib.LLQ_EINVAL, b"bad shape"),
    (dict(), -1, _lib.LLQ_EINVAL, b"bad shape"),
    (dict(bits=3), 4, _lib.LLQ_EUNSUPPORTED, b"bits"),
    (dict(), 33, _lib.LLQ_EUNSUPPORTED, b"at most 32 tokens"),
    (dict(E=257), 4, _lib.LLQ_EUNSUPPORTED, b"E <= 256"),
    (dict(E=64, k=33), 4, _lib.LLQ_EUNSUPPORTED, b"k <= 32"),
    (dict(H=264), 4, _lib.LLQ_EUNSUPPORTED, b"multiples of 32"),
    (dict(I=120), 4, _lib.LLQ_EUNSUPPORTED, b"multiples of 32"),
    (dict(H=65536), 4, _lib.LLQ_EUNSUPPORTED, b"8192"),
    (dict(group_size=64), 4, _lib.LLQ_EUNSUPPORTED, b"multiples of 128"),
    (dict(qw1=None), 4, _lib.LLQ_EINVAL, b"null"),
    (dict(qw2=24), 4, _lib.LLQ_EINVAL, b"16-byte"),
    (dict(), 4, _lib.LLQ_ENOSPACE, b"workspace"),
])
def test_c_refusals_need_no_gpu(kw, T, code, text):
    import ctypes
    lib = _lib.load()
    rc = lib.llq_moe_few(ctypes.byref(_c_layer(**kw)), 16, T, None, 16, 16, 16, 256, 1, None)
    assert rc == code and text in lib.llq_last_error(), lib.llq_last_error()


def test_c_edges_need_no_gpu():
    import ctypes
    lib = _lib.load()
    assert lib.llq_moe_few(None, 16, 1, None, 16, 16, 16, 16, 1, None) == _lib.LLQ_EINVAL
    assert lib.llq_moe_few(ctypes.byref(_c_layer()), None, 0, None, None, None, None, None, 0, None) == _lib.LLQ_OK
    assert lib.llq_moe_few_workspace_size(0, 8, 64, 2048, 1024) == 0
    assert lib.llq_moe_few_workspace_size(32, 8, 64, 2048, 1024) >= 32 * 8 * 1024 * 4


def test_python_refusals_need_no_gpu(monkeypatch):
    from llada_quant_b200 import ops
    from llada_quant_b200.few_tokens import FewTokenMoE
    layer, x, gate, weights, ids = make_layer(4, 8, 256, 128, 2, 4, 128, device="cpu")
    with pytest.raises(RuntimeError, match="CUDA"):
        FewTokenMoE(packed_of(layer, 128), gate, 2)
    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: None)
    packed = packed_of(layer, 128)
    moe = FewTokenMoE(packed, gate, 2)
    for bad in (x[0], x[:, :128], x.float()):
        with pytest.raises(ValueError, match="x must be"):
            moe(bad)
    with pytest.raises(RuntimeError, match="no backward"):
        moe(x.clone().requires_grad_())
    with pytest.raises(ValueError, match="routing must be"):
        moe.routed(x, weights[:, :1], ids)
    with pytest.raises(ValueError, match="int32 or int64"):
        moe.routed(x, weights, ids.to(torch.int16))
    with pytest.raises(RuntimeError, match="no backward"):
        moe.routed(x, weights.clone().requires_grad_(), ids)
    with pytest.raises(ValueError, match="without gate_w"):
        FewTokenMoE(packed, None, 2)(x)
    with pytest.raises(ValueError, match="gate_w must be"):
        FewTokenMoE(packed, gate[:, :128], 2)
    with pytest.raises(ValueError, match="bias must be"):
        FewTokenMoE(packed, gate, 2, bias=torch.zeros(7))
    for k in (0, 9):
        with pytest.raises(ValueError, match="top_k"):
            FewTokenMoE(packed, gate, k)
    q1, s1, q2, s2, _ = layer
    for args, text in (((q1, s1, q2[:, :, :32], s2), "not one layer"), ((q1, s1, q2, s2.half()), "float32 scales"),
                       ((q1, s1[:, :, :1].contiguous(), q2, s2.expand(8, 256, 3).contiguous()), "scales for rows"),
                       ((q1.to(torch.int16), s1, q2, s2), "int8")):
        with pytest.raises(ValueError, match=text):
            ops.few_layer(*args, 2, 4)
