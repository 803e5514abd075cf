"""The decoding step's operators where a value is held between kernels or between calls."""

from __future__ import annotations

import ctypes
import gc
import weakref

import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 8, 9, 10, 12, 32])  # segments of 1 to 8 tokens, alone and behind full ones
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("inter", [32, 160, 384])
def test_h_keeps_the_bits_of_fp32(T, bits, inter):
    """out = h0 - h1 for two fp32 numbers that agree in their upper 16 bits: the lower 8, exactly.

    Every feature has a = 32 and b = 2^-5, so h = silu(a) b w = w in fp32 (exp(-32) < 2^-24).  Expert 0 adds the h of one
    feature to each output and expert 1 takes it away.  w0 has 24 bits in [1, 1.5) and w1 is w0 without its lower 8, so
    that parts of either, and any sum of them, are multiples of 2^-23 below 2: fp32 sums in any order are exact, and the
    8 bits that are left are a bf16 number.
    """
    from llada_quant_b200.few_tokens import FewTokenMoE
    from llada_quant_b200.moe import PackedExperts
    H, one = 64, 1 if bits == 8 else 0x01
    w1 = torch.zeros(2, 2 * inter, H * bits // 8, dtype=torch.int8)
    w1[:, :, 0] = one
    s1 = torch.cat([torch.full((2, inter, 1), 32.0), torch.full((2, inter, 1), 2.0 ** -5)], 1)
    w2 = torch.zeros(2, H, inter, dtype=torch.int8)
    for r in range(H):
        w2[0, r, r * 37 % inter], w2[1, r, r * 37 % inter] = 1, -1
    if bits == 4:
        w2 = (w2[..., 0::2] & 15) | (w2[..., 1::2] << 4)
    packed = PackedExperts(w1.cuda(), s1.cuda(), w2.contiguous().cuda(), torch.ones(2, H, 1, device="cuda"), bits, -1)
    x = torch.zeros(T, H, dtype=torch.bfloat16, device="cuda")
    x[:, 0] = 1
    low = torch.randint(1, 256, (T,), generator=torch.Generator().manual_seed(T))
    high = torch.randint(2 ** 15, 3 * 2 ** 14, (T,), generator=torch.Generator().manual_seed(T + 1)) * 256
    weights = (torch.stack([high + low, high], 1).double() * 2.0 ** -23).float().cuda()
    ids = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda").repeat(T, 1)
    out = FewTokenMoE(packed, None, 2).routed(x, weights, ids)
    want = (low.double() * 2.0 ** -23).cuda()[:, None].expand(T, H)
    assert torch.equal(out.double(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("T", [1, 2])
def test_an_infinite_h_of_one_or_two_tokens_stays_infinite(T, bits):
    """The parts of h side by side in one plane: infinity and zeros, no NaN."""
    from llada_quant_b200.few_tokens import FewTokenMoE
    from llada_quant_b200.moe import PackedExperts
    one = torch.full((2, 64, 32 if bits == 8 else 16), 1 if bits == 8 else 0x11, dtype=torch.int8, device="cuda")
    packed = PackedExperts(one, torch.ones(2, 64, 1, device="cuda"), one[:, :32].contiguous(), torch.ones(2, 32, 1, device="cuda"),
                           bits, -1)
    x = torch.full((T, 32), 1e30, dtype=torch.bfloat16, device="cuda")
    out = FewTokenMoE(packed, None, 1).routed(x, torch.ones(T, 1, device="cuda"), torch.ones(T, 1, dtype=torch.int32, device="cuda"))
    assert bool((out == float("inf")).all())


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 12, 32])
@pytest.mark.parametrize("bits", [4, 8])
def test_what_the_workspace_held_before_does_not_count(T, bits):
    """Every byte set: NaN in each place of h and of the partial sums that the call does not write."""
    from llada_quant_b200 import _lib, ops
    from llada_quant_b200.few_tokens import FewTokenMoE
    from tests.test_few_tokens import check, make_layer, packed_of
    layer, x, _, weights, ids = make_layer(T, 3, 160, 352, 2, bits, -1)
    want = FewTokenMoE(packed_of(layer, -1), None, 2).routed(x, weights, ids)
    check(want, x, layer, weights, ids)
    lib, desc = _lib.load(), ops.few_layer(*layer[:4], 2, bits)
    nbytes = lib.llq_moe_few_workspace_size(T, 2, 3, 160, 352)
    ws = torch.full((nbytes + 256,), 0xFF, dtype=torch.uint8, device="cuda")
    out = torch.full_like(x, float("nan"))
    _lib.check(lib.llq_moe_few(ctypes.byref(desc), x.data_ptr(), T, None, weights.data_ptr(), ids.data_ptr(), out.data_ptr(),
                               ws.data_ptr(), nbytes, ops._stream(x)))
    assert torch.equal(out, want) and bool((ws[nbytes:] == 0xFF).all())


# ---------------------------------------------------------------------------
# operands that change between calls
# ---------------------------------------------------------------------------

def layer_parts(device):
    from llada_quant_b200.moe import PackedExperts
    from tests.test_few_tokens import make_layer
    layer, x, gate, weights, ids = make_layer(4, 8, 256, 128, 2, 4, 128, device=device)
    return PackedExperts(*layer[:4], 4, 128), x, gate, weights, ids


def test_exchanged_operands_reach_the_next_call_without_a_gpu(monkeypatch):
    """The addresses that a call passes are those of the operands at the call."""
    from llada_quant_b200 import ops
    from llada_quant_b200.few_tokens import FewTokenMoE
    passed = []
    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: None)
    monkeypatch.setattr(ops, "few_call", lambda layer, x, *a: passed.append(layer) or x)
    packed, x, gate, weights, ids = layer_parts("cpu")
    router = torch.nn.Linear(256, 8, bias=False, dtype=torch.bfloat16).requires_grad_(False)
    router.weight.copy_(gate)
    bias = torch.zeros(8)
    moe = FewTokenMoE(packed, router.weight, 2, bias)
    moe(x)
    old = router.weight.data_ptr()
    router.float()
    with pytest.raises(ValueError, match="gate_w must be"):
        moe(x)
    router.bfloat16()
    moe(x)
    assert passed[0].gate_w == old and passed[1].gate_w == router.weight.data_ptr()
    for t, name in ((packed.qw1, "qw1"), (packed.sw1, "sw1"), (packed.qw2, "qw2"), (packed.sw2, "sw2"), (bias, "bias")):
        t.data = t.data.clone()
        moe.with_logits(x)
        assert getattr(passed[-1], name) == t.data_ptr(), name
        moe.routed(x, weights, ids)
        assert name == "bias" or getattr(passed[-1], name) == t.data_ptr(), name
    router.weight.data = router.weight.data[:, 128:]
    with pytest.raises(ValueError, match="gate_w must be"):
        moe(x)
    router.weight.data = gate.clone()
    moe(x)
    router.weight.data.untyped_storage().resize_(0)
    with pytest.raises(ValueError, match="no memory"):
        moe(x)


@pytest.mark.gpu
def test_exchanged_operands_reach_the_next_call():
    from llada_quant_b200.few_tokens import FewTokenMoE
    packed, x, gate, weights, ids = layer_parts("cuda")
    router = torch.nn.Linear(256, 8, bias=False, dtype=torch.bfloat16, device="cuda").requires_grad_(False)
    router.weight.copy_(gate)
    moe = FewTokenMoE(packed, router.weight, 2)
    want = moe(x)
    router.float()  # the bf16 storage is given back
    fill = [torch.full((8, 256), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(8)]
    with pytest.raises(ValueError, match="gate_w must be"):
        moe(x)
    router.bfloat16()
    assert all(torch.equal(a, b) for a, b in zip(moe(x), want))
    router.weight.data = gate.flip(0).contiguous()
    assert torch.equal(moe(x)[2], 7 - want[2])
    was = moe.routed(x, weights, ids)
    packed.sw2.data = packed.sw2 * 2
    assert torch.equal(moe.routed(x, weights, ids), was * 2)
    del fill


def odd_router(gate, bias):
    """gate_w between other columns, and a bias that is exact in bf16: both have to be copied."""
    wide = torch.zeros(gate.shape[0], gate.shape[1] + 7, dtype=gate.dtype, device=gate.device)
    wide[:, 3:3 + gate.shape[1]] = gate
    return wide[:, 3:3 + gate.shape[1]], bias.to(torch.bfloat16)


def test_copied_operands_are_copied_for_each_call_without_a_gpu(monkeypatch):
    from llada_quant_b200 import ops
    from llada_quant_b200.few_tokens import FewTokenMoE
    seen = []

    def call(layer, x, *a):
        seen.append((list((ctypes.c_float * 8).from_address(layer.bias)),
                     list((ctypes.c_int16 * 2048).from_address(layer.gate_w))))
        return x

    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: None)
    monkeypatch.setattr(ops, "few_call", call)
    packed, x, gate, _, _ = layer_parts("cpu")
    g, b = odd_router(gate, torch.arange(8) / 8)
    moe = FewTokenMoE(packed, g, 2, b)
    for change in (lambda: None, lambda: b.fill_(3), lambda: g.mul_(2)):
        change()
        for run in (moe, moe.with_logits):
            run(x)
            assert seen[-1] == (b.tolist(), g.contiguous().view(torch.int16).flatten().tolist())


@pytest.mark.gpu
def test_operands_changed_in_place_reach_calls_and_replays():
    from llada_quant_b200.few_tokens import FewTokenMoE
    packed, x, gate, _, _ = layer_parts("cuda")
    plain = torch.arange(8, device="cuda") / 8
    for g, b in ((gate.clone(), plain.clone()), odd_router(gate, plain)):
        moe, graph = FewTokenMoE(packed, g, 2, b), torch.cuda.CUDAGraph()
        moe(x)
        with torch.cuda.graph(graph):
            held = moe(x)
        eager = moe(x)  # before any replay
        for change in (lambda: None, lambda: b.copy_(plain.flip(0)), lambda: g.copy_(gate.flip(0))):
            change()
            want = FewTokenMoE(packed, g.contiguous(), 2, b.float())(x)
            graph.replay()
            for got in (moe(x), held):
                assert all(torch.equal(p, q) for p, q in zip(got, want))
        assert all(torch.equal(p, q) for p, q in zip(eager, FewTokenMoE(packed, gate, 2, plain)(x)))


def linear_of(device, bias_dtype=torch.bfloat16, compute=torch.bfloat16):
    """An Fp8Linear 256 -> 40 on random bytes, with a bias that is exact in every type."""
    from llada_quant_b200.fp8 import Fp8Linear
    m = Fp8Linear(256, 40, bias=True, compute_dtype=compute)
    g = torch.Generator().manual_seed(1)
    m.qweight.copy_(torch.randint(0, 0x70, m.qweight.shape, generator=g, dtype=torch.uint8))
    m.scale.copy_(torch.rand(m.scale.shape, generator=g) / 64)
    m.bias = (torch.arange(40) / 4).to(bias_dtype)
    return m.to(device)


def odd_buffers(m):
    """Replaces each buffer of m by one that has to be copied."""
    bad = torch.empty(m.qweight.numel() + 1, dtype=torch.uint8, device=m.qweight.device)[1:].view(m.qweight.shape)
    m.qweight = bad.copy_(m.qweight)
    m.scale = m.scale.t().contiguous().t() if m.scale.shape[0] > 1 else m.scale.repeat_interleave(2, 1)[:, ::2]
    m.bias = m.bias.float()
    return m


def test_copied_buffers_are_copied_for_each_call_without_a_gpu(monkeypatch):
    """The operand of a call holds what the buffers hold at the call, whether they are read in place or copied."""
    from llada_quant_b200 import ops
    seen = []
    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: None)
    monkeypatch.setattr(ops.Fp8Weight, "multiply", lambda w, x, s=None: seen.append(
        (w.codes.view(torch.uint8).clone(), w.scale.clone(), w.bias.float())) or x.new_zeros(x.shape[0], w.N))
    x = torch.zeros(3, 256)
    one_by_one = [lambda m: setattr(m, "bias", m.bias.float()), lambda m: setattr(m, "scale", odd_buffers(linear_of("cpu")).scale)]
    for make in (lambda m: None, odd_buffers, *one_by_one):
        m = linear_of("cpu")
        make(m)
        for change in (lambda: None, lambda: m.bias.fill_(3), lambda: m.scale.mul_(2), lambda: m.qweight.fill_(8),
                       lambda: m.load_state_dict(linear_of("cpu").state_dict())):
            change()
            m(x)
            assert all(torch.equal(a, b) for a, b in zip(seen[-1], (m.qweight, m.scale, m.bias.float())))


@pytest.mark.gpu
def test_buffers_changed_in_place_reach_calls_and_replays():
    from tests.test_fp8 import check_product
    from llada_quant_b200.fp8 import quantize_fp8
    x = torch.randn(5, 256, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    q = quantize_fp8(x)
    for make in (lambda m: m, odd_buffers):
        m, graph = make(linear_of("cuda")), torch.cuda.CUDAGraph()
        make(linear_of("cuda"))(x)
        with torch.cuda.graph(graph):
            held = m(x)  # the module's first call
        eager = m(x)  # before any replay
        check_product(eager, q.codes, q.scale, m.weight, m.bias)
        for change in (lambda: None, lambda: m.bias.fill_(3), lambda: m.scale.mul_(2), lambda: m.qweight.sub_(8).clamp_(0, 0x70)):
            change()
            graph.replay()
            assert torch.equal(held, m(x))
            check_product(held, q.codes, q.scale, m.weight, m.bias)


def test_a_changed_compute_dtype_reaches_the_next_call_without_a_gpu(monkeypatch):
    from llada_quant_b200 import ops
    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: None)
    monkeypatch.setattr(ops.Fp8Weight, "multiply", lambda w, x, s=None: x.new_zeros(x.shape[0], w.N, dtype=w.dtype))
    m, x = linear_of("cpu"), torch.zeros(3, 256)
    for dtype in (torch.bfloat16, torch.float32, torch.float16, torch.bfloat16):
        m.compute_dtype = dtype
        assert m(x).dtype == dtype and m(x).dtype == dtype


def test_replaced_buffers_are_given_back_without_a_gpu(monkeypatch):
    """Moved, loaded by assignment or set: nothing keeps what the buffers were until the next call."""
    from llada_quant_b200 import ops
    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: None)
    fresh = linear_of("cpu")
    for replace in (lambda m: m.to_empty(device="cpu"), lambda m: m.load_state_dict(fresh.state_dict(), assign=True),
                    lambda m: [setattr(m, n, getattr(fresh, n).clone()) for n in ("qweight", "scale", "bias")]):
        m = linear_of("cpu")
        w = m._multiplier()
        assert w is m._multiplier()
        old = [weakref.ref(t) for t in (m.qweight, m.scale, m.bias, w.codes, w.scale, w.bias)]
        del w
        replace(m)
        gc.collect()
        assert all(r() is None for r in old)


@pytest.mark.gpu
def test_a_moved_module_gives_its_memory_back():
    from llada_quant_b200.fp8 import Fp8Linear
    m = Fp8Linear(4096, 4096).cuda()
    x = torch.ones(1, 4096, dtype=torch.bfloat16, device="cuda")
    y = m(x)
    before = torch.cuda.memory_allocated()
    m.cpu()
    assert before - torch.cuda.memory_allocated() >= 4096 * 4096
    assert torch.equal(m.cuda()(x), y)


# ---------------------------------------------------------------------------
# registered operators
# ---------------------------------------------------------------------------

def operator_calls(device):
    """name -> (operator, arguments), with x transposed, sliced or wide where a caller may have it so."""
    from llada_quant_b200 import ops  # noqa: F401
    from llada_quant_b200.fp8 import quantize_fp8
    packed, x, gate, weights, ids = layer_parts(device)
    p = (packed.qw1, packed.sw1, packed.qw2, packed.sw2)
    calls = {}
    wide = torch.zeros(4, 300, dtype=torch.bfloat16, device=device)
    for name, v in (("plain", x), ("transposed", x.t().contiguous().t()), ("sliced", wide[:, 7:263])):
        calls[f"moe_few {name}"] = (torch.ops.llada_quant.moe_few, (v, gate, None, True, *p, 2, 4))
        calls[f"moe_few_routed {name}"] = (torch.ops.llada_quant.moe_few_routed, (v, *p, weights, ids, 4))
        for rows in (1, 128):
            calls[f"fp8_quantize {name} {rows}"] = (torch.ops.llada_quant.fp8_quantize, (v[:, :201], rows))
        if device == "cuda":
            w, q = quantize_fp8(gate, 128), quantize_fp8(v)
            for out in (torch.bfloat16, torch.float32):
                calls[f"fp8_linear values {name} {out}"] = (torch.ops.llada_quant.fp8_linear,
                                                            (v, None, w.codes, w.scale, gate[:, 0].to(out), out))
                calls[f"fp8_linear codes {name} {out}"] = (torch.ops.llada_quant.fp8_linear,
                                                           (q.codes, q.scale, w.codes, w.scale, None, out))
    return calls


def test_fake_outputs_are_laid_out_like_the_real_ones():
    from torch._subclasses.fake_tensor import FakeTensorMode
    calls = operator_calls("cpu")
    with FakeTensorMode(allow_non_fake_inputs=True):
        for name, (op, args) in calls.items():
            out = op(*args)
            for t in out if isinstance(out, tuple) else (out,):
                assert t.stride(1) == 1 and t.stride(0) in (t.shape[1], -(-t.shape[1] // 16) * 16), name


@pytest.mark.gpu
def test_registered_operators_hold_to_their_contract():
    """Fake outputs against real ones; schema and a traced graph where no tensor is float8, which those checks multiply."""
    for name, (op, args) in operator_calls("cuda").items():
        more = ("test_schema", "test_aot_dispatch_static") if name.startswith("moe") else ()
        torch.library.opcheck(op.default, args, test_utils=("test_faketensor", *more))


@pytest.mark.gpu
def test_registered_operators_equal_the_python_entry_points():
    from llada_quant_b200.few_tokens import FewTokenMoE
    from llada_quant_b200.fp8 import Fp8Tensor, fp8_linear, quantize_fp8
    packed, _, gate, _, _ = layer_parts("cuda")
    moe = FewTokenMoE(packed, gate, 2, renormalize=True)
    for name, (op, args) in operator_calls("cuda").items():
        got, x = op(*args), args[0]
        if name.startswith("moe_few_routed"):
            want = (moe.routed(x, *args[5:7]),)
        elif name.startswith("moe_few"):
            want = moe.with_logits(x)
        elif name.startswith("fp8_quantize"):
            q = quantize_fp8(*args)
            want, got = (q.codes.float(), q.scale), (got[0].float(), got[1])
        else:
            x = Fp8Tensor(x, args[1], 1) if args[1] is not None else x
            want = (fp8_linear(x, Fp8Tensor(args[2], args[3], 128), args[4], args[5]),)
        got = got if isinstance(got, tuple) else (got,)
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and len(got) == len(want), name


@pytest.mark.gpu
@pytest.mark.parametrize("bias_dtype", [torch.float32, torch.bfloat16])
def test_captured_logits_are_those_before_the_bias(bias_dtype):
    """As the layer for many tokens records them; with_logits adds the bias."""
    from llada_quant_b200.few_tokens import FewTokenMoE
    from llada_quant_b200.fused_moe import moe_layer
    from llada_quant_b200.router_capture import RouterCapture
    from tests.test_few_tokens import logits64
    packed, x, gate, _, _ = layer_parts("cuda")
    bias = torch.arange(8, device="cuda").to(bias_dtype)
    bias[3] = -torch.inf
    z, dz = logits64(x, gate, None)
    for name, impl, step in (("few", "few", 0.0), ("many", "auto", 2.0 ** -8)):
        cap = RouterCapture()
        moe_layer(x, gate, packed, 2, bias, impl=impl, capture=cap, name=name)
        off = (cap.gates[name].double().cuda() - z).abs()
        assert bool((off <= dz + step * (z.abs() + dz)).all()), (name, off.max().item())
    logits = FewTokenMoE(packed, gate, 2, bias).with_logits(x)[3].double()
    zb, dzb = logits64(x, gate, bias)
    assert bool((((logits - zb).abs() <= dzb) | (torch.isinf(zb) & (logits == zb))).all())
    assert bool((logits[:, 3] == -torch.inf).all())
    with torch.no_grad():
        moe = FewTokenMoE(packed, gate, 2, bias.clone().requires_grad_())
    assert not moe.with_logits(x)[3].requires_grad


# ---------------------------------------------------------------------------
# quantizer and product through their module
# ---------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("M,K", [(1, 1), (1, 16), (3, 127), (5, 128), (129, 129)])
@pytest.mark.parametrize("rows", [1, 128])
def test_codes_have_their_shape_and_an_aligned_pitch(M, K, rows):
    from llada_quant_b200.fp8 import quantize_fp8
    q = quantize_fp8(torch.ones(M, K, device="cuda"), rows)
    assert q.codes.shape == q.shape == (M, K) and q.scale.shape == (-(-M // rows), -(-K // 128))
    assert M == 1 or q.codes.stride() == (-(-K // 16) * 16, 1)
    assert bool((q.codes.float() == 448).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
def test_from_linear_holds_the_quantized_weight_and_multiplies_by_it(dtype):
    from llada_quant_b200.fp8 import Fp8Linear, quantize_fp8
    from tests.test_fp8 import check_product, plain_quantize
    g = torch.Generator().manual_seed(5)
    lin = torch.nn.Linear(1040, 520, bias=True, dtype=dtype)
    with torch.no_grad():
        lin.weight.copy_(torch.randn(520, 1040, generator=g) * 0.02)
        lin.bias.copy_((torch.randn(520, generator=g) * 0.1).bfloat16())  # exact in the module's type
    m = Fp8Linear.from_linear(lin.cuda())
    code, scale = plain_quantize(lin.weight.detach().float(), 128)
    assert torch.equal(m.qweight.cpu(), code.view(torch.uint8)) and torch.equal(m.scale.cpu(), scale)
    for M in (1, 6, 40):
        x = torch.randn(M, 1040, generator=g).to(torch.bfloat16).cuda()
        q = quantize_fp8(x)
        check_product(m(x), q.codes, q.scale, m.weight, lin.bias.detach().bfloat16())
        check_product(m(q), q.codes, q.scale, m.weight, lin.bias.detach().bfloat16())


@pytest.mark.gpu
def test_few_token_layer_without_tokens_records_nothing():
    from llada_quant_b200.fused_moe import moe_layer
    from llada_quant_b200.router_capture import RouterCapture
    from llada_quant_b200.routing_stats import RoutingRecorder
    packed, x, gate, _, _ = layer_parts("cuda")
    rec, cap = RoutingRecorder(8, "cuda"), RouterCapture()
    assert moe_layer(x[:0], gate, packed, 2, impl="few", recorder=rec, capture=cap, name="l").shape == (0, 256)
    assert rec.stats().counts == [0] * 8 and cap.gates["l"].shape == (0, 8) and cap.topk_ids["l"].shape == (0, 2)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_codes_are_the_nearest_within_the_quotients_rounding(rows, dtype):
    """In 64 bits: bf16 and fp16 exactly the nearest, fp32 up to 2^-23 of the value (two fp32 roundings)."""
    from llada_quant_b200.fp8 import quantize_fp8
    x = torch.randn(256, 1024, generator=torch.Generator("cuda").manual_seed(4), device="cuda")
    x[:, ::128] = 4.0
    # 448 x / 4 next to borders between codes, from both sides
    edge = torch.tensor([(8 + m + 0.5) * 2.0 ** e / 112 for e in range(-9, 4) for m in range(8)], device="cuda")
    for i in range(64):
        x[i, 1:1 + edge.numel()] = edge * (1 + (i - 32) * 2.0 ** -24)
    x[128, :128] = 0.9962565898895264 / 4
    x[128, :2] = torch.tensor([0.9962565898895264, 4.1261671867687255e-05], device="cuda")
    x = x.to(dtype)
    q = quantize_fp8(x, rows)
    amax = x.double().view(256 // rows, rows, 8, 128).abs().amax((1, 3))
    v = x.double() * 448 / amax.repeat_interleave(rows, 0).repeat_interleave(128, 1)
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    slack = 2.0 ** -23 if dtype == torch.float32 else 0.0
    assert bool(((q.codes.double() - v).abs() <= step / 2 + (slack + 2.0 ** -50) * v.abs()).all())
