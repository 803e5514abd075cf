"""The e4m3 quantizer and product against their definitions, and their refusals.

Quantizer: the definition's fp32 steps (IEEE division, nearest-even rounding) give the same codes and scales
bit for bit, on the CPU too.

Product: v in fp64 from the codes.  A block's sum of exact products runs through at most 16 + 8 fp32 steps on
mma.sync (16 inside an MMA, 8 MMAs) and 32 + 4 on tcgen05; two steps per block follow (scale, sum; the product of
the two scales one more), one per partial that meets it and the bias.  With u = 2^-23 for a rounded or truncated step,
    dv <= (64 + 3 G) u sum of |products|,   |out - v| <= dv + half (|v| + dv) (+ the type's smallest step / 2)
where half is eps / 2 of the output's type.
"""

from __future__ import annotations

import pytest
import torch

from llada_quant_b200 import _lib

U = 2.0 ** -23
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def plain_quantize(x, rows):
    """codes (float8) and scales in fp32 steps, on the CPU."""
    x = x.cpu()
    M, K = x.shape
    R, G = -(-M // rows), -(-K // 128)
    v = torch.zeros(R * rows, G * 128)
    v[:M, :K] = x.float()
    v = v.view(R, rows, G, 128)
    amax = v.abs().amax((1, 3), keepdim=True).clamp(min=448 * 2.0 ** -60)
    code = ((v * 0.4375) / (amax * 2.0 ** -10)).view(R * rows, -1)[:M, :K].to(torch.float8_e4m3fn)
    return code, (amax / 448.0).view(R, G)


def spread(scale, rows, M, K):
    return scale.double().repeat_interleave(rows, 0)[:M].repeat_interleave(128, 1)[:, :K]


def same_bits(q, code, scale):
    assert torch.equal(q.codes.cpu().contiguous().view(torch.uint8), code.contiguous().view(torch.uint8))
    assert torch.equal(q.scale.cpu().view(torch.int32), scale.view(torch.int32))


def check_product(out, xc, xs, w, bias=None):
    from llada_quant_b200.fp8 import Fp8Tensor
    assert isinstance(w, Fp8Tensor)
    (M, K), N = xc.shape, w.shape[0]
    a = xc.double() * spread(xs, 1, M, K)
    b = w.codes.double() * spread(w.scale, 128, N, K)
    v, mag = a @ b.t(), a.abs() @ b.abs().t()
    if bias is not None:
        v, mag = v + bias.double(), mag + bias.double().abs()
    dv = (64 + 3 * -(-K // 128)) * U * mag
    fin = torch.finfo(out.dtype)
    bound = dv + fin.eps / 2 * (v.abs() + dv) + fin.smallest_normal * fin.eps / 2
    off = (out.double() - v).abs()
    assert out.shape == (M, N)
    assert bool((off <= bound).all()), (off - bound).max().item()


def values(M, K, dtype, seed, device="cuda"):
    g = torch.Generator(device).manual_seed(seed)
    x = torch.randn(M, K, generator=g, device=device)
    return (x * torch.exp(torch.randn(K, generator=g, device=device))).to(dtype)


# ---------------------------------------------------------------------------
# quantizer
# ---------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 16), (3, 127), (5, 128), (129, 129), (128, 256), (300, 1000), (2, 8200),
                                 (257, 2048), (1000, 136)])
def test_quantizer_equals_its_definition(M, K, rows, dtype):
    from llada_quant_b200.fp8 import quantize_fp8
    x = values(M, K, dtype, M + K)
    q = quantize_fp8(x, rows)
    assert q.codes.shape == (M, K) and q.codes.stride(0) % 16 == 0 or M == 1
    same_bits(q, *plain_quantize(x, rows))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantizer_with_many_groups_per_warp(dtype):
    from llada_quant_b200.fp8 import quantize_fp8
    x = values(1200, 4104, dtype, 9)  # 39600 groups, and a tail of 8 in every row
    same_bits(quantize_fp8(x), *plain_quantize(x, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 128])
def test_quantizer_at_the_ends_of_the_range(rows):
    """Zeros, the smallest and largest numbers, exact ties, NaN and infinities; each in rows of its own."""
    from llada_quant_b200.fp8 import quantize_fp8
    g = torch.Generator("cuda").manual_seed(3)
    base = torch.randn(128, 384, generator=g, device="cuda")
    big, tiny = torch.finfo(torch.float32).max, 2.0 ** -149
    for fill in (0.0, tiny, 1e-38, 2.0 ** -55, 1e30, big / 8):
        x = base * fill
        x[:, 200] = fill
        same_bits(quantize_fp8(x, rows), *plain_quantize(x, rows))
    x = base.clone()
    x[:, 130] = big
    same_bits(quantize_fp8(x, rows), *plain_quantize(x, rows))
    # 448 largest: the quotient is the value; halves of every spacing are ties
    steps = torch.arange(0, 384, device="cuda").float()
    x = (steps * 2.0 ** -10).repeat(128, 1)
    x[:, ::128] = 448.0
    same_bits(quantize_fp8(x, rows), *plain_quantize(x, rows))
    ties = torch.tensor([(8 + m + 0.5) * 2.0 ** e for e in range(-9, 6) for m in range(8)], device="cuda")
    x = torch.zeros(128, 384, device="cuda")
    x[:, 1:1 + 120] = ties[:120]
    x[:, ::128] = 448.0
    same_bits(quantize_fp8(x, rows), *plain_quantize(x, rows))
    for bad in (float("nan"), float("inf"), -float("inf")):
        x = base.clone()
        x[5, 140] = bad
        q = quantize_fp8(x, rows)
        v = q.dequantize()
        hurt = torch.zeros(128, 384, dtype=torch.bool, device="cuda")
        hurt[5 if rows == 1 else slice(None), 128:256] = True
        assert torch.equal(v.isnan(), hurt)
        code, scale = plain_quantize(x, rows)
        assert torch.equal(q.scale.cpu().isnan(), scale.isnan())
        clean, _ = plain_quantize(base, rows)
        ok = ~hurt.cpu()
        assert torch.equal(q.codes.cpu().float()[ok], clean.float()[ok])


@pytest.mark.gpu
def test_quantizer_strides_and_untouched_bytes():
    from llada_quant_b200 import ops
    from llada_quant_b200.fp8 import quantize_fp8
    big = values(40, 700, torch.bfloat16, 1)
    for x in (big[:, 3:603], big[::2, :130], big[:, ::2], big.t(), big[7:8], big[:, 8:16]):
        same_bits(quantize_fp8(x), *plain_quantize(x, 1))
        same_bits(quantize_fp8(x, 128), *plain_quantize(x, 128))
    x = values(6, 130, torch.float16, 2)
    codes = torch.full((7, 144), 0x55, dtype=torch.uint8, device="cuda")
    scale = torch.full((7, 2), -1.0, device="cuda")
    _lib.check(_lib.load().llq_fp8_quantize(x.data_ptr(), _lib.LLQ_F16, 6, 130, 130, 1, codes.data_ptr(), 144,
                                            scale.data_ptr(), ops._stream(x)))
    torch.cuda.synchronize()
    assert bool((codes[:, 130:] == 0x55).all()) and bool((codes[6] == 0x55).all()) and bool((scale[6] == -1).all())
    assert quantize_fp8(x[:0]).codes.shape == (0, 130)


# ---------------------------------------------------------------------------
# product
# ---------------------------------------------------------------------------

PRODUCTS = [
    # M, N, K
    (1, 1, 16), (1, 2048, 2048), (2, 17, 48), (7, 130, 144), (8, 16, 128), (9, 1000, 272), (16, 256, 1024),
    (17, 384, 2048), (31, 48, 4000), (33, 1000, 1360), (64, 2048, 512), (65, 128, 128), (127, 129, 1040),
    (128, 256, 256), (129, 512, 2048), (200, 77, 80), (256, 1024, 640), (300, 2000, 2064), (1000, 384, 304),
]


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_product_of_codes(M, N, K):
    from llada_quant_b200.fp8 import fp8_linear, quantize_fp8
    x, w = values(M, K, torch.float32, M), quantize_fp8(values(N, K, torch.float32, N + 1) * 0.05, 128)
    q = quantize_fp8(x)
    for dtype in DTYPES:
        check_product(fp8_linear(q, w, out_dtype=dtype), q.codes, q.scale, w)
    bias = values(1, N, torch.bfloat16, 5)[0]
    check_product(fp8_linear(q, w, bias), q.codes, q.scale, w, bias)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_product_of_values(M, N, K, dtype):
    """Quantized on the way as by the quantizer: the same codes, the same product."""
    from llada_quant_b200.fp8 import Fp8Linear, quantize_fp8
    x, w = values(M, K, dtype, M + 3), quantize_fp8(values(N, K, torch.float32, N + 1) * 0.05, 128)
    bias = values(1, N, dtype, 6)[0] if N % 2 else None
    out = Fp8Linear.from_codes(w, bias, dtype)(x)
    q = quantize_fp8(x)
    check_product(out, q.codes, q.scale, w, bias)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(1, 130, 16384), (2, 1000, 16400), (8, 4500, 1040), (16, 2050, 2048), (24, 4352, 4096),
                                   (8, 5001, 1040), (3, 9000, 144), (17, 5000, 512), (48, 300, 4096), (200, 512, 4096)])
def test_product_on_either_side_of_each_choice(M, N, K):
    """Rows quantized by the product or before it; few rows with a large weight."""
    from llada_quant_b200.fp8 import fp8_linear, quantize_fp8
    x, w = values(M, K, torch.bfloat16, M), quantize_fp8(values(N, K, torch.float32, N + 1) * 0.05, 128)
    q = quantize_fp8(x)
    check_product(fp8_linear(x, w), q.codes, q.scale, w)
    check_product(fp8_linear(q, w, out_dtype=torch.float32), q.codes, q.scale, w)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [5000, 5003])
@pytest.mark.parametrize("dtype", DTYPES)
def test_product_with_many_tiles_per_sm(N, dtype):
    """Three waves of the widest tile, the last of every row partly or wholly behind N; rows that are 16-byte aligned or not."""
    from llada_quant_b200 import ops
    from llada_quant_b200.fp8 import fp8_linear, quantize_fp8
    w = quantize_fp8(values(N, 400, torch.float32, 2) * 0.05, 128)
    q = quantize_fp8(values(2500, 400, torch.bfloat16, 1))
    bias = values(1, N, dtype, 3)[0]
    out = fp8_linear(q, w, bias, dtype)
    check_product(out, q.codes, q.scale, w, bias)
    assert torch.equal(fp8_linear(q, w, bias, dtype), out)
    assert ops.device_error() == 0


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """2.2 G values in and out: the last rows equal a call of their own."""
    from llada_quant_b200.fp8 import Fp8Tensor, fp8_linear, quantize_fp8
    rows = values(300, 32768, torch.bfloat16, 1)
    x = rows.repeat(220, 1)  # 66000 x 32768
    for r in (1, 128):
        q, part = quantize_fp8(x, r), quantize_fp8(rows[-80:], r)  # (66000 = 515 * 128 + 80)
        assert torch.equal(q.codes.view(torch.uint8)[-80:], part.codes.view(torch.uint8))
        assert torch.equal(q.scale[-part.scale.shape[0]:], part.scale)
        del q
    del x
    q = quantize_fp8(values(66000, 128, torch.bfloat16, 2))
    w = quantize_fp8(values(33024, 128, torch.float32, 3) * 0.05, 128)
    last = Fp8Tensor(q.codes[-80:], q.scale[-80:], 1)
    assert torch.equal(fp8_linear(q, w)[-80:], fp8_linear(last, w))


@pytest.mark.gpu
def test_linear_module_against_the_layer_it_replaces():
    from llada_quant_b200.fp8 import Fp8Linear
    g = torch.Generator().manual_seed(5)
    lin = torch.nn.Linear(1024, 520, bias=True)
    with torch.no_grad():
        lin.weight.copy_(torch.randn(520, 1024, generator=g) * 0.02)
        lin.bias.copy_(torch.randn(520, generator=g) * 0.1)
    m = Fp8Linear.from_linear(lin.cuda())
    x = torch.randn(2, 3, 1024, generator=g).to(torch.bfloat16).cuda()
    y = m(x)
    assert y.shape == (2, 3, 520) and y.dtype == torch.bfloat16
    # both operands are off by at most half an e4m3 step, 2^-4 of a value or 2^-10 of the block's amax / 448
    ref = torch.nn.functional.linear(x.double(), lin.weight.double(), lin.bias.double())
    wide = torch.nn.functional.linear(x.double().abs(), lin.weight.double().abs())
    amax = x.double().abs().amax() * lin.weight.double().abs().amax() * 1024 * 2.0 ** -10 / 448 * 2
    assert bool(((y.double() - ref).abs() <= wide * (2 * 2.0 ** -4 + 2.0 ** -8) + amax + 2.0 ** -8 * ref.abs() + 1e-6).all())
    state = {k: v.clone() for k, v in m.state_dict().items()}
    other = Fp8Linear(1024, 520, bias=True).cuda()
    other.load_state_dict(state)
    assert torch.equal(other(x), y)
    other.half()  # the bytes stay bytes; a scale that is no longer fp32 is refused
    assert other.qweight.dtype == torch.uint8
    with pytest.raises(ValueError, match="float32"):
        other(x)
    assert m.storage_bytes() == 520 * 1024 + 5 * 8 * 4 + 520 * 2
    assert torch.equal(m(x[:, :0]), y[:, :0])


@pytest.mark.gpu
def test_linear_module_copied_pickled_and_changed_in_place():
    import copy
    import io
    from llada_quant_b200.fp8 import Fp8Linear, quantize_fp8
    m = Fp8Linear.from_codes(quantize_fp8(values(200, 256, torch.float32, 1), 128), values(1, 200, torch.bfloat16, 2)[0])
    x = values(5, 256, torch.bfloat16, 3)
    y = m(x)
    twin, file = copy.deepcopy(m), io.BytesIO()
    torch.save(m, file)
    file.seek(0)
    for other in (twin, torch.load(file, weights_only=False)):
        assert other.qweight.data_ptr() != m.qweight.data_ptr() and torch.equal(other(x), y)
    twin.scale.mul_(2)
    twin.bias.mul_(2)
    assert torch.equal(twin(x), y * 2) and torch.equal(m(x), y)
    twin.qweight = m.qweight.clone().zero_()
    assert torch.equal(twin(x), twin.bias.expand(5, 200))


@pytest.mark.gpu
def test_zero_rows_nan_rows_and_strides():
    from llada_quant_b200.fp8 import Fp8Linear, fp8_linear, quantize_fp8
    w = quantize_fp8(values(300, 384, torch.float32, 1), 128)
    for M in (5, 150):
        x = values(M, 384, torch.bfloat16, 2)
        x[1] = 0
        x[3, 200] = float("nan")
        y = fp8_linear(x, w)
        keep = [i for i in range(M) if i != 3]
        q = quantize_fp8(x[keep])
        check_product(y[keep], q.codes, q.scale, w)
        assert bool((y[1] == 0).all()) and bool(y[3].isnan().all())
        big = torch.zeros(M, 500, dtype=torch.bfloat16, device="cuda")
        big[:, 5:389] = x
        assert torch.equal(fp8_linear(big[:, 5:389], w)[keep], y[keep])
        codes = torch.zeros(M, 401, dtype=torch.uint8, device="cuda")  # a pitch the kernel cannot read: copied
        q = quantize_fp8(x)
        codes[:, :384] = q.codes.view(torch.uint8)
        from llada_quant_b200.fp8 import Fp8Tensor
        odd = Fp8Tensor(codes[:, :384].view(torch.float8_e4m3fn), q.scale, 1)
        assert torch.equal(fp8_linear(odd, w)[keep], fp8_linear(q, w)[keep])
    assert Fp8Linear.from_codes(w)(x[:0]).shape == (0, 300)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [3, 40, 300])
def test_product_captured_and_on_two_streams(M):
    from llada_quant_b200.fp8 import Fp8Linear, quantize_fp8
    m = Fp8Linear.from_codes(quantize_fp8(values(640, 1024, torch.float32, 1), 128))
    xs = [values(M, 1024, torch.bfloat16, s) for s in range(4)]
    want = [m(x) for x in xs]
    ins, outs, graphs = [torch.empty_like(xs[0]) for _ in range(2)], [], []
    for v in ins:
        v.copy_(xs[0])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(m(v))
        graphs.append(g)
    for a, b in ((0, 1), (2, 3), (3, 0)):
        ins[0].copy_(xs[a])
        ins[1].copy_(xs[b])
        torch.cuda.synchronize()
        for g in graphs:
            with torch.cuda.stream(torch.cuda.Stream()):
                g.replay()
        eager = m(xs[b])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[a]) and torch.equal(outs[1], want[b]) and torch.equal(eager, want[b])


@pytest.mark.gpu
def test_a_step_of_both_kinds():
    """Projection in e4m3, experts for few tokens, projection back: as a decoding step runs them, captured."""
    from llada_quant_b200.few_tokens import FewTokenMoE
    from llada_quant_b200.fp8 import Fp8Linear, quantize_fp8
    from tests.test_few_tokens import check, make_layer, packed_of
    layer, x, gate, _, _ = make_layer(12, 16, 512, 256, 4, 4, 128)
    moe = FewTokenMoE(packed_of(layer, 128), gate, 4)
    up = Fp8Linear.from_codes(quantize_fp8(values(512, 512, torch.float32, 1) * 0.03, 128))
    head = Fp8Linear.from_codes(quantize_fp8(values(1000, 512, torch.float32, 2) * 0.03, 128), compute_dtype=torch.float32)

    def step(v):
        a = up(v)
        b, w, ids = moe(a)
        return a, b, w, ids, head(a + b)

    g = torch.cuda.CUDAGraph()
    warm = step(x)
    with torch.cuda.graph(g):
        got = step(x)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, warm))
    a, b, w, ids, y = got
    q = quantize_fp8(x)
    check_product(a, q.codes, q.scale, up.weight)
    check(b, a, layer, w, ids)
    q = quantize_fp8(a + b)
    check_product(y, q.codes, q.scale, head.weight)


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------

def test_c_refusals_need_no_gpu():
    lib = _lib.load()

    def quant(x=16, dt=_lib.LLQ_BF16, M=4, K=100, ldx=100, rows=1, codes=16, ldc=112, scale=16):
        return lib.llq_fp8_quantize(x, dt, M, K, ldx, rows, codes, ldc, scale, None), lib.llq_last_error()

    for kw, code, text in ((dict(M=-1), _lib.LLQ_EINVAL, b"bad shape"), (dict(K=0), _lib.LLQ_EINVAL, b"bad shape"),
                           (dict(ldx=99), _lib.LLQ_EINVAL, b"bad shape"), (dict(ldc=96), _lib.LLQ_EINVAL, b"bad shape"),
                           (dict(rows=64), _lib.LLQ_EUNSUPPORTED, b"128 x 128"), (dict(ldc=104), _lib.LLQ_EINVAL, b"16-byte"),
                           (dict(codes=8), _lib.LLQ_EINVAL, b"16-byte"), (dict(x=None), _lib.LLQ_EINVAL, b"null"),
                           (dict(dt=_lib.LLQ_E4M3), _lib.LLQ_EUNSUPPORTED, b"dtype")):
        rc, msg = quant(**kw)
        assert rc == code and text in msg, (kw, msg)
    assert quant(M=0, x=None)[0] == _lib.LLQ_OK

    def lin(x=16, dt=_lib.LLQ_E4M3, xs=16, M=4, K=128, ldx=128, w=16, ws=16, N=64, ldw=128, bias=None, out=16,
            ot=_lib.LLQ_BF16, wk=None, nb=0):
        return lib.llq_fp8_linear(x, dt, xs, M, K, ldx, w, ws, N, ldw, bias, out, ot, wk, nb, None), lib.llq_last_error()

    for kw, code, text in ((dict(M=-1), _lib.LLQ_EINVAL, b"bad shape"), (dict(N=0), _lib.LLQ_EINVAL, b"bad shape"),
                           (dict(ldw=112), _lib.LLQ_EINVAL, b"bad shape"), (dict(ot=_lib.LLQ_E4M3), _lib.LLQ_EUNSUPPORTED, b"output"),
                           (dict(K=120), _lib.LLQ_EUNSUPPORTED, b"multiples of 16"), (dict(ldw=136), _lib.LLQ_EINVAL, b"16-byte"),
                           (dict(w=8), _lib.LLQ_EINVAL, b"16-byte"), (dict(xs=None), _lib.LLQ_EINVAL, b"scales"),
                           (dict(ldx=136), _lib.LLQ_EINVAL, b"16-byte"), (dict(dt=9), _lib.LLQ_EUNSUPPORTED, b"dtype"),
                           (dict(K=2 ** 30 + 16, ldx=2 ** 31, ldw=2 ** 31), _lib.LLQ_EINVAL, b"K too large"),
                           (dict(dt=_lib.LLQ_BF16, M=17, xs=None), _lib.LLQ_ENOSPACE, b"workspace"),
                           (dict(out=None), _lib.LLQ_EINVAL, b"null")):
        rc, msg = lin(**kw)
        assert rc == code and text in msg, (kw, msg)
    assert lin(M=0, x=None, out=None)[0] == _lib.LLQ_OK


def test_python_refusals_need_no_gpu(monkeypatch):
    from llada_quant_b200 import ops
    from llada_quant_b200.fp8 import Fp8Linear, Fp8Tensor, fp8_linear, quantize_fp8
    x = torch.randn(4, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        quantize_fp8(x)
    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: None)
    for bad, rows, text in ((x[0], 1, "takes fp32"), (x.double(), 1, "takes fp32"), (x[:, :0], 1, "takes fp32"), (x, 64, "block_rows")):
        with pytest.raises(ValueError, match=text):
            quantize_fp8(bad, rows)
    with pytest.raises(RuntimeError, match="no backward"):
        quantize_fp8(x.clone().requires_grad_())
    w = Fp8Tensor(torch.zeros(32, 64, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.ones(1, 1), 128)
    r = Fp8Tensor(torch.zeros(4, 64, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.ones(4, 1), 1)
    for a, b, kw, text in ((x, r, {}, "128 x 128"), (w, w, {}, "128 values"), (x[:, :32], w, {}, "got"),
                           (x.double(), w, {}, "rows must be"), (x, w, dict(out_dtype=torch.float64), "gives"),
                           (x, w, dict(bias=torch.zeros(31)), "bias"),
                           (x, Fp8Tensor(w.codes, torch.ones(2, 1), 128), {}, "scales must be"),
                           (Fp8Tensor(r.codes, torch.ones(1, 4), 1), w, {}, "scales must be")):
        with pytest.raises(ValueError, match=text):
            fp8_linear(a, b, **kw)
    with pytest.raises(RuntimeError, match="no backward"):
        fp8_linear(x.clone().requires_grad_(), w)
    for n in (8, 100):
        with pytest.raises(ValueError, match="multiples of 16"):
            Fp8Linear(n, 32)
    with pytest.raises(ValueError, match="compute_dtype"):
        Fp8Linear(64, 32, compute_dtype=torch.float64)
