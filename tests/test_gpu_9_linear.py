"""INT8 projections on the GPU against their definitions in float64.

Tolerances.  A code is rint(y * (127 / max|y|)) with two fp32 roundings before the rint, so it lies within half a step of the
exact quotient, plus 127 * 2^-23 for those roundings and whatever error y itself has.  A product is an exact integer, converted
(one rounding), scaled twice, added to up to twice (2^-24 of the operands' magnitude each) and rounded once to the output's type
(half a step: finfo.eps / 2)."""
import numpy as np
import pytest
import torch

from triattention_b200.kernels.linear import Int8Ops, Int8Rows

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
TYPES = (BF16, FP16, FP32)
U = 2.0 ** -24          # half a step of fp32, relative


@pytest.fixture(scope="module")
def ops(module):
    return Int8Ops(module)


def randn(*shape, seed=0, dtype=BF16, outliers=False):
    gen = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn(*shape, generator=gen, device="cuda")
    if outliers:
        x = x * torch.where(torch.rand(shape[-1], generator=gen, device="cuda") < 0.02, 20.0, 1.0)
    return x.to(dtype)


def check_codes(rows, y, slack=0.0):
    """rows against the exact values y (float64 [T,H]); slack: relative error that y itself may have in fp32."""
    codes, scales = rows.codes.reshape(y.shape).double(), rows.scales.reshape(-1).double()
    largest = y.abs().amax(1)
    assert rows.codes.dtype == torch.int8 and rows.scales.dtype == FP32
    torch.testing.assert_close(scales, largest / 127, rtol=slack + 4 * U, atol=0)
    quotient = torch.where(largest[:, None] > 0, y / largest[:, None] * 127, 0.0)
    assert float((codes - quotient).abs().max()) <= 0.5 + 127 * (2 * U + 2 * slack)
    assert int(codes.abs().max()) <= 127


WIDTHS = [(1, 1), (1, 7), (3, 16), (2, 129), (5, 1000), (4, 1024), (33, 4096), (2, 5001), (3, 8192), (2, 14336), (2, 16384),
          (2, 32768), (1, 40000), (1, 131071), (700, 128), (1500, 65)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", WIDTHS)
def test_quantize_rows(ops, rows, width, dtype):
    x = randn(rows, width, seed=rows + width, dtype=dtype, outliers=True)
    check_codes(ops.quantize_rows(x), x.double())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", WIDTHS)
def test_silu_mul(ops, rows, width, dtype):
    gate, up = 3 * randn(rows, width, seed=1, dtype=dtype), randn(rows, width, seed=2, dtype=dtype, outliers=True)
    g, u = gate.double(), up.double()
    # __expf: 2 + 1.173 |x| steps of 2^-23; __fdividef: 2 steps; the sum and the product half a step each
    slack = (2 + 1.173 * float(g.abs().max()) + 2 + 1) * 2 * U
    check_codes(ops.silu_mul(gate, up), g * torch.sigmoid(g) * u, slack)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", WIDTHS)
@pytest.mark.parametrize("residual", (False, True))
def test_rms_norm(ops, rows, width, dtype, residual):
    x, w = randn(rows, width, seed=3, dtype=dtype, outliers=True), (1 + 0.2 * randn(width, seed=4, dtype=FP32)).to(dtype)
    r = 3 * randn(rows, width, seed=5, dtype=dtype) if residual else None
    got = ops.rms_norm(x, w, 1e-5, residual=r)
    h = x
    if residual:
        got, total = got
        h = (x.float() + r.float()).to(dtype)
        assert total.dtype == dtype and torch.equal(total, h)
    h = h.double()
    y = h / (h.square().mean(1, keepdim=True) + 1e-5).sqrt() * w.double()
    # h * w, rsqrt, division, products: half a step each; the sum of squares: at most a few steps (partial sums by thread)
    check_codes(got, y, slack=(8 + width / 256 + 16) * U)


def test_rows_that_hold_nothing_or_too_much(ops):
    inf, nan = float("inf"), float("nan")
    for dtype in TYPES:
        for width in (24, 333, 4096, 40000):
            x = randn(9, width, seed=6, dtype=dtype)
            x[1] = 0
            x[2, width - 1] = nan
            x[3, 0] = inf
            x[4, width // 2] = -inf
            x[5] = -0.0
            x[6] = torch.finfo(dtype).max
            x[7], x[7, 3] = 0, -torch.finfo(dtype).max
            rows = ops.quantize_rows(x)
            assert rows.scales[[1, 5]].tolist() == [0, 0] and not rows.codes[[1, 2, 3, 4, 5]].any()
            assert torch.isnan(rows.scales[2:5]).all()
            ok = [0, 6, 7, 8]
            check_codes(Int8Rows(rows.codes[ok], rows.scales[ok]), x[ok].double())
            back = ops.dequantize(rows, FP32)
            assert torch.isnan(back[2:5]).all() and not back[[1, 5]].any() and torch.isfinite(back[ok]).all()
            gated = ops.silu_mul(x, torch.ones_like(x))
            assert gated.scales[[1, 5]].tolist() == [0, 0] and torch.isnan(gated.scales[2:5]).all()
            assert not gated.codes[[1, 2, 3, 4, 5]].any()
            for eps in (1e-5, 0.0):
                normed = ops.rms_norm(x, torch.ones(width, dtype=dtype, device="cuda"), eps)
                assert normed.scales[[1, 5]].tolist() == [0, 0] and torch.isnan(normed.scales[2:5]).all()
                assert not normed.codes[[1, 2, 3, 4, 5]].any()
                h = x[ok].double()
                check_codes(Int8Rows(normed.codes[ok], normed.scales[ok]), h / (h.square().mean(1, keepdim=True) + eps).sqrt(),
                            slack=(24 + width / 256) * U)


@pytest.mark.parametrize("size", (1e30, 1e19, 1e-15, 1e-25, 1e-30))
@pytest.mark.parametrize("eps", (0.0, 1e-6))
@pytest.mark.parametrize("residual", (False, True))
def test_norm_of_rows_whose_squares_leave_fp32(ops, size, eps, residual):
    x = (randn(4, 777, seed=7, dtype=FP32) * size).to(BF16)
    w = torch.full((777,), 0.5, dtype=BF16, device="cuda")
    r = (randn(4, 777, seed=8, dtype=FP32) * size).to(BF16) if residual else None
    got = ops.rms_norm(x, w, eps, residual=r)
    h = (x if r is None else x + r).double()
    y = h / (h.square().mean(1, keepdim=True) + eps).sqrt() * 0.5
    check_codes(got if r is None else got[0], y, slack=32 * U)
    # in place: the new residual over the old one
    if residual:
        codes, scales = torch.empty(4, 784, dtype=torch.int8, device="cuda")[:, :777], torch.empty(4, device="cuda")
        ops.module.rms_norm_rows(x, w, eps, codes, scales, r, r)
        assert torch.equal(r, got[1]) and torch.equal(codes, got[0].codes) and torch.equal(scales, got[0].scales)


def test_rows_strided_offset_and_shaped(ops):
    """Halves of one tensor, every offset of the first element, a broadcast row, leading dimensions, an empty batch."""
    wide = randn(40, 3 * 1000 + 8, seed=9)
    for off in range(9):
        x = wide[:, off:off + 1000]
        got, want = ops.quantize_rows(x), ops.quantize_rows(x.contiguous())
        assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)
        up = wide[:, 2000 + off // 2:3000 + off // 2]
        got, want = ops.silu_mul(x, up), ops.silu_mul(x.contiguous(), up.contiguous())
        assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)
        w = wide[0, 3 + off:1003 + off]
        (got, total), (want, sums) = ops.rms_norm(x, w, 1e-6, residual=up), ops.rms_norm(x.contiguous(), w.clone(), 1e-6, residual=up.contiguous())
        # Codes do not depend on the sum of squares; scales do, and rows that lie differently are summed in another order: at most
        # 32 terms in turn and a tree of 10 (42 half steps) on each side, halved by the root, and four roundings after it.
        assert torch.equal(got.codes, want.codes) and torch.equal(total, sums)
        torch.testing.assert_close(got.scales, want.scales, rtol=46 * U, atol=0)
    one = randn(1, 96, seed=10)
    many = ops.quantize_rows(one.expand(5, 96))
    assert torch.equal(many.codes, ops.quantize_rows(one).codes.expand(5, 96))
    x = randn(2, 3, 130, seed=11)
    rows = ops.quantize_rows(x)
    assert rows.shape == (2, 3, 130) and rows.scales.shape == (2, 3) and rows.dtype == BF16
    assert torch.equal(rows.codes.reshape(6, 130), ops.quantize_rows(x.reshape(6, 130)).codes)
    assert ops.dequantize(rows).shape == x.shape and ops.dequantize(rows).dtype == BF16
    flat = ops.quantize_rows(x[0, 0])
    assert flat.shape == (130,) and flat.scales.shape == () and torch.equal(flat.codes, rows.codes[0, 0])
    none = ops.quantize_rows(x[:0])
    assert none.shape == (0, 3, 130) and ops.dequantize(none).shape == (0, 3, 130)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 129), (17, 4096), (2, 16400), (1000, 65)])
def test_dequantize(ops, rows, width, dtype):
    got = ops.quantize_rows(randn(rows, width, seed=12))
    out = ops.dequantize(got, dtype)
    assert out.dtype == dtype and torch.equal(out, (got.codes.float() * got.scales[:, None]).to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", [(1, 1), (2, 3), (5, 9), (700, 31), (33, 250), (700, 257), (400, 1003), (9, 2049), (320, 8195), (4, 9001),
                                        (310, 16391), (3, 20001), (2, 33333)])
def test_rows_that_start_anywhere(ops, rows, width, dtype):
    """Inputs between NaN, outputs between guards: nothing beside a row is used, nothing beside it is written; in place too."""
    def room(seed, off, fill):
        whole = torch.full((rows + 2, width + 11), fill, dtype=dtype, device="cuda")
        view = whole[1:-1, off:off + width]
        view.copy_(randn(rows, width, seed=seed, dtype=dtype))
        return whole, view

    def code_room():
        whole = torch.full((rows + 2, -(-width // 16) * 16 + 32), 99, dtype=torch.int8, device="cuda")
        return whole, whole[1:-1, 16:16 + width], torch.empty(rows, device="cuda")

    def beside(whole, view, fill):
        view.fill_(fill)
        assert bool((whole == fill).all())

    nan, m = float("nan"), ops.module
    (_, x), (_, u), (_, r) = room(70, 3, nan), room(71, 6, nan), room(72, 1, nan)
    w = randn(width + 1, seed=73, dtype=dtype)[1:]
    whole, codes, scales = code_room()
    m.quantize_rows(x, codes, scales)
    check_codes(Int8Rows(codes, scales), x.double())
    values_room, values = room(0, 5, 7.0)
    m.dequantize_rows(codes, scales, values)
    assert torch.equal(values, (codes.float() * scales[:, None]).to(dtype))
    beside(values_room, values, 7.0), beside(whole, codes, 99)
    whole, codes, scales = code_room()
    m.silu_mul_rows(x, u, codes, scales)
    g = x.double()
    check_codes(Int8Rows(codes, scales), g * torch.sigmoid(g) * u.double(), slack=(2 + 1.173 * float(g.abs().max()) + 2 + 1) * 2 * U)
    beside(whole, codes, 99)
    h = (x.float() + r.float()).to(dtype)
    y = h.double() / (h.double().square().mean(1, keepdim=True) + 1e-5).sqrt() * w.double()
    whole, codes, scales = code_room()
    total_room, total = room(0, 2, 7.0)
    m.rms_norm_rows(x, w, 1e-5, codes, scales, r, total)
    check_codes(Int8Rows(codes, scales), y, slack=(8 + width / 256 + 16) * U)
    assert torch.equal(total, h)
    again, again_scales = code_room()[1:]
    m.rms_norm_rows(x, w, 1e-5, again, again_scales, r, r)
    assert torch.equal(r, h) and torch.equal(again, codes) and torch.equal(again_scales, scales)
    beside(total_room, total, 7.0), beside(whole, codes, 99)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("stride", (0, 1, 3, 5, 9))
def test_rows_that_overlap(ops, stride, dtype):
    """One row for many, and windows of a sequence: rows less than 16 bytes apart."""
    for width in (37, 515):
        x = randn(9 * stride + width, seed=74, dtype=dtype).as_strided((10, width), (stride, 1))
        u = randn(9 * stride + width, seed=75, dtype=dtype).as_strided((10, width), (stride, 1))
        w = randn(width, seed=76, dtype=dtype)
        for call in (lambda x, u: ops.quantize_rows(x), lambda x, u: ops.silu_mul(x, u), lambda x, u: ops.rms_norm(x, w, 1e-6, residual=u)[0]):
            got, want = call(x, u), call(x.contiguous(), u.contiguous())
            assert torch.equal(got.codes, want.codes)
            torch.testing.assert_close(got.scales, want.scales, rtol=46 * U, atol=0)


# ---- products --------------------------------------------------------------------------------------------------------

def codes_rows(rows, width, seed, low=-127, high=128, extra=0):
    """Random code rows whose rows lie `extra` more 16-byte units apart than they must."""
    gen = torch.Generator("cuda").manual_seed(seed)
    pitch = (-(-width // 16) + extra) * 16
    codes = torch.randint(low, high, (rows, pitch), generator=gen, device="cuda", dtype=torch.int8)[:, :width]
    return Int8Rows(codes, torch.rand(rows, generator=gen, device="cuda") * 0.01 + 1e-4)


def check_linear(ops, x, w, dtype=BF16, bias=None, residual=None, got=None):
    if got is None:
        got = ops.linear(x, w, bias=bias, residual=residual, dtype=dtype)
    total = x.codes.double() @ w.codes.double().T               # exact: below 2^53
    y = total * w.scales.double() * x.scales.double()[:, None]
    size = y.abs() * 3
    for more in (bias, residual):
        if more is not None:
            y = y + more.double()
            size = size + more.double().abs() + y.abs()
    far = (got.double() - y).abs() - (U * 2 * size + y.abs() * torch.finfo(dtype).eps / 2 + 2.0 ** -25 * (dtype == FP16))
    assert got.dtype == dtype and got.shape == y.shape
    assert not far.numel() or float(far.max()) <= 0, (float(far.max()), int((far > 0).sum()))
    return got


SHAPES = [(1, 1, 1), (1, 17, 33), (2, 8, 16), (3, 128, 64), (7, 130, 127), (1, 4096, 4096), (8, 512, 1024), (16, 256, 4096),
          (16, 1000, 4099), (17, 129, 160), (31, 384, 8192), (32, 4608, 3584), (33, 96, 96), (64, 300, 1000), (65, 127, 2000),
          (100, 2000, 500), (127, 640, 2048), (128, 128, 128), (129, 257, 2051), (200, 1111, 777), (255, 256, 512), (256, 4096, 1024),
          (257, 513, 130), (300, 1000, 100), (511, 384, 384), (512, 512, 512), (777, 1003, 1051), (1000, 640, 512), (1500, 2048, 256),
          (1, 9001, 4099), (1, 5000, 2047), (1, 30001, 31), (1, 40, 131071), (1, 3, 2), (1, 700, 14336),
          (2049, 1025, 129), (4096, 512, 640), (3, 20000, 48), (5000, 3, 48), (700, 5000, 17), (2, 2, 30000), (24, 24, 131071)]


@pytest.mark.parametrize("tokens,outputs,width", SHAPES)
def test_linear(ops, tokens, outputs, width):
    x, w = codes_rows(tokens, width, 1), codes_rows(outputs, width, 2)
    check_linear(ops, x, w)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,outputs,width", [(1, 4096, 512), (5, 333, 1000), (48, 640, 4096), (130, 1001, 300), (600, 777, 1024),
                                                  (2048, 1024, 512)])
@pytest.mark.parametrize("with_bias,with_residual", [(True, False), (False, True), (True, True)])
def test_linear_types_bias_residual(ops, tokens, outputs, width, dtype, with_bias, with_residual):
    x, w = codes_rows(tokens, width, 3, low=-128), codes_rows(outputs, width, 4, low=-128, extra=1)
    check_linear(ops, x, w, dtype, randn(outputs, seed=5, dtype=dtype) if with_bias else None,
                 randn(tokens, outputs, seed=6, dtype=dtype) if with_residual else None)


@pytest.mark.parametrize("tokens,outputs", [(2, 130), (200, 140)])
def test_linear_largest_sums(ops, tokens, outputs):
    """Every product at its largest, at the widest row: 131071 * 128 * 128 = 2^31 - 16384."""
    x, w = codes_rows(tokens, 131071, 7), codes_rows(outputs, 131071, 8)
    x.codes.fill_(-128), w.codes.fill_(-128)
    x.scales.fill_(1), w.scales.fill_(1)
    assert torch.equal(ops.linear(x, w, dtype=FP32), torch.full((tokens, outputs), 2147467264.0, device="cuda"))
    w.codes.fill_(127)
    assert torch.equal(ops.linear(x, w, dtype=FP32), torch.full((tokens, outputs), -128.0 * 127 * 131071, device="cuda"))


@pytest.mark.parametrize("tokens", (1, 40, 300, 1100))
def test_linear_writes_its_rows_only(ops, tokens):
    """Output, residual and codes inside wider buffers: nothing beside the rows is written, nothing beside them is read."""
    outputs, width = 333, 250
    x, w = codes_rows(tokens, width, 9, extra=2), codes_rows(outputs, width, 10, extra=3)
    for rows in (x.codes, w.codes):      # what lies between the rows changes nothing
        base = rows.as_strided((rows.shape[0], rows.stride(0)), (rows.stride(0), 1))
        base[:, width:] = 77
    room = torch.full((tokens + 2, outputs + 9), 7.0, dtype=BF16, device="cuda")
    out = room[1:-1, 5:5 + outputs]
    residual = randn(tokens, outputs + 3, seed=11)[:, 2:-1]
    ops.module.int8_linear(x.codes, x.scales, w.codes, w.scales, out, residual=residual)
    check_linear(ops, x, w, residual=residual, got=out)
    kept = torch.full_like(room, 7.0)
    kept[1:-1, 5:5 + outputs] = out
    assert torch.equal(room, kept)
    want = out.clone()
    out.copy_(residual)                  # the residual stream updated in place
    ops.module.int8_linear(x.codes, x.scales, w.codes, w.scales, out, residual=out)
    assert torch.equal(out, want)


@pytest.mark.parametrize("tokens", (3, 70, 700))
def test_linear_keeps_a_bad_row_to_itself(ops, tokens):
    x, w = codes_rows(tokens, 512, 12), codes_rows(200, 512, 13)
    x.scales[1] = float("nan")
    x.codes[2].zero_()
    x.scales[2] = 0
    got = ops.linear(x, w, bias=torch.ones(200, dtype=BF16, device="cuda"))
    assert torch.isnan(got[1]).all() and (got[2] == 1).all()
    keep = [t for t in range(tokens) if t != 1]
    check_linear(ops, Int8Rows(x.codes[keep], x.scales[keep]), w, bias=torch.ones(200, dtype=BF16, device="cuda"), got=got[keep])


def test_linear_shapes_and_empty_batch(ops):
    x, w = codes_rows(6, 160, 14), codes_rows(64, 160, 15)
    flat = ops.linear(x, w)
    cube = Int8Rows(x.codes.view(2, 3, 160), x.scales.view(2, 3))
    got = ops.linear(cube, w, residual=torch.zeros(2, 3, 64, dtype=BF16, device="cuda"))
    assert got.shape == (2, 3, 64) and torch.equal(got.view(6, 64), flat)
    assert ops.linear(Int8Rows(x.codes[:0], x.scales[:0]), w).shape == (0, 64)
    one = ops.linear(Int8Rows(x.codes[0], x.scales[0]), w)
    assert one.shape == (64,) and torch.equal(one, ops.linear(Int8Rows(x.codes[:1], x.scales[:1]), w)[0])


def test_same_bits_every_time(ops):
    """The sums are integers, so no order of the work shows in the result."""
    for tokens, outputs, width in ((1, 4096, 8192), (40, 1000, 14336), (520, 1000, 4096)):
        x, w = codes_rows(tokens, width, 16), codes_rows(outputs, width, 17)
        first = ops.linear(x, w)
        assert all(torch.equal(ops.linear(x, w), first) for _ in range(5))


@pytest.mark.parametrize("outputs,width", [(4096, 4096), (1000, 14336), (333, 2051), (130, 500)])
def test_a_row_has_the_same_bits_in_every_batch(ops, outputs, width):
    """Whatever tile, split or pairing a batch gets, with bias and residual."""
    x, w = codes_rows(1100, width, 60), codes_rows(outputs, width, 61)
    bias, residual = randn(outputs, seed=62), randn(1100, outputs, seed=63)
    whole = ops.linear(x, w, bias=bias, residual=residual)
    for lo, hi in ((0, 1), (1, 17), (17, 81), (81, 281), (281, 700), (500, 1100)):
        part = Int8Rows(x.codes[lo:hi], x.scales[lo:hi])
        assert torch.equal(ops.linear(part, w, bias=bias, residual=residual[lo:hi]), whole[lo:hi]), (lo, hi)


@pytest.mark.parametrize("width", (64, 500, 4096, 5001, 14336))
def test_a_row_has_the_same_codes_in_every_batch(ops, width):
    """Rows of one layout: whatever number of them a call gets."""
    x, u, r, w = randn(900, width, seed=64, outliers=True), randn(900, width, seed=65), randn(900, width, seed=66), randn(width, seed=67)
    for call in (lambda lo, hi: ops.quantize_rows(x[lo:hi]), lambda lo, hi: ops.silu_mul(x[lo:hi], u[lo:hi]),
                 lambda lo, hi: ops.rms_norm(x[lo:hi], w, 1e-6, residual=r[lo:hi])[0]):
        whole = call(0, 900)
        for lo, hi in ((0, 1), (0, 37), (0, 400), (400, 900)):
            part = call(lo, hi)
            assert torch.equal(part.codes, whole.codes[lo:hi]) and torch.equal(part.scales, whole.scales[lo:hi])


# ---- together, and as programs use them ------------------------------------------------------------------------------

def layer(ops, state, x, residual):
    normed, residual = ops.rms_norm(x, state["norm"], 1e-5, residual=residual)
    both = ops.linear(normed, state["gate_up"])
    half = both.shape[-1] // 2
    return ops.linear(ops.silu_mul(both[..., :half], both[..., half:]), state["down"], bias=state["bias"], residual=residual)


def layer_state(ops, hidden=384, inner=1000):
    weight = lambda n, k, seed: ops.quantize_rows(0.05 * randn(n, k, seed=seed, dtype=FP32))
    return dict(norm=(1 + 0.1 * randn(hidden, seed=20, dtype=FP32)).to(BF16), gate_up=weight(2 * inner, hidden, 21),
                down=weight(hidden, inner, 22), bias=randn(hidden, seed=23))


@pytest.mark.parametrize("tokens", (1, 19, 300))
def test_a_feed_forward_block(ops, tokens):
    """Norm, gate and up, gated activation, down with bias and residual in one run: every stage is the exact function (float64) of
    what the stage before it gave, within that stage's own roundings, and the run's result has the last stage's bits."""
    state = layer_state(ops)
    x, residual = randn(tokens, 384, seed=24), randn(tokens, 384, seed=25)
    got = layer(ops, state, x, residual)
    normed, total = ops.rms_norm(x, state["norm"], 1e-5, residual=residual)
    assert torch.equal(total, (x.float() + residual.float()).to(BF16))
    h = total.double()
    check_codes(normed, h / (h.square().mean(1, keepdim=True) + 1e-5).sqrt() * state["norm"].double(), slack=32 * U)
    both = check_linear(ops, normed, state["gate_up"])
    g, u = both[:, :1000].double(), both[:, 1000:].double()
    gated = ops.silu_mul(both[:, :1000], both[:, 1000:])
    check_codes(gated, g * torch.sigmoid(g) * u, (5 + 1.173 * float(g.abs().max())) * 2 * U)
    check_linear(ops, gated, state["down"], bias=state["bias"], residual=total, got=got)


def test_captured_replayed_and_on_other_streams(ops):
    """Two graphs of one block over inputs of their own, replayed in turn and at the same time on two streams."""
    state = layer_state(ops)
    xs = [randn(t, 384, seed=30 + t) for t in (1, 40, 300)]
    rs = [randn(t, 384, seed=60 + t) for t in (1, 40, 300)]
    wants = [layer(ops, state, x, r) for x, r in zip(xs, rs)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x, r in zip(xs, rs):
            layer(ops, state, x, r)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for x, r in zip(xs, rs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(layer(ops, state, x, r))
        graphs.append(graph)
    for _ in range(3):
        for out in outs:
            out.zero_()
        side.wait_stream(torch.cuda.current_stream())
        for i, graph in enumerate(graphs):
            with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
                graph.replay()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(o, w) for o, w in zip(outs, wants))
    xs[1].copy_(xs[1].flip(0)), rs[1].copy_(rs[1].flip(0))
    graphs[1].replay()
    assert torch.equal(outs[1], wants[1].flip(0))
    ops.module.check_device_error()


def test_many_calls_at_once(ops):
    """Three streams with calls of every kind in flight at the same time (clusters that split the width, two CTAs per SM, pairs, rows):
    each gives what it gives alone."""
    jobs = []
    for i, (tokens, outputs, width) in enumerate(((1, 4096, 4096), (40, 2000, 8192), (300, 1000, 4096), (900, 4096, 1024), (16, 20000, 512),
                                                  (2500, 3000, 640))):
        x, w = codes_rows(tokens, width, 70 + i), codes_rows(outputs, width, 80 + i)
        jobs.append((x, w, ops.linear(x, w)))
    acts = randn(700, 8192, seed=90)
    want = ops.quantize_rows(acts)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for turn in range(20):
        for i, (x, w, y) in enumerate(jobs):
            with torch.cuda.stream(streams[(turn + i) % 3]):
                got.append((ops.linear(x, w), y))
        with torch.cuda.stream(streams[turn % 3]):
            got.append((ops.quantize_rows(acts).codes, want.codes))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in got)
    ops.module.check_device_error()


def test_refusals_on_the_gpu(ops):
    x, w = codes_rows(4, 64, 40), codes_rows(32, 64, 41)
    y = randn(4, 64, seed=42)
    with pytest.raises(RuntimeError, match="codes"):
        ops.linear(x, codes_rows(32, 80, 41))
    with pytest.raises(RuntimeError, match="16-byte"):
        ops.module.int8_linear(x.codes[:, 1:], x.scales, w.codes[:, 1:], w.scales, torch.empty(4, 32, dtype=BF16, device="cuda"))
    with pytest.raises(RuntimeError, match="bias"):
        ops.linear(x, w, bias=torch.zeros(32, device="cuda"))
    with pytest.raises(RuntimeError, match="bias"):
        ops.linear(x, w, bias=torch.zeros(31, dtype=BF16, device="cuda"))
    with pytest.raises(RuntimeError, match="residual"):
        ops.linear(x, w, residual=torch.zeros(4, 33, dtype=BF16, device="cuda"))
    with pytest.raises(RuntimeError, match="contiguous features"):
        ops.quantize_rows(y.T)
    with pytest.raises(RuntimeError, match="one shape"):
        ops.silu_mul(y, y[:3])
    with pytest.raises(RuntimeError, match="weight"):
        ops.rms_norm(y, torch.ones(63, dtype=BF16, device="cuda"), 1e-5)
    with pytest.raises(RuntimeError, match="eps"):
        ops.rms_norm(y, torch.ones(64, dtype=BF16, device="cuda"), -1.0)
    with pytest.raises(RuntimeError, match="no backward"):
        ops.quantize_rows(y.clone().requires_grad_())
    with torch.no_grad():
        ops.quantize_rows(y.clone().requires_grad_())


# ---- in a model ------------------------------------------------------------------------------------------------------

class DefinedOps:
    """The operators' definitions in float64, results in the types of Int8Ops: what the model computes with INT8 projections."""

    class Rows:
        def __init__(self, y, dtype):
            largest = y.abs().amax(-1, keepdim=True)
            step = torch.where(largest > 0, largest / 127, torch.ones_like(largest))
            self.values, self.dtype, self.shape = torch.round(y / step) * step, dtype, y.shape

    def quantize_rows(self, x):
        return self.Rows(x.double(), x.dtype)

    def silu_mul(self, gate, up):
        g = gate.double()
        return self.Rows(g * torch.sigmoid(g) * up.double(), gate.dtype)

    def rms_norm(self, x, weight, eps, residual=None):
        kept = x if residual is None else (x.float() + residual.float()).to(x.dtype)
        h = kept.double()
        rows = self.Rows(h / (h.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double(), x.dtype)
        return rows if residual is None else (rows, kept)

    def linear(self, rows, weight, bias=None, residual=None, dtype=None):
        y = rows.values @ weight.values.T
        for more in (bias, residual):
            if more is not None:
                y = y + more.double()
        return y.to(dtype or rows.dtype)


def toy_llama():
    from transformers import LlamaConfig, LlamaForCausalLM
    torch.manual_seed(0)
    cfg = LlamaConfig(hidden_size=512, intermediate_size=1000, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=2,
                      head_dim=128, vocab_size=1024, max_position_embeddings=1024, rope_theta=500000.0, attention_bias=True)
    return LlamaForCausalLM(cfg).to(BF16).cuda().eval()


@torch.inference_mode()
def test_model_with_int8_projections_is_what_the_definitions_say():
    """Both forms round at the same places, so they differ where a number lies next to a rounding border: per stage at most one
    element in 2^13 by a bf16 step (2^-8) and one code in 2^14 by 1/127 of a row's largest element (some 4 times its root mean
    square): 3e-4 of a stage's norm.  30 stages, each worth twice its error in what follows: 2 % of the logits' norm."""
    import copy
    from triattention_b200.models import int8_projections
    model = toy_llama()
    model.set_attn_implementation("sdpa")
    ids = torch.randint(0, 1024, (3, 50), generator=torch.Generator().manual_seed(1)).cuda()
    plain = model(input_ids=ids, use_cache=False).logits.float()
    defined = int8_projections(copy.deepcopy(model), DefinedOps())
    want = defined(input_ids=ids, use_cache=False).logits.float()
    got = int8_projections(model)(input_ids=ids, use_cache=False).logits.float()
    assert float((got - want).norm() / want.norm()) < 0.02
    assert float((got - plain).norm()) > 0          # (it is not the bf16 model)


@torch.inference_mode()
def test_generate_with_int8_projections(module):
    """Prompt pass, eager steps and the captured step over the quantised attention: the same tokens either way, whichever of the
    two is put into the model first."""
    from triattention_b200.maps import per_kv_head
    from triattention_b200.models import TriAttention, int8_projections
    ids = torch.randint(0, 1024, (3, 150), generator=torch.Generator().manual_seed(5)).cuda()
    rows = []
    for first in (True, False):
        model = toy_llama()
        if first:
            int8_projections(model)
        engine = TriAttention(model, per_kv_head(["int8", "int4"], 2), max_new_tokens=20)
        if not first:
            int8_projections(model)
        rows.append(engine.generate(ids, 20, eos=()))
        assert engine.generate(ids, 20, eos=(), cuda_graph=True) == rows[-1]
    assert rows[0] == rows[1] and all(len(r) == 20 for r in rows[0])
    module.check_device_error()


def test_a_first_call_inside_a_capture_is_refused(ops, monkeypatch):
    """The error word would be allocated from the capture's pool: the call says so instead."""
    x, w = codes_rows(2, 64, 50), codes_rows(16, 64, 51)
    ops.linear(x, w)
    kept = dict(ops.module._errors)
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph):
            ops.module._errors.clear()
            with pytest.raises(RuntimeError, match="outside of a stream capture"):
                ops.linear(x, w)
            ops.module._errors.update(kept)
            out = ops.linear(x, w)
    finally:
        ops.module._errors.update(kept)
    graph.replay()
    assert torch.equal(out, ops.linear(x, w))


@pytest.mark.skipif("torch.cuda.device_count() < 2")
def test_on_another_device_than_the_current_one(ops):
    x, w = codes_rows(5, 200, 52), codes_rows(70, 200, 53)
    def move(rows):
        codes = torch.zeros(rows.shape[0], 208, dtype=torch.int8, device="cuda:1")[:, :200]
        return Int8Rows(codes.copy_(rows.codes), rows.scales.to("cuda:1"))

    assert torch.equal(ops.linear(move(x), move(w)).cpu(), ops.linear(x, w).cpu())


# ---- the norm's second try -----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", (BF16, FP32))
@pytest.mark.parametrize("rows,width", [(5, 8), (700, 24), (300, 128), (300, 256), (5, 1024), (300, 4096), (3, 8704), (3, 16384), (2, 40000)])
@pytest.mark.parametrize("size", (1e30, 1e19, 1e-15, 1e-30))
def test_norm_of_aligned_rows_whose_squares_leave_fp32(ops, rows, width, size, dtype):
    """Rows of one warp and of many, with a residual: the second try reads the new residual that other threads have just written.
    Between rows that fit, beside rows that hold a NaN or an infinity, and in place."""
    x, r = ((randn(rows, width, seed=s, dtype=FP32) * size).to(dtype) for s in (110, 111))
    x[1::4], r[1::4] = randn(rows, width, seed=112, dtype=dtype)[1::4], randn(rows, width, seed=113, dtype=dtype)[1::4]
    w = (1 + 0.1 * randn(width, seed=114, dtype=FP32)).to(dtype)
    if rows > 3:
        x[2, width // 3], r[3, width - 1] = float("nan"), float("-inf")
    h = (x.float() + r.float()).to(dtype)
    good = torch.isfinite(h).all(1)
    wide = h.double()[good]
    y = wide / (wide.square().mean(1, keepdim=True) + 1e-6).sqrt() * w.double()

    def check(rows_of_codes, total):
        assert torch.equal(total.view(torch.int16 if dtype == BF16 else torch.int32)[good], h.view(torch.int16 if dtype == BF16 else torch.int32)[good])
        assert torch.isnan(rows_of_codes.scales[~good]).all() and not rows_of_codes.codes[~good].any()
        check_codes(Int8Rows(rows_of_codes.codes[good], rows_of_codes.scales[good]), y, slack=(8 + width / 256 + 16) * U)

    got, total = ops.rms_norm(x, w, 1e-6, residual=r)
    check(got, total)
    for place in ("residual", "x"):             # the new residual over the old one, or over x
        x2, r2 = x.clone(), r.clone()
        codes, scales = torch.empty(rows, -(-width // 16) * 16, dtype=torch.int8, device="cuda")[:, :width], torch.empty(rows, device="cuda")
        ops.module.rms_norm_rows(x2, w, 1e-6, codes, scales, r2, r2 if place == "residual" else x2)
        check(Int8Rows(codes, scales), r2 if place == "residual" else x2)


# ---- codes next to a tie -------------------------------------------------------------------------------------------------

# Every way through the row kernels: a warp a row, one warp a row with a ring, several warps (whole and with a remainder), two and
# four vectors a thread, rows that start anywhere, rows too wide for registers; a few rows and long batches.
TIE_SHAPES = [(5, 8), (3, 24), (700, 256), (900, 512), (5, 777), (400, 1000), (3, 4096), (500, 4096), (700, 4095), (2, 9000),
              (400, 8704), (2, 14336), (310, 14336), (310, 16391), (2, 40000)]


def rows_of_ties(rows, width, seed):
    """Whole numbers of which the largest is 254, so that every odd one's quotient, y / 2, lies on a tie."""
    gen = torch.Generator("cuda").manual_seed(seed)
    y = torch.randint(-253, 254, (rows, width), generator=gen, device="cuda").float()
    y[torch.arange(rows), torch.randint(0, width, (rows,), generator=gen, device="cuda")] = 254
    return y


def fp32_codes(y):
    """Scales and codes of y as the formulas have them, each operation in IEEE fp32: s = max|y| * fl(1/127), rint(y / s)."""
    assert y.dtype == FP32
    scales = y.abs().amax(1) * torch.tensor(1 / 127, device="cuda")
    return scales, torch.round(y / scales[:, None]).to(torch.int8)


def silu_mul_fp32(gate, up):
    """gate / (1 + e^-gate) * up in IEEE fp32; zero where the sum passes 2^126, as the kernels have it."""
    g, u = gate.float(), up.float()
    d = 1 + torch.exp(-g)
    return torch.where(d > 2.0 ** 126, 0 * g * u, g / d * u)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", TIE_SHAPES)
def test_plain_codes_are_those_of_fp32(ops, rows, width, dtype):
    """Bit for bit: on rows full of ties (where s = fl(fl(1/127) * 254) decides the side), and on rows as they come."""
    for y in (rows_of_ties(rows, width, 90), 1.4140625 * rows_of_ties(rows, width, 91), randn(rows, width, seed=92, dtype=FP32, outliers=True)):
        x = y.to(dtype)
        got, (scales, codes) = ops.quantize_rows(x), fp32_codes(x.float())
        assert torch.equal(got.scales, scales) and torch.equal(got.codes, codes)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", TIE_SHAPES)
def test_gated_codes_are_those_of_fp32(ops, rows, width, dtype):
    """Bit for bit, although most elements go by a fast exponential.  From a gate of 18 on 1 + e^-gate is 1 in fp32, so gates of 32 give
    y = 32 up: rows full of ties.  Then gates as they come, gates below -16 (where the exponential's error is largest) and beyond
    -87.3 (where the product counts as zero), and rows of nothing else."""
    gen = torch.Generator("cuda").manual_seed(93)
    ties = rows_of_ties(rows, width, 94) / 32
    spread = 90 * torch.rand(rows, width, generator=gen, device="cuda") * torch.where(torch.rand(rows, width, generator=gen, device="cuda") < 0.7, -1, 1)
    far = -14 - 70 * torch.rand(rows, width, generator=gen, device="cuda")
    for gate, up in ((torch.full_like(ties, 32), ties), (torch.full_like(ties, 32), 1.4140625 * ties),
                     (3 * randn(rows, width, seed=95, dtype=FP32), randn(rows, width, seed=96, dtype=FP32, outliers=True)),
                     (spread, randn(rows, width, seed=97, dtype=FP32)), (far, randn(rows, width, seed=98, dtype=FP32) * 1e20 if dtype != FP16 else ties)):
        gate, up = gate.to(dtype), up.to(dtype)
        y = silu_mul_fp32(gate, up)
        got, (scales, codes) = ops.silu_mul(gate, up), fp32_codes(y)
        live = y.abs().amax(1) >= 2.0 ** -119
        assert bool(live.any()) and torch.equal(got.scales, torch.where(live, scales, 0.0))
        assert torch.equal(got.codes, torch.where(live[:, None], codes, 0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", TIE_SHAPES)
@pytest.mark.parametrize("residual", (False, True))
def test_norm_codes_next_to_ties(ops, rows, width, dtype, residual):
    """A norm's code is rint(q), q = 127 y / max|y| rounded to fp32 once (2^-24 of q), y = fl(h * weight), ties to even: as exact arithmetic
    has it on rows of ties (multiples of half a weight), with powers of two in front that send the squares out of fp32's range,
    and on the ties among rows as they come."""
    y = rows_of_ties(rows, width, 99)
    gen = torch.Generator("cuda").manual_seed(100)
    w = 2.0 ** torch.randint(-1, 2, (width,), generator=gen, device="cuda")
    cases = [(y / w * 2.0 ** power, factor * w, torch.round(y / w) * 2.0 ** power)    # h - r is a half at most: exact in every type
             for power, factor in (((0, 1), (-30, 1.4140625), (66, 1.0078125), (-66, 1.7265625)) if dtype != FP16 else ((0, 1), (5, 1.4140625)))]
    cases.append((randn(rows, width, seed=101, dtype=FP32, outliers=True), 1 + 0.1 * randn(width, seed=102, dtype=FP32), 3 * randn(rows, width, seed=103, dtype=FP32)))
    for h, weight, r in cases:
        x, weight, r = (h - r if residual else h).to(dtype), weight.to(dtype), r.to(dtype)
        got = ops.rms_norm(x, weight, 1e-6, residual=r if residual else None)
        if residual:
            x = (x.float() + r.float()).to(dtype)
            assert torch.equal(got[1], x)
            got = got[0]
        z = (x.float() * weight.float()).double()
        q = z * 127 / z.abs().amax(1, keepdim=True)       # 127 z has 31 bits: a tie in float64 where the exact quotient is one, else 2^-32 away
        code = got.codes.double()
        assert float(((code - q).abs() - q.abs() * U).max()) <= 0.5
        tie = (q - q.floor()) == 0.5
        assert torch.equal(code[tie], torch.round(q[tie])) and (h is cases[-1][0] or bool(tie.any()))


# ---- copies --------------------------------------------------------------------------------------------------------------

def test_products_of_copied_and_saved_rows(ops):
    """A copy is read where it lies: what becomes of the original's memory does not show."""
    import copy
    import io
    w, x = ops.quantize_rows(randn(300, 1000, seed=120)), ops.quantize_rows(randn(5, 1000, seed=121))
    want = ops.linear(x, w)
    saved = io.BytesIO()
    torch.save(w, saved)
    saved.seek(0)
    others = [copy.deepcopy(w), torch.load(saved, weights_only=False)]
    w.codes.zero_(), w.scales.fill_(float("nan"))
    for other in others:
        assert torch.equal(ops.linear(x, other), want)


@torch.inference_mode()
def test_a_copied_model_runs_on_its_own_weights(ops):
    import copy
    from triattention_b200.models import int8_projections
    ids = torch.arange(40).cuda()[None]
    model = int8_projections(toy_llama(), ops)
    want = model(input_ids=ids, use_cache=False).logits
    other = copy.deepcopy(model)
    for layer in model.model.layers:
        layer.down.rows.codes.zero_()
    assert torch.equal(other(input_ids=ids, use_cache=False).logits, want)


# ---- subnormal numbers -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,outputs,width", [(1, 200, 512), (2, 640, 4096), (40, 200, 512), (300, 640, 300), (5000, 4096, 256)])
def test_linear_keeps_subnormal_numbers(ops, tokens, outputs, width, dtype):
    """IEEE arithmetic down to the smallest numbers of each type: products of powers of two, residuals and biases come out as they are."""
    least = torch.finfo(dtype).smallest_normal / 2 ** 4
    x, w = codes_rows(tokens, width, 130), codes_rows(outputs, width, 131)
    x.codes.zero_(), w.codes.fill_(1)
    residual, bias = (randn(*shape, seed=s, dtype=FP32).mul(least).to(dtype) for shape, s in (((tokens, outputs), 132), ((outputs,), 133)))
    assert bool(residual.any()) and float(residual.abs().max()) < torch.finfo(dtype).smallest_normal
    assert torch.equal(ops.linear(x, w, residual=residual, dtype=dtype), residual)
    assert torch.equal(ops.linear(x, w, bias=bias, dtype=dtype), bias.expand(tokens, outputs))
    x.codes[:, 0] = 3
    x.scales.fill_(2.0 ** -60), w.scales.fill_(least * 2.0 ** 60)        # (2^-60 each way: 3 * 2^60 * 2^-60 * least)
    assert torch.equal(ops.linear(x, w, dtype=dtype), torch.full((tokens, outputs), 3 * least, dtype=FP32, device="cuda").to(dtype))


# ---- the largest tensors, broadcast residuals --------------------------------------------------------------------------------

@pytest.mark.parametrize("width", (32768, 32765))
def test_rows_past_32_bits(ops, width):
    """2.3e9 elements, 4.6 GB an operand: the last rows are what they are alone."""
    rows = 70001
    x, u = (torch.empty(rows, width, dtype=BF16, device="cuda") for _ in range(2))
    for t, seed in ((x, 140), (u, 141)):
        t.copy_(randn(1, width, seed=seed).expand(rows, width))
        t[-3:] = randn(3, width, seed=seed + 2)
    w = (1 + 0.1 * randn(width, seed=144, dtype=FP32)).to(BF16)
    last = slice(rows - 3, rows)
    for call in (lambda p: ops.quantize_rows(x[p]), lambda p: ops.silu_mul(x[p], u[p]), lambda p: ops.rms_norm(x[p], w, 1e-6, residual=u[p])):
        got, want = call(slice(None)), call(last)
        if isinstance(got, tuple):
            assert torch.equal(got[1][last], want[1])
            got, want = got[0], want[0]
        assert torch.equal(got.codes[last], want.codes) and torch.equal(got.codes[1], got.codes[rows - 4])
        if width % 8 == 0:                      # (rows that lie alike)
            assert torch.equal(got.scales[last], want.scales)
        else:
            torch.testing.assert_close(got.scales[last], want.scales, rtol=46 * U, atol=0)
        part = Int8Rows(got.codes[last], got.scales[last])
        assert torch.equal(ops.dequantize(got)[last], ops.dequantize(part))
        del got, want, part


@pytest.mark.parametrize("tokens,outputs,width", [(40001, 65536, 48), (40001, 65533, 48)])
def test_linear_results_past_32_bits(ops, tokens, outputs, width):
    x, w = codes_rows(tokens, width, 150), codes_rows(outputs, width, 151)
    bias, residual = randn(outputs, seed=152), randn(1, outputs, seed=153).expand(tokens, outputs)
    got = ops.linear(x, w, bias=bias, residual=residual)
    for lo in (0, 32760, tokens - 5):
        part = slice(lo, lo + 5)
        assert torch.equal(got[part], ops.linear(Int8Rows(x.codes[part], x.scales[part]), w, bias=bias, residual=residual[part]))
    ops.module.check_device_error()


def test_linear_weights_past_32_bits(ops):
    outputs, width = 200003, 16384
    w = codes_rows(outputs, width, 154)
    last = Int8Rows(w.codes[-300:], w.scales[-300:])
    for tokens in (1, 7, 300):
        x = codes_rows(tokens, width, 155 + tokens)
        assert torch.equal(ops.linear(x, w)[:, -300:], ops.linear(x, last))
        check_linear(ops, x, last)


@pytest.mark.parametrize("tokens", (1, 3, 40, 300, 2500))
def test_linear_residuals_that_lie_otherwise(ops, tokens):
    """One row for all tokens, rows further apart, odd offsets, a transposed batch: the values count."""
    x, w = codes_rows(tokens, 260, 160), codes_rows(520, 260, 161)
    for residual in (randn(1, 520, seed=162).expand(tokens, 520), randn(tokens, 1100, seed=163)[:, 5:525], randn(tokens, 528, seed=164)[:, 8:]):
        assert torch.equal(ops.linear(x, w, residual=residual), ops.linear(x, w, residual=residual.contiguous()))
    if tokens % 4 == 0:
        cube = Int8Rows(x.codes.view(4, tokens // 4, 260), x.scales.view(4, tokens // 4))
        turned = randn(tokens // 4, 4, 520, seed=165).transpose(0, 1)
        assert torch.equal(ops.linear(cube, w, residual=turned).view(tokens, 520), ops.linear(x, w, residual=turned.reshape(tokens, 520)))
