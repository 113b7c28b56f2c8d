"""Row quantisation and the 8-bit linear against plain 64-bit arithmetic."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def ops():
    from pixal3d.cpp_b200 import ops as o
    return o


def L():
    from pixal3d.cpp_b200 import _lib
    return _lib


def quantised64(x):
    """(q, scale): the definition, on the CPU in 64 bits (a scale is an f32)."""
    x = x.double().cpu()
    scale = torch.clamp((x.abs().amax(1) / 127.0).float(), min=2.0 ** -126)
    return torch.round(x / scale.double()[:, None]).to(torch.int8), scale


def check_quantised(x):
    q, s = ops().quantize_rows(x)
    wq, ws = quantised64(x)
    assert torch.equal(s.cpu(), ws)
    assert torch.equal(q.cpu(), wq)
    return q, s


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k", [(1, 1), (1, 16), (3, 7), (5, 130), (33, 773), (2, 1024), (7, 1025), (9, 4096), (4, 8192), (3, 8200),
                                 (2, 20001), (300, 64)])
def test_quantize_rows_exact(dtype, m, k):
    g = torch.Generator(device="cuda").manual_seed(m * 1000 + k)
    x = torch.randn((m, k), device="cuda", generator=g) * torch.exp(3 * torch.randn((m, 1), device="cuda", generator=g))
    check_quantised(x.to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k", [8, 31, 129, 256, 257, 1000, 1024, 1031, 2048, 2060, 4099, 8192, 16400])
def test_quantize_rows_every_width(dtype, k):
    """Rows enough for the per-row thread counts of large calls, rows that
    start inside a 16-byte word among them."""
    g = torch.Generator(device="cuda").manual_seed(k)
    x = torch.randn((301, k), device="cuda", generator=g).to(dtype)
    check_quantised(x)
    wide = torch.randn((301, k + 3), device="cuda", generator=g).to(dtype)
    wide[:, 0] = math.nan  # beside the rows, in the words they begin in
    wide[:, k + 1:] = math.inf
    check_quantised(wide[:, 1:k + 1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad,off", [(1, 0), (3, 1), (8, 8), (27, 0), (16, 3)])
def test_quantize_rows_strided(dtype, pad, off):
    """Rows inside wider ones, at any alignment; q beside its columns stays as it was."""
    m, k = 37, 203
    x = torch.randn((m, k + pad + off), device="cuda").to(dtype)[:, off:off + k]
    out = torch.full((m, k + pad), 55, dtype=torch.int8, device="cuda")
    q, s = ops().quantize_rows(x, out=out[:, :k])
    wq, ws = quantised64(x)
    assert torch.equal(q.cpu(), wq) and torch.equal(s.cpu(), ws)
    assert bool((out[:, k:] == 55).all())


def test_quantize_rows_ties_and_borders():
    """Multiples of half a scale (exact ties among them), the neighbours of
    every border, halves of the largest value, subnormal and huge rows."""
    rows = []
    for amax in (127.0, 1.0, 0.3, 254.0, 3.0e38, 1e-30, 2.0 ** -126, 2.0 ** -133, 1.4e-45, 7 * 1.4e-45, 200 * 1.4e-45):
        a = np.float32(amax)
        s = np.maximum(np.float32(np.float64(a) / 127), np.float32(2.0 ** -126))
        border = (np.arange(-127, 127) + 0.5) * np.float64(s)
        v = border.astype(np.float32)
        v = np.concatenate([v, np.nextafter(v, np.float32(np.inf)), np.nextafter(v, np.float32(-np.inf)),
                            np.float32([a, -a, a / 2, -a / 2, a / 4, 0.0, -0.0])])
        rows.append(np.clip(v, -a, a))
    check_quantised(torch.from_numpy(np.stack(rows)).cuda())


def test_quantize_rows_zero_and_nonfinite_rows():
    for dtype in TYPES:
        x = torch.randn((6, 40), device="cuda").to(dtype)
        x[1] = 0
        x[2, 39] = math.inf
        x[3, 0] = -math.inf
        x[4, 17] = math.nan
        q, s = ops().quantize_rows(x)
        assert float(s[1]) == 2.0 ** -126 and not bool(q[1].any())
        for r in (2, 3, 4):
            assert math.isnan(float(s[r])) and not bool(q[r].any())
        wq, ws = quantised64(x[[0, 5]])
        assert torch.equal(q[[0, 5]].cpu(), wq) and torch.equal(s[[0, 5]].cpu(), ws)


def product64(x, xs, w, ws, bias, epi):
    """(y, size of the product's terms) in 64 bits."""
    y = x.double() @ w.double().t() * xs.double()[:, None] * ws.double()
    size = y.abs()
    if bias is not None:
        y = y + bias.double()
    pre = y
    if epi & L().EPI_GELU_TANH:
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    elif epi & L().EPI_SILU:
        y = y * torch.sigmoid(y)
    return y, size, pre


def check_linear(m, n, k, out_dtype, epi=0, bias=True, low=-127, high=127):
    g = torch.Generator(device="cuda").manual_seed(m + 31 * n + 7 * k)
    pitch = (k + 15) // 16 * 16
    # what follows the k columns is not part of the operands
    x = torch.randint(low, high + 1, (m, pitch), device="cuda", generator=g).to(torch.int8)[:, :k]
    w = torch.randint(low, high + 1, (n, pitch), device="cuda", generator=g).to(torch.int8)[:, :k]
    xs = torch.rand(m, device="cuda", generator=g) + 0.01
    ws = (torch.rand(n, device="cuda", generator=g) + 0.01) / (127 * 127 * math.sqrt(k) / 3)
    b = torch.randn(n, device="cuda", generator=g) if bias else None
    got = ops().linear_i8(x, xs, w, ws, b, out_dtype=out_dtype, epilogue=epi)
    y, size, pre = product64(x, xs, w, ws, b, epi)
    # f32: the sum and its two scalings round three times, the bias' addition once
    tol = 2.0 ** -24 * (3 * size + pre.abs()) * 1.01
    if epi:
        # activations: slope at most 1.13; in f32 the exponential's argument (at most 2.1 |y|^3 units)
        # and its 2^-22; the hardware tanh 2^-10.9 of half the value
        tol = 1.13 * tol + y.abs() * 2.0 ** -22 * (4 + 2 * pre.abs() + 0.2 * pre.abs() ** 3)
        if epi & L().EPI_GELU_TANH and out_dtype != torch.float32:
            tol = tol + 0.5 * pre.abs() * 2.0 ** -10.9
    if out_dtype != torch.float32:
        tol = tol + torch.finfo(out_dtype).eps / 2 * (y.abs() + tol) + 2.0 ** -25
    else:
        tol = tol + 2.0 ** -149
    err = (got.double() - y).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("out_dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 64, 64), (2, 6144, 1024), (3, 100, 33), (4, 130, 4096), (8, 257, 500), (9, 64, 128),
                                   (17, 48, 1000), (127, 129, 127), (128, 256, 128), (129, 257, 384), (200, 40, 16), (1029, 384, 320),
                                   (2050, 520, 96), (300, 1024, 2048), (4133, 96, 64)])
def test_linear_i8_shapes(m, n, k, out_dtype):
    check_linear(m, n, k, out_dtype)


@pytest.mark.parametrize("epi", [1, 2])
@pytest.mark.parametrize("out_dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(2, 96, 100), (300, 200, 160), (1500, 512, 96)])
def test_linear_i8_activations(m, n, k, out_dtype, epi):
    check_linear(m, n, k, out_dtype, epi)
    check_linear(m, n, k, out_dtype, epi, bias=False)


@pytest.mark.parametrize("m", [1, 130])
def test_linear_i8_sums_are_exact(m):
    """All operands -128 at the largest k: the sum is 2^31 - 2^14, and it is
    right to its last bit; an odd k leaves bytes behind that are not used."""
    n, k = 40, 131071
    x = torch.full((m, 131072), -128, dtype=torch.int8, device="cuda")[:, :k]
    w = torch.full((n, 131072), -128, dtype=torch.int8, device="cuda")[:, :k]
    one = torch.ones(max(m, n), device="cuda")
    got = ops().linear_i8(x, one[:m], w, one[:n], out_dtype=torch.float32)
    assert bool((got == float(np.float32(128 * 128 * k))).all())
    w[:, 1::2] = 127
    got = ops().linear_i8(x, one[:m], w, one[:n], out_dtype=torch.float32)
    assert bool((got == float(np.float32(128 * 128 * 65536 - 128 * 127 * 65535))).all())


@pytest.mark.parametrize("m,n,k", [(3, 70, 40), (700, 300, 200), (515, 256, 1024)])
@pytest.mark.parametrize("gated", [False, True])
def test_linear_i8_residual(m, n, k, gated):
    x = torch.randint(-127, 128, (m, (k + 15) // 16 * 16), device="cuda").to(torch.int8)[:, :k]
    w = torch.randint(-127, 128, (n, (k + 15) // 16 * 16), device="cuda").to(torch.int8)[:, :k]
    xs, ws = torch.rand(m, device="cuda"), torch.rand(n, device="cuda") / (5000 * math.sqrt(k))
    b = torch.randn(n, device="cuda")
    res = torch.randn((m, n + 12), device="cuda")
    off = torch.tensor([0, m // 3, m // 3, m], dtype=torch.int32, device="cuda")
    gate = torch.randn((3, n + 4), device="cuda")[:, :n] if gated else None
    out = res.clone()
    ops().linear_i8(x, xs, w, ws, b, out=out[:, :n], epilogue=L().EPI_RESIDUAL, gate=gate, batch_offsets=off if gated else None)
    y, size, pre = product64(x, xs, w, ws, b, 0)
    item = torch.bucketize(torch.arange(m, device="cuda"), off[1:].long(), right=True)
    gg = gate.double()[item] if gated else torch.ones((m, n), dtype=torch.float64, device="cuda")
    want = res[:, :n].double() + gg * y
    tol = 2.0 ** -24 * (gg.abs() * (3 * size + 2 * pre.abs()) + want.abs()) * 1.01
    assert bool(((out[:, :n].double() - want).abs() <= tol).all())
    assert torch.equal(out[:, n:], res[:, n:])


def test_linear_i8_output_view_keeps_the_rest():
    for m in (2, 200):
        x, w = torch.ones((m, 32), dtype=torch.int8, device="cuda"), torch.ones((50, 32), dtype=torch.int8, device="cuda")
        for t in TYPES:
            big = torch.full((m + 2, 75), 7.0, device="cuda").to(t)
            ops().linear_i8(x, torch.ones(m, device="cuda"), w, torch.ones(50, device="cuda"), out=big[1:m + 1, 5:55])
            want = torch.full((m + 2, 75), 7.0, device="cuda").to(t)
            want[1:m + 1, 5:55] = 32
            assert torch.equal(big, want)


def test_linear_i8_nan_scale_stays_in_its_row():
    for m in (4, 150):
        x, w = torch.ones((m, 64), dtype=torch.int8, device="cuda"), torch.ones((70, 64), dtype=torch.int8, device="cuda")
        xs = torch.ones(m, device="cuda")
        xs[2] = math.nan
        got = ops().linear_i8(x, xs, w, torch.ones(70, device="cuda"))
        assert bool(got[2].isnan().all()) and int(got.isnan().sum()) == 70


def test_quantised_linear_is_near_the_real_one():
    """Quantise, multiply: within the quantisation's half steps of x W^T."""
    m, n, k = 260, 192, 1000
    x, w = torch.randn((m, k), device="cuda"), torch.randn((n, k), device="cuda") / 30
    (xq, xs), (wq, ws) = ops().quantize_rows(x), ops().quantize_rows(w)
    got = ops().linear_i8(xq, xs, wq, ws, out_dtype=torch.float32).double()
    x, w = x.double(), w.double()
    tol = (xs.double()[:, None] / 2 * w.abs().sum(1) + x.abs().sum(1)[:, None] * ws.double() / 2 +
           k * xs.double()[:, None] * ws.double() / 4) * 1.0001
    assert bool(((got - x @ w.t()).abs() <= tol).all())


def test_refusals():
    o, l = ops(), L()
    x = torch.zeros((4, 32), dtype=torch.int8, device="cuda")
    w = torch.zeros((8, 32), dtype=torch.int8, device="cuda")
    a, b = torch.ones(4, device="cuda"), torch.ones(8, device="cuda")
    f = torch.zeros((4, 32), device="cuda")
    for bad in (lambda: o.quantize_rows(f.t()[:, ::2]), lambda: o.quantize_rows(f, out=x[:3]), lambda: o.quantize_rows(f, scale=b),
                lambda: o.quantize_rows(f[:, :0]),
                lambda: o.quantize_rows(f.cpu()), lambda: o.quantize_rows(f, out=x.float()),
                lambda: o.linear_i8(x, a, w[:, :16], b), lambda: o.linear_i8(x, b, w, b), lambda: o.linear_i8(x, a, w, b, a),
                lambda: o.linear_i8(x, a, w.cpu(), b), lambda: o.linear_i8(x.float(), a, w, b),
                lambda: o.linear_i8(x, a, w, b, epilogue=l.EPI_RESIDUAL), lambda: o.linear_i8(x, a, w, b, out=f),
                lambda: o.linear_i8(x, a.double(), w, b)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        o.quantize_rows(f.double())
    odd = torch.zeros((4, 40), dtype=torch.int8, device="cuda")
    out = torch.zeros((4, 8), device="cuda")
    k = 131072
    for bad, status in ((lambda: o.linear_i8(odd[:, :32], a, w, b), l.P3D_ERR_INVALID),           # pitch 40
                        (lambda: o.linear_i8(odd.view(5, 32)[:4, :], a, odd.view(-1)[8:136].view(4, 32), a), l.P3D_ERR_INVALID),
                        (lambda: o.linear_i8(x, a, w, b, epilogue=3), l.P3D_ERR_INVALID),          # two activations
                        (lambda: o.linear_i8(x, a, w, b, epilogue=64), l.P3D_ERR_INVALID),
                        (lambda: o.linear_i8(x, a, w, b, out=out.half(), epilogue=l.EPI_RESIDUAL), l.P3D_ERR_INVALID),
                        (lambda: o.linear_i8(torch.zeros((1, k), dtype=torch.int8, device="cuda"), a[:1],
                                             torch.zeros((1, k), dtype=torch.int8, device="cuda"), a[:1]), l.P3D_ERR_UNSUPPORTED)):
        with pytest.raises(l.P3DError) as e:
            bad()
        assert e.value.status == status
    q, s = o.quantize_rows(f[:0])
    assert q.shape == (0, 32) and s.shape == (0,)
    assert o.linear_i8(x[:0], a[:0], w, b).shape == (0, 8)


@pytest.mark.parametrize("out_dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(2, 900, 64), (5, 5000, 40), (400, 700, 100), (1300, 1024, 96)])
def test_linear_i8_gelu_is_right_to_a_step_everywhere(m, n, k, out_dtype):
    """GELU between -10 and 4 against its own size: its values left of -2 are small,
    and a small one's sign and size are as good as a large one's."""
    g = torch.Generator(device="cuda").manual_seed(n)
    pitch = (k + 15) // 16 * 16
    x = torch.randint(-20, 21, (m, pitch), device="cuda", generator=g).to(torch.int8)[:, :k]
    w = torch.randint(-20, 21, (n, pitch), device="cuda", generator=g).to(torch.int8)[:, :k]
    xs, ws = torch.rand(m, device="cuda", generator=g) + 0.5, torch.full((n,), 1.0 / (1500 * math.sqrt(k)), device="cuda")
    b = torch.linspace(-10, 4, n, device="cuda")
    got = ops().linear_i8(x, xs, w, ws, b, out_dtype=out_dtype, epilogue=L().EPI_GELU_TANH)
    y = x.double() @ w.double().t() * xs.double()[:, None] * ws.double()
    size, c = y.abs(), math.sqrt(2 / math.pi)
    p = (y + b.double()).requires_grad_()
    z = 2 * c * (p + 0.044715 * p ** 3)
    want = p * torch.sigmoid(z)
    slope = torch.autograd.grad(want.sum(), p)[0].abs()
    p, z, want = p.detach(), z.detach(), want.detach()
    # the argument: three roundings of the product and one of the sum, carried by the slope (and its
    # change over that little distance: below 2 times its square).  The form x / (1 + exp(-z)): z is off
    # by five roundings of itself (2^-24 each) of which exp makes |z| times as much, the exponential's 2^-22 and its
    # own argument's rounding, the division's 2^-22; denominators past 2^126 count as infinite
    dp = 2.0 ** -24 * (3 * size + p.abs()) * 1.01
    tol = slope * dp + 2 * dp ** 2 + want.abs() * 2.0 ** -22 * (4 + 2 * z.abs()) + p.abs() * 2.0 ** -125
    u = torch.finfo(out_dtype).eps / 2 if out_dtype != torch.float32 else 0.0
    tol = tol + u * (want.abs() + tol) + (2.0 ** -25 if out_dtype == torch.float16 else 0.0)
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
