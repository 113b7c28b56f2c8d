"""Rotary positions against plain 64-bit arithmetic."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def ops():
    from pixal3d.cpp_b200 import ops as o
    return o


def turned64(x, freqs, heads, dim, positions, layout, amplitude):
    n, half = x.shape[0], freqs.shape[0]
    y = x.double().reshape(n, heads, dim).clone()
    at = torch.arange(half, device=x.device)
    a, b = (at, at + half) if layout == "half" else (2 * at, 2 * at + 1)
    t = (positions.double()[:, None] * freqs)[:, None, :]
    u, w = y[..., a].clone(), y[..., b].clone()
    y[..., a] = amplitude * (u * torch.cos(t) - w * torch.sin(t))
    y[..., b] = amplitude * (u * torch.sin(t) + w * torch.cos(t))
    size = torch.zeros_like(y)
    size[..., a] = size[..., b] = u.abs() + w.abs()
    return y.reshape(x.shape), size.reshape(x.shape)


def check(got, x, freqs, heads, dim, positions, layout, amplitude=1.0):
    y, size = turned64(x, freqs, heads, dim, positions, layout, amplitude)
    # the angle: 2^-25 turns from its rounding to f32 and 2^-53 of itself, twice; sine and cosine 2 ulp;
    # amplitude, products and their sum round once each (2^-24)
    angle = 2 * math.pi * 2.0 ** -25 + 2.0 ** -51 * float((positions.abs().max() * freqs.abs().max()).item() if len(positions) else 0)
    tol = amplitude * size * (angle + 2.0 ** -22 + 4 * 2.0 ** -24)
    tol = tol + torch.finfo(x.dtype).eps / 2 * (y.abs() + tol) + (2.0 ** -25 if x.dtype == torch.float16 else 0.0)
    err = (got.double() - y).abs()
    assert bool((err <= tol).all()), float((err / tol.clamp_min(1e-30)).max())


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,heads,dim,rot", [(1, 1, 2, 2), (1, 40, 128, 128), (3, 2, 64, 48), (5, 3, 64, 64), (17, 1, 80, 30), (100, 5, 96, 64),
                                             (7, 2, 512, 512), (130, 12, 64, 32), (2, 7, 9, 4), (1000, 3, 32, 16)])
def test_rotary(n, heads, dim, rot, dtype, layout):
    o = ops()
    x = torch.randn((n, heads * dim), device="cuda").to(dtype)
    freqs, amp = o.rotary_frequencies(rot)
    assert amp == 1.0
    pos = torch.randint(-5000, 1 << 20, (n,), device="cuda", dtype=torch.int32)
    got = o.rotary(x, freqs, heads, dim, pos, layout=layout)
    check(got, x, freqs, heads, dim, pos, layout)
    rest = got.reshape(n, heads, dim)[..., rot:], x.reshape(n, heads, dim)[..., rot:]
    assert torch.equal(*rest)  # bits
    # the same in place
    y = x.clone()
    assert o.rotary(y, freqs, heads, dim, pos, layout=layout, out=y) is y
    assert torch.equal(y, got)


def test_rotary_default_positions_and_far_ends():
    o = ops()
    freqs, _ = o.rotary_frequencies(64, base=500000.0)
    for off in (0, 70000, 2 ** 31 - 20):
        x = torch.randn((19, 128), device="cuda")
        got = o.rotary(x, freqs, 2, 64, position_offset=off)
        check(got, x, freqs, 2, 64, torch.arange(off, off + 19, device="cuda"), "half")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad,off", [(64, 0), (8, 8), (3, 0), (5, 1)])
def test_rotary_views(dtype, pad, off):
    """Heads inside wider rows, at any alignment; what lies beside them stays."""
    o = ops()
    n, heads, dim = 29, 3, 32
    width = heads * dim
    freqs, _ = o.rotary_frequencies(dim)
    pos = torch.arange(29, device="cuda", dtype=torch.int32) * 37
    wide = torch.randn((n, width + pad + off), device="cuda").to(dtype)
    before = wide.clone()
    x = wide[:, off:off + width]
    for layout in ("half", "interleaved"):
        check(o.rotary(x, freqs, heads, dim, pos, layout=layout), x, freqs, heads, dim, pos, layout)
    o.rotary(x, freqs, heads, dim, pos, out=x)
    check(x, before[:, off:off + width], freqs, heads, dim, pos, "half")
    assert torch.equal(wide[:, :off], before[:, :off]) and torch.equal(wide[:, off + width:], before[:, off + width:])


def test_rotary_stretched_frequencies():
    """Interpolation by parts: fast pairs as before, slow ones slowed by the
    factor, and the turned rows follow the returned frequencies."""
    o = ops()
    plain, _ = o.rotary_frequencies(128)
    freqs, amp = o.rotary_frequencies(128, stretch=16.0, original_length=4096)
    assert abs(amp - (0.1 * math.log(16.0) + 1.0)) < 1e-15
    turns = 4096 * plain / (2 * math.pi)
    assert torch.equal(freqs[turns > 32], plain[turns > 32])
    assert torch.allclose(freqs[turns < 1], plain[turns < 1] / 16, rtol=1e-14, atol=0)
    mixed = (turns > 1) & (turns < 32)
    assert bool(mixed.any()) and bool(((freqs < plain) & (freqs > plain / 16))[mixed].all())
    x = torch.randn((50, 256), device="cuda").half()
    pos = torch.randint(0, 65536, (50,), device="cuda", dtype=torch.int32)
    check(o.rotary(x, freqs, 2, 128, pos, amplitude=amp), x, freqs, 2, 128, pos, "half", amp)


def test_rotary_keeps_scores_of_equal_distance():
    """The score of a turned query and key depends on their distance alone."""
    o = ops()
    freqs, _ = o.rotary_frequencies(64)
    q, k = (torch.randn((1, 64), device="cuda").expand(300, 64).contiguous() for _ in range(2))
    near, far = torch.arange(300, device="cuda", dtype=torch.int32), torch.arange(300, device="cuda", dtype=torch.int32) + 900001
    a = (o.rotary(q, freqs, 1, 64, near).double() * o.rotary(k, freqs, 1, 64, near + 12).double()).sum(1)
    b = (o.rotary(q, freqs, 1, 64, far).double() * o.rotary(k, freqs, 1, 64, far + 12).double()).sum(1)
    # two turned rows, each off by 6e-7 of its pairs' sizes (the bound above)
    tol = 2 * 6e-7 * 2 * float((q[0].norm() * k[0].norm()).double()) * 2
    assert float((a - b).abs().max()) <= tol and float((a - a[0]).abs().max()) <= tol


def test_rotary_nonfinite_values_stay_in_their_pair():
    o = ops()
    freqs, _ = o.rotary_frequencies(16)
    x = torch.randn((4, 64), device="cuda")
    x[1, 3] = math.nan
    x[2, 40] = math.inf
    got = o.rotary(x, freqs, 2, 32)
    bad = ~got.isfinite()
    want = torch.zeros_like(bad)
    want[1, 3] = want[1, 11] = want[2, 40] = want[2, 32] = True
    assert torch.equal(bad, want)


def test_rotary_refusals():
    from pixal3d.cpp_b200 import _lib as l
    o = ops()
    x = torch.zeros((4, 64), device="cuda")
    f, _ = o.rotary_frequencies(32)
    for bad in (lambda: o.rotary(x, f, 2, 16), lambda: o.rotary(x, f.float(), 2, 32), lambda: o.rotary(x, f, 2, 32, layout="other"),
                lambda: o.rotary(x, f, 2, 32, torch.zeros(3, dtype=torch.int32, device="cuda")),
                lambda: o.rotary(x, f, 2, 32, torch.zeros(4, device="cuda")), lambda: o.rotary(x, f, 2, 32, out=x.half()),
                lambda: o.rotary(x, f.cpu(), 2, 32), lambda: o.rotary(x.cpu(), f, 2, 32), lambda: o.rotary(x.t().contiguous().t(), f, 2, 32),
                lambda: o.rotary_frequencies(7), lambda: o.rotary_frequencies(8, stretch=0.5)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: o.rotary(x, o.rotary_frequencies(66)[0], 2, 32), lambda: o.rotary(torch.zeros((2, 600), device="cuda"), f, 1, 600),
                lambda: o.rotary(x[:, :32], f, 1, 32, out=x[:, 16:48])):  # overlapping columns
        with pytest.raises(l.P3DError) as e:
            bad()
        assert e.value.status == l.P3D_ERR_INVALID
    # beside one another in the same rows is no overlap
    o.rotary(x[:, :32], f, 1, 32, out=x[:, 32:])
    assert o.rotary(x[:0], f, 2, 32).shape == (0, 64)
