"""Masked attention against plain 64-bit arithmetic."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def ops():
    from pixal3d.cpp_b200 import ops as o
    return o


def cu(lens):
    return torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device="cuda")


def attention64(q, k, v, lens, heads, kv_heads, scale, causal=False, prefix=None, doc_q=None, doc_k=None, slopes=None, softcap=0.0):
    """(out, tolerance) of every query row, row by row of the definition."""
    d = q.shape[1] // heads
    u = torch.finfo(q.dtype).eps / 2
    out, tol = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    q0 = k0 = 0
    for s, (lq, lk) in enumerate(lens):
        at_q, at_k = torch.arange(lq, device="cuda") + lk - lq, torch.arange(lk, device="cuda")
        seen = torch.ones((lq, lk), dtype=torch.bool, device="cuda")
        if causal:
            seen &= at_k[None, :] <= at_q[:, None]
        if doc_q is not None:
            seen &= doc_q[q0:q0 + lq, None] == doc_k[None, k0:k0 + lk]
        if prefix is not None:
            seen |= (at_k < int(prefix[s]))[None, :]
        for h in range(heads if lq and lk else 0):
            hk = h // (heads // kv_heads)
            qq = q[q0:q0 + lq, h * d:(h + 1) * d].double()
            kk, vv = (t[k0:k0 + lk, hk * d:(hk + 1) * d].double() for t in (k, v))
            x = qq @ kk.t() * scale
            # scores: f32 products and sums (2^-23 of the terms each way), the cap's 2^-21
            dx = (qq.abs() @ kk.abs().t()) * scale * 2.0 ** -22 + softcap * 2.0 ** -21
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            if slopes is not None:
                apart = (at_q[:, None] - at_k[None, :]).abs()
                x = x - slopes[h].double() * apart
                dx = dx + slopes[h].double() * apart * 2.0 ** -22
            x = x.masked_fill(~seen, -math.inf)
            top = x.amax(1, keepdim=True).clamp_min(-1e300)
            w = torch.exp(x - top)
            l = w.sum(1, keepdim=True)
            o = w @ vv / l.clamp_min(1e-300)
            out[q0:q0 + lq, h * d:(h + 1) * d] = o
            # each weight is off by 2 dx (its score and the maximum's), the exponential's 2^-21 with the
            # distance's rounding, and its rounding to 16 bits (u); each moves the mean by at most
            # weight * (|v| + |o|).  f16 weights below 2^-14 are off by 2^-25 instead.  The f32 sums of
            # lk terms add lk 2^-24 of their size, the result its rounding.
            rel = w * (2 * dx + 2.0 ** -20 + (top - x).clamp(0, 200).nan_to_num(0.0) * 2.0 ** -22 + u * 1.01)
            t = (rel @ vv.abs() + rel.sum(1, keepdim=True) * o.abs()) / l.clamp_min(1e-300)
            mean = w @ vv.abs() / l.clamp_min(1e-300) + o.abs()
            t = t + mean * (lk * 2.0 ** -24 + 2.0 ** -21)
            if q.dtype == HF:
                t = t + seen.sum(1, keepdim=True) * 2.0 ** -25 * (vv.abs().amax() + o.abs())
            tol[q0:q0 + lq, h * d:(h + 1) * d] = t + u * (o.abs() + t) + 2.0 ** -25
        q0, k0 = q0 + lq, k0 + lk
    return out, tol


def run(lens, heads, kv_heads, d, dtype, seed=0, sharp=2.0, poison=None, spare=0, **rules):
    o = ops()
    g = torch.Generator(device="cuda").manual_seed(seed)
    nq, nk = sum(a for a, _ in lens), sum(b for _, b in lens)
    q = (torch.randn((nq + spare, heads * d), device="cuda", generator=g) * sharp).to(dtype)
    k = torch.randn((nk + spare, kv_heads * d), device="cuda", generator=g).to(dtype)
    v = torch.randn((nk + spare, kv_heads * d), device="cuda", generator=g).to(dtype)
    scale = 1.0 / math.sqrt(d)
    want, tol = attention64(q, k, v, lens, heads, kv_heads, scale, **rules)
    if poison is not None:
        poison(q, k, v)
    out = torch.full((nq + spare, heads * d), 3.0, device="cuda").to(dtype)
    got = o.masked_attention(q, k, v, cu([a for a, _ in lens]), cu([b for _, b in lens]), max(a for a, _ in lens),
                             max(b for _, b in lens), heads, scale, kv_heads=kv_heads, out=out, **rules)
    o.ctx().sync_check()
    err = (got.double() - want).abs()[:nq]
    assert bool((err <= tol[:nq]).all()), (float((err / tol[:nq]).max()), int((~(err <= tol[:nq])).sum()))
    assert bool((got[nq:] == 3.0).all())
    return got


LENGTHS = [
    [(1, 1)], [(1, 0), (2, 3)], [(1, 17), (1, 300), (1, 64)], [(1, 5000)], [(3, 1000), (1, 15), (5, 2049)], [(64, 64)], [(65, 129)],
    [(128, 128), (1, 200), (0, 5), (130, 130)], [(200, 77)], [(77, 200)], [(513, 513), (300, 300)], [(1100, 1100)],
]


@pytest.mark.parametrize("d,dtype", [(64, HF), (64, BF), (128, HF), (128, BF)])
@pytest.mark.parametrize("lens", LENGTHS)
def test_plain_and_causal(lens, d, dtype):
    run(lens, 4, 4, d, dtype)
    run(lens, 6, 2, d, dtype, causal=True, spare=3)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 1), (20, 1), (40, 2), (12, 4), (34, 2)])
def test_shared_heads(heads, kv_heads):
    run([(1, 700), (1, 65)], heads, kv_heads, 64, BF)
    run([(150, 150)], heads, kv_heads, 128, HF, causal=True)


@pytest.mark.parametrize("softcap", [0.0, 5.0, 50.0])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("lens", [[(1, 900)], [(2, 40), (1, 513)], [(333, 333)], [(140, 400)]])
def test_score_rules(lens, bias, softcap):
    slopes = torch.tensor([0.5, 0.0625, 0.0, 2.0], device="cuda") if bias else None
    run(lens, 4, 2, 64, HF, softcap=softcap, slopes=slopes, sharp=6.0)
    run(lens, 4, 2, 128, BF, softcap=softcap, slopes=slopes, sharp=6.0, causal=True)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d,dtype", [(64, HF), (128, BF)])
def test_prefix(d, dtype, causal):
    prefix = torch.tensor([0, 30, 1000, -4, 129], dtype=torch.int32, device="cuda")
    lens = [(40, 40), (100, 100), (70, 200), (65, 65), (300, 300)]
    run(lens, 4, 2, d, dtype, causal=causal, prefix=prefix)
    run([(1, b) for _, b in lens], 4, 2, d, dtype, causal=causal, prefix=prefix)


def documents(lens, cuts):
    """Sorted document numbers for keys, the queries' being those at their positions."""
    dk = [torch.bucketize(torch.arange(b), torch.tensor(cuts), right=True).int() for _, b in lens]
    return torch.cat([x[b - a:] if a <= b else torch.cat([x.new_full((a - b,), -9), x]) for x, (a, b) in zip(dk, lens)]).cuda(), torch.cat(dk).cuda()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d,dtype", [(64, HF), (128, BF)])
@pytest.mark.parametrize("lens", [[(300, 300), (90, 90)], [(700, 700)], [(100, 350)], [(1, 400), (2, 100)], [(30, 12)]])
def test_documents(lens, d, dtype, causal):
    dq, dk = documents(lens, [1, 70, 128, 200, 201, 333])
    run(lens, 4, 2, d, dtype, causal=causal, doc_q=dq, doc_k=dk)
    prefix = torch.full((len(lens),), 20, dtype=torch.int32, device="cuda")
    run(lens, 4, 2, d, dtype, causal=causal, doc_q=dq, doc_k=dk, prefix=prefix, slopes=torch.rand(4, device="cuda"))


def test_documents_in_any_order():
    """Documents need not be runs, and a query's may have no key: zeros then."""
    g = torch.Generator(device="cuda").manual_seed(5)
    for lens in ([(400, 400)], [(1, 333), (1, 5)], [(130, 700)]):
        nq, nk = sum(a for a, _ in lens), sum(b for _, b in lens)
        dq = torch.randint(-3, 5, (nq,), device="cuda", generator=g).int()
        dk = torch.randint(-2, 4, (nk,), device="cuda", generator=g).int()
        got = run(lens, 4, 4, 64, BF, doc_q=dq, doc_k=dk)
        for i in (dq == 4).nonzero().flatten().tolist() + (dq == -3).nonzero().flatten().tolist():
            assert not bool(got[i].any())
        none = torch.full_like(dq, 77)
        assert not bool(run(lens, 4, 4, 64, BF, doc_q=none, doc_k=dk).any())


def test_more_queries_than_keys_under_causal_mask():
    """The first queries stand before the first key and see nothing."""
    for lens in ([(50, 20)], [(300, 100), (4, 1), (2, 0)]):
        got = run(lens, 4, 2, 64, HF, causal=True)
        assert not bool(got[:lens[0][0] - lens[0][1]].any())


@pytest.mark.parametrize("d,dtype", [(64, HF), (128, BF)])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_hidden_values_do_not_matter(d, dtype, value):
    """NaN and infinities in keys and values that no query of a tile sees, that
    only some of its queries see not, and in rows behind the last sequence."""
    lens = [(1, 500), (200, 200), (3, 90)]
    dq, dk = documents(lens, [40, 130])

    def behind(q, k, v):
        for t in (q, k, v):
            t[-70:] = value
    run(lens, 4, 2, d, dtype, spare=70, poison=behind)

    def pad_document(q, k, v):
        bad = dk == 99
        k[:len(dk)][bad] = value
        v[:len(dk)][bad] = value
    dk99, dq99 = dk.clone(), dq.clone()
    dk99[::7] = 99
    run(lens, 4, 2, d, dtype, doc_q=dq99, doc_k=dk99, poison=lambda q, k, v: (k[dk99 == 99].fill_(value), k.__setitem__(dk99 == 99, value), v.__setitem__(dk99 == 99, value)))


@pytest.mark.parametrize("d,dtype", [(64, HF), (128, BF)])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_future_values_do_not_reach_earlier_queries(d, dtype, value):
    """A non-finite value row reaches the queries that see it, and no other."""
    n, at = 300, 170
    got = {}
    for bad in (False, True):
        g = torch.Generator(device="cuda").manual_seed(3)
        q, k, v = (torch.randn((n, 2 * d), device="cuda", generator=g).to(dtype) for _ in range(3))
        if bad:
            v[at, 3] = value
            v[at, d + 5] = -value
        got[bad] = ops().masked_attention(q, k, v, cu([n]), cu([n]), n, n, 2, 0.1, causal=True)
    want = got[False].clone()
    want[at:, 3] = value
    want[at:, d + 5] = -value
    assert torch.equal(got[True].nan_to_num(7.5, 1e4, -1e4), want.nan_to_num(7.5, 1e4, -1e4))


def test_views_of_a_packed_projection():
    """q, k, v as columns of one projection, out as columns of a wider row."""
    heads, kv, d, n = 6, 2, 64, 260
    qkv = torch.randn((n, (heads + 2 * kv) * d + 8), device="cuda").half()
    q, k, v = qkv[:, :heads * d], qkv[:, heads * d:(heads + kv) * d], qkv[:, (heads + kv) * d:(heads + 2 * kv) * d]
    wide = torch.full((n, heads * d + 16), 9.0, device="cuda").half()
    o = ops()
    for lens in ([(n, n)], [(1, n - 4), (1, 4)]):
        nq = sum(a for a, _ in lens)
        got = o.masked_attention(q[:nq], k, v, cu([a for a, _ in lens]), cu([b for _, b in lens]), nq, n, heads, 0.2, kv_heads=kv,
                                 causal=True, out=wide[:nq, 8:8 + heads * d])
        same = o.masked_attention(q[:nq].contiguous(), k.contiguous(), v.contiguous(), cu([a for a, _ in lens]),
                                  cu([b for _, b in lens]), nq, n, heads, 0.2, kv_heads=kv, causal=True)
        assert torch.equal(got, same)
        assert bool((wide[:, :8] == 9).all()) and bool((wide[:, 8 + heads * d:] == 9).all())


def test_scores_that_differ_widely():
    """A maximum that rises late and by much, and keys whose weight vanishes."""
    d, n = 64, 900
    for lq in (1, n):
        q = torch.ones((lq, d), device="cuda").half()
        k = torch.zeros((n, d), device="cuda").half()
        k[:, 0] = torch.linspace(-300, 300, n, device="cuda").half()
        v = torch.randn((n, d), device="cuda").half()
        want, tol = attention64(q, k, v, [(lq, n)], 1, 1, 1.0)
        got = ops().masked_attention(q, k, v, cu([lq]), cu([n]), lq, n, 1, 1.0)
        assert bool(((got.double() - want).abs() <= tol).all())


def test_matches_the_unmasked_operator():
    """No rule set: the same function as varlen_attention (its 16-bit exponents
    are coarser: 2^-9 of an exponent up to 16, 1 % of a weight)."""
    o = ops()
    q, k, v = (torch.randn((500, 256), device="cuda").half() for _ in range(3))
    c = cu([200, 300])
    a = o.masked_attention(q, k, v, c, c, 300, 300, 4, 0.125)
    b = o.varlen_attention(q, k, v, c, c, 300, 4, 0.125)
    assert float((a.float() - b.float()).abs().max()) <= 0.02


def test_calls_on_other_streams_and_in_graphs():
    o = ops()
    for lens in ([(1, 3000), (1, 2000)], [(400, 400), (100, 100)]):
        nq, nk = sum(a for a, _ in lens), sum(b for _, b in lens)
        q, k, v = (torch.randn((n, 256), device="cuda").half() for n in (nq, nk, nk))
        cq, ck = cu([a for a, _ in lens]), cu([b for _, b in lens])
        dq, dk = documents(lens, [10, 300])
        args = (cq, ck, max(a for a, _ in lens), max(b for _, b in lens), 4, 0.125)
        rules = dict(causal=True, doc_q=dq, doc_k=dk)
        want = o.masked_attention(q, k, v, *args, **rules)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            other = o.masked_attention(q, k, v, *args, **rules)
        side.synchronize()
        assert torch.equal(other, want)
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = o.masked_attention(q, k, v, *args, **rules)
            graphs.append((graph, out))
        q2 = torch.randn_like(q)
        want2 = o.masked_attention(q2, k, v, *args, **rules)
        q.copy_(q2)
        for graph, out in graphs + graphs:
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want2)


def test_offsets_out_of_range_are_clamped():
    """Offsets are device data: wrong ones read nothing outside the buffers."""
    o = ops()
    q, k, v = (torch.randn((64, 128), device="cuda").half() for _ in range(3))
    out = torch.zeros_like(q)
    bad = torch.tensor([-50, 90000, 32, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    o.masked_attention(q, k, v, bad, bad, 64, 64, 2, 0.1, out=out)
    o.masked_attention(q[:2], k, v, bad[:2], bad[:2], 2, 64, 2, 0.1, out=out[:2])
    o.ctx().sync_check()


def test_refusals():
    from pixal3d.cpp_b200 import _lib as l
    o = ops()
    q = torch.zeros((4, 128), device="cuda").half()
    c = cu([4])
    for bad in (lambda: o.masked_attention(q, q, q.bfloat16(), c, c, 4, 4, 2, 1.0), lambda: o.masked_attention(q.float(), q, q, c, c, 4, 4, 2, 1.0),
                lambda: o.masked_attention(q, q, q, c, c, 4, 4, 3, 1.0), lambda: o.masked_attention(q, q, q, c, c, 4, 4, 2, 1.0, kv_heads=1),
                lambda: o.masked_attention(q, q, q, c, c.long(), 4, 4, 2, 1.0), lambda: o.masked_attention(q, q, q, c, c[:1], 4, 4, 2, 1.0),
                lambda: o.masked_attention(q, q, q.cpu(), c, c, 4, 4, 2, 1.0),
                lambda: o.masked_attention(q, q, q, c, c, 4, 4, 2, 1.0, doc_q=torch.zeros(4, dtype=torch.int32, device="cuda")),
                lambda: o.masked_attention(q, q, q, c, c, 4, 4, 2, 1.0, prefix=c), lambda: o.masked_attention(q, q, q, c, c, 4, 4, 2, 1.0, slopes=c.float()[:1]),
                lambda: o.masked_attention(q, q, q, c, c, 4, 4, 2, 1.0, out=q[:3])):
        with pytest.raises(ValueError):
            bad()
    wide = torch.zeros((4, 132), device="cuda").half()
    for bad, status in ((lambda: o.masked_attention(q, q, q, c, c, 4, 4, 4, 1.0), l.P3D_ERR_UNSUPPORTED),          # head_dim 32
                        (lambda: o.masked_attention(q, q, q, c, c, 4, 4, 2, 0.0), l.P3D_ERR_INVALID),
                        (lambda: o.masked_attention(q, q, q, c, c, 4, 4, 2, math.inf), l.P3D_ERR_INVALID),
                        (lambda: o.masked_attention(q, q, q, c, c, 4, 4, 2, 1.0, softcap=-1.0), l.P3D_ERR_INVALID),
                        (lambda: o.masked_attention(q, q, q, c, c, 4, 4, 2, 1.0, softcap=math.nan), l.P3D_ERR_INVALID),
                        (lambda: o.masked_attention(wide[:, :128], q, q, c, c, 4, 4, 2, 1.0), l.P3D_ERR_INVALID),   # 264-byte rows
                        (lambda: o.masked_attention(q, wide.view(-1)[4:516].view(4, 128), q, c, c, 4, 4, 2, 1.0), l.P3D_ERR_INVALID)):
        with pytest.raises(l.P3DError) as e:
            bad()
        assert e.value.status == status
    assert o.masked_attention(q[:0], q, q, c, c, 4, 4, 2, 1.0).shape == (0, 128)


LONG = [[(1, 3000)], [(1, 700), (1, 0), (2, 5000), (8, 513)], [(5, 1200), (0, 900), (3, 2)], [(2, 4100)] * 5, [(1, 600)] * 40, [(8, 2000), (8, 5)]]


@pytest.mark.parametrize("d,dtype", [(64, HF), (128, BF)])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (8, 2), (12, 1), (40, 1)])
@pytest.mark.parametrize("lens", LONG)
def test_few_queries_over_long_keys(lens, heads, kv_heads, d, dtype):
    """Up to 8 queries a sequence over keys that are shared out over the GPU:
    items of 8 to 32 rows and more, whole and cut ones."""
    run(lens, heads, kv_heads, d, dtype, causal=True, spare=5)
    run(lens, heads, kv_heads, d, dtype, slopes=torch.rand(heads, device="cuda") * 0.01, softcap=20.0)


@pytest.mark.parametrize("d,dtype", [(64, HF), (128, BF)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("value", [0.0, math.nan, math.inf])
def test_few_queries_over_long_keys_masked(d, dtype, causal, value):
    lens = [(1, 900), (4, 1500), (8, 640), (3, 1)]
    g = torch.Generator(device="cuda").manual_seed(11)
    nq, nk = sum(a for a, _ in lens), sum(b for _, b in lens)
    dk = torch.randint(0, 3, (nk,), device="cuda", generator=g).int()
    dk[::5] = 99  # nobody's
    dq = torch.randint(0, 4, (nq,), device="cuda", generator=g).int()  # 3 has no key
    prefix = torch.tensor([0, 100, 640, 1], dtype=torch.int32, device="cuda")

    def hide(hidden):
        def poison(q, k, v):
            if value != 0.0:
                k[hidden.nonzero().flatten()] = value
                v[hidden.nonzero().flatten()] = value
        return poison
    run(lens, 8, 2, d, dtype, causal=causal, doc_q=dq, doc_k=dk, poison=hide(dk == 99))
    at = torch.cat([torch.arange(b) for _, b in lens]).cuda()
    shared = at < torch.cat([prefix[i].repeat(b) for i, (_, b) in enumerate(lens)])
    run(lens, 8, 2, d, dtype, causal=causal, doc_q=dq, doc_k=dk, prefix=prefix, slopes=torch.rand(8, device="cuda") * 0.01,
        poison=hide((dk == 99) & ~shared))


@pytest.mark.parametrize("d,dtype", [(64, HF), (128, BF)])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_later_keys_of_few_queries(d, dtype, value):
    """Of the last keys some queries see a non-finite value and others do not."""
    n, lq = 1000, 6
    got = {}
    for bad in (False, True):
        g = torch.Generator(device="cuda").manual_seed(3)
        q = torch.randn((lq, 4 * d), device="cuda", generator=g).to(dtype)
        k, v = (torch.randn((n, 2 * d), device="cuda", generator=g).to(dtype) for _ in range(2))
        if bad:
            v[n - 3, 3] = value  # seen from query 3 on
            v[n - 2, d + d - 1] = -value
        got[bad] = ops().masked_attention(q, k, v, cu([lq]), cu([n]), lq, n, 4, 0.1, kv_heads=2, causal=True)
    want = got[False].clone()
    want[3:, 3] = want[3:, d + 3] = value
    want[4:, 3 * d - 1] = want[4:, 4 * d - 1] = -value
    ok = want.isfinite()
    assert torch.equal(got[True].isfinite(), ok) and torch.equal(got[True].isnan(), want.isnan())
    assert torch.equal(got[True][~ok].nan_to_num(7.5, 1e4, -1e4), want[~ok].nan_to_num(7.5, 1e4, -1e4))
    assert torch.equal(got[True][ok], want[ok])


@pytest.mark.parametrize("d,dtype", [(64, HF), (128, BF)])
@pytest.mark.parametrize("lens", [[(9, 1100)], [(64, 5000), (30, 700)], [(200, 3000)], [(130, 1024), (0, 3), (1, 2500)]])
def test_many_queries_over_long_keys(lens, d, dtype):
    """Few tiles over long keys: the key blocks are split and joined."""
    run(lens, 4, 2, d, dtype, causal=True, spare=4)
    run(lens, 4, 2, d, dtype, softcap=30.0, slopes=torch.rand(4, device="cuda"))
    dq, dk = documents(lens, [100, 640, 1000])
    run(lens, 4, 2, d, dtype, causal=True, doc_q=dq, doc_k=dk)
    dq[::3] = 55  # see the prefix alone, or nothing
    run(lens, 4, 2, d, dtype, doc_q=dq, doc_k=dk)
    prefix = torch.full((len(lens),), 70, dtype=torch.int32, device="cuda")
    bad = torch.zeros(len(dk), dtype=torch.bool, device="cuda")
    at = torch.cat([torch.arange(b) for _, b in lens]).cuda()
    dk[(at >= 70) & (at % 4 == 0)] = 77
    bad[dk == 77] = True
    run(lens, 4, 2, d, dtype, doc_q=dq, doc_k=dk, prefix=prefix,
        poison=lambda q, k, v: (k.__setitem__(bad.nonzero().flatten(), math.nan), v.__setitem__(bad.nonzero().flatten(), math.inf)))


@pytest.mark.parametrize("d,dtype", [(64, HF), (128, BF)])
@pytest.mark.parametrize("lens", [[(1, 300)], [(2, 900)], [(150, 200)]])
def test_large_and_small_caps(lens, d, dtype):
    """A cap far above the scores changes them by 2.4e-6 of themselves (and the
    tanh by nothing): the uncapped result.  One far below them flattens them."""
    g = torch.Generator(device="cuda").manual_seed(1)
    nq, nk = lens[0]
    q, k, v = (torch.randn((n, 2 * d), device="cuda", generator=g).to(dtype) for n in (nq, nk, nk))
    q = q * 4
    args = (cu([nq]), cu([nk]), nq, nk, 2, 1 / math.sqrt(d))
    want, tol = attention64(q, k, v, lens, 2, 2, 1 / math.sqrt(d))
    score = float((q.double().reshape(nq, 2, d).norm(dim=2).max() * k.double().reshape(nk, 2, d).norm(dim=2).max()) / math.sqrt(d))
    for cap in (1e5, 1e6):
        got = ops().masked_attention(q, k, v, *args, softcap=cap)
        assert bool(((got.double() - want).abs() <= tol + 2 * 2.4e-6 * score * 2 * v.double().abs().amax()).all())
    got = ops().masked_attention(q, k, v, *args, softcap=1e-6)
    mean = v.double().mean(0)
    u = torch.finfo(dtype).eps / 2
    # every weight is 1 within 2e-6 and its rounding; the mean's own rounding; f32 sums
    bound = (u * 1.01 + 4e-6 + nk * 2.0 ** -24) * 2 * v.double().abs().mean(0) + u * mean.abs() + 2.0 ** -24
    assert bool(((got.double() - mean).abs() <= bound).all())


def test_more_refusals():
    from pixal3d.cpp_b200 import _lib as l
    o = ops()
    q = torch.zeros((4, 128), device="cuda").half()
    c = cu([4])
    for bad in (dict(softcap=1e7), dict(softcap=1e-9), dict(softcap=math.inf)):
        with pytest.raises(l.P3DError) as e:
            o.masked_attention(q, q, q, c, c, 4, 4, 2, 1.0, **bad)
        assert e.value.status == l.P3D_ERR_INVALID
    for bad in (lambda: o.masked_attention(q, q, q, c, c, -1, 4, 2, 1.0), lambda: o.masked_attention(q, q, q, c, c, 4, -1, 2, 1.0),
                lambda: o.masked_attention(q, q, q, c, c, 4, 4, 0, 1.0), lambda: o.masked_attention(q, q[:, :64], q, c, c, 4, 4, 2, 1.0),
                lambda: o.masked_attention(q, q.t().contiguous().t(), q, c, c, 4, 4, 2, 1.0)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        o.masked_attention(q, q, None, c, c, 4, 4, 2, 1.0)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d,dtype", [(64, HF), (128, BF)])
@pytest.mark.parametrize("lens", [[(1100, 1100), (0, 40), (300, 700), (9, 0)], [(9, 30)] * 31])
def test_documents_of_more_tiles_than_places(lens, d, dtype, causal):
    """Tiles are taken in the order of their key blocks: sorted documents, numbers in any order, empty tiles and sequences."""
    g = torch.Generator(device="cuda").manual_seed(11)
    dq, dk = documents(lens, [3, 70, 500, 620, 1000])
    prefix = torch.arange(len(lens), dtype=torch.int32, device="cuda") * 7 - 5
    run(lens, 10, 5, d, dtype, causal=causal, doc_q=dq, doc_k=dk, prefix=prefix)
    dq, dk = (torch.randint(-3, 5, x.shape, device="cuda", generator=g).int() for x in (dq, dk))
    got = run(lens, 12, 1, d, dtype, causal=causal, doc_q=dq, doc_k=dk)
    assert torch.equal(got, run(lens, 12, 1, d, dtype, causal=causal, doc_q=dq, doc_k=dk))


@pytest.mark.parametrize("sequences", [1024, 1025])
def test_documents_of_many_sequences(sequences):
    """The most tiles that are ordered, and one more."""
    lens = [(9 + i % 3, 11 + i % 70) for i in range(sequences)]
    dq, dk = documents(lens, [5, 40, 64])
    run(lens, 1, 1, 64, HF, doc_q=dq, doc_k=dk)


def test_ordered_documents_in_graphs_and_on_streams():
    """One workspace, two captured calls replayed in turn and a call on another stream: each call counts its tiles anew."""
    o = ops()
    n, heads, d = 1500, 30, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn((n, heads * d), device="cuda", generator=g).half() for _ in range(3))
    doc = torch.bucketize(torch.arange(n), torch.tensor([100, 900, 1000]), right=True).int().cuda()

    def call(doc):
        return o.masked_attention(q, k, v, cu([n]), cu([n]), n, n, heads, 0.125, doc_q=doc, doc_k=doc)

    other = doc.flip(0).contiguous()
    want = call(doc), call(other)
    c = cu([n])
    graphs = []
    for x in (doc, other):
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = o.masked_attention(q, k, v, c, c, n, n, heads, 0.125, doc_q=x, doc_k=x)
        graphs.append((gr, out))
    for _ in range(3):
        for (gr, out), w in zip(graphs, want):
            out.fill_(1.0)
            gr.replay()
            assert torch.equal(out, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = call(other)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want[1])
    o.ctx().sync_check()


@pytest.mark.parametrize("d,dtype", [(64, HF), (128, BF)])
def test_documents_that_come_late(d, dtype):
    """Inputs far from the SMs: loads of masks end before or after those of keys, and no wait runs out."""
    o = ops()
    g = torch.Generator(device="cuda").manual_seed(9)
    n, heads = 1300, 30
    q, k, v = (torch.randn((n, heads * d), device="cuda", generator=g).to(dtype) for _ in range(3))
    doc = torch.bucketize(torch.arange(n), torch.tensor([64, 200, 210, 700]), right=True).int().cuda()
    slopes = torch.rand(heads, device="cuda", generator=g)
    flush = torch.empty(64 << 20, dtype=torch.int32, device="cuda")
    c = cu([n])
    want = o.masked_attention(q, k, v, c, c, n, n, heads, 0.1, doc_q=doc, doc_k=doc, slopes=slopes)
    o.ctx().sync_check()
    for i in range(40):
        flush.fill_(i)
        got = o.masked_attention(q, k, v, c, c, n, n, heads, 0.1, doc_q=doc, doc_k=doc, slopes=slopes)
        o.ctx().sync_check()
        assert torch.equal(got, want)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d,dtype", [(64, HF), (64, BF), (128, HF), (128, BF)])
def test_caps_near_and_far_from_the_scores(d, dtype, causal):
    """Blocks whose scores all lie within half the cap, blocks with a row beyond it, and the largest score on either side of it."""
    for softcap, sharp in ((50.0, 1.0), (50.0, 6.0), (8.0, 1.0), (3.0, 0.3), (1000.0, 4.0)):
        run([(300, 300), (140, 500)], 4, 2, d, dtype, softcap=softcap, sharp=sharp, causal=causal)


@pytest.mark.parametrize("d,dtype", [(64, HF), (128, BF)])
def test_split_keys_in_longer_buffers(d, dtype):
    """Splits are joined by the sequences' places, whatever rows lie behind them."""
    run([(64, 5000), (30, 700), (0, 9), (9, 2)], 4, 2, d, dtype, causal=True, spare=3000)
    run([(1, 30), (100, 4000)], 6, 3, d, dtype, slopes=torch.rand(6, device="cuda"), spare=500)


@pytest.mark.parametrize("d,dtype", [(64, HF), (128, BF)])
def test_sequences_longer_than_max_k(d, dtype):
    """A max_k below the longest sequence costs time only, and a cache of many
    more rows than the sequences have costs nothing."""
    o = ops()
    lens = [(1, 40000), (3, 700), (2, 5000), (1, 0), (1, 9)]
    nq, nk = sum(a for a, _ in lens), sum(b for _, b in lens)
    g = torch.Generator(device="cuda").manual_seed(17)
    q = torch.randn((nq, 8 * d), device="cuda", generator=g).to(dtype)
    k, v = (torch.randn((nk + 100000, 2 * d), device="cuda", generator=g).to(dtype) for _ in range(2))
    want, tol = attention64(q, k, v, lens, 8, 2, 0.1, causal=True)
    for max_k in (513, 600, 3000, 40000):
        got = o.masked_attention(q, k, v, cu([a for a, _ in lens]), cu([b for _, b in lens]), 3, max_k, 8, 0.1, kv_heads=2, causal=True)
        o.ctx().sync_check()
        assert bool(((got.double() - want).abs() <= tol).all()), max_k


@pytest.mark.parametrize("extra", [(1, 1), (1, 600), (9, 20)])
def test_the_most_sequences(extra):
    """65535 sequences, all but one of a single query and key: its value."""
    o = ops()
    n, d = 65534, 64
    g = torch.Generator(device="cuda").manual_seed(2)
    q, k, v = (torch.randn((n + e, d), device="cuda", generator=g).half() for e in (extra[0], extra[1], extra[1]))
    at = [torch.cat([torch.arange(n + 1), torch.tensor([n + e])]).int().cuda() for e in extra]
    got = o.masked_attention(q, k, v, at[0], at[1], extra[0], extra[1], 1, 0.125)
    o.ctx().sync_check()
    assert torch.equal(got[:n], v[:n])
    want, tol = attention64(q[n:], k[n:], v[n:], [extra], 1, 1, 0.125)
    assert bool(((got[n:].double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [HF, BF])
@pytest.mark.parametrize("lens,heads,kv_heads", [([(5, 12000)] * 3, 16, 4), ([(1, 9000)] * 16, 24, 1), ([(6, 44000), (2, 3000), (0, 7)], 12, 3)])
def test_passes_of_24_rows(lens, heads, kv_heads, dtype):
    """17 to 24 rows a K/V head over many keys: one pass over them."""
    run(lens, heads, kv_heads, 64, dtype, causal=True, softcap=30.0)
