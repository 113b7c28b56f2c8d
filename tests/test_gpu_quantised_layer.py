"""The quantised attention layer as it is run: quantise rows, 8-bit qkv, rotary
positions in place, masked attention, quantise, 8-bit output projection added
into the residual; for packed prompts and token by token over a cache."""
import math

import pytest

torch = pytest.importorskip("torch")

from tests.test_gpu_masked_attention import attention64, cu
from tests.test_gpu_rotary import turned64

pytestmark = pytest.mark.gpu

H, KV, D, C = 8, 2, 64, 320


def ops():
    from pixal3d.cpp_b200 import ops as o
    return o


def weights(seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    o = ops()
    wq, ws = o.quantize_rows(torch.randn(((H + 2 * KV) * D, C), device="cuda", generator=g) / math.sqrt(C))
    wo, wos = o.quantize_rows(torch.randn((C, H * D), device="cuda", generator=g) / math.sqrt(H * D))
    return wq, ws, torch.randn((H + 2 * KV) * D, device="cuda", generator=g) * 0.1, wo, wos


def layer(x, w, freqs, pos, cu_q, cu_k, max_q, max_k, cache=None, rows=None, **rules):
    """x f32 [n, C] residual stream, updated in place; returns the parts."""
    from pixal3d.cpp_b200 import _lib as L
    o = ops()
    wq, ws, bias, wo, wos = w
    xq, xs = o.quantize_rows(x)
    qkv = o.linear_i8(xq, xs, wq, ws, bias, out_dtype=torch.bfloat16)
    plain = qkv.clone()
    heads = qkv[:, :(H + KV) * D]
    o.rotary(heads, freqs, H + KV, D, pos, out=heads)
    k, v = qkv[:, H * D:(H + KV) * D], qkv[:, (H + KV) * D:]
    if cache is not None:
        cache[0][rows], cache[1][rows] = k, v
        k, v = cache
    a = o.masked_attention(qkv[:, :H * D], k, v, cu_q, cu_k, max_q, max_k, H, 1 / math.sqrt(D), kv_heads=KV, causal=True, **rules)
    aq, as_ = o.quantize_rows(a)
    o.linear_i8(aq, as_, wo, wos, out=x, epilogue=L.EPI_RESIDUAL)
    return dict(xq=xq, xs=xs, plain=plain, qkv=qkv, k=k, v=v, a=a, aq=aq, as_=as_)


def test_layer_stage_by_stage():
    """Every stage against 64-bit arithmetic on what it was given."""
    o = ops()
    w = weights()
    lens = [(200, 200), (77, 77), (1, 1)]
    n = sum(a for a, _ in lens)
    x = torch.randn((n, C), device="cuda")
    x0 = x.clone()
    freqs, amp = o.rotary_frequencies(D, stretch=4.0)
    pos = torch.cat([torch.arange(a) for a, _ in lens]).int().cuda()
    c = cu([a for a, _ in lens])
    doc = torch.zeros(n, dtype=torch.int32, device="cuda")
    doc[120:200] = 1
    s = layer(x, w, freqs, pos, c, c, 200, 200, doc_q=doc, doc_k=doc, softcap=30.0)
    u = 2.0 ** -8  # half a step of bf16
    y = (s["xq"].double() @ w[0].double().t()) * s["xs"].double()[:, None] * w[1].double() + w[2].double()
    assert bool(((s["plain"].double() - y).abs() <= u * y.abs() * 1.001 + 1e-6).all())
    turned, size = turned64(s["plain"][:, :(H + KV) * D], freqs, H + KV, D, pos, "half", 1.0)
    got = s["qkv"][:, :(H + KV) * D].double()
    assert bool(((got - turned).abs() <= u * turned.abs() * 1.001 + 2e-6 * size).all())
    assert torch.equal(s["qkv"][:, (H + KV) * D:], s["plain"][:, (H + KV) * D:])
    want, tol = attention64(s["qkv"][:, :H * D], s["k"], s["v"], lens, H, KV, 1 / math.sqrt(D), causal=True, doc_q=doc, doc_k=doc,
                            softcap=30.0)
    assert bool(((s["a"].double() - want).abs() <= tol).all())
    z = (s["aq"].double() @ w[3].double().t()) * s["as_"].double()[:, None] * w[4].double()
    assert bool(((x.double() - x0.double() - z).abs() <= 2.0 ** -22 * (z.abs() + x.abs() + x0.abs())).all())


def test_tokens_one_by_one_match_the_prompt():
    """The cache filled token by token gives the prompt's rows: the same
    integers and turned heads, and attention within its tolerance, which the
    output projection carries on."""
    o = ops()
    w = weights(1)
    n = 140
    x = torch.randn((n, C), device="cuda")
    freqs, _ = o.rotary_frequencies(D)
    c = cu([n])
    full = x.clone()
    s = layer(full, w, freqs, torch.arange(n, dtype=torch.int32, device="cuda"), c, c, n, n)
    want, tol = attention64(s["qkv"][:, :H * D], s["k"], s["v"], [(n, n)], H, KV, 1 / math.sqrt(D), causal=True)
    # the cache's unwritten rows hold what memory holds: NaN here
    cache = [torch.full((n, KV * D), math.nan, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for t in range(n):
        one = x[t:t + 1].clone()
        p = layer(one, w, freqs, None if t == 0 else torch.tensor([t], dtype=torch.int32, device="cuda"), cu([1]), cu([t + 1]), 1, t + 1,
                  cache=cache, rows=slice(t, t + 1))
        assert torch.equal(p["qkv"], s["qkv"][t:t + 1])
        assert bool(((p["a"].double() - want[t:t + 1]).abs() <= tol[t:t + 1]).all()), t


def test_layer_in_a_graph():
    """Captured once, replayed on new inputs beside a second captured copy."""
    o = ops()
    w = weights(2)
    n = 300
    freqs, _ = o.rotary_frequencies(D)
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    c = cu([120, 180])
    doc = (torch.arange(n, device="cuda") // 50).int()
    args = (freqs, pos, c, c, 180, 180)
    x = torch.randn((n, C), device="cuda")
    layer(x.clone(), w, *args, doc_q=doc, doc_k=doc)
    torch.cuda.synchronize()
    runs = []
    for _ in range(2):
        buf = torch.zeros_like(x)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            layer(buf, w, *args, doc_q=doc, doc_k=doc)
        runs.append((g, buf))
    for seed in range(3):
        x = torch.randn((n, C), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
        want = x.clone()
        layer(want, w, *args, doc_q=doc, doc_k=doc)
        for g, buf in runs:
            buf.copy_(x)
        torch.cuda.synchronize()
        for g, _ in runs:
            g.replay()
        torch.cuda.synchronize()
        for _, buf in runs:
            assert torch.equal(buf, want)


def test_two_threads_on_their_own_streams():
    """Calls of two host threads on their own streams do not mix."""
    import threading
    o = ops()
    w = weights(3)
    freqs, _ = o.rotary_frequencies(D)
    results, errors = {}, []

    def work(k, stream):
        try:
            n = 64 + 40 * k
            g = torch.Generator(device="cuda").manual_seed(k)
            with torch.cuda.stream(stream):
                x0 = torch.randn((n, C), device="cuda", generator=g)
                c, pos = cu([n]), torch.arange(n, dtype=torch.int32, device="cuda")
                for _ in range(30):
                    x = x0.clone()
                    layer(x, w, freqs, pos, c, c, n, n)
                results[k] = (x0, x)
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(k, torch.cuda.Stream())) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    torch.cuda.synchronize()
    for x0, x in results.values():
        n = x0.shape[0]
        want = x0.clone()
        c = cu([n])
        layer(want, w, freqs, torch.arange(n, dtype=torch.int32, device="cuda"), c, c, n, n)
        assert torch.equal(x, want)
