"""Operators on buffers whose element offsets pass 32 bits: the same results as
on small copies of the rows."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

BIG = 2 ** 31 + 2 ** 27  # elements


def ops():
    from pixal3d.cpp_b200 import ops as o
    return o


def cu(*at):
    return torch.tensor(at, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("lq,lk", [(1, 20000), (3, 300), (200, 2500)])
def test_attention_at_the_end_of_a_long_cache(lq, lk):
    heads, kv, d = 16, 8, 128
    rows = BIG // (kv * d)
    g = torch.Generator(device="cuda").manual_seed(lq)
    cache = torch.empty((rows, kv * d), dtype=torch.bfloat16, device="cuda")
    cache[-lk:] = torch.randn((lk, kv * d), device="cuda", generator=g).to(cache.dtype)
    q = torch.randn((lq, heads * d), device="cuda", generator=g).to(cache.dtype)
    doc_q, doc_k = torch.zeros(lq, dtype=torch.int32, device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda")
    doc_k[-lk::5] = 1
    small = cache[-lk:].clone()
    for docs in (False, True):
        a = dict(doc_q=doc_q, doc_k=doc_k) if docs else {}
        b = dict(doc_q=doc_q, doc_k=doc_k[-lk:].contiguous()) if docs else {}
        got = ops().masked_attention(q, cache, cache, cu(0, lq), cu(rows - lk, rows), lq, lk, heads, 0.1, kv_heads=kv, causal=True, **a)
        want = ops().masked_attention(q, small, small, cu(0, lq), cu(0, lk), lq, lk, heads, 0.1, kv_heads=kv, causal=True, **b)
        assert torch.equal(got, want)
    ops().ctx().sync_check()


def test_wide_pitches():
    m = 2100
    pitch = BIG // m // 16 * 16
    g = torch.Generator(device="cuda").manual_seed(0)
    big = torch.empty((m, pitch), dtype=torch.bfloat16, device="cuda")
    x = torch.randn((m, 512), device="cuda", generator=g).to(big.dtype)
    big[:, :512] = x
    o = ops()
    q, s = o.quantize_rows(big[:, :512])
    wq, ws = o.quantize_rows(x)
    assert torch.equal(q, wq) and torch.equal(s, ws)
    f, _ = o.rotary_frequencies(64)
    want = o.rotary(x, f, 8, 64)
    assert torch.equal(o.rotary(big[:, :512], f, 8, 64, out=big[:, :512]), want)
    w, wsc = o.quantize_rows(torch.randn((70, 512), device="cuda", generator=g))
    want = o.linear_i8(wq, ws, w, wsc)
    assert torch.equal(o.linear_i8(wq, ws, w, wsc, out=big[:, :70]), want)
    assert torch.equal(o.linear_i8(wq[:3], ws[:3], w, wsc, out=big[:3, 1:71]), o.linear_i8(wq[:3], ws[:3], w, wsc))
    i8 = big.view(torch.int8)[:, :512]
    i8.copy_(wq)
    assert torch.equal(o.linear_i8(i8, ws, w, wsc), want)
    q8, _ = o.quantize_rows(x, out=big.view(torch.int8)[:, 600:1112])
    assert torch.equal(q8, wq)
