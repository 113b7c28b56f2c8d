"""Masked attention where roundings on the way could show."""
import math

import pytest

torch = pytest.importorskip("torch")

from tests.test_gpu_masked_attention import BF, HF, attention64, cu, documents, ops

pytestmark = pytest.mark.gpu


def capped(lens, d, dtype, cap, doc_q=None, doc_k=None, causal=False, poison=None, rows=None):
    """A cap far above all scores but those of query rows `rows`: near scores
    are at most 2.4e-6 of themselves off whatever lies beside them, so nothing
    in the tolerance grows with the cap (the tanh itself takes s^3 / (3 cap^2),
    below 1e-6 here)."""
    o = ops()
    g = torch.Generator(device="cuda").manual_seed(7)
    nq, nk = sum(a for a, _ in lens), sum(b for _, b in lens)
    q = torch.randn((nq + 9, 2 * d), device="cuda", generator=g).to(dtype)
    k, v = (torch.randn((nk + 9, 2 * d), device="cuda", generator=g).to(dtype) for _ in range(2))
    scale = 1 / math.sqrt(d)
    rules = dict(causal=causal, doc_q=doc_q, doc_k=doc_k)
    want, tol = attention64(q, k, v, lens, 2, 2, scale, **rules)
    score = float(q[:nq].double().reshape(nq, 2, d).norm(dim=2).max() * k[:nk].double().reshape(nk, 2, d).norm(dim=2).max()) * scale
    tol = tol + 2 * (2.4e-6 * score + 1e-6) * 2 * v[:nk].double().abs().amax()
    if poison is not None:
        poison(q, k, v)
    got = o.masked_attention(q, k, v, cu([a for a, _ in lens]), cu([b for _, b in lens]), max(a for a, _ in lens), max(b for _, b in lens),
                             2, scale, softcap=cap, **rules)
    o.ctx().sync_check()
    keep = torch.ones(nq, dtype=torch.bool, device="cuda")
    if rows is not None:
        keep[rows] = False
    err = (got.double() - want).abs()[:nq][keep]
    assert bool((err <= tol[:nq][keep]).all()), float((err / tol[:nq][keep]).max())


CAPPED = [(64, HF), (64, BF), (128, HF), (128, BF)]


@pytest.mark.parametrize("cap", [1e5, 1e6])
@pytest.mark.parametrize("d,dtype", CAPPED)
@pytest.mark.parametrize("lens", [[(200, 200), (90, 130)], [(30, 1500)], [(3, 700)], [(2, 100)]])
def test_hidden_keys_leave_capped_scores_alone(lens, d, dtype, cap):
    """One infinite element in hidden keys, and in rows behind the last sequence."""
    dq, dk = documents(lens, [10 ** 6])
    dk[5::9] = 99
    dq, dk = torch.cat([dq, dq.new_full((9,), 7)]), torch.cat([dk, dk.new_full((9,), 7)])

    def poison(q, k, v):
        hidden = (dk == 99).nonzero().flatten()
        k[hidden, 3] = k[hidden, d + 3] = math.inf
        for t in (q, k, v):
            t[-9:] = 3e4
    capped(lens, d, dtype, cap, doc_q=dq, doc_k=dk, poison=poison)


@pytest.mark.parametrize("cap", [3e4, 1e5])
@pytest.mark.parametrize("d,dtype", CAPPED)
@pytest.mark.parametrize("lens,row", [([(200, 200), (90, 130)], 37), ([(130, 400)], 129), ([(5, 700)], 2)])
def test_far_scores_of_one_query_leave_the_others_alone(lens, row, d, dtype, cap):
    """A query whose scores reach the cap beside queries whose scores do not."""
    def poison(q, k, v):
        q[row] = 6e4 * torch.sign(q[row].float()).to(dtype)
    capped(lens, d, dtype, cap, poison=poison, rows=[row])


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq,n", [(1, 400), (7, 3000), (40, 3000), (1000, 900)])
def test_f16_weights_far_below_the_largest(lq, n, d):
    """Every sixteenth key has the largest weight and no value, the others 2^-18
    to 2^-24 of it and large values.  Weights are rounded to f16 with the
    largest at 2^7 or above: half a step of the smallest is 2^-32 of it."""
    o = ops()
    g = torch.Generator(device="cuda").manual_seed(d)
    q, k, v = (torch.zeros((m, 2 * d), device="cuda") for m in (lq, n, n))
    t = torch.linspace(12.5, 16.5, 2 * lq, device="cuda").reshape(lq, 2).half()
    q[:, 0], q[:, d] = t[:, 0], t[:, 1]
    k[:, 0] = k[:, d] = -1
    v[:] = 500 + 1000 * torch.rand((1, 2 * d), device="cuda", generator=g)
    k[5::16] = v[5::16] = 0
    q, k, v = q.half(), k.half(), v.half()
    got = o.masked_attention(q, k, v, cu([lq]), cu([n]), lq, n, 2, 1.0)
    o.ctx().sync_check()
    top = len(range(5, n, 16))
    e = torch.exp(-t.double())[:, :, None]
    want = e * (n - top) / (top + e * (n - top)) * v[0].double().reshape(2, d)
    # a weight: half its step (2^-11 of it, or 2^-32 of the largest) and the exponential's 2^-19; it counts once in
    # the mean and once in the sum; f32 sums of n terms; the result's own half step
    rel = 2 * (2.0 ** -11 + 2.0 ** -32 / e + 2.0 ** -19 + n * 2.0 ** -24)
    tol = want * (rel + 2.0 ** -11) * 1.01 + 2.0 ** -25
    err = (got.double().reshape(lq, 2, d) - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("d,dtype", [(64, HF), (64, BF), (128, HF), (128, BF)])
@pytest.mark.parametrize("lq,n", [(1, 100), (7, 90), (8, 1400), (200, 300), (64, 1500), (900, 900)])
@pytest.mark.parametrize("rules", [dict(), dict(causal=True, softcap=50.0)])
def test_values_that_are_alike_average_to_themselves(lq, n, d, dtype, rules):
    """Whatever the weights are, a weighted mean of equal numbers is that number:
    the weights are summed as the product with V takes them.  f32 sums of n <=
    1500 terms are n 2^-24 off, below half a step of the result."""
    o = ops()
    q, k, v = (torch.zeros((m, 2 * d), device="cuda") for m in (lq, n, n))
    q[:, 0] = q[:, d] = torch.linspace(0.1, 3.0, lq, device="cuda")
    q[:, 1] = q[:, d + 1] = torch.linspace(0.0, 0.01, lq, device="cuda")
    k[:, 0] = k[:, d] = -1
    k[:, 1] = k[:, d + 1] = torch.linspace(-1, 1, n, device="cuda")
    k[0] = 0
    v[:] = torch.rand((1, 2 * d), device="cuda", generator=torch.Generator(device="cuda").manual_seed(d)) * 4 - 2
    q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    got = o.masked_attention(q, k, v, cu([lq]), cu([n]), lq, n, 2, 1.0, **rules)
    o.ctx().sync_check()
    assert torch.equal(got, v[:1].expand_as(got)), float((got.double() / v[0].double() - 1).abs().max())


@pytest.mark.parametrize("softcap", [0.0, 20.0])
@pytest.mark.parametrize("d,dtype", [(64, HF), (64, BF), (128, HF), (128, BF)])
@pytest.mark.parametrize("lens", [[(200, 200)], [(70, 900), (5, 5)], [(300, 4000)], [(3, 700), (8, 900)], [(2, 100)]])
def test_what_lies_beside_changes_no_bit(lens, d, dtype, softcap):
    """Rows behind the last sequence and hidden keys may hold anything: the same
    outputs to the last bit."""
    o = ops()
    g = torch.Generator(device="cuda").manual_seed(23)
    nq, nk = sum(a for a, _ in lens), sum(b for _, b in lens)
    q = torch.randn((nq + 140, 2 * d), device="cuda", generator=g).to(dtype)
    k, v = (torch.randn((nk + 140, 2 * d), device="cuda", generator=g).to(dtype) for _ in range(2))
    cq, ck = cu([a for a, _ in lens]), cu([b for _, b in lens])
    doc = torch.zeros(nk + 140, dtype=torch.int32, device="cuda")
    doc[7:nk // 2:11] = 99
    dq = torch.zeros(nq + 140, dtype=torch.int32, device="cuda")
    hidden = (doc == 99).nonzero().flatten()
    for rules in (dict(), dict(causal=True), dict(doc_q=dq, doc_k=doc)):
        got = []
        for value in (0.0, 3e4, math.inf, math.nan):
            for t in (q[nq:], k[nk:], v[nk:]):
                t.fill_(value)
            if "doc_q" in rules:
                k[hidden] = v[hidden] = value
            out = o.masked_attention(q, k, v, cq, ck, max(a for a, _ in lens), max(b for _, b in lens), 2, 0.2, softcap=softcap, **rules)
            got.append(out[:nq])
        o.ctx().sync_check()
        assert all(torch.equal(got[0], x) for x in got[1:]), (rules.keys(), [int((got[0] != x).sum()) for x in got])
