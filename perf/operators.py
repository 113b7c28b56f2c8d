"""Cases, inputs, plain forms and 64-bit values of the operators of a quantised transformer block on packed rows:

  quantize  rows to 8-bit integers with one scale for each row
  linear    matrix product of 8-bit integers with scales for each row and output channel, bias and activation
  rotary    rotary positions of packed heads: half and interleaved pairs, part of the head, stretched frequencies
  attend    attention over packed sequences with capped scores, distance bias, causal, prefix and document masks

`run` computes them by elementary torch operations, or, where `own` is true, by the framework's entry points.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    q = dict(op="quantize", pad=0)
    i8 = dict(op="linear", bias=True)
    at = dict(op="attend", cap=0.0, slopes=False, causal=False, prefix=0, docs=0)
    return [
        # the modulation vector of one image, before its int8 projection: latency
        dict(q, name="quantize_token", m=1, k=1024, dtype="bf16"),
        # the MLP's hidden rows of a flow trunk step with classifier-free guidance
        dict(q, name="quantize_hidden", m=8184, k=4096, dtype="f16"),
        # voxel features beside projected image channels: odd width, f32, rows inside wider ones
        dict(q, name="quantize_voxels", m=21766, k=773, dtype="f32", pad=27),
        # the six modulation vectors of a conditional and an unconditional item: latency, all weights
        dict(i8, name="linear_modulation", m=2, k=1024, n=6144, out="f32", act="none"),
        # keys and values of one image's condition tokens (1024 patches and 5 more)
        dict(i8, name="linear_context", m=1029, k=1024, n=2048, out="f16", act="none"),
        # the trunk's MLP, up and down
        dict(i8, name="linear_mlp_up", m=8184, k=1024, n=4096, out="bf16", act="gelu"),
        dict(i8, name="linear_mlp_down", m=8184, k=4096, n=1024, out="f32", act="none"),
        # one new token far into a long context, stretched frequencies: latency
        dict(op="rotary", name="rotary_token", n=1, heads=40, dim=128, rot=128, layout="half", dtype="bf16", far=1 << 20,
             stretch=16.0, pad=1024),
        # query and key heads of packed rows, three quarters of the head turned
        dict(op="rotary", name="rotary_packed", n=16368, heads=32, dim=64, rot=48, layout="interleaved", dtype="f16",
             far=32768, stretch=1.0, pad=1024),
        # one new token of each of several sequences over its keys and values, shared heads, capped scores
        dict(at, name="attend_token", seqs=5, lq=1, lk=16381, ragged=True, heads=32, kv=8, dim=128, dtype="bf16", cap=50.0,
             causal=True),
        # condition tokens seen by all as a prefix, the rest causal, capped scores
        dict(at, name="attend_prefix", seqs=2, lq=4092, lk=4092, ragged=True, heads=16, kv=16, dim=64, dtype="f16", cap=30.0,
             causal=True, prefix=1029),
        # many items packed into one long sequence behind a shared prefix, distance bias, shared heads
        dict(at, name="attend_documents", seqs=1, lq=16384, lk=16384, ragged=False, heads=16, kv=4, dim=128, dtype="bf16",
             slopes=True, prefix=130, docs=5),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["quantize", "linear", "rotary", "attend", "attend"])
    if op == "quantize":
        k = log(16, 4096)
        return dict(op=op, m=min(log(1, 43532), 33_000_000 // k), k=k, dtype=rng.choice(list(TYPES)), pad=rng.choice([0, 0, 1, 8, 40]))
    if op == "linear":
        k, n = log(32, 4096), log(32, 6144)
        return dict(op=op, m=max(1, min(log(1, 8184), 34_000_000_000 // (k * n))), k=k, n=n, out=rng.choice(list(TYPES)),
                    act=rng.choice(["none", "gelu", "silu"]), bias=rng.random() < 0.7)
    if op == "rotary":
        dim = rng.choice([32, 64, 80, 128])
        heads = rng.randint(1, 40)
        return dict(op=op, n=min(log(1, 16368), 33_000_000 // (heads * dim)), heads=heads, dim=dim, rot=2 * rng.randint(1, dim // 2),
                    layout=rng.choice(["half", "interleaved"]), dtype=rng.choice(list(TYPES)), far=log(64, 1 << 21),
                    stretch=rng.choice([1.0, 4.0, 32.0]), pad=rng.choice([0, 0, 8, 1024]))
    heads, kv = rng.choice([(16, 16), (12, 12), (16, 4), (32, 8), (10, 2), (6, 1)])
    case = dict(op=op, heads=heads, kv=kv, dim=rng.choice([64, 128]), dtype=rng.choice(["bf16", "f16"]),
                cap=rng.choice([0.0, 0.0, 30.0, 50.0]), slopes=rng.random() < 0.4, causal=rng.random() < 0.6,
                seqs=rng.randint(1, 6), ragged=rng.random() < 0.7)
    if rng.random() < 0.5:
        lk = log(1, 16384)
        return dict(case, lq=min(lk, rng.choice([1, 1, 1, 2, 5])), lk=lk, prefix=0, docs=0)
    lk = log(16, 8192 // case["seqs"])
    return dict(case, lq=lk if rng.random() < 0.6 else log(8, lk), lk=lk, prefix=rng.choice([0, 0, lk // 5]), docs=rng.choice([0, 0, 3, 7]))


# ------------------------------------------------------------------- inputs

def lengths(case):
    """(queries, keys) of each sequence."""
    n, lq, lk = case["seqs"], case["lq"], case["lk"]
    keys = [max(1, lk - (i * lk) // (2 * n)) if case["ragged"] else lk for i in range(n)]
    return [(min(lq, k) if lq < lk else k, k) for k in keys]


def documents(case, n):
    """The document of each of n positions: uneven runs."""
    d = max(1, case["docs"])
    cuts = [int(n * ((i + 1) / d) ** 1.3) for i in range(d - 1)]
    return np.searchsorted(np.array(cuts, dtype=np.int64), np.arange(n), side="right").astype(np.int32)


def frequencies(rot, stretch, base=10000.0, original=4096, fast=32.0, slow=1.0):
    """Angles per position in 64 bits; for stretch > 1, pairs that turn fewer than `slow` times in the original length
    are slowed by the factor, those that turn more than `fast` times are kept, those between are mixed."""
    f = base ** (-np.arange(0, rot, 2, dtype=np.float64) / rot)
    if stretch > 1.0:
        keep = np.clip((original * f / (2 * math.pi) - slow) / (fast - slow), 0.0, 1.0)
        f = f / stretch * (1.0 - keep) + f * keep
    return f


def amplitude(stretch):
    return 1.0 if stretch <= 1.0 else 0.1 * math.log(stretch) + 1.0


def rows(shape, width, dtype, gen, scale=1.0):
    """Random rows as a view of wider ones."""
    m, k = shape
    return (torch.randn((m, width), generator=gen, device="cuda") * scale).to(dtype)[:, :k]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    st = dict(op=case["op"])
    if case["op"] == "quantize":
        m, k = case["m"], case["k"]
        x = rows((m, k), k + case["pad"], torch.float32, gen)
        x = x * torch.exp(torch.randn((m, 1), generator=gen, device="cuda"))  # rows of different size
        x[:, :: max(1, k // 7)] *= 8.0  # and channels that stand out, as activations have
        wide = torch.zeros((m, k + case["pad"]), dtype=TYPES[case["dtype"]], device="cuda")
        wide[:, :k] = x
        st.update(x=wide[:, :k])
    elif case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        pitch = (k + 15) // 16 * 16  # rows of whole 16-byte words
        x = (rows((m, pitch), pitch, torch.float32, gen) * 36.0).round().clamp(-127, 127).to(torch.int8)
        w = (rows((n, pitch), pitch, torch.float32, gen) * 42.0).round().clamp(-127, 127).to(torch.int8)
        xs = torch.exp(0.5 * torch.randn(m, generator=gen, device="cuda")) / 36.0
        ws = torch.exp(0.3 * torch.randn(n, generator=gen, device="cuda")) / (42.0 * math.sqrt(k))
        st.update(x=x[:, :k], w=w[:, :k], xs=xs, ws=ws, out=TYPES[case["out"]], act=case["act"],
                  bias=0.3 * torch.randn(n, generator=gen, device="cuda") if case["bias"] else None)
    elif case["op"] == "rotary":
        width = case["heads"] * case["dim"]
        st.update(x=rows((case["n"], width), width + case["pad"], TYPES[case["dtype"]], gen, 1.5),
                  positions=torch.randint(0, case["far"], (case["n"],), generator=gen, device="cuda", dtype=torch.int32),
                  freqs=torch.from_numpy(frequencies(case["rot"], case["stretch"])).cuda(), amplitude=amplitude(case["stretch"]),
                  heads=case["heads"], dim=case["dim"], layout=case["layout"])
    else:
        h, kv, d, t = case["heads"], case["kv"], case["dim"], TYPES[case["dtype"]]
        lens = lengths(case)
        cu = [np.concatenate([[0], np.cumsum([p[i] for p in lens])]).astype(np.int32) for i in (0, 1)]
        if all(a == b for a, b in lens):  # one packed projection, as a self-attention has
            qkv = rows((int(cu[0][-1]), (h + 2 * kv) * d), (h + 2 * kv) * d, t, gen)
            qkv[:, : h * d] *= 2.5
            q, k, v = qkv[:, : h * d], qkv[:, h * d : (h + kv) * d], qkv[:, (h + kv) * d :]
        else:
            q = rows((int(cu[0][-1]), h * d), h * d, t, gen, 2.5)
            k, v = (rows((int(cu[1][-1]), kv * d), kv * d, t, gen) for _ in range(2))
        st.update(q=q, k=k, v=v, heads=h, kv=kv, dim=d, cap=case["cap"], causal=case["causal"], scale=1.0 / math.sqrt(d),
                  starts_q=cu[0].tolist(), starts_k=cu[1].tolist(), cu_q=torch.from_numpy(cu[0]).cuda(),
                  cu_k=torch.from_numpy(cu[1]).cuda(), max_q=max(p[0] for p in lens), max_k=max(p[1] for p in lens),
                  slopes=2.0 ** (-8.0 * (torch.arange(h, device="cuda", dtype=torch.float32) + 1) / h) if case["slopes"] else None,
                  prefix=torch.tensor([min(case["prefix"], p[1]) for p in lens], dtype=torch.int32, device="cuda") if case["prefix"] else None,
                  doc_q=None, doc_k=None)
        if case["docs"]:
            of = [documents(case, p[1]) for p in lens]
            st.update(doc_k=torch.from_numpy(np.concatenate(of)).cuda(),
                      doc_q=torch.from_numpy(np.concatenate([x[p[1] - p[0] :] for x, p in zip(of, lens)])).cuda())
    return st


# -------------------------------------------------------------- plain forms

def activate(y, act):
    if act == "gelu":
        return 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    return y / (1.0 + torch.exp(-y)) if act == "silu" else y


def plain_quantize(st):
    x = st["x"]
    # 64 bits: a scale is amax / 127 rounded once, and quotients lie next to halves (half the row's largest gives 63.5)
    scale = (x.float().abs().amax(1).double() / 127.0).float().clamp_min(2.0 ** -126)
    q = torch.round(x.double() / scale.double()[:, None])
    return q.float() * scale[:, None], scale


def plain_linear(st):
    y = (st["x"].float() @ st["w"].float().t()) * st["xs"][:, None] * st["ws"]
    if st["bias"] is not None:
        y = y + st["bias"]
    return activate(y, st["act"]).to(st["out"])


def plain_rotary(st):
    x, half = st["x"], st["freqs"].numel()
    angle = st["positions"].double()[:, None] * st["freqs"]
    c, s = ((f(angle) * st["amplitude"]).float()[:, None, :] for f in (torch.cos, torch.sin))
    h = x.float().reshape(x.shape[0], st["heads"], st["dim"])
    turned, rest = h[..., : 2 * half], h[..., 2 * half :]
    if st["layout"] == "half":
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat([a * c - b * s, a * s + b * c], -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    return torch.cat([turned, rest], -1).reshape(x.shape).to(x.dtype)


def plain_attend(st):
    q, k, v, d, group = st["q"], st["k"], st["v"], st["dim"], st["heads"] // st["kv"]
    out = torch.zeros((q.shape[0], st["heads"] * d), dtype=q.dtype, device=q.device)
    for i in range(len(st["starts_q"]) - 1):
        q0, q1, k0, k1 = st["starts_q"][i], st["starts_q"][i + 1], st["starts_k"][i], st["starts_k"][i + 1]
        at_k = torch.arange(k1 - k0, device=q.device)
        at_q = torch.arange(q1 - q0, device=q.device) + (k1 - k0) - (q1 - q0)
        seen = torch.ones((q1 - q0, k1 - k0), dtype=torch.bool, device=q.device)
        if st["causal"]:
            seen &= at_k <= at_q[:, None]
        if st["doc_q"] is not None:
            seen &= st["doc_k"][k0:k1] == st["doc_q"][q0:q1, None]
        if st["prefix"] is not None:
            seen |= at_k < st["prefix"][i]
        apart = (at_q[:, None] - at_k).abs().float()
        for j in range(st["kv"]):
            heads = slice(j * group * d, (j + 1) * group * d)
            qs = q[q0:q1, heads].float().reshape(q1 - q0, group, d).transpose(0, 1)
            s = (qs @ k[k0:k1, j * d : (j + 1) * d].float().t()) * st["scale"]
            if st["cap"] > 0.0:
                s = st["cap"] * torch.tanh(s / st["cap"])
            if st["slopes"] is not None:
                s = s - st["slopes"][j * group : (j + 1) * group, None, None] * apart
            s = s.masked_fill(~seen, -math.inf)
            p = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e30))
            o = (p @ v[k0:k1, j * d : (j + 1) * d].float()) / p.sum(-1, keepdim=True).clamp_min(1e-30)
            out[q0:q1, heads] = o.transpose(0, 1).reshape(q1 - q0, group * d).to(q.dtype)
    return out


def run(state):
    st = state
    if own:
        from pixal3d.cpp_b200 import _lib as L
        from pixal3d.cpp_b200 import ops
        if st["op"] == "quantize":
            q, scale = ops.quantize_rows(st["x"])
            return q * scale[:, None], scale
        if st["op"] == "linear":
            return ops.linear_i8(st["x"], st["xs"], st["w"], st["ws"], st["bias"], out_dtype=st["out"],
                                 epilogue={"none": L.EPI_NONE, "gelu": L.EPI_GELU_TANH, "silu": L.EPI_SILU}[st["act"]])
        if st["op"] == "rotary":
            return ops.rotary(st["x"], st["freqs"], st["heads"], st["dim"], st["positions"], layout=st["layout"],
                              amplitude=st["amplitude"])
        return ops.masked_attention(st["q"], st["k"], st["v"], st["cu_q"], st["cu_k"], st["max_q"], st["max_k"], st["heads"],
                                    st["scale"], kv_heads=st["kv"], causal=st["causal"], prefix=st["prefix"], doc_q=st["doc_q"],
                                    doc_k=st["doc_k"], slopes=st["slopes"], softcap=st["cap"])
    return {"quantize": plain_quantize, "linear": plain_linear, "rotary": plain_rotary, "attend": plain_attend}[st["op"]](st)


# ------------------------------------------------------------ work and truth

def pairs(case):
    """Visible (query, key) pairs of one head."""
    total = 0
    for lq, lk in lengths(case):
        at = np.arange(lq) + lk - lq
        doc = documents(case, lk)
        first, last = np.searchsorted(doc, doc[lk - lq :], "left"), np.searchsorted(doc, doc[lk - lq :], "right")
        end = np.minimum(last, at + 1) if case["causal"] else last
        p = min(case["prefix"], lk)
        total += int((p + np.maximum(0, end - np.maximum(first, p))).sum())
    return total


def work(case):
    if case["op"] == "quantize":
        m, k = case["m"], case["k"]
        # the integers come back as the values they stand for, 4 bytes each
        return {"bytes": m * k * (SIZES[case["dtype"]] + 4) + 4 * m, "flops": 2 * m * k}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + m * n * SIZES[case["out"]] + 4 * m + 4 * n * (2 if case["bias"] else 1), "flops": 2 * m * n * k}
    if case["op"] == "rotary":
        e = case["n"] * case["heads"] * case["dim"]
        return {"bytes": 2 * e * SIZES[case["dtype"]] + 4 * case["n"], "flops": 3 * case["n"] * case["heads"] * case["rot"]}
    lens, d, s = lengths(case), case["dim"], SIZES[case["dtype"]]
    nq, nk = sum(p[0] for p in lens), sum(p[1] for p in lens)
    return {"bytes": 2 * nq * case["heads"] * d * s + 2 * nk * case["kv"] * d * s + (4 * (nq + nk) if case["docs"] else 0),
            "flops": 4 * d * case["heads"] * pairs(case)}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "quantize":
        x = st["x"].double()
        scale = torch.clamp((x.abs().max(1).values / 127.0).float(), min=2.0 ** -126)  # a scale is a 32-bit number
        return torch.round(x / scale.double().unsqueeze(1)) * scale.double().unsqueeze(1), scale.double()
    if case["op"] == "linear":
        y = torch.mm(st["x"].double(), st["w"].double().T)
        y *= torch.outer(st["xs"].double(), st["ws"].double())
        y += 0.0 if st["bias"] is None else st["bias"].double()
        if case["act"] == "gelu":
            y = y * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * y * (1.0 + 0.044715 * y.square()))
        elif case["act"] == "silu":
            y = y * torch.sigmoid(y)
        return y
    if case["op"] == "rotary":
        n, h, d, half = case["n"], case["heads"], case["dim"], case["rot"] // 2
        x = st["x"].double().reshape(n, h, d)
        pair = torch.arange(half, device="cuda")
        a, b = (pair, pair + half) if case["layout"] == "half" else (2 * pair, 2 * pair + 1)
        turn = st["amplitude"] * torch.exp(1j * torch.outer(st["positions"].double(), st["freqs"]))
        z = torch.complex(x[:, :, a], x[:, :, b]) * turn.unsqueeze(1)
        y = x.clone()
        y[:, :, a], y[:, :, b] = z.real, z.imag
        return y.reshape(n, h * d)
    h, kv, d = case["heads"], case["kv"], case["dim"]
    q, k, v = (st[t].double().reshape(st[t].shape[0], -1, d) for t in "qkv")
    out = torch.zeros((q.shape[0], h, d), dtype=torch.float64, device="cuda")
    at_q = at_k = 0
    for i, (lq, lk) in enumerate(lengths(case)):
        where = torch.arange(lk - lq, lk, device="cuda").unsqueeze(1) - torch.arange(lk, device="cuda").unsqueeze(0)
        hidden = (where < 0) if case["causal"] else torch.zeros_like(where, dtype=torch.bool)
        if case["docs"]:
            doc = torch.from_numpy(documents(case, lk)).cuda()
            hidden = hidden | (doc[lk - lq :].unsqueeze(1) != doc.unsqueeze(0))
        hidden[:, : min(case["prefix"], lk)] = False
        for j in range(h):
            s = torch.einsum("qd,kd->qk", q[at_q : at_q + lq, j], k[at_k : at_k + lk, j * kv // h]) * st["scale"]
            if case["cap"]:
                s = torch.tanh(s / case["cap"]) * case["cap"]
            if case["slopes"]:
                s -= float(st["slopes"][j]) * where.abs()
            s[hidden] = -math.inf
            out[at_q : at_q + lq, j] = torch.nan_to_num(torch.softmax(s, -1), nan=0.0) @ v[at_k : at_k + lk, j * kv // h]
        at_q, at_k = at_q + lq, at_k + lk
    return out.reshape(q.shape[0], h * d)
