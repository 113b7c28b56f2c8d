"""Host threads on their own streams, in calls of both bindings."""
import threading

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def test_threads_mix_both_bindings():
    """Each thread runs masked attention over documents (several dependent
    launches a call, native binding) between linear and varlen_attention (ctypes),
    on its own stream, and reads its results there without waiting for others."""
    from pixal3d.cpp_b200 import ops as o
    H, D = 12, 64
    cu = [torch.tensor([0, n], dtype=torch.int32, device="cuda") for n in (1500, 1400, 1300)]

    def chain(k, x, w, doc):
        n = x.shape[0]
        for _ in range(3):
            y = o.linear(x, w, None, out_dtype=torch.float16)
            q = y[:, :H * D]
            a = o.masked_attention(q, y[:, H * D:2 * H * D], y[:, 2 * H * D:], cu[k], cu[k], n, n, H, 0.125, doc_q=doc, doc_k=doc)
            b = o.varlen_attention(q, y[:, H * D:2 * H * D], y[:, 2 * H * D:], cu[k], cu[k], n, H, 0.125)
            xq, s = o.quantize_rows(a)
            x = (x + 0.5 * a + 0.5 * b + 0.01 * xq.half() * s[:, None].half()).half()
        return x

    g = torch.Generator(device="cuda").manual_seed(1)
    cases = []
    for n in (1500, 1400, 1300):
        x = torch.randn((n, H * D), device="cuda", generator=g).half()
        w = (torch.randn((3 * H * D, H * D), device="cuda", generator=g) / 30).half()
        cases.append((x, w, torch.bucketize(torch.arange(n), torch.tensor([100, 640, 1000]), right=True).int().cuda()))
    want = [chain(k, *c) for k, c in enumerate(cases)]
    launches = o.ctx().launches
    chain(0, *cases[0])
    each = o.ctx().launches - launches
    torch.cuda.synchronize()
    launches = o.ctx().launches
    got, errors = {}, []

    def work(k):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                out = [chain(k, *cases[k]) for _ in range(10)]
                o.ctx().sync_check()
            got[k] = out
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    torch.cuda.synchronize()
    for k, out in got.items():
        for x in out:
            assert torch.equal(x, want[k])
    assert o.ctx().launches - launches == 30 * each  # counted for the device, whatever the thread
    o.ctx().sync_check()


def test_flow_runs_on_the_calling_threads_stream():
    """A model made by one thread and run by another follows the latter's stream."""
    import numpy as np
    from oracle import oracle as O
    from pixal3d.cpp_b200 import _lib as L
    from tests.test_gpu_flow import make, two_item_coords
    coords = two_item_coords()
    n = coords.shape[0]
    _, model = make(O.FlowHParams(in_channels=8, out_channels=8, model_channels=128, cond_channels=64, num_blocks=2, num_heads=2,
                                  mlp_ratio=4.0), seed=1)
    rng = np.random.default_rng(2)
    x = torch.from_numpy(rng.standard_normal((n, 8)).astype(np.float32)).cuda()
    cond = torch.from_numpy(rng.standard_normal((77, 64)).astype(np.float32)).cuda()
    t = torch.tensor([500.0, 500.0], device="cuda")
    model.prepare(torch.from_numpy(coords).cuda(), 2, (16, 16, 16), [0, 40, 77])
    want = model.forward(x, t, cond)
    torch.cuda.synchronize()
    seen = {}

    def work():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            out = model.forward(x, t, cond)
            seen.update(on=L.lib.p3d_ctx_stream(model.ctx.h), stream=s.cuda_stream, out=out)
        s.synchronize()

    th = threading.Thread(target=work)
    th.start()
    th.join()
    assert seen["on"] == seen["stream"]
    assert torch.equal(seen["out"], want)
