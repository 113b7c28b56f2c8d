"""Argument checks of the quantised-block operators that need no device."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from pixal3d.cpp_b200 import _lib as L
from pixal3d.cpp_b200 import ops


def test_tensors_off_the_device_are_refused():
    x = torch.zeros((4, 64))
    i8, one, c = x.to(torch.int8), torch.ones(4), torch.tensor([0, 4], dtype=torch.int32)
    for bad in (lambda: ops.quantize_rows(x), lambda: ops.linear_i8(i8, one, i8, one),
                lambda: ops.rotary(x, torch.ones(16, dtype=torch.float64), 2, 32),
                lambda: ops.masked_attention(x.half(), x.half(), x.half(), c, c, 4, 4, 1, 1.0)):
        with pytest.raises(ValueError, match="CUDA"):
            bad()


def test_null_context_is_refused():
    assert L.lib.p3d_quantize_rows(None, None, 0, 1, 1, 0, None, 0, None) == L.P3D_ERR_INVALID
    assert L.lib.p3d_linear_i8(None, None, 0, None, None, 0, None, None, 1, 1, 1, None, 0, 0, 0, None, 0, None, 0) == L.P3D_ERR_INVALID
    assert L.lib.p3d_rotary(None, None, 0, 1, 1, 2, 2, 0, None, 0, None, 1.0, None, 0, 0) == L.P3D_ERR_INVALID
    assert L.lib.p3d_masked_attention(None, None, 0, None, 0, None, 0, None, 0, None, None, 1, 1, 1, 1, 1, 1, 1, 64, 1.0,
                                      C.byref(L.AttentionRules()), None, 0, 1) == L.P3D_ERR_INVALID


def test_masked_attention_workspace():
    ws = L.lib.p3d_masked_attention_workspace
    assert ws(0, 1, 1, 1, 1, 1, 1, 64, 0) == 0 and ws(1, 0, 1, 1, 1, 1, 1, 64, 0) == 0
    token = ws(1, 1, 16384, 1, 16384, 16, 4, 128, 0)
    assert token >= 2 * 16 * 128 * 4  # one token over a long cache: its keys are split
    assert token <= ws(1, 1, 65536, 1, 65536, 16, 4, 128, 0)
    assert ws(3, 500, 500, 1500, 1500, 16, 4, 128, 0) == 0
    assert ws(3, 500, 500, 1500, 1500, 16, 4, 128, 1) >= 8 * (1500 // 64 + 3 + 1)  # a range for every block of keys


def test_rotary_frequencies_on_the_host():
    f, amp = ops.rotary_frequencies(8, base=10.0, device="cpu")
    assert amp == 1.0 and f.dtype == torch.float64
    assert torch.allclose(f, 10.0 ** -torch.tensor([0, 0.25, 0.5, 0.75], dtype=torch.float64), rtol=1e-15, atol=0)
    with pytest.raises(ValueError):
        ops.rotary_frequencies(8, fast=1.0, slow=1.0, device="cpu")


def test_masked_attention_workspace_does_not_grow_with_spare_query_rows():
    """64 queries over 8192 keys, split between blocks, in a q of 64 rows and of
    32768: the same results to join, so the same workspace."""
    ws = L.lib.p3d_masked_attention_workspace
    for documents in (0, 1):
        assert 0 < ws(1, 64, 8192, 32768, 8192, 16, 16, 128, documents) == ws(1, 64, 8192, 64, 8192, 16, 16, 128, documents)
    for nseq, max_q, heads in ((1, 9, 1), (1, 2000, 4), (3, 200, 6), (100, 100, 1)):
        assert ws(nseq, max_q, 16384, 1 << 30, 16384 * nseq, heads, heads, 128, 0) <= 296 * 128 * (128 + 2) * 4 + 512


def test_masked_attention_workspace_does_not_grow_with_spare_key_rows():
    """One token over 1024 keys that lie in a cache of 2^20 rows: as over 1024."""
    ws = L.lib.p3d_masked_attention_workspace
    assert 0 < ws(1, 1, 1024, 1, 1 << 20, 32, 8, 128, 0) <= ws(1, 1, 1024, 1, 1024, 32, 8, 128, 0)
    assert 0 < ws(4, 2, 3000, 9, 1 << 24, 32, 8, 64, 0) <= ws(4, 2, 3000, 9, 4 * 3000, 32, 8, 64, 0)
