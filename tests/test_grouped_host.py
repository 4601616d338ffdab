"""CPU: argument checks of the grouped and MXFP4 entry points.  Every refusal
here is decided before the first CUDA call; no kernel is launched."""

from __future__ import annotations

import ctypes

import pytest

P = 1 << 20  # a well-aligned address that is never read


def _lib():
    import tinym_b200

    return tinym_b200.capi()


def _fp8(x=P, w=P, y=P, ldy=64, rows=4, experts=2, n=64, k=64, offsets=P, alpha=P, count=1, flags=0):
    return _lib().tinym_fp8_gemm_grouped(x, w, y, ldy, rows, experts, n, k, offsets, alpha, count,
                                         flags, None)


def _mx(x=P, xs=P, w=P, ws=P, y=P, ldy=64, rows=4, experts=2, n=64, k=64, offsets=P, alpha=P,
        count=1, flags=0):
    return _lib().tinym_mxfp4_gemm_grouped(x, xs, w, ws, y, ldy, rows, experts, n, k, offsets, alpha,
                                           count, flags, None)


@pytest.mark.parametrize("call", [_fp8, _mx])
@pytest.mark.parametrize("bad,status,words", [
    (dict(x=None), 1, "non-null"),
    (dict(w=None), 1, "non-null"),
    (dict(y=None), 1, "non-null"),
    (dict(rows=0), 1, "positive"),
    (dict(experts=0), 1, "positive"),
    (dict(n=-1), 1, "positive"),
    (dict(k=0), 1, "positive"),
    (dict(k=40), 2, "multiple of"),
    (dict(experts=1025), 2, "experts"),
    (dict(rows=1 << 31), 2, "32-bit"),
    (dict(offsets=None), 1, "offsets"),
    (dict(ldy=63), 1, "ldy"),
    (dict(x=P + 8), 3, "16-byte"),
    (dict(w=P + 4), 3, "16-byte"),
    (dict(y=P + 1), 3, "2-byte"),
    (dict(offsets=P + 2), 3, "4-byte"),
    (dict(alpha=P + 2), 3, "4-byte"),
    (dict(count=3), 1, "alpha"),
    (dict(flags=1), 1, "flags"),
])
def test_grouped_refusals(call, bad, status, words):
    assert call(**bad) == status
    assert words in _lib().tinym_last_error().decode()


def test_mxfp4_gemm_refusals():
    for bad, status, words in [(dict(xs=None), 1, "scales"), (dict(ws=None), 1, "scales"),
                               (dict(xs=P + 4), 3, "scales"), (dict(k=48), 2, "multiple of 32")]:
        assert _mx(**bad) == status
        assert words in _lib().tinym_last_error().decode()
    assert _lib().tinym_mxfp4_gemm(P, P, P, P, P, 64, 0, 64, 64, None, None) == 1


def test_selftest_rejects_bad_timeout():
    for ns in (0, 10 ** 11):
        assert _lib().tinym_selftest_grouped_timeout(P, P, P, 4, 2, 64, 64, P, ns, None) == 1


@pytest.mark.parametrize("batch,rows,k,want", [
    (1, 1, 32, 512), (1, 128, 128, 512), (1, 129, 128, 1024), (1, 1, 160, 1024), (3, 200, 6144, 3 * 2 * 48 * 512),
])
def test_mxfp4_scale_bytes(batch, rows, k, want):
    out = ctypes.c_int64(0)
    assert _lib().tinym_mxfp4_scale_bytes(batch, rows, k, ctypes.byref(out)) == 0
    assert out.value == want


def test_mxfp4_quantize_refusals():
    lib = _lib()
    out = ctypes.c_int64(0)
    assert lib.tinym_mxfp4_scale_bytes(1, 4, 48, ctypes.byref(out)) == 2
    assert lib.tinym_mxfp4_scale_bytes(1, 0, 64, ctypes.byref(out)) == 1
    assert lib.tinym_mxfp4_scale_bytes(1 << 20, 1 << 20, 64, ctypes.byref(out)) == 2
    assert lib.tinym_mxfp4_scale_bytes(1, 4, 64, None) == 1
    for fn, args in ((lib.tinym_mxfp4_quantize, lambda a, d, c, s: (a, d, c, s)),
                     (lib.tinym_mxfp4_dequantize, lambda a, d, c, s: (c, s, a, d))):
        assert fn(*args(None, 1, P, P), 1, 4, 64, None) == 1
        assert fn(*args(P, 1, None, P), 1, 4, 64, None) == 1
        assert fn(*args(P, 1, P, None), 1, 4, 64, None) == 1
        assert fn(*args(P, 3, P, P), 1, 4, 64, None) == 1
        assert fn(*args(P, 1, P, P), 1, 4, 40, None) == 2
        assert fn(*args(P + 8, 1, P, P), 1, 4, 64, None) == 3
        assert fn(*args(P, 1, P + 8, P), 1, 4, 64, None) == 3
        assert fn(*args(P, 1, P, P + 8), 1, 4, 64, None) == 3


def test_ops_refuse_cpu_tensors():
    import torch

    import candidate_kernel as ck

    a = torch.zeros(4, 64, dtype=torch.uint8)
    s = torch.zeros(1, 1, 512, dtype=torch.uint8)
    with pytest.raises(NotImplementedError):
        ck.mxfp4_quantize(torch.zeros(4, 64))
    with pytest.raises(NotImplementedError):
        ck.mxfp4_dequantize(a, s)
    with pytest.raises(NotImplementedError):
        ck.mxfp4_gemm(a, s, a, s)
