"""GPU: the grouped and MXFP4 kernels where two of them meet, and where a wait
runs out."""

from __future__ import annotations

import pytest

from test_gpu_grouped import fp8, offsets_of, quantized

pytestmark = pytest.mark.gpu


# (rows, experts, n, k): stream, folded and pair kernel, K of fewer and of more
# stages than the ring holds
LOST = [(40, 4, 300, 160), (40, 4, 300, 6144), (2, 2, 1000, 2048), (2, 2, 1000, 16384), (700, 2, 600, 96),
        (700, 2, 600, 4096)]


@pytest.mark.parametrize("rows,experts,n,k", LOST)
@pytest.mark.parametrize("lost", [0, 1, 2])
@pytest.mark.parametrize("mx", [False, True])
def test_lost_copies_products_and_commits_are_reported(cuda_device, rows, experts, n, k, lost, mx):
    """Whatever does not happen: every wait for it ends after its limit, what
    is in flight is waited for, the next call raises, and the one after that is
    right again."""
    import torch

    import candidate_kernel as ck
    import tinym_b200 as t

    off = offsets_of([1] * (experts - 1) + [rows - experts + 1])
    if mx:
        a, sa = quantized((rows, k), 1)
        b, sb = quantized((experts, n, k), 2)
        call = lambda: ck.mxfp4_gemm_grouped(a, sa, b, sb, off)
    else:
        a, b, sa, sb = fp8((rows, k), 1), fp8((experts, n, k), 2), None, None
        one = torch.ones(1, device="cuda")
        call = lambda: ck.fp8_gemm_grouped(a, b, one, off)
    want = call()
    torch.cuda.synchronize()
    assert t.device_status(clear=True) == 0
    y = torch.empty_like(want)
    lib = t.capi()
    for _ in range(2):
        st = lib.tinym_selftest_grouped_lost(lost, a.data_ptr(), sa.data_ptr() if mx else None, b.data_ptr(),
                                             sb.data_ptr() if mx else None, y.data_ptr(), rows, experts, n, k,
                                             off.data_ptr(), 2_000_000, torch.cuda.current_stream().cuda_stream)
        assert st == 0, lib.tinym_last_error()
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="TINYM_ERR_DEVICE_TIMEOUT"):
            call()
    assert torch.equal(call(), want)
    assert t.device_status(clear=True) != 0
    assert t.device_status() == 0 and t.pending_errors() == 0
