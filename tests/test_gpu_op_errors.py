"""GPU: a refused torch-op call whose message holds numbers raises RuntimeError."""

from __future__ import annotations

import pytest


@pytest.mark.gpu
def test_packed_size_mismatch_raises(cuda_device):
    import torch

    import candidate_kernel as ck

    ck.build()
    a = torch.zeros(1, 256, device=cuda_device).to(torch.float8_e4m3fn)
    packed = torch.zeros(1000, dtype=torch.uint8, device=cuda_device)
    with pytest.raises(RuntimeError, match="1000 bytes"):
        torch.ops.sm120_fp8_gemm.run_packed(a, packed, 128, 256, torch.ones(1, device=cuda_device))
