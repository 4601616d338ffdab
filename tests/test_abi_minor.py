"""CPU: a caller can tell which entry points a library has: those added since
TINYM_ABI_VERSION was raised last have a minor number."""

from __future__ import annotations

import re

from test_capi_host import HEADER


def test_minor_number():
    import tinym_b200

    text = HEADER.read_text()
    minor = int(re.search(r"#define TINYM_ABI_MINOR (\d+)", text).group(1))
    lib = tinym_b200.capi()
    assert lib.tinym_abi_minor() == minor >= 1
    # the header says which entry points came with which minor number
    block = text[:text.index("#define TINYM_ABI_MINOR")][-700:]
    for name in ("tinym_fp8_gemm_grouped", "tinym_mxfp4_gemm_grouped", "tinym_mxfp4_gemm",
                 "tinym_mxfp4_quantize", "tinym_mxfp4_dequantize", "tinym_mxfp4_scale_bytes",
                 "tinym_selftest_grouped_timeout", "tinym_selftest_grouped_lost", "tinym_abi_minor",
                 "TINYM_FLAG_ZERO_REST"):
        assert name in block, name
