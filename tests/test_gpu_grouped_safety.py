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


@pytest.mark.parametrize("mx", [False, True])
def test_short_pair_products_on_three_streams(cuda_device, mx):
    """Pair kernels of one chunk of K, beside each other and beside split-K
    clusters and stream kernels: every call ends and is right."""
    import torch

    import candidate_kernel as ck

    def make(counts, n, k, seed):
        off = offsets_of(counts)
        if mx:
            a, sa = quantized((sum(counts), k), seed)
            b, sb = quantized((len(counts), n, k), seed + 1)
            return lambda: ck.mxfp4_gemm_grouped(a, sa, b, sb, off)
        a, b = fp8((sum(counts), k), seed), fp8((len(counts), n, k), seed + 1)
        one = torch.ones(1, device="cuda")
        return lambda: ck.fp8_gemm_grouped(a, b, one, off)

    x, w = fp8((9, 6144), 7), fp8((5120, 6144), 8)
    alpha = torch.tensor([0.01], device="cuda")
    lanes = [[make([700, 0, 300], 2000, 96, 1)],
             [make([130], 5120, 64, 3), make([3, 5], 700, 128, 5)],
             [lambda: ck.fp8_gemm(x, w, alpha), make([400], 1000, 128, 9)]]
    want = [[f() for f in lane] for lane in lanes]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in lanes]
    got = []
    for _ in range(30):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, [f() for f in lanes[i]]))
    torch.cuda.synchronize()
    for i, outs in got:
        assert all(torch.equal(o, w) for o, w in zip(outs, want[i]))


@pytest.mark.parametrize("rows", [6, 50, 400, 1000])
def test_chain_of_kernels_that_start_early(cuda_device, rows):
    """quantise -> grouped product -> quantise -> product, each launched while
    the one before ends, captured and replayed on changing X and groups: no
    step sees what its buffers held before (folded, stream and pair plans)."""
    import torch

    import candidate_kernel as ck

    k, n = 512, 768
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.randn(rows, k, generator=g, device="cuda").bfloat16()
    w1, s1 = ck.mxfp4_quantize(torch.randn(4, n, k, generator=g, device="cuda"))
    w2, s2 = ck.mxfp4_quantize(torch.randn(k, n, generator=g, device="cuda"))
    off = offsets_of([rows - 3, 0, 2, 1])

    def step(wait):
        wait()
        a, sa = ck.mxfp4_quantize(x)
        wait()
        up = ck.mxfp4_gemm_grouped(a, sa, w1, s1, off)
        wait()
        d, sd = ck.mxfp4_quantize(up)
        wait()
        return up, d, ck.mxfp4_gemm(d, sd, w2, s2)

    step(torch.cuda.synchronize)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(lambda: None)
    for i in range(12):
        x.copy_(torch.randn(rows, k, generator=g, device="cuda") * 2.0 ** (i - 6))
        off.copy_(offsets_of([i % 4, rows - 3 - i % 4, 0, 3 if i % 2 else 1]))
        graph.replay()
        graph.replay()
        torch.cuda.synchronize()
        for have, want in zip(got, step(torch.cuda.synchronize)):
            assert torch.equal(have, want), i


@pytest.mark.parametrize("op", ["quantize", "dequantize"])
def test_conversions_raise_after_a_wait_that_ran_out(cuda_device, op):
    """The output of a product whose wait ran out is unspecified: quantising or
    expanding it raises, as every op does, instead of passing it on."""
    import torch

    import candidate_kernel as ck
    import tinym_b200 as t

    a, b, off = fp8((4, 512), 1), fp8((2, 64, 512), 2), offsets_of([2, 2])
    y = ck.fp8_gemm_grouped(a, b, torch.ones(1, device="cuda"), off)
    codes, scales = ck.mxfp4_quantize(y)
    call = {"quantize": lambda: ck.mxfp4_quantize(y), "dequantize": lambda: ck.mxfp4_dequantize(codes, scales)}[op]
    torch.cuda.synchronize()
    assert t.device_status(clear=True) == 0
    st = t.capi().tinym_selftest_grouped_lost(0, a.data_ptr(), None, b.data_ptr(), None, y.data_ptr(), 4, 2, 64,
                                              512, off.data_ptr(), 2_000_000,
                                              torch.cuda.current_stream().cuda_stream)
    assert st == 0
    torch.cuda.synchronize()
    try:
        with pytest.raises(RuntimeError, match="TINYM_ERR_DEVICE_TIMEOUT"):
            call()
        call()
    finally:
        t.device_status(clear=True)


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("rows,n", [(4, 8192), (40, 2000), (700, 1024)])
def test_sums_are_kept_in_32_bits(cuda_device, rows, n, mx):
    """Root mean square error against 64 bits, for the folded, stream and pair
    kernel.  BF16 rounds a value of [2^e, 2^(e + 1)) to a step of 2^(e - 7), so
    the rounding's rms is 2^(e - 8) / sqrt(3) <= 2^-8 / sqrt(3) of the value
    (5 % more for the spread of 30,000 values and more); each of K additions is
    off by at most 2^-23 of a partial sum, whose rms is at most the whole
    sum's, and rms values add up: K 2^-23.  An accumulator of 14 bits would be
    off by ten times as much."""
    import torch

    import candidate_kernel as ck
    from test_gpu_grouped import mx_values

    k = 6144
    if mx:
        a, sa = quantized((rows, k), 31)
        b, sb = quantized((n, k), 32)
        y, want = ck.mxfp4_gemm(a, sa, b, sb), mx_values(a, sa) @ mx_values(b, sb).T
    else:
        a, b = fp8((rows, k), 33), fp8((1, n, k), 34)
        y = ck.fp8_gemm_grouped(a, b, torch.ones(1, device="cuda"), offsets_of([rows]))
        want = a.double() @ b[0].double().T
    rms = lambda v: float(v.square().mean().sqrt())
    assert rms(y.double() - want) <= (1.05 * 2.0 ** -8 / 3 ** 0.5 + k * 2.0 ** -23) * rms(want)
