"""GPU: grouped FP8 product, MXFP4 quantise / dequantise, MXFP4 products.

Products are compared with 64-bit ones of the same operands.  Tolerance, per
value: the rounding to BF16 is off by at most 2^-8 of the value; the FP32 sum
of K products of magnitude |a_k b_k|, each addition off by at most 2^-23 of
its result (2^-24 for rounding, twice that for truncation), by at most
K 2^-23 sum |a_k b_k|; alpha's product by 2^-24 of the value, inside the
slack between 2^-8 and the BF16 half step 2^-9.  Quantisation is exact.
"""

from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- 64-bit references
LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def mx_values(codes, scales):
    """[R, K/2] codes and their blocked scales -> float64 values."""
    import torch

    lv = torch.tensor(LEVELS + [-v for v in LEVELS], dtype=torch.float64, device=codes.device)
    v = torch.stack([lv[(codes & 15).long()], lv[(codes >> 4).long()]], -1).reshape(codes.shape[0], -1)
    r = torch.arange(v.shape[0], device=codes.device)[:, None]
    c = torch.arange(v.shape[1] // 32, device=codes.device)[None, :]
    s = scales[r // 128, c // 4, (r % 32) * 16 + (r // 32 % 4) * 4 + c % 4].double()
    s = torch.where(s == 255, torch.nan, torch.exp2(s - 127))
    return v * s.repeat_interleave(32, 1)


def mx_codes(x):
    """float [R, K] -> (codes, scale bytes [R, K/32]) by the definition, in 64 bits."""
    import torch

    v = x.double().reshape(x.shape[0], -1, 32)
    top = v.abs().amax(-1)
    bad = ~torch.isfinite(v).all(-1)
    e = torch.frexp(torch.where(bad | (top == 0), 1.0, top))[1] - 3
    e = torch.where(top == 0, -127, e.clamp(-127, 127))
    u = v / torch.exp2(e.double())[..., None]
    u = torch.where(bad[..., None], 0.0, u)
    levels = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)
    d = (u.abs().clamp(max=6.0)[..., None] - levels).abs()
    near = d.amin(-1, keepdim=True) == d
    even = torch.arange(8, device=x.device) % 2 == 0  # ties go to the even code
    code = torch.where((near & even).any(-1), (near & even).int().argmax(-1), near.int().argmax(-1))
    code = code | (torch.signbit(v) & ~bad[..., None]).long() << 3
    code = code.reshape(x.shape[0], -1)
    byte = torch.where(bad, 255, e + 127)
    return (code[:, 0::2] | code[:, 1::2] << 4).to(torch.uint8), byte.to(torch.uint8)


def row_scales(scales, rows, cols):
    import torch

    r = torch.arange(rows, device=scales.device)[:, None]
    c = torch.arange(cols, device=scales.device)[None, :]
    return scales[r // 128, c // 4, (r % 32) * 16 + (r // 32 % 4) * 4 + c % 4]


def scale_block(byte):
    """Row scales [R, C] in the blocked layout."""
    import torch

    r, c = byte.shape
    full = torch.zeros(-(-r // 128) * 128, -(-c // 4) * 4, dtype=torch.uint8, device=byte.device)
    full[:r, :c] = byte
    return full.reshape(-1, 4, 32, full.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).reshape(
        -1, full.shape[1] // 4, 512).contiguous()


def check(y, a, b, alpha=1.0):
    """y [R, N] against alpha a b^T of float64 a [R, K], b [N, K]."""
    import torch

    want = alpha * (a @ b.T)
    tol = 2.0 ** -8 * want.abs() + a.shape[1] * 2.0 ** -23 * abs(alpha) * (a.abs() @ b.abs().T)
    bad = ~((y.double() - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), y[bad][:4], want[bad][:4])


def gen(seed):
    import torch

    return torch.Generator("cuda").manual_seed(seed)


def fp8(shape, seed):
    import torch

    return (torch.randn(shape, generator=gen(seed), device="cuda") * 3).to(torch.float8_e4m3fn)


def offsets_of(counts, first=0):
    import torch

    o = [first]
    for c in counts:
        o.append(o[-1] + c)
    return torch.tensor(o, dtype=torch.int32, device="cuda")


def quantized(shape, seed):
    """Random MXFP4 operand with the framework's layout, from random codes and
    scales (every code, scales over 2^-6 .. 2^6)."""
    import torch

    g = gen(seed)
    *lead, rows, k = shape
    codes = torch.randint(0, 256, (*lead, rows, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.randint(121, 134, (*lead, -(-rows // 128), -(-k // 128), 512), generator=g,
                           device="cuda", dtype=torch.uint8)
    return codes, scales


# (counts, spare, n, k): one row to hundreds per group, empty groups, odd sizes
GROUPS = [
    ([1], 0, 1, 32),
    ([1, 0, 1], 0, 64, 512),
    ([3, 0, 17, 1], 2, 200, 1024),
    ([0, 0, 5], 0, 2050, 2080),
    ([16, 33, 0, 64, 7], 1, 130, 1184),
    ([2] * 40, 0, 257, 544),
    ([0] * 70 + [1, 2], 3, 96, 4096),
    ([128], 0, 128, 256),
    ([300, 0, 57, 129], 5, 333, 672),
    ([257], 0, 1000, 1568),
    ([1, 700], 0, 384, 4128),
    ([130], 0, 1, 32),
    ([0, 191, 193, 385], 0, 129, 96),
    # few rows, K of whole 128-byte chunks: segments of K side by side in an MMA
    ([1], 0, 2050, 6144),
    ([16], 0, 1000, 1536),
    ([7], 1, 640, 3584),
    ([1, 0, 0, 2, 0, 1, 0, 0], 0, 1024, 2048),
    ([0, 3, 17, 0, 1], 2, 500, 1024),
    ([0] * 9 + [9], 0, 333, 768),
    ([0] * 1000 + [3, 0, 70, 1], 0, 24, 160),
]


@pytest.mark.parametrize("counts,spare,n,k", GROUPS)
@pytest.mark.parametrize("per_expert", [False, True])
def test_fp8_gemm_grouped(cuda_device, counts, spare, n, k, per_expert):
    import torch

    import candidate_kernel as ck

    if k % 256:
        k += 16  # K a multiple of 16 only
    rows, e = sum(counts) + spare, len(counts)
    a, b = fp8((rows, k), 1), fp8((e, n, k), 2)
    alpha = torch.rand(e if per_expert else 1, generator=gen(3), device="cuda") / 64
    off = offsets_of(counts)
    y = ck.fp8_gemm_grouped(a, b, alpha, off)
    assert y.dtype == torch.bfloat16 and y.shape == (rows, n)
    at = 0
    for i, c in enumerate(counts):
        check(y[at:at + c], a[at:at + c].double(), b[i].double(), float(alpha[i if per_expert else 0]))
        at += c
    assert not y[at:].any()


@pytest.mark.parametrize("counts,spare,n,k", GROUPS)
def test_mxfp4_gemm_grouped(cuda_device, counts, spare, n, k):
    import torch

    import candidate_kernel as ck

    rows, e = sum(counts) + spare, len(counts)
    a, sa = quantized((rows, k), 1)
    b, sb = quantized((e, n, k), 2)
    alpha = torch.rand(e, generator=gen(3), device="cuda")
    y = ck.mxfp4_gemm_grouped(a, sa, b, sb, offsets_of(counts), alpha)
    va = mx_values(a, sa)
    at = 0
    for i, c in enumerate(counts):
        check(y[at:at + c], va[at:at + c], mx_values(b[i], sb[i]), float(alpha[i]))
        at += c
    assert not y[at:].any()


@pytest.mark.parametrize("m,n,k", [(1, 1, 32), (1, 5120, 6144), (3, 100, 96), (16, 129, 128), (17, 2000, 160),
                                   (64, 300, 2048), (65, 1000, 1056), (193, 257, 512), (512, 384, 1312)])
def test_mxfp4_gemm(cuda_device, m, n, k):
    import torch

    import candidate_kernel as ck

    a, sa = quantized((m, k), 4)
    b, sb = quantized((n, k), 5)
    check(ck.mxfp4_gemm(a, sa, b, sb), mx_values(a, sa), mx_values(b, sb))
    alpha = torch.tensor([-0.37], device="cuda")
    check(ck.mxfp4_gemm(a, sa, b, sb, alpha), mx_values(a, sa), mx_values(b, sb), float(alpha))


@pytest.mark.parametrize("byte", [0, 40, 100, 254])
def test_mxfp4_scale_range(cuda_device, byte):
    """Scales far from 1: the other side's are chosen so that the products fit FP32."""
    import candidate_kernel as ck

    a, sa = quantized((20, 256), 4)
    b, sb = quantized((140, 256), 5)
    sa.fill_(byte)
    sb.fill_(254 - byte)
    check(ck.mxfp4_gemm(a, sa, b, sb), mx_values(a, sa), mx_values(b, sb))


# ---------------------------------------------------------------- quantisation
@pytest.mark.parametrize("dtype_name", ["bfloat16", "float32"])
@pytest.mark.parametrize("shape", [(1, 32), (3, 96), (130, 160), (128, 128), (257, 6144), (2, 5, 64), (3, 129, 416)])
def test_mxfp4_quantize(cuda_device, dtype_name, shape):
    import torch

    import candidate_kernel as ck

    x = torch.randn(shape, generator=gen(6), device="cuda")
    x *= torch.exp2(torch.randint(-20, 20, (*shape[:-1], 1), generator=gen(7), device="cuda").float())
    x = x.to(getattr(torch, dtype_name))
    codes, scales = ck.mxfp4_quantize(x)
    flat = [(x, codes, scales)] if x.dim() == 2 else list(zip(x, codes, scales))
    for xi, ci, si in flat:
        want, byte = mx_codes(xi)
        assert torch.equal(ci, want)
        assert torch.equal(row_scales(si, *byte.shape), byte)
        rows, cols = si.shape[0] * 128, si.shape[1] * 4
        every = row_scales(si, rows, cols)
        assert not every[byte.shape[0]:].any() and not every[:, byte.shape[1]:].any()  # padding
        for out in (torch.bfloat16, torch.float32):
            assert torch.equal(ck.mxfp4_dequantize(ci, si, out).double(), mx_values(ci, si))
    back = ck.mxfp4_dequantize(codes, scales, torch.float32)
    assert back.shape == x.shape


def test_mxfp4_quantize_special_values(cuda_device):
    """Ties, zeros of both signs, the ends of the range, NaN and infinity."""
    import torch

    import candidate_kernel as ck

    rows = []
    ties = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.99, 0.0, -0.0, 4.0]
    for scale in (1.0, 2.0 ** -126, 2.0 ** 120):
        rows.append([v * scale for v in ties] + [-v * scale for v in ties] + [4.0 * scale] * 6)
    rows.append([0.0] * 31 + [-0.0])
    rows.append([2.0 ** -149] * 16 + [-(2.0 ** -140)] * 16)
    rows.append([2.0 ** -127, 2.0 ** -128, 2.0 ** -129, 3 * 2.0 ** -128] + [0.0] * 28)
    rows.append([3.4028234663852886e38, -3.4028234663852886e38, 2.0 ** 127] + [1.0] * 29)
    rows.append([1.0, math.nan] + [2.0] * 30)
    rows.append([math.inf] + [1.0] * 31)
    rows.append([1.0] * 31 + [-math.inf])
    x = torch.tensor(rows, dtype=torch.float32, device="cuda")
    x = torch.cat([x, torch.ones_like(x)], 1)  # a neighbour block is not touched
    codes, scales = ck.mxfp4_quantize(x)
    want, byte = mx_codes(x)
    assert torch.equal(codes, want)
    assert torch.equal(row_scales(scales, *byte.shape), byte)
    back = ck.mxfp4_dequantize(codes, scales, torch.float32)
    assert torch.equal(back.isnan(), mx_values(codes, scales).isnan())
    keep = ~back.isnan()
    assert torch.equal(back[keep].double(), mx_values(codes, scales)[keep])


@pytest.mark.parametrize("dtype_name", ["bfloat16", "float32"])
def test_mxfp4_dequantize_every_code_and_scale(cuda_device, dtype_name):
    """Exact wherever the type can hold the value (6 * 2^127 becomes infinite)."""
    import torch

    import candidate_kernel as ck

    dtype = getattr(torch, dtype_name)
    codes = torch.arange(256, device="cuda").to(torch.uint8).reshape(16, 16).repeat(16, 8)  # [256, 128]
    scales = torch.arange(256, device="cuda").to(torch.uint8)  # row r: scale r
    rows = scales[:, None].expand(256, 8)
    blocked = rows.reshape(2, 4, 32, 2, 4).permute(0, 3, 2, 1, 4).reshape(2, 2, 512).contiguous()
    got = ck.mxfp4_dequantize(codes, blocked, dtype)
    want = mx_values(codes, blocked).to(dtype)
    nan = want.isnan()
    assert torch.equal(got.isnan(), nan) and nan.any() and want.isinf().any()
    assert torch.equal(got[~nan], want[~nan])


def test_nan_stays_in_its_row(cuda_device):
    """NaN in one row of X reaches that row alone; NaN in an expert without
    rows, in spare rows and in the scales' padding reaches nothing."""
    import torch

    import candidate_kernel as ck

    counts, n, k = [5, 0, 40], 300, 224
    off = offsets_of(counts)
    x = torch.randn(48, k, generator=gen(8), device="cuda")
    x[7, 3] = math.nan
    x[45:] = math.nan
    a, sa = ck.mxfp4_quantize(x)
    w = torch.randn(3, n, k, generator=gen(9), device="cuda")
    w[1] = math.nan
    b, sb = ck.mxfp4_quantize(w)
    for s, rows in ((sa, 48), (sb[0], n), (sb[2], n)):  # fill the padding with NaN scales
        full = torch.full((s.shape[0] * 128, s.shape[1] * 4), 255, dtype=torch.uint8, device="cuda")
        full[:rows, :k // 32] = row_scales(s, rows, k // 32)
        s.copy_(full.reshape(s.shape[0], 4, 32, s.shape[1], 4).permute(0, 3, 2, 1, 4).reshape(s.shape))
    y = ck.mxfp4_gemm_grouped(a, sa, b, sb, off)
    nan = y.isnan()
    assert nan[7].all() and not nan[:7].any() and not nan[8:].any()
    assert not y[45:].any()
    a8 = x.nan_to_num(0.0).to(torch.float8_e4m3fn)
    a8[7, 3] = math.nan
    b8 = w.to(torch.float8_e4m3fn)
    y = ck.fp8_gemm_grouped(a8, b8, torch.ones(1, device="cuda"), off)
    nan = y.isnan()
    assert nan[7].all() and not nan[:7].any() and not nan[8:].any()


# ---------------------------------------------------------------- how they are called
@pytest.mark.parametrize("counts", [[2, 0, 3], [100, 0, 150]])
def test_out_keeps_rows_of_no_group(cuda_device, counts):
    """out= with a wider row stride: rows of no group and columns past N stay."""
    import torch

    import candidate_kernel as ck

    n, k, rows = 70, 320, sum(counts) + 6
    off = offsets_of(counts, first=2)
    a, b = fp8((rows, k), 1), fp8((3, n, k), 2)
    alpha = torch.tensor([0.01], device="cuda")
    wide = torch.full((rows, n + 9), 7.0, dtype=torch.bfloat16, device="cuda")
    got = ck.fp8_gemm_grouped(a, b, alpha, off, out=wide[:, :n])
    assert got.data_ptr() == wide.data_ptr()
    fresh = ck.fp8_gemm_grouped(a, b, alpha, off)
    last = 2 + sum(counts)
    assert torch.equal(wide[2:last, :n], fresh[2:last])
    assert (wide[:2] == 7).all() and (wide[last:] == 7).all() and (wide[:, n:] == 7).all()
    assert not fresh[:2].any() and not fresh[last:].any()
    ac, sa = ck.mxfp4_quantize(a.float())
    bc, sb = ck.mxfp4_quantize(b.float())
    wide.fill_(7.0)
    ck.mxfp4_gemm_grouped(ac, sa, bc, sb, off, out=wide[:, :n])
    assert torch.equal(wide[2:last, :n], ck.mxfp4_gemm_grouped(ac, sa, bc, sb, off)[2:last])
    assert (wide[:2] == 7).all() and (wide[last:] == 7).all() and (wide[:, n:] == 7).all()
    one = torch.full((rows, n + 9), 7.0, dtype=torch.bfloat16, device="cuda")
    ck.mxfp4_gemm(ac, sa, bc[0], sb[0], out=one[:, :n])
    assert torch.equal(one[:, :n], ck.mxfp4_gemm(ac, sa, bc[0], sb[0])) and (one[:, n:] == 7).all()


@pytest.mark.parametrize("n", [1024, 1003])
def test_padded_batch(cuda_device, n):
    """A row buffer of which a few rows are in use, in the middle: the others
    are zeros, whatever X holds there."""
    import torch

    import candidate_kernel as ck

    k, rows = 512, 900
    off = offsets_of([3, 0, 70], first=400)
    x = torch.full((rows, k), math.nan, device="cuda")
    x[400:473] = torch.randn(73, k, generator=gen(1), device="cuda")
    w = torch.randn(3, n, k, generator=gen(2), device="cuda")
    a, b = x.to(torch.float8_e4m3fn), w.to(torch.float8_e4m3fn)
    y = ck.fp8_gemm_grouped(a, b, torch.ones(1, device="cuda"), off)
    assert not y[:400].any() and not y[473:].any()
    check(y[400:403], a[400:403].double(), b[0].double())
    check(y[403:473], a[403:473].double(), b[2].double())
    (ac, sa), (bc, sb) = ck.mxfp4_quantize(x), ck.mxfp4_quantize(w)
    y = ck.mxfp4_gemm_grouped(ac, sa, bc, sb, off)
    assert not y[:400].any() and not y[473:].any()
    check(y[400:403], mx_values(ac, sa)[400:403], mx_values(bc[0], sb[0]))
    check(y[403:473], mx_values(ac, sa)[403:473], mx_values(bc[2], sb[2]))


@pytest.mark.parametrize("rows", [12, 400])
def test_offsets_outside_the_rows(cuda_device, rows):
    """Offsets that are not sorted or point outside are clamped, as documented."""
    import torch

    import candidate_kernel as ck

    n, k = 96, 256
    a, b = fp8((rows, k), 1), fp8((4, n, k), 2)
    one = torch.ones(1, device="cuda")
    raw = [-5, rows // 3, 1, rows // 2, rows + 1000]
    fixed, top = [], 0
    for v in raw:
        top = max(top, min(max(v, 0), rows))
        fixed.append(top)
    y = ck.fp8_gemm_grouped(a, b, one, torch.tensor(raw, dtype=torch.int32, device="cuda"))
    for i in range(4):
        check(y[fixed[i]:fixed[i + 1]], a[fixed[i]:fixed[i + 1]].double(), b[i].double())


def test_empty(cuda_device):
    import torch

    import candidate_kernel as ck

    one = torch.ones(1, device="cuda")
    off = torch.zeros(3, dtype=torch.int32, device="cuda")
    assert ck.fp8_gemm_grouped(fp8((0, 64), 1), fp8((2, 8, 64), 2), one, off).shape == (0, 8)
    assert not ck.fp8_gemm_grouped(fp8((5, 64), 1), fp8((2, 8, 64), 2), one, off).any()
    codes, scales = ck.mxfp4_quantize(torch.zeros(0, 64, device="cuda"))
    assert codes.shape == (0, 32) and scales.shape == (0, 1, 512)
    assert ck.mxfp4_dequantize(codes, scales).shape == (0, 64)
    b, sb = ck.mxfp4_quantize(torch.ones(8, 64, device="cuda"))
    assert ck.mxfp4_gemm(codes, scales, b, sb).shape == (0, 8)


@pytest.mark.parametrize("rows", [4, 24, 600])
def test_results_are_reproducible(cuda_device, rows):
    """The same bits in every run, and for a row whatever groups the other rows
    of the call are in."""
    import torch

    import candidate_kernel as ck

    n, k = 1100, 1536
    a, sa = quantized((rows, k), 1)
    b, sb = quantized((3, n, k), 2)
    a8, b8 = fp8((rows, k), 3), fp8((3, n, k), 4)
    one = torch.ones(1, device="cuda")
    first = rows // 4
    off = offsets_of([first, rows - first, 0])
    y, y8 = ck.mxfp4_gemm_grouped(a, sa, b, sb, off), ck.fp8_gemm_grouped(a8, b8, one, off)
    for _ in range(3):
        assert torch.equal(y, ck.mxfp4_gemm_grouped(a, sa, b, sb, off))
        assert torch.equal(y8, ck.fp8_gemm_grouped(a8, b8, one, off))
    for second in (1, rows // 2):
        off = offsets_of([first, second, rows - first - second])
        assert torch.equal(y[:first + second], ck.mxfp4_gemm_grouped(a, sa, b, sb, off)[:first + second])
        assert torch.equal(y8[:first + second], ck.fp8_gemm_grouped(a8, b8, one, off)[:first + second])


def test_captured_graph_replays_with_other_groups(cuda_device):
    import torch

    import candidate_kernel as ck

    n, k, rows = 520, 512, 40
    x = torch.randn(rows, k, generator=gen(1), device="cuda").bfloat16()
    w, sw = ck.mxfp4_quantize(torch.randn(4, n, k, generator=gen(2), device="cuda").bfloat16())
    b = fp8((4, n, k), 3)
    alpha = torch.full((4,), 0.01, device="cuda")
    off = offsets_of([10, 10, 10, 10])

    def step():
        codes, scales = ck.mxfp4_quantize(x)
        return (ck.mxfp4_gemm_grouped(codes, scales, w, sw, off),
                ck.fp8_gemm_grouped(x.to(torch.float8_e4m3fn), b, alpha, off),
                ck.mxfp4_dequantize(codes, scales))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for counts in ([10, 10, 10, 10], [0, 1, 33, 2], [40, 0, 0, 0], [0, 0, 0, 3]):
        off.copy_(offsets_of(counts))
        x.copy_(torch.randn(rows, k, generator=gen(sum(counts) + 7), device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        for g, want in zip(got, step()):
            assert torch.equal(g, want), counts


def test_two_streams_at_once(cuda_device):
    import torch

    import candidate_kernel as ck

    cases = [([1, 2, 0, 5], 1000, 2048), ([200, 0, 90, 30], 640, 1024)]
    made = []
    for i, (counts, n, k) in enumerate(cases):
        a, sa = quantized((sum(counts), k), 10 + i)
        b, sb = quantized((len(counts), n, k), 20 + i)
        made.append((a, sa, b, sb, offsets_of(counts)))
    want = [ck.mxfp4_gemm_grouped(*m) for m in made]
    streams = [torch.cuda.Stream() for _ in made]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ck.mxfp4_gemm_grouped(*made[i]))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, y) for y in g)


def test_offsets_past_32_bits(cuda_device):
    """Values of Y, bytes of W and values of X behind 2^32."""
    import torch

    import candidate_kernel as ck

    n, k, rows = 8192, 128, 530_000  # Y: 4.3e9 values
    a, b = fp8((rows, k), 1), fp8((2, n, k), 2)
    one, off = torch.ones(1, device="cuda"), offsets_of([rows - 300, 300])
    y = ck.fp8_gemm_grouped(a, b, one, off)
    check(y[-300:], a[-300:].double(), b[1].double())
    check(y[-600:-300], a[-600:-300].double(), b[0].double())
    del y
    torch.cuda.empty_cache()
    experts, n, k = 40, 8192, 14336  # W: 4.7e9 bytes
    b = torch.zeros(experts, n, k, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)
    b[-1] = fp8((n, k), 3)
    for c in (2, 100):
        a = fp8((c, k), 4)
        off = offsets_of([0] * (experts - 1) + [c])
        check(ck.fp8_gemm_grouped(a, b, one, off), a.double(), b[-1].double())
    del b
    torch.cuda.empty_cache()
    x = torch.zeros(700_000, 6144, device="cuda", dtype=torch.bfloat16)  # 4.3e9 values
    x[-200:] = torch.randn(200, 6144, generator=gen(5), device="cuda").bfloat16()
    codes, scales = ck.mxfp4_quantize(x)
    want, byte = mx_codes(x[-200:])
    assert torch.equal(codes[-200:], want)
    tail = row_scales(scales[-3:], 3 * 128, 192)
    last = x.shape[0] - (scales.shape[0] - 3) * 128
    assert torch.equal(tail[last - 200:last], byte)
    del x
    back = ck.mxfp4_dequantize(codes, scales)
    assert torch.equal(back[-200:].double(), mx_values(codes[-200:], scale_block(byte)))


@pytest.mark.parametrize("rows,experts,n,k", [(2, 2, 1000, 2048), (40, 4, 300, 1024), (700, 2, 600, 1024)])
def test_waits_that_run_out_are_reported(cuda_device, rows, experts, n, k):
    """Folded, stream and pair kernel: without copies every wait ends after its
    limit, the next call raises, and the one after that is right again."""
    import torch

    import candidate_kernel as ck
    import tinym_b200 as t

    a, b = fp8((rows, k), 1), fp8((experts, n, k), 2)
    one, off = torch.ones(1, device="cuda"), offsets_of([1] * (experts - 1) + [rows - experts + 1])
    want = ck.fp8_gemm_grouped(a, b, one, off)
    torch.cuda.synchronize()
    assert t.device_status(clear=True) == 0
    y = torch.empty_like(want)
    lib = t.capi()
    st = lib.tinym_selftest_grouped_timeout(a.data_ptr(), b.data_ptr(), y.data_ptr(), rows, experts, n, k,
                                            off.data_ptr(), 2_000_000,
                                            torch.cuda.current_stream().cuda_stream)
    assert st == 0, lib.tinym_last_error()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="TINYM_ERR_DEVICE_TIMEOUT"):
        ck.fp8_gemm_grouped(a, b, one, off)
    assert torch.equal(ck.fp8_gemm_grouped(a, b, one, off), want)
    assert t.device_status(clear=True) != 0
    assert t.device_status() == 0 and t.pending_errors() == 0


def test_refusals(cuda_device):
    import torch

    import candidate_kernel as ck

    a, b = fp8((8, 64), 1), fp8((2, 32, 64), 2)
    one, off = torch.ones(1, device="cuda"), offsets_of([4, 4])
    bad = [
        (a.float(), b, one, off), (a, b.float(), one, off), (a[:, :32], b, one, off), (a, b[0], one, off),
        (a, fp8((2, 32, 80), 1), one, off), (a, b, one.double(), off), (a, b, torch.ones(3, device="cuda"), off),
        (a, b, one.cpu(), off), (a, b, one, off.long()), (a, b, one, off[:2]), (a, b, one, off.cpu()),
        (a.T, b, one, off), (fp8((8, 40), 1), fp8((2, 32, 40), 1), one, off),
        (fp8((8 * 64 + 8,), 1)[8:].view(8, 64), b, one, off),  # 8-byte aligned
    ]
    for args in bad:
        with pytest.raises((RuntimeError, NotImplementedError)):
            ck.fp8_gemm_grouped(*args)
    for out in (torch.empty(8, 32, device="cuda"), torch.empty(8, 31, device="cuda").bfloat16(),
                torch.empty(32, 8, device="cuda").bfloat16().T, torch.empty(8, 32).bfloat16(),
                torch.empty(1, 32, device="cuda").bfloat16().expand(8, 32)):
        with pytest.raises(RuntimeError):
            ck.fp8_gemm_grouped(a, b, one, off, out=out)
    for x in (torch.zeros(4, 48, device="cuda"), torch.zeros(64, device="cuda"),
              torch.zeros(4, 64, device="cuda").half(), torch.zeros(64, 4, device="cuda").T):
        with pytest.raises(RuntimeError):
            ck.mxfp4_quantize(x)
    c, s = ck.mxfp4_quantize(torch.ones(8, 64, device="cuda"))
    w, sw = ck.mxfp4_quantize(torch.ones(2, 32, 64, device="cuda"))
    for args in [(c.int(), s), (c, s[:, :, :256]), (c[:, :8], s), (c, s.float()), (c, s, torch.float16), (c, s.cpu())]:
        with pytest.raises(RuntimeError):
            ck.mxfp4_dequantize(*args)
    for args in [(c, s, w, sw), (c, s, w[0], sw), (c, s, w[0, :, :16].contiguous(), sw[0]),
                 (c, s, w[0], sw[0], torch.ones(2, device="cuda"))]:
        with pytest.raises(RuntimeError):
            ck.mxfp4_gemm(*args)
    for args in [(c, s, w[0], sw[0], off), (c, s, w, sw[0], off), (c, s, w, sw, off[:2]),
                 (c, s, w, sw, off, torch.ones(3, device="cuda"))]:
        with pytest.raises(RuntimeError):
            ck.mxfp4_gemm_grouped(*args)


def test_mixture_of_experts_layer(cuda_device):
    """The operators as a layer uses them: route, sort the rows by expert,
    quantise, two grouped products with an activation between, weigh and add.
    Compared with the same layer in 64 bits on the dequantised operands; every
    product adds the tolerance above, the second one also the first's error
    through its quantisation, so the layer is compared product by product."""
    import torch

    import candidate_kernel as ck

    tokens, top, experts, k, h = 37, 2, 6, 512, 768
    x = torch.randn(tokens, k, generator=gen(1), device="cuda").bfloat16()
    w1, s1 = ck.mxfp4_quantize(torch.randn(experts, 2 * h, k, generator=gen(2), device="cuda").bfloat16())
    w2, s2 = ck.mxfp4_quantize(torch.randn(experts, k, h, generator=gen(3), device="cuda").bfloat16())
    weight, expert = torch.randn(tokens, experts, generator=gen(4), device="cuda").softmax(-1).topk(top)
    order = expert.flatten().argsort(stable=True)
    off = torch.zeros(experts + 1, dtype=torch.int32, device="cuda")
    off[1:] = torch.bincount(expert.flatten(), minlength=experts).cumsum(0)
    rows = x[order // top]
    a, sa = ck.mxfp4_quantize(rows)
    up = ck.mxfp4_gemm_grouped(a, sa, w1, s1, off)
    act = (torch.nn.functional.silu(up[:, :h].float()) * up[:, h:].float()).bfloat16()
    d, sd = ck.mxfp4_quantize(act)
    down = ck.mxfp4_gemm_grouped(d, sd, w2, s2, off)
    y = torch.zeros(tokens, k, device="cuda").index_add_(
        0, order // top, down.float() * weight.flatten()[order][:, None])
    assert torch.isfinite(y).all()
    o = off.tolist()
    for e in range(experts):
        r = slice(o[e], o[e + 1])
        check(up[r], mx_values(a, sa)[r], mx_values(w1[e], s1[e]))
        check(down[r], mx_values(d, sd)[r], mx_values(w2[e], s2[e]))
    # the same rows through the E4M3 path
    sx = rows.float().abs().amax() / 448
    sw = ck.mxfp4_dequantize(w1, s1, torch.float32)
    scale = sw.abs().amax((1, 2)) / 448
    b8 = (sw / scale[:, None, None]).to(torch.float8_e4m3fn)
    a8 = (rows.float() / sx).to(torch.float8_e4m3fn)
    up8 = ck.fp8_gemm_grouped(a8, b8, sx * scale, off)
    for e in range(experts):
        r = slice(o[e], o[e + 1])
        check(up8[r], a8[r].double(), b8[e].double(), float((sx * scale)[e]))
