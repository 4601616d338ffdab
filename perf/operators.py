"""Measured cases of the grouped FP8 product and of the microscaled 4-bit (MXFP4) operators.

Operators (the framework's calls are those of ``candidate_kernel``):

* ``fp8_gemm_grouped``   rows of X sorted by expert, one E4M3 weight per expert;
* ``mxfp4_quantize`` and ``mxfp4_dequantize``: E2M1 elements, one power-of-two scale per 32;
* ``mxfp4_gemm``         product of two MXFP4 matrices;
* ``mxfp4_gemm_grouped`` the same with one weight per expert.

MXFP4 in memory: two E2M1 codes per byte, the even column in the low nibble.
A scale is an E8M0 byte (2^(byte - 127), 255 = NaN).  Scales lie in blocks of
128 rows x 4 scales (128 columns), 512 bytes each, [ceil(rows / 128)]
[ceil(K / 128)][32][4][4]: byte 16 * (r % 32) + 4 * (r // 32 % 4) + s of a block
is row r's scale s; bytes past the matrix are zero.

``run`` computes the plain form (elementary torch operations in 32 bits)
unless ``own`` is set.
"""

from __future__ import annotations

import math

import torch

own = False

_LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---------------------------------------------------------------- cases
def listed():
    return [
        # one token routed to two of eight small experts: launch latency
        {"name": "fp8 grouped one token", "op": "fp8_grouped", "experts": 8, "active": 2, "rows": 2,
         "spare": 0, "n": 2048, "k": 2048},
        # a decode batch over many experts, in a row buffer with spare rows
        {"name": "fp8 grouped decode", "op": "fp8_grouped", "experts": 32, "active": 28, "rows": 128,
         "spare": 8, "n": 2048, "k": 5120},
        # a prefill chunk over eight experts of the repository's 6144 x 5120 weight
        {"name": "fp8 grouped prefill", "op": "fp8_grouped", "experts": 8, "active": 8, "rows": 8192,
         "spare": 0, "n": 5120, "k": 6144},
        # an activation of one token
        {"name": "mxfp4 round trip row", "op": "round_trip", "experts": 0, "m": 1, "k": 6144,
         "dtype": "bfloat16"},
        # a ragged FP32 activation, K no multiple of 128
        {"name": "mxfp4 round trip odd", "op": "round_trip", "experts": 0, "m": 777, "k": 5152,
         "dtype": "float32"},
        # the weights of eight experts, laid out once at load time
        {"name": "mxfp4 round trip weights", "op": "round_trip", "experts": 8, "m": 5120, "k": 6144,
         "dtype": "bfloat16"},
        # decode of one token through the 6144 -> 5120 projection
        {"name": "mxfp4 gemm one row", "op": "gemm", "m": 1, "n": 5120, "k": 6144},
        # a decode batch, odd in every dimension
        {"name": "mxfp4 gemm odd batch", "op": "gemm", "m": 37, "n": 8190, "k": 5152},
        # a prefill chunk through the 5120 -> 16384 projection
        {"name": "mxfp4 gemm prefill", "op": "gemm", "m": 4096, "n": 16384, "k": 5120},
        # one token over sixteen small experts of odd sizes
        {"name": "mxfp4 grouped one token", "op": "mx_grouped", "experts": 16, "active": 2, "rows": 2,
         "spare": 0, "n": 2050, "k": 2080},
        # a decode batch over many experts
        {"name": "mxfp4 grouped decode", "op": "mx_grouped", "experts": 64, "active": 60, "rows": 256,
         "spare": 0, "n": 2000, "k": 4096},
        # a ragged prefill chunk, one expert without rows
        {"name": "mxfp4 grouped prefill", "op": "mx_grouped", "experts": 16, "active": 15, "rows": 7999,
         "spare": 1, "n": 5120, "k": 6144},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["fp8_grouped", "round_trip", "gemm", "mx_grouped"])
    step = 16 if op == "fp8_grouped" else 32
    k = max(step, _log(rng, 256, 8192) // step * step)
    if op == "round_trip":
        experts = rng.choice([0, 0, rng.randint(1, 8)])
        m = _log(rng, 1, 2 ** 26 // (k * max(1, experts)))
        return {"op": op, "experts": experts, "m": m, "k": k,
                "dtype": rng.choice(["bfloat16", "float32"])}
    n = _log(rng, 64, 8192)
    if op == "gemm":
        return {"op": op, "m": _log(rng, 1, 4096), "n": n, "k": k}
    experts = _log(rng, 1, max(1, min(64, 2 ** 28 // (n * k))))
    rows = _log(rng, 1, 6000)
    return {"op": op, "experts": experts, "active": rng.randint(1, min(experts, rows)), "rows": rows,
            "spare": rng.choice([0, 0, rng.randint(1, 64)]), "n": n, "k": k}


def work(case):
    op, k = case["op"], case["k"]
    if op == "round_trip":
        values = max(1, case["experts"]) * case["m"] * k
        wide = 2 if case["dtype"] == "bfloat16" else 4
        # quantise: values in, codes and scales out; dequantise: the reverse
        return {"bytes": 2 * values * wide + 2 * (values / 2 + values / 32), "flops": 4 * values}
    n = case["n"]
    per = 1.0 if op == "fp8_grouped" else 0.5 + 1 / 32  # bytes of an operand's element
    rows, weights = (case["m"], 1) if op == "gemm" else (case["rows"], case["active"])
    spare = case.get("spare", 0)
    return {"bytes": per * k * (rows + weights * n) + 2 * (rows + spare) * n,
            "flops": 2 * rows * n * k}


# ---------------------------------------------------------------- inputs
def _quantize(x):
    """MXFP4 codes (two per byte) and blocked scales of the last axis of x."""
    v = x.float()
    lead, k = v.shape[:-1], v.shape[-1]
    v = v.reshape(*lead, k // 32, 32)
    top = v.abs().amax(-1, keepdim=True)
    e = torch.where(top > 0, torch.frexp(top)[1] - 3, -127).clamp(-127, 127)
    u = torch.ldexp(v, -e).abs()
    # nearest level, ties to the even code
    code = ((u > 0.25).to(torch.uint8) + (u >= 0.75) + (u > 1.25) + (u >= 1.75) + (u > 2.5)
            + (u >= 3.5) + (u > 5.0)) | (torch.signbit(v).to(torch.uint8) << 3)
    code = code.reshape(*lead, k)
    return code[..., 0::2] | (code[..., 1::2] << 4), _block((e + 127).to(torch.uint8).reshape(*lead, k // 32))


def _block(s):
    rows, cols = s.shape[-2:]
    s = torch.nn.functional.pad(s, (0, -cols % 4, 0, -rows % 128))
    s = s.reshape(*s.shape[:-2], -1, 4, 32, s.shape[-1] // 4, 4)
    return s.transpose(-4, -2).reshape(*s.shape[:-5], s.shape[-5], s.shape[-2], 512).contiguous()


def _unblock(s, rows, cols):
    s = s.reshape(*s.shape[:-1], 32, 4, 4).transpose(-4, -2)
    return s.reshape(*s.shape[:-5], s.shape[-5] * 128, s.shape[-2] * 4)[..., :rows, :cols]


def _offsets(case, seed):
    """Row offsets of the experts: `active` of them have rows, unevenly."""
    g = torch.Generator().manual_seed(seed)
    e, a = case["experts"], case["active"]
    share = torch.rand(a, generator=g) ** 2 + 0.05
    count = torch.ones(a, dtype=torch.int64)
    more = torch.multinomial(share, case["rows"] - a, replacement=True, generator=g) if case["rows"] > a else count[:0]
    count += torch.bincount(more, minlength=a)
    full = torch.zeros(e, dtype=torch.int64)
    full[torch.randperm(e, generator=g)[:a]] = count
    return torch.cat([full.new_zeros(1), full.cumsum(0)]), int(full.max())


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    k = case["k"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    state = {"op": case["op"]}
    if case["op"] == "round_trip":
        shape = (case["m"], k) if not case["experts"] else (case["experts"], case["m"], k)
        x = normal(*shape)
        # a few columns are much larger, as in activations
        x *= 1 + 30 * (torch.rand(k, generator=g, device="cuda") < 0.01)
        state["x"] = x.to(getattr(torch, case["dtype"]))
        return state
    if case["op"] == "gemm":
        state["a"], state["sa"] = _quantize(normal(case["m"], k))
        state["b"], state["sb"] = _quantize(normal(case["n"], k) / math.sqrt(k))
        return state
    offsets, state["most"] = _offsets(case, seed)
    state["offsets"] = offsets.to("cuda", torch.int32)
    x = normal(case["rows"] + case["spare"], k)
    if case["op"] == "mx_grouped":
        state["a"], state["sa"] = _quantize(x)
        b = [_quantize(normal(case["n"], k) / math.sqrt(k)) for _ in range(case["experts"])]
        state["b"], state["sb"] = (torch.stack(t) for t in zip(*b))
        return state
    sx = x.abs().amax() / 448
    state["a"] = (x / sx).to(torch.float8_e4m3fn)
    b, alpha = [], []
    for _ in range(case["experts"]):
        w = normal(case["n"], k) / math.sqrt(k)
        sw = w.abs().amax() / 448
        b.append((w / sw).to(torch.float8_e4m3fn))
        alpha.append(sx * sw)
    state["b"], state["alpha"] = torch.stack(b), torch.stack(alpha)
    return state


# ---------------------------------------------------------------- one pass
def _values(codes, scales):
    """FP32 values of MXFP4 codes and blocked scales."""
    level = torch.tensor(_LEVELS + tuple(-v for v in _LEVELS), device=codes.device)
    v = torch.stack([level[(codes & 15).int()], level[(codes >> 4).int()]], -1)
    rows, k = codes.shape[-2], codes.shape[-1] * 2
    s = _unblock(scales, rows, k // 32).int()
    # 2^(s - 127) in two factors: 2^-127 is below FP32's normal range
    v = v.reshape(*codes.shape[:-1], k // 32, 32)
    v = torch.ldexp(torch.ldexp(v, ((s - 127) // 2).unsqueeze(-1)), (s - 127 - (s - 127) // 2).unsqueeze(-1))
    return v.reshape(*codes.shape[:-1], k)


def _grouped(x, w, offsets, most, alpha=None):
    """out[r] = w[expert of r] x[r]; zero for rows of no expert."""
    row = torch.arange(x.shape[0], device=x.device)
    expert = (row[:, None] >= offsets[None, 1:]).sum(1)
    kept = expert < w.shape[0]
    expert = expert.clamp(max=w.shape[0] - 1)
    at = torch.where(kept, row - offsets[expert], most)
    wide = x.new_zeros(w.shape[0], most + 1, x.shape[1])
    wide[expert, at] = x
    y = torch.bmm(wide, w.transpose(1, 2))[expert, at]
    if alpha is not None:
        y = y * alpha[expert, None]
    return torch.where(kept[:, None], y, 0.0).bfloat16()


def run(state):
    if own:
        return _run_own(state)
    op = state["op"]
    if op == "round_trip":
        return _values(*_quantize(state["x"])).to(state["x"].dtype)
    if op == "fp8_grouped":
        return _grouped(state["a"].float(), state["b"].float(), state["offsets"], state["most"], state["alpha"])
    a, b = _values(state["a"], state["sa"]), _values(state["b"], state["sb"])
    if op == "gemm":
        return (a @ b.T).bfloat16()
    return _grouped(a, b, state["offsets"], state["most"])


def _run_own(state):
    import candidate_kernel as ck

    op = state["op"]
    if op == "round_trip":
        codes, scales = ck.mxfp4_quantize(state["x"])
        return ck.mxfp4_dequantize(codes, scales, state["x"].dtype)
    if op == "fp8_grouped":
        return ck.fp8_gemm_grouped(state["a"], state["b"], state["alpha"], state["offsets"])
    if op == "gemm":
        return ck.mxfp4_gemm(state["a"], state["sa"], state["b"], state["sb"])
    return ck.mxfp4_gemm_grouped(state["a"], state["sa"], state["b"], state["sb"], state["offsets"])


# ---------------------------------------------------------------- 64 bits
def _decode64(codes, scales):
    """sign * (2^(e-1) (1 + m/2), or m/2 for e = 0) * 2^(scale - 127)."""
    out = torch.empty(codes.shape[0], codes.shape[1] * 2, dtype=torch.float64, device=codes.device)
    for half in (0, 1):
        c = (codes >> (4 * half)).long() & 15
        e, m = (c >> 1) & 3, (c & 1).double()
        mag = torch.where(e > 0, torch.exp2((e - 1).double()) * (1 + m / 2), m / 2)
        out[:, half::2] = torch.where(c >= 8, -mag, mag)
    rows = torch.arange(codes.shape[0], device=codes.device)[:, None]
    col = torch.arange(out.shape[1], device=codes.device)[None, :] // 32
    byte = scales[rows // 128, col // 4, (rows % 32) * 16 + (rows // 32 % 4) * 4 + col % 4]
    return out * torch.exp2(byte.double() - 127)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "round_trip":
        x = state["x"]
        v = x.double().reshape(*x.shape[:-1], -1, 32)
        top = v.abs().amax(-1, keepdim=True)
        e = torch.floor(torch.log2(top)) - 2
        e = torch.where(torch.exp2(e + 3) <= top, e + 1, torch.where(torch.exp2(e + 2) > top, e - 1, e))
        unit = torch.exp2(e.clamp(-127, 127).nan_to_num(neginf=-127.0))
        u = (v / unit).clamp(-6, 6)
        # spacing of E2M1 around |u|: 1/2 below 2, 1 below 4, 2 from there; round() ties to even
        step = 0.5 * (1 + (u.abs() >= 2) + 2 * (u.abs() >= 4))
        return (torch.round(u / step) * step * unit).reshape(x.shape)
    if case["op"] == "gemm":
        return _decode64(state["a"], state["sa"]) @ _decode64(state["b"], state["sb"]).T
    off = state["offsets"].tolist()
    a = state["a"].double() if case["op"] == "fp8_grouped" else _decode64(state["a"], state["sa"])
    y = a.new_zeros(a.shape[0], case["n"])
    for e in range(case["experts"]):
        r = slice(off[e], off[e + 1])
        if off[e + 1] > off[e]:
            if case["op"] == "fp8_grouped":
                y[r] = a[r] @ state["b"][e].double().T * state["alpha"][e].double()
            else:
                y[r] = a[r] @ _decode64(state["b"][e], state["sb"][e]).T
    return y
