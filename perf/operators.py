"""Workloads of the products grouped by expert and of the microscaled 4-bit format.

Five paths, each as a program calls it:

  grouped       y[t] = x[t] W[e]^T for the rows t of group e (tokens sorted by expert)
  grouped_grad  the gradients of that product: dx[t] = dy[t] W[e] and dW[e] = sum_t dy[t]^T x[t]
  quantize      bf16 to MXFP4 (blocks of 32 along K, one power-of-two scale each) and back
  mx            a linear layer in 4 bits: the activations are quantised, then multiplied with
                weights that are held in MXFP4
  grouped_mx    the same with one 4-bit weight matrix per expert

`own` chooses between the plain form (elementary torch operations in 32 bits) and the calls of
`gemm_b200.ops`.
"""
import math
import random

import torch

own = False

#: The sixteen values of an E2M1 code (sign bit 3, exponent bits 2-1, mantissa bit 0).
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


# ---------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # Two tokens of a small model on eight experts: launch latency.
        dict(name="grouped tiny", op="grouped", groups=8, rows=2, n=1024, k=1024, spare=0),
        # One decoding step, eight rows over sixteen experts: the chosen weights are streamed once.
        dict(name="grouped decode", op="grouped", groups=16, rows=8, n=3584, k=2048, spare=0),
        # A mixed batch of a serving loop, ragged, with rows behind the last group (padded batch).
        dict(name="grouped mixed", op="grouped", groups=32, rows=1001, n=3584, k=2048, spare=23),
        # The experts' projection in training or prefill.
        dict(name="grouped prefill", op="grouped", groups=8, rows=16384, n=4096, k=4096, spare=0),
        # Gradients of a short ragged batch.
        dict(name="grad short", op="grouped_grad", groups=8, rows=513, n=1024, k=2048, spare=7),
        # Gradients of the large batch.
        dict(name="grad long", op="grouped_grad", groups=8, rows=16384, n=4096, k=4096, spare=0),
        # Activations of one decoding step.
        dict(name="quantize rows", op="quantize", rows=16, k=8192),
        # A weight matrix, as it is converted when a model is loaded.
        dict(name="quantize weight", op="quantize", rows=28672, k=8192),
        # The decode shape in 4 bits.
        dict(name="mx decode", op="mx", rows=16, n=28672, k=8192),
        # The square benchmark shape in 4 bits.
        dict(name="mx square", op="mx", rows=8192, n=8192, k=8192),
        # One decoding step of a batch over 4-bit experts.
        dict(name="grouped mx decode", op="grouped_mx", groups=32, rows=64, n=3584, k=2048, spare=0),
        # Prefill over 4-bit experts.
        dict(name="grouped mx prefill", op="grouped_mx", groups=8, rows=8191, n=4096, k=4096, spare=1),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("grouped", "grouped_grad", "quantize", "mx", "grouped_mx"))
    if op == "quantize":
        return dict(op=op, rows=_log(rng, 1, 20000), k=32 * _log(rng, 1, 256))
    n, k = 8 * _log(rng, 8, 512), 8 * _log(rng, 8, 512)
    if op == "mx":
        return dict(op=op, rows=_log(rng, 1, 8000), n=n + rng.randrange(8), k=64 * _log(rng, 1, 128))
    if op == "grouped_mx":
        k = 64 * _log(rng, 1, 64)
    groups = _log(rng, 1, 64)
    while groups > 1 and groups * n * k > 32 * 3584 * 2048:
        groups //= 2
    return dict(op=op, groups=groups, rows=_log(rng, 1, 12000), n=n, k=k,
                spare=rng.choice((0, 0, rng.randrange(1, 200))))


def work(case):
    if case["op"] == "quantize":
        m, k = case["rows"], case["k"]
        packed = m * k // 2 + m * k // 32
        return {"bytes": 2 * m * k + 2 * packed + 2 * m * k, "flops": 2 * m * k}
    m, n, k = case["rows"], case["n"], case["k"]
    if case["op"] == "mx":
        return {"bytes": 2 * m * k + n * k // 2 + n * k // 32 + 2 * m * n, "flops": 2 * m * n * k}
    # A group without rows needs no weights: the expected number of groups that have some.
    used = sum(1 for c in _counts(case, 0) if c)
    if case["op"] == "grouped":
        return {"bytes": 2 * (m * k + used * n * k + m * n), "flops": 2 * m * n * k}
    if case["op"] == "grouped_mx":
        return {"bytes": 2 * m * k + used * (n * k // 2 + n * k // 32) + 2 * m * n,
                "flops": 2 * m * n * k}
    return {"bytes": 2 * (2 * m * k + 2 * m * n + used * n * k + case["groups"] * n * k),
            "flops": 4 * m * n * k}


# ---------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------
def _counts(case, seed):
    """Rows of every group: a router's uneven load, some groups without any."""
    rng = random.Random(seed * 7919 + 11)
    g, weight, got = case["groups"], [], [0] * case["groups"]
    for _ in range(g):
        weight.append(math.exp(0.6 * rng.gauss(0.0, 1.0)))
    for e in rng.choices(range(g), weights=weight, k=case["rows"]):
        got[e] += 1
    return got


def _normal(gen, *shape, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(torch.bfloat16)


def _mx_weights(gen, *shape):
    """Random weights in the MXFP4 format: codes [.., rows, K/2] with two E2M1 codes to a byte (the
    even k in the low four bits) and E8M0 scales in tiles of 128 rows x 4 blocks,
    [.., ceil(rows/128), ceil(K/128), 32, 4, 4], indexed by (row % 32, row % 128 // 32, block % 4).
    The codes' spread is that of normal values quantised with a block's largest magnitude."""
    *lead, rows, k = shape
    w = torch.randn(*lead, rows, k // 32, 32, generator=gen, device="cuda")
    w /= math.sqrt(k)
    exponent = torch.frexp(w.abs().amax(-1))[1] - 3          # floor(log2(amax)) - 2
    mag = (w.abs() * torch.exp2(-exponent.float())[..., None]).clamp(max=6.0)
    step = torch.where(mag < 2.0, 0.5, torch.where(mag < 4.0, 1.0, 2.0))
    mag = torch.round(mag / step) * step
    code = (mag * 2).to(torch.int32)                          # 0 1 2 3 4 6 8 12 -> 0 .. 7
    code = code - (code > 5).int() - (code > 7).int() - 3 * (code > 11).int()
    code = (code + 8 * (w < 0).int()).to(torch.uint8).view(*lead, rows, k // 2, 2)
    codes = code[..., 0] | (code[..., 1] << 4)
    rb, kb = -(-rows // 128), -(-k // 128)
    grid = torch.zeros(*lead, rb * 128, kb * 4, dtype=torch.uint8, device="cuda")
    grid[..., :rows, :k // 32] = (exponent + 127).to(torch.uint8)
    n = len(lead)
    scales = grid.view(*lead, rb, 4, 32, kb, 4).permute(*range(n), n, n + 3, n + 2, n + 1, n + 4)
    return codes.contiguous(), scales.contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, rows, k = case["op"], case["rows"], case["k"]
    state = dict(op=op)
    if op == "quantize":
        # A few channels are far larger than the rest, as in activations.
        loud = torch.exp(torch.randn(k, generator=gen, device="cuda"))
        state["x"] = _normal(gen, rows, k).mul_(loud.to(torch.bfloat16))
        return state
    n = case["n"]
    if op == "mx":
        state["x"] = _normal(gen, rows, k)
        state["codes"], state["scales"] = _mx_weights(gen, n, k)
        return state
    counts = _counts(case, seed)
    total = rows + case["spare"]
    ends = [0]
    for c in counts:
        ends.append(ends[-1] + c)
    state["offsets"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
    state["longest"] = max(counts)       # a program that pads its groups knows its capacity
    state["x"] = _normal(gen, total, k)
    if op == "grouped_mx":
        state["codes"], state["scales"] = _mx_weights(gen, case["groups"], n, k)
        return state
    state["w"] = _normal(gen, case["groups"], n, k, scale=1.0 / math.sqrt(k))
    if op == "grouped_grad":
        state["dy"] = _normal(gen, total, n)
    return state


# ---------------------------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------------------------
def _pad_index(offsets, longest, total):
    """For every group and every place up to the longest group: the row, and whether there is one."""
    place = torch.arange(max(longest, 1), device=offsets.device)
    row = offsets[:-1, None].long() + place[None, :]
    return row.clamp(max=total - 1), row < offsets[1:, None].long()


def _into_groups(x, row, there):
    return x.float()[row] * there[..., None]


def _out_of_groups(padded, row, there, total):
    """Rows back to their places; rows of no group are zero."""
    out = torch.zeros(total + 1, padded.shape[-1], dtype=torch.float32, device=padded.device)
    out[torch.where(there, row, total)] = padded
    return out[:total]


def _plain_quantize(x):
    """(magnitudes with sign in units of the block's scale, biased exponent of the scale)."""
    blocks = x.float().view(*x.shape[:-1], -1, 32)
    amax = blocks.abs().amax(-1)
    exponent = (amax.view(torch.int32) >> 23).clamp(min=2) - 2      # floor(log2) - 2, biased
    # 2^-(exponent - 127), in two factors so that neither leaves the range of normal numbers
    half = (127 - exponent) // 2
    up = torch.exp2(half.float()) * torch.exp2((127 - exponent - half).float())
    scaled = blocks * up[..., None]
    mag = scaled.abs().clamp(max=6.0)
    step = torch.where(mag < 2.0, 0.5, torch.where(mag < 4.0, 1.0, 2.0))
    mag = torch.round(mag / step) * step                            # ties to the even code
    return torch.copysign(mag, scaled), exponent


def _times_scale(units, exponent):
    half = (exponent - 127) // 2
    v = units * torch.exp2(half.float())[..., None]
    v = v * torch.exp2((exponent - 127 - half).float())[..., None]
    return v.flatten(-2)


def _scale_tiles(exponent):
    """Scale bytes [rows, K/32] in the format's tiles; padding is zero."""
    rows, blocks = exponent.shape
    rb, kb = -(-rows // 128), -(-blocks // 4)
    grid = torch.zeros(rb * 128, kb * 4, dtype=torch.uint8, device=exponent.device)
    grid[:rows, :blocks] = exponent.to(torch.uint8)
    return grid.view(rb, 4, 32, kb, 4).permute(0, 3, 2, 1, 4).contiguous()


def _unpack(codes, scales):
    """MXFP4 to fp32 values [.., rows, K]."""
    rows, k = codes.shape[-2], 2 * codes.shape[-1]
    table = torch.tensor(E2M1, device=codes.device)
    pair = torch.stack((codes & 15, codes >> 4), dim=-1)
    units = table[pair.int()].view(*codes.shape[:-1], k // 32, 32)
    s = scales.movedim(-2, -4)                 # [.., rb, 4, kb, 32, 4]
    s = s.movedim(-2, -3)                      # [.., rb, 4, 32, kb, 4]
    s = s.reshape(*s.shape[:-5], s.shape[-5] * 128, s.shape[-2] * 4)[..., :rows, :k // 32]
    return _times_scale(units, s.int())


def _plain(state):
    op, x = state["op"], state["x"]
    if op == "quantize":
        units, exponent = _plain_quantize(x)
        return {"values": _times_scale(units, exponent).to(torch.bfloat16),
                "scales": _scale_tiles(exponent)}
    if op == "mx":
        xq = _times_scale(*_plain_quantize(x))
        return (xq @ _unpack(state["codes"], state["scales"]).t()).to(torch.bfloat16)
    total = x.shape[0]
    row, there = _pad_index(state["offsets"], state["longest"], total)
    if op == "grouped_mx":
        xq = _into_groups(_times_scale(*_plain_quantize(x)), row, there)
        y = xq @ _unpack(state["codes"], state["scales"]).transpose(1, 2)
        return _out_of_groups(y, row, there, total).to(torch.bfloat16)
    w = state["w"].float()
    xg = _into_groups(x, row, there)
    if op == "grouped":
        return _out_of_groups(xg @ w.transpose(1, 2), row, there, total).to(torch.bfloat16)
    dyg = _into_groups(state["dy"], row, there)
    return {"dx": _out_of_groups(dyg @ w, row, there, total).to(torch.bfloat16),
            "dw": (dyg.transpose(1, 2) @ xg).to(torch.bfloat16)}


def run(state):
    if not own:
        return _plain(state)
    from gemm_b200 import ops
    op, x = state["op"], state["x"]
    if op == "grouped":
        return ops.grouped_matmul(x, state["w"], state["offsets"])
    if op == "grouped_grad":
        return {"dx": ops.grouped_matmul_dx(state["dy"], state["w"], state["offsets"]),
                "dw": ops.grouped_matmul_dw(state["dy"], x, state["offsets"])}
    q = ops.quantize_mxfp4(x)
    if op == "quantize":
        return {"values": ops.dequantize_mxfp4(q), "scales": q.scales}
    w = ops.MxFp4(state["codes"], state["scales"])
    if op == "mx":
        return ops.matmul_mxfp4(q, w)
    return ops.grouped_matmul_mxfp4(q, w, state["offsets"])


# ---------------------------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------------------------
def _exact_round(x):
    """bf16 [rows, K] -> (values of the MXFP4 tensor, scale exponents) in 64 bits."""
    b = x.double().reshape(x.shape[0], -1, 32)
    top = b.abs().amax(-1)
    e = torch.frexp(top)[1].double() - 3
    e = torch.where(top == 0, torch.full_like(e, -127), e).clamp(-127, 127)
    s = torch.ldexp(torch.ones_like(e), e)[..., None]
    grid = torch.tensor(E2M1[:8], dtype=torch.float64, device=x.device)
    u = (b / s).abs()
    middle = (grid[1:] + grid[:-1]) / 2
    below = torch.bucketize(u, middle)                  # a tie falls to the lower code ...
    above = torch.bucketize(u, middle, right=True)      # ... or to the upper one
    code = torch.where(below % 2 == 0, below, above)    # the even one of the two
    return (grid[code] * s * torch.sign(b)).flatten(1), e


def _exact_unpack(codes, scales):
    rows, k = codes.shape[-2], codes.shape[-1] * 2
    grid = torch.tensor(E2M1, dtype=torch.float64, device=codes.device)
    v = torch.empty(*codes.shape[:-1], k, dtype=torch.float64, device=codes.device)
    v[..., 0::2] = grid[(codes % 16).long()]
    v[..., 1::2] = grid[(codes // 16).long()]
    r = torch.arange(rows, device=codes.device)[:, None]
    b = torch.arange(k // 32, device=codes.device)[None, :]
    s = scales[..., r // 128, b // 4, r % 32, r % 128 // 32, b % 4].double() - 127
    return v * torch.exp2(s).repeat_interleave(32, dim=-1)


def exact(case, seed):
    state = prepare(case, seed)
    op, x = state["op"], state["x"]
    if op == "quantize":
        v, e = _exact_round(x)
        rows, blocks = e.shape
        tiles = torch.zeros(-(-rows // 128), -(-blocks // 4), 32, 4, 4, dtype=torch.uint8,
                            device=x.device)
        r = torch.arange(rows, device=x.device)[:, None]
        b = torch.arange(blocks, device=x.device)[None, :]
        tiles[r // 128, b // 4, r % 32, r % 128 // 32, b % 4] = (e + 127).to(torch.uint8)
        return {"values": v, "scales": tiles}
    if op == "mx":
        return _exact_round(x)[0] @ _exact_unpack(state["codes"], state["scales"]).t()
    ends = state["offsets"].tolist()
    v = _exact_round(x)[0] if op == "grouped_mx" else x.double()
    if op == "grouped_grad":
        dy = state["dy"].double()
        dx = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
        dw = torch.zeros(state["w"].shape, dtype=torch.float64, device=x.device)
        for g, (a, b) in enumerate(zip(ends, ends[1:])):
            dx[a:b] = dy[a:b] @ state["w"][g].double()
            dw[g] = dy[a:b].t() @ v[a:b]
        return {"dx": dx, "dw": dw}
    y = torch.zeros(x.shape[0], case["n"], dtype=torch.float64, device=x.device)
    for g, (a, b) in enumerate(zip(ends, ends[1:])):
        w = (_exact_unpack(state["codes"][g], state["scales"][g]) if op == "grouped_mx"
             else state["w"][g].double())
        y[a:b] = v[a:b] @ w.t()
    return y
