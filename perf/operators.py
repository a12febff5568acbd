"""Cases of the MXFP4 operators: quantisation, SwiGLU with quantisation, the product of two MXFP4 operands, and the same product
grouped by expert.

MXFP4 holds a row as blocks of 32 elements: 32 E2M1 codes (two in a byte, the even element in the low half) and one E8M0 byte e, the
scale 2^(e - 127). Quantised outputs are returned as the values that they stand for (bf16, which holds every one of them exactly).

The products take their scales as the framework's tiled layout holds them: [ceil(K / 128), rows, 4], the four scale bytes of a row's
128-element stretch side by side and consecutive rows next to one another, zero where K ends inside a stretch.
"""
import math

import torch

own = False

# the gpt-oss activation's constants, as the f32 numbers that the operators take
ALPHA, LIMIT = float(torch.tensor(1.702, dtype=torch.float32)), 7.0
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one token's hidden state, quantised ahead of a 4-bit layer: latency
        {"name": "quantise one token", "op": "quantise", "rows": 1, "cols": 2880, "ld": 2880, "dtype": "bf16", "rule": "floor", "row_scale": False},
        # a prompt's hidden states, 8192 tokens of gpt-oss-20b
        {"name": "quantise prompt", "op": "quantise", "rows": 8192, "cols": 2880, "ld": 2880, "dtype": "bf16", "rule": "floor", "row_scale": False},
        # f32 weights of 16 experts' gate/up rows made into a checkpoint's MXFP4, with scales that never clip
        {"name": "quantise weights", "op": "quantise", "rows": 16 * 5760, "cols": 2880, "ld": 2880, "dtype": "f32", "rule": "noclip", "row_scale": False},
        # expert-major f16 rows with a scale for each, a column range of wider rows, an odd number of them
        {"name": "quantise scaled rows", "op": "quantise", "rows": 2731, "cols": 4096, "ld": 5120, "dtype": "f16", "rule": "floor", "row_scale": True},
        # the activation between the two expert products: 8 tokens with 4 experts each
        {"name": "swiglu decode", "op": "swiglu", "rows": 32, "cols": 2880, "ld": 5760, "dtype": "f32", "rule": "floor"},
        # the same for a prompt of 8192 tokens
        {"name": "swiglu prompt", "op": "swiglu", "rows": 32768, "cols": 2880, "ld": 5760, "dtype": "bf16", "rule": "floor"},
        # one token through the q/k/v projection
        {"name": "product one token", "op": "product", "m": 1, "n": 5120, "k": 2880, "out": "bf16", "bias": True},
        # 64 sequences' logits
        {"name": "product logits", "op": "product", "m": 64, "n": 201088, "k": 2880, "out": "f32", "bias": False},
        # an odd prompt through the output projection
        {"name": "product odd prompt", "op": "product", "m": 1037, "n": 2880, "k": 4096, "out": "bf16", "bias": True},
        # 8192 tokens through the q/k/v projection
        {"name": "product prompt", "op": "product", "m": 8192, "n": 5120, "k": 2880, "out": "bf16", "bias": True},
        # 8 tokens with 4 of 32 experts each: gate/up products of one decode step
        {"name": "grouped decode", "op": "grouped", "groups": 32, "m": 32, "n": 5760, "k": 2880, "skew": 0.5, "out": "f32", "bias": True},
        # 8192 tokens with 4 of 32 experts each: gate/up products of a prompt, skewed loads
        {"name": "grouped prompt", "op": "grouped", "groups": 32, "m": 32768, "n": 5760, "k": 2880, "skew": 0.5, "out": "bf16", "bias": True},
    ]


def draw(rng):
    def size(lo, hi, step=1):  # spread over the logarithm
        return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))) // step * step))) if hi > lo else lo

    op = rng.choice(["quantise", "swiglu", "product", "grouped"])
    if op in ("quantise", "swiglu"):
        cols = size(32, 8192, 32)
        width = cols * (2 if op == "swiglu" else 1)
        case = {"op": op, "rows": size(1, min(65536, 90_000_000 // width)), "cols": cols, "ld": width + rng.choice([0, 0, 8, 64, 1000]),
                "dtype": rng.choice(["bf16", "f32", "f16"]), "rule": rng.choice(["floor", "noclip"])}
        if op == "quantise":
            case["row_scale"] = rng.random() < 0.3
        return case
    if op == "product":
        n, k = size(64, 32768), size(64, 8192, 32)
        return {"op": op, "m": size(1, min(8192, 120_000_000_000 // (n * k))), "n": n, "k": k, "out": rng.choice(["bf16", "f32"]), "bias": rng.random() < 0.5}
    groups, n, k = size(1, 64), size(64, 5760), size(64, 4096, 32)
    return {"op": op, "groups": groups, "m": size(1, min(32768, 200_000_000_000 // (n * k))), "n": n, "k": k, "skew": round(rng.uniform(0.0, 0.8), 2),
            "out": rng.choice(["bf16", "f32"]), "bias": rng.random() < 0.5}


def rows_of_groups(case):
    """Rows of each group from the busiest down: shares that fall like rank^-skew, whole numbers with the case's sum."""
    g, m = case["groups"], case["m"]
    share = [(r + 1) ** -case["skew"] for r in range(g)]
    share = [m * s / sum(share) for s in share]
    got = [int(s) for s in share]
    for r in sorted(range(g), key=lambda r: got[r] - share[r])[: m - sum(got)]:
        got[r] += 1
    return got


def work(case):
    if case["op"] in ("quantise", "swiglu"):
        n, size = case["rows"] * case["cols"], DTYPES[case["dtype"]].itemsize
        read = n * size * (2 if case["op"] == "swiglu" else 1) + (4 * case["rows"] if case.get("row_scale") else 0)
        # codes and scales written, and the bf16 values that they are returned as
        return {"bytes": read + n // 2 + n // 32 + 2 * n, "flops": n * (12 if case["op"] == "swiglu" else 3)}
    m, n, k = case["m"], case["n"], case["k"]
    held = sum(c > 0 for c in rows_of_groups(case)) if case["op"] == "grouped" else 1
    read = (m + held * n) * (k // 2 + k // 32) + (2 * held * n if case["bias"] else 0)
    return {"bytes": read + m * n * DTYPES[case["out"]].itemsize, "flops": 2 * m * n * k}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def integers(low, high, *shape):
        return torch.randint(low, high, shape, generator=gen, device="cuda", dtype=torch.uint8)

    if case["op"] in ("quantise", "swiglu"):
        rows, width = case["rows"], case["cols"] * (2 if case["op"] == "swiglu" else 1)
        x = normal(rows, case["ld"])
        x *= 0.05 if case["rule"] == "noclip" else 2.0
        if case["op"] == "quantise" and case["rule"] == "floor":  # some of a hidden state's channels are far larger than the others
            x *= torch.exp(normal(case["ld"]))
        state = {"case": dict(case), "x": x.to(DTYPES[case["dtype"]])[:, :width]}
        if case.get("row_scale"):
            state["row_scale"] = torch.exp2(torch.randint(-3, 4, (rows,), generator=gen, device="cuda").float())
        return state
    groups, m, n, k = case.get("groups", 1), case["m"], case["n"], case["k"]
    lead = (groups,) if case["op"] == "grouped" else ()
    state = {"case": dict(case), "a": integers(0, 256, m, k // 2), "a_scales": tiled_scales(integers, m, k, (), 127),
             "b": integers(0, 256, *lead, n, k // 2), "b_scales": tiled_scales(integers, n, k, lead, 121),
             "bias": normal(*lead, n).to(torch.bfloat16) if case["bias"] else None}
    if case["op"] == "grouped":
        order = torch.randperm(groups, generator=gen, device="cuda")  # which expert is the busy one
        counts = torch.tensor(rows_of_groups(case), dtype=torch.int32, device="cuda")
        state["counts"], state["most"] = counts[order].contiguous(), max(rows_of_groups(case))
    return state


def tiled_scales(integers, rows, k, lead, around):
    """Scale bytes near `around`, tiled: [*lead, ceil(k / 128), rows, 4]."""
    s = integers(around - 2, around + 3, *lead, (k + 127) // 128, rows, 4)
    if k % 128:
        s[..., -1, :, k % 128 // 32:] = 0
    return s


def run(state):
    case = state["case"]
    if own:
        from oxidized_gpt_oss_b200 import ffn, mxfp4
        if case["op"] in ("quantise", "swiglu"):
            if case["op"] == "quantise":
                blocks, scales = mxfp4.quantize_mxfp4(state["x"], row_scale=state.get("row_scale"), scale_rule=case["rule"])
            else:
                blocks, scales = ffn.swiglu_quantize_mxfp4(state["x"], ALPHA, LIMIT, scale_rule=case["rule"])
            return mxfp4.dequantize_mxfp4(blocks, scales, case["rows"], case["cols"]).view(torch.bfloat16).view(case["rows"], case["cols"])
        if case["op"] == "product":
            return mxfp4.mxfp4_matmul(state["a"], state["a_scales"], state["b"], state["b_scales"], bias=state["bias"], out_dtype=DTYPES[case["out"]])
        return mxfp4.mxfp4_grouped_matmul(state["a"], state["a_scales"], state["counts"], state["b"], state["b_scales"], bias=state["bias"],
                                          out_dtype=DTYPES[case["out"]])
    if case["op"] == "quantise":
        x = state["x"].float()
        return plain_quantise(x * state["row_scale"][:, None] if "row_scale" in state else x, case["rule"])
    if case["op"] == "swiglu":  # in 64 bits: a value next to a border between two codes has to fall on its own side
        gate, up = state["x"][:, 0::2].double().clamp(max=LIMIT), state["x"][:, 1::2].double().clamp(-LIMIT, LIMIT)
        return plain_quantise(gate / (1 + torch.exp(-ALPHA * gate)) * (up + 1), case["rule"])
    a, b = plain_values(state["a"], state["a_scales"]), plain_values(state["b"], state["b_scales"])
    if case["op"] == "product":
        y = a @ b.T
        return (y if state["bias"] is None else y + state["bias"].float()).to(DTYPES[case["out"]])
    # each group's rows, padded to the busiest group's, times its own matrix
    counts = state["counts"].long()
    at = torch.arange(state["most"], device=a.device)[None, :]
    held = at < counts[:, None]
    index = torch.where(held, counts.cumsum(0)[:, None] - counts[:, None] + at, 0)
    y = torch.bmm(a[index], b.transpose(1, 2))
    if state["bias"] is not None:
        y += state["bias"].float()[:, None, :]
    return y[held].to(DTYPES[case["out"]])


def plain_quantise(x, rule):
    """[rows, cols] to the nearest MXFP4 values, ties to the even code, as bf16."""
    v = x.view(x.shape[0], -1, 32)
    part, e = torch.frexp(v.abs().amax(-1, keepdim=True))  # part in [1/2, 1)
    e = e - 3 + ((part > 0.75).to(e.dtype) if rule == "noclip" else 0)  # the largest lands in [4, 8), or in (3, 6]
    e = e.clamp(min=-126)
    r = torch.ldexp(v.double(), -e)
    a = r.abs()
    code = (a > 0.25).to(torch.int32) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    return torch.ldexp(torch.copysign(table[code], r), e).view(x.shape).to(torch.bfloat16)


def plain_values(blocks, scales):
    """Packed codes [..., rows, K / 2] and tiled scales as f32 values [..., rows, K]."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=blocks.device)
    table = torch.cat([table, -table])
    codes = torch.stack([blocks & 15, blocks >> 4], -1).flatten(-2)
    k = codes.shape[-1]
    s = torch.exp2(scales.transpose(-3, -2).flatten(-2)[..., : k // 32].float() - 127)
    return (table[codes.int()].unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] in ("quantise", "swiglu"):
        x = state["x"].double()
        if "row_scale" in state:
            x = x * state["row_scale"].double()[:, None]
        if case["op"] == "swiglu":
            g, u = torch.minimum(x[:, ::2], torch.full_like(x[:, ::2], LIMIT)), torch.clamp(x[:, 1::2], -LIMIT, LIMIT)
            x = g * torch.sigmoid(ALPHA * g) * (u + 1)
        top = x.reshape(x.shape[0], -1, 32).abs().amax(2).clamp(min=2.0 ** -300)
        e = torch.floor(torch.log2(top) + 1e-11)  # log2 of a power of two may come out just below the whole number
        step = e - 2 + ((top > 1.5 * torch.ldexp(torch.ones_like(e), e.int())).double() if case["rule"] == "noclip" else 0)
        scale = torch.ldexp(torch.ones_like(step), step.clamp(min=-126).int()).repeat_interleave(32, 1)
        a = (x / scale).abs()
        # E2M1 counts in halves below 2, in ones from 2 to 4, in twos above; torch.round takes ties to even
        near = torch.where(a < 2, torch.round(2 * a) / 2, torch.where(a < 4, torch.round(a), 2 * torch.round(a / 2))).clamp(max=6)
        return near * scale * torch.sign(x)
    values = []
    for blocks, scales in ((state["a"], state["a_scales"]), (state["b"], state["b_scales"])):
        v = torch.empty(*blocks.shape[:-1], 2 * blocks.shape[-1], dtype=torch.float64, device=blocks.device)
        for half in (0, 1):
            c = (blocks >> (4 * half)) & 15
            mag, man = (c >> 1) & 3, (c & 1).double()
            w = torch.where(mag == 0, man / 2, (1 + man / 2) * torch.exp2(mag.double() - 1))
            v[..., half::2] = torch.where(c > 7, -w, w)
        for block in range(v.shape[-1] // 32):
            v[..., 32 * block: 32 * block + 32] *= torch.exp2(scales[..., block // 4, :, block % 4].double() - 127)[..., None]
        values.append(v)
    a, b = values
    if case["op"] == "product":
        y = a @ b.mT
        return y if state["bias"] is None else y + state["bias"].double()
    out, first = [], 0
    for group, count in enumerate(state["counts"].tolist()):
        y = a[first: first + count] @ b[group].mT
        out.append(y if state["bias"] is None else y + state["bias"][group].double())
        first += count
    return torch.cat(out)
