"""Operators of a token table, in their plain form and through this package, with what they cannot do without.

A token table is trained (lookup of scaled rows, gradient of the rows), published in 4 bits with one scale and bias per
group of a row, and served from those bytes (lookup, and products of a few hidden states with all rows).  ``listed()``
names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes what a program holds before the call,
``run`` is one pass: elementary torch operations in fp32 where ``own`` is false, the package's operators where it is true.

A 4-bit row of D elements in groups of g is ``[D / 2 bytes of codes, low nibble first][fp16 scale, fp16 bias per group]``,
padded to a multiple of 16 bytes; an element is code * scale + bias.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"fp32": 4, "fp16": 2, "bf16": 2}
CODES = {"fp32": 0, "fp16": 1, "bf16": 5}      # the package's output_dtype numbers
DEVICE = "cuda"


def _lookup(name, tokens, rows, dim, table, output, scale, bits, pruned=0.0):
    return {"name": name, "kind": "lookup", "tokens": tokens, "rows": rows, "dim": dim, "table": table, "output": output, "scale": scale,
            "bits": bits, "pruned": pruned}


def _grad(name, tokens, rows, dim, grad, output, scale, bits, into, hot=0.0, padding=-1, pruned=0.0):
    """``into``: the gradient is added into a buffer that the program keeps, instead of written whole.  ``hot``: the
    share of tokens that are one and the same token."""
    return {"name": name, "kind": "grad", "tokens": tokens, "rows": rows, "dim": dim, "grad": grad, "output": output, "scale": scale, "bits": bits,
            "into": into, "hot": hot, "padding": padding, "pruned": pruned}


def _packed(name, tokens, rows, dim, group, output, scale, bits):
    return {"name": name, "kind": "packed", "tokens": tokens, "rows": rows, "dim": dim, "group": group, "output": output, "scale": scale, "bits": bits}


def _publish(name, rows, dim, group, table, output):
    return {"name": name, "kind": "publish", "rows": rows, "dim": dim, "group": group, "table": table, "output": output}


def _linear(name, states, rows, dim, group, hidden, output, bias):
    return {"name": name, "kind": "linear", "states": states, "rows": rows, "dim": dim, "group": group, "hidden": hidden, "output": output, "bias": bias}


def listed():
    return [
        # A few tokens of an odd-sized table, as a decoding step looks up: latency, unaligned rows, pruned tokens.
        _lookup("few_odd_rows", 33, 50_021, 1001, "fp32", "bf16", 1.0, 32, 0.1),
        # The tokens of a batch of prompts, rows scaled by the root of their width.
        _lookup("prompt_rows", 16_384, 131_072, 4096, "bf16", "bf16", 64.0, 64),
        # The same from the table published in 4 bits.
        _packed("packed_rows", 16_384, 131_072, 4096, 128, "bf16", 64.0, 64),
        # The gradient of a small table: the smallest training step.
        _grad("small_step", 512, 8_192, 512, "fp32", "fp32", 1.0, 64, False),
        # An ordinary training step: the whole gradient of a large vocabulary is written.
        _grad("train_step", 16_384, 131_072, 2048, "bf16", "bf16", 1.0, 64, False),
        # A further micro-batch added into the fp32 gradient that the program keeps: only the rows met are touched.
        _grad("accumulate", 32_768, 131_072, 4096, "bf16", "fp32", 64.0, 64, True),
        # Ragged: one token is a third of the batch, padding and pruned tokens, an odd width.
        _grad("hot_token", 65_537, 32_003, 1001, "fp16", "fp16", 0.5, 32, False, 0.3, 3, 0.05),
        # A trained table put into 4-bit rows and read back.
        _publish("publish", 65_536, 4096, 128, "bf16", "bf16"),
        # A small one, short last groups.
        _publish("publish_small", 4_099, 1000, 32, "fp32", "fp32"),
        # One state through a square layer: the smallest product, a single token's step.
        _linear("one_state", 1, 4096, 4096, 128, "bf16", "bf16", False),
        # Scores of a small batch over the vocabulary: the largest table.
        _linear("scores", 8, 131_072, 4096, 128, "bf16", "fp32", False),
        # An odd number of rows and states, short last groups, a bias.
        _linear("odd_layer", 5, 11_003, 5000, 32, "fp16", "fp16", True),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _dim(rng, step, hi=8192):
    d = _log(rng, 64, hi)
    return max(step, d // step * step)


def draw(rng):
    kind = rng.choice(["lookup", "grad", "grad", "packed", "publish", "linear", "linear"])
    rows = _log(rng, 256, 262_144)
    dim = _dim(rng, 8 if kind in ("packed", "publish", "linear") else rng.choice([1, 8, 64]))
    rows = max(1, min(rows, 500_000_000 // dim))
    tokens = max(1, min(_log(rng, 1, 131_072), 130_000_000 // dim))
    scale, bits, group = rng.choice([1.0, round(math.sqrt(dim), 3)]), rng.choice([32, 64]), rng.choice([32, 64, 128, 256])
    table, output = rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.choice(["bf16", "fp16", "fp32"])
    if kind == "lookup":
        c = _lookup("", tokens, rows, dim, table, rng.choice([table, output]), scale, bits, rng.choice([0.0, 0.1]))
    elif kind == "grad":
        into = rng.random() < 0.4
        c = _grad("", tokens, rows, dim, table, "fp32" if into else rng.choice([table, output]), scale, bits, into,
                  rng.choice([0.0, 0.0, 0.3]), rng.choice([-1, -1, 0]), rng.choice([0.0, 0.05]))
    elif kind == "packed":
        c = _packed("", tokens, rows, dim, group, output, scale, bits)
    elif kind == "publish":
        c = _publish("", max(1, min(rows, 250_000_000 // dim)), dim, group, table, output)
    else:
        states = rng.choice([1, 1, 2, 4, 8, rng.randint(1, 16)])
        c = _linear("", states, rows, dim, group, table, rng.choice([table, output]), rng.random() < 0.3)
    del c["name"]
    return c


# ---- what a case is made of -------------------------------------------------------------------------------------

def _weights(n):
    """Shares of n tokens by rank: Zipf's law with exponent 1.05, as words of a text have."""
    w = 1.0 / np.arange(1, n + 1) ** 1.05
    return w / w.sum()


def _tokens(case, gen):
    n, rows = case["tokens"], case["rows"]
    cdf = torch.from_numpy(np.cumsum(_weights(rows))).to(DEVICE)
    rank = torch.searchsorted(cdf, torch.rand(n, dtype=torch.float64, device=DEVICE, generator=gen)).clamp_(max=rows - 1)
    t = torch.randperm(rows, device=DEVICE, generator=gen)[rank]
    for share, value in ((case.get("hot", 0.0), rows // 2), (case.get("pruned", 0.0), -1)):
        if share:
            t[torch.rand(n, device=DEVICE, generator=gen) < share] = value
    return t.to(torch.int32 if case["bits"] == 32 else torch.int64)


def _group_rows(values, g):
    """fp32 [E, D] -> the bytes of 4-bit rows, and the fp32 numbers that those stand for."""
    E, D = values.shape
    G = -(-D // g)
    pad = G * g - D
    x = torch.cat([values, values[:, -1:].expand(E, pad)], 1) if pad else values      # a repeated value moves neither end of its group
    x = x.view(E, G, g)
    bias = x.amin(2).half()
    span = x.amax(2) - bias.float()
    scale = torch.where(span == 0, torch.ones_like(span), span / torch.full_like(span, 15.0)).half()   # a division: by a plain 15 torch multiplies by its inverse
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    inverse = 1.0 / scale.float()
    scale = torch.where(torch.isinf(inverse), torch.ones_like(scale), scale)
    inverse = torch.where(torch.isinf(inverse), torch.ones_like(inverse), inverse)
    q = ((x - bias.float()[..., None]) * inverse[..., None]).round().clamp(0, 15)
    back = (q * scale.float()[..., None] + bias.float()[..., None]).view(E, G * g)[:, :D]
    q = q.view(E, G * g)[:, :D].to(torch.uint8)
    head = torch.stack([scale, bias], 2).view(E, 2 * G).view(torch.uint8)
    out = torch.zeros(E, _row_bytes(D, g), dtype=torch.uint8, device=values.device)
    out[:, :D // 2] = q[:, 0::2] | (q[:, 1::2] << 4)
    out[:, D // 2:D // 2 + 4 * G] = head
    return out, back


def _values(rows, D, g):
    """The fp32 numbers that 4-bit rows stand for."""
    E, G = rows.shape[0], -(-D // g)
    byte = rows[:, :D // 2]
    q = torch.stack([byte & 15, byte >> 4], 2).view(E, D).float()
    head = rows[:, D // 2:D // 2 + 4 * G].contiguous().view(torch.float16).float().view(E, G, 2)
    of = torch.arange(D, device=rows.device) // g
    return q * head[:, of, 0] + head[:, of, 1]


def _row_bytes(D, g):
    return -(-(D // 2 + 4 * -(-D // g)) // 16) * 16


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    kind = case["kind"]

    def normal(n, d, dtype, std):
        return torch.empty(n, d, dtype=DTYPES[dtype], device=DEVICE).normal_(0.0, std, generator=gen)

    s = {"case": case}
    if kind == "lookup":
        s["weight"] = normal(case["rows"], case["dim"], case["table"], 0.02)
        s["tokens"] = _tokens(case, gen)
    elif kind == "grad":
        s["grad"] = normal(case["tokens"], case["dim"], case["grad"], 0.01)
        s["tokens"] = _tokens(case, gen)
        if case["into"]:
            s["into"] = normal(case["rows"], case["dim"], "fp32", 0.01)
    elif kind == "publish":
        s["weight"] = normal(case["rows"], case["dim"], case["table"], 0.02)
    else:
        step = max(1, 40_000_000 // case["dim"])
        s["rows"] = torch.cat([_group_rows(normal(min(step, case["rows"] - r), case["dim"], "fp32", 0.02), case["group"])[0]
                               for r in range(0, case["rows"], step)])
        if kind == "packed":
            s["tokens"] = _tokens(case, gen)
        else:
            s["hidden"] = normal(case["states"], case["dim"], case["hidden"], 1.0)
            s["bias"] = normal(1, case["rows"], case["output"], 0.1)[0] if case["bias"] else None
    return s


def run(s):
    c = s["case"]
    kind = c["kind"]
    if own:
        import fbgemm_ascend_b200  # noqa: F401  (registers the operators)
        ops = torch.ops.tbe_b200
        if kind == "lookup":
            return ops.token_embedding(s["weight"], s["tokens"], scale=c["scale"], output_dtype=CODES[c["output"]])
        if kind == "grad":
            padding = None if c["padding"] < 0 else c["padding"]
            if c["into"]:
                return ops.token_embedding_grad_(s["into"], s["grad"], s["tokens"], scale=c["scale"], padding_idx=padding)
            return ops.token_embedding_grad(s["grad"], s["tokens"], c["rows"], scale=c["scale"], padding_idx=padding, output_dtype=CODES[c["output"]])
        if kind == "packed":
            return ops.group_row_embedding(s["rows"], s["tokens"], c["dim"], c["group"], scale=c["scale"], output_dtype=CODES[c["output"]])
        if kind == "publish":
            return ops.group_rows_to_float(ops.quantize_to_group_rows(s["weight"], c["group"]), c["dim"], c["group"], output_dtype=CODES[c["output"]])
        return ops.group_row_linear(s["hidden"], s["rows"], c["group"], bias=s["bias"], output_dtype=CODES[c["output"]])

    if kind == "publish":
        return _group_rows(s["weight"].float(), c["group"])[1].to(DTYPES[c["output"]])
    if kind == "linear":
        y = s["hidden"].float() @ _values(s["rows"], c["dim"], c["group"]).t()
        return (y if s["bias"] is None else y + s["bias"].float()).to(DTYPES[c["output"]])
    t = s["tokens"].long()
    met = (t >= 0) & (t < c["rows"])
    if kind == "grad":
        met &= t != c["padding"]
        add = torch.where(met[:, None], s["grad"].float(), 0.0) * c["scale"]
        into = s["into"] if c["into"] else torch.zeros(c["rows"], c["dim"], dtype=torch.float32, device=t.device)
        into.index_add_(0, torch.where(met, t, 0), add)
        return into if c["into"] else into.to(DTYPES[c["output"]])
    at = torch.where(met, t, 0)
    rows = s["weight"][at].float() if kind == "lookup" else _values(s["rows"][at], c["dim"], c["group"])
    return torch.where(met[:, None], rows * c["scale"], 0.0).to(DTYPES[c["output"]])


# ---- what a pass cannot do without ------------------------------------------------------------------------------

def _distinct(case):
    """How many different rows the tokens are expected to name."""
    n = case["tokens"] * (1.0 - case.get("hot", 0.0)) * (1.0 - case.get("pruned", 0.0))
    return float(-np.expm1(n * np.log1p(-np.minimum(_weights(case["rows"]), 1 - 1e-12))).sum())


def work(case):
    D, kind = case["dim"], case["kind"]
    if kind == "publish":
        row = _row_bytes(D, case["group"])      # written by the one operator, read by the other
        return {"bytes": case["rows"] * (D * (SIZES[case["table"]] + SIZES[case["output"]]) + 2.0 * row), "flops": 4.0 * case["rows"] * D}
    if kind == "linear":
        m, n = case["states"], case["rows"]
        return {"bytes": float(n * _row_bytes(D, case["group"]) + m * D * SIZES[case["hidden"]] + (m + case["bias"]) * n * SIZES[case["output"]]),
                "flops": 2.0 * m * n * D}
    n = case["tokens"]
    out = SIZES[case["output"]]
    if kind == "lookup":
        return {"bytes": _distinct(case) * D * SIZES[case["table"]] + n * (D * out + case["bits"] / 8), "flops": float(n * D)}
    if kind == "packed":
        return {"bytes": _distinct(case) * _row_bytes(D, case["group"]) + n * (D * out + case["bits"] / 8), "flops": 3.0 * n * D}
    rows = 2 * _distinct(case) if case["into"] else case["rows"]
    return {"bytes": rows * D * out + n * (D * SIZES[case["grad"]] + case["bits"] / 8), "flops": 2.0 * n * D}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------

def _wide_rows(rows, D, g):
    """4-bit rows as numbers of 64 bits, group by group."""
    parts = []
    for k in range(-(-D // g)):
        lo, hi = k * g, min(D, (k + 1) * g)
        codes = rows[:, lo // 2:hi // 2].to(torch.int32)
        head = rows[:, D // 2 + 4 * k:D // 2 + 4 * k + 4].contiguous().view(torch.float16).double()
        part = torch.empty(rows.shape[0], hi - lo, dtype=torch.float64, device=rows.device)
        part[:, 0::2] = (codes % 16).double()
        part[:, 1::2] = (codes // 16).double()
        parts.append(part.mul_(head[:, :1]).add_(head[:, 1:]))
    return torch.cat(parts, 1)


def exact(case, seed):
    s = prepare(case, seed)
    D, kind = case["dim"], case["kind"]
    if kind == "publish":
        x, parts = s["weight"].double(), []
        for lo in range(0, D, case["group"]):
            v = x[:, lo:lo + case["group"]]
            bias = v.min(1, keepdim=True).values.half().double()
            # scale and codes are defined by these roundings to fp32 (the 4-bit rows of the whole package are): at a border
            # between two codes they decide, and a product with more bits would name the other one
            scale = ((v.max(1, keepdim=True).values - bias).float().double() / 15).float().half().double()
            scale[scale == 0] = 1.0
            steps = (v - bias).float().double() * (1.0 / scale).float().double()
            parts.append(torch.clamp(torch.round(steps.float().double()), 0, 15) * scale + bias)
        return torch.cat(parts, 1)
    if kind == "linear":
        out = torch.empty(case["states"], case["rows"], dtype=torch.float64, device=DEVICE)
        step = max(1, 100_000_000 // D)
        for r in range(0, case["rows"], step):
            out[:, r:r + step] = torch.einsum("mk,nk->mn", s["hidden"].double(), _wide_rows(s["rows"][r:r + step], D, case["group"]))
        return out if s["bias"] is None else out + s["bias"].double()
    t = s["tokens"].long()
    met = (t >= 0) & (t < case["rows"])
    if kind == "grad":
        met &= t != case["padding"]
        out = s["into"].double() if case["into"] else torch.zeros(case["rows"], D, dtype=torch.float64, device=DEVICE)
        return out.index_put_((t[met],), s["grad"][met].double() * case["scale"], accumulate=True)
    out = torch.zeros(case["tokens"], D, dtype=torch.float64, device=DEVICE)
    picked = s["weight"][t[met]].double() if kind == "lookup" else _wide_rows(s["rows"][t[met]], D, case["group"])
    out[met] = picked * case["scale"]
    return out
