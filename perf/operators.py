"""Cases of the 8-bit float operators: RMS norm with a block-quantised output, the quantiser with its activations, the
block-scaled product, and the product grouped by expert.

`run` computes a case in plain torch operations (`own` false) or through the package's operators (`own` true)."""
import math
import random

import torch

own = False

BLOCK = 128          # columns of one scale
TOP = 448.0          # the largest e4m3 value
LEAST = 2.0 ** -100  # block maxima below this count as this
F8 = torch.float8_e4m3fn
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}

_f8 = None


def _ops():
    global _f8
    if _f8 is None:
        from futon_b200 import f8
        _f8 = f8
    return _f8


def listed():
    return [
        # The norm before a product, one token: a call's latency.
        {"name": "norm token", "op": "norm", "rows": 1, "k": 4096, "type": "bf16", "residual": True},
        # A batch of packed tokens at the hidden width of the nomic and arctic packs.
        {"name": "norm batch", "op": "norm", "rows": 32768, "k": 768, "type": "f16", "residual": True},
        # A width that ends inside a block of 128, f32 rows without a residual.
        {"name": "norm odd", "op": "norm", "rows": 4099, "k": 5000, "type": "f32", "residual": False},
        # Between the two products of a SwiGLU feed-forward block, a batch of packed tokens.
        {"name": "quantize swiglu", "op": "quantize", "rows": 16384, "k": 1536, "type": "f16", "act": "swiglu", "block_rows": 1},
        # A weight matrix laid out in 128 x 128 blocks.
        {"name": "quantize weights", "op": "quantize", "rows": 4096, "k": 4096, "type": "f32", "act": "none", "block_rows": 128},
        # One token through a square projection: the weights are all there is to read.
        {"name": "product token", "op": "product", "m": 1, "n": 4096, "k": 4096, "out": "bf16", "bias": False},
        # A short query through the qkv projection of a small encoder, with its bias.
        {"name": "product short", "op": "product", "m": 37, "n": 1152, "k": 384, "out": "f32", "bias": True},
        # A batch of a few short texts.
        {"name": "product middle", "op": "product", "m": 500, "n": 4096, "k": 2048, "out": "f16", "bias": False},
        # A long batch: the tensor cores are the bound.
        {"name": "product large", "op": "product", "m": 8192, "n": 8192, "k": 4096, "out": "bf16", "bias": False},
        # Experts with a token or two each: all their weights are read.
        {"name": "experts tokens", "op": "grouped", "groups": 32, "m": 64, "n": 2048, "k": 2048, "type": "e4m3", "out": "bf16", "rest": 0},
        # Experts over a long batch, ragged, some of them empty.
        {"name": "experts batch", "op": "grouped", "groups": 16, "m": 8192, "n": 4096, "k": 2048, "type": "e4m3", "out": "bf16", "rest": 0},
        # The same in f16 with rows behind the last group, at an encoder's widths.
        {"name": "experts f16", "op": "grouped", "groups": 8, "m": 6001, "n": 1536, "k": 768, "type": "f16", "out": "f16", "rest": 29},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["norm", "quantize", "product", "grouped"])
    if op == "norm":
        k = rng.choice([8 * log(8, 1024), log(1, 9000)])
        return {"op": op, "rows": log(1, min(40000, (1 << 26) // k)), "k": k, "type": rng.choice(["f32", "f16", "bf16"]),
                "residual": rng.random() < 0.7}
    if op == "quantize":
        k = rng.choice([8 * log(4, 1024), log(1, 9000)])
        act, block_rows = rng.choice([("none", 1), ("none", BLOCK), ("gelu", 1), ("swiglu", 1)])
        return {"op": op, "rows": log(1, min(20000, (1 << 25) // k)), "k": k, "type": rng.choice(["f32", "f16", "bf16"]),
                "act": act, "block_rows": block_rows}
    k = rng.choice([16 * log(2, 512), 64 * log(1, 100), log(1, 3000)])
    n = rng.choice([128 * log(1, 64), log(1, 8192)])
    out = rng.choice(["f32", "f16", "bf16"])
    if op == "product":
        return {"op": op, "m": log(1, min(16384, (1 << 37) // (n * k))), "n": n, "k": k, "out": out, "bias": rng.random() < 0.5}
    groups = log(1, max(1, min(64, (1 << 28) // (n * k))))
    m = log(1, min(12000, (1 << 35) // (n * k)))
    return {"op": op, "groups": groups, "m": m, "n": n, "k": k, "type": rng.choice(["e4m3", "e4m3", "f16", "bf16"]), "out": out,
            "rest": rng.choice([0, 0, min(3, m - 1)])}


def work(case):
    op = case["op"]
    if op in ("norm", "quantize"):
        e, r, k = SIZE[case["type"]], case["rows"], case["k"]
        nb = -(-k // BLOCK)
        if op == "norm":
            return {"bytes": r * k * (e * (3 if case["residual"] else 1) + 1) + 4 * r * nb + 4 * k, "flops": 6 * r * k}
        scales = -(-r // case["block_rows"]) * nb
        return {"bytes": r * k * (e * (2 if case["act"] == "swiglu" else 1) + 1) + 4 * scales,
                "flops": r * k * {"none": 3, "gelu": 12, "swiglu": 10}[case["act"]]}
    m, n, k = case["m"], case["n"], case["k"]
    nb, nn = -(-k // BLOCK), -(-n // BLOCK)
    if op == "product":
        return {"bytes": m * k + n * k + 4 * nb * (m + nn) + m * n * SIZE[case["out"]] + (4 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    e = SIZE[case["type"]]
    used = min(case["groups"], m - case["rest"])
    rows = m - case["rest"]
    scales = 4 * nb * (rows + used * nn) if e == 1 else 0
    return {"bytes": rows * k * e + used * n * k * e + scales + rows * n * SIZE[case["out"]] + 4 * (case["groups"] + 1),
            "flops": 2 * rows * n * k}


def _quantised(y, block_rows):
    """y [r, k] in 32 bits -> its e4m3 codes and the scales of its blocks."""
    r, k = y.shape
    y = torch.nn.functional.pad(y, (0, -k % BLOCK, 0, -r % block_rows))
    b = y.view(y.shape[0] // block_rows, block_rows, y.shape[1] // BLOCK, BLOCK)
    top = b.abs().amax(dim=(1, 3), keepdim=True).clamp_min(LEAST)
    codes = (b * (TOP / top)).to(F8)
    return codes.view(y.shape)[:r, :k], (top / TOP).view(top.shape[0], top.shape[2])


def _values(q, scales, block_rows):
    """The values that codes and scales stand for, in 32 bits."""
    r, k = q.shape[-2:]
    s = scales.repeat_interleave(BLOCK, -1)[..., :k]
    return q.float() * (s if block_rows == 1 else s.repeat_interleave(block_rows, -2)[..., :r, :])


def _pitched(t):
    """t with rows that begin at multiples of 16 bytes, as the products take them."""
    k = t.shape[-1]
    wide = -(-k * t.element_size() // 16) * 16 // t.element_size()
    if wide == k:
        return t.contiguous()
    room = torch.zeros(*t.shape[:-1], wide, dtype=torch.float32, device=t.device).to(t.dtype)
    room[..., :k] = t
    return room[..., :k]


def _activations(g, rows, k):
    """Rows as a trained encoder has them: a spread of row sizes and a few loud channels."""
    x = torch.randn(rows, k, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(rows, 1, generator=g, device="cuda"))
    loud = torch.rand(k, generator=g, device="cuda") < 0.01
    return x * torch.where(loud, 20.0, 1.0)


def _weights(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda") * 0.02


def _sizes(case, seed):
    """Rows of each group: ragged, some empty, none over four times the mean (or 8 rows)."""
    rng, rows, n = random.Random(seed), case["m"] - case["rest"], case["groups"]
    most = max(8, -(-4 * rows // n))
    share = [0.0 if n > 2 and rng.random() < 0.1 else rng.expovariate(1.0) + 0.02 for _ in range(n)]
    if not any(share):
        share[0] = 1.0
    total = sum(share)
    sizes = [min(most, int(rows * s / total)) for s in share]
    left = rows - sum(sizes)
    while left:
        i = rng.randrange(n)
        if sizes[i] < most:
            add = min(left, most - sizes[i], max(1, left // 4))
            sizes[i] += add
            left -= add
    return sizes


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, s = case["op"], {"case": case}
    if op == "norm":
        r, k, t = case["rows"], case["k"], TYPES[case["type"]]
        s["x"] = _activations(g, r, k).to(t)
        s["weight"] = 1.0 + 0.1 * torch.randn(k, generator=g, device="cuda")
        s["residual"] = (2.0 * torch.randn(r, k, generator=g, device="cuda")).to(t) if case["residual"] else None
        s["eps"] = 1e-6
        wide = -(-k // 16) * 16
        s["q"] = torch.zeros(r, wide, dtype=torch.uint8, device="cuda").view(F8)[:, :k]
        s["scales"] = torch.zeros(r, -(-k // BLOCK), device="cuda")
        s["sum"] = torch.zeros_like(s["x"]) if case["residual"] else None
    elif op == "quantize":
        r, k, t = case["rows"], case["k"], TYPES[case["type"]]
        if case["block_rows"] == 1:
            s["src"] = _activations(g, r, 2 * k if case["act"] == "swiglu" else k).to(t)
        else:
            s["src"] = _weights(g, r, k).to(t)
        wide = -(-k // 16) * 16
        s["q"] = torch.zeros(r, wide, dtype=torch.uint8, device="cuda").view(F8)[:, :k]
        s["scales"] = torch.zeros(-(-r // case["block_rows"]), -(-k // BLOCK), device="cuda")
    elif op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        a, s["a_scales"] = _quantised(_activations(g, m, k), 1)
        b, s["b_scales"] = _quantised(_weights(g, n, k), BLOCK)
        s["a"], s["b"] = _pitched(a), _pitched(b)
        s["bias"] = torch.randn(n, generator=g, device="cuda") if case["bias"] else None
        s["out"] = torch.zeros(m, n, dtype=TYPES[case["out"]], device="cuda")
    else:
        m, n, k, e = case["m"], case["n"], case["k"], case["groups"]
        sizes = _sizes(case, seed)
        s["most"] = max(sizes)
        s["offsets"] = torch.tensor([sum(sizes[:i]) for i in range(e + 1)], dtype=torch.int32, device="cuda")
        a, w = _activations(g, m, k), _weights(g, e, n, k)
        if case["type"] == "e4m3":
            q, s["a_scales"] = _quantised(a, 1)
            rows = -(-n // BLOCK) * BLOCK
            w = torch.nn.functional.pad(w, (0, 0, 0, rows - n))
            wq, ws = _quantised(w.view(e * rows, k), BLOCK)
            s["b_scales"] = ws.view(e, rows // BLOCK, -1)
            s["a"], s["b"] = _pitched(q), _pitched(wq.reshape(e, rows, k)[:, :n])
        else:
            t = TYPES[case["type"]]
            s["a"], s["b"], s["a_scales"], s["b_scales"] = _pitched(a.to(t)), _pitched(w.to(t)), None, None
        s["out"] = torch.full((m, n), 3.0, dtype=TYPES[case["out"]], device="cuda")
    return s


def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    case, ops = s["case"], _ops()
    op = case["op"]
    if op == "norm":
        ops.rms_norm_f8(s["x"], s["weight"], s["eps"], residual=s["residual"], residual_out=s["sum"], out=(s["q"], s["scales"]))
        return [s["q"], s["scales"], s["sum"]]
    if op == "quantize":
        return list(ops.quantize_f8(s["src"], activation=case["act"], block_rows=case["block_rows"], out=(s["q"], s["scales"])))
    if op == "product":
        return ops.matmul_t_f8(s["a"], s["a_scales"], s["b"], s["b_scales"], bias=s["bias"], out=s["out"])
    return ops.matmul_t_grouped(s["a"], s["b"], s["offsets"], a_scales=s["a_scales"], b_scales=s["b_scales"], out=s["out"])


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op == "norm":
        h = s["x"].float()
        if s["residual"] is not None:
            h = h + s["residual"].float()
        y = h * torch.rsqrt((h * h).mean(dim=1, keepdim=True) + s["eps"]) * s["weight"]
        q, scales = _quantised(y, 1)
        return [q, scales, h.to(s["x"].dtype) if s["residual"] is not None else None]
    if op == "quantize":
        y = s["src"].float()
        if case["act"] == "gelu":
            y = 0.5 * y * torch.special.erfc(y * -math.sqrt(0.5))
        elif case["act"] == "swiglu":
            up, gate = y.chunk(2, dim=1)
            y = up * (gate / (1.0 + torch.exp(-gate)))
        return list(_quantised(y, case["block_rows"]))
    if op == "product":
        d = _values(s["a"], s["a_scales"], 1) @ _values(s["b"], s["b_scales"], BLOCK).t()
        if s["bias"] is not None:
            d = d + s["bias"]
        return d.to(s["out"].dtype)
    # Grouped: the rows of each group in a slab of its own, one batched product, and back.
    e8 = case["type"] == "e4m3"
    a = _values(s["a"], s["a_scales"], 1) if e8 else s["a"].float()
    b = _values(s["b"], s["b_scales"], BLOCK) if e8 else s["b"].float()
    off = s["offsets"].long()
    row = torch.arange(case["m"] - case["rest"], device=a.device)
    group = torch.bucketize(row, off[1:], right=True)
    at = row - off[group]
    slabs = torch.zeros(case["groups"], max(1, s["most"]), case["k"], device=a.device)
    slabs[group, at] = a[: row.numel()]
    d = torch.bmm(slabs, b.transpose(1, 2))
    out = torch.full_like(s["out"], 3.0)
    out[: row.numel()] = d[group, at].to(out.dtype)
    return out


def exact(case, seed):
    """The definitions in 64 bits; codes come unrounded, as the numbers that the 8 bits are nearest to."""
    s = prepare(case, seed)
    op = case["op"]

    def blockwise(y, rows):
        r, k = y.shape
        codes, scales = torch.empty_like(y), torch.empty(-(-r // rows), -(-k // 128), dtype=torch.float64, device=y.device)
        for c in range(scales.shape[1]):
            part = y[:, 128 * c:128 * (c + 1)].abs().max(dim=1).values
            part = torch.nn.functional.pad(part, (0, -r % rows)).view(-1, rows).max(dim=1).values
            top = torch.maximum(part, torch.full_like(part, 2.0 ** -100))
            scales[:, c] = top / 448
            codes[:, 128 * c:128 * (c + 1)] = y[:, 128 * c:128 * (c + 1)] * (448 / top).repeat_interleave(rows)[:r, None]
        return codes, scales

    def widened(q, scales, rows):
        r, k = q.shape
        v = q.double()
        for c in range(scales.shape[1]):
            v[:, 128 * c:128 * (c + 1)] *= scales[:, c].double().repeat_interleave(rows)[:r, None]
        return v

    if op == "norm":
        h = s["x"].double() if s["residual"] is None else s["x"].double() + s["residual"].double()
        y = h / torch.sqrt(h.square().sum(dim=1, keepdim=True) / case["k"] + s["eps"]) * s["weight"].double()
        return [*blockwise(y, 1), None if s["residual"] is None else h]
    if op == "quantize":
        y = s["src"].double()
        if case["act"] == "gelu":
            y = y * torch.special.erfc(-y / math.sqrt(2)) / 2
        elif case["act"] == "swiglu":
            y = y[:, :case["k"]] * y[:, case["k"]:] * torch.sigmoid(y[:, case["k"]:])
        return list(blockwise(y, case["block_rows"]))
    if op == "product":
        d = torch.matmul(widened(s["a"], s["a_scales"], 1), widened(s["b"], s["b_scales"], 128).t())
        return d if s["bias"] is None else d + s["bias"].double()
    out, off = s["out"].double(), s["offsets"].tolist()
    for i in range(case["groups"]):
        lo, hi = off[i], off[i + 1]
        if hi > lo:
            if case["type"] == "e4m3":
                a, b = widened(s["a"][lo:hi], s["a_scales"][lo:hi], 1), widened(s["b"][i], s["b_scales"][i], 128)
            else:
                a, b = s["a"][lo:hi].double(), s["b"][i].double()
            out[lo:hi] = torch.matmul(a, b.t())
    return out
