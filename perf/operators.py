"""Cases of the scalar-quantised row operators: what is timed, with a plain form of each.

A store of scalar-quantised rows holds `capacity` rows of `d` values as 8-bit or
4-bit codes and one fp32 scale for each group of a row:

    scale = fp32(max |x| over the group / L)         L = 127 (8 bits) or 7 (4 bits)
    code  = round-half-even(x / scale), within [-L, L]; 0 where the scale is 0
    value = code * scale

`write`   rows go to their slots of the store (a slot outside the store is left
          out, of two rows with one slot the later stays); the store is then read back
`read`    rows of the store are gathered and turned back into values
`matmul`  8-bit product: (a . b) * a_scale[row of a] * b_scale[row of b] + bias[row of b]
`scores`  floating rows, quantised one scale a row, then that product with every row of a store
"""
import math
import os
import sys

import torch

own = False

F32, F16, BF16 = "float32", "float16", "bfloat16"


def _library():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "insituann-opensource_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import insitu_b200

    return insitu_b200


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one embedding inserted online into a small store: latency
        {"name": "write 1x128 f32", "op": "write", "n": 1, "capacity": 64, "d": 128, "type": F32, "bits": 8,
         "group": 0, "repeats": False},
        # a query batch of unit vectors, every row to a slot of its own
        {"name": "write 10000x96 f32", "op": "write", "n": 10000, "capacity": 10000, "d": 96, "type": F32, "bits": 8,
         "group": 0, "repeats": False},
        # 4-bit groups, a width that no group divides, slots that repeat or are left out
        {"name": "write 4099x1000 f16 4 bits", "op": "write", "n": 4099, "capacity": 5000, "d": 1000, "type": F16,
         "bits": 4, "group": 64, "repeats": True},
        # a million embeddings loaded in an order of their own
        {"name": "write 1Mx128 bf16", "op": "write", "n": 1000000, "capacity": 1100000, "d": 128, "type": BF16,
         "bits": 8, "group": 0, "repeats": False},
        # the 512 candidates of each of 10000 queries, read back for a rerank
        {"name": "read 5.12Mx128 bf16", "op": "read", "n": 5120000, "capacity": 2000000, "d": 128, "type": BF16,
         "bits": 8, "group": 0},
        # 4-bit rows read back in fp32
        {"name": "read 65537x96 f32 4 bits", "op": "read", "n": 65537, "capacity": 100000, "d": 96, "type": F32,
         "bits": 4, "group": 32},
        # a few tokens against a weight of a layer: bound by reading the weight
        {"name": "matmul 16x16384x4096 bf16", "op": "matmul", "m": 16, "n": 16384, "k": 4096, "type": BF16,
         "bias": False, "packed": False},
        # odd sizes, rows one after another without padding (no 16-byte alignment)
        {"name": "matmul 333x10007x1031 f16", "op": "matmul", "m": 333, "n": 10007, "k": 1031, "type": F16,
         "bias": True, "packed": True},
        # the largest square product: bound by the tensor cores
        {"name": "matmul 8192x8192x8192 bf16", "op": "matmul", "m": 8192, "n": 8192, "k": 8192, "type": BF16,
         "bias": True, "packed": False},
        # one query against 65536 rows: latency
        {"name": "scores 1x65536x128 f32", "op": "scores", "m": 1, "n": 65536, "k": 128, "type": F32, "out": F32},
        # a query batch against 4096 rows
        {"name": "scores 10000x4096x96 f32", "op": "scores", "m": 10000, "n": 4096, "k": 96, "type": F32, "out": F32},
        # 256 queries against a million rows: bound by writing the scores
        {"name": "scores 256x1Mx128 bf16", "op": "scores", "m": 256, "n": 1000000, "k": 128, "type": BF16,
         "out": F32},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm; now and then a multiple of 16."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.3 and v > 16:
        v = v // 16 * 16
    return min(hi, max(lo, v))


def draw(rng):
    op = rng.choice(["write", "read", "matmul", "scores"])
    kind = rng.choice([F32, F16, BF16])
    if op in ("write", "read"):
        d = _log(rng, 1, 2048)
        n = _log(rng, 1, min(1000000, (1 << 27) // d))
        bits = rng.choice([8, 8, 4])
        group = rng.choice([0, 0, 32, 64, 128])
        case = {"op": op, "n": n, "capacity": n + rng.randrange(n // 8 + 2), "d": d, "type": kind, "bits": bits,
                "group": group}
        if op == "write":
            case["repeats"] = rng.random() < 0.4
        return case
    k = _log(rng, 1, 8192)
    m = _log(rng, 1, 8192)
    n = _log(rng, 1, min(1000000, (1 << 27) // m, (1 << 37) // (m * k), (1 << 28) // k))
    if op == "matmul":
        return {"op": op, "m": m, "n": n, "k": k, "type": kind, "bias": rng.random() < 0.5,
                "packed": rng.random() < 0.3}
    return {"op": op, "m": m, "n": n, "k": k, "type": kind, "out": rng.choice([F32, F16, BF16])}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _type(name):
    return getattr(torch, name)


def _rows(n, d, kind, g):
    """Embeddings: a few directions stronger than the others, rows of different lengths, some rows of zeros."""
    x = torch.randn(n, d, generator=g, device="cuda")
    x *= 1.0 + 4.0 * (torch.rand(d, generator=g, device="cuda") < 0.03)
    x *= torch.exp(0.5 * torch.randn(n, 1, generator=g, device="cuda")) / math.sqrt(d)
    x *= torch.rand(n, 1, generator=g, device="cuda") >= 0.01 if n > 16 else 1.0
    return x.to(_type(kind))


def _codes(n, k, top, g, packed=False):
    """[n, k] codes of int8, bell-shaped as the codes of embeddings; rows 16-byte aligned unless packed."""
    ld = k if packed else (k + 15) // 16 * 16
    c = torch.zeros(n, ld, dtype=torch.int8, device="cuda")
    step = max(1, (1 << 27) // max(k, 1))
    for i in range(0, n, step):
        r = torch.randn(min(step, n - i), k, generator=g, device="cuda")
        c[i:i + step, :k] = (r * (top / 3.5)).round_().clamp_(-top, top).to(torch.int8)
    return c[:, :k]


def _scales(shape, g):
    return torch.exp(0.5 * torch.randn(shape, generator=g, device="cuda")) * 1e-3


def _groups(d, group):
    return -(-d // group) if group else 1


def _pack(codes, bits):
    """Codes as the store holds them: int8, or two 4-bit codes a byte, the even one in the low half."""
    if bits == 8:
        return codes
    lo = codes[:, 0::2].to(torch.uint8) & 15
    hi = torch.zeros_like(lo)
    hi[:, :codes.shape[1] // 2] = codes[:, 1::2].to(torch.uint8) & 15
    return lo | (hi << 4)


def _row_bytes(d, bits):
    return ((d if bits == 8 else (d + 1) // 2) + 15) // 16 * 16


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    s = dict(case)
    if case["op"] == "write":
        n, cap, d = case["n"], case["capacity"], case["d"]
        s["x"] = _rows(n, d, case["type"], g)
        slots = torch.randperm(cap, generator=g, device="cuda")[:n]
        if case["repeats"]:
            u = torch.rand(n, generator=g, device="cuda")
            slots = torch.where(u < 0.1, slots[torch.randint(0, n, (n,), generator=g, device="cuda")], slots)
            slots = torch.where(u > 0.95, -1, slots)
        s["slots"] = slots
        s["codes"] = torch.zeros(cap, _row_bytes(d, case["bits"]), dtype=torch.int8 if case["bits"] == 8 else torch.uint8,
                                 device="cuda")
        s["scales"] = torch.zeros(cap, _groups(d, case["group"]), device="cuda")
    elif case["op"] == "read":
        n, cap, d, top = case["n"], case["capacity"], case["d"], 127 if case["bits"] == 8 else 7
        packed = _pack(_codes(cap, d, top, g), case["bits"])
        s["codes"] = torch.zeros(cap, _row_bytes(d, case["bits"]), dtype=packed.dtype, device="cuda")
        s["codes"][:, :packed.shape[1]] = packed
        s["scales"] = _scales((cap, _groups(d, case["group"])), g)
        s["slots"] = torch.randint(0, cap, (n,), generator=g, device="cuda")
    else:
        m, n, k = case["m"], case["n"], case["k"]
        packed = bool(case.get("packed"))
        s["b"] = _codes(n, k, 127, g, packed)
        s["b_scale"] = _scales((n,), g)
        if case["op"] == "matmul":
            s["a"] = _codes(m, k, 127, g, packed)
            s["a_scale"] = _scales((m,), g)
            s["bias"] = torch.randn(n, generator=g, device="cuda") if case["bias"] else None
        else:
            s["x"] = _rows(m, k, case["type"], g)
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

def _quantise(x, bits, group):
    """(codes int8 [n, d], scales fp32 [n, groups]) of floating rows."""
    n, d = x.shape
    top = 127.0 if bits == 8 else 7.0
    width, groups = (group, _groups(d, group)) if group else (d, 1)
    v = torch.nn.functional.pad(x.float(), (0, groups * width - d)).view(n, groups, width)
    amax = v.abs().amax(2)
    scale = amax / torch.full_like(amax, top)
    # the quotient in 64 bits: in 32 a value next to a border between two codes may fall on it
    q = torch.round(v.double() / scale.double()[:, :, None]).clamp(-top, top)
    q = torch.where(scale[:, :, None] > 0, q, 0.0)
    return q.view(n, -1)[:, :d].to(torch.int8), scale


def _values(codes, scales, d, bits, group, kind):
    """Values of rows as the store holds them."""
    if bits == 4:
        lo = (codes & 15).to(torch.int8)
        hi = (codes >> 4).to(torch.int8)
        q = torch.stack((lo, hi), 2).view(codes.shape[0], -1)
        q = torch.where(q > 7, q - 16, q)
    else:
        q = codes
    s = scales.repeat_interleave(group, 1)[:, :d] if group else scales
    return (q[:, :d].float() * s).to(_type(kind))


def _plain_write(s):
    x, slots, bits, group, d = s["x"], s["slots"], s["bits"], s["group"], s["d"]
    codes, scales = _quantise(x, bits, group)
    row = torch.arange(x.shape[0], device=x.device)
    inside = (slots >= 0) & (slots < s["capacity"])
    at = torch.where(inside, slots, s["capacity"])
    last = torch.full((s["capacity"] + 1,), -1, device=x.device).scatter_reduce(0, at, row, "amax")[:-1]
    to = torch.nonzero(last >= 0)[:, 0]
    stored = _pack(codes, bits)
    s["codes"][to, :stored.shape[1]] = stored[last[to]]
    s["scales"][to] = scales[last[to]]
    return {"values": _values(s["codes"], s["scales"], d, bits, group, s["type"]), "scales": s["scales"]}


def _product(a, a_scale, b, b_scale, bias, kind):
    # the sums of products in 64 bits: in 32 they are whole up to 2^24 only
    y = (a.double() @ b.double().t()) * a_scale.double()[:, None] * b_scale.double()
    if bias is not None:
        y = y + bias.double()
    return y.to(_type(kind))


def run(state):
    s = state
    if own:
        return _run_own(s)
    if s["op"] == "write":
        return _plain_write(s)
    if s["op"] == "read":
        return _values(s["codes"][s["slots"]], s["scales"][s["slots"]], s["d"], s["bits"], s["group"], s["type"])
    if s["op"] == "matmul":
        return _product(s["a"], s["a_scale"], s["b"], s["b_scale"], s["bias"], s["type"])
    a, a_scale = _quantise(s["x"], 8, 0)
    return _product(a, a_scale[:, 0], s["b"], s["b_scale"], None, s["out"])


def _run_own(s):
    ib = _library()
    if s["op"] == "matmul":
        return ib.sq_matmul(s["a"], s["a_scale"], s["b"], s["b_scale"], bias=s["bias"],
                            dtype=_type(s["type"]))
    if "rows" not in s:   # the store that a program keeps
        if s["op"] == "scores":
            s["rows"] = ib.SQRows.from_arrays(s["b"], s["b_scale"][:, None], s["k"])
        else:
            s["rows"] = ib.SQRows.from_arrays(s["codes"], s["scales"], s["d"], bits=s["bits"], group=s["group"])
    rows = s["rows"]
    if s["op"] == "write":
        rows.write(s["x"], s["slots"])
        return {"values": rows.read(dtype=s["x"].dtype), "scales": rows.scales}
    if s["op"] == "read":
        return rows.read(s["slots"], dtype=_type(s["type"]))
    return rows.scores(s["x"], dtype=_type(s["out"]))


# ---------------------------------------------------------------------------
# the least work, and the definition in 64 bits
# ---------------------------------------------------------------------------

def work(case):
    size = {F32: 4, F16: 2, BF16: 2}
    if case["op"] in ("write", "read"):
        n, cap, d = case["n"], case["capacity"], case["d"]
        held = (d * case["bits"] + 7) // 8 + 4 * _groups(d, case["group"])
        value = d * size[case["type"]]
        if case["op"] == "write":
            # rows and slots in, codes and scales out; the store in and its values out
            return {"bytes": n * (value + 8 + held) + cap * (held + value), "flops": 3 * n * d + cap * d}
        # a row that several slots name is read once
        distinct = min(n, cap)
        return {"bytes": n * (8 + value) + distinct * held, "flops": n * d}
    m, n, k = case["m"], case["n"], case["k"]
    out = size[case.get("out", case["type"])]
    a = k + 4 if case["op"] == "matmul" else k * size[case["type"]]
    return {"bytes": m * a + n * (k + 4) + (4 * n if case.get("bias") else 0) + m * n * out,
            "flops": 2 * m * n * k + 2 * m * n}


def _exact_codes(x, top):
    """(codes, scales) of the groups [..., width] in 64 bits; the scale is rounded to the 32 bits it is held in."""
    x = x.to(torch.float64)
    scale = (x.abs().max(-1, keepdim=True).values / top).to(torch.float32).to(torch.float64)
    inv = torch.where(scale > 0, scale, torch.ones_like(scale))
    return torch.clamp((x / inv).round(), -top, top) * (scale > 0), scale


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "write":
        d, cap, top = case["d"], case["capacity"], 127 if case["bits"] == 8 else 7
        width = case["group"] or d
        values = torch.zeros(cap, d, dtype=torch.float64, device="cuda")
        scales = torch.zeros(cap, _groups(d, case["group"]), dtype=torch.float64, device="cuda")
        # the row that stays in each slot: the last one that names it
        order = torch.sort(s["slots"], stable=True)
        ends = torch.ones_like(order.values, dtype=torch.bool)
        ends[:-1] = order.values[1:] != order.values[:-1]
        keep = ends & (order.values >= 0) & (order.values < cap)
        slot, row = order.values[keep], order.indices[keep]
        for j, lo in enumerate(range(0, d, width)):
            q, scale = _exact_codes(s["x"][:, lo:lo + width], top)
            values[slot, lo:lo + width] = (q * scale)[row]
            scales[slot, j] = scale[row, 0]
        return {"values": values, "scales": scales}
    if case["op"] == "read":
        d, width = case["d"], case["group"] or case["d"]
        held, scale = s["codes"].to(torch.int64), s["scales"].to(torch.float64)
        place = torch.arange(d, device="cuda")
        if case["bits"] == 4:
            nibble = (held[:, place // 2] >> (4 * (place % 2))) & 15
            q = nibble - 16 * (nibble >= 8)
        else:
            q = held[:, :d]
        return (q * scale[:, place // width])[s["slots"]]
    if case["op"] == "matmul":
        a = s["a"].to(torch.float64) * s["a_scale"].to(torch.float64)[:, None]
        y = torch.matmul(a, (s["b"].to(torch.float64) * s["b_scale"].to(torch.float64)[:, None]).t())
        return y if s["bias"] is None else y + s["bias"]
    q, scale = _exact_codes(s["x"], 127)
    return torch.matmul(q * scale, (s["b"].to(torch.float64) * s["b_scale"].to(torch.float64)[:, None]).t())
