"""What is measured of the mixture-of-experts operators: routing, dispatch and combine (with their
gradients), quantisation to 8 bits, and the 8-bit matrix product with a scale for each block of 128.

``run`` computes them in their plain form, or (``own``) through the package's entry points.
"""
from __future__ import annotations

import functools
import math

import torch

own = False

BLOCK = 128
FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0
SCALE_MIN = 2.0 ** -120
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
WIDTH = {"bf16": 2, "f32": 4}


def _ceil(a: int, b: int) -> int:
    return -(-a // b)


def _rows(case: dict) -> int:
    """Rows of the sorted buffer: the case's own number, or what holds every routing outcome."""
    if case.get("rows"):
        return case["rows"]
    n, block = case["tokens"] * case["choices"], case["block"]
    return (n + min(case["experts"], n) * (block - 1)) // block * block


# ---------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------

def listed() -> list[dict]:
    return [
        # one token through a linear layer whose weight is held in 8 bits: the weight's bytes count
        {"name": "gemm-token", "op": "gemm", "m": 1, "n": 4096, "k": 4096, "out": "bf16"},
        # a short prompt against a layer whose sizes fill no tile; the f32 output of a last layer
        {"name": "gemm-ragged", "op": "gemm", "m": 333, "n": 2056, "k": 1040, "out": "f32"},
        # a batch of prompts: the tensor cores count
        {"name": "gemm-prompts", "op": "gemm", "m": 8192, "n": 8192, "k": 4096, "out": "bf16"},
        # 32 sequences, one token each, four experts of 64: about two rows an expert
        {"name": "experts-decode", "op": "experts", "tokens": 32, "choices": 4, "experts": 64, "n": 2048, "k": 2048,
         "out": "bf16"},
        # prompts of 8192 tokens over 32 experts of unequal load
        {"name": "experts-prompts", "op": "experts", "tokens": 8192, "choices": 4, "experts": 32, "n": 4096, "k": 2048,
         "out": "bf16"},
        # the activations of a batch of prompts before an 8-bit product
        {"name": "quantize-tokens", "op": "quantize", "m": 8192, "k": 8192, "block_rows": 1, "input": "bf16"},
        # a weight when it is loaded: 128 x 128 blocks, from f32
        {"name": "quantize-weight", "op": "quantize", "m": 4096, "k": 4096, "block_rows": 128, "input": "f32"},
        # 16 sequences, one token each, routed and sorted straight into 8 bits
        {"name": "dispatch-decode", "op": "dispatch", "tokens": 16, "choices": 8, "experts": 128, "width": 4096,
         "block": 1, "form": "fp8", "input": "bf16", "train": False, "rows": 0, "dropped": 0.0},
        # odd sizes, f32, and entries that belong to another rank's experts; with the gradient
        {"name": "dispatch-ragged", "op": "dispatch", "tokens": 1001, "choices": 3, "experts": 10, "width": 1004,
         "block": 16, "form": "rows", "input": "f32", "train": True, "rows": 0, "dropped": 0.3},
        # a training step's tokens, padded for the grouped product's 128-row tiles; with the gradient
        {"name": "dispatch-train", "op": "dispatch", "tokens": 8192, "choices": 4, "experts": 32, "width": 4096,
         "block": 128, "form": "rows", "input": "bf16", "train": True, "rows": 0, "dropped": 0.0},
        # 16 sequences, one token each, coming back
        {"name": "combine-decode", "op": "combine", "tokens": 16, "choices": 8, "experts": 128, "width": 4096,
         "block": 1, "input": "bf16", "train": False, "rows": 0, "dropped": 0.0},
        # a training step's tokens coming back, with the gradients of rows and weights
        {"name": "combine-train", "op": "combine", "tokens": 8192, "choices": 4, "experts": 32, "width": 4096,
         "block": 128, "input": "bf16", "train": True, "rows": 0, "dropped": 0.0},
    ]


def _spread(rng, low: int, high: int, step: int = 1) -> int:
    """A multiple of `step` in [low, high], even over the logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high + 1)))
    return min(high, max(low, int(v / step) * step if v >= step else step))


def draw(rng) -> dict:
    while True:
        op = rng.choice(["gemm", "gemm", "experts", "quantize", "dispatch", "dispatch", "combine"])
        kind = rng.choice(["bf16", "bf16", "f32"])
        if op == "gemm":
            case = {"op": op, "m": _spread(rng, 1, 8192), "n": _spread(rng, 64, 8192, 8), "k": _spread(rng, 64, 8192, 16),
                    "out": kind}
            if case["m"] * case["n"] * case["k"] <= 8192 * 8192 * 4096:
                return case
            continue
        if op == "quantize":
            return {"op": op, "m": _spread(rng, 1, 8192), "k": _spread(rng, 64, 8192, 16),
                    "block_rows": rng.choice([1, 1, 128]), "input": kind}
        experts = _spread(rng, 1, 256)
        case = {"op": op, "tokens": _spread(rng, 1, 8192), "choices": rng.randint(1, min(8, experts)), "experts": experts}
        if op == "experts":
            case.update(n=_spread(rng, 64, 4096, 8), k=_spread(rng, 64, 4096, 16), out=kind)
            entries = case["tokens"] * case["choices"]
            if entries * case["n"] * case["k"] <= 32768 * 4096 * 2048 and experts * case["n"] * case["k"] <= 2 ** 29:
                return case
            continue
        case.update(block=rng.choice([1, 8, 16, 64, 128]), input=kind, train=rng.random() < 0.6, rows=0,
                    dropped=rng.choice([0.0, 0.0, 0.3, 0.9]))
        case["width"] = _spread(rng, 64, 8192, 16)
        if op == "dispatch":
            case["form"] = rng.choice(["rows", "fp8"])
            if case["form"] == "fp8":
                case["train"] = False
        if rng.random() < 0.25:          # a buffer that may be too small for all entries
            case["rows"] = _ceil(max(1, int(_rows(case) * rng.uniform(0.3, 0.9))), case["block"]) * case["block"]
        if _rows(case) * case["width"] <= 32768 * 4096:
            return case


# ---------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------

def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)


def _ids(case: dict, g) -> torch.Tensor:
    """Distinct experts for each token, drawn from a skewed distribution; some entries dropped."""
    load = torch.randn(case["experts"], generator=g, device="cuda")
    noise = -torch.empty(case["tokens"], case["experts"], device="cuda").exponential_(generator=g).log()
    ids = (load + noise).topk(case["choices"], dim=-1).indices.to(torch.int32)
    if case.get("dropped"):
        away = torch.rand(ids.shape, generator=g, device="cuda") < case["dropped"]
        ids = torch.where(away, torch.full_like(ids, -1), ids)
    return ids


def _fp8_values(shape, g) -> torch.Tensor:
    """8-bit values as a quantised bell curve has them: the largest of a block near 448."""
    q = torch.empty(shape, dtype=FP8, device="cuda")
    flat = q.view(-1, shape[-1])
    step = max(1, (1 << 26) // shape[-1])
    for i in range(0, flat.shape[0], step):
        part = flat[i:i + step]
        part.copy_((torch.randn(part.shape, generator=g, device="cuda") * 140.0).clamp(-FP8_MAX, FP8_MAX))
    return q


def _scales(shape, g, unit: float) -> torch.Tensor:
    """Scales of neighbouring blocks differ by a factor of a few."""
    return torch.exp2(torch.randn(shape, generator=g, device="cuda")) * unit


def _values(shape, g, dtype) -> torch.Tensor:
    """Activations: a bell curve with a few wide columns."""
    wide = 1.0 + 20.0 * (torch.rand(shape[-1], generator=g, device="cuda") < 0.01)
    return (torch.randn(shape, generator=g, device="cuda") * wide).to(dtype)


def _inputs(case: dict, seed: int) -> dict:
    g = _generator(seed)
    op = case["op"]
    if op == "gemm":
        m, n, kb = case["m"], case["n"], _ceil(case["k"], BLOCK)
        return {"a": _fp8_values((m, case["k"]), g), "sa": _scales((m, kb), g, 1.0 / 140.0),
                "b": _fp8_values((n, case["k"]), g),
                "sb": _scales((_ceil(n, BLOCK), kb), g, 1.0 / 140.0 / math.sqrt(case["k"]))}
    if op == "experts":
        n, k, experts, kb = case["n"], case["k"], case["experts"], _ceil(case["k"], BLOCK)
        rows = case["tokens"] * case["choices"]
        counts = torch.zeros(experts, dtype=torch.int32, device="cuda")
        ids = _ids(case, g).reshape(-1)
        counts.scatter_add_(0, ids.long(), torch.ones_like(ids))
        offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0, dtype=torch.int32)])
        return {"a": _fp8_values((rows, k), g), "sa": _scales((rows, kb), g, 1.0 / 140.0),
                "b": _fp8_values((experts * n, k), g),
                "sb": _scales((experts * _ceil(n, BLOCK), kb), g, 1.0 / 140.0 / math.sqrt(k)), "offsets": offsets}
    dtype = DTYPES[case["input"]]
    if op == "quantize":
        return {"x": _values((case["m"], case["k"]), g, dtype)}
    ids = _ids(case, g)
    if op == "dispatch":
        s = {"ids": ids, "x": _values((case["tokens"], case["width"]), g, dtype)}
        if case["train"]:
            s["grad"] = _values((_rows(case), case["width"]), g, dtype)
        return s
    row_of, entry_of, _ = _plain_route(ids, case["experts"], case["block"], _rows(case))
    s = {"y": _values((_rows(case), case["width"]), g, dtype), "row_of": row_of, "entry_of": entry_of,
         "weights": torch.softmax(torch.randn(ids.shape, generator=g, device="cuda"), dim=-1)}
    if case["train"]:
        s["grad"] = _values((case["tokens"], case["width"]), g, dtype)
    return s


@functools.lru_cache(maxsize=None)
def _kernels(*key):
    """The kernel objects that a program builds once for its sizes."""
    from pyptx_b200.examples.blackwell import fp8_gemm, moe
    from pyptx_b200.types import bf16, f32
    types = {"bf16": bf16, "f32": f32}
    op, *sizes = key
    if op == "gemm":
        m, n, k, out = sizes
        return (fp8_gemm.build_fp8_gemm(m, n, k, out_dtype=types[out]),)
    if op == "experts":
        rows, experts, n, k, out = sizes
        return (fp8_gemm.build_fp8_grouped_gemm_varlen(experts, rows, n, k, out_dtype=types[out]),)
    if op == "quantize":
        m, k, block_rows, kind = sizes
        return (fp8_gemm.build_fp8_quantize(m, k, block_rows=block_rows, in_dtype=types[kind]),)
    if op == "dispatch":
        tokens, choices, experts, width, block, rows, form, kind, train = sizes
        route = moe.build_moe_route(tokens, choices, experts, block=block, rows=rows)
        if form == "fp8":
            return route, moe.build_moe_dispatch_fp8(tokens, choices, rows, width, in_dtype=types[kind]), None
        back = moe.build_moe_dispatch_bwd(tokens, choices, rows, width, dtype=types[kind]) if train else None
        return route, moe.build_moe_dispatch(tokens, choices, rows, width, dtype=types[kind]), back
    tokens, choices, width, rows, kind, train = sizes
    back = moe.build_moe_combine_bwd(tokens, choices, rows, width, dtype=types[kind]) if train else None
    return moe.build_moe_combine(tokens, choices, rows, width, dtype=types[kind]), back


def prepare(case: dict, seed: int) -> dict:
    state = _inputs(case, seed)
    state["case"] = case
    if own:
        op = case["op"]
        if op == "gemm":
            state["kernels"] = _kernels(op, case["m"], case["n"], case["k"], case["out"])
        elif op == "experts":
            state["kernels"] = _kernels(op, case["tokens"] * case["choices"], case["experts"], case["n"], case["k"],
                                        case["out"])
        elif op == "quantize":
            state["kernels"] = _kernels(op, case["m"], case["k"], case["block_rows"], case["input"])
        elif op == "dispatch":
            state["kernels"] = _kernels(op, case["tokens"], case["choices"], case["experts"], case["width"],
                                        case["block"], _rows(case), case["form"], case["input"], case["train"])
        else:
            state["kernels"] = _kernels(op, case["tokens"], case["choices"], case["width"], _rows(case), case["input"],
                                        case["train"])
    return state


# ---------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------

def run(state: dict):
    op = state["case"]["op"]
    if own:
        return _run_own(op, state)
    return _run_plain(op, state)


def _run_own(op: str, s: dict):
    k = s["kernels"]
    if op == "gemm":
        return k[0](s["a"], s["sa"], s["b"], s["sb"])
    if op == "experts":
        return k[0](s["a"], s["sa"], s["b"], s["sb"], s["offsets"])
    if op == "quantize":
        return k[0](s["x"])
    if op == "dispatch":
        route, dispatch, back = k
        row_of, entry_of, offsets = route(s["ids"])
        out = [row_of, entry_of, offsets]
        if s["case"]["form"] == "fp8":
            out += list(dispatch(s["x"], row_of, entry_of))
        else:
            out.append(dispatch(s["x"], row_of, entry_of))
        if back is not None:
            out.append(back(row_of, s["grad"]))
        return out
    combine, back = k
    out = [combine(s["y"], s["weights"], s["row_of"])]
    if back is not None:
        out += list(back(s["y"], s["weights"], s["row_of"], s["entry_of"], s["grad"]))
    return out


def _dequantized(q, scale, block_rows: int) -> torch.Tensor:
    rows, cols = q.shape
    x = scale.repeat_interleave(BLOCK, dim=1)[:, :cols]
    if block_rows > 1:
        x = x.repeat_interleave(block_rows, dim=0)[:rows]
    return q.float() * x


def _plain_quantize(x, block_rows: int):
    rows, cols = x.shape
    rb, cb = _ceil(rows, block_rows), _ceil(cols, BLOCK)
    v = torch.nn.functional.pad(x.float(), (0, cb * BLOCK - cols, 0, rb * block_rows - rows))
    v = v.view(rb, block_rows, cb, BLOCK)
    amax = v.abs().amax(dim=(1, 3), keepdim=True)
    scale = (amax / torch.full_like(amax, FP8_MAX)).clamp_min(SCALE_MIN)
    q = (v * torch.reciprocal(scale)).clamp(-FP8_MAX, FP8_MAX).to(FP8)
    return q.view(rb * block_rows, cb * BLOCK)[:rows, :cols].contiguous(), scale.view(rb, cb)


def _plain_route(ids, experts: int, block: int, rows: int):
    flat = ids.reshape(-1).long()
    n = flat.numel()
    key = torch.where((flat >= 0) & (flat < experts), flat, torch.full_like(flat, experts))
    counts = torch.zeros(experts + 1, dtype=torch.int64, device=flat.device)
    counts.scatter_add_(0, key, torch.ones_like(key))
    start = counts.cumsum(0) - counts
    padded = (counts[:experts] + block - 1) // block * block
    ends = padded.cumsum(0)
    base = torch.cat([ends - padded, ends.new_full((1,), rows)])
    order = torch.argsort(key, stable=True)
    sorted_key = key[order]
    row = base[sorted_key] + torch.arange(n, device=flat.device) - start[sorted_key]
    kept = (sorted_key < experts) & (row < rows)
    row_of = torch.empty(n, dtype=torch.int32, device=flat.device)
    row_of[order] = torch.where(kept, row, torch.full_like(row, -1)).to(torch.int32)
    entry_of = torch.full((rows + 1,), -1, dtype=torch.int32, device=flat.device)
    entry_of[torch.where(kept, row, torch.full_like(row, rows))] = order.to(torch.int32)
    offsets = torch.cat([ends.new_zeros(1), ends]).clamp_max(rows).to(torch.int32)
    return row_of.view(ids.shape), entry_of[:rows].contiguous(), offsets


def _plain_gather(x, entry_of, choices: int):
    """x of each row's token in 32 bits, zeros in rows that no entry owns."""
    owned = entry_of >= 0
    token = torch.where(owned, entry_of, torch.zeros_like(entry_of)).long() // choices
    return torch.where(owned[:, None], x[token].float(), x.new_zeros((), dtype=torch.float32))


def _plain_back(rows, row_of, weights=None):
    """For each token the sum over its choices of (weight times) the choice's row."""
    total = torch.zeros(row_of.shape[0], rows.shape[1], dtype=torch.float32, device=rows.device)
    for j in range(row_of.shape[1]):
        r = row_of[:, j].long()
        part = rows[r.clamp_min(0)].float()
        if weights is not None:
            part = part * weights[:, j:j + 1]
        total += torch.where((r >= 0)[:, None], part, torch.zeros_like(part))
    return total


def _run_plain(op: str, s: dict):
    case = s["case"]
    if op == "gemm":
        return (_dequantized(s["a"], s["sa"], 1) @ _dequantized(s["b"], s["sb"], BLOCK).T).to(DTYPES[case["out"]])
    if op == "experts":
        n, nb = case["n"], _ceil(case["n"], BLOCK)
        out = torch.empty(s["a"].shape[0], n, dtype=DTYPES[case["out"]], device="cuda")
        ends = s["offsets"].tolist()
        for e in range(case["experts"]):
            lo, hi = ends[e], ends[e + 1]
            if lo < hi:
                w = _dequantized(s["b"][e * n:(e + 1) * n], s["sb"][e * nb:(e + 1) * nb], BLOCK)
                out[lo:hi] = (_dequantized(s["a"][lo:hi], s["sa"][lo:hi], 1) @ w.T).to(out.dtype)
        return out
    if op == "quantize":
        return _plain_quantize(s["x"], case["block_rows"])
    if op == "dispatch":
        row_of, entry_of, offsets = _plain_route(s["ids"], case["experts"], case["block"], _rows(case))
        rows = _plain_gather(s["x"], entry_of, case["choices"])
        out = [row_of, entry_of, offsets]
        if case["form"] == "fp8":
            q, scale = _plain_quantize(rows, 1)
            out += [q, torch.where((entry_of >= 0)[:, None], scale, torch.zeros_like(scale))]
        else:
            out.append(rows.to(s["x"].dtype))
        if case["train"]:
            out.append(_plain_back(s["grad"], row_of).to(s["grad"].dtype))
        return out
    out = [_plain_back(s["y"], s["row_of"], s["weights"]).to(s["y"].dtype)]
    if case["train"]:
        entry, y, grad = s["entry_of"], s["y"].float(), s["grad"]
        owned = entry >= 0
        at = torch.where(owned, entry, torch.zeros_like(entry)).long()
        dout = grad[at // case["choices"]].float()
        dy = torch.where(owned[:, None], dout * s["weights"].reshape(-1)[at][:, None], torch.zeros_like(dout))
        dot = (y * dout).sum(dim=-1)
        dw = torch.zeros(s["weights"].numel() + 1, dtype=torch.float32, device="cuda")
        dw[torch.where(owned, at, torch.full_like(at, dw.numel() - 1))] = dot
        out += [dy.to(s["y"].dtype), dw[:-1].view(s["weights"].shape).contiguous()]
    return out


# ---------------------------------------------------------------------------------------------
# Work and exact values
# ---------------------------------------------------------------------------------------------

def work(case: dict) -> dict:
    op = case["op"]
    if op in ("gemm", "experts"):
        n, k, kb = case["n"], case["k"], _ceil(case["k"], BLOCK)
        experts = case.get("experts", 1)
        m = case["m"] if op == "gemm" else case["tokens"] * case["choices"]
        used = min(experts, m)           # experts without rows need not be read
        return {"bytes": m * k + 4 * m * kb + used * (n * k + 4 * kb * _ceil(n, BLOCK)) + m * n * WIDTH[case["out"]],
                "flops": 2 * m * n * k}
    size = WIDTH[case["input"]]
    if op == "quantize":
        m, k = case["m"], case["k"]
        return {"bytes": m * k * (size + 1) + 4 * _ceil(m, case["block_rows"]) * _ceil(k, BLOCK), "flops": 3 * m * k}
    entries, rows, width, tokens = case["tokens"] * case["choices"], _rows(case), case["width"], case["tokens"]
    held = min(rows, int(entries * (1.0 - case["dropped"])))
    if op == "dispatch":
        out = rows * (width + 4 * _ceil(width, BLOCK)) if case["form"] == "fp8" else rows * width * size
        total = 4 * entries + 4 * entries + 4 * rows + 4 * (case["experts"] + 1) + tokens * width * size + out
        flops = 3 * rows * width if case["form"] == "fp8" else 0
        if case["train"]:
            total += (held + tokens) * width * size
            flops += held * width
        return {"bytes": total, "flops": flops}
    total, flops = (held + tokens) * width * size + 8 * entries, 2 * held * width
    if case["train"]:
        total += (held + tokens + rows) * width * size + 12 * entries + 4 * rows
        flops += 3 * held * width
    return {"bytes": total, "flops": flops}


def _round_f32(x: torch.Tensor) -> torch.Tensor:
    return x.to(torch.float32).to(torch.float64)


def _e4m3(x: torch.Tensor) -> torch.Tensor:
    """The nearest value with four significant bits (ties to even), steps of 2^-9 at least, 448 at most."""
    _, e = torch.frexp(x)
    step = torch.exp2((e - 4).clamp_min(-9).to(torch.float64))
    return (torch.round(x / step) * step).clamp(-FP8_MAX, FP8_MAX)


def _exact_quantize(x: torch.Tensor, block_rows: int):
    """Scale, reciprocal and product are defined as f32 numbers: each is formed in 64 bits and rounded once."""
    q = torch.empty(x.shape, dtype=torch.float32, device=x.device)
    scales = torch.empty(_ceil(x.shape[0], block_rows), _ceil(x.shape[1], BLOCK), dtype=torch.float64, device=x.device)
    for c in range(scales.shape[1]):
        part = x[:, c * BLOCK:(c + 1) * BLOCK].double()
        top = part.abs().amax(dim=1)
        top = torch.nn.functional.pad(top, (0, scales.shape[0] * block_rows - top.numel()))
        top = top.view(-1, block_rows).amax(dim=1)
        scale = torch.maximum(_round_f32(top / FP8_MAX), torch.full_like(top, SCALE_MIN))
        inverse = _round_f32(1.0 / scale).repeat_interleave(block_rows)[:x.shape[0], None]
        q[:, c * BLOCK:(c + 1) * BLOCK] = _e4m3(_round_f32(part * inverse)).float()
        scales[:, c] = scale
    return q, scales


def _exact_route(case: dict, ids: torch.Tensor):
    rows, block, choices = _rows(case), case["block"], case["choices"]
    lists = [[] for _ in range(case["experts"])]
    flat = ids.reshape(-1).tolist()
    for i, e in enumerate(flat):
        if 0 <= e < case["experts"]:
            lists[e].append(i)
    row_of, entry_of, offsets, at = [-1] * len(flat), [-1] * rows, [0], 0
    for entries in lists:
        for r, i in enumerate(entries, at):
            if r < rows:
                row_of[i], entry_of[r] = r, i
        at += _ceil(len(entries), block) * block
        offsets.append(min(at, rows))
    whole = [torch.tensor(v, dtype=torch.int32, device=ids.device) for v in (row_of, entry_of, offsets)]
    return whole[0].view(-1, choices), whole[1], whole[2]


def exact(case: dict, seed: int):
    s = _inputs(case, seed)
    op = case["op"]
    if op in ("gemm", "experts"):
        n, nb, k = case["n"], _ceil(case["n"], BLOCK), case["k"]
        ends = [0, s["a"].shape[0]] if op == "gemm" else s["offsets"].tolist()
        out = torch.zeros(s["a"].shape[0], n, dtype=torch.float64, device="cuda")
        for e in range(len(ends) - 1):
            lo, hi = ends[e], ends[e + 1]
            for b in range(_ceil(k, BLOCK) if lo < hi else 0):
                cols = slice(b * BLOCK, (b + 1) * BLOCK)
                left = s["a"][lo:hi, cols].double() * s["sa"][lo:hi, b:b + 1].double()
                weight = s["b"][e * n:(e + 1) * n, cols].double()
                sb = s["sb"][e * nb:(e + 1) * nb, b].double().repeat_interleave(BLOCK)[:n]
                out[lo:hi].addmm_(left, (weight * sb[:, None]).T)
        return out
    if op == "quantize":
        return _exact_quantize(s["x"], case["block_rows"])
    choices, rows = case["choices"], _rows(case)
    if op == "dispatch":
        row_of, entry_of, offsets = _exact_route(case, s["ids"])
        owned = torch.nonzero(entry_of >= 0).view(-1)
        token = torch.div(entry_of[owned].long(), choices, rounding_mode="floor")
        out = [row_of, entry_of, offsets]
        if case["form"] == "fp8":
            q1, s1 = _exact_quantize(s["x"], 1)
            q = torch.zeros(rows, case["width"], dtype=torch.float32, device="cuda")
            scale = torch.zeros(rows, s1.shape[1], dtype=torch.float64, device="cuda")
            q[owned], scale[owned] = q1[token], s1[token]
            out += [q, scale]
        else:
            xs = torch.zeros(rows, case["width"], dtype=torch.float64, device="cuda")
            xs[owned] = s["x"].double()[token]
            out.append(xs)
        if case["train"]:
            dx = torch.zeros(case["tokens"], case["width"], dtype=torch.float64, device="cuda")
            out.append(dx.index_add_(0, token, s["grad"][owned].double()))
        return out
    owned = torch.nonzero(s["entry_of"] >= 0).view(-1)
    entry = s["entry_of"][owned].long()
    token = torch.div(entry, choices, rounding_mode="floor")
    weight = s["weights"].reshape(-1)[entry].double()
    y = s["y"][owned].double()
    out = [torch.zeros(case["tokens"], case["width"], dtype=torch.float64, device="cuda")
           .index_add_(0, token, y * weight[:, None])]
    if case["train"]:
        dout = s["grad"].double()[token]
        dy = torch.zeros(rows, case["width"], dtype=torch.float64, device="cuda")
        dy[owned] = dout * weight[:, None]
        dw = torch.zeros(s["weights"].numel(), dtype=torch.float64, device="cuda")
        dw[entry] = (y * dout).sum(dim=-1)
        out += [dy, dw.view(s["weights"].shape)]
    return out
