"""The operators of a dense block in 8-bit integers: their calls, their plain forms and their values in 64 bits.

A model runner brings a token's (or a prompt's) hidden state through a residual addition and a root-mean-square norm
into 8-bit rows, multiplies them with 8-bit weights that carry one scale a channel, and feeds the gated feed-forward
block of a dense layer from the same rows.  The kinds of case:

norm     hidden' = hidden + delta, the norm of hidden', and its output: rows in the hidden state's type, Q8_K blocks (what
         the K-quant products read) or int8 rows with one scale each (what the int8 product reads)
product  int8 rows x int8 channels with a scale for each row and channel, optionally added to a residual
gated    silu(gate) * up of two such products
block    norm, gated product, quantization of its rows, product into the residual: one dense feed-forward block
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5
LEAST = 2.0 ** -126   # a scale below this is zero


def listed():
    return [
        # One decoded token in front of its projections: all latency.
        {"name": "norm_token_i8", "kind": "norm", "tokens": 1, "n": 4096, "type": "f32", "residual": True, "out": "i8"},
        # A decode batch in front of a mixture-of-experts block: the router takes the rows, the experts the Q8_K blocks.
        {"name": "norm_batch_64_q8_k", "kind": "norm", "tokens": 64, "n": 4096, "type": "f32", "residual": True,
         "out": "q8_k"},
        # A ragged prompt without a residual (the embedding's rows), norm alone, of an odd width.
        {"name": "norm_prompt_333_odd", "kind": "norm", "tokens": 333, "n": 7167, "type": "f32", "residual": False,
         "out": "rows"},
        # A long prompt in 16 bits: bandwidth.
        {"name": "norm_prompt_6007_i8", "kind": "norm", "tokens": 6007, "n": 4096, "type": "bf16", "residual": True,
         "out": "i8"},
        # One token through a wide projection: the weights stream once.
        {"name": "product_token", "kind": "product", "tokens": 1, "rows": 12288, "k": 4096, "type": "f32",
         "residual": False},
        # A ragged decode batch through a square output projection, added to the residual.
        {"name": "product_batch_37", "kind": "product", "tokens": 37, "rows": 4096, "k": 4096, "type": "bf16",
         "residual": True},
        # A prefill chunk of the ordinary size.
        {"name": "product_prefill_512", "kind": "product", "tokens": 512, "rows": 12288, "k": 4096, "type": "f32",
         "residual": False},
        # The largest chunk: several prompts together.
        {"name": "product_prefill_4096", "kind": "product", "tokens": 4096, "rows": 12288, "k": 4096, "type": "bf16",
         "residual": False},
        # The dense layer's gate and up projections for one token, and for a ragged prompt chunk.
        {"name": "gated_token", "kind": "gated", "tokens": 1, "rows": 13312, "k": 4096, "type": "f32"},
        {"name": "gated_prefill_1500", "kind": "gated", "tokens": 1500, "rows": 13312, "k": 4096, "type": "bf16"},
        # The dense layer's whole feed-forward block: a decode batch, and a prefill chunk.
        {"name": "block_batch_16", "kind": "block", "tokens": 16, "n": 4096, "rows": 13312, "type": "bf16"},
        {"name": "block_prefill_1024", "kind": "block", "tokens": 1024, "n": 4096, "rows": 13312, "type": "bf16"},
    ]


MOST = 4096 * 12288 * 4096   # multiplications of the largest product


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A row length: mostly multiples of 16 as models have them, at times any number."""
    k = _log(rng, lo, hi)
    return k if rng.random() < 0.2 else max(16, k // 16 * 16)


def draw(rng):
    kind = rng.choice(("norm", "norm", "product", "product", "product", "gated", "gated", "block"))
    ty = rng.choice(("f32", "f16", "bf16"))
    if kind == "norm":
        out = rng.choice(("rows", "q8_k", "i8", "i8"))
        n = 256 * rng.randint(1, 52) if out == "q8_k" else _width(rng, 64, 13312)
        return {"kind": kind, "tokens": _log(rng, 1, min(8192, 24_000_000 // n)), "n": n, "type": ty,
                "residual": rng.random() < 0.7, "out": out}
    k = _width(rng, 256, 13312)
    if kind == "block":
        n = 16 * rng.randint(32, 256)
        rows = _width(rng, 512, 13312)
        return {"kind": kind, "tokens": _log(rng, 1, min(2048, MOST // (3 * n * rows))), "n": n, "rows": rows,
                "type": rng.choice(("f16", "bf16"))}
    rows = _log(rng, 64, 14000)
    parts = 2 if kind == "gated" else 1
    case = {"kind": kind, "tokens": _log(rng, 1, min(4096, MOST // (parts * rows * k))), "rows": rows, "k": k, "type": ty}
    if kind == "product":
        case["residual"] = rng.random() < 0.5
    return case


# ------------------------------------------------------------------ inputs


def _hidden(gen, tokens, n, ty):
    """Rows of a residual stream: channels of unequal size, one in 512 of them large."""
    size = torch.exp(0.4 * torch.randn(n, device=DEVICE, generator=gen))
    size[torch.randint(0, n, (max(1, n // 512),), device=DEVICE, generator=gen)] *= 20.0
    return (torch.randn(tokens, n, device=DEVICE, generator=gen) * size).to(TYPES[ty])


def _norm_inputs(gen, tokens, n, ty, residual):
    return {"hidden": _hidden(gen, tokens, n, ty),
            "delta": (0.3 * torch.randn(tokens, n, device=DEVICE, generator=gen)).to(TYPES[ty]) if residual else None,
            "weight": 1.0 + 0.2 * torch.randn(n, device=DEVICE, generator=gen)}


def _rows(gen, tokens, k):
    """int8 rows whose largest value is 127, with their scales."""
    x = torch.randn(tokens, k, device=DEVICE, generator=gen)
    top = x.abs().amax(1, keepdim=True)
    scale = 0.5 + torch.rand(tokens, device=DEVICE, generator=gen)
    return torch.round(x * (127.0 / top)).to(torch.int8), scale * (4.0 / 127.0)


def _channels(gen, rows, k):
    """int8 weights of unit size after the product, with their scales."""
    w = torch.empty(rows, k, dtype=torch.int8, device=DEVICE)
    for at in range(0, rows, 2048):
        part = torch.randn(min(2048, rows - at), k, device=DEVICE, generator=gen)
        w[at:at + 2048] = torch.round(part * 30.0).clamp_(-127, 127).to(torch.int8)
    return w, (0.5 + torch.rand(rows, device=DEVICE, generator=gen)) / (30.0 * math.sqrt(k))


def _inputs(case, seed):
    """Every raw input of a case, made from the seed alone."""
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    kind, tokens = case["kind"], case["tokens"]
    if kind == "norm":
        return _norm_inputs(gen, tokens, case["n"], case["type"], case["residual"])
    if kind == "block":
        s = _norm_inputs(gen, tokens, case["n"], case["type"], True)
        for name, r, k in (("gate", case["rows"], case["n"]), ("up", case["rows"], case["n"]),
                           ("down", case["n"], case["rows"])):
            s[name] = _channels(gen, r, k)
        return s
    s = {"x": _rows(gen, tokens, case["k"])}
    if kind == "gated":
        s["gate"], s["up"] = _channels(gen, case["rows"], case["k"]), _channels(gen, case["rows"], case["k"])
        return s
    s["w"] = _channels(gen, case["rows"], case["k"])
    if case["residual"]:
        s["residual"] = (2.0 * torch.randn(tokens, case["rows"], device=DEVICE, generator=gen)).to(TYPES[case["type"]])
    return s


_backend = None


def _be():
    """The framework's backend, opened once as a program does."""
    global _backend
    if _backend is None:
        package = str(Path(__file__).resolve().parent.parent / "lightbridge-engine_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        import lbhip
        _backend = lbhip.HipBackend(0)
    return _backend


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:   # the weights as the framework keeps them, and the workspace of the largest call
        be, tokens = _be(), case["tokens"]
        s["be"] = be
        need = [16]
        if "gate" in s:
            s["pair"] = be.upload_i8_gated(*s["gate"], *s["up"])
            need.append(be.gemm_i8_workspace_bytes(s["pair"], tokens))
        for name in ("w", "down"):
            if name in s:
                s["m"] = be.upload_i8(*s[name])
                need.append(be.gemm_i8_workspace_bytes(s["m"], tokens))
        s["workspace"] = torch.zeros(max(need), dtype=torch.uint8, device=DEVICE)
    return s


# ------------------------------------------------------------------ plain forms


def _values(v):
    """int8 rows of 64-bit values and their scales in 32 bits: (q, scale), the rounding done in 64 bits."""
    scale = (v.abs().amax(1, keepdim=True) / 127.0).float()
    scale = torch.where(scale < LEAST, torch.zeros_like(scale), scale)
    q = torch.round(v / torch.where(scale > 0, scale, torch.ones_like(scale)).double())
    return torch.where(scale > 0, q.clamp(-127, 127), torch.zeros_like(q)), scale


def _plain_norm(s):
    """(hidden', the normed rows in 64 bits)"""
    h = s["hidden"]
    if s["delta"] is not None:
        h = (h.float() + s["delta"].float()).to(h.dtype)
    v = h.double()
    return h, v * torch.rsqrt((v * v).mean(1, keepdim=True) + EPS) * s["weight"].double()


def _plain_q8_k(x):
    """Q8_K blocks of 256 of 32-bit rows: the values they stand for, and the sums of 16 quants each."""
    b = x.reshape(x.shape[0], -1, 256)
    at = b.abs().argmax(2, keepdim=True)
    top = torch.gather(b, 2, at)
    some = top != 0
    inverse = torch.where(some, torch.full_like(top, -127.0) / torch.where(some, top, torch.ones_like(top)),
                          torch.zeros_like(top))   # a true quotient: a number over a tensor is reciprocal times number
    q = torch.round(inverse * b).clamp(max=127.0)
    d = torch.where(some, 1.0 / torch.where(some, inverse, torch.ones_like(inverse)), torch.zeros_like(inverse))
    return q * d, q.reshape(*q.shape[:2], 16, 16).sum(3).to(torch.int16)


def _plain_product(x, w):
    (q, xs), (m, ws) = x, w
    return (q.float() @ m.float().t()) * xs.reshape(-1, 1) * ws


def _plain_gated(x, gate, up):
    g = _plain_product(x, gate)
    return g / (1.0 + torch.exp(-g)) * _plain_product(x, up)


def _plain(s):
    case, ty = s["case"], TYPES[s["case"]["type"]]
    kind = case["kind"]
    if kind == "product":
        y = _plain_product(s["x"], s["w"])
        return (y + s["residual"].float() if case["residual"] else y).to(ty)
    if kind == "gated":
        return _plain_gated(s["x"], s["gate"], s["up"]).to(ty)
    h, v = _plain_norm(s)
    if kind == "block":
        q, scale = _values(v)
        q, scale = _values(_plain_gated((q, scale), s["gate"], s["up"]).double())
        return {"hidden": h, "out": (h.float() + _plain_product((q, scale), s["down"])).to(ty)}
    got = {"hidden": h} if case["residual"] else {}
    if case["out"] == "i8":
        q, scale = _values(v)
        return {**got, "values": q.float() * scale}
    if case["out"] == "q8_k":
        x = v.float()
        values, sums = _plain_q8_k(x)
        return {**got, "rows": x, "values": values, "sums": sums}
    return {**got, "rows": v.to(ty)}


# ------------------------------------------------------------------ the framework's calls


def _own_norm_i8(s):
    h = s["hidden"]
    after = torch.empty_like(h) if s["delta"] is not None else None
    q = torch.empty(h.shape, dtype=torch.int8, device=DEVICE)
    scale = torch.empty(h.shape[0], device=DEVICE)
    s["be"].rms_norm_i8_rows(h, s["weight"], EPS, q, scale, delta=s["delta"], hidden_out=after)
    return after, q, scale


def _own(s):
    case, be, ty = s["case"], s["be"], TYPES[s["case"]["type"]]
    kind, tokens = case["kind"], case["tokens"]
    if kind == "product":
        y = torch.empty(tokens, case["rows"], dtype=ty, device=DEVICE)
        be.gemm_i8(s["m"], *s["x"], y, s["workspace"], residual=s.get("residual"))
        return y
    if kind == "gated":
        y = torch.empty(tokens, case["rows"], dtype=ty, device=DEVICE)
        be.gemm_i8_swiglu(s["pair"], *s["x"], y, s["workspace"])
        return y
    if kind == "block":
        after, q, scale = _own_norm_i8(s)
        y = torch.empty(tokens, case["rows"], device=DEVICE)   # 32 bits until its own quantization
        be.gemm_i8_swiglu(s["pair"], q, scale, y, s["workspace"])
        q, scale = torch.empty(y.shape, dtype=torch.int8, device=DEVICE), torch.empty_like(scale)
        be.quantize_i8_rows(y, q, scale)
        out = torch.empty_like(after)
        be.gemm_i8(s["m"], q, scale, out, s["workspace"], residual=after)
        return {"hidden": after, "out": out}
    if case["out"] == "i8":
        after, q, scale = _own_norm_i8(s)
        got = {"values": torch.mul(q, scale.unsqueeze(1))}
    else:
        h = s["hidden"]
        after = torch.empty_like(h) if case["residual"] else None
        if case["out"] == "q8_k":
            blocks = torch.empty(tokens, case["n"] // 256, 292, dtype=torch.uint8, device=DEVICE)
            rows = torch.empty(h.shape, device=DEVICE)
            be.rms_norm_q8_k_rows(h, s["weight"], EPS, blocks, y=rows, delta=s["delta"], hidden_out=after)
            got = {"rows": rows, "sums": blocks[:, :, 260:].view(torch.int16),
                   "values": torch.mul(blocks[:, :, 4:260].view(torch.int8), blocks[:, :, :4].view(torch.float32))}
        else:
            rows = torch.empty_like(h)
            be.rms_norm_rows(h, s["weight"], EPS, rows, delta=s["delta"], hidden_out=after)
            got = {"rows": rows}
    return {**got, "hidden": after} if case["residual"] else got


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    kind, t = case["kind"], case["tokens"]
    e = SIZE[case["type"]]

    def norm(n, out):
        return t * n * (e * (3 if case.get("residual", True) else 1) + out) + 4 * n

    if kind == "norm":
        n = case["n"]
        out = {"rows": e, "i8": 1 + 4 / n, "q8_k": 4 + 292 / 256}[case["out"]]
        return {"bytes": norm(n, out), "flops": 6 * t * n}
    rows = case["rows"]
    if kind == "block":
        n = case["n"]
        return {"bytes": 3 * rows * n + 8 * rows + 4 * n + norm(n, 1) + t * (n + 2 * rows + 2 * e * rows + 2 * e * n),
                "flops": 6 * t * rows * n}
    k, parts = case["k"], 2 if kind == "gated" else 1
    return {"bytes": parts * rows * (k + 4) + t * (k + 4) + t * rows * e * (2 if case.get("residual") else 1),
            "flops": 2 * parts * t * rows * k}


# ------------------------------------------------------------------ the results in 64 bits


def _exact_product(q, scale, w, w_scale):
    """[tokens, rows], in pieces of rows that keep the 64-bit copies small."""
    a = q.double()
    parts = [torch.mm(a, w[at:at + 4096].double().t().contiguous()) for at in range(0, w.shape[0], 4096)]
    return torch.cat(parts, 1) * w_scale.double()[None, :] * scale.double()[:, None]


def _exact_silu(g):
    return g * torch.sigmoid(g)


def _exact_norm(raw, ty):
    h = raw["hidden"]
    if raw["delta"] is not None:   # the stored state is the sum in 32 bits, in the state's type
        h = torch.add(h.float(), raw["delta"].float()).to(TYPES[ty])
    d = h.double()
    root = torch.sqrt(torch.sum(d.square(), dim=1) / d.shape[1] + EPS)
    return h, d * raw["weight"].double()[None, :] / root[:, None]


def _exact_i8(v):
    """Nearest integers of v / scale, ties to even, the scale being the 32-bit value that the rows carry."""
    top = torch.maximum(v.amax(dim=1), -v.amin(dim=1))
    scale = (top / 127).to(torch.float32).double()
    live = scale >= LEAST
    per = torch.where(live, 1 / torch.where(live, scale, 1.0), 0.0)
    ratio = v * per[:, None]
    low = torch.floor(ratio)
    over = ratio - low
    up = (over > 0.5) | ((over == 0.5) & (torch.remainder(low, 2) == 1))
    return torch.clamp(low + up, -127, 127), torch.where(live, scale, 0.0)


def exact(case, seed):
    raw, kind = _inputs(case, seed), case["kind"]
    if kind == "product":
        y = _exact_product(*raw["x"], *raw["w"])
        return y + raw["residual"].double() if case["residual"] else y
    if kind == "gated":
        return _exact_silu(_exact_product(*raw["x"], *raw["gate"])) * _exact_product(*raw["x"], *raw["up"])
    h, v = _exact_norm(raw, case["type"])
    if kind == "block":
        q, scale = _exact_i8(v)
        y = _exact_silu(_exact_product(q, scale, *raw["gate"])) * _exact_product(q, scale, *raw["up"])
        q, scale = _exact_i8(y)
        return {"hidden": h.double(), "out": _exact_product(q, scale, *raw["down"]) + h.double()}
    got = {"hidden": h.double()} if case["residual"] else {}
    if case["out"] == "rows":
        return {**got, "rows": v}
    if case["out"] == "i8":
        q, scale = _exact_i8(v)
        return {**got, "values": q * scale[:, None]}
    # Q8_K's definition is in 32-bit steps (scale, inverse, product), each rounded once: done here block by block with
    # the rounding of a 64-bit result to 32 bits in each place.
    x = v.float()
    b = x.double().reshape(x.shape[0], -1, 256)
    hi, lo = b.max(dim=2), b.min(dim=2)
    first = (hi.values > -lo.values) | ((hi.values == -lo.values) & (hi.indices < lo.indices))
    top = torch.where(first, hi.values, lo.values)
    live = top != 0
    inverse = torch.where(live, -127.0 / torch.where(live, top, 1.0), 0.0).float().double()
    q = torch.minimum(torch.round((b * inverse[:, :, None]).float()).double(), torch.tensor(127.0, device=DEVICE).double())
    d = torch.where(live, 1.0 / torch.where(live, inverse, 1.0), 0.0).float().double()
    return {**got, "rows": v, "values": q * d[:, :, None], "sums": None}
