"""The operators of a mixture-of-experts layer in 8-bit integers: their calls, their plain forms and their values in 64
bits.

A model runner brings a block's output back into the residual stream (normed, gated and scaled where the model says so)
and norms the stream for the next block in the same step, routes the normed rows to experts, sends their int8 rows
through the routed and the shared experts, and has projections with a bias and an activation around them.  The kinds of
case:

norm     h = hidden + scale * act(gate) * norm(block), norm of h: rows in the hidden state's type, or int8 rows with one
         scale each
product  residual + scale * act(int8 rows x int8 channels + bias), or act(gate + bias) * (up + bias) of a gated pair
route    rows x router weights, the selection of the best experts and their coefficients
moe      residual + sum of coefficient * down(silu(gate) * up) over a token's experts, + the shared expert's
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
POST_EPS, EPS = 1e-6, 1e-5
LEAST = 2.0 ** -126   # a scale below this is zero
FLOOR = 2.0 ** -14    # the least sum of a token's sigmoid scores
ACTS = ("none", "relu", "relu2", "silu", "gelu", "gelu_tanh")


def listed():
    return [
        # One decoded token between two blocks of a model with norms on both sides of a block: all latency.
        {"name": "norm_token", "kind": "norm", "tokens": 1, "n": 4096, "type": "f32", "post": True, "gate": "none",
         "out": "i8"},
        # A ragged prompt whose block output has a gate row a token, of an odd width, no norm behind the block.
        {"name": "norm_prompt_333_odd", "kind": "norm", "tokens": 333, "n": 4095, "type": "f16", "post": False,
         "gate": "sigmoid", "out": "rows"},
        # A prefill chunk with everything: bandwidth.
        {"name": "norm_prefill_4096", "kind": "norm", "tokens": 4096, "n": 4096, "type": "bf16", "post": True,
         "gate": "silu", "out": "i8"},
        # One token through a projection with a bias: the weights stream once.
        {"name": "product_token", "kind": "product", "tokens": 1, "rows": 8192, "k": 4096, "type": "f32", "act": "none",
         "gated": False, "residual": True},
        # A ragged decode batch through a gated pair with biases.
        {"name": "gated_batch_37", "kind": "product", "tokens": 37, "rows": 1536, "k": 4096, "type": "bf16",
         "act": "gelu_tanh", "gated": True, "residual": False},
        # A prefill chunk through the first matrix of a block without a gate.
        {"name": "product_prefill_2048", "kind": "product", "tokens": 2048, "rows": 13312, "k": 4096, "type": "bf16",
         "act": "gelu", "gated": False, "residual": False},
        # Routing: one decoded token by softmax, a ragged prompt chunk by biased sigmoid scores.
        {"name": "route_token", "kind": "route", "tokens": 1, "experts": 192, "n": 4096, "top_k": 8, "mode": 0,
         "type": "f32"},
        {"name": "route_prompt_1000", "kind": "route", "tokens": 1000, "experts": 192, "n": 4096, "top_k": 8, "mode": 1,
         "type": "bf16"},
        # The layer's experts: one decoded token, a ragged handful and a batch of requests; the last without a shared
        # expert.  `hot` of a token's experts are the same for all.
        {"name": "moe_token", "kind": "moe", "tokens": 1, "experts": 192, "top_k": 8, "hot": 0, "n": 4096, "ffn": 1536,
         "shared": 4096, "type": "f32"},
        {"name": "moe_tokens_5", "kind": "moe", "tokens": 5, "experts": 192, "top_k": 8, "hot": 1, "n": 4096, "ffn": 1536,
         "shared": 1536, "type": "bf16"},
        {"name": "moe_tokens_16", "kind": "moe", "tokens": 16, "experts": 192, "top_k": 8, "hot": 1, "n": 4096,
         "ffn": 1536, "shared": 4096, "type": "f32"},
        {"name": "moe_tokens_64", "kind": "moe", "tokens": 64, "experts": 192, "top_k": 8, "hot": 2, "n": 4096,
         "ffn": 1536, "shared": 0, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A row length: mostly multiples of 16 as models have them, at times any number."""
    k = _log(rng, lo, hi)
    return k if rng.random() < 0.2 else max(16, k // 16 * 16)


def draw(rng):
    kind = rng.choice(("norm", "norm", "product", "product", "route", "moe", "moe"))
    ty = rng.choice(("f32", "f16", "bf16"))
    if kind == "norm":
        n = _width(rng, 64, 16384)
        return {"kind": kind, "tokens": _log(rng, 1, min(4096, 16_000_000 // n)), "n": n, "type": ty,
                "post": rng.random() < 0.7, "gate": rng.choice(("none", "row", "sigmoid", "silu")),
                "out": rng.choice(("i8", "i8", "rows"))}
    if kind == "product":
        gated = rng.random() < 0.4
        rows, k = _log(rng, 64, 13312), _width(rng, 256, 8192)
        most = 2048 * 13312 * 4096 // ((2 if gated else 1) * rows * k)
        return {"kind": kind, "tokens": _log(rng, 1, min(4096, most)), "rows": rows, "k": k, "type": ty,
                "act": rng.choice(ACTS), "gated": gated, "residual": not gated and rng.random() < 0.5}
    if kind == "route":
        experts = rng.randint(8, 256)
        return {"kind": kind, "tokens": _log(rng, 1, 4096), "experts": experts, "n": 256 * rng.randint(2, 16),
                "top_k": rng.randint(1, min(16, experts)), "mode": rng.randint(0, 1), "type": ty}
    experts, top_k = rng.randint(8, 192), rng.choice((1, 2, 4, 6, 8))
    return {"kind": kind, "tokens": _log(rng, 1, 64), "experts": experts, "top_k": top_k,
            "hot": rng.randint(0, min(2, top_k)), "n": _width(rng, 256, 4096), "ffn": _width(rng, 128, 1536),
            "shared": rng.choice((0, _width(rng, 256, 4096))), "type": ty}


# ------------------------------------------------------------------ inputs


def _rows(gen, tokens, k):
    """int8 rows whose largest value is 127, with their scales."""
    x = torch.randn(tokens, k, device=DEVICE, generator=gen)
    top = x.abs().amax(1, keepdim=True)
    scale = 0.5 + torch.rand(tokens, device=DEVICE, generator=gen)
    return torch.round(x * (127.0 / top)).to(torch.int8), scale * (4.0 / 127.0)


def _channels(gen, *shape):
    """int8 weights [..., rows, k] of unit size after the product, with their scales [..., rows]."""
    w = torch.randn(shape, device=DEVICE, generator=gen).mul_(30.0).round_().clamp_(-127, 127).to(torch.int8)
    return w, (0.5 + torch.rand(shape[:-1], device=DEVICE, generator=gen)) / (30.0 * math.sqrt(shape[-1]))


def _stream(gen, tokens, n, ty):
    """Rows of a residual stream: channels of unequal size, one in 512 of them large."""
    size = torch.exp(0.4 * torch.randn(n, device=DEVICE, generator=gen))
    size[torch.randint(0, n, (max(1, n // 512),), device=DEVICE, generator=gen)] *= 20.0
    return (torch.randn(tokens, n, device=DEVICE, generator=gen) * size).to(TYPES[ty])


def _norm_inputs(gen, case):
    tokens, n, ty = case["tokens"], case["n"], case["type"]

    def weight():
        return 1.0 + 0.2 * torch.randn(n, device=DEVICE, generator=gen)

    return {"hidden": _stream(gen, tokens, n, ty),
            "block": torch.randn(tokens, n, device=DEVICE, generator=gen).to(TYPES[ty]),
            "post": weight() if case["post"] else None,
            # "row": one row of gates for every token
            "gate": None if case["gate"] == "none" else
            torch.randn(1 if case["gate"] == "row" else tokens, n, device=DEVICE, generator=gen).to(TYPES[ty]),
            "weight": weight(), "scale": 0.22}


def _product_inputs(gen, case):
    rows, k = case["rows"], case["k"]
    s = {"x": _rows(gen, case["tokens"], k), "w": _channels(gen, rows, k),
         "bias": 0.3 * torch.randn(rows, device=DEVICE, generator=gen), "scale": 1.0}
    if case["gated"]:
        s |= {"up": _channels(gen, rows, k), "up_bias": 0.3 * torch.randn(rows, device=DEVICE, generator=gen)}
    if case["residual"]:
        s |= {"residual": (2.0 * torch.randn(case["tokens"], rows, device=DEVICE, generator=gen)).to(TYPES[case["type"]]),
              "scale": 0.22}
    return s


def _route_inputs(gen, case):
    n, experts = case["n"], case["experts"]
    return {"x": torch.randn(case["tokens"], n, device=DEVICE, generator=gen).to(TYPES[case["type"]]),
            "router": torch.randn(experts, n, device=DEVICE, generator=gen) / math.sqrt(n),
            "bias": 0.1 * torch.randn(experts, device=DEVICE, generator=gen), "weight_scale": 2.5}


def _moe_inputs(gen, case):
    tokens, n, ffn, experts, top_k = case["tokens"], case["n"], case["ffn"], case["experts"], case["top_k"]
    s = {"x": _rows(gen, tokens, n), "gate": _channels(gen, experts, ffn, n), "up": _channels(gen, experts, ffn, n),
         "down": _channels(gen, experts, n, ffn),
         "residual": (2.0 * torch.randn(tokens, n, device=DEVICE, generator=gen)).to(TYPES[case["type"]])}
    if case["shared"]:
        s |= {"shared_gate": _channels(gen, case["shared"], n), "shared_up": _channels(gen, case["shared"], n),
              "shared_down": _channels(gen, n, case["shared"])}
    rank = torch.rand(tokens, experts, device=DEVICE, generator=gen)
    rank[:, torch.randperm(experts, device=DEVICE, generator=gen)[:case["hot"]]] += 2.0
    s["ids"] = rank.topk(top_k, 1).indices.sort(1).values.to(torch.int32)
    s["coefs"] = torch.softmax(torch.randn(tokens, top_k, device=DEVICE, generator=gen), 1)
    return s


INPUTS = {"norm": _norm_inputs, "product": _product_inputs, "route": _route_inputs, "moe": _moe_inputs}


def _inputs(case, seed):
    """Every raw input of a case, made from the seed alone."""
    return INPUTS[case["kind"]](torch.Generator(device=DEVICE).manual_seed(int(seed)), case)


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
    if own:   # the weights as the framework keeps them, and the workspace of the call
        be, kind, tokens = _be(), case["kind"], case["tokens"]
        s["be"], need = be, 16
        if kind == "product":
            s["m"] = be.upload_i8_gated(*s.pop("w"), *s.pop("up")) if case["gated"] else be.upload_i8(*s.pop("w"))
            need = be.gemm_i8_workspace_bytes(s["m"], tokens)
        elif kind == "route":
            s["m"] = be.router(s["router"].cpu().numpy(), s["bias"].cpu().numpy())
            need = be.route_rows_workspace_bytes(s["m"], tokens)
        elif kind == "moe":
            (g, gs), (u, us), (d, ds) = s.pop("gate"), s.pop("up"), s.pop("down")
            experts = [(be.upload_i8_gated(g[e], gs[e], u[e], us[e]), be.upload_i8(d[e], ds[e]))
                       for e in range(case["experts"])]
            shared = (be.upload_i8_gated(*s.pop("shared_gate"), *s.pop("shared_up")),
                      be.upload_i8(*s.pop("shared_down"))) if case["shared"] else None
            s["m"] = be.moe_i8_create(experts, shared)
            need = be.moe_i8_workspace_bytes(s["m"], tokens, case["top_k"])
        s["workspace"] = torch.zeros(max(need, 16), dtype=torch.uint8, device=DEVICE)
    return s


# ------------------------------------------------------------------ plain forms


def _values(v):
    """int8 rows of 64-bit values and their scales in 32 bits: (q, scale), the rounding done in 64 bits."""
    scale = (v.abs().amax(-1, keepdim=True) / 127.0).float()
    scale = torch.where(scale < LEAST, torch.zeros_like(scale), scale)
    q = torch.round(v / torch.where(scale > 0, scale, torch.ones_like(scale)).double())
    return torch.where(scale > 0, q.clamp(-127, 127), torch.zeros_like(q)), scale


def _norm(v, weight, eps):
    return v * torch.rsqrt((v * v).mean(1, keepdim=True) + eps) * weight.double()


def _plain_norm(s):
    """In 64 bits: the int8 values are next to borders."""
    case, h = s["case"], s["hidden"]
    p = s["block"].double()
    if case["post"]:
        p = _norm(p, s["post"], POST_EPS)
    if case["gate"] != "none":
        g = s["gate"].double()
        open_ = 1.0 / (1.0 + torch.exp(-g))
        p = p * (g if case["gate"] == "row" else open_ if case["gate"] == "sigmoid" else g * open_)
    h = (h.double() + s["scale"] * p).float().to(h.dtype)
    v = _norm(h.double(), s["weight"], EPS)
    if case["out"] == "rows":
        return {"hidden": h, "rows": v.float().to(h.dtype)}
    q, scale = _values(v)
    return {"hidden": h, "values": q.float() * scale}


def _sums(x, w):
    """int8 rows x int8 channels: whole numbers far below 2^24, which 32 bits add exactly."""
    return x.float() @ w.float().t()


def _act(v, act):
    if act == "relu":
        return v.clamp(min=0.0)
    if act == "relu2":
        return v.clamp(min=0.0) ** 2
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    return v


def _plain_product(s):
    case = s["case"]
    (q, xs), (w, ws) = s["x"], s["w"]
    v = _act(_sums(q, w) * xs.reshape(-1, 1) * ws + s["bias"], case["act"])
    if case["gated"]:
        u, us = s["up"]
        v = v * (_sums(q, u) * xs.reshape(-1, 1) * us + s["up_bias"])
    if case["residual"]:
        v = s["residual"].float() + s["scale"] * v
    return v.to(TYPES[case["type"]])


def _plain_route(s):
    """In 64 bits: two experts' scores may be next to each other."""
    case = s["case"]
    logits = s["x"].double() @ s["router"].double().t().contiguous()
    score = torch.sigmoid(logits) + s["bias"].double() if case["mode"] else logits
    ids = torch.sort(score, dim=1, descending=True, stable=True).indices[:, :case["top_k"]].sort(1).values
    best = torch.gather(logits, 1, ids)
    if case["mode"]:
        open_ = torch.sigmoid(best)
        coefs = open_ / open_.sum(1, keepdim=True).clamp(min=FLOOR)
    else:
        e = torch.exp(best - best.amax(1, keepdim=True))
        coefs = e / e.sum(1, keepdim=True)
    return {"ids": ids.to(torch.int32), "coefs": (coefs * s["weight_scale"]).float(), "logits": logits.float()}


def _pair_sums(w, ids, x):
    """Sums of each (token, expert) pair's matrix and row: exact in 32 bits, as above."""
    return torch.bmm(w[ids].float(), x.float().unsqueeze(2)).squeeze(2).double()


def _plain_expert(g, u):
    """silu(g) * u as the int8 rows that the second product reads."""
    return _values((g / (1.0 + torch.exp(-g)) * u).float().double())


def _plain_moe(s):
    case, (q, xs) = s["case"], s["x"]
    tokens, top_k = s["ids"].shape
    ids = s["ids"].reshape(-1).long()
    x, scale = q.repeat_interleave(top_k, 0), xs.double().repeat_interleave(top_k).unsqueeze(1)
    (gw, gs), (uw, us), (dw, ds) = s["gate"], s["up"], s["down"]
    h, hs = _plain_expert(_pair_sums(gw, ids, x) * scale * gs[ids].double(), _pair_sums(uw, ids, x) * scale * us[ids].double())
    y = _pair_sums(dw, ids, h) * hs.double() * ds[ids].double() * s["coefs"].reshape(-1, 1).double()
    y = y.reshape(tokens, top_k, -1).sum(1)
    if case["shared"]:
        (gw, gs), (uw, us), (dw, ds) = s["shared_gate"], s["shared_up"], s["shared_down"]
        scale = xs.double().unsqueeze(1)
        h, hs = _plain_expert(_sums(q, gw).double() * scale * gs.double(), _sums(q, uw).double() * scale * us.double())
        y = y + _sums(h, dw).double() * hs.double() * ds.double()
    return (s["residual"].double() + y).float().to(TYPES[case["type"]])


PLAIN = {"norm": _plain_norm, "product": _plain_product, "route": _plain_route, "moe": _plain_moe}


# ------------------------------------------------------------------ the framework's calls


def _own_norm(s):
    case, h = s["case"], s["hidden"]
    after = torch.empty_like(h)
    args = {"post_weight": s["post"], "post_eps": POST_EPS, "gate": s["gate"],
            "gate_act": "none" if case["gate"] in ("none", "row") else case["gate"], "scale": s["scale"],
            "weight": s["weight"], "eps": EPS}
    if case["out"] == "rows":
        rows = torch.empty_like(h)
        s["be"].block_norm_rows(s["block"], h, after, y=rows, **args)
        return {"hidden": after, "rows": rows}
    q = torch.empty(h.shape, dtype=torch.int8, device=DEVICE)
    scales = torch.empty(h.shape[0], device=DEVICE)
    s["be"].block_norm_rows(s["block"], h, after, q=q, scales=scales, **args)
    return {"hidden": after, "values": torch.mul(q, scales.unsqueeze(1))}


def _own_product(s):
    case = s["case"]
    y = torch.empty(case["tokens"], case["rows"], dtype=TYPES[case["type"]], device=DEVICE)
    s["be"].gemm_i8_act(s["m"], *s["x"], y, case["act"], s["workspace"], bias=s["bias"], up_bias=s.get("up_bias"),
                        residual=s.get("residual"), scale=s["scale"])
    return y


def _own_route(s):
    case = s["case"]
    ids = torch.empty(case["tokens"], case["top_k"], dtype=torch.int32, device=DEVICE)
    coefs = torch.empty(ids.shape, device=DEVICE)
    logits = torch.empty(case["tokens"], case["experts"], device=DEVICE)
    s["be"].route_rows(s["m"], s["x"], ids, coefs, s["workspace"], mode=case["mode"], weight_scale=s["weight_scale"],
                       logits=logits)
    return {"ids": ids, "coefs": coefs, "logits": logits}


def _own_moe(s):
    y = torch.empty_like(s["residual"])
    s["be"].moe_i8_forward(s["m"], *s["x"], s["ids"], s["coefs"], y, s["workspace"], residual=s["residual"])
    return y


OWN = {"norm": _own_norm, "product": _own_product, "route": _own_route, "moe": _own_moe}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["kind"]](state)


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    kind, t = case["kind"], case["tokens"]
    e = SIZE[case["type"]]
    if kind == "norm":
        n = case["n"]
        gates = {"none": 0, "row": 1}.get(case["gate"], t)
        return {"bytes": t * n * (3 * e + (e if case["out"] == "rows" else 1)) + gates * n * e + 4 * n * (2 if case["post"] else 1),
                "flops": 14 * t * n}
    if kind == "product":
        rows, k, parts = case["rows"], case["k"], 2 if case["gated"] else 1
        return {"bytes": parts * rows * (k + 8) + t * (k + 4) + t * rows * e * (2 if case["residual"] else 1),
                "flops": 2 * parts * t * rows * k}
    n, experts, top_k = case["n"], case["experts"], case["top_k"]
    if kind == "route":
        return {"bytes": 4 * experts * (n + 1) + t * (n * e + 4 * experts + 8 * top_k), "flops": 2 * t * experts * n}
    # The experts that at least one token has: the hot ones, and of the others what is to be expected.
    hot, ffn, shared = case["hot"], case["ffn"], case["shared"]
    others = experts - hot
    used = hot + (others * (1.0 - (1.0 - (top_k - hot) / others) ** t) if others else 0)
    return {"bytes": int(used * (3 * n * ffn + 8 * ffn + 4 * n)) + 3 * n * shared + 8 * shared + t * (n * (1 + 2 * e) + 4 + 8 * top_k),
            "flops": 6 * t * n * (top_k * ffn + shared)}


# ------------------------------------------------------------------ the results in 64 bits


def _exact_rms(v, weight, eps):
    return v * weight.double()[None, :] / torch.sqrt(torch.sum(v.square(), dim=1) / v.shape[1] + eps)[:, None]


def _exact_i8(v):
    """Nearest integers of v / scale, ties to even, the scale being the 32-bit value that the rows carry."""
    top = torch.maximum(v.amax(dim=1), -v.amin(dim=1))
    scale = (top / 127).to(torch.float32).double()
    live = scale >= LEAST
    ratio = v / torch.where(live, scale, 1.0)[:, None]
    low = torch.floor(ratio)
    over = ratio - low
    up = (over > 0.5) | ((over == 0.5) & (torch.remainder(low, 2) == 1))
    return torch.where(live[:, None], torch.clamp(low + up, -127, 127), 0.0), torch.where(live, scale, 0.0)


def _exact_norm(raw, case):
    p = raw["block"].double()
    if raw["post"] is not None:
        p = _exact_rms(p, raw["post"], POST_EPS)
    if raw["gate"] is not None:
        g = raw["gate"].double()
        p = p * {"row": lambda: g, "sigmoid": lambda: torch.sigmoid(g), "silu": lambda: g * torch.sigmoid(g)}[case["gate"]]()
    h = torch.add(raw["hidden"].double(), p, alpha=raw["scale"]).to(torch.float32).to(TYPES[case["type"]])
    v = _exact_rms(h.double(), raw["weight"], EPS)
    if case["out"] == "rows":
        return {"hidden": h.double(), "rows": v}
    q, scale = _exact_i8(v)
    return {"hidden": h.double(), "values": q * scale[:, None]}


def _exact_sums(q, scale, w, w_scale):
    """[tokens, rows], in pieces of rows that keep the 64-bit copies small."""
    a = q.double()
    parts = [torch.mm(a, w[at:at + 4096].double().t().contiguous()) for at in range(0, w.shape[0], 4096)]
    return torch.cat(parts, 1) * w_scale.double()[None, :] * scale.double()[:, None]


def _exact_act(v, act):
    root = math.sqrt(2.0 / math.pi)
    return {"none": lambda: v, "relu": lambda: torch.where(v > 0, v, 0.0), "relu2": lambda: torch.where(v > 0, v * v, 0.0),
            "silu": lambda: v * torch.sigmoid(v), "gelu": lambda: v * 0.5 * torch.special.erfc(-v / math.sqrt(2.0)),
            "gelu_tanh": lambda: v * torch.sigmoid(2.0 * root * (v + 0.044715 * v ** 3))}[act]()


def _exact_product(raw, case):
    y = _exact_act(_exact_sums(*raw["x"], *raw["w"]) + raw["bias"].double(), case["act"])
    if case["gated"]:
        y = y * (_exact_sums(*raw["x"], *raw["up"]) + raw["up_bias"].double())
    return y * raw["scale"] + raw["residual"].double() if case["residual"] else y


def _exact_route(raw, case):
    logits = torch.mm(raw["x"].double(), raw["router"].double().t().contiguous())
    score = logits if case["mode"] == 0 else 1.0 / (1.0 + torch.exp(-logits)) + raw["bias"].double()
    ids = torch.argsort(-score, dim=1, stable=True)[:, :case["top_k"]].sort(1).values
    best = logits.gather(1, ids)
    if case["mode"] == 0:
        coefs = torch.softmax(best, 1)
    else:
        w = 1.0 / (1.0 + torch.exp(-best))
        coefs = w / torch.clamp(w.sum(1, keepdim=True), min=FLOOR)
    return {"ids": ids.to(torch.int32), "coefs": coefs * raw["weight_scale"], "logits": logits}


def _exact_expert(q, scale, gate, up, down):
    """down(silu(gate) * up) of int8 rows; the rows between them are 32-bit floats before they are int8."""
    g = _exact_sums(q, scale, *gate)
    hq, hs = _exact_i8((g * torch.sigmoid(g) * _exact_sums(q, scale, *up)).to(torch.float32).double())
    return _exact_sums(hq, hs, *down)


def _exact_moe(raw, case):
    q, scale = raw["x"]
    y = raw["residual"].double()
    if case["shared"]:
        y = y + _exact_expert(q, scale, raw["shared_gate"], raw["shared_up"], raw["shared_down"])
    for e in torch.unique(raw["ids"]).tolist():
        t, slot = (raw["ids"] == e).nonzero(as_tuple=True)
        out = _exact_expert(q[t], scale[t], *((raw[m][0][e], raw[m][1][e]) for m in ("gate", "up", "down")))
        y.index_add_(0, t, out * raw["coefs"][t, slot].double()[:, None])
    return y


def exact(case, seed):
    return {"norm": _exact_norm, "product": _exact_product, "route": _exact_route, "moe": _exact_moe}[case["kind"]](
        _inputs(case, seed), case)
