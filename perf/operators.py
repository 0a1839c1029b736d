"""Operators of mixture-of-experts feed-forward layers outside a stack, as cases that can be timed and compared.

* ``route``: router logits to selected experts, their weights and the grouping of the selections by expert;
* ``quantize``: rows to MXFP4 (E2M1 codes, one power-of-two scale per 32 columns), with the values the codes stand for;
* ``matmul``: a dense W4A4 projection, the activations quantised on the way;
* ``experts``: the same by expert groups, for gathered token rows, with the gate's activation applied to the up rows;
* ``combine``: the weighted sum of each token's expert rows.

``run`` with ``own`` false states them in elementary torch operations; with ``own`` true it calls the library.  Sizes are
those of the repository's benchmark configurations (hidden 2816, 128 experts of 704, top-8; hidden 5120, 64 experts of 1536,
top-4; projections of 4096 x 4096 and of the dense branch, 2112 x 2816) and generic ones.
"""
from __future__ import annotations

import importlib
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 32


def listed():
    small = {"hidden": 2816, "inter": 704, "experts": 128, "topk": 8}
    large = {"hidden": 5120, "inter": 1536, "experts": 64, "topk": 4}
    plain = {"groups": 1, "top_groups": 1, "group_top": 1}
    return [
        # the next token of one chat: nothing but latency
        dict(plain, name="route-token", op="route", tokens=1, experts=128, topk=8, scoring="softmax", bias=False, renorm=True,
             dtype="f32"),
        # a prompt chunk of a model that balances its experts by a bias and limits a token to half of the groups
        dict(name="route-prompt-groups", op="route", tokens=4099, experts=256, topk=8, scoring="sigmoid", bias=True, renorm=True,
             dtype="bf16", groups=8, top_groups=4, group_top=2),
        # activations of a small decode batch
        {"name": "quantize-batch", "op": "quantize", "tokens": 16, "cols": 5120, "fan": 0, "dtype": "bf16"},
        # the rows of a prompt in the order of their experts, each token eight times
        {"name": "quantize-prompt-gather", "op": "quantize", "tokens": 1999, "cols": 2816, "fan": 8, "dtype": "f32"},
        # one projection of the next token
        {"name": "matmul-token", "op": "matmul", "tokens": 1, "rows": 4096, "cols": 4096, "dtype": "bf16"},
        # the dense branch beside the experts for a few streams with draft tokens
        {"name": "matmul-drafts", "op": "matmul", "tokens": 37, "rows": 2112, "cols": 2816, "dtype": "f32"},
        # a projection of a long prompt
        {"name": "matmul-prompt", "op": "matmul", "tokens": 4096, "rows": 5120, "cols": 5120, "dtype": "bf16"},
        # gate and up of the next token's experts
        dict(large, name="experts-token", op="experts", tokens=1, gated=True, dtype="bf16"),
        # gate and up of a decode batch: most experts with a few tokens each
        dict(small, name="experts-batch", op="experts", tokens=64, gated=True, dtype="f32"),
        # gate and up of a prompt of ragged length
        dict(large, name="experts-prompt", op="experts", tokens=1999, gated=True, dtype="bf16"),
        # the experts' rows of a decode batch and of a prompt, back in token order
        {"name": "combine-batch", "op": "combine", "tokens": 64, "cols": 2816, "topk": 8, "dtype": "f32"},
        {"name": "combine-prompt", "op": "combine", "tokens": 1999, "cols": 5120, "topk": 4, "dtype": "bf16"},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["route", "quantize", "matmul", "matmul", "experts", "experts", "experts", "combine"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "route":
        grouped = rng.random() < 0.5
        groups = rng.choice([4, 8, 16]) if grouped else 1
        per = _spread(rng, 8, 384 // groups)
        top_groups = rng.randint(max(1, -(-16 // per)), groups) if grouped else 1
        return {"op": op, "tokens": _spread(rng, 1, 4099), "experts": groups * per, "groups": groups, "top_groups": min(groups, top_groups),
                "group_top": rng.choice([1, 2]), "topk": rng.randint(1, 8), "scoring": rng.choice(["softmax", "sigmoid"]),
                "bias": rng.random() < 0.5, "renorm": rng.random() < 0.7, "dtype": dtype}
    if op == "quantize":
        fan = rng.choice([0, 2, 4, 8])
        return {"op": op, "tokens": _spread(rng, 1, 16000 // max(fan, 1)), "cols": BLOCK * _spread(rng, 8, 160), "fan": fan, "dtype": dtype}
    if op == "matmul":
        return {"op": op, "tokens": _spread(rng, 1, 4096), "rows": _spread(rng, 200, 5120), "cols": BLOCK * _spread(rng, 8, 160),
                "dtype": dtype}
    if op == "experts":
        gated = rng.random() < 0.6
        return {"op": op, "tokens": _spread(rng, 1, 1999), "hidden": BLOCK * _spread(rng, 16, 160), "inter": BLOCK * _spread(rng, 8, 48),
                "experts": rng.choice([8, 31, 64]), "topk": rng.choice([1, 2, 4]), "gated": gated, "dtype": dtype}
    return {"op": op, "tokens": _spread(rng, 1, 1999), "cols": _spread(rng, 200, 5120), "topk": rng.choice([1, 2, 4, 6, 8]), "dtype": dtype}


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _grid():
    return torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device="cuda")


def _mx_weights(g, rows, cols, out_codes, out_scales):
    """A trained matrix as it is stored: normal values, larger in some columns, quantised by the format's rule."""
    w = torch.randn(rows, cols, device="cuda", generator=g) * (1.0 / math.sqrt(cols))
    w *= torch.exp(0.5 * torch.randn(1, cols, device="cuda", generator=g))
    values, scale = _quantized(w)
    code = torch.bucketize(values.abs(), _grid()).to(torch.uint8) | (torch.signbit(w).to(torch.uint8) << 3)
    code = code.view(rows, cols // 2, 2)
    out_codes.copy_(code[:, :, 0] | (code[:, :, 1] << 4))
    out_scales.copy_(scale.to(torch.uint8))


def _activations(g, rows, cols, dtype):
    """Normalised hidden states: unit rows with a few channels far above the others."""
    x = torch.randn(rows, cols, device="cuda", generator=g)
    x[:, torch.randperm(cols, device="cuda", generator=g)[:max(1, cols // 200)]] *= 12.0
    return x.to(DTYPES[dtype])


def _choices(g, tokens, experts, topk):
    """Distinct experts of every token, ascending, and their grouping."""
    ids = torch.rand(tokens, experts, device="cuda", generator=g).topk(topk, dim=1).indices.sort(dim=1).values
    return ids, *_grouping(ids, experts)


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, T = case["op"], case["tokens"]
    s = {"case": case}
    if op == "route":
        E = case["experts"]
        s["logits"] = (2.0 * torch.randn(T, E, device="cuda", generator=g)).to(DTYPES[case["dtype"]])
        s["bias"] = 0.2 * torch.randn(E, device="cuda", generator=g) if case["bias"] else None
    elif op == "quantize":
        s["x"] = _activations(g, T, case["cols"], case["dtype"])
        n = T * max(case["fan"], 1)
        s["index"] = torch.randperm(n, device="cuda", generator=g).to(torch.int32) if case["fan"] else None
    elif op == "matmul":
        R, C = case["rows"], case["cols"]
        s["codes"] = torch.empty(1, R, C // 2, dtype=torch.uint8, device="cuda")
        s["scales"] = torch.empty(1, R, C // BLOCK, dtype=torch.uint8, device="cuda")
        _mx_weights(g, R, C, s["codes"][0], s["scales"][0])
        s["x"] = _activations(g, T, C, case["dtype"])
    elif op == "experts":
        H, M, E = case["hidden"], case["inter"], case["experts"]
        R, C = (M, H) if case["gated"] else (H, M)
        for name in ("codes", "up_codes") if case["gated"] else ("codes",):
            s[name] = torch.empty(E, R, C // 2, dtype=torch.uint8, device="cuda")
            s[name.replace("codes", "scales")] = torch.empty(E, R, C // BLOCK, dtype=torch.uint8, device="cuda")
            for e in range(E):
                _mx_weights(g, R, C, s[name][e], s[name.replace("codes", "scales")][e])
        _, s["offsets"], s["index"], _ = _choices(g, T, E, case["topk"])
        # gate and up read the tokens' rows through the grouping, down the rows that gate and up left in grouped order
        s["x"] = _activations(g, T if case["gated"] else T * case["topk"], C, case["dtype"])
    else:
        s["rows"] = _activations(g, T * case["topk"], case["cols"], case["dtype"])
        s["index"] = torch.randperm(T * case["topk"], device="cuda", generator=g).to(torch.int32)
        w = torch.rand(T, case["topk"], device="cuda", generator=g) + 0.05
        s["weights"] = w / w.sum(dim=1, keepdim=True)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if not own:
        return s
    lib = importlib.import_module("salt-core_b200.experts")
    op, T, out = case["op"], case["tokens"], DTYPES[case["dtype"]]

    def new(*shape, dtype):
        return torch.empty(*shape, dtype=dtype, device="cuda")

    if op == "route":
        n = T * case["topk"]
        s["spec"] = lib.RouteSpec(case["experts"], case["topk"], scoring=case["scoring"], n_groups=case["groups"],
                                  topk_groups=case["top_groups"], group_top=case["group_top"], renormalize=case["renorm"])
        s["out"] = [new(T, case["topk"], dtype=torch.int32), new(T, case["topk"], dtype=torch.float32),
                    new(case["experts"] + 1, dtype=torch.int32), new(n, dtype=torch.int32), new(n, dtype=torch.int32)]
    elif op == "combine":
        s["y"] = new(T, case["cols"], dtype=out)
    else:
        if op == "quantize":
            C, n = case["cols"], T * max(case["fan"], 1)
            s["values"] = new(n, C, dtype=out)
        else:
            R, C = s["codes"].shape[1], s["codes"].shape[2] * 2
            n = s["index"].numel() if op == "experts" else T
            s["weights"] = lib.Mxfp4Weights(R, C, s["codes"].shape[0], s["codes"].data_ptr(), s["scales"].data_ptr(),
                                            up_codes=s["up_codes"].data_ptr() if "up_codes" in s else 0,
                                            up_scales=s["up_scales"].data_ptr() if "up_scales" in s else 0, activation="silu")
            s["y"] = new(n, R, dtype=out)
        s["x_codes"] = new(n, C // 2, dtype=torch.uint8)
        s["x_scales"] = new(n, lib.scale_pitch(C), dtype=torch.uint8)
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------------

def _quantized(x):
    """Values of the E2M1 codes of x's blocks of 32 (before the scale), and the blocks' scale exponents."""
    b = x.float().view(x.shape[0], -1, BLOCK)
    top = b.abs().amax(dim=2)
    scale = ((top.view(torch.int32) >> 23) - 2).clamp(min=0)
    u = b * ((254 - scale) << 23).view(torch.float32)[:, :, None]
    a = u.abs().clamp(max=6.0)
    step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0))
    return torch.copysign(torch.round(a / step) * step, u).view(x.shape), scale


def _power(scale):
    return (scale.to(torch.int32) << 23).view(torch.float32)


def _quantized_values(x):
    values, scale = _quantized(x)
    return values * _power(scale).repeat_interleave(BLOCK, dim=1)


def _weights(codes, scales):
    """The matrices that packed codes and scale bytes stand for, in 32 bits."""
    both = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).to(torch.int32)
    values = _grid()[both & 7] * (1 - 2 * (both >> 3))
    return values * _power(scales).repeat_interleave(BLOCK, dim=-1)


def _grouping(ids, experts):
    flat = ids.reshape(-1)
    order = torch.sort(flat, stable=True).indices
    counts = torch.bincount(flat, minlength=experts)
    offsets = torch.cat((counts.new_zeros(1), counts.cumsum(0)))
    back = torch.empty_like(order)
    back[order] = torch.arange(order.numel(), device=order.device)
    return offsets.to(torch.int32), order.to(torch.int32), back.to(torch.int32)


def _route(s):
    c = s["case"]
    logits = s["logits"].double()
    scores = torch.softmax(logits, dim=1) if c["scoring"] == "softmax" else 1.0 / (1.0 + torch.exp(-logits))
    keys = scores if s["bias"] is None else scores + s["bias"].double()
    if c["groups"] > 1:
        best = keys.view(len(keys), c["groups"], -1).sort(dim=2, descending=True).values[:, :, :c["group_top"]].sum(dim=2)
        stay = best.sort(dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
        mask = torch.zeros_like(best, dtype=torch.bool).scatter_(1, stay, True)
        keys = keys.masked_fill(~mask.repeat_interleave(c["experts"] // c["groups"], dim=1), -math.inf)
    ids = keys.sort(dim=1, descending=True, stable=True).indices[:, :c["topk"]].sort(dim=1).values
    w = scores.gather(1, ids)
    if c["renorm"]:
        w = w / w.sum(dim=1, keepdim=True)
    return [ids.to(torch.int32), w.float(), *_grouping(ids, c["experts"])]


def _experts(s):
    """Every expert's rows padded to the longest group, one batched product."""
    c = s["case"]
    x = _quantized_values(s["x"])
    if c["gated"]:
        x = x[s["index"].long() // c["topk"]]
    offsets = s["offsets"].long()
    counts = offsets[1:] - offsets[:-1]
    used = counts.nonzero()[:, 0]
    group = torch.repeat_interleave(torch.arange(used.numel(), device="cuda"), counts[used])
    place = torch.arange(x.shape[0], device="cuda") - offsets[used][group]
    padded = x.new_zeros(used.numel(), int(counts.max()), x.shape[1])
    padded[group, place] = x
    y = torch.bmm(padded, _weights(s["codes"][used], s["scales"][used]).transpose(1, 2))[group, place]
    if c["gated"]:
        up = torch.bmm(padded, _weights(s["up_codes"][used], s["up_scales"][used]).transpose(1, 2))[group, place]
        y = y / (1.0 + torch.exp(-y)) * up
    return y.to(s["x"].dtype)


def _plain(s):
    c = s["case"]
    if c["op"] == "route":
        return _route(s)
    if c["op"] == "quantize":
        x = s["x"] if s["index"] is None else s["x"][s["index"].long() // c["fan"]]
        return _quantized_values(x).to(x.dtype)
    if c["op"] == "matmul":
        return (_quantized_values(s["x"]) @ _weights(s["codes"][0], s["scales"][0]).t()).to(s["x"].dtype)
    if c["op"] == "experts":
        return _experts(s)
    rows = s["rows"].float()[s["index"].long()].view(c["tokens"], c["topk"], -1)
    return (rows * s["weights"][:, :, None]).sum(dim=1).to(s["rows"].dtype)


def run(state):
    if not own:
        return _plain(state)
    s, c = state, state["case"]
    lib = importlib.import_module("salt-core_b200.experts")
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "route":
        bias = 0 if s["bias"] is None else s["bias"].data_ptr()
        rc = lib.route(s["spec"], s["logits"].data_ptr(), c["tokens"], *[t.data_ptr() for t in s["out"]], dtype=c["dtype"],
                       d_bias=bias, stream=stream)
        out = s["out"]
    elif c["op"] == "combine":
        rc = lib.combine(s["rows"].data_ptr(), s["rows"].shape[0], c["cols"], s["index"].data_ptr(), s["weights"].data_ptr(), c["tokens"],
                         c["topk"], s["y"].data_ptr(), dtype=c["dtype"], y_dtype=c["dtype"], stream=stream)
        out = s["y"]
    else:
        x, gather = s["x"], s.get("index")
        if c["op"] == "experts" and not c["gated"]:
            gather = None
        rc = lib.quantize(x.data_ptr(), x.shape[0], x.shape[1], s["x_codes"].data_ptr(), s["x_scales"].data_ptr(), dtype=c["dtype"],
                          rows=s["x_codes"].shape[0], d_row_index=0 if gather is None else gather.data_ptr(),
                          index_div=c.get("fan") or c.get("topk") or 1,
                          d_values=s["values"].data_ptr() if "values" in s else 0, stream=stream)
        out = s.get("values", s.get("y"))
        if rc == 0 and c["op"] == "matmul":
            rc = s["weights"].matmul(s["x_codes"].data_ptr(), s["x_scales"].data_ptr(), c["tokens"], out.data_ptr(), y_dtype=c["dtype"],
                                     stream=stream)
        elif rc == 0 and c["op"] == "experts":
            rc = s["weights"].experts(s["x_codes"].data_ptr(), s["x_scales"].data_ptr(), s["offsets"].data_ptr(), out.shape[0],
                                      out.data_ptr(), y_dtype=c["dtype"], stream=stream)
    if rc != 0:
        raise RuntimeError(f"{c['op']} was refused")
    return out


# ---- definition in 64 bits, written apart ---------------------------------------------------------------------------

def _exact_quantized(x):
    """Nearest point of the E2M1 grid by search, the even code where two are equally near."""
    b = x.double().view(-1, BLOCK)
    top = b.abs().amax(dim=1, keepdim=True)
    power = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top))))
    power = torch.where(torch.exp2(power) > top, power - 1, torch.where(torch.exp2(power + 1) <= top, power + 1, power))
    unit = torch.exp2((power - 2).clamp(min=-127.0))
    unit = torch.where(top > 0, unit, torch.full_like(unit, 2.0 ** -127))
    a = (b / unit).abs().clamp(max=6.0)
    points = _grid().double()
    above = torch.searchsorted(points, a).clamp(1, 7)
    low, high = points[above - 1], points[above]
    up = (a - low > high - a) | ((a - low == high - a) & (above % 2 == 0))
    return (torch.where(up, high, low) * torch.sign(b) * unit).view(x.shape)


def _exact_weights(codes, scales):
    table = torch.cat((_grid(), -_grid())).double()
    pairs = torch.stack((table[(codes % 16).long()], table[(codes // 16).long()]), dim=2)
    return (pairs.view(codes.shape[0], -1, BLOCK) * torch.exp2(scales.double() - 127.0)[:, :, None]).view(codes.shape[0], -1)


def _exact_route(s):
    c = s["case"]
    T, E, G = c["tokens"], c["experts"], c["groups"]
    l = s["logits"].double()
    if c["scoring"] == "softmax":
        p = torch.exp(l - l.amax(dim=1, keepdim=True))
        p = p / p.sum(dim=1, keepdim=True)
    else:
        p = torch.sigmoid(l)
    key = p + (0.0 if s["bias"] is None else s["bias"].double())
    left = torch.ones(T, E, dtype=torch.bool, device=l.device)
    if G > 1:
        grouped, total = key.view(T, G, E // G).clone(), 0.0
        for _ in range(c["group_top"]):
            best, at = grouped.max(dim=2)
            total = total + best
            grouped.scatter_(2, at[:, :, None], -math.inf)
        kept = torch.zeros(T, G, dtype=torch.bool, device=l.device)
        for _ in range(c["top_groups"]):
            kept.scatter_(1, total.masked_fill(kept, -math.inf).argmax(dim=1, keepdim=True), True)
        left = kept[:, :, None].expand(T, G, E // G).reshape(T, E).clone()
    chosen = torch.zeros_like(left)
    for _ in range(c["topk"]):
        chosen.scatter_(1, key.masked_fill(~left | chosen, -math.inf).argmax(dim=1, keepdim=True), True)
    token, expert = chosen.nonzero(as_tuple=True)
    ids = expert.view(T, c["topk"])
    w = p[token, expert].view(T, c["topk"])
    if c["renorm"]:
        w = w / w.sum(dim=1, keepdim=True)
    canonical = torch.arange(T * c["topk"], device=l.device).view(T, c["topk"])
    by_expert = torch.argsort(expert * T + token)
    counts = (expert[None] == torch.arange(E, device=l.device)[:, None]).sum(dim=1)
    offsets = torch.zeros(E + 1, dtype=torch.long, device=l.device)
    offsets[1:] = torch.cumsum(counts, 0)
    return [ids.int(), w, offsets.int(), canonical.view(-1)[by_expert].int(), torch.argsort(by_expert).int()]


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op == "route":
        return _exact_route(s)
    if op == "quantize":
        x = s["x"] if s["index"] is None else s["x"].repeat_interleave(case["fan"], dim=0)[s["index"].long()]
        return _exact_quantized(x)
    if op == "matmul":
        return _exact_quantized(s["x"]) @ _exact_weights(s["codes"][0], s["scales"][0]).T
    if op == "combine":
        y = torch.zeros(case["tokens"], case["cols"], dtype=torch.float64, device="cuda")
        for j in range(case["topk"]):
            y += s["weights"][:, j:j + 1].double() * s["rows"][s["index"].view(-1, case["topk"])[:, j].long()].double()
        return y
    x = _exact_quantized(s["x"])
    if case["gated"]:
        x = x.repeat_interleave(case["topk"], dim=0)[s["index"].long()]
    bounds = s["offsets"].tolist()
    parts = []
    for e in range(case["experts"]):
        rows = x[bounds[e]:bounds[e + 1]]
        y = rows @ _exact_weights(s["codes"][e], s["scales"][e]).T
        if case["gated"]:
            y = y * torch.sigmoid(y) * (rows @ _exact_weights(s["up_codes"][e], s["up_scales"][e]).T)
        parts.append(y)
    return torch.cat(parts)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def work(case):
    T, size = case["tokens"], {"f32": 4, "bf16": 2, "f16": 2}[case["dtype"]]
    op = case["op"]
    if op == "route":
        n, E = T * case["topk"], case["experts"]
        return {"bytes": T * E * size + (4 * E if case["bias"] else 0) + 16 * n + 4 * (E + 1), "flops": 10 * T * E}
    if op == "quantize":
        C, n = case["cols"], T * max(case["fan"], 1)
        return {"bytes": T * C * size + (4 * n if case["fan"] else 0) + n * C * (size + 0.5 + 1 / BLOCK), "flops": 3 * n * C}
    if op == "combine":
        C, n = case["cols"], T * case["topk"]
        return {"bytes": (n + T) * C * size + 8 * n, "flops": 2 * n * C}
    if op == "matmul":
        R, C = case["rows"], case["cols"]
        return {"bytes": R * C * (0.5 + 1 / BLOCK) + T * (C + R) * size, "flops": 2 * T * R * C}
    H, M, E, n = case["hidden"], case["inter"], case["experts"], T * case["topk"]
    R, C = (M, H) if case["gated"] else (H, M)
    matrices = 2 if case["gated"] else 1
    reached = E * (1.0 - (1.0 - case["topk"] / E) ** T)          # experts that at least one token selects, on average
    return {"bytes": reached * matrices * R * C * (0.5 + 1 / BLOCK) + ((T if case["gated"] else n) * C + n * R) * size + 8 * E,
            "flops": 2 * n * matrices * R * C}
