"""The operators around the routed experts of a layer, as they are measured: routing to the
experts, the norms before and after a block with its gate and residual, and the matrix
product in 8-bit integers of the shared expert and the dense projections.

`own` selects the side: the plain forms (elementary torch operations) or the calls a user
makes of crosslane_b200. The definitions both sides follow:

route   s = sigmoid(l), softmax(l) or sqrt(softplus(l)) of a token's logits l, correctly
        rounded to fp32. An expert is ranked by fl(s + bias); without a bias by l itself (s
        rises with l). Experts with l = -inf are not available. With groups, a group's value
        is its largest rank value, or the fp32 sum of its two largest s + bias (s without a
        bias), and only the best `top_groups` groups stay. The k best are picked, ties to the
        lower id; places that are left over take the other ids in ascending order with weight
        0. w = s, over the picks' sum (+ 1e-20) if renormalised, times the scale.
norm    h' = r h + b g z with z = y or RMSNorm(y) w_post, g one, a vector over the channels, a
        number for each token or a full tensor, or its sigmoid; x = RMSNorm(h') w_pre.
int8    each row of x: scale s = fl(max |x| / 127), q = x / s rounded to the nearest integer
        (ties to even); y[t, n] = s[t] sw[n] sum_k q[t, k] w[n, k] + bias[n].
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # one token of a decode step through the expert bank's layer: 384 experts, top 6
        {"name": "route_one", "op": "route", "tokens": 1, "experts": 384, "k": 6, "score": "sigmoid", "bias": True,
         "groups": 1, "top_groups": 1, "pair": False, "renorm": True, "scale": 2.5, "type": "f32", "masked": 0.0},
        # a decode batch with group-limited routing and 16-bit logits, a few sequences short of 64
        {"name": "route_groups", "op": "route", "tokens": 61, "experts": 384, "k": 8, "score": "sigmoid", "bias": True,
         "groups": 8, "top_groups": 4, "pair": True, "renorm": True, "scale": 2.5, "type": "bf16", "masked": 0.0},
        # a prompt of 2048 tokens with the square-root scores of the GPU stage
        {"name": "route_prompt", "op": "route", "tokens": 2048, "experts": 384, "k": 6, "score": "sqrt_softplus",
         "bias": True, "groups": 1, "top_groups": 1, "pair": False, "renorm": True, "scale": 1.5, "type": "f32",
         "masked": 0.0},
        # many prompts at once, softmax scores, experts masked out in places and padding rows
        {"name": "route_padded", "op": "route", "tokens": 16383, "experts": 256, "k": 8, "score": "softmax",
         "bias": False, "groups": 1, "top_groups": 1, "pair": False, "renorm": False, "scale": 1.0, "type": "f32",
         "masked": 0.05},
        # the residual step of one decoded token: norm after the block, norm before the next
        {"name": "norm_one", "op": "norm", "tokens": 1, "dim": 7168, "post": True, "pre": True, "gate": "none",
         "sigmoid": False, "h": "f32", "y": "f32", "x": "f32", "pad": 0},
        # the same for a prompt, with a learned scale on each channel
        {"name": "norm_prompt", "op": "norm", "tokens": 2048, "dim": 7168, "post": True, "pre": True,
         "gate": "channel", "sigmoid": False, "h": "f32", "y": "f32", "x": "f32", "pad": 0},
        # many prompts in 16 bits with a gate computed from the input (its logits)
        {"name": "norm_gated", "op": "norm", "tokens": 8192, "dim": 5120, "post": True, "pre": True, "gate": "full",
         "sigmoid": True, "h": "bf16", "y": "bf16", "x": "bf16", "pad": 0},
        # an odd width in rows of a wider buffer, a gate for each token, no norm after the block
        {"name": "norm_odd", "op": "norm", "tokens": 777, "dim": 2311, "post": False, "pre": True, "gate": "token",
         "sigmoid": True, "h": "f32", "y": "f16", "x": "f16", "pad": 5},
        # one token through the shared expert's gate matrix
        {"name": "int8_one", "op": "int8", "tokens": 1, "k": 7168, "n": 1536, "x": "f32", "out": "f32", "bias": False,
         "pad": 0},
        # a decode batch through the wider shared expert
        {"name": "int8_batch", "op": "int8", "tokens": 64, "k": 5120, "n": 2304, "x": "bf16", "out": "bf16",
         "bias": False, "pad": 0},
        # a prompt, one token short of its tile, through the shared expert's down matrix
        {"name": "int8_prompt", "op": "int8", "tokens": 2047, "k": 1536, "n": 7168, "x": "f32", "out": "f32",
         "bias": True, "pad": 0},
        # many prompts through a square projection
        {"name": "int8_large", "op": "int8", "tokens": 4096, "k": 7168, "n": 7168, "x": "bf16", "out": "bf16",
         "bias": False, "pad": 0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["route", "norm", "int8"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * _log(rng, 8, 512 // groups)
        top = rng.randint((groups + 1) // 2, groups)
        score = rng.choice(["sigmoid", "softmax", "sqrt_softplus"])
        return {"op": op, "tokens": _log(rng, 1, min(16384, 16383 * 256 // experts)), "experts": experts,
                "k": rng.randint(1, min(16, top * (experts // groups))), "score": score, "bias": rng.random() < 0.5,
                "groups": groups, "top_groups": top, "pair": rng.random() < 0.5, "renorm": rng.random() < 0.7,
                "scale": rng.choice([1.0, 1.5, 2.5]), "type": rng.choice(["f32", "f32", "bf16", "f16"]),
                "masked": rng.choice([0.0, 0.0, 0.05])}
    if op == "norm":
        dim = _log(rng, 64, 16384)
        if rng.random() < 0.6:
            dim = (dim + 7) // 8 * 8
        post = rng.random() < 0.8
        return {"op": op, "tokens": _log(rng, 1, min(8192, 8192 * 5120 // dim)), "dim": dim, "post": post,
                "pre": not post or rng.random() < 0.8, "gate": rng.choice(["none", "channel", "token", "full"]),
                "sigmoid": rng.random() < 0.5, "h": rng.choice(["f32", "bf16", "f16"]),
                "y": rng.choice(["f32", "bf16", "f16"]), "x": rng.choice(["f32", "bf16", "f16"]),
                "pad": rng.choice([0, 0, 5, 8])}
    k, n = _log(rng, 64, 8192), _log(rng, 64, 8192)
    if rng.random() < 0.6:
        k = (k + 15) // 16 * 16
    return {"op": op, "tokens": _log(rng, 1, min(4096, 4096 * 7168 * 7168 // (k * n))), "k": k, "n": n,
            "x": rng.choice(["f32", "bf16", "f16"]), "out": rng.choice(["f32", "bf16", "f16"]),
            "bias": rng.random() < 0.3, "pad": rng.choice([0, 0, 5, 8])}


def _rows(gen, tokens, width, dtype, pad, scale=1.0):
    """[tokens][width] normal values in rows of a buffer that is `pad` elements wider."""
    buf = torch.randn((tokens, width + pad), generator=gen, device="cuda") * scale
    return buf.to(dtype)[:, :width]


def _empty(tokens, width, dtype, pad):
    return torch.empty((tokens, width + pad), dtype=dtype, device="cuda")[:, :width]


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": case}
    T = case["tokens"]
    if case["op"] == "route":
        E = case["experts"]
        logits = torch.randn((T, E), generator=gen, device="cuda") * 1.5
        if case["masked"]:
            logits.masked_fill_(torch.rand((T, E), generator=gen, device="cuda") < case["masked"], -math.inf)
            logits.masked_fill_(torch.rand((T, 1), generator=gen, device="cuda") < 0.01, -math.inf)  # padding rows
        s["logits"] = logits.to(TYPES[case["type"]])
        s["bias"] = torch.randn(E, generator=gen, device="cuda") * 0.05 if case["bias"] else None
    elif case["op"] == "norm":
        D, pad = case["dim"], case["pad"]
        # a residual stream has channels far above the others
        lift = torch.where(torch.rand(D, generator=gen, device="cuda") < 0.01, 12.0, 1.0)
        s["h"] = _empty(T, D, TYPES[case["h"]], pad)
        s["h"].copy_(torch.randn((T, D), generator=gen, device="cuda") * lift * 2.0)
        s["y"] = _rows(gen, T, D, TYPES[case["y"]], pad, 0.3)
        shape = {"none": None, "channel": (D,), "token": (T,), "full": (T, D)}[case["gate"]]
        s["gate"] = None if shape is None else torch.randn(shape, generator=gen, device="cuda").to(TYPES[case["y"]])
        s["w_post"] = 1.0 + 0.2 * torch.randn(D, generator=gen, device="cuda") if case["post"] else None
        s["w_pre"] = 1.0 + 0.2 * torch.randn(D, generator=gen, device="cuda") if case["pre"] else None
    else:
        K, N = case["k"], case["n"]
        lift = torch.where(torch.rand(K, generator=gen, device="cuda") < 0.002, 8.0, 1.0)
        s["x"] = _empty(T, K, TYPES[case["x"]], case["pad"])
        s["x"].copy_(torch.randn((T, K), generator=gen, device="cuda") * lift)
        w = torch.randn((N, K), generator=gen, device="cuda") * 0.02
        s["w_scale"] = w.abs().amax(dim=1).div_(127.0)
        # stored with a row pitch of a multiple of 16 bytes, as the weights of a loaded model are
        s["w"] = torch.zeros((N, (K + 15) // 16 * 16), dtype=torch.int8, device="cuda")[:, :K]
        s["w"].copy_(w.div_(s["w_scale"][:, None]).round_())
        s["bias"] = torch.randn(N, generator=gen, device="cuda") * 0.1 if case["bias"] else None
    return s


RESIDUAL, BLOCK, EPS = 1.0, 0.5, 1e-6  # a block's output enters the residual stream at half its size


def prepare(case, seed):
    s = _inputs(case, seed)
    T = case["tokens"]
    if case["op"] == "route":
        s["ids"] = torch.empty((T, case["k"]), dtype=torch.int32, device="cuda")
        s["w"] = torch.empty((T, case["k"]), dtype=torch.float32, device="cuda")
    elif case["op"] == "norm":
        s["h_out"] = _empty(T, case["dim"], TYPES[case["h"]], case["pad"])
        s["x"] = _empty(T, case["dim"], TYPES[case["x"]], case["pad"]) if case["pre"] else None
    else:
        s["out"] = torch.empty((T, case["n"]), dtype=TYPES[case["out"]], device="cuda")
    if own:
        import crosslane_b200 as cb
        if case["op"] == "route":
            s["op"] = cb.ExpertRoute(case["experts"], case["k"], score=case["score"], n_groups=case["groups"],
                                     top_groups=case["top_groups"], group_score="pair" if case["pair"] else "max",
                                     renormalize=case["renorm"], scale=case["scale"])
        elif case["op"] == "norm":
            s["op"] = cb.BlockNorm(case["dim"], post=case["post"], pre=case["pre"], eps=EPS, gate=case["gate"],
                                   gate_sigmoid=case["sigmoid"], residual_scale=RESIDUAL, block_scale=BLOCK)
        else:
            s["op"] = cb.Int8Linear(s["w"], s["w_scale"], s["bias"])
            s["ws"] = torch.empty(s["op"].workspace_bytes(T), dtype=torch.uint8, device="cuda")
    return s


def run(state):
    op = state["case"]["op"]
    if own:
        if op == "route":
            state["op"].run(state["logits"], state["ids"], state["w"], d_bias=state["bias"])
            return state["ids"], state["w"]
        if op == "norm":
            state["op"].run(state["h"], d_y=state["y"], d_gate=state["gate"], d_w_post=state["w_post"],
                            d_w_pre=state["w_pre"], d_h_out=state["h_out"], d_x=state["x"])
            return (state["h_out"], state["x"]) if state["x"] is not None else (state["h_out"],)
        state["op"].run(state["x"], state["out"], d_ws=state["ws"])
        return state["out"]
    return {"route": _route, "norm": _norm, "int8": _int8}[op](state)


# -- the plain forms ---------------------------------------------------------------------

def _route(s):
    c = s["case"]
    l = s["logits"].float()
    T, E = l.shape
    G, k = c["groups"], c["k"]
    there = l > -math.inf
    v = l.double()
    if c["score"] == "sigmoid":
        score = torch.sigmoid(v)
    elif c["score"] == "softmax":
        top = v.amax(dim=1, keepdim=True)
        e = torch.exp(v - torch.where(top > -math.inf, top, 0.0))
        score = e / e.sum(dim=1, keepdim=True).clamp_min(1e-300)
    else:
        score = torch.sqrt(v.clamp_min(0.0) + torch.log1p(torch.exp(-v.abs())))
    score = score.float()
    rank = torch.where(there, l if s["bias"] is None else score + s["bias"], -math.inf)
    if G > 1:
        if c["pair"]:
            value = torch.where(there, score, -math.inf) if s["bias"] is None else rank
            best = torch.sort(value.view(T, G, E // G), dim=2, descending=True).values[:, :, :2]
            value = best[:, :, 0] + (torch.where(best[:, :, 1] > -math.inf, best[:, :, 1], 0.0) if E > G else 0.0)
        else:
            value = rank.view(T, G, E // G).amax(dim=2)
        kept = torch.sort(value, dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
        keep = torch.zeros((T, G), dtype=torch.bool, device=l.device).scatter_(1, kept, True)
        rank = torch.where(keep.repeat_interleave(E // G, dim=1), rank, -math.inf)
    ordered = torch.sort(rank, dim=1, descending=True, stable=True)
    ids = ordered.indices[:, :k]
    w = torch.where(ordered.values[:, :k] > -math.inf, score.gather(1, ids), 0.0)
    if c["renorm"]:
        w = w / (w.sum(dim=1, keepdim=True) + 1e-20)
    return ids.to(torch.int32), w * c["scale"]


def _norm(s):
    c = s["case"]
    h, z = s["h"].float(), s["y"].float()
    if c["post"]:
        z = z * torch.rsqrt(z.square().mean(dim=1, keepdim=True) + EPS) * s["w_post"]
    if s["gate"] is not None:
        g = s["gate"].float()
        g = torch.sigmoid(g) if c["sigmoid"] else g
        z = z * (g[:, None] if c["gate"] == "token" else g)
    h = RESIDUAL * h + BLOCK * z
    out = (h.to(s["h"].dtype),)
    if c["pre"]:
        out += ((h * torch.rsqrt(h.square().mean(dim=1, keepdim=True) + EPS) * s["w_pre"]).to(TYPES[c["x"]]),)
    return out


def _int8(s):
    x = s["x"].float()
    scale = (x.abs().amax(dim=1, keepdim=True).double() / 127.0).float()
    # the quotient in 64 bits: in 32 it rounds onto the border between two integers
    q = torch.where(scale > 0, torch.round(x.double() / scale.double()), 0.0).clamp_(-127.0, 127.0).float()
    y = (q @ s["w"].float().t()) * scale * s["w_scale"]
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(TYPES[s["case"]["out"]])


# -- what a pass cannot do without -------------------------------------------------------

def work(case):
    T = case["tokens"]
    if case["op"] == "route":
        E, k = case["experts"], case["k"]
        return {"bytes": T * E * BYTES[case["type"]] + (4 * E if case["bias"] else 0) + T * k * 8, "flops": 8 * T * E}
    if case["op"] == "norm":
        D = case["dim"]
        gate = {"none": 0, "channel": D, "token": T, "full": T * D}[case["gate"]] * BYTES[case["y"]]
        moved = T * D * (2 * BYTES[case["h"]] + BYTES[case["y"]] + (BYTES[case["x"]] if case["pre"] else 0))
        return {"bytes": moved + gate + 4 * D * (case["post"] + case["pre"]), "flops": 12 * T * D}
    K, N = case["k"], case["n"]
    moved = T * K * BYTES[case["x"]] + N * K + T * N * BYTES[case["out"]] + 4 * N * (2 if case["bias"] else 1)
    return {"bytes": moved, "flops": 2 * T * K * N}


# -- the same from the definitions, in 64 bits -------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed)
    return {"route": _exact_route, "norm": _exact_norm, "int8": _exact_int8}[case["op"]](case, s)


def _exact_route(c, s):
    l = s["logits"].float().cpu().numpy().astype(np.float64)
    T, E = l.shape
    G, k = c["groups"], c["k"]
    there = ~np.isneginf(l)
    m = np.where(there, l, -1e30).max(axis=1, keepdims=True)
    low = np.where(there, l, 0.0)
    p = {"sigmoid": lambda: 1.0 / (1.0 + np.exp(-low)), "softmax": lambda: np.where(there, np.exp(low - m), 0.0),
         "sqrt_softplus": lambda: np.sqrt(np.logaddexp(0.0, low))}[c["score"]]()
    if c["score"] == "softmax":
        p = p / np.maximum(p.sum(axis=1, keepdims=True), 1e-300)
    held = p.astype(np.float32)  # the ranks are defined on the fp32 scores
    rank = l.astype(np.float32) if s["bias"] is None else held + s["bias"].cpu().numpy()[None, :]
    rank = np.where(there, rank, np.float32(-np.inf))
    if G > 1:
        per = np.where(there, held, np.float32(-np.inf)) if c["pair"] and s["bias"] is None else rank
        per = -np.sort(-per.reshape(T, G, E // G), axis=2)
        value = per[:, :, 0]
        if c["pair"] and E > G:
            value = value + np.where(np.isneginf(per[:, :, 1]), np.float32(0), per[:, :, 1])
        place = np.argsort(np.argsort(-value, axis=1, kind="stable"), axis=1, kind="stable")
        rank = np.where(np.repeat(place < c["top_groups"], E // G, axis=1), rank, np.float32(-np.inf))
    ids = np.argsort(-rank, axis=1, kind="stable")[:, :k]
    w = np.where(np.isneginf(np.take_along_axis(rank, ids, 1)), 0.0, np.take_along_axis(p, ids, 1))
    if c["renorm"]:
        w = w / (w.sum(axis=1, keepdims=True) + 1e-20)
    return ids.astype(np.int32), w * c["scale"]


def _exact_norm(c, s):
    wide = {n: s[n].to(torch.float64) for n in ("h", "y", "gate", "w_post", "w_pre") if s[n] is not None}
    D = c["dim"]
    add = wide["y"]
    if c["post"]:
        add = wide["w_post"] * add / torch.sqrt((add * add).sum(1) / D + EPS)[:, None]
    if "gate" in wide:
        g = 1.0 / (1.0 + torch.exp(-wide["gate"])) if c["sigmoid"] else wide["gate"]
        add = add * g.reshape((-1, 1) if c["gate"] == "token" else (-1, D))
    h = wide["h"] * RESIDUAL + add * BLOCK
    if not c["pre"]:
        return (h,)
    return h, wide["w_pre"] * h / torch.sqrt((h * h).sum(1) / D + EPS)[:, None]


def _exact_int8(c, s):
    x = s["x"].to(torch.float64)
    step = (torch.maximum(x.max(1).values, -x.min(1).values) / 127.0).to(torch.float32).to(torch.float64)  # held in fp32
    q = torch.clamp(torch.round(x / step.clamp_min(1e-300)[:, None]), -127, 127)
    q[step == 0] = 0
    y = torch.matmul(q, s["w"].to(torch.float64).T) * s["w_scale"].to(torch.float64)[None, :] * step[:, None]
    return y if s["bias"] is None else y + s["bias"].to(torch.float64)
