"""What rotary positions, differential attention and the norms around a block are judged by: calls of decoders, of conditioned
transformers and of their training, from one token to long sequences, each in a plain form and through this package's entry points.

A case is a dict of plain values.  `op` says what one pass is:

    rotary        rotary_embedding of q [B, H, L, D] and k [B, Hkv, L, D]; "views": both are parts of one projection [B, L, (H + Hkv) D]
    rotary_train  the same with the gradients of q and k
    diff          differential_attention: q [B, 2H, Lq, D], k [B, 2Hkv, Lk, D], v [B, Hkv, Lk, Dv], lam [H]
    diff_train    the same with the gradients of q, k, v and lam
    norm          residual_norm: r = a x + act(gate) * post_norm(y), h = norm(r), x and y [B, T, C]
    norm_train    the same with the gradients of everything that goes in

Masks over the keys as batches have them: "ragged" rows end anywhere in their second half, "random" drops 8 % of the keys, "none" is no
mask.  A causal call's queries are the last Lq of the Lk tokens.  Gates, weights and biases of a norm are one row for all tokens
("channel", [C]), for the tokens of a sequence ("batch", [B, 1, C]) or every token's own ("token", [B, T, C]).
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _rotary(name, B, H, Hkv, L, D, rotary, dtype="bf16", interleaved=False, base=10000.0, factor=1.0, positions="offset", views=False, op="rotary"):
    return {"name": name, "op": op, "B": B, "H": H, "Hkv": Hkv, "L": L, "D": D, "rotary": rotary, "dtype": dtype, "interleaved": interleaved, "base": base, "factor": factor,
            "positions": positions, "views": views}


def _diff(name, B, H, Hkv, Lq, Lk, D, Dv, dtype="bf16", mask="none", causal=False, op="diff"):
    return {"name": name, "op": op, "B": B, "H": H, "Hkv": Hkv, "Lq": Lq, "Lk": Lk, "D": D, "Dv": Dv, "dtype": dtype, "mask": mask, "causal": causal}


def _norm(name, B, T, C, dtype="bf16", norm="rms", post="none", gate="none", activation="none", weight="channel", bias="none", scale=1.0, stream=True, op="norm"):
    return {"name": name, "op": op, "B": B, "T": T, "C": C, "dtype": dtype, "norm": norm, "post": post, "gate": gate, "activation": activation, "weight": weight, "bias": bias,
            "scale": scale, "stream": stream}


def listed():
    return [
        # a decoder's step of a batch of requests, each at a position of its own: launches and host time
        _rotary("rotary_token_b32", 32, 16, 4, 1, 128, 128, positions="requests"),
        # a long prompt behind the fused projection of its queries and keys, frequencies stretched to four times the trained length
        _rotary("rotary_prompt_n4096", 4, 32, 8, 4096, 128, 128, base=500000.0, factor=4.0, views=True),
        # a training step in full precision, interleaved pairs, half of the head turned, an odd length
        _rotary("rotary_train_n1491", 2, 12, 12, 1491, 64, 32, dtype="fp32", interleaved=True, op="rotary_train"),
        # a decoder's step over the caches of a batch of requests of many lengths
        _diff("diff_token_b32_k1491", 32, 16, 4, 1, 1491, 64, 128, mask="ragged"),
        # one request's step over a long cache, wide heads
        _diff("diff_token_k8192", 1, 16, 4, 1, 8192, 128, 256),
        # a long prompt
        _diff("diff_prompt_n4096", 2, 16, 4, 4096, 4096, 64, 128, causal=True),
        # queries to states of another length, in full precision, with dropped keys
        _diff("diff_fp32_n200_k768", 4, 8, 8, 200, 768, 32, 64, dtype="fp32", mask="random"),
        # a training step of a decoder's layer
        _diff("diff_train_n1024", 4, 12, 12, 1024, 1024, 64, 128, causal=True, op="diff_train"),
        # the end of one block and the beginning of the next for one token of each request: launches and host time
        _norm("norm_token_b32", 32, 1, 2048, post="rms"),
        # a conditioned transformer's tokens in training: sigmoid gates, weights and biases of every token's own
        _norm("norm_train_conditioned_n768", 8, 768, 768, norm="layer", gate="token", activation="sigmoid", weight="token", bias="token", op="norm_train"),
        # a wide decoder's layer in training: norms on both sides of the block, a learned gate by channel
        _norm("norm_train_n2048_c4096", 4, 2048, 4096, post="rms", gate="channel", op="norm_train"),
        # in full precision, odd numbers of tokens, a gate and a weight by sequence
        _norm("norm_train_fp32_n259_c384", 6, 259, 384, dtype="fp32", norm="layer", gate="batch", weight="batch", bias="channel", scale=0.5, op="norm_train"),
    ]


def _log(rng, low, high):
    """A whole number between low and high, spread over its logarithm; odd ones among them, and multiples of 8 as often as not."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.4:
        n = (n + 7) // 8 * 8
    return max(low, min(high, n))


def draw(rng):
    op = rng.choice(["rotary", "rotary_train", "diff", "diff", "token", "diff_train", "diff_train", "norm", "norm_train", "norm_train"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    if op in ("rotary", "rotary_train"):
        Hkv, G, D = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4]), rng.choice([32, 64, 80, 96, 128, 256])
        B = _log(rng, 1, 48)
        L = 1 if op == "rotary" and rng.random() < 0.3 else _log(rng, 2, min(16384, 2 ** 24 // (B * Hkv * (G + 1) * D)))
        rotary = rng.choice([D, D, D // 2, D // 4 // 2 * 2])
        return {k: v for k, v in _rotary("", B, Hkv * G, Hkv, L, D, rotary, dtype, rng.random() < 0.4, rng.choice([10000.0, 500000.0]), rng.choice([1.0, 4.0, 16.0]),
                                         rng.choice(["offset", "requests"]), rng.random() < 0.5, op).items() if k != "name"}
    if op in ("norm", "norm_train"):
        C = _log(rng, 64, 8192)
        B = _log(rng, 1, 32)
        T = 1 if op == "norm" and rng.random() < 0.3 else _log(rng, 2, min(8192, 2 ** 23 // (B * C)))
        kind = lambda *more: rng.choice(["channel", "channel", "batch", "token", *more])
        norm = rng.choice(["rms", "rms", "layer", "none"])
        gate = kind("none", "none")
        case = _norm("", B, T, C, dtype, norm, rng.choice(["none", "rms", "layer"]), gate, rng.choice(["none", "sigmoid"]) if gate != "none" else "none",
                     kind("none") if norm != "none" else "none", kind("none", "none") if norm != "none" else "none", rng.choice([1.0, 1.0, 0.7]), rng.random() < 0.8, op)
        return {k: v for k, v in case.items() if k != "name"}
    Hkv, G = rng.choice([1, 2, 4, 8]), rng.choice([1, 1, 2, 4])
    D = rng.choice([16, 24, 32, 48, 64, 64, 80, 128] if dtype == "bf16" else [16, 32, 48, 64])
    Dv = rng.choice([2 * D, 2 * D, 2 * D, D])
    mask = rng.choice(["none", "ragged", "random"])
    if op == "token":
        B = _log(rng, 1, 32)
        case = _diff("", B, Hkv * G, Hkv, rng.choice([1, 1, 2, 5]), _log(rng, 16, min(8192, 10 ** 8 // (B * Hkv * (2 * D + Dv)))), D, Dv, dtype, mask, rng.random() < 0.5)
    elif op == "diff":
        Lq = _log(rng, 16, 1491)
        case = _diff("", rng.randint(1, 4), Hkv * G, Hkv, Lq, _log(rng, 16, 2048), D, Dv, dtype, mask, rng.random() < 0.6)
    else:
        case = _diff("", rng.randint(1, 4), Hkv * G, Hkv, _log(rng, 16, 768), _log(rng, 16, 1024), D, Dv, dtype, mask, rng.random() < 0.6, op="diff_train")
    if case["causal"] and case["Lk"] < case["Lq"]:
        case["Lk"] = case["Lq"]
    case.pop("name")
    return case


# ---- inputs ---------------------------------------------------------------------------------------------------------------
def _frequencies(case):
    """base^(-2 i / n) for pair i of n / 2, the slow ones divided by the factor (a ramp between 32 turns and 1 within 2048 tokens), and the cosines' scale."""
    n, base, factor = case["rotary"], case["base"], case["factor"]
    plain = [base ** (-2.0 * i / n) for i in range(n // 2)]
    if factor == 1.0:
        return plain, 1.0
    place = lambda turns: n * math.log(2048 / (turns * 2 * math.pi)) / (2 * math.log(base))
    low, high = max(math.floor(place(32.0)), 0), min(math.ceil(place(1.0)), n - 1)
    ramp = [min(max((i - low) / max(high - low, 1e-3), 0.0), 1.0) for i in range(n // 2)]
    return [f / factor * r + f * (1.0 - r) for f, r in zip(plain, ramp)], 0.1 * math.log(factor) + 1.0


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    s = {"case": case}
    B = case["B"]
    leaves = []
    if case["op"] in ("rotary", "rotary_train"):
        H, Hkv, L, D = case["H"], case["Hkv"], case["L"], case["D"]
        if case["views"]:
            both = normal(B, L, H + Hkv, D).transpose(1, 2)
            s["q"], s["k"] = both[:, :H], both[:, H:]
        else:
            s["q"], s["k"] = normal(B, H, L, D), normal(B, Hkv, L, D)
        f, s["scale"] = _frequencies(case)
        s["frequencies"] = torch.tensor(f, dtype=torch.float64, device="cuda")
        s["offset"] = int(torch.randint(0, 30000, (1,), generator=gen, device="cuda")) if L > 1 else 701
        # (requests: each batch row goes on from a place of its own)
        s["positions"] = torch.randint(0, 8192, (B, 1), generator=gen, device="cuda") + torch.arange(L, device="cuda") if case["positions"] == "requests" else None
        if case["op"] == "rotary_train":
            leaves = ["q", "k"]
            s["q"], s["k"] = s["q"].detach(), s["k"].detach()
            s["grads"] = normal(B, H, L, D), normal(B, Hkv, L, D)
    elif case["op"] in ("diff", "diff_train"):
        H, Hkv, Lq, Lk, D, Dv = (case[n] for n in ("H", "Hkv", "Lq", "Lk", "D", "Dv"))
        s["q"], s["k"], s["v"] = normal(B, 2 * H, Lq, D), normal(B, 2 * Hkv, Lk, D), normal(B, Hkv, Lk, Dv)
        s["lam"] = (0.2 + 0.6 * torch.rand(H, generator=gen, device="cuda")).to(dtype)
        s["mask"] = None
        if case["mask"] == "random":
            s["mask"] = torch.rand(B, Lk, generator=gen, device="cuda") < 0.92
            s["mask"][:, 0] = True
        elif case["mask"] == "ragged":
            s["mask"] = torch.arange(Lk, device="cuda") < (Lk * (0.5 + 0.5 * torch.rand(B, 1, generator=gen, device="cuda"))).ceil()
        if case["op"] == "diff_train":
            leaves = ["q", "k", "v", "lam"]
            s["grads"] = (normal(B, H, Lq, Dv),)
    else:
        T, C = case["T"], case["C"]
        shape = {"channel": (C,), "batch": (B, 1, C), "token": (B, T, C)}
        s["x"], s["y"] = normal(B, T, C) if case["stream"] else None, normal(B, T, C)
        s["gate"] = normal(*shape[case["gate"]]) if case["gate"] != "none" else None
        s["weight"] = (1.0 + 0.2 * normal(*shape[case["weight"]])).to(dtype) if case["weight"] != "none" else None
        s["bias"] = 0.2 * normal(*shape[case["bias"]]) if case["bias"] != "none" else None
        s["post_weight"] = (1.0 + 0.2 * normal(C)).to(dtype) if case["post"] != "none" else None
        if case["op"] == "norm_train":
            leaves = [n for n in ("x", "y", "gate", "weight", "bias", "post_weight") if s[n] is not None]
            s["grads"] = (normal(B, T, C), normal(B, T, C)) if case["norm"] != "none" else (normal(B, T, C),)
    for name in leaves:
        s[name].requires_grad_(True)
    s["leaves"] = leaves
    return s


# ---- the plain forms --------------------------------------------------------------------------------------------------------
def _plain_turn(x, cos, sin, interleaved, sign):
    """Every pair of a head's turned part by its angle; cos, sin [.., 1, L, pairs]."""
    n = 2 * cos.shape[-1]
    x = x.detach().float()
    part = x[..., :n]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., : n // 2], part[..., n // 2:])
    c, d = a * cos - sign * b * sin, sign * a * sin + b * cos
    turned = torch.stack((c, d), -1).flatten(-2) if interleaved else torch.cat((c, d), -1)
    return torch.cat((turned, x[..., n:]), -1)


def _plain_rotary(s):
    case, dtype = s["case"], _TYPES[s["case"]["dtype"]]
    at = s["positions"] if s["positions"] is not None else torch.arange(case["L"], device="cuda")[None] + s["offset"]
    angles = at.double()[:, None, :, None] * s["frequencies"]
    cos, sin = (torch.cos(angles) * s["scale"]).float(), (torch.sin(angles) * s["scale"]).float()
    out = [_plain_turn(s[n], cos, sin, case["interleaved"], 1.0).to(dtype) for n in ("q", "k")]
    if case["op"] == "rotary_train":
        out += [_plain_turn(g, cos, sin, case["interleaved"], -1.0).to(dtype) for g in s["grads"]]
    return out


def _plain_diff(s):
    case, dtype = s["case"], _TYPES[s["case"]["dtype"]]
    B, H, Hkv, Lq, Lk, D, Dv = (case[n] for n in ("B", "H", "Hkv", "Lq", "Lk", "D", "Dv"))
    G, scale = H // Hkv, D ** -0.5
    # [map, B, Hkv, G * Lq or Lk, D]
    q = s["q"].detach().float().view(B, Hkv, G, 2, Lq, D).permute(3, 0, 1, 2, 4, 5).reshape(2, B, Hkv, G * Lq, D)
    k = s["k"].detach().float().view(B, Hkv, 2, Lk, D).permute(2, 0, 1, 3, 4).contiguous()
    v, lam = s["v"].detach().float(), s["lam"].detach().float()
    dropped = torch.zeros(B, 1, 1, Lq, Lk, dtype=torch.bool, device="cuda")
    if s["mask"] is not None:
        dropped = dropped | ~s["mask"][:, None, None, None, :]
    if case["causal"]:
        dropped = dropped | (torch.arange(Lk, device="cuda") > torch.arange(Lq, device="cuda")[:, None] + (Lk - Lq))
    maps = []
    for i in range(2):
        x = torch.matmul(q[i] * scale, k[i].transpose(2, 3).contiguous()).view(B, Hkv, G, Lq, Lk).masked_fill_(dropped, -math.inf)
        x = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e30))
        total = x.sum(-1, keepdim=True)
        maps.append((x / torch.where(total == 0, 1.0, total)).view(B, Hkv, G * Lq, Lk))
    each = lam.view(Hkv, G, 1).expand(Hkv, G, Lq).reshape(Hkv, G * Lq, 1)
    first, second = torch.matmul(maps[0], v), torch.matmul(maps[1], v)
    out = (first - each * second).view(B, H, Lq, Dv).to(dtype)
    if case["op"] == "diff":
        return out
    g = s["grads"][0].float().view(B, Hkv, G * Lq, Dv)
    dv = torch.matmul((maps[0] - each * maps[1]).transpose(2, 3).contiguous(), g)
    dp = torch.matmul(g, v.transpose(2, 3).contiguous())
    dq, dk = [], []
    for i, (o, weight) in enumerate(((first, 1.0), (second, -each))):
        ds = weight * maps[i] * (dp - (g * o).sum(-1, keepdim=True)) * scale
        dq.append(torch.matmul(ds, k[i]).view(B, Hkv, G, Lq, D))
        dk.append(torch.matmul(ds.transpose(2, 3).contiguous(), q[i]))
    dlam = -(g * second).view(B, H, Lq * Dv).sum((0, 2), dtype=torch.float64)
    return [out, torch.stack(dq, 3).view(B, 2 * H, Lq, D).to(dtype), torch.stack(dk, 2).view(B, 2 * Hkv, Lk, D).to(dtype), dv.to(dtype), dlam.to(dtype)]


def _plain_standard(x, kind, eps):
    """The normalised rows and 1 / their root."""
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    root = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
    return x * root, root


def _plain_back(g, normed, root, kind):
    g = g - normed * (g * normed).mean(-1, keepdim=True)
    if kind == "layer":
        g = g - g.mean(-1, keepdim=True)
    return g * root


def _plain_share(g, like):
    """The gradient of what was broadcast: sums over the tokens it was for."""
    if like.dim() == 1:
        return g.sum((0, 1), dtype=torch.float64)
    return g.sum(1, keepdim=True, dtype=torch.float64) if like.shape[1] == 1 and g.shape[1] != 1 else g


def _plain_norm(s):
    case, dtype = s["case"], _TYPES[s["case"]["dtype"]]
    f = {n: s[n].detach().float() if s[n] is not None else None for n in ("x", "y", "gate", "weight", "bias", "post_weight")}
    z, post_root = _plain_standard(f["y"], case["post"], 1e-5) if case["post"] != "none" else (f["y"], None)
    zw = z if f["post_weight"] is None else z * f["post_weight"]
    gate = f["gate"]
    if gate is not None and case["activation"] == "sigmoid":
        gate = 1.0 / (1.0 + torch.exp(-gate))
    r = zw if gate is None else gate * zw
    if f["x"] is not None:
        r = r + case["scale"] * f["x"]
    out = [r.to(dtype)]
    if case["norm"] != "none":
        n, root = _plain_standard(r, case["norm"], 1e-5)
        h = n if f["weight"] is None else n * f["weight"]
        out.append((h if f["bias"] is None else h + f["bias"]).to(dtype))
    if case["op"] == "norm":
        return out
    grads = {}
    dr = s["grads"][0].float()
    if case["norm"] != "none":
        dh = s["grads"][1].float()
        grads["bias"], grads["weight"] = dh, dh * n
        dr = dr + _plain_back(dh if f["weight"] is None else dh * f["weight"], n, root, case["norm"])
    grads["x"] = case["scale"] * dr
    grads["gate"] = dr * zw * (gate * (1.0 - gate) if case["activation"] == "sigmoid" else 1.0)
    dz = dr if gate is None else dr * gate
    grads["post_weight"] = dz * z
    if case["post"] != "none":
        dz = _plain_back(dz * f["post_weight"], z, post_root, case["post"])
    grads["y"] = dz
    return out + [_plain_share(grads[n], s[n]).to(dtype) for n in s["leaves"]]


# ---- through the entry points -----------------------------------------------------------------------------------------------
def _run_own(s):
    import af3_kernels_amd as af3
    case = s["case"]
    if case["op"] in ("rotary", "rotary_train"):
        out = af3.rotary_embedding(s["q"], s["k"], s["frequencies"], s["positions"], offset=s["offset"], interleaved=case["interleaved"], scale=s["scale"])
    elif case["op"] in ("diff", "diff_train"):
        out = (af3.differential_attention(s["q"], s["k"], s["v"], s["lam"], s["mask"], causal=case["causal"], q_offset=case["Lk"] - case["Lq"]),)
    else:
        out = af3.residual_norm(s["x"], s["y"], s["weight"], s["bias"], s["gate"], s["post_weight"], norm=case["norm"], post_norm=case["post"],
                                gate_activation=case["activation"], residual_scale=case["scale"])
        if case["norm"] == "none":
            out = out[:1]
    if not s["leaves"]:
        return list(out) if len(out) > 1 else out[0] if case["op"] == "diff" else list(out)
    return [o.detach() for o in out] + list(torch.autograd.grad(out, [s[n] for n in s["leaves"]], s["grads"]))


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    return _plain_rotary(state) if op.startswith("rotary") else _plain_diff(state) if op.startswith("diff") else _plain_norm(state)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    train = case["op"].endswith("_train")
    B = case["B"]
    if case["op"] in ("rotary", "rotary_train"):
        n = B * (case["H"] + case["Hkv"]) * case["L"] * case["D"]
        places = 8 * B * case["L"] if case["positions"] == "requests" else 0
        return {"bytes": size * n * (4 if train else 2) + places, "flops": 3 * n * (2 if train else 1)}
    if case["op"] in ("diff", "diff_train"):
        H, Hkv, Lq, Lk, D, Dv = (case[n] for n in ("H", "Hkv", "Lq", "Lk", "D", "Dv"))
        live = {"none": 1.0, "random": 0.92, "ragged": 0.75}[case["mask"]]
        queries, states, result = 2 * B * H * Lq * D, B * Hkv * Lk * (2 * D + Dv), B * H * Lq * Dv
        nbytes = size * (queries + states * live + result) + (B * Lk if case["mask"] != "none" else 0)
        pairs = B * H * (Lq * (Lk - Lq) + Lq * (Lq + 1) // 2 if case["causal"] else Lq * Lk) * live
        flops = pairs * (4 * D + 4 * Dv)
        if train:
            nbytes += size * (queries + states + result)
            flops += pairs * (12 * D + 4 * Dv)   # S and the output again are not counted: 2 maps of S, dQ and dK, one dP, one dV
        return {"bytes": int(nbytes), "flops": int(flops)}
    rows = {"none": 0, "channel": 1, "batch": B, "token": B * case["T"]}
    tokens, C = B * case["T"], case["C"]
    streams = 2 if case["stream"] else 1
    params = sum(rows[case[n]] for n in ("gate", "weight", "bias")) + (case["post"] != "none")
    results = 2 if case["norm"] != "none" else 1
    moved = streams * tokens + params + results * tokens
    if train:
        moved += (streams + results) * tokens + params
    return {"bytes": size * C * moved, "flops": tokens * C * (30 if train else 12)}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------------
def _exact_rotary(s):
    case, f64 = s["case"], torch.float64
    L, n = case["L"], case["rotary"]
    places = (s["positions"] if s["positions"] is not None else (torch.arange(L, device="cuda") + s["offset"]).expand(case["B"], L)).to(f64)
    turn = torch.polar(torch.full((), s["scale"], dtype=f64, device="cuda").expand(case["B"], L, n // 2), places[..., None] * s["frequencies"])

    def turned(x, by):
        x = x.detach().to(f64)
        out = x.clone()
        for h in range(x.shape[1]):
            if case["interleaved"]:
                w = torch.complex(x[:, h, :, 0:n:2], x[:, h, :, 1:n:2]) * by
                out[:, h, :, 0:n:2], out[:, h, :, 1:n:2] = w.real, w.imag
            else:
                w = torch.complex(x[:, h, :, : n // 2], x[:, h, :, n // 2: n]) * by
                out[:, h, :, : n // 2], out[:, h, :, n // 2: n] = w.real, w.imag
        return out

    out = [turned(s["q"], turn), turned(s["k"], turn)]
    return out + [turned(g, turn.conj()) for g in s["grads"]] if s["leaves"] else out


def _exact_diff(s):
    case, f64 = s["case"], torch.float64
    B, H, Hkv, Lq, Lk, D, Dv = (case[n] for n in ("B", "H", "Hkv", "Lq", "Lk", "D", "Dv"))
    wide = {n: s[n].detach().to(f64) for n in ("q", "k", "v", "lam")}
    out = torch.empty(B, H, Lq, Dv, dtype=f64, device="cuda")
    train = bool(s["leaves"])
    grads = {n: torch.zeros_like(t) for n, t in wide.items()} if train else {}
    hidden = torch.ones(Lq, Lk, dtype=torch.bool, device="cuda").triu(Lk - Lq + 1) if case["causal"] else None
    for b in range(B):
        for h in range(H):
            kv = h // (H // Hkv)
            live = s["mask"][b].nonzero()[:, 0] if s["mask"] is not None else torch.arange(Lk, device="cuda")
            v, lam = wide["v"][b, kv][live], wide["lam"][h]
            maps = []
            for i in range(2):
                x = wide["q"][b, 2 * h + i] @ wide["k"][b, 2 * kv + i][live].t() / math.sqrt(D)
                if hidden is not None:
                    x[hidden[:, live]] = -math.inf
                maps.append(torch.nan_to_num(torch.softmax(x, -1), nan=0.0))   # (a query without a key: zeros)
            weights = maps[0] - lam * maps[1]
            out[b, h] = weights @ v
            if not train:
                continue
            g = s["grads"][0][b, h].to(f64)
            grads["v"][b, kv].index_add_(0, live, weights.t() @ g)
            dw = g @ v.t()
            grads["lam"][h] -= (dw * maps[1]).sum()
            for i, dp in enumerate((dw, -lam * dw)):
                ds = maps[i] * (dp - (maps[i] * dp).sum(-1, keepdim=True)) / math.sqrt(D)
                grads["q"][b, 2 * h + i] = ds @ wide["k"][b, 2 * kv + i][live]
                grads["k"][b, 2 * kv + i].index_add_(0, live, ds.t() @ wide["q"][b, 2 * h + i])
    return [out] + [grads[n] for n in s["leaves"]] if train else out


def _exact_norm(s):
    case, f64 = s["case"], torch.float64
    t = {n: s[n].detach().to(f64).requires_grad_(True) for n in ("x", "y", "gate", "weight", "bias", "post_weight") if s[n] is not None}

    def norm(a, kind):
        centre = a.mean(-1, keepdim=True) if kind == "layer" else 0.0
        return (a - centre) / torch.sqrt(((a - centre) ** 2).mean(-1, keepdim=True) + 1e-5)

    branch = t["y"] if case["post"] == "none" else norm(t["y"], case["post"]) * t["post_weight"]
    if "gate" in t:
        branch = branch * (torch.sigmoid(t["gate"]) if case["activation"] == "sigmoid" else t["gate"])
    r = branch + case["scale"] * t["x"] if "x" in t else branch
    out = [r]
    if case["norm"] != "none":
        out.append(norm(r, case["norm"]) * t.get("weight", 1.0) + t.get("bias", 0.0))
    grads = torch.autograd.grad(out, [t[n] for n in s["leaves"]], [g.to(f64) for g in s["grads"]]) if s["leaves"] else ()
    return [o.detach() for o in out] + list(grads)


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_rotary(s) if case["op"].startswith("rotary") else _exact_diff(s) if case["op"].startswith("diff") else _exact_norm(s)
