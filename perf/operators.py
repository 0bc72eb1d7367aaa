"""What the attention to states of another length and the learned relative position bias are judged by: calls of encoders,
decoders and their training, from one token to long sequences, each in a plain form and through this package's entry points.

A case is a dict of plain values.  `op` says what one pass is:

    attend       cross_attention forward: q [B, H, Lq, D] to k, v [B, Hkv, Lk, D]
    train        the same with the gradients of q, k, v and, where there is one, of the bias; "bias": "table" makes that bias with
                 relative_position_bias within the pass and takes the gradient through to the table
    bias         relative_position_bias forward, [H, Lq, Lk]
    bias_train   the same with the table's gradient

Masks over the keys: "ragged" rows end anywhere in their second half (padding to the longest), "random" drops 8 % of the keys, "empty"
is ragged with one batch row that keeps no key at all, "none" is no mask.  Positions: "tokens" are 0, 1, 2, ... (a decoder's
queries begin at an offset), "residues" are numbers of residues with gaps between chains.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _attend(name, B, H, Hkv, Lq, Lk, D, dtype="bf16", mask="ragged", bias="none"):
    return {"name": name, "op": "attend", "B": B, "H": H, "Hkv": Hkv, "Lq": Lq, "Lk": Lk, "D": D, "dtype": dtype, "mask": mask, "bias": bias}


def _train(name, *sizes, **kinds):
    return {**_attend(name, *sizes, **kinds), "op": "train"}


def _bias(name, op, H, Lq, Lk, buckets, scheme="log", both=True, distance=128, positions="tokens", offset=0, dtype="bf16"):
    return {"name": name, "op": op, "H": H, "Lq": Lq, "Lk": Lk, "buckets": buckets, "scheme": scheme, "both": both, "distance": distance,
            "positions": positions, "offset": offset, "dtype": dtype}


def listed():
    return [
        # one query over the conditioning of a short peptide: launches and host time are all there is to it
        _attend("token_k37", 1, 4, 4, 1, 37, 32),
        # a decoder's step over the encoder's states of a batch of requests of many lengths
        _attend("token_b32_k1491", 32, 16, 16, 1, 1491, 64),
        # a short prompt over a long document whose key heads are shared
        _attend("prompt_n37_k8192", 1, 16, 4, 37, 8192, 128, mask="none"),
        # tokens of a middling crop over atoms, an odd number of them, with a pair bias
        _attend("cross_n384_k1491", 4, 16, 16, 384, 1491, 48, mask="random", bias="given"),
        # the longest of them: shared key heads, long states
        _attend("cross_n1491_k4096", 8, 16, 4, 1491, 4096, 128),
        # in full precision
        _attend("cross_fp32_n200_k768", 4, 8, 8, 200, 768, 32, dtype="fp32", bias="given"),
        # a training step of a decoder's layer
        _train("train_n768_k1024", 8, 16, 16, 768, 1024, 64),
        # a training step of an encoder's layer, whose bias is learned by buckets
        _train("train_table_n512", 8, 12, 12, 512, 512, 64, bias="table"),
        # a training step in full precision, with the gradient of a pair bias
        _train("train_fp32_n259_k384", 2, 8, 8, 259, 384, 32, dtype="fp32", mask="random", bias="given"),
        # the bias of one decoded token: far positions back, none ahead
        _bias("bias_token_k701", "bias", 12, 1, 701, 32, both=False, offset=700),
        # the bias of a long sequence
        _bias("bias_n4096", "bias", 16, 4096, 4096, 32),
        # residue offsets of a training crop, limited to 32 either way, with the table's gradient
        _bias("bias_train_residues_n768", "bias_train", 16, 768, 768, 65, scheme="clip", distance=32, positions="residues", dtype="fp32"),
    ]


def _log(rng, low, high):
    """A whole number between low and high, spread over its logarithm; odd ones among them, and multiples of 8 as often as not."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.4:
        n = (n + 7) // 8 * 8
    return max(low, min(high, n))


def draw(rng):
    op = rng.choice(["attend", "attend", "token", "train", "train", "bias", "bias_train"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    if op in ("bias", "bias_train"):
        scheme = rng.choice(["log", "clip"])
        both = rng.random() < 0.6
        top = 4096 if op == "bias" else 2048
        Lq, Lk = (1, _log(rng, 2, 8192)) if op == "bias" and rng.random() < 0.3 else (_log(rng, 2, top), _log(rng, 2, top))
        distance = rng.choice([32, 64, 128, 256])
        buckets = rng.choice([16, 32, 64] if distance > 32 else [16, 32]) if scheme == "log" else 2 * distance + 1 if both else distance + 1
        positions = rng.choice(["tokens", "residues"]) if Lq > 1 else "tokens"
        case = _bias("", op, rng.choice([4, 8, 12, 16]), Lq, Lk, buckets, scheme, both, distance, positions, rng.randint(0, Lk) if positions == "tokens" else 0, dtype)
    else:
        Hkv, G = rng.choice([2, 4, 8]), rng.choice([1, 1, 2, 4])
        mask = rng.choice(["none", "ragged", "random", "empty"])
        if op == "token":
            sizes = (_log(rng, 1, 48), Hkv * G, Hkv, rng.choice([1, 1, 2, 5]), _log(rng, 16, 8192))
        elif op == "attend":
            sizes = (rng.randint(1, 8), Hkv * G, Hkv, _log(rng, 16, 1491), _log(rng, 16, 4096))
        else:
            sizes = (rng.randint(1, 6), Hkv * G, Hkv, _log(rng, 16, 768), _log(rng, 16, 1024))
        D = rng.choice([24, 32, 48, 64, 80, 128])
        bias = rng.choice(["none", "given"] if op != "train" else ["none", "given", "table"])
        case = _attend("", *sizes, D, dtype=dtype, mask=mask, bias=bias)
        case["op"] = "train" if op == "train" else "attend"
    case.pop("name")
    return case


# ---- inputs ---------------------------------------------------------------------------------------------------------------
_TABLE = {"buckets": 32, "scheme": "log", "both": True, "distance": 128}   # of a training step with a learned bias


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    H, Lq, Lk = case["H"], case["Lq"], case["Lk"]
    s = {"case": case}
    if case["op"] in ("bias", "bias_train"):
        s["table"] = normal(case["buckets"], H)
        if case["positions"] == "residues":
            def numbers(n):   # mostly the next number, now and then a gap
                step = torch.ones(n, dtype=torch.int64, device="cuda")
                return torch.cumsum(step + 40 * (torch.rand(n, generator=gen, device="cuda") < 0.01), 0)
            s["q_positions"] = numbers(Lq)
            s["k_positions"] = s["q_positions"] if Lk == Lq else numbers(Lk)
        if case["op"] == "bias_train":
            s["table"].requires_grad_(True)
            s["grad"] = normal(H, Lq, Lk)
        return s
    B, Hkv, D = case["B"], case["Hkv"], case["D"]
    s["q"], s["k"], s["v"] = normal(B, H, Lq, D), normal(B, Hkv, Lk, D), normal(B, Hkv, Lk, D)
    if case["mask"] == "random":
        s["mask"] = torch.rand(B, Lk, generator=gen, device="cuda") < 0.92
        s["mask"][:, 0] = True
    elif case["mask"] != "none":
        lengths = (Lk * (0.5 + 0.5 * torch.rand(B, 1, generator=gen, device="cuda"))).ceil()
        s["mask"] = torch.arange(Lk, device="cuda") < lengths
        if case["mask"] == "empty":
            s["mask"][B // 2] = False
    else:
        s["mask"] = None
    s["bias"] = normal(H, Lq, Lk) if case["bias"] == "given" else None
    s["table"] = normal(_TABLE["buckets"], H) if case["bias"] == "table" else None
    if case["op"] == "train":
        s["grad"] = normal(B, H, Lq, D)
        for name in ("q", "k", "v", "bias", "table"):
            if s[name] is not None:
                s[name].requires_grad_(True)
    return s


# ---- the plain forms --------------------------------------------------------------------------------------------------------
def _borders(buckets, scheme, both, distance):
    """The smallest distance of each bucket but the first on one side."""
    if scheme == "clip":
        return list(range(1, distance + 1))
    n = buckets // 2 if both else buckets
    near = n // 2
    far = n - near
    out = list(range(1, near + 1))
    for i in range(1, far):
        # the smallest d with far * log(d / near) / log(distance / near) >= i, in whole numbers: (d / near)^far >= (distance / near)^i
        d = near
        while d ** far < distance ** i * near ** (far - i):
            d += 1
        out.append(d)
    return out


def _buckets(rel, p):
    """Bucket of key position minus query position (whole numbers)."""
    side = torch.tensor(_borders(p["buckets"], p["scheme"], p["both"], p["distance"]), device=rel.device)
    if p["scheme"] == "clip":
        return (-rel).clamp(-p["distance"] if p["both"] else 0, p["distance"]) + (p["distance"] if p["both"] else 0)
    d = rel.abs() if p["both"] else (-rel).clamp(min=0)
    b = torch.bucketize(d, side, right=True)
    return b + (rel > 0) * (p["buckets"] // 2) if p["both"] else b


def _positions(s):
    case = s["case"]
    if s.get("q_positions") is not None:
        return s["q_positions"], s["k_positions"]
    dev = s["table"].device
    return torch.arange(case["Lq"], device=dev) + case.get("offset", 0), torch.arange(case["Lk"], device=dev)


def _plain_bias(s, p):
    q, k = _positions(s)
    b = _buckets(k[None, :] - q[:, None], p)
    return b, s["table"].detach().float()[b].permute(2, 0, 1)


def _plain_table_gradient(b, g, n):
    """Sums of g [H, Lq, Lk] by bucket, in 64 bits: a bucket holds millions of terms."""
    return torch.stack([torch.where(b == i, g, 0.0).sum((1, 2), dtype=torch.float64) for i in range(n)])


def _plain_attention(s, bias, gradients):
    """softmax(q.k^T D^-1/2 + bias) v over the live keys, in 32 bits, and the gradients of q, k, v and the bias."""
    q, k, v = (s[n].detach().float() for n in ("q", "k", "v"))
    B, H, Lq, D = q.shape
    Hkv, Lk = k.shape[1:3]
    G = H // Hkv
    scale = D ** -0.5
    logits = torch.matmul(q.reshape(B, Hkv, G * Lq, D) * scale, k.transpose(2, 3).contiguous()).view(B, H, Lq, Lk)
    if bias is not None:
        logits += bias[None]
    if s["mask"] is not None:
        dropped = ~s["mask"][:, None, None, :]
        # (a batch row without a live key: every key alike)
        logits = logits.masked_fill_(dropped, -1e30)
    logits = torch.exp(logits - logits.amax(-1, keepdim=True))
    p = logits / logits.sum(-1, keepdim=True)
    pg = p.view(B, Hkv, G * Lq, Lk)
    out = torch.matmul(pg, v)
    if not gradients:
        return out.view(B, H, Lq, D), None
    g = s["grad"].float().view(B, Hkv, G * Lq, D)
    dv = torch.matmul(pg.transpose(2, 3).contiguous(), g)
    ds = torch.matmul(g, v.transpose(2, 3).contiguous())
    ds = pg * (ds - (g * out).sum(-1, keepdim=True))
    if s["mask"] is not None:
        ds = ds.view(B, H, Lq, Lk).masked_fill_(dropped, 0.0).view(B, Hkv, G * Lq, Lk)
    dq = torch.matmul(ds, k) * scale
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q.view(B, Hkv, G * Lq, D)) * scale
    dbias = ds.view(B, H, Lq, Lk).sum(0) if bias is not None else None
    return out.view(B, H, Lq, D), (dq.view(B, H, Lq, D), dk, dv, dbias)


def _run_plain(s):
    case = s["case"]
    dtype = _TYPES[case["dtype"]]
    if case["op"] in ("bias", "bias_train"):
        b, bias = _plain_bias(s, case)
        bias = bias.to(dtype, memory_format=torch.contiguous_format)
        if case["op"] == "bias":
            return bias
        return bias, _plain_table_gradient(b, s["grad"], case["buckets"]).to(dtype)
    bias = s["bias"].detach().float() if s["bias"] is not None else None
    if s["table"] is not None:
        b, bias = _plain_bias(s, _TABLE)
    out, grads = _plain_attention(s, bias, case["op"] == "train")
    if grads is None:
        return out.to(dtype)
    dq, dk, dv, dbias = grads
    result = [out.to(dtype), dq.to(dtype), dk.to(dtype), dv.to(dtype)]
    if s["bias"] is not None:
        result.append(dbias.to(dtype))
    if s["table"] is not None:
        result.append(_plain_table_gradient(b, dbias, _TABLE["buckets"]).to(dtype))
    return result


# ---- through the entry points -----------------------------------------------------------------------------------------------
def _run_own(s):
    import af3_kernels_amd as af3
    case = s["case"]

    def position_bias(p):
        return af3.relative_position_bias(s["table"], case["Lq"], case["Lk"], scheme=p["scheme"], bidirectional=p["both"], max_distance=p["distance"],
                                          q_positions=s.get("q_positions"), k_positions=s.get("k_positions"), q_offset=case.get("offset", 0))

    if case["op"] in ("bias", "bias_train"):
        bias = position_bias(case)
        if case["op"] == "bias":
            return bias
        return bias.detach(), torch.autograd.grad(bias, s["table"], s["grad"])[0]
    bias = position_bias(_TABLE) if s["table"] is not None else s["bias"]
    out = af3.cross_attention(s["q"], s["k"], s["v"], s["mask"], bias)
    if case["op"] == "attend":
        return out
    leaves = [t for t in (s["q"], s["k"], s["v"], s["bias"], s["table"]) if t is not None]
    return [out.detach(), *torch.autograd.grad(out, leaves, s["grad"])]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    H, Lq, Lk = case["H"], case["Lq"], case["Lk"]
    if case["op"] in ("bias", "bias_train"):
        train = case["op"] == "bias_train"
        places = 8 * (Lq + Lk) if case["positions"] == "residues" else 0
        return {"bytes": size * (H * Lq * Lk * (2 if train else 1) + case["buckets"] * H * (2 if train else 1)) + places, "flops": H * Lq * Lk if train else 0}
    B, Hkv, D = case["B"], case["Hkv"], case["D"]
    live = {"none": 1.0, "random": 0.92}.get(case["mask"], 0.75)
    train = case["op"] == "train"
    rows, states = B * H * Lq * D, B * Hkv * Lk * D * live
    # forward: q, k, v in and the result out; training: the result's gradient in, three gradients out (those of dropped keys too, zeros)
    nbytes = size * ((4 if train else 2) * rows + 2 * states + (2 * B * Hkv * Lk * D if train else 0)) + (B * Lk if case["mask"] != "none" else 0)
    if case["bias"] == "given":
        nbytes += size * H * Lq * Lk * (2 if train else 1)
    return {"bytes": int(nbytes), "flops": int((14 if train else 4) * rows * Lk * live)}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------------
def _exact_bucket_table(p, reach):
    """bucket of every offset -reach .. reach of a key from its query, one by one in Python."""
    out = []
    for rel in range(-reach, reach + 1):
        if p["scheme"] == "clip":
            r = p["distance"]
            out.append(min(max(-rel, -r), r) + r if p["both"] else min(max(-rel, 0), r))
            continue
        n = p["buckets"] // 2 if p["both"] else p["buckets"]
        first = n if p["both"] and rel > 0 else 0
        d = abs(rel) if p["both"] else max(-rel, 0)
        near = n // 2
        if d < near:
            out.append(first + d)
            continue
        far = n - near
        i = int(far * math.log(d / near) / math.log(p["distance"] / near))
        # the logarithm is off by a rounding at the borders: i is the largest whole number with (distance / near)^i <= (d / near)^far
        while i < far and p["distance"] ** (i + 1) * near ** (far - i - 1) <= d ** far:
            i += 1
        while 0 < i <= far and p["distance"] ** i * near ** (far - i) > d ** far:
            i -= 1
        out.append(first + min(near + i, n - 1))
    return out


def _exact_buckets(s, p):
    q, k = _positions(s)
    reach = p["distance"] + 1
    table = torch.tensor(_exact_bucket_table(p, reach), device=q.device)
    return table[(k[None, :] - q[:, None]).clamp(-reach, reach) + reach]


def _exact_sums(b, g, n):
    flat = b.reshape(-1)
    return torch.stack([torch.zeros(n, dtype=torch.float64, device=g.device).index_add_(0, flat, g[h].reshape(-1).double()) for h in range(g.shape[0])], 1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("bias", "bias_train"):
        b = _exact_buckets(s, case)
        bias = torch.stack([s["table"].detach()[:, h][b] for h in range(case["H"])]).double()
        return bias if case["op"] == "bias" else (bias, _exact_sums(b, s["grad"], case["buckets"]))
    f64 = torch.float64
    train = case["op"] == "train"
    B, H, Lq, D = s["q"].shape
    G = H // case["Hkv"]
    bias = s["bias"].detach().to(f64) if s["bias"] is not None else None
    if s["table"] is not None:
        b = _exact_buckets(s, _TABLE)
        bias = torch.stack([s["table"].detach()[:, h][b] for h in range(H)]).to(f64)
    out = torch.empty(B, H, Lq, D, dtype=f64, device="cuda")
    if train:
        dq, dk, dv = torch.zeros_like(out), torch.zeros(s["k"].shape, dtype=f64, device="cuda"), torch.zeros(s["v"].shape, dtype=f64, device="cuda")
        dbias = torch.zeros_like(bias) if bias is not None else None
    for i in range(B):
        live = s["mask"][i].nonzero()[:, 0] if s["mask"] is not None else torch.arange(case["Lk"], device="cuda")
        for h in range(H):
            q, k, v = s["q"][i, h].detach().to(f64), s["k"][i, h // G].detach().to(f64), s["v"][i, h // G].detach().to(f64)
            if len(live) == 0:   # no live key: the mean of the values
                out[i, h] = v.mean(0)
                if train:
                    dv[i, h // G] += s["grad"][i, h].to(f64).sum(0) / case["Lk"]
                continue
            k, v = k[live], v[live]
            x = q @ k.t() / math.sqrt(D)
            if bias is not None:
                x = x + bias[h][:, live]
            p = torch.softmax(x, -1)
            o = p @ v
            out[i, h] = o
            if train:
                g = s["grad"][i, h].to(f64)
                dp = g @ v.t()
                ds = p * (dp - (p * dp).sum(-1, keepdim=True))
                dq[i, h] = ds @ k / math.sqrt(D)
                dk[i, h // G].index_add_(0, live, ds.t() @ q / math.sqrt(D))
                dv[i, h // G].index_add_(0, live, p.t() @ g)
                if bias is not None:
                    dbias[h].index_add_(1, live, ds)
    if not train:
        return out
    result = [out, dq, dk, dv]
    if s["bias"] is not None:
        result.append(dbias)
    if s["table"] is not None:
        result.append(_exact_sums(b, dbias, _TABLE["buckets"]))
    return result
