"""rotary_embedding, differential_attention and residual_norm on the GPU against their formulas in 64 bits on the CPU, on the numbers the device saw.

Tolerances are bounds per element, worked out from the roundings before anything ran: sums of n terms in 32 bits are off by at most n 2^-24 of the sum of the terms'
magnitudes, a rounding to bf16 by 2^-8 of the value.  Rotary: angles in 64 bits, cosine and sine and the turn in 32.  Attention (`diff_formula`): P in 16 bits of significand or
as fp16 in the forward pass, dS and P1 - lam P2 rounded to bf16 in front of their products, results once.  Norms (`Num`): every operation's rounding carried along.
"""
import gc
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
E32 = 2.0 ** -24
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
TYPES = pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
HOSTS = pytest.mark.parametrize("native", [True, False], ids=["native", "python"])
half_step = lambda dtype: torch.finfo(dtype).eps / 2


class _NoNativeHost:
    def __getattr__(self, name):
        return lambda *args: None


@pytest.fixture(scope="module")
def af3():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    import af3_kernels_amd
    af3_kernels_amd._lib.load()
    return af3_kernels_amd


@pytest.fixture
def host(monkeypatch):
    """host(False): the calls that follow are prepared in Python."""
    from af3_kernels_amd import layers

    def choose(native):
        if not native:
            monkeypatch.setattr(layers, "_host", _NoNativeHost())
    return choose


def wide(t):
    return None if t is None else t.detach().double().cpu()


def within(name, got, value, bound):
    got = got.detach().double().cpu()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    assert torch.isfinite(got).all(), f"{name}: not finite"
    excess = ((got - value).abs() - bound - 1e-30)
    assert excess.numel() == 0 or excess.max().item() <= 0, f"{name}: {excess.max().item()} beyond the bound, error {(got - value).abs().max().item()}"


# ---- rotary positions ---------------------------------------------------------------------------------------------------------
def turned(x, frequencies, places, interleaved, scale, inverse=False):
    """The formula and its bound: |error| <= scale (|a| + |b|) 2^-21 (cosine and sine to 2^-22 with the scale, two products and their sum), one rounding."""
    x = wide(x)
    n = 2 * len(frequencies)
    angle = places.double().view(-1, 1, x.shape[2], 1) * frequencies.double().cpu() * (-1 if inverse else 1)
    a, b = (x[..., 0:n:2], x[..., 1:n:2]) if interleaved else (x[..., : n // 2], x[..., n // 2: n])
    c, d = scale * (a * angle.cos() - b * angle.sin()), scale * (a * angle.sin() + b * angle.cos())
    err = abs(scale) * (a.abs() + b.abs()) * 2.0 ** -21
    put = lambda c, d: torch.cat((torch.stack((c, d), -1).flatten(-2) if interleaved else torch.cat((c, d), -1), x[..., n:]), -1)
    return put(c, d), torch.cat((put(err, err)[..., :n], torch.zeros_like(x[..., n:])), -1)


def check_turned(name, got, x, frequencies, places, interleaved, scale, inverse=False):
    value, bound = turned(x, frequencies, places, interleaved, scale, inverse)
    n = 2 * len(frequencies)
    within(name, got, value, bound + half_step(got.dtype) * (value.abs() + bound))
    assert torch.equal(got[..., n:].cpu(), x[..., n:].cpu()), "the elements behind the turned ones"


@TYPES
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "interleaved"])
@pytest.mark.parametrize("B,H,Hkv,L,D,n", [(1, 1, 0, 1, 2, 2), (2, 4, 1, 1, 64, 64), (3, 5, 2, 37, 128, 64), (1, 3, 3, 130, 80, 80), (2, 2, 1, 9, 30, 10), (1, 8, 8, 257, 24, 24),
                                           (2, 3, 1, 5, 1024, 1024), (1, 2, 2, 11, 7, 6), (4, 16, 4, 70, 256, 128), (1, 1, 1, 3, 1000, 996)])
def test_rotary_and_gradients(af3, B, H, Hkv, L, D, n, interleaved, dtype):
    g = torch.Generator().manual_seed(B + L + D)
    q = torch.randn(B, H, L, D, generator=g).to(dtype).cuda().requires_grad_(True)
    k = torch.randn(B, Hkv, L, D, generator=g).to(dtype).cuda().requires_grad_(True) if Hkv else None
    f, scale = af3.rotary_frequencies(n, scaling="yarn", factor=4.0, original_length=2048, device="cuda") if n > 2 else (torch.tensor([0.37], dtype=F64, device="cuda"), -1.5)
    tensors = [q] + ([k] if Hkv else [])
    for positions, offset in ((None, 0), (None, 100003), (torch.randint(-5000, 200000, (L,), generator=g), 0), (torch.randint(0, 9000, (B, L), generator=g).int(), 0)):
        out = af3.rotary_embedding(q, k, f, None if positions is None else positions.cuda(), offset, interleaved, scale)
        assert (out[1] is None) == (k is None) and all(o.is_contiguous() for o in out if o is not None)
        places = torch.arange(L) + offset if positions is None else positions
        grads = [torch.randn(t.shape, generator=g).to(dtype).cuda() for t in tensors]
        back = torch.autograd.grad([o for o in out if o is not None], tensors, grads)
        for t, o, go, gi in zip(tensors, out, grads, back):
            check_turned("out", o, t, f, places, interleaved, scale)
            check_turned("gradient", gi, go, f, places, interleaved, scale, True)


@TYPES
def test_rotary_views_casts_and_lengths(af3, dtype):
    g = torch.Generator().manual_seed(5)
    B, H, Hkv, L, D = 2, 4, 2, 33, 64
    both = torch.randn(B, L, H + Hkv + 1, D + 1, generator=g).to(dtype).cuda()
    f, scale = af3.rotary_frequencies(D, device="cuda")
    views = (both.transpose(1, 2)[:, :H, :, :D], both.transpose(1, 2)[:, H:H + Hkv, :, 1:])       # (one element into a row: no 16-byte loads)
    repeated = (both.transpose(1, 2)[:1, :1, :, :D].expand(B, H, L, D), both.transpose(1, 2)[:, :Hkv, :1, :D].expand(B, Hkv, L, D))
    columns = (both[:, :, :H, :D].permute(0, 2, 3, 1).contiguous().transpose(2, 3), both[:, :, :Hkv, :D].transpose(1, 2))
    for q, k in (views, repeated, columns):
        for interleaved in (False, True):
            for x, o in zip((q, k), af3.rotary_embedding(q, k, f.float(), offset=7, interleaved=interleaved)):
                check_turned("view", o, x, f.float(), torch.arange(L) + 7, interleaved, 1.0)
    # positions that are strided, or one row for the batch; k of another type
    places = torch.randint(0, 500, (B, 2 * L), generator=g)
    q, k = views
    a = af3.rotary_embedding(q, k, f, places.cuda()[:, ::2])
    check_turned("strided", a[0], q, f, places[:, ::2], False, 1.0)
    b = af3.rotary_embedding(q, k, f, places.cuda()[:, :L][:1])
    check_turned("one row", b[1], k, f, places[0, :L], False, 1.0)
    other = F32 if dtype == BF16 else BF16
    assert torch.equal(af3.rotary_embedding(q, k.to(other), f)[1], af3.rotary_embedding(q, k.to(other).to(dtype), f)[1])
    # gradients that are views, and one of two results alone
    x, y = q.detach().clone().requires_grad_(True), k.detach().clone().requires_grad_(True)
    out = af3.rotary_embedding(x, y, f)
    check_turned("expanded gradient", torch.autograd.grad(out[0], x, torch.ones(1, 1, 1, 1, dtype=dtype, device="cuda").expand(out[0].shape), retain_graph=True)[0],
                 torch.ones(out[0].shape, dtype=dtype), f, torch.arange(L), False, 1.0, True)
    assert torch.autograd.grad(out[0].sum(), y, allow_unused=True)[0] is None
    # nothing to turn
    for shape in ((0, H, L, D), (B, 0, L, D), (B, H, 0, D)):
        e = torch.zeros(shape, dtype=dtype, device="cuda", requires_grad=True)
        o = af3.rotary_embedding(e, None, f)[0]
        assert o.shape == e.shape and torch.autograd.grad(o.sum(), e)[0].shape == e.shape
    o = af3.rotary_embedding(torch.zeros(B, 0, L, D, dtype=dtype, device="cuda"), k, f)
    assert o[0].shape == (B, 0, L, D)
    check_turned("k alone", o[1], k, f, torch.arange(L), False, 1.0)


def test_rotary_far_positions_and_rows(af3):
    """Angles of 2^40 turns are exact to 64 bits' last places; rows and heads more than 4 GB apart."""
    f = torch.tensor([1.0, 0.1, 1e-3, 1e-9], dtype=F64, device="cuda")
    x = torch.randn(1, 1, 3, 8, device="cuda")
    places = torch.tensor([(1 << 30) + 1, -(1 << 30), 12345678901])
    # (2^34 radians in 64 bits: 2^-19 radians where the product is rounded, in the formula as in the kernel, which may differ by that)
    value, bound = turned(x, f, places, False, 1.0)
    within("far", af3.rotary_embedding(x, None, f, places.cuda())[0], value, bound + 2.0 ** -18 * x.abs().sum().item())
    free = torch.cuda.mem_get_info()[0]
    if free > 12 << 30:
        base = torch.empty((4 << 30) // 2 + 4096, dtype=BF16, device="cuda")
        far = base.as_strided((2, 2, 2, 64), ((1 << 31), 64, 256, 1))
        far.copy_(torch.randn(2, 2, 2, 64))
        g = af3.rotary_frequencies(64, device="cuda")[0]
        check_turned("far rows", af3.rotary_embedding(far, None, g, offset=3)[0], far.contiguous(), g, torch.arange(2) + 3, False, 1.0)
        del base, far
        gc.collect()
        torch.cuda.empty_cache()


def test_rotary_refuses(af3):
    q = torch.zeros(2, 4, 3, 16, device="cuda")
    f = torch.zeros(8, dtype=F64, device="cuda")
    bad = [((q[0], None, f), "q must be"), ((q, q[:1], f), "q must be"), ((q.half(), None, f), "unsupported dtype"), ((q, None, f[:0]), "frequencies"), ((q, None, f.repeat(2)), "frequencies"),
           ((q, None, f.long()), "frequencies"), ((q, None, f.view(2, 4)), "frequencies"), ((q, None, f, torch.zeros(4, device="cuda", dtype=torch.int64)), "positions"),
           ((q, None, f, torch.zeros(3, device="cuda")), "positions"), ((q, None, f, torch.zeros(3, 3, device="cuda", dtype=torch.int64)), "positions"),
           ((q, None, f, None, (1 << 62) + 1), "2\\^62"), ((q, None, f, None, 0, False, math.inf), "scale"), ((q, None, f, None, 0, False, math.nan), "scale"),
           ((torch.zeros(1, 1, 1, 1025, device="cuda"), None, f), "head_dim"), ((q[..., :1], None, f), "head_dim")]
    for args, match in bad:
        with pytest.raises(ValueError, match=match):
            af3.rotary_embedding(*args)
    with pytest.raises(ValueError, match="no gradient"):
        af3.rotary_embedding(q, None, f.clone().requires_grad_(True))
    for args in ((q, q.cpu(), f), (q, None, f.cpu()), (q, None, f, torch.zeros(3, dtype=torch.int64))):
        with pytest.raises((RuntimeError, ValueError)):
            af3.rotary_embedding(*args)


# ---- differential attention ---------------------------------------------------------------------------------------------------
def diff_formula(q, k, v, lam, keep, causal, offset, scale, grad=None):
    """{name: (value, bound)} of out and, with grad, dq, dk, dv, dlam."""
    bf = q.dtype == BF16
    up_f, up, uo = (2.0 ** -11, 2.0 ** -8, 2.0 ** -8) if bf else (0.0, 0.0, E32)      # P in the forward pass; dS and P1 - lam P2; results
    q, k, v, lam = (wide(t) for t in (q, k, v, lam))
    B, H, Lq, D = q.shape[0], q.shape[1] // 2, q.shape[2], q.shape[3]
    Hkv, Lk, Dv = v.shape[1:]
    G = H // Hkv
    lam = lam.reshape(-1).expand(H).view(1, H, 1, 1)
    live = torch.ones(B, 1, Lq, Lk, dtype=torch.bool) if keep is None else keep.cpu().bool().view(-1, 1, 1, Lk).expand(B, 1, Lq, Lk).clone()
    seen = live[:, 0].any(1)[:, None, :, None]
    if causal:
        live &= torch.arange(Lk) <= torch.arange(Lq)[:, None] + offset
    k, v = k.masked_fill(~seen, 0.0), v.masked_fill(~seen, 0.0)
    heads = lambda t: t.repeat_interleave(G, 1)
    group = lambda t: t.reshape(B, Hkv, G, *t.shape[2:]).sum(2)
    vh = heads(v)
    q1, q2, k1, k2 = q[:, 0::2], q[:, 1::2], heads(k[:, 0::2]), heads(k[:, 1::2])
    # (V as fp16 is off by 2^-25 of its tile's unit at most, 2^-18 of what is largest in it; P as fp16 by 2^-25 of the row's largest)
    tiles = vh.abs().reshape(B, H, Lk, Dv)
    tiles = torch.cat([t.amax(2, keepdim=True).expand_as(t) for t in tiles.split(128, 2)], 2) if Lk else tiles
    small = (2.0 ** -17 * tiles, 2.0 ** -24 * vh.abs().sum(2, keepdim=True)) if bf else (0.0 * tiles, 0.0 * vh.abs().sum(2, keepdim=True))
    maps, eps, results, errors = [], [], [], []
    for qi, ki in ((q1, k1), (q2, k2)):
        x = torch.matmul(qi, ki.transpose(2, 3)) * scale
        size = (torch.matmul(qi.abs(), ki.abs().transpose(2, 3)) * scale).masked_fill(~live, 0.0)
        x = x.masked_fill(~live, -math.inf)
        top = x.amax(-1, keepdim=True)
        e = torch.exp(x - torch.where(torch.isinf(top), torch.zeros((), dtype=F64), top))
        total = e.sum(-1, keepdim=True)
        p = torch.where(total == 0, torch.zeros((), dtype=F64), e / torch.where(total == 0, torch.ones((), dtype=F64), total))
        ep = 2 * (D + 8) * E32 * size.amax(-1, keepdim=True) + (Lk + 16) * E32
        o = torch.matmul(p, vh)
        maps.append(p), eps.append(ep), results.append(o)
        errors.append(torch.matmul(p, vh.abs()) * (ep + (Lk + 8) * E32 + up_f) + torch.matmul(p, small[0]) + p.amax(-1, keepdim=True) * small[1])
    p1, p2 = maps
    out = results[0] - lam * results[1]
    err = errors[0] + lam.abs() * errors[1] + 2 * E32 * (results[0].abs() + (lam * results[1]).abs())
    r = {"out": (out, err + uo * (out.abs() + err))}
    if grad is None:
        return r
    g = wide(grad)
    n = G * Lq
    dp = torch.matmul(g, vh.transpose(2, 3))
    sums = torch.matmul(g.abs(), vh.abs().transpose(2, 3))
    weights = p1 - lam * p2
    dv = group(torch.matmul(weights.transpose(2, 3), g))
    terms = p1 * (eps[0] + (n + 8) * E32) + lam.abs() * p2 * (eps[1] + (n + 8) * E32) + up * weights.abs()
    dv_err = group(torch.matmul(terms.transpose(2, 3), g.abs()))
    r["dv"] = (dv, dv_err + uo * (dv.abs() + dv_err))
    kept = 2.0 ** -16 if bf else E32                                   # of a result and what its rounding lost
    lost = [errors[0] + kept * (out.abs() + (lam * results[1]).abs()), errors[1] + kept * results[1].abs()]
    lost[0] = lost[0] + lam.abs() * lost[1] + err
    dq, dk, dq_err, dk_err = [], [], [], []
    for i, (p, qi, ki, w) in enumerate(((p1, q1, k1, torch.ones_like(lam)), (p2, q2, k2, -lam))):
        delta = (p * dp).sum(-1, keepdim=True)
        to_delta = (g.abs() * lost[i]).sum(-1, keepdim=True) + (Dv + 4) * E32 * (g * results[i]).abs().sum(-1, keepdim=True)
        ds = w * p * (dp - delta)
        ds_err = w.abs() * p * ((eps[i] + 6 * E32) * (dp.abs() + delta.abs()) + (Dv + 4) * E32 * sums + to_delta) * 1.01
        f = ds_err + (up + 4 * E32) * (ds.abs() + ds_err)
        a = torch.matmul(ds, ki) * scale
        ea = scale * torch.matmul(f + (Lk + 4) * E32 * ds.abs(), ki.abs())
        b = group(torch.matmul(ds.transpose(2, 3), qi)) * scale
        eb = scale * group(torch.matmul((f + (n + 4) * E32 * ds.abs()).transpose(2, 3), qi.abs()))
        dq.append(a), dk.append(b), dq_err.append(ea + uo * (a.abs() + ea)), dk_err.append(eb + uo * (b.abs() + eb))
    both = lambda a: torch.stack(a, 2).flatten(1, 2)
    r["dq"], r["dk"] = (both(dq), both(dq_err)), (both(dk), both(dk_err))
    # lam's gradient: row sums of P2 dP in 32 bits, less what the row sum that was taken off missed
    dlam = -(p2 * dp).sum((0, 2, 3))
    each = (p2 * ((2 * eps[1] + (Lk + 24) * E32) * (dp.abs() + (p2 * dp).sum(-1, keepdim=True).abs()) + 2 * (Dv + 4) * E32 * sums)).sum((0, 2, 3))
    each = each + (B * Lq + 8) * E32 * (p2 * dp).sum(-1).abs().sum((0, 2)) + E32 * (g * results[1]).abs().sum((0, 2, 3)) * (Dv + 8)
    r["dlam"] = (dlam, each)                                               # (its own rounding: `compare`)
    return r


def diff_inputs(B, H, Hkv, Lq, Lk, D, Dv, dtype, seed, mask="none"):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()
    q, k, v, grad = n(B, 2 * H, Lq, D), n(B, 2 * Hkv, Lk, D), n(B, Hkv, Lk, Dv), n(B, H, Lq, Dv)
    lam = (torch.rand(H, generator=g) * 1.2 - 0.2).cuda()
    m = None
    if mask == "random":
        m = torch.rand(B, Lk, generator=g) < 0.7
    elif mask == "one":
        m = torch.zeros(B, Lk, dtype=torch.bool)
        m[torch.arange(B), torch.randint(Lk, (B,), generator=g)] = True
    elif mask in ("ragged", "empty"):
        m = torch.arange(Lk) < torch.randint(1, Lk + 1, (B, 1), generator=g)
        if mask == "empty":
            m[B // 2] = False
    return q, k, v, lam, (m.cuda() if m is not None else None), grad


def diff_run(af3, q, k, v, lam, m, grad, **kw):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, lam)]
    out = af3.differential_attention(*leaves, m, **kw)
    return dict(zip(["out", "dq", "dk", "dv", "dlam"], [out, *torch.autograd.grad(out, leaves, grad)]))


def diff_compare(got, q, k, v, lam, m, grad, causal=False, q_offset=0, softmax_scale=None):
    want = diff_formula(q, k, v, lam, m, causal, q_offset, q.shape[3] ** -0.5 if softmax_scale is None else softmax_scale, grad if "dq" in got else None)
    for name, t in got.items():
        value, bound = want[name]
        if name == "dlam":
            if tuple(t.shape) != tuple(value.shape):
                value, bound = value.sum().reshape(t.shape), bound.sum().reshape(t.shape) + (len(value) - 1) * E32 * value.abs().sum()
            bound = bound + half_step(t.dtype) * (value.abs() + bound)
        within(name, t, value, bound)


DIFF_SIZES = [
    # B, H, Hkv, Lq, Lk, D, Dv
    (1, 1, 1, 1, 1, 8, 16),
    (1, 1, 1, 1, 1, 1, 1),
    (2, 4, 4, 1, 37, 32, 64),
    (3, 4, 2, 1, 300, 64, 128),
    (2, 8, 2, 5, 129, 64, 64),
    (1, 6, 1, 33, 64, 24, 48),
    (2, 2, 2, 37, 1, 64, 128),
    (2, 2, 1, 64, 65, 48, 33),
    (1, 3, 3, 130, 257, 20, 100),
    (2, 16, 1, 1, 70, 64, 128),
    (2, 4, 1, 17, 200, 33, 65),
    (1, 2, 1, 200, 120, 7, 3),
]


@TYPES
@pytest.mark.parametrize("B,H,Hkv,Lq,Lk,D,Dv", DIFF_SIZES)
def test_differential_attention_and_gradients(af3, B, H, Hkv, Lq, Lk, D, Dv, dtype):
    for i, mask in enumerate(("none", "random", "one", "empty")):
        t = diff_inputs(B, H, Hkv, Lq, Lk, D, Dv, dtype, 10 * i + B, mask)
        for kw in ({}, {"causal": True, "q_offset": Lk - Lq}):
            got = diff_run(af3, *t, **kw)
            diff_compare(got, *t, **kw)
            alone = af3.differential_attention(*t[:5], **kw)
            assert torch.equal(alone, got["out"]), "the gradient's wish changes the result"


@pytest.mark.parametrize("B,H,Hkv,Lq,Lk,D,Dv,mask", [(1, 2, 1, 1, 400, 128, 256, "random"), (2, 2, 2, 40, 150, 128, 256, "empty"), (1, 4, 2, 200, 300, 100, 200, "ragged"),
                                                      (1, 1, 1, 70, 70, 128, 40, "none"), (1, 2, 2, 90, 66, 16, 256, "random"), (1, 2, 2, 65, 40, 72, 144, "one")])
def test_differential_attention_of_wide_heads(af3, B, H, Hkv, Lq, Lk, D, Dv, mask):
    t = diff_inputs(B, H, Hkv, Lq, Lk, D, Dv, BF16, 3, mask)
    for kw in ({}, {"causal": True, "q_offset": Lk - Lq}):
        diff_compare(diff_run(af3, *t, **kw), *t, **kw)


@TYPES
@pytest.mark.parametrize("B,H,Hkv,Lq,Lk,D", [(9, 4, 4, 640, 130, 64), (9, 8, 8, 520, 97, 32), (40, 4, 2, 300, 90, 64), (5, 4, 4, 700, 140, 128)])
def test_differential_attention_of_many_rows(af3, B, H, Hkv, Lq, Lk, D, dtype):
    """Workgroups whose wavefronts share no rows, V as fp16 among them."""
    if dtype == F32 and D > 64:
        D = 48
    t = diff_inputs(B, H, Hkv, Lq, Lk, D, 2 * D, dtype, 4, "empty")
    for kw in ({}, {"causal": True, "q_offset": 5}):
        diff_compare(diff_run(af3, *t, **kw), *t, **kw)


@TYPES
@pytest.mark.parametrize("Lq", [1, 3, 40])
def test_a_long_axis_of_keys_in_parts(af3, Lq, dtype):
    B, H, Hkv, D = 1, 4, 2, 64
    t = list(diff_inputs(B, H, Hkv, Lq, 6000, D, 128, dtype, 6, "random"))
    diff_compare(diff_run(af3, *t), *t)
    t[4][:, 128:5900] = False                     # parts without a live key
    diff_compare(diff_run(af3, *t), *t)
    t[4][:] = False
    got = diff_run(af3, *t)
    assert all((x == 0).all() for x in got.values())


@pytest.mark.parametrize("B,H,Hkv,L,D,dtype", [(2, 8, 4, 1100, 32, BF16), (3, 3, 3, 900, 64, BF16), (1, 16, 8, 700, 128, BF16), (1, 8, 8, 500, 32, F32), (1, 11, 11, 400, 16, F32), (2, 2, 1, 1300, 64, BF16)])
def test_causal_tiles_of_every_length(af3, B, H, Hkv, L, D, dtype):
    """However the tiles of a causal launch are dealt out: pairs in eights, more than eight, fewer; parts of the long axes among them."""
    t = diff_inputs(B, H, Hkv, L, L, D, 2 * D, dtype, 23, "none")
    diff_compare(diff_run(af3, *t, causal=True), *t, causal=True)


def test_a_long_axis_of_queries_in_parts(af3):
    for dtype in (BF16, F32):
        t = diff_inputs(1, 2, 1, 4000, 33, 32, 64, dtype, 7, "random")
        diff_compare(diff_run(af3, *t), *t)


@TYPES
@pytest.mark.parametrize("Lq,B", [(1, 2), (60, 2), (300, 40), (640, 9)])
def test_nothing_at_a_dropped_key_matters(af3, Lq, B, dtype):
    q, k, v, lam, m, g = diff_inputs(B, 4, 4, Lq, 150, 64, 128, dtype, 8, "random")
    m[:, 0] = True
    clean = diff_run(af3, q, k, v, lam, m, g)
    for worst in (math.nan, math.inf, -math.inf, torch.finfo(dtype).max, torch.finfo(dtype).min):
        k2, v2 = (t.clone() for t in (k, v))
        k2.masked_fill_(~m[:, None, :, None], worst), v2.masked_fill_(~m[:, None, :, None], worst)
        dirty = diff_run(af3, q, k2, v2, lam, m, g)
        for name in clean:
            assert torch.equal(clean[name], dirty[name]), (name, worst)
    for name in ("dk", "dv"):
        assert (clean[name].masked_select(~m[:, None, :, None]) == 0).all()


@TYPES
@pytest.mark.parametrize("offset", [-1000, -40, -3, 0, 7, 49, 10 ** 9])
def test_causal_offsets(af3, offset, dtype):
    """Queries in front of the first key give zeros and have no gradient."""
    for sizes in ((2, 4, 2, 40, 50, 64, 128), (1, 4, 4, 3, 50, 32, 64)):
        t = diff_inputs(*sizes, dtype, 9, "random")
        got = diff_run(af3, *t, causal=True, q_offset=offset)
        diff_compare(got, *t, causal=True, q_offset=offset)
        dead = -offset if offset < 0 else 0
        assert (got["out"][:, :, :dead] == 0).all() and (got["dq"][:, :, :dead] == 0).all()


@TYPES
def test_a_prompt_in_chunks(af3, dtype):
    """Queries whose keys end inside a tile, chunk by chunk over one cache: each chunk like the rows of the whole."""
    q, k, v, lam, _, _ = diff_inputs(2, 4, 2, 190, 190, 64, 128, dtype, 11)
    value, bound = diff_formula(q, k, v, lam, None, True, 0, 0.125)["out"]
    at = 0
    for n in (1, 63, 64, 1, 2, 40, 19):
        out = af3.differential_attention(q[:, :, at:at + n], k[:, :, :at + n], v[:, :, :at + n], lam, causal=True, q_offset=at)
        within(f"{at}..{at + n}", out, value[:, :, at:at + n], bound[:, :, at:at + n])
        at += n


@pytest.mark.parametrize("Lq,B", [(1, 1), (40, 2), (640, 9)])
def test_values_of_very_different_sizes(af3, Lq, B):
    """Tiles of V that are 2^200 apart, a column of tiny ones beside large ones, and V that is zero."""
    t = list(diff_inputs(B, 4, 4, Lq, 400, 64, 128, BF16, 12, "random"))
    g = torch.Generator().manual_seed(1)
    v0 = t[2].clone()
    for unit in (2.0 ** torch.randint(-100, 100, (400 // 50, 1), generator=g).double(), torch.tensor([[2.0 ** 60], [2.0 ** -60]] * 4, dtype=F64), torch.tensor([[2.0 ** -120]] * 8, dtype=F64),
                 torch.tensor([[2.0 ** 110]] * 8, dtype=F64), torch.zeros(8, 1, dtype=F64)):
        t[2] = (v0.double() * unit.expand(8, 50).reshape(400, 1).cuda()).to(BF16)
        diff_compare({"out": af3.differential_attention(*t[:5])}, *t)
    t[2] = v0.clone()
    t[2][..., ::7] *= 2.0 ** -12
    diff_compare({"out": af3.differential_attention(*t[:5])}, *t)


@TYPES
@pytest.mark.parametrize("Lq,B", [(1, 2), (40, 2), (640, 9)])
def test_large_logits_and_other_scales(af3, Lq, B, dtype):
    q, k, v, lam, m, g = diff_inputs(B, 4, 4, Lq, 100, 64, 128, dtype, 13, "random")
    for factor, scale in ((30.0, None), (1.0, 2.5), (1e-3, 1e-3), (1.0, 1e-30)):
        t = (q * factor, k, v, lam, m, g)
        diff_compare(diff_run(af3, *t, softmax_scale=scale), *t, softmax_scale=scale)
    # rows whose logits are all far from zero, either side
    for far in (1e3, 1e6, 1e10):
        for sign in (1.0, -1.0):
            q2, k2 = torch.zeros_like(q), torch.zeros_like(k)
            q2[..., 0], k2[..., 0], k2[..., 1] = 1.0, sign * far, 0.0
            out = af3.differential_attention(q2, k2, v, lam, m, softmax_scale=1.0)
            # all logits alike: the mean over live keys, times 1 - lam
            live = m.sum(1).clamp(min=1)[:, None, None].double()
            mean = (v.double() * m[:, None, :, None]).sum(2) / live * (1 - lam.double())[None, :, None]
            size = (v.double().abs() * m[:, None, :, None]).sum(2) / live * (1 + lam.double().abs())[None, :, None]
            limit = size * (2.0 ** -11 if dtype == BF16 else 200 * E32) + half_step(dtype) * mean.abs() + 2.0 ** -17 * v.abs().max().item() * 2.2 * (dtype == BF16)
            assert ((out.double() - mean[:, :, None]).abs() <= limit[:, :, None]).all(), (far, sign)


@TYPES
def test_views_broadcasts_and_odd_layouts(af3, dtype):
    B, H, Hkv, Lq, Lk, D, Dv = 2, 4, 2, 33, 70, 32, 64
    g = torch.Generator().manual_seed(14)
    n = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()
    lam = torch.rand(H, generator=g).cuda()
    lay = [
        (n(B, Lq, 2 * H, D).transpose(1, 2), n(B, Lk, 2 * Hkv, D).transpose(1, 2), n(B, Lk, Hkv, Dv).transpose(1, 2)),
        (n(B, 2 * H, Lq, D + 1)[..., 1:], n(B, 2 * Hkv, Lk, D + 3)[..., 2:D + 2], n(B, Hkv, Lk, Dv + 1)[..., :Dv]),
        (n(1, 1, Lq, D).expand(B, 2 * H, Lq, D), n(B, 1, Lk, D).expand(B, 2 * Hkv, Lk, D), n(1, Hkv, Lk, Dv).expand(B, Hkv, Lk, Dv)),
        (n(B, 2 * H, 1, D).expand(B, 2 * H, Lq, D), n(B, 2 * Hkv, 1, D).expand(B, 2 * Hkv, Lk, D), n(B, Hkv, 1, Dv).expand(B, Hkv, Lk, Dv)),
        (n(B, 2 * H, D, Lq).transpose(2, 3), n(B, 2 * Hkv, D, Lk).transpose(2, 3), n(B, Hkv, Dv, Lk).transpose(2, 3)),
        (n(B, 2 * H, 2 * Lq, D)[:, :, ::2], n(B, 2 * Hkv, 3 * Lk, D)[:, :, 1::3], n(2 * B, Hkv, Lk, Dv)[::2]),
    ]
    for q, k, v in lay:
        for grad in (n(B, H, Lq, Dv), n(B, Lq, H, Dv).transpose(1, 2), n(B, H, Lq, Dv + 1)[..., 1:], n(1, 1, 1, Dv).expand(B, H, Lq, Dv), n(B, H, Dv, Lq).transpose(2, 3)):
            m = (torch.rand(B, 2 * Lk, generator=g) < 0.8).cuda()[:, ::2]
            t = (q, k, v, lam, m, grad)
            diff_compare(diff_run(af3, *t), *t)
        for step in (q[:, :, :1], q[:, :, 5:7]):
            diff_compare({"out": af3.differential_attention(step, k, v, lam, m)}, step, k, v, lam, m, None)
    # gradients of what was broadcast, summed by torch
    one = n(1, 1, Lk, D).requires_grad_(True)
    q, _, v = lay[0]
    out = af3.differential_attention(q, one.expand(B, 2 * Hkv, Lk, D), v, lam)
    want = diff_formula(q, one.expand(B, 2 * Hkv, Lk, D), v, lam, None, False, 0, D ** -0.5, torch.ones_like(out))["dk"]
    extra = (half_step(dtype) * 2 + 8 * E32) * (want[0].abs() + want[1]).sum((0, 1), keepdim=True)
    within("broadcast k", torch.autograd.grad(out, one, torch.ones_like(out))[0], want[0].sum((0, 1), keepdim=True), want[1].sum((0, 1), keepdim=True) + extra)


@HOSTS
def test_forms_of_lam_masks_and_types(af3, host, native):
    host(native)
    q, k, v, lam, m, g = diff_inputs(2, 4, 2, 20, 40, 32, 64, BF16, 15, "random")
    for form in (lam, lam.to(BF16), lam[:1], lam[0], lam.double(), lam.half(), lam.repeat_interleave(3)[::3], lam[:1].expand(4)):
        seen = form if form.dtype in (BF16, F32) else form.float()
        leaf = form.detach().clone().requires_grad_(True) if form.dim() == 0 or form.stride(0) == 1 else form.detach().requires_grad_(True)
        out = af3.differential_attention(q, k, v, leaf, m)
        diff_compare({"out": out}, q, k, v, seen, m, None)
        d = torch.autograd.grad(out, leaf, g)[0]
        assert d.shape == form.shape and d.dtype == form.dtype
        value, bound = diff_formula(q, k, v, seen, m, False, 0, 32 ** -0.5, g)["dlam"]
        if form.numel() == 1:
            value, bound = value.sum().reshape(form.shape), bound.sum().reshape(form.shape) + (2 * half_step(seen.dtype) + 8 * E32) * value.abs().sum()
        within("dlam", d, value, bound + (half_step(form.dtype) + half_step(seen.dtype)) * (value.abs() + bound))
    base = af3.differential_attention(q, k, v, lam, m)
    for form in (m[:, None, None, :], m.to(torch.uint8), m.int() * 7, m.float()):
        assert torch.equal(base, af3.differential_attention(q, k, v, lam, form))
    row = m[0]
    assert torch.equal(af3.differential_attention(q, k, v, lam, row), af3.differential_attention(q, k, v, lam, row.expand(2, 40)))
    assert torch.equal(af3.differential_attention(q, k.float(), v.half(), lam), af3.differential_attention(q, k.float().to(BF16), v.half().to(BF16), lam))
    # one number for all heads, given as such or repeated
    leaf = lam[:1].clone().requires_grad_(True)
    a = torch.autograd.grad(af3.differential_attention(q, k, v, leaf, m), leaf, g)[0]
    b = torch.autograd.grad(af3.differential_attention(q, k, v, leaf.expand(4), m), leaf, g)[0]
    assert torch.equal(a, b)


@HOSTS
def test_no_queries_no_keys_no_batch(af3, host, native):
    host(native)
    for B, Lq, Lk in ((0, 5, 5), (2, 0, 5), (2, 5, 0)):
        t = diff_inputs(B, 2, 1, Lq, Lk, 16, 32, F32, 16)
        got = diff_run(af3, *t)
        assert got["out"].shape == (B, 2, Lq, 32) and all((x == 0).all() for x in got.values())
        assert got["dk"].shape == (B, 2, Lk, 16) and got["dlam"].shape == (2,)


def test_only_the_gradients_asked_for(af3):
    for dtype in (BF16, F32):
        q, k, v, lam, m, g = diff_inputs(2, 4, 2, 50, 60, 32, 64, dtype, 17, "random")
        whole = diff_run(af3, q, k, v, lam, m, g)
        for i, name in enumerate(("dq", "dk", "dv", "dlam")):
            args = [t.detach() for t in (q, k, v, lam)]
            args[i].requires_grad_(True)
            assert torch.equal(torch.autograd.grad(af3.differential_attention(*args, m), args[i], g)[0], whole[name]), name


def test_gradients_agree_with_differences(af3):
    """fp32: (f(x + h d) - f(x - h d)) / 2 h along random directions; h^2 of the third derivative and 2^-24 / h of f are what it may miss."""
    q, k, v, lam, m, g = diff_inputs(1, 2, 1, 9, 20, 16, 32, F32, 18, "random")
    got = diff_run(af3, q, k, v, lam, m, g)
    gen = torch.Generator().manual_seed(2)
    f = lambda *a: (af3.differential_attention(*a, m).double() * g.double()).sum().item()
    h = 2.0 ** -7
    for i, name in enumerate(("dq", "dk", "dv", "dlam")):
        args = [q, k, v, lam]
        d = torch.randn(args[i].shape, generator=gen).cuda()
        d /= d.norm()
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + h * d, args[i] - h * d
        difference = (f(*up) - f(*down)) / (2 * h)
        slope = (got[name].double() * d.double()).sum().item()
        # |f'''| <= 4 |g| |v| along a direction of length 1 whose logits move by |k| / 4 < 2 at most; f itself to 2^-20 |g| |out|
        room = 4 * 8 * h * h / 6 * g.norm().item() * v.abs().max().item() + 2.0 ** -20 / h * g.norm().item() * got["out"].norm().item()
        assert abs(difference - slope) <= room, (name, difference, slope, room)


def test_the_same_bits_every_time(af3):
    for sizes in ((3, 4, 2, 100, 300, 64, 128), (1, 8, 2, 1, 5000, 64, 128), (9, 4, 4, 640, 70, 64, 128)):
        t = diff_inputs(*sizes, BF16, 19, "random")
        first = diff_run(af3, *t)
        for _ in range(2):
            assert all(torch.equal(a, b) for a, b in zip(first.values(), diff_run(af3, *t).values()))


def test_keys_and_gradients_far_apart(af3):
    """Rows, heads and batches more than 4 GB apart, in the forward pass and as gradients of results."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of free memory")
    q, k, v, lam, m, g = diff_inputs(2, 2, 1, 40, 50, 32, 64, BF16, 20, "random")
    want = diff_run(af3, q, k, v, lam, m, g)

    def spread(t, axis):
        """t with one axis's stride beyond 2^31 elements / its length, so that its last entry is more than 4 GB away."""
        strides = [s for s in t.contiguous().stride()]
        strides[axis] = (1 << 31) // max(t.shape[axis] - 1, 1) + 4096
        strides[axis] -= strides[axis] % 64
        reach = sum((n - 1) * s for n, s in zip(t.shape, strides)) + 1
        out = torch.empty(reach, dtype=t.dtype, device="cuda").as_strided(t.shape, strides)
        out.copy_(t)
        return out
    for axis in (0, 1, 2):
        moved = [spread(t, axis) if t.shape[axis] > 1 else t for t in (q, k, v)]
        got = diff_run(af3, *moved, lam, m, spread(g, axis))
        assert all(torch.equal(a, b) for a, b in zip(want.values(), got.values())), axis
        del moved, got
        gc.collect()
        torch.cuda.empty_cache()


@HOSTS
def test_gradients_of_results_with_far_rows(af3, host, native):
    """Rows 2^23 elements apart and more are laid out anew on the way in."""
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB of free memory")
    host(native)
    q, k, v, lam, m, g = diff_inputs(1, 1, 1, 5, 20, 32, 64, BF16, 21, "random")
    far = torch.empty(4 * ((1 << 23) + 64) + 64, dtype=BF16, device="cuda").as_strided((1, 1, 5, 64), (64, 64, (1 << 23) + 64, 1))
    far.copy_(g)
    assert all(torch.equal(a, b) for a, b in zip(diff_run(af3, q, k, v, lam, m, g).values(), diff_run(af3, q, k, v, lam, m, far).values()))


@HOSTS
def test_differential_attention_refuses(af3, host, native):
    host(native)
    q, k, v, lam, _, _ = diff_inputs(2, 4, 2, 3, 5, 16, 32, F32, 22)
    z = lambda *s: torch.zeros(*s, device="cuda")
    bad = [((q[0], k, v, lam), {}, "q must be"), ((q[:, :7], k, v, lam), {}, "q must be"), ((q, k[:, :3], v, lam), {}, "q must be"), ((q, k, v[:1], lam), {}, "q must be"),
           ((q, k, v[:, :, :4], lam), {}, "q must be"), ((q, k[..., :8], v, lam), {}, "q must be"), ((z(2, 6, 3, 16), k, v, lam), {}, "multiple"),
           ((q.half(), k, v, lam), {}, "unsupported dtype"), ((z(1, 2, 3, 65), z(1, 2, 3, 65), z(1, 1, 3, 8), lam[:1]), {}, "head_dim"),
           ((z(1, 2, 3, 8), z(1, 2, 3, 8), z(1, 1, 3, 129), lam[:1]), {}, "head_dim"), ((q, k, v, lam[:3]), {}, "lam"), ((q, k, v, lam[None]), {}, "lam"),
           ((q, k, v, lam, torch.ones(4, device="cuda")), {}, "mask"), ((q, k, v, lam, torch.ones(3, 5, device="cuda")), {}, "mask"),
           ((q, k, v, lam), {"q_offset": 1 << 40}, "2\\^40"), ((q, k, v, lam), {"q_offset": -(1 << 40)}, "2\\^40")]
    bad += [((q, k, v, lam), {"softmax_scale": s}, "softmax_scale") for s in (0.0, -1.0, math.inf, math.nan)]
    for args, kw, match in bad:
        with pytest.raises(ValueError, match=match):
            af3.differential_attention(*args, **kw)
    with pytest.raises((RuntimeError, ValueError)):
        af3.differential_attention(q, k.cpu(), v, lam)
    with pytest.raises(TypeError, match="lam must be a tensor"):
        af3.differential_attention(q, k, v, 0.8)


# ---- norms around a block -----------------------------------------------------------------------------------------------------
class Num:
    """A number in 64 bits and how far the kernel's own, in 32, may be from it.  `depth`: how many additions lie on a term's way through a sum (16 channels of a thread, 6
    exchanges in a wavefront, 16 wavefronts, and some room)."""

    def __init__(self, v, e=0.0):
        self.v, self.e = v, e + torch.zeros_like(v)

    @staticmethod
    def of(x):
        return x if isinstance(x, Num) else Num(torch.as_tensor(x, dtype=F64))

    def _rounded(self, v, e):
        return Num(v, e + E32 * (v.abs() + e))

    def __add__(self, o):
        o = Num.of(o)
        return self._rounded(self.v + o.v, self.e + o.e)

    def __sub__(self, o):
        o = Num.of(o)
        return self._rounded(self.v - o.v, self.e + o.e)

    def __mul__(self, o):
        o = Num.of(o)
        return self._rounded(self.v * o.v, self.v.abs() * o.e + o.v.abs() * self.e + self.e * o.e)

    __radd__, __rmul__ = __add__, __mul__

    def mean(self):
        return Num(self.v.mean(-1, keepdim=True), self.e.mean(-1, keepdim=True) + 64 * E32 * (self.v.abs() + self.e).mean(-1, keepdim=True))

    def sum(self, dims, keepdim=False):
        n = math.prod(self.v.shape[d] for d in dims)
        size = (self.v.abs() + self.e).sum(dims, keepdim=keepdim)
        return Num(self.v.sum(dims, keepdim=keepdim), self.e.sum(dims, keepdim=keepdim) + n * E32 * size)

    def inverse_root(self):
        v = self.v.rsqrt()
        return Num(v, 0.5 * self.e * v ** 3 * 1.1 + 4 * E32 * v)

    def logistic(self):
        s = torch.sigmoid(self.v)
        return Num(s, s * (1 - s) * (self.e + 4 * E32 * self.v.abs()) + 8 * E32 * s)

    def rounded(self, dtype):
        return self.v, self.e + half_step(dtype) * (self.v.abs() + self.e)


def standard(a, kind, eps):
    if kind == "layer":
        a = a - a.mean()
    root = ((a * a).mean() + eps).inverse_root()
    return a * root, root


def back(g, normed, root, kind):
    d = g - normed * (g * normed).mean()
    if kind == "layer":
        d = d - g.mean()          # (the mean of normed is zero)
    return d * root


def norm_formula(t, grads=None, norm="rms", post_norm="none", gate_activation="none", residual_scale=1.0, eps=1e-5):
    """{name: Num}: out, normed and, with grads (of out, of normed), those of every tensor in t."""
    f = {n: Num(wide(x)) if x is not None else None for n, x in t.items()}
    s, eps = float(torch.tensor(residual_scale, dtype=F32)), float(torch.tensor(eps, dtype=F32))
    z, post_root = standard(f["y"], post_norm, eps) if post_norm != "none" else (f["y"], None)
    zw = z * f["post_weight"] if f["post_weight"] is not None else z
    gate = f["gate"]
    if gate is not None and gate_activation == "sigmoid":
        gate = gate.logistic()
    r = zw * gate if gate is not None else zw
    if f["x"] is not None:
        r = r + f["x"] * s
    res = {"out": r}
    if norm != "none":
        n, root = standard(r, norm, eps)
        h = n * f["weight"] if f["weight"] is not None else n
        res["normed"] = h + f["bias"] if f["bias"] is not None else h
    if grads is None:
        return res
    zero = torch.zeros_like(f["y"].v)
    d = Num(wide(grads[0])) if grads[0] is not None else Num(zero)
    to = {}
    if norm != "none" and grads[1] is not None:
        dh = Num(wide(grads[1]))
        to["bias"], to["weight"] = dh, dh * n
        d = d + back(dh * f["weight"] if f["weight"] is not None else dh, n, root, norm)
    to["x"] = d * s
    if gate is not None:
        to["gate"] = d * zw
        if gate_activation == "sigmoid":
            to["gate"] = to["gate"] * (gate * (Num.of(1.0) - gate))
        d = d * gate
    to["post_weight"] = d * z
    if f["post_weight"] is not None:
        d = d * f["post_weight"]
    to["y"] = back(d, z, post_root, post_norm) if post_norm != "none" else d
    for name, x in t.items():
        if x is None:
            continue
        g = to.get(name, Num(torch.zeros_like(f[name].v)))
        if g.v.shape != x.shape:
            lead = g.v.dim() - x.dim()
            g = g.sum(tuple(range(lead)) + tuple(i + lead for i in range(x.dim()) if x.shape[i] == 1 and g.v.shape[i + lead] != 1), keepdim=False) if x.dim() == 1 else \
                g.sum(tuple(i for i in range(x.dim()) if x.shape[i] == 1 and g.v.shape[i] != 1), keepdim=True) if any(x.shape[i] != g.v.shape[i] for i in range(x.dim())) else g
        res["d" + name] = g
    return res


NAMES = ("x", "y", "weight", "bias", "gate", "post_weight")


def norm_inputs(shape, dtype, seed, x=True, weight="channel", bias="none", gate="none", post=False):
    g = torch.Generator().manual_seed(seed)
    C = shape[-1]
    forms = {"channel": (C,), "row": shape, "batch": (shape[0], *[1] * (len(shape) - 2), C), "one": (*[1] * (len(shape) - 1), C)}
    n = lambda s: torch.randn(s, generator=g).to(dtype).cuda()
    t = {"x": n(shape) if x else None, "y": n(shape), "weight": n(forms[weight]) if weight != "none" else None, "bias": n(forms[bias]) if bias != "none" else None,
         "gate": n(forms[gate]) if gate != "none" else None, "post_weight": n((C,)) if post else None}
    return t, (n(shape), n(shape))


def norm_run(af3, t, grads, **kw):
    leaves = {n: x.detach().requires_grad_(True) for n, x in t.items() if x is not None}
    out, normed = af3.residual_norm(*(leaves.get(n) for n in NAMES), **kw)
    got = {"out": out, "normed": normed}
    pairs = [(o, g) for o, g in zip((out, normed), grads) if o is not None and g is not None]
    d = torch.autograd.grad([o for o, _ in pairs], list(leaves.values()), [g for _, g in pairs])
    return got | {"d" + n: x for n, x in zip(leaves, d)}


def norm_compare(got, t, grads=None, **kw):
    want = norm_formula(t, grads, **kw)
    for name, x in got.items():
        if x is None:
            assert name not in want
            continue
        within(name, x, *want[name].rounded(x.dtype))


@TYPES
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 3, 8), (1, 1, 64), (3, 37, 100), (2, 65, 384), (1, 5, 513), (2, 1030, 1024), (1, 3, 1023), (2, 9, 2048), (1, 33, 2050), (2, 7, 4096), (1, 5, 8192),
                                   (1, 3, 10000), (1, 2, 16384)], ids=str)
def test_residual_norm_and_gradients(af3, shape, dtype):
    settings = [
        (dict(), dict()),
        (dict(x=False, weight="none"), dict(norm="layer")),
        (dict(weight="row", bias="row", gate="row"), dict(norm="layer", gate_activation="sigmoid", residual_scale=0.7)),
        (dict(weight="batch", bias="batch", gate="batch", post=True), dict(norm="layer", post_norm="rms", residual_scale=-1.3)),
        (dict(weight="channel", bias="channel", gate="channel", post=True), dict(post_norm="layer", eps=1e-2)),
        (dict(weight="none", gate="batch", post=True), dict(norm="none", post_norm="rms")),
        (dict(x=False, weight="none", post=True), dict(norm="none", post_norm="rms")),
        (dict(x=False, weight="none", gate="row"), dict(norm="none", gate_activation="sigmoid")),
        (dict(weight="one", bias="batch", gate="row"), dict()),
        (dict(post=False), dict(post_norm="layer")),
    ]
    for i, (form, kw) in enumerate(settings):
        if shape[-1] == 1 and ("layer" in kw.values()):
            continue                       # (one channel less its mean)
        t, grads = norm_inputs(shape, dtype, 100 + i, **form)
        got = norm_run(af3, t, grads, **kw)
        norm_compare(got, t, grads, **kw)
        alone = af3.residual_norm(*(t[n] for n in NAMES), **kw)
        assert all(a is b is None or torch.equal(a, b) for a, b in zip(alone, (got["out"], got["normed"]))), "the gradient's wish changes the result"


@TYPES
@HOSTS
def test_residual_norm_forms_of_parameters(af3, host, native, dtype):
    """Parameters repeated over other axes than the last ones, several lengths of repetition in one call, other types, rows of two, three and four axes."""
    host(native)
    g = torch.Generator().manual_seed(31)
    n = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()
    for shape, forms in (((3, 4, 5, 24), ((3, 1, 1, 24), (3, 4, 1, 24), (1, 4, 1, 24))), ((3, 4, 24), ((1, 4, 24), (3, 1, 24), (24,))), ((6, 24), ((1, 24), (6, 24), (24,))), ((24,), ((24,), (24,), (24,))),
                         ((2, 3, 4, 5, 24), ((2, 1, 4, 1, 24), (1, 1, 1, 1, 24), (2, 3, 1, 1, 24)))):
        gate, weight, bias = (n(*f) for f in forms)
        for gate, weight, bias in ((gate, weight, bias), (weight, bias, gate), (bias, gate, weight)):
            t = {"x": n(*shape), "y": n(*shape), "weight": weight, "bias": bias, "gate": gate, "post_weight": None}
            grads = (n(*shape), n(*shape))
            got = norm_run(af3, t, grads, norm="layer", gate_activation="sigmoid")
            want = norm_formula(t, grads, norm="layer", gate_activation="sigmoid")
            for name, x in got.items():
                value, bound = want[name].rounded(x.dtype)
                if name in ("dgate", "dweight", "dbias") and x.shape != torch.Size(shape):      # (laid out for more rows than it has, its sums may be torch's, of rounded rows)
                    full = norm_formula({k: v.expand(shape) if k == name[1:] and v.dim() > 1 else v for k, v in t.items()}, grads, norm="layer", gate_activation="sigmoid")
                    size = (full[name].v.abs() + full[name].e)
                    dims = tuple(i for i in range(size.dim()) if x.dim() == size.dim() and x.shape[i] == 1 and size.shape[i] != 1)
                    bound = bound + half_step(dtype) * (size.sum(dims, keepdim=True) if dims else size)
                within(name, x, value, bound)
    t, grads = norm_inputs((2, 5, 40), dtype, 32, bias="batch", gate="row", post=True)
    other = F32 if dtype == BF16 else BF16
    cast = {k: v if k == "y" else v.to(other) for k, v in t.items()}
    back_again = {k: v.to(dtype) for k, v in cast.items()}
    kw = dict(post_norm="rms")
    for a, b in zip(af3.residual_norm(*(cast[k] for k in NAMES), **kw), af3.residual_norm(*(back_again[k] for k in NAMES), **kw)):
        assert torch.equal(a, b)


@TYPES
@HOSTS
def test_residual_norm_views(af3, host, native, dtype):
    host(native)
    g = torch.Generator().manual_seed(33)
    n = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()
    w = n(72)
    for x, y in ((n(3, 5, 73)[..., 1:], n(3, 5, 80)[..., :72]), (n(5, 3, 72).transpose(0, 1), n(3, 10, 72)[:, ::2]), (n(1, 1, 72).expand(3, 5, 72), n(3, 1, 72).expand(3, 5, 72)),
                 (n(3, 72, 5).transpose(1, 2), n(72, 3, 5).permute(1, 2, 0)), (n(3, 5, 72), n(1, 5, 72).expand(3, 5, 72))):
        for gate in (None, n(144)[::2], n(3, 1, 73)[..., 1:], n(3, 5, 73)[..., 1:]):
            t = {"x": x, "y": y, "weight": n(73)[1:], "bias": n(1, 1, 72).expand(3, 5, 72), "gate": gate, "post_weight": w}
            for grads in ((n(3, 5, 73)[..., 1:], n(5, 3, 72).transpose(0, 1)), (n(1, 1, 1).expand(3, 5, 72), n(3, 5, 72))):
                got = norm_run(af3, t, grads, post_norm="rms")
                norm_compare(got, t, grads, post_norm="rms")


@HOSTS
def test_residual_norm_gradients_of_one_result(af3, host, native):
    host(native)
    for dtype in (BF16, F32):
        t, grads = norm_inputs((2, 6, 100), dtype, 34, bias="channel", gate="batch", post=True)
        kw = dict(post_norm="layer")
        for pair in ((grads[0], None), (None, grads[1])):
            got = norm_run(af3, t, pair, **kw)
            if pair[1] is None:
                assert (got["dweight"] == 0).all() and (got["dbias"] == 0).all()
            norm_compare(got, t, pair, **kw)
        whole = norm_run(af3, t, grads, **kw)
        for name in NAMES:
            args = {k: v.detach() for k, v in t.items()}
            args[name].requires_grad_(True)
            got = torch.autograd.grad(af3.residual_norm(*(args[k] for k in NAMES), **kw), args[name], grads)[0]
            assert torch.equal(got, whole["d" + name]), name
        # the same tensor as stream and as the block's result, and for all parameters
        x = t["y"].detach().requires_grad_(True)
        d = torch.autograd.grad(af3.residual_norm(x, x, t["weight"]), x, grads)[0]
        two = norm_run(af3, {"x": t["y"], "y": t["y"], "weight": t["weight"], "bias": None, "gate": None, "post_weight": None}, grads)
        assert torch.equal(d, two["dx"] + two["dy"])
        same = t["weight"].detach().requires_grad_(True)
        d = torch.autograd.grad(af3.residual_norm(None, t["y"], same, same, same, same, post_norm="rms"), same, grads)[0]
        each = norm_run(af3, {"x": None, "y": t["y"], "weight": t["weight"], "bias": t["weight"], "gate": t["weight"], "post_weight": t["weight"]}, grads, post_norm="rms")
        terms = [each[n].double() for n in ("dweight", "dbias", "dgate", "dpost_weight")]
        assert ((d.double() - sum(terms)).abs() <= 3 * half_step(dtype) * 1.01 * sum(x.abs() for x in terms)).all()


@HOSTS
def test_residual_norm_of_nothing(af3, host, native):
    host(native)
    for shape in ((0, 5, 16), (3, 0, 16), (0, 16)):
        t, grads = norm_inputs(shape, F32, 35, bias="channel", gate="channel", post=True)
        got = norm_run(af3, t, grads, post_norm="rms")
        assert got["out"].shape == shape and got["normed"].shape == shape and (got["dweight"] == 0).all() and got["dweight"].shape == (16,)


def test_residual_norm_rows_that_are_not_finite_stay_alone(af3):
    for dtype in (BF16, F32):
        for C in (100, 1000, 4096):
            t, _ = norm_inputs((1, 9, C), dtype, 36, bias="channel", gate="channel", post=True)
            want = af3.residual_norm(*(t[n] for n in NAMES), post_norm="rms")
            t["y"][0, 4, 7], t["x"][0, 2, 3] = math.nan, math.inf
            got = af3.residual_norm(*(t[n] for n in NAMES), post_norm="rms")
            ok = [0, 1, 3, 5, 6, 7, 8]
            assert all(torch.equal(a[:, ok], b[:, ok]) for a, b in zip(got, want)) and got[1][0, 4].isnan().any()


@pytest.mark.parametrize("C,rows", [(64, 20000), (1024, 5000), (4096, 3000)])
def test_residual_norm_sums_over_many_rows(af3, C, rows):
    t, grads = norm_inputs((1, rows, C), BF16, 37, bias="channel", gate="channel", post=True)
    kw = dict(post_norm="rms", norm="layer")
    got = norm_run(af3, t, grads, **kw)
    norm_compare(got, t, grads, **kw)
    again = norm_run(af3, t, grads, **kw)
    assert all(torch.equal(a, b) for a, b in zip(got.values(), again.values()))


def test_residual_norm_gradients_agree_with_differences(af3):
    t, grads = norm_inputs((2, 3, 40), F32, 38, bias="batch", gate="row", post=True)
    kw = dict(norm="layer", post_norm="rms", gate_activation="sigmoid", residual_scale=0.6)
    got = norm_run(af3, t, grads, **kw)
    f = lambda a: sum((o.double() * g.double()).sum().item() for o, g in zip(af3.residual_norm(*(a[n] for n in NAMES), **kw), grads))
    gen, h = torch.Generator().manual_seed(3), 2.0 ** -7
    size = sum(o.norm().item() * g.norm().item() for o, g in zip((got["out"], got["normed"]), grads))
    for name in NAMES:
        d = torch.randn(t[name].shape, generator=gen).cuda()
        d /= d.norm()
        difference = (f(t | {name: t[name] + h * d}) - f(t | {name: t[name] - h * d})) / (2 * h)
        slope = (got["d" + name].double() * d.double()).sum().item()
        # third derivatives of a normalised row along a direction of length 1: 16 |grad| / its root mean square^3 (which is not far below 1/2 here); f to 2^-20
        assert abs(difference - slope) <= 16 * 8 * h * h / 6 * (grads[0].norm() + grads[1].norm()).item() + 2.0 ** -20 / h * size, (name, difference, slope)


def test_residual_norm_rows_far_apart(af3):
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB of free memory")
    t, grads = norm_inputs((3, 64), BF16, 39)
    want = norm_run(af3, t, grads)
    far = torch.empty((2 << 30) + 4096, dtype=BF16, device="cuda").as_strided((3, 64), (1 << 30, 1))
    far.copy_(t["y"])
    assert all(torch.equal(a, b) for a, b in zip(want.values(), norm_run(af3, t | {"y": far}, grads).values()))
    far.copy_(grads[1])
    assert all(torch.equal(a, b) for a, b in zip(want.values(), norm_run(af3, t, (grads[0], far)).values()))
    del far
    gc.collect()
    torch.cuda.empty_cache()


def test_residual_norm_of_more_rows_than_a_grid_has_on_one_side(af3):
    rows, C = (1 << 28) + 5, 8
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of free memory")
    y = torch.empty(rows, C, dtype=BF16, device="cuda")
    piece = torch.randn(1 << 20, C).to(BF16).cuda()
    for at in range(0, rows, 1 << 20):
        n = min(1 << 20, rows - at)
        y[at:at + n] = piece[:n]
    want = af3.residual_norm(None, piece)[1]
    y.requires_grad_(True)
    out, normed = af3.residual_norm(None, y)
    for at in (0, 1 << 27, rows - 5):
        n = min(1 << 20, rows - at)
        assert torch.equal(out[at:at + n], piece[:n]) and torch.equal(normed[at:at + n], want[:n])
    d = torch.autograd.grad(normed, y, y.detach())[0]
    del out, normed
    leaf = piece.detach().requires_grad_(True)
    back = torch.autograd.grad(af3.residual_norm(None, leaf)[1], leaf, piece)[0]
    for at in (0, 1 << 27, rows - 5):
        n = min(1 << 20, rows - at)
        assert torch.equal(d[at:at + n], back[:n])
    del d, y
    gc.collect()
    torch.cuda.empty_cache()


@HOSTS
def test_residual_norm_refuses(af3, host, native):
    host(native)
    y, w = torch.zeros(2, 3, 16, device="cuda"), torch.zeros(16, device="cuda")
    bad = [((None, y.half()), {}, "unsupported dtype"), ((None, y), {"norm": "batch"}, "norm must be"), ((None, y), {"post_norm": "l2"}, "post_norm must be"),
           ((None, y, None, None, w), {"gate_activation": "tanh"}, "gate_activation"), ((None, y), {"gate_activation": "sigmoid"}, "needs a gate"), ((y[:1], y), {}, "x must have"),
           ((None, y, w), {"norm": "none"}, "belong to a norm"), ((None, y, None, w), {"norm": "none"}, "belong to a norm"), ((None, y, None, None, None, w), {}, "belongs to a post_norm"),
           ((None, y, None, None, None, y), {"post_norm": "rms"}, "post_weight must be"), ((None, y, w[:8]), {}, "weight must be"), ((None, y, w[None]), {}, "weight must be"),
           ((None, y, None, y[:, :2]), {}, "bias must be"), ((None, y, None, None, y[:, :, :1]), {}, "gate must be"), ((None, torch.zeros(2, 16385, device="cuda")), {}, "C of 1"),
           ((None, torch.zeros(2, 0, device="cuda")), {}, "C of 1"), ((None, y), {"eps": -1.0}, "eps"), ((None, y), {"eps": math.nan}, "eps"), ((y, y), {"residual_scale": math.inf}, "residual_scale")]
    for args, kw, match in bad:
        with pytest.raises(ValueError, match=match):
            af3.residual_norm(*args, **kw)
    with pytest.raises((RuntimeError, ValueError)):
        af3.residual_norm(y.cpu(), y)


# ---- together, and as a program uses them --------------------------------------------------------------------------------------
def layer_parts(C, H, Hkv, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)
    w = {"norm1": 1 + 0.1 * n(C), "to_q": n(C, 2 * H * D) / C ** 0.5, "to_k": n(C, 2 * Hkv * D) / C ** 0.5, "to_v": n(C, Hkv * 2 * D) / C ** 0.5, "o": n(H * 2 * D, C) / (2 * H * D) ** 0.5,
         "head": 1 + 0.1 * n(2 * D), "norm2": 1 + 0.1 * n(C), "post": 1 + 0.1 * n(C), "gate": n(C)}
    return {k: t.to(dtype).cuda().requires_grad_(True) for k, t in w.items()} | {"lam": (torch.rand(H, generator=g)).cuda().requires_grad_(True)}


def layer(af3, w, x, y, f, cache, offset, H, Hkv, D, mask=None):
    """A decoder's attention layer between its two norms: (everything it made); cache: (k, v) of the tokens so far, or None."""
    B, L, C = y.shape
    x1, n1 = af3.residual_norm(x, y, w["norm1"])
    split = lambda t, h: t.view(B, L, h, -1).transpose(1, 2)
    q0, k0, v = (split(n1.view(-1, C) @ w[n], h) for n, h in (("to_q", 2 * H), ("to_k", 2 * Hkv), ("to_v", Hkv)))
    q, k = af3.rotary_embedding(q0, k0, f, offset=offset)
    K, V = (k, v) if cache is None else (torch.cat((cache[0], k), 2), torch.cat((cache[1], v), 2))
    a = af3.differential_attention(q, K, V, w["lam"], mask, causal=True, q_offset=offset)
    a2 = af3.residual_norm(None, a, post_weight=w["head"], post_norm="rms", norm="none")[0]      # (each head's own norm, as such layers have it)
    y2 = (a2.transpose(1, 2).reshape(B * L, -1) @ w["o"]).view(B, L, C)
    x2, n2 = af3.residual_norm(x1, y2, w["norm2"], None, w["gate"], w["post"], norm="layer", post_norm="rms", gate_activation="sigmoid")
    return dict(x1=x1, n1=n1, q0=q0, k0=k0, v=v, q=q, k=k, a=a, a2=a2, y2=y2, x2=x2, n2=n2)


@TYPES
def test_a_layer_with_its_gradients(af3, dtype):
    """Every operator against its formula on what the others gave it, forwards and backwards."""
    B, L, C, H, Hkv, D = 2, 75, 96, 4, 2, 32
    w = layer_parts(C, H, Hkv, D, dtype, 41)
    g = torch.Generator().manual_seed(42)
    x, y, g1, g2 = (torch.randn(B, L, C, generator=g).to(dtype).cuda() for _ in range(4))
    x.requires_grad_(True), y.requires_grad_(True)
    mask = (torch.arange(L) < torch.tensor([[L], [41]])).cuda()
    f, scale = af3.rotary_frequencies(D, device="cuda")
    r = layer(af3, w, x, y, f, None, 0, H, Hkv, D, mask)
    names = list(r)
    got = dict(zip(names + list(w) + ["x", "y"], torch.autograd.grad([r["x2"], r["n2"]], [r[n] for n in names] + list(w.values()) + [x, y], [g1, g2])))
    none = dict.fromkeys(NAMES)
    norm_compare({"out": r["x1"], "normed": r["n1"], "dx": got["x"], "dy": got["y"], "dweight": got["norm1"]}, none | {"x": x, "y": y, "weight": w["norm1"]}, (got["x1"], got["n1"]))
    for a, b, da, db in (("q0", "q", got["q0"], got["q"]), ("k0", "k", got["k0"], got["k"])):
        check_turned(b, r[b], r[a], f, torch.arange(L), False, scale)
        check_turned("d" + a, da, db, f, torch.arange(L), False, scale, True)
    diff_compare({"out": r["a"], "dq": got["q"], "dk": got["k"], "dv": got["v"], "dlam": got["lam"]}, r["q"], r["k"], r["v"], w["lam"], mask, got["a"], True, 0)
    norm_compare({"out": r["a2"], "dy": got["a"], "dpost_weight": got["head"]}, none | {"y": r["a"], "post_weight": w["head"]}, (got["a2"], None), norm="none", post_norm="rms")
    norm_compare({"out": r["x2"], "normed": r["n2"], "dx": got["x1"], "dy": got["y2"], "dgate": got["gate"], "dweight": got["norm2"], "dpost_weight": got["post"]},
                 none | {"x": r["x1"], "y": r["y2"], "weight": w["norm2"], "gate": w["gate"], "post_weight": w["post"]}, (g1, g2), norm="layer", post_norm="rms", gate_activation="sigmoid")


@TYPES
def test_a_decoder_token_by_token(af3, dtype):
    """A prompt and then single tokens over its cache: each step's operators against their formulas, and the same as the whole sequence at once within both sides' bounds of the last norm."""
    B, L, C, H, Hkv, D = 3, 30, 64, 4, 2, 16
    w = {k: t.detach() for k, t in layer_parts(C, H, Hkv, D, dtype, 43).items()}
    g = torch.Generator().manual_seed(44)
    x, y = (torch.randn(B, L, C, generator=g).to(dtype).cuda() for _ in range(2))
    f, _ = af3.rotary_frequencies(D, device="cuda")
    whole = layer(af3, w, x, y, f, None, 0, H, Hkv, D)
    r = layer(af3, w, x[:, :20], y[:, :20], f, None, 0, H, Hkv, D)
    K, V = r["k"], r["v"]
    for t in range(20, L):
        r = layer(af3, w, x[:, t:t + 1], y[:, t:t + 1], f, (K, V), t, H, Hkv, D)
        check_turned("q", r["q"], r["q0"], f, torch.tensor([t]), False, 1.0)
        K, V = torch.cat((K, r["k"]), 2), torch.cat((V, r["v"]), 2)
        diff_compare({"out": r["a"]}, r["q"], K, V, w["lam"], None, None, True, t)
        norm_compare({"out": r["x2"], "normed": r["n2"]}, {"x": r["x1"], "y": r["y2"], "weight": w["norm2"], "bias": None, "gate": w["gate"], "post_weight": w["post"]}, norm="layer",
                     post_norm="rms", gate_activation="sigmoid")
        # (the norms' rows are alike to the bit: a row does not depend on those beside it)
        assert torch.equal(r["x1"], whole["x1"][:, t:t + 1]) and torch.equal(r["n1"], whole["n1"][:, t:t + 1])


def test_calls_prepared_in_python_give_the_same_bits(af3, monkeypatch):
    from af3_kernels_amd import layers
    for dtype in (BF16, F32):
        w = layer_parts(64, 4, 2, 16, dtype, 45)
        x, y, g = (torch.randn(2, 37, 64, device="cuda", dtype=dtype) for _ in range(3))
        f, _ = af3.rotary_frequencies(16, device="cuda")
        mask = torch.rand(2, 37, device="cuda") < 0.8

        def everything():
            r = layer(af3, w, x, y, f, None, 0, 4, 2, 16, mask)
            return [*r.values(), *torch.autograd.grad([r["x2"], r["n2"]], list(w.values()), [g, g])]
        native = everything()
        with monkeypatch.context() as m:
            m.setattr(layers, "_host", _NoNativeHost())
            python = everything()
        assert all(torch.equal(a, b) for a, b in zip(native, python))


CALLS = {
    "rotary": lambda af3, a, b: af3.rotary_embedding(a[:, :, :, :8], b[:, :, :, :8], torch.ones(4, dtype=F64, device="cuda"))[0],
    "diff": lambda af3, a, b: af3.differential_attention(a, b, b[:, :2].repeat(1, 1, 1, 2), torch.ones(2, device="cuda")),
    "norm": lambda af3, a, b: af3.residual_norm(a, b)[1],
}


@HOSTS
@pytest.mark.parametrize("name", list(CALLS))
def test_no_second_derivative_and_no_forward_mode(af3, host, native, name):
    host(native)
    a, b = (torch.randn(2, 4, 5, 16, device="cuda").requires_grad_(True) for _ in range(2))
    g = torch.autograd.grad((CALLS[name](af3, a, b) ** 2).sum(), a, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="second derivative" if native else None):
        g.sum().backward()
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            CALLS[name](af3, forward_ad.make_dual(a.detach(), torch.ones_like(a)), b.detach())


@HOSTS
@pytest.mark.parametrize("name", ["diff", "norm"])
def test_inputs_changed_between_forward_and_backward_are_noticed(af3, host, native, name):
    host(native)
    a, b = torch.randn(2, 4, 5, 16, device="cuda").requires_grad_(True), torch.randn(2, 4, 5, 16, device="cuda")
    out = CALLS[name](af3, a, b)
    if name == "norm":
        b.mul_(2)
    else:
        with torch.no_grad():
            a.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.sum().backward()


def step_of(af3, dtype=BF16, B=2, L=60):
    C, H, Hkv, D = 64, 4, 2, 32
    w = layer_parts(C, H, Hkv, D, dtype, 51)
    g = torch.Generator().manual_seed(52)
    x, y, grad = (torch.randn(B, L, C, generator=g).to(dtype).cuda() for _ in range(3))
    f, _ = af3.rotary_frequencies(D, device="cuda")
    mask = (torch.rand(B, L, generator=g) < 0.8).cuda()

    def forward():
        with torch.no_grad():
            r = layer(af3, w, x, y, f, None, 0, H, Hkv, D, mask)
        return [r["x2"], r["n2"]]

    def train(w=w):
        r = layer(af3, w, x, y, f, None, 0, H, Hkv, D, mask)
        return [r["x2"].detach(), r["n2"].detach(), *torch.autograd.grad([r["x2"], r["n2"]], list(w.values()), [grad, grad])]
    return forward, train, (x, y, mask), w


def test_on_another_stream(af3):
    _, train, _, _ = step_of(af3)
    want = train()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = train()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    # two streams at once
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                results.append(train())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in results for a, b in zip(want, r))


def test_captured_and_replayed(af3):
    """Two graphs of the same calls, replayed in turn with eager work between them, inputs changed in place."""
    forward, _, inputs, _ = step_of(af3)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        forward()
    s.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(forward())
    for i in range(4):
        inputs[0].copy_(torch.randn_like(inputs[0])), inputs[2].copy_(torch.rand(inputs[2].shape, device="cuda") < 0.6)
        for graph in graphs:
            graph.replay()
        want = forward()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(want, out)), i


@pytest.mark.parametrize("kind", ["token", "parts", "half"])
def test_each_kind_of_attention_captured(af3, kind):
    sizes = {"token": (3, 8, 2, 1, 900, 64, 128), "parts": (1, 4, 2, 40, 5000, 64, 128), "half": (9, 4, 4, 640, 70, 64, 128)}[kind]
    q, k, v, lam, m, _ = diff_inputs(*sizes, BF16, 53, "random")
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        af3.differential_attention(q, k, v, lam, m)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = af3.differential_attention(q, k, v, lam, m)
    for _ in range(3):
        v.copy_(torch.randn_like(v.float()).to(BF16))
        graph.replay()
        want = af3.differential_attention(q, k, v, lam, m)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_a_training_step_captured_and_replayed(af3):
    _, train, inputs, w = step_of(af3)
    own = lambda: {n: t.detach().clone().requires_grad_(True) for n, t in w.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train(own())
    torch.cuda.current_stream().wait_stream(side)
    static = own()
    gc.collect()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = train(static)
    for i in range(4):
        inputs[1].copy_(torch.randn_like(inputs[1].float()))
        want = train(own())
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want)), i


@HOSTS
def test_a_capture_that_would_wait_for_another_stream_is_refused(af3, monkeypatch, native):
    """Leaves that an eager result still holds: captured, their gradient would end the process."""
    from af3_kernels_amd import layers

    class Only(_NoNativeHost):
        check_capture = staticmethod(layers._host.check_capture)
    if not native:
        monkeypatch.setattr(layers, "_host", Only())
    a, b = (torch.randn(2, 4, 5, 16, device="cuda").requires_grad_(True) for _ in range(2))
    f, lam, v = torch.ones(4, dtype=F64, device="cuda"), torch.ones(2, device="cuda"), torch.randn(2, 2, 5, 32, device="cuda")
    calls = (lambda a, b: af3.rotary_embedding(a, b, f)[0], lambda a, b: af3.differential_attention(a, b, v, lam), lambda a, b: af3.residual_norm(a, b)[1])
    eager = [call(a, b) for call in calls]
    refused, plain = 0, []
    gc.collect()      # (a graph that the collector frees while another is captured ends the process; for the same reason no exception, and with it this frame, is kept here)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in calls:
            with pytest.raises(RuntimeError, match="captured"):
                call(a, b)
            refused += 1
            plain.append(call(a.detach(), b.detach()))      # a call without a gradient is captured as ever
    assert refused == 3
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, e) for p, e in zip(plain, eager))
    del eager
