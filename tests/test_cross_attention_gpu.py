"""cross_attention and relative_position_bias on the GPU against their formulas in 64 bits on the CPU, on the numbers the device saw.

Tolerances are bounds per element, worked out from the roundings before anything ran (`bounds` below): fp32 sums of n terms are
off by at most n 2^-24 of the sum of the terms' magnitudes, a rounding to bf16 by 2^-8 of the value; P and dS are rounded to bf16 in front of
the products that follow them (bf16 calls), results once at the end.
"""
import gc
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
E32 = 2.0 ** -24
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def af3():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    import af3_kernels_amd
    af3_kernels_amd._lib.load()
    return af3_kernels_amd


# ---- the formulas in 64 bits ------------------------------------------------------------------------------------------------
def spread(t, H):
    """[B, Hkv, ...] -> [B, H, ...]: every query head's own copy of its key head."""
    return t.repeat_interleave(H // t.shape[1], dim=1)


def formula(q, k, v, keep, bias, grad, scale):
    """out, dq, dk, dv, dbias and the bounds of their errors as functions of (u_p, u_o), the roundings of P / dS and of results."""
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    B, H, Lq, D = q.shape
    Hkv, Lk = k.shape[1:3]
    keep = torch.ones(B, Lk, dtype=torch.bool) if keep is None else keep.cpu().bool().expand(B, Lk)
    live = keep.any(1)
    gone = (~keep & live[:, None])[:, None, None, :]          # a batch row without a live key: all of them, alike
    kh, vh = spread(k, H), spread(v, H)
    kh, vh = (t.masked_fill(gone.transpose(2, 3), 0.0) for t in (kh, vh))
    x = torch.matmul(q, kh.transpose(2, 3)) * scale
    size = torch.matmul(q.abs(), kh.abs().transpose(2, 3)) * scale
    if bias is not None:
        bias = bias.detach().double().cpu()
        x, size = x + bias, size + bias.abs()
    x = x.masked_fill(gone, -math.inf)
    dead = ~live[:, None, None, None]
    x, size = torch.where(dead, torch.zeros((), dtype=torch.float64), x), torch.where(dead | gone | ~torch.isfinite(size) | ~torch.isfinite(x), torch.zeros((), dtype=torch.float64), size)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(torch.isinf(top) & (top < 0), torch.zeros((), dtype=torch.float64), top))
    total = e.sum(-1, keepdim=True)
    p = torch.where(total == 0, torch.zeros((), dtype=torch.float64), e / total)
    out = torch.matmul(p, vh)
    # relative error of P: logits (products of D terms, scaling, adding), their distance to the maximum, exp2's argument, the sum
    worst = size.clamp(max=1e30).amax(-1, keepdim=True)
    ep = 2 * (D + 8) * E32 * worst + (Lk + 16) * E32
    r = {}
    err_out = torch.matmul(p, vh.abs()) * (ep + Lk * E32)
    r["out"] = (out, lambda up, uo: err_out + up * torch.matmul(p, vh.abs()) + uo * out.abs())
    if grad is None:
        return r
    g = grad.detach().double().cpu()
    group = lambda t: t.view(B, Hkv, H // Hkv, *t.shape[2:]).sum(2)
    dv = group(torch.matmul(p.transpose(2, 3), g))
    dv_size = lambda f: group(torch.matmul((p * f).transpose(2, 3), g.abs()))
    n = H // Hkv * Lq
    r["dv"] = (dv, lambda up, uo: dv_size(ep + n * E32 + up) + uo * dv.abs())
    dp = torch.matmul(g, vh.transpose(2, 3))
    delta = (g * out).sum(-1, keepdim=True)
    frozen = dead | gone
    ds = (p * (dp - delta)).masked_fill(frozen, 0.0)
    sums = torch.matmul(g.abs(), vh.abs().transpose(2, 3))

    def ds_error(up, uo):
        to_delta = (g.abs() * r["out"][1](up, uo)).sum(-1, keepdim=True) + D * E32 * (g * out).abs().sum(-1, keepdim=True)
        return (p * ((ep + 4 * E32) * (dp.abs() + delta.abs()) + (D + 2) * E32 * sums + to_delta)).masked_fill(frozen, 0.0)

    dq = torch.matmul(ds, kh) * scale
    r["dq"] = (dq, lambda up, uo: scale * torch.matmul(ds_error(up, uo) + (up + (Lk + 4) * E32) * ds.abs(), kh.abs()) + uo * dq.abs())
    dk = group(torch.matmul(ds.transpose(2, 3), q)) * scale
    r["dk"] = (dk, lambda up, uo: scale * group(torch.matmul((ds_error(up, uo) + (up + (n + 4) * E32) * ds.abs()).transpose(2, 3), q.abs())) + uo * dk.abs())
    if bias is not None:
        dbias = ds.sum(0)
        r["dbias"] = (dbias, lambda up, uo: ds_error(up, uo).sum(0) + (B + 2) * E32 * ds.abs().sum(0) + uo * dbias.abs())
    return r


def check(name, got, want, dtype):
    up, uo = (2.0 ** -8, 2.0 ** -8) if dtype == BF16 else (0.0, E32)
    value, bound = want
    got = got.detach().double().cpu()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    assert torch.isfinite(got).all(), f"{name}: not finite"
    excess = ((got - value).abs() - bound(up, uo) - 1e-30).max().item()
    assert excess <= 0, f"{name}: {excess} beyond the bound, error {(got - value).abs().max().item()}"


def make(B, H, Hkv, Lq, Lk, D, dtype, seed, mask="none", bias="none"):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()
    q, k, v, grad = n(B, H, Lq, D), n(B, Hkv, Lk, D), n(B, Hkv, Lk, D), n(B, H, Lq, D)
    b = n(H, Lq, Lk) if bias != "none" else None
    m = None
    if mask == "random":
        m = torch.rand(B, Lk, generator=g) < 0.7
        m[:, int(torch.randint(Lk, (1,), generator=g))] = True
    elif mask == "one":          # a single live key
        m = torch.zeros(B, Lk, dtype=torch.bool)
        m[torch.arange(B), torch.randint(Lk, (B,), generator=g)] = True
    elif mask in ("ragged", "empty"):
        m = torch.arange(Lk) < torch.randint(1, Lk + 1, (B, 1), generator=g)
        if mask == "empty":
            m[B // 2] = False
    return q, k, v, (m.cuda() if m is not None else None), b, grad


def run(af3, q, k, v, m, b, grad, scale=None):
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (q, k, v, b)]
    out = af3.cross_attention(leaves[0], leaves[1], leaves[2], m, leaves[3], softmax_scale=scale)
    wanted = [t for t in leaves if t is not None]
    return dict(zip(["out", "dq", "dk", "dv", "dbias"], [out, *torch.autograd.grad(out, wanted, grad)]))


def compare(got, q, k, v, m, b, grad, scale=None, dtype=None):
    want = formula(q, k, v, m, b, grad, q.shape[3] ** -0.5 if scale is None else scale)
    for name, t in got.items():
        check(name, t, want[name], dtype or q.dtype)


SIZES = [
    # B, H, Hkv, Lq, Lk, D
    (1, 1, 1, 1, 1, 8),
    (2, 4, 4, 1, 37, 32),
    (3, 4, 2, 1, 300, 64),
    (2, 8, 2, 5, 129, 128),
    (1, 6, 1, 33, 64, 24),
    (2, 2, 2, 37, 1, 64),
    (2, 2, 1, 64, 65, 48),
    (1, 3, 3, 130, 257, 80),
    (2, 2, 2, 200, 77, 96),
    (1, 2, 2, 31, 1000, 64),
    (1, 2, 1, 500, 31, 64),
    (2, 3, 3, 45, 70, 7),
    (1, 2, 2, 40, 50, 33),
    (1, 2, 2, 20, 40, 1),
    (1, 2, 1, 70, 130, 121),
]


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("B,H,Hkv,Lq,Lk,D", SIZES)
def test_cross_attention_and_gradients(af3, B, H, Hkv, Lq, Lk, D, dtype):
    for i, (mask, bias) in enumerate([("none", "none"), ("ragged", "given"), ("random", "none"), ("empty", "given"), ("one", "given")]):
        t = make(B, H, Hkv, Lq, Lk, D, dtype, 100 + i, mask, bias)
        print((B, H, Hkv, Lq, Lk, D), dtype, mask, bias, flush=True)
        got = run(af3, *t)
        compare(got, *t)
        plain = af3.cross_attention(*t[:5])
        assert torch.equal(plain, got["out"])      # without a graph the same bits


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("B,H,Hkv,Lq,Lk,D", [
    (9, 16, 16, 384, 200, 64),     # enough workgroups: 128 query rows each, 128 keys each in the gradient
    (9, 16, 4, 150, 384, 32),
    (20, 16, 16, 140, 150, 128),
    (20, 16, 16, 140, 150, 96),
])
def test_workgroups_of_128_rows(af3, B, H, Hkv, Lq, Lk, D, dtype):
    t = make(B, H, Hkv, Lq, Lk, D, dtype, 7, "empty", "given")
    compare(run(af3, *t), *t)
    t = make(B, H, Hkv, Lq, Lk, D, dtype, 8, "random", "none")
    compare(run(af3, *t), *t)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
def test_a_long_key_axis_in_parts(af3, dtype):
    """One query over 40000 keys: the key axis is cut over the workgroups and longer than what one of them looks at at a time."""
    t = make(1, 2, 2, 1, 40000, 64, dtype, 3, "random", "given")
    compare(run(af3, *t), *t)
    q, k, v, m, b, g = make(2, 2, 1, 3, 17000, 32, dtype, 4, "ragged", "none")
    m[0] = False
    m[1, :16500] = False
    m[1, 16900] = True
    compare(run(af3, q, k, v, m, b, g), q, k, v, m, b, g)
    many = make(64, 8, 8, 1, 20000, 16, dtype, 5, "ragged", "none")      # whole rows in one workgroup, in two stretches
    want = formula(many[0][:2], many[1][:2], many[2][:2], many[3][:2], None, None, 0.25)
    check("out", af3.cross_attention(*many[:4])[:2], want["out"], dtype)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("Lq,B", [(1, 2), (60, 2), (300, 40)])
def test_nothing_at_a_dropped_key_matters(af3, Lq, B, dtype):
    """Infinities, NaN and huge values in k, v and bias where the mask drops the key: the same bits as with zeros there, zeros as gradients."""
    q, k, v, m, b, g = make(B, 8, 4, Lq, 200, 48, dtype, 11, "random", "given")
    clean = [t.clone() for t in (k, v)]
    for t in clean:
        t.masked_fill_(~m[:, None, :, None], 0.0)
    cb = b.clone()
    common = ~m.any(0)
    k, v, b = k.clone(), v.clone(), b.clone()
    for i, bad in enumerate((float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).max)):
        sel = (~m & (torch.arange(200, device="cuda") % 4 == i))[:, None, :, None]
        k.masked_fill_(sel, bad), v.masked_fill_(sel, bad)
    m[:, 17], m[:, 18] = False, False
    b[:, :, 17], b[:, :, 18] = float("nan"), float("inf")
    cb[:, :, 17:19] = 0.0
    got = run(af3, q, k, v, m, b, g)
    want = run(af3, q, *clean, m, cb, g)
    for name in got:
        assert torch.equal(got[name], want[name]), name
    assert not got["dk"].masked_select(~m[:, None, :, None]).any() and not got["dv"].masked_select(~m[:, None, :, None]).any()
    assert not got["dbias"][:, :, 17:19].any()


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("Lq,Lk,B", [(1, 40, 2), (40, 150, 2), (300, 90, 40)])
def test_masks_through_the_bias(af3, Lq, Lk, B, dtype):
    low = torch.finfo(dtype).min
    q, k, v, m, b, g = make(B, 4, 4, Lq, Lk, 32, dtype, 12, "ragged", "given")
    b[0, :, ::3] = -float("inf")          # every third key for no query of head 0
    b[1, Lq // 2] = -float("inf")         # a query that its bias leaves no key
    b[2, Lq // 2] = low                   # ... and one that it weights alike
    b[3, :, 1::2] = low
    compare(run(af3, q, k, v, m, b, g), q, k, v, m, b, g)
    out = af3.cross_attention(q, k, v, m, b)
    assert not out[:, 1, Lq // 2].any()
    b = torch.zeros_like(b)
    b[0, 0, 0], b[1, 0, 0] = float("nan"), float("inf")     # at a live key: the formula gives NaN, to that row alone
    out = af3.cross_attention(q, k, v, m, b)
    assert out[:, :2, 0].isnan().all() and out[:, 2:].isfinite().all() and out[:, :, 1:].isfinite().all()


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
def test_large_logits_and_other_scales(af3, dtype):
    q, k, v, m, b, g = make(2, 4, 2, 70, 333, 64, dtype, 13, "random", "given")
    for scale in (1.0, 3.5, 1e-3):
        t = (q * 4, k, v, m, None, g)
        compare(run(af3, *t, scale=scale), *t, scale=scale)
    ramp = (torch.arange(333, device="cuda") * 3.0).to(dtype)       # the maximum moves with every tile
    t = (q, k, v, m, (b + ramp).contiguous(), g)
    compare(run(af3, *t), *t)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
def test_strides_views_and_broadcasts(af3, dtype):
    B, H, Hkv, Lq, Lk, D = 2, 4, 2, 50, 90, 40
    g = torch.Generator().manual_seed(5)
    n = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()
    # heads inside the token ([B, L, H, D]), k and v out of one packed projection at odd offsets
    q = n(B, Lq, H, D).transpose(1, 2)
    packed = n(B, Lk, Hkv, 2 * D + 3)
    k, v = packed[..., 1:D + 1].transpose(1, 2), packed[..., D + 2:2 * D + 2].transpose(1, 2)
    bias = n(H, Lq + 3, Lk + 5)
    grad = n(B, Lq, H, D).transpose(1, 2)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, bias)]
    out = af3.cross_attention(*leaves[:3], None, leaves[3])
    grads = torch.autograd.grad(out, leaves, grad)
    want = formula(q, k, v, None, bias[:, :Lq, :Lk], grad, D ** -0.5)
    for name, t in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        check(name, t, want[name], dtype)
    check("dbias", grads[3][:, :Lq, :Lk], want["dbias"], dtype)
    assert not grads[3][:, Lq:].any() and not grads[3][:, :, Lk:].any()
    # inputs that repeat: one k and v for the batch, one bias row for all queries, one bias for all heads, gradients that repeat
    k1, v1, b1, b2 = n(1, Hkv, Lk, D), n(1, 1, Lk, D), n(H, 1, Lk), n(1, Lq, Lk)
    for b0 in (b1, b2):
        leaves = [t.detach().requires_grad_(True) for t in (q, k1, v1, b0)]
        out = af3.cross_attention(leaves[0], leaves[1].expand(B, Hkv, Lk, D), leaves[2].expand(B, Hkv, Lk, D), None, leaves[3].expand(H, Lq, Lk))
        grads = torch.autograd.grad(out.sum(), leaves)
        want = formula(q, k1.expand(B, Hkv, Lk, D), v1.expand(B, Hkv, Lk, D), None, b0.expand(H, Lq, Lk), torch.ones(B, H, Lq, D, dtype=dtype), D ** -0.5)
        check("out", out, want["out"], dtype)
        check("dq", grads[0], want["dq"], dtype)
        up, uo = (2.0 ** -8, 2.0 ** -8) if dtype == BF16 else (0.0, E32)
        for got, name, dims in ((grads[1], "dk", (0,)), (grads[2], "dv", (0, 1)), (grads[3], "dbias", (1,) if b0 is b1 else (0,))):
            value, bound = want[name]
            # each summand as bounded, then torch's sum of them, rounded once more
            limit = bound(up, uo).sum(dims, keepdim=True) + (uo + 400 * E32) * value.abs().sum(dims, keepdim=True)
            assert ((got.double().cpu() - value.sum(dims, keepdim=True)).abs() <= limit + 1e-30).all(), name


def test_other_types_are_cast_and_masks_of_every_rank(af3):
    q, k, v, m, b, g = make(2, 4, 4, 30, 60, 32, BF16, 21, "random", "given")
    base = af3.cross_attention(q, k, v, m, b)
    assert torch.equal(af3.cross_attention(q, k.float(), v.half().to(BF16), m.int(), b.float()), base)
    assert torch.equal(af3.cross_attention(q, k, v, m[:, None, None, :], b), base)
    one = m[0]
    assert torch.equal(af3.cross_attention(q, k, v, one, b), af3.cross_attention(q, k, v, one.expand(2, 60), b))
    f = b.float().requires_grad_(True)
    grad = torch.autograd.grad(af3.cross_attention(q, k, v, m, f), f, g)[0]
    assert grad.dtype == torch.float32 and torch.equal(grad.to(BF16), run(af3, q, k, v, m, b, g)["dbias"])


def test_no_queries_no_keys_no_batch(af3):
    for B, Lq, Lk in ((2, 0, 5), (2, 3, 0), (0, 3, 5), (2, 0, 0)):
        q, k = (torch.randn(B, 4, n, 16, device="cuda").requires_grad_(True) for n in (Lq, Lk))
        v = torch.randn(B, 4, Lk, 16, device="cuda").requires_grad_(True)
        bias = torch.randn(4, Lq, Lk, device="cuda").requires_grad_(True)
        out = af3.cross_attention(q, k, v, None, bias)
        assert out.shape == q.shape and not out.any()
        for t, g in zip((q, k, v, bias), torch.autograd.grad(out, (q, k, v, bias), torch.ones_like(out))):
            assert g.shape == t.shape and not g.any()


def test_only_the_gradients_asked_for(af3):
    t = make(2, 4, 2, 50, 150, 64, BF16, 22, "ragged", "given")
    everything = run(af3, *t)
    names = ["dq", "dk", "dv", "dbias"]
    for chosen in ([0], [1], [2], [3], [1, 2], [0, 3]):
        leaves = [x.detach().requires_grad_(i in chosen) for i, x in zip((0, 1, 2, 3), (*t[:3], t[4]))]
        out = af3.cross_attention(leaves[0], leaves[1], leaves[2], t[3], leaves[3])
        for i, g in zip(chosen, torch.autograd.grad(out, [leaves[i] for i in chosen], t[5])):
            assert torch.equal(g, everything[names[i]]), names[i]


def test_gradients_agree_with_differences(af3):
    """Central differences of the call itself, in fp32 along one direction of every input at once."""
    q, k, v, m, b, g = make(1, 2, 1, 20, 45, 16, F32, 23, "random", "given")
    got = run(af3, q, k, v, m, b, g)
    gen = torch.Generator().manual_seed(1)
    for name, t in (("dq", q), ("dk", k), ("dv", v), ("dbias", b)):
        way = torch.randn(t.shape, generator=gen).cuda()
        step = 2.0 ** -6

        def at(x):
            args = [x if y is t else y for y in (q, k, v)]
            return (af3.cross_attention(*args, m, x if t is b else b).double() * g.double()).sum().item()
        slope = (at(t + step * way) - at(t - step * way)) / (2 * step)
        want = (got[name].double() * way.double()).sum().item()
        # third derivatives: step^2 / 6 times a sum over 640 outputs of order 10; the function's own fp32 errors divided by the step
        assert abs(slope - want) <= 1e-2 * max(1.0, abs(want)), (name, slope, want)


def test_the_same_bits_every_time(af3):
    for sizes in ((2, 8, 4, 1, 3000, 64), (2, 8, 2, 130, 500, 64), (10, 16, 16, 200, 200, 64)):
        for dtype in (BF16, F32):
            t = make(*sizes, dtype, 31, "ragged", "given")
            first = run(af3, *t)
            for _ in range(3):
                again = run(af3, *t)
                assert all(torch.equal(first[n], again[n]) for n in first)


def test_keys_more_than_4_gb_apart(af3):
    """Rows of k and v far enough apart that offsets pass 32 bits, in elements and bytes."""
    Lk, D, apart = 600, 64, 1 << 23
    room = torch.empty(Lk * apart + D, dtype=BF16, device="cuda")       # 10 GB
    q, k, v, m, b, g = make(1, 2, 2, 40, Lk, D, BF16, 41, "random", "none")
    kk, vv = (room.as_strided((1, 2, Lk, D), (0, 128, apart, 1), at) for at in (0, 1024))
    kk.copy_(k), vv.copy_(v)
    want, got = run(af3, q, k, v, m, b, g), run(af3, q, kk, vv, m, b, g)
    assert all(torch.equal(want[n], got[n]) for n in want)
    del room, kk, vv
    torch.cuda.empty_cache()


def test_streams(af3):
    t = make(4, 8, 8, 100, 400, 64, BF16, 51, "ragged", "given")
    want = run(af3, *t)
    side = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s in side:       # two calls at once, on streams that are not the tensors' own
        with torch.cuda.stream(s):
            got.append(run(af3, *t))
    torch.cuda.synchronize()
    assert all(torch.equal(g[n], want[n]) for g in got for n in want)


def test_captured_and_replayed(af3):
    B, H, Lq, Lk, D = 2, 8, 1, 700, 64
    q, k, v, m, b, g = make(B, H, H, Lq, Lk, D, BF16, 61, "ragged", "given")
    graphs = []
    for _ in range(2):        # two graphs of the same call side by side
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            af3.cross_attention(q, k, v, m, b)
        torch.cuda.current_stream().wait_stream(side)
        gc.collect()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = af3.cross_attention(q, k, v, m, b)
        graphs.append((graph, out))
    for i in range(4):
        q.normal_(), v.normal_()
        want = af3.cross_attention(q, k, v, m, b)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out, want), i


def test_a_training_step_captured_and_replayed(af3):
    q, k, v, m, _, g = make(2, 4, 4, 100, 150, 64, BF16, 62, "ragged", "none")
    table = torch.randn(32, 4, device="cuda", dtype=BF16)

    def step(leaves):
        bias = af3.relative_position_bias(leaves[3], 100, 150)
        out = af3.cross_attention(leaves[0], leaves[1], leaves[2], m, bias)
        return [out.detach(), *torch.autograd.grad(out, leaves, g)]

    data = [q, k, v, table]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step([t.detach().requires_grad_(True) for t in data])
    torch.cuda.current_stream().wait_stream(side)
    static = [t.detach().clone().requires_grad_(True) for t in data]
    gc.collect()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(static)
    for i in range(4):
        with torch.no_grad():
            for t in static:
                t.normal_()
        want = step([t.detach().clone().requires_grad_(True) for t in static])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want)), i


def test_cross_attention_refuses(af3):
    q, k = torch.randn(2, 4, 8, 16, device="cuda"), torch.randn(2, 2, 9, 16, device="cuda")
    for bad, message in [
        (lambda: af3.cross_attention(q.cpu(), k, k), "device"),
        (lambda: af3.cross_attention(q.half(), k, k), "dtype"),
        (lambda: af3.cross_attention(q[0], k, k), "q must be"),
        (lambda: af3.cross_attention(q, k[:1], k[:1]), "k and v must be"),
        (lambda: af3.cross_attention(q, k, k[:, :, :8]), "k and v must be"),
        (lambda: af3.cross_attention(q[:, :3], k, k), "multiple"),
        (lambda: af3.cross_attention(q, k[..., :8], k[..., :8]), "k and v must be"),
        (lambda: af3.cross_attention(torch.randn(1, 1, 2, 130, device="cuda"), torch.randn(1, 1, 2, 130, device="cuda"), torch.randn(1, 1, 2, 130, device="cuda")), "head_dim"),
        (lambda: af3.cross_attention(q, k, k, torch.ones(8, dtype=torch.bool, device="cuda")), "mask"),
        (lambda: af3.cross_attention(q, k, k, torch.ones(3, 9, dtype=torch.bool, device="cuda")), "mask"),
        (lambda: af3.cross_attention(q, k, k, None, torch.randn(4, 8, 8, device="cuda")), "bias"),
        (lambda: af3.cross_attention(q, k, k, None, torch.randn(2, 8, 9, device="cuda")), "bias"),
        (lambda: af3.cross_attention(q, k, k, softmax_scale=0.0), "softmax_scale"),
        (lambda: af3.cross_attention(q, k, k, softmax_scale=float("nan")), "softmax_scale"),
    ]:
        with pytest.raises((ValueError, RuntimeError), match=message):
            bad()


# ---- relative position bias ---------------------------------------------------------------------------------------------------
def bucket(rel, buckets, scheme, both, r):
    """The bucket of key position - query position, in whole numbers."""
    if scheme == "clip":
        return min(max(-rel, -r), r) + r if both else min(max(-rel, 0), r)
    n = buckets // 2 if both else buckets
    first = n if both and rel > 0 else 0
    d = abs(rel) if both else max(-rel, 0)
    near, far = n // 2, n - n // 2
    if d < near:
        return first + d
    i = 0
    while i < far - 1 and d ** far >= r ** (i + 1) * near ** (far - i - 1):
        i += 1
    return first + near + i


SETTINGS = [
    # buckets, scheme, bidirectional, max_distance
    (32, "log", True, 128), (32, "log", False, 128), (64, "log", True, 33), (2, "log", False, 5), (4, "log", True, 2), (16, "log", False, 5000), (576, "log", False, 300),
    (65, "clip", True, 32), (33, "clip", False, 32), (3, "clip", True, 1), (513, "clip", True, 256), (2, "clip", False, 1), (575, "clip", True, 287),
]


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("buckets,scheme,both,r", SETTINGS)
def test_relative_position_bias(af3, buckets, scheme, both, r, dtype):
    gen = torch.Generator().manual_seed(buckets + r)
    for H, Lq, Lk, offset in ((3, 70, 300, 0), (1, 1, 1, 0), (2, 1, 613, 600), (4, 37, 61, -20), (2, 300, 5, 100000)):
        table = torch.randn(buckets, H, generator=gen).to(dtype).cuda().requires_grad_(True)
        grad = torch.randn(H, Lq, Lk, generator=gen).to(dtype).cuda()
        print(buckets, scheme, both, r, (H, Lq, Lk, offset), flush=True)
        out = af3.relative_position_bias(table, Lq, Lk, scheme, both, r, q_offset=offset)
        got = torch.autograd.grad(out, table, grad)[0]
        of = {rel: bucket(rel, buckets, scheme, both, r) for rel in range(-offset - Lq, Lk - offset + 1)}
        b = torch.tensor([[of[j - i - offset] for j in range(Lk)] for i in range(Lq)])
        assert torch.equal(out.cpu(), table.detach().cpu()[b].permute(2, 0, 1)), (H, Lq, Lk)
        assert out.is_contiguous()
        check_sums(got, grad, b, buckets, dtype)


def check_sums(got, grad, b, buckets, dtype):
    g = grad.double().cpu().reshape(grad.shape[0], -1)
    n = torch.zeros(buckets, dtype=torch.float64).index_add_(0, b.reshape(-1), torch.ones(b.numel(), dtype=torch.float64))
    want = torch.zeros(buckets, g.shape[0], dtype=torch.float64).index_add_(0, b.reshape(-1), g.t())
    size = torch.zeros(buckets, g.shape[0], dtype=torch.float64).index_add_(0, b.reshape(-1), g.t().abs())
    bound = n[:, None] * E32 * size + (2.0 ** -8 if dtype == BF16 else E32) * want.abs()
    assert ((got.double().cpu() - want).abs() <= bound + 1e-30).all()


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("buckets,scheme,both,r", [(32, "log", True, 128), (65, "clip", True, 32), (16, "log", False, 5000)])
def test_given_positions(af3, buckets, scheme, both, r, dtype):
    gen = torch.Generator().manual_seed(9)
    H, Lq, Lk = 3, 90, 131
    qp, kp = torch.randint(-50, 400, (Lq,), generator=gen), torch.randint(-50, 400, (Lk,), generator=gen)
    qp[:3], kp[:3] = torch.tensor([2 ** 62, -2 ** 63, 2 ** 63 - 1]), torch.tensor([2 ** 62 - 7, 2 ** 63 - 1, -2 ** 63])
    table = torch.randn(buckets, H, generator=gen).to(dtype).cuda().requires_grad_(True)
    grad = torch.randn(H, Lq, Lk, generator=gen).to(dtype).cuda()
    out = af3.relative_position_bias(table, Lq, Lk, scheme, both, r, q_positions=qp.cuda(), k_positions=kp.cuda())
    got = torch.autograd.grad(out, table, grad)[0]
    known = {}
    def of(rel):
        rel = min(max(rel, -r - 1), r + 1)
        if rel not in known:
            known[rel] = bucket(rel, buckets, scheme, both, r)
        return known[rel]
    b = torch.tensor([[of(j - i) for j in kp.tolist()] for i in qp.tolist()])
    assert torch.equal(out.cpu(), table.detach().cpu()[b].permute(2, 0, 1))
    check_sums(got, grad, b, buckets, dtype)
    # int32, and one side only
    small = qp.clamp(-1000, 1000).to(torch.int32)
    a = af3.relative_position_bias(table, Lq, Lk, scheme, both, r, q_positions=small.cuda())
    c = af3.relative_position_bias(table, Lq, Lk, scheme, both, r, q_positions=small.long().cuda(), k_positions=torch.arange(Lk, device="cuda"))
    assert torch.equal(a, c)
    d = af3.relative_position_bias(table, Lq, Lk, scheme, both, r, q_offset=5)
    e = af3.relative_position_bias(table, Lq, Lk, scheme, both, r, q_offset=5, k_positions=torch.arange(Lk, device="cuda", dtype=torch.int32))
    assert torch.equal(d, e)


def test_position_bias_strides_and_large_sums(af3):
    gen = torch.Generator().manual_seed(10)
    table = torch.randn(8, 32, generator=gen).cuda().t()[:, ::2].requires_grad_(True)      # [32, 4], strides of a transposed slice
    out = af3.relative_position_bias(table, 40, 50)
    plain = table.detach().contiguous().requires_grad_(True)
    assert torch.equal(out, af3.relative_position_bias(plain, 40, 50))
    g = torch.randn(1, 40, 50, generator=gen).cuda().expand(4, 40, 50)
    assert torch.equal(torch.autograd.grad(out, table, g)[0], torch.autograd.grad(af3.relative_position_bias(plain, 40, 50), plain, g.contiguous())[0])
    # millions of terms to a bucket, all of one sign
    big = torch.rand(2, 2000, 2100, generator=gen).cuda()
    plain = torch.randn(32, 2, device="cuda").requires_grad_(True)
    got = torch.autograd.grad(af3.relative_position_bias(plain, 2000, 2100), plain, big)[0].double()
    rel = torch.arange(2100)[None] - torch.arange(2000)[:, None]
    known = torch.tensor([bucket(x, 32, "log", True, 128) for x in range(-130, 131)])
    b = known[rel.clamp(-130, 130) + 130].cuda()
    for h in range(2):
        want = torch.stack([torch.where(b == i, big[h].double(), 0.0).sum() for i in range(32)])
        # 4096 terms at most in a row in fp32, the rest in 64 bits
        assert ((got[:, h] - want).abs() <= 5000 * E32 * want).all()


def test_a_bias_of_more_than_4_billion_entries(af3):
    """Places past 32 bits, in the bias and in its gradient."""
    n = 46400
    table = torch.randn(32, 2, device="cuda", dtype=BF16).requires_grad_(True)
    out = af3.relative_position_bias(table, n, n)                       # 8.6 GB
    assert out.numel() > 2 ** 32
    rows = torch.tensor([0, 1, 12345, n - 2, n - 1])
    known = torch.tensor([bucket(x, 32, "log", True, 128) for x in range(-130, 131)])
    b = known[(torch.arange(n)[None] - rows[:, None]).clamp(-130, 130) + 130].cuda()
    for h in range(2):
        assert torch.equal(out[h, rows.cuda()], table.detach()[:, h][b])
    got = torch.autograd.grad(out, table, torch.ones(1, 1, n, device="cuda", dtype=BF16).expand(2, n, n))[0].double().cpu()
    offsets = torch.arange(-(n - 1), n)
    counts = torch.zeros(32, dtype=torch.float64).index_add_(0, known[offsets.clamp(-130, 130) + 130], (n - offsets.abs()).double())
    assert ((got - counts[:, None]).abs() <= 2.0 ** -8 * counts[:, None]).all()      # ones add up exactly in fp32 as far as a part goes
    del out
    torch.cuda.empty_cache()


def test_relative_position_bias_refuses(af3):
    t = torch.randn(32, 4, device="cuda")
    for bad, message in [
        (lambda: af3.relative_position_bias(t.cpu(), 4, 4), "device"),
        (lambda: af3.relative_position_bias(t[0], 4, 4), "table"),
        (lambda: af3.relative_position_bias(t.half(), 4, 4), "dtype"),
        (lambda: af3.relative_position_bias(t, -1, 4), "q_len"),
        (lambda: af3.relative_position_bias(t, 4, 4, "linear"), "scheme"),
        (lambda: af3.relative_position_bias(t, 4, 4, "clip", True, 32), "buckets"),
        (lambda: af3.relative_position_bias(t[:31], 4, 4), "even"),
        (lambda: af3.relative_position_bias(t, 4, 4, max_distance=8), "max_distance"),
        (lambda: af3.relative_position_bias(t[:2], 4, 4), "max_distance"),
        (lambda: af3.relative_position_bias(t, 4, 4, max_distance=0), "max_distance"),
        (lambda: af3.relative_position_bias(t, 4, 4, q_offset=2 ** 63), "q_offset"),
        (lambda: af3.relative_position_bias(torch.randn(578, 4, device="cuda"), 4, 4), "buckets"),
        (lambda: af3.relative_position_bias(t, 4, 4, q_positions=torch.arange(5, device="cuda")), "q_positions"),
        (lambda: af3.relative_position_bias(t, 4, 4, k_positions=torch.arange(4.0, device="cuda")), "k_positions"),
        (lambda: af3.relative_position_bias(t, 4, 4, q_positions=torch.arange(4)), "device"),
    ]:
        with pytest.raises((ValueError, RuntimeError), match=message):
            bad()
    assert af3.relative_position_bias(t, 0, 4).shape == (4, 0, 4)
    empty = t.clone().requires_grad_(True)
    assert not torch.autograd.grad(af3.relative_position_bias(empty, 3, 0), empty, torch.zeros(4, 3, 0, device="cuda"))[0].any()


# ---- together -------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
def test_an_encoder_layer_and_a_decoder_step(af3, dtype):
    """The table's bias into the attention of a layer and gradients back to the table; then a decoder that takes its tokens one by one gives
    what the whole sequence gives."""
    B, H, L, D = 3, 4, 75, 32
    q, k, v, m, _, g = make(B, H, H, L, L, D, dtype, 71, "ragged", "none")
    table = torch.randn(32, H).to(dtype).cuda()
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, table)]
    bias = af3.relative_position_bias(leaves[3], L, L)
    out = af3.cross_attention(*leaves[:3], m, bias)
    grads = torch.autograd.grad(out, leaves, g)
    want = formula(q, k, v, m, bias, g, D ** -0.5)
    for name, t in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        check(name, t, want[name], dtype)
    b = torch.tensor([[bucket(j - i, 32, "log", True, 128) for j in range(L)] for i in range(L)]).reshape(-1)
    up, uo = (2.0 ** -8, 2.0 ** -8) if dtype == BF16 else (0.0, E32)
    add = lambda t: torch.zeros(32, H, dtype=torch.float64).index_add_(0, b, t.reshape(H, -1).t().contiguous())
    value, bound = want["dbias"]
    limit = add(bound(up, uo)) + (uo + b.numel() * E32) * add(value.abs())
    assert ((grads[3].double().cpu() - add(value)).abs() <= limit + 1e-30).all()
    # single tokens: causal through the keys that exist so far
    causal = torch.full((L, L), -math.inf, device="cuda", dtype=dtype).triu(1)
    one_way = af3.relative_position_bias(table, L, L, bidirectional=False)
    whole = formula(q, k, v, None, one_way + causal, None, D ** -0.5)["out"]
    check("whole", af3.cross_attention(q, k, v, None, one_way + causal), whole, dtype)
    for t in (0, 1, 40, L - 1):
        step = af3.cross_attention(q[:, :, t:t + 1], k[:, :, :t + 1], v[:, :, :t + 1], None, af3.relative_position_bias(table, 1, t + 1, bidirectional=False, q_offset=t))
        check(f"token {t}", step, (whole[0][:, :, t:t + 1], lambda up, uo: whole[1](up, uo)[:, :, t:t + 1]), dtype)


@pytest.mark.parametrize("native", [True, False], ids=["native", "python"])
def test_a_table_behind_bf16_attention_loses_nothing_to_the_biass_gradient(af3, monkeypatch, native):
    """The rows of dS sum to zero, so that a bucket's sum is small beside its terms: rounding each of them to bf16 would be felt.  The bias's own gradient is
    still that of a bf16 tensor, and a bias that was changed on the way takes the plain route."""
    from af3_kernels_amd import cross
    if not native:
        monkeypatch.setattr(cross, "_host", _NoNativeHost())
    B, H, L, D = 4, 4, 200, 64
    q, k, v, m, _, g = make(B, H, H, L, L, D, BF16, 73, "ragged", "none")
    table = torch.randn(32, H).to(BF16).cuda().requires_grad_(True)
    bias = af3.relative_position_bias(table, L, L)
    out = af3.cross_attention(q, k, v, m, bias)
    dbias, dtable = torch.autograd.grad(out, (bias, table), g, retain_graph=True)
    want = formula(q, k, v, m, bias, g, D ** -0.5)
    check("dbias", dbias, want["dbias"], BF16)
    leaf = bias.detach().requires_grad_(True)
    assert torch.equal(dbias, torch.autograd.grad(af3.cross_attention(q, k, v, m, leaf), leaf, g)[0])
    b = torch.tensor([[bucket(j - i, 32, "log", True, 128) for j in range(L)] for i in range(L)]).reshape(-1)
    add = lambda t: torch.zeros(32, H, dtype=torch.float64).index_add_(0, b, t.reshape(H, -1).t().contiguous())
    value, bound = want["dbias"]
    # no rounding of the terms to bf16 (of P or dS neither: dbias is not behind a second product), out known to 16 bits; two sums rounded to bf16, then theirs
    limit = add(bound(0.0, 0.0)) + add(value.abs()) * (2.0 ** -16 + L * L * E32) + 3 * 2.0 ** -8 * add(value).abs() + 2.0 ** -16 * add(value.abs())
    rest = want["out"][1](2.0 ** -8, 2.0 ** -16)      # ... but P was rounded for out, which delta is made of
    x = torch.matmul(q.double().cpu(), spread(k, H).double().cpu().transpose(2, 3)) * D ** -0.5 + bias.detach().double().cpu()
    p = torch.softmax(x.masked_fill(~m.cpu()[:, None, None, :], -math.inf), -1)
    limit = limit + add((p * (g.double().cpu().abs() * rest).sum(-1, keepdim=True)).sum(0))
    assert ((dtable.double().cpu() - add(value)).abs() <= limit).all()
    # (and without the second way: the sums of the rounded gradient)
    changed = torch.autograd.grad(af3.cross_attention(q, k, v, m, bias * 1), table, g)[0]
    assert ((changed.double().cpu() - add(dbias.double().cpu())).abs() <= 2 * 2.0 ** -8 * add(value).abs() + L * L * E32 * add(value.abs()) + 1e-3).all()
    error = lambda t: ((t.double().cpu() - add(value)).norm() / add(value).norm()).item()
    print("table's gradient off by", error(dtable), "and by the plain route", error(changed))


@pytest.mark.parametrize("H,Hkv,Lq,Lk,D", [(2, 2, 200, 200, 64), (2, 1, 9, 1500, 32), (96, 48, 300, 130, 64), (1, 1, 1, 1, 16), (3, 1, 40, 777, 100)])
def test_the_rows_of_the_biass_gradient_sum_to_zero(af3, H, Hkv, Lq, Lk, D):
    """... although delta comes from a result whose probabilities were rounded to bf16: a table's gradient is made of what is left of these sums.  The same bits whether the
    gradients of q, k and v are wanted or not."""
    from af3_kernels_amd import cross
    q, k, v, m, bias, g = make(1, H, Hkv, Lq, Lk, D, BF16, 83, "random", "given")
    scale = D ** -0.5
    out, stats, lost = cross._forward(q, k, v, m, bias, scale, True)
    alone, whole = (cross._backward(g, q, k, v, m, bias, out, stats, lost, scale, (w, w, w, True, True)) for w in (False, True))
    assert all(torch.equal(a, b) for a, b in zip(alone[3:], whole[3:]))
    rows = (alone[3].double() + alone[4].double()).sum(-1).cpu()
    Q, K, V, X, G = (t.double().cpu() for t in (q[0], spread(k, H)[0], spread(v, H)[0], bias, g[0]))
    gone = ~m.cpu().expand(1, Lk)
    x = (torch.matmul(Q, K.transpose(1, 2)) * scale + X).masked_fill(gone, -math.inf)
    size = (torch.matmul(Q.abs(), K.abs().transpose(1, 2)) * scale + X.abs()).masked_fill(gone, 0.0)
    p = torch.softmax(x, -1)
    dp = torch.matmul(G, V.transpose(1, 2))
    delta = (p * dp).sum(-1, keepdim=True)
    ep = 2 * (D + 8) * E32 * size.amax(-1, keepdim=True) + (Lk + 16) * E32
    # P twice (where the row is summed and where dS is made), its sum's distance from one, dP twice, the sum of Lk terms, dbias and its residual rounded to bf16 each
    limit = (p * ((2 * ep + (Lk + 24) * E32) * (dp.abs() + delta.abs()) + 2 * (D + 2) * E32 * torch.matmul(G.abs(), V.abs().transpose(1, 2)) + 2.0 ** -16 * (dp - delta).abs())).sum(-1)
    assert (rows.abs() <= limit).all(), (rows.abs() / limit).max()


@pytest.mark.parametrize("H,L,buckets,scheme,both,r", [(4, 200, 32, "log", True, 128), (1, 17, 3, "clip", True, 1), (3, 131, 575, "clip", True, 287), (2, 301, 16, "log", False, 5000)])
def test_the_sums_of_a_rounded_gradient_and_its_residual_round_once(af3, H, L, buckets, scheme, both, r):
    """What goes to the table directly makes up for both roundings: of the terms, and of the sums that go the usual way."""
    from af3_kernels_amd import cross
    gen = torch.Generator().manual_seed(81)
    exact = torch.randn(H, L, L, generator=gen) - 0.3
    grad = exact.to(BF16)
    rest = (exact - grad.float()).to(BF16)
    settings = (scheme, both, r, 0)
    own, missed = (cross._position_sums(grad.cuda(), x, (buckets, H), settings, None, None).double().cpu() for x in (None, rest.cuda()))
    b = torch.tensor([[bucket(j - i, buckets, scheme, both, r) for j in range(L)] for i in range(L)]).reshape(-1)
    add = lambda t: torch.zeros(buckets, H, dtype=torch.float64).index_add_(0, b, t.double().reshape(H, -1).t().contiguous())
    want, size = add(grad.double() + rest.double()), add(grad.double().abs() + rest.double().abs())
    # the second call's answer rounded to bf16, the terms added in 32 bits
    assert ((own + missed - want).abs() <= 2.0 ** -8 * missed.abs() + 2 * L * L * E32 * size).all()
    assert (missed.abs() <= 2.0 ** -8 * (own.abs() + size) * 1.01 + 2 * L * L * E32 * size).all()
    # sums that are not finite stay what they are
    grad[0, 0, 0] = math.inf
    own, missed = (cross._position_sums(grad.cuda(), x, (buckets, H), settings, None, None).float().cpu() for x in (None, rest.cuda()))
    at = bucket(0, buckets, scheme, both, r)
    assert own[at, 0] == math.inf and missed[at, 0] == 0 and missed.isfinite().all()


def test_the_bias_feeds_the_other_attention_calls(af3, oracle):
    """relative_position_bias into dot_product_attention_cpp, which takes q_len == k_len: the same result as cross_attention's within both bounds."""
    q, k, v, m, _, _ = make(4, 4, 4, 96, 96, 32, F32, 72, "random", "none")
    bias = af3.relative_position_bias(torch.randn(65, 4, device="cuda"), 96, 96, "clip", True, 32)
    a, b = af3.cross_attention(q, k, v, m, bias), af3.dot_product_attention_cpp(q, k, v, m, bias)
    want = oracle.dpa_formula(*(t.cpu().numpy() for t in (q, k, v)), m.cpu().numpy(), bias.cpu().numpy())
    for t in (a, b):
        assert abs(t.cpu().numpy() - want).max() <= 1e-4


# ---- the two host sides, and what autograd may not do ------------------------------------------------------------------------------
class _NoNativeHost:
    def __getattr__(self, name):
        return lambda *args: None


def test_calls_prepared_in_python_give_the_same_bits(af3, monkeypatch):
    from af3_kernels_amd import cross
    for dtype, sizes, bias in ((BF16, (2, 4, 2, 70, 150, 64), "given"), (F32, (3, 2, 2, 1, 400, 32), "none")):
        t = make(*sizes, dtype, 81, "empty", bias)
        table = torch.randn(32, 4, device="cuda", dtype=dtype).requires_grad_(True)
        grad = torch.randn(4, 30, 50, device="cuda", dtype=dtype)
        args = dict(q_positions=torch.arange(30, device="cuda") * 3, k_positions=torch.arange(50, device="cuda") * 2)

        def everything():
            b = af3.relative_position_bias(table, 30, 50, **args)
            return [*run(af3, *t).values(), af3.cross_attention(*t[:5]), b, torch.autograd.grad(b, table, grad)[0]]
        native = everything()
        with monkeypatch.context() as m:
            m.setattr(cross, "_host", _NoNativeHost())
            python = everything()
        assert all(torch.equal(a, b) for a, b in zip(native, python))


@pytest.mark.parametrize("native", [True, False], ids=["native", "python"])
def test_no_second_derivative(af3, monkeypatch, native):
    from af3_kernels_amd import cross
    if not native:
        monkeypatch.setattr(cross, "_host", _NoNativeHost())
    q = torch.randn(1, 2, 4, 16, device="cuda").requires_grad_(True)
    g = torch.autograd.grad(af3.cross_attention(q, q, q).sum(), q, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="second derivative" if native else None):
        g.sum().backward()
    with pytest.raises(RuntimeError):       # (not a gradient that is silently zero either)
        torch.autograd.grad(g.sum(), q)
    table = torch.randn(32, 2, device="cuda").requires_grad_(True)
    g = torch.autograd.grad(af3.relative_position_bias(table, 4, 4).sum(), table, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="second derivative" if native else None):
        g.sum().backward()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), table)


def test_inputs_changed_between_forward_and_backward_are_noticed(af3):
    q, k, v, m, b, g = make(1, 2, 2, 10, 20, 16, F32, 82, "random", "given")
    q.requires_grad_(True)
    for t in (k, m):
        out = af3.cross_attention(q, k, v, m, b)
        t.zero_()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(out, q, g)


def test_a_table_may_change_before_its_gradient_is_taken(af3):
    table = torch.randn(32, 2, device="cuda", dtype=BF16).requires_grad_(True)
    q = torch.randn(1, 2, 30, 16, device="cuda", dtype=BF16)
    bias = af3.relative_position_bias(table, 30, 30)
    out = af3.cross_attention(q, q, q, None, bias)
    want = torch.autograd.grad(out.sum(), table, retain_graph=True)[0]
    with torch.no_grad():
        table.mul_(2)
    assert torch.equal(torch.autograd.grad(out.sum(), table)[0], want)
    # the bias's graph is freed now: another call with it works, its gradient does not
    again = af3.cross_attention(q, q, q, None, bias)
    with pytest.raises(RuntimeError, match="second time"):
        again.sum().backward()


@pytest.mark.parametrize("native", [True, False], ids=["native", "python"])
def test_a_table_changed_in_place_behind_its_bias(af3, monkeypatch, native):
    """The bias's gradient goes to what the table was, not to what it became: the same bits as with a table of its own for each."""
    from af3_kernels_amd import cross
    if not native:
        monkeypatch.setattr(cross, "_host", _NoNativeHost())
    q, k, v, _, _, g = make(2, 2, 2, 60, 60, 32, BF16, 84)
    w = torch.randn(32, 2, dtype=BF16).cuda().requires_grad_(True)
    table = w * 1
    bias = af3.relative_position_bias(table, 60, 60)
    table.mul_(1000)
    got = torch.autograd.grad(af3.cross_attention(q, k, v, None, bias), w, g)[0]
    want = torch.autograd.grad(af3.cross_attention(q, k, v, None, af3.relative_position_bias(w, 60, 60) * 1), w, g)[0]
    assert torch.equal(got, want)


@pytest.mark.parametrize("native", [True, False], ids=["native", "python"])
def test_a_capture_that_would_wait_for_another_stream_is_refused(af3, monkeypatch, native):
    """The leaf's gradient is accumulated on the default stream while an eager result holds the leaf: captured, that would end the process."""
    from af3_kernels_amd import cross

    class Only:
        check_capture = staticmethod(cross._host.check_capture)

        def __getattr__(self, name):
            return lambda *args: None
    if not native:
        monkeypatch.setattr(cross, "_host", Only())
    q = torch.randn(1, 2, 4, 16, device="cuda").requires_grad_(True)
    table = torch.randn(32, 2, device="cuda").requires_grad_(True)
    eager = af3.cross_attention(q, q, q), af3.relative_position_bias(table, 4, 4)
    refused = 0
    gc.collect()      # (a graph that the collector frees while another is captured ends the process; for the same reason no exception, and with it this frame, is kept here)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: af3.cross_attention(q, q, q), lambda: af3.cross_attention(q * 2, q.detach(), q.detach()), lambda: af3.relative_position_bias(table, 4, 4)):
            with pytest.raises(RuntimeError, match="captured"):
                call()
            refused += 1
        plain = af3.cross_attention(q.detach(), q.detach(), q.detach())      # a call without a gradient is captured as ever
    assert refused == 3
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(plain, eager[0])
    del eager


# ---- the table's gradient behind bf16 attention: rounded once where the bias's gradient arrives as the call made it ----------------------
def _table_case(seed, B=3, H=4, L=90, D=32):
    q, k, v, m, _, g = make(B, H, H, L, L, D, BF16, seed, "ragged", "none")
    gen = torch.Generator().manual_seed(seed + 1)
    return q, k, v, m, g, torch.randn(32, H, generator=gen).to(BF16).cuda().requires_grad_(True)


def _plain_sums(af3, table, grad):
    """The sums by bucket of a bias's gradient as it stands, in bfloat16."""
    bias = af3.relative_position_bias(table, *grad.shape[1:])
    return torch.autograd.grad(bias, table, grad)[0]


def test_a_tables_gradient_with_one_attention_call_is_rounded_once(af3):
    """own + missed: the sums of the bias's gradient, and what they and that gradient lost.  In every way of asking for it."""
    from af3_kernels_amd import cross
    q, k, v, m, g, table = _table_case(91)
    bias = af3.relative_position_bias(table, 90, 90)
    out = af3.cross_attention(q, k, v, m, bias)
    keep, scale = m.view(torch.uint8), 32 ** -0.5
    kernel = cross._forward(q, k, v, keep, bias.detach(), scale, True)
    grads = cross._backward(g, q, k, v, keep, bias.detach(), *kernel, scale, (False, False, False, True, True))
    settings = ("log", True, 128, 0)
    own, missed = (cross._position_sums(grads[3], x, table.shape, settings, None, None) for x in (None, grads[4]))
    want = own + missed
    assert not torch.equal(own, want)
    once = torch.autograd.grad(out, table, g, retain_graph=True)[0]
    assert torch.equal(once, want) and torch.equal(torch.autograd.grad(out, table, g, retain_graph=True)[0], want)
    both = torch.autograd.grad(out, (bias, table), g, retain_graph=True)
    assert torch.equal(both[0], grads[3]) and torch.equal(both[1], want)
    # the bias's gradient alone, and then the table's from it: a gradient like any other
    dbias = torch.autograd.grad(out, bias, g, retain_graph=True)[0]
    assert torch.equal(dbias, grads[3]) and torch.equal(torch.autograd.grad(bias, table, dbias, retain_graph=True)[0], own)
    bias.retain_grad()
    out.backward(g, retain_graph=True)
    assert torch.equal(bias.grad, grads[3]) and torch.equal(table.grad, want)
    # a gradient that has a graph is made of the one that arrives
    graph = torch.autograd.grad(out, table, g, create_graph=True)[0]
    assert torch.equal(graph, own)


@pytest.mark.parametrize("where", ["tensor", "node", "attention"])
@pytest.mark.parametrize("change", ["zeros", "in place", "behind torch's back", "one head", "half", "none"])
def test_a_hook_on_the_biass_gradient_has_the_last_word(af3, where, change):
    q, k, v, m, g, table = _table_case(92)
    bias = af3.relative_position_bias(table, 90, 90)
    out = af3.cross_attention(q, k, v, m, bias)
    dbias = torch.autograd.grad(out, bias, g, retain_graph=True)[0].clone()

    def changed(t):
        if change == "zeros":
            return torch.zeros_like(t)
        if change == "in place":
            t.zero_()
            return None
        if change == "behind torch's back":      # no version counter sees this
            t.data.zero_()
            return None
        if change == "one head":
            return torch.cat([torch.zeros_like(t[:1]), t[1:]])
        return t * 0.5 if change == "half" else None

    arrives = dbias.clone()
    replaced = changed(arrives)
    arrives = arrives if replaced is None else replaced
    if where == "tensor":
        bias.register_hook(changed)
    elif where == "node":
        def before(grads):
            new = changed(grads[0])
            return None if new is None else (new,)
        bias.grad_fn.register_prehook(before)
    else:
        def after(grads, _):
            new = changed(grads[3])
            return None if new is None else (*grads[:3], new, *grads[4:])
        out.grad_fn.register_hook(after)
    got = torch.autograd.grad(out, table, g)[0]
    assert torch.equal(got, _plain_sums(af3, table, arrives))
    if change in ("zeros", "in place", "behind torch's back"):
        assert not got.any()
    if change == "one head":
        assert not got[:, 0].any() and got[:, 1:].any()


@pytest.mark.parametrize("native", [True, False], ids=["native", "python"])
@pytest.mark.parametrize("layers", [2, 3, 12])
def test_a_bias_that_a_stack_of_layers_shares(af3, monkeypatch, layers, native):
    """The bias's gradients are added in bf16 before the table sees them: its gradient is the sums of what arrives, to the bit."""
    from af3_kernels_amd import cross
    if not native:
        monkeypatch.setattr(cross, "_host", _NoNativeHost())
    q, k, v, m, g, table = _table_case(93)

    def stack(bias):
        x = q
        for _ in range(layers):
            x = af3.cross_attention(x, k, v, m, bias)
        return x
    bias = af3.relative_position_bias(table, 90, 90)
    got = torch.autograd.grad(stack(bias), (bias, table), g)
    plain = af3.relative_position_bias(table, 90, 90)
    want = torch.autograd.grad(stack(plain * 1), (plain, table), g)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(got[1], _plain_sums(af3, table, got[0]))


def test_a_bias_that_something_else_has_too(af3):
    q, k, v, m, g, table = _table_case(94)
    w = torch.randn(4, 90, 90, device="cuda", dtype=BF16)
    for order in (0, 1):
        bias = af3.relative_position_bias(table, 90, 90)
        parts = [lambda: (af3.cross_attention(q, k, v, m, bias).float() * g.float()).sum(), lambda: (bias * w).float().sum()]
        loss = parts[order]() + parts[1 - order]()
        dbias, got = torch.autograd.grad(loss, (bias, table))
        assert torch.equal(got, _plain_sums(af3, table, dbias))


def test_a_bias_of_another_stream(af3):
    """The bias is made on one stream, the attention runs on another: the same bits, also where memory is handed round at once."""
    q, k, v, m, g, table = _table_case(95)
    want = torch.autograd.grad(af3.cross_attention(q, k, v, m, af3.relative_position_bias(table, 90, 90)), table, g)[0]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(10):
        bias = af3.relative_position_bias(table, 90, 90)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            out = af3.cross_attention(q, k, v, m, bias)
            got = torch.autograd.grad(out, table, g)[0]
            torch.full_like(bias, 1e4), torch.full_like(bias, -1e4)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want)


def test_a_table_that_is_changed_by_what_its_bias_led_to_is_freed(af3):
    """Nothing in the bias's graph holds the table's own: in place, that would be a circle."""
    import weakref
    w = torch.randn(32, 2, device="cuda", dtype=BF16).requires_grad_(True)
    table = w * 1
    bias = af3.relative_position_bias(table, 40, 40)
    table.add_(bias.float().mean().to(BF16))
    gone = weakref.ref(table)
    node = table.grad_fn
    seen = []
    node.metadata["witness"] = type("witness", (), {"__del__": lambda self: seen.append(1)})()
    del table, bias, node
    gc.collect()
    assert gone() is None and seen == [1]


def test_a_tables_gradient_does_not_depend_on_how_its_calls_come(af3):
    """int32 positions, lengths of another integer type, masks of numbers, other types of k and v, other strides: each call is prepared in Python first and
    gives the bits that the plain ones give together, whichever of the two it is."""
    import numpy
    q, k, v, m, g, table = _table_case(96)
    at = torch.arange(90, device="cuda")
    plain = (lambda: af3.relative_position_bias(table, 90, 90, q_positions=at, k_positions=at), lambda b: af3.cross_attention(q, k, v, m, b))

    def gradient(bias, attend):
        return torch.autograd.grad(attend(bias()), table, g)[0]
    want = gradient(*plain)
    assert not torch.equal(want, gradient(plain[0], lambda b: plain[1](b * 1)))
    biases = {"int32 positions": lambda: af3.relative_position_bias(table, 90, 90, q_positions=at.int(), k_positions=at.int()),
              "numpy lengths": lambda: af3.relative_position_bias(table, numpy.int64(90), numpy.int64(90), q_positions=at, k_positions=at)}
    odd = q.transpose(2, 3).contiguous().transpose(2, 3)
    attends = {"a mask of numbers": lambda b: af3.cross_attention(q, k, v, m.int(), b), "a mask of rank 4": lambda b: af3.cross_attention(q, k, v, m.float()[:, None, None, :], b),
               "keys in fp32": lambda b: af3.cross_attention(q, k.float(), v, m, b), "other strides": lambda b: af3.cross_attention(odd, k, v, m, b),
               "a scale of numpy's": lambda b: af3.cross_attention(q, k, v, m, b, softmax_scale=numpy.float64(32 ** -0.5))}
    for name, bias in biases.items():
        assert torch.equal(gradient(bias, plain[1]), want), name
    for name, attend in attends.items():
        assert torch.equal(gradient(plain[0], attend), want), name
    assert torch.equal(gradient(biases["int32 positions"], attends["a mask of numbers"]), want)


@pytest.mark.parametrize("native", [True, False], ids=["native", "python"])
def test_no_forward_mode(af3, monkeypatch, native):
    """A result without a tangent would say that it does not depend on the input; with and without a graph of its own."""
    from torch.autograd import forward_ad
    from af3_kernels_amd import cross
    if not native:
        monkeypatch.setattr(cross, "_host", _NoNativeHost())
    q, k, v, m, b, _ = make(1, 2, 2, 10, 20, 16, F32, 97, "random", "given")
    table = torch.randn(32, 2, device="cuda")
    want = af3.cross_attention(q, k, v, m, b), af3.relative_position_bias(table, 4, 5)
    for requires_grad in (False, True):
        with forward_ad.dual_level():
            for name, t in {"q": q, "k": k, "v": v, "bias": b}.items():
                dual = forward_ad.make_dual(t.detach().requires_grad_(requires_grad), torch.ones_like(t))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    af3.cross_attention(**({"q": q, "k": k, "v": v, "mask": m, "bias": b} | {name: dual}))
            dual = forward_ad.make_dual(table.detach().requires_grad_(requires_grad), torch.ones_like(table))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                af3.relative_position_bias(dual, 4, 5)
            # (a call without tangents runs inside such a context as ever)
            assert torch.equal(af3.cross_attention(q, k, v, m, b), want[0]) and torch.equal(af3.relative_position_bias(table, 4, 5), want[1])
    leaf, leaf_table = q.detach().requires_grad_(True), table.detach().requires_grad_(True)
    for out, x in ((af3.cross_attention(leaf, k, v, m, b), leaf), (af3.relative_position_bias(leaf_table, 4, 5), leaf_table)):
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(out, x, dual)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: af3.cross_attention(x, k, v, m, b), (q,), (q,))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda x: af3.cross_attention(x, k, v, m, b))(q[None])


@pytest.mark.parametrize("native", [True, False], ids=["native", "python"])
def test_sizes_without_a_gradient(af3, monkeypatch, native):
    """Refused before the forward pass, not behind it; without a graph such calls run."""
    from af3_kernels_amd import cross
    if not native:
        monkeypatch.setattr(cross, "_host", _NoNativeHost())
    n = 64 * 4096
    q, k = (torch.zeros(1, 1, 1, 8, device="cuda", dtype=BF16).expand(1, 1, n, 8) for _ in range(2))
    bias = torch.zeros(1, 1, n, device="cuda", dtype=BF16).requires_grad_(True)
    with pytest.raises(ValueError, match="gradient of a bias"):
        af3.cross_attention(q, k, k, None, bias.expand(1, n, n))
    leaf = torch.zeros(1 << 10, 4, 1, 8, device="cuda", dtype=BF16).requires_grad_(True)
    many = torch.ones(1, 1, 1, 8, device="cuda", dtype=BF16).expand(1 << 10, 4, 1 << 17, 8)
    with pytest.raises(ValueError, match="Hkv"):
        af3.cross_attention(leaf, many, many)
    assert (af3.cross_attention(leaf.detach(), many, many) == 1).all()


def test_without_the_native_host_no_gradient_is_captured(af3, monkeypatch, tmp_path):
    from af3_kernels_amd import _lib, cross
    monkeypatch.setattr(_lib, "HOST_PATH", str(tmp_path / "_host.so"))
    monkeypatch.setattr(_lib._Host, "_warned", True)
    monkeypatch.setattr(cross, "_host", _lib._Host())
    q, table = torch.randn(1, 2, 4, 16, device="cuda"), torch.randn(32, 2, device="cuda")
    want = af3.cross_attention(q, q, q, None, af3.relative_position_bias(table, 4, 4))
    leaf, leaf_table = q.clone().requires_grad_(True), table.clone().requires_grad_(True)
    refused = 0
    gc.collect()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: af3.cross_attention(leaf, q, q), lambda: af3.relative_position_bias(leaf_table, 4, 4)):
            with pytest.raises(RuntimeError, match="native host side"):
                call()
            refused += 1
        plain = af3.cross_attention(q, q, q, None, af3.relative_position_bias(table, 4, 4))
    assert refused == 2
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(plain, want)
    # ... and outside of a capture it flows
    assert torch.autograd.grad(af3.cross_attention(leaf, q, q).sum(), leaf)[0].isfinite().all()


def test_a_captured_gradient_of_what_was_made_outside_is_refused(af3):
    """The leaves' gradients belong to the capturing stream here, an operation between them and the call does not: it would run on its own stream, which is not captured."""
    capturing, aside = torch.cuda.Stream(), torch.cuda.Stream()
    q, k = torch.randn(1, 2, 4, 16, device="cuda").requires_grad_(True), torch.randn(1, 2, 5, 16, device="cuda")
    table = torch.randn(32, 2, device="cuda").requires_grad_(True)
    torch.cuda.synchronize()
    with torch.cuda.stream(capturing):
        held = q * 1, table * 1            # the leaves come into a graph here first
    torch.cuda.synchronize()
    outside = [q * 2, af3.relative_position_bias(table, 4, 5)]
    with torch.cuda.stream(aside):
        outside.append(q * 3)
    torch.cuda.synchronize()
    want = af3.cross_attention(outside[0].detach(), k, k, None, outside[1].detach())
    calls = [lambda: af3.cross_attention(outside[0], k, k), lambda: af3.cross_attention(q.detach(), k, k, None, outside[1]), lambda: af3.cross_attention(outside[2], k, k),
             lambda: af3.relative_position_bias(table * 1 + held[1].sum() + outside[1].sum(), 4, 5)]
    refused = 0
    gc.collect()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=capturing):
        for call in calls:
            with pytest.raises(RuntimeError, match="outside of the capture"):
                call()
            refused += 1
        plain = af3.cross_attention(outside[0].detach(), k, k, None, outside[1].detach())
        # recorded on another stream of the same capture: taken
        aside.wait_stream(capturing)
        with torch.cuda.stream(aside):
            branch = q * 2
        capturing.wait_stream(aside)
        assert af3.cross_attention(branch, k, k).requires_grad
    assert refused == 4
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(plain, want)
    del held, outside


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("B,H,Hkv,Lq,Lk,D,live", [
    # whole rows in one workgroup, which goes through them in two stretches of 16384 keys, in every kernel
    (64, 8, 8, 1, 20000, 16, [0, 5, 9000, 16383, 16384, 16500, 19999]),
    (64, 8, 8, 3, 17000, 32, [16383, 16384]),
    (64, 8, 8, 1, 33000, 8, [40, 16384, 32767, 32768]),      # three of them
    (16, 16, 16, 200, 17000, 32, [16383, 16384, 16400]),     # 128 rows to a workgroup
    # a key axis in parts: live keys in a few of them, at their ends among others
    (1, 2, 2, 1, 40000, 64, [3, 639, 640, 5000, 20011, 39999]),
    (1, 4, 2, 20, 40000, 128, [0, 12799, 12800, 33333]),
    (2, 2, 1, 3, 17000, 32, [100, 16384, 16999]),
])
def test_few_live_keys_of_a_long_axis(af3, B, H, Hkv, Lq, Lk, D, live, dtype):
    """Few enough that each of them shows: a result without any one of them is off by more than it may be (of the formula's own results; nothing is planted in the kernels)."""
    gen = torch.Generator("cuda").manual_seed(98)
    n = lambda *s: torch.randn(s, generator=gen, device="cuda", dtype=dtype)
    q, k, v, b, g = n(B, H, Lq, D), n(B, Hkv, Lk, D), n(B, Hkv, Lk, D), n(H, Lq, Lk), n(B, H, Lq, D)
    mask = torch.zeros(B, Lk, dtype=torch.bool, device="cuda")
    mask[:, live] = True
    got = run(af3, q, k, v, mask, b, g)
    few = lambda keys: formula(q, k[:, :, keys], v[:, :, keys], None, b[:, :, keys], g, D ** -0.5)
    want = few(live)
    up, uo = (2.0 ** -8, 2.0 ** -8) if dtype == BF16 else (0.0, E32)
    for name in ("dk", "dv", "dbias"):
        rest = got[name].clone()
        rest.index_fill_(2, torch.tensor(live, device="cuda"), 0.0)
        assert not rest.any(), name
        got[name] = got[name][:, :, live]
    for name, t in got.items():
        check(name, t, want[name], dtype)
    for gone in range(len(live)):
        others = few(live[:gone] + live[gone + 1:])
        for name in ("out", "dq"):
            value, bound = want[name]
            assert ((others[name][0] - value).abs() > bound(up, uo)).any(), (name, live[gone])
        for name in ("dk", "dv", "dbias"):
            value, bound = want[name]
            assert (value.abs() > bound(up, uo))[:, :, gone].any(), (name, live[gone])


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("far", [3000.0, 1e5, 1e7, 1e9, 1e10, 1e20, 1e30, 3.3e38])
@pytest.mark.parametrize("sign", [1, -1], ids=["high", "low"])
def test_rows_whose_logits_are_all_far_from_zero(af3, dtype, far, sign):
    """A bias that is the same for all keys of a query changes nothing, and keys that lie far below the others have no weight: -1e9 as a mask of a padded query, say.
    The queries are zeros there, so that every logit is the bias, to the bit, and P what it is without it."""
    c = torch.tensor(sign * far).to(dtype)
    for B, H, Hkv, Lq, Lk, D in ((2, 2, 2, 40, 150, 32), (1, 2, 1, 1, 1700, 64), (2, 2, 2, 64, 300, 128), (9, 16, 16, 140, 150, 64), (9, 16, 4, 300, 70, 128)):
        q, k, v, m, b, g = make(B, H, Hkv, Lq, Lk, D, dtype, 99, "ragged", "given")
        rows = torch.arange(0, Lq, 3, device="cuda")
        q[:, 0, rows] = 0.0
        plain = b.clone()
        for bias, here, there in ((b, c, c / 2 if sign > 0 else c * 2), (plain, 0.0, -math.inf)):
            bias[0, rows] = here
            bias[0, rows[:, None], torch.arange(1, Lk, 2, device="cuda")] = there
        print((B, H, Hkv, Lq, Lk, D), flush=True)
        got = run(af3, q, k, v, m, b, g)
        want = formula(q, k, v, m, plain, g, D ** -0.5)
        for name, t in got.items():
            check(name, t, want[name], dtype)
