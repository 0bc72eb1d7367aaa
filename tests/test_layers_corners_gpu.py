"""The layer operators where little or nothing is left: results that no gradient reaches, values far below one, queries without a key.

Formulas, bounds and inputs are those of test_layers_gpu.py.
"""
import math

import pytest
import torch

from test_layers_gpu import BF16, HOSTS, NAMES, TYPES, af3, diff_compare, diff_inputs, diff_run, host, norm_inputs  # noqa: F401

pytestmark = pytest.mark.gpu


class Drops(torch.autograd.Function):
    """A consumer through which no gradient flows back."""
    @staticmethod
    def forward(ctx, *tensors):
        ctx.count = len(tensors)
        return sum(t.double().sum() for t in tensors)

    @staticmethod
    def backward(ctx, grad):
        return (None,) * ctx.count


def dropped(results, leaves):
    """The leaves' gradients behind `Drops`, with memory of their sizes in the allocator's hands that holds NaN."""
    junk = [torch.full_like(t, math.nan) for t in leaves for _ in range(4)]
    torch.cuda.synchronize()
    del junk
    return torch.autograd.grad(Drops.apply(*results), leaves, allow_unused=True)


@HOSTS
@TYPES
def test_residual_norm_of_which_no_gradient_comes(af3, host, native, dtype):
    host(native)
    for kw in ({"post_norm": "layer"}, {"post_norm": "rms", "gate_activation": "sigmoid"}):
        t, _ = norm_inputs((2, 6, 100), dtype, 34, bias="channel", gate="batch", post=True)
        leaves = [t[n].detach().requires_grad_(True) for n in NAMES]
        got = dropped(af3.residual_norm(*leaves, **kw), leaves)
        for name, leaf, g in zip(NAMES, leaves, got):
            assert g is None or (g.shape == leaf.shape and (g == 0).all()), name
    # one result alone, and parameters of which nothing is wanted
    x, y = (t[n].detach().requires_grad_(True) for n in ("x", "y"))
    assert all(g is None or (g == 0).all() for g in dropped(af3.residual_norm(x, y, norm="none")[:1], [x, y]))
    assert all(g is None or (g == 0).all() for g in dropped(af3.residual_norm(x, y.detach(), t["weight"]), [x]))


@HOSTS
@TYPES
def test_other_layers_of_which_no_gradient_comes(af3, host, native, dtype):
    host(native)
    f, _ = af3.rotary_frequencies(32, device="cuda")
    q, k = (torch.randn(2, h, 9, 32, device="cuda").to(dtype).requires_grad_(True) for h in (4, 2))
    assert all(g is None or (g == 0).all() for g in dropped(af3.rotary_embedding(q, k, f), [q, k]))
    leaves = [t.detach().requires_grad_(True) for t in diff_inputs(2, 4, 2, 9, 40, 32, 64, dtype, 35)[:4]]
    assert all(g is None or (g == 0).all() for g in dropped([af3.differential_attention(*leaves)], leaves))


# ---- values far below one -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("few", [True, False], ids=["few keys", "most keys"])
@pytest.mark.parametrize("Lq,B", [(1, 2), (40, 2), (640, 9)])
def test_small_values_and_smaller_columns(af3, Lq, B, few):
    """A column of V 2^-14 of the others is as exact where V is small as where it is not, in calls of every length.

    (Held as fp16 in units of a tile whose largest value is at least 2^8 units, a value is off by 2^-25 units: 2^-33 of the tile's largest, which is below 5 standard deviations here: 1.3 times 2^-17 of the
    column's own, within the 2^-17 of the column's largest of 128 keys that the bound has.)"""
    q, k, v, lam, m, _ = diff_inputs(B, 4, 4, Lq, 400, 64, 128, BF16, 41, "random")
    if few:
        m &= torch.rand(m.shape, generator=torch.Generator().manual_seed(1)).cuda() < 0.03
        m[:, 7] = True
    v[..., ::3] *= 2.0 ** -14
    for unit in (1.0, 2.0 ** -5, 2.0 ** -11, 2.0 ** -16, 2.0 ** -17, 1e-9, 2.0 ** 20):
        t = (q, k, (v * unit).to(BF16), lam, m, None)
        diff_compare({"out": af3.differential_attention(*t[:5])}, *t)


@pytest.mark.parametrize("Lq,B", [(1, 2), (40, 2), (640, 9)])
def test_zeros_beside_the_smallest_values(af3, Lq, B):
    """A tile of V that holds nothing but zeros says nothing of the sizes of others."""
    q, k, v, lam, m, _ = diff_inputs(B, 4, 4, Lq, 400, 64, 128, BF16, 42, "random")
    for unit in (2.0 ** -60, 2.0 ** -70, 2.0 ** -85):
        for zeros in (slice(0, 128), slice(128, 256), slice(256, 400)):
            small = (v * unit).to(BF16)
            small[:, :, zeros] = 0.0
            t = (q, k, small, lam, m, None)
            diff_compare({"out": af3.differential_attention(*t[:5])}, *t)


# ---- queries without a key ----------------------------------------------------------------------------------------------------
@HOSTS
@TYPES
@pytest.mark.parametrize("Lq,Lk,B", [(1, 40, 2), (1, 5000, 2), (16, 40, 3), (40, 70, 2), (40, 5000, 2), (640, 150, 9)])
def test_queries_without_a_key_whatever_lam_is(af3, host, native, Lq, Lk, B, dtype):
    host(native)
    q, k, v, _, _, _ = diff_inputs(B, 4, 4, Lq, Lk, 64, 128, dtype, 43)
    m = torch.ones(B, Lk, dtype=torch.bool, device="cuda")
    m[1] = False
    for worst in (math.inf, -math.inf, math.nan):
        out = af3.differential_attention(q, k, v, torch.full((4,), worst, device="cuda"), m)
        assert (out[1] == 0).all(), worst


@TYPES
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("Lq,Lk,B", [(1, 40, 2), (40, 700, 2), (640, 150, 9)])
def test_gradients_of_queries_without_a_key_whatever_lam_is(af3, Lq, Lk, B, D, dtype):
    D = D if dtype == BF16 else min(D, 64)
    q, k, v, _, _, g = diff_inputs(B, 4, 4, Lq, Lk, D, 2 * D, dtype, 44)
    m = torch.ones(B, Lk, dtype=torch.bool, device="cuda")
    m[1] = False
    for worst in (math.inf, math.nan):
        got = diff_run(af3, q, k, v, torch.full((4,), worst, device="cuda"), m, g)
        for name in ("out", "dq", "dk", "dv"):
            assert (got[name][1] == 0).all(), (name, worst)


@TYPES
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("Lq,Lk,B", [(8, 40, 2), (8, 5000, 2), (40, 70, 2), (40, 5000, 2), (640, 400, 9)])
def test_queries_without_a_key_beside_values_that_are_not_finite(af3, Lq, Lk, B, D, dtype):
    D = D if dtype == BF16 else min(D, 64)
    q, k, v, lam, _, _ = diff_inputs(B, 4, 4, Lq, Lk, D, 2 * D, dtype, 45)
    for worst in (math.nan, math.inf):
        v2 = v.clone()
        v2[:, :, ::3] = worst
        out = af3.differential_attention(q, k, v2, lam, causal=True, q_offset=-5)
        assert (out[:, :, :5] == 0).all(), worst
        # a sequence that is padded in front: its first queries see dropped keys alone
        m = torch.ones(B, Lk, dtype=torch.bool, device="cuda")
        m[-1, :5] = False
        out = af3.differential_attention(q, k, v2, lam, m, causal=True)
        assert (out[-1, :, :5] == 0).all(), worst


@TYPES
@pytest.mark.parametrize("H,Hkv,Lq,Lk,B,D", [(4, 4, 8, 40, 2, 64), (4, 2, 40, 70, 3, 32), (4, 4, 150, 150, 9, 64), (8, 8, 300, 300, 9, 64), (4, 1, 130, 130, 2, 128), (6, 2, 260, 700, 9, 32), (8, 8, 260, 600, 9, 128)])
def test_queries_without_a_key_have_no_part_in_a_gradient(af3, H, Hkv, Lq, Lk, B, D, dtype):
    D = D if dtype == BF16 else min(D, 64)
    q, k, v, lam, _, g = diff_inputs(B, H, Hkv, Lq, Lk, D, 2 * D, dtype, 46)
    padded = torch.ones(B, Lk, dtype=torch.bool, device="cuda")
    padded[0, :6] = False
    padded[-1, :3] = False
    for m, kw, dead in ((None, dict(causal=True, q_offset=-5), [5] * B), (padded, dict(causal=True), [6] + [0] * (B - 2) + [3])):
        gone = (torch.arange(Lq)[None] < torch.tensor(dead)[:, None]).cuda()[:, None, :, None]
        clean = diff_run(af3, q, k, v, lam, m, g, **kw)
        diff_compare(clean, q, k, v, lam, m, g, **kw)
        for worst in (math.nan, math.inf):
            dirty = diff_run(af3, q.masked_fill(gone, worst), k, v, lam, m, g.masked_fill(gone, worst), **kw)
            for name in clean:
                assert torch.equal(clean[name], dirty[name]), (name, worst)
            assert (dirty["dq"].masked_select(gone) == 0).all() and (dirty["out"].masked_select(gone) == 0).all()


# ---- one lam for all heads ----------------------------------------------------------------------------------------------------
@HOSTS
def test_one_lam_of_few_bits_for_all_heads(af3, host, native):
    """Its gradient is a sum over heads, and rounded once."""
    host(native)
    for seed in range(16):
        q, k, v, lam, m, g = diff_inputs(2, 8, 4, 30, 40, 32, 64, BF16, 47 + seed, "random")
        for form in (lam[:1], lam[0]):
            few = form.detach().to(BF16).requires_grad_(True)
            more = few.detach().float().requires_grad_(True)
            a, b = (af3.differential_attention(q, k, v, x, m) for x in (few, more))
            assert torch.equal(a, b)
            a, b = torch.autograd.grad(a, few, g)[0], torch.autograd.grad(b, more, g)[0]
            assert a.dtype == BF16 and torch.equal(a, b.to(BF16))


# ---- many queries of few keys -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("D,Dv", [(64, 128), (32, 1), (24, 64), (128, 7)])
@pytest.mark.parametrize("Lk", [1, 2, 15, 63, 64, 65, 127, 130])
def test_many_queries_of_few_keys(af3, Lk, D, Dv):
    """Long calls whose keys do not fill a tile, with masks that leave a sequence empty or hold back most of its keys."""
    for seed, mask in ((51, "none"), (52, "empty"), (53, "one")):
        t = diff_inputs(9, 8, 8, 530, Lk, D, Dv, BF16, seed, mask)
        for unit in (1.0, 2.0 ** -13):
            few = (t[0], t[1], (t[2] * unit).to(BF16), *t[3:])
            diff_compare({"out": af3.differential_attention(*few[:5])}, *few)
    diff_compare(diff_run(af3, *t, causal=True, q_offset=-3), *t, causal=True, q_offset=-3)
