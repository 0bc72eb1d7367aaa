"""The layer operators where little or nothing is left.

Formulas, bounds and inputs are those of test_layers_gpu.py.
"""
import math

import pytest
import torch

from test_layers_gpu import HOSTS, NAMES, TYPES, af3, diff_inputs, host, norm_inputs  # noqa: F401

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
