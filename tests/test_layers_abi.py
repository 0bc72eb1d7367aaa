"""The C entry points of rotary positions, differential attention and the norms around a block, as far as the host goes: layouts, refusals, workspaces; and the frequencies.  No GPU."""
import ctypes
import math
import os
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
i64x3 = ctypes.c_int64 * 3
BASE = 1 << 40   # (addresses that nothing follows)


@pytest.fixture
def lib():
    from af3_kernels_amd import _lib
    return _lib.load()


def _put(p, values):
    for name, value in values.items():
        setattr(p, name, value)
    return p


def _diff(B=2, H=4, Hkv=2, Lq=50, Lk=70, D=32, Dv=64, **kw):
    from af3_kernels_amd import _lib
    return _put(_lib.DiffAttentionParams(q=BASE, k=2 * BASE, v=3 * BASE, lam=4 * BASE, out=5 * BASE, stats=6 * BASE, second=7 * BASE, B=B, H=H, Hkv=Hkv, Lq=Lq, Lk=Lk, D=D, Dv=Dv,
                                         q_stride=i64x3(2 * H * Lq * D, Lq * D, D), k_stride=i64x3(2 * Hkv * Lk * D, Lk * D, D), v_stride=i64x3(Hkv * Lk * Dv, Lk * Dv, Dv),
                                         out_stride=i64x3(H * Lq * Dv, Lq * Dv, Dv), lam_stride=1, dtype=_lib.AF3_BF16, lam_dtype=_lib.AF3_F32, softmax_scale=0.25,
                                         workspace=BASE, workspace_bytes=1 << 50), kw)


def _diff_grads(**kw):
    from af3_kernels_amd import _lib
    return _put(_lib.DiffAttentionGrads(grad_out=8 * BASE, grad_out_stride=i64x3(12800, 3200, 64), grad_q=9 * BASE, grad_k=10 * BASE, grad_v=11 * BASE, grad_lam=12 * BASE,
                                        workspace=13 * BASE, workspace_bytes=1 << 50), kw)


def _rotary(B=2, L=5, D=16, rotary=16, heads=(4, 2), **kw):
    from af3_kernels_amd import _lib
    p = _lib.RotaryParams(frequencies=BASE, B=B, L=L, D=D, rotary=rotary, dtype=_lib.AF3_BF16, scale=1.0)
    for i in range(2):
        p.x[i], p.out[i], p.heads[i] = (2 + i) * BASE, (4 + i) * BASE, heads[i]
        p.x_stride[i] = p.out_stride[i] = i64x3(max(heads[i], 1) * L * D, L * D, D)
    return _put(p, kw)


def _norm(rows=6, C=64, **kw):
    from af3_kernels_amd import _lib
    return _put(_lib.ResidualNormParams(x=BASE, y=2 * BASE, out=3 * BASE, normed=4 * BASE, stats=5 * BASE, rows=rows, C=C, x_stride=C, y_stride=C, norm=_lib.NORMS["rms"],
                                        dtype=_lib.AF3_F32, eps=1e-5, residual_scale=1.0), kw)


def _norm_grads(C=64, **kw):
    from af3_kernels_amd import _lib
    return _put(_lib.ResidualNormGrads(grad_out=6 * BASE, grad_normed=7 * BASE, grad_out_stride=C, grad_normed_stride=C, grad_y=8 * BASE, workspace=9 * BASE, workspace_bytes=1 << 50), kw)


def test_struct_mirrors_match_what_a_c_compiler_lays_out(tmp_path):
    from af3_kernels_amd import _lib
    mirrors = {"af3_diff_attention_params": _lib.DiffAttentionParams, "af3_diff_attention_grads": _lib.DiffAttentionGrads, "af3_rotary_params": _lib.RotaryParams,
               "af3_residual_norm_params": _lib.ResidualNormParams, "af3_residual_norm_grads": _lib.ResidualNormGrads}
    values = {"AF3_ROTARY_MAX_HEAD_DIM": _lib.ROTARY_MAX_HEAD_DIM, "AF3_RESIDUAL_NORM_MAX_CHANNELS": _lib.RESIDUAL_NORM_MAX_CHANNELS, "AF3_DIFF_ATTENTION_GRAD_ROW_BYTES": _lib.DIFF_ATTENTION_GRAD_ROW_BYTES,
              "AF3_NORM_NONE": _lib.NORMS["none"], "AF3_NORM_RMS": _lib.NORMS["rms"], "AF3_NORM_LAYER": _lib.NORMS["layer"], "AF3_SHARE_CHANNEL": _lib.SHARE_CHANNEL,
              "AF3_SHARE_GROUP": _lib.SHARE_GROUP, "AF3_SHARE_ROW": _lib.SHARE_ROW}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "af3_dpa.h"', "int main(void) {"]
    for name, cls in mirrors.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    lines += [f'printf("{name} %d\\n", (int){name});' for name in values] + ["return 0; }"]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    found = dict(l.rsplit(" ", 1) for l in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.splitlines())
    for name, cls in mirrors.items():
        assert int(found[name]) == ctypes.sizeof(cls)
        for f, _ in cls._fields_:
            assert int(found[f"{name}.{f}"]) == getattr(cls, f).offset, (name, f)
    for name, value in values.items():
        assert int(found[name]) == value, name


def test_differential_attention_validates_on_the_host(lib):
    from af3_kernels_amd import _lib
    fwd = lambda p: lib.af3_diff_attention_forward(ctypes.byref(p), None)
    size = lambda p: lib.af3_diff_attention_workspace_bytes(ctypes.byref(p))
    assert lib.af3_diff_attention_forward(None, None) == -1
    for name in ("q", "k", "v", "lam", "out"):
        assert fwd(_diff(**{name: None})) == -1, name
    assert fwd(_diff(stats=None)) == -1 and fwd(_diff(second=None)) == -1      # both or neither
    assert fwd(_diff(dtype=_lib.AF3_FP8_E4M3)) == -2 and fwd(_diff(lam_dtype=_lib.AF3_FP8_E4M3)) == -2
    assert fwd(_diff(dtype=_lib.AF3_F32, residuals=BASE)) in (-1, -2)          # (nothing is lost)
    for name in ("B", "H", "Hkv", "Lq", "Lk", "D", "Dv"):
        for value in (0, -1):
            assert fwd(_diff(**{name: value})) in (-3, -5) and size(_diff(**{name: value})) in (-3, -5), name
    assert fwd(_diff(H=4, Hkv=3)) == -3
    for over in ({"Lk": 1 << 30}, {"Lq": 1 << 30}, {"H": 1 << 15, "Hkv": 1}, {"H": 1 << 14, "Hkv": 1, "Lq": 1 << 16}, {"B": 1 << 24}, {"B": 1 << 12, "Lk": 1 << 17}):
        assert fwd(_diff(**over)) == -3 and size(_diff(**over)) == -3, over
    assert size(_diff(B=1 << 12, Lk=1 << 17, stats=None, second=None)) >= 0    # (a forward pass alone takes more keys)
    for D, Dv, dtype in ((129, 64, _lib.AF3_BF16), (64, 257, _lib.AF3_BF16), (65, 64, _lib.AF3_F32), (64, 129, _lib.AF3_F32)):
        assert fwd(_diff(D=D, Dv=Dv, dtype=dtype)) == -5
    for name in ("q_stride", "k_stride", "v_stride", "out_stride"):
        assert fwd(_diff(**{name: i64x3(-1, 64, 64)})) == -4, name
    for shared in (i64x3(12800, 3200, 63), i64x3(0, 3200, 64), i64x3(12800, 0, 64)):      # results that share a place
        assert fwd(_diff(out_stride=shared)) == -4
    assert fwd(_diff(lam_stride=-1)) == -4 and fwd(_diff(key_mask=BASE, key_mask_stride_b=-1)) == -4
    for scale in (0.0, -1.0, math.inf, math.nan):
        assert fwd(_diff(softmax_scale=scale)) == -7
    assert fwd(_diff(causal=1, q_offset=1 << 40)) in (-3, -7) and fwd(_diff(causal=1, q_offset=-(1 << 40))) in (-3, -7)
    # one query over many keys needs room for the parts' results, rows that are not 16 bytes apart for themselves
    for p in (lambda **kw: _diff(B=1, H=2, Lq=1, Lk=40000, **kw), lambda **kw: _diff(D=31, **kw), lambda **kw: _diff(B=40, Lq=1000, **kw)):
        need = size(p())
        assert need > 0 and need % 4 == 0
        for bad in ({"workspace": None}, {"workspace": BASE + 4}, {"workspace_bytes": need - 1}):
            assert fwd(p(**bad)) == -7, bad


def test_differential_attention_backward_validates_on_the_host(lib):
    bwd = lambda p, g: lib.af3_diff_attention_backward(ctypes.byref(p), ctypes.byref(g), None)
    assert lib.af3_diff_attention_backward(ctypes.byref(_diff()), None, None) == -1
    assert bwd(_diff(stats=None, second=None), _diff_grads()) == -1
    assert bwd(_diff(), _diff_grads(grad_out=None)) == -1
    assert bwd(_diff(), _diff_grads(grad_q=None, grad_k=None, grad_v=None, grad_lam=None)) == -1
    assert bwd(_diff(), _diff_grads(grad_out_stride=i64x3(1, -1, 1))) == -4
    assert bwd(_diff(), _diff_grads(grad_out_stride=i64x3(64, 64, 1 << 23), workspace=None)) == -4
    assert bwd(_diff(), _diff_grads(grad_out_stride=i64x3(64, 64, (1 << 23) - 1), workspace=None)) == -7
    assert bwd(_diff(Lq=0), _diff_grads()) == -3
    need = lib.af3_diff_attention_backward_workspace_bytes(ctypes.byref(_diff()))
    assert need >= 2 * 4 * 50 * 4 * 2
    for bad in ({"workspace": None}, {"workspace": BASE + 8}, {"workspace_bytes": need - 1}):
        assert bwd(_diff(), _diff_grads(**bad)) == -7
    assert lib.af3_diff_attention_backward_workspace_bytes(ctypes.byref(_diff(D=0))) in (-3, -5)


def test_differential_attention_sizes_at_their_limits(lib):
    size = lambda **kw: lib.af3_diff_attention_workspace_bytes(ctypes.byref(_diff(**kw)))
    back = lambda **kw: lib.af3_diff_attention_backward_workspace_bytes(ctypes.byref(_diff(**kw)))
    full = 1 << 24
    for under, over in (({"B": full // 4 - 1, "H": 4, "Hkv": 1, "Lq": 32, "Lk": 1}, {"B": full // 4, "H": 4, "Hkv": 1, "Lq": 32, "Lk": 1}),
                        ({"B": (1 << 23) - 1, "H": 1, "Hkv": 1, "Lq": 20, "Lk": 1}, {"B": 1 << 23, "H": 1, "Hkv": 1, "Lq": 20, "Lk": 1}),
                        ({"B": 1, "H": (1 << 15) - 1, "Hkv": 1, "Lq": 1, "Lk": 1}, {"B": 1, "H": 1 << 15, "Hkv": 1, "Lq": 1, "Lk": 1}),
                        ({"B": 1, "H": 511, "Hkv": 1, "Lq": 1 << 20, "Lk": 1}, {"B": 1, "H": 1 << 10, "Hkv": 1, "Lq": 1 << 20, "Lk": 1}),
                        ({"B": 1, "H": 1, "Hkv": 1, "Lq": 1, "Lk": (1 << 29) - 32}, {"B": 1, "H": 1, "Hkv": 1, "Lq": 1, "Lk": 1 << 30})):
        assert size(**under) >= 0 and back(**under) > 0, under
        assert size(**over) == -3 and back(**over) == -3, over


def test_rotary_validates_on_the_host(lib):
    from af3_kernels_amd import _lib
    call = lambda p: lib.af3_rotary_embedding(ctypes.byref(p), None)
    assert lib.af3_rotary_embedding(None, None) == -1 and call(_rotary(frequencies=None)) == -1
    for i in range(2):
        for name in ("x", "out"):
            p = _rotary()
            getattr(p, name)[i] = None
            assert call(p) == -1, (name, i)
    assert call(_rotary(dtype=_lib.AF3_FP8_E4M3)) == -2
    for bad in ({"B": 0}, {"L": 0}, {"D": 0}, {"rotary": 0}, {"rotary": 3}, {"rotary": 18}, {"D": 1025}, {"heads": (0, 2)}, {"heads": (4, -1)}, {"heads": (1 << 15, 1 << 15)}, {"B": 1 << 15, "L": 1 << 15}):
        assert call(_rotary(**bad)) in (-3, -5), bad
    for name in ("x_stride", "out_stride"):
        p = _rotary()
        getattr(p, name)[0] = i64x3(64, -16, 16)
        assert call(p) == -4, name
    p = _rotary(positions=BASE, position_stride_b=-1)
    assert call(p) == -4
    for bad in ({"scale": math.inf}, {"scale": math.nan}, {"offset": (1 << 62) + 1}, {"offset": -(1 << 62) - 1}):
        assert call(_rotary(**bad)) == -7, bad


def test_residual_norm_validates_on_the_host(lib):
    from af3_kernels_amd import _lib
    fwd = lambda p: lib.af3_residual_norm_forward(ctypes.byref(p), None)
    bwd = lambda p, g: lib.af3_residual_norm_backward(ctypes.byref(p), ctypes.byref(g), None)
    assert lib.af3_residual_norm_forward(None, None) == -1
    for name in ("y", "out", "normed"):
        assert fwd(_norm(**{name: None})) == -1, name
    assert fwd(_norm(dtype=_lib.AF3_FP8_E4M3)) == -2
    for bad in ({"rows": 0}, {"rows": 1 << 30}, {"C": 0}, {"C": 16385}):
        assert fwd(_norm(**bad)) in (-3, -5), bad
    assert fwd(_norm(x_stride=-1)) == -4 and fwd(_norm(y_stride=-1)) == -4
    for bad in ({"norm": 3}, {"norm": -1}, {"post_norm": 3}, {"eps": -1.0}, {"eps": math.nan}, {"eps": math.inf}, {"residual_scale": math.inf}, {"gate": BASE}, {"gate": BASE, "gate_share": 4},
                {"gate_share": 1}, {"weight": BASE}, {"norm": 0, "weight": BASE, "weight_share": 1}, {"post_weight": BASE}, {"gate": BASE, "gate_share": _lib.SHARE_GROUP, "group": 4},
                {"gate": BASE, "gate_share": _lib.SHARE_GROUP, "group": 0}):
        assert fwd(_norm(**bad)) < 0, bad
    assert fwd(_norm(stats=5 * BASE + 8)) == -7
    assert bwd(_norm(stats=None), _norm_grads()) == -1
    assert bwd(_norm(), _norm_grads(grad_out=None, grad_normed=None)) == -1
    assert bwd(_norm(), _norm_grads(grad_y=None)) == -1
    assert bwd(_norm(), _norm_grads(grad_out_stride=-1)) == -4
    shared = dict(weight=BASE, weight_share=_lib.SHARE_CHANNEL)
    assert bwd(_norm(**shared), _norm_grads(grad_normed=None, grad_weight=BASE)) < 0
    for wanted in ({"grad_x": BASE, "x": None}, {"grad_gate": BASE}, {"grad_weight": BASE}, {"grad_bias": BASE}, {"grad_post_weight": BASE}):       # gradients of what is not there
        params = {k: v for k, v in wanted.items() if k == "x"}
        assert bwd(_norm(**params), _norm_grads(**{k: v for k, v in wanted.items() if k != "x"})) == -1, wanted
    p, g = _norm(**shared), _norm_grads(grad_weight=BASE)
    need = lib.af3_residual_norm_backward_workspace_bytes(ctypes.byref(p), ctypes.byref(g))
    assert need > 0 and lib.af3_residual_norm_backward_workspace_bytes(ctypes.byref(_norm()), ctypes.byref(_norm_grads())) == 0
    for bad in ({"workspace": None}, {"workspace": BASE + 8}, {"workspace_bytes": need - 1}):
        assert bwd(p, _norm_grads(grad_weight=BASE, **bad)) == -7, bad


def test_wrappers_reject_cpu_tensors():
    import af3_kernels_amd as af3
    q = torch.zeros(1, 2, 2, 8)
    for call in (lambda: af3.rotary_embedding(q, q, torch.zeros(4, dtype=torch.float64)), lambda: af3.differential_attention(q, q, q[:, :1], torch.zeros(1)), lambda: af3.residual_norm(q, q)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_forward_mode_is_refused():
    import af3_kernels_amd as af3
    from torch.autograd import forward_ad
    a = torch.randn(1, 2, 3, 8)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(a, torch.ones_like(a))
        for call in (lambda: af3.rotary_embedding(a, d, torch.zeros(4, dtype=torch.float64)), lambda: af3.differential_attention(a, a, d[:, :1], torch.zeros(1)), lambda: af3.residual_norm(d, a),
                     lambda: af3.residual_norm(None, a, gate=d)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_rotary_frequencies():
    from af3_kernels_amd import rotary_frequencies
    f, scale = rotary_frequencies(8)
    assert scale == 1.0 and f.dtype == torch.float64 and f.tolist() == [10000.0 ** (-i / 4) for i in range(4)]
    assert rotary_frequencies(8, 500.0)[0].tolist() == [500.0 ** (-i / 4) for i in range(4)]
    assert rotary_frequencies(8, scaling="linear", factor=4.0)[0].tolist() == [x / 4.0 for x in f.tolist()]
    n = rotary_frequencies(8, scaling="ntk", factor=4.0)[0]
    assert n[0] == 1.0 and abs(n[3] * 4.0 / f[3] - 1.0) < 1e-14        # the slowest by the factor, the fastest not at all
    # "yarn": fast pairs as they are, slow ones by the factor, a ramp between; the scale
    f = rotary_frequencies(128)[0]
    y, scale = rotary_frequencies(128, scaling="yarn", factor=8.0, original_length=4096)
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(y[turns > 33], f[turns > 33]) and torch.allclose(y[turns < 0.9], f[turns < 0.9] / 8.0, rtol=1e-14)
    ratio = y / f
    assert ((ratio[1:] - ratio[:-1]) <= 1e-15).all() and scale == 0.1 * math.log(8.0) + 1.0
    same, one = rotary_frequencies(128, scaling="yarn", factor=1.0, original_length=4096)
    assert torch.allclose(same, f, rtol=1e-15) and one == 1.0
    # nothing is slowed where every pair turns often enough, everything where none does
    assert torch.allclose(rotary_frequencies(16, scaling="yarn", factor=4.0, original_length=1 << 30)[0][:-1], rotary_frequencies(16)[0][:-1], rtol=1e-14)
    assert torch.allclose(rotary_frequencies(16, scaling="yarn", factor=4.0, original_length=1)[0][1:], rotary_frequencies(16)[0][1:] / 4.0, rtol=1e-14)
    for args, kw in (((7,), {}), ((0,), {}), ((1026,), {}), ((8, 1.0), {}), ((8, math.inf), {}), ((8, math.nan), {}), ((8,), {"scaling": "ntk-aware"}), ((8,), {"factor": 2.0}),
                     ((8,), {"scaling": "linear", "factor": 0.5}), ((8,), {"scaling": "linear", "factor": math.nan}), ((2,), {"scaling": "ntk", "factor": 2.0}),
                     ((8,), {"scaling": "yarn", "factor": 2.0}), ((8,), {"scaling": "yarn", "factor": 2.0, "original_length": 64, "beta_fast": 1.0, "beta_slow": 2.0})):
        with pytest.raises(ValueError):
            rotary_frequencies(*args, **kw)


def test_sizes_without_a_gradient_are_refused_before_the_forward_pass(monkeypatch):
    import af3_kernels_amd as af3
    from af3_kernels_amd import layers
    monkeypatch.setattr(layers, "_same_device", lambda *t: None)
    thin = lambda *shape: torch.zeros(1).expand(*shape)
    q = torch.zeros(1 << 10, 8, 1, 8).requires_grad_(True)
    with pytest.raises(ValueError, match="gradients take"):
        af3.differential_attention(q, thin(1 << 10, 8, 1 << 17, 8), thin(1 << 10, 4, 1 << 17, 8), torch.zeros(4))
