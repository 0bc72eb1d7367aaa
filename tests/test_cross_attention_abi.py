"""The C entry points of cross attention and of the relative position bias, as far as the host goes: layouts, refusals, workspaces.  No GPU."""
import ctypes
import math
import os
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
i64x2, i64x3 = ctypes.c_int64 * 2, ctypes.c_int64 * 3
BASE = 1 << 40   # (addresses that nothing follows)


def _cross(B=2, H=4, Hkv=2, Lq=50, Lk=70, D=32, **kw):
    from af3_kernels_amd import _lib
    p = _lib.CrossAttentionParams(q=BASE, k=2 * BASE, v=3 * BASE, out=4 * BASE, stats=5 * BASE, B=B, H=H, Hkv=Hkv, Lq=Lq, Lk=Lk, D=D,
                                  q_stride=i64x3(H * Lq * D, Lq * D, D), k_stride=i64x3(Hkv * Lk * D, Lk * D, D), v_stride=i64x3(Hkv * Lk * D, Lk * D, D),
                                  out_stride=i64x3(H * Lq * D, Lq * D, D), dtype=_lib.AF3_BF16, softmax_scale=0.25)
    for name, value in kw.items():
        setattr(p, name, value)
    return p


def _grads(**kw):
    from af3_kernels_amd import _lib
    g = _lib.CrossAttentionGrads(grad_out=6 * BASE, grad_out_stride=i64x3(6400, 1600, 32), grad_q=7 * BASE, grad_k=8 * BASE, grad_v=9 * BASE, workspace=10 * BASE, workspace_bytes=1 << 40)
    for name, value in kw.items():
        setattr(g, name, value)
    return g


def _position(buckets=32, H=4, Lq=10, Lk=20, scheme=0, bidirectional=1, max_distance=128, **kw):
    from af3_kernels_amd import _lib
    p = _lib.PositionBiasParams(table=BASE, out=2 * BASE, grad=3 * BASE, table_stride=i64x2(H, 1), grad_stride=i64x2(Lq * Lk, Lk), buckets=buckets, H=H, Lq=Lq, Lk=Lk,
                                max_distance=max_distance, scheme=scheme, bidirectional=bidirectional, dtype=_lib.AF3_F32, workspace=4 * BASE, workspace_bytes=1 << 40)
    for name, value in kw.items():
        setattr(p, name, value)
    return p


def test_struct_mirrors_match_what_a_c_compiler_lays_out(tmp_path):
    from af3_kernels_amd import _lib
    mirrors = {"af3_cross_attention_params": _lib.CrossAttentionParams, "af3_cross_attention_grads": _lib.CrossAttentionGrads, "af3_position_bias_params": _lib.PositionBiasParams}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "af3_dpa.h"', "int main(void) {"]
    for name, cls in mirrors.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    lines.append('printf("buckets %d\\n", AF3_POSITION_BIAS_MAX_BUCKETS); return 0; }')
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    found = dict(l.rsplit(" ", 1) for l in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.splitlines())
    for name, cls in mirrors.items():
        assert int(found[name]) == ctypes.sizeof(cls)
        for f, _ in cls._fields_:
            assert int(found[f"{name}.{f}"]) == getattr(cls, f).offset, (name, f)
    assert int(found["buckets"]) == _lib.POSITION_BIAS_MAX_BUCKETS


def test_cross_attention_validates_on_the_host():
    from af3_kernels_amd import _lib
    lib = _lib.load()
    fwd = lambda p: lib.af3_cross_attention_forward(ctypes.byref(p), None)
    assert lib.af3_cross_attention_forward(None, None) == -1
    for name in ("q", "k", "v", "out"):
        assert fwd(_cross(**{name: None})) == -1
    assert fwd(_cross(dtype=_lib.AF3_FP8_E4M3)) == -2
    for name in ("B", "H", "Hkv", "Lq", "Lk", "D"):
        for value in (0, -1):
            assert fwd(_cross(**{name: value})) in (-3, -5), name
    assert fwd(_cross(H=4, Hkv=3)) == -3
    assert fwd(_cross(Lk=1 << 30)) == -3
    assert fwd(_cross(B=1 << 24)) == -3
    assert fwd(_cross(Lq=1 << 29, H=64, Hkv=64)) == -3
    assert fwd(_cross(D=129)) == -5
    for name in ("q_stride", "k_stride", "v_stride", "out_stride"):
        assert fwd(_cross(**{name: i64x3(-1, 32, 32)})) == -4
    for shared in (i64x3(6400, 1600, 31), i64x3(0, 1600, 32), i64x3(6400, 0, 32)):      # results that share a place
        assert fwd(_cross(out_stride=shared)) == -4
    assert fwd(_cross(bias=BASE, bias_stride=i64x2(-1, 1))) == -4
    assert fwd(_cross(key_mask=BASE, key_mask_stride_b=-1)) == -4
    for scale in (0.0, -1.0, math.inf, math.nan):
        assert fwd(_cross(softmax_scale=scale)) == -7
    # one query over many keys needs room for the parts' results
    long = _cross(B=1, H=2, Lq=1, Lk=40000)
    need = lib.af3_cross_attention_workspace_bytes(ctypes.byref(long))
    assert need > 0 and need % 4 == 0 and fwd(long) == -7
    long.workspace, long.workspace_bytes = BASE, need - 1
    assert fwd(long) == -7
    long.workspace, long.workspace_bytes = BASE + 4, need
    assert fwd(long) == -7
    assert lib.af3_cross_attention_workspace_bytes(ctypes.byref(_cross(B=64, H=16, Hkv=16, Lq=512))) == 0
    assert lib.af3_cross_attention_workspace_bytes(ctypes.byref(_cross(D=0))) == -3


def test_cross_attention_backward_validates_on_the_host():
    from af3_kernels_amd import _lib
    lib = _lib.load()
    bwd = lambda p, g: lib.af3_cross_attention_backward(ctypes.byref(p), ctypes.byref(g), None)
    assert lib.af3_cross_attention_backward(ctypes.byref(_cross()), None, None) == -1
    assert bwd(_cross(stats=None), _grads()) == -1
    assert bwd(_cross(), _grads(grad_out=None)) == -1
    assert bwd(_cross(), _grads(grad_q=None, grad_k=None, grad_v=None)) == -1
    assert bwd(_cross(), _grads(grad_bias=BASE)) == -1          # the gradient of a bias that is not there
    assert bwd(_cross(bias=BASE), _grads(grad_bias_residual=BASE)) == -1      # what the rounding of no gradient lost
    assert bwd(_cross(), _grads(grad_out_stride=i64x3(1, -1, 1))) == -4
    assert bwd(_cross(Lq=0), _grads()) == -3
    need = lib.af3_cross_attention_backward_workspace_bytes(ctypes.byref(_cross()))
    assert need >= 2 * 4 * 50 * 4
    assert bwd(_cross(), _grads(workspace_bytes=need - 1)) == -7
    assert bwd(_cross(), _grads(workspace=None)) == -7
    assert bwd(_cross(), _grads(workspace=BASE + 8)) == -7
    assert bwd(_cross(H=1 << 15, Hkv=1, B=1, Lq=1 << 15, Lk=1 << 28, bias=BASE), _grads(grad_bias=BASE)) == -3


def test_position_bias_validates_on_the_host():
    from af3_kernels_amd import _lib
    lib = _lib.load()
    fwd, bwd = (lambda p, f=f: f(ctypes.byref(p), None) for f in (lib.af3_position_bias_forward, lib.af3_position_bias_backward))
    for call in (fwd, bwd):
        assert call(_position(dtype=_lib.AF3_FP8_E4M3)) == -2
        for bad in ({"buckets": 0}, {"buckets": 577}, {"H": 0}, {"H": 1 << 16}, {"Lq": 0}, {"Lk": 1 << 30}):
            assert call(_position(**bad)) == -3, bad
        assert call(_position(table_stride=i64x2(-1, 1))) == -4
        for bad in ({"max_distance": 0}, {"max_distance": 1 << 30}, {"max_distance": 8}, {"scheme": 2}, {"buckets": 31}, {"buckets": 2}, {"buckets": 1, "bidirectional": 0},
                    {"scheme": 1, "max_distance": 32}, {"scheme": 1, "max_distance": 32, "buckets": 64}, {"q_offset": (1 << 62) + 1}, {"q_offset": -(1 << 62) - 1}):
            assert call(_position(**bad)) == -7, bad
        assert call(_position(out=None)) == -1
    assert lib.af3_position_bias_forward(None, None) == -1 and lib.af3_position_bias_backward(None, None) == -1
    assert fwd(_position(table=None)) == -1
    assert bwd(_position(grad=None)) == -1 and bwd(_position(workspace=None)) == -1
    assert bwd(_position(grad_stride=i64x2(-1, 1))) == -4
    assert bwd(_position(table_stride=i64x2(0, 1))) == -4 and bwd(_position(table_stride=i64x2(1, 0))) == -4
    need = lib.af3_position_bias_workspace_bytes(ctypes.byref(_position()))
    assert need > 0 and bwd(_position(workspace_bytes=need - 1)) == -7 and bwd(_position(workspace=BASE + 4)) == -7
    # with what the gradient's rounding lost: room for both sums, and half the heads at most
    both = lib.af3_position_bias_workspace_bytes(ctypes.byref(_position(grad_residual=5 * BASE)))
    assert both == 2 * need and bwd(_position(grad_residual=5 * BASE, workspace_bytes=both - 1)) == -7
    for call in (bwd, lambda p: lib.af3_position_bias_workspace_bytes(ctypes.byref(p))):
        assert call(_position(grad_residual=5 * BASE, H=1 << 15)) == -3


def test_wrappers_reject_cpu_tensors():
    import af3_kernels_amd as af3
    q = torch.zeros(1, 1, 2, 8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        af3.cross_attention(q, q, q)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        af3.relative_position_bias(torch.zeros(32, 1), 2, 2)


def test_a_stale_library_says_so_and_does_not_keep_the_package_from_being_imported(tmp_path):
    """A library built before a symbol was added: importing works (or `python -m af3_kernels_amd.build` could not), calls raise."""
    import shutil
    import sys
    copy = tmp_path / "af3_kernels_amd"
    shutil.copytree(os.path.join(ROOT, "af3_kernels_amd"), copy, ignore=shutil.ignore_patterns("csrc", "*.so", "__pycache__"))
    (tmp_path / "old.c").write_text("int af3_abi_version(void) { return 4; }")
    subprocess.run(["gcc", "-shared", "-fPIC", str(tmp_path / "old.c"), "-o", str(copy / "libaf3_dpa.so")], check=True)
    (copy / "_host.so").write_bytes(b"")
    code = "import af3_kernels_amd as a\ntry:\n    a._lib.load()\nexcept ImportError as e:\n    print('said:', 'rebuild' in str(e))"
    r = subprocess.run([sys.executable, "-c", code], cwd=tmp_path, capture_output=True, text=True)
    assert r.returncode == 0 and "said: True" in r.stdout, r.stdout + r.stderr


def test_forward_mode_is_refused():
    """A tangent would be lost without a word: refused before anything else is looked at."""
    import af3_kernels_amd as af3
    from torch.autograd import forward_ad
    plain = {"q": torch.randn(1, 2, 3, 8), "k": torch.randn(1, 2, 4, 8), "v": torch.randn(1, 2, 4, 8), "bias": torch.randn(2, 3, 4)}
    with forward_ad.dual_level():
        for name, t in plain.items():
            args = plain | {name: forward_ad.make_dual(t, torch.ones_like(t))}
            with pytest.raises(NotImplementedError, match="forward-mode"):
                af3.cross_attention(**args)
        table = torch.randn(32, 2)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            af3.relative_position_bias(forward_ad.make_dual(table, torch.ones_like(table)), 3, 4)


def test_sizes_at_their_limits():
    """The limits that the header states, from either side; nothing is launched (size queries, and calls that lack their workspace)."""
    from af3_kernels_amd import _lib
    lib = _lib.load()
    ws = lambda **kw: lib.af3_cross_attention_workspace_bytes(ctypes.byref(_cross(**kw)))
    gws = lambda **kw: lib.af3_cross_attention_backward_workspace_bytes(ctypes.byref(_cross(**kw)))
    bwd = lambda g, **kw: lib.af3_cross_attention_backward(ctypes.byref(_cross(**kw)), ctypes.byref(_grads(workspace=None, **g)), None)
    full = 1 << 24
    for under, over in (({"B": full // 2 - 1, "H": 2, "Hkv": 1, "Lq": 32, "Lk": 1}, {"B": full // 2, "H": 2, "Hkv": 1, "Lq": 32, "Lk": 1}),
                        ({"B": 1, "H": 255, "Hkv": 1, "Lq": 1 << 21, "Lk": 1}, {"B": 1, "H": 256, "Hkv": 1, "Lq": 1 << 21, "Lk": 1}),
                        ({"B": 1, "H": 255, "Hkv": 1, "Lq": 1 << 21, "Lk": 1}, {"B": 1, "H": 255, "Hkv": 1, "Lq": (1 << 21) + (1 << 15), "Lk": 1}),
                        ({"B": 255, "H": 65535, "Hkv": 1, "Lq": 1, "Lk": 1}, {"B": 1, "H": 65536, "Hkv": 1, "Lq": 1, "Lk": 1}),
                        ({"B": 1, "H": 1, "Hkv": 1, "Lq": 1, "Lk": (1 << 29) - 32}, {"B": 1, "H": 1, "Hkv": 1, "Lq": 1, "Lk": 1 << 30})):
        assert ws(**under) >= 0 and gws(**under) > 0 and bwd({}, **under) == -7, under
        assert ws(**over) == -3 and gws(**over) == -3 and bwd({}, **over) == -3, over
    # keys: a forward pass alone takes more of them than one with its gradient
    under, over = ({"B": 1 << 10, "H": 4, "Hkv": 4, "Lq": 1, "Lk": n} for n in ((1 << 17) - 32, 1 << 17))
    assert ws(**under) >= 0 and gws(**under) > 0 and bwd({}, **under) == -7
    assert ws(**over) == -3 and gws(**over) == -3 and bwd({}, **over) == -3 and lib.af3_cross_attention_forward(ctypes.byref(_cross(**over)), None) == -3
    assert ws(stats=None, **over) >= 0 and gws(stats=None, **over) == -3
    # a bias's gradient: tiles of 64 x 64 for every head
    under, over = ({"B": 1, "H": 1, "Hkv": 1, "Lq": 64 * n, "Lk": 64 * 4096, "bias": BASE} for n in (4095, 4096))
    for sizes, wanted, rc in ((under, BASE, -7), (over, BASE, -3), (over, None, -7)):
        assert ws(**sizes) >= 0 and gws(**sizes) > 0 and bwd({"grad_bias": wanted}, **sizes) == rc


def test_sizes_without_a_gradient_are_refused_before_the_forward_pass():
    from af3_kernels_amd import cross
    thin = lambda *shape: torch.zeros(1).expand(*shape)
    q, k = thin(1, 2, 64, 8), thin(1, 2, 64, 8)
    cross._check_gradient(q, k, None)
    cross._check_gradient(thin(1 << 10, 4, 1, 8), thin(1 << 10, 4, (1 << 17) - 32, 8), None)
    with pytest.raises(ValueError, match="Hkv"):
        cross._check_gradient(thin(1 << 10, 4, 1, 8), thin(1 << 10, 4, 1 << 17, 8), None)
    long, longer = thin(1, 1, 64 * 4095, 8), thin(1, 1, 64 * 4096, 8)
    leaf = torch.zeros(1, 1, 64 * 4096).requires_grad_(True)
    cross._check_gradient(long, longer, leaf.expand(1, 64 * 4095, -1))
    cross._check_gradient(longer, longer, leaf.detach().expand(1, 64 * 4096, -1))
    with pytest.raises(ValueError, match="gradient of a bias"):
        cross._check_gradient(longer, longer, leaf.expand(1, 64 * 4096, -1))


def test_what_fp32_does_not_lose_is_not_asked_for():
    """grad_bias_residual of an fp32 call would be left as it was: refused."""
    from af3_kernels_amd import _lib
    lib = _lib.load()
    bwd = lambda p: lib.af3_cross_attention_backward(ctypes.byref(p), ctypes.byref(_grads(grad_bias=BASE, grad_bias_residual=2 * BASE, workspace=None)), None)
    assert bwd(_cross(bias=BASE, dtype=_lib.AF3_F32)) == -2
    assert bwd(_cross(bias=BASE)) == -7      # (as far as its missing workspace)


def test_without_the_native_host_no_gradient_is_captured(monkeypatch, tmp_path):
    from af3_kernels_amd import _lib
    host = _lib._Host()
    monkeypatch.setattr(_lib, "HOST_PATH", str(tmp_path / "_host.so"))
    monkeypatch.setattr(_lib._Host, "_warned", True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    assert host.cross_attention() is None       # (the Python implementation's turn)
    with pytest.raises(RuntimeError, match="native host side"):
        host.check_capture()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    assert host.check_capture() is None
    # found later: the module's own
    monkeypatch.undo()
    from af3_kernels_amd import _host
    assert host.cross_attention is _host.cross_attention and host.check_capture is _host.check_capture
