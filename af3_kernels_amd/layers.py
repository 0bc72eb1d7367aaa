"""What a decoder's or a conditioned transformer's layer is made of, beside cross_attention.

    rotary_frequencies, rotary_embedding   positions as turns of the pairs of a head, instead of a bias
    differential_attention                 the difference of two softmax maps over one set of values
    residual_norm                          the end of one block and the beginning of the next: norm, gate, residual stream, norm

All work under autograd (first derivatives).  The reference has none of them; its LayerNorm is torch's (src/af3_kernels/Attention.py:51).  Every computation on
the device happens in libaf3_dpa.so (af3_rotary_embedding, af3_diff_attention_*, af3_residual_norm_*); there is no CPU path.
"""
import ctypes
import math
from typing import Optional, Tuple

import torch

from . import _lib, ops
from ._lib import DiffAttentionGrads, DiffAttentionParams, ResidualNormGrads, ResidualNormParams, RotaryParams
from .cross import _DTYPES, _inner_contig, _no_tangents, _same_device

_host = ops._host
_i64x3 = ctypes.c_int64 * 3
_LIMIT = 3.4028234663852886e38   # the largest float32


def _finite(x, name):
    x = float(x)
    if not abs(x) <= _LIMIT:
        raise ValueError(f"{name} must be finite in float32, got {x}")
    return x


# ---- rotary positions -----------------------------------------------------------------------------------------------------
def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0, original_length: int = 0, beta_fast: float = 32.0,
                       beta_slow: float = 1.0, device=None) -> Tuple[torch.Tensor, float]:
    """(frequencies, scale) for rotary_embedding: float64 [rotary_dim // 2], radians per position, and what the turned elements are multiplied with.

    Pair i turns with base^(-2 i / rotary_dim).  For contexts longer than the trained ones:
    "linear": all frequencies divided by `factor`; "ntk": base * factor^(rotary_dim / (rotary_dim - 2)) in place of base (the slowest pair is slowed by `factor`, the
    fastest not at all); "yarn": pairs that turn more than beta_fast times within original_length keep their frequency, those that turn less than beta_slow times
    have it divided by `factor`, a ramp in between, and scale = 0.1 log(factor) + 1.  To be made once and kept (host arithmetic and one copy to the device)."""
    n = int(rotary_dim)
    if n < 2 or n % 2 or n > _lib.ROTARY_MAX_HEAD_DIM:
        raise ValueError(f"rotary_dim must be even, 2 to {_lib.ROTARY_MAX_HEAD_DIM}, got {rotary_dim}")
    if scaling not in ("none", "linear", "ntk", "yarn"):
        raise ValueError(f"scaling must be 'none', 'linear', 'ntk' or 'yarn', got {scaling!r}")
    base, factor = float(base), float(factor)
    if not 1.0 < base < math.inf:
        raise ValueError(f"base must be above 1 and finite, got {base}")
    if not 1.0 <= factor < math.inf:
        raise ValueError(f"factor must be at least 1 and finite, got {factor}")
    if scaling == "none" and factor != 1.0:
        raise ValueError("a factor belongs to a scaling: 'linear', 'ntk' or 'yarn'")
    scale = 1.0
    if scaling == "ntk":
        if n == 2:
            raise ValueError("scaling 'ntk' needs a rotary_dim of at least 4")
        base *= factor ** (n / (n - 2))
    frequencies = [base ** (-2.0 * i / n) for i in range(n // 2)]
    if scaling == "linear":
        frequencies = [f / factor for f in frequencies]
    elif scaling == "yarn":
        if int(original_length) < 1:
            raise ValueError(f"scaling 'yarn' needs the trained length as original_length, got {original_length}")
        if not 0.0 < beta_slow < beta_fast < math.inf:
            raise ValueError(f"beta_fast must be above beta_slow and both positive, got {beta_fast} and {beta_slow}")

        def pair_of(turns):   # the pair that turns so often within original_length (a real number)
            return n * math.log(original_length / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))
        low, high = max(math.floor(pair_of(beta_fast)), 0), min(math.ceil(pair_of(beta_slow)), n - 1)
        for i, f in enumerate(frequencies):
            slowed = min(max((i - low) / max(high - low, 1e-3), 0.0), 1.0) if original_length * f >= beta_slow * 2.0 * math.pi else 1.0   # (within a few tokens not even pair 0 turns so often)
            frequencies[i] = f / factor * slowed + f * (1.0 - slowed)
        scale = 0.1 * math.log(factor) + 1.0
    return torch.tensor(frequencies, dtype=torch.float64, device=device), scale


def _turn(tensors, frequencies, positions, offset, interleaved, scale, inverse):
    """The tensors [B, heads, L, D] (None: left out) turned, in one launch."""
    p, outs, n = RotaryParams(), [], 0
    for t in tensors:
        if t is None or t.numel() == 0:
            outs.append(None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device))
            continue
        out = torch.empty(t.shape, dtype=t.dtype, device=t.device)
        p.x[n], p.out[n], p.heads[n] = t.data_ptr(), out.data_ptr(), t.shape[1]
        p.x_stride[n], p.out_stride[n] = _i64x3(*t.stride()[:3]), _i64x3(*out.stride()[:3])
        p.B, p.L, p.D, p.dtype = t.shape[0], t.shape[2], t.shape[3], _DTYPES[t.dtype]
        outs.append(out)
        n += 1
    if n:
        p.frequencies, p.rotary = frequencies.data_ptr(), 2 * frequencies.shape[0]
        if positions is not None:
            p.positions, p.position_stride_b = positions.data_ptr(), 0 if positions.dim() == 1 or positions.shape[0] == 1 else positions.stride(0)
        p.offset, p.interleaved, p.inverse, p.scale = offset, int(interleaved), int(inverse), scale
        with ops._on_device(frequencies.device):
            _lib.check(_lib.load().af3_rotary_embedding(ctypes.byref(p), ops._stream_ptr(frequencies.device)), "af3_rotary_embedding")
    return outs


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, frequencies, positions, offset, interleaved, scale):
        ctx.save_for_backward(frequencies, positions)
        ctx.settings = (offset, interleaved, scale)
        ctx.set_materialize_grads(False)
        return tuple(_turn((q, k), frequencies, positions, offset, interleaved, scale, False))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        _no_tangents("the gradient of rotary_embedding", *grads)
        frequencies, positions = ctx.saved_tensors
        grads = [_inner_contig(g) if g is not None and need else None for g, need in zip(grads, ctx.needs_input_grad)]
        return (*_turn(grads, frequencies, positions, *ctx.settings, True), None, None, None, None, None)


def rotary_embedding(q: torch.Tensor, k: Optional[torch.Tensor], frequencies: torch.Tensor, positions: Optional[torch.Tensor] = None, offset: int = 0,
                     interleaved: bool = False, scale: float = 1.0) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Queries and keys with their positions: (q, k) with every pair of elements turned by position * frequency.

    q [B, H, L, D] and k [B, Hkv, L, D] (or None), float32 or bfloat16 (k is cast to q's dtype), any strides, D up to 1024.  The first
    n = 2 * len(frequencies) <= D elements of a head are turned, the others are handed through: pair i is elements (i, i + n / 2), or (2 i, 2 i + 1) if `interleaved`,
        (x, y) -> scale * (x cos a - y sin a, x sin a + y cos a),  a = position * frequencies[i]
    with angles in 64 bits, the rest in fp32, one rounding at the end.  frequencies, scale: from rotary_frequencies, or any float64 [n / 2] (float32 is cast).  Positions are
    offset, offset + 1, ... (a decoder's token t: L = 1, offset = t), or what `positions` holds: [L], or [B, L] for rows at positions of their own
    (int64 or int32).  New contiguous tensors; (q, None) without k.

    Gradients flow to q and k (turned back), not to frequencies, which must not ask for one; a second derivative and forward mode raise.  In a HIP graph: as
    cross_attention."""
    out = _host.rotary(q, k, frequencies, positions, offset, interleaved, scale)
    if out is not None:
        return out if out.__class__ is not int else _lib.check(out, "af3_rotary_embedding")
    _no_tangents("rotary_embedding", q, k, frequencies)
    _same_device(q, k, frequencies, positions)
    if q.dim() != 4 or (k is not None and (k.dim() != 4 or k.shape[0] != q.shape[0] or k.shape[2:] != q.shape[2:])):
        raise ValueError(f"q must be [B, H, L, D] and k [B, Hkv, L, D], got {tuple(q.shape)} and {None if k is None else tuple(k.shape)}")
    if q.dtype not in _DTYPES:
        raise ValueError(f"unsupported dtype {q.dtype}: float32 or bfloat16")
    B, _, L, D = q.shape
    if not 2 <= D <= _lib.ROTARY_MAX_HEAD_DIM:
        raise ValueError(f"head_dim must be 2 to {_lib.ROTARY_MAX_HEAD_DIM}, got {D}")
    if frequencies.dim() != 1 or frequencies.dtype not in (torch.float64, torch.float32) or not 2 <= 2 * frequencies.shape[0] <= D:
        raise ValueError(f"frequencies must be float64 or float32 [n / 2] with n of 2 to head_dim {D}, got {frequencies.dtype} {tuple(frequencies.shape)}")
    if frequencies.requires_grad:
        raise ValueError("frequencies have no gradient here: detach them")
    if positions is not None and (positions.dtype not in (torch.int64, torch.int32) or positions.dim() not in (1, 2) or positions.shape[-1] != L
                                  or (positions.dim() == 2 and positions.shape[0] not in (1, B))):
        raise ValueError(f"positions must be int64 or int32 [L] or [B, L] with B={B}, L={L}, got {positions.dtype} {tuple(positions.shape)}")
    offset, interleaved, scale = int(offset), bool(interleaved), _finite(scale, "scale")
    if abs(offset) > 1 << 62:
        raise ValueError(f"offset must lie within 2^62, got {offset}")
    q, frequencies = _inner_contig(q), frequencies.to(torch.float64).contiguous()
    k = None if k is None else _inner_contig(k if k.dtype == q.dtype else k.to(q.dtype))
    positions = None if positions is None else _inner_contig(positions.to(torch.int64))
    with ops._on_device(q.device):   # (as a plain call)
        out = _host.rotary(q, k, frequencies, positions, offset, interleaved, scale)
    if out is not None:
        return out if out.__class__ is not int else _lib.check(out, "af3_rotary_embedding")
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        with ops._on_device(q.device):
            _host.check_capture(q, k)
        return _Rotary.apply(q, k, frequencies, positions, offset, interleaved, scale)
    return tuple(_turn((q, k), frequencies, positions, offset, interleaved, scale, False))


# ---- differential attention -------------------------------------------------------------------------------------------------
def _diff_block(q, k, v, lam, keep, out, stats, second, lost, causal, offset, scale) -> DiffAttentionParams:
    p = DiffAttentionParams()
    p.q, p.k, p.v, p.lam, p.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), lam.data_ptr(), out.data_ptr()
    p.B, p.H, p.Lq, p.Dv = out.shape
    p.D, p.Hkv, p.Lk = q.shape[3], v.shape[1], v.shape[2]
    p.q_stride, p.k_stride, p.v_stride, p.out_stride = (_i64x3(*t.stride()[:3]) for t in (q, k, v, out))
    if keep is not None:
        p.key_mask, p.key_mask_stride_b = keep.data_ptr(), 0 if keep.shape[0] == 1 else keep.stride(0)
    if stats is not None:
        p.stats, p.second = stats.data_ptr(), second.data_ptr()
    if lost is not None:
        p.residuals = lost.data_ptr()
    p.lam_stride, p.lam_dtype, p.dtype = lam.stride(0), _DTYPES[lam.dtype], _DTYPES[q.dtype]
    p.causal, p.q_offset, p.softmax_scale = int(causal), offset, scale
    return p


def _diff_forward(q, k, v, lam, keep, causal, offset, scale, want_stats):
    """(out, stats, second, lost): where the gradient will be asked for, stats [B, 2H, Lq, 2], the second map's own result, and what the two lost by their rounding to bfloat16."""
    B, H, Lq = q.shape[0], q.shape[1] // 2, q.shape[2]
    out = torch.empty(B, H, Lq, v.shape[3], dtype=q.dtype, device=q.device)
    if out.numel() == 0 or k.shape[2] == 0:
        return out.zero_(), None, None, None
    stats = torch.empty(B, 2 * H, Lq, 2, dtype=torch.float32, device=q.device) if want_stats else None
    second = torch.empty_like(out) if want_stats else None
    lost = torch.empty(2, *out.shape, dtype=out.dtype, device=out.device) if want_stats and out.dtype == torch.bfloat16 else None
    p = _diff_block(q, k, v, lam, keep, out, stats, second, lost, causal, offset, scale)
    lib = _lib.load()
    with ops._on_device(q.device):
        need = lib.af3_diff_attention_workspace_bytes(ctypes.byref(p))
        if need > 0:
            ws = torch.empty(need, dtype=torch.uint8, device=q.device)
            p.workspace, p.workspace_bytes = ws.data_ptr(), need
        _lib.check(lib.af3_diff_attention_forward(ctypes.byref(p), ops._stream_ptr(q.device)), "af3_diff_attention_forward")
    return out, stats, second, lost


class _DifferentialAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lam, keep, causal, offset, scale):
        out, stats, second, lost = _diff_forward(q, k, v, lam, keep, causal, offset, scale, True)
        ctx.save_for_backward(q, k, v, lam, keep, out, stats, second, lost)
        ctx.settings = (causal, offset, scale)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        _no_tangents("the gradient of differential_attention", grad)
        q, k, v, lam, keep, out, stats, second, lost = ctx.saved_tensors
        wants = ctx.needs_input_grad[:4]
        if stats is None:
            return (*(torch.zeros(t.shape, dtype=t.dtype, device=t.device) if w else None for t, w in zip((q, k, v, lam), wants)), None, None, None, None)
        grads = [torch.empty(t.shape, dtype=t.dtype, device=t.device) if w else None for t, w in zip((q, k, v, lam), wants)]
        grad = _inner_contig(grad)
        grad = grad if grad.stride(2) * grad.element_size() < _lib.DIFF_ATTENTION_GRAD_ROW_BYTES else grad.contiguous()
        p, g = _diff_block(q, k, v, lam, keep, out, stats, second, lost, *ctx.settings), DiffAttentionGrads()
        g.grad_out, g.grad_out_stride = grad.data_ptr(), _i64x3(*grad.stride()[:3])
        g.grad_q, g.grad_k, g.grad_v, g.grad_lam = (0 if t is None else t.data_ptr() for t in grads)
        lib = _lib.load()
        with ops._on_device(q.device):
            need = lib.af3_diff_attention_backward_workspace_bytes(ctypes.byref(p))
            ws = torch.empty(max(need, 16), dtype=torch.uint8, device=q.device)
            g.workspace, g.workspace_bytes = ws.data_ptr(), need
            _lib.check(lib.af3_diff_attention_backward(ctypes.byref(p), ctypes.byref(g), ops._stream_ptr(q.device)), "af3_diff_attention_backward")
        return (*grads, None, None, None, None)


def differential_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lam: torch.Tensor, mask: Optional[torch.Tensor] = None, causal: bool = False, q_offset: int = 0,
                           softmax_scale: Optional[float] = None) -> torch.Tensor:
    """(softmax(q1.k1^T * softmax_scale) - lam * softmax(q2.k2^T * softmax_scale)) . v for every head: what two attention maps have in common cancels.

    q [B, 2 H, Lq, D]: query heads 2 h and 2 h + 1 are the two maps of head h; k [B, 2 Hkv, Lk, D] likewise; v [B, Hkv, Lk, Dv] with H a multiple of Hkv (head h uses key
    head h // (H // Hkv)); the result is [B, H, Lq, Dv].  lam [H], or one number for all heads (a tensor of one element): float32 or q's dtype, anything else is cast to float32.
    bfloat16: D up to 128, Dv up to 256; float32: half of that.  mask [Lk], [B, Lk] or [B, 1, 1, Lk], truthy = attend; causal: key j counts for query i if j <= i + q_offset (a
    decoder's token t: Lq = 1, q_offset = t).  softmax_scale: D^-1/2 unless given.  float32 (fp32 throughout) or bfloat16 (bf16 products, fp32 accumulation and softmax; the
    probabilities and, in the gradient, dS are rounded to bf16 for the products that follow; in long calls the probabilities and v go as fp16, v in units of its tile of 64 or 128 keys: values
    below 2^-25 of the tile's largest are rounded, by 2^-33 of it at most, and results below 2^-70 of the largest v of a call lose bits); k and v are cast to q's dtype.  Any strides; a new contiguous tensor.

    A key that `mask` drops has no part in the result or its gradient, whatever k and v hold there.  A query that is left without a key, by mask and causality, gives zeros and
    has no gradient (not the mean of its values as in cross_attention: of a difference nothing is left).  Keys behind a causal query have weight zero for it, which NaN and
    infinities in their k and v do not heed where other queries of the call see those keys.  Lk == 0 gives zeros.

    Gradients flow to q, k, v and lam (the same bits every time); a second derivative and forward mode raise.  In a HIP graph: as cross_attention."""
    out = _host.differential_attention(q, k, v, lam, mask, causal, q_offset, softmax_scale)
    if out is not None:
        return out if out.__class__ is not int else _lib.check(out, "af3_diff_attention_forward")
    if not isinstance(lam, torch.Tensor):
        raise TypeError(f"lam must be a tensor, [H] or of one element, got {type(lam).__name__}")
    _no_tangents("differential_attention", q, k, v, lam)
    _same_device(q, k, v, lam, mask)
    if q.dtype not in _DTYPES:
        raise ValueError(f"unsupported dtype {q.dtype}: float32 or bfloat16")
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError(f"q must be [B, 2 H, Lq, D], k [B, 2 Hkv, Lk, D] and v [B, Hkv, Lk, Dv], got {tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    B, H, Lq, D = q.shape[0], q.shape[1] // 2, q.shape[2], q.shape[3]
    Hkv, Lk, Dv = v.shape[1], k.shape[2], v.shape[3]
    if q.shape[1] % 2 or tuple(k.shape) != (B, 2 * Hkv, Lk, D) or v.shape[0] != B or v.shape[2] != Lk:
        raise ValueError(f"q must be [B, 2 H, Lq, D], k [B, 2 Hkv, Lk, D] and v [B, Hkv, Lk, Dv], got {tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    if Hkv == 0 or H % Hkv != 0:
        raise ValueError(f"the heads must be a multiple of the key heads, got {H} and {Hkv}")
    most = 64 if q.dtype == torch.float32 else 128
    if not 1 <= D <= most or not 1 <= Dv <= 2 * most:
        raise ValueError(f"head_dim must be 1 to {most} and v's 1 to {2 * most} in {q.dtype}, got {D} and {Dv}")
    if lam.numel() != 1 and tuple(lam.shape) != (H,):
        raise ValueError(f"lam must be [H] with H={H}, or one number, got {tuple(lam.shape)}")
    keep = ops._lift_mask(mask, None) if mask is not None else None
    if keep is not None and (keep.shape[1] != Lk or keep.shape[0] not in (1, B)):
        raise ValueError(f"mask must be [Lk], [B, Lk] or [B, 1, 1, Lk] with B={B}, Lk={Lk}, got {tuple(mask.shape)}")
    causal, q_offset = bool(causal), int(q_offset)
    if abs(q_offset) >= 1 << 40:
        raise ValueError(f"q_offset must lie within 2^40, got {q_offset}")
    scale = float(D) ** -0.5 if softmax_scale is None else float(softmax_scale)
    if not 0.0 < scale <= _LIMIT:
        raise ValueError(f"softmax_scale must be positive and finite, got {scale}")
    dtype = q.dtype
    q, k, v = _inner_contig(q), _inner_contig(k if k.dtype == dtype else k.to(dtype)), _inner_contig(v if v.dtype == dtype else v.to(dtype))
    shared = tuple(lam.shape) != (H,)
    # (one number for all heads: its gradient is rounded once, behind their sum)
    if lam.dtype not in (dtype, torch.float32) or (shared and lam.dtype != torch.float32 and lam.requires_grad and torch.is_grad_enabled()):
        lam = lam.to(torch.float32)
    lam = lam.reshape(1).expand(H) if shared else lam
    graph = torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, lam))
    if graph and B * Hkv * -(-Lk // 32) >= 1 << 24:
        raise ValueError(f"gradients take B * Hkv * ceil(Lk / 32) below 2^24, got {B} * {Hkv} * ceil({Lk} / 32)")
    with ops._on_device(q.device):   # (as a plain call)
        out = _host.differential_attention(q, k, v, lam, None if keep is None else keep.view(torch.bool), causal, q_offset, scale)
    if out is not None:
        return out if out.__class__ is not int else _lib.check(out, "af3_diff_attention_forward")
    if graph:
        with ops._on_device(q.device):
            _host.check_capture(q, k, v, lam)
        return _DifferentialAttention.apply(q, k, v, lam, keep, causal, q_offset, scale)
    return _diff_forward(q, k, v, lam, keep, causal, q_offset, scale, False)[0]


# ---- norms around a block ---------------------------------------------------------------------------------------------------
def _row_stride(t):
    """The distance of a tensor's rows [.., C] where they are equally far apart, None otherwise."""
    stride, behind = None, 1
    for size, step in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size == 1:
            continue
        if stride is None:
            stride = step
        elif step != stride * behind:
            return None
        behind *= size
    return t.shape[-1] if stride is None else stride


def _rows(t):
    return t if t is None or (t.stride(-1) == 1 and _row_stride(t) is not None) else t.contiguous()


def _shared_by(t, y):
    """How many consecutive rows of y a row of the parameter t is for: all of them, some, 1; None: not a parameter for y, or one that is repeated otherwise."""
    rows, lead = y.numel() // y.shape[-1], t.shape[:-1]
    if t.dim() == 1 or (t.dim() == y.dim() and t.numel() == t.shape[-1]):
        return rows
    if t.dim() != y.dim():
        return None
    i = 0
    while i < len(lead) and lead[i] == y.shape[i]:
        i += 1
    return math.prod(y.shape[i:-1]) if all(n == 1 for n in lead[i:]) else None


def _norm_block(x, y, weight, bias, gate, post_weight, kinds, scale, eps) -> ResidualNormParams:
    p = ResidualNormParams()
    p.C, p.rows = y.shape[-1], y.numel() // y.shape[-1]
    p.y, p.y_stride = y.data_ptr(), _row_stride(y)
    if x is not None:
        p.x, p.x_stride = x.data_ptr(), _row_stride(x)
    for name, t in (("gate", gate), ("weight", weight), ("bias", bias)):
        if t is not None:
            each = _shared_by(t, y)
            share = _lib.SHARE_CHANNEL if t.dim() == 1 or each == p.rows else _lib.SHARE_ROW if each == 1 else _lib.SHARE_GROUP
            if share == _lib.SHARE_GROUP:
                p.group = each
            setattr(p, name, t.data_ptr())
            setattr(p, name + "_share", share)
    if post_weight is not None:
        p.post_weight = post_weight.data_ptr()
    p.norm, p.post_norm, p.gate_sigmoid = kinds
    p.dtype, p.eps, p.residual_scale = _DTYPES[y.dtype], eps, scale
    return p


def _norm_forward(x, y, weight, bias, gate, post_weight, kinds, scale, eps, want_stats):
    out = torch.empty(y.shape, dtype=y.dtype, device=y.device)
    normed = torch.empty_like(out) if kinds[0] else None
    if y.numel() == 0:
        return out, normed, None
    stats = torch.empty(y.numel() // y.shape[-1], 4, dtype=torch.float32, device=y.device) if want_stats else None
    p = _norm_block(x, y, weight, bias, gate, post_weight, kinds, scale, eps)
    p.out, p.normed, p.stats = out.data_ptr(), 0 if normed is None else normed.data_ptr(), 0 if stats is None else stats.data_ptr()
    with ops._on_device(y.device):
        _lib.check(_lib.load().af3_residual_norm_forward(ctypes.byref(p), ops._stream_ptr(y.device)), "af3_residual_norm_forward")
    return out, normed, stats


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, weight, bias, gate, post_weight, kinds, scale, eps):
        out, normed, stats = _norm_forward(x, y, weight, bias, gate, post_weight, kinds, scale, eps, True)
        ctx.save_for_backward(x, y, weight, bias, gate, post_weight, stats)
        ctx.settings = (kinds, scale, eps)
        ctx.set_materialize_grads(False)
        return out, normed

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out, grad_normed):
        _no_tangents("the gradient of residual_norm", grad_out, grad_normed)
        *tensors, stats = ctx.saved_tensors
        y = tensors[1]
        # (without a gradient of the normed rows those of weight and bias are zeros)
        reached = (grad_out is not None or grad_normed is not None, grad_normed is not None)
        grads = [None if t is None or not need else torch.empty(t.shape, dtype=t.dtype, device=t.device) for t, need in zip(tensors, ctx.needs_input_grad)]
        for i, g in enumerate(grads):
            if g is not None and (stats is None or not reached[i in (2, 3)]):
                g.zero_()
        wanted = [g if stats is not None and reached[i in (2, 3)] else None for i, g in enumerate(grads)]
        if any(g is not None for g in wanted):
            p, o = _norm_block(*tensors, *ctx.settings), ResidualNormGrads()
            p.stats = stats.data_ptr()
            grad_out, grad_normed = _rows(grad_out), _rows(grad_normed)
            if grad_out is not None:
                o.grad_out, o.grad_out_stride = grad_out.data_ptr(), _row_stride(grad_out)
            if grad_normed is not None:
                o.grad_normed, o.grad_normed_stride = grad_normed.data_ptr(), _row_stride(grad_normed)
            o.grad_x, o.grad_y, o.grad_weight, o.grad_bias, o.grad_gate, o.grad_post_weight = (0 if g is None else g.data_ptr() for g in wanted)
            lib = _lib.load()
            with ops._on_device(y.device):
                need = lib.af3_residual_norm_backward_workspace_bytes(ctypes.byref(p), ctypes.byref(o))
                _lib.check(min(need, 0), "af3_residual_norm_backward_workspace_bytes")
                ws = torch.empty(max(need, 16), dtype=torch.uint8, device=y.device)
                o.workspace, o.workspace_bytes = ws.data_ptr(), need
                _lib.check(lib.af3_residual_norm_backward(ctypes.byref(p), ctypes.byref(o), ops._stream_ptr(y.device)), "af3_residual_norm_backward")
        return (*grads, None, None, None)


def residual_norm(x: Optional[torch.Tensor], y: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                  post_weight: Optional[torch.Tensor] = None, norm: str = "rms", post_norm: str = "none", gate_activation: str = "none", residual_scale: float = 1.0,
                  eps: float = 1e-5) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The end of one block and the beginning of the next in one pass: (out, normed) with
        out    = residual_scale * x + gate * post_norm(y) * post_weight
        normed = norm(out) * weight + bias
    x: the residual stream [.., C] (None: no stream); y: the block's result [.., C].  norm, post_norm: "rms", "layer" (biased variance) or "none"; norm="none" gives
    (out, None).  A norm alone is residual_norm(None, y, post_weight=w, post_norm="rms", norm="none")[0].  gate_activation="sigmoid" takes the logistic function of the gate.

    gate, weight and bias are [C], or have y's number of axes with 1 where they are repeated: [B, 1, C] for all tokens of a sequence, [B, T, C] for
    every token (a conditioned transformer's), [C] for all.  post_weight [C].  One left out counts as ones (a bias as zeros).  float32 or bfloat16, everything else cast to y's
    dtype; arithmetic in fp32, out and normed rounded once each (normed is made of out before its rounding).  C up to 16384; x, y: any strides.  New contiguous tensors.
    (A parameter that is repeated along an axis in front of one that it is not repeated along, [1, T, C], goes as one with a row for every token: torch adds those rows' gradients up, rounded to y's dtype.)

    Gradients flow to all tensors (the same bits every time); a second derivative and forward mode raise.  In a HIP graph: as cross_attention."""
    kinds = _lib.NORMS.get(norm, -1), _lib.NORMS.get(post_norm, -1), gate_activation == "sigmoid"
    out = _host.residual_norm(x, y, weight, bias, gate, post_weight, *kinds, residual_scale, eps) if gate_activation in ("none", "sigmoid") else None
    if out is not None:
        return out if out.__class__ is not int else _lib.check(out, "af3_residual_norm_forward")
    _no_tangents("residual_norm", x, y, weight, bias, gate, post_weight)
    _same_device(y, x, weight, bias, gate, post_weight)
    if y.dtype not in _DTYPES:
        raise ValueError(f"unsupported dtype {y.dtype}: float32 or bfloat16")
    for name, kind in (("norm", norm), ("post_norm", post_norm)):
        if kind not in _lib.NORMS:
            raise ValueError(f"{name} must be 'none', 'rms' or 'layer', got {kind!r}")
    if gate_activation not in ("none", "sigmoid"):
        raise ValueError(f"gate_activation must be 'none' or 'sigmoid', got {gate_activation!r}")
    if y.dim() < 1 or not 1 <= y.shape[-1] <= _lib.RESIDUAL_NORM_MAX_CHANNELS:
        raise ValueError(f"y must be [.., C] with C of 1 to {_lib.RESIDUAL_NORM_MAX_CHANNELS}, got {tuple(y.shape)}")
    if x is not None and x.shape != y.shape:
        raise ValueError(f"x must have y's shape {tuple(y.shape)}, got {tuple(x.shape)}")
    if norm == "none" and (weight is not None or bias is not None):
        raise ValueError("weight and bias belong to a norm, and norm is 'none'")
    if post_norm == "none" and post_weight is not None:
        raise ValueError("post_weight belongs to a post_norm, and post_norm is 'none'")
    if gate_activation != "none" and gate is None:
        raise ValueError("gate_activation needs a gate")
    if post_weight is not None and tuple(post_weight.shape) != (y.shape[-1],):
        raise ValueError(f"post_weight must be [C] with C={y.shape[-1]}, got {tuple(post_weight.shape)}")
    C, shared = y.shape[-1], {}
    for name, t in (("gate", gate), ("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.dim() < 1 or t.shape[-1] != C or not (t.dim() == 1 or (t.dim() == y.dim() and all(n in (1, m) for n, m in zip(t.shape, y.shape)))):
            raise ValueError(f"{name} must be [C] or have y's axes, of y's sizes or 1, and C channels, got {tuple(t.shape)} for y {tuple(y.shape)}")
        shared[name] = _shared_by(t, y)
    residual_scale, eps = _finite(residual_scale, "residual_scale"), _finite(eps, "eps")
    if eps < 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    # Parameters that are repeated along an axis in front of one they are not repeated along have a row for every row of y; of several lengths of repetition the shortest is taken for all.
    rows = y.numel() // C
    groups = [n for n in shared.values() if n is not None and 1 < n < rows]

    def laid_out(name, t):
        if t is None:
            return None
        if t.dtype != y.dtype:
            t = t.to(y.dtype)
        if name in shared:
            if shared[name] is None:
                t = t.expand(y.shape)
            elif 1 < shared[name] < rows and shared[name] != min(groups):
                size, each = list(t.shape), 1   # (as many of the last axes stay repeated as the shortest has)
                for i in range(y.dim() - 2, -1, -1):
                    if each >= min(groups):
                        size[i] = y.shape[i]
                    each *= y.shape[i]
                t = t.expand(size)
        return t.contiguous()
    gate, weight, bias, post_weight = (laid_out(n, t) for n, t in (("gate", gate), ("weight", weight), ("bias", bias), ("post_weight", post_weight)))
    y, x = _rows(y), None if x is None else _rows(x if x.dtype == y.dtype else x.to(y.dtype))
    with ops._on_device(y.device):   # (as a plain call)
        out = _host.residual_norm(x, y, weight, bias, gate, post_weight, *kinds, residual_scale, eps)
    if out is not None:
        return out if out.__class__ is not int else _lib.check(out, "af3_residual_norm_forward")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, y, weight, bias, gate, post_weight)):
        with ops._on_device(y.device):
            _host.check_capture(x, y, weight, bias, gate, post_weight)
        return _ResidualNorm.apply(x, y, weight, bias, gate, post_weight, kinds, residual_scale, eps)
    return _norm_forward(x, y, weight, bias, gate, post_weight, kinds, residual_scale, eps, False)[:2]
