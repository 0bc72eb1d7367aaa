"""Attention of queries to states of another length, its gradient, and the learned relative position bias it takes.

    cross_attention          softmax(q.k^T scale + bias, mask).v for q [B, H, Lq, D] and k, v [B, Hkv, Lk, D]
    relative_position_bias   bias[h, i, j] = table[bucket(position of key j - position of query i), h]

Both work under autograd (first derivatives).  The reference has neither: its attention takes q_len == k_len
(src/csrc/dot_product_attention.cpp:50-52) and no gradient.  Every computation happens in libaf3_dpa.so
(af3_cross_attention_*, af3_position_bias_*); there is no CPU path.
"""
import ctypes
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _lib, ops
from ._lib import CrossAttentionGrads, CrossAttentionParams, PositionBiasParams

_host = ops._host
_i64x2, _i64x3 = ctypes.c_int64 * 2, ctypes.c_int64 * 3
_DTYPES = {torch.float32: _lib.AF3_F32, torch.bfloat16: _lib.AF3_BF16}


def _same_device(first, *others):
    ops._require_device(first, *others)
    for t in others:
        if t is not None and t.device != first.device:
            raise ValueError(f"all tensors must be on one device, got {first.device} and {t.device}")


def _no_tangents(what, *tensors):
    """Forward-mode differentiation is refused: the result would come without a tangent, as if it did not depend on these."""
    for t in tensors:
        if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{what} has no forward-mode derivative")


def _inner_contig(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


# ---- attention ----------------------------------------------------------------------------------------------------------
def _fill(q, k, v, keep, bias, out, stats, lost, scale) -> CrossAttentionParams:
    p = CrossAttentionParams()
    p.q, p.k, p.v, p.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    p.B, p.H, p.Lq, p.D = q.shape
    p.Hkv, p.Lk = k.shape[1], k.shape[2]
    p.q_stride, p.k_stride, p.v_stride, p.out_stride = (_i64x3(*t.stride()[:3]) for t in (q, k, v, out))
    if bias is not None:
        p.bias, p.bias_stride = bias.data_ptr(), _i64x2(bias.stride(0), bias.stride(1))
    if keep is not None:
        p.key_mask, p.key_mask_stride_b = keep.data_ptr(), 0 if keep.shape[0] == 1 else keep.stride(0)
    if stats is not None:
        p.stats = stats.data_ptr()
    if lost is not None:
        p.out_residual = lost.data_ptr()
    p.dtype, p.softmax_scale = _DTYPES[q.dtype], scale
    return p


def _forward(q, k, v, keep, bias, scale, want_stats):
    """(out, stats, lost): where the gradient will be asked for, stats [B, H, Lq, 2] and what out lost by its rounding to bfloat16."""
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if out.numel() == 0 or k.shape[2] == 0:
        return out.zero_(), None, None
    stats = torch.empty(*q.shape[:3], 2, dtype=torch.float32, device=q.device) if want_stats else None
    lost = torch.empty_like(out) if want_stats and q.dtype == torch.bfloat16 else None
    p = _fill(q, k, v, keep, bias, out, stats, lost, scale)
    lib = _lib.load()
    with ops._on_device(q.device):
        need = lib.af3_cross_attention_workspace_bytes(ctypes.byref(p))
        if need > 0:
            ws = torch.empty(need, dtype=torch.uint8, device=q.device)
            p.workspace, p.workspace_bytes = ws.data_ptr(), need
        _lib.check(lib.af3_cross_attention_forward(ctypes.byref(p), ops._stream_ptr(q.device)), "af3_cross_attention_forward")
    return out, stats, lost


def _backward(grad, q, k, v, keep, bias, out, stats, lost, scale, wants):
    """Gradients of q, k, v and bias, None for those not wanted, and with wants[4] what the bias's lost by its rounding."""
    bias_shape = None if bias is None else (q.shape[1], q.shape[2], k.shape[2])
    shapes = (q.shape, k.shape, v.shape, bias_shape, bias_shape)
    if stats is None:
        return tuple(torch.zeros(s, dtype=q.dtype, device=q.device) if w else None for s, w in zip(shapes, wants))
    grads = tuple(torch.empty(s, dtype=q.dtype, device=q.device) if w else None for s, w in zip(shapes, wants))
    grad = _inner_contig(grad)
    p = _fill(q, k, v, keep, bias, out, stats, lost, scale)
    g = CrossAttentionGrads()
    g.grad_out, g.grad_out_stride = grad.data_ptr(), _i64x3(*grad.stride()[:3])
    g.grad_q, g.grad_k, g.grad_v, g.grad_bias, g.grad_bias_residual = (0 if t is None else t.data_ptr() for t in grads)
    lib = _lib.load()
    with ops._on_device(q.device):
        need = lib.af3_cross_attention_backward_workspace_bytes(ctypes.byref(p))
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device=q.device)
        g.workspace, g.workspace_bytes = ws.data_ptr(), need
        _lib.check(lib.af3_cross_attention_backward(ctypes.byref(p), ctypes.byref(g), ops._stream_ptr(q.device)), "af3_cross_attention_backward")
    return grads


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, keep, bias, scale):
        out, stats, lost = _forward(q, k, v, keep, bias, scale, True)
        ctx.save_for_backward(q, k, v, keep, bias, out, stats, lost)
        ctx.scale = scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        _no_tangents("the gradient of cross_attention", grad)
        q, k, v, keep, bias, out, stats, lost = ctx.saved_tensors
        needs = ctx.needs_input_grad
        # (what the bias's gradient loses by its rounding is not asked for: the native host side knows whether it may be handed on to a table, this side does not)
        dq, dk, dv, dbias, _ = _backward(grad, q, k, v, keep, bias, out, stats, lost, ctx.scale, (needs[0], needs[1], needs[2], needs[4], False))
        return dq, dk, dv, None, dbias, None


def _check_cross(q, k, v, keep, bias):
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError(f"q must be [B, H, Lq, D], k and v [B, Hkv, Lk, D], got {tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    B, H, Lq, D = q.shape
    Hkv, Lk = k.shape[1], k.shape[2]
    if tuple(k.shape) != (B, Hkv, Lk, D) or tuple(v.shape) != (B, Hkv, Lk, D):
        raise ValueError(f"k and v must be [B, Hkv, Lk, D] with B={B}, D={D}, got {tuple(k.shape)} and {tuple(v.shape)}")
    if Hkv == 0 or H % Hkv != 0:
        raise ValueError(f"the query heads must be a multiple of the key heads, got {H} and {Hkv}")
    if D < 1 or D > 128:
        raise ValueError(f"head_dim must be 1 to 128, got {D}")
    if bias is not None and (bias.dim() != 3 or bias.shape[0] != H or bias.shape[1] < Lq or bias.shape[2] < Lk):
        raise ValueError(f"bias must be [H, Lq, Lk] (or larger in its last two axes) with H={H}, Lq={Lq}, Lk={Lk}, got {tuple(bias.shape)}")
    if keep is not None and (keep.shape[1] != Lk or keep.shape[0] not in (1, B)):
        raise ValueError(f"mask must be [Lk], [B, Lk] or [B, 1, 1, Lk] with B={B}, Lk={Lk}, got {tuple(keep.shape)}")


def _check_gradient(q, k, bias):
    """Sizes whose gradients would be refused (af3_cross_attention_backward), before the forward pass."""
    B, H, Lq, _ = q.shape
    Hkv, Lk = k.shape[1], k.shape[2]
    if B * Hkv * -(-Lk // 32) >= 1 << 24:
        raise ValueError(f"gradients take B * Hkv * ceil(Lk / 32) below 2^24, got {B} * {Hkv} * ceil({Lk} / 32)")
    if bias is not None and bias.requires_grad and H * -(-Lq // 64) * -(-Lk // 64) >= 1 << 24:
        raise ValueError(f"the gradient of a bias takes H * ceil(Lq / 64) * ceil(Lk / 64) below 2^24, got {H} * ceil({Lq} / 64) * ceil({Lk} / 64)")


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mask: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                    softmax_scale: Optional[float] = None) -> torch.Tensor:
    """softmax(q.k^T * softmax_scale + bias, mask) . v for queries and keys of any two lengths, down to a single query token.

    q [B, H, Lq, D]; k, v [B, Hkv, Lk, D] with H a multiple of Hkv (query head h uses key head h // (H // Hkv)); D up to 128.  mask [Lk], [B, Lk]
    or [B, 1, 1, Lk], truthy = attend; bias [H, Lq, Lk] shared by the batch (or larger: its first Lq and Lk entries count), e.g. from
    relative_position_bias.  softmax_scale: D^-1/2 unless given.  float32 (fp32 throughout) or bfloat16 (bf16 products, fp32 accumulation and
    softmax; the probabilities and, in the gradient, dS are rounded to bf16 for the products that follow); k, v and bias are cast to q's dtype.
    Any strides; the result is a new contiguous tensor.

    A key that `mask` drops has no part in the result or its gradient, whatever k, v and bias hold there; a batch row without any
    live key gives the mean of its v rows, like the package's other attention calls (and their gradient).  A bias of -inf drops a key for
    that query; a query left without a live key by that gives zeros and no gradient.  The lowest finite bias does as the formula
    says: a row of nothing else weights its live keys alike.  Lk == 0 gives zeros.

    Gradients flow to q, k, v and bias (the same bits every time); a second derivative and forward mode raise.  In a HIP graph: capture forward and backward
    together, and whatever leads to the inputs, with leaves that no result of an earlier call on another stream still holds.  Their gradients would be worked out or
    accumulated on that stream, outside of the capture, so such a call raises RuntimeError."""
    out = _host.cross_attention(q, k, v, mask, bias, softmax_scale)
    if out is not None:
        return out if out.__class__ is not int else _lib.check(out, "af3_cross_attention_forward")
    _no_tangents("cross_attention", q, k, v, bias)
    _same_device(q, k, v, mask, bias)
    if q.dtype not in _DTYPES:
        raise ValueError(f"unsupported dtype {q.dtype}: float32 or bfloat16")
    keep = ops._lift_mask(mask, None) if mask is not None else None
    _check_cross(q, k, v, keep, bias)
    Lq, Lk = q.shape[2], k.shape[2]
    dtype = q.dtype
    q, k, v = _inner_contig(q), _inner_contig(k if k.dtype == dtype else k.to(dtype)), _inner_contig(v if v.dtype == dtype else v.to(dtype))
    if bias is not None:
        if bias.shape[1] != Lq or bias.shape[2] != Lk:
            bias = bias[:, :Lq, :Lk]
        bias = _inner_contig(bias if bias.dtype == dtype else bias.to(dtype))
    scale = float(q.shape[3]) ** -0.5 if softmax_scale is None else float(softmax_scale)
    if not 0.0 < scale < float("inf"):
        raise ValueError(f"softmax_scale must be positive and finite, got {scale}")
    graph = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (bias is not None and bias.requires_grad))
    if graph:
        _check_gradient(q, k, bias)
    with ops._on_device(q.device):   # (the call as a plain one: what it gives, gradients too, is not a question of how it came)
        out = _host.cross_attention(q, k, v, None if keep is None else keep.view(torch.bool), bias, scale)
    if out is not None:
        return out if out.__class__ is not int else _lib.check(out, "af3_cross_attention_forward")
    if graph:
        with ops._on_device(q.device):
            _host.check_capture(q, k, v, bias)
        return _CrossAttention.apply(q, k, v, keep, bias, scale)
    return _forward(q, k, v, keep, bias, scale, False)[0]


# ---- relative position bias ---------------------------------------------------------------------------------------------------
def _position_params(table_shape, strides, dtype, q_len, k_len, settings, q_positions, k_positions) -> PositionBiasParams:
    scheme, bidirectional, max_distance, q_offset = settings
    p = PositionBiasParams()
    p.buckets, p.H = table_shape
    p.table_stride = _i64x2(*strides)
    p.Lq, p.Lk, p.max_distance, p.q_offset = q_len, k_len, max_distance, q_offset
    p.scheme, p.bidirectional, p.dtype = _lib.POSITION_SCHEMES[scheme], int(bidirectional), _DTYPES[dtype]
    if q_positions is not None:
        p.q_positions = q_positions.data_ptr()
    if k_positions is not None:
        p.k_positions = k_positions.data_ptr()
    return p


def _position_forward(table, q_len, k_len, settings, q_positions, k_positions):
    out = torch.empty(table.shape[1], q_len, k_len, dtype=table.dtype, device=table.device)
    if out.numel() == 0:
        return out
    p = _position_params(table.shape, table.stride(), table.dtype, q_len, k_len, settings, q_positions, k_positions)
    p.table, p.out = table.data_ptr(), out.data_ptr()
    with ops._on_device(table.device):
        _lib.check(_lib.load().af3_position_bias_forward(ctypes.byref(p), ops._stream_ptr(table.device)), "af3_position_bias_forward")
    return out


def _position_sums(grad, lost, table_shape, settings, q_positions, k_positions):
    """The table's gradient of a gradient [H, Lq, Lk] of the bias; with what that one's rounding lost (laid out like it): what the first call misses."""
    out = torch.empty(table_shape, dtype=grad.dtype, device=grad.device)
    if grad.numel() == 0:
        return out.zero_()
    grad = _inner_contig(grad)
    p = _position_params(table_shape, out.stride(), grad.dtype, grad.shape[1], grad.shape[2], settings, q_positions, k_positions)
    p.grad, p.grad_stride, p.out = grad.data_ptr(), _i64x2(grad.stride(0), grad.stride(1)), out.data_ptr()
    if lost is not None:
        p.grad_residual = lost.data_ptr()
    lib = _lib.load()
    with ops._on_device(grad.device):
        need = lib.af3_position_bias_workspace_bytes(ctypes.byref(p))
        _lib.check(min(need, 0), "af3_position_bias_workspace_bytes")
        ws = torch.empty(need, dtype=torch.uint8, device=grad.device)
        p.workspace, p.workspace_bytes = ws.data_ptr(), need
        _lib.check(lib.af3_position_bias_backward(ctypes.byref(p), ops._stream_ptr(grad.device)), "af3_position_bias_backward")
    return out


class _PositionBias(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, q_len, k_len, settings, q_positions, k_positions):
        ctx.save_for_backward(q_positions, k_positions)
        ctx.table_shape, ctx.settings = table.shape, settings
        return _position_forward(table, q_len, k_len, settings, q_positions, k_positions)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        _no_tangents("the gradient of relative_position_bias", grad)
        q_positions, k_positions = ctx.saved_tensors
        return _position_sums(grad, None, ctx.table_shape, ctx.settings, q_positions, k_positions), None, None, None, None, None


def _check_settings(buckets, scheme, bidirectional, max_distance, q_offset):
    if scheme not in _lib.POSITION_SCHEMES:
        raise ValueError(f"scheme must be 'log' or 'clip', got {scheme!r}")
    if not 1 <= max_distance < 1 << 30:
        raise ValueError(f"max_distance must be 1 to 2^30 - 1, got {max_distance}")
    if abs(q_offset) > 1 << 62:
        raise ValueError(f"q_offset must lie within 2^62, got {q_offset}")
    if not 1 <= buckets <= _lib.POSITION_BIAS_MAX_BUCKETS:
        raise ValueError(f"the table must have 1 to {_lib.POSITION_BIAS_MAX_BUCKETS} buckets, got {buckets}")
    if scheme == "clip":
        want = max_distance * (2 if bidirectional else 1) + 1
        if buckets != want:
            raise ValueError(f"scheme 'clip' with max_distance={max_distance}, bidirectional={bool(bidirectional)} takes {want} buckets, the table has {buckets}")
    else:
        if bidirectional and buckets % 2:
            raise ValueError(f"a bidirectional table of scheme 'log' has an even number of buckets, got {buckets}")
        near = (buckets // 2 if bidirectional else buckets) // 2
        if near < 1 or max_distance <= near:
            raise ValueError(f"scheme 'log' gives the first half of a side's buckets one distance each: with {buckets} buckets max_distance must be above {near} (and {near} at least 1), got {max_distance}")


def _positions_of(t, n, name):
    if t is None:
        return None
    if t.dim() != 1 or t.shape[0] != n or t.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{name} must be int64 or int32 of shape [{n}], got {t.dtype} {tuple(t.shape)}")
    return t.to(torch.int64).contiguous()


def relative_position_bias(table: torch.Tensor, q_len: int, k_len: int, scheme: str = "log", bidirectional: bool = True, max_distance: int = 128,
                           q_positions: Optional[torch.Tensor] = None, k_positions: Optional[torch.Tensor] = None, q_offset: int = 0) -> torch.Tensor:
    """The learned bias [H, q_len, k_len] of a table [buckets, H] (float32 or bfloat16, an Embedding's weight), in the layout and dtype that the
    attention calls take: bias[h, i, j] = table[bucket(i, j), h] for the distance between query i and key j.

    scheme "log": every side has n = buckets / 2 (bidirectional) or buckets; distances below near = n // 2 have a bucket each, from there
    near + floor((n - near) log(d / near) / log(max_distance / near)), at most n - 1, worked out in whole numbers so that distances at a
    border fall where the formula puts them.  Bidirectional: keys ahead of the query take the second n buckets; otherwise they count as
    distance 0.  scheme "clip": bucket = position of the query - position of the key limited to -max_distance .. max_distance, plus max_distance
    (2 max_distance + 1 buckets), or limited to 0 .. max_distance (max_distance + 1 buckets) if not bidirectional; with residue numbers
    as positions that is what AlphaFold 3's relative residue encoding does within a chain (pairs of different chains, which have a bucket of their own
    there, fall where their numbers put them here).

    Positions are 0, 1, 2, ... for keys and q_offset, q_offset + 1, ... for queries (a decoder's token t: q_len=1, q_offset=t), or what q_positions [q_len]
    and k_positions [k_len] hold (int64 or int32, on the table's device; q_offset then does not count for queries).
    The gradient flows to the table: the sums by bucket, in a fixed order, of the gradient that arrives at the bias.  That of a bfloat16 bias has been rounded to bfloat16 by
    then, which a sum of such terms feels; a bias that one cross_attention call and nothing else has, with no hook on the way of its gradient, has its table's gradient from
    what there was before that rounding instead (not without the native host module, nor if the table was changed in place in between, nor for a gradient with a graph)."""
    out = _host.position_bias(table, q_len, k_len, _lib.POSITION_SCHEMES.get(scheme, -1), bidirectional, max_distance, q_positions, k_positions, q_offset)
    if out is not None:
        return out if out.__class__ is not int else _lib.check(out, "af3_position_bias_forward")
    _no_tangents("relative_position_bias", table)
    _same_device(table, q_positions, k_positions)
    if table.dim() != 2:
        raise ValueError(f"table must be [buckets, H], got {tuple(table.shape)}")
    if table.dtype not in _DTYPES:
        raise ValueError(f"unsupported dtype {table.dtype}: float32 or bfloat16")
    q_len, k_len, max_distance, q_offset = int(q_len), int(k_len), int(max_distance), int(q_offset)
    if q_len < 0 or k_len < 0 or q_len >= 1 << 30 or k_len >= 1 << 30:
        raise ValueError(f"q_len and k_len must be 0 to 2^30 - 1, got {q_len} and {k_len}")
    _check_settings(table.shape[0], scheme, bidirectional, max_distance, q_offset)
    q_positions, k_positions = _positions_of(q_positions, q_len, "q_positions"), _positions_of(k_positions, k_len, "k_positions")
    settings = (scheme, bool(bidirectional), max_distance, q_offset)
    with ops._on_device(table.device):   # (as a plain call)
        out = _host.position_bias(table, q_len, k_len, _lib.POSITION_SCHEMES[scheme], settings[1], max_distance, q_positions, k_positions, q_offset)
    if out is not None:
        return out if out.__class__ is not int else _lib.check(out, "af3_position_bias_forward")
    if torch.is_grad_enabled() and table.requires_grad:
        with ops._on_device(table.device):
            _host.check_capture(table)
        return _PositionBias.apply(table, q_len, k_len, settings, q_positions, k_positions)
    return _position_forward(table, q_len, k_len, settings, q_positions, k_positions)
