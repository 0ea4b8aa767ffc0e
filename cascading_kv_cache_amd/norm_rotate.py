"""RMSNorm of every head's queries and keys and their rotation at the tokens' positions, one launch of the library, with gradients.

    q, k = norm_rotate(q, k, q_weight, k_weight, positions, inv_freq, eps)
    out, scores = attention(q, k, v, True, scale, mask, beta)

Models that norm their heads do so between the projections and the rotation.  In front of the dense operator ``attention``, which takes
rotated queries and keys, both are done here; in front of a cascade cache, which keeps keys un-rotated and rotates them at every call, the
norm alone (no ``positions``).  Where the mixin's ``rope`` (cascade/models/cascade_attention.py:343-353) rounds angle, cos, sin and products
to the tensor dtype on the way, everything here is float32, the angle the exact product of position and frequency, rounded once at the end.
"""
import ctypes as C

import torch
from torch.autograd.function import once_differentiable

from . import _abi
from .cascading_cache import _require_device, on_device, raw_stream

MAX_HEAD_DIM = 256


def _describe(q, k, q_weight, k_weight, positions, inv_freq, eps):
    a = _abi.NormRotateArgs()
    a.q, a.k = q.data_ptr(), k.data_ptr()
    _abi.set_strides(a.q_stride, q)
    _abi.set_strides(a.k_stride, k)
    a.q_stride[3] = a.k_stride[3] = 1   # of a single head dim torch may say anything
    if q_weight is not None:
        a.q_weight, a.k_weight = q_weight.data_ptr(), k_weight.data_ptr()
    if inv_freq is not None:
        a.positions, a.inv_freq = positions.data_ptr(), inv_freq.data_ptr()
        a.pos_stride = positions.stride(0) if positions.ndim == 2 and positions.size(0) > 1 else 0
        a.rot = 2 * inv_freq.numel()
    a.B, a.H, a.n, a.D = q.shape
    a.KVH = k.size(1)
    a.eps = float(eps)
    a.dtype = _abi.dtype_code(q.dtype)
    return a


def _forward(q, k, q_weight, k_weight, positions, inv_freq, eps, out=None):
    # not torch.empty_like: the inputs are usually parts of one wider buffer, and may be expanded
    q_out, k_out = out or (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k))
    a = _describe(q, k, q_weight, k_weight, positions, inv_freq, eps)
    a.q_out, a.k_out = q_out.data_ptr(), k_out.data_ptr()
    _abi.set_strides(a.q_out_stride, q_out)
    _abi.set_strides(a.k_out_stride, k_out)
    a.q_out_stride[3] = a.k_out_stride[3] = 1
    with on_device(q.device):
        _abi.check(_abi.lib().ckv_norm_rotate(C.byref(a), C.c_void_p(raw_stream(q.device))), "ckv_norm_rotate")
    return q_out, k_out


class _NormRotate(torch.autograd.Function):

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, inv_freq, eps):
        ctx.save_for_backward(q, k, q_weight, k_weight, positions, inv_freq)
        ctx.eps = eps
        return _forward(q, k, q_weight, k_weight, positions, inv_freq, eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, q_grad, k_grad):
        q, k, q_weight, k_weight, positions, inv_freq = ctx.saved_tensors
        # a gradient may be an expanded scalar, or in an order of its own
        q_grad, k_grad = (g if g.stride(-1) == 1 or g.size(-1) == 1 else g.contiguous() for g in (q_grad.to(q.dtype), k_grad.to(q.dtype)))
        a = _describe(q, k, q_weight, k_weight, positions, inv_freq, ctx.eps)
        a.q_grad, a.k_grad = q_grad.data_ptr(), k_grad.data_ptr()
        dq, dk = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k))
        a.dq, a.dk = dq.data_ptr(), dk.data_ptr()
        for field, t in ((a.q_grad_stride, q_grad), (a.k_grad_stride, k_grad), (a.dq_stride, dq), (a.dk_stride, dk)):
            _abi.set_strides(field, t)
            field[3] = 1
        dqw = dkw = None
        lib = _abi.lib()
        with on_device(q.device):
            if q_weight is not None:
                dqw, dkw = torch.empty_like(q_weight), torch.empty_like(k_weight)
                a.dq_weight, a.dk_weight = dqw.data_ptr(), dkw.data_ptr()
                # of this call alone: a graph that records it must share its scratch with nobody
                ws = torch.empty(lib.ckv_norm_rotate_workspace_bytes(a.D), dtype=torch.uint8, device=q.device)
                a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
            _abi.check(lib.ckv_norm_rotate_bwd(C.byref(a), C.c_void_p(raw_stream(q.device))), "ckv_norm_rotate_bwd")
        return dq, dk, dqw, dkw, None, None, None


def _check(q, k, q_weight, k_weight, positions, inv_freq):
    if q.ndim != 4 or k.ndim != 4:
        raise ValueError("queries and keys are (batch, heads, tokens, head_dim)")
    B, H, n, D = q.shape
    if (k.size(0), k.size(2), k.size(3)) != (B, n, D) or H == 0 or k.size(1) == 0:
        raise ValueError(f"queries {tuple(q.shape)} and keys {tuple(k.shape)} differ in more than their heads, or have none")
    if not 0 < D <= MAX_HEAD_DIM:
        raise ValueError(f"head_dim is 1 to {MAX_HEAD_DIM}, got {D}")
    _abi.dtype_code(q.dtype)
    if (q_weight is None) != (k_weight is None):
        raise ValueError("weights of the norm for queries and keys come together")
    if (positions is None) != (inv_freq is None):
        raise ValueError("positions and inv_freq come together")
    if q_weight is None and positions is None:
        raise ValueError("nothing to do: neither weights nor positions")
    for name, t, dtype in (("k", k, q.dtype), ("q_weight", q_weight, q.dtype), ("k_weight", k_weight, q.dtype),
                           ("positions", positions, torch.int64), ("inv_freq", inv_freq, torch.float32)):
        if t is not None and t.dtype != dtype:
            raise TypeError(f"{name} is {t.dtype}, expected {dtype}")
    for name, t in (("q", q), ("k", k), ("q_weight", q_weight), ("k_weight", k_weight), ("positions", positions), ("inv_freq", inv_freq)):
        if t is not None:
            _require_device(t, name)
            if t.device != q.device:
                raise ValueError(f"{name} lives on {t.device}, the queries on {q.device}")
    if q_weight is not None and (q_weight.shape != (D,) or k_weight.shape != (D,)):
        raise ValueError(f"weights of the norm have shapes {tuple(q_weight.shape)} and {tuple(k_weight.shape)}, expected ({D},)")
    if positions is not None:
        if positions.shape not in ((n,), (1, n), (B, n)):
            raise ValueError(f"positions have shape {tuple(positions.shape)}; expected ({n},) or ({B}, {n})")
        if inv_freq.ndim != 1 or 2 * inv_freq.numel() > D or inv_freq.numel() == 0:
            raise ValueError(f"inv_freq has shape {tuple(inv_freq.shape)}: a frequency for each of at most {D // 2} pairs")
        if inv_freq.requires_grad:
            raise ValueError("inv_freq has no gradient here")


def _check_out(out, q, k):
    for name, t, like in (("queries", out[0], q), ("keys", out[1], k)):
        if t.dtype != like.dtype or t.device != like.device or t.shape != like.shape:
            raise ValueError(f"out holds {name} {tuple(t.shape)} of {t.dtype} on {t.device}; expected {tuple(like.shape)} of {like.dtype} on {like.device}")
        if t.size(-1) > 1 and t.stride(-1) != 1:
            raise ValueError("the head dims of out are not adjacent")
        if any(s == 0 for n, s in zip(t.shape, t.stride()) if n > 1):
            raise ValueError("out is expanded: its rows are not its own")


def norm_rotate(q, k, q_weight=None, k_weight=None, positions=None, inv_freq=None, eps=1e-6, out=None):
    """``(q, k)`` with every head's row normed and rotated, contiguous, or written to ``out``: two tensors of their shapes, apart from the inputs
    or the inputs themselves (a decoding step has no other use for them); such a call has no gradients.

    q ``(B, H, n, D)`` and k ``(B, KVH, n, D)``, float32, float16 or bfloat16, any strides.  ``q_weight``, ``k_weight`` ``(D,)``, dtype of q: the
    weights of the norm, or None for no norm.  ``positions`` int64 ``(n,)`` or ``(B, n)`` and ``inv_freq`` float32 ``(R / 2,)``: the first
    R <= D dims are rotated, dim j with dim j + R / 2 by ``position * inv_freq[j]``; or None for no rotation.  Gradients go back to q, k
    and the weights (once: not a second time).  Works under graph capture; nothing is kept between calls."""
    _check(q, k, q_weight, k_weight, positions, inv_freq)
    q, k = (t if t.stride(-1) == 1 or t.size(-1) == 1 else t.contiguous() for t in (q, k))
    q_weight, k_weight, inv_freq = (None if t is None else t.contiguous() for t in (q_weight, k_weight, inv_freq))
    if positions is not None and positions.stride(-1) != 1:
        positions = positions.contiguous()
    followed = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight))
    if out is not None:
        if followed:
            raise ValueError("no gradients go through out")
        _check_out(out, q, k)
        return _forward(q, k, q_weight, k_weight, positions, inv_freq, eps, tuple(out))
    if followed:
        return _NormRotate.apply(q, k, q_weight, k_weight, positions, inv_freq, float(eps))
    return _forward(q, k, q_weight, k_weight, positions, inv_freq, eps)
