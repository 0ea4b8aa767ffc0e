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

from . import _abi
from .cascading_cache import _require_device, on_device, raw_stream
from .row_products import refuse_followers

MAX_HEAD_DIM = 256


# What is known of a call by its tensors' sizes, strides, types and devices alone: that the checks passed, and the argument block without
# pointers.  Nothing of a tensor's address or contents.  A single token's call is bound by the host: 19 us with all of this every time.
_LAYOUTS = {}


class _Layout:
    def __init__(self, q, k, q_weight, k_weight, positions, inv_freq, out):
        a = _abi.NormRotateArgs()
        self._strides(a, q_stride=q, k_stride=k)
        if inv_freq is not None:
            a.pos_stride = positions.stride(0) if positions.ndim == 2 and positions.size(0) > 1 else 0
            a.rot = 2 * inv_freq.numel()
        a.B, a.H, a.n, a.D = q.shape
        a.KVH = k.size(1)
        a.dtype = _abi.dtype_code(q.dtype)
        self.common = bytes(a)
        # not torch.empty_like: the inputs are usually parts of one wider buffer, and may be expanded
        self._strides(a, **dict(zip(("q_out_stride", "k_out_stride"), out or (q.new_empty(q.shape), k.new_empty(k.shape)))))
        self.forward = bytes(a)
        self.backward = {}
        self.scratch = _abi.lib().ckv_norm_rotate_workspace_bytes(a.D)

    @staticmethod
    def _strides(a, **tensors):
        for field, t in tensors.items():
            array = getattr(a, field)
            _abi.set_strides(array, t)
            array[3] = 1   # of a single head dim torch may say anything

    def block(self, grads=None, dq=None, dk=None):
        """A copy of the block (the backward runs on a thread of autograd's own)."""
        if grads is None:
            return _abi.NormRotateArgs.from_buffer_copy(self.forward)
        key = (grads[0].stride(), grads[1].stride())
        known = self.backward.get(key)
        if known is None:
            a = _abi.NormRotateArgs.from_buffer_copy(self.common)
            self._strides(a, q_grad_stride=grads[0], k_grad_stride=grads[1], dq_stride=dq, dk_stride=dk)
            if len(self.backward) > 64:
                self.backward.clear()
            known = self.backward[key] = bytes(a)
        return _abi.NormRotateArgs.from_buffer_copy(known)


def _point(a, q, k, q_weight, k_weight, positions, inv_freq, eps):
    a.q, a.k = q.data_ptr(), k.data_ptr()
    if q_weight is not None:
        a.q_weight, a.k_weight = q_weight.data_ptr(), k_weight.data_ptr()
    if inv_freq is not None:
        a.positions, a.inv_freq = positions.data_ptr(), inv_freq.data_ptr()
    a.eps = eps


def _forward(layout, q, k, q_weight, k_weight, positions, inv_freq, eps, out=None):
    q_out, k_out = out or (q.new_empty(q.shape), k.new_empty(k.shape))
    a = layout.block()
    _point(a, q, k, q_weight, k_weight, positions, inv_freq, eps)
    a.q_out, a.k_out = q_out.data_ptr(), k_out.data_ptr()
    device = q.device
    with on_device(device):
        _abi.check(_abi.lib().ckv_norm_rotate(C.byref(a), raw_stream(device)), "ckv_norm_rotate")
    return q_out, k_out


class _Refused(torch.autograd.Function):

    @staticmethod
    def forward(ctx, many, *tensors):
        return tuple(t.view_as(t) for t in tensors[:many])

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("gradients of this operator have none of their own (once_differentiable)")


def once(results, tensors):
    """Gradients in a graph that is made of them: as ``torch.autograd.function.once_differentiable``, which lets a second time pass as if nothing led from
    the operator's inputs to its gradients where the gradient handed to it has no graph, but refused on every way to ``tensors``."""
    there = [r for r in results if r is not None]
    refused = iter(_Refused.apply(len(there), *there, *(t for t in tensors if t is not None and t.requires_grad)))
    return tuple(None if r is None else next(refused) for r in results)


class _NormRotate(torch.autograd.Function):

    @staticmethod
    def forward(ctx, layout, eps, q, k, q_weight, k_weight, positions, inv_freq):
        ctx.save_for_backward(q, k, q_weight, k_weight, positions, inv_freq)
        ctx.layout, ctx.eps = layout, eps
        return _forward(layout, q, k, q_weight, k_weight, positions, inv_freq, eps)

    @staticmethod
    def backward(ctx, *grads):
        if not torch.is_grad_enabled():
            return _gradients(ctx, *grads)
        with torch.no_grad():
            results = _gradients(ctx, *grads)
        return once(results, (*ctx.saved_tensors, *grads))


def _gradients(ctx, *grads):
    q, k, q_weight, k_weight, positions, inv_freq = ctx.saved_tensors
    refuse_followers("norm_rotate's backward pass", *grads)
    # a gradient may be an expanded scalar, or in an order of its own
    q_grad, k_grad = (g if g.stride(-1) == 1 or g.size(-1) == 1 else g.contiguous() for g in grads)
    dq, dk = q.new_empty(q.shape), k.new_empty(k.shape)
    a = ctx.layout.block((q_grad, k_grad), dq, dk)
    _point(a, q, k, q_weight, k_weight, positions, inv_freq, ctx.eps)
    a.q_grad, a.k_grad, a.dq, a.dk = q_grad.data_ptr(), k_grad.data_ptr(), dq.data_ptr(), dk.data_ptr()
    dqw = dkw = None
    device = q.device
    with on_device(device):
        if q_weight is not None:
            dqw, dkw = q_weight.new_empty(q_weight.shape), k_weight.new_empty(k_weight.shape)
            a.dq_weight, a.dk_weight = dqw.data_ptr(), dkw.data_ptr()
            # of this call alone: a graph that records it must share its scratch with nobody
            ws = torch.empty(ctx.layout.scratch, dtype=torch.uint8, device=device)
            a.workspace, a.workspace_bytes = ws.data_ptr(), ctx.layout.scratch
        _abi.check(_abi.lib().ckv_norm_rotate_bwd(C.byref(a), raw_stream(device)), "ckv_norm_rotate_bwd")
    return None, None, dq, dk, dqw, dkw, None, None


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
    if len(out) != 2:
        raise ValueError(f"out is {len(out)} tensors; expected one for the queries and one for the keys")
    for name, t, like in (("queries", out[0], q), ("keys", out[1], k)):
        if t.dtype != like.dtype or t.device != like.device or t.shape != like.shape:
            raise ValueError(f"out holds {name} {tuple(t.shape)} of {t.dtype} on {t.device}; expected {tuple(like.shape)} of {like.dtype} on {like.device}")
        if t.size(-1) > 1 and t.stride(-1) != 1:
            raise ValueError("the head dims of out are not adjacent")
        if any(s == 0 for n, s in zip(t.shape, t.stride()) if n > 1):
            raise ValueError("out is expanded: its rows are not its own")


def _written(out, tensors):
    """What a call that writes ``out`` asks of where its tensors lie, and its announcement to whoever has saved one of them."""
    if out[0].numel():
        at = [None if t is None else t.data_ptr() for t in tensors]
        for i, t in enumerate(out):
            own, here = tensors[i], t.data_ptr()
            if here in at[:i] + at[i + 1:] or here == out[1 - i].data_ptr():
                raise ValueError("out lies where something else is: the queries' may be the queries, the keys' the keys")
            if here == at[i] and any(n > 1 and a != b for n, a, b in zip(t.shape, t.stride(), own.stride())):
                raise ValueError("out begins where its input does, in another order")
    for t in out:
        if not t.is_inference():   # those have no versions
            torch.autograd.graph.increment_version(t)


def norm_rotate(q, k, q_weight=None, k_weight=None, positions=None, inv_freq=None, eps=1e-6, out=None):
    """``(q, k)`` with every head's row normed and rotated, contiguous, or written to ``out``: two tensors of their shapes, apart from the inputs
    and each other, or the inputs themselves (a decoding step has no other use for them); such a call has no gradients, and counts as one of torch's
    operations in place: who has saved one of the two for a backward pass is told.

    q ``(B, H, n, D)`` and k ``(B, KVH, n, D)``, float32, float16 or bfloat16, any strides.  ``q_weight``, ``k_weight`` ``(D,)``, dtype of q: the
    weights of the norm, or None for no norm.  ``positions`` int64 ``(n,)`` or ``(B, n)`` and ``inv_freq`` float32 ``(R / 2,)``: the first
    R <= D dims are rotated, dim j with dim j + R / 2 by ``position * inv_freq[j]``; or None for no rotation.  Gradients go back to q, k
    and the weights (once: not a second time, and not by forward mode, torch.func's transforms or a trace, which are refused).  Works under graph capture; nothing of the tensors is kept between calls.  Recorded into a graph, a
    backward pass wants no eager graph of the same leaves alive: torch would have the recording wait for it."""
    tensors = q, k, q_weight, k_weight, positions, inv_freq
    refuse_followers("norm_rotate", *tensors)
    followed = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors[:4])
    if out is not None:
        out = tuple(out)
        if followed or (torch.is_grad_enabled() and any(t.requires_grad for t in out)):
            raise ValueError("no gradients go through out")
        refuse_followers("norm_rotate", *out)
    key = [(t.shape, t.stride(), t.dtype, t.device) if t is not None else None for t in (tensors if out is None else tensors + out)]
    key = tuple(key)
    layout = _LAYOUTS.get(key)
    if layout is None or (inv_freq is not None and inv_freq.requires_grad):
        _check(*tensors)
        if out is not None:
            _check_out(out, q, k)
        q, k = (t if t.stride(-1) == 1 or t.size(-1) == 1 else t.contiguous() for t in (q, k))
        q_weight, k_weight, inv_freq = (None if t is None else t.contiguous() for t in (q_weight, k_weight, inv_freq))
        if positions is not None and positions.stride(-1) != 1:
            positions = positions.contiguous()
        layout = _Layout(q, k, q_weight, k_weight, positions, inv_freq, out)
        if all(a is b for a, b in zip(tensors, (q, k, q_weight, k_weight, positions, inv_freq))):   # nothing to lay out at the next call either
            if len(_LAYOUTS) > 256:
                _LAYOUTS.clear()
            _LAYOUTS[key] = layout
    if followed:
        return _NormRotate.apply(layout, float(eps), q, k, q_weight, k_weight, positions, inv_freq)
    if out is not None:
        _written(out, tensors)
    return _forward(layout, q, k, q_weight, k_weight, positions, inv_freq, float(eps), out)
