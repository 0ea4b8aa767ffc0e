"""The first half of a gated MLP in one launch of the library, with gradients: ``silu(x Wg^T) * (x Wu^T)``.

    hidden = gated_feed_forward(x, w_gate_up)      # what GatedMLP keeps in one buffer: gate rows, then up rows
    y = down_proj(hidden)

The reference's models run three of torch's operations there (cascade/models/llama/modeling_llama.py, LlamaMLP).  Everything is float32 and
rounded once, where ``gated_silu`` behind a product, and the fused products of a decoding step (``row_products.py``), keep the bits of those
operations and round three times.
"""
import torch

from . import _abi
from .cascading_cache import _require_device, on_device, raw_stream
from .norm_rotate import once
from .row_products import refuse_followers


def _scratch(nbytes, device):
    # of this call alone: a graph that records it must share its scratch with nobody
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _at(t):
    return None if t is None else t.data_ptr()


def _forward(x, w, both):
    rows, k = x.shape
    inter = w.size(0) // 2
    lib, code = _abi.lib(), _abi.dtype_code(x.dtype)
    out = torch.empty(rows, inter, dtype=x.dtype, device=x.device)
    gate_up = torch.empty(rows, 2 * inter, dtype=torch.float32, device=x.device) if both else None
    with on_device(x.device):
        ws = _scratch(lib.ckv_gated_linear_workspace_bytes(rows, inter, k, code), x.device)
        _abi.check(lib.ckv_gated_linear(_at(x), _at(w), _at(out), _at(gate_up), rows, inter, k, x.stride(0) if rows > 1 else k, code, _at(ws),
                                        0 if ws is None else ws.numel(), raw_stream(x.device)), "ckv_gated_linear")
    return out, gate_up


class _GatedFeedForward(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, w):
        out, gate_up = _forward(x, w, True)
        ctx.save_for_backward(x, w, gate_up)
        return out

    @staticmethod
    def backward(ctx, dout):
        if not torch.is_grad_enabled():
            return _gradients(ctx, dout)
        with torch.no_grad():
            results = _gradients(ctx, dout)
        return once(results, (*ctx.saved_tensors[:2], dout))


def _gradients(ctx, dout):
    x, w, gate_up = ctx.saved_tensors
    refuse_followers("gated_feed_forward's backward pass", dout)
    rows, k = x.shape
    inter = w.size(0) // 2
    lib, code = _abi.lib(), _abi.dtype_code(x.dtype)
    dout = dout.to(x.dtype).contiguous()
    dx = torch.empty(rows, k, dtype=x.dtype, device=x.device) if ctx.needs_input_grad[0] else None
    dw = torch.empty(w.shape, dtype=w.dtype, device=w.device) if ctx.needs_input_grad[1] else None
    with on_device(x.device):
        ws = _scratch(lib.ckv_gated_linear_bwd_workspace_bytes(rows, inter, k, code), x.device)
        _abi.check(lib.ckv_gated_linear_bwd(_at(x), _at(w), _at(gate_up), _at(dout), _at(dx), _at(dw), rows, inter, k,
                                            x.stride(0) if rows > 1 else k, code, _at(ws), 0 if ws is None else ws.numel(),
                                            raw_stream(x.device)), "ckv_gated_linear_bwd")
    return dx, dw


def gated_feed_forward(x, w_gate_up):
    """``silu(gate) * up`` of ``gate | up = x w_gate_up^T``: x ``(..., K)``, w_gate_up ``(2 I, K)``, one type of float32, float16 and
    bfloat16; returns ``(..., I)``.  Gradients go back to both (once: not a second time, and not by forward mode, torch.func's transforms or a
    trace, which are refused); the projections are kept for that in
    float32, ``2 I`` elements a row; their gradients are rounded to the tensor type for the two products (float16: times a power of two a row,
    so that none of them is above its end, or below its beginning beside the row's others).  In 16 bits, sizes, strides
    and addresses of whole eight elements are what it is fast for; others are multiplied on float32's instructions, some ten times slower.  Works under graph
    capture; nothing is kept between calls.  Recorded into a graph, a backward pass wants no eager graph of the same leaves alive: torch would have the recording
    wait for it."""
    refuse_followers("gated_feed_forward", x, w_gate_up)
    if w_gate_up.ndim != 2 or w_gate_up.size(0) % 2 or w_gate_up.size(0) == 0 or w_gate_up.size(1) == 0:
        raise ValueError(f"weights have shape {tuple(w_gate_up.shape)}; expected (2 * intermediate, hidden)")
    if x.ndim == 0 or x.size(-1) != w_gate_up.size(1):
        raise ValueError(f"rows have shape {tuple(x.shape)}; expected (..., {w_gate_up.size(1)})")
    _abi.dtype_code(x.dtype)
    if w_gate_up.dtype != x.dtype:
        raise TypeError(f"rows are {x.dtype}, the weights {w_gate_up.dtype}")
    _require_device(x, "x")
    _require_device(w_gate_up, "w_gate_up")
    if w_gate_up.device != x.device:
        raise ValueError(f"rows live on {x.device}, the weights on {w_gate_up.device}")
    rows = x.reshape(-1, x.size(-1))
    if rows.stride(1) != 1 and rows.size(1) > 1 or rows.size(0) > 1 and rows.stride(0) < rows.size(1):
        rows = rows.contiguous()
    w = w_gate_up.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad):
        out = _GatedFeedForward.apply(rows, w)
    else:
        out = _forward(rows, w, False)[0]
    return out.view(*x.shape[:-1], out.size(-1))
