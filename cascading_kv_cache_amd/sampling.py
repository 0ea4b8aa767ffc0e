"""Tokens drawn from logits by temperature, top-k, top-p and min-p, with random numbers of the caller's.

    tokens, logprobs = sample_tokens(logits, torch.rand(batch, device=logits.device), temperature=0.8, top_p=0.95)

The reference's generation loop is greedy (cascade/models/cascade_attention.py:473-499); ``decoder.generate`` draws through this function
when it is given settings.  The random numbers are inputs, so that a draw can be repeated, recorded into a graph, or checked.
"""
import ctypes as C

import torch

from . import _abi
from .cascading_cache import _require_device, on_device, raw_stream
from .row_products import refuse_followers

MAX_VOCAB = (1 << 19) - 1

#: setting: (field of one number, field of one a row, type of the array)
_SETTINGS = {"temperature": ("temperature", "temperatures", torch.float32), "top_k": ("top_k", "top_ks", torch.int64),
             "top_p": ("top_p", "top_ps", torch.float32), "min_p": ("min_p", "min_ps", torch.float32)}


@torch.no_grad()
def sample_tokens(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """``(tokens int64 (rows,), logprobs float32 (rows,))`` from logits ``(rows, vocab)`` of float32, float16 or bfloat16 and one float32
    number of [0, 1) a row.

    Tokens are ordered by falling logit, equal ones by rising index, and weigh ``exp((logit - largest) / temperature)``.  Kept are the first
    ``top_k`` (0: all); of those the ones with less than ``top_p`` of their weight in front of them (1: all); of those the ones that weigh at
    least ``min_p`` of the first one; the first one always.  The token is the first whose running kept weight exceeds the row's number times
    all of it, ``logprobs`` the logarithm of its share.  Every setting is a number or a tensor with one a row (float32, top_k int64) on the
    logits' device; those are not checked, what lies outside their ranges means the nearest in it.  ``temperature`` 0: the largest logit,
    whatever the number.  Logits of NaN and minus infinity are no tokens; a row without any gives -1 and NaN.  No gradients; traces and torch.func's
    transforms are refused.  Works under graph capture; nothing is kept between calls."""
    refuse_followers("sample_tokens", logits, uniforms, *(t for t in (temperature, top_k, top_p, min_p) if isinstance(t, torch.Tensor)))
    if logits.ndim != 2 or uniforms.shape != logits.shape[:1]:
        raise ValueError(f"logits {tuple(logits.shape)} and random numbers {tuple(uniforms.shape)}; expected (rows, vocab) and (rows,)")
    rows, vocab = logits.shape
    if not 0 < vocab <= MAX_VOCAB:
        raise ValueError(f"{vocab} tokens to draw from; 1 to {MAX_VOCAB} can be")
    a = _abi.SampleArgs()
    a.dtype = _abi.dtype_code(logits.dtype)
    if uniforms.dtype != torch.float32:
        raise TypeError(f"random numbers are {uniforms.dtype}, expected float32")
    dev = logits.device
    held = []   # contiguous copies, until the launch is on its way
    for name, value in (("temperature", temperature), ("top_k", top_k), ("top_p", top_p), ("min_p", min_p)):
        number, array, dtype = _SETTINGS[name]
        if not isinstance(value, torch.Tensor):
            if value != value:
                raise ValueError(f"{name} is not a number")
            # limits beyond 64 bits are none
            setattr(a, number, int(max(0, min(value, MAX_VOCAB + 1))) if name == "top_k" else float(value))
            continue
        if value.dtype != dtype:
            raise TypeError(f"{name} is {value.dtype}, expected {dtype}")
        if value.shape != (rows,):
            raise ValueError(f"{name} has shape {tuple(value.shape)}; expected a number or ({rows},)")
        if value.device != dev:
            raise ValueError(f"{name} lives on {value.device}, the logits on {dev}")
        held.append(value.contiguous())
        setattr(a, array, held[-1].data_ptr())
    _require_device(logits, "logits")
    if uniforms.device != dev:
        raise ValueError(f"random numbers live on {uniforms.device}, the logits on {dev}")
    if logits.stride(1) != 1 and vocab > 1:
        logits = logits.contiguous()
    uniforms = uniforms.contiguous()
    tokens = torch.empty(rows, dtype=torch.int64, device=dev)
    logprobs = torch.empty(rows, dtype=torch.float32, device=dev)
    a.logits, a.uniforms, a.tokens, a.logprobs = logits.data_ptr(), uniforms.data_ptr(), tokens.data_ptr(), logprobs.data_ptr()
    a.logit_stride = logits.stride(0) if rows > 1 else vocab
    a.rows, a.vocab = rows, vocab
    lib = _abi.lib()
    with on_device(dev):
        need = lib.ckv_sample_workspace_bytes(rows, vocab)
        if need:   # of this call alone: a graph that records it must share its scratch with nobody
            ws = torch.empty(need, dtype=torch.uint8, device=dev)
            a.workspace, a.workspace_bytes = ws.data_ptr(), need
        _abi.check(lib.ckv_sample(C.byref(a), C.c_void_p(raw_stream(dev))), "ckv_sample")
    return tokens, logprobs
