"""What the operators around attention refuse, before anything reaches a device."""
import ctypes as C
import os

import pytest
import torch

from cascading_kv_cache_amd import _abi
from cascading_kv_cache_amd.feed_forward import gated_feed_forward
from cascading_kv_cache_amd.norm_rotate import norm_rotate
from cascading_kv_cache_amd.sampling import sample_tokens


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_abi.LIB_PATH):
        from cascading_kv_cache_amd import build

        build.build(verbose=False)
    return _abi.lib()


def heads(**change):
    a = dict(q=torch.zeros(2, 4, 3, 8), k=torch.zeros(2, 2, 3, 8), q_weight=torch.ones(8), k_weight=torch.ones(8),
             positions=torch.arange(3), inv_freq=torch.ones(4))
    a.update(change)
    return a


@pytest.mark.parametrize("change,error,text", [
    (dict(q=torch.zeros(4, 3, 8)), ValueError, "batch, heads"),
    (dict(k=torch.zeros(2, 2, 4, 8)), ValueError, "differ"),
    (dict(k=torch.zeros(1, 2, 3, 8)), ValueError, "differ"),
    (dict(k=torch.zeros(2, 0, 3, 8)), ValueError, "have none"),
    (dict(q=torch.zeros(2, 4, 3, 257), k=torch.zeros(2, 2, 3, 257)), ValueError, "head_dim"),
    (dict(q=torch.zeros(2, 4, 3, 8, dtype=torch.float64)), TypeError, "float64"),
    (dict(k=torch.zeros(2, 2, 3, 8, dtype=torch.float16)), TypeError, "k is"),
    (dict(q_weight=torch.ones(8, dtype=torch.bfloat16)), TypeError, "q_weight"),
    (dict(q_weight=None), ValueError, "together"),
    (dict(positions=None), ValueError, "together"),
    (dict(q_weight=None, k_weight=None, positions=None, inv_freq=None), ValueError, "nothing to do"),
    (dict(positions=torch.arange(3, dtype=torch.int32)), TypeError, "positions"),
    (dict(inv_freq=torch.ones(4, dtype=torch.float64)), TypeError, "inv_freq"),
    (dict(), _abi.CkvError, "no CPU fallback"),
])
def test_norm_rotate(change, error, text):
    with pytest.raises(error, match=text):
        norm_rotate(**heads(**change))


@pytest.mark.gpu
@pytest.mark.parametrize("change,error,text", [
    (dict(q_weight=torch.ones(4), k_weight=torch.ones(4)), ValueError, "shapes"),
    (dict(positions=torch.arange(4)), ValueError, "positions"),
    (dict(positions=torch.zeros(3, 3, dtype=torch.int64)), ValueError, "positions"),
    (dict(inv_freq=torch.ones(5)), ValueError, "inv_freq"),
    (dict(inv_freq=torch.ones(0)), ValueError, "inv_freq"),
    (dict(inv_freq=torch.ones(4).requires_grad_()), ValueError, "gradient"),
])
def test_norm_rotate_on_the_device(change, error, text):
    args = {n: t.detach().cuda().requires_grad_(t.requires_grad) for n, t in heads(**change).items()}
    with pytest.raises(error, match=text):
        norm_rotate(**args)
    with pytest.raises((ValueError, _abi.CkvError)):
        norm_rotate(**{n: t.cuda() if n != "k_weight" else t for n, t in heads().items()})


def test_norm_rotate_in_c(lib):
    a = _abi.NormRotateArgs()
    assert lib.ckv_norm_rotate(None, None) == -1
    a.dtype = 9
    assert lib.ckv_norm_rotate(C.byref(a), None) == -4
    a.dtype, a.B, a.H, a.KVH, a.n, a.D = _abi.CKV_BF16, 1, 4, 2, 3, 64
    for name, value, status in (("rot", 66, -2), ("rot", 3, -2), ("H", 0, -2), ("n", -1, -2), ("D", 512, -6)):
        was = getattr(a, name)
        setattr(a, name, value)
        assert lib.ckv_norm_rotate(C.byref(a), None) == status, name
        setattr(a, name, was)
    assert lib.ckv_norm_rotate(C.byref(a), None) == -1               # no tensors
    a.q_weight = 16
    assert lib.ckv_norm_rotate(C.byref(a), None) == -1               # one weight of two
    a.k_weight = a.dq_weight = a.dk_weight = 16
    assert lib.ckv_norm_rotate_bwd(C.byref(a), None) == -5           # no workspace
    a.q_weight = a.k_weight = None
    a.q = a.k = a.q_out = a.k_out = 16
    a.rot = 8
    assert lib.ckv_norm_rotate(C.byref(a), None) == -1               # no positions
    a.rot = 0
    a.q_stride[3] = 2
    assert lib.ckv_norm_rotate(C.byref(a), None) == -3
    assert lib.ckv_norm_rotate_workspace_bytes(0) == lib.ckv_norm_rotate_workspace_bytes(300) == 0 < lib.ckv_norm_rotate_workspace_bytes(128)
    f = C.CDLL(_abi.LIB_PATH).ckv_sizeof_norm_rotate_args
    f.restype = C.c_int64
    assert f() == C.sizeof(_abi.NormRotateArgs)


@pytest.mark.parametrize("x,w,error", [
    (torch.zeros(2, 8), torch.zeros(7, 8), ValueError),
    (torch.zeros(2, 8), torch.zeros(8), ValueError),
    (torch.zeros(2, 8), torch.zeros(0, 8), ValueError),
    (torch.zeros(2, 0), torch.zeros(4, 0), ValueError),
    (torch.zeros(2, 9), torch.zeros(4, 8), ValueError),
    (torch.zeros(()), torch.zeros(4, 8), ValueError),
    (torch.zeros(2, 8, dtype=torch.float64), torch.zeros(4, 8, dtype=torch.float64), TypeError),
    (torch.zeros(2, 8), torch.zeros(4, 8, dtype=torch.float16), TypeError),
    (torch.zeros(2, 8), torch.zeros(4, 8), _abi.CkvError),
])
def test_gated_feed_forward(x, w, error):
    with pytest.raises(error):
        gated_feed_forward(x, w)


def test_gated_linear_in_c(lib):
    forward = lambda **c: lib.ckv_gated_linear(*{**dict(x=16, w=16, out=16, both=None, rows=2, inter=4, k=8, stride=8, dtype=_abi.CKV_BF16,   # noqa: E731
                                                        ws=None, n=0, stream=None), **c}.values())
    assert forward(dtype=7) == -4
    assert forward(rows=-1) == forward(inter=0) == forward(k=0) == forward(stride=7) == -2
    assert forward(inter=1 << 31) == -6
    assert forward(x=None) == forward(w=None) == forward(out=None) == -1
    assert forward(rows=0) == 0
    backward = lambda **c: lib.ckv_gated_linear_bwd(*{**dict(x=16, w=16, both=16, dout=16, dx=16, dw=16, rows=2, inter=4, k=8, stride=8,   # noqa: E731
                                                             dtype=_abi.CKV_F32, ws=None, n=0, stream=None), **c}.values())
    assert backward(dtype=7) == -4 and backward(stride=7) == -2
    assert backward(x=None) == backward(both=None) == backward(dout=None) == -1
    assert backward(dx=None, dw=None) == 0
    assert lib.ckv_gated_linear_workspace_bytes(0, 4, 8, 0) == lib.ckv_gated_linear_bwd_workspace_bytes(4, 4, 8, 7) == 0


@pytest.mark.parametrize("change,error,text", [
    (dict(logits=torch.zeros(8)), ValueError, "rows, vocab"),
    (dict(logits=torch.zeros(3, 8)), ValueError, "rows, vocab"),
    (dict(uniforms=torch.zeros(2, 1)), ValueError, "rows, vocab"),
    (dict(logits=torch.zeros(2, 0)), ValueError, "to draw from"),
    (dict(logits=torch.empty(2, 1 << 20, device="meta")), ValueError, "to draw from"),
    (dict(logits=torch.zeros(2, 8, dtype=torch.float64)), TypeError, "float64"),
    (dict(uniforms=torch.zeros(2, dtype=torch.float64)), TypeError, "random numbers"),
    (dict(temperature=float("nan")), ValueError, "temperature"),
    (dict(top_p=float("nan")), ValueError, "top_p"),
    (dict(top_k=torch.zeros(2)), TypeError, "top_k"),
    (dict(min_p=torch.zeros(2, dtype=torch.float64)), TypeError, "min_p"),
    (dict(temperature=torch.ones(3)), ValueError, "temperature"),
    (dict(temperature=torch.ones(2, device="meta")), ValueError, "temperature"),
    (dict(), _abi.CkvError, "no CPU fallback"),
])
def test_sample_tokens(change, error, text):
    args = dict(logits=torch.zeros(2, 8), uniforms=torch.zeros(2))
    args.update(change)
    with pytest.raises(error, match=text):
        sample_tokens(**args)


def test_sample_in_c(lib):
    assert lib.ckv_sample(None, None) == -1
    a = _abi.SampleArgs()
    a.dtype = 5
    assert lib.ckv_sample(C.byref(a), None) == -4
    a.dtype, a.rows, a.vocab, a.logit_stride = _abi.CKV_F32, 2, 8, 8
    for name, value, status in (("rows", -1, -2), ("vocab", 0, -2), ("logit_stride", -8, -2), ("vocab", 1 << 20, -6)):
        was = getattr(a, name)
        setattr(a, name, value)
        assert lib.ckv_sample(C.byref(a), None) == status, name
        setattr(a, name, was)
    assert lib.ckv_sample(C.byref(a), None) == -1
    a.rows = 0
    assert lib.ckv_sample(C.byref(a), None) == 0
    assert lib.ckv_sample_workspace_bytes(0, 8) == lib.ckv_sample_workspace_bytes(2, 1 << 20) == 0
    f = C.CDLL(_abi.LIB_PATH).ckv_sizeof_sample_args
    f.restype = C.c_int64
    assert f() == C.sizeof(_abi.SampleArgs)
