"""Who follows torch's operations on an operator's inputs, other than for gradients: the operators, which go by address, refuse them, and a decoder's MLP
takes torch's operations."""
from dataclasses import replace

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from cascading_kv_cache_amd.decoder import PRESETS, CascadeDecoder, GatedMLP
from cascading_kv_cache_amd.feed_forward import gated_feed_forward
from cascading_kv_cache_amd.norm_rotate import norm_rotate
from cascading_kv_cache_amd.row_products import followed, followed_beyond_gradients
from cascading_kv_cache_amd.sampling import sample_tokens


class Elsewhere(torch.Tensor):
    """A subclass whose own storage holds nothing."""

    @staticmethod
    def __new__(cls, like):
        return torch.Tensor._make_wrapper_subclass(cls, like.shape, dtype=like.dtype, device=like.device)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise AssertionError(func)


def norm(t):
    return norm_rotate(t, t, torch.ones(8), torch.ones(8))[0]


def weight_of_norm(t):
    x = torch.ones(1, 2, 3, 8)
    return norm_rotate(x, x, t, t)[0]


def ffn(t):
    return gated_feed_forward(t, torch.ones(6, 8))


def weight_of_ffn(t):
    return gated_feed_forward(torch.ones(2, 8), t)


def sample(t):
    return sample_tokens(t, torch.full((2,), 0.5))[1]


def temperature(t):
    return sample_tokens(torch.ones(2, 8), torch.full((2,), 0.5), temperature=t)[1]


CALLS = [(norm, (1, 2, 3, 8)), (weight_of_norm, (8,)), (ffn, (2, 8)), (weight_of_ffn, (6, 8)), (sample, (2, 8)), (temperature, (2,))]
ids = [c.__name__ for c, _ in CALLS]


@pytest.mark.parametrize("call,shape", CALLS, ids=ids)
def test_refused(call, shape):
    x = torch.ones(shape)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward mode"):
        call(forward_ad.make_dual(x, x))
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(call, x, check_trace=False)
    with pytest.raises(RuntimeError, match="traced"):
        make_fx(call)(x)
    with pytest.raises(RuntimeError, match="transforms"):
        torch.vmap(call)(torch.ones(3, *shape))
    with pytest.raises(RuntimeError, match="transforms"):
        torch.func.jvp(call, (x,), (x,))
    with pytest.raises(RuntimeError, match="transforms"):
        torch.func.grad(lambda t: call(t).sum())(x)
    with pytest.raises(TypeError, match="Elsewhere"):
        call(Elsewhere(x))


@pytest.mark.parametrize("call,shape", CALLS, ids=ids)
def test_others_are_not_in_the_way(call, shape):
    """A level or a mode that none of the inputs belongs to, a parameter, a subclass with data of its own: the call goes on to the next check."""
    x = torch.ones(shape)

    class Named(torch.Tensor):
        pass

    for t in (torch.nn.Parameter(x), x.as_subclass(Named)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call(t)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="no CPU fallback"):
        call(x)
    with torch.utils._python_dispatch.TorchDispatchMode(), pytest.raises(RuntimeError):
        call(x)


def mlp(fused):
    torch.manual_seed(0)
    m = GatedMLP(PRESETS["tiny"], torch.float32, "cpu")
    if fused:
        m.fuse_projections()
        m.one_launch = True
    return m


def test_a_decoders_mlp_goes_back_to_torchs_operations():
    """The product of 256 terms of both weights at a time has sums of another order: half a step of float32 of each, 256 * 2^-24 of their sizes."""
    plain, fused = mlp(False), mlp(True)
    x, t = torch.randn(3, 256), torch.randn(3, 256)
    with torch.no_grad():
        with forward_ad.dual_level():
            want, got = (forward_ad.unpack_dual(m(forward_ad.make_dual(x, t))) for m in (plain, fused))
        for a, b in zip(got, want):
            assert b is not None and torch.allclose(a, b, rtol=1e-4, atol=1e-5)
        traced = torch.jit.trace(fused, x, check_trace=False)
        y = torch.randn(3, 256)
        assert torch.allclose(traced(y), plain(y), rtol=1e-4, atol=1e-5)
        assert torch.allclose(make_fx(fused)(x)(y), plain(y), rtol=1e-4, atol=1e-5)
        many = torch.randn(4, 3, 256)
        assert torch.allclose(torch.vmap(fused)(many), plain(many), rtol=1e-4, atol=1e-5)
        with pytest.raises(RuntimeError, match="no CPU fallback"):   # which nobody follows
            fused(x)


def test_who_follows():
    x = torch.ones(2)
    assert followed(x) and not followed_beyond_gradients(x)
    with torch.no_grad():
        assert not followed(x) and followed(x.requires_grad_()) and not followed_beyond_gradients(x)
        x = torch.ones(2)
        with forward_ad.dual_level():
            assert followed(x) and followed_beyond_gradients(x)


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["norm_rotate", "gated_feed_forward"])
def test_backward_passes_of_followed_gradients(which):
    if which == "norm_rotate":
        x = torch.randn(1, 2, 3, 8, device="cuda", requires_grad=True)
        w = torch.ones(8, device="cuda")
        out = norm_rotate(x, x, w, w)[0]
    else:
        x = torch.randn(3, 8, device="cuda", requires_grad=True)
        out = gated_feed_forward(x, torch.ones(16, 8, device="cuda"))
    one = torch.ones_like(out)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward mode"):
        torch.autograd.grad(out, x, forward_ad.make_dual(one, one), retain_graph=True)
    with pytest.raises(RuntimeError, match="transforms|data pointer"):
        torch.autograd.grad(out, x, one.expand(2, *one.shape), is_grads_batched=True, retain_graph=True)
    assert torch.autograd.grad(out, x, one)[0].isfinite().all()


@pytest.mark.gpu
def test_a_decoders_mlp_on_the_device():
    plain, fused = mlp(False).cuda(), mlp(False).cuda()
    fused.fuse_projections()
    fused.one_launch = True
    x, t, y = (torch.randn(3, 256, device="cuda") for _ in range(3))
    with torch.no_grad():
        with forward_ad.dual_level():
            want, got = (forward_ad.unpack_dual(m(forward_ad.make_dual(x, t))) for m in (plain, fused))
        for a, b in zip(got, want):
            assert b is not None and torch.allclose(a, b, rtol=1e-4, atol=1e-5)
        assert torch.allclose(torch.jit.trace(fused, x, check_trace=False)(y), fused(y), rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("hidden,inter,whole", [(256, 512, True), (256, 510, False), (252, 512, False)])
def test_layers_that_the_operator_is_slow_for_keep_torchs_products(hidden, inter, whole, dtype):
    model = CascadeDecoder(replace(PRESETS["tiny"], hidden_size=hidden, intermediate_size=inter), dtype, "cpu")
    assert all(layer.mlp.one_launch == (whole or dtype == torch.float32) for layer in model.fuse_projections(feed_forward=True).layers)
