"""A decoder's MLP whose projections share a buffer, in training: gradients reach the parameters."""
from copy import deepcopy

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch import nn

from cascading_kv_cache_amd.decoder import PRESETS, GatedMLP


def pair(dtype, device, one_launch):
    torch.manual_seed(0)
    plain = GatedMLP(PRESETS["tiny"], dtype, device)
    fused = deepcopy(plain)
    fused.fuse_projections()
    fused.one_launch = one_launch
    return plain, fused


def exact(plain, x, dy):
    """Outputs and gradients in 64 bits: x, gate, up, down."""
    m = deepcopy(plain).double()
    x = x.detach().double().requires_grad_()
    y = m(x)
    return [y, *torch.autograd.grad(y, (x, m.gate_proj.weight, m.up_proj.weight, m.down_proj.weight), dy.double())]


def step(m, x, dy):
    for p in m.parameters():
        p.grad = None
    x = x.detach().requires_grad_()
    y = m(x)
    y.backward(dy)
    return [y.detach(), x.grad, m.gate_proj.weight.grad, m.up_proj.weight.grad, m.down_proj.weight.grad]


def close(got, want, dtype):
    """Three products in a row of up to 512 terms and the roundings between them, each at most 2^-8 (2^-24) of what it adds up, whose sizes are up to
    8 times the sums: against the largest of a tensor 8 * 6 * 2^-9 of bfloat16, 8 * 3 * 512 * 2^-24 of float32."""
    limit = 8 * 6 * 2.0 ** -9 if dtype == torch.bfloat16 else 8 * 3 * 512 * 2.0 ** -24
    for i, (a, b) in enumerate(zip(got, want)):
        assert a is not None, i
        assert (a.double() - b).abs().max() <= limit * b.abs().max(), i


CASES = [pytest.param(torch.float32, "cpu", False),
         *(pytest.param(d, "cuda", o, marks=pytest.mark.gpu) for d in (torch.float32, torch.bfloat16) for o in (False, True))]


@pytest.mark.parametrize("dtype,device,one_launch", CASES)
def test_gradients_reach_the_projections(dtype, device, one_launch):
    plain, fused = pair(dtype, device, one_launch)
    x, dy = torch.randn(2, 21, 256, device=device).to(dtype), torch.randn(2, 21, 256, device=device).to(dtype)
    close(step(fused, x, dy), exact(plain, x, dy), dtype)
    with torch.no_grad():      # a step of an optimizer: the buffer is what the parameters are
        for p in (*plain.parameters(), *fused.parameters()):
            p.mul_(1.25)
    close(step(fused, x, dy), exact(plain, x, dy), dtype)
    fused.gate_proj.weight.requires_grad_(False)
    got, want = step(fused, x, dy), exact(plain, x, dy)
    assert got.pop(2) is None
    del want[2]
    close(got, want, dtype)


@pytest.mark.parametrize("dtype,device,one_launch", CASES)
def test_parameters_that_have_moved(dtype, device, one_launch):
    plain, fused = pair(dtype, device, one_launch)
    x, dy = torch.randn(5, 256, device=device).to(dtype), torch.randn(5, 256, device=device).to(dtype)
    for m in (plain, fused):
        m.up_proj.weight = nn.Parameter(m.up_proj.weight.detach() * 0.5)
    close(step(fused, x, dy), exact(plain, x, dy), dtype)
    assert fused._w_gate_up is None
    with torch.no_grad():
        y = fused(x)
    close([y], exact(plain, x, dy)[:1], dtype)
    plain, fused = pair(dtype, device, one_launch)
    other = {"gate_proj.weight": (plain.gate_proj.weight.detach() * 2).requires_grad_()}
    y = torch.func.functional_call(fused, other, (x,))
    got, = torch.autograd.grad(y, other["gate_proj.weight"], dy)
    with torch.no_grad():
        plain.gate_proj.weight.mul_(2)
    close([got], [exact(plain, x, dy)[2]], dtype)
    assert fused._w_gate_up is not None


@pytest.mark.parametrize("dtype,device,one_launch", CASES)
def test_a_copy_learns(dtype, device, one_launch):
    """A copy's parameters have storage of their own: what a step has taught them is there without gradients too."""
    plain, fused = (deepcopy(m) for m in pair(dtype, device, one_launch))
    x, dy = torch.randn(5, 256, device=device).to(dtype), torch.randn(5, 256, device=device).to(dtype)
    close(step(fused, x, dy), exact(plain, x, dy), dtype)
    with torch.no_grad():
        for p in (*plain.parameters(), *fused.parameters()):
            p.mul_(1.5)
        y = fused(x)
    close([y], exact(plain, x, dy)[:1], dtype)


def test_forward_mode_of_the_weights():
    plain, fused = pair(torch.float32, "cpu", False)
    x, t = torch.randn(5, 256), torch.randn_like(plain.gate_proj.weight)
    with forward_ad.dual_level():
        want, got = (forward_ad.unpack_dual(torch.func.functional_call(m, {"gate_proj.weight": forward_ad.make_dual(m.gate_proj.weight.detach(), t)}, (x,)))
                     for m in (plain, fused))
    assert got.tangent is not None and torch.allclose(got.tangent, want.tangent, rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("dtype,device,one_launch", CASES)
def test_written_to_in_between(dtype, device, one_launch):
    _, fused = pair(dtype, device, one_launch)
    y = fused(torch.randn(5, 256, device=device).to(dtype))
    with torch.no_grad():
        fused.gate_proj.weight.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
