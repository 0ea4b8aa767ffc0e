"""What ``norm_rotate`` writes over: by whom it may be, and who is told."""
import pytest
import torch

from cascading_kv_cache_amd.norm_rotate import _written, norm_rotate


def buffer(device="cpu"):
    """Queries and keys as a fused projection leaves them, and what else a call reads."""
    rows = torch.randn(2, 5, 6, 8, device=device)
    q, k = rows[:, :, :4].transpose(1, 2), rows[:, :, 4:].transpose(1, 2)
    return q, k, torch.rand(8, device=device), torch.rand(8, device=device)


def test_places():
    q, k, qw, kw = buffer()
    tensors = q, k, qw, kw, None, None
    _written((q, k), tensors)
    _written((torch.empty_like(q), k), tensors)
    _written((q[:, :, :, :], k.view_as(k)), tensors)
    one = q[:1, :, :1].as_strided((1, 4, 1, 8), (7, 8, 9, 1)), k[:1, :, :1]       # of what there is one of, strides say nothing
    _written(one, (q[:1, :, :1], k[:1, :, :1], qw, kw, None, None))
    square = torch.randn(2, 2, 5, 8), torch.randn(2, 2, 5, 8)
    for out in (square[::-1], (square[0], square[0]), (square[1], torch.empty_like(square[1])), (square[0].transpose(0, 1), square[1])):
        with pytest.raises(ValueError, match="out"):
            _written(out, (*square, qw, kw, None, None))
    with pytest.raises(ValueError, match="something else"):
        _written((qw.view(1, 1, 1, 8), kw.new_empty(1, 1, 1, 8)), (torch.ones(1, 1, 1, 8), torch.ones(1, 1, 1, 8), qw, kw, None, None))


def test_versions():
    q, k, qw, kw = buffer()
    before = q._version
    _written((q, k), (q, k, qw, kw, None, None))
    assert q._version > before and q._version == q._base._version
    with torch.inference_mode():
        a, b = torch.ones(1, 2, 3, 8), torch.ones(1, 2, 3, 8)
        _written((a, b), (a, b, qw, kw, None, None))
        before = q._version
        _written((q, k), (q, k, qw, kw, None, None))
        assert q._version > before
    _written((q[:0], k[:0]), (q[:0], k[:0], qw, kw, None, None))


@pytest.mark.gpu
def test_a_backward_pass_is_told():
    q, k, qw, kw = buffer("cuda")
    leaf = torch.ones(2, 4, 5, 8, device="cuda", requires_grad=True)
    y = (leaf * q).sum()
    with torch.no_grad():
        norm_rotate(q, k, qw, kw, out=(q, k))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    y = (leaf * q).sum()
    norm_rotate(q, k, qw, kw)            # writes to nobody
    y.backward()
    assert torch.equal(leaf.grad, q)


@pytest.mark.gpu
def test_refused_on_the_device():
    q, k, qw, kw = buffer("cuda")
    q2, k2 = k.clone(), k.clone()
    was = q2.clone()
    for args, out in (((q2, k2), (k2, q2)), ((q2, k2), (q2, q2)), ((q2, k2), (torch.empty_like(q2), q2)),
                      ((q, k), (torch.empty_like(q).requires_grad_(), torch.empty_like(k)))):
        for _ in range(2):               # what a layout is known by does not let it pass
            with pytest.raises(ValueError, match="out"):
                norm_rotate(*args, qw, kw, out=out)
    assert torch.equal(q2, was) and torch.equal(k2, k)
    with torch.no_grad():                # as torch has it of its own operations
        a, b = norm_rotate(q, k, qw, kw, out=(torch.empty_like(q).requires_grad_(), torch.empty_like(k)))
    for got, want in zip((a, b), norm_rotate(q, k, qw, kw)):
        assert torch.equal(got, want)
