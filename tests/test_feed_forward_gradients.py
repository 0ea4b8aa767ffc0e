"""Gradients of ``gated_feed_forward`` in float16's range and their precision, against the formulas in 64 bits.

float16: a row m of the projections' gradients [dg du] is kept as float16 numbers times 2^e, e such that its largest lies in [2^14, 2^15) 2^e, and
dW is made of x_m 2^(e - T), T the largest of e and the exponent of x's row, found the same way.  An element is off by half a step of its own, or by half
the smallest step, 2^-25, where it is below 2^-14 there: 2^(e - 25) <= 2^-39 of the largest of its row.  x so is off by 2^(T - e - 25) at most, which meets
|dg| <= 2^(e + 15): 2^(T - 10) a row of dW's sums, where 2^T <= 2^-28 max over rows of (largest of [dg du] times largest of x)."""
import pytest
import torch

from cascading_kv_cache_amd import _abi
from cascading_kv_cache_amd.feed_forward import gated_feed_forward

U = 2.0 ** -24                                   # half a step of float32, relative
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -149}   # half the smallest step


def exact(x, w, dtype, dh):
    """{name: (value, limit with the last rounding)}; float32 sums and slopes as in test_gpu_feed_forward.py, the projections float32."""
    x, w, dh = x.double(), w.double(), dh.double()
    (m, k), inter, half = x.shape, w.size(0) // 2, torch.finfo(dtype).eps / 2
    proj, off = x @ w.T, (k + 2) * U * (x.abs() @ w.abs().T) + 2.0 ** -149
    (g, u), (og, ou) = proj.split(inter, -1), off.split(inter, -1)
    s = torch.sigmoid(g)
    slope, act = s * (1 + g * (1 - s)), g * s
    d = torch.cat((dh * u * slope, dh * act), -1)
    od = torch.cat((dh.abs() * (1.1 * ou + u.abs() * (0.5 * og + 0.2 * og * og) + 0.5 * og * ou) + 32 * U * (dh * u).abs(),
                    dh.abs() * 1.1 * og + 16 * U * (dh * act).abs()), -1)
    top = (d.abs() + od).where(d.isfinite(), 0.0).amax(-1, keepdim=True)   # of the numbers
    lost = 0.0
    if dtype == torch.float16:
        od = od + half * (d.abs() + od) + 2.0 ** -39 * top
        lost = m * 2.0 ** -38 * (top[:, 0] * x.abs().amax(-1)).max()
    elif dtype == torch.bfloat16:
        od = od + half * (d.abs() + od) + TINY[dtype]
    res = {"dx": (d @ w, od @ w.abs() + (2 * inter + 2) * U * ((d.abs() + od) @ w.abs())),
           "dw": (d.T @ x, od.T @ x.abs() + (m + 2) * U * ((d.abs() + od).T @ x.abs()) + lost)}
    return {n: (v, o + half * (v.abs() + o) + TINY[dtype]) for n, (v, o) in res.items()}


def beyond(got, want):
    """How many elements are further off than the limit; where the value is about the type's end, infinity is as good, and what is no number has to
    be none."""
    value, limit = want
    most = torch.finfo(got.dtype).max
    off = (got.double() - value).abs()
    ends = (got.isinf() & (value.abs() + limit >= most) & (got.double().sign() == value.sign())) | (off <= limit)
    ends = torch.where(value.isfinite(), ends, ~got.isfinite())
    return int((~ends).sum())


def inputs(m, k, i, dtype, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g).to(device)   # noqa: E731
    return rand(m, k).to(dtype), (rand(2 * i, k) * k ** -0.5).to(dtype), rand(m, i)


def gradients(x, w, dh):
    x, w = x.clone().requires_grad_(), w.clone().requires_grad_()
    return torch.autograd.grad(gated_feed_forward(x, w), (x, w), dh)


def check(x, w, dh, what):
    want = exact(x, w, x.dtype, dh)
    for name, got in zip(("dx", "dw"), gradients(x, w, dh)):
        bad = beyond(got, want[name])
        assert not bad, f"{what}: {name}: {bad} of {got.numel()} beyond the limit"


# one tile or more, shares of the sums, sizes that no tile of 16 bits takes, layers whose rows are longer than what a workgroup holds of one
SIZES = [(64, 256, 512), (300, 520, 264), (33, 77, 55), (5, 64, 21000), (3, 40, 9001), (4, 32, 25608), (2, 24, 17003), (1, 8, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("scale", [2e4, 1e-4, 1e-6])
def test_large_and_small_gradients_in_float16(scale, size):
    """Those of a scaled loss: [dg du] would be infinite, or a few steps."""
    x, w, dh = inputs(*size, torch.float16, "cuda")
    dh = (dh * scale).clamp(-65504, 65504).half()
    dx, dw = gradients(x, w, dh)
    want = exact(x, w, torch.float16, dh)
    if scale > 1:      # inside the type, though dg is not
        dg = dh.double() * (x.double() @ w.double().T)[:, size[2]:]
        assert size[0] < 30 or dg.abs().max() > 65504
    assert not beyond(dx, want["dx"]) and not beyond(dw, want["dw"])


@pytest.mark.gpu
@pytest.mark.parametrize("size", SIZES[:7], ids=str)
def test_rows_of_all_sizes_in_float16(size):
    """Tokens whose loss is weighed, masked or scaled each by itself, and rows of x of any size beside them."""
    m, k, i = size
    x, w, dh = inputs(*size, torch.float16, "cuda", seed=1)
    by = torch.tensor([1.0, 2.0 ** -12, 0.0, 2.0 ** 14, 2.0 ** -20, 2.0 ** 7], device="cuda").repeat(m // 6 + 1)[:m, None]
    check(x, w, (dh * by).half(), "gradients")
    turned = torch.tensor([2.0 ** 5, 1.0, 2.0 ** -9, 0.0, 2.0 ** -13], device="cuda").repeat(m // 5 + 1)[:m, None]
    check((x.float() * turned).half(), w, (dh * by).half(), "gradients and rows")
    check(x, w, torch.zeros_like(dh).half(), "none")
    x[0, :2] = torch.tensor([6e4, -6e4], device="cuda").half()
    check(x, w, dh.half(), "an outlier")


@pytest.mark.gpu
def test_orders_of_float16_rows():
    m, k, i = 70, 128, 96
    x, w, dh = inputs(m, k, i, torch.float16, "cuda", seed=2)
    dh = (dh * 2e4).clamp(-65504, 65504).half()
    want = exact(x, w, torch.float16, dh)
    wide = torch.zeros(m, 2, k + 9, dtype=torch.float16, device="cuda")
    wide[:, 1, 4:4 + k] = x
    off = torch.zeros(m * i + 1, dtype=torch.float16, device="cuda")[1:].view(m, i).copy_(dh)
    for name, a, d in (("inside a wider buffer", wide[:, 1, 4:4 + k], dh), ("dh off alignment", x, off), ("columns first", x.t().contiguous().t(), dh)):
        a, b = a.detach().requires_grad_(), w.detach().requires_grad_()
        for got, what in zip(torch.autograd.grad(gated_feed_forward(a, b), (a, b), d), ("dx", "dw")):
            assert not beyond(got, want[what]), (name, what)
    b = w.detach().requires_grad_()
    assert not beyond(torch.autograd.grad(gated_feed_forward(x, b), b, dh)[0], want["dw"])
    a = x.detach().requires_grad_()
    assert not beyond(torch.autograd.grad(gated_feed_forward(a, w), a, dh)[0], want["dx"])


@pytest.mark.gpu
def test_float16_gradients_that_are_no_numbers():
    """As a loss scaler looks for them: they stay what they are, and where they are."""
    m, k, i = 40, 64, 72
    x, w, dh = inputs(m, k, i, torch.float16, "cuda", seed=3)
    dh = dh.half()
    clean = gradients(x, w, dh)
    for spoil in (float("inf"), float("nan")):
        d = dh.clone()
        d[7, 5] = spoil
        dx, dw = gradients(x, w, d)
        assert not dx[7].isfinite().any() and torch.equal(dx[:7], clean[0][:7]) and torch.equal(dx[8:], clean[0][8:])
        rows = torch.zeros(2 * i, dtype=torch.bool, device="cuda")
        rows[5] = rows[i + 5] = True
        assert not dw[rows].isfinite().any() and not beyond(dw[~rows], tuple(t[~rows] for t in exact(x, w, torch.float16, dh)["dw"]))


# One row: an element of dW is one product, so what its two factors were rounded by stands in it undiluted.
ONE = (1, 64, 4096)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_projections_are_kept_in_float32(dtype):
    x, w, dh = inputs(*ONE, dtype, "cuda", seed=4)
    check(x, w, dh.to(dtype), "one row")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_the_limit_tells_projections_of_16_bits(dtype):
    """The operator restated on the CPU: as it is, and with projections rounded to the tensor type."""
    x, w, dh = inputs(*ONE, dtype, "cpu", seed=4)
    dh = dh.to(dtype)
    value = exact(x, w, dtype, dh)["dw"]
    for rounded in (False, True):
        proj = x.float() @ w.float().T
        g, u = (proj.to(dtype).float() if rounded else proj).chunk(2, -1)
        s = torch.sigmoid(g)
        d = torch.cat((dh.float() * u * s * (1 + g * (1 - s)), dh.float() * g * s), -1).to(dtype).float()
        many = beyond((d.T @ x.float()).to(dtype), value)
        assert (many > 100) if rounded else many == 0


# Rows that a wavefront's lanes share out between several of them, and more rows than one look at the exponents takes
SHORT = [(65, 40, 24), (1001, 24, 5), (130, 64, 1000), (9, 48, 8), (70001, 16, 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("size", SHORT, ids=str)
def test_short_rows_in_float16(size):
    m, k, i = size
    x, w, dh = inputs(*size, torch.float16, "cuda", seed=5)
    by = torch.tensor([1.0, 2.0 ** -12, 0.0, 2.0 ** 13, 2.0 ** -20], device="cuda").repeat(m // 5 + 1)[:m, None]
    for d in (dh * 2e4, dh * 1e-6, dh * by):
        check(x, w, d.clamp(-65504, 65504).half(), "gradients")


def test_a_workspace_that_exponents_cannot_lie_in():
    lib = _abi.lib()
    assert lib.ckv_gated_linear_bwd(16, 16, 16, 16, 16, 16, 2, 8, 8, 8, _abi.CKV_F16, 18, 1 << 30, None) == -5
