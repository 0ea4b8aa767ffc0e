"""``gated_feed_forward`` against the formulas in 64 bits, with limits counted from the roundings on the way."""
import pytest
import torch

from cascading_kv_cache_amd.feed_forward import gated_feed_forward

pytestmark = pytest.mark.gpu

U = 2.0 ** -24                                   # half a step of float32, relative
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -149}   # half the smallest step
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def exact(x, w, dtype, dh=None):
    """{name: (value, limit without the last rounding)}.  A float32 sum of n products in any order is off by n U of the sum of their sizes;
    the activation's slope is at most 1.1, its second derivative at most 0.5, its third at most 0.4."""
    x, w = x.double(), w.double()
    k, inter, half = x.size(1), w.size(0) // 2, torch.finfo(dtype).eps / 2
    proj, off = x @ w.T, (k + 2) * U * (x.abs() @ w.abs().T) + 2.0 ** -149
    g, u = proj.split(inter, -1)
    og, ou = off.split(inter, -1)
    s = torch.sigmoid(g)
    act = g * s
    res = {"out": (act * u, 1.1 * og * u.abs() + (act.abs() + 1.1 * og) * ou + 16 * U * (act * u).abs())}
    if dh is not None:
        dh = dh.double()
        og, ou = og + half * (g.abs() + og) + TINY[dtype], ou + half * (u.abs() + ou) + TINY[dtype]   # they are kept in the tensor type
        slope = s * (1 + g * (1 - s))
        dg, du = dh * u * slope, dh * act
        odg = dh.abs() * (1.1 * ou + u.abs() * (0.5 * og + 0.2 * og * og) + 0.5 * og * ou) + 32 * U * (dh * u).abs()
        odu = dh.abs() * 1.1 * og + 16 * U * du.abs()
        odg, odu = odg + half * (dg.abs() + odg) + TINY[dtype], odu + half * (du.abs() + odu) + TINY[dtype]
        d, od = torch.cat((dg, du), -1), torch.cat((odg, odu), -1)
        m = x.size(0)
        res["dx"] = (d @ w, od @ w.abs() + (2 * inter + 2) * U * ((d.abs() + od) @ w.abs()))
        res["dw"] = (d.T @ x, od.T @ x.abs() + (m + 2) * U * ((d.abs() + od).T @ x.abs()))
    return res


def close(got, want, dtype, what):
    value, limit = want
    limit = limit + torch.finfo(dtype).eps / 2 * (value.abs() + limit) + TINY[dtype]
    bad = ~((got.double() - value).abs() <= limit)
    assert got.dtype == dtype and got.shape == value.shape, what
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, by {((got.double() - value).abs() / limit)[bad].max().item():.2f} limits"


def inputs(m, k, i, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*s):
        return torch.randn(*s, generator=g, device="cuda")

    return rand(m, k).to(dtype), (rand(2 * i, k) * k ** -0.5).to(dtype), rand(m, i).to(dtype)


SIZES = [  # rows, k, inter
    (1, 1, 1), (3, 7, 5), (2, 64, 16), (1, 256, 512), (17, 130, 66), (65, 129, 63), (129, 512, 64), (16, 4096, 32), (130, 72, 200),
    (255, 1000, 136), (1030, 136, 8200), (4104, 4104, 72), (77, 4104, 2056), (513, 2056, 4104), (40, 3592, 9480), (130, 1544, 9480), (300, 64, 1000), (64, 4096, 264), (513, 264, 520), (5, 2056, 8), (257, 8, 256), (1000, 2048, 16), (9, 520, 2048),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_against_float64(size, dtype):
    x, w, dh = inputs(*size, dtype)
    alone = gated_feed_forward(x, w)
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    out = gated_feed_forward(xs, ws)
    dx, dw = torch.autograd.grad(out, (xs, ws), dh)
    want = exact(x, w, dtype, dh)
    close(alone, want["out"], dtype, "output alone")
    close(out.detach(), want["out"], dtype, "output")
    close(dx, want["dx"], dtype, "dx")
    close(dw, want["dw"], dtype, "dw")


@pytest.mark.parametrize("dtype", TYPES[:2])
@pytest.mark.parametrize("size", [(50, 328, 18952), (100, 328, 18952), (64, 64, 17000), (33, 1032, 25608), (128, 520, 25608), (64, 456, 31000),
                                  (40, 520, 11016), (90, 776, 9736), (50, 2056, 22024), (100, 2056, 22024), (100, 2056, 28680), (20, 1536, 9728),
                                  (200, 1032, 14344), (250, 520, 18952), (140, 264, 11016), (300, 520, 18952), (300, 456, 5640), (700, 328, 5640), (520, 1032, 17416),
                                  (390, 264, 2824)], ids=str)
def test_few_rows_and_wide_layers(size, dtype):
    """Columns that leave compute units idle, or are more than a round of them, in tiles of one width or another."""
    x, w, dh = inputs(*size, dtype)
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    out = gated_feed_forward(xs, ws)
    dx, dw = torch.autograd.grad(out, (xs, ws), dh)
    want = exact(x, w, dtype, dh)
    close(gated_feed_forward(x, w), want["out"], dtype, "output alone")
    close(out.detach(), want["out"], dtype, "output")
    close(dx, want["dx"], dtype, "dx")
    close(dw, want["dw"], dtype, "dw")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 3, 40])
def test_orders_and_alignment(rows, dtype):
    k, i = 128, 96
    x, w, dh = inputs(rows, k, i, dtype)
    want = exact(x, w, dtype, dh)
    wide = torch.zeros(rows, 2, k + 8, dtype=dtype, device="cuda")
    wide[:, 1, 4:4 + k] = x
    off_x = torch.zeros(rows * k + 1, dtype=dtype, device="cuda")[1:].view(rows, k).copy_(x)
    off_w = torch.zeros(2 * i * k + 1, dtype=dtype, device="cuda")[1:].view(2 * i, k).copy_(w)
    turned = x.t().contiguous().t()
    across = w.t().contiguous().t()
    odd = torch.zeros(rows, k + 1, dtype=dtype, device="cuda")
    odd[:, :k] = x
    for name, a, b in (("inside a wider buffer", wide[:, 1, 4:4 + k], w), ("rows off alignment", off_x, w), ("weights off alignment", x, off_w),
                       ("columns first", turned, across), ("an odd stride", odd[:, :k], w)):
        a, b = a.detach().requires_grad_(), b.detach().requires_grad_()
        out = gated_feed_forward(a, b)
        dx, dw = torch.autograd.grad(out, (a, b), dh)
        close(out.detach(), want["out"], dtype, name)
        close(dx, want["dx"], dtype, name)
        close(dw, want["dw"], dtype, name)
    batched = gated_feed_forward(x.view(1, rows, 1, k), w)
    assert batched.shape == (1, rows, 1, i) and torch.equal(batched.view(rows, i), gated_feed_forward(x, w))


@pytest.mark.parametrize("dtype", TYPES)
def test_one_row_for_all_and_gradients_of_one_side(dtype):
    x, w, dh = inputs(1, 64, 40, dtype)
    dh = dh.expand(6, 40)
    x.requires_grad_()
    out = gated_feed_forward(x.expand(6, 64), w)
    dx, = torch.autograd.grad(out, x, dh)
    value, limit = exact(x.detach().expand(6, 64), w, dtype, dh)["dx"]
    half = torch.finfo(dtype).eps / 2
    limit = limit + half * (value.abs() + limit) + TINY[dtype]       # rounded before torch adds the six up, in the tensor type or float32
    want = (value.sum(0, keepdim=True), limit.sum(0, keepdim=True) + 6 * half * (value.abs() + limit).sum(0, keepdim=True))
    close(dx, want, dtype, "dx of an expanded row")
    xs = torch.randn(5, 64, device="cuda").to(dtype)
    ws = w.clone().requires_grad_()
    dw, = torch.autograd.grad(gated_feed_forward(xs, ws), ws, dh[:5])
    close(dw, exact(xs, w, dtype, dh[:5])["dw"], dtype, "dw alone")


def test_gradients_against_differences():
    """As the outputs change along a direction; the limit is what the same difference is off in 64 bits and the outputs' rounding."""
    x, w, dh = inputs(9, 48, 40, torch.float32)
    h = 2.0 ** -7
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    grads = torch.autograd.grad(gated_feed_forward(xs, ws), (xs, ws), dh)

    def loss(a, b, op):
        return (op(a, b).double() * dh.double()).sum().item()

    def in64(a, b):
        return exact(a, b, torch.float32)["out"][0]

    for which, t in enumerate((x, w)):
        d = h * torch.sign(torch.randn_like(t))
        sides = [(x + s * d, w) if which == 0 else (x, w + s * d) for s in (1, -1)]
        step = (sides[0][which].double() - sides[1][which].double()) / 2
        fine = [(x.double() + s * 2.0 ** -12 * step, w) if which == 0 else (x, w.double() + s * 2.0 ** -12 * step) for s in (1, -1)]
        true = (loss(*fine[0], in64) - loss(*fine[1], in64)) / 2 ** -11
        bent = (loss(*sides[0], in64) - loss(*sides[1], in64)) / 2
        got = (loss(*sides[0], gated_feed_forward) - loss(*sides[1], gated_feed_forward)) / 2
        slope = (grads[which].double() * step).sum().item()
        size = sum((exact(a, b, torch.float32)["out"][1] * dh.double().abs()).sum().item() for a, b in sides)
        own = (exact(x, w, torch.float32, dh)[("dx", "dw")[which]][1] * step.abs()).sum().item()
        assert abs(got - slope) <= abs(bent - true) * 1.01 + size + own, which


@pytest.mark.parametrize("dtype", TYPES)
def test_no_rows(dtype):
    x, w, _ = inputs(4, 64, 32, dtype)
    x = x[:0].requires_grad_()
    w.requires_grad_()
    out = gated_feed_forward(x.view(2, 0, 64), w)
    assert out.shape == (2, 0, 32)
    dx, dw = torch.autograd.grad(out.sum(), (x, w))
    assert dx.shape == (0, 64) and (dw == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [(70, 200, 96), (300, 256, 264)], ids=str)
def test_a_row_that_is_not_a_number_stays_alone(size, dtype):
    m, k, i = size
    x, w, _ = inputs(*size, dtype)
    clean = gated_feed_forward(x, w)
    x[m - 2, 3] = float("nan")
    x[1, k - 1] = float("inf")
    out = gated_feed_forward(x, w)
    same = torch.ones(m, dtype=torch.bool, device="cuda")
    same[m - 2] = same[1] = False
    assert out[m - 2].isnan().all() and torch.equal(out[same], clean[same])
    assert not out[1].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [(300, 256, 264), (3, 2048, 64)], ids=str)
def test_another_stream_and_replays_of_a_graph(size, dtype):
    x, w, dh = inputs(*size, dtype)
    x.requires_grad_()
    w.requires_grad_()

    def step():
        out = gated_feed_forward(x, w)
        return [out.detach(), *torch.autograd.grad(out, (x, w), dh)]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = step()
    for rep in range(4):
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
        graph.replay()
        fresh = step()          # the program's own work between two replays
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(recorded, fresh)), rep
