"""``norm_rotate`` against the formulas in 64 bits, with limits counted from the roundings on the way."""
import pytest
import torch

from cascading_kv_cache_amd.norm_rotate import norm_rotate

pytestmark = pytest.mark.gpu

U = 2.0 ** -24                                   # half a step of float32, relative
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -149}   # half the smallest step


def angles(positions, inv_freq):
    return positions.double()[..., None] * inv_freq.double()


def turn(y, positions, inv_freq, back=False):
    """Rotated rows ``(B, H, n, D)`` and the size of what each element is made of."""
    if inv_freq is None:
        return y, y.abs()
    h = inv_freq.numel()
    ang = angles(positions, inv_freq)
    ang = ang[:, None] if ang.dim() == 3 else ang
    c, s = ang.cos(), ang.sin() * (-1 if back else 1)
    a, b, rest = y[..., :h], y[..., h:2 * h], y[..., 2 * h:]
    size = a.abs() + b.abs()
    return torch.cat((a * c - b * s, b * c + a * s, rest), -1), torch.cat((size, size, rest.abs()), -1)


def exact(x, w, positions, inv_freq, eps, g=None):
    """{name: (value, limit without the last rounding)} of one side."""
    x, d = x.double(), x.size(-1)
    c = (d + 32) * U        # sum of d squares, root, and a few products and sums; sin and cos are off by less than 4 U
    if w is None:
        out, size = turn(x, positions, inv_freq)
        res = {"out": (out, c * size)}
        if g is not None:
            dx, size = turn(g.double(), positions, inv_freq, back=True)
            res["dx"] = (dx, c * size)
        return res
    w = w.double()
    r = (x.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    unit = x * r
    out, size = turn(unit * w, positions, inv_freq)
    res = {"out": (out, c * size)}
    if g is not None:
        g, gsize = turn(g.double(), positions, inv_freq, back=True)
        res["dx"] = (r * (g * w - unit * (g * w * unit).mean(-1, keepdim=True)),
                     2 * c * r * (gsize * w.abs() + unit.abs() * (gsize * w.abs() * unit.abs()).mean(-1, keepdim=True)))
        rows = x.numel() // d
        res["dw"] = ((g * unit).sum((0, 1, 2)), (rows + d + 32) * U * (gsize * unit.abs()).sum((0, 1, 2)))
    return res


def close(got, want, dtype, what):
    value, limit = want
    limit = limit + torch.finfo(dtype).eps / 2 * (value.abs() + limit) + TINY[dtype]
    bad = ~((got.double() - value).abs() <= limit)
    assert got.dtype == dtype and got.shape == value.shape, what
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, by {((got.double() - value).abs() / limit)[bad].max().item():.2f} limits"


def freqs(r, theta=5e5):
    return (1.0 / theta ** (torch.arange(0, r, 2, dtype=torch.int64).float() / r)).cuda() if r else None


def inputs(B, H, KVH, n, D, dtype, layout, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*s):
        return torch.randn(*s, generator=g, device="cuda").mul(2).to(dtype)

    if layout == "projected":       # parts of one buffer, tokens outermost
        both = rand(B, n, H + 2 * KVH, D)
        q, k = both[:, :, :H].transpose(1, 2), both[:, :, H:H + KVH].transpose(1, 2)
    elif layout == "odd":           # an element off any alignment
        q = rand(B * H * n * D + 1)[1:].view(B, H, n, D)
        k = rand(B * KVH * n * (D + 3) + 1)[1:].view(B, KVH, n, D + 3)[..., :D]
    elif layout == "expanded":      # one batch row for all, and head dims apart
        q = rand(1, H, n, D).expand(B, H, n, D)
        k = rand(B, KVH, D, n).transpose(2, 3)
    else:
        q, k = rand(B, H, n, D), rand(B, KVH, n, D)
    w = [(1 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(dtype) for _ in range(2)]
    grads = rand(B, H, n, D), rand(B, KVH, n, D)
    return q, k, w[0], w[1], grads


CASES = [  # B, H, KVH, n, D, rotated dims, layout
    (1, 32, 8, 1, 128, 128, "projected"),
    (1, 4, 2, 1, 128, 0, "projected"),
    (2, 28, 4, 37, 128, 128, "projected"),
    (2, 8, 8, 65, 64, 64, "dense"),
    (1, 3, 1, 130, 256, 256, "projected"),
    (2, 2, 1, 33, 96, 96, "projected"),
    (3, 5, 5, 17, 80, 40, "projected"),
    (2, 3, 2, 9, 80, 0, "dense"),
    (2, 3, 2, 19, 128, 128, "odd"),
    (2, 2, 1, 21, 256, 254, "odd"),
    (2, 3, 2, 11, 255, 2, "odd"),
    (1, 2, 2, 7, 5, 4, "odd"),
    (2, 1, 1, 3, 1, 0, "odd"),
    (2, 2, 1, 5, 2, 2, "dense"),
    (3, 4, 2, 13, 64, 32, "expanded"),
    (1, 1, 1, 300, 8, 8, "dense"),
    (9, 40, 8, 211, 128, 128, "projected"),     # a backward pass whose blocks come to several tokens
    (1, 300, 1, 2, 16, 16, "dense"),            # more heads than chunks of a backward pass
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("weights", [True, False])
def test_against_float64(case, weights, dtype):
    B, H, KVH, n, D, r, layout = case
    if not weights and not r:
        pytest.skip("nothing to do: the call is refused")
    q, k, qw, kw, (gq, gk) = inputs(B, H, KVH, n, D, dtype, layout)
    if not weights:
        qw = kw = None
    inv_freq = freqs(r)
    positions = None
    if r:
        positions = torch.randint(0, 100000, (B, n) if layout == "projected" else (n,), device="cuda")
    with torch.no_grad():
        alone = norm_rotate(q, k, qw, kw, positions, inv_freq, 1e-5)
    ins = [t if t is None else t.detach().requires_grad_() for t in (q, k, qw, kw)]
    outs = norm_rotate(*ins, positions, inv_freq, 1e-5)
    assert all(o.is_contiguous() and torch.equal(o, a) for o, a in zip(outs, alone))
    grads = torch.autograd.grad(outs, [t for t in ins if t is not None], (gq, gk))
    for i, (x, w, g) in enumerate(((q, qw, gq), (k, kw, gk))):
        want = exact(x, w, positions, inv_freq, 1e-5, g)
        close(outs[i], want["out"], dtype, f"output {i}")
        close(grads[i], want["dx"], dtype, f"gradient {i}")
        if weights:
            close(grads[2 + i], want["dw"], dtype, f"weight gradient {i}")


@pytest.mark.parametrize("start", [0, 131071, 10 ** 7, 2 ** 33, 2 ** 40])
def test_far_positions(start):
    """The angle is the exact product; beside it float32 has no digits left for a far position (10^7 radians: a step of one).  In 64 bits
    a product of 2^40 is off by 2^-13 of a radian, which the limit has to grant."""
    q, k, qw, kw, _ = inputs(1, 2, 1, 50, 128, torch.float32, "dense")
    pos, inv_freq = start + torch.arange(50, device="cuda"), freqs(128)
    out = norm_rotate(q, k, qw, kw, pos, inv_freq)[0]
    want, limit = exact(q, qw, pos, inv_freq, 1e-6)["out"]
    close(out, (want, limit + 2 * start * 2.0 ** -53 * 4 * limit / ((128 + 32) * U)), torch.float32, "far")


def test_gradients_against_differences():
    """The outputs' change along a direction against the gradient's product with it.  The limit is what the same difference is off in 64 bits
    and the outputs' own rounding over the step."""
    q, k, qw, kw, (gq, gk) = inputs(2, 3, 2, 5, 64, torch.float32, "dense")
    pos, inv_freq, h = torch.arange(5, device="cuda") * 1000, freqs(64), 2.0 ** -7
    ins = [t.clone().requires_grad_() for t in (q, k, qw, kw)]
    grads = torch.autograd.grad(norm_rotate(*ins, pos, inv_freq), ins, (gq, gk))

    def loss(ts, op):
        oq, ok = op(ts)
        return ((oq.double() * gq.double()).sum() + (ok.double() * gk.double()).sum()).item()

    def in64(ts):
        return [exact(ts[i], ts[i + 2], pos, inv_freq, 1e-6)["out"][0] for i in range(2)]

    for which in range(4):
        d = torch.sign(torch.randn_like(ins[which]))   # exact in every type
        up = [t.detach() + h * d if i == which else t.detach() for i, t in enumerate(ins)]
        down = [t.detach() - h * d if i == which else t.detach() for i, t in enumerate(ins)]
        step = ((up[which].double() - down[which].double()) * 0.5)        # what the rounded sums really stepped
        slope = (grads[which].double() * step).sum().item()
        fine = [[t.double() + s * 2.0 ** -12 * (step if i == which else 0) for i, t in enumerate(ins)] for s in (1, -1)]
        true = (loss(fine[0], in64) - loss(fine[1], in64)) / 2 ** -11
        bent = (loss(up, in64) - loss(down, in64)) / 2
        got = (loss(up, lambda t: norm_rotate(*t, pos, inv_freq)) - loss(down, lambda t: norm_rotate(*t, pos, inv_freq))) / 2
        size = sum((exact(ts[i], ts[i + 2], pos, inv_freq, 1e-6)["out"][1] * g.double().abs()).sum().item()
                   for ts in (up, down) for i, g in enumerate((gq, gk)))
        assert abs(got - slope) <= abs(bent - true) * 1.01 + size, which


def test_rows_of_zeros_and_rows_that_are_not_numbers():
    q, k, qw, kw, (gq, gk) = inputs(1, 2, 1, 8, 128, torch.bfloat16, "dense")
    q[0, 0, 3] = 0
    q[0, 1, 5, 7] = float("nan")
    k[0, 0, 2, 9] = float("inf")
    clean_q, clean_k = q.clone(), k.clone()
    clean_q[0, 1, 5], clean_k[0, 0, 2] = 1, 1
    pos, inv_freq = torch.arange(8, device="cuda"), freqs(128)
    a, b = norm_rotate(q, k, qw, kw, pos, inv_freq), norm_rotate(clean_q, clean_k, qw, kw, pos, inv_freq)
    assert (a[0][0, 0, 3] == 0).all() and a[0][0, 1, 5].isnan().all() and a[1][0, 0, 2].isnan().any()
    same = torch.ones(1, 2, 8, dtype=torch.bool)
    same[0, 1, 5] = False
    assert torch.equal(a[0][same.cuda()], b[0][same.cuda()])
    assert torch.equal(a[1][0, 0, [0, 1, 3, 4, 5, 6, 7]], b[1][0, 0, [0, 1, 3, 4, 5, 6, 7]])


@pytest.mark.parametrize("shape", [(0, 4, 2, 5), (2, 4, 2, 0)])
def test_nothing_to_norm(shape):
    B, H, KVH, n = shape
    q, k, qw, kw, _ = inputs(B, H, KVH, n, 64, torch.float16, "dense")
    ins = [t.requires_grad_() for t in (q, k, qw, kw)]
    pos = torch.arange(n, device="cuda")
    oq, ok = norm_rotate(*ins, pos, freqs(64))
    assert oq.shape == q.shape and ok.shape == k.shape
    grads = torch.autograd.grad(oq.sum() + ok.sum(), ins)
    assert grads[0].shape == q.shape and (grads[2] == 0).all() and (grads[3] == 0).all()


def test_gradients_of_sums_and_of_one_output():
    """A sum's gradient is one number expanded; an output that nobody used has none."""
    q, k, qw, kw, _ = inputs(2, 3, 1, 6, 64, torch.float32, "projected")
    pos, inv_freq = torch.arange(6, device="cuda"), freqs(64)
    ins = [t.detach().requires_grad_() for t in (q, k, qw, kw)]
    grads = torch.autograd.grad(norm_rotate(*ins, pos, inv_freq)[0].sum(), ins)
    want = exact(q, qw, pos, inv_freq, 1e-6, torch.ones(2, 3, 6, 64, device="cuda"))
    close(grads[0], want["dx"], torch.float32, "dq")
    close(grads[2], want["dw"], torch.float32, "dw")
    assert (grads[1] == 0).all() and (grads[3] == 0).all()


def test_another_stream_and_replays_of_a_graph():
    q, k, qw, kw, (gq, gk) = inputs(2, 8, 2, 40, 128, torch.bfloat16, "projected")
    pos, inv_freq = torch.arange(40, device="cuda"), freqs(128)
    ins = [t.detach().clone().requires_grad_() for t in (q, k, qw, kw)]

    def step():
        outs = norm_rotate(*ins, pos, inv_freq)
        return [o.detach() for o in outs] + list(torch.autograd.grad(outs, ins, (gq, gk)))

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
            ins[0].copy_(torch.randn_like(ins[0]))
            ins[3].copy_(torch.randn_like(ins[3]))
        graph.replay()
        fresh = step()          # the program's own work between two replays
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(recorded, fresh)), rep


def test_written_over_the_inputs_and_elsewhere():
    for layout, D in (("projected", 128), ("dense", 64), ("odd", 80)):
        q, k, qw, kw, _ = inputs(2, 4, 2, 7, D, torch.bfloat16, layout)
        pos, inv_freq = torch.arange(7, device="cuda"), freqs(D)
        want = norm_rotate(q, k, qw, kw, pos, inv_freq)
        there = torch.zeros(7, 2, 4, D, dtype=q.dtype, device="cuda").permute(1, 2, 0, 3), torch.zeros_like(k)
        for out in (there, (q, k)):
            got = norm_rotate(q, k, qw, kw, pos, inv_freq, out=out)
            assert got[0] is out[0] and torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_outputs_that_cannot_be_written_to():
    q, k, qw, kw, _ = inputs(2, 4, 2, 7, 64, torch.float32, "dense")
    for out in ((q[:, :3], k), (q, k.half()), (q.transpose(2, 3).contiguous().transpose(2, 3), k), (q[:1].expand(2, -1, -1, -1), k), (q.cpu(), k)):
        with pytest.raises(ValueError):
            norm_rotate(q, k, qw, kw, out=out)
    with pytest.raises(ValueError, match="gradients"):
        norm_rotate(q, k, qw.requires_grad_(), kw, out=(q, k))


def test_calls_alike_are_not_one_another():
    """The same sizes and strides again and again, with other tensors, eps and positions, with gradients and without, in place and not."""
    for dtype in (torch.bfloat16, torch.float32):
        for seed in range(4):
            q, k, qw, kw, (gq, gk) = inputs(2, 4, 2, 9, 64, dtype, "projected", seed)
            pos, inv_freq, eps = torch.randint(0, 1000, (9,), device="cuda"), freqs(64, 1e4 * (seed + 1)), 10.0 ** (-seed - 1)
            ins = [t.detach().requires_grad_() for t in (q, k, qw, kw)]
            outs = norm_rotate(*ins, pos, inv_freq, eps)
            grads = torch.autograd.grad(outs, ins, (gq, gk) if seed % 2 else (gq.transpose(1, 2).contiguous().transpose(1, 2), gk))
            alone = norm_rotate(q, k, qw, kw, pos, inv_freq, eps)
            for i, (x, w, g) in enumerate(((q, qw, gq), (k, kw, gk))):
                want = exact(x, w, pos, inv_freq, eps, g)
                close(outs[i], want["out"], dtype, "output")
                close(grads[i], want["dx"], dtype, "gradient")
                close(grads[2 + i], want["dw"], dtype, "weight gradient")
            norm_rotate(q, k, qw, kw, pos, inv_freq, eps, out=(q, k))
            assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(outs, alone, (q, k)))
            with pytest.raises(ValueError, match="no gradient"):
                norm_rotate(q, k, qw, kw, pos, inv_freq.clone().requires_grad_(), eps)
            with pytest.raises(ValueError):
                norm_rotate(q, k, qw, kw, pos, inv_freq, eps, out=(q,))


@pytest.mark.parametrize("n", [1, 3])
def test_many_heads(n):
    q, k, qw, kw, (gq, gk) = inputs(1, 70000, 3, n, 4, torch.float16, "dense")
    pos, inv_freq = torch.arange(n, device="cuda"), freqs(4)
    ins = [t.detach().requires_grad_() for t in (q, k, qw, kw)]
    outs = norm_rotate(*ins, pos, inv_freq, 1e-5)
    grads = torch.autograd.grad(outs, ins, (gq, gk))
    for i, (x, w, g) in enumerate(((q, qw, gq), (k, kw, gk))):
        want = exact(x, w, pos, inv_freq, 1e-5, g)
        close(outs[i], want["out"], torch.float16, "output")
        close(grads[i], want["dx"], torch.float16, "gradient")
        close(grads[2 + i], want["dw"], torch.float16, "weight gradient")
