"""``sample_tokens`` against the definition in 64 bits: the same tokens, and their logarithms within what is counted below."""
import math

import numpy as np
import pytest
import torch

from cascading_kv_cache_amd.sampling import sample_tokens

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def plain(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The definition, a row at a time."""
    rows, vocab = logits.shape
    each = [v.double().cpu().numpy() if torch.is_tensor(v) else np.full(rows, float(v)) for v in (temperature, top_k, top_p, min_p)]
    tokens, logs = [], []
    for row, u, t, k, p, least in zip(logits.double().cpu().numpy(), uniforms.double().cpu().numpy(), *each):
        row = np.where(np.isnan(row), -np.inf, row)
        order = np.argsort(-row, kind="stable")
        top = row[order[0]]
        if top == -np.inf:
            tokens.append(-1)
            logs.append(math.nan)
            continue
        if not t > 0:
            k, t = 1, 1.0
        with np.errstate(invalid="ignore", over="ignore"):
            x = np.where(row[order] == top, 0.0, (row[order] - top) / t)
        x[np.isnan(x)] = -np.inf
        w = np.exp(x)
        many = vocab if k <= 0 else min(int(k), vocab)
        before = np.cumsum(w) - w
        if p < 1:
            many = min(many, max(1, int((before < p * w[:many].sum()).sum())))
        many = min(many, max(1, int((w >= min(least, 1.0)).sum())))
        running = np.cumsum(w[:many])
        above = running > (u if u > 0 else 0.0) * running[-1]
        last = int(np.flatnonzero(w[:many] > 0)[-1])
        place = int(above.argmax()) if above.any() else last
        tokens.append(int(order[place]))
        logs.append(x[place] - math.log(running[-1]))
    return torch.tensor(tokens), torch.tensor(logs, dtype=torch.float64)


def check(logits, uniforms, **settings):
    tokens, logs = sample_tokens(logits, uniforms, **settings)
    want, exact = plain(logits, uniforms, **settings)
    assert tokens.dtype == torch.int64 and logs.dtype == torch.float32
    wrong = (tokens.cpu() != want).nonzero().flatten().tolist()
    assert not wrong, [(i, int(tokens[i]), int(want[i])) for i in wrong[:5]]
    # a mass is off by 2^-31 of itself and 2^-45 of the first one's, the sum by as many of those
    limit = 2.0 ** -24 * exact.abs() + 2.0 ** -30 + logits.size(1) * 2.0 ** -44
    off = (logs.double().cpu() - exact).abs()
    assert ((off <= limit) | (exact.isnan() & logs.cpu().isnan())).all(), off.max()
    return tokens


def normal(rows, vocab, dtype, spread, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(rows, vocab, generator=g, device="cuda") * spread).to(dtype), torch.rand(rows, generator=g, device="cuda")


SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=7), dict(top_k=50, top_p=0.9), dict(top_p=0.95), dict(top_p=0.3, temperature=1.3),
            dict(min_p=0.05), dict(top_k=40, top_p=0.99, min_p=0.02, temperature=0.9), dict(top_k=100000, top_p=0.999), dict(temperature=0.0, top_p=0.5)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,spread", [(1, 1, 1.0), (3, 2, 1.0), (2, 17, 2.0), (5, 1000, 3.0), (1, 4099, 3.0), (4, 32001, 2.0), (1, 128256, 3.0),
                                               (130, 5001, 2.0), (200, 300, 0.1)])
@pytest.mark.parametrize("settings", SETTINGS, ids=str)
def test_against_the_definition(rows, vocab, spread, settings, dtype):
    logits, u = normal(rows, vocab, dtype, spread)
    check(logits, u, **settings)


@pytest.mark.parametrize("rows", [3, 140])
@pytest.mark.parametrize("dtype", TYPES)
def test_every_row_its_own_settings(rows, dtype):
    logits, u = normal(rows, 20000, dtype, 2.5, 3)
    g = torch.Generator(device="cuda").manual_seed(4)
    draw = lambda *values: torch.tensor(values, device="cuda")[torch.randint(0, len(values), (rows,), generator=g, device="cuda")]   # noqa: E731
    check(logits, u, temperature=draw(0.0, 0.5, 1.0, 2.0), top_k=draw(0, 1, 30, 500, 10 ** 12, -5), top_p=draw(0.0, 0.5, 0.9, 1.0, 2.0),
          min_p=draw(0.0, 0.01, 0.5, 1.0, 3.0))
    check(logits, u, temperature=0.8, top_p=draw(0.3, 0.8))


@pytest.mark.parametrize("vocab", [64, 5000, 40000])
@pytest.mark.parametrize("rows", [2, 150])
@pytest.mark.parametrize("settings", [dict(), dict(top_k=37), dict(top_p=0.5), dict(top_k=3001, top_p=0.25), dict(min_p=1.0)], ids=str)
def test_ties(rows, vocab, settings):
    """Equal logits, more of them than are sorted: the lowest index first."""
    u = torch.arange(rows, device="cuda") / rows
    check(torch.zeros(rows, vocab, device="cuda"), u, **settings)
    g = torch.Generator(device="cuda").manual_seed(5)
    few = torch.randint(0, 3, (rows, vocab), generator=g, device="cuda").bfloat16()
    check(few, u, **settings)
    near = 1 + torch.randint(0, 4, (rows, vocab), generator=g, device="cuda") * 2.0 ** -20     # one bin, several values
    check(near, u, **settings)
    zeros = torch.where(torch.rand(rows, vocab, generator=g, device="cuda") < 0.5, -0.0, 0.0)
    check(zeros, u, **settings)


@pytest.mark.parametrize("rows", [1, 160])
@pytest.mark.parametrize("dtype", TYPES)
def test_masked_logits_and_rows_without_a_token(rows, dtype):
    logits, u = normal(rows, 3001, dtype, 2.0)
    low = torch.finfo(dtype).min
    for spoil in (float("-inf"), float("nan"), low):
        some = logits.clone()
        some[:, ::3] = spoil
        some[:, :100] = spoil
        for settings in (dict(), dict(top_k=20, top_p=0.8), dict(top_k=2999), dict(temperature=1e30)):
            check(some, u, **settings)
    one = torch.full_like(logits, float("-inf"))
    one[:, 1234] = -3.0
    assert (check(one, u) == 1234).all() and (check(one, u, top_k=5, temperature=0.0) == 1234).all()
    check(torch.full_like(logits, low), u)
    for nothing in (float("-inf"), float("nan")):
        tokens, logs = sample_tokens(torch.full_like(logits, nothing), u, top_k=3)
        assert (tokens == -1).all() and logs.isnan().all()
    much = logits.clone()
    much[:, [5, 2000]] = float("inf")
    check(much, u)
    check(much, u, temperature=1e-30)
    if rows > 1:    # in one row alone
        much = logits.clone()
        much[3] = float("nan")
        got = check(much, u, top_p=0.9)
        keep = torch.arange(rows, device="cuda") != 3
        assert got[3] == -1 and torch.equal(got[keep], sample_tokens(logits, u, top_p=0.9)[0][keep])


@pytest.mark.parametrize("rows", [5, 140])
def test_numbers_at_and_beyond_the_ends(rows):
    logits, _ = normal(rows, 9000, torch.float32, 2.0)
    for value in (0.0, -1.0, 1.0, 2.0, 1 - 2.0 ** -24, 2.0 ** -149, float("inf"), float("nan")):
        u = torch.full((rows,), value, device="cuda")
        for settings in (dict(), dict(top_k=11), dict(top_p=0.7), dict(min_p=0.1)):
            tokens = sample_tokens(logits, u, **settings)[0]
            if value <= 0 or value != value:
                assert torch.equal(tokens, logits.argmax(-1))
            elif value >= 1 and settings:     # the last one that is kept
                beyond = plain(logits, torch.full((rows,), 1.0), **settings)[0]
                assert torch.equal(tokens.cpu(), beyond)
            assert ((tokens >= 0) & (tokens < 9000)).all()


def test_extreme_temperatures():
    logits, u = normal(4, 6000, torch.float32, 2.0)
    logits[:, 77] = logits[:, 33] = 50.0
    assert set(sample_tokens(logits, u, temperature=1e-310)[0].tolist()) <= {33, 77}
    check(logits, u, temperature=1e-6)
    check(logits, u, temperature=1e8)
    check(logits, u, temperature=float("inf"))
    check(logits * 1e37, u, temperature=1e37)


def test_orders_and_alignment():
    base, u = normal(6, 2 * 5003, torch.float16, 2.0)
    for view in (base[:, 1:5002], base[::2], base[:, ::2], base.t().contiguous().t(), base[:1].expand(6, -1)):
        n = view.size(0)
        assert torch.equal(sample_tokens(view, u[:n], top_p=0.9)[0], sample_tokens(view.contiguous(), u[:n], top_p=0.9)[0])
        check(view, u[:n], top_k=300)
    wide = torch.rand(12, device="cuda")[::2]
    check(base, wide, temperature=torch.full((12,), 0.5, device="cuda")[::2])
    assert sample_tokens(base[:0], u[:0])[0].shape == (0,)


def test_frequencies():
    """As often as the distribution says: 20000 numbers a 20000th apart take every token its share of times, one more or less."""
    logits, _ = normal(1, 50, torch.float32, 1.5)
    n = 20000
    u = (torch.arange(n, device="cuda") + 0.5) / n
    tokens = sample_tokens(logits.expand(n, -1), u, temperature=1.2)[0]
    share = torch.softmax(logits.double() / 1.2, -1)[0]
    assert ((tokens.bincount(minlength=50) - n * share).abs() <= 1 + n * 2.0 ** -24).all()


@pytest.mark.parametrize("rows", [2, 140])
def test_another_stream_and_replays_of_a_graph(rows):
    logits, u = normal(rows, 30000, torch.bfloat16, 2.5)
    settings = dict(temperature=torch.full((rows,), 0.9, device="cuda"), top_k=50, top_p=0.95)
    want = sample_tokens(logits, u, **settings)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sample_tokens(logits, u, **settings)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = sample_tokens(logits, u, **settings)
    for rep in range(5):
        logits.copy_(torch.randn_like(logits) * 2)
        u.copy_(torch.rand_like(u))
        graph.replay()
        fresh = sample_tokens(logits, u, **settings)       # the program's own work between two replays
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(recorded, fresh)), rep


def test_no_limit_in_any_number():
    logits, u = normal(3, 500, torch.float32, 2.0)
    want = sample_tokens(logits, u)
    for k in (0, -1, 500, 10 ** 30, float("inf")):
        got = sample_tokens(logits, u, top_k=k)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    with pytest.raises(ValueError):
        sample_tokens(logits, u, top_k=float("nan"))


@pytest.mark.parametrize("rows", [1, 3, 140])
def test_two_streams_at_a_time(rows):
    a, b = normal(rows, 90001, torch.bfloat16, 3.0, 1), normal(rows, 90001, torch.bfloat16, 3.0, 2)
    settings = dict(top_k=60, top_p=0.9)
    want = [sample_tokens(*x, **settings) for x in (a, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for s, x, g in zip(streams, (a, b), got):
            with torch.cuda.stream(s):
                g.append(sample_tokens(*x, **settings))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(t, w[0]) and torch.equal(l, w[1]) for t, l in g)


@pytest.mark.parametrize("settings", [dict(), dict(top_k=37), dict(top_p=0.5), dict(top_k=60001, top_p=0.25), dict(min_p=1.0), dict(top_k=50, top_p=0.95)], ids=str)
def test_ties_in_long_rows(settings):
    test_ties(2, 150001, settings)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [70001, 128256])
def test_long_rows_alone_are_those_of_a_batch(vocab, dtype):
    """In slices or not: the same tokens and the same logarithms."""
    logits, u = normal(131, vocab, dtype, 2.5, 7)
    low = torch.finfo(dtype).min
    for i, spoil in enumerate((float("-inf"), float("nan"), low, float("inf"))):
        logits[i, ::3] = spoil
        logits[i, :9000] = spoil
    logits[4] = float("nan")
    logits[5] = float("-inf")
    logits[6] = float("-inf")
    logits[6, vocab - 1] = 2.0
    logits[7] = 0.25
    logits[8] = logits[8].clamp(max=1.0)      # a tie of many at the top
    u[9:15] = torch.tensor([0.0, -1.0, 1.0, 2.0, 1 - 2.0 ** -24, float("nan")])
    g = torch.Generator(device="cuda").manual_seed(8)
    draw = lambda *values: torch.tensor(values, device="cuda")[torch.randint(0, len(values), (131,), generator=g, device="cuda")]   # noqa: E731
    each = dict(temperature=draw(0.0, 0.5, 1.0, 2.0), top_k=draw(0, 1, 30, 500, 50000), top_p=draw(0.0, 0.5, 0.9, 1.0), min_p=draw(0.0, 0.01, 0.5, 1.0))
    for settings in (dict(), dict(top_k=40), dict(top_p=0.9, temperature=0.8), dict(min_p=0.02), each):
        tokens, logs = sample_tokens(logits, u, **settings)
        for first, many in [(i, 1) for i in range(16)] + [(16, 3), (40, 33), (100, 31)]:
            own = {n: v[first:first + many] if torch.is_tensor(v) else v for n, v in settings.items()}
            t, l = sample_tokens(logits[first:first + many], u[first:first + many], **own)
            assert torch.equal(t, tokens[first:first + many]), (settings, first)
            assert torch.equal(l.view(torch.int32), logs[first:first + many].view(torch.int32)), (settings, first)
    few = slice(9, 20)
    check(logits[16:22], u[16:22], top_k=40, top_p=0.9)
    check(logits[few], torch.rand(11, generator=g, device="cuda"), top_p=0.95)
