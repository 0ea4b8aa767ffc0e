"""``sample_tokens`` of rows that several workgroups share, recorded into a graph: maxima, bins, counters of arrivals and lists begin anew every time."""
import pytest
import torch

from cascading_kv_cache_amd import _abi
from cascading_kv_cache_amd.sampling import sample_tokens

pytestmark = pytest.mark.gpu

SHAPES = [(1, 128256), (3, 90001), (33, 152064)]


def rows_of(kind, shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    logits = torch.randn(*shape, generator=g, device="cuda") * (1.5 + seed % 3)
    if kind == "ties":            # more of one value than a list of elements holds: the row is read again
        logits = (logits * 2).round() / 2
    elif kind == "gaps":
        logits[:, ::3] = float("-inf")
        logits[:, 1::7] = float("nan")
        if seed % 2:
            logits[0] = float("nan")
    return logits.to(dtype), torch.rand(shape[0], generator=g, device="cuda")


@pytest.mark.parametrize("kind", ["normal", "ties", "gaps"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_replays_of_long_rows(shape, dtype, kind):
    rows = shape[0]
    assert _abi.lib().ckv_sample_workspace_bytes(*shape) > 0      # else nothing here is shared out
    logits, u = rows_of(kind, shape, dtype, 0)
    each = dict(temperature=torch.linspace(0.5, 1.5, rows, device="cuda"), top_k=torch.arange(rows, device="cuda") * 40 + 20,
                top_p=torch.full((rows,), 0.95, device="cuda"), min_p=torch.full((rows,), 0.001, device="cuda"))
    settings = [dict(top_k=50, top_p=0.95), dict(), each]
    sample_tokens(logits, u)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = [sample_tokens(logits, u, **s) for s in settings]
    for rep in range(6):
        fresh_logits, fresh_u = rows_of(kind, shape, dtype, rep + 1)
        logits.copy_(fresh_logits)
        u.copy_(fresh_u)
        graph.replay()
        fresh = [sample_tokens(logits, u, **s) for s in settings]       # the program's own work between two replays
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(recorded, fresh)):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1].view(torch.int32), b[1].view(torch.int32)), (rep, i)
    assert ((recorded[0][0] >= 0) & (recorded[0][0] < shape[1])).sum() >= rows - 1


def test_replays_of_two_graphs_at_a_time():
    """Each has scratch of its own."""
    inputs = [rows_of("normal", (3, 90001), torch.bfloat16, s) for s in (1, 2)]
    want = [sample_tokens(*x, top_k=60, top_p=0.9) for x in inputs]
    graphs, recorded = [], []
    for x in inputs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            recorded.append(sample_tokens(*x, top_k=60, top_p=0.9))
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for rep in range(8):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for got, right in zip(recorded, want):
            assert torch.equal(got[0], right[0]) and torch.equal(got[1], right[1]), rep
            got[0].fill_(-7)
