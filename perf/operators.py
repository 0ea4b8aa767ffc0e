"""What the speed of the operators around attention is measured on, through their public entry points.

Three operators:

* ``norm``: ``norm_rotate``, the norm of every head's queries and keys and their rotation at the token's position, alone (a decoding step,
  a chunk of a prompt) or with its gradients (a training step in front of ``attention``);
* ``ffn``: ``gated_feed_forward``, the two projections of a gated MLP, the activation and their product, alone or with its gradients;
* ``sample``: ``sample_tokens``, a token a row from logits by temperature, top-k, top-p and min-p with given random numbers.

``listed()`` names the cases, ``draw(rng)`` gives one more of the same ranges, ``prepare`` makes what a program holds before the call, ``run``
is one pass: elementary torch operations in 32 bits, or the framework's operators where ``own`` is true; ``exact`` is the operator's
definition in 64 bits and ``work`` counts what a pass cannot do without.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-6


def _norm(batch, heads, kv_heads, tokens, dim, rotated, dtype, backward, start):
    return dict(kind="norm", batch=batch, heads=heads, kv_heads=kv_heads, tokens=tokens, dim=dim, rotated=rotated, dtype=dtype,
                backward=backward, start=start)


def _ffn(rows, hidden, inter, dtype, backward):
    return dict(kind="ffn", rows=rows, hidden=hidden, inter=inter, dtype=dtype, backward=backward)


def _sample(batch, vocab, dtype, temperature, top_k, top_p, min_p, spread, each=False):
    return dict(kind="sample", batch=batch, vocab=vocab, dtype=dtype, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p,
                spread=spread, each=each)


def listed():
    return [
        # a decoding step of one stream far into a long context: 40 head rows, bound by the launch
        dict(_norm(1, 32, 8, 1, 128, 128, "bf16", False, 131071), name="norm_token"),
        # a 4096-token chunk of a prompt, queries and keys as the fused projection leaves them
        dict(_norm(1, 32, 8, 4096, 128, 128, "bf16", False, 0), name="norm_chunk"),
        # a training step with seven query heads a kv head and a ragged length
        dict(_norm(4, 28, 4, 2047, 128, 128, "bf16", True, 0), name="norm_train"),
        # float32, heads of 80 dims of which the first 40 are rotated, with gradients
        dict(_norm(2, 8, 8, 1001, 80, 40, "f32", True, 0), name="norm_part_f32"),
        # a decoding step of one stream: the weights have to come in
        dict(_ffn(1, 4096, 14336, "bf16", False), name="ffn_token"),
        # a decoding step of a served batch, odd in number
        dict(_ffn(77, 3584, 18944, "bf16", False), name="ffn_batch"),
        # a 4096-token chunk of a prompt
        dict(_ffn(4096, 4096, 14336, "bf16", False), name="ffn_chunk"),
        # the largest: a training step of 2048 tokens
        dict(_ffn(2048, 3584, 18944, "f16", True), name="ffn_train"),
        # float32, the precision parity runs are made in, with gradients and sizes that are no multiple of anything
        dict(_ffn(509, 1023, 2731, "f32", True), name="ffn_train_f32"),
        # one stream with the settings of a chat
        dict(_sample(1, 128256, "bf16", 0.8, 50, 0.95, 0.0, 3.0), name="sample_one"),
        # a served batch, every row with settings of its own, logits in float32
        dict(_sample(33, 152064, "f32", 1.0, 0, 0.9, 0.02, 2.5, each=True), name="sample_batch"),
        # 256 rows from the whole distribution, as reinforcement learning draws them
        dict(_sample(256, 128256, "bf16", 1.0, 0, 1.0, 0.0, 2.0), name="sample_whole"),
    ]


MOST_NORM = 4 * 32 * 2047 * 128 * 3        # elements moved by the largest listed norm
MOST_FFN = 6 * 2048 * 2 * 3584 * 18944     # operations of the largest listed feed-forward block
MOST_SAMPLE = 256 * 128256


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm"] * 4 + ["ffn"] * 5 + ["sample"] * 4)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "norm":
        while True:
            heads, kv_heads = rng.choice([(32, 8), (28, 4), (8, 8), (16, 2), (4, 1)])
            dim = rng.choice([128, 128, 128, 64, 256, 80, 96])
            c = _norm(_spread(rng, 1, 16), heads, kv_heads, _spread(rng, 1, 8192), dim, rng.choice([dim, dim, dim // 2 // 2 * 2, 0]), dtype,
                      rng.random() < 0.5, _spread(rng, 1, 1000000) - 1)
            moved = c["batch"] * (heads + kv_heads) * c["tokens"] * dim * (3 if c["backward"] else 1) * (2 if dtype == "f32" else 1)
            if moved <= MOST_NORM:
                return c
    if kind == "ffn":
        while True:
            hidden, inter = rng.choice([(4096, 14336), (3584, 18944), (256, 512), (_spread(rng, 64, 4096), _spread(rng, 64, 16384)),
                                        (_spread(rng, 8, 512) * 8, _spread(rng, 8, 2048) * 8)])
            c = _ffn(_spread(rng, 1, 4096), hidden, inter, dtype, rng.random() < 0.5)
            if work(c)["flops"] * (12 if dtype == "f32" else 1) <= MOST_FFN:
                return c
    while True:
        c = _sample(_spread(rng, 1, 256), rng.choice([128256, 152064, _spread(rng, 2, 200000)]), dtype, round(rng.uniform(0.3, 1.5), 3),
                    rng.choice([0, 0, 1, 20, 50, 1000]), rng.choice([1.0, 0.95, 0.9, 0.5, 0.999]), rng.choice([0.0, 0.0, 0.05, 0.2]),
                    round(rng.uniform(0.5, 5.0), 2), rng.random() < 0.3)
        if c["batch"] * c["vocab"] * (2 if dtype == "f32" else 1) <= MOST_SAMPLE:
            return c


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device=DEVICE) * scale).to(dtype)

    if case["kind"] == "norm":
        b, h, kv, n, d = (case[x] for x in ("batch", "heads", "kv_heads", "tokens", "dim"))
        qkv = normal(b, n, h + 2 * kv, d, scale=2.0)   # as the fused projection leaves them
        state = dict(case, q=qkv[:, :, :h].transpose(1, 2), k=qkv[:, :, h:h + kv].transpose(1, 2),
                     q_weight=1 + normal(d, scale=0.2), k_weight=1 + normal(d, scale=0.2), positions=None, inv_freq=None)
        if case["rotated"]:
            r = case["rotated"]
            state["positions"] = torch.arange(case["start"], case["start"] + n, device=DEVICE)
            state["inv_freq"] = (1.0 / (5e5 ** (torch.arange(0, r, 2, dtype=torch.int64).float() / r))).to(DEVICE)
        if case["backward"]:
            state["dq"], state["dk"] = normal(b, h, n, d), normal(b, kv, n, d)
        return state
    if case["kind"] == "ffn":
        state = dict(case, x=normal(case["rows"], case["hidden"]), w=normal(2 * case["inter"], case["hidden"], scale=0.02))
        if case["backward"]:
            state["dh"] = normal(case["rows"], case["inter"])
        return state
    b, v = case["batch"], case["vocab"]
    state = dict(case, logits=normal(b, v, scale=case["spread"]), uniforms=torch.rand(b, generator=gen, device=DEVICE))
    settings = {x: case[x] for x in ("temperature", "top_k", "top_p", "min_p")}
    if case["each"]:   # rows differ: every other row has a higher temperature and a limit of its own
        odd = torch.arange(b, device=DEVICE) % 2
        settings["temperature"] = case["temperature"] * (1 + 0.25 * odd.float())
        settings["top_k"] = torch.where(odd == 1, case["top_k"] + 40, case["top_k"])
        settings["top_p"] = torch.full((b,), case["top_p"], device=DEVICE)
        settings["min_p"] = case["min_p"] * odd.float()
    state["settings"] = settings
    return state


# ---- the plain forms -------------------------------------------------------------------------------------------------------------------

def _norm_rows(x, w, state):
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    if state["inv_freq"] is None:
        return x
    half = state["rotated"] // 2
    angles = state["positions"].double()[:, None] * state["inv_freq"].double()   # far positions lose their angle in 32 bits
    cos, sin = angles.cos().float(), angles.sin().float()
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, rest), dim=-1)


def _plain_norm(state):
    dtype = state["q"].dtype
    names = ("q", "k", "q_weight", "k_weight")
    ins = {x: state[x].float().requires_grad_(state["backward"]) for x in names}
    outs = _norm_rows(ins["q"], ins["q_weight"], state), _norm_rows(ins["k"], ins["k_weight"], state)
    result = [o.detach().to(dtype) for o in outs]
    if state["backward"]:
        grads = torch.autograd.grad(outs, [ins[x] for x in names], [state["dq"].float(), state["dk"].float()])
        result += [g.to(dtype) for g in grads]
    return result


def _plain_ffn(state):
    dtype, back = state["x"].dtype, state["backward"]
    x, w = state["x"].float().requires_grad_(back), state["w"].float().requires_grad_(back)
    gate, up = (x @ w.T).chunk(2, dim=-1)
    h = gate / (1 + torch.exp(-gate)) * up
    result = [h.detach().to(dtype)]
    if back:
        result += [g.to(dtype) for g in torch.autograd.grad(h, [x, w], state["dh"].float())]
    return result


def _column(value, like, dtype):
    value = value if torch.is_tensor(value) else torch.full((like.size(0),), value, dtype=dtype, device=like.device)
    return value.to(dtype)[:, None]


def _plain_sample(state):
    logits, s = state["logits"].float(), state["settings"]
    vocab = logits.size(1)
    temperature, top_k = _column(s["temperature"], logits, torch.float64), _column(s["top_k"], logits, torch.int64)
    top_p, min_p = _column(s["top_p"], logits, torch.float64), _column(s["min_p"], logits, torch.float64)
    ordered, index = torch.sort(logits, dim=-1, descending=True, stable=True)
    # in 64 bits: a token's place beside a border of the running sum decides
    scaled = (ordered.double() - ordered[:, :1].double()) / temperature
    weights = torch.exp(scaled)
    rank = torch.arange(vocab, device=logits.device)
    kept = (top_k <= 0) | (rank < top_k)
    weights_k = weights * kept
    before = torch.cumsum(weights_k, -1) - weights_k
    kept &= (top_p >= 1) | (before < top_p * weights_k.sum(-1, keepdim=True)) | (rank == 0)
    kept &= (weights >= min_p) | (rank == 0)
    running = torch.cumsum(weights * kept, -1)
    total = running[:, -1:]
    above = running > state["uniforms"].double()[:, None] * total
    place = torch.where(above.any(-1), above.int().argmax(-1), kept.sum(-1) - 1)[:, None]
    return [index.gather(1, place)[:, 0], (scaled.gather(1, place) - torch.log(total))[:, 0].float()]


PLAIN = {"norm": _plain_norm, "ffn": _plain_ffn, "sample": _plain_sample}


# ---- the framework's operators ---------------------------------------------------------------------------------------------------------

def _own_norm(state):
    from cascading_kv_cache_amd.norm_rotate import norm_rotate

    names = ("q", "k", "q_weight", "k_weight")
    ins = [state[x] for x in names]
    if state["backward"]:
        ins = [t.detach().requires_grad_() for t in ins]
    outs = norm_rotate(*ins, positions=state["positions"], inv_freq=state["inv_freq"], eps=EPS)
    if not state["backward"]:
        return list(outs)
    return [o.detach() for o in outs] + list(torch.autograd.grad(outs, ins, [state["dq"], state["dk"]]))


def _own_ffn(state):
    from cascading_kv_cache_amd.feed_forward import gated_feed_forward

    if not state["backward"]:
        return [gated_feed_forward(state["x"], state["w"])]
    x, w = state["x"].detach().requires_grad_(), state["w"].detach().requires_grad_()
    h = gated_feed_forward(x, w)
    return [h.detach(), *torch.autograd.grad(h, [x, w], state["dh"])]


def _own_sample(state):
    from cascading_kv_cache_amd.sampling import sample_tokens

    return list(sample_tokens(state["logits"], state["uniforms"], **state["settings"]))


OWN = {"norm": _own_norm, "ffn": _own_ffn, "sample": _own_sample}


def run(state):
    return (OWN if own else PLAIN)[state["kind"]](state)


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------------------

def _exact_norm_rows(x, w, g, c):
    """Outputs and gradients of rows ``x (B, heads, n, d)`` from the formulas; the rotation is a product with complex numbers."""
    x, w = x.double(), w.double()
    r = (x.pow(2).sum(-1, keepdim=True) / x.size(-1) + EPS).pow(-0.5)
    unit = x * r
    half = c["rotated"] // 2 if c["inv_freq"] is not None else 0
    turn = None
    if half:
        angle = torch.outer(c["positions"].double(), c["inv_freq"].double())
        turn = torch.polar(torch.ones_like(angle), angle)

    def rotate(y, by):
        if by is None:
            return y
        z = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * by
        return torch.cat((z.real, z.imag, y[..., 2 * half:]), -1)

    out = rotate(unit * w, turn)
    if g is None:
        return out, None, None
    g = rotate(g.double(), None if turn is None else turn.conj())
    dw = (g * unit).sum((0, 1, 2))
    dx = r * (g * w - unit * (g * w * unit).mean(-1, keepdim=True))
    return out, dx, dw


def _exact_norm(s):
    q, dq, dqw = _exact_norm_rows(s["q"], s["q_weight"], s.get("dq"), s)
    k, dk, dkw = _exact_norm_rows(s["k"], s["k_weight"], s.get("dk"), s)
    return [q, k, dq, dk, dqw, dkw] if s["backward"] else [q, k]


def _exact_ffn(s):
    x, w = s["x"].double(), s["w"].double()
    inter = s["inter"]
    gate, up = x @ w[:inter].T, x @ w[inter:].T
    sig = torch.sigmoid(gate)
    h = gate * sig * up
    if not s["backward"]:
        return [h]
    dh = s["dh"].double()
    dgate = dh * up * sig * (1 + gate * (1 - sig))
    dup = dh * gate * sig
    dx = dgate @ w[:inter] + dup @ w[inter:]
    return [h, dx, torch.cat((dgate.T @ x, dup.T @ x))]


def _exact_sample(s):
    logits, uniforms = s["logits"].double().cpu().numpy(), s["uniforms"].double().cpu().numpy()
    each = {x: (v.cpu().numpy().tolist() if torch.is_tensor(v) else [v] * len(logits)) for x, v in s["settings"].items()}
    tokens, logprobs = [], []
    for row, u, t, k, p, least in zip(logits, uniforms, each["temperature"], each["top_k"], each["top_p"], each["min_p"]):
        order = np.argsort(-row, kind="stable")
        if k > 0:
            order = order[:k]
        scaled = (row[order] - row[order[0]]) / t
        weight = np.exp(scaled)
        many = len(order)
        if p < 1:
            many = max(1, int(np.searchsorted(np.cumsum(weight), p * weight.sum(), side="left")) + 1)
        many = min(many, max(1, int((weight >= least).sum())))
        running = np.cumsum(weight[:many])
        place = min(int(np.searchsorted(running, u * running[-1], side="right")), many - 1)
        tokens.append(int(order[place]))
        logprobs.append(scaled[place] - math.log(running[-1]))
    return [torch.tensor(tokens), torch.tensor(logprobs, dtype=torch.float64)]


EXACT = {"norm": _exact_norm, "ffn": _exact_ffn, "sample": _exact_sample}


def exact(case, seed):
    return EXACT[case["kind"]](prepare(case, seed))


def work(case):
    size = BYTES[case["dtype"]]
    if case["kind"] == "norm":
        d, rows = case["dim"], case["batch"] * (case["heads"] + case["kv_heads"]) * case["tokens"]
        half = case["rotated"] // 2
        positions = case["tokens"] * 8 + half * 4 if half else 0
        moved, ops = 2, 4 * d + 6 * half
        if case["backward"]:
            moved, ops = 4, 12 * d + 12 * half   # the rows are read once, the gradients of both sides come and go
        return {"bytes": rows * d * size * moved + positions + 2 * d * size * (2 if case["backward"] else 1), "flops": rows * ops}
    if case["kind"] == "ffn":
        m, k, i = case["rows"], case["hidden"], case["inter"]
        moved, flops = m * k + 2 * i * k + m * i, 2 * m * k * 2 * i
        if case["backward"]:
            moved, flops = 2 * moved, 3 * flops
        return {"bytes": moved * size, "flops": flops}
    n = case["batch"] * case["vocab"]
    return {"bytes": n * size + case["batch"] * (4 + 8 + 4), "flops": 4 * n}
