"""The operators around attention as a decoder and a training step use them."""
from dataclasses import replace

import pytest
import torch

from cascading_kv_cache_amd.decoder import PRESETS, CascadeDecoder, generate
from cascading_kv_cache_amd.feed_forward import gated_feed_forward
from cascading_kv_cache_amd.flash_attention import attention
from cascading_kv_cache_amd.norm_rotate import norm_rotate
from cascading_kv_cache_amd.sampling import sample_tokens
from oracle.attention import OracleCascadeAttention
from oracle.update import OracleCache

pytestmark = pytest.mark.gpu

META = ("mask", "sink_mask", "pos", "sink_pos", "stored_tokens", "start_indices", "stored_sinks", "og_pos")


def spread_norms(model, seed=9):
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for layer in model.layers:
            for w in (layer.self_attn.q_norm_weight, layer.self_attn.k_norm_weight):
                w.copy_(1 + 0.3 * torch.randn(w.shape, generator=g))
    return model


def normed(x, w, eps):
    xf = x.float()
    return (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps) * w.float()).to(x.dtype)


def oracle_logits(model, oracles, caches, ids):
    cfg = model.cfg
    B, q = ids.shape
    x = model.embed_tokens(ids)
    for layer, attn_o, cache in zip(model.layers, oracles, caches):
        a, h = layer.self_attn, layer.input_layernorm(x)
        qs, ks, vs = a.qkv(h, (B, q, cfg.num_heads, cfg.head_dim), (B, q, cfg.num_kv_heads, cfg.head_dim))
        qs, ks = normed(qs, a.q_norm_weight, cfg.rms_eps), normed(ks, a.k_norm_weight, cfg.rms_eps)
        x = x + a.o_proj(attn_o.forward(qs, ks, vs, cache).transpose(1, 2).reshape(B, q, -1))
        x = x + layer.mlp(layer.post_attention_layernorm(x))
    return model.lm_head(model.norm(x[:, -1:]))


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_decoder_with_normed_heads_against_the_oracle(dtype, fused):
    """As tests/test_gpu_decoder.py compares the decoder without norms: logits within 3 % of their scale, metadata equal."""
    cfg = replace(PRESETS["tiny"], qk_norm=True)
    gpu = spread_norms(CascadeDecoder(cfg, dtype=dtype, device="cuda:0", seed=3))
    cpu = spread_norms(CascadeDecoder(cfg, dtype=dtype, device="cpu", seed=3))
    if fused:
        gpu.fuse_projections(feed_forward=True)
    B, NS, W, C = 2, 4, 64, 2      # the stream below stays inside the window: no eviction, so no score ties decide
    cache = gpu.new_cache(W * C, C, batch=B, num_sink_tokens=NS)
    caches = [OracleCache(window_length=W, num_sink_tokens=NS, max_batch_size=B, heads=cfg.num_kv_heads, dim=cfg.head_dim, max_seq_len=W * C,
                          dtype=dtype) for _ in range(cfg.num_layers)]
    oracles = [OracleCascadeAttention(cfg.num_heads, cfg.num_kv_heads, cfg.head_dim, rope_theta=cfg.rope_theta,
                                      head_reduction=cfg.head_reduction) for _ in range(cfg.num_layers)]
    ids = torch.randint(0, cfg.vocab_size, (B, 70), generator=torch.Generator().manual_seed(4))
    with torch.no_grad():
        for n, chunk in enumerate([ids[:, 0:32], ids[:, 32:64], ids[:, 64:70]] + [ids[:, i:i + 1] for i in range(5)]):
            lg, lc = gpu(chunk.cuda(), cache).float().cpu(), oracle_logits(cpu, oracles, caches, chunk).float()
            scale = lc.abs().max().item()
            assert (lg - lc).abs().max().item() <= 3e-2 * scale + 1e-3, n
    for i, oc in enumerate(caches):
        for name in META:
            assert torch.equal(getattr(cache, name)[i].cpu(), getattr(oc, name)), f"layer {i}: {name}"


def test_norms_in_place_are_norms():
    """The fused decoder norms its heads where the projections wrote them; with gradients on, beside them: the same logits."""
    model = spread_norms(CascadeDecoder(replace(PRESETS["tiny"], qk_norm=True), device="cuda:0", seed=3)).fuse_projections()
    a, b = (model.new_cache(64, 2, batch=2, num_sink_tokens=4) for _ in range(2))
    ids = torch.randint(0, 512, (2, 40), generator=torch.Generator().manual_seed(4)).cuda()
    seen = []
    model.layers[0].self_attn.o_proj.register_forward_pre_hook(lambda m, args: seen.append(args[0].detach().clone()))
    for chunk in (ids[:, :33], ids[:, 33:34], ids[:, 34:]):
        with torch.no_grad():
            model(chunk, a)
        model(chunk, b)
        assert torch.equal(seen[-1], seen[-2])
    for i in range(2):
        assert torch.equal(a.key_cache[i], b.key_cache[i]) and torch.equal(a.value_cache[i], b.value_cache[i])


def test_layers_saved_without_norms_run():
    model = CascadeDecoder(PRESETS["tiny"], device="cuda:0", seed=3)
    for layer in model.layers:
        assert not layer.self_attn.qk_norm and "q_norm_weight" not in dict(layer.self_attn.named_parameters())
        vars(layer.mlp).pop("one_launch", None)
        vars(layer.self_attn).pop("qk_norm", None)
    with torch.no_grad():
        model(torch.zeros(1, 3, dtype=torch.int64, device="cuda"), model.new_cache(64, 2))


def test_feed_forward_of_a_decoder():
    """One rounding instead of three: logits within the 2 % that fused norms are granted, and the products of a step untouched."""
    plain, fused = (CascadeDecoder(PRESETS["tiny"], device="cuda:0", seed=5).fuse_projections(feed_forward=f) for f in (False, True))
    x = torch.randn(2, 33, 256, device="cuda").bfloat16()
    with torch.no_grad():
        mlp = fused.layers[0].mlp
        assert torch.equal(mlp(x), mlp.down_proj(gated_feed_forward(x, mlp._w_gate_up)))
        with torch.autocast("cuda", torch.float16):
            assert mlp(x).dtype == torch.float16     # autocast's products
        ids = torch.randint(0, 512, (2, 60), generator=torch.Generator().manual_seed(6)).cuda()
        la, lb = (m(ids, m.new_cache(64, 2, batch=2, num_sink_tokens=4)).float() for m in (plain, fused))
        assert (la - lb).abs().max() <= 2e-2 * la.abs().max() + 1e-3
    x.requires_grad_()
    mlp(x).float().sum().backward()
    assert x.grad.isfinite().all() and (x.grad != 0).any()


def test_generate_draws_what_sample_tokens_draws():
    model = CascadeDecoder(PRESETS["tiny"], device="cuda:0", seed=5).fuse_projections()
    ids = torch.randint(0, 512, (3, 50), generator=torch.Generator().manual_seed(6)).cuda()
    fresh = lambda: model.new_cache(64, 2, batch=3, num_sink_tokens=4)   # noqa: E731
    greedy = generate(model, ids, fresh(), 32, 9)
    assert torch.equal(greedy, generate(model, ids, fresh(), 32, 9, sampling=dict(temperature=0.0)))
    assert torch.equal(greedy, generate(model, ids, fresh(), 32, 9, sampling=dict(top_k=1)))
    each = dict(temperature=torch.tensor([0.5, 1.0, 1.5], device="cuda"), top_k=40, top_p=0.95)
    gen = lambda seed: torch.Generator(device="cuda").manual_seed(seed)   # noqa: E731
    out = generate(model, ids, fresh(), 32, 9, sampling=each, generator=gen(1))
    assert torch.equal(out, generate(model, ids, fresh(), 32, 9, sampling=each, generator=gen(1)))
    assert not torch.equal(out, generate(model, ids, fresh(), 32, 9, sampling=each, generator=gen(2)))
    cache, g = fresh(), gen(1)
    with torch.no_grad():
        for i in range(0, 50, 32):
            logits = model(ids[:, i:i + 32], cache)
        for step in range(9):
            nxt = sample_tokens(logits[:, -1], torch.rand(3, generator=g, device="cuda"), **each)[0]
            assert torch.equal(nxt, out[:, 50 + step])
            logits = model(nxt[:, None], cache)


def test_logits_that_are_not_numbers_end_no_stream():
    model = CascadeDecoder(PRESETS["tiny"], device="cuda:0", seed=5)
    with torch.no_grad():
        model.lm_head.weight.fill_(float("nan"))
    out = generate(model, torch.zeros(1, 5, dtype=torch.int64, device="cuda"), model.new_cache(64, 2), 5, 3, sampling=dict(top_p=0.9))
    assert (out[:, 5:] == 0).all()


def test_a_layers_gradients():
    """Projection, norm and rotation, attention, feed-forward: gradients in float32 against the same layer in 64 bits.  Six products in a
    row, of up to 256 terms, each off by up to 256 U of the sizes it adds up, which are up to 8 times the sums: 6 * 256 * 8 * 2^-24 < 1e-3."""
    B, n, H, KVH, D, hidden, inter = 2, 45, 4, 2, 64, 256, 136
    g = torch.Generator(device="cuda").manual_seed(0)
    rand = lambda *s, scale=1.0: torch.randn(*s, generator=g, device="cuda") * scale   # noqa: E731
    x, dy = rand(B, n, hidden), rand(B, n, inter)
    params = [rand((H + 2 * KVH) * D, hidden, scale=hidden ** -0.5), 1 + 0.2 * rand(D), 1 + 0.2 * rand(D),
              rand(hidden, H * D, scale=(H * D) ** -0.5), rand(2 * inter, hidden, scale=hidden ** -0.5)]
    pos = torch.arange(n, device="cuda") * 17
    inv_freq = (1.0 / 5e5 ** (torch.arange(0, D, 2, dtype=torch.int64).float() / D)).cuda()

    def layer(x, wqkv, qw, kw, wo, wgu, own):
        qkv = (x @ wqkv.T).view(B, n, H + 2 * KVH, D).transpose(1, 2)
        q, k, v = qkv.split((H, KVH, KVH), 1)
        if own:
            q, k = norm_rotate(q, k, qw, kw, pos, inv_freq)
        else:
            ang = pos.double()[:, None] * inv_freq.double()
            ang = torch.cat((ang, ang), -1)
            half = lambda t: torch.cat((-t[..., D // 2:], t[..., :D // 2]), -1)   # noqa: E731
            q, k = (t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + 1e-6) * w for t, w in ((q, qw), (k, kw)))
            q, k = (t * ang.cos() + half(t) * ang.sin() for t in (q, k))
        k, v = (t.repeat_interleave(H // KVH, 1) for t in (k, v))
        if own:
            o = attention(q, k.contiguous(), v.contiguous(), True, D ** -0.5, None, 0.99)[0]
        else:
            p = q @ k.transpose(-1, -2).contiguous() * D ** -0.5
            p = p.masked_fill(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), float("-inf")).softmax(-1)
            o = p @ v
        h = x + o.transpose(1, 2).reshape(B, n, H * D) @ wo.T
        if own:
            return gated_feed_forward(h, wgu)
        gate, up = (h @ wgu.T).chunk(2, -1)
        return torch.nn.functional.silu(gate) * up

    results = []
    for own in (True, False):
        ins = [t.clone().requires_grad_() if own else t.double().requires_grad_() for t in (x, *params)]
        out = layer(*ins, own)
        results.append([out.detach(), *torch.autograd.grad(out, ins, dy if own else dy.double())])
    for i, (got, want) in enumerate(zip(*results)):
        assert (got - want).abs().max() <= 1e-3 * want.abs().max(), i


def test_rows_further_apart_than_31_bits():
    """Logits, heads and rows of a buffer of 2^32 elements, of which only theirs are written."""
    far = 2 ** 31
    base = torch.empty(2 * far + 4096, dtype=torch.bfloat16, device="cuda")
    small = torch.randn(3, 4096, device="cuda").bfloat16()
    wide = base.as_strided((3, 4096), (far, 1))
    wide.copy_(small)
    u = torch.rand(3, device="cuda")
    assert all(torch.equal(a, b) for a, b in zip(sample_tokens(wide, u, top_p=0.9), sample_tokens(small, u, top_p=0.9)))
    w = (torch.randn(512, 4096, device="cuda") / 64).bfloat16()
    torch.testing.assert_close(gated_feed_forward(wide, w), gated_feed_forward(small, w), rtol=2.0 ** -7, atol=1e-6)   # half a step each, another order
    q, far_q = small.view(1, 3, 32, 128).transpose(1, 2), wide.unflatten(1, (32, 128))[None].transpose(1, 2)
    weight, pos = torch.rand(128, device="cuda").bfloat16(), torch.arange(3, device="cuda")
    inv_freq = 1.0 / 1e4 ** (torch.arange(0, 128, 2, device="cuda").float() / 128)
    near = norm_rotate(q, q, weight, weight, pos, inv_freq)
    assert all(torch.equal(a, b) for a, b in zip(norm_rotate(far_q, far_q, weight, weight, pos, inv_freq), near))
    norm_rotate(q, q, weight, weight, pos, inv_freq, out=(far_q, torch.empty_like(q)))
    assert torch.equal(far_q, near[0])


def test_a_layer_on_two_streams():
    """Forward and backward of two layers' worth of operators at a time, each with scratch of its own."""
    def step(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        q, k = (torch.randn(2, h, 33, 64, generator=g, device="cuda").bfloat16().requires_grad_() for h in (8, 2))
        qw, kw = (torch.rand(64, generator=g, device="cuda").bfloat16().requires_grad_() for _ in range(2))
        x = torch.randn(66, 264, generator=g, device="cuda").bfloat16().requires_grad_()
        w = (torch.randn(528, 264, generator=g, device="cuda") / 16).bfloat16().requires_grad_()
        qs, ks = norm_rotate(q, k, qw, kw)
        h = gated_feed_forward(x, w)
        grads = torch.autograd.grad((qs, ks, h), (q, k, qw, kw, x, w), (torch.ones_like(qs), torch.ones_like(ks), torch.ones_like(h)))
        return [t.detach() for t in (qs, ks, h)] + list(grads)

    want = [step(s) for s in (1, 2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(i + 1))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for one in g for a, b in zip(one, w))


def test_a_graph_of_the_gradients_can_be_made_and_not_gone_through():
    q, k = (torch.randn(1, h, 5, 64, device="cuda", requires_grad=True) for h in (4, 2))
    qw, kw = (torch.rand(64, device="cuda", requires_grad=True) for _ in range(2))
    x, w = torch.randn(6, 32, device="cuda", requires_grad=True), torch.randn(32, 32, device="cuda", requires_grad=True)
    for leaves, outs in (((q, k, qw, kw), norm_rotate(q, k, qw, kw)), ((x, w), (gated_feed_forward(x, w),))):
        once = torch.autograd.grad(outs, leaves, [torch.ones_like(o) for o in outs], retain_graph=True)
        made = torch.autograd.grad(outs, leaves, [torch.ones_like(o) for o in outs], create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(once, made))
        for which in (0, -1):
            with pytest.raises(RuntimeError, match="once_differentiable"):
                torch.autograd.grad(made[which].sum() + leaves[0].sum(), leaves[0], retain_graph=True)
