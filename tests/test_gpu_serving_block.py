"""A block's way from the residual stream to attention for many requests, as it is used: the residual's addition with the norm,
projections with each request's adapter, rotary positions of three axes, the store, attention over the cache
(`add_norm_quantize`, then `cached_attention(..., rope=..., adapters=...)`)."""
import types

import pytest
import torch

import vdn_fp8
from vdn_fp8 import Adapters, RopeAxes
from vdn_fp8.softmax_attention import cached_attention

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
HIDDEN, HQ, H, D = 1024, 8, 2, 128


def model(device, seed=1):
    g = torch.Generator(device).manual_seed(seed)

    def linear(n):
        lin = torch.nn.Linear(HIDDEN, n, bias=False, device=device, dtype=BF16)
        lin.weight.data.normal_(0, HIDDEN ** -0.5, generator=g)
        return vdn_fp8.Fp8Linear(lin)

    def norm(n):
        return types.SimpleNamespace(weight=(1 + 0.1 * torch.randn(n, device=device, generator=g)).to(BF16), eps=1e-6)

    def bank(n):
        return Adapters((torch.randn(3, 16, HIDDEN, device=device, generator=g) / 32).to(BF16),
                        (torch.randn(3, n, 16, device=device, generator=g) / 4).to(BF16), torch.ones(3, device=device))

    return types.SimpleNamespace(projections=(linear(HQ * D), linear(H * D), linear(H * D)), norm=norm(HIDDEN), norm_q=norm(D), norm_k=norm(D),
                                 banks=(bank(HQ * D), None, bank(H * D)), rope=RopeAxes.make((24, 20, 20), device=device))


def state(device, tokens, seed):
    g = torch.Generator(device).manual_seed(seed)
    return tuple(torch.randn(tokens, HIDDEN, device=device, generator=g).to(BF16) for _ in "rb")


def cache_of(device, B, W):
    cache = vdn_fp8.KvCache.empty(B * W, H, D, device)
    table = torch.arange(B * W, device=device, dtype=torch.int32).view(W, B).T.contiguous()
    return cache, table


def test_a_prompt_and_steps(device):
    """Three requests (one without adapter): ragged prompts, then steps of one token each. Every call's result has the bits of its
    parts, called one by one, and is what attention in 64 bits over the same keys and values gives, to the cache's own rounding."""
    m = model(device)
    news = [70, 1, 130]
    cache, table = cache_of(device, 3, 4)
    other, _ = cache_of(device, 3, 4)
    lengths = torch.zeros(3, dtype=torch.int32, device=device)
    kept = [[], [], []]
    for step in range(3):
        n = news if step == 0 else [1, 1, 1]
        T = sum(n)
        start = torch.tensor([0, n[0], n[0] + n[1], T], dtype=torch.int32, device=device)
        at = torch.cat([torch.arange(c, device=device) + int(length) for c, length in zip(n, lengths.tolist())]).int()
        positions = torch.stack([at // 64, at // 8 % 8, at % 8], 1)
        request = torch.repeat_interleave(torch.arange(3), torch.tensor(n))
        index = torch.tensor([2, -1, 0], dtype=torch.int32)[request].to(device)
        lengths += start[1:] - start[:-1]
        r, b = state(device, T, 10 + step)
        hidden, codes, scale, x = vdn_fp8.add_norm_quantize(r, b, m.norm.weight, m.norm.eps, return_normed=True)
        kw = dict(causal=True, q_start=start)
        got = cached_attention(x, *m.projections, m.norm_q, m.norm_k, cache, table, lengths, rope=m.rope, positions=positions,
                               adapters=m.banks, index=index, **kw)
        q, k, v = (p(x) if bank is None else p(x, adapters=bank, index=index) for p, bank in zip(m.projections, m.banks))
        q, k, v = (t.unflatten(1, (-1, D)) for t in (q, k, v))
        q, k = vdn_fp8.qk_prep_axes(q, k, (m.norm_q.weight, 1e-6), (m.norm_k.weight, 1e-6), m.rope, positions)
        vdn_fp8.kv_append(k, v, other, table, lengths, q_start=start)
        want = vdn_fp8.kv_attention(q, other, table, lengths, **kw)
        assert torch.equal(got, want.flatten(1))
        # in 64 bits over the keys and values before the cache's rounding to e4m3 (half a step 2^-4): a key's relative error moves a
        # score by at most 2^-4 |q| |k| / sqrt(d), weights by the factor exp of twice that
        for b_ in range(3):
            mine = request == b_
            kept[b_].append((k[mine].double(), v[mine].double()))
            K, V = (torch.cat([p[i] for p in kept[b_]]) for i in range(2))
            Q = q[mine].double()
            assert K.shape[0] == int(lengths[b_])
            for h in range(HQ):
                s = Q[:, h] @ K[:, h // 4].T * D ** -0.5
                seen = torch.arange(K.shape[0], device=device)[None] <= (K.shape[0] - Q.shape[0] + torch.arange(Q.shape[0], device=device))[:, None]
                shift = 2.0 ** -4 * (Q[:, h].abs() @ K[:, h // 4].abs().T) * D ** -0.5
                p = torch.softmax(s.masked_fill(~seen, -float("inf")), 1)
                exact = p @ V[:, h // 4]
                spread = (torch.exp(2 * shift.masked_fill(~seen, 0).amax(1, keepdim=True)) - 1) * (p @ V[:, h // 4].abs())
                room = spread + 2 * (2.0 ** -4 * p @ V[:, h // 4].abs()) + 2.0 ** -8 * exact.abs() + 2.0 ** -9 * 448 ** -1 * V.abs().amax()
                assert torch.all((got[mine].unflatten(1, (HQ, D))[:, h].double() - exact).abs() <= room)


def test_refusals_come_before_the_store(device):
    m = model(device)
    cache, table = cache_of(device, 1, 2)
    lengths = torch.full((1,), 4, dtype=torch.int32, device=device)
    for t in cache:
        t.view(torch.uint8).fill_(7)
    x = state(device, 4, 3)[0]
    pos, index = torch.zeros(4, 3, dtype=torch.int32, device=device), torch.zeros(4, dtype=torch.int32, device=device)
    base = (x, *m.projections, m.norm_q, m.norm_k, cache, table, lengths)
    for kw, needle in ((dict(rope=m.rope), "go together"), (dict(positions=pos), "go together"),
                       (dict(rope=m.rope, positions=pos, rotary_emb=(pos, pos)), "in place of"), (dict(adapters=m.banks), "go together"),
                       (dict(index=index), "go together"), (dict(adapters=m.banks[:2], index=index), "go together"),
                       (dict(rope=m.rope, positions=pos[:3]), "positions"), (dict(adapters=m.banks, index=index[:3]), "index"),
                       (dict(rope=m.rope, positions=pos, scale=-1.0), "scale")):
        with pytest.raises(ValueError, match=needle):
            cached_attention(*base, **kw)
    torch.cuda.synchronize()
    assert all(bool((t.view(torch.uint8) == 7).all()) for t in cache)


def test_a_projection_that_returns_a_buffer_of_its_own_keeps_it(device):
    m = model(device)
    cache, table = cache_of(device, 1, 2)
    lengths = torch.full((1,), 4, dtype=torch.int32, device=device)
    x = state(device, 4, 3)[0]
    outputs = [p(x) for p in m.projections]
    before = [t.clone() for t in outputs]
    index = torch.zeros(4, dtype=torch.int32, device=device)
    cached_attention(x, *[lambda _, t=t: t for t in outputs], m.norm_q, m.norm_k, cache, table, lengths, adapters=m.banks, index=index)
    assert all(torch.equal(a, b) for a, b in zip(before, outputs))


def test_a_step_in_a_graph(device):
    """The whole way captured, and replayed with other rows, requests, positions and lengths."""
    m = model(device)
    B = 5
    g = torch.Generator().manual_seed(3)
    mine, other = cache_of(device, B, 3), cache_of(device, B, 3)
    r, b = state(device, B, 1)
    lengths, positions = torch.full((B,), 1, dtype=torch.int32, device=device), torch.zeros(B, 3, dtype=torch.int32, device=device)
    index = torch.zeros(B, dtype=torch.int32, device=device)

    def step(cache, table):
        hidden, _, _, x = vdn_fp8.add_norm_quantize(r, b, m.norm.weight, m.norm.eps, return_normed=True)
        return hidden, cached_attention(x, *m.projections, m.norm_q, m.norm_k, cache, table, lengths, rope=m.rope, positions=positions,
                                        adapters=m.banks, index=index, causal=True)

    step(*mine), step(*other)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*mine)
    for n in range(1, 7):
        new = state(device, B, 20 + n)
        r.copy_(new[0]), b.copy_(new[1])
        lengths.fill_(n)
        positions.copy_(torch.randint(0, 99, (B, 3), generator=g).int())
        index.copy_(torch.randint(-1, 3, (B,), generator=g).int())
        graph.replay()
        want = step(*other)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b_) for a, b_ in zip(out, want)), n


@pytest.mark.parametrize("choice", [{}, {"top": 2, "query_block": 32}], ids=["dense", "top"])
def test_rows_that_attention_refuses_are_refused_before_the_store(device, choice):
    """float32 rows, which the rotation and the store take and attention does not: with `rope` nothing is stored either."""
    m = model(device)
    cache, table = cache_of(device, 1, 2)
    lengths = torch.full((1,), 4, dtype=torch.int32, device=device)
    for t in cache:
        t.view(torch.uint8).fill_(7)
    x = torch.randn(4, HIDDEN, device=device)
    projections = [torch.nn.Linear(HIDDEN, n * D, bias=False, device=device).requires_grad_(False) for n in (HQ, H, H)]
    norms = [types.SimpleNamespace(weight=torch.ones(D, device=device), eps=1e-6) for _ in "qk"]
    positions = torch.zeros(4, 3, dtype=torch.int32, device=device)
    with pytest.raises(ValueError, match="bfloat16, float16"):
        cached_attention(x, *projections, *norms, cache, table, lengths, rope=m.rope, positions=positions, **choice)
    torch.cuda.synchronize()
    assert all(bool((t.view(torch.uint8) == 7).all()) for t in cache)


def test_float16_rows(device):
    """A float16 block by `rope`: each call's result has the bits of its parts."""
    m = model(device)
    g = torch.Generator(device).manual_seed(2)
    cache, table = cache_of(device, 2, 2)
    other, _ = cache_of(device, 2, 2)
    weights = [(torch.randn(n * D, HIDDEN, device=device, generator=g) / 32).half() for n in (HQ, H, H)]
    projections = [lambda t, w=w: t @ w.T for w in weights]
    norms = [types.SimpleNamespace(weight=torch.ones(D, device=device, dtype=torch.float16), eps=1e-6) for _ in "qk"]
    for length in (30, 31):
        T = 60 if length == 30 else 2
        x = torch.randn(T, HIDDEN, device=device, generator=g).half()
        lengths = torch.full((2,), length, dtype=torch.int32, device=device)
        positions = torch.arange(T, device=device, dtype=torch.int32)[:, None].expand(T, 3)
        got = cached_attention(x, *projections, *norms, cache, table, lengths, rope=m.rope, positions=positions, causal=True)
        q, k, v = (p(x).unflatten(1, (-1, D)) for p in projections)
        q, k = vdn_fp8.qk_prep_axes(q, k, *((n.weight, n.eps) for n in norms), m.rope, positions)
        vdn_fp8.kv_append(k, v, other, table, lengths)
        want = vdn_fp8.kv_attention(q, other, table, lengths, causal=True)
        assert got.dtype == torch.float16 and torch.equal(got, want.flatten(1))
