"""The 8-bit key/value cache on the GPU at the sizes where its kernels change their ways: batches of
more sequences than a wave has lanes, several heads to a workgroup, more pages than a workgroup looks
up at a time, tables without columns, graphs whose batch changes between replays, and the attention
branch over a cache."""
import numpy as np
import pytest
import torch
import torch.nn as nn

import kv_reference as R
import vdn_fp8
from kv_reference import PAGE
from test_gpu_kv_cache import attention_case, i32, near, same_cache, starts_of, tables

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def ragged(B, most, seed):
    """Rows and lengths of B sequences, some empty, some without rows."""
    rng = np.random.default_rng(seed)
    news = rng.integers(0, most + 1, B)
    return news.tolist(), (news + rng.integers(0, 150, B) * (rng.random(B) < 0.8)).tolist()


# -- batches ---------------------------------------------------------------------------------

@pytest.mark.parametrize("B,most", [(64, 1), (65, 2), (200, 3)])
def test_append_of_many_sequences(device, B, most):
    print(f"append B={B}", flush=True)
    H, d = 2, 64
    news, lengths = ragged(B, most, B)
    g, T = torch.Generator().manual_seed(B), sum(news)
    pages = sum(-(-n // PAGE) for n in lengths) + 1
    table = tables(lengths, pages, 2)
    key, value = (torch.randn(T, H, d, generator=g).to(BF16) for _ in range(2))
    want = R.Cache(pages, H, d, seed=3)
    for c in (want.k, want.v):
        u = c.view(torch.uint8)
        u[(u & 0x7F) == 0x7F] = 0x42
    got = vdn_fp8.KvCache(*want.tensors(device))
    R.append(want, key, value, table, lengths, starts_of(news))
    vdn_fp8.kv_append(key.to(device), value.to(device), got, i32(table, device), i32(lengths, device), q_start=i32(starts_of(news), device))
    torch.cuda.synchronize()
    same_cache(got, want)


@pytest.mark.parametrize("B,most,group,max_query", [(64, 1, 2, 1), (65, 3, 5, 3), (200, 3, 1, None), (130, 40, 1, 40)])
def test_attention_of_many_sequences(device, B, most, group, max_query):
    print(f"attention B={B} most={most} group={group}", flush=True)
    news, lengths = ragged(B, most, B + most)
    attention_case(device, BF16, 2 * group, 2, 64, news, lengths, True, seed=B, ragged=True, max_query=max_query)


@pytest.mark.parametrize("block", [1, 128])
def test_select_of_many_sequences(device, block):
    B, H, d = 130, 1, 64
    news, lengths = ragged(B, 3 if block == 1 else 150, block)
    starts = starts_of(news)
    pages = sum(-(-n // PAGE) for n in lengths) + 1
    table, cache = tables(lengths, pages, 4), R.Cache(pages, H, d, seed=5)
    q = torch.randn(sum(news), H, d, generator=torch.Generator().manual_seed(3)).to(BF16)
    want = R.select(cache, q, table, lengths, starts, 2, block, 1, 1, True, True)
    got = vdn_fp8.kv_select(q.to(device), vdn_fp8.KvCache(*cache.tensors(device)), i32(table, device), i32(lengths, device), 2, query_block=block,
                            causal=True, q_start=i32(starts, device))
    assert np.array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("d,Hq,H,news,lengths", [(64, 24, 2, [1, 2], [300, 90]), (256, 12, 1, [1], [500]), (128, 9, 1, [3, 3], [700, 2]), (256, 2, 2, [1, 1, 1], [64, 0, 1000])])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("causal", [False, True])
def test_single_queries_choose_and_attend(device, d, Hq, H, news, lengths, dtype, causal):
    """Each query its own pages, groups above and below eight heads, every head size."""
    print(f"single queries {dtype} d={d} {Hq}/{H} {news} of {lengths} causal={causal}", flush=True)
    starts, ragged_ = starts_of(news), len(set(news)) != 1
    pages = sum(-(-n // PAGE) for n in lengths) + 2
    table, cache = tables(lengths, pages, 1), R.Cache(pages, H, d, seed=6)
    g = torch.Generator().manual_seed(d + Hq)
    key, value = (torch.randn(sum(lengths), H, d, generator=g).to(BF16) for _ in range(2))
    R.append(cache, key, value, table, lengths, starts_of(lengths))
    q = torch.randn(sum(news), Hq, d, generator=g).to(dtype)
    want = R.select(cache, q, table, lengths, starts, 3, 1, 1, 1, causal, ragged_)
    got = vdn_fp8.kv_select(q.to(device), vdn_fp8.KvCache(*cache.tensors(device)), i32(table, device), i32(lengths, device), 3, query_block=1,
                            causal=causal, q_start=i32(starts, device) if ragged_ else None)
    assert np.array_equal(got.cpu().numpy(), want)
    attention_case(device, dtype, Hq, H, d, news, lengths, causal, cache=cache, table=table, q=q, blocks=want, block=1, max_query=max(news))


def test_more_single_queries_than_a_launch_numbers(device):
    """Past 65535 single queries the page scores take the way of the blocks; the choice is the same."""
    n, H, d, length = 66000, 1, 64, 330
    g = torch.Generator().manual_seed(15)
    pages = -(-length // PAGE)
    cache, table = R.Cache(pages, H, d, seed=6), [list(range(pages))]
    q = torch.randn(n, H, d, generator=g).to(BF16)
    got = vdn_fp8.kv_select(q.to(device), vdn_fp8.KvCache(*cache.tensors(device)), i32(table, device), i32([length], device), 3, query_block=1)
    for rows in (slice(0, 40), slice(65510, 65560), slice(n - 30, n)):
        part = q[rows]
        want = R.select(cache, part, table, [length], [0, len(part)], 3, 1, 1, 1, False)
        assert np.array_equal(got[rows].cpu().numpy(), want)


# -- workgroups ------------------------------------------------------------------------------

@pytest.mark.parametrize("H,d,T", [(10, 64, 9000), (9, 128, 7000), (6, 256, 6000)])
def test_append_of_several_heads_a_workgroup(device, H, d, T):
    """Enough tokens for workgroups that take several heads, the last of them fewer."""
    print(f"append {T} tokens of {H} heads of {d}", flush=True)
    g = torch.Generator().manual_seed(T)
    lengths, pages = [T + 21], -(-(T + 21) // PAGE) + 1
    table = tables(lengths, pages, 6)
    key, value = (torch.randn(T, H, d, generator=g).to(BF16) for _ in range(2))
    key[T // 3] = 0
    key[T // 2, :, 5], value[T // 2 + 70, 1] = float("nan"), float("inf")
    want = R.Cache(pages, H, d, seed=7)
    for c in (want.k, want.v):
        u = c.view(torch.uint8)
        u[(u & 0x7F) == 0x7F] = 0x42
    got = vdn_fp8.KvCache(*want.tensors(device))
    R.append(want, key, value, table, lengths, [0, T])
    vdn_fp8.kv_append(key.to(device), value.to(device), got, i32(table, device), i32(lengths, device))
    torch.cuda.synchronize()
    same_cache(got, want)


def test_prep_append_of_many_tokens_has_the_bits_of_its_parts(device):
    T, Hq, H, d = 3001, 40, 10, 128
    g = torch.Generator(device=device).manual_seed(8)
    q, k, v = (torch.randn(T, n, d, device=device, generator=g).to(BF16) for n in (Hq, H, H))
    angle = 6.28 * torch.rand(T, d // 2, device=device, generator=g)
    cos, sin = (torch.cat([f(angle), f(angle)], 1) for f in (torch.cos, torch.sin))
    norm = (1 + 0.1 * torch.randn(d, device=device, generator=g).to(BF16), 1e-6)
    pages = -(-T // PAGE)
    table, lengths = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).to(torch.int32).to(device)[None], i32([T], device)
    caches = []
    for _ in range(2):
        caches.append(vdn_fp8.KvCache.empty(pages, H, d, device))
        for t in caches[-1]:
            t.view(torch.uint8).zero_()   # (codes behind the last token stay as they were)
    out = vdn_fp8.qk_prep_append(q, k, v, norm, norm, caches[0], table, lengths, cos=cos, sin=sin)
    assert torch.equal(out, vdn_fp8.qk_prep(q, *norm, cos, sin))
    vdn_fp8.kv_append(vdn_fp8.qk_prep(k, *norm, cos, sin), v, caches[1], table, lengths)
    for a, b in zip(*caches):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("n,B,H,group", [(1, 1100, 1, 3), (130, 300, 1, 1)])
def test_more_pages_than_a_workgroup_looks_up(device, n, B, H, group):
    """So many sequences that no key axis is split, of more pages than are looked up at a time; a NaN
    value that the last rows alone see. The pages are shared: every sequence attends to the same."""
    d, length = 64, 257 * PAGE + 70
    print(f"{B} sequences of {n} rows on {length}", flush=True)
    g = torch.Generator().manual_seed(n)
    cache, pages = R.Cache(261, H, d, seed=1), 259
    order = torch.randperm(261, generator=g)[:pages].tolist()
    key, value = (torch.randn(length, H, d, generator=g).to(BF16) for _ in range(2))
    value[length - 2, 0, 3] = float("nan")
    R.append(cache, key, value, [order], [length], [0, length])
    q = torch.randn(B * n, H * group, d, generator=g).to(BF16)
    kc = vdn_fp8.KvCache(*cache.tensors(device))
    out, z = vdn_fp8.kv_attention(q.to(device), kc, i32([order], device).expand(B, pages), i32([length] * B, device), causal=True, return_lse=True)
    for b in (0, B // 2, B - 1):
        rows = slice(b * n, (b + 1) * n)
        want, wz, tol, tol_z = R.attend(cache, q[rows], [order], [length], [0, n], d ** -0.5, True)
        near(out[rows], want, tol, BF16)
        assert bool(((z[rows].double().cpu() - wz).abs() <= tol_z).all())


@pytest.mark.parametrize("rows", [1, 20, 150])
@pytest.mark.parametrize("order", [[0, 1, 2, 3], [3, 2, 1, 0], [1, 3, 0, 2]])
def test_scales_of_values_further_apart_than_a_float(device, rows, order):
    """Pages of zeros and tiny values beside pages of enormous ones: the former take no less of the weight,
    whichever come first, in one pass and where the keys are split."""
    H, d = 1, 64
    g = torch.Generator().manual_seed(14)
    for pages in (4, 64):
        sizes = [0.0, 1e-24, 1.0, 1e33] * (pages // 4)
        value = torch.cat([torch.randn(PAGE, H, d, generator=g) * sizes[(w // 4) * 4 + order[w % 4]] for w in range(pages)]).to(BF16)
        n = pages * PAGE
        cache, table = R.Cache(pages, H, d, seed=2), [list(range(pages))]
        R.append(cache, torch.randn(n, H, d, generator=g).to(BF16), value, table, [n], [0, n])
        print(f"far apart rows={rows} pages={pages} {order}", flush=True)
        q = torch.randn(rows, 2, d, generator=g).to(BF16)
        attention_case(device, BF16, 2, H, d, [rows], [n], False, cache=cache, table=table, q=q)
        attention_case(device, BF16, 2, H, d, [rows], [n], False, cache=cache, table=table, q=q, scale=2.0)


@pytest.mark.parametrize("n", [1, 40])
def test_a_table_without_columns(device, n):
    """No sequence has a page: nothing is stored, every row is zeros, every list empty."""
    H, d = 2, 128
    kc = vdn_fp8.KvCache(*R.Cache(3, H, d, seed=1).tensors(device))
    before = [t.clone() for t in kc]
    table, lengths = i32([[], []], device).reshape(2, 0), i32([0, 0], device)
    x = torch.randn(2 * n, H, d, device=device).to(BF16)
    vdn_fp8.kv_append(x, x, kc, table, lengths)
    for a, b in zip(before, kc):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    out, z = vdn_fp8.kv_attention(x, kc, table, lengths, causal=True, return_lse=True)
    assert not bool(out.any()) and bool((z == -float("inf")).all())
    for block in (1, 128):
        lists = vdn_fp8.kv_select(x, kc, table, lengths, 2, query_block=block)
        assert bool((lists == -1).all())
        assert not bool(vdn_fp8.kv_attention(x, kc, table, lengths, blocks=lists, query_block=block).any())


# -- graphs ----------------------------------------------------------------------------------

def test_a_captured_batch_that_changes(device):
    """One graph of a padded batch, replayed with other rows, lengths and pages: each replay equals the
    eager call, the rows behind the last sequence included."""
    H, d, T, B = 2, 128, 300, 4
    g = torch.Generator().manual_seed(9)
    base = R.Cache(64, H, d, seed=8)
    for c in (base.k, base.v):
        c.view(torch.uint8).bitwise_and_(0x3F)
    caches = [vdn_fp8.KvCache(*base.tensors(device)) for _ in range(2)]
    table, lengths, start = (torch.zeros(s, dtype=torch.int32, device=device) for s in ((B, 16), (B,), (B + 1,)))
    key, value, query = (torch.zeros(T, h, d, device=device, dtype=BF16) for h in (H, H, 2 * H))

    def calls(cache):
        vdn_fp8.kv_append(key, value, cache, table, lengths, q_start=start)
        lists = vdn_fp8.kv_select(query, cache, table, lengths, 3, query_block=64, causal=True, q_start=start)
        return (lists, *vdn_fp8.kv_attention(query, cache, table, lengths, causal=True, q_start=start, return_lse=True),
                vdn_fp8.kv_attention(query, cache, table, lengths, causal=True, q_start=start, blocks=lists, query_block=64))

    def fill(news, olds):
        now = [a + b for a, b in zip(news, olds)]
        table.copy_(torch.tensor([r + [-1] * (16 - len(r)) for r in tables(now, 64, sum(news), extra=0)], dtype=torch.int32))
        lengths.copy_(torch.tensor(now, dtype=torch.int32))
        start.copy_(torch.tensor(starts_of(news), dtype=torch.int32))
        for t in (key, value, query):
            t.copy_(torch.randn(t.shape, generator=g))

    fill([1, 1, 1, 1], [0, 5, 64, 100])
    calls(caches[1])
    caches[1] = vdn_fp8.KvCache(*base.tensors(device))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = calls(caches[0])
    for news, olds in (([1, 1, 1, 1], [0, 5, 64, 100]), ([0, 299, 0, 1], [30, 400, 0, 0]), ([0, 0, 0, 0], [1, 2, 3, 4]), ([75, 75, 75, 75], [1, 0, 200, 63])):
        fill(news, olds)
        want = calls(caches[1])
        graph.replay()
        (query.float().sum() + 1).item()
        for i, (a, b) in enumerate(zip(out, want)):
            assert torch.equal(a, b), (news, i)
        for a, b in zip(*caches):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), news


# -- the branch ------------------------------------------------------------------------------

def _linear(n, k, g, device):
    lin = nn.Linear(k, n, dtype=BF16, device="meta")
    lin.weight = nn.Parameter((0.02 * torch.randn(n, k, generator=g)).to(BF16).to(device), requires_grad=False)
    lin.bias = nn.Parameter((0.01 * torch.randn(n, generator=g)).to(BF16).to(device), requires_grad=False)
    return vdn_fp8.Fp8Linear(lin)


@pytest.mark.parametrize("chosen", [False, True])
def test_the_branch_over_a_cache(device, chosen):
    """`cached_attention` chunk by chunk: the bits of its parts (`qkv`, `kv_append`, `kv_select`,
    `kv_attention`), and a plain attention over everything stored."""
    from vdn_fp8 import softmax_attention as SA
    Hq, H, d, C, chunk = 4, 2, 128, 512, 128
    g = torch.Generator().manual_seed(12)
    to_q, to_k, to_v = (_linear(n * d, C, g, device) for n in (Hq, H, H))
    norm_q, norm_k = (nn.RMSNorm(d, eps=1e-6, dtype=BF16).to(device) for _ in range(2))
    norm_q.weight.data.copy_(1 + 0.1 * torch.randn(d, generator=g))
    caches = []
    for _ in range(2):
        caches.append(vdn_fp8.KvCache.empty(8, H, d, device))
        for t in caches[-1]:
            t.view(torch.uint8).zero_()
    table, lengths = [[6, 1, 0, 7, 3, 2, 5]], i32([0], device)
    pages = i32(table, device)
    more = dict(top=3, query_block=64) if chosen else {}
    for _ in range(3):
        x = torch.randn(chunk, C, generator=g).to(BF16).to(device)
        angle = 6.28 * torch.rand(chunk, d // 2, generator=g)
        rope = tuple(torch.cat([f(angle), f(angle)], 1).to(device) for f in (torch.cos, torch.sin))
        lengths += chunk
        with torch.no_grad():
            out = SA.cached_attention(x, to_q, to_k, to_v, norm_q, norm_k, caches[0], pages, lengths, rotary_emb=rope, **more)
            codes, scales = vdn_fp8.quantize_activation(x)
            q, k, v = (p.forward_quantized(codes, scales).unflatten(-1, (-1, d)) for p in (to_q, to_k, to_v))
            q, k = (vdn_fp8.qk_prep(t, n.weight, n.eps, *rope) for t, n in ((q, norm_q), (k, norm_k)))
            vdn_fp8.kv_append(k, v, caches[1], pages, lengths)
            lists = vdn_fp8.kv_select(q, caches[1], pages, lengths, 3, query_block=64) if chosen else None
            want = vdn_fp8.kv_attention(q, caches[1], pages, lengths, blocks=lists, query_block=64 if chosen else None)
        assert out.shape == (chunk, Hq * d) and torch.equal(out, want.flatten(1))
        for a, b in zip(*caches):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        plain = R.Cache(8, H, d, seed=0)
        plain.k, plain.v = caches[1].k.cpu(), caches[1].v.cpu()
        plain.ek, plain.ev = (t.cpu().view(torch.uint8).int() - 127 for t in (caches[1].k_scale, caches[1].v_scale))
        exact, _, tol, _ = R.attend(plain, q.cpu(), table, lengths.tolist(), [0, chunk], d ** -0.5, False, None if lists is None else lists.cpu(),
                                    64 if chosen else None)
        near(want, exact, tol, BF16)


def test_the_branch_with_other_projections(device):
    """Projections that are not `Fp8Linear`, no rotation, a ragged batch; `top` alone is refused."""
    from vdn_fp8 import softmax_attention as SA
    H, d, C = 2, 64, 96
    g = torch.Generator().manual_seed(13)
    projections = [nn.Linear(C, H * d, dtype=BF16).to(device).requires_grad_(False) for _ in range(3)]
    norm = nn.RMSNorm(d, eps=1e-6, dtype=BF16).to(device)
    x = torch.randn(70, C, generator=g).to(BF16).to(device)
    table, lengths, start = i32([[0, 1], [2, -1]], device), i32([67, 3], device), i32([0, 67, 70], device)
    caches = [vdn_fp8.KvCache.empty(3, H, d, device) for _ in range(2)]
    with torch.no_grad():
        out = SA.cached_attention(x, *projections, norm, norm, caches[0], table, lengths, causal=True, scale=0.2, q_start=start, max_query=67)
        q, k, v, _ = SA.qkv(x, *projections, H, norm, norm)
        vdn_fp8.kv_append(k, v, caches[1], table, lengths, q_start=start)
        want = vdn_fp8.kv_attention(q, caches[1], table, lengths, causal=True, scale=0.2, q_start=start, max_query=67)
    assert torch.equal(out, want.flatten(1))
    with pytest.raises(ValueError, match="query_block"):
        SA.cached_attention(x, *projections, norm, norm, caches[0], table, lengths, q_start=start, top=2)
