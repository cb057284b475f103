"""The 8-bit key/value cache on the GPU at the edges of what its entry points allow: the largest blocks of
queries, weights far below a row's largest, hints that are wrong, batches without tokens."""
import numpy as np
import pytest
import torch

import kv_reference as R
import vdn_fp8
from kv_reference import PAGE
from test_gpu_kv_cache import attention_case, i32, near

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("group", [2048, 4096])
def test_blocks_of_more_rows_than_32_bits_count(device, group):
    """The largest query_block with large groups: a block has 2^31 and 2^32 rows, the call a few thousand."""
    print(f"block rows 2^20 x {group}", flush=True)
    blocks = np.array([[[0, 2, -1]]], np.int32)
    attention_case(device, BF16, group, 1, 64, [3], [170], True, seed=41, blocks=blocks, block=1 << 20)


# -- weights far below a row's largest ---------------------------------------------------------

def attend_by_channel(cache, q, table, length, scale, causal=False):
    """Attention of one sequence's last rows over one key/value head, in 64 bits, and a bound in which each
    channel answers for its own values: (out, lse, bound of out, bound of lse). q [n, Hq, d], H = 1.

    A page's largest weight P' = p 2^ev (p the weight, 2^ev the page's value scale) is held as 2^-5 at least, and
    as 2^5 where it moves the row's unit, which it does when it is more than 2^20 from every other page's (the unit
    is within 2^10 of the page before). Rounded to binary16 each is off by 2^-11 of itself or by 2^-25 there: 2^-20,
    or 2^-30, of the page's largest. A unit comes down by 2^60 and stays where it is
    within 2^10 of that: 2^-25 is then 2^-30 of a unit of 2^-50, 2^-80 of the row's largest at most. The products'
    sum is N / 16 sums one after another of 16 products each (four more levels), a few joins, and a power and a product
    for each page that moves the unit: N / 16 + N / 32 + 22 roundings (2^-23, should they truncate) of the magnitudes.
    Scores as in kv_reference.attend."""
    n, Hq, d = q.shape
    pages = -(-length // PAGE)
    k = torch.cat([R.decode(cache.k[p, 0], cache.ek[p, 0]) for p in table[:pages]])[:length]
    v = torch.cat([R.decode(cache.v[p, 0], cache.ev[p, 0]).T for p in table[:pages]])[:length]
    x = q.double().reshape(n * Hq, d)
    s = scale * (x @ k.T)
    if causal:
        limit = length - n + torch.arange(n).repeat_interleave(Hq)
        s.masked_fill_(torch.arange(length)[None] > limit[:, None], -float("inf"))
    z = torch.logsumexp(s, 1)
    p = torch.exp(s - z[:, None])
    out, a = p @ v, p @ v.abs()
    pad = pages * PAGE - length
    most = torch.nn.functional.pad(p, (0, pad)).reshape(-1, pages, PAGE).amax(2)
    ev = torch.stack([cache.ev[p, 0] for p in table[:pages]]).double()
    size = torch.nn.functional.pad(v.abs(), (0, 0, 0, pad)).reshape(pages, PAGE, d).sum(1) * torch.exp2(-ev)[:, None]   # of codes
    unit = most * torch.exp2(ev)
    first, second = unit.topk(min(2, pages), 1).values.T[[0, -1]]
    alone = (unit == first[:, None]) & (first > 2.0 ** 20 * second)[:, None]
    held = torch.where(alone, 2.0 ** -30, 2.0 ** -20) * unit + 2.0 ** -80 * first[:, None]
    es = scale * 2.0 ** -18 * (x.abs() @ k.abs().T).amax(1)
    tol = (2.0 ** -11 + 2.0 ** -18 + 2.0 ** -23 * (length / 16 + length / 32 + 22) + 2 * es)[:, None] * a + held @ size
    return out.reshape(n, Hq, d), z.reshape(n, Hq), tol.reshape(n, Hq, d), (2 * es + 2.0 ** -20 + 2.0 ** -22 * z.abs()).reshape(n, Hq)


def sink_cache(d, length, nats, outlier, at, amount=8.0):
    """One head: `length` tokens, of which number `at` has a score `nats` above the others' middle for queries whose
    first element is `amount`, and a value of zeros but for `outlier` in channel 5; the others' values are about 1."""
    g = torch.Generator().manual_seed(int(10 * nats) + d)
    key, value = torch.randn(length, 1, d, generator=g), 1 + 0.3 * torch.randn(length, 1, d, generator=g)
    key[:, 0, 0] = 0
    key[at], value[at] = 0, 0
    key[at, 0, 0] = nats * d ** 0.5 / amount
    value[at, 0, 5] = outlier
    pages = -(-length // PAGE)
    cache, table = R.Cache(pages, 1, d, seed=2), torch.randperm(pages, generator=g).tolist()
    R.append(cache, key.to(BF16), value.to(BF16), [table], [length], [0, length])
    return cache, table


def sink_queries(n, heads, d, seed=0, amount=8.0):
    q = torch.randn(n, heads, d, generator=torch.Generator().manual_seed(seed + n)).to(F16)
    q[:, :, 0] = amount
    return q


# (sequences of one table, rows of each, query heads): k_kv_attn_rows whole and split, k_kv_attn_step whole and split
FORMS = [(300, 20, 1), (1, 150, 1), (1100, 1, 2), (2, 1, 5)]


@pytest.mark.parametrize("nats,outlier", [(14.0, 0.0), (17.5, 0.0), (20.0, 0.0), (30.0, 0.0), (10.0, 1000.0), (11.5, 200.0), (3.0, 3e4)])
@pytest.mark.parametrize("B,n,heads", FORMS)
def test_weights_far_below_the_largest(device, nats, outlier, B, n, heads):
    """A token that takes most of the weight and has little of the value (and, in one channel, the largest of
    its page): the others' part of each channel keeps its bits, wherever the token stands."""
    d, length = 64, 30011
    for at in (0, length // 2 + 3, length - 1):
        print(f"sink {nats} nats, outlier {outlier}, at {at}, {B} x {n} rows of {heads}", flush=True)
        cache, table = sink_cache(d, length, nats, outlier, at)
        q = sink_queries(B * n, heads, d)
        out, z = vdn_fp8.kv_attention(q.to(device), vdn_fp8.KvCache(*cache.tensors(device)), i32([table], device).expand(B, len(table)),
                                      i32([length] * B, device), return_lse=True)
        for b in {0, B - 1}:
            rows = slice(b * n, (b + 1) * n)
            want, wz, tol, tol_z = attend_by_channel(cache, q[rows], table, length, d ** -0.5)
            near(out[rows], want, tol, F16)
            assert bool(((z[rows].double().cpu() - wz).abs() <= tol_z).all())


@pytest.mark.parametrize("d,dtype", [(128, F16), (256, F16), (128, BF16)])
@pytest.mark.parametrize("rows", [1, 60])
def test_weights_far_below_the_largest_of_every_size(device, d, dtype, rows):
    for nats, outlier in ((18.0, 0.0), (10.0, 1000.0)):
        print(f"sink d={d} {dtype} rows={rows} {nats} {outlier}", flush=True)
        cache, table = sink_cache(d, 9000, nats, outlier, 70)
        q = sink_queries(rows, 2, d).to(dtype)
        got = vdn_fp8.kv_attention(q.to(device), vdn_fp8.KvCache(*cache.tensors(device)), i32([table], device), i32([9000], device), causal=True)
        want, _, tol, _ = attend_by_channel(cache, q, table, 9000, d ** -0.5, True)
        near(got, want, tol, dtype)


@pytest.mark.parametrize("B,n", [(300, 20), (1100, 1)])
def test_scores_that_climb_and_fall(device, B, n):
    """Pages whose largest scores rise and fall by tens of nats, sizes of values with and against them."""
    d, pages = 64, 48
    g = torch.Generator().manual_seed(44)
    step = torch.tensor([0, 30, 5, 60, 59, 0, 44, 80, 81, 20, 2, 79], dtype=torch.float32).repeat(pages // 12).repeat_interleave(PAGE)
    for sign in (0.0, 0.4, -0.4):
        print(f"climb {B} x {n} sign {sign}", flush=True)
        key, value = torch.randn(pages * PAGE, 1, d, generator=g), torch.randn(pages * PAGE, 1, d, generator=g)
        key[:, 0, 0] = step * d ** 0.5 / 8
        value *= torch.exp(sign * step)[:, None, None]
        cache, table = R.Cache(pages, 1, d, seed=3), list(range(pages))
        R.append(cache, key.to(BF16), value.to(BF16), [table], [pages * PAGE], [0, pages * PAGE])
        q = sink_queries(B * n, 1, d).to(BF16)
        out, z = vdn_fp8.kv_attention(q.to(device), vdn_fp8.KvCache(*cache.tensors(device)), i32([table], device).expand(B, pages),
                                      i32([pages * PAGE] * B, device), return_lse=True)
        for b in (0, B - 1):
            rows = slice(b * n, (b + 1) * n)
            want, wz, tol, tol_z = attend_by_channel(cache, q[rows], table, pages * PAGE, d ** -0.5)
            near(out[rows], want, tol, BF16)
            assert bool(((z[rows].double().cpu() - wz).abs() <= tol_z).all())


def test_the_sum_of_many_pages_of_zeros(device):
    """Values of zeros have the least scale; the sum of weights of 2.5 million tokens of them stays a number."""
    d, pages, B, n = 64, 40000, 300, 20
    key, value = torch.zeros(2 * PAGE, 1, d), torch.zeros(2 * PAGE, 1, d)
    key[PAGE:, 0, 0] = 5.25
    cache = R.Cache(2, 1, d, seed=1)
    R.append(cache, key.to(BF16), value.to(BF16), [[0, 1]], [2 * PAGE], [0, 2 * PAGE])
    q = torch.zeros(B * n, 1, d, dtype=BF16)
    q[:, :, 0] = 1.0
    table = i32([[0] + [1] * (pages - 1)], device).expand(B, pages)
    out, z = vdn_fp8.kv_attention(q.to(device), vdn_fp8.KvCache(*cache.tensors(device)), table, i32([pages * PAGE] * B, device), scale=1.0,
                                  return_lse=True)
    top = float(R.decode(cache.k[1, 0], cache.ek[1, 0])[0, 0])
    want = top + np.log(64.0 * (pages - 1) + 64.0 * np.exp(-top))
    assert not bool(out.any())
    # one sum a page in binary32, and the logarithm's rounding (the unit moves once)
    assert bool(((z.double() - want).abs() <= pages * 2.0 ** -24 + 2.0 ** -20).all())


# -- hints and empty batches -------------------------------------------------------------------

@pytest.mark.parametrize("d,Hq,H", [(64, 3, 1), (128, 10, 2), (256, 4, 2)])
@pytest.mark.parametrize("news,lengths", [([1, 5, 40], [90, 5, 700]), ([0, 17, 1], [70, 3000, 1]), ([33], [4100])])
@pytest.mark.parametrize("causal", [False, True])
def test_more_rows_than_max_query(device, d, Hq, H, news, lengths, causal):
    """max_query chooses a kernel; rows beyond it are attended to all the same."""
    for most in (1, 2):
        print(f"max_query {most} of {news} d={d} {Hq}/{H} causal={causal}", flush=True)
        torch.full((1 << 22,), float("nan"), device=device)   # (what an allocation of the call may find)
        attention_case(device, BF16, Hq, H, d, news, lengths, causal, seed=43, ragged=True, max_query=most)


def test_choice_of_a_batch_without_tokens(device):
    """No tokens, sequences with q_start: each has a row of the list that no block takes."""
    H, d = 2, 128
    kc = vdn_fp8.KvCache(*R.Cache(3, H, d, seed=1).tensors(device))
    q, table, lengths = torch.zeros(0, 4, d, dtype=BF16, device=device), i32([[0, 1], [2, -1]], device), i32([100, 30], device)
    for block, rows in ((128, 2), (1, 0)):
        torch.full((rows * H * 3,), 7, dtype=torch.int32, device=device)   # (what the allocation may find)
        lists = vdn_fp8.kv_select(q, kc, table, lengths, 3, query_block=block, q_start=i32([0, 0, 0], device))
        assert lists.shape == (rows, H, 3) and bool((lists == -1).all())


# -- splits of short key axes ------------------------------------------------------------------

@pytest.mark.parametrize("d,Hq,H,B,n,pages,split", [
    (128, 40, 8, 1, 1, 16, False), (128, 40, 8, 1, 1, 24, True), (256, 32, 4, 1, 1, 16, True), (64, 16, 2, 1, 1, 24, False),
    (64, 12, 12, 3, 77, 8, False), (64, 12, 12, 3, 77, 12, True), (64, 12, 12, 3, 77, 31, True), (128, 8, 8, 4, 300, 14, False), (128, 8, 8, 4, 300, 24, True),
])
def test_short_key_axes_are_split_where_that_pays(device, d, Hq, H, B, n, pages, split):
    """Below 32 pages too, where the pages spared outweigh the parts; the workspace tells which way a call goes."""
    import ctypes

    import vdn_fp8._lib as L
    if torch.cuda.get_device_properties(device).multi_processor_count != 256:
        pytest.skip("the sizes are those of 256 compute units")
    size = ctypes.c_int64(-1)
    c = L.KvCacheStruct(*[1 << 20] * 5, pages, H, d)
    b = L.KvBatchStruct(1 << 20, pages, pages, 1 << 20, None, B, B * n)
    assert L.load().vdn_fp8_kv_attention_workspace_size(c, b, Hq, 0, 0, 0, ctypes.byref(size)) == L.OK
    assert (size.value > 0) == split
    if B == 1 or n < 100:
        print(f"split {pages} pages d={d} {Hq}/{H}", flush=True)
        attention_case(device, BF16, Hq, H, d, [n] * B, [pages * PAGE - 5 * b for b in range(B)], True, seed=45, extra=0)


# -- the branch --------------------------------------------------------------------------------

def branch(device, H, d, C, seed=51):
    g = torch.Generator().manual_seed(seed)
    to = [torch.nn.Linear(C, H * d, dtype=BF16) for _ in range(3)]
    for m in to:
        m.weight.data.copy_(0.1 * torch.randn(m.weight.shape, generator=g))
    norm = torch.nn.RMSNorm(d, eps=1e-6, dtype=BF16).to(device)
    return [m.to(device).requires_grad_(False) for m in to], norm.requires_grad_(False), g


def test_the_branch_refuses_sizes_before_it_stores(device):
    """What only the library knows to refuse: more sequences than a choice of pages numbers, more workgroups than a
    launch holds."""
    from vdn_fp8.softmax_attention import cached_attention
    H, d, C, B = 1, 64, 16, 70000
    to, norm, g = branch(device, H, d, C)
    x = torch.randn(B, C, generator=g).to(BF16).to(device)
    kc = vdn_fp8.KvCache.empty(2, H, d, device)
    for t in kc:
        t.view(torch.uint8).zero_()
    table, lengths = i32([[0]], device).expand(B, 1), torch.zeros(B, dtype=torch.int32, device=device)
    lengths[0] = 1
    with pytest.raises(ValueError, match="65535"):
        cached_attention(x, *to, norm, norm, kc, table, lengths, top=2, query_block=1)
    assert not any(bool(t.view(torch.uint8).any()) for t in kc)
    # (a head's units of rows and one behind the last sequence, 2^24 of them with 4096 heads of few tokens each)
    heads = 4096
    wide = vdn_fp8.KvCache.empty(1, heads, d, device)
    rows = torch.zeros(5000, heads, d, dtype=BF16, device=device)
    start, table = torch.arange(5001, dtype=torch.int32, device=device), i32([[0]], device).expand(5000, 1)
    with pytest.raises(ValueError, match="2\\^24"):
        vdn_fp8.kv_cache.check_attention(rows, wide, table, torch.ones(5000, dtype=torch.int32, device=device), q_start=start)


def test_the_branch_over_one_page(device):
    """top = 1: the newest page alone, or the best one."""
    from vdn_fp8 import softmax_attention as SA
    H, d, C, n = 2, 64, 48, 128
    to, norm, g = branch(device, H, d, C)
    table = i32([[4, 0, 2, 3]], device)
    caches = []
    for _ in range(2):
        caches.append(vdn_fp8.KvCache.empty(5, H, d, device))
        for t in caches[-1]:
            t.view(torch.uint8).zero_()
    lengths = i32([0], device)
    for first, last in ((0, 1), (0, 0)):
        x = torch.randn(n, C, generator=g).to(BF16).to(device)
        lengths += n
        out = SA.cached_attention(x, *to, norm, norm, caches[0], table, lengths, top=1, query_block=128, first=first, last=last)
        q, k, v, _ = SA.qkv(x, *to, H, norm, norm)
        vdn_fp8.kv_append(k, v, caches[1], table, lengths)
        lists = vdn_fp8.kv_select(q, caches[1], table, lengths, 1, query_block=128, first=first, last=last)
        assert torch.equal(out, vdn_fp8.kv_attention(q, caches[1], table, lengths, blocks=lists, query_block=128).flatten(1))
        assert last == 0 or bool((lists == lengths.item() // PAGE - 1).all())


@pytest.mark.parametrize("block", [0, -64])
def test_lists_of_no_queries_are_refused(device, block):
    H, d = 2, 64
    kc = vdn_fp8.KvCache.empty(2, H, d, device)
    q, blocks = torch.zeros(3, H, d, dtype=BF16, device=device), torch.zeros(1, H, 1, dtype=torch.int32, device=device)
    for start in (None, i32([0, 3], device)):
        with pytest.raises(ValueError, match="query_block"):
            vdn_fp8.kv_attention(q, kc, i32([[0]], device), i32([3], device), q_start=start, blocks=blocks, query_block=block)
