"""The 8-bit key/value cache on the GPU against plain 64-bit implementations (kv_reference.py):
codes, scales and means bit for bit, attention within a bound that counts its roundings,
chosen pages exactly; the entry points' run together; streams, graphs and padded batches."""
import numpy as np
import pytest
import torch

import kv_reference as R
import vdn_fp8
from kv_reference import PAGE

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def tables(lengths, pages, seed, extra=1, hole=None):
    """Page lists of the sequences (with `extra` unused entries), scattered over the pool."""
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=g).tolist()
    out, W = [], max([-(-n // PAGE) for n in lengths] + [0]) + extra
    for n in lengths:
        need = -(-n // PAGE)
        out.append([order.pop() for _ in range(need)] + [-1] * (W - need))
    if hole is not None:
        out[hole[0]][hole[1]] = hole[2]
    return out


def starts_of(news):
    return [sum(news[:b]) for b in range(len(news) + 1)]


def same_cache(got, want, touched=None):
    k, v, ks, vs, mean = (t.cpu() for t in got)
    for a, b in ((k, want.k), (v, want.v)):
        x, y = a.view(torch.uint8), b.view(torch.uint8)
        nan = ((x & 0x7F) == 0x7F) & ((y & 0x7F) == 0x7F)
        assert torch.equal(torch.where(nan, y, x), y)
    assert torch.equal(ks.view(torch.uint8).int() - 127, want.ek.int())
    assert torch.equal(vs.view(torch.uint8).int() - 127, want.ev.int())
    x, y = mean.float(), want.mean.float()
    assert torch.equal(x.nan_to_num(1e30), y.nan_to_num(1e30)) and torch.equal(x.isnan(), y.isnan())


def near(got, want, tol, dtype):
    """got within tol of want before one rounding to dtype."""
    got = got.double().cpu()
    half = torch.finfo(dtype).eps / 2
    bound = tol + half * (want.abs() + tol) + torch.finfo(dtype).smallest_normal * half
    assert torch.equal(got.isnan(), want.isnan())
    ok = want.isnan() | ((got - want).abs() <= bound)
    assert bool(ok.all()), float(((got - want).abs() / bound).nan_to_num(0).max())


# -- storing ---------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("H,d", [(1, 64), (3, 128), (2, 256)])
@pytest.mark.parametrize("news,olds", [
    ([1], [0]), ([1], [63]), ([1], [64]), ([64], [0]), ([65], [63]), ([130], [5]), ([3, 1, 200, 64, 0], [0, 127, 33, 64, 70]),
])
def test_append(device, dtype, H, d, news, olds):
    print(f"append {dtype} H={H} d={d} {news} behind {olds}", flush=True)
    g = torch.Generator().manual_seed(d + sum(news))
    lengths, starts, T = [a + b for a, b in zip(news, olds)], starts_of(news), sum(news)
    pages = sum(-(-n // PAGE) for n in lengths) + 2
    table = tables(lengths, pages, 3)
    # rows as slices of a wider projection; a token of zeros, sizes that differ by orders
    wide = torch.randn(T, 2 * H * d + 8 * H, generator=g) * torch.exp(3 * torch.randn(T, 1, generator=g))
    wide[T // 2] = 0
    wide = wide.to(dtype)
    key, value = wide[:, :H * d].unflatten(1, (H, d)), wide[:, H * d:2 * H * d].unflatten(1, (H, d))
    want = R.Cache(pages, H, d, seed=T)
    # kept tokens: finite codes
    for c in (want.k, want.v):
        u = c.view(torch.uint8)
        u[(u & 0x7F) == 0x7F] = 0x42
    got = vdn_fp8.KvCache(*want.tensors(device))
    R.append(want, key, value, table, lengths, starts)
    wd = wide.to(device)
    uniform = len(set(news)) == 1
    vdn_fp8.kv_append(wd[:, :H * d].unflatten(1, (H, d)), wd[:, H * d:2 * H * d].unflatten(1, (H, d)), got, i32(table, device), i32(lengths, device),
                      q_start=None if uniform else i32(starts, device))
    torch.cuda.synchronize()
    same_cache(got, want)


def test_append_values_at_the_edges(device):
    """Infinities, NaN, the largest and smallest magnitudes, amax at a power of two times 448, zeros."""
    d = 64
    rows = [torch.zeros(d), torch.full((d,), 448.0), torch.full((d,), 450.0), torch.full((d,), 1e-38), torch.full((d,), 3e38),
            torch.full((d,), 2.0 ** -94), torch.full((d,), 448.0 * 2.0 ** -100)]
    rows += [torch.full((d,), 1.0) for _ in range(3)]
    rows[7][3], rows[8][5], rows[9][7] = float("inf"), float("-inf"), float("nan")
    x = torch.stack(rows)[:, None].float()
    for dtype in (F32, BF16):
        xs = x.to(dtype)
        lengths, starts = [1] * len(rows), list(range(len(rows) + 1))
        table = tables(lengths, len(rows) + 1, 5)
        want = R.Cache(len(rows) + 1, 1, d, seed=1)
        got = vdn_fp8.KvCache(*want.tensors(device))
        R.append(want, xs, xs, table, lengths, starts)
        vdn_fp8.kv_append(xs.to(device), xs.to(device), got, i32(table, device), i32(lengths, device))
        torch.cuda.synchronize()
        same_cache(got, want)


def test_append_leaves_out_what_has_no_place(device):
    """Positions below 0 and beyond the table, absent pages, rows behind the last sequence; no k_mean."""
    H, d, pages = 2, 128, 6
    g = torch.Generator().manual_seed(0)
    news, lengths = [10, 70, 40, 5], [4, 200, 64, 2]     # the first shorter than its rows, the second beyond its table
    starts = starts_of(news)
    table = [[0, 1], [2, 99], [-1, 3], [4, 5]]
    key, value = torch.randn(starts[-1] + 9, H, d, generator=g).to(BF16), torch.randn(starts[-1] + 9, H, d, generator=g).to(BF16)
    want = R.Cache(pages, H, d, seed=9)
    got = vdn_fp8.KvCache(*want.tensors(device))
    R.append(want, key, value, table, lengths, starts)
    kept = got.k_mean.clone()
    vdn_fp8.kv_append(key.to(device), value.to(device), got._replace(k_mean=None), i32(table, device), i32(lengths, device), q_start=i32(starts, device))
    torch.cuda.synchronize()
    assert torch.equal(kept, got.k_mean)
    want.mean = kept.cpu()
    same_cache(got, want)


def test_append_twice_is_append_once(device):
    """Storing the same tokens again (a replayed step) changes nothing."""
    H, d = 2, 128
    g = torch.Generator().manual_seed(1)
    key, value = (torch.randn(3, H, d, generator=g).to(BF16).to(device) * 20 for _ in range(2))
    table, lengths = i32([[2, 0]], device), i32([67], device)
    got = vdn_fp8.KvCache(*R.Cache(3, H, d, seed=2).tensors(device))
    got.k.view(torch.uint8).bitwise_and_(0x3F), got.v.view(torch.uint8).bitwise_and_(0x3F)
    vdn_fp8.kv_append(key, value, got, table, lengths)
    once = [t.clone() for t in got]
    vdn_fp8.kv_append(key, value, got, table, lengths)
    for a, b in zip(once, got):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("d,Hq,H,R_dim,table_dtype", [(64, 3, 3, 64, F32), (128, 40, 8, 128, F32), (128, 5, 1, 64, BF16),
                                                     (256, 6, 2, 256, F32), (128, 9, 3, 0, None), (256, 130, 2, 128, BF16)])
@pytest.mark.parametrize("news,olds", [([1, 1, 1], [0, 63, 200]), ([70], [30]), ([5, 66, 1], [0, 0, 64])])
def test_prep_append_has_the_bits_of_its_parts(device, d, Hq, H, R_dim, table_dtype, news, olds):
    print(f"prep append d={d} {Hq}/{H} R={R_dim} {news}", flush=True)
    T, g = sum(news), torch.Generator().manual_seed(d + Hq)
    qkv = torch.randn(T, (Hq + 2 * H) * d, generator=g).to(BF16).to(device)
    q, k, v = (t.unflatten(1, (-1, d)) for t in qkv.split((Hq * d, H * d, H * d), 1))
    norm_q = ((1 + 0.1 * torch.randn(d, generator=g)).to(BF16).to(device), 1e-6)
    norm_k = (None, 1e-5)
    cos = sin = None
    if R_dim:
        a = 6.28 * torch.rand(T, R_dim // 2, generator=g)
        cos, sin = (torch.cat([f(a), f(a)], 1).to(table_dtype).to(device) for f in (torch.cos, torch.sin))
    lengths = [a + b for a, b in zip(news, olds)]
    pages = sum(-(-n // PAGE) for n in lengths) + 1
    table, start = i32(tables(lengths, pages, 7), device), None if len(set(news)) == 1 else i32(starts_of(news), device)
    base = R.Cache(pages, H, d, seed=4)
    one, two = vdn_fp8.KvCache(*base.tensors(device)), vdn_fp8.KvCache(*base.tensors(device))
    out = vdn_fp8.qk_prep_append(q, k, v, norm_q, norm_k, one, table, i32(lengths, device), cos=cos, sin=sin, q_start=start)
    for h in range(0, Hq, 16384 // d):   # (as many heads as qk_prep takes)
        part = slice(h, min(Hq, h + 16384 // d))
        assert torch.equal(out[:, part], vdn_fp8.qk_prep(q[:, part].contiguous(), *norm_q, cos, sin))
    vdn_fp8.kv_append(vdn_fp8.qk_prep(k, *norm_k, cos, sin), v, two, table, i32(lengths, device), q_start=start)
    for a, b in zip(one, two):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


# -- attention -------------------------------------------------------------------------------

def attention_case(device, dtype, Hq, H, d, news, lengths, causal, seed=0, ragged=None, scale=None, hole=None, lse=True, max_query=None,
                   blocks=None, block=None, cache=None, table=None, q=None, extra=1):
    g = torch.Generator().manual_seed(seed + d + Hq)
    starts, T = starts_of(news), sum(news)
    if cache is None:
        pages = sum(-(-n // PAGE) for n in lengths) + 2
        table = tables(lengths, pages, seed, extra=extra, hole=hole)
        cache = R.Cache(pages, H, d, seed=seed)
        key, value = torch.randn(sum(lengths), H, d, generator=g).to(BF16), torch.randn(sum(lengths), H, d, generator=g).to(BF16)
        value[:, :, ::7] *= 30
        R.append(cache, key, value, table, lengths, starts_of(lengths))
    if q is None:
        q = (1.5 * torch.randn(T, Hq, d, generator=g)).to(dtype)
    ragged = len(set(news)) != 1 if ragged is None else ragged
    scale_ = d ** -0.5 if scale is None else scale
    out, z, tol, tol_z = R.attend(cache, q, table, lengths, starts, scale_, causal, blocks, block, ragged)
    kc = vdn_fp8.KvCache(*cache.tensors(device))
    got = vdn_fp8.kv_attention(q.to(device), kc, i32(table, device), i32(lengths, device), scale=scale, causal=causal,
                               q_start=i32(starts, device) if ragged else None, max_query=max_query, return_lse=lse,
                               blocks=None if blocks is None else torch.as_tensor(blocks, dtype=torch.int32, device=device), query_block=block)
    torch.cuda.synchronize()
    got, got_z = got if lse else (got, None)
    assert got.dtype == dtype and got.shape == q.shape
    near(got, out, tol, dtype)
    if lse:
        got_z = got_z.double().cpu()
        assert torch.equal(got_z.isinf(), z.isinf())
        live = z.isfinite()
        assert bool(((got_z - z).abs() <= tol_z)[live].all()), float((got_z - z).abs()[live].max())
    return got


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("Hq,H,news,lengths", [
    (1, 1, [1], [1]), (5, 1, [1], [64]), (8, 2, [1, 1, 1], [65, 1, 500]), (40, 1, [1], [130]),        # one token
    (6, 2, [3, 3], [3, 200]), (1, 1, [31], [700]),                                                    # a few
    (2, 2, [129], [129]), (3, 1, [50], [391]), (1, 1, [300], [1000]), (4, 2, [7, 140, 64, 1], [7, 150, 300, 5]),
])
@pytest.mark.parametrize("causal", [False, True])
def test_attention(device, d, dtype, Hq, H, news, lengths, causal):
    print(f"attention {dtype} {Hq}/{H} d={d} {news} of {lengths} causal={causal}", flush=True)
    attention_case(device, dtype, Hq, H, d, news, lengths, causal, seed=len(lengths) + sum(news))


@pytest.mark.parametrize("news", [[1, 1, 1, 1], [40, 40, 40, 40], [3, 0, 200, 0]])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_rows_without_keys(device, news, causal):
    """Empty sequences, sequences shorter than their rows, a page that is not there."""
    lengths = [0, 2, 230, 0]
    print(f"rows without keys {news} causal={causal}", flush=True)
    got = attention_case(device, BF16, 4, 2, 128, news, lengths, causal, seed=3, hole=(2, 1, 1 << 20))
    assert not bool(got[:news[0]].any())


def test_attention_absent_pages_only(device):
    attention_case(device, BF16, 2, 1, 128, [1], [64], True, seed=5, hole=(0, 0, -7))
    attention_case(device, BF16, 2, 1, 128, [130], [130], False, seed=5, hole=(0, 0, -1))


@pytest.mark.parametrize("form", ["step", "rows"])
def test_attention_of_a_pool_without_pages(device, form):
    n = 1 if form == "step" else 70
    kc = vdn_fp8.KvCache.empty(0, 2, 128, device)
    table = i32([[0, 3]], device)
    for blocks, block in ((None, None), (i32([[[0], [1]]], device).expand(1, 2, 1), 128 if n > 1 else 1)):
        out = vdn_fp8.kv_attention(torch.randn(n, 2, 128, device=device).to(BF16), kc, table, i32([90], device), blocks=blocks, query_block=block)
        assert not bool(out.any())
    assert vdn_fp8.kv_attention(torch.zeros(0, 2, 128, device=device, dtype=BF16), kc, table, i32([90], device)).shape == (0, 2, 128)


@pytest.mark.parametrize("news,lengths", [([1], [200]), ([100], [200]), ([200], [200])])
def test_nan_reaches_the_rows_that_attend_to_it(device, news, lengths):
    """NaN and infinities among the stored keys and values, some behind a causal row's last key and
    some behind the sequence; a NaN query."""
    H, d = 2, 128
    g = torch.Generator().manual_seed(11)
    key, value = torch.randn(200, H, d, generator=g).to(BF16), torch.randn(200, H, d, generator=g).to(BF16)
    key[150, 0, 3] = float("nan")
    value[180, 1, 5], value[130, 0, 9], value[199, 0, 0] = float("nan"), float("inf"), float("nan")
    cache, table = R.Cache(6, H, d, seed=1), [[4, 0, 2, 5]]
    R.append(cache, key, value, table, [200], [0, 200])
    q = torch.randn(sum(news), 4, d, generator=g).to(BF16)
    if news[0] > 1:
        q[3, 1, 7] = float("nan")
    for causal in (True, False):
        print(f"nan {news} causal={causal}", flush=True)
        attention_case(device, BF16, 4, H, d, news, lengths, causal, cache=cache, table=table, q=q, lse=False)


def test_scales_far_apart(device):
    """Pages whose scales differ by orders, keys of zeros, values of zeros, and large scores."""
    H, d, n = 1, 128, 320
    g = torch.Generator().manual_seed(13)
    key, value = torch.randn(n, H, d, generator=g), torch.randn(n, H, d, generator=g)
    value[:64] *= 1e-6
    value[64:128] *= 1e5
    value[128:192] = 0
    key[192:256] *= 8
    key[256:] = 0
    cache, table = R.Cache(6, H, d, seed=2), [[3, 1, 0, 5, 2]]
    R.append(cache, key.to(BF16), value.to(BF16), table, [n], [0, n])
    for rows in (1, 150):
        for scale in (0.02, 3.0):
            print(f"scales rows={rows} scale={scale}", flush=True)
            q = torch.randn(rows, 2, d, generator=g).to(BF16)
            attention_case(device, BF16, 2, H, d, [rows], [n], True, cache=cache, table=table, q=q, scale=scale)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attention_splits_long_caches(device, dtype):
    """Few rows of long caches: the key axis is split and joined; a table far wider than the sequences."""
    for news, lengths, extra in (([1, 1], [5000, 321], 0), ([90], [4500], 3), ([1], [100], 500)):
        print(f"splits {dtype} {news} {lengths} +{extra}", flush=True)
        attention_case(device, dtype, 4, 2, 128, news, lengths, True, seed=17, extra=extra)


def test_rows_of_a_strided_view_and_other_orders(device):
    """A query that is a column slice, misaligned rows, a padded table, an expanded table."""
    H, d, n = 2, 64, 100
    cache, g = R.Cache(4, H, d, seed=3), torch.Generator().manual_seed(4)
    table = [[2, 0]]
    R.append(cache, torch.randn(n, H, d, generator=g).to(BF16), torch.randn(n, H, d, generator=g).to(BF16), table, [n], [0, n])
    kc = vdn_fp8.KvCache(*cache.tensors(device))
    wide = torch.randn(2, 3 * H * d, generator=g).to(BF16).to(device)
    q = wide[:, H * d:2 * H * d].unflatten(1, (H, d))
    lengths = i32([n, n], device)
    t = i32(table, device).expand(2, 2)
    want = vdn_fp8.kv_attention(q.contiguous(), kc, t.contiguous(), lengths)
    assert torch.equal(want, vdn_fp8.kv_attention(q, kc, t, lengths))
    padded = torch.full((2, 9), 77, dtype=torch.int32, device=device)
    padded[:, :2] = t
    assert torch.equal(want, vdn_fp8.kv_attention(q, kc, padded[:, :2], lengths))
    odd = torch.zeros(2 * (H * d + 3) + 1, dtype=BF16, device=device)[1:].as_strided((2, H, d), (H * d + 3, d, 1))
    odd.copy_(q)
    assert torch.equal(want, vdn_fp8.kv_attention(odd, kc, padded[:, :2], lengths))
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(want, vdn_fp8.kv_attention(heads_first, kc, padded[:, :2], lengths))


@pytest.mark.parametrize("n", [1, 70])
def test_rows_behind_the_last_sequence(device, n):
    """A padded batch: rows that q_start leaves out are zeros, -inf in the log-sum-exp, -1 in the lists."""
    H, d = 2, 128
    cache, g = R.Cache(8, H, d, seed=3), torch.Generator().manual_seed(4)
    lengths, table = [100, 130], [[2, 0, 1], [4, 5, 6]]
    R.append(cache, torch.randn(230, H, d, generator=g).to(BF16), torch.randn(230, H, d, generator=g).to(BF16), table, lengths, [0, 100, 230])
    kc = vdn_fp8.KvCache(*cache.tensors(device))
    q = torch.randn(2 * n + 300, 4, d, generator=g).to(BF16).to(device)
    start = i32([0, n, 2 * n], device)
    args = (kc, i32(table, device), i32(lengths, device))
    for most in (None, n):
        out, z = vdn_fp8.kv_attention(q, *args, q_start=start, max_query=most, return_lse=True)
        want, wz = vdn_fp8.kv_attention(q[:2 * n].contiguous(), *args, return_lse=True)
        tol = 2.0 ** -6 * want.float().abs().max()
        assert float((out[:2 * n].float() - want.float()).abs().max()) <= tol and torch.allclose(z[:2 * n], wz, atol=1e-3)
        assert not bool(out[2 * n:].any()) and bool((z[2 * n:] == -float("inf")).all())
    for block in (1, 64):
        lists = vdn_fp8.kv_select(q, *args, 2, query_block=block, q_start=start)
        used = set()
        for b in range(2):
            base = b * n if block == 1 else b * n // block + b
            used |= set(range(base, base + -(-n // block)))
        assert all((int(lists[r].max()) >= 0) == (r in used) for r in range(lists.shape[0]))
        out = vdn_fp8.kv_attention(q, *args, q_start=start, max_query=n, blocks=lists, query_block=block)
        assert bool(out[:2 * n].any()) and not bool(out[2 * n:].any())


# -- chosen pages ----------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d,Hq,H,news,lengths,block,top,first,last", [
    (128, 4, 4, [1, 1], [900, 64], 1, 5, 1, 1), (64, 10, 2, [300], [2000], 128, 8, 1, 1), (256, 2, 2, [129, 129], [700, 130], 128, 3, 0, 0),
    (128, 8, 1, [40, 3, 17], [640, 3, 500], 16, 4, 2, 1), (128, 2, 1, [2, 0, 5], [300, 0, 90], 1, 2, 0, 2), (128, 1, 1, [1], [3000], 1, 100, 1, 1),
])
@pytest.mark.parametrize("causal", [False, True])
def test_select(device, dtype, d, Hq, H, news, lengths, block, top, first, last, causal):
    print(f"select {dtype} d={d} {Hq}/{H} {news} block={block} top={top} causal={causal}", flush=True)
    g = torch.Generator().manual_seed(d + sum(news))
    starts, ragged = starts_of(news), len(set(news)) != 1
    pages = sum(-(-n // PAGE) for n in lengths) + 2
    table = tables(lengths, pages, 1, hole=(0, 1, -1))
    cache = R.Cache(pages, H, d, seed=6)
    q = torch.randn(sum(news), Hq, d, generator=g).to(dtype)
    want = R.select(cache, q, table, lengths, starts, top, block, first, last, causal, ragged)
    got = vdn_fp8.kv_select(q.to(device), vdn_fp8.KvCache(*cache.tensors(device)), i32(table, device), i32(lengths, device), top, query_block=block,
                            first=first, last=last, causal=causal, q_start=i32(starts, device) if ragged else None)
    torch.cuda.synchronize()
    assert np.array_equal(got.cpu().numpy(), want)


def test_select_ties_and_nan(device):
    """Equal scores go to the lower page, +0 and -0 are equal, NaN comes last; long lists."""
    H, d = 1, 64
    for W, top in ((40, 7), (2500, 300)):
        cache = R.Cache(W, H, d, seed=6)
        g = torch.Generator().manual_seed(W)
        cache.mean.zero_()
        cache.mean[:, 0, 0] = torch.randint(-1, 2, (W,), generator=g).to(BF16)
        cache.mean[::3, 0, 1] = -0.0
        cache.mean[5, 0, 2], cache.mean[6, 0, 0] = float("nan"), float("-inf")
        q = torch.zeros(1, 1, d).to(BF16)
        q[0, 0, 0] = 2.0
        for sign in (1, -1):
            table, lengths = [list(range(W))], [W * PAGE - 3]
            want = R.select(cache, sign * q, table, lengths, [0, 1], top, 1, 0, 0, False)
            got = vdn_fp8.kv_select((sign * q).to(device), vdn_fp8.KvCache(*cache.tensors(device)), i32(table, device), i32(lengths, device), top,
                                    query_block=1, first=0, last=0)
            assert np.array_equal(got.cpu().numpy(), want), (W, sign)


@pytest.mark.parametrize("dtype,d,Hq,H,news,lengths,block", [
    (BF16, 128, 2, 2, [200], [900], 128), (F16, 64, 8, 2, [40, 70], [500, 640], 32), (BF16, 256, 1, 1, [129], [300], 128),
    (BF16, 128, 5, 1, [1, 1, 1], [700, 100, 64], 1), (F16, 128, 40, 1, [2, 1], [400, 90], 1),
])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_over_listed_pages(device, dtype, d, Hq, H, news, lengths, block, causal):
    """Lists with -1, pages outside the sequence, a page twice, and pages that a causal row does not see."""
    print(f"listed {dtype} d={d} {Hq}/{H} {news} block={block} causal={causal}", flush=True)
    ragged = len(set(news)) != 1
    rows = R.listed_rows(starts_of(news), block, ragged)[1]
    rng = np.random.default_rng(d + rows)
    W = max(-(-n // PAGE) for n in lengths)
    blocks = np.sort(np.stack([[rng.permutation(W + 1)[:4] for _ in range(H)] for _ in range(rows)]).astype(np.int32), 2)
    blocks[rng.random(blocks.shape) < 0.15] = -1
    blocks[0, 0, :2] = 0
    blocks[-1, -1] = [1 << 30, -5, W - 1, 7000]
    attention_case(device, dtype, Hq, H, d, news, lengths, causal, seed=23, blocks=blocks, block=block, ragged=ragged, max_query=max(news))


# -- together --------------------------------------------------------------------------------

def test_a_run_of_them(device):
    """A prompt stored and attended to, then steps of one token each, dense and over chosen pages, as a
    causal model uses them: each step against a plain attention of all tokens so far."""
    Hq, H, d, B = 4, 2, 128, 2
    g = torch.Generator().manual_seed(31)
    prompt, steps = [150, 70], 5
    news = prompt
    cache = vdn_fp8.KvCache.empty(9, H, d, device)
    plain = R.Cache(9, H, d, seed=0)
    plain.k, plain.v = cache.k.cpu(), cache.v.cpu()
    plain.ek, plain.ev = (t.cpu().view(torch.uint8).int() - 127 for t in (cache.k_scale, cache.v_scale))
    plain.mean = cache.k_mean.cpu()
    table = [[8, 3, 1, -1], [0, 7, -1, -1]]
    lengths = i32([0, 0], device)
    norm = ((1 + 0.1 * torch.randn(d, generator=g)).to(BF16).to(device), 1e-6)
    pages = i32(table, device)
    for step in range(steps + 1):
        starts, T = starts_of(news), sum(news)
        q, k, v = (torch.randn(T, n, d, generator=g).to(BF16).to(device) for n in (Hq, H, H))
        angle = 6.28 * torch.rand(T, d // 2, generator=g)
        cos, sin = (torch.cat([f(angle), f(angle)], 1).to(device) for f in (torch.cos, torch.sin))
        lengths += i32(news, device)
        start = None if step else i32(starts, device)
        query = vdn_fp8.qk_prep_append(q, k, v, norm, norm, cache, pages, lengths, cos=cos, sin=sin, q_start=start)
        out = vdn_fp8.kv_attention(query, cache, pages, lengths, causal=True, q_start=start)
        n = lengths.tolist()
        R.append(plain, vdn_fp8.qk_prep(k, *norm, cos, sin).cpu(), v.cpu(), table, n, starts)
        want, _, tol, _ = R.attend(plain, query.cpu(), table, n, starts, d ** -0.5, True)
        near(out, want, tol, BF16)
        if step:
            lists = vdn_fp8.kv_select(query, cache, pages, lengths, 2, query_block=1, causal=True)
            assert np.array_equal(lists.cpu().numpy(), R.select(plain, query.cpu(), table, n, starts, 2, 1, 1, 1, True))
            out = vdn_fp8.kv_attention(query, cache, pages, lengths, causal=True, blocks=lists, query_block=1)
            want, _, tol, _ = R.attend(plain, query.cpu(), table, n, starts, d ** -0.5, True, lists.cpu(), 1)
            near(out, want, tol, BF16)
        news = [1] * B
    same_cache(cache, plain)


def test_captured_steps(device):
    """A step captured into two graphs and replayed, with lengths that grow between the replays and eager
    work among them: every replay equals the eager result."""
    Hq, H, d = 8, 2, 128
    g = torch.Generator(device=device).manual_seed(5)
    base = R.Cache(40, H, d, seed=8)
    for c in (base.k, base.v):
        c.view(torch.uint8).bitwise_and_(0x3F)
    caches = [vdn_fp8.KvCache(*base.tensors(device)) for _ in range(2)]
    pages = torch.randperm(40, generator=torch.Generator().manual_seed(1))[:36].to(torch.int32).to(device).view(2, 18)
    lengths = i32([900, 70], device)
    qkv = torch.randn(2, (Hq + 2 * H) * d, device=device, generator=g).to(BF16)
    norm = (None, 1e-6)

    def step(cache, length):
        q, k, v = (t.unflatten(1, (-1, d)) for t in qkv.split((Hq * d, H * d, H * d), 1))
        query = vdn_fp8.qk_prep_append(q, k, v, norm, norm, cache, pages, length)
        lists = vdn_fp8.kv_select(query, cache, pages, length, 4, query_block=1, causal=True)
        return (vdn_fp8.kv_attention(query, cache, pages, length, causal=True),
                vdn_fp8.kv_attention(query, cache, pages, length, causal=True, blocks=lists, query_block=1))

    step(caches[1], lengths.clone())
    caches[1] = vdn_fp8.KvCache(*base.tensors(device))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(caches[0], lengths)
        graphs.append((graph, out))
    eager_lengths = lengths.clone()
    for i in range(6):
        lengths += 1
        eager_lengths += 1
        qkv.copy_(torch.randn(qkv.shape, device=device, generator=g))
        want = step(caches[1], eager_lengths)
        graph, out = graphs[i % 2]
        graph.replay()
        (qkv.float().sum() + i).item()
        for a, b in zip(out, want):
            assert torch.equal(a, b), i
        for a, b in zip(*caches):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), i


def test_calls_on_two_streams(device):
    """Calls that overlap on two streams have workspaces of their own."""
    H, d, n = 2, 128, 3000
    g = torch.Generator(device=device).manual_seed(6)
    kc = vdn_fp8.KvCache.empty(50, H, d, device)
    table, lengths = torch.arange(50, dtype=torch.int32, device=device)[None], i32([n], device)
    vdn_fp8.kv_append(torch.randn(n, H, d, device=device, generator=g).to(BF16), torch.randn(n, H, d, device=device, generator=g).to(BF16), kc, table, lengths)
    qs = [torch.randn(1, 8, d, device=device, generator=g).to(BF16) for _ in range(2)]
    want = [vdn_fp8.kv_attention(q, kc, table, lengths) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(vdn_fp8.kv_attention(qs[i], kc, table, lengths))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_repeats_have_the_same_bits(device):
    H, d, n = 4, 128, 2000
    g = torch.Generator(device=device).manual_seed(7)
    kc = vdn_fp8.KvCache.empty(40, H, d, device)
    table, lengths = torch.randperm(40, generator=torch.Generator().manual_seed(2))[:32].to(torch.int32).to(device)[None], i32([n], device)
    vdn_fp8.kv_append(torch.randn(n, H, d, device=device, generator=g).to(BF16), torch.randn(n, H, d, device=device, generator=g).to(BF16), kc, table, lengths)
    for rows in (1, 300):
        q = torch.randn(rows, 8, d, device=device, generator=g).to(BF16)
        first = vdn_fp8.kv_attention(q, kc, table, lengths, causal=True)
        for _ in range(5):
            assert torch.equal(first, vdn_fp8.kv_attention(q, kc, table, lengths, causal=True))


def test_offsets_beyond_32_bits(device):
    """A pool of more than 2^32 bytes of keys, pages at its end."""
    H, d = 8, 256
    pages = (1 << 32) // (H * 64 * d) + 40
    kc = vdn_fp8.KvCache.empty(pages, H, d, device)
    small = vdn_fp8.KvCache.empty(4, H, d, device)
    g = torch.Generator(device=device).manual_seed(8)
    n = 200
    key, value = (torch.randn(n, H, d, device=device, generator=g).to(BF16) for _ in range(2))
    far, near_ = i32([[pages - 1, pages - 9, pages - 20, pages - 3]], device), i32([[0, 1, 2, 3]], device)
    lengths = i32([n], device)
    for cache, table in ((kc, far), (small, near_)):
        vdn_fp8.kv_append(key, value, cache, table, lengths)
    for rows in (1, 100):
        q = torch.randn(rows, H, d, device=device, generator=g).to(BF16)
        assert torch.equal(vdn_fp8.kv_attention(q, kc, far, lengths, causal=True), vdn_fp8.kv_attention(q, small, near_, lengths, causal=True))
    q = torch.randn(1, H, d, device=device, generator=g).to(BF16)
    assert torch.equal(vdn_fp8.kv_select(q, kc, far, lengths, 2, query_block=1), vdn_fp8.kv_select(q, small, near_, lengths, 2, query_block=1))
