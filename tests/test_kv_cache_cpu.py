"""The 8-bit key/value cache without a GPU: the plain reference's own properties, and every
refusal of the C entry points and of the Python layer."""
import ctypes

import pytest
import torch

import kv_reference as R
import vdn_fp8
import vdn_fp8._lib as L

FAKE = 1 << 20        # never dereferenced: every call below fails its checks first
CACHE = dict(k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, k_mean=FAKE, pages=4, heads=2, head_dim=128)
BATCH = dict(page_table=FAKE, ldtable=3, max_pages=3, lengths=FAKE, q_start=None, batch=2, tokens=4)


def cache(**kw):
    return L.KvCacheStruct(**{**CACHE, **kw})


def batch(**kw):
    return L.KvBatchStruct(**{**BATCH, **kw})


def append(c=None, b=None, key=FAKE, ldk=256, value=FAKE, ldv=256, dtype=0):
    return L.load().vdn_fp8_kv_append(c or cache(), b or batch(), key, ldk, value, ldv, dtype, None)


def prep(q=FAKE, heads=4, ldq=512, eps=1e-6, cos=FAKE, sin=FAKE, R=128, ldcs=128, out=FAKE, ldo=512, **kw):
    return L.load().vdn_fp8_qk_prep_append(cache(), batch(), q, heads, ldq, FAKE, 256, FAKE, 256, kw.get("weight"), eps, None, 1e-6, cos, sin,
                                           R, ldcs, 0, out, ldo, None)


def attention(c=None, b=None, q=FAKE, dtype=0, heads=4, ldq=512, most=0, scale=1.0, blocks=None, top=0, block=0, out=FAKE, ws=None, n=0):
    return L.load().vdn_fp8_kv_attention(c or cache(), b or batch(), q, dtype, heads, ldq, most, scale, 0, blocks, top, block, out, None, ws, n, None)


def select(c=None, b=None, q=FAKE, dtype=0, heads=4, ldq=512, top=4, first=1, last=1, block=64, out=FAKE, ws=FAKE, n=1 << 40):
    return L.load().vdn_fp8_kv_select(c or cache(), b or batch(), q, dtype, heads, ldq, 0, top, first, last, block, out, ws, n, None)


@pytest.mark.parametrize("call,needle", [
    (lambda: append(cache(head_dim=96)), "head dim"),
    (lambda: append(cache(heads=0)), "heads"),
    (lambda: append(cache(pages=-1)), "pages"),
    (lambda: append(cache(k=None)), "null cache"),
    (lambda: append(cache(v=FAKE + 8)), "aligned"),
    (lambda: append(b=batch(tokens=-1)), "tokens"),
    (lambda: append(b=batch(tokens=5)), "divide"),
    (lambda: append(b=batch(batch=0)), "empty batch"),
    (lambda: append(b=batch(lengths=None)), "null page table or lengths"),
    (lambda: append(b=batch(page_table=None)), "null page table or lengths"),
    (lambda: append(b=batch(ldtable=-1)), "ldtable"),
    (lambda: append(b=batch(max_pages=-1)), "max_pages"),
    (lambda: append(b=batch(lengths=FAKE + 2)), "4-byte"),
    (lambda: append(key=None), "null pointer"),
    (lambda: append(ldk=248), "ldk"),
    (lambda: append(ldv=260), "multiples of 8"),
    (lambda: append(value=FAKE + 8), "aligned"),
    (lambda: append(dtype=3), "dtype"),
    (lambda: prep(q=None), "null pointer"),
    (lambda: prep(heads=0), "query heads"),
    (lambda: prep(R=72), "multiple of 16"),
    (lambda: prep(R=144), "multiple of 16"),
    (lambda: prep(cos=None), "tables"),
    (lambda: prep(ldcs=64), "tables"),
    (lambda: prep(ldq=504), "ldq"),
    (lambda: prep(eps=-1.0), "eps"),
    (lambda: prep(eps=float("nan")), "eps"),
    (lambda: prep(weight=FAKE + 4), "misaligned"),
    (lambda: prep(ldcs=130), "misaligned"),
    (lambda: attention(dtype=2), "dtype"),
    (lambda: attention(heads=3), "query heads"),
    (lambda: attention(q=None), "null pointer"),
    (lambda: attention(out=None), "null pointer"),
    (lambda: attention(ldq=256), "ldq"),
    (lambda: attention(out=FAKE + 2), "misaligned"),
    (lambda: attention(scale=0.0), "scale"),
    (lambda: attention(scale=float("inf")), "scale"),
    (lambda: attention(scale=3e38), "scale"),   # (times log2(e) it is beyond binary32)
    (lambda: attention(scale=float("nan")), "scale"),
    (lambda: attention(most=-1), "max_query"),
    (lambda: attention(b=batch(tokens=1 << 30)), "2^30"),
    (lambda: attention(blocks=FAKE, top=0, block=1), "top"),
    (lambda: attention(blocks=FAKE, top=4, block=0), "query_block"),
    (lambda: attention(blocks=FAKE, top=4, block=100), "multiple of 128"),
    (lambda: select(cache(k_mean=None)), "k_mean"),
    (lambda: select(heads=5), "query heads"),
    (lambda: select(dtype=2), "dtype"),
    (lambda: select(block=65), "multiple of 128"),
    (lambda: select(top=1), "first + last"),
    (lambda: select(first=-1), "first and last"),
    (lambda: select(out=None), "null pointer"),
    (lambda: select(ws=None), "workspace"),
    (lambda: select(n=16), "workspace"),
    (lambda: select(q=FAKE + 4), "misaligned"),
    (lambda: select(b=batch(batch=1 << 17, tokens=1 << 17)), "batch"),
])
def test_contract_violations_are_einval(call, needle):
    assert call() == L.EINVAL
    assert needle in L.load().vdn_fp8_last_error().decode()


def test_null_structs_are_einval():
    assert L.load().vdn_fp8_kv_append(None, batch(), FAKE, 256, FAKE, 256, 0, None) == L.EINVAL
    assert L.load().vdn_fp8_kv_append(cache(), None, FAKE, 256, FAKE, 256, 0, None) == L.EINVAL
    assert L.load().vdn_fp8_kv_attention_workspace_size(cache(), batch(), 4, 0, 0, 0, None) == L.EINVAL
    assert L.load().vdn_fp8_kv_select_workspace_size(cache(), batch(), 4, 1, None) == L.EINVAL


def test_empty_calls_are_no_ops():
    none = batch(tokens=0)
    assert append(b=none, key=None, value=None) == L.OK
    assert attention(b=none, q=None, out=None) == L.OK
    assert select(b=none, q=None, out=None) == L.OK
    n = ctypes.c_int64(7)
    assert L.load().vdn_fp8_kv_attention_workspace_size(cache(), none, 4, 0, 0, 0, ctypes.byref(n)) == L.OK and n.value == 0


def test_select_workspace_holds_scores_and_sums():
    n = ctypes.c_int64(0)
    assert L.load().vdn_fp8_kv_select_workspace_size(cache(), batch(), 4, 1, ctypes.byref(n)) == L.OK
    assert n.value == 4 * 2 * (3 * 8 + 128 * 4)


def test_select_counts_rows_as_attention_does():
    n, many = ctypes.c_int64(0), batch(batch=1, tokens=1 << 28)
    for rows, ok in (((1 << 28) - 1, L.OK), (1 << 28, L.EINVAL)):
        assert L.load().vdn_fp8_kv_select_workspace_size(cache(), batch(batch=1, tokens=rows), 4, 1 << 20, ctypes.byref(n)) == ok
    assert "2^30" in L.load().vdn_fp8_last_error().decode()
    assert attention(b=many) == L.EINVAL and "2^30" in L.load().vdn_fp8_last_error().decode()


def pool(**kw):
    c = vdn_fp8.KvCache.empty(3, 2, 64, "cpu")
    return c._replace(**kw)


def test_python_layer_refuses():
    x, table, lengths = torch.zeros(2, 2, 64, dtype=torch.bfloat16), torch.zeros(1, 3, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: vdn_fp8.kv_append(x, x, pool(), table, lengths), lambda: vdn_fp8.kv_attention(x, pool(), table, lengths),
                 lambda: vdn_fp8.kv_select(x, pool(), table, lengths, 2, query_block=1),
                 lambda: vdn_fp8.qk_prep_append(x, x, x, (None, 1e-6), (None, 1e-6), pool(), table, lengths)):
        with pytest.raises(ValueError, match="GPU"):
            call()
    with pytest.raises(ValueError, match="64, 128 or 256"):
        vdn_fp8.KvCache.empty(3, 2, 80, "cpu")


@pytest.mark.parametrize("change,needle", [
    (dict(k=torch.zeros(3, 2, 32, 64).to(R.E4M3)), "cache.k"),
    (dict(v=torch.zeros(3, 2, 32, 64).to(R.E4M3)), "cache.v"),
    (dict(k_scale=torch.zeros(3, 2)), "k_scale"),
    (dict(v_scale=torch.zeros(3, 1).to(R.E8M0)), "k_scale"),
    (dict(k_mean=torch.zeros(3, 2, 64)), "k_mean"),
    (dict(k=torch.zeros(3, 64, 2, 64).to(R.E4M3).transpose(1, 2)), "contiguous"),
])
def test_cache_checks(change, needle):
    from vdn_fp8 import kv_cache as K
    with pytest.raises(ValueError, match=needle):
        K._cache(pool(**change), torch.device("cpu"))


def test_the_branch_refuses_before_it_stores():
    """What a later part of `cached_attention` would refuse is refused before anything is stored."""
    from vdn_fp8.softmax_attention import cached_attention
    x, table, lengths = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(1, 3, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    to = [torch.nn.Linear(8, n, dtype=torch.bfloat16) for n in (128, 128, 128)]
    norm = torch.nn.RMSNorm(64, eps=1e-6, dtype=torch.bfloat16)
    odd = torch.nn.Linear(8, 192, dtype=torch.bfloat16)
    for args, more, needle in (((*to, norm, norm, pool()), dict(top=2), "query_block"), ((*to, norm, norm, pool()), dict(query_block=64), "query_block"),
                               ((*to, norm, norm, pool(k_mean=None)), dict(top=2, query_block=64), "k_mean"),
                               ((odd, *to[1:], norm, norm, pool()), {}, "query heads"), ((*to, norm, norm, pool()), {}, "GPU")):
        with pytest.raises(ValueError, match=needle):
            cached_attention(x, *args, table, lengths, **more)


@pytest.mark.parametrize("more,needle", [
    (dict(top=1, query_block=128), "top must be"), (dict(top=0, query_block=128), "top must be"), (dict(top=4, query_block=128, first=3, last=2), "top must be"),
    (dict(top=4, query_block=128, first=-1), "top must be"), (dict(top=4, query_block=65), "query_block must be"), (dict(top=4, query_block=0), "query_block must be"),
    (dict(top=4, query_block=-128), "query_block must be"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(scale=3e38), "scale"), (dict(max_query=-1), "max_query"),
])
def test_the_branch_stores_nothing_when_it_refuses(monkeypatch, more, needle):
    from vdn_fp8 import kv_cache as K
    from vdn_fp8.softmax_attention import cached_attention
    stored = []
    monkeypatch.setattr(K, "qk_prep_append", lambda query, *a, **kw: stored.append(query) or query)
    x, table, lengths = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(1, 3, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    to = [torch.nn.Linear(8, 128, dtype=torch.bfloat16) for _ in range(3)]
    norm = torch.nn.RMSNorm(64, eps=1e-6, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match=needle):
        cached_attention(x, *to, norm, norm, pool(), table, lengths, **more)
    assert not stored


def test_batch_checks():
    from vdn_fp8 import kv_cache as K
    cpu, table, lengths = torch.device("cpu"), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    start = torch.zeros(3, dtype=torch.int32)
    assert K._batch(table, lengths, start, 5, 3, cpu).tokens == 5
    for args, needle in (((table.long(), lengths, None, 4), "page_table"), ((table, lengths.float(), None, 4), "lengths"),
                         ((table, lengths[:1], None, 4), "lengths"), ((table, lengths, start[:2], 4), "q_start"),
                         ((table, lengths, None, 5), "divide"), ((table[:0], lengths[:0], None, 5), "empty"),
                         ((table.t().contiguous().t(), lengths, None, 4), "stride")):
        with pytest.raises(ValueError, match=needle):
            K._batch(*args, 3, cpu)
    before = vdn_fp8.set_index_checks(True)
    try:
        with pytest.raises(IndexError, match="lengths"):
            K._batch(table, lengths + 193, None, 4, 3, cpu)
        with pytest.raises(IndexError, match="q_start"):
            K._batch(table, lengths, start + 5, 4, 3, cpu)
    finally:
        vdn_fp8.set_index_checks(before)


def test_reference_exponent():
    for amax, e in ((448.0, 0), (448.1, 1), (224.0, -1), (225.0, 0), (1.0, -8), (0.0, -100), (1e-38, -100), (3e38, 120)):
        got = R.exponent(torch.tensor([amax, -amax, float("nan"), float("inf")]))
        assert got == e, (amax, got, e)
        if amax and e > -100:
            assert amax * 2.0 ** -e <= 448 and (amax * 2.0 ** -(e - 1) > 448)


def test_reference_attention_is_a_softmax():
    """The plain attention against torch's softmax on dense keys, and its bound's size."""
    g = torch.Generator().manual_seed(0)
    H, d, n = 2, 64, 130
    key, value = torch.randn(n, H, d, generator=g).to(torch.bfloat16), torch.randn(n, H, d, generator=g).to(torch.bfloat16)
    c, table = R.Cache(4, H, d), [[3, 0, 2]]
    R.append(c, key, value, table, [n], [0, n])
    q = torch.randn(n, 4, d, generator=g).to(torch.bfloat16)
    out, lse, tol, tol_lse = R.attend(c, q, table, [n], [0, n], 0.125, True)
    k = torch.cat([R.decode(c.k, c.ek)[p] for p in table[0]], 1)[:, :n].repeat_interleave(2, 0)
    v = torch.cat([R.decode(c.v, c.ev).transpose(2, 3)[p] for p in table[0]], 1)[:, :n].repeat_interleave(2, 0)
    s = (q.double().transpose(0, 1) @ k.transpose(1, 2)) * 0.125
    s = s.masked_fill(~torch.tril(torch.ones(n, n, dtype=torch.bool)), float("-inf"))
    assert torch.allclose(out, (s.softmax(-1) @ v).transpose(0, 1)) and torch.allclose(lse, s.logsumexp(-1).T)
    assert float(tol.max()) < 0.01 and float(tol_lse.max()) < 1e-3


def test_reference_append_by_pieces():
    """Tokens stored one by one differ from the same tokens stored at once by their page's least steps at
    most: half of 2^-9 at each of the scales that the page went through."""
    g = torch.Generator().manual_seed(2)
    n, d = 64, 64
    x = torch.randn(n, 1, d, generator=g) * torch.exp(2 * torch.randn(n, 1, 1, generator=g))
    once, steps = R.Cache(1, 1, d), R.Cache(1, 1, d)
    R.append(once, x, x, [[0]], [n], [0, n])
    for i in range(n):
        R.append(steps, x[i:i + 1], x[i:i + 1], [[0]], [i + 1], [0, 1])
    assert int(once.ek[0, 0]) == int(steps.ek[0, 0])
    a, b = (R.decode(c.k, c.ek) for c in (once, steps))
    assert float((a - b).abs().max()) <= 2 * 2.0 ** -10 * 2.0 ** int(once.ek[0, 0])
