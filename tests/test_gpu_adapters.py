"""Low-rank adapters of many requests (`adapter_add`, `Fp8Linear.forward(adapters=...)`) against the formula in 64 bits.

Bound. With u = 2^-24 (binary32's half step): h[r] is a sum of K exact products in some order, and of up to 32 parts: off by
(K + 32) u' of sum |x a|, u' = 2 u, should the matrix cores truncate. It enters the second product off by 2^-17 of itself (bf16; float16:
2^-22 of the token's largest, and 2^-24 of it below float16's normal range: 2^-21 together), whose up to 128 * 2 products add 260 u'
of sum |h b|. Scale and sum round once each in binary32, the result once to its type."""
import pytest
import torch

import vdn_fp8
from vdn_fp8 import Adapters, adapter_add

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
U = 2.0 ** -23


def bank(device, L, R, K, N, dtype, seed):
    g = torch.Generator(device).manual_seed(seed)
    a = (torch.randn(L, R, K, device=device, generator=g) * K ** -0.5).to(dtype)
    b = (torch.randn(L, N, R, device=device, generator=g) * R ** -0.5).to(dtype)
    return Adapters(a, b, 0.3 + torch.rand(L, device=device, generator=g))


def rows(device, T, K, N, dtype, seed):
    g = torch.Generator(device).manual_seed(seed)
    return torch.randn(T, K, device=device, generator=g).to(dtype), torch.randn(T, N, device=device, generator=g).to(dtype)


def formula(x, base, ad, index):
    """(result, bound before its own rounding) in 64 bits."""
    want, bound = base.double(), torch.zeros(base.shape, dtype=torch.float64, device=base.device)
    K, R = x.shape[1], ad.a.shape[1]
    for i in range(ad.a.shape[0]):
        mine = (index == i).nonzero()[:, 0]
        if not len(mine):
            continue
        xi, a, b, s = x[mine].double(), ad.a[i].double(), ad.b[i].double(), float(ad.scale[i])
        h, size = xi @ a.T, xi.abs() @ a.abs().T
        eh = (K + 32) * U * size
        eh = eh + (2.0 ** -17 * h.abs() if x.dtype == BF16 else 2.0 ** -21 * h.abs().amax(1, keepdim=True))
        delta = h @ b.T
        want[mine] += s * delta
        bound[mine] = abs(s) * (eh @ b.abs().T + 260 * U * (h.abs() + eh) @ b.abs().T) + U * (abs(s) * delta.abs() + base[mine].double().abs())
    return want, bound


def check(got, x, base, ad, index):
    want, bound = formula(x, base, ad, index)
    assert got.dtype == base.dtype and got.shape == base.shape
    room = bound + torch.finfo(x.dtype).eps / 2 * (want.abs() + bound) + (2.0 ** -25 if x.dtype == F16 else 0.0)
    bad = (got.double() - want).abs() > room
    if x.dtype == F16:
        # float16 ends at 65504, and half a step beyond it, 65520, is where a value rounds to infinity
        bad &= ~(got.isinf() & (want.abs() + bound >= 65520) & (got.sign() == want.sign()))
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), float((got.double() - want).abs().max()))
    none = (index < 0) | (index >= ad.a.shape[0])
    assert torch.equal(got[none].view(torch.int16), base[none].view(torch.int16))


def choose(device, T, L, form, seed):
    g = torch.Generator().manual_seed(seed)
    if form == "one":
        i = torch.full((T,), min(1, L - 1))
    elif form == "random":
        i = torch.randint(-1, L, (T,), generator=g)
    elif form == "each":
        i = torch.arange(T) % L
    else:   # runs of a request's tokens, of any lengths
        cuts = torch.cat([torch.zeros(1).long(), torch.randint(0, T + 1, (6,), generator=g).sort().values, torch.tensor([T])])
        i = torch.cat([torch.full((int(b - a),), int(torch.randint(-1, L, (1,), generator=g))) for a, b in zip(cuts[:-1], cuts[1:])])
    return i.int().to(device)


@pytest.mark.parametrize("T", [1, 2, 15, 17, 63, 64, 65, 129, 500, 1024, 1025, 1217, 2100])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("form", ["one", "random", "runs", "each"])
def test_tokens_and_orders(device, T, dtype, form):
    L, R, K, N = 7, 32, 328, 296
    print(f"adapters {T} {dtype} {form}", flush=True)
    x, base = rows(device, T, K, N, dtype, T)
    ad = bank(device, L, R, K, N, dtype, T + 1)
    index = choose(device, T, L, form, T + 2)
    got = adapter_add(x, base, ad, index)
    check(got, x, base, ad, index)
    # in place, and again: the same bits
    mine = base.clone()
    assert adapter_add(x, mine, ad, index, out=mine) is mine
    assert torch.equal(mine, got)


@pytest.mark.parametrize("R", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("K,N", [(8, 8), (16, 40), (72, 264), (1032, 1040), (4104, 104), (5120, 2056)])
@pytest.mark.parametrize("T", [5, 1100])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_ranks_and_widths(device, R, K, N, T, dtype):
    print(f"adapters R={R} K={K} N={N} T={T} {dtype}", flush=True)
    x, base = rows(device, T, K, N, dtype, R + K)
    ad = bank(device, 3, R, K, N, dtype, R + N)
    index = choose(device, T, 3, "random" if T < 100 else "runs", R)
    check(adapter_add(x, base, ad, index), x, base, ad, index)


@pytest.mark.parametrize("L,T", [(1, 40), (64, 64), (70, 200), (300, 1500), (1, 1500)])
def test_many_adapters(device, L, T):
    x, base = rows(device, T, 520, 136, BF16, L)
    ad = bank(device, L, 16, 520, 136, BF16, L + 1)
    for form in ("random", "each"):
        index = choose(device, T, L, form, 4)
        check(adapter_add(x, base, ad, index), x, base, ad, index)


def test_indices_outside_and_banks_without_adapters(device):
    x, base = rows(device, 70, 64, 72, BF16, 1)
    ad = bank(device, 2, 16, 64, 72, BF16, 2)
    index = torch.tensor([-1, 0, 1, 2, -2 ** 31, 2 ** 31 - 1, 5] * 10, device=device, dtype=torch.int32)
    check(adapter_add(x, base, ad, index), x, base, ad, index)
    none = torch.full((70,), -1, device=device, dtype=torch.int32)
    assert torch.equal(adapter_add(x, base, ad, none), base)
    empty = Adapters(ad.a[:0], ad.b[:0], ad.scale[:0])
    assert torch.equal(adapter_add(x, base, empty, index), base)
    assert adapter_add(x[:0], base[:0], ad, index[:0]).shape == (0, 72)


@pytest.mark.parametrize("T", [40, 1200])
def test_strides_and_shapes(device, T):
    x, base = rows(device, T, 136, 88, BF16, 1)
    ad = bank(device, 3, 16, 136, 88, BF16, 2)
    index = choose(device, T, 3, "random", 3)
    want = adapter_add(x, base, ad, index)
    wide = torch.randn(T, 400, device=device).to(BF16)
    wide[:, 16:152], wide[:, 160:248] = x, base
    before = wide.clone()
    assert torch.equal(adapter_add(wide[:, 16:152], wide[:, 160:248], ad, index), want)
    view = wide[:, 160:248]
    adapter_add(wide[:, 16:152], view, ad, index, out=view)
    assert torch.equal(view, want)
    before[:, 160:248] = want
    assert torch.equal(wide, before)      # nothing beside the slice
    odd = torch.randn(T, 137, device=device).to(BF16)
    odd[:, 1:] = x
    assert torch.equal(adapter_add(odd[:, 1:], base, ad, index), want)
    cube = adapter_add(x.view(T // 4, 4, 136), base.view(T // 4, 4, 88), ad, index)
    assert torch.equal(cube.view(T, 88), want)
    with pytest.raises(ValueError, match="in place"):
        bad = torch.randn(T, 89, device=device).to(BF16)[:, 1:]
        adapter_add(x, bad, ad, index, out=bad)


@pytest.mark.parametrize("T", [50, 1300])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_token_depends_on_its_own_row_alone(device, T, dtype):
    """Infinities, NaN and other values in some rows leave the others' bits as they were."""
    x, base = rows(device, T, 264, 104, dtype, 1)
    ad = bank(device, 4, 32, 264, 104, dtype, 2)
    index = choose(device, T, 4, "random", 3)
    want = adapter_add(x, base, ad, index)
    y = x.clone()
    y[3, 5], y[11, 100], y[20] = float("nan"), float("inf"), 60000.0
    got = adapter_add(y, base, ad, index)
    other = torch.ones(T, dtype=torch.bool, device=device)
    other[[3, 11, 20]] = False
    assert torch.equal(got[other], want[other])
    for t in (3, 11):
        assert index[t] < 0 or not got[t].isfinite().any()
    if index[20] >= 0:
        check(got[20:21], y[20:21], base[20:21], ad, index[20:21])


def test_products_beyond_float16(device):
    """h beyond float16's largest, with a small B: the result is in range."""
    x, base = rows(device, 6, 1024, 64, F16, 1)
    x = x.abs() * 200
    a = torch.full((2, 16, 1024), 3.0, device=device, dtype=F16)
    b = torch.full((2, 64, 16), 1e-6, device=device, dtype=F16)
    ad = Adapters(a, b, torch.ones(2, device=device))
    index = torch.tensor([0, 1, 0, -1, 1, 0], device=device, dtype=torch.int32)
    assert float((x.float() @ a[0].float().T).max()) > 65504
    check(adapter_add(x, base, ad, index), x, base, ad, index)


def test_graph_with_other_requests(device):
    T = 48
    x, base = rows(device, T, 512, 264, BF16, 1)
    ad = bank(device, 5, 32, 512, 264, BF16, 2)
    index = torch.zeros(T, device=device, dtype=torch.int32)
    adapter_add(x, base, ad, index)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = adapter_add(x, base, ad, index)
        graphs.append((graph, out))
    for step in range(6):
        index.copy_(choose(device, T, 5, ("random", "each", "one")[step % 3], step))
        x.copy_(rows(device, T, 512, 8, BF16, 50 + step)[0])
        graph, out = graphs[step % 2]
        graph.replay()
        want = adapter_add(x, base, ad, index)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        check(out, x, base, ad, index)


def test_two_streams_at_once(device):
    sets = [rows(device, 700, 1024, 520, BF16, s) for s in (1, 2)]
    ad = bank(device, 5, 64, 1024, 520, BF16, 3)
    index = choose(device, 700, 5, "runs", 4)
    want = [adapter_add(*s, ad, index) for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], [None, None]
    for _ in range(5):
        for i, (s, stream) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(stream):
                got[i] = adapter_add(*s, ad, index)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_beside_an_fp8_linear(device, dtype):
    g = torch.Generator(device).manual_seed(1)
    lin = torch.nn.Linear(512, 384, device=device, dtype=dtype)
    lin.requires_grad_(False)
    f = vdn_fp8.Fp8Linear(lin)
    x = torch.randn(3, 11, 512, device=device, generator=g).to(dtype)
    ad = bank(device, 3, 16, 512, 384, dtype, 2)
    index = choose(device, 33, 3, "random", 3)
    base = f(x)
    got = f(x, adapters=ad, index=index)
    assert got.shape == base.shape
    assert torch.equal(got, adapter_add(x, base, ad, index))
    check(got.view(33, 384), x.view(33, 512), base.view(33, 384), ad, index)
    with pytest.raises(ValueError, match="go together"):
        f(x, adapters=ad)
    with pytest.raises(ValueError, match="epilogue"):
        f(x, adapters=ad, index=index, epilogue="gelu_tanh")


def test_banks_from_adapter_files(device):
    """`Adapters.pack` of several ranks and types, and of the states that `load_external_lora` returns, is the sum that merging
    each adapter alone gives."""
    g = torch.Generator().manual_seed(1)
    states = []
    for rank in (4, 20, 32):
        states.append(({"blk.to_q.lora_A.weight": 0.1 * torch.randn(rank, 128, generator=g),
                        "blk.to_q.lora_B.weight": 0.1 * torch.randn(96, rank, generator=g),
                        "blk.to_k.lora_A.weight": torch.zeros(rank, 128), "blk.to_k.lora_B.weight": torch.zeros(96, rank)}, 16.0 / rank))
    ad = Adapters.of_states(states, "blk.to_q", device=device)
    assert ad.a.shape == (3, 32, 128) and ad.b.shape == (3, 96, 32) and ad.scale.tolist() == [4.0, pytest.approx(0.8), 0.5]
    x, base = rows(device, 30, 128, 96, BF16, 2)
    index = choose(device, 30, 3, "each", 0)
    got = adapter_add(x, base, ad, index)
    check(got, x, base, ad, index)
    for i, (state, scale) in enumerate(states):
        a, b = state["blk.to_q.lora_A.weight"].to(BF16), state["blk.to_q.lora_B.weight"].to(BF16)
        assert torch.equal(ad.a[i, :a.shape[0]].cpu(), a) and torch.equal(ad.b[i, :, :a.shape[0]].cpu(), b)
        assert not ad.a[i, a.shape[0]:].any() and not ad.b[i, :, a.shape[0]:].any()


@pytest.mark.parametrize("R", [16, 32, 48, 64])
@pytest.mark.parametrize("form", ["one", "random", "runs", "each"])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_one_launch_at_its_limits(device, R, form, dtype):
    """64 tokens, up to all of one adapter, and the widest rows that one launch takes; columns that end inside a workgroup's."""
    T, K, N = 64, 7168, 1544
    x, base = rows(device, T, K, N, dtype, R)
    ad = bank(device, 16, R, K, N, dtype, R + 1)
    index = choose(device, T, 16, form, R + 2)
    got = adapter_add(x, base, ad, index)
    check(got, x, base, ad, index)
    mine = base.clone()
    adapter_add(x, mine, ad, index, out=mine)
    assert torch.equal(mine, got)


@pytest.mark.parametrize("T", [9, 200, 1200])
def test_shared_memory(device, T):
    """out over x is refused (others still read those rows); x itself as the base, with a new out, is not."""
    x, _ = rows(device, T, 64, 64, BF16, 1)
    ad = bank(device, 4, 16, 64, 64, BF16, 2)
    index = choose(device, T, 4, "random", 3)
    kept = x.clone()
    with pytest.raises(ValueError, match="overlap x"):
        adapter_add(x, x, ad, index, out=x)
    wide = torch.zeros(T, 96, device=device, dtype=BF16)
    with pytest.raises(ValueError, match="overlap x"):
        part = wide[:, 32:]
        adapter_add(wide[:, :64], part, ad, index, out=part)
    assert torch.equal(x, kept) and not wide.any()
    check(adapter_add(x, x, ad, index), x, x, ad, index)


def test_offsets_beyond_32_bits(device):
    """33000 rows of 65544 columns, 4.3 GB: the last tokens' are what they are alone."""
    T, K, N = 33000, 64, 65544
    ad = bank(device, 2, 16, K, N, BF16, 2)
    x = rows(device, T, K, 8, BF16, 1)[0]
    base = torch.empty(T, N, device=device, dtype=BF16)
    base.fill_(0.5)
    tail = slice(T - 1300, T)
    base[tail] = rows(device, 1300, 8, N, BF16, 3)[1]
    index = choose(device, T, 2, "each", 0)
    want = adapter_add(x[tail], base[tail].clone(), ad, index[tail])
    check(want[-64:], x[-64:], base[-64:], ad, index[-64:])
    got = adapter_add(x, base, ad, index)
    assert torch.equal(got[tail], want)
    adapter_add(x, base, ad, index, out=base)
    assert torch.equal(base, got)


def test_rows_of_float32_are_refused(device):
    f = vdn_fp8.Fp8Linear(torch.nn.Linear(512, 384, device=device, dtype=torch.float32).requires_grad_(False))
    with pytest.raises(ValueError, match="bfloat16 or float16"):
        f(torch.randn(4, 512, device=device), adapters=bank(device, 2, 16, 512, 384, BF16, 2),
          index=torch.zeros(4, device=device, dtype=torch.int32))


@pytest.mark.parametrize("T", [300, 1300])
def test_graphs_of_the_other_forms(device, T):
    """A step and a prompt, captured, replayed with other requests and rows between eager calls (which take workspaces of their own)."""
    x, base = rows(device, T, 1024, 520, BF16, 1)
    ad = bank(device, 4, 96, 1024, 520, BF16, 2)
    index = torch.zeros(T, device=device, dtype=torch.int32)
    adapter_add(x, base, ad, index)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = adapter_add(x, base, ad, index)
        twice = adapter_add(x, out, ad, index)
    for step in range(5):
        index.copy_(choose(device, T, 4, ("random", "runs", "one")[step % 3], step))
        x.copy_(rows(device, T, 1024, 8, BF16, 50 + step)[0])
        graph.replay()
        want = adapter_add(x, base, ad, index)
        want_twice = adapter_add(x, want, ad, index)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(twice, want_twice)
        check(out, x, base, ad, index)


# Values in [1, 2) of 18 bits. Both 16-bit parts of one are multiples of 2^-17, as it is itself, so every sum below is one of a
# few such multiples of at most 4 and is exact in binary32 in any order: what is off is the split alone, 2^-17 at most.
@pytest.mark.parametrize("T", [40, 500, 1500])
@pytest.mark.parametrize("R", [16, 48, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_what_the_second_product_gets_of_the_first(device, T, R, dtype):
    """h in three ranks: a value, less its two largest 16-bit parts. What is left of the sum is below 2^-17, and so is what the
    kernel may lose of the value."""
    g = torch.Generator().manual_seed(R)
    h = 1 + torch.randint(0, 1 << 17, (T,), generator=g).double() / (1 << 17)
    h[:4] = torch.tensor([1 + 2.0 ** -8 + 2.0 ** -16, 1 + 2.0 ** -7 - 2.0 ** -17, 1 + 2.0 ** -8 + 3 * 2.0 ** -17, 2 - 2.0 ** -17])
    top = h.to(BF16).double()
    middle = (h - top).to(BF16).double()
    rest = h - top - middle
    assert float(rest.abs().max()) <= 2.0 ** -17
    K, N = 8, 136
    x = torch.zeros(T, K, dtype=torch.float64)
    x[:, 0], x[:, 1], x[:, 2] = top, middle, rest
    a, b = torch.zeros(1, R, K), torch.zeros(1, N, R)
    a[0, 0, :3] = 1
    a[0, 1, 0] = a[0, 2, 1] = -1
    b[0, :, :3] = 1
    assert torch.equal(x.to(dtype).double(), x)
    ad = Adapters(a.to(dtype).to(device), b.to(dtype).to(device), torch.ones(1, device=device))
    index, base = torch.zeros(T, dtype=torch.int32, device=device), torch.zeros(T, N, dtype=dtype, device=device)
    got = adapter_add(x.to(dtype).to(device), base, ad, index).double().cpu()
    # (the result is rounded to its type: half a step of what is at most 2^-16)
    assert torch.all((got - rest[:, None]).abs() <= 2.0 ** -17 + 2.0 ** -16 * torch.finfo(dtype).eps / 2), float((got - rest[:, None]).abs().max() * 2 ** 17)


@pytest.mark.parametrize("T", [40, 500, 1500])
def test_products_beyond_bfloat16(device, T):
    """h between bfloat16's largest and binary32's, with a small B: the result is in range, with h's own accuracy."""
    top = float(torch.finfo(BF16).max)
    x, base = torch.zeros(T, 8, device=device, dtype=BF16), torch.zeros(T, 72, device=device, dtype=BF16)
    x[:, 0] = top
    x[:, 1] = 2.0 ** 119 * (1 + torch.arange(T, device=device) % 64 / 64)          # (below 2^120: h below 2^128)
    x[1::2] *= -1
    a, b = torch.zeros(1, 16, 8, device=device, dtype=BF16), torch.full((1, 72, 16), 2.0 ** -20, device=device, dtype=BF16)
    a[0, 0, :2] = 1
    ad = Adapters(a, b, torch.ones(1, device=device))
    assert float((x.double() @ a[0].double().T).abs().max()) > top
    index = torch.zeros(T, device=device, dtype=torch.int32)
    check(adapter_add(x, base, ad, index), x, base, ad, index)


@pytest.mark.parametrize("K,T", [(7176, 7), (7176, 300), (13824, 1), (13824, 40), (13824, 64), (13824, 65), (13824, 700), (13824, 1100), (41000, 30),
                                 (41000, 520), (41000, 1100), (1 << 17, 3), (1 << 17, 130), (1 << 17, 1030)])
@pytest.mark.parametrize("R", [16, 48, 64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_long_rows(device, K, T, R, dtype):
    """Rows that the form of one launch does not take, those of a feed-forward's down projection and the longest; more than 32 parts of
    the first product."""
    print(f"adapters K={K} T={T} R={R} {dtype}", flush=True)
    N = 136
    x, base = rows(device, T, K, N, dtype, K + T)
    ad = bank(device, 3, R, K, N, dtype, R)
    index = choose(device, T, 3, "random" if T < 100 else "runs", R)
    got = adapter_add(x, base, ad, index)
    check(got, x, base, ad, index)
    mine = base.clone()
    adapter_add(x, mine, ad, index, out=mine)
    assert torch.equal(mine, got)
