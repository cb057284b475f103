"""The residual's addition, the norm and the codes in one pass (`add_norm_quantize`) against the formulas in 64 bits.

The new stream is compared exactly: a product of two 16-bit values and its sum with a third are formed by one fma,
that is as the 64-bit sum rounded to binary32, then rounded to the stream's type (a binary32 stream's product
of binary32 values is exact to 2^-53 in 64 bits: one step of binary32 is allowed there).

The normed rows' bound. With u = 2^-24: the sum of squares takes at most 8 * 8 fused steps of a lane, 6 of a wave and 16
of the waves (relative error 90 u, all terms positive), the quotient by K, eps, root and reciprocal 4 u: rstd is off by
45 u + 4 u. h rstd, w (1 + scale), their product and the shift's sum round 5 times. So n is off by no more than
ERR = 56 u of |h rstd w (1 + scale)| + |shift|."""
import pytest
import torch

import vdn_fp8
import vdn_fp8._lib as L

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
E4M3 = torch.float8_e4m3fn
ERR = 56 * 2.0 ** -24
TYPES = [(BF16, BF16), (F16, F16), (F32, BF16), (F32, F16), (F32, F32)]


def inputs(device, M, K, stream, dtype, rows, seed):
    g = torch.Generator().manual_seed(seed)
    channel = torch.exp(0.5 * torch.randn(K, generator=g))
    r = (3 * torch.randn(M, K, generator=g) * channel).to(stream)
    b = torch.randn(M, K, generator=g).to(dtype)
    w = (1 / channel + 0.05 * torch.randn(K, generator=g)).to(dtype)
    gate, sc, sh = ((0.5 * torch.randn(rows, K, generator=g)).to(dtype) for _ in range(3))
    index = torch.randint(0, rows, (M,), generator=g).to(torch.int32)
    return [t.to(device) for t in (r, b, w, gate, sc, sh, index)]


def formula(r, b, w, eps, gate=None, scale=None, shift=None, index=None):
    """hidden (its type), n and the bound of n in 64 bits."""
    i = torch.zeros(r.shape[0], dtype=torch.long, device=r.device) if index is None else index.long()
    total = r.double() + (b.double() if gate is None else gate.double()[i] * b.double())
    hidden = total.float().to(r.dtype)
    h = hidden.double()
    n = h / (h.square().mean(1, keepdim=True) + eps).sqrt()
    if w is not None:
        n = n * w.double()
    size = n.abs()
    if scale is not None:
        n = n * (1 + scale.double()[i])
        size = n.abs() + shift.double()[i].abs()
        n = n + shift.double()[i]
    return hidden, n, ERR * size


def check(got, want, dtype):
    hidden, n, err = want
    out, codes, s = got[:3]
    assert out.dtype == hidden.dtype and codes.dtype == E4M3 and s.shape == (n.shape[0], 1)
    if hidden.dtype == F32:
        assert torch.all((out.double() - hidden.double()).abs() <= 2.0 ** -23 * hidden.double().abs())
    else:
        assert torch.equal(out, hidden)
    size = (n.abs().amax(1, keepdim=True) / 448).clamp_min(1e-12)
    assert torch.all((s.double() - size).abs() <= err.amax(1, keepdim=True) / 448 + 2.0 ** -23 * size)
    # a code is that of a value within the bound of n, over the scale that came back (its quotient rounds once more)
    quotient, slack = n / s.double(), (err / s.double()) + 2.0 ** -23 * (n / s.double()).abs()
    low = (quotient - slack).clamp(-448, 448).float().to(E4M3).float()
    high = (quotient + slack).clamp(-448, 448).float().to(E4M3).float()
    c = codes.float()
    assert torch.all((low <= c) & (c <= high))
    if len(got) == 4:
        assert got[3].dtype == dtype
        room = err + torch.finfo(dtype).eps / 2 * (n.abs() + err) + (2.0 ** -25 if dtype == F16 else 0.0)   # (float16 below 2^-14)
        assert torch.all((got[3].double() - n).abs() <= room)


@pytest.mark.parametrize("M,K", [(1, 8), (3, 72), (2, 512), (5, 1024), (7, 1032), (1, 4104), (16, 5120), (33, 5376), (9, 7168), (2, 16384), (700, 2056),
                                 (515, 8200)])
@pytest.mark.parametrize("stream,dtype", TYPES)
def test_sizes_and_types(device, M, K, stream, dtype):
    print(f"add_norm {M} x {K} {stream} {dtype}", flush=True)
    r, b, w, gate, sc, sh, index = inputs(device, M, K, stream, dtype, 5, M * K)
    got = vdn_fp8.add_norm_quantize(r, b, w, 1e-6, gate=gate, scale=sc, shift=sh, indices=index, return_normed=True)
    check(got, formula(r, b, w, 1e-6, gate, sc, sh, index), dtype)
    got = vdn_fp8.add_norm_quantize(r, b, None, 1e-5)
    check(got, formula(r, b, None, 1e-5), dtype)


@pytest.mark.parametrize("gate,table,index,weight", [(True, False, True, True), (False, True, True, False), (True, True, False, True),
                                                     (False, True, False, True), (True, False, False, False)])
def test_forms(device, gate, table, index, weight):
    r, b, w, g, sc, sh, i = inputs(device, 37, 1288, F32, BF16, 1 if not index else 4, 3)
    kw = dict(gate=g if gate else None, scale=sc if table else None, shift=sh if table else None)
    got = vdn_fp8.add_norm_quantize(r, b, w if weight else None, 1e-6, indices=i if index else None, return_normed=True, **kw)
    want = formula(r, b, w if weight else None, 1e-6, kw["gate"], kw["scale"], kw["shift"], i if index else None)
    check(got, want, BF16)
    # without the normed rows the others have the same bits
    again = vdn_fp8.add_norm_quantize(r, b, w if weight else None, 1e-6, indices=i if index else None, **kw)
    for x, y in zip(got, again):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_shapes_strides_and_indices(device):
    r, b, w, gate, sc, sh, index = inputs(device, 24, 256, BF16, BF16, 6, 5)
    want = vdn_fp8.add_norm_quantize(r, b, w, 1e-6, gate=gate, scale=sc, shift=sh, indices=index)
    wide = torch.randn(24, 640, device=device).to(BF16)
    wide[:, 8:264], wide[:, 304:560] = r, b
    odd = torch.randn(24, 259, device=device).to(BF16)
    odd[:, 1:257] = b
    forms = {"column slices": (wide[:, 8:264], wide[:, 304:560]), "odd strides": (r, odd[:, 1:257]),
             "transposed": (r.T.contiguous().T, b), "three dimensions": (r.view(2, 12, 256), b.view(2, 12, 256))}
    for name, (x, y) in forms.items():
        got = vdn_fp8.add_norm_quantize(x, y, w, 1e-6, gate=gate, scale=sc, shift=sh, indices=index)
        assert got[0].shape == x.shape and got[1].shape == (24, 256), name
        for p, q in zip(got, want):
            assert torch.equal(p.reshape(q.shape).view(torch.uint8), q.view(torch.uint8)), name
    # indices of other integer types, and outside the tables: clamped
    out = index.long() * 0 + torch.tensor([-3, 0, 7, 1 << 40, 5, -(1 << 40)] * 4, device=device)
    a = vdn_fp8.add_norm_quantize(r, b, w, 1e-6, gate=gate, scale=sc, shift=sh, indices=out)
    c = vdn_fp8.add_norm_quantize(r, b, w, 1e-6, gate=gate, scale=sc, shift=sh, indices=out.clamp(0, 5).int())
    assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(a, c))
    empty = vdn_fp8.add_norm_quantize(r[:0], b[:0], w, 1e-6, return_normed=True)
    assert [t.shape[0] for t in empty] == [0] * 4


@pytest.mark.parametrize("K", [64, 5120])
@pytest.mark.parametrize("stream,dtype", TYPES)
def test_edge_rows(device, K, stream, dtype):
    """Rows of zeros (codes of zero at the least scale), one value in a row, infinities and NaN, that reach their own
    row alone; eps of zero."""
    M = 8
    r, b = torch.zeros(M, K, device=device, dtype=stream), torch.zeros(M, K, device=device, dtype=dtype)
    w = torch.ones(K, device=device, dtype=dtype)
    g = torch.Generator(device).manual_seed(1)
    r[1:] = torch.randn(M - 1, K, device=device, generator=g).to(stream)
    r[2] = 0
    r[2, K // 3] = 5.0
    r[3, 7], r[4, 0], b[5, K - 1] = float("inf"), float("nan"), float("-inf")
    r[6] *= 1e-3
    for eps in (1e-6, 0.0):
        hidden, codes, s, normed = vdn_fp8.add_norm_quantize(r, b, w, eps, return_normed=True)
        total = r.float() + b.float()
        assert torch.equal(torch.nan_to_num(hidden.float(), 77.0), torch.nan_to_num(total.to(stream).float(), 77.0))
        for row in (3, 4, 5):
            assert s[row].isnan().all() and codes[row].float().isnan().all()
        if eps:
            assert torch.all(codes[0].float() == 0) and abs(float(s[0]) - 1e-12) < 1e-18
            keep = [0, 1, 2, 6, 7]
        else:
            assert normed[0].isnan().all() and s[0].isnan().all()
            keep = [1, 2, 6, 7]
        want = formula(r[keep], b[keep], w, eps)
        check((hidden[keep], codes[keep], s[keep], normed[keep]), want, dtype)


def test_graphs_and_streams(device):
    """Captured and replayed with other rows, with eager calls between; on a stream that is not the default one."""
    sets = [inputs(device, 40, 5120, BF16, BF16, 3, s) for s in (11, 12, 13)]
    static = [t.clone() for t in sets[0]]

    def call(r, b, w, gate, sc, sh, index):
        return vdn_fp8.add_norm_quantize(r, b, w, 1e-6, gate=gate, scale=sc, shift=sh, indices=index, return_normed=True)

    want = [call(*s) for s in sets]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(*static)
    for k in (1, 2, 0, 1):
        for t, u in zip(static, sets[k]):
            t.copy_(u)
        graph.replay()
        call(*sets[0])
        torch.cuda.synchronize()
        assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(out, want[k])), k
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = call(*sets[2])
    side.synchronize()
    assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(got, want[2]))


def test_codes_feed_the_next_projection(device):
    """The codes and scales are what `Fp8Linear.forward_quantized` takes: its product is the one of the dequantized rows."""
    r, b, w, gate, sc, sh, index = inputs(device, 50, 512, BF16, BF16, 3, 9)
    hidden, codes, s = vdn_fp8.add_norm_quantize(r, b, w, 1e-6, gate=gate, scale=sc, shift=sh, indices=index)
    lin = torch.nn.Linear(512, 256, bias=False, device=device, dtype=BF16)
    f = vdn_fp8.Fp8Linear(lin)
    got = f.forward_quantized(codes, s).double()
    x = codes.double() * s.double()
    q = f.weight_fp8.double() * f.weight_scale.double().T
    want, size = x @ q.T, x.abs() @ q.abs().T
    # the product's rounding to bf16, half a step of 2^-7 (it has 8 significant bits), and 512 sums and two scales in binary32
    # (2^-23 each, should the matrix cores truncate)
    room = 514 * 2.0 ** -23 * size
    assert torch.all((got - want).abs() <= 2.0 ** -8 * (want.abs() + room) + room)


def test_offsets_beyond_32_bits(device):
    """300000 rows of 8192, 4.9 GB a tensor, the last of them. (Their bits are not those of a call of 40 rows, whose waves sum squares
    in another order.)"""
    M, K = 300000, 8192
    r, b, w, gate, sc, sh, index = inputs(device, 40, K, BF16, BF16, 3, 1)
    residual, branch = (torch.empty(M, K, device=device, dtype=BF16) for _ in range(2))
    residual.fill_(1.0)
    branch.fill_(0.25)
    residual[-40:], branch[-40:] = r, b
    far = torch.zeros(M, device=device, dtype=torch.int32)
    far[-40:] = index
    got = vdn_fp8.add_norm_quantize(residual, branch, w, 1e-6, gate=gate, scale=sc, shift=sh, indices=far)
    check([t[-40:] for t in got], formula(r, b, w, 1e-6, gate, sc, sh, index), BF16)


@pytest.mark.parametrize("K", [64, 5120])
def test_squares_beyond_binary32(device, K):
    """Sums of squares that overflow (1 / inf: n is the shift itself) or are subnormal (no accuracy is left, but no NaN either)."""
    g = torch.Generator(device).manual_seed(1)
    r = torch.randn(6, K, device=device, generator=g)
    r[:3] *= 1e25
    r[3:] *= 1e-22
    b, w, sc = torch.zeros(6, K, device=device, dtype=BF16), torch.ones(K, device=device, dtype=BF16), torch.zeros(K, device=device, dtype=BF16)
    sh = torch.randn(K, device=device, generator=g).to(BF16)
    hidden, codes, s, normed = vdn_fp8.add_norm_quantize(r, b, w, 0.0, scale=sc, shift=sh, return_normed=True)
    assert torch.equal(hidden, r)
    assert torch.equal(normed[:3], sh.expand(3, K))
    alone, s_alone = vdn_fp8.quantize_rows(sh[None])
    assert torch.equal(s[:3], s_alone.expand(3, 1)) and torch.equal(codes[:3].float(), alone.float().expand(3, K))
    assert normed[3:].isfinite().all() and codes[3:].float().isfinite().all() and s[3:].isfinite().all()


def test_equal_maxima(device):
    """Rows in which many elements are the largest, in other waves: the same bits in every call, and the formula's."""
    g = torch.Generator(device).manual_seed(1)
    r = torch.randint(-2, 3, (600, 5120), device=device, generator=g).to(BF16)
    b = torch.zeros_like(r)
    w = (1 + torch.randint(0, 2, (5120,), device=device, generator=g).float() / 128).to(BF16)
    sc, sh = (torch.randint(0, 2, (5120,), device=device, generator=g).float() / 64).to(BF16), torch.zeros(5120, device=device, dtype=BF16)
    for tables in ({}, {"scale": sc, "shift": sh}):
        first = vdn_fp8.add_norm_quantize(r, b, w, 1e-6, return_normed=True, **tables)
        check(first, formula(r, b, w, 1e-6, scale=sc[None] if tables else None, shift=sh[None] if tables else None), BF16)
        for _ in range(20):
            again = vdn_fp8.add_norm_quantize(r, b, w, 1e-6, return_normed=True, **tables)
            assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(first, again))


def test_more_rows_than_a_launch_takes(device):
    M, K = (1 << 21) + 37, 8
    r, b, w, gate, sc, sh, index = inputs(device, M, K, BF16, BF16, 5, 1)
    got = vdn_fp8.add_norm_quantize(r, b, w, 1e-6, gate=gate, scale=sc, shift=sh, indices=index, return_normed=True)
    check(got, formula(r, b, w, 1e-6, gate, sc, sh, index), BF16)


@pytest.mark.parametrize("kind,rows", [(torch.uint8, 300), (torch.uint8, 20), (torch.int8, 200), (torch.int8, 128), (torch.int8, 129),
                                       (torch.int16, 33000), (torch.bool, 2), (torch.bool, 1), (torch.int64, 300)])
def test_indices_narrower_than_the_table(device, kind, rows):
    """Indices of any integer type (or truth values), also of one that does not hold the table's last row: clamped as others are."""
    g = torch.Generator().manual_seed(rows)
    M, K = 40, 64
    r, b, gate = (torch.randn(n, K, generator=g).to(BF16).to(device) for n in (M, M, rows))
    index = torch.randint(-128, 128, (M,), generator=g).to(kind).to(device)
    got = vdn_fp8.add_norm_quantize(r, b, None, 1e-6, gate=gate, indices=index)
    want = vdn_fp8.add_norm_quantize(r, b, None, 1e-6, gate=gate, indices=index.long().clamp(0, rows - 1).int())
    assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(got, want))


def call(r, b, w, hidden, y, s, normed):
    """The C entry point, without tables."""
    M, K = r.shape
    types = {BF16: L.DTYPE_BF16, F16: L.DTYPE_F16, F32: L.DTYPE_F32}
    L.check(L.load().vdn_fp8_add_norm_quantize(
        r.data_ptr(), types[r.dtype], r.stride(0), b.data_ptr(), types[b.dtype], b.stride(0), M, K, None, 0, w.data_ptr(), 1e-6, None, None, 0, None,
        0, hidden.data_ptr(), hidden.stride(0), y.data_ptr(), y.stride(0), s.data_ptr(), normed.data_ptr(), normed.stride(0),
        torch.cuda.current_stream().cuda_stream), "add_norm_quantize")


@pytest.mark.parametrize("M,K", [(1, 264), (16, 5120), (700, 4104)])
@pytest.mark.parametrize("stream,dtype,over", [(*t, over) for t in TYPES for over in ("residual", "branch", "both") if over != "both" or t[0] is t[1]])
def test_hidden_in_place(device, M, K, stream, dtype, over):
    """hidden over residual, over a branch of its type, over both where they are one: the bits of a new tensor. Rows lie apart, and
    what lies between them stays."""
    r, b, w, *_ = inputs(device, M, K, stream, dtype, 1, M + K)
    wide = [torch.full((M, K + 24), 7.0, device=device, dtype=t.dtype) for t in (r, b)]
    if over == "both":
        b = r.clone()
        wide[1] = wide[0]
    rows = [t[:, 8:8 + K] for t in wide]
    rows[0].copy_(r), rows[1].copy_(b)
    want = vdn_fp8.add_norm_quantize(r, b, w, 1e-6, return_normed=True)
    y, s, normed = torch.empty(M, K, device=device, dtype=E4M3), torch.empty(M, 1, device=device), torch.empty(M, K, device=device, dtype=dtype)
    hidden = rows[over == "branch"]
    if over == "branch" and stream is not dtype:
        kept = [t.clone() for t in wide]
        with pytest.raises(ValueError, match="with its stride and type"):
            call(*rows, w, hidden, y, s, normed)
        assert all(torch.equal(t, k) for t, k in zip(wide, kept))
        return
    call(*rows, w, hidden, y, s, normed)
    for got, t in zip((hidden, y, s, normed), want):
        assert torch.equal(got.contiguous().view(torch.uint8), t.view(torch.uint8))
    assert all(bool((t[:, :8] == 7).all() and (t[:, 8 + K:] == 7).all()) for t in wide)
