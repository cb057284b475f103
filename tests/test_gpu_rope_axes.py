"""QK-norm and rotary positions with several axes (`qk_prep_axes`) against the formulas in 64 bits.

Bound. With u = 2^-24: a head's sum of squares takes 8 products and sums of a lane and up to 5 of the lanes (21 u of it), the
quotient, eps, root and reciprocal 4 u, the two products 2 u: n is off by 17 u. Cosine and sine: the angle's remainder of a quarter
turn, at most pi / 4, rounds once, the series (errors below 2^-28) about 3 times: 4 u. Product and sum: 2 u. Together 24 u of
|n lo| + |n hi|, and the reference's own angle (the product of position and frequency rounds once in 64 bits, pi / 2's multiple
once): 2^-51 of the angle. The result rounds once."""
import pytest
import torch

import vdn_fp8
import vdn_fp8._lib as L
from vdn_fp8 import RopeAxes

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def formula(x, norm, rope, positions):
    """(result, bound before its own rounding) in 64 bits."""
    n = x.double()
    if norm is not None:
        w, eps = norm
        n = n / (n.square().mean(2, keepdim=True) + eps).sqrt() * (1.0 if w is None else w.double())
    half = rope.inv_freq.numel()
    p = positions.double()
    p = p[:, None] if p.dim() == 1 else p
    angle = p[:, rope.axis.long()] * rope.inv_freq
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    at = torch.arange(half, device=x.device)
    lo, hi = (2 * at, 2 * at + 1) if rope.pairs else (at, at + half)
    out, size = n.clone(), n.abs()
    a, b = n[..., lo], n[..., hi]
    out[..., lo], out[..., hi] = a * c - b * s, b * c + a * s
    both = a.abs() + b.abs()
    bound = 24 * 2.0 ** -24 * size
    turned = both * (24 * 2.0 ** -24 + 2.0 ** -51 * angle.abs()[:, None])
    bound[..., lo], bound[..., hi] = turned, turned
    return out, bound


def check(got, x, norm, rope, positions):
    want, bound = formula(x, norm, rope, positions)
    assert got.dtype == x.dtype and got.shape == x.shape and got.is_contiguous()
    room = bound + torch.finfo(x.dtype).eps / 2 * (want.abs() + bound) + (2.0 ** -25 if x.dtype == F16 else 0.0)
    bad = (got.double() - want).abs() > room
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())


def heads(device, T, Hq, H, d, dtype, seed, norm=True):
    g = torch.Generator(device).manual_seed(seed)
    qkv = torch.randn(T, (Hq + 2 * H) * d, device=device, generator=g).to(dtype)
    q, k, _ = (t.unflatten(1, (-1, d)) for t in qkv.split((Hq * d, H * d, H * d), 1))
    nq, nk = (((1 + 0.2 * torch.randn(d, device=device, generator=g)).to(dtype), 1e-6) if norm else None for _ in range(2))
    return q, k, nq, nk


@pytest.mark.parametrize("T,Hq,H,d,sections,pairs", [
    (1, 1, 1, 64, (32,), False), (1, 40, 8, 128, (24, 20, 20), False), (3, 12, 12, 64, (5, 11), True), (17, 7, 1, 128, (1, 2, 3, 2), True),
    (130, 40, 40, 128, (16, 24, 24), False), (65, 5, 3, 256, (64, 32, 32), True), (9, 33, 11, 256, (40, 48, 40), False),
    (1025, 12, 12, 64, (8, 8, 8), False), (1300, 56, 56, 128, (22, 21, 21), True), (1027, 9, 2, 256, (16,), False),
    (40, 4, 2, 128, (1, 1, 1, 1, 1, 1, 1, 1), True)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_sizes_types_and_layouts(device, T, Hq, H, d, sections, pairs, dtype):
    print(f"rope {T} {Hq}/{H} x {d} {sections} {pairs} {dtype}", flush=True)
    q, k, nq, nk = heads(device, T, Hq, H, d, dtype, T + d)
    rope = RopeAxes.make(sections, pairs=pairs, device=device)
    pos = torch.randint(0, 3000, (T, len(sections)), device=device).int()
    for norms in ((nq, nk), (None, None), ((None, 1e-5), nk)):
        got = vdn_fp8.qk_prep_axes(q, k, *norms, rope, pos)
        check(got[0], q, norms[0], rope, pos)
        check(got[1], k, norms[1], rope, pos)


@pytest.mark.parametrize("kind", ["int32", "int64", "float32"])
def test_positions(device, kind):
    """Far, negative and fractional positions; strided ones; one axis as a vector."""
    q, k, nq, nk = heads(device, 48, 6, 2, 128, F32, 5)
    rope = RopeAxes.make((32, 32), theta=1e6, device=device)
    g = torch.Generator(device).manual_seed(3)
    far = torch.randint(-2 ** 31, 2 ** 31 - 1, (48, 2), device=device, generator=g)
    if kind == "float32":
        pos = torch.cat([(far[:24] / 1000.0).float(), torch.rand(24, 2, device=device, generator=g) * 50])
    elif kind == "int64":
        pos = far * 256
    else:
        pos = far.int()
        pos[0], pos[1] = 2 ** 31 - 1, -2 ** 31
    got = vdn_fp8.qk_prep_axes(q, k, nq, nk, rope, pos)
    check(got[0], q, nq, rope, pos)
    check(got[1], k, nk, rope, pos)
    wide = torch.zeros(48, 7, device=device, dtype=pos.dtype)
    wide[:, ::4] = pos
    again = vdn_fp8.qk_prep_axes(q, k, nq, nk, rope, wide[:, ::4])
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    one = RopeAxes.make((64,), device=device)
    got = vdn_fp8.qk_prep_axes(q, k, nq, nk, one, pos[:, 0])
    check(got[0], q, nq, one, pos[:, 0])


def test_axes_that_share_one_sequence_of_frequencies(device):
    """`shared`: on equal positions of every axis it is the rotation of one axis; axes in any order."""
    q, k, nq, nk = heads(device, 20, 4, 4, 128, BF16, 7)
    pos = torch.arange(20, device=device).int() * 37
    one = vdn_fp8.qk_prep_axes(q, k, nq, nk, RopeAxes.make((64,), device=device), pos)
    three = RopeAxes.make((16, 24, 24), shared=True, device=device)
    got = vdn_fp8.qk_prep_axes(q, k, nq, nk, three, pos[:, None].expand(-1, 3))
    assert all(torch.equal(a, b) for a, b in zip(one, got))
    mixed = RopeAxes(three.inv_freq, (torch.arange(64, device=device) % 3).int())
    p = torch.randint(0, 99, (20, 3), device=device).int()
    got = vdn_fp8.qk_prep_axes(q, k, nq, nk, mixed, p)
    check(got[0], q, nq, mixed, p)
    # an axis that is not there is the nearest that is
    a = vdn_fp8.qk_prep_axes(q, k, nq, nk, RopeAxes(three.inv_freq, mixed.axis + 1), p)
    b = vdn_fp8.qk_prep_axes(q, k, nq, nk, RopeAxes(three.inv_freq, (mixed.axis + 1).clamp(max=2)), p)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_no_pairs_is_the_norm_alone(device):
    q, k, nq, nk = heads(device, 11, 3, 2, 64, BF16, 8)
    rope = RopeAxes(torch.zeros(0, dtype=torch.float64, device=device), torch.zeros(0, dtype=torch.int32, device=device))
    pos = torch.zeros(11, 1, device=device).int()
    got = vdn_fp8.qk_prep_axes(q, k, nq, nk, rope, pos)
    check(got[0], q, nq, rope, pos)
    assert torch.equal(got[0], vdn_fp8.qk_prep(q, *nq))


def test_edge_values(device):
    """Infinities and NaN stay in their head; a position that is no number in its token; rows of zeros."""
    q, k, nq, nk = heads(device, 6, 4, 2, 128, F32, 9)
    q, k = q.clone(), k.clone()
    rope = RopeAxes.make((64,), device=device)
    pos = torch.arange(6, device=device).float()
    clean = vdn_fp8.qk_prep_axes(q, k, nq, nk, rope, pos)
    q[1, 2, 5], q[3, 0, 100], k[4] = float("nan"), float("inf"), 0.0
    pos[5] = float("nan")
    got = vdn_fp8.qk_prep_axes(q, k, nq, nk, rope, pos)
    touched = torch.zeros(6, 4, dtype=torch.bool, device=device)
    touched[1, 2] = touched[3, 0] = True
    touched[5] = True
    assert torch.equal(got[0][~touched], clean[0][~touched])
    assert got[0][1, 2].isnan().all() and got[0][3, 0].isnan().any() and got[0][5].isnan().all()
    assert torch.all(got[1][4] == 0)
    empty = vdn_fp8.qk_prep_axes(q[:0], k[:0], nq, nk, rope, pos[:0])
    assert empty[0].shape == (0, 4, 128) and empty[1].shape == (0, 2, 128)


def test_graph_with_other_positions(device):
    q, k, nq, nk = heads(device, 16, 40, 8, 128, BF16, 10)
    rope = RopeAxes.make((24, 20, 20), device=device)
    pos = torch.zeros(16, 3, device=device).int()
    graph = torch.cuda.CUDAGraph()
    vdn_fp8.qk_prep_axes(q, k, nq, nk, rope, pos)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = vdn_fp8.qk_prep_axes(q, k, nq, nk, rope, pos)
    for step in (5, 100000, 7, 123):
        pos.fill_(step)
        graph.replay()
        want = vdn_fp8.qk_prep_axes(q, k, nq, nk, rope, pos)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_offsets_beyond_32_bits(device):
    """300000 tokens of 64 + 1 heads of 128, 4.9 GB of queries: the last tokens' results are what they are alone."""
    T, d, rope = 300000, 128, RopeAxes.make((24, 20, 20), device=device)
    q, k, nq, nk = heads(device, 40, 64, 1, d, BF16, 1)
    query, key = torch.empty(T, 64, d, device=device, dtype=BF16), torch.empty(T, 1, d, device=device, dtype=BF16)
    query.fill_(1.0)
    key.fill_(1.0)
    query[-40:], key[-40:] = q, k
    positions = torch.arange(3 * T, device=device, dtype=torch.int32).view(T, 3)
    got = vdn_fp8.qk_prep_axes(query, key, nq, nk, rope, positions)
    for out, x, norm in zip(got, (q, k), (nq, nk)):
        check(out[-40:], x, norm, rope, positions[-40:])


def test_more_tokens_than_a_launch_takes(device):
    T, rope = (1 << 25) + 70, RopeAxes.make((8, 12, 12), device=device)
    q, _, nq, _ = heads(device, 100, 1, 1, 64, BF16, 1)
    query = torch.empty(T, 1, 64, device=device, dtype=BF16)
    query.fill_(1.0)
    query[-100:] = q
    positions = torch.arange(T, device=device, dtype=torch.int32)[:, None].expand(T, 3)
    out, none = vdn_fp8.qk_prep_axes(query, query[:, :0], nq, None, rope, positions)
    assert none.shape == (T, 0, 64)
    check(out[-100:], q, nq, rope, positions[-100:])


@pytest.mark.parametrize("T", [1, 16, 1500])
@pytest.mark.parametrize("d,dtype,pairs", [(64, F16, True), (128, BF16, False), (256, F32, False)])
def test_outputs_in_place(device, T, d, dtype, pairs):
    """The C entry with each output in its input's place, column slices of one fused matrix: the bits of new tensors, and the
    columns of the values stay."""
    Hq, H = 5, 3
    rope = RopeAxes.make((d // 4, d // 4), pairs=pairs, device=device)
    qkv = torch.randn(T, (Hq + 2 * H) * d, device=device).to(dtype)
    before = qkv.clone()
    q, k, v = (t.unflatten(1, (-1, d)) for t in qkv.split((Hq * d, H * d, H * d), 1))
    w = (1 + 0.2 * torch.randn(d, device=device)).to(dtype)
    pos = torch.randint(0, 3000, (T, 2), device=device).int()
    want = vdn_fp8.qk_prep_axes(q, k, (w, 1e-6), None, rope, pos)
    ld, kind = qkv.stride(0), {BF16: L.DTYPE_BF16, F16: L.DTYPE_F16, F32: L.DTYPE_F32}[dtype]
    L.check(L.load().vdn_fp8_qk_prep_axes(
        q.data_ptr(), Hq, ld, k.data_ptr(), H, ld, T, d, kind, 1, w.data_ptr(), 1e-6, 0, None, 0.0, rope.inv_freq.data_ptr(), rope.axis.data_ptr(), d,
        int(pairs), pos.data_ptr(), L.POSITION_I32, 2, 2, q.data_ptr(), ld, k.data_ptr(), ld, torch.cuda.current_stream().cuda_stream), "qk_prep_axes")
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(v, before.split((Hq * d, H * d, H * d), 1)[2].unflatten(1, (-1, d)))
