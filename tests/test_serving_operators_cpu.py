"""Refusals of `add_norm_quantize`, `adapter_add` and `qk_prep_axes`, in C and in Python, without a GPU."""
import ctypes

import pytest
import torch

import vdn_fp8
import vdn_fp8._lib as L
from vdn_fp8 import Adapters, RopeAxes

FAKE = 1 << 20        # never dereferenced: every call below fails its checks first
OTHER = 1 << 30


def norm(r=FAKE, stream=0, ldr=64, b=FAKE, dtype=0, ldb=64, M=4, K=64, gate=None, ldgate=64, w=None, eps=1e-6, sc=None, sh=None, ldmod=64,
         index=None, rows=0, h=FAKE, ldh=64, y=FAKE, ldy=64, s=FAKE, n=None, ldn=64):
    return L.load().vdn_fp8_add_norm_quantize(r, stream, ldr, b, dtype, ldb, M, K, gate, ldgate, w, eps, sc, sh, ldmod, index, rows, h, ldh, y, ldy,
                                              s, n, ldn, None)


def adapt(x=FAKE, dtype=0, ldx=64, base=FAKE, ldbase=32, T=4, K=64, N=32, a=FAKE, b=FAKE, scale=FAKE, banks=2, R=16, index=FAKE, out=OTHER, ldo=32,
          ws=FAKE, n=1 << 40):
    return L.load().vdn_fp8_adapter_add(x, dtype, ldx, base, ldbase, T, K, N, a, b, scale, banks, R, index, out, ldo, ws, n, None)


def rope(q=FAKE, hq=4, ldq=512, k=FAKE, hk=2, ldk=256, T=4, d=128, dtype=0, wq=None, eq=1e-6, wk=None, ek=1e-6, freq=FAKE, axis=FAKE, R=128, pairs=0,
         pos=FAKE, kind=0, axes=3, ldpos=3, oq=FAKE, ldoq=512, ok=FAKE, ldok=256):
    return L.load().vdn_fp8_qk_prep_axes(q, hq, ldq, k, hk, ldk, T, d, dtype, 1, wq, eq, 1, wk, ek, freq, axis, R, pairs, pos, kind, axes, ldpos, oq,
                                         ldoq, ok, ldok, None)


@pytest.mark.parametrize("call,needle", [
    (lambda: norm(M=-1), "negative"), (lambda: norm(K=60, ldr=64), "multiple of 8"), (lambda: norm(K=0), "multiple of 8"),
    (lambda: norm(K=16392, ldr=16392, ldb=16392, ldh=16392, ldy=16392), "16384"), (lambda: norm(dtype=3, stream=3), "dtype"),
    (lambda: norm(stream=1), "dtype"), (lambda: norm(stream=0, dtype=2), "dtype"), (lambda: norm(r=None), "null"), (lambda: norm(s=None), "null"),
    (lambda: norm(sc=FAKE), "together"), (lambda: norm(eps=-1.0), "eps"), (lambda: norm(eps=float("nan")), "eps"),
    (lambda: norm(gate=FAKE), "at least 1 row"), (lambda: norm(index=FAKE), "index"), (lambda: norm(ldr=56), "strides"),
    (lambda: norm(ldb=68), "strides"), (lambda: norm(n=FAKE, ldn=8), "strides"), (lambda: norm(gate=FAKE, rows=2, ldgate=8), "strides"),
    (lambda: norm(sc=FAKE, sh=FAKE, rows=2, ldmod=60), "strides"), (lambda: norm(h=FAKE + 8), "misaligned"), (lambda: norm(y=FAKE + 4), "misaligned"),
    (lambda: norm(w=FAKE + 2), "misaligned"),
    (lambda: adapt(T=-1), "negative"), (lambda: adapt(T=(1 << 23) + 1), "2^23"), (lambda: adapt(banks=(1 << 23) + 1), "2^23"),
    (lambda: adapt(K=60), "multiples of 8"), (lambda: adapt(N=0), "multiples of 8"), (lambda: adapt(K=(1 << 17) + 8), "2^17"),
    (lambda: adapt(R=8), "rank"), (lambda: adapt(R=24), "rank"), (lambda: adapt(R=144), "rank"), (lambda: adapt(dtype=2), "dtype"),
    (lambda: adapt(x=None), "null"), (lambda: adapt(index=None), "null"), (lambda: adapt(b=None), "null"), (lambda: adapt(ldx=56), "strides"),
    (lambda: adapt(ldbase=36), "strides"), (lambda: adapt(ldo=(1 << 23) + 8), "strides"), (lambda: adapt(x=FAKE + 8), "misaligned"),
    (lambda: adapt(index=FAKE + 2), "misaligned"),
    # (a call of few tokens has no workspace)
    (lambda: adapt(T=9, ws=None), "workspace"), (lambda: adapt(T=9, n=16), "workspace"), (lambda: adapt(T=9, ws=FAKE + 8), "workspace"),
    # out over x: the same rows, rows of another stride, one that begins in x's last row, columns that meet in it, that wrap into it
    (lambda: adapt(N=64, ldbase=64, ldo=64, out=FAKE), "overlap x"), (lambda: adapt(out=FAKE + 3 * 128), "overlap x"),
    (lambda: adapt(x=OTHER, out=OTHER - 3 * 64), "overlap x"), (lambda: adapt(ldx=96, ldo=96, x=OTHER, out=OTHER + 112), "overlap x"),
    (lambda: adapt(ldx=96, ldo=96, x=OTHER + 96, out=OTHER + 64), "overlap x"),
    (lambda: adapt(ldo=64, out=FAKE + (1 << 16), base=FAKE + (1 << 16)), "base itself"),
    (lambda: adapt(base=FAKE + (1 << 16), out=FAKE + (1 << 16) + 64), "base itself"),
    (lambda: rope(T=-1), "negative"), (lambda: rope(dtype=3), "dtype"), (lambda: rope(d=96), "head dim"), (lambda: rope(hq=513, ldq=1 << 17), "65536"),
    (lambda: rope(R=136), "multiple of 16"), (lambda: rope(R=24), "multiple of 16"), (lambda: rope(R=12, pairs=1), "multiple of 8"),
    (lambda: rope(R=-16), "multiple of 16"), (lambda: rope(freq=None), "null"), (lambda: rope(pos=None), "null"), (lambda: rope(axes=0), "axes"),
    (lambda: rope(axes=9, ldpos=9), "axes"), (lambda: rope(ldpos=2), "axes"), (lambda: rope(kind=3), "positions"), (lambda: rope(kind=-1), "positions"),
    (lambda: rope(freq=FAKE + 4), "misaligned"), (lambda: rope(pos=FAKE + 4, kind=1), "misaligned"), (lambda: rope(eq=-1.0), "eps"),
    (lambda: rope(ek=float("nan")), "eps"), (lambda: rope(q=None), "rows"), (lambda: rope(ldq=504), "rows"), (lambda: rope(ldk=260), "rows"),
    (lambda: rope(ok=FAKE + 8), "rows"), (lambda: rope(wk=FAKE + 2), "misaligned"),
])
def test_contract_violations_are_einval(call, needle):
    assert call() == L.EINVAL
    assert needle in L.load().vdn_fp8_last_error().decode()


def test_empty_calls_do_nothing():
    assert norm(M=0, r=None, b=None, h=None, y=None, s=None) == L.OK
    assert adapt(T=0, x=None, base=None, out=None, index=None, ws=None) == L.OK
    assert rope(T=0, q=None, k=None, oq=None, ok=None) == L.OK
    assert rope(hq=0, hk=0, q=None, k=None, oq=None, ok=None) == L.OK


def test_adapter_workspace_sizes():
    lib, size = L.load(), ctypes.c_int64(-1)
    ask = lambda *a: lib.vdn_fp8_adapter_add_workspace_size(*a, ctypes.byref(size))   # noqa: E731
    assert ask(0, 64, 64, 2, 16) == L.OK and size.value == 0
    assert ask(5, 64, 64, 0, 16) == L.OK and size.value == 0
    for T in (17, 64, 1024, 1025, 32760):
        for R in (16, 48, 128):
            assert ask(T, 5120, 5120, 4, R) == L.OK
            whole = -(-T // 64) * 64 * R * 4       # h of whole tiles, in up to 32 parts
            assert size.value > 0 and size.value % whole == 0 and size.value // whole <= 32
    # few tokens of an adapter, ranks and widths that one launch takes: none
    for T, R, K, none in ((1, 64, 7168, True), (16, 64, 5120, True), (16, 80, 5120, False), (16, 64, 7176, False), (17, 16, 64, False)):
        assert ask(T, K, 5120, 4, R) == L.OK and (size.value == 0) == none
    assert ask(5, 64, 64, 2, 17) == L.EINVAL
    assert lib.vdn_fp8_adapter_add_workspace_size(5, 64, 64, 2, 16, None) == L.EINVAL


def test_cpu_tensors_are_refused():
    r = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        vdn_fp8.add_norm_quantize(r, r, None, 1e-6)
    with pytest.raises(ValueError, match="GPU"):
        vdn_fp8.adapter_add(r, r, Adapters(torch.zeros(1, 16, 64).bfloat16(), torch.zeros(1, 64, 16).bfloat16(), torch.ones(1)),
                            torch.zeros(4, dtype=torch.int32))
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        vdn_fp8.qk_prep_axes(q, q, None, None, RopeAxes.make((32,), device="cpu"), torch.zeros(4, 1, dtype=torch.int32))


def test_banks():
    f = torch.randn(5, 24), torch.randn(16, 5), 2.0
    ad = Adapters.pack([f, (torch.randn(33, 24), torch.randn(16, 33), 1.0)], device="cpu", dtype=torch.float16)
    assert ad.a.shape == (2, 48, 24) and ad.b.shape == (2, 16, 48) and ad.scale.tolist() == [2.0, 1.0]
    assert torch.equal(ad.a[0, :5], f[0].half()) and not ad.a[0, 5:].any() and not ad.b[0, :, 5:].any()
    for bad, needle in (([], "at least one"), ([f, (torch.randn(4, 25), torch.randn(16, 4), 1.0)], "fit"),
                        ([(torch.randn(129, 8), torch.randn(8, 129), 1.0)], "128")):
        with pytest.raises(ValueError, match=needle):
            Adapters.pack(bad, device="cpu")
    with pytest.raises(ValueError, match="bfloat16 or float16"):
        Adapters.pack([f], dtype=torch.float32, device="cpu")
    with pytest.raises(KeyError):
        Adapters.of_states([({"a.lora_A.weight": f[0], "a.lora_B.weight": f[1]}, 1.0)], "b", device="cpu")


def test_rope_axes():
    rope = RopeAxes.make((2, 4, 2), theta=100.0, device="cpu")
    assert rope.axis.tolist() == [0, 0, 1, 1, 1, 1, 2, 2] and rope.axis.dtype == torch.int32 and rope.inv_freq.dtype == torch.float64
    want = [1.0, 100 ** -0.5, 1.0, 100 ** -0.25, 100 ** -0.5, 100 ** -0.75, 1.0, 100 ** -0.5]
    assert rope.inv_freq.tolist() == pytest.approx(want, rel=1e-15)
    shared = RopeAxes.make((2, 4, 2), theta=100.0, shared=True, device="cpu")
    assert shared.inv_freq.tolist() == pytest.approx([100 ** (-j / 8) for j in range(8)], rel=1e-15)
    for bad in ((), (0,), (-1, 9)):
        with pytest.raises(ValueError):
            RopeAxes.make(bad, device="cpu")


def test_one_bank_for_three_projections_is_refused():
    """A bank is a tuple of three itself: refused before a projection runs, not taken apart."""
    bank = Adapters(torch.zeros(1, 16, 64).bfloat16(), torch.zeros(1, 64, 16).bfloat16(), torch.ones(1))
    cache = vdn_fp8.KvCache.empty(1, 1, 64, "cpu")

    def unreached(x):
        raise AssertionError("a projection ran")

    with pytest.raises(ValueError, match="three banks"):
        vdn_fp8.softmax_attention.cached_attention(torch.zeros(4, 64).bfloat16(), unreached, unreached, unreached, None, None, cache,
                                                   torch.zeros(1, 1, dtype=torch.int32), torch.full((1,), 4, dtype=torch.int32),
                                                   adapters=bank, index=torch.zeros(4, dtype=torch.int32))


def apart(**over):
    """`norm` of four rows of 64 in places of their own (bf16), less what `over` puts elsewhere."""
    return norm(**{**dict(r=FAKE, b=FAKE + (1 << 16), h=OTHER, y=OTHER + (1 << 16), s=OTHER + (1 << 18)), **over})


@pytest.mark.parametrize("over,needle", [
    # hidden over residual or branch with another stride, or in part: rows, columns that meet, columns that wrap into a row
    (dict(h=FAKE, ldh=72), "residual or branch itself"), (dict(h=FAKE + (1 << 16), ldh=72), "residual or branch itself"),
    (dict(h=FAKE + 128), "residual or branch itself"), (dict(h=FAKE + (1 << 16) + 3 * 128), "residual or branch itself"),
    (dict(h=FAKE + 64, ldr=96, ldh=96), "residual or branch itself"), (dict(r=OTHER, h=OTHER + 112, ldr=96, ldh=96), "residual or branch itself"),
    # a binary32 stream over a branch of 16 bits: a row of it is two of the branch's
    (dict(h=FAKE + (1 << 16), stream=2), "residual or branch itself"), (dict(h=FAKE + (1 << 16), stream=2, M=1), "residual or branch itself"),
    (dict(h=FAKE + (1 << 16), stream=2, dtype=1), "residual or branch itself"),
    (dict(r=FAKE, h=FAKE, b=FAKE, stream=2), "residual or branch itself"),
    # in place, and the other rows over them
    (dict(h=FAKE, y=FAKE), "y and normed"), (dict(y=FAKE + 128), "y and normed"), (dict(y=FAKE + (1 << 16) + 3 * 128 + 120), "y and normed"),
    (dict(y=OTHER), "y and normed"), (dict(n=FAKE), "y and normed"), (dict(n=FAKE + (1 << 16)), "y and normed"), (dict(n=OTHER), "y and normed"),
    (dict(n=OTHER + (1 << 16) + 240), "y and normed"),
])
def test_rows_that_share_memory_are_einval(over, needle):
    assert apart(**over) == L.EINVAL
    assert needle in L.load().vdn_fp8_last_error().decode()


@pytest.mark.parametrize("over", [
    # an output over its own input with another stride, or in part
    dict(oq=FAKE, ldoq=520), dict(ok=FAKE + (1 << 16), ldok=264), dict(oq=FAKE + 1024), dict(oq=FAKE + 3 * 1024 + 1008),
    dict(ok=FAKE + (1 << 16) - 496), dict(ldk=272, ldok=272, ok=FAKE + (1 << 16) + 32),
    # over the other side's input or output, also in place
    dict(oq=FAKE + (1 << 16)), dict(ok=FAKE), dict(ok=OTHER), dict(ok=OTHER + 3 * 1024), dict(k=FAKE, oq=FAKE), dict(oq=FAKE, ok=FAKE + 512),
    dict(k=FAKE + 768, ldq=640, ldk=640, oq=FAKE, ldoq=640),
])
def test_rotated_rows_that_share_memory_are_einval(over):
    """Four tokens of 4 + 2 heads of 128 bf16 in places of their own, less what `over` puts elsewhere."""
    assert rope(**{**dict(q=FAKE, k=FAKE + (1 << 16), oq=OTHER, ok=OTHER + (1 << 16)), **over}) == L.EINVAL
    assert "own input" in L.load().vdn_fp8_last_error().decode()
