"""QK preparation for the softmax attention branch, MI355X-native.

Mirrors `_qk_prep` of the reference's `src.models.softmax_attention.kernels`
(kernels.py:8-45): everything between the q (or k) projection and the attention
call -- the per-head RMSNorm (`norm_q` / `norm_k`) and the rotary embedding -- in one
pass over [T, H, d], as `HybridAttention._qkv` uses it at inference
(hybrid_attention.py:128-130). The reference compiles the pair with inductor; here
it is a hand-written HIP kernel (`vdn_fp8_qk_prep`). Numerics follow the compiled
kernel: binary32 throughout, the cos/sin tables rounded to bf16 first
(`cos.to(x.dtype)`), one rounding at the store -- not bitwise with the eager chain,
which rounds after every op, exactly as the reference notes for its own kernel.

`qk_prep_axes` is the same preparation of q and k at positions of several axes (time, height, width), the
angles computed in the kernel.

`cached_attention` is the branch over tokens of earlier calls, kept in 8 bits
(`vdn_fp8.kv_cache`).
"""
from typing import NamedTuple

import torch

from . import _lib
from .fp8_linear import _DTYPES, _aligned16, _ptr, _stream
from .kv_cache import _rows


def qk_prep(t, weight, eps, cos=None, sin=None):
    """RMSNorm over the last dim (weight, eps), then rotary embedding with
    (cos, sin) of shape [T, R] (R <= d; the first R channels rotate as two halves,
    the rest pass through). t bf16 [T, H, d] (heads contiguous; any token stride)
    -> a new contiguous bf16 [T, H, d]."""
    if not t.is_cuda:
        raise ValueError("qk_prep runs on the GPU (a HIP kernel); got a CPU tensor")
    if t.dim() != 3 or t.dtype != torch.bfloat16:
        raise ValueError(f"qk_prep wants a bfloat16 [T, H, d] tensor (got {t.dtype} {tuple(t.shape)})")
    T, H, d = t.shape
    if t.stride(2) != 1 or t.stride(1) != d:
        t = t.contiguous()
    if t.data_ptr() % 16 or t.stride(0) % 8:
        t = t.contiguous()
    dev = t.device
    w = None
    if weight is not None:
        if weight.numel() != d or weight.dtype != torch.bfloat16:
            raise ValueError("weight must be a bfloat16 [d] tensor")
        w = _aligned16(weight.detach().to(dev).reshape(d).contiguous())
    R, ldcs, cs_bf16 = 0, 0, 0
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin go together")
    if cos is not None:
        cos = cos.detach().to(dev).reshape(-1, cos.shape[-1])
        sin = sin.detach().to(dev).reshape(-1, sin.shape[-1])
        if cos.shape != sin.shape or cos.shape[0] != T or cos.dtype != sin.dtype:
            raise ValueError(f"cos/sin must both be [T={T}, R] of one dtype (got {tuple(cos.shape)}, "
                             f"{tuple(sin.shape)})")
        if cos.dtype not in (torch.float32, torch.bfloat16):
            cos, sin = cos.float(), sin.float()
        cos, sin = _aligned16(cos.contiguous()), _aligned16(sin.contiguous())
        R, ldcs, cs_bf16 = cos.shape[1], cos.shape[1], int(cos.dtype == torch.bfloat16)
    out = torch.empty(T, H, d, device=dev, dtype=torch.bfloat16)
    lib = _lib.load()
    _lib.check(lib.vdn_fp8_qk_prep(_ptr(t), T, H, d, t.stride(0), _ptr(w), float(eps), _ptr(cos), _ptr(sin),
                                   R, ldcs, cs_bf16, _ptr(out), H * d, _stream(t)), "qk_prep")
    return out


# The reference's name (softmax_attention/kernels.py:33).
_qk_prep = qk_prep


class RopeAxes(NamedTuple):
    """A rotary embedding over positions of several axes: pair j of a head turns by positions[axis[j]] *
    inv_freq[j]. inv_freq float64 [R / 2] (radians a position), axis int32 [R / 2]; pairs: pair j is elements
    (2 j, 2 j + 1) of the head, else (j, j + R / 2). Elements from R on pass through."""
    inv_freq: torch.Tensor
    axis: torch.Tensor
    pairs: bool = False

    @classmethod
    def make(cls, sections, *, theta=10000.0, shared=False, pairs=False, device="cuda"):
        """`sections` pairs for each axis in turn. Each axis has frequencies of its own, theta ** -(i / n) for its
        n pairs, or with `shared` all take the one sequence theta ** -(j / sum(sections))."""
        sections = [int(n) for n in sections]
        if not sections or min(sections) < 0 or not sum(sections):
            raise ValueError(f"sections must be pairs for each axis (got {sections})")
        at = torch.arange(sum(sections), dtype=torch.float64) / sum(sections) if shared else \
            torch.cat([torch.arange(n, dtype=torch.float64) / max(n, 1) for n in sections])
        axis = torch.repeat_interleave(torch.arange(len(sections), dtype=torch.int32), torch.tensor(sections))
        return cls((float(theta) ** -at).to(device), axis.to(device), bool(pairs))


_POSITIONS = {torch.int32: _lib.POSITION_I32, torch.int64: _lib.POSITION_I64, torch.float32: _lib.POSITION_F32}
_MOST_AXES = 8


def _axes_norm(norm, d, dtype, at, name):
    """(normed, weight, eps) of a norm (weight or None, eps) or None."""
    if norm is None:
        return 0, None, 0.0
    weight, eps = norm
    if weight is None:
        return 1, None, float(eps)
    if weight.numel() != d or weight.dtype is not dtype or weight.get_device() != at:
        raise ValueError(f"{name}'s weight must be a {str(dtype).replace('torch.', '')} [{d}] tensor on the rows' device "
                         f"(got {weight.dtype} {tuple(weight.shape)} on {weight.device})")
    if not weight.is_contiguous() or weight.data_ptr() % 16:
        weight = weight.clone(memory_format=torch.contiguous_format)
    return 1, weight, float(eps)


def qk_prep_axes(query, key, norm_q, norm_k, rope, positions):
    """RMSNorm over each head, then the rotation of `rope` (`RopeAxes`) at `positions` int32, int64 or float32
    [T, axes] (up to 8 axes, or [T] for one), of query [T, q_heads, d] and key [T, heads, d] in one launch. norm_q and
    norm_k are (weight or None, eps), or None for no norm. bf16, float16 or float32 (weights of the same type), d 64,
    128 or 256; heads contiguous, any token stride (column slices of one projection's output are fine).

    Angles are formed in binary64, so that far positions keep their fraction of a turn; cosine and sine are
    binary32, and the result is rounded once. Returns new contiguous query and key."""
    # (the kernel is short for few tokens: each of a tensor's properties is read once, and nothing is called that can be done without)
    dtype, shape, at = query.dtype, query.shape, query.get_device()
    if at >= 0 and torch._C._cuda_getDevice() != at:
        with torch.cuda.device(at):
            return qk_prep_axes(query, key, norm_q, norm_k, rope, positions)
    if dtype not in _DTYPES:
        raise ValueError(f"qk_prep_axes takes bfloat16, float16 or float32 (got {dtype})")
    if len(shape) != 3 or shape[2] not in (64, 128, 256):
        raise ValueError(f"query must be [T, heads, 64, 128 or 256] (got {tuple(shape)})")
    T, q_heads, d = shape
    kinds = (dtype,)
    query, key = _rows(query, None, d, "query", kinds), _rows(key, None, d, "key", kinds)
    of_key = key.shape
    if key.get_device() != at or of_key[0] != T:
        raise ValueError("query and key must have the same rows on one device")
    k_heads = of_key[1]
    inv_freq, axis, pairs = rope
    of_freq = inv_freq.shape
    if inv_freq.dtype is not torch.float64 or axis.dtype is not torch.int32 or len(of_freq) != 1 or axis.shape != of_freq:
        raise ValueError(f"rope must hold float64 inv_freq [R / 2] and int32 axis [R / 2] (got {inv_freq.dtype} {tuple(of_freq)}, "
                         f"{axis.dtype} {tuple(axis.shape)})")
    half = of_freq[0]
    if 2 * half > d or half % (4 if pairs else 8):
        raise ValueError(f"rope must turn at most {d // 2} pairs, a multiple of {4 if pairs else 8} (got {half})")
    kind, of_positions = positions.dtype, positions.shape
    if kind not in _POSITIONS or len(of_positions) not in (1, 2) or of_positions[0] != T:
        raise ValueError(f"positions must be int32, int64 or float32 [{T}, axes] (got {kind} {tuple(of_positions)})")
    axes = of_positions[1] if len(of_positions) == 2 else 1
    if not 1 <= axes <= _MOST_AXES:
        raise ValueError(f"positions of 1 to {_MOST_AXES} axes (got {axes})")
    if positions.get_device() != at or inv_freq.get_device() != at or axis.get_device() != at:
        raise ValueError(f"positions and rope must be on {query.device}")
    positions, inv_freq, axis = positions.contiguous(), inv_freq.contiguous(), axis.contiguous()
    nq, wq, eps_q = _axes_norm(norm_q, d, dtype, at, "norm_q")
    nk, wk, eps_k = _axes_norm(norm_k, d, dtype, at, "norm_k")
    # (empty_like is the shortest way to a new tensor, 1.1 us; of rows that lie apart it makes a contiguous one)
    out_q, out_k = torch.empty_like(query), torch.empty_like(key)
    of_q, of_k = q_heads * d, k_heads * d
    status = _lib.load().vdn_fp8_qk_prep_axes(
        query.data_ptr(), q_heads, query.stride(0) if T > 1 else of_q, key.data_ptr(), k_heads, key.stride(0) if T > 1 else of_k, T, d,
        _DTYPES[dtype], nq, None if wq is None else wq.data_ptr(), eps_q, nk, None if wk is None else wk.data_ptr(), eps_k,
        inv_freq.data_ptr(), axis.data_ptr(), 2 * half, 1 if pairs else 0, positions.data_ptr(), _POSITIONS[kind], axes, axes,
        out_q.data_ptr(), of_q, out_k.data_ptr(), of_k, torch._C._cuda_getCurrentRawStream(at))
    if status:
        _lib.check(status, "qk_prep_axes")
    return out_q, out_k


def _project(x, projections):
    """Every projection of x; fp8 ones share one quantization of it."""
    from .fp8_linear import Fp8Linear, quantize_activation

    if all(isinstance(p, Fp8Linear) for p in projections):
        x_fp8, x_scale = quantize_activation(x)
        return [p.forward_quantized(x_fp8, x_scale, out_dtype=x.dtype) for p in projections]
    return [p(x) for p in projections]


def qkv(x, to_q, to_k, to_v, heads, norm_q, norm_k, rotary_emb=None):
    """The inference body of `HybridAttention._qkv` (hybrid_attention.py:108-137) on this
    library: with fp8 projections x is quantized ONCE and shared by the three GEMMs
    (hybrid_attention.py:118-124), then QK-norm + rope run as one pass each (`_qk_prep`,
    :128-130). x [T, hidden] bf16; to_q/k/v the projection modules (Fp8Linear or any
    callable); norm_q/norm_k modules with `.weight` and `.eps` (RMSNorm); rotary_emb
    (cos, sin) [T, R] or None. Returns (query, key, value, (query_raw, key_raw, value)),
    everything [T, heads, d] -- the raw q/k are the ones the linear branch consumes.
    Without rotary_emb the norms alone run (the same kernel with no rotation), as the
    reference's eager branch would apply them."""
    out = _project(x, (to_q, to_k, to_v))
    query_raw, key_raw, value = (t.unflatten(-1, (heads, -1)) for t in out)
    cos, sin = (None, None) if rotary_emb is None else rotary_emb
    query = qk_prep(query_raw, norm_q.weight, norm_q.eps, cos, sin)
    key = qk_prep(key_raw, norm_k.weight, norm_k.eps, cos, sin)
    return query, key, value, (query_raw, key_raw, value)


def cached_attention(x, to_q, to_k, to_v, norm_q, norm_k, cache, page_table, lengths, *, rotary_emb=None, causal=False,
                     scale=None, q_start=None, max_query=None, top=None, query_block=None, first=1, last=1, rope=None, positions=None,
                     adapters=None, index=None):
    """`qkv` and the attention behind it where earlier tokens are kept in a `KvCache`: one quantization
    of x for the three GEMMs, then QK-norm, rope and the store of k and v in one launch
    (`qk_prep_append`), then `kv_attention` over each sequence's cache, its new tokens included. The cache's
    shape gives the heads; to_q may have more of them (a multiple of the cache's). x [T, hidden] bf16;
    projections, norms and rotary_emb as in `qkv`; page_table, lengths, q_start, max_query, causal and scale
    as in `kv_attention`. With `top`, each block of `query_block` queries attends to the `top` pages
    that `kv_select` finds for it (`first` and `last` as there). What any part refuses is refused before
    anything is stored. Returns [T, q_heads * d], what the output projection takes.

    rope, positions: a `RopeAxes` and each token's positions, in place of rotary_emb (`qk_prep_axes`, then the store).
    adapters, index: the low-rank adapters of to_q, to_k and to_v (three `Adapters`, or None for one without) and
    each token's own (`adapter_add`)."""
    from .kv_cache import check_attention, kv_append, kv_attention, kv_select, qk_prep_append

    d = cache.k.shape[-1]
    if (rope is None) != (positions is None) or (rope is not None and rotary_emb is not None):
        raise ValueError("rope and positions go together, in place of rotary_emb")
    if (adapters is None) != (index is None) or (adapters is not None and len(adapters) != 3):
        raise ValueError("adapters (of to_q, to_k and to_v) and index go together")
    if adapters is not None and any(isinstance(bank, torch.Tensor) for bank in adapters):   # (one bank has three parts as well)
        raise ValueError("adapters must be three banks, of to_q, to_k and to_v (or None for one without); got the tensors of one")
    out = _project(x, (to_q, to_k, to_v))
    if adapters is not None:
        from .fp8_linear import Fp8Linear
        from .lora import adapter_add

        # in place where the output is a new tensor for certain (another callable may return x, or a buffer of its own)
        out = [t if bank is None else adapter_add(x, t, bank, index, out=t if isinstance(p, Fp8Linear) else None)
               for t, p, bank in zip(out, (to_q, to_k, to_v), adapters)]
    query, key, value = (t.unflatten(-1, (-1, d)) for t in out)
    check_attention(query, cache, page_table, lengths, scale=scale, q_start=q_start, max_query=max_query, top=top, query_block=query_block,
                    first=first, last=last)
    if rope is not None:
        query, key = qk_prep_axes(query, key, (norm_q.weight, norm_q.eps), (norm_k.weight, norm_k.eps), rope, positions)
        kv_append(key, value, cache, page_table, lengths, q_start=q_start)
    else:
        cos, sin = (None, None) if rotary_emb is None else rotary_emb
        query = qk_prep_append(query, key, value, (norm_q.weight, norm_q.eps), (norm_k.weight, norm_k.eps), cache, page_table, lengths,
                               cos=cos, sin=sin, q_start=q_start)
    blocks = None
    if top is not None:
        blocks = kv_select(query, cache, page_table, lengths, top, query_block=query_block, first=first, last=last, causal=causal,
                           q_start=q_start)
    out = kv_attention(query, cache, page_table, lengths, scale=scale, causal=causal, q_start=q_start, max_query=max_query, blocks=blocks,
                       query_block=query_block)
    return out.flatten(1)
