"""Keys and values kept in 8 bits, and the attention that reads them, on MI355X.

The reference attends within one call (`HybridAttention`, src/models/hybrid_attention.py:108-137,
and src/models/softmax_attention); here the keys and values of earlier calls -- the frames
before a chunk, a prompt, the tokens of a causal text model -- stay in a cache of e4m3 codes, half
of their bf16 size, with a power-of-two scale for each page of 64 tokens and each head:

  qk_prep_append   QK-norm and rope of q and k (`qk_prep`) and the store of k and v, one launch
  kv_append        the store alone, for keys that are ready (bf16, float16 or float32)
  kv_attention     softmax attention over a sequence's cache, for chunks, prompts and single tokens
  kv_select        the pages that a block of queries attends to, by a cheap score;
                   `kv_attention(..., blocks=...)` then reads those alone

A call takes a batch of sequences: `page_table` int32 [B, W] lists the pool pages of each (entries
outside the pool, such as -1, are pages that are not there), `lengths` int32 [B] counts each one's
tokens in the cache, the call's own INCLUDED, and the call's rows are packed: T / B for each sequence,
or rows [q_start[b], q_start[b + 1]) of sequence b with `q_start` int32 [B + 1]. They are a sequence's
last positions. Nothing is read back to the host, so every call can be captured into a graph and
replayed with other lengths and tables in the same buffers.

Everything runs on torch's current stream of the tensors' device, in hand-written kernels
(include/vdn_fp8.h); there is no CPU path and no autograd.
"""
import contextlib
import ctypes
from typing import NamedTuple, Optional

import torch

from . import _lib
from .fp8_linear import _DTYPES, FP8_DTYPE, _aligned16, _ptr, _stream, check_index_range

KV_PAGE = 64
SCALE_DTYPE = torch.float8_e8m0fnu


class KvCache(NamedTuple):
    """The pool: k e4m3 [pages, heads, 64, d], v e4m3 [pages, heads, d, 64] (a page's tokens
    contiguous), k_scale and v_scale e8m0 [pages, heads] (code * scale is the value), k_mean
    bf16 [pages, heads, d], the mean key of each page (None: not kept, and no `kv_select`)."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor
    k_mean: Optional[torch.Tensor] = None

    @classmethod
    def empty(cls, pages, heads, head_dim, device, means=True):
        """A pool of `pages` pages; what it holds before the first store is never read."""
        if head_dim not in (64, 128, 256):
            raise ValueError(f"the cache takes heads of 64, 128 or 256 elements (got {head_dim})")
        return cls(torch.empty(pages, heads, KV_PAGE, head_dim, device=device, dtype=FP8_DTYPE),
                   torch.empty(pages, heads, head_dim, KV_PAGE, device=device, dtype=FP8_DTYPE),
                   torch.empty(pages, heads, device=device, dtype=torch.uint8).view(SCALE_DTYPE),
                   torch.empty(pages, heads, device=device, dtype=torch.uint8).view(SCALE_DTYPE),
                   torch.empty(pages, heads, head_dim, device=device, dtype=torch.bfloat16) if means else None)


def _cache(cache, device):
    """The C struct of a cache, checked. (Each of a tensor's properties read once: 0.1 us a piece.)"""
    k, v, ks, vs, mean = cache
    shape = k.shape
    if k.dtype is not FP8_DTYPE or len(shape) != 4 or shape[2] != KV_PAGE:
        raise ValueError(f"cache.k must be float8_e4m3fn [pages, heads, {KV_PAGE}, d] (got {k.dtype} {tuple(shape)})")
    P, H, _, d = shape
    if v.dtype is not FP8_DTYPE or v.shape != (P, H, d, KV_PAGE):
        raise ValueError(f"cache.v must be float8_e4m3fn [{P}, {H}, {d}, {KV_PAGE}] (got {v.dtype} {tuple(v.shape)})")
    each = (P, H)
    if ks.dtype is not SCALE_DTYPE or vs.dtype is not SCALE_DTYPE or ks.shape != each or vs.shape != each:
        raise ValueError(f"cache.k_scale and v_scale must be float8_e8m0fnu [{P}, {H}]")
    at = _index(device)
    here = (k.get_device() == at and v.get_device() == at and ks.get_device() == at and vs.get_device() == at and
            k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous())
    mean_ptr = None
    if mean is not None:
        if mean.dtype is not torch.bfloat16 or mean.shape != (P, H, d):
            raise ValueError(f"cache.k_mean must be bfloat16 [{P}, {H}, {d}]")
        here = here and mean.get_device() == at and mean.is_contiguous()
        mean_ptr = mean.data_ptr()
    if not here:
        raise ValueError(f"the cache's tensors must be contiguous, on {device}")
    return _lib.KvCacheStruct(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), mean_ptr, P, H, d)


def _heads(cache):
    """Heads and their size (whatever else is wrong with the cache, `_cache` says)."""
    shape = cache.k.shape
    return (shape[1], shape[3]) if len(shape) == 4 else (1, 0)


def _index(device):
    """What get_device() gives for tensors on `device` (cheaper to compare than devices are)."""
    return device.index if device.type == "cuda" else -1


def _batch(page_table, lengths, q_start, tokens, pages, device):
    """The C struct of a batch, checked (and what it points to, to be kept until the launch)."""
    shape = page_table.shape
    if page_table.dtype is not torch.int32 or len(shape) != 2:
        raise ValueError("page_table must be int32 [B, W] with unit column stride")
    B, W = shape
    ld, unit = page_table.stride()
    if unit != 1 and W > 1:
        raise ValueError("page_table must be int32 [B, W] with unit column stride")
    if lengths.dtype is not torch.int32 or lengths.shape != (B,) or not lengths.is_contiguous():
        raise ValueError(f"lengths must be a contiguous int32 [{B}] tensor")
    at = _index(device)
    here = page_table.get_device() == at and lengths.get_device() == at
    start = None
    if q_start is not None:
        if q_start.dtype is not torch.int32 or q_start.shape != (B + 1,) or not q_start.is_contiguous():
            raise ValueError(f"q_start must be a contiguous int32 [{B + 1}] tensor")
        here = here and q_start.get_device() == at
        start = q_start.data_ptr()
    if not here:
        raise ValueError(f"page_table, lengths and q_start must be on {device}")
    if tokens and not B:
        raise ValueError(f"{tokens} tokens of an empty batch")
    if start is None and B and tokens % B:
        raise ValueError(f"{tokens} tokens do not divide among {B} sequences: pass q_start")
    check_index_range(lengths, W * KV_PAGE + 1, "lengths")
    if q_start is not None:
        check_index_range(q_start, tokens + 1, "q_start")
    return _lib.KvBatchStruct(page_table.data_ptr(), ld if B > 1 else W, W, lengths.data_ptr(), start, B, tokens)


def _not_rows(t, heads, d, name, dtypes):
    names = ", ".join(str(x).replace("torch.", "") for x in dtypes)
    return ValueError(f"{name} must be a {names} [T, {'heads' if heads is None else heads}, {d}] tensor "
                      f"(got {t.dtype} {tuple(t.shape)})")


def _rows(t, heads, d, name, dtypes):
    """[T, heads, d] with contiguous heads on the GPU, 16-byte aligned rows; a copy where it is not."""
    if not t.is_cuda:
        raise ValueError(f"the cache's kernels run on the GPU; {name} is a CPU tensor")
    shape = t.shape
    if len(shape) != 3 or t.dtype not in dtypes or shape[2] != d or (heads is not None and shape[1] != heads):
        raise _not_rows(t, heads, d, name, dtypes)
    token, head, unit = t.stride()
    if unit != 1 or head != d or token % 8 or token < shape[1] * d or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _ld(t):
    rows, heads, d = t.shape
    return t.stride(0) if rows > 1 else max(t.stride(0), heads * d)


_HERE = contextlib.nullcontext()


def _on(device):
    """The tensors' device as the current one, for a launch (nothing where it is already)."""
    return _HERE if torch._C._cuda_getDevice() == device.index else torch.cuda.device(device)


def kv_append(key, value, cache, page_table, lengths, *, q_start=None):
    """Stores key and value [T, heads, d] (bf16, float16 or float32; any token stride) at their
    positions in `cache`: sequence b's n rows go to positions lengths[b] - n .. lengths[b] - 1.

    A page's scale is the least power of two that brings its largest finite element to 448 or less,
    and no smaller than before where the page keeps earlier tokens (their codes then move to
    the new scale); each element is rounded once; infinities and NaN are stored as NaN. Positions
    below 0, beyond the table, or in a page that is not there are left out; a page may receive
    tokens of one sequence only, at one place of its table."""
    heads, d = _heads(cache)
    key = _rows(key, heads, d, "key", tuple(_DTYPES))
    value = _rows(value, heads, d, "value", (key.dtype,))
    dev, T = key.device, key.shape[0]
    if value.device != dev or value.shape[0] != T:
        raise ValueError("key and value must have the same rows on one device")
    c = _cache(cache, dev)
    b = _batch(page_table, lengths, q_start, T, c.pages, dev)
    with _on(dev):
        _lib.check(_lib.load().vdn_fp8_kv_append(c, b, key.data_ptr(), _ld(key), value.data_ptr(), _ld(value), _DTYPES[key.dtype],
                                                 _stream(key)), "kv_append")


def _norm(norm, d, device, name):
    weight, eps = norm
    if weight is None:
        return None, float(eps)
    if weight.shape == (d,) and weight.dtype == torch.bfloat16 and weight.device == device and weight.stride(0) == 1:
        return _aligned16(weight), float(eps)
    if weight.numel() != d or weight.dtype != torch.bfloat16:
        raise ValueError(f"{name}'s weight must be a bfloat16 [{d}] tensor")
    return _aligned16(weight.detach().to(device).reshape(d).contiguous()), float(eps)


def qk_prep_append(query, key, value, norm_q, norm_k, cache, page_table, lengths, *, cos=None, sin=None, q_start=None):
    """`qk_prep` of query and of key -- the RMSNorm over each head, norm_q = (weight, eps) and norm_k
    likewise, then the rotation by cos, sin [T, R] -- and `kv_append` of that key and the value, in one
    launch with the same bits. query bf16 [T, q_heads, d], key and value bf16 [T, heads, d] (column
    slices of one projection's output are fine). Returns the prepared query, a new [T, q_heads, d]."""
    heads, d = _heads(cache)
    bf16 = (torch.bfloat16,)
    query = _rows(query, None, d, "query", bf16)
    key, value = _rows(key, heads, d, "key", bf16), _rows(value, heads, d, "value", bf16)
    dev, T, q_heads = query.device, query.shape[0], query.shape[1]
    if key.device != dev or value.device != dev or key.shape[0] != T or value.shape[0] != T:
        raise ValueError("query, key and value must have the same rows on one device")
    wq, eps_q = _norm(norm_q, d, dev, "norm_q")
    wk, eps_k = _norm(norm_k, d, dev, "norm_k")
    R = ldcs = bf16_table = 0
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin go together")
    if cos is not None:
        at = _index(dev)
        if cos.dim() != 2 or cos.get_device() != at or sin.dim() != 2 or sin.get_device() != at:
            cos, sin = cos.detach().to(dev).reshape(-1, cos.shape[-1]), sin.detach().to(dev).reshape(-1, sin.shape[-1])
        shape, kind = cos.shape, cos.dtype
        if sin.shape != shape or shape[0] != T or sin.dtype is not kind:
            raise ValueError(f"cos/sin must both be [T={T}, R] of one dtype (got {tuple(cos.shape)}, {tuple(sin.shape)})")
        if kind is not torch.float32 and kind is not torch.bfloat16:
            cos, sin = cos.float(), sin.float()
        cos, sin = _aligned16(cos.contiguous()), _aligned16(sin.contiguous())
        R = ldcs = shape[1]
        bf16_table = int(kind is torch.bfloat16)
    c = _cache(cache, dev)
    b = _batch(page_table, lengths, q_start, T, c.pages, dev)
    out = torch.empty(T, q_heads, d, device=dev, dtype=torch.bfloat16)
    with _on(dev):
        _lib.check(_lib.load().vdn_fp8_qk_prep_append(
            c, b, query.data_ptr(), q_heads, _ld(query), key.data_ptr(), _ld(key), value.data_ptr(), _ld(value), _ptr(wq), eps_q, _ptr(wk),
            eps_k, _ptr(cos), _ptr(sin), R, ldcs, bf16_table, out.data_ptr(), q_heads * d, _stream(query)), "qk_prep_append")
    return out


_QUERY_DTYPES = (torch.bfloat16, torch.float16)


def _block_rows(T, B, query_block, ragged):
    """Rows of a block list (include/vdn_fp8.h, vdn_fp8_kv_attention)."""
    if query_block == 1:
        return T
    return T // query_block + B if ragged else B * -(-(T // B) // query_block) if B else 0


_WORKSPACES = {}


def _workspace(entry, c, b, args, dev):
    """Bytes of workspace of a call, asked of the library once per shape."""
    key = (entry, dev.index, c.pages > 0, c.heads, c.head_dim, b.max_pages, b.batch, b.tokens, b.q_start is None, args)
    got = _WORKSPACES.get(key)
    if got is None:
        if len(_WORKSPACES) >= 4096:
            _WORKSPACES.clear()
        size = ctypes.c_int64(0)
        _lib.check(getattr(_lib.load(), entry)(c, b, *args, ctypes.byref(size)), entry)
        got = _WORKSPACES[key] = size.value
    return got


def _check_scale(scale, d):
    scale = float(d ** -0.5 if scale is None else scale)
    if not 0 < scale <= 2e38:   # (NaN too)
        raise ValueError(f"scale must be positive, and 2e38 at most (got {scale})")
    return scale


def _check_choice(group, top, query_block, first, last):
    if query_block < 1 or (query_block > 1 and query_block * group % 128):
        raise ValueError(f"query_block must be 1, or such that query_block * {group} (heads of a group) is a multiple of 128 (got {query_block})")
    if top < 1 or first < 0 or last < 0 or first + last > top:
        raise ValueError(f"top must be at least 1 and hold the first {first} and last {last} pages (got {top})")


def check_attention(query, cache, page_table, lengths, *, scale=None, q_start=None, max_query=None, top=None, query_block=None, first=1, last=1):
    """Raises what `kv_attention` of these arguments would -- with `top`, over the pages of `kv_select` --
    and launches nothing: for callers that store before they attend."""
    dev, (T, q_heads, _) = query.device, query.shape
    c = _cache(cache, dev)
    heads, d = c.heads, c.head_dim
    if q_heads % heads or not q_heads:
        raise ValueError(f"{q_heads} query heads for a cache of {heads}")
    if (top is None) != (query_block is None):
        raise ValueError("top and query_block go together")
    _check_scale(scale, d)
    if top is not None:
        if cache.k_mean is None:
            raise ValueError("top needs a cache that keeps k_mean")
        _check_choice(q_heads // heads, top, query_block, first, last)
    if max_query is not None and max_query < 0:
        raise ValueError(f"max_query must not be negative (got {max_query})")
    if not query.is_cuda:
        raise ValueError("the cache's kernels run on the GPU; query is a CPU tensor")
    if query.dtype not in _QUERY_DTYPES or query.shape[2] != d:
        raise _not_rows(query, None, d, "query", _QUERY_DTYPES)
    # what the library refuses by sizes
    b = _batch(page_table, lengths, q_start, T, c.pages, dev)
    with _on(dev):
        _workspace("vdn_fp8_kv_attention_workspace_size", c, b, (q_heads, int(max_query or 0), top or 0, query_block or 0), dev)
        if top is not None:
            _workspace("vdn_fp8_kv_select_workspace_size", c, b, (q_heads, query_block), dev)


def kv_attention(query, cache, page_table, lengths, *, scale=None, causal=False, q_start=None, max_query=None, blocks=None,
                 query_block=None, return_lse=False):
    """Softmax attention of query [T, q_heads, d] (bf16 or float16; any token stride) over the cached
    tokens of each row's sequence -- with `causal` those up to the row's own position -- as a new
    [T, q_heads, d] of query's type. q_heads is a multiple of the cache's heads; scale defaults to
    d ** -0.5. A row that sees no token (an empty sequence, pages that are not there) gets zeros.

    return_lse: also log(sum exp(scores)), float32 [T, q_heads] (-inf for such a row), by which
    results over different keys join.
    max_query: with q_start, the rows of the longest sequence, if known: a few rows per sequence take
    another kernel (in which a sequence of more rows than that takes longer).
    blocks, query_block: int32 [rows, heads, top] from `kv_select` (or a caller's own list; entries
    outside the sequence are skipped, one listed twice counts twice): only those pages are read."""
    heads, d = _heads(cache)
    query = _rows(query, None, d, "query", _QUERY_DTYPES)
    dev, (T, q_heads, _) = query.device, query.shape
    if q_heads % heads or not q_heads:
        raise ValueError(f"{q_heads} query heads for a cache of {heads}")
    c = _cache(cache, dev)
    b = _batch(page_table, lengths, q_start, T, c.pages, dev)
    top = 0
    if blocks is not None:
        if query_block is None:
            raise ValueError("blocks need query_block, the queries that share a list")
        if query_block < 1:
            raise ValueError(f"query_block must be at least 1 (got {query_block})")
        rows = _block_rows(T, b.batch, query_block, q_start is not None)
        if blocks.dim() != 3 or blocks.shape[:2] != (rows, heads) or blocks.dtype != torch.int32 or blocks.device != dev or not blocks.shape[2]:
            raise ValueError(f"blocks must be int32 [{rows}, {heads}, top] on {dev} (got {blocks.dtype} {tuple(blocks.shape)})")
        blocks = blocks.contiguous()
        top = blocks.shape[2]
    out = torch.empty(T, q_heads, d, device=dev, dtype=query.dtype)
    lse = torch.empty(T, q_heads, device=dev, dtype=torch.float32) if return_lse else None
    size = (q_heads, int(max_query or 0), top, query_block if top else 0)
    with _on(dev):
        n = _workspace("vdn_fp8_kv_attention_workspace_size", c, b, size, dev)
        ws = torch.empty(n, device=dev, dtype=torch.uint8) if n else None
        _lib.check(_lib.load().vdn_fp8_kv_attention(
            c, b, query.data_ptr(), _DTYPES[query.dtype], q_heads, _ld(query), size[1], _check_scale(scale, d),
            int(bool(causal)), _ptr(blocks), top, size[3], out.data_ptr(), _ptr(lse), _ptr(ws), n, _stream(query)), "kv_attention")
    return (out, lse) if return_lse else out


def kv_select(query, cache, page_table, lengths, top, *, query_block, first=1, last=1, causal=False, q_start=None):
    """The pages that each block of `query_block` consecutive queries of a sequence attends to, for each
    of the cache's heads: the `top` best by the product of the block's summed queries with the pages'
    mean keys, the first `first` and last `last` of those that the block sees among them, ties to
    the lower page. Returns int32 [rows, heads, top], ascending, then -1, for `kv_attention`.

    query_block is 1 (each query its own pages) or a number of which query_block * q_heads / heads is
    a multiple of 128. rows: T for query_block = 1; B * ceil(T / B / query_block) without q_start,
    T // query_block + B with it (sequence b's blocks from q_start[b] // query_block + b on; rows that
    no block takes hold -1)."""
    heads, d = _heads(cache)
    query = _rows(query, None, d, "query", _QUERY_DTYPES)
    dev, (T, q_heads, _) = query.device, query.shape
    if q_heads % heads or not q_heads:
        raise ValueError(f"{q_heads} query heads for a cache of {heads}")
    if cache.k_mean is None:
        raise ValueError("kv_select needs a cache that keeps k_mean")
    _check_choice(q_heads // heads, top, query_block, first, last)
    c = _cache(cache, dev)
    b = _batch(page_table, lengths, q_start, T, c.pages, dev)
    blocks = torch.empty(_block_rows(T, b.batch, query_block, q_start is not None), heads, top, device=dev, dtype=torch.int32)
    with _on(dev):
        n = _workspace("vdn_fp8_kv_select_workspace_size", c, b, (q_heads, query_block), dev)
        ws = torch.empty(n, device=dev, dtype=torch.uint8) if n else None
        _lib.check(_lib.load().vdn_fp8_kv_select(
            c, b, query.data_ptr(), _DTYPES[query.dtype], q_heads, _ld(query), int(bool(causal)), top, first, last, query_block,
            blocks.data_ptr(), _ptr(ws), n, _stream(query)), "kv_select")
    return blocks
