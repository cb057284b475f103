"""What is measured of the key/value cache in 8 bits: storing a chunk's keys and values (after
QK-norm and rope, or as they are), attention over the cache for chunks, prompts and single
tokens, the choice of the cache pages that a block of queries attends to, and attention over
those pages alone.

Sizes are those of the two DiTs that the workloads name (40 or 56 heads of 128; latent frames of
1560 tokens, 21 of them 32760) and of encoded prompts (800 to 3485 tokens), next to generic
grouped heads of 64, 128 and 256.

A cache page holds 64 tokens of every key/value head: e4m3 codes k [pages, H, 64, d] and
v [pages, H, d, 64], their scales (powers of two) [pages, H], and the page's mean key.
`lengths` counts a sequence's tokens in the cache, those of the call at hand included.
"""
import math
import os
import sys

import torch

own = False

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vdn-minimax-h3_amd"))

DEV = "cuda:0"
BF16 = torch.bfloat16
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
DTYPES = {"bf16": BF16, "f16": torch.float16, "f32": torch.float32}
PAGE = 64
EPS = 1e-6
FRAME = 1560                    # tokens of one latent frame (30 x 52 patches)
LEAST_E, MOST_E = -100, 120     # exponents of a page's scale

# (query heads, key/value heads) of the DiTs, and generic groups
HEADS = ((40, 40), (56, 56), (40, 8), (32, 8), (32, 4), (16, 2), (12, 12))

# a drawn case costs no more than the largest listed ones
MOST_SCORES = 3120 * 32760 * 40          # query-key pairs of all heads, at 128 elements each
MOST_CACHE = 8 * 98304 * 8 * 128         # elements of k
MOST_NEW = 3120 * 40 * 128               # elements of k stored by a call


def listed():
    return [
        # a step of 16 sequences, one token each: QK-norm, rope and the store in one call; latency counts
        {"name": "store_step", "kind": "prep", "B": 16, "n": 1, "len": 4000, "spread": 3900, "Hq": 40, "H": 8, "d": 128, "R": 128},
        # two latent frames behind nine others
        {"name": "store_frames", "kind": "prep", "B": 1, "n": 2 * FRAME, "len": 11 * FRAME, "spread": 0, "Hq": 40, "H": 40, "d": 128, "R": 128},
        # prompts of different lengths, float16, stored as they are
        {"name": "store_prompts_f16", "kind": "store", "lens": "3485,1299,821,800,64,1", "news": "3485,1299,821,800,64,1",
         "Hq": 16, "H": 16, "d": 64, "dtype": "f16"},
        # one token behind a prompt: the smallest attention
        {"name": "attn_step_prompt", "kind": "attn", "B": 1, "n": 1, "len": 821, "spread": 0, "Hq": 40, "H": 8, "d": 128, "dtype": "bf16"},
        # one token each behind eight long caches
        {"name": "attn_step_long", "kind": "attn", "B": 8, "n": 1, "len": 131072, "spread": 60000, "Hq": 40, "H": 8, "d": 128, "dtype": "bf16"},
        # two latent frames that attend to all 21: the largest
        {"name": "attn_frames", "kind": "attn", "B": 1, "n": 2 * FRAME, "len": 21 * FRAME, "spread": 0, "Hq": 40, "H": 40, "d": 128, "dtype": "bf16"},
        # ragged causal prompts with grouped heads, with the log-sum-exp that joins them to another part
        {"name": "attn_prompts", "kind": "attn", "lens": "3485,1299,821,800", "news": "3485,1299,821,800", "Hq": 32, "H": 8, "d": 128,
         "dtype": "bf16", "causal": True, "lse": True},
        # a few tokens of a small float16 model at once (a draft's check), odd lengths
        {"name": "attn_few_f16", "kind": "attn", "B": 3, "n": 77, "len": 5001, "spread": 2111, "Hq": 12, "H": 12, "d": 64, "dtype": "f16", "causal": True},
        # the pages that each block of 128 queries of two frames attends to
        {"name": "select_frames", "kind": "select", "B": 1, "n": 2 * FRAME, "len": 21 * FRAME, "spread": 0, "Hq": 40, "H": 40, "d": 128,
         "dtype": "bf16", "block": 128, "top": 64},
        # the pages that one token each of eight long caches attends to
        {"name": "select_step", "kind": "select", "B": 8, "n": 1, "len": 131072, "spread": 60000, "Hq": 40, "H": 8, "d": 128,
         "dtype": "bf16", "block": 1, "top": 64, "causal": True},
        # attention over those pages alone
        {"name": "sparse_frames", "kind": "sparse", "B": 1, "n": 2 * FRAME, "len": 21 * FRAME, "spread": 0, "Hq": 40, "H": 40, "d": 128,
         "dtype": "bf16", "block": 128, "top": 64},
        {"name": "sparse_step", "kind": "sparse", "B": 8, "n": 1, "len": 131072, "spread": 60000, "Hq": 40, "H": 8, "d": 128,
         "dtype": "bf16", "block": 1, "top": 64, "causal": True},
    ]


def _log(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    kind = rng.choice(("prep", "store", "attn", "attn", "attn", "select", "sparse", "sparse"))
    Hq, H = rng.choice(HEADS)
    d = rng.choice((64, 128, 128, 128, 256))
    c = {"kind": kind, "Hq": Hq, "H": H, "d": d}
    if kind in ("prep", "store"):
        most = max(2, min(8 * FRAME, MOST_NEW // (H * d)))
        B = _log(rng, 1, 32)
        if rng.random() < 0.5:
            n = _log(rng, 1, max(2, most // B))
            c.update(B=B, n=n, len=n + _log(rng, 1, min(20000, MOST_CACHE // (2 * B * H * d))), spread=0)
            c["spread"] = rng.randint(0, c["len"] - n)
        else:
            news = [_log(rng, 1, max(2, most // B)) for _ in range(B)]
            c.update(news=",".join(map(str, news)), lens=",".join(str(n + rng.choice((0, _log(rng, 1, min(9000, MOST_CACHE // (2 * B * H * d)))))) for n in news))
        if kind == "prep":
            c["R"] = rng.choice((0, d // 2, d, d))
        else:
            c["dtype"] = rng.choice(("bf16", "f16", "f32"))
        return c
    c["dtype"] = rng.choice(("bf16", "bf16", "f16"))
    c["causal"] = rng.random() < 0.5
    pairs = MOST_SCORES // Hq * 128 // max(d, 128)
    if kind == "attn":
        form = rng.choice(("step", "chunk", "ragged"))
        if form == "step":
            B = _log(rng, 1, 64)
            most = min(200000, MOST_CACHE // (B * H * d))
            c.update(B=B, n=1, len=_log(rng, 64, most))
            c["spread"] = rng.randint(0, c["len"] - 1)
        elif form == "chunk":
            B = _log(rng, 1, 8)
            n = _log(rng, 2, 4000 // B)
            c.update(B=B, n=n, len=n + _log(rng, 1, max(2, min(32760, pairs // (B * n), MOST_CACHE // (B * H * d)) - n)),
                     spread=0)
            c["spread"] = rng.randint(0, c["len"] - n)
        else:
            B = rng.randint(2, 6)
            most = min(3485, math.isqrt(pairs // B))
            news = [_log(rng, 1, most) for _ in range(B)]
            c.update(news=",".join(map(str, news)), lens=",".join(str(n + rng.choice((0, 0, rng.randint(1, 300)))) for n in news))
        c["lse"] = rng.random() < 0.5
        return c
    if rng.random() < 0.5:
        B = _log(rng, 1, 16)
        c.update(B=B, n=1, len=_log(rng, 1000, min(200000, MOST_CACHE // (B * H * d))), block=1, spread=0)
    else:
        n = _log(rng, 65, 2 * FRAME)
        c.update(B=1, n=n, len=n + _log(rng, 1000, min(32760, pairs // n) - n), block=rng.choice((128, 128, 256)), spread=0)
    c["spread"] = rng.randint(0, (c["len"] - c["n"]) // 2)
    c["top"] = min(_log(rng, 4, 128), max(3, -(-c["len"] // PAGE) // 2))
    return c


def _plan(case):
    """(tokens in the cache, tokens of the call) of each sequence."""
    if "news" in case:
        return [int(x) for x in case["lens"].split(",")], [int(x) for x in case["news"].split(",")]
    B = case["B"]
    return [case["len"] - (b * 7919 * 613) % (case["spread"] + 1) for b in range(B)], [case["n"]] * B


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------

def _scale_exponent(amax):
    """The least e with amax <= 448 * 2^e."""
    mantissa, exponent = torch.frexp(amax)
    e = exponent - 9 + (mantissa > 0.875).to(exponent.dtype)
    return torch.where(amax > 0, e, LEAST_E).clamp(LEAST_E, MOST_E)


def _e8m0(e):
    return (e + 127).to(torch.uint8).view(E8M0)


def _encode(x, e):
    return (x * torch.exp2(-e.float())).to(E4M3)


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(int(seed))

    def normal(*shape, std=1.0, dtype=BF16):
        return torch.empty(*shape, device=DEV).normal_(0.0, std, generator=g).to(dtype)

    lens, news = _plan(case)
    B, T, Hq, H, d = len(lens), sum(news), case["Hq"], case["H"], case["d"]
    dtype = DTYPES[case.get("dtype", "bf16")]
    need = [-(-n // PAGE) for n in lens]
    pages, W = sum(need) + 3, max(need)
    # the pool's pages in the order in which sequences that grow in turn come by them
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((B, W), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    s = {"table": table, "lengths": torch.tensor(lens, dtype=torch.int32, device=DEV), "ragged": "news" in case, "n": max(news),
         "q_start": None, "causal": case.get("causal", False)}
    if s["ragged"]:
        s["q_start"] = torch.tensor([sum(news[:b]) for b in range(B + 1)], dtype=torch.int32, device=DEV)
    # keys of neighbouring tokens (a page's) are alike; channels differ in size
    channel = torch.exp(0.5 * torch.empty(d, device=DEV).normal_(generator=g))

    def codes(std):
        x = torch.empty(pages, H, PAGE, d, device=DEV).normal_(0.0, std, generator=g)
        if std > 0.5:
            x += torch.empty(pages, H, 1, d, device=DEV).normal_(0.0, 0.7, generator=g)
            x *= channel
        e = _scale_exponent(x.abs().amax((2, 3)))
        return _encode(x, e[:, :, None, None]), e

    k, ek = codes(0.8)
    v, ev = codes(0.3)
    mean = (k.float().sum(2) / PAGE * torch.exp2(ek.float())[:, :, None]).to(BF16)
    s["cache"] = (k, v.transpose(2, 3).contiguous(), _e8m0(ek), _e8m0(ev), mean)
    if case["kind"] in ("prep", "store"):
        # the projections of one fused linear, as column slices of its output
        qkv = normal(T, (Hq + 2 * H) * d, dtype=dtype)
        s["query"], s["key"], s["value"] = (t.unflatten(1, (-1, d)) for t in qkv.split((Hq * d, H * d, H * d), 1))
    else:
        s["query"] = (normal(T, Hq, d) * (channel.reciprocal() * 2.0)).to(dtype)
    if case["kind"] == "prep":
        s["norm_q"], s["norm_k"] = ((1.0 + normal(d, std=0.1)).to(BF16), EPS), ((1.0 + normal(d, std=0.1)).to(BF16), EPS)
        s["cos"] = s["sin"] = None
        if case["R"]:
            freq = 10000.0 ** (-torch.arange(case["R"] // 2, device=DEV) * 2.0 / case["R"])
            at = torch.cat([torch.arange(n - m, n, device=DEV) for n, m in zip(lens, news)])
            angle = at[:, None].double() * freq.double()
            s["cos"], s["sin"] = torch.cat([angle, angle], 1).cos().float(), torch.cat([angle, angle], 1).sin().float()
    s["block"], s["top"], s["lse"] = case.get("block"), case.get("top"), case.get("lse", False)
    if case["kind"] == "sparse":
        # distinct pages in ascending order, the last one (the newest tokens) among them
        rows = sum(-(-n // s["block"]) for n in news)
        have = torch.tensor([need[b] for b, n in enumerate(news) for _ in range(-(-n // s["block"]))], device=DEV)
        lot = torch.rand(rows, H, W, generator=g, device=DEV)
        page = torch.arange(W, device=DEV)
        lot = torch.where(page == have[:, None, None] - 1, 2.0, torch.where(page < have[:, None, None], lot, -1.0))
        score, pick = lot.topk(s["top"], 2)
        pick = torch.where(score >= 0, pick, W).sort(2).values
        s["blocks"] = torch.where(pick < W, pick, -1).to(torch.int32)
    s["kind"] = case["kind"]
    return s


# ---------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------

def _tokens(s):
    """Each token's sequence, its position in the cache, and each sequence's first position."""
    T, B = s["query"].shape[0], s["lengths"].numel()
    start = s["q_start"] if s["ragged"] else torch.arange(B + 1, device=DEV, dtype=torch.int32) * (T // B)
    seq = torch.searchsorted(start[1:], torch.arange(T, device=DEV, dtype=torch.int32), right=True)
    first = s["lengths"] - (start[1:] - start[:-1])
    return seq, (first[seq] + torch.arange(T, device=DEV) - start[seq]).long(), first.long(), start.long()


def _store(s, key, value):
    k, v, ks, vs, mean = s["cache"]
    seq, pos, first, _ = _tokens(s)
    page = s["table"][seq, pos // PAGE].long()
    off = pos % PAGE
    lengths = s["lengths"].long()
    # pages that the call begins inside of keep their earlier tokens, at a scale no smaller
    kept = (first % PAGE > 0).nonzero()[:, 0]
    kept_page = s["table"][kept, first[kept] // PAGE].long()
    before = torch.arange(PAGE, device=DEV) < (first[kept] % PAGE)[:, None]
    tail = s["table"][torch.arange(len(lengths), device=DEV), (lengths - 1) // PAGE].long()
    count = torch.full((k.shape[0],), PAGE, device=DEV)
    count[tail] = (lengths - 1) % PAGE + 1
    touched = torch.zeros(k.shape[0], dtype=torch.bool, device=DEV)
    touched[page] = True
    new = []
    for x, codes, scale in ((key, k, ks), (value, v.transpose(2, 3), vs)):
        x = x.float()
        amax = torch.zeros(scale.shape, device=DEV).index_reduce_(0, page, x.abs().amax(2), "amax")
        e = _scale_exponent(amax)
        old = scale.view(torch.uint8).int() - 127
        e[kept_page] = torch.maximum(e[kept_page], old[kept_page])
        e = torch.where(touched[:, None], e, old)
        shifted = _encode(codes[kept_page].float(), (e - old)[kept_page][:, :, None, None])
        kept_codes = torch.where(before[:, None, :, None], shifted.view(torch.uint8), codes[kept_page].view(torch.uint8))
        codes.view(torch.uint8)[kept_page] = kept_codes
        codes.view(torch.uint8)[page, :, off] = _encode(x, e[page][:, :, None]).view(torch.uint8)
        scale.view(torch.uint8).copy_(e + 127)
        new.append(e)
    at = touched.nonzero()[:, 0]
    inside = torch.arange(PAGE, device=DEV) < count[at][:, None]
    total = (k[at].float() * inside[:, None, :, None]).sum(2)
    mean[at] = (total / count[at][:, None, None] * torch.exp2(new[0][at].float())[:, :, None]).to(BF16)


def _norm_rope(x, norm, cos, sin):
    weight, eps = norm
    x = x.double()
    n = x / (x.square().mean(2, keepdim=True) + eps).sqrt() * weight.double()
    if cos is None:
        return n.to(BF16)
    R = cos.shape[1]
    c, s = (t.to(BF16).double()[:, None] for t in (cos, sin))
    lo, hi = n[..., :R // 2], n[..., R // 2:R]
    turned = torch.cat([lo * c[..., :R // 2] - hi * s[..., :R // 2], hi * c[..., R // 2:] + lo * s[..., R // 2:], n[..., R:]], 2)
    return turned.to(BF16)


def _items(s, block):
    """The queries as items of `block` tokens (a sequence's last one padded): tokens [I, block], which
    of them are real, their positions, each item's sequence."""
    seq, pos, first, start = _tokens(s)
    n = start[1:] - start[:-1]
    rows = (n + block - 1) // block
    end = rows.cumsum(0)
    item = torch.arange(s["items"], device=DEV)
    of = torch.searchsorted(end, item, right=True)
    at = (item - (end - rows)[of])[:, None] * block + torch.arange(block, device=DEV)
    return (start[of][:, None] + at).clamp(max=len(seq) - 1), at < n[of][:, None], first[of][:, None] + at, of


def _decode(codes, scale):
    return codes.float() * scale.float()[..., None, None]


def _attend(s):
    """Softmax attention of each item of queries over its pages: all of its sequence, or those listed."""
    k, v, ks, vs, _ = s["cache"]
    query, table, lengths = s["query"], s["table"], s["lengths"]
    H, d = k.shape[1], k.shape[3]
    block = s["block"] if s["kind"] == "sparse" else s["n"]
    B, T = lengths.numel(), query.shape[0]
    s["items"] = s["blocks"].shape[0] if s["kind"] == "sparse" else B
    token, real, pos, of = _items(s, block)
    I, n, G = token.shape[0], token.shape[1], query.shape[1] // H
    pages = table[of].long()
    if s["kind"] == "sparse":
        index = s["blocks"].long()                                                        # [I, H, top]
        slot = pages.gather(1, index.clamp(min=0).flatten(1)).view(index.shape)
        head = torch.arange(H, device=DEV)[:, None]
        keys, values = _decode(k[slot, head], ks[slot, head]), _decode(v[slot, head], vs[slot, head])   # [I, H, top, ...]
        where = index[..., None] * PAGE + torch.arange(PAGE, device=DEV)                  # positions of the keys
        seen = ((index >= 0)[..., None] & (where < lengths[of][:, None, None, None])).flatten(2)
        where = where.flatten(2)
    else:
        slot = pages.clamp(min=0)
        keys = _decode(k[slot], ks[slot]).transpose(1, 2)                                 # [I, H, W, 64, d]
        values = _decode(v[slot], vs[slot]).transpose(1, 2)
        where = torch.arange(pages.shape[1] * PAGE, device=DEV).expand(I, 1, -1)
        seen = where < lengths[of][:, None, None]
    keys = keys.reshape(I, H, -1, d)
    values = values.transpose(3, 4).reshape(I, H, -1, d)
    q = query[token].view(I, n, H, G, d).permute(0, 2, 1, 3, 4).reshape(I, H, n * G, d).float() * d ** -0.5
    score = (q @ keys.transpose(2, 3)).view(I, H, n, G, -1)
    mask = seen[:, :, None]
    if s["causal"]:
        mask = mask & (where[:, :, None] <= pos[:, None, :, None])
    score.masked_fill_(~mask[:, :, :, None], -math.inf)
    top = score.amax(4, keepdim=True)
    top = torch.where(top.isinf(), 0.0, top)
    score.sub_(top).exp_()
    total = score.sum(4, keepdim=True)
    out = (score.view(I, H, n * G, -1) @ values).view(I, H, n, G, d)
    out = torch.where(total > 0, out / total, 0.0).to(query.dtype).permute(0, 2, 1, 3, 4).reshape(I, n, H * G, d)
    lse = (top + total.log())[..., 0].permute(0, 2, 1, 3).reshape(I, n, H * G)
    back = torch.empty_like(query)
    back[token[real]] = out[real]
    if not s["lse"]:
        return back
    lse_back = torch.empty(T, H * G, device=DEV)
    lse_back[token[real]] = lse[real]
    return back, lse_back


def _select(s):
    """Each item's best pages by the product of its queries' sum with the pages' mean keys."""
    mean, table, lengths, query = s["cache"][4], s["table"], s["lengths"].long(), s["query"]
    H, d = mean.shape[1], mean.shape[2]
    start = _tokens(s)[3]
    B, block = lengths.numel(), s["block"]
    s["items"] = B * -(-s["n"] // block)
    token, real, pos, of = _items(s, block)
    I, W = token.shape[0], table.shape[1]
    q = (query[token].double() * real[..., None, None]).sum(1).view(I, H, -1, d).sum(2).float().double()
    score = torch.einsum("ihd,iwhd->ihw", q, mean[table[of].long().clamp(min=0)].double())
    last = torch.where(real, pos, -1).amax(1) if s["causal"] else lengths[of] - 1
    have = (last // PAGE + 1)[:, None, None]
    page = torch.arange(W, device=DEV)
    score = torch.where((page == 0) | (page == have - 1), math.inf, score)
    score = torch.where(page < have, score, -math.inf)
    best, pick = score.sort(dim=2, descending=True, stable=True)
    pick = torch.where(best[..., :s["top"]] > -math.inf, pick[..., :s["top"]], W).sort(2).values
    return torch.where(pick < W, pick, -1).to(torch.int32)


def run(s):
    if own:
        import vdn_fp8
        cache = vdn_fp8.KvCache(*s["cache"])
        if s["kind"] == "prep":
            query = vdn_fp8.qk_prep_append(s["query"], s["key"], s["value"], s["norm_q"], s["norm_k"], cache, s["table"], s["lengths"],
                                           cos=s["cos"], sin=s["sin"], q_start=s["q_start"])
            return (query, *cache)
        if s["kind"] == "store":
            vdn_fp8.kv_append(s["key"], s["value"], cache, s["table"], s["lengths"], q_start=s["q_start"])
            return tuple(cache)
        if s["kind"] == "select":
            return vdn_fp8.kv_select(s["query"], cache, s["table"], s["lengths"], s["top"], query_block=s["block"], first=1, last=1,
                                     causal=s["causal"], q_start=s["q_start"])
        return vdn_fp8.kv_attention(s["query"], cache, s["table"], s["lengths"], causal=s["causal"], q_start=s["q_start"],
                                    max_query=s["n"], blocks=s["blocks"] if s["kind"] == "sparse" else None,
                                    query_block=s["block"], return_lse=s["lse"])
    if s["kind"] == "prep":
        query, key = _norm_rope(s["query"], s["norm_q"], s["cos"], s["sin"]), _norm_rope(s["key"], s["norm_k"], s["cos"], s["sin"])
        _store(s, key, s["value"])
        return (query, *s["cache"])
    if s["kind"] == "store":
        _store(s, s["key"], s["value"])
        return s["cache"]
    return _select(s) if s["kind"] == "select" else _attend(s)


# ---------------------------------------------------------------------------------------
# work and 64-bit results
# ---------------------------------------------------------------------------------------

def _pairs(case):
    """Query-key pairs of one head, and the tokens of the cache that are read for each key/value head."""
    lens, news = _plan(case)
    pairs = seen = 0
    for n, m in zip(lens, news):
        if case["kind"] == "sparse":
            blocks = -(-m // case["block"])
            kept = min(case["top"] * PAGE, n)
            pairs += m * kept
            seen += min(n, blocks * kept)
        else:
            pairs += m * n - (m * (m - 1) // 2 if case.get("causal") else 0)
            seen += n
    return pairs, seen


def work(case):
    lens, news = _plan(case)
    T, Hq, H, d = sum(news), case["Hq"], case["H"], case["d"]
    size = {"bf16": 2, "f16": 2, "f32": 4}[case.get("dtype", "bf16")]
    if case["kind"] in ("prep", "store"):
        pages = sum(-(-n // PAGE) - (n - m) // PAGE for n, m in zip(lens, news))
        moved = T * H * d * (2 * size + 2) + pages * H * (2 * d + 2)
        if case["kind"] == "prep":
            moved += T * Hq * d * 4 + T * case["R"] * 8
        return {"bytes": moved, "flops": 10 * T * (Hq + 2 * H) * d}
    if case["kind"] == "select":
        rows = sum(-(-m // case["block"]) for m in news)
        pages = [-(-n // PAGE) for n in lens]
        return {"bytes": T * Hq * d * size + sum(pages) * H * d * 2 + rows * H * case["top"] * 4,
                "flops": 2 * H * d * sum(w * -(-m // case["block"]) for w, m in zip(pages, news)) + T * Hq * d}
    pairs, seen = _pairs(case)
    return {"bytes": 2 * T * Hq * d * size + seen * H * 2 * d, "flops": 4 * pairs * Hq * d}


def exact(case, seed):
    s = prepare(case, seed)
    lens, news = _plan(case)
    k, v, ks, vs, mean = s["cache"]
    H, d, G = case["H"], case["d"], case["Hq"] // case["H"]
    query = s["query"].double()
    if case["kind"] == "select":
        return None       # whole numbers
    if case["kind"] in ("prep", "store"):
        def prep(x, norm):
            x = x.double()
            if case["kind"] == "store":
                return x
            x = x * torch.rsqrt(x.pow(2).sum(-1, keepdim=True) / d + norm[1]) * norm[0].double()
            R = case["R"]
            if R:
                z = torch.complex(x[..., :R // 2], x[..., R // 2:R]) * torch.complex(
                    s["cos"].to(BF16).double(), s["sin"].to(BF16).double())[:, None, :R // 2]
                x = torch.cat([z.real, z.imag, x[..., R:]], -1)
            return x
        query = prep(s["query"], s.get("norm_q"))
        key = prep(s["key"], s.get("norm_k"))
        # what is stored: bf16 keys in e4m3 steps; here by the pages, one sequence after the other
        key = key.to(BF16).double() if case["kind"] == "prep" else key
        out = [[c.double() for c in (k, v.transpose(2, 3))], [t.double() for t in (ks, vs)], mean.double()]
        at = 0
        for b, (n, m) in enumerate(zip(lens, news)):
            slots = s["table"][b].tolist()
            for w in range((n - m) // PAGE, -(-n // PAGE)):
                lo, hi = max(0, n - m - w * PAGE), min(PAGE, n - w * PAGE)
                first = at + w * PAGE + lo - (n - m)
                for side, x in enumerate((key, s["value"].double())):
                    new = x[first:first + hi - lo].transpose(0, 1)                      # [H, tokens, d]
                    codes, scale = out[0][side][slots[w]], out[1][side][slots[w]]
                    size = torch.exp2(torch.ceil(torch.log2(new.abs().amax((1, 2)) / 448)).clamp(LEAST_E, MOST_E))
                    if lo:
                        bigger = torch.maximum(size, scale)
                        codes[:, :lo] = (codes[:, :lo] * (scale / bigger)[:, None, None]).float().to(E4M3).double()
                        size = bigger
                    codes[:, lo:hi] = (new / size[:, None, None]).float().to(E4M3).double()
                    scale.copy_(size)
                    if side == 0:
                        out[2][slots[w]] = codes[:, :hi].mean(1) * size[:, None]
            at += m
        caches = [out[0][0], out[0][1].transpose(2, 3).contiguous(), out[1][0], out[1][1], out[2]]
        return [query, *caches] if case["kind"] == "prep" else caches
    out = torch.zeros(query.shape, dtype=torch.float64, device=DEV)
    lse = torch.full(query.shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    at = row = 0
    for b, (n, m) in enumerate(zip(lens, news)):
        W = -(-n // PAGE)
        slots = s["table"][b, :W].long()
        block = case["block"] if case["kind"] == "sparse" else max(1, min(m, 4096))
        for i in range(0, m, block):
            hi = min(m, i + block)
            for h in range(H):
                pick = s["blocks"][row, h] if case["kind"] == "sparse" else torch.arange(W, device=DEV)
                pick = pick[pick >= 0].long()
                K = k[slots[pick], h].double() * ks[slots[pick], h].double()[:, None, None]
                V = v[slots[pick], h].double() * vs[slots[pick], h].double()[:, None, None]
                place = (pick[:, None] * PAGE + torch.arange(PAGE, device=DEV)).flatten()
                live = place[None] < n
                if case.get("causal"):
                    live = live & (place[None] <= n - m + torch.arange(i, hi, device=DEV)[:, None])
                q = query[at + i:at + hi, h * G:(h + 1) * G].transpose(0, 1)            # [G, rows, d]
                x = (q.reshape(-1, d) @ K.flatten(0, 1).T / math.sqrt(d)).view(G, hi - i, -1).masked_fill(~live, -math.inf)
                z = torch.logsumexp(x, 2)
                p = torch.exp(x - z[..., None]).nan_to_num(0.0)
                out[at + i:at + hi, h * G:(h + 1) * G] = (p.flatten(0, 1) @ V.transpose(1, 2).flatten(0, 1)).view(G, hi - i, d).transpose(0, 1)
                lse[at + i:at + hi, h * G:(h + 1) * G] = z.T
            row += 1
        at += m
    return (out, lse) if case.get("lse") else out
