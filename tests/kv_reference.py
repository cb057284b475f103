"""Plain 64-bit implementations of the 8-bit key/value cache's operators, on the CPU, for its
tests: storing, attention with its error bound, and the choice of pages. Written from the
definitions in include/vdn_fp8.h, one sequence, head and token at a time."""
import math

import numpy as np
import torch

PAGE = 64
E4M3 = torch.float8_e4m3fn
E8M0 = torch.float8_e8m0fnu


def decode(codes, exponents):
    """e4m3 [..., n, m] with exponents [...] -> float64 values."""
    return codes.double() * torch.exp2(exponents.double())[..., None, None]


def encode(x, e):
    """e4m3(x 2^-e), one rounding (x float32-representable, the product exact)."""
    return (x.double() * 2.0 ** -float(e)).float().to(E4M3)


def exponent(x):
    """Least e with amax <= 448 * 2^e over the finite elements, in [-100, 120]."""
    x = x.double()
    x = x[torch.isfinite(x)].abs()
    amax = float(x.max()) if x.numel() else 0.0
    if amax == 0.0:
        return -100
    m, e = math.frexp(amax)
    return max(-100, min(120, e - 9 + (m > 0.875)))


class Cache:
    """k [P, H, 64, d] and v [P, H, d, 64] codes, exponents [P, H], means [P, H, d] (bf16)."""

    def __init__(self, pages, heads, d, seed=0):
        g = torch.Generator().manual_seed(seed)
        # what an earlier owner left: any bytes, NaN codes among them
        self.k = torch.randint(0, 256, (pages, heads, PAGE, d), generator=g, dtype=torch.uint8).view(E4M3)
        self.v = torch.randint(0, 256, (pages, heads, d, PAGE), generator=g, dtype=torch.uint8).view(E4M3)
        self.ek = torch.randint(-9, 9, (pages, heads), generator=g)
        self.ev = torch.randint(-9, 9, (pages, heads), generator=g)
        self.mean = torch.randn(pages, heads, d, generator=g).to(torch.bfloat16)

    def tensors(self, device):
        s = [(e + 127).to(torch.uint8).view(E8M0).to(device) for e in (self.ek, self.ev)]
        return [self.k.to(device), self.v.to(device), *s, self.mean.to(device)]

    def copy(self):
        c = Cache.__new__(Cache)
        c.k, c.v, c.ek, c.ev, c.mean = (t.clone() for t in (self.k, self.v, self.ek, self.ev, self.mean))
        return c


def spans(starts, lengths):
    """(sequence, its first row, rows, position of the first row) of each sequence."""
    return [(b, starts[b], starts[b + 1] - starts[b], lengths[b] - (starts[b + 1] - starts[b])) for b in range(len(lengths))]


def append(cache, key, value, table, lengths, starts):
    """Stores key, value [T, H, d]; table: lists of pages; starts: row offsets of the sequences."""
    P, H = cache.ek.shape
    for b, row, n, first in spans(starts, lengths):
        end = min(lengths[b], len(table[b]) * PAGE)
        for w in range(max(first, 0) // PAGE, -(-end // PAGE)):
            lo, hi = max(0, first - w * PAGE), min(PAGE, end - w * PAGE)
            page = int(table[b][w])
            if lo >= hi or not 0 <= page < P:
                continue
            rows = slice(row + w * PAGE + lo - first, row + w * PAGE + hi - first)
            for h in range(H):
                for x, codes, e in ((key, cache.k[page, h], cache.ek), (value, cache.v[page, h].T, cache.ev)):
                    new = exponent(x[rows, h])
                    if lo:
                        old = int(e[page, h])
                        new = max(new, old)
                        codes.view(torch.uint8)[:lo] = encode(codes[:lo].double(), new - old).view(torch.uint8)
                    codes.view(torch.uint8)[lo:hi] = encode(x[rows, h], new).view(torch.uint8)
                    e[page, h] = new
                total = cache.k[page, h, :hi].double().sum(0).float() / torch.tensor(float(hi))
                cache.mean[page, h] = (total * 2.0 ** int(cache.ek[page, h])).to(torch.bfloat16)


def listed_rows(starts, block, ragged):
    """Row of the block list where each sequence's blocks begin, and the rows in all."""
    B, T = len(starts) - 1, starts[-1]
    if block == 1:
        return list(starts[:-1]), T
    if ragged:
        return [starts[b] // block + b for b in range(B)], T // block + B
    each = -(-(T // B) // block)
    return [b * each for b in range(B)], B * each


def attend(cache, q, table, lengths, starts, scale, causal=False, blocks=None, block=None, ragged=False):
    """(out, lse, bound of out's error before its rounding, bound of lse's) in float64; q [T, Hq, d]."""
    T, Hq, d = q.shape
    P, H = cache.ek.shape
    G = Hq // H
    q = q.double()
    out, lse = torch.zeros(T, Hq, d, dtype=torch.float64), torch.full((T, Hq), -math.inf, dtype=torch.float64)
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    base = listed_rows(starts, block, ragged)[0] if blocks is not None else None
    K, V = decode(cache.k, cache.ek), decode(cache.v, cache.ev).transpose(2, 3)
    for b, row, n, first in spans(starts, lengths):
        end = max(0, min(lengths[b], len(table[b]) * PAGE))
        chunk = block if blocks is not None else max(n, 1)
        for i in range(0, n, chunk):
            rows = torch.arange(i, min(n, i + chunk))
            for h in range(H):
                pages = range(-(-end // PAGE)) if blocks is None else [
                    int(w) for w in blocks[base[b] + i // chunk, h] if 0 <= w < -(-end // PAGE)]
                pages = [w for w in pages if 0 <= int(table[b][w]) < P]
                place = torch.tensor([w * PAGE + t for w in pages for t in range(PAGE)], dtype=torch.long)
                keep = place < end
                place = place[keep]
                if not len(place):
                    continue
                k = torch.cat([K[table[b][w], h] for w in pages])[keep]
                v = torch.cat([V[table[b][w], h] for w in pages])[keep]
                seen = torch.ones(len(rows), len(place), dtype=torch.bool)
                if causal:
                    seen = place[None] <= first + rows[:, None]
                for gh in range(h * G, (h + 1) * G):
                    x = q[row + rows, gh]
                    s = torch.where(seen, scale * (x @ k.T), -math.inf)
                    live = seen.any(1)
                    z = torch.logsumexp(s, 1)
                    p = torch.where(seen, torch.exp(s - torch.where(live, z, 0.0)[:, None]), 0.0)
                    o = p @ v.nan_to_num(0)
                    # (a NaN value reaches the rows that see it; a NaN score makes its whole row NaN)
                    o = torch.where((seen.double() @ v.isnan().double()) > 0, math.nan, o)
                    o = torch.where(live[:, None], o, 0.0)
                    out[row + rows, gh], lse[row + rows, gh] = o, torch.where(live, z, -math.inf)
                    # Weights are rounded to binary16: 2^-11 of each, and 2^-25 where it is below that
                    # type's normal range, next to a largest one of at least 1 (in units of the largest
                    # value times 2^e, so at most 2^-24 of the largest value for each token). Scores:
                    # products are exact; their sum is d / 16 sums one after another, at most 16, of 16
                    # products each (four more levels), so at most 20 roundings (2^-23 each, should they
                    # truncate) of the magnitudes' sum, and two more for the scale: below 2^-18 of |q|.|k|.
                    es = scale * 2.0 ** -18 * (x.abs() @ k.abs().nan_to_num(0).T).amax(1)
                    a = p.nan_to_num(0) @ v.nan_to_num(0).abs()
                    tol[row + rows, gh] = (2.0 ** -11 + 2.0 ** -18 + 2 * es)[:, None] * a + len(place) * 2.0 ** -24 * float(v.abs().nan_to_num(0).max())
                    tol_lse[row + rows, gh] = 2 * es + 2.0 ** -20 + 2.0 ** -22 * z.abs().nan_to_num(0, 0, 0)
    return out, lse, tol, tol_lse


def select(cache, q, table, lengths, starts, top, block, first, last, causal, ragged=False):
    """Block lists, numpy int32 [rows, H, top]."""
    T, Hq, d = q.shape
    P, H = cache.ek.shape
    base, total = listed_rows(starts, block, ragged)
    got = np.full((total, H, top), -1, np.int32)
    mean = cache.mean.double()
    for b, row, n, at in spans(starts, lengths):
        for i in range(0, n, block):
            hi = min(n, i + block)
            end = max(0, min(lengths[b], len(table[b]) * PAGE))
            if causal:
                end = min(end, max(0, at + hi))
            have = -(-end // PAGE)
            x = q[row + i:row + hi].double().reshape(hi - i, H, Hq // H, d).sum((0, 2)).float().double()
            for h in range(H):
                order = []
                for w in range(have):
                    page = int(table[b][w])
                    if not 0 <= page < P:
                        continue
                    score = float(x[h] @ mean[page, h])
                    if math.isnan(score):
                        score = -math.inf
                    forced = w < first or w >= have - last
                    order.append((0 if forced else 1, -score, w))
                pick = sorted(w for _, _, w in sorted(order)[:top])
                got[base[b] + i // block, h, :len(pick)] = pick
    return got
