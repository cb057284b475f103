"""What is measured of a block that serves many requests at once, from the residual stream to attention's
queries and keys: the residual's addition with the root-mean-square norm and the 8-bit rows of the next
projection; low-rank adapters of many requests beside a shared projection; QK-norm and rotary positions
with several axes.

Sizes are those of the two DiTs that the workloads name (hidden 5120 and 5376, 40 or 56 heads of 128, frames
of 30 x 52 tokens, 21 of them 32760; feed-forward 13824), of encoded prompts (800 to 3485 tokens), and
generic grouped heads of 64, 128 and 256.
"""
import math
import os
import random
import sys

import torch

own = False

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vdn-minimax-h3_amd"))

DEV = "cuda:0"
E4M3 = torch.float8_e4m3fn
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-6
TOKENS = 32760                  # 21 latent frames of 30 x 52

# (query heads, key heads) of the DiTs, and generic groups
HEADS = ((40, 40), (56, 56), (40, 8), (32, 8), (32, 4), (16, 2), (12, 12))

# a drawn case costs no more than the largest listed ones
MOST_NORM = TOKENS * 5376 * 7           # bytes
MOST_ADAPT = TOKENS * (5120 + 2 * 15360) * 2
MOST_ROPE = TOKENS * 80 * 128 * 4


def listed():
    return [
        # a step of 16 sequences: the residual's addition, the norm and the codes, with the normed rows that adapters read; latency counts
        {"name": "norm_step", "kind": "norm", "M": 16, "K": 5120, "stream": "bf16", "dtype": "bf16", "gate": False, "affine": False, "rows": 1,
         "normed": True},
        # all tokens of a video, gated and modulated by the row of their frame
        {"name": "norm_frames", "kind": "norm", "M": TOKENS, "K": 5376, "stream": "bf16", "dtype": "bf16", "gate": True, "affine": True, "rows": 21,
         "normed": False},
        # a prompt, the residual stream in float32
        {"name": "norm_prompt_f32", "kind": "norm", "M": 3485, "K": 5120, "stream": "f32", "dtype": "bf16", "gate": False, "affine": False,
         "rows": 1, "normed": True},
        # a short prompt of a float16 model, an odd width
        {"name": "norm_odd_f16", "kind": "norm", "M": 821, "K": 4104, "stream": "f16", "dtype": "f16", "gate": True, "affine": True, "rows": 5,
         "normed": False},
        # one token of one request: the smallest
        {"name": "adapt_one", "kind": "adapt", "news": "1", "L": 4, "used": 1, "R": 16, "K": 5120, "N": 5120, "dtype": "bf16"},
        # a step of 32 requests with 12 adapters, some requests without one
        {"name": "adapt_step", "kind": "adapt", "news": ",".join(["1"] * 32), "L": 16, "used": 12, "R": 32, "K": 5120, "N": 7168, "dtype": "bf16"},
        # prompts of several requests, float16, adapters of rank 128
        {"name": "adapt_prompts_f16", "kind": "adapt", "news": "3485,1299,821,800,64,1", "L": 8, "used": 4, "R": 128, "K": 5376, "N": 7168,
         "dtype": "f16"},
        # a video each for four requests, at the fused QKV projection: the largest
        {"name": "adapt_frames", "kind": "adapt", "news": "12480,9360,6240,4680", "L": 4, "used": 3, "R": 64, "K": 5120, "N": 15360, "dtype": "bf16"},
        # a step of 16 sequences at far positions, three axes
        {"name": "rope_step", "kind": "rope", "T": 16, "Hq": 40, "H": 8, "d": 128, "sections": "24,20,20", "pairs": False, "norm": True,
         "pos": "int32", "far": 100000, "dtype": "bf16"},
        # all tokens of a video
        {"name": "rope_frames", "kind": "rope", "T": TOKENS, "Hq": 40, "H": 40, "d": 128, "sections": "22,21,21", "pairs": True, "norm": True,
         "pos": "int32", "far": 0, "dtype": "bf16"},
        # images of a float16 model without norms, two axes, part of the head rotates
        {"name": "rope_images_f16", "kind": "rope", "T": 5329, "Hq": 16, "H": 16, "d": 64, "sections": "12,12", "pairs": False, "norm": False,
         "pos": "int64", "far": 0, "dtype": "f16"},
        # ragged prompts in float32, times in seconds (fractions)
        {"name": "rope_prompts_f32", "kind": "rope", "T": 6405, "Hq": 32, "H": 8, "d": 128, "sections": "16,24,24", "pairs": False, "norm": True,
         "pos": "float32", "far": 3000, "dtype": "f32"},
    ]


def _log(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    kind = rng.choice(("norm", "adapt", "adapt", "rope"))
    if kind == "norm":
        stream, dtype = rng.choice((("bf16", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("f32", "f32")))
        K = rng.choice((4096, 5120, 5376, 7168, 8 * rng.randint(8, 1024)))
        normed = rng.random() < 0.5
        M = _log(rng, 1, min(40000, MOST_NORM // (K * (2 * SIZES[stream] + SIZES[dtype] * (1 + normed) + 1))))
        return {"kind": kind, "M": M, "K": K, "stream": stream, "dtype": dtype, "gate": rng.random() < 0.5, "affine": rng.random() < 0.5,
                "rows": _log(rng, 1, 40), "normed": normed}
    if kind == "adapt":
        K, N = rng.choice((4096, 5120, 5376, 16 * rng.randint(16, 500))), rng.choice((4096, 5120, 7168, 13824, 15360, 8 * rng.randint(32, 1000)))
        L = _log(rng, 1, 32)
        used = rng.randint(1, L)
        most = min(TOKENS, MOST_ADAPT // ((K + 2 * N) * 2))
        if rng.random() < 0.5:
            news = [1] * _log(rng, 1, 256)           # a step: one token of each request
        else:
            B = _log(rng, 1, 16)
            news = [_log(rng, 1, most // B) for _ in range(B)]
        return {"kind": kind, "news": ",".join(map(str, news)), "L": L, "used": used, "R": rng.choice((16, 16, 32, 48, 64, 128)), "K": K, "N": N,
                "dtype": rng.choice(("bf16", "bf16", "f16"))}
    Hq, H = rng.choice(HEADS)
    d = rng.choice((64, 128, 128, 128, 256))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    half = rng.choice((d // 2, d // 2, d // 4))
    axes = rng.randint(1, 4)
    cuts = sorted(rng.sample(range(1, half), axes - 1))
    sections = [b - a for a, b in zip([0] + cuts, cuts + [half])]
    return {"kind": kind, "T": _log(rng, 1, min(40000, MOST_ROPE // ((Hq + H) * d * 2 * SIZES[dtype]))), "Hq": Hq, "H": H, "d": d,
            "sections": ",".join(map(str, sections)), "pairs": rng.random() < 0.5, "norm": rng.random() < 0.7,
            "pos": rng.choice(("int32", "int32", "int64", "float32")), "far": rng.choice((0, _log(rng, 1, 1000000))), "dtype": dtype}


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------

def _adapters_of(case):
    """Each request's adapter, those from `used` on having none."""
    rng = random.Random(len(case["news"]) * 1009 + case["L"])
    news = [int(n) for n in case["news"].split(",")]
    which = [b if b < case["used"] else rng.randint(0, case["used"]) for b in range(len(news))]
    rng.shuffle(which)
    return news, [a if a < case["used"] else -1 for a in which]


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(int(seed))

    def normal(*shape, std=1.0, dtype=torch.float32):
        return torch.empty(*shape, device=DEV).normal_(0.0, std, generator=g).to(dtype)

    dtype = DTYPES[case["dtype"]]
    s = {"kind": case["kind"]}
    if case["kind"] == "norm":
        M, K, rows = case["M"], case["K"], case["rows"]
        channel = torch.exp(0.5 * normal(K))            # channels of a residual stream differ in size
        s["residual"] = (normal(M, K) * channel * 3.0).to(DTYPES[case["stream"]])
        s["branch"] = normal(M, K, dtype=dtype)
        s["weight"] = (1.0 / channel + normal(K, std=0.05)).to(dtype)
        s["gate"] = normal(rows, K, std=0.7, dtype=dtype) if case["gate"] else None
        s["scale"], s["shift"] = (normal(rows, K, std=0.3, dtype=dtype) for _ in "ab") if case["affine"] else (None, None)
        # frames one after the other
        s["indices"] = (torch.arange(M, device=DEV) * rows // M).to(torch.int32) if case["gate"] or case["affine"] else None
        s["normed"] = case["normed"]
    elif case["kind"] == "adapt":
        news, which = _adapters_of(case)
        T, L, R, K, N = sum(news), case["L"], case["R"], case["K"], case["N"]
        s["x"], s["base"] = normal(T, K, dtype=dtype), normal(T, N, dtype=dtype)
        s["a"], s["b"] = normal(L, R, K, std=K ** -0.5, dtype=dtype), normal(L, N, R, std=0.5 * R ** -0.5, dtype=dtype)
        s["alpha"] = 0.5 + torch.rand(L, generator=g, device=DEV)
        # the batch may come in any order of requests: each seed has another adapter for each
        turn = int(torch.randint(0, case["used"], (1,), generator=g, device=DEV))
        each = torch.tensor([(a + turn) % case["used"] if a >= 0 else -1 for a in which], dtype=torch.int32)
        s["index"] = each.repeat_interleave(torch.tensor(news)).to(DEV)
        total = [sum(n for n, a in zip(news, which) if a == u) for u in range(case["used"])]
        s["most"], s["used"] = max(1, *total), case["used"]
    else:
        T, Hq, H, d = case["T"], case["Hq"], case["H"], case["d"]
        sections = [int(n) for n in case["sections"].split(",")]
        qkv = normal(T, (Hq + 2 * H) * d, dtype=dtype)      # the projections of one fused linear
        s["query"], s["key"], _ = (t.unflatten(1, (-1, d)) for t in qkv.split((Hq * d, H * d, H * d), 1))
        s["norm_q"], s["norm_k"] = (((1.0 + normal(d, std=0.1)).to(dtype), EPS) if case["norm"] else None for _ in "qk")
        s["freq"] = torch.cat([10000.0 ** (-torch.arange(n, device=DEV, dtype=torch.float64) / n) for n in sections])
        s["axis"] = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections)).to(torch.int32).to(DEV)
        at = torch.arange(T, device=DEV, dtype=torch.float64)
        grid = [at // 1560, at // 52 % 30, at % 52, at % 7][: len(sections)]
        p = torch.stack(grid, 1) + case["far"] + torch.randint(0, 50, (1, len(sections)), generator=g, device=DEV)
        s["positions"] = (p * 24.0 / 7.0).float() if case["pos"] == "float32" else p.to(getattr(torch, case["pos"]))
        s["pairs"] = case["pairs"]
    return s


# ---------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------

def _add_norm_quantize(s):
    r, b = s["residual"].float(), s["branch"].float()
    index = None if s["indices"] is None else s["indices"].long()
    if s["gate"] is not None:
        b = s["gate"].float()[index] * b
    hidden = (r + b).to(s["residual"].dtype)
    h = hidden.float()
    weight, eps = s["weight"].float(), EPS
    n = h * (1.0 / (h.square().mean(1, keepdim=True) + eps).sqrt()) * weight
    if s["scale"] is not None:
        n = n * (1.0 + s["scale"].float()[index]) + s["shift"].float()[index]
    scale = (n.abs().amax(1, keepdim=True) / 448.0).clamp_min(1e-12)
    codes = (n / scale).clamp(-448.0, 448.0).to(E4M3)
    return (hidden, codes, scale, n.to(s["branch"].dtype)) if s["normed"] else (hidden, codes, scale)


def _adapter_add(s):
    x, index, used = s["x"], s["index"].long(), s["used"]
    T, K = x.shape
    # the tokens of each adapter side by side, every adapter's padded to the most
    order = torch.sort(index, stable=True).indices
    sorted_index = index[order]
    first = torch.searchsorted(sorted_index, torch.arange(-1, used, device=DEV))
    place = torch.arange(T, device=DEV) - first[sorted_index + 1]
    slot = torch.where(sorted_index < 0, used * s["most"], sorted_index * s["most"] + place)
    rows = torch.zeros(used * s["most"] + 1, K, device=DEV)
    rows[slot] = torch.where(sorted_index < 0, 0.0, 1.0)[:, None] * x[order].float()
    rows = rows[:-1].view(used, s["most"], K)
    low = rows @ s["a"][:used].float().transpose(1, 2).contiguous()
    delta = low @ s["b"][:used].float().transpose(1, 2).contiguous() * s["alpha"][:used, None, None]
    out = s["base"].float()
    has = sorted_index >= 0
    taken = delta.flatten(0, 1)[slot.clamp(max=used * s["most"] - 1)]
    out[order] += torch.where(has[:, None], taken, 0.0)
    return out.to(s["base"].dtype)


def _rope(x, norm, cos, sin, pairs):
    n = x.float()
    if norm is not None:
        weight, eps = norm
        n = n * (1.0 / (n.square().mean(2, keepdim=True) + eps).sqrt()) * weight.float()
    half = cos.shape[1]
    if pairs:
        lo, hi = n[..., 0:2 * half:2], n[..., 1:2 * half:2]
        turned = torch.stack([lo * cos[:, None] - hi * sin[:, None], hi * cos[:, None] + lo * sin[:, None]], 3).flatten(2)
    else:
        lo, hi = n[..., :half], n[..., half:2 * half]
        turned = torch.cat([lo * cos[:, None] - hi * sin[:, None], hi * cos[:, None] + lo * sin[:, None]], 2)
    return torch.cat([turned, n[..., 2 * half:]], 2).to(x.dtype)


def _qk_prep_axes(s):
    angle = s["positions"].double()[:, s["axis"].long()] * s["freq"]
    cos, sin = angle.cos().float(), angle.sin().float()
    return _rope(s["query"], s["norm_q"], cos, sin, s["pairs"]), _rope(s["key"], s["norm_k"], cos, sin, s["pairs"])


def run(s):
    if own:
        import vdn_fp8
        if s["kind"] == "norm":
            return vdn_fp8.add_norm_quantize(s["residual"], s["branch"], s["weight"], EPS, gate=s["gate"], scale=s["scale"], shift=s["shift"],
                                             indices=s["indices"], return_normed=s["normed"])
        if s["kind"] == "adapt":
            return vdn_fp8.adapter_add(s["x"], s["base"], vdn_fp8.Adapters(s["a"], s["b"], s["alpha"]), s["index"])
        return vdn_fp8.qk_prep_axes(s["query"], s["key"], s["norm_q"], s["norm_k"], vdn_fp8.RopeAxes(s["freq"], s["axis"], s["pairs"]),
                                    s["positions"])
    if s["kind"] == "norm":
        return _add_norm_quantize(s)
    return _adapter_add(s) if s["kind"] == "adapt" else _qk_prep_axes(s)


# ---------------------------------------------------------------------------------------
# work and 64-bit results
# ---------------------------------------------------------------------------------------

def work(case):
    size = SIZES[case["dtype"]]
    if case["kind"] == "norm":
        M, K = case["M"], case["K"]
        moved = M * K * (2 * SIZES[case["stream"]] + size * (1 + case["normed"]) + 1) + 4 * M + K * size
        moved += case["rows"] * K * size * (case["gate"] + 2 * case["affine"])
        return {"bytes": moved, "flops": 12 * M * K}
    if case["kind"] == "adapt":
        news, which = _adapters_of(case)
        T, R, K, N = sum(news), case["R"], case["K"], case["N"]
        adapted = sum(n for n, a in zip(news, which) if a >= 0)
        distinct = len({a for a in which if a >= 0})
        return {"bytes": (adapted * K + 2 * T * N + distinct * R * (K + N)) * size + 4 * T, "flops": 2 * adapted * R * (K + N)}
    elements = case["T"] * (case["Hq"] + case["H"]) * case["d"]
    axes = case["sections"].count(",") + 1
    return {"bytes": 2 * elements * size + case["T"] * axes * (8 if case["pos"] == "int64" else 4), "flops": 10 * elements}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        index = torch.zeros(case["M"], dtype=torch.long, device=DEV) if s["indices"] is None else s["indices"].long()
        hidden = s["residual"].double() + (s["branch"].double() if s["gate"] is None else s["branch"].double() * s["gate"].double()[index])
        if case["stream"] != "f32":
            # the stream that is kept, and normed: the sum in 32 bits, then the stream's own rounding
            hidden = hidden.float().to(DTYPES[case["stream"]]).double()
        n = hidden / torch.sqrt(hidden.pow(2).sum(1, keepdim=True) / case["K"] + EPS)
        n.mul_(s["weight"].double())
        if case["affine"]:
            n.mul_(s["scale"].double()[index] + 1.0).add_(s["shift"].double()[index])
        size = torch.maximum(n.abs().amax(1, keepdim=True) / 448.0, torch.full((1, 1), 1e-12, dtype=torch.float64, device=DEV))
        codes = (n / size).float().to(E4M3).double()
        return (hidden, codes, size, n) if case["normed"] else (hidden, codes, size)
    if case["kind"] == "adapt":
        out = s["base"].double()
        for adapter in range(case["used"]):
            mine = (s["index"] == adapter).nonzero()[:, 0]
            low = torch.mm(s["x"][mine].double(), s["a"][adapter].double().T)
            out[mine] += torch.mm(low, s["b"][adapter].double().T) * s["alpha"][adapter].double()
        return out
    half = s["freq"].numel()
    p = s["positions"].double()
    turns = torch.empty(case["T"], half, dtype=torch.complex128, device=DEV)
    for j, (axis, freq) in enumerate(zip(s["axis"].tolist(), s["freq"].tolist())):
        turns[:, j] = torch.polar(torch.ones_like(p[:, axis]), p[:, axis] * freq)
    got = []
    for x, norm in ((s["query"], s["norm_q"]), (s["key"], s["norm_k"])):
        x = x.double()
        if norm is not None:
            x = x / torch.sqrt(x.pow(2).sum(2, keepdim=True) / case["d"] + norm[1]) * norm[0].double()
        at = torch.arange(half, device=DEV)
        lo, hi = (2 * at, 2 * at + 1) if case["pairs"] else (at, at + half)
        z = torch.complex(x[..., lo], x[..., hi]) * turns[:, None]
        x[..., lo], x[..., hi] = z.real, z.imag
        got.append(x)
    return tuple(got)
