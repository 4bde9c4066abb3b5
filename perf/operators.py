"""The measured cases of the operators for a packed batch of requests: per-head norm with
rotation, attention over a key range per query row, and a projection with per-row low-rank adapters.

A user who serves several requests at once packs their tokens into one [rows, ...] buffer: every
row has its request's adapter, its own position, and sees the keys of its own request only.
`run` computes one operator in its plain form (fp32, elementary torch operations), or through the
library's entry points where `own` is set; `exact` restates the definitions in fp64.
"""
import math
import os
import sys

import torch

own = False

BF16 = torch.bfloat16
DEV = "cuda"


# ---------------------------------------------------------------------------- cases
def listed():
    return [
        # one new token of one request: 24 query and 24 key heads, the latency of the smallest call
        {"name": "norm_one_token", "op": "norm", "rows": 1, "hq": 24, "hk": 24, "dim": 128, "rot": 128, "inter": True,
         "positions": 9000},
        # an odd packed batch of short requests, grouped heads of 64, half-split pairs, part of the head rotated
        {"name": "norm_packed_grouped", "op": "norm", "rows": 1999, "hq": 32, "hk": 8, "dim": 64, "rot": 48,
         "inter": False, "positions": 777},
        # the q and k sections of a whole video step's fused projection: 2 x 7854 tokens
        {"name": "norm_video", "op": "norm", "rows": 15708, "hq": 24, "hk": 24, "dim": 128, "rot": 128, "inter": True,
         "positions": 7854},
        # one token of one request over a short cache: latency
        {"name": "attn_one_token", "op": "attn", "batch": 1, "q_len": 1, "kv_len": 1031, "hq": 24, "hk": 24, "dim": 128,
         "mask": "cache", "docs": 1, "block": 1, "prefix": 0, "cap": 0.0, "bias": "none", "reach": 0},
        # the next token of 16 requests with caches of unequal lengths, three query heads to a key head
        {"name": "attn_decode_batch", "op": "attn", "batch": 16, "q_len": 1, "kv_len": 4096, "hq": 24, "hk": 8,
         "dim": 128, "mask": "cache", "docs": 1, "block": 1, "prefix": 0, "cap": 0.0, "bias": "slopes", "reach": 0},
        # a text encoder's layer: 512-token prompts with padding, 64 heads of 64, relative-position bias table
        {"name": "attn_text_encoder", "op": "attn", "batch": 2, "q_len": 512, "kv_len": 512, "hq": 64, "hk": 64,
         "dim": 64, "mask": "padded", "docs": 1, "block": 1, "prefix": 0, "cap": 0.0, "bias": "table", "reach": 128},
        # packed documents with a prefix that every token of its document sees, capped scores, grouped heads
        {"name": "attn_packed_prefix_cap", "op": "attn", "batch": 1, "q_len": 5003, "kv_len": 5003, "hq": 16, "hk": 4,
         "dim": 128, "mask": "documents", "docs": 7, "block": 1, "prefix": 97, "cap": 30.0, "bias": "none", "reach": 0},
        # two videos packed, each frame (17 x 22 tokens) sees its own and all earlier frames
        {"name": "attn_video_frames", "op": "attn", "batch": 1, "q_len": 10846, "kv_len": 10846, "hq": 24, "hk": 24,
         "dim": 128, "mask": "documents", "docs": 2, "block": 374, "prefix": 0, "cap": 0.0, "bias": "none", "reach": 0},
        # a step of four single-token requests with an adapter each (one without): reading the weight bounds it
        {"name": "lora_four_rows", "op": "lora", "rows": 4, "k": 4096, "n": 4096, "adapters": 8, "rank": 16,
         "sorted": False, "epi": "bias"},
        # short prompts of many requests, rows of 16 adapters interleaved
        {"name": "lora_mixed_rows", "op": "lora", "rows": 509, "k": 4096, "n": 2048, "adapters": 16, "rank": 16,
         "sorted": False, "epi": "bias"},
        # an FFN up-projection with GELU over the token shard of one GPU, three requests
        {"name": "lora_ffn_up", "op": "lora", "rows": 1964, "k": 2048, "n": 8192, "adapters": 3, "rank": 32,
         "sorted": True, "epi": "gelu"},
        # an output projection into the fp32 residual stream over a whole video batch, four requests
        {"name": "lora_video_residual", "op": "lora", "rows": 15708, "k": 4096, "n": 4096, "adapters": 4, "rank": 64,
         "sorted": True, "epi": "res"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "attn", "attn", "lora"])
    if op == "norm":
        dim = rng.choice([64, 128])
        hk = rng.choice([1, 2, 4, 8, 24])
        hq = hk * rng.choice([1, 1, 2, 3])
        rows = _log_int(rng, 1, min(15708, 15708 * 48 * 128 // ((hq + hk) * dim)))
        return {"op": "norm", "rows": rows, "hq": hq, "hk": hk, "dim": dim,
                "rot": rng.choice([dim, dim, dim // 2, 3 * dim // 4]), "inter": rng.random() < 0.5,
                "positions": _log_int(rng, 1, 9000)}
    if op == "attn":
        dim = rng.choice([64, 128])
        hk = rng.choice([2, 4, 8, 12])
        hq = hk * rng.choice([1, 1, 2, 3])
        case = {"op": "attn", "hq": hq, "hk": hk, "dim": dim, "docs": 1, "block": 1, "prefix": 0, "reach": 0,
                "cap": rng.choice([0.0, 0.0, 20.0, 50.0]), "bias": rng.choice(["none", "none", "slopes", "table"])}
        if case["bias"] == "table":
            case["reach"] = rng.choice([32, 128, 500])
        kind = rng.choice(["cache", "padded", "documents", "documents"])
        if kind == "cache":
            q_len = rng.choice([1, 1, 2, 5, 40])
            kv = _log_int(rng, q_len + 1, 8000)
            return {**case, "mask": "cache", "batch": rng.randint(1, 12), "q_len": q_len, "kv_len": kv}
        if kind == "padded":
            n = _log_int(rng, 2, 1500)
            return {**case, "mask": "padded", "batch": rng.randint(1, 4), "q_len": n, "kv_len": n}
        n = _log_int(rng, 30, 6000)
        return {**case, "mask": "documents", "batch": 1, "q_len": n, "kv_len": n, "docs": rng.randint(1, min(12, n // 2)),
                "block": rng.choice([1, 1, 16, 374]), "prefix": rng.choice([0, 0, 60])}
    rows = _log_int(rng, 1, 8000)
    rank = rng.choice([8, 16, 24, 32, 64])
    return {"op": "lora", "rows": rows, "k": 64 * rng.randint(4, 64), "n": 32 * rng.randint(8, 128),
            "adapters": rng.randint(1, 16), "rank": rank, "sorted": rng.random() < 0.5,
            "epi": rng.choice(["bias", "gelu", "res"])}


# ---------------------------------------------------------------------------- inputs
def _key_ranges(case, gen):
    """lo, hi, pos [B or 1, q_len] int32: query row i sees keys lo <= j < hi and sits at key position pos."""
    n, kv, b = case["q_len"], case["kv_len"], case["batch"]
    if case["mask"] == "cache":  # the last q_len tokens of each request's cache, causal among themselves
        lens = torch.randint(max(n, kv // 4), kv + 1, (b, 1), generator=gen)
        pos = lens - n + torch.arange(n)[None]
        lo, hi = torch.zeros_like(pos), pos + 1
    elif case["mask"] == "padded":  # prompts of unequal lengths; the padded rows see nothing
        lens = torch.randint(max(1, n // 8), n + 1, (b, 1), generator=gen)
        pos = torch.arange(n)[None].expand(b, n)
        lo, hi = torch.zeros_like(pos), torch.where(pos < lens, lens, torch.zeros_like(lens))
    else:  # packed documents, block-causal inside each, with a prefix seen by all of its document
        cuts = torch.randperm(n - 1, generator=gen)[:case["docs"] - 1].sort().values + 1
        edges = torch.cat([torch.zeros(1, dtype=torch.int64), cuts, torch.tensor([n])])
        i = torch.arange(n)
        doc = torch.bucketize(i, edges, right=True) - 1
        lo, end = edges[doc], edges[doc + 1]
        hi = lo + ((i - lo) // case["block"] + 1) * case["block"]
        hi = torch.minimum(torch.maximum(hi, lo + case["prefix"]), end)
        lo, hi, pos = lo[None], hi[None], i[None]
    return [t.to(torch.int32).contiguous().to(DEV) for t in (lo, hi, pos)]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)

    def randn(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device=DEV).mul_(scale).to(BF16)

    s = {"case": case}
    if case["op"] == "norm":
        m, hq, hk, d = case["rows"], case["hq"], case["hk"], case["dim"]
        # the q, k and v sections of one fused projection; the v columns stay behind
        s["qkv"] = randn(m, (hq + 2 * hk) * d)
        s["out"] = torch.zeros(m, (hq + hk) * d, dtype=BF16, device=DEV)
        s["gq"] = (1 + 0.1 * torch.randn(d, generator=g, device=DEV)).to(BF16)
        s["gk"] = (1 + 0.1 * torch.randn(d, generator=g, device=DEV)).to(BF16)
        p = case["positions"]
        freq = 10000.0 ** (-torch.arange(case["rot"] // 2, device=DEV, dtype=torch.float64) * 2 / case["rot"])
        angle = torch.arange(p, device=DEV, dtype=torch.float64)[:, None] * freq
        s["cos"], s["sin"] = angle.cos().float().contiguous(), angle.sin().float().contiguous()
        start = torch.randint(0, p, (1,), generator=cpu).item()
        s["pos"] = ((torch.arange(m, device=DEV) + start) % p).to(torch.int32)
    elif case["op"] == "attn":
        b, d = case["batch"], case["dim"]
        s["q"] = randn(b, case["q_len"], case["hq"], d, scale=1.5)
        s["k"] = randn(b, case["kv_len"], case["hk"], d, scale=1.5)
        s["v"] = randn(b, case["kv_len"], case["hk"], d)
        s["lo"], s["hi"], s["pos"] = _key_ranges(case, cpu)
        s["slopes"] = s["table"] = None
        if case["bias"] == "slopes":
            s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, case["hq"] + 1, device=DEV) / case["hq"])
        if case["bias"] == "table":
            s["table"] = torch.randn(case["hq"], 2 * case["reach"] + 1, generator=g, device=DEV)
    else:
        m, k, n, na, r = case["rows"], case["k"], case["n"], case["adapters"], case["rank"]
        s["x"] = randn(m, k)
        s["w"] = randn(n, k, scale=k ** -0.5)
        s["bias"] = randn(n, scale=0.1)
        s["down"] = randn(na, r, k, scale=k ** -0.5)
        s["up"] = randn(n, na, r, scale=0.3 * r ** -0.5)
        s["scales"] = torch.rand(na, generator=g, device=DEV) + 0.5
        if case["sorted"]:  # whole requests one after the other, adapter -1 = none
            ids = torch.randint(-1, na, (max(1, min(m, na)),), generator=cpu).repeat_interleave(-(-m // max(1, min(m, na))))[:m]
        else:
            ids = torch.randint(-1, na, (m,), generator=cpu)
        s["ids"] = ids.to(torch.int32).to(DEV)
        s["res"] = torch.randn(m, n, generator=g, device=DEV) if case["epi"] == "res" else None
    return s


# ---------------------------------------------------------------------------- plain forms
def _rotate(y, cos, sin, rot, inter):
    """The pairs of the first rot channels of y [..., dim] turned by the row's angles [rows, rot / 2]."""
    c, s = cos[:, None], sin[:, None]
    r = y[..., :rot]
    a, b = (r[..., 0::2], r[..., 1::2]) if inter else (r[..., :rot // 2], r[..., rot // 2:])
    ra, rb = a * c - b * s, a * s + b * c
    r = torch.stack([ra, rb], -1).flatten(-2) if inter else torch.cat([ra, rb], -1)
    return torch.cat([r, y[..., rot:]], -1)


def _norm_plain(s):
    c = s["case"]
    m, hq, hk, d = c["rows"], c["hq"], c["hk"], c["dim"]
    cos, sin = s["cos"][s["pos"].long()], s["sin"][s["pos"].long()]
    x = s["qkv"][:, :(hq + hk) * d].float().view(m, hq + hk, d)
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    gain = torch.cat([s["gq"].float().expand(hq, d), s["gk"].float().expand(hk, d)])
    return _rotate(y * gain, cos, sin, c["rot"], c["inter"]).to(BF16).view(m, -1)


def _attn_plain(s):
    c = s["case"]
    group = c["hq"] // c["hk"]
    q = s["q"].float().transpose(1, 2)
    k = s["k"].float().transpose(1, 2).repeat_interleave(group, 1)
    v = s["v"].float().transpose(1, 2).repeat_interleave(group, 1)
    t = (q * c["dim"] ** -0.5) @ k.transpose(2, 3)
    if c["cap"] > 0:
        t = c["cap"] * torch.tanh(t / c["cap"])
    j = torch.arange(c["kv_len"], device=DEV)
    dist = j - s["pos"][..., None].long()  # [B or 1, q, kv]
    if c["bias"] == "slopes":
        t = t - s["slopes"][:, None, None] * dist.abs()[:, None]
    if c["bias"] == "table":
        t = t + s["table"][:, dist.clamp(-c["reach"], c["reach"]) + c["reach"]].transpose(0, 1)
    seen = ((j >= s["lo"][..., None]) & (j < s["hi"][..., None]))[:, None]
    t = t.masked_fill(~seen, -math.inf)
    top = t.amax(-1, keepdim=True)
    e = torch.exp(t - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    o = (e @ v) / torch.where(total == 0, torch.ones_like(total), total)
    return o.transpose(1, 2).to(BF16).contiguous()


def _lora_plain(s):
    c = s["case"]
    x = s["x"].float()
    y = x @ s["w"].float().t() + s["bias"].float()
    na, r = c["adapters"], c["rank"]
    use = torch.where(s["ids"][:, None] == torch.arange(na, device=DEV), s["scales"], torch.zeros_like(s["scales"]))
    h = (x @ s["down"].float().view(na * r, -1).t()).view(-1, na, r) * use[..., None]
    y = y + h.view(-1, na * r) @ s["up"].float().view(-1, na * r).t()
    if c["epi"] == "gelu":
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    if c["epi"] == "res":
        return s["res"] + y
    return y.to(BF16)


# ---------------------------------------------------------------------------- the library's calls
def _library():
    """wanb200.ops; the package lies one folder below the repository's root."""
    folder = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "wan2-ti2v-5b_b200")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    from wanb200 import ops
    return ops


def _norm_own(s):
    ops = _library()
    c = s["case"]
    ops.head_norm_rope(s["qkv"], [(0, c["hq"], s["gq"]), (c["hq"] * c["dim"], c["hk"], s["gk"])], c["dim"], out=s["out"],
                       cos=s["cos"], sin=s["sin"], positions=s["pos"], interleaved=c["inter"])
    return s["out"]


def _attn_own(s):
    ops = _library()
    return ops.range_attention(s["q"], s["k"], s["v"], s["lo"], s["hi"], pos=s["pos"], softcap=s["case"]["cap"],
                               slopes=s["slopes"], dist_bias=s["table"])


def _lora_own(s):
    ops = _library()
    epi = {"bias": ops.L.EPI_BIAS, "gelu": ops.L.EPI_BIAS_GELU, "res": ops.L.EPI_BIAS_RES}[s["case"]["epi"]]
    out = torch.empty_like(s["res"]) if s["res"] is not None else None
    return ops.lora_linear(s["x"], s["w"], s["bias"], s["down"], s["up"], s["ids"], scales=s["scales"], epilogue=epi,
                           residual=s["res"], out=out)


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _norm_own, "attn": _attn_own, "lora": _lora_own}[op](state)
    return {"norm": _norm_plain, "attn": _attn_plain, "lora": _lora_plain}[op](state)


# ---------------------------------------------------------------------------- work and definitions
def work(case):
    if case["op"] == "norm":
        vals = case["rows"] * (case["hq"] + case["hk"]) * case["dim"]
        table = min(case["rows"], case["positions"]) * case["rot"] * 4
        return {"bytes": 4 * vals + table + 4 * case["rows"] + 4 * case["dim"], "flops": 8 * vals}
    if case["op"] == "attn":
        # pairs: the (row, key) pairs that are seen; keys: those that any row sees (means over the drawn lengths)
        b, n, kv = case["batch"], case["q_len"], case["kv_len"]
        if case["mask"] == "cache":
            keys = b * 0.625 * kv
            pairs = keys * n
        elif case["mask"] == "padded":
            keys = b * 0.5625 * kv
            pairs = b * n * n * 0.38
        else:
            keys = kv
            squares = 2 * n * n / (case["docs"] + 1)  # the documents' lengths squared, for random cuts
            pairs = min(squares, (squares + n * case["block"]) / 2)
        qo = 2 * 2 * b * n * case["hq"] * case["dim"]
        return {"bytes": qo + 2 * 2 * keys * case["hk"] * case["dim"], "flops": 4 * pairs * case["hq"] * case["dim"]}
    m, k, n, r = case["rows"], case["k"], case["n"], case["rank"]
    used = min(m, case["adapters"])
    out = 8 if case["epi"] == "res" else 2
    return {"bytes": 2 * (m * k + n * k + n + used * r * (k + n)) + out * m * n,
            "flops": 2 * m * n * k + 2 * m * r * (k + n)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        m, d, rot = case["rows"], case["dim"], case["rot"]
        out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
        cos, sin = s["cos"].double()[s["pos"].long()], s["sin"].double()[s["pos"].long()]
        half = rot // 2
        first = torch.arange(half, device=DEV) * 2 if case["inter"] else torch.arange(half, device=DEV)
        second = first + 1 if case["inter"] else first + half
        for h in range(case["hq"] + case["hk"]):
            x = s["qkv"][:, h * d:(h + 1) * d].double()
            gain = (s["gq"] if h < case["hq"] else s["gk"]).double()
            y = gain * x / (x.pow(2).sum(1, keepdim=True) / d + 1e-6).sqrt()
            z = y.clone()
            z[:, first] = cos * y[:, first] - sin * y[:, second]
            z[:, second] = sin * y[:, first] + cos * y[:, second]
            out[:, h * d:(h + 1) * d] = z
        return out
    if case["op"] == "attn":
        b, n, kv, d = case["batch"], case["q_len"], case["kv_len"], case["dim"]
        out = torch.zeros(b, n, case["hq"], d, dtype=torch.float64, device=DEV)
        j = torch.arange(kv, device=DEV)
        for i in range(b):
            m = i if s["lo"].shape[0] > 1 else 0
            lo, hi, pos = (s[x][m].long()[:, None] for x in ("lo", "hi", "pos"))
            hidden = (j < lo) | (j >= hi)
            some = (hi > lo).squeeze(1)
            for h in range(case["hq"]):
                kh = h // (case["hq"] // case["hk"])
                t = s["q"][i, :, h].double() @ s["k"][i, :, kh].double().t() / math.sqrt(d)
                if case["cap"] > 0:
                    t = torch.tanh(t / case["cap"]) * case["cap"]
                if case["bias"] == "slopes":
                    t -= s["slopes"][h].double() * (j - pos).abs()
                if case["bias"] == "table":
                    t += s["table"][h].double()[torch.clamp(j - pos + case["reach"], 0, 2 * case["reach"])]
                t[hidden] = -math.inf
                p = torch.softmax(t, 1)
                p[~some] = 0
                out[i, :, h] = p @ s["v"][i, :, kh].double()
        return out
    x = s["x"].double()
    y = x @ s["w"].double().t() + s["bias"].double()
    for a in range(case["adapters"]):
        rows = (s["ids"] == a).nonzero().squeeze(1)
        if rows.numel():
            y[rows] += s["scales"][a].double() * ((x[rows] @ s["down"][a].double().t()) @ s["up"][:, a].double().t())
    if case["epi"] == "gelu":
        y = y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y.pow(3)))
    if case["epi"] == "res":
        y += s["res"].double()
    return y
