"""Cases of the paged-cache attention operators: head norms with the position rotation
(norm_rope), appending keys and values to a paged cache (append), and attention of new tokens
over that cache (attention). `run` computes them in elementary torch operations, or, where
`own` is true, with the calls of this package."""
import math
import os
import sys

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


def listed():
    return [
        # One new patch of one series: q and k of the forecast geometry (12 heads of 64); latency.
        {"name": "norm_rope_one_token", "op": "norm_rope", "type": "f16", "tokens": 1, "q_heads": 12, "k_heads": 12,
         "head_dim": 64, "rope_dim": 64, "table": 2113},
        # The chunk of a long prompt, grouped heads of 128.
        {"name": "norm_rope_prompt", "op": "norm_rope", "type": "bf16", "tokens": 16384, "q_heads": 32, "k_heads": 8,
         "head_dim": 128, "rope_dim": 128, "table": 32768},
        # An odd number of tokens, half of each head rotated.
        {"name": "norm_rope_partial_odd", "op": "norm_rope", "type": "f16", "tokens": 4099, "q_heads": 12, "k_heads": 12,
         "head_dim": 64, "rope_dim": 32, "table": 2113},
        # One new patch of one series goes into its cache; latency.
        {"name": "append_one_token", "op": "append", "type": "f16", "seqs": 1, "chunk": 1, "context": 1055, "kv_heads": 12,
         "head_dim": 64, "page": 16, "rope": True, "ragged": False},
        # Prompts of many requests, of different lengths, go into the cache.
        {"name": "append_prompts_ragged", "op": "append", "type": "bf16", "seqs": 64, "chunk": 512, "context": 4000,
         "kv_heads": 8, "head_dim": 128, "page": 64, "rope": True, "ragged": True},
        # A block of patches of every row of a forecast batch, rotated already.
        {"name": "append_forecast_rows", "op": "append", "type": "f16", "seqs": 2048, "chunk": 16, "context": 64,
         "kv_heads": 12, "head_dim": 64, "page": 16, "rope": False, "ragged": False},
        # One new patch of one series against its longest row; latency.
        {"name": "attention_one_token", "op": "attention", "type": "f16", "seqs": 1, "chunk": 1, "context": 1055,
         "q_heads": 12, "kv_heads": 12, "head_dim": 64, "page": 16, "window": 0, "masked": False, "gate": False,
         "ragged": False},
        # Decoding for many requests of different lengths, grouped heads: bound by the cache's bytes.
        {"name": "attention_decode_batch", "op": "attention", "type": "bf16", "seqs": 64, "chunk": 1, "context": 8191,
         "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "window": 0, "masked": False, "gate": False,
         "ragged": True},
        # Decoding for one request with a long past: the cache's length is all there is to share out.
        {"name": "attention_decode_long", "op": "attention", "type": "bf16", "seqs": 1, "chunk": 1, "context": 131071,
         "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page": 128, "window": 0, "masked": False, "gate": False,
         "ragged": False},
        # A decode block of a forecast batch: new patches and decoder tokens of every row over its
        # cached patches, some of them unobserved, with the sigmoid gate.
        {"name": "attention_forecast_rows", "op": "attention", "type": "f16", "seqs": 2048, "chunk": 16, "context": 64,
         "q_heads": 12, "kv_heads": 12, "head_dim": 64, "page": 16, "window": 0, "masked": True, "gate": True,
         "ragged": False},
        # A chunk of a long prompt over what is cached of it: bound by the products.
        {"name": "attention_prompt_chunk", "op": "attention", "type": "bf16", "seqs": 1, "chunk": 2048, "context": 32768,
         "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "window": 0, "masked": False, "gate": False,
         "ragged": False},
        # Prompts and single tokens in one batch, five query heads to a cached head, a sliding window.
        {"name": "attention_mixed_window", "op": "attention", "type": "f16", "seqs": 7, "chunk": 300, "context": 5003,
         "q_heads": 20, "kv_heads": 4, "head_dim": 128, "page": 16, "window": 1000, "masked": False, "gate": False,
         "ragged": True},
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["norm_rope", "append", "attention", "attention"])
    while True:
        kind = rng.choice(["f16", "bf16"])
        hd = rng.choice([64, 128])
        kvh = rng.choice([1, 2, 3, 4, 8, 12])
        page = rng.choice([8, 16, 32, 64, 128, 256])
        if op == "norm_rope":
            c = {"op": op, "type": kind, "tokens": _log(rng, 1, 16384), "q_heads": kvh * rng.choice([1, 2, 3, 4]),
                 "k_heads": kvh, "head_dim": hd, "rope_dim": rng.choice([32, hd, hd]), "table": _log(rng, 128, 32768)}
            if work(c)["bytes"] <= 330e6:
                return c
        elif op == "append":
            c = {"op": op, "type": kind, "seqs": _log(rng, 1, 2048), "chunk": _log(rng, 1, 512), "context": _log(rng, 1, 8000),
                 "kv_heads": kvh, "head_dim": hd, "page": page, "rope": rng.random() < 0.6, "ragged": rng.random() < 0.6}
            pool = sum(-(-x // page) * page for x in _spread(c)[1]) * kvh * hd * 4
            if work(c)["bytes"] <= 200e6 and pool <= 1.5e9:
                return c
        else:
            c = {"op": op, "type": kind, "seqs": _log(rng, 1, 2048), "chunk": rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 2, 2048)]),
                 "context": _log(rng, 1, 131071), "q_heads": kvh * rng.choice([1, 1, 2, 4, 5, 8]), "kv_heads": kvh,
                 "head_dim": hd, "page": page, "window": rng.choice([0, 0, 0, _log(rng, 1, 4096)]),
                 "masked": rng.random() < 0.25, "gate": rng.random() < 0.25, "ragged": rng.random() < 0.6}
            longest = c["context"] + c["chunk"]
            scores = c["seqs"] * c["q_heads"] * c["chunk"] * longest
            if scores <= 1e9 and c["seqs"] * longest * kvh * hd <= 4e8 and c["seqs"] * c["chunk"] <= 65536 and work(c)["flops"] <= 1.1e12:
                return c


def _spread(c):
    """New tokens of each sequence, and its length with them: all alike, or spread over their range."""
    n = c["seqs"]
    if not c["ragged"]:
        return [c["chunk"]] * n, [c["context"] + c["chunk"]] * n
    new = [1 + (i * 7919) % c["chunk"] for i in range(n)]
    new[-1] = c["chunk"]
    return new, [c["context"] - (i * 10473) % (c["context"] // 2 + 1) + x for i, x in enumerate(new)]


def work(c):
    """Each input read once and each output written once; the products over the keys that are seen."""
    hd = c["head_dim"]
    if c["op"] == "norm_rope":
        heads = c["tokens"] * (c["q_heads"] + c["k_heads"])
        rows = min(c["tokens"], c["table"])
        return {"bytes": heads * hd * 4 + rows * c["rope_dim"] * 4 + c["tokens"] * 4 + hd * 8,
                "flops": heads * (4 * hd + 3 * c["rope_dim"])}
    new, lengths = _spread(c)
    tokens = sum(new)
    if c["op"] == "append":
        table = sum(-(-x // c["page"]) for x in lengths)
        angles = max(new) * hd * 4 if c["rope"] else 0
        return {"bytes": tokens * c["kv_heads"] * hd * 8 + angles + 4 * table + 8 * c["seqs"],
                "flops": tokens * c["kv_heads"] * hd * 3 if c["rope"] else 0}
    seen, pairs = 0, 0
    for x, length in zip(new, lengths):
        w = c["window"] or length
        seen += min(length, w + x - 1)
        first = length - x + 1                     # keys that the first and the last new token see
        if w >= length:
            pairs += x * (first + length) // 2
        else:
            full = max(0, min(x, length - w))      # tokens that see a whole window
            rest = x - full
            pairs += full * w + rest * (first + first + rest - 1) // 2
    share = 0.9 if c["masked"] else 1.0
    out = tokens * c["q_heads"] * hd * 2 * (3 if c["gate"] else 2)
    return {"bytes": int(seen * c["kv_heads"] * hd * 4 * share) + out + 4 * c["seqs"] * 2,
            "flops": int(4 * hd * c["q_heads"] * pairs * share)}


def _rotation(rows, dim):
    """cos and sin of row * 10000^(-2 i / dim), the angles in 64 bits."""
    angle = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * torch.exp(
        torch.arange(dim // 2, device="cuda", dtype=torch.float64) * (-2 * math.log(10000.0) / dim))
    return torch.cos(angle).float(), torch.sin(angle).float()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    dt, hd = TYPES[case["type"]], case["head_dim"]

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dt)

    if case["op"] == "norm_rope":
        t, qh, kh = case["tokens"], case["q_heads"], case["k_heads"]
        fused = normal(t, (qh + 2 * kh) * hd, scale=1.5)            # a projection's output: q | k | v of a token
        cos, sin = _rotation(case["table"], case["rope_dim"])
        return {"case": case, "q": fused[:, :qh * hd].unflatten(1, (qh, hd)),
                "k": fused[:, qh * hd:(qh + kh) * hd].unflatten(1, (kh, hd)),
                "q_out": torch.empty(t, qh, hd, device="cuda", dtype=dt), "k_out": torch.empty(t, kh, hd, device="cuda", dtype=dt),
                "q_weight": 1 + 0.2 * torch.randn(hd, generator=g, device="cuda"),
                "k_weight": 1 + 0.2 * torch.randn(hd, generator=g, device="cuda"), "cos": cos, "sin": sin,
                "positions": (torch.randint(0, case["table"], (1,), generator=g, device="cuda")
                              + torch.arange(t, device="cuda")).remainder(case["table"]).int()}
    new, lengths = _spread(case)
    n, page, kvh = case["seqs"], case["page"], case["kv_heads"]
    pages = [-(-x // page) for x in lengths]
    total, widest = sum(pages), max(pages)
    order = torch.randperm(total + 3, generator=g, device="cuda").int()       # pages lie anywhere in the pool
    width = torch.tensor(pages, device="cuda")
    first = torch.cumsum(width, 0) - width
    at = first[:, None] + torch.arange(widest, device="cuda")
    used = torch.arange(widest, device="cuda") < width[:, None]
    table = torch.where(used, order[at.clamp(max=total)], torch.full_like(at, -1, dtype=torch.int32)).contiguous()
    s = {"case": case, "table": table, "lengths": torch.tensor(lengths, device="cuda", dtype=torch.int32),
         "q_start": torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), device="cuda", dtype=torch.int32),
         "max_chunk": max(new), "max_length": max(lengths),
         "k_pool": normal(total + 3, kvh, page, hd), "v_pool": normal(total + 3, kvh, page, hd)}
    t = sum(new)
    if case["op"] == "append":
        fused = normal(t, 2 * kvh * hd)
        s["k"], s["v"] = fused[:, :kvh * hd].unflatten(1, (kvh, hd)), fused[:, kvh * hd:].unflatten(1, (kvh, hd))
        s["cos"], s["sin"] = _rotation(max(lengths), hd) if case["rope"] else (None, None)
        return s
    s["q"] = normal(t, case["q_heads"], hd, scale=1.5)
    s["out"] = torch.empty_like(s["q"])
    s["gate"] = torch.rand(t, case["q_heads"], hd, generator=g, device="cuda").to(dt) if case["gate"] else None
    s["key_valid"] = None
    if case["masked"]:                                # bit p % 32 of word p / 32: patch p is observed
        words = -(-max(lengths) // 32)
        bits = (torch.rand(n, words, 32, generator=g, device="cuda") < 0.9).long() << torch.arange(32, device="cuda")
        s["key_valid"] = bits.sum(2).to(torch.int32) if words else None
    s["workspace"] = torch.empty(64 << 20, device="cuda", dtype=torch.uint8)
    return s


def run(state):
    c = state["case"]
    if own:
        return _own(state, c)
    if c["op"] == "norm_rope":
        return [_norm_rope(state["q"], state["q_weight"], state), _norm_rope(state["k"], state["k_weight"], state)]
    if c["op"] == "append":
        return _append(state, c)
    return _attention(state, c)


def _own(s, c):
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "timestral.cpp_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import timestral_b200 as tb
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "norm_rope":
        tb.norm_rope(s["q"], s["q_out"], s["k"], s["k_out"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS,
                     cos=s["cos"], sin=s["sin"], positions=s["positions"], stream=stream)
        return [s["q_out"], s["k_out"]]
    cache = tb.PagedCache(s["k_pool"], s["v_pool"], s["table"])
    batch = tb.PagedBatch(s["q_start"], s["lengths"], s["max_chunk"], s["max_length"])
    if c["op"] == "append":
        tb.paged_append(cache, batch, s["k"], s["v"], cos=s["cos"], sin=s["sin"], stream=stream)
        return [s["k_pool"], s["v_pool"]]
    tb.paged_attention(cache, batch, s["q"], s["out"], window=c["window"], key_valid=s["key_valid"], gate=s["gate"],
                       self_visible=c["masked"], workspace=s["workspace"], stream=stream)
    return [s["out"]]


def _rotate(x, cos, sin):
    """x [tokens, heads, d] in 32 bits; the first 2 * half values of a head turn by their token's angles."""
    half = cos.shape[1]
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    cos, sin = cos[:, None], sin[:, None]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _norm_rope(x, weight, s):
    y = x.float()
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * weight
    at = s["positions"].long()
    return _rotate(y, s["cos"][at], s["sin"][at]).to(x.dtype)


def _token_rows(s):
    """Of each new token: its sequence, its place among that sequence's new tokens, its place in the cache."""
    start, lengths = s["q_start"].long(), s["lengths"].long()
    token = torch.arange(s["k"].shape[0] if "k" in s else s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(start[1:], token, right=True)
    place = token - start[seq]
    return seq, place, lengths[seq] - (start[seq + 1] - start[seq]) + place


def _append(s, c):
    seq, _, position = _token_rows(s)
    k = s["k"]
    if c["rope"]:
        k = _rotate(k.float(), s["cos"][position], s["sin"][position]).to(k.dtype)
    page = s["table"][seq, position // c["page"]].long()
    s["k_pool"][page, :, position % c["page"]] = k
    s["v_pool"][page, :, position % c["page"]] = s["v"]
    return [s["k_pool"], s["v_pool"]]


def _attention(s, c):
    n, qh, kvh, hd = c["seqs"], c["q_heads"], c["kv_heads"], c["head_dim"]
    chunk, longest, group = s["max_chunk"], s["max_length"], c["q_heads"] // c["kv_heads"]
    seq, place, _ = _token_rows(s)
    q = torch.zeros(n, chunk, kvh, group, hd, device="cuda")
    q[seq, place] = s["q"].float().view(-1, kvh, group, hd)
    q = q.permute(0, 2, 3, 1, 4).reshape(n, kvh, group * chunk, hd)
    key = torch.arange(longest, device="cuda")
    page = s["table"][:, key // c["page"]].long().clamp(min=0)             # [n, longest]
    slot = (key % c["page"]).expand(n, longest)
    k = s["k_pool"][page, :, slot].float().permute(0, 2, 3, 1)              # [n, kvh, hd, longest]
    scores = torch.matmul(q, k).view(n, kvh, group, chunk, longest)
    del k
    scores *= 1 / math.sqrt(hd)
    new = (s["q_start"][1:] - s["q_start"][:-1]).long()
    position = (s["lengths"].long() - new)[:, None] + torch.arange(chunk, device="cuda")
    position = torch.where(torch.arange(chunk, device="cuda") < new[:, None], position, torch.full_like(position, -1))
    seen = key <= position[:, :, None]                                      # [n, chunk, longest]
    if c["window"]:
        seen &= key > position[:, :, None] - c["window"]
    if c["masked"]:
        bit = (s["key_valid"][:, key // 32] >> (key % 32)) & 1
        seen &= (bit[:, None, :] != 0) | (key == position[:, :, None])
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores -= torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    scores.exp_()
    total = scores.sum(-1, keepdim=True)
    v = s["v_pool"][page, :, slot].float().permute(0, 2, 1, 3)              # [n, kvh, longest, hd]
    out = torch.matmul(scores.view(n, kvh, group * chunk, longest), v).view(n, kvh, group, chunk, hd)
    out = out / torch.where(total > 0, total, torch.ones_like(total))
    out = out.permute(0, 3, 1, 2, 4)[seq, place].reshape(-1, qh, hd)
    if s["gate"] is not None:
        out = out * s["gate"].float()
    return [out.to(s["q"].dtype)]


def exact(case, seed):
    """The same from the definitions in 64 bits, sequence by sequence and head by head."""
    s = prepare(case, seed)
    hd = case["head_dim"]
    if case["op"] == "norm_rope":
        c, n = s["cos"].double()[s["positions"].long()], s["sin"].double()[s["positions"].long()]
        outs = []
        for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
            out = torch.empty(x.shape, device="cuda", dtype=torch.float64)
            for h in range(x.shape[1]):
                y = x[:, h].double()
                y = y / (y.square().mean(1) + EPS).sqrt()[:, None] * w.double()
                half = case["rope_dim"] // 2
                z = torch.complex(y[:, :half], y[:, half:2 * half]) * torch.complex(c, n)
                out[:, h] = torch.cat([z.real, z.imag, y[:, 2 * half:]], 1)
            outs.append(out)
        return outs
    new, lengths = _spread(case)
    page, kvh = case["page"], case["kv_heads"]
    if case["op"] == "append":
        pools = [s["k_pool"].double(), s["v_pool"].double()]
        table = s["table"].cpu().tolist()
        rows, slots, positions = [], [], []
        for i, (x, length) in enumerate(zip(new, lengths)):
            for p in range(length - x, length):
                rows.append(table[i][p // page])
                slots.append(p % page)
                positions.append(p)
        rows, slots = torch.tensor(rows, device="cuda"), torch.tensor(slots, device="cuda")
        for h in range(kvh):
            y = s["k"][:, h].double()
            if case["rope"]:
                at = torch.tensor(positions, device="cuda")
                z = torch.complex(y[:, :hd // 2], y[:, hd // 2:]) * torch.complex(s["cos"].double()[at], s["sin"].double()[at])
                y = torch.cat([z.real, z.imag], 1)
            pools[0][rows, h, slots] = y
            pools[1][rows, h, slots] = s["v"][:, h].double()
        return pools
    if case["seqs"] > 4000:
        return None
    out = torch.empty(s["q"].shape, device="cuda", dtype=torch.float64)
    group, first = case["q_heads"] // kvh, 0
    for i, (x, length) in enumerate(zip(new, lengths)):
        place = torch.arange(length, device="cuda")
        at = s["table"][i].long()[place // page]
        mine = place[length - x:, None]
        hidden = place > mine
        if case["window"]:
            hidden |= place <= mine - case["window"]
        if case["masked"]:
            observed = (s["key_valid"][i].long()[place // 32] >> (place % 32)) & 1
            hidden |= (observed == 0) & (place != mine)
        few = max(1, min(kvh, 200_000_000 // (group * x * length)))       # cached heads at a time
        for h in range(0, kvh, few):
            heads = range(h, min(kvh, h + few))
            k, v = (torch.stack([pool[at, j, place % page] for j in heads]).double() for pool in (s["k_pool"], s["v_pool"]))
            q = s["q"][first:first + x, h * group:(h + len(heads)) * group].double().unflatten(1, (len(heads), group))
            logits = torch.einsum("thgd,hkd->hgtk", q, k).div_(math.sqrt(hd)).masked_fill_(hidden, -math.inf)
            mean = torch.einsum("hgtk,hkd->thgd", torch.softmax(logits, 3), v)
            out[first:first + x, h * group:(h + len(heads)) * group] = mean.flatten(1, 2)
        first += x
    return [out * s["gate"].double() if s["gate"] is not None else out]
