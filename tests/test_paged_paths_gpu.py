"""Ways through the operators over a paged cache that need larger calls: two heads a thread in norm, rotation
and append, and prompts of more row tiles than the GPU has SMs, whose last items alone are split."""
import math

import pytest
import torch

import paged_ref as ref
import timestral_b200 as tb

pytestmark = pytest.mark.gpu


def stream():
    return torch.cuda.current_stream().cuda_stream


def word():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("tokens, qh, kh, hd, rd", [(4001, 13, 7, 64, 64), (5003, 5, 3, 128, 64), (6007, 1, 6, 96, 96), (3001, 5, 2, 256, 32),
                                                    (19001, 7, 1, 32, 16), (25013, 9, 4, 16, 16)])
@pytest.mark.parametrize("norm, turn", [(True, True), (True, False), (False, True)])
def test_norm_rope_of_many_heads(dt, tokens, qh, kh, hd, rd, norm, turn):
    """Odd numbers of heads where a thread has two of them, at every number of threads a head."""
    dt = ref.DT[dt]
    threads = 1 << (hd // 16 - 1).bit_length()
    assert tokens * (qh + kh) * threads >= 148 * 2048
    g = torch.Generator(device="cuda").manual_seed(hd)
    fused = (2 * torch.randn(tokens, (qh + kh) * hd, generator=g, device="cuda")).to(dt)
    q, k = fused[:, :qh * hd].unflatten(1, (qh, hd)), fused[:, qh * hd:].unflatten(1, (kh, hd))
    w = [1 + 0.3 * torch.randn(hd, generator=g, device="cuda") for _ in range(2)] if norm else [None, None]
    cos, sin = ref.rotation(300, rd, "cuda") if turn else (None, None)
    pos = torch.randint(0, 300, (tokens,), generator=g, device="cuda", dtype=torch.int32) if turn else None
    q_out, k_out, err = torch.empty(tokens, qh, hd, device="cuda", dtype=dt), torch.empty(tokens, kh, hd, device="cuda", dtype=dt), word()
    kw = dict(q_weight=w[0], k_weight=w[1], eps=1e-5, cos=cos, sin=sin, positions=pos, error=err, stream=stream())
    tb.norm_rope(q, q_out, k, k_out, **kw)
    for x, o, wt in ((q, q_out, w[0]), (k, k_out, w[1])):
        y, size = ref.norm_rope(x, wt, 1e-5, cos, sin, pos)
        ref.within(o, y, ref.norm_rope_tolerance(y, size, dt))
    tb.norm_rope(q, q, k, k, **kw)
    assert torch.equal(q, q_out) and torch.equal(k, k_out) and err.item() == 0


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kvh", [2, 5])
@pytest.mark.parametrize("norm, rd, explicit", [(True, 64, False), (True, 0, False), (False, 32, False), (True, 32, True)])
def test_append_of_many_heads(dt, hd, kvh, norm, rd, explicit):
    """Norm and rotation on the way where a thread has two cached heads (the last one of an odd number alone)."""
    dt, page = ref.DT[dt], 32
    chunk = -(-148 * 2048 // (9 * kvh * (hd // 16))) + 3
    new = [chunk, 7, 0, chunk - 1, 33, chunk // 2, 1, chunk, 500]
    lengths = [n + extra for n, extra in zip(new, (0, 40, 9, 1, 0, 77, 12, 31, 0))]
    assert max(new) * len(new) * kvh * (hd // 16) >= 148 * 2048
    b = ref.Batch(new, lengths, kvh, kvh, hd, page, dt, extra_rows=2)
    w = 1 + 0.3 * torch.randn(hd, device="cuda") if norm else None
    rows = max(lengths)
    cos, sin = ref.rotation(rows, rd, "cuda") if rd else (None, None)
    at = torch.cat([torch.arange(m - n, m) for n, m in zip(new, lengths)]).int().cuda()
    if explicit:
        at = (at * 7 + 3) % rows
    seq = torch.cat([torch.full((n,), i) for i, n in enumerate(new)]).cuda()
    place = torch.cat([torch.arange(m - n, m) for n, m in zip(new, lengths)]).cuda()
    pages, slots = b.table[seq, place // page].long(), place % page
    k_before, v_before, err = b.k_pool.clone(), b.v_pool.clone(), word()
    tb.paged_append(tb.PagedCache(b.k_pool, b.v_pool, b.table), tb.PagedBatch(b.q_start, b.lengths, b.max_chunk, b.max_length), b.k, b.v,
                    k_weight=w, eps=1e-5, cos=cos, sin=sin,
                    positions=torch.cat([at, torch.full((2,), -1, dtype=torch.int32, device="cuda")]) if explicit else None,
                    error=err, stream=stream())
    y, size = ref.norm_rope(b.k[:b.tokens], w, 1e-5, cos, sin, at)
    ref.within(b.k_pool[pages, :, slots], y, ref.norm_rope_tolerance(y, size, dt))
    v_before[pages, :, slots] = b.v[:b.tokens]
    assert torch.equal(b.v_pool, v_before) and err.item() == 0
    b.k_pool[pages, :, slots] = k_before[pages, :, slots]
    assert torch.equal(b.k_pool, k_before)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new, lengths, qh, kvh, split", [
    ([2500], [2500], 16, 8, True), ([1300, 257, 700, 1], [1300, 900, 701, 2000], 24, 12, False),
    ([1300, 257, 700, 1], [1300, 900, 701, 2000], 16, 8, True), ([2100, 2100], [2100, 2600], 10, 5, True)])
def test_attention_of_whole_and_split_items(dt, hd, new, lengths, qh, kvh, split):
    """More than a round of row tiles: as many as fill the SMs are whole, the keys of the others are split
    and joined, in one call; also with less workspace than it would like, and none. (split False: too many are
    left over for that, and all stay whole.)"""
    b = ref.Batch(new, lengths, qh, kvh, hd, 64, ref.DT[dt], seed=hd, extra_rows=2)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    row_tiles = -(-max(new) * (qh // kvh) // 256)             # of the longest chunk, and those of all that can hold rows:
    assert min(row_tiles * len(new), b.tokens * (qh // kvh) // 256 + len(new)) * kvh > sms
    cache, batch = tb.PagedCache(b.k_pool, b.v_pool, b.table), tb.PagedBatch(b.q_start, b.lengths, b.max_chunk, b.max_length)
    full = tb.paged_attention_workspace(cache, batch, b.q.shape[0], qh)
    item = 256 * (hd * 4 + 8)                              # partial results of one item of one split
    assert (full >= 2 * item) == split
    g = torch.Generator(device="cuda").manual_seed(2)
    bits = torch.rand(len(new), -(-max(lengths) // 32) * 32, generator=g, device="cuda") < 0.7
    for kw in ({}, {"bits": bits, "self_visible": True, "gate": b.gate}):
        want, tol = ref.attention(b, **kw)
        args = dict(gate=kw.get("gate"), key_valid=ref.words(bits) if kw else None, self_visible=bool(kw))
        for size in (full, full // 2, 0) if split else (0,):
            ws = torch.full((size // 4,), float("nan"), device="cuda") if size else None
            out, err = torch.full_like(b.q, 7.0), word()
            tb.paged_attention(cache, batch, b.q, out, workspace=ws, error=err, stream=stream(), **args)
            ref.within(out[:b.tokens], want, tol)
            assert (out[b.tokens:] == 7).all() and err.item() == 0


@pytest.mark.parametrize("new, lengths", [([1, 1], [40, 3000]), ([4, 1], [4, 900]), ([150, 1], [2000, 30]), ([1, 1], [5, 96])])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("sign", [1, -1])
def test_attention_of_infinite_scores(dt, new, lengths, sign):
    """A score of plus infinity gives NaN in its row (inf - inf) and nowhere else, however the keys are split; one of
    minus infinity is a key of weight 0."""
    b = ref.Batch(new, lengths, 4, 2, 128, 16, ref.DT[dt])
    first = b.sequence(0, b.k_pool)
    b.q[:new[0]] = b.q[:new[0]].abs() + 0.1                       # positive, so that the sign of the score is the key's
    hit = torch.zeros(b.tokens, 4, dtype=torch.bool, device="cuda")
    hit[:new[0], :2] = True                                       # the heads that read cached head 0 of sequence 0
    if sign < 0:
        # weight 0: the other keys alone
        bits = torch.ones(b.n, -(-max(lengths) // 32) * 32, dtype=torch.bool, device="cuda")
        bits[0, 0] = False
        masked, mtol = ref.attention(b, bits=bits)
    want, tol = ref.attention(b)
    first[0, 0] = sign * math.inf
    b.put(0, b.k_pool, first)
    cache, batch = tb.PagedCache(b.k_pool, b.v_pool, b.table), tb.PagedBatch(b.q_start, b.lengths, b.max_chunk, b.max_length)
    size = tb.paged_attention_workspace(cache, batch, b.tokens, 4)
    for workspace in (None, torch.empty(size, dtype=torch.uint8, device="cuda") if size else None):
        out = torch.full_like(b.q, 7.0)
        tb.paged_attention(cache, batch, b.q, out, workspace=workspace, stream=stream())
        ref.within(out[~hit], want[~hit], tol[~hit])
        if sign > 0:
            assert torch.isnan(out[hit]).all()
            continue
        alone = hit.clone()
        alone[:, :2] &= torch.tensor([n == length for n, length in zip(new, lengths)], device="cuda").repeat_interleave(
            torch.tensor(new, device="cuda"))[:, None] & (torch.arange(b.tokens, device="cuda") == 0)[:, None]
        see = hit & ~alone                                        # (a row that sees that key alone is left out)
        ref.within(out[see], masked[see], mtol[see])
