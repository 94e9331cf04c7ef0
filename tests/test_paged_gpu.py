"""The operators over a paged cache on the GPU against 64-bit restatements (paged_ref)."""
import math

import pytest
import torch

import paged_ref as ref
import timestral_b200 as tb

pytestmark = pytest.mark.gpu
NAN = float("nan")


def stream():
    return torch.cuda.current_stream().cuda_stream


def word():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


def handles(b, max_chunk=None, max_length=None):
    return (tb.PagedCache(b.k_pool, b.v_pool, b.table),
            tb.PagedBatch(b.q_start, b.lengths, b.max_chunk if max_chunk is None else max_chunk,
                          b.max_length if max_length is None else max_length))


# ---- norm_rope ---------------------------------------------------------------------------

@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("tokens, qh, kh, hd, rd", [
    (1, 12, 12, 64, 64), (1, 1, 0, 16, 16), (5, 3, 1, 48, 32), (33, 4, 4, 96, 96), (257, 12, 12, 64, 32), (100, 8, 2, 128, 128),
    (64, 2, 2, 256, 256), (31, 5, 1, 256, 64), (17, 3, 3, 240, 16), (1025, 32, 8, 128, 64), (7, 0, 3, 64, 64)])
@pytest.mark.parametrize("norm, turn", [(True, True), (True, False), (False, True)])
def test_norm_rope(dt, tokens, qh, kh, hd, rd, norm, turn):
    dt = ref.DT[dt]
    g = torch.Generator(device="cuda").manual_seed(tokens + hd)
    fused = (2 * torch.randn(tokens, (qh + 2 * kh) * hd, generator=g, device="cuda")).to(dt)
    q, k = fused[:, :qh * hd].unflatten(1, (qh, hd)), fused[:, qh * hd:(qh + kh) * hd].unflatten(1, (kh, hd)) if kh else None
    w = [1 + 0.3 * torch.randn(hd, generator=g, device="cuda") for _ in range(2)] if norm else [None, None]
    cos, sin = ref.rotation(300, rd, "cuda") if turn else (None, None)
    pos = torch.randint(0, 300, (tokens,), generator=g, device="cuda", dtype=torch.int32) if turn else None
    q_out, k_out, err = torch.empty(tokens, qh, hd, device="cuda", dtype=dt), torch.empty(tokens, kh, hd, device="cuda", dtype=dt), word()
    before = fused.clone()
    tb.norm_rope(q, q_out, k, k_out if kh else None, q_weight=w[0], k_weight=w[1], eps=1e-5, cos=cos, sin=sin, positions=pos,
                 error=err, stream=stream())
    for x, o, wt in ((q, q_out, w[0]), (k, k_out, w[1])):
        if x is not None and x.shape[1]:
            y, size = ref.norm_rope(x, wt, 1e-5, cos, sin, pos)
            ref.within(o, y, ref.norm_rope_tolerance(y, size, dt))
    assert err.item() == 0 and torch.equal(before, fused)
    # in place, through the strides of the fused projection: the same bits; the values' part as it was
    tb.norm_rope(q, q, k, k, q_weight=w[0], k_weight=w[1], eps=1e-5, cos=cos, sin=sin, positions=pos, stream=stream())
    assert torch.equal(q, q_out) and (k is None or torch.equal(k, k_out))
    assert torch.equal(fused[:, (qh + kh) * hd:], before[:, (qh + kh) * hd:])


def test_norm_rope_neither_is_a_copy_and_zero_rows_stay_zero():
    x = torch.randn(9, 3, 64, device="cuda").half()
    o = torch.empty_like(x)
    tb.norm_rope(x, o, stream=stream())
    assert torch.equal(x, o)
    z = torch.zeros(9, 3, 64, device="cuda", dtype=torch.float16)
    tb.norm_rope(z, o, q_weight=torch.ones(64, device="cuda"), eps=1e-6, stream=stream())
    assert torch.equal(o, z)


@pytest.mark.parametrize("scale", [2.0 ** -12, 3e4])
def test_norm_rope_small_and_large_values(scale):
    """The squares are summed in f32: neither end of the f16 range leaves it."""
    x = (scale * (0.5 + torch.rand(64, 4, 128, device="cuda"))).half()
    w = torch.ones(128, device="cuda")
    o = torch.empty_like(x)
    tb.norm_rope(x, o, q_weight=w, eps=1e-12, stream=stream())
    y, size = ref.norm_rope(x, w, 1e-12, None, None, None)
    ref.within(o, y, ref.norm_rope_tolerance(y, size, torch.float16))


def test_norm_rope_bad_positions_are_reported_and_skipped():
    q = torch.randn(6, 2, 64, device="cuda").half()
    out = torch.full_like(q, 7.0)
    cos, sin = ref.rotation(10, 64, "cuda")
    pos = torch.tensor([0, -1, 9, 10, 2 ** 31 - 1, 3], dtype=torch.int32, device="cuda")
    err = word()
    tb.norm_rope(q, out, cos=cos, sin=sin, positions=pos, error=err, stream=stream())
    good = torch.tensor([0, 2, 5], device="cuda")
    y, size = ref.norm_rope(q[good], None, 0, cos, sin, pos[good])
    ref.within(out[good], y, ref.norm_rope_tolerance(y, size, torch.float16))
    assert (out[[1, 3, 4]] == 7).all() and err.item() == 6
    tb.norm_rope(q, out, cos=cos, sin=sin, positions=pos, stream=stream())     # no word to report to


# ---- paged_append -------------------------------------------------------------------------

def appended(b, k, v):
    """The pools with k, v [tokens, heads, hd] at the new positions."""
    kp, vp = b.k_pool.clone(), b.v_pool.clone()
    t = 0
    for i in range(b.n):
        for p in range(b.len[i] - b.new[i], b.len[i]):
            page = int(b.table[i, p // b.page])
            kp[page, :, p % b.page], vp[page, :, p % b.page] = k[t], v[t]
            t += 1
    return kp, vp


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("order", [(0, 1, 2), (0, 2, 1), (1, 0, 2)])
@pytest.mark.parametrize("new, lengths, kvh, hd, page", [
    ([1], [1], 1, 64, 8), ([1], [1056], 12, 64, 16), ([3, 0, 7, 1], [3, 0, 20, 130], 2, 128, 16),
    ([0, 0], [5, 0], 3, 64, 8), ([65, 17, 64], [65, 1000, 64], 5, 128, 64), ([33], [33], 8, 64, 1024)])
def test_append_copies_bits(dt, order, new, lengths, kvh, hd, page):
    b = ref.Batch(new, lengths, kvh, kvh, hd, page, ref.DT[dt], order=order, extra_rows=2, pool_fill=NAN)
    b.v[0, 0, 0] = NAN
    b.k[0, 0, 1] = -math.inf
    kp, vp = appended(b, b.k, b.v)
    err = word()
    cache, batch = handles(b)
    tb.paged_append(cache, batch, b.k, b.v, error=err, stream=stream())
    assert same_bits(b.k_pool, kp) and same_bits(b.v_pool, vp) and err.item() == 0


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("norm, rd, explicit", [(False, 64, False), (True, 32, False), (True, 0, False), (True, 64, True)])
def test_append_norms_and_turns_the_keys(dt, norm, rd, explicit):
    b = ref.Batch([5, 1, 0, 40], [5, 77, 9, 40], 3, 3, 64, 16, ref.DT[dt])
    w = 1 + 0.3 * torch.randn(64, device="cuda") if norm else None
    cos, sin = ref.rotation(200, rd, "cuda") if rd else (None, None)
    at = torch.tensor([p for n, m in zip(b.new, b.len) for p in range(m - n, m)], dtype=torch.int32, device="cuda")
    if explicit:
        at = (at * 7 + 3) % 200
    fused = torch.randn(b.tokens, 2 * 3 * 64, device="cuda").to(b.dt)          # k | v of a token in one row
    k, v = fused[:, :192].unflatten(1, (3, 64)), fused[:, 192:].unflatten(1, (3, 64))
    before = b.k_pool.clone()
    cache, batch = handles(b)
    tb.paged_append(cache, batch, k, v, k_weight=w, eps=1e-5, cos=cos, sin=sin, positions=at if explicit else None, stream=stream())
    y, size = ref.norm_rope(k, w, 1e-5, cos, sin, at)
    written = torch.zeros(b.k_pool.shape[:3], dtype=torch.bool, device="cuda")
    t = 0
    for i in range(b.n):
        for p in range(b.len[i] - b.new[i], b.len[i]):
            page, slot = int(b.table[i, p // 16]), p % 16
            ref.within(b.k_pool[page, :, slot], y[t], ref.norm_rope_tolerance(y[t], size[t], b.dt))
            assert torch.equal(b.v_pool[page, :, slot], v[t])
            written[page, :, slot] = True
            t += 1
    assert torch.equal(b.k_pool[~written], before[~written])


def test_append_reports_bad_entries_and_skips_them():
    b = ref.Batch([4, 2, 3, 5], [20, 2, 10, 5], 2, 2, 64, 8, torch.float16)
    good = ref.Batch([4, 2, 3, 5], [20, 2, 10, 5], 2, 2, 64, 8, torch.float16)
    cache, batch = handles(b)
    # the page of positions 16..23 of sequence 0 lies outside the pool: its tokens are not written
    b.table[0, 2] = b.k_pool.shape[0]
    kp, vp = appended(good, b.k, b.v)
    bad = int(good.table[0, 2])
    kp[bad], vp[bad] = good.k_pool[bad], good.v_pool[bad]
    err = word()
    tb.paged_append(cache, batch, b.k, b.v, error=err, stream=stream())
    assert same_bits(b.k_pool, kp) and same_bits(b.v_pool, vp) and err.item() == 11
    # lengths below the new tokens, above the bound and negative, and starts that go backwards
    for name, at, value in (("lengths", 1, 1), ("lengths", 1, 21), ("lengths", 1, -5), ("q_start", 2, 2 ** 31 - 1), ("q_start", 1, -2 ** 31)):
        b = ref.Batch([4, 2, 3, 5], [20, 2, 10, 5], 2, 2, 64, 8, torch.float16)
        getattr(b, name)[at] = value
        kp, vp = appended(good, b.k, b.v)
        skipped = [1] if name == "lengths" else [1, 2] if at == 2 else [0, 1]
        for i in skipped:
            for p in good.table[i].tolist():
                if p >= 0:
                    kp[p], vp[p] = good.k_pool[p], good.v_pool[p]
        err = word()
        cache, batch = handles(b)
        tb.paged_append(cache, batch, b.k, b.v, error=err, stream=stream())
        assert same_bits(b.k_pool, kp) and same_bits(b.v_pool, vp) and err.item() == 10, name


# ---- paged_attention ------------------------------------------------------------------------

def attend(b, gate=None, workspace="full", bits=None, positions=None, max_chunk=None, max_length=None, out=None, **kw):
    cache, batch = handles(b, max_chunk, max_length)
    if workspace == "full":
        size = tb.paged_attention_workspace(cache, batch, b.q.shape[0], b.qh, kw.get("window", 0))
        workspace = torch.full((size // 4 + 4,), NAN, device="cuda")       # what it holds does not matter
    elif isinstance(workspace, int):
        workspace = torch.full((workspace // 4,), NAN, device="cuda")
    out = torch.full_like(b.q, 7.0) if out is None else out
    tb.paged_attention(cache, batch, b.q, out, gate=gate, workspace=workspace,
                       key_valid=None if bits is None else ref.words(bits), key_valid_positions=positions, stream=stream(), **kw)
    return out


BATCHES = [
    # new, lengths, q heads, kv heads, page
    ([1], [1], 1, 1, 8),
    ([1], [64], 12, 12, 16),
    ([1], [1056], 12, 12, 16),
    ([1], [5000], 8, 2, 64),
    ([1, 1, 1, 1, 1], [1, 63, 65, 700, 129], 4, 4, 32),
    ([1, 0, 1], [300, 5, 8], 20, 4, 8),
    ([2, 1, 0, 3], [2, 100, 0, 515], 6, 3, 16),
    ([16, 16, 9], [80, 16, 73], 3, 3, 16),
    ([31], [95], 2, 1, 128),
    ([7, 64], [999, 64], 5, 1, 256),
    ([64, 1, 130], [64, 1, 258], 4, 2, 64),
    ([200], [333], 3, 3, 16),
    ([257, 3], [1300, 40], 8, 2, 1024),
]


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("case", range(len(BATCHES)))
def test_attention(dt, hd, case):
    new, lengths, qh, kvh, page = BATCHES[case]
    b = ref.Batch(new, lengths, qh, kvh, hd, page, ref.DT[dt], seed=case, extra_rows=2)
    want, tol = ref.attention(b)
    for workspace in ("full", None):
        out = attend(b, workspace=workspace)
        ref.within(out[:b.tokens], want, tol)
        assert (out[b.tokens:] == 7).all()                 # rows behind the last sequence


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window", [1, 5, 64, 100, 1000])
@pytest.mark.parametrize("new, lengths", [([1, 1], [1500, 3]), ([20, 5], [400, 5]), ([150, 300], [150, 1024])])
def test_attention_window(hd, window, new, lengths):
    b = ref.Batch(new, lengths, 4, 2, hd, 16, torch.float16, seed=window)
    want, tol = ref.attention(b, window=window)
    # pages that slid out of every window may be gone from the table, their slots may hold anything
    for i, (n, m) in enumerate(zip(new, lengths)):
        gone = max(0, m - n - window + 1)
        for p in range(gone):
            b.k_pool[b.table[i, p // 16], :, p % 16] = NAN
            b.v_pool[b.table[i, p // 16], :, p % 16] = NAN
        b.table[i, :gone // 16] = -5
    err = word()
    for workspace in ("full", None):
        ref.within(attend(b, window=window, workspace=workspace, error=err), want, tol)
    assert err.item() == 0


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("self_visible", [False, True])
@pytest.mark.parametrize("share", [0.0, 0.02, 0.9])
@pytest.mark.parametrize("new, lengths, qh, kvh", [([1, 1, 1], [1, 64, 900], 4, 2), ([16, 9], [80, 73], 3, 3), ([150, 40], [700, 40], 4, 1)])
def test_attention_key_valid(hd, self_visible, share, new, lengths, qh, kvh):
    """Rows whose mask leaves nothing give zeros; masked keys may hold anything."""
    b = ref.Batch(new, lengths, qh, kvh, hd, 16, torch.float16, seed=int(100 * share))
    g = torch.Generator(device="cuda").manual_seed(5)
    m = -(-max(lengths) // 32) * 32
    bits = torch.rand(len(new), m, generator=g, device="cuda") < share
    want, tol = ref.attention(b, bits=bits, self_visible=self_visible)
    gated, gtol = ref.attention(b, bits=bits, self_visible=self_visible, gate=b.gate)
    for i, n in enumerate(lengths):                         # masked for every query of the sequence
        for p in range(n - (new[i] if self_visible else 0)):
            if not bits[i, p]:
                b.k_pool[b.table[i, p // 16], :, p % 16] = NAN
                b.v_pool[b.table[i, p // 16], :, p % 16] = math.inf
    for workspace in ("full", None):
        ref.within(attend(b, bits=bits, self_visible=self_visible, workspace=workspace), want, tol)
        ref.within(attend(b, bits=bits, self_visible=self_visible, workspace=workspace, gate=b.gate), gated, gtol)
    # bits for the first positions alone: the later ones count as set
    few = 37
    part = bits.clone()
    part[:, few:] = True
    if share == 0.9:
        b2 = ref.Batch(new, lengths, qh, kvh, hd, 16, torch.float16, seed=3)
        want, tol = ref.attention(b2, bits=part, self_visible=self_visible)
        ref.within(attend(b2, bits=bits, positions=few, self_visible=self_visible), want, tol)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("new, lengths, qh, kvh", [([50], [90], 4, 1), ([90, 3, 40], [96, 70, 40], 4, 2), ([64], [300], 4, 1),
                                                   ([100, 0, 31], [577, 5, 31], 2, 2), ([33, 2], [97, 1000], 14, 2), ([8] * 40, [120] * 40, 16, 2)])
def test_attention_several_row_tiles_over_few_keys(hd, window, new, lengths, qh, kvh):
    """65 to 256 rows of a problem: more than one tile of rows, each with keys of its own."""
    b = ref.Batch(new, lengths, qh, kvh, hd, 16, torch.float16, seed=window, extra_rows=3)
    g = torch.Generator(device="cuda").manual_seed(2)
    bits = torch.rand(len(new), -(-max(lengths) // 32) * 32, generator=g, device="cuda") < 0.7
    for kw in ({}, {"bits": bits, "self_visible": True, "gate": b.gate}):
        want, tol = ref.attention(b, window=window, **kw)
        for workspace in ("full", None):
            out = attend(b, window=window, workspace=workspace, **kw)
            ref.within(out[:b.tokens], want, tol)
            assert (out[b.tokens:] == 7).all()


@pytest.mark.parametrize("seqs", [1, 2, 3, 5, 9, 14, 20, 37, 75, 150])
@pytest.mark.parametrize("hd, qh, kvh", [(64, 2, 1), (128, 12, 1), (128, 8, 2), (64, 20, 1)])
def test_attention_any_number_of_problems(seqs, hd, qh, kvh):
    """From many splits of few problems over clusters of every size to one team a problem."""
    lengths = [700 - 3 * (i % 50) for i in range(seqs)]
    b = ref.Batch([1] * seqs, lengths, qh, kvh, hd, 32, torch.bfloat16, seed=seqs)
    want, tol = ref.attention(b)
    for workspace in ("full", None):
        ref.within(attend(b, workspace=workspace), want, tol)
    assert torch.equal(attend(b), attend(b))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new, lengths", [([1, 1], [77, 300]), ([5, 30], [5, 131]), ([129, 70], [129, 400])])
def test_attention_unused_slots_hold_anything(hd, new, lengths):
    """NaN in every slot that no sequence owns, and pages that end inside a tile."""
    b = ref.Batch(new, lengths, 4, 2, hd, 32, torch.float16, table_fill=-7)
    own_k, own_v = [b.sequence(i, b.k_pool) for i in range(b.n)], [b.sequence(i, b.v_pool) for i in range(b.n)]
    want, tol = ref.attention(b)
    b.k_pool.fill_(NAN)
    b.v_pool.fill_(NAN)
    for i in range(b.n):
        b.put(i, b.k_pool, own_k[i])
        b.put(i, b.v_pool, own_v[i])
    err = word()
    for workspace in ("full", None):
        ref.within(attend(b, workspace=workspace, error=err), want, tol)
    assert err.item() == 0


@pytest.mark.parametrize("new, lengths", [([1, 4], [200, 90]), ([140, 4], [500, 90])])
@pytest.mark.parametrize("order", [(0, 2, 1), (1, 0, 2), (2, 0, 1)])
def test_attention_strides_scale_and_output_in_place(new, lengths, order):
    b = ref.Batch(new, lengths, 6, 2, 128, 16, torch.bfloat16, order=order)
    fused = torch.randn(b.tokens, 10 * 128, device="cuda").bfloat16()
    b.q = fused[:, 256:256 + 768].unflatten(1, (6, 128))
    want, tol = ref.attention(b, scale=0.2)
    out = torch.empty(6, b.tokens, 128, device="cuda", dtype=torch.bfloat16).transpose(0, 1)
    attend(b, scale=0.2, out=out)
    ref.within(out, want, tol)
    other = out.clone()
    attend(b, scale=0.2, out=b.q)
    assert torch.equal(b.q, other)


@pytest.mark.parametrize("new, lengths, wanted", [([1], [3000], False), ([4, 1], [900, 2000], False), ([4, 1], [900, 9000], True),
                                                  ([150], [2000], True), ([1], [30000], True)])
def test_attention_splits_as_far_as_the_workspace_goes(new, lengths, wanted):
    """A few splits join without a workspace (wanted False); more want one, and take what there is."""
    b = ref.Batch(new, lengths, 4, 2, 128, 64, torch.float16)
    want, tol = ref.attention(b)
    full = tb.paged_attention_workspace(*handles(b), b.tokens, b.qh)
    assert (full > 0) == wanted
    for size in (0, 4, full // 4, full // 2, max(full - 4, 0), "full"):
        a = attend(b, workspace=size)
        ref.within(a, want, tol)
        assert torch.equal(a, attend(b, workspace=size))          # the same bits every time


def test_attention_bounds_above_the_batch():
    """One set of bounds, as a captured graph has them, for any batch within them."""
    for new, lengths in (([1, 1], [5, 40]), ([16, 0], [100, 0]), ([0, 0], [0, 0]), ([3, 50], [3, 333])):
        b = ref.Batch(new, lengths, 4, 2, 64, 16, torch.float16)
        if b.table.shape[1] < 32:
            b.table = torch.cat([b.table, torch.full((2, 32 - b.table.shape[1]), -1, dtype=torch.int32, device="cuda")], 1)
        if not b.tokens:
            continue
        want, tol = ref.attention(b)
        for chunk in (50, 64, 200):
            ref.within(attend(b, max_chunk=chunk, max_length=512), want, tol)


@pytest.mark.parametrize("new, lengths", [([1, 1, 1], [40, 100, 64]), ([100, 40, 64], [140, 100, 64])])
def test_attention_reports_bad_entries(new, lengths):
    def fresh():
        return ref.Batch(new, lengths, 4, 2, 64, 16, torch.float16)
    good = fresh()
    want, tol = ref.attention(good)
    starts = [0, new[0], new[0] + new[1], sum(new)]
    for i, value in ((1, -1), (1, max(lengths) + 1), (1, 0)):
        b = fresh()
        b.lengths[i] = value
        for workspace in ("full", None):
            err = word()
            out = attend(b, workspace=workspace, error=err)
            assert err.item() == 10 and (out[starts[i]:starts[i + 1]] == 7).all()
            keep = torch.ones(b.tokens, dtype=torch.bool, device="cuda")
            keep[starts[i]:starts[i + 1]] = False
            ref.within(out[keep], want[keep], tol[keep])
    # a page outside the pool: its keys and values read as zeros
    for page in (-1, 2 ** 31 - 1, good.k_pool.shape[0]):
        b = fresh()
        b.table[0, 1] = page
        z = fresh()
        p = z.table[0, 1]
        z.k_pool[p], z.v_pool[p] = 0, 0
        w2, t2 = ref.attention(z)
        err = word()
        ref.within(attend(b, error=err), w2, t2)
        assert err.item() == 11


def test_attention_far_offsets():
    """A pool of more than 2^31 values, its last pages in use."""
    pages, kvh, page, hd = 70000, 4, 64, 128
    pool = torch.zeros(pages, 2, kvh, page, hd, device="cuda", dtype=torch.float16)      # 4.6e9 values
    b = ref.Batch([1, 40], [700, 130], 8, kvh, hd, page, torch.float16)
    used = b.k_pool.shape[0]
    at = torch.arange(pages - used, pages, device="cuda")
    pool[at, 0], pool[at, 1] = b.k_pool, b.v_pool
    want, tol = ref.attention(b)
    b.k_pool, b.v_pool = pool[:, 0], pool[:, 1]
    b.table = torch.where(b.table >= 0, b.table + pages - used, b.table)
    ref.within(attend(b), want, tol)
    kp = pool[at, 0].clone()
    cache, batch = handles(b)
    tb.paged_append(cache, batch, b.k, b.v, stream=stream())
    last = int(b.table[1, 129 // 64])
    assert torch.equal(b.k_pool[last, :, 129 % 64], b.k[40]) and torch.equal(b.v_pool[last, :, 129 % 64], b.v[40])
    assert not torch.equal(pool[at, 0], kp)


def test_attention_large_scores_and_repeated_maxima():
    """Scores far apart (the running maximum moves late) and all alike."""
    for new, m in ((1, 2000), (150, 2000)):
        b = ref.Batch([new], [m], 4, 2, 128, 64, torch.float16)
        k = b.sequence(0, b.k_pool)
        b.put(0, b.k_pool, k * torch.linspace(0, 6, m, device="cuda")[None, :, None].double())
        want, tol = ref.attention(b, scale=0.5)
        ref.within(attend(b, scale=0.5), want, tol)
        b.k_pool.zero_()
        want, tol = ref.attention(b)
        ref.within(attend(b), want, tol)


@pytest.mark.parametrize("new, lengths", [([1, 1], [40, 3000]), ([4, 1], [4, 900]), ([150, 1], [2000, 30]), ([1, 1], [5, 96])])
def test_attention_hands_on_what_is_not_a_number(new, lengths):
    """A query or a visible key that is NaN gives NaN in its rows, however the keys are split, and nowhere
    else; an infinite score does too (inf - inf)."""
    for bad in (NAN, math.inf):
        b = ref.Batch(new, lengths, 4, 2, 128, 16, torch.float16)
        want, tol = ref.attention(b)
        b.q[0, 1] = NAN                                            # one head of the first token
        if math.isinf(bad):
            b.q[0, 1] = 1.0
            b.k_pool[b.table[0, 0], 0, 0] = bad                    # seen by every token of sequence 0, heads 0 and 1
        hit = torch.zeros(b.tokens, 4, dtype=torch.bool, device="cuda")
        if math.isinf(bad):
            hit[:new[0], :2] = True
        else:
            hit[0, 1] = True
        for workspace in ("full", None):
            out = attend(b, workspace=workspace)
            if not math.isinf(bad):
                assert torch.isnan(out[hit]).all()
            ref.within(out[~hit], want[~hit], tol[~hit])


def test_calls_refuse_other_memory():
    b = ref.Batch([1, 4], [20, 9], 4, 2, 64, 16, torch.float16)
    cache, batch = handles(b)
    with pytest.raises(tb.TimestralError, match="q is not device memory"):
        tb.paged_attention(cache, batch, b.q.cpu(), b.q)
    with pytest.raises(tb.TimestralError, match="table is not device memory"):
        tb.paged_attention(tb.PagedCache(b.k_pool, b.v_pool, b.table.cpu()), batch, b.q, b.q)
    with pytest.raises(tb.TimestralError, match="lengths is not device memory"):
        tb.paged_append(cache, tb.PagedBatch(b.q_start, b.lengths.cpu(), 4, 20), b.k, b.v)
    with pytest.raises(tb.TimestralError, match="q_weight is not device memory"):
        tb.norm_rope(b.q, b.q, q_weight=torch.ones(64))
    with pytest.raises(tb.TimestralError, match="workspace is not device memory"):
        tb.paged_attention(cache, batch, b.q, b.q, workspace=torch.empty(1 << 20, dtype=torch.uint8).pin_memory())


def test_another_stream_and_graphs_with_new_lengths():
    """Captured once at the bounds, replayed for longer and longer sequences; a second graph with a
    workspace of its own at the same time."""
    b = ref.Batch([1, 1], [700, 300], 8, 2, 128, 16, torch.float16)
    side = torch.cuda.Stream()
    graphs = []
    cos, sin = ref.rotation(b.max_length, 128, "cuda")
    cache, batch = handles(b)
    for _ in range(2):
        ws = torch.empty(max(16, tb.paged_attention_workspace(cache, batch, 2, 8)), dtype=torch.uint8, device="cuda")
        out = torch.empty_like(b.q)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            tb.paged_append(cache, batch, b.k, b.v, cos=cos, sin=sin, stream=stream())
            tb.paged_attention(cache, batch, b.q, out, workspace=ws, stream=stream())
        graphs.append((g, out, ws))
    for first, second in ((1, 16), (17, 250), (699, 299), (700, 300)):
        b.len = [first, second]
        b.lengths.copy_(torch.tensor(b.len, dtype=torch.int32))
        b.q.normal_()
        b.k.normal_()
        torch.cuda.synchronize()
        for i, (g, _, _) in enumerate(graphs):
            with torch.cuda.stream(side if i else torch.cuda.default_stream()):
                g.replay()
        torch.cuda.synchronize()
        want, tol = ref.attention(b)
        for _, out, _ in graphs:
            ref.within(out, want, tol)
        at = torch.tensor([first - 1, second - 1], dtype=torch.int32, device="cuda")
        y, size = ref.norm_rope(b.k, None, 0, cos, sin, at)
        for i in range(2):
            got = b.sequence(i, b.k_pool)[:, -1]
            ref.within(got, y[i], ref.norm_rope_tolerance(y[i], size[i], b.dt))


@pytest.mark.parametrize("dt, qh, kvh, hd", [("f16", 12, 12, 64), ("bf16", 8, 2, 128), ("f16", 10, 2, 128)])
def test_the_operators_together(dt, qh, kvh, hd):
    """A layer's attention as it is served: prompts in chunks, then token by token, for sequences of
    different lengths, against attention over the whole sequences in 64 bits."""
    dt, page, total = ref.DT[dt], 16, [150, 77, 203]
    torch.manual_seed(0)
    cos, sin = ref.rotation(max(total), hd, "cuda")
    qw, kw = 1 + 0.2 * torch.randn(hd, device="cuda"), 1 + 0.2 * torch.randn(hd, device="cuda")
    projected = [torch.randn(t, (qh + 2 * kvh) * hd, device="cuda").to(dt) for t in total]
    pages = [-(-t // page) for t in total]
    pool = torch.full((sum(pages), 2, page, kvh, hd), NAN, device="cuda", dtype=dt)
    k_pool, v_pool = pool[:, 0].transpose(1, 2), pool[:, 1].transpose(1, 2)
    table = torch.full((3, max(pages)), -1, dtype=torch.int32, device="cuda")
    for i, p in enumerate(torch.randperm(sum(pages), device="cuda").int().split(pages)):
        table[i, :pages[i]] = p
    err, results, queries, done = word(), [[] for _ in total], [[] for _ in total], [0, 0, 0]
    for step in ([100, 40, 90], [37, 30, 0], [12, 6, 112], [1, 1, 1]):
        new = step
        length = [d + n for d, n in zip(done, new)]
        q_start = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
        lengths = torch.tensor(length, dtype=torch.int32, device="cuda")
        x = torch.cat([projected[i][done[i]:length[i]] for i in range(3)])
        at = torch.cat([torch.arange(done[i], length[i], device="cuda") for i in range(3)]).int()
        q, k, v = (y.unflatten(1, (-1, hd)) for y in x.split([qh * hd, kvh * hd, kvh * hd], 1))
        cache, batch = tb.PagedCache(k_pool, v_pool, table), tb.PagedBatch(q_start, lengths, max(new), max(length))
        tb.norm_rope(q, q, q_weight=qw, eps=1e-6, cos=cos, sin=sin, positions=at, error=err, stream=stream())
        tb.paged_append(cache, batch, k, v, k_weight=kw, eps=1e-6, cos=cos, sin=sin, error=err, stream=stream())
        ws = torch.empty(tb.paged_attention_workspace(cache, batch, q.shape[0], qh), dtype=torch.uint8, device="cuda")
        out = torch.empty(q.shape, dtype=dt, device="cuda")
        tb.paged_attention(cache, batch, q, out, workspace=ws if ws.numel() else None, error=err, stream=stream())
        for i, (o, y) in enumerate(zip(out.split(new), q.split(new))):
            results[i].append(o)
            queries[i].append(y)
        done = length
    assert err.item() == 0 and done == total
    for i, t in enumerate(total):
        # the stored queries, keys and values against the projections', and the results against
        # attention over what is stored (`projected` still holds what x was cut from)
        b = ref.Batch([t], [t], qh, kvh, hd, page, dt)
        q, k, v = (y.unflatten(1, (-1, hd)) for y in projected[i].split([qh * hd, kvh * hd, kvh * hd], 1))
        at = torch.arange(t, device="cuda")
        b.q = torch.cat(queries[i])
        b.k_pool, b.v_pool, b.table = k_pool, v_pool, table[i:i + 1]
        for got, x, w in ((b.q, q, qw), (b.sequence(0, k_pool).transpose(0, 1), k, kw)):
            y, size = ref.norm_rope(x, w, 1e-6, cos, sin, at)
            ref.within(got, y, ref.norm_rope_tolerance(y, size, dt))
        assert torch.equal(b.sequence(0, v_pool).transpose(0, 1), v.double())
        want, tol = ref.attention(b)
        ref.within(torch.cat(results[i]), want, tol)
