"""Pages whose positions no new token sees because their bits are clear may be gone from the table."""
import pytest
import torch

import paged_ref as ref
import timestral_b200 as tb

pytestmark = pytest.mark.gpu


def stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("self_visible", [False, True])
@pytest.mark.parametrize("page", [8, 16, 64, 256])
@pytest.mark.parametrize("hd, new, lengths, qh, kvh", [
    (64, [1, 3], [70, 96], 2, 2), (64, [1, 1], [900, 77], 4, 2), (128, [1], [6000], 8, 1), (128, [5, 9], [300, 1000], 4, 2),
    (64, [150, 40], [700, 300], 4, 1), (128, [300], [900], 3, 3)])
def test_pages_behind_clear_bits_are_not_read(hd, new, lengths, qh, kvh, page, self_visible):
    """Entries of such pages name no page of the pool: no fault is reported and the results are those of
    the masked keys. A page with one visible position still has to be there."""
    b = ref.Batch(new, lengths, qh, kvh, hd, page, torch.float16, seed=page)
    g = torch.Generator(device="cuda").manual_seed(1)
    m = -(-max(lengths) // 32) * 32
    bits = torch.rand(len(new), m, generator=g, device="cuda") < 0.5
    gone = []
    for i, (n, length) in enumerate(zip(new, lengths)):
        pages = -(-length // page)
        for p in range(pages):
            first, end = p * page, min((p + 1) * page, length)
            # every second page, unless a new token sees itself there
            if p % 2 == 0 and not (self_visible and end > length - n):
                bits[i, first:min((p + 1) * page, m)] = False
                gone.append((i, p))
            else:
                bits[i, first] = True
    want, tol = ref.attention(b, bits=bits, self_visible=self_visible)
    for j, (i, p) in enumerate(gone):
        b.table[i, p] = (-1, 2 ** 31 - 1, b.k_pool.shape[0])[j % 3]
    cache, batch = tb.PagedCache(b.k_pool, b.v_pool, b.table), tb.PagedBatch(b.q_start, b.lengths, b.max_chunk, b.max_length)
    size = tb.paged_attention_workspace(cache, batch, b.tokens, qh)
    for workspace in (None, torch.empty(size, dtype=torch.uint8, device="cuda") if size else None):
        out, err = torch.full_like(b.q, 7.0), torch.zeros(1, dtype=torch.int32, device="cuda")
        tb.paged_attention(cache, batch, b.q, out, key_valid=ref.words(bits), self_visible=self_visible, workspace=workspace,
                           error=err, stream=stream())
        ref.within(out, want, tol)
        assert err.item() == 0
    if not gone:                                              # (every page holds new tokens, which see themselves)
        return
    # one visible position on a page that is not there
    i, p = gone[-1]
    bits[i, p * page] = True
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    tb.paged_attention(cache, batch, b.q, out, key_valid=ref.words(bits), self_visible=self_visible, error=err, stream=stream())
    assert err.item() == 11
