"""paged_attention where most of a row's weight lies in many keys of small probabilities each (a long
past behind one key that stands out): f16 probabilities must not lose them."""
import math

import pytest
import torch

import paged_ref as ref
import timestral_b200 as tb

pytestmark = pytest.mark.gpu


def stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("seqs, new", [(1500, 1), (160, 300)])
@pytest.mark.parametrize("ahead", [26, 30])
def test_many_small_probabilities(dt, hd, seqs, new, ahead):
    """The first key's score is `ahead` (in log2 units), all others' 0, the first value 0, all others' 1:
    out = w / (1 + w), w = (keys seen - 1) 2^-ahead. Enough problems that no keys are split, so that the
    first key is the reference of all others; the sequences share their pages.

    Tolerance: one rounding of the result; 2^-17 for the exponent and 2^-24 a key for the sums, as
    paged_ref; and a 16-bit probability's own rounding. The largest probability is held as at least 2^7,
    so f16's half step of 2^-25 for small ones is 2^-32 of it, for each of the keys."""
    dt, keys, page = ref.DT[dt], 32768, 1024
    k_pool = torch.zeros(keys // page, 1, page, hd, device="cuda", dtype=dt)
    v_pool = torch.ones_like(k_pool)
    k_pool[0, 0, 0] = ahead / hd                              # exact: q is 1
    v_pool[0, 0, 0] = 0
    table = torch.arange(keys // page, dtype=torch.int32, device="cuda").repeat(seqs, 1)
    q_start = torch.arange(0, seqs * new + 1, new, dtype=torch.int32, device="cuda")
    lengths = torch.full((seqs,), keys, dtype=torch.int32, device="cuda")
    q = torch.ones(seqs * new, 1, hd, device="cuda", dtype=dt)
    out, err = torch.full_like(q, 7.0), torch.zeros(1, dtype=torch.int32, device="cuda")
    tb.paged_attention(tb.PagedCache(k_pool, v_pool, table), tb.PagedBatch(q_start, lengths, new, keys), q, out,
                       scale=math.log(2), error=err, stream=stream())
    seen = keys - new + 1 + torch.arange(new, device="cuda", dtype=torch.float64)
    w = ((seen - 1) * 2.0 ** -ahead).repeat(seqs)[:, None, None].expand(out.shape)
    want = w / (1 + w)
    e = (2 * 2.0 ** -17 + keys * 2.0 ** -24) * want + (keys * 2.0 ** -32 if dt == torch.float16 else ref.half_step(dt) * want)
    ref.within(out, want, e + (ref.half_step(dt) + 2.0 ** -23) * (want + e) + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps)
    assert err.item() == 0
