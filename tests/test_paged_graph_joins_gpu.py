"""Captured calls of paged_attention whose splits join through the workspace in a second kernel."""
import pytest
import torch

import paged_ref as ref
import timestral_b200 as tb

pytestmark = pytest.mark.gpu


def stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("hd, qh, kvh, new, lengths, later", [
    (128, 8, 2, [1], [30000], ([4097], [29999])), (128, 4, 2, [4, 1], [900, 9000], ([900, 3], [17, 8999])),
    (128, 4, 2, [150], [2000], ([1999], [151]))])
def test_captured_joins_with_other_lengths(hd, qh, kvh, new, lengths, later):
    """Two graphs over one cache with workspaces of their own, replayed at the same time on two streams, and an eager
    call beside them."""
    b = ref.Batch(new, lengths, qh, kvh, hd, 64, torch.float16)
    cache, batch = tb.PagedCache(b.k_pool, b.v_pool, b.table), tb.PagedBatch(b.q_start, b.lengths, b.max_chunk, b.max_length)
    size = tb.paged_attention_workspace(cache, batch, b.tokens, qh)
    assert size > 0
    side, graphs = torch.cuda.Stream(), []
    for _ in range(2):
        ws, out = torch.full((size // 4,), float("nan"), device="cuda"), torch.empty_like(b.q)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            tb.paged_attention(cache, batch, b.q, out, workspace=ws, stream=stream())
        graphs.append((g, out, ws))
    eager = torch.empty(size // 4, device="cuda"), torch.empty_like(b.q)
    for at in (lengths,) + later:
        b.len = [max(n, x) for n, x in zip(b.new, at)]
        b.lengths.copy_(torch.tensor(b.len, dtype=torch.int32))
        b.q.normal_()
        torch.cuda.synchronize()
        for i, (g, _, _) in enumerate(graphs):
            with torch.cuda.stream(side if i else torch.cuda.default_stream()):
                for _ in range(3):
                    g.replay()
        other = torch.cuda.Stream()
        with torch.cuda.stream(other):
            tb.paged_attention(cache, batch, b.q, eager[1], workspace=eager[0], stream=stream())
        torch.cuda.synchronize()
        want, tol = ref.attention(b)
        for out in (graphs[0][1], graphs[1][1], eager[1]):
            ref.within(out, want, tol)
            assert torch.equal(out, eager[1])
