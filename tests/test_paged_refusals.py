"""The operators over a paged cache refuse bad arguments before any device work (no GPU)."""
import ctypes as C

import pytest
import torch

import timestral_b200 as tb


def arrays(dt=torch.float16, tokens=4, qh=4, kvh=2, hd=64, page=16, pages=6, seqs=2, width=3):
    return dict(q=torch.zeros(tokens, qh, hd, dtype=dt), out=torch.zeros(tokens, qh, hd, dtype=dt),
                k=torch.zeros(tokens, kvh, hd, dtype=dt), v=torch.zeros(tokens, kvh, hd, dtype=dt),
                k_pool=torch.zeros(pages, kvh, page, hd, dtype=dt), v_pool=torch.zeros(pages, kvh, page, hd, dtype=dt),
                table=torch.zeros(seqs, width, dtype=torch.int32), q_start=torch.tensor([0, 2, 4], dtype=torch.int32),
                lengths=torch.tensor([2, 2], dtype=torch.int32))


def handles(a, max_chunk=2, max_length=8):
    return tb.PagedCache(a["k_pool"], a["v_pool"], a["table"]), tb.PagedBatch(a["q_start"], a["lengths"], max_chunk, max_length)


def refused(call, *words):
    with pytest.raises(tb.TimestralError) as e:
        call()
    for w in words:
        assert w in str(e.value), str(e.value)


@pytest.mark.parametrize("change, word", [
    (dict(k_pool=torch.zeros(6, 2, 16, 64)), "float32"),
    (dict(v_pool=torch.zeros(6, 2, 16, 64, dtype=torch.bfloat16)), "different types"),
    (dict(v_pool=torch.zeros(6, 2, 8, 64, dtype=torch.float16)), "alike"),
    (dict(k_pool=torch.zeros(6, 2, 64, 16, dtype=torch.float16).transpose(2, 3)), "last axis"),
    (dict(table=torch.zeros(2, 3, dtype=torch.int64)), "int32"),
    (dict(table=torch.zeros(3, dtype=torch.int32)), "entries"),
    (dict(q_start=torch.tensor([0, 4], dtype=torch.int32)), "q_start"),
])
def test_handles_refuse(change, word):
    a = arrays()
    a.update(change)
    refused(lambda: handles(a), word)


@pytest.mark.parametrize("make, word", [
    (dict(page=12), "page_size 12"), (dict(page=4), "page_size 4"), (dict(page=2048), "page_size 2048"),
    (dict(hd=96), "head_dim 96"), (dict(qh=3), "q_heads 3"), (dict(pages=0), "0 pages"),
])
def test_attention_refuses_geometry(make, word):
    a = arrays(**make)
    cache, batch = handles(a)
    refused(lambda: tb.paged_attention(cache, batch, a["q"], a["out"]), word)


def test_attention_refuses_arguments():
    a = arrays()
    cache, batch = handles(a)
    run = lambda **kw: tb.paged_attention(cache, batch, kw.pop("q", a["q"]), kw.pop("out", a["out"]), **kw)  # noqa: E731
    refused(lambda: run(q=a["q"].bfloat16()), "unlike")
    refused(lambda: run(out=a["out"][:3]), "shape")
    refused(lambda: run(q=torch.zeros(4, 4, 32, dtype=torch.float16)), "shape")
    refused(lambda: run(window=-1), "window")
    refused(lambda: run(scale=float("nan")), "scale")
    refused(lambda: run(gate=a["q"].transpose(1, 2).contiguous().transpose(1, 2)), "last axis")
    refused(lambda: run(out=a["out"][:1].expand(4, 4, 64)), "overlap")
    base = torch.zeros(4 * 4 * 64 + 8, dtype=torch.float16)
    refused(lambda: run(q=base[1:1 + 4 * 4 * 64].view(4, 4, 64)), "aligned")
    refused(lambda: run(q=torch.zeros(4, 4 * 64 + 4, dtype=torch.float16)[:, :256].unflatten(1, (4, 64))), "multiple of 8")
    refused(lambda: run(key_valid=torch.zeros(1, 1, dtype=torch.int32)), "key_valid")
    refused(lambda: run(key_valid=torch.zeros(2, 1, dtype=torch.int32), key_valid_positions=33), "32 bits")
    refused(lambda: run(key_valid=torch.zeros(2, 1, dtype=torch.int64)), "int32")
    refused(lambda: run(error=torch.zeros(1, dtype=torch.int64)), "int32")
    refused(lambda: run(workspace=torch.zeros(64, 2, dtype=torch.uint8)[:, :1]), "dense")
    long = tb.PagedBatch(a["q_start"], a["lengths"], 2, 49)
    refused(lambda: tb.paged_attention(cache, long, a["q"], a["out"]), "max_length 49")
    more = tb.PagedBatch(torch.zeros(4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), 2, 8)
    refused(lambda: tb.paged_attention(cache, more, a["q"], a["out"]), "3 sequences")
    refused(lambda: tb.paged_attention(cache, tb.PagedBatch(a["q_start"], a["lengths"], -1, 8), a["q"], a["out"]), "negative")


def test_append_refuses():
    a = arrays()
    cache, batch = handles(a)
    cos = torch.zeros(8, 32)
    run = lambda **kw: tb.paged_append(cache, batch, kw.pop("k", a["k"]), kw.pop("v", a["v"]), **kw)  # noqa: E731
    refused(lambda: run(k=a["q"]), "shape")
    refused(lambda: run(v=a["v"][:2]), "shape")
    refused(lambda: run(cos=cos), "missing")
    refused(lambda: run(cos=cos, sin=torch.zeros(8, 16)), "alike")
    refused(lambda: run(cos=torch.zeros(8, 40), sin=torch.zeros(8, 40)), "rope_dim 80")
    refused(lambda: run(cos=torch.zeros(8, 4), sin=torch.zeros(8, 4)), "rope_dim 8")
    refused(lambda: run(cos=torch.zeros(0, 32), sin=torch.zeros(0, 32)), "0 rows")
    refused(lambda: run(cos=cos.double(), sin=cos.double()), "float32")
    refused(lambda: run(cos=torch.zeros(8, 34)[:, :32], sin=torch.zeros(8, 34)[:, :32]), "stride")
    refused(lambda: run(cos=cos, sin=cos, positions=torch.zeros(3, dtype=torch.int32)), "positions")
    refused(lambda: run(k_weight=torch.zeros(32)), "k_weight")
    refused(lambda: run(k_weight=torch.zeros(64), eps=-1.0), "eps")


def test_norm_rope_refuses():
    q = torch.zeros(3, 4, 64, dtype=torch.float16)
    cos, pos = torch.zeros(8, 32), torch.zeros(3, dtype=torch.int32)
    refused(lambda: tb.norm_rope(q, q.bfloat16()), "unlike")
    refused(lambda: tb.norm_rope(q, q[:2]), "shape")
    refused(lambda: tb.norm_rope(q.float(), q.float()), "float32")
    refused(lambda: tb.norm_rope(q, q, q[:2], q), "shape")
    refused(lambda: tb.norm_rope(q, q, cos=cos, sin=cos), "positions")
    refused(lambda: tb.norm_rope(q, q, q_weight=torch.zeros(64), eps=float("inf")), "eps")
    refused(lambda: tb.norm_rope(q, q, q_weight=torch.zeros(64, dtype=torch.float64)), "float32")
    for hd in (24, 272, 8):
        z = torch.zeros(3, 4, hd, dtype=torch.float16)
        refused(lambda: tb.norm_rope(z, z), f"head_dim {hd}")
    refused(lambda: tb.norm_rope(q, q[:1].expand(3, 4, 64), cos=cos, sin=cos, positions=pos), "overlap")


def test_outputs_in_place_keep_the_layout():
    """The input's address with other strides: a block would write what another has not read yet."""
    a = arrays()
    cache, batch = handles(a)
    q = torch.zeros(4, 4, 64, dtype=torch.float16)
    refused(lambda: tb.paged_attention(cache, batch, q, q.transpose(0, 1)), "other strides")
    refused(lambda: tb.norm_rope(q, q.transpose(0, 1)), "q_out is its input")
    refused(lambda: tb.norm_rope(q, q, q, q.transpose(0, 1)), "k_out is its input")


def test_c_entries_refuse_null():
    L = tb.lib()
    assert L.tsb_norm_rope(None, None) == tb.TSB_ERR_ARG
    assert L.tsb_paged_append(None, None) == tb.TSB_ERR_ARG
    assert L.tsb_paged_attention(None, None) == tb.TSB_ERR_ARG
    assert b"args is NULL" in L.timestral_capi_last_error(None)
    assert L.tsb_paged_attention_workspace(None) == 0
    assert L.tsb_paged_attention(C.byref(tb.PagedAttentionArgs()), None) == tb.TSB_ERR_ARG
    assert b"cache is NULL" in L.timestral_capi_last_error(None)


def test_nothing_to_do_needs_no_device():
    """No token or no sequence: the calls succeed, whatever the machine."""
    a = arrays(tokens=0)
    cache, _ = handles(a)
    none = tb.PagedBatch(torch.zeros(1, dtype=torch.int32), torch.zeros(0, dtype=torch.int32), 0, 0)
    tb.paged_attention(cache, none, a["q"], a["out"])
    tb.paged_append(cache, none, a["k"], a["v"])
    tb.norm_rope(a["q"], a["out"])


def test_struct_layouts(tmp_path):
    """The ctypes structures have the header's sizes and offsets."""
    import shutil
    import subprocess
    from pathlib import Path
    cc = shutil.which("gcc") or shutil.which("cc")
    if not cc:
        pytest.skip("no C compiler")
    structs = {"tsb_heads": tb.Heads, "tsb_paged_cache": tb.PagedCacheArgs, "tsb_paged_batch": tb.PagedBatchArgs,
               "tsb_rotation": tb.Rotation, "tsb_norm_rope_args": tb.NormRopeArgs,
               "tsb_paged_append_args": tb.PagedAppendArgs, "tsb_paged_attention_args": tb.PagedAttentionArgs}
    lines, want = [], []
    for name, s in structs.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(C.sizeof(s))
        for f in s._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {f[0]}));')
            want.append(getattr(s, f[0]).offset)
    src = tmp_path / "s.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "timestral_b200.h"\nint main(void){' + "\n".join(lines) + "return 0;}\n")
    inc = Path(__file__).resolve().parents[1] / "include"
    subprocess.run([cc, "-std=c99", "-Wall", "-Werror", f"-I{inc}", str(src), "-o", str(tmp_path / "s")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == want
