"""Serving operators without a GPU: the rotary table, what the entry points refuse (in Python and behind the C ABI, before anything is launched)."""
import ctypes

import pytest
import torch

from ralf_amd import _lib, ops
from ralf_amd._abi import RalfLogitsDesc, RalfPagedAttnDesc, RalfPagedKV, RalfRopeDesc

FAKE = 1 << 20      # an aligned address that nothing may follow


def test_rope_table():
    f, a = ops.rope_table((2, 3), theta=100.0)
    assert a.tolist() == [0, 0, 1, 1, 1] and f.dtype == torch.float64
    assert torch.allclose(f, 100.0 ** (-torch.arange(5, dtype=torch.float64) / 5), rtol=1e-15)
    f, a = ops.rope_table((2, 3), theta=100.0, ladder="axis")
    assert torch.allclose(f, torch.tensor([1.0, 100 ** -0.5, 1.0, 100 ** (-1 / 3), 100 ** (-2 / 3)], dtype=torch.float64), rtol=1e-15)
    assert ops.rope_table((1, 3, 2), order="round")[1].tolist() == [0, 1, 2, 1, 2, 1]
    for bad in (dict(sections=()), dict(sections=(0,)), dict(sections=(-1, 2)), dict(sections=(1,), ladder="x"), dict(sections=(1,), order="x")):
        with pytest.raises(AssertionError):
            ops.rope_table(**bad)


def rope_args(**kw):
    f, a = ops.rope_table((4, 4))
    d = dict(x=torch.zeros(3, 2, 16), pos=torch.zeros(2, 3, dtype=torch.int64), freq=f, axis=a)
    d.update(kw)
    return d


@pytest.mark.parametrize("kw,says", [
    (dict(x=torch.zeros(3, 2, 16, dtype=torch.float16)), "dtype"), (dict(x=torch.zeros(3, 32)), "heads"), (dict(x=torch.zeros(3, 16, 2).transpose(1, 2)), "contiguous"),
    (dict(pos=torch.zeros(2, 3, dtype=torch.int32)), "pos"), (dict(pos=torch.zeros(2, 4, dtype=torch.int64)), "pos"), (dict(freq=torch.zeros(8)), "freq"),
    (dict(x=torch.zeros(3, 2, 14)), "pairs"), (dict(out=torch.zeros(3, 2, 17)), "shape"), (dict(out=torch.zeros(3, 2, 16, dtype=torch.bfloat16)), "type"), (dict(), "GPU")])
def test_rope_refuses(kw, says):
    kw = rope_args(**kw)
    with pytest.raises(AssertionError, match=says):
        ops.rope_axes(kw.pop("x"), kw.pop("pos"), kw.pop("freq"), kw.pop("axis"), **kw)


def test_rope_refuses_a_leaf_in_a_capture(monkeypatch):
    from ralf_amd import functional

    a = rope_args(x=torch.zeros(3, 2, 16, requires_grad=True))
    monkeypatch.setattr(functional, "_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="inverse=True"):
        functional.rope_axes(a["x"], a["pos"], a["freq"], a["axis"])
    monkeypatch.undo()
    with pytest.raises(AssertionError, match="GPU"):
        functional.rope_axes(a["x"], a["pos"], a["freq"], a["axis"])
    monkeypatch.setattr(functional, "_capturing", lambda: True)
    with torch.no_grad(), pytest.raises(AssertionError, match="GPU"):        # (no gradient asked for: on to the ordinary checks)
        functional.rope_axes(a["x"], a["pos"], a["freq"], a["axis"])


def paged(store=torch.bfloat16, n=4, page=16, heads=2, dim=32, B=2):
    return dict(pool=ops.paged_kv_pool(n, page, heads, dim, store, device="cpu"), table=torch.zeros(B, 2, dtype=torch.int32), q_start=torch.tensor([0, 1, 3], dtype=torch.int32),
                kv_len=torch.tensor([5, 9], dtype=torch.int32))


def test_pool():
    p = ops.paged_kv_pool(3, 16, 2, 32, torch.float8_e4m3fn, device="cpu")
    assert p.k.shape == (3, 2, 16, 32) and p.k.dtype == torch.float8_e4m3fn and p.v_exp.shape == (3, 2, 16) and p.k_exp.dtype == torch.uint8
    assert ops.paged_kv_pool(3, 16, 2, 32, torch.float32, device="cpu").k_exp is None
    with pytest.raises(AssertionError):
        ops.paged_kv_pool(3, 16, 2, 32, torch.float16, device="cpu")


@pytest.mark.parametrize("kw,says", [
    (dict(table=torch.zeros(2, 2, dtype=torch.int64)), "table"), (dict(kv_len=torch.zeros(3, dtype=torch.int32)), "kv_len"), (dict(kv_len=torch.zeros(2, dtype=torch.int64)), "kv_len"),
    (dict(q_start=torch.zeros(2, dtype=torch.int32)), "q_start"), (dict(table=torch.zeros(1, 2, dtype=torch.int32).expand(2, 2)), "overlap"), (dict(), "GPU"),
    (dict(pool=ops.PagedKV(torch.zeros(4, 2, 16, 32), torch.zeros(4, 2, 16, 32, dtype=torch.bfloat16))), "cache"),
    (dict(pool=ops.PagedKV(torch.zeros(4, 2, 16, 32, dtype=torch.int8), torch.zeros(4, 2, 16, 32, dtype=torch.int8))), "exponents"),
    (dict(pool=ops.PagedKV(torch.zeros(4, 2, 32, 16).transpose(2, 3), torch.zeros(4, 2, 32, 16).transpose(2, 3))), "contiguous")])
def test_paged_refuses(kw, says):
    a = paged()
    a.update(kw)
    k = torch.zeros(3, 2, 32, dtype=torch.bfloat16)
    with pytest.raises(AssertionError, match=says):
        ops.paged_kv_write(a["pool"], k, k, a["table"], a["q_start"], a["kv_len"])
    with pytest.raises(AssertionError, match=says.replace("q_start", "start")):
        ops.paged_kv_read(a["pool"], a["table"], a["kv_len"], a["q_start"], 3)
    if a["pool"].k.dtype == torch.bfloat16:
        with pytest.raises(AssertionError, match=says):
            ops.paged_attention(torch.zeros(3, 4, 32, dtype=torch.bfloat16), a["pool"], a["table"], a["q_start"], a["kv_len"])


def test_paged_rows_refused():
    a = paged()
    k = torch.zeros(3, 2, 32, dtype=torch.bfloat16)
    for kk, vv, says in ((k.half(), k.half(), "float16"), (k, k.float(), "v"), (k[:, :1], k[:, :1], "rows"), (k[..., :16], k[..., :16], "rows")):
        with pytest.raises(AssertionError, match=says):
            ops.paged_kv_write(a["pool"], kk, vv, a["table"], a["q_start"], a["kv_len"])
    q = torch.zeros(3, 4, 32, dtype=torch.bfloat16)
    for qq, kw, says in ((q.float(), {}, "queries"), (q[:, :3], {}, "heads"), (q[..., :16], {}, "heads"), (q, dict(window=-1), "negative"), (q, dict(max_q=-1), "negative"),
                         (q, dict(out=torch.zeros(3, 4, 32)), "out"), (q.half(), {}, "dtype")):
        with pytest.raises(AssertionError, match=says):
            ops.paged_attention(qq, a["pool"], a["table"], a["q_start"], a["kv_len"], **kw)
    with pytest.raises(AssertionError, match="out"):
        ops.paged_kv_read(a["pool"], a["table"], a["kv_len"], a["q_start"], 3, out=(torch.zeros(3, 2, 32), torch.zeros(4, 2, 32)))


@pytest.mark.parametrize("kw,says", [
    (dict(logits=torch.zeros(2, 5, dtype=torch.float16)), "logits"), (dict(logits=torch.zeros(5, 2).t()), "logits"), (dict(tokens=torch.zeros(2, 3, dtype=torch.int32)), "tokens"),
    (dict(lens=torch.zeros(2, dtype=torch.int64)), "lens"), (dict(lens=None), "penalties"), (dict(repetition=torch.ones(3)), "repetition"), (dict(bias=torch.zeros(6)), "bias"),
    (dict(bias=torch.zeros(5, dtype=torch.bfloat16)), "bias"), (dict(mask=torch.zeros(3, 1, dtype=torch.int32)), "mask"), (dict(mask_row=torch.zeros(2, dtype=torch.int32)), "mask_row"),
    (dict(mask=torch.zeros(2, 0, dtype=torch.int32)), "mask"), (dict(out=torch.zeros(2, 6)), "out"), (dict(), "GPU")])
def test_logits_refuses(kw, says):
    a = dict(logits=torch.zeros(2, 5), tokens=torch.zeros(2, 3, dtype=torch.int64), lens=torch.zeros(2, dtype=torch.int32), repetition=torch.ones(2))
    a.update(kw)
    with pytest.raises(AssertionError, match=says):
        ops.logits_process(a.pop("logits"), a.pop("tokens"), a.pop("lens"), **a)


def refused(rc, says):
    assert rc < 0
    assert says in _lib.lib().ralf_last_error().decode()


def test_c_entries_refuse():
    """the C entries check what they are given by themselves: every call below returns its error before a kernel could be launched"""
    L = _lib.lib()

    def rope(**kw):
        d = RalfRopeDesc(x=FAKE, y=FAKE, pos=FAKE, freq=FAKE, axis=FAKE, T=4, x_ts=64, x_hs=32, y_ts=64, y_hs=32, pos_as=4, H=2, D=32, R=32, A=2)
        for n, v in kw.items():
            setattr(d, n, v)
        return L.ralf_rope_axes(ctypes.byref(d), None)

    refused(L.ralf_rope_axes(None, None), "null")
    for kw, says in ((dict(x=None), "null"), (dict(axis=None), "null"), (dict(dtype=2), "dtype"), (dict(R=34), "rotated"), (dict(R=3), "rotated"), (dict(R=0), "rotated"), (dict(A=0), "sizes"),
                     (dict(T=-1), "sizes"), (dict(x_ts=-8), "stride"), (dict(y_ts=0), "overlap"), (dict(y_ts=128), "in place"), (dict(T=1 << 60, y=2 * FAKE), "too many")):
        refused(rope(**kw), says)
    assert rope(T=0, x=None) == 0

    def kv(**kw):
        d = RalfPagedKV(k=FAKE, v=FAKE, k_exp=FAKE, v_exp=FAKE, table=FAKE, kv_len=FAKE, n_pages=4, table_ld=2, page=16, heads=2, dim=32, store=1, B=2, max_pages=2)
        for n, v in kw.items():
            setattr(d, n, v)
        return d

    bad = [(dict(page=24), "page"), (dict(dim=48), "dim"), (dict(store=4), "store"), (dict(heads=0), "heads"), (dict(B=-1), "size"), (dict(table=None), "table"), (dict(table_ld=1), "table"),
           (dict(k=None), "cache"), (dict(v=FAKE + 8), "unaligned"), (dict(kv_len=None), "kv_len"), (dict(store=2, k_exp=None), "exponents"), (dict(n_pages=1 << 31), "pages"),
           (dict(max_pages=1 << 27, table_ld=1 << 27), "pages")]
    for kw, says in bad:
        d = kv(**kw)
        refused(L.ralf_paged_kv_write(ctypes.byref(d), 1, FAKE, FAKE, 64, 32, 64, 32, FAKE, 3, None), says)
        refused(L.ralf_paged_kv_read(ctypes.byref(d), 1, FAKE, FAKE, FAKE, 3, None), says)
        a = RalfPagedAttnDesc(kv=d, q=FAKE, o=FAKE, q_start=FAKE, T=3, q_ts=128, q_hs=32, o_ts=128, o_hs=32, q_heads=4, dtype=1, causal=1, scale=1.0)
        refused(L.ralf_paged_attention(ctypes.byref(a), None, 0, None), says)
        assert L.ralf_paged_attention_workspace_bytes(ctypes.byref(a)) == 0
    d = kv()
    refused(L.ralf_paged_kv_write(None, 1, FAKE, FAKE, 64, 32, 64, 32, FAKE, 3, None), "null")
    refused(L.ralf_paged_kv_write(ctypes.byref(d), 0, FAKE, FAKE, 64, 32, 64, 32, FAKE, 3, None), "own type")
    refused(L.ralf_paged_kv_write(ctypes.byref(d), 1, None, FAKE, 64, 32, 64, 32, FAKE, 3, None), "null")
    refused(L.ralf_paged_kv_write(ctypes.byref(d), 1, FAKE, FAKE, 60, 32, 64, 32, FAKE, 3, None), "multiples")
    refused(L.ralf_paged_kv_write(ctypes.byref(d), 1, FAKE + 2, FAKE, 64, 32, 64, 32, FAKE, 3, None), "multiples")
    refused(L.ralf_paged_kv_write(ctypes.byref(d), 1, FAKE, FAKE, 64, 32, -64, 32, FAKE, 3, None), "negative")
    refused(L.ralf_paged_kv_write(ctypes.byref(d), 2, FAKE, FAKE, 64, 32, 64, 32, FAKE, 3, None), "dtype")
    refused(L.ralf_paged_kv_write(ctypes.byref(d), 1, FAKE, FAKE, 64, 32, 64, 32, FAKE, -1, None), "rows")
    refused(L.ralf_paged_kv_read(ctypes.byref(d), 1, FAKE, None, FAKE, 3, None), "null")
    refused(L.ralf_paged_kv_read(ctypes.byref(d), 7, FAKE, FAKE, FAKE, 3, None), "dtype")
    assert L.ralf_paged_kv_write(ctypes.byref(d), 1, None, None, 64, 32, 64, 32, None, 0, None) == 0
    assert L.ralf_paged_kv_read(ctypes.byref(d), 1, None, None, None, 0, None) == 0

    def attn(ws=None, n=0, **kw):
        a = RalfPagedAttnDesc(kv=d, q=FAKE, o=FAKE, q_start=FAKE, T=3, q_ts=128, q_hs=32, o_ts=128, o_hs=32, q_heads=4, dtype=1, causal=1, scale=1.0)
        for name, v in kw.items():
            setattr(a, name, v)
        return L.ralf_paged_attention(ctypes.byref(a), ws, n, None)

    for kw, says in ((dict(q=None), "null"), (dict(q_start=None), "null"), (dict(q_heads=3), "heads"), (dict(q_heads=0), "heads"), (dict(dtype=0), "own type"), (dict(dtype=3), "dtype"),
                     (dict(window=-1), "negative"), (dict(T=-1), "rows"), (dict(T=1 << 31), "rows"), (dict(q_ts=100), "multiples"), (dict(o=FAKE + 8), "multiples")):
        refused(attn(**kw), says)
    refused(L.ralf_paged_attention(None, None, 0, None), "null")
    assert attn(T=0, q=None) == 0
    d = kv(max_pages=4096, table_ld=4096, n_pages=4096)          # a long axis and three rows: split, so a workspace is asked for
    a = RalfPagedAttnDesc(kv=d, T=3, q_heads=4, dtype=1)
    need = L.ralf_paged_attention_workspace_bytes(ctypes.byref(a))
    assert need > 0
    refused(attn(kv=d), "workspace")
    refused(attn(kv=d, ws=FAKE, n=need - 1), "workspace")

    def logits(**kw):
        g = RalfLogitsDesc(logits=FAKE, out=FAKE, tokens=FAKE, len=FAKE, repetition=FAKE, ld_in=8, ld_out=8, tok_ld=3, B=2, V=8, L=3)
        for n, v in kw.items():
            setattr(g, n, v)
        return L.ralf_logits_process(ctypes.byref(g), None)

    refused(L.ralf_logits_process(None, None), "null")
    for kw, says in ((dict(logits=None), "null"), (dict(ld_in=7), "shorter"), (dict(dtype=5), "dtype"), (dict(V=0), "sizes"), (dict(V=1 << 30), "sizes"), (dict(B=-1), "sizes"), (dict(len=None), "history"),
                     (dict(tok_ld=2), "history"), (dict(tokens=None), "history"), (dict(bias=FAKE, bias_ld=3), "bias"), (dict(mask=FAKE, mask_ld=0, mask_rows=2), "mask"),
                     (dict(mask=FAKE, mask_ld=1, mask_rows=1), "mask"), (dict(ld_out=9), "in place")):
        refused(logits(**kw), says)
    assert logits(B=0, logits=None) == 0
