"""Serving operators without a GPU: calls that the C entries refuse before anything is launched, and what they plan."""
import ctypes

import pytest

from ralf_amd import _lib
from ralf_amd._abi import RalfLogitsDesc, RalfPagedAttnDesc, RalfPagedKV, RalfRopeDesc

FAKE = 1 << 20      # an aligned address that nothing may follow


def refused(rc, says):
    assert rc < 0
    assert says in _lib.lib().ralf_last_error().decode()


def paged(**kw):
    d = RalfPagedKV(k=FAKE, v=FAKE, k_exp=FAKE, v_exp=FAKE, table=FAKE, kv_len=FAKE, n_pages=4, table_ld=2, page=16, heads=2, dim=32, store=1, B=2, max_pages=2)
    for n, v in kw.items():
        setattr(d, n, v)
    return d


def attention(**kw):
    d = RalfPagedAttnDesc(kv=paged(), q=FAKE, o=2 * FAKE, q_start=FAKE, T=3, q_ts=128, q_hs=32, o_ts=128, o_hs=32, q_heads=4, dtype=1, causal=1, scale=1.0)
    for n, v in kw.items():
        setattr(d, n, v)
    return d


def rope(**kw):
    d = RalfRopeDesc(x=FAKE, y=2 * FAKE, pos=FAKE, freq=FAKE, axis=FAKE, T=4, x_ts=64, x_hs=32, y_ts=64, y_hs=32, pos_as=4, H=2, D=32, R=32, A=2)
    for n, v in kw.items():
        setattr(d, n, v)
    return d


# (strides of [T, heads, 32]: expanded over tokens, over heads; rows that begin within others)
OVERLAPPING = [(0, 32), (128, 0), (0, 0), (64, 32), (128, 24), (120, 32), (32, 64), (8, 8)]


@pytest.mark.parametrize("ts,hs", OVERLAPPING)
def test_outputs_whose_rows_overlap(ts, hs):
    """two rows of the output in one place: refused (a workgroup each would write it)"""
    L = _lib.lib()
    refused(L.ralf_paged_attention(ctypes.byref(attention(o_ts=ts, o_hs=hs)), None, 0, None), "overlap")
    refused(L.ralf_rope_axes(ctypes.byref(rope(H=4, x_ts=128, y_ts=ts, y_hs=hs)), None), "overlap")


@pytest.mark.parametrize("size,dtype", [(4, 0), (2, 1)])
def test_outputs_that_overlap_their_inputs(size, dtype):
    """an output that lies across its input without being it: refused (some workgroup would read what another has written)"""
    L = _lib.lib()
    # x [4, 4, 32] with steps 128, 32: shifted by elements, by a head, by a token, back by a token, by half a byte's element; then with other steps
    for off, ts, hs in ((size, 128, 32), (32 * size, 128, 32), (128 * size, 128, 32), (-128 * size, 128, 32), (511 * size, 128, 32), (1, 256, 64), (0, 256, 32), (64 * size, 32, 128)):
        refused(L.ralf_rope_axes(ctypes.byref(rope(H=4, x_ts=128, y=FAKE + off, y_ts=ts, y_hs=hs, dtype=dtype)), None), "in place" if off == 0 else "overlap")
    # queries in a wider projection, the output over its neighbouring heads
    for off in (-32 * size, 32 * size, 96 * size, 224 * size):
        refused(L.ralf_paged_attention(ctypes.byref(attention(kv=paged(store=dtype), q_ts=256, o=FAKE + off, o_ts=256, dtype=dtype)), None, 0, None), "overlap")
    refused(L.ralf_paged_attention(ctypes.byref(attention(kv=paged(store=dtype), q_ts=256, o=FAKE, o_ts=128, dtype=dtype)), None, 0, None), "overlap")
    for off, ld in ((size, 8), (-8 * size, 8), (15 * size, 8), (4 * size, 16)):
        refused(L.ralf_logits_process(ctypes.byref(RalfLogitsDesc(logits=FAKE, out=FAKE + off, ld_in=8 if ld == 8 else 16, ld_out=ld, B=2, V=8, dtype=dtype)), None), "overlap")


@pytest.mark.parametrize("dtype,T,max_q", [(0, 3, 0), (1, 3, 0), (1, 3000, 0), (1, 3000, 1)])
def test_the_widest_windows_plan_like_none(dtype, T, max_q):
    """windows up to 2^31 - 1, to which larger ones are cut: the split of the keys (seen in the workspace) is the one without a window"""
    need = lambda w: _lib.lib().ralf_paged_attention_workspace_bytes(ctypes.byref(attention(kv=paged(store=dtype, B=2, max_pages=4096, table_ld=4096, n_pages=4096), dtype=dtype, T=T, max_q=max_q, window=w)))    # noqa: E731
    assert need(0) > 0
    for w in (2 ** 31 - 1, 2 ** 31 - 256, 2 ** 31 - 257, 65536):
        assert need(w) == need(0)
    assert need(1) < need(0)


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 3.4e38])
def test_scales_that_are_not_finite(scale):
    """refused, as is one that is not finite once log2(e) is in it (empty rows would be NaN on many rows and zeros on few)"""
    L = _lib.lib()
    for kw in (dict(scale=scale), dict(scale=-scale), dict(scale=scale, T=0)):
        refused(L.ralf_paged_attention(ctypes.byref(attention(**kw)), None, 0, None), "scale")
    assert L.ralf_paged_attention_workspace_bytes(ctypes.byref(attention(kv=paged(max_pages=4096, table_ld=4096, n_pages=4096), scale=scale))) == 0


@pytest.mark.parametrize("T", [1 << 61, 1 << 62, (1 << 62) + 1, (1 << 63) - 1])
def test_row_counts_whose_products_wrap(T):
    """counts that pass 2^63 once multiplied are refused like other large ones"""
    L = _lib.lib()
    refused(L.ralf_rope_axes(ctypes.byref(rope(T=T)), None), "too many")
    refused(L.ralf_paged_attention(ctypes.byref(attention(T=T)), None, 0, None), "rows")
    assert L.ralf_paged_attention_workspace_bytes(ctypes.byref(attention(T=T))) == 0
    refused(L.ralf_rope_axes(ctypes.byref(rope(D=(1 << 31) - 1, R=2, T=1)), None), "sizes")


def test_single_tokens_beside_a_chunk_keep_their_splits():
    """one token on 131 072 keys has them cut into as many pieces beside a chunk of 2048 as alone (the workspace holds the pieces of up to 64 rows of every sequence and key head)"""
    L = _lib.lib()

    def need(T, B, max_q, max_kv=131072):
        c = paged(B=B, heads=8, dim=128, page=64, max_pages=2048, table_ld=2048, n_pages=4096)
        return L.ralf_paged_attention_workspace_bytes(ctypes.byref(attention(kv=c, q_heads=32, T=T, max_q=max_q, max_kv=max_kv)))

    alone = need(1, 1, 1) // (1 * 32 * (128 + 2) * 4)
    assert alone > 8
    beside = need(2049, 2, 2048)
    assert beside % (2 * 64 * 8 * (128 + 2) * 4) == 0 and alone // 2 <= beside // (2 * 64 * 8 * (128 + 2) * 4) <= alone
    c = lambda T: need(T, 40, 100, 8192)    # noqa: E731
    assert c(139) % (139 * 32 * (128 + 2) * 4) == 0 and 0 < c(139) <= 16 * 139 * 32 * (128 + 2) * 4        # by token where those are fewer
    assert need(2049, 2, 2 ** 31 - 1) == beside
    assert need(4096, 2, 2048) == 0             # two chunks of 2048: no short sequence
    assert need(2049, 2, 2048, 512) == 0        # short axes stay whole
