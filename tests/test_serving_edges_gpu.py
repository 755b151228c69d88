"""Serving operators on the GPU at the edges of their definitions, against the 64-bit oracle (tests/serving_oracle.py)."""
import math

import pytest
import torch

import serving_oracle as O
from test_serving_gpu import BF16, E4M3, F32, I8, bits, gen, make, rnd

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------- attention: the weights' precision
@pytest.mark.parametrize("lens,new,Hq,heads,dim,kw", [
    ([37, 1, 70, 16, 2], [5, 1, 13, 16, 2], 4, 2, 64, {}), ([51], [1], 8, 8, 32, {}), ([300, 517], [1, 1], 8, 2, 128, {}), ([9000], [1], 4, 1, 128, dict(max_q=1, max_kv=9000)), ([130, 65], [8, 1], 2, 1, 256, {}),
    ([200, 90], [7, 3], 4, 2, 64, dict(window=13)), ([200, 90], [7, 3], 4, 2, 64, dict(causal=False))])
@pytest.mark.parametrize("store", [BF16, E4M3, I8])
def test_few_rows_round_only_their_result(lens, new, Hq, heads, dim, kw, store):
    """bf16 queries, few rows: the weights count with two bf16 parts (off by 2^-8 of 2^-8), so that what is left is the result's own rounding"""
    from ralf_amd import ops

    pool, table, q_start, kv_len = make(lens, new, heads, dim, 16, store, BF16, seed=dim + len(lens))
    T = int(q_start[-1])
    q, k, v = (rnd(T, h, dim, seed=i, dtype=BF16) for i, h in ((1, Hq), (2, heads), (3, heads)))
    args = (pool, table.cuda(), q_start.cuda(), kv_len.cuda())
    ops.paged_kv_write(pool, k.cuda(), v.cuda(), *args[1:])
    out = ops.paged_attention(q.cuda(), *args, **kw)
    want, e, _ = O.attention(q, *O.pool_values(pool), table, q_start, kv_len, dim ** -0.5, p_step=O.half_step(BF16) ** 2, causal=kw.get("causal", True), window=kw.get("window", 0))
    O.check(out, want, e + O.half_step(BF16) * (want.abs() + e) + 1e-37, "two parts")


# ---------------------------------------------------------------------------------------------- attention: values near fp32's end
@pytest.mark.parametrize("store,dtype", [(F32, F32), (BF16, BF16), (E4M3, BF16), (E4M3, F32), (I8, BF16), (I8, F32)])
@pytest.mark.parametrize("n,past", [(1, 60), (100, 60), (300, 300), (1, 5000), (100, 5000)])
@pytest.mark.parametrize("rising", [False, True])
def test_attention_large_values_stay_finite(store, dtype, n, past, rising):
    """Finite values whose weighted sum is finite give it.  rising: scores that grow along the keys by 6 nats, so that the softmax's reference has to follow them; values of 2^120 times up
    to 2 (their sum over the 5100 keys at most would pass 2^128 for weights of 1: all but 100 keys have a score of 20 less)."""
    from ralf_amd import ops

    L, heads, dim = past + n, 1, 64
    pool, table, q_start, kv_len = make([L], [L], heads, dim, 16, store, dtype, seed=5)
    q, k = torch.zeros(L, 2, dim), torch.zeros(L, heads, dim)
    q[:, :, 0] = 8.0                                       # times 64 ** -0.5: scores are k's first element
    near = torch.arange(L) % max(1, L // 50) == 0
    k[:, 0, 0] = torch.where(near, 6.0 * torch.arange(L) / L if rising else torch.zeros(L), -20.0)
    v = 2.0 ** 120 * (1 + torch.rand(L, heads, dim, generator=gen(n)))
    q, k, v = (t.to(dtype) for t in (q, k, v))
    ops.paged_kv_write(pool, k.cuda(), v.cuda(), table.cuda(), q_start.cuda(), kv_len.cuda())
    start = torch.tensor([0, n], dtype=torch.int32)
    out = ops.paged_attention(q[-n:].cuda(), pool, table.cuda(), start.cuda(), kv_len.cuda(), max_q=n, max_kv=L)
    want, e, _ = O.attention(q[-n:], *O.pool_values(pool), table, start, kv_len, dim ** -0.5, p_step=O.half_step(BF16) if dtype == BF16 else 0.0)
    assert torch.isfinite(want).all() and torch.isfinite(out).all()
    O.check(out, want, e + O.half_step(dtype) * (want.abs() + e), "large values")


@pytest.mark.parametrize("store,dtype", [(F32, F32), (BF16, BF16), (E4M3, BF16), (E4M3, F32), (I8, BF16), (I8, F32)])
@pytest.mark.parametrize("n", [1, 100])
def test_attention_mean_of_large_values(store, dtype, n):
    """the mean of up to 200 values of 2^127 is one of them, whatever their sum is"""
    from ralf_amd import ops

    pool, table, q_start, kv_len = make([200], [200], 1, 64, 16, store, dtype, seed=5)
    v = torch.full((200, 1, 64), 2.0 ** 127, dtype=dtype)
    ops.paged_kv_write(pool, torch.zeros_like(v).cuda(), v.cuda(), table.cuda(), q_start.cuda(), kv_len.cuda())
    out = ops.paged_attention(rnd(n, 2, 64, seed=1, dtype=dtype).cuda(), pool, table.cuda(), torch.tensor([0, n], dtype=torch.int32).cuda(), kv_len.cuda())
    # equal weights, their sum and the value's sum off by a step of fp32 a key at most; the division by two
    assert ((out.double() / 2.0 ** 127 - 1).abs() <= (2 * 200 + 2) * O.U32 + O.half_step(dtype)).all()
