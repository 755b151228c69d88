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
