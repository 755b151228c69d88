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


@pytest.mark.parametrize("store,dtype", [(F32, F32), (BF16, BF16), (E4M3, BF16), (I8, F32)])
@pytest.mark.parametrize("n,past", [(1, 300), (3, 300), (100, 600), (1, 5000)])
@pytest.mark.parametrize("kw", [{}, dict(causal=False)])
def test_infinities_that_every_row_sees(store, dtype, n, past, kw):
    """infinite values far behind the newest tokens: infinities of their sign for all rows, NaN where both signs meet (8-bit rows that hold one: NaN), and the other columns as they are"""
    from ralf_amd import ops

    L = past + n
    pool, table, q_start, kv_len = make([L], [L], 2, 64, 16, store, dtype, seed=3)
    k, v, q = rnd(L, 2, 64, seed=1, dtype=dtype), rnd(L, 2, 64, seed=2, dtype=dtype), rnd(n, 4, 64, seed=4, dtype=dtype)
    for t, c, x in ((5, 1, math.inf), (70, 2, -math.inf), (71, 3, math.inf), (150, 3, -math.inf), (200, 4, math.nan), (201, 63, math.inf)):
        v[t, 0, c] = x
    ops.paged_kv_write(pool, k.cuda(), v.cuda(), table.cuda(), q_start.cuda(), kv_len.cuda())
    start = torch.tensor([0, n], dtype=torch.int32)
    out = ops.paged_attention(q.cuda(), pool, table.cuda(), start.cuda(), kv_len.cuda(), **kw)
    want, e, _ = O.attention(q, *O.pool_values(pool), table, start, kv_len, 0.125, p_step=O.half_step(BF16) if dtype == BF16 else 0.0, **kw)
    if store.itemsize > 1:
        assert want[:, :2].isinf().sum() == n * 2 * 3 and want[:, :2].isnan().sum() == n * 2 * 2
    O.check(out, want, (e + O.half_step(dtype) * (want.abs() + e)).nan_to_num(), "infinities")


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


# ---------------------------------------------------------------------------------------------- the 8-bit stores: no value past fp32's
LARGEST_FINITE = {E4M3: (240.0, 120), I8: (63.0, 122)}      # the largest code at the exponent that fp32's largest numbers take: 256 and 64 would be 2^128


@pytest.mark.parametrize("store", [E4M3, I8])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_cache_holds_no_value_past_fp32(store, dtype):
    from ralf_amd import ops

    top = torch.finfo(dtype).max
    x = rnd(4, 2, 64, seed=1)
    x[0, 0, 3], x[0, 1, 0], x[1, 0, 5], x[1, 1, 7] = top, -top, 3.3e38, -3.37e38
    x[2, 0], x[3, 1, 0] = top, 1.2e38
    x = x.to(dtype)
    pool, table, q_start, kv_len = make([4], [4], 2, 64, 16, store, dtype, seed=2)
    ops.paged_kv_write(pool, x.cuda(), -x.cuda(), table.cuda(), q_start.cuda(), kv_len.cuda())
    code, e = LARGEST_FINITE[store]
    for sign, got, exp in ((1, pool.k, pool.k_exp), (-1, pool.v, pool.v_exp)):
        for t in range(4):
            c, byte = O.quantise(sign * x[t], store)
            c = torch.where((byte == 127 + e)[:, None], c.clamp(-code, code), c)       # (the nearest that fp32 holds)
            assert torch.equal(exp[int(table[0, 0]), :, t].cpu(), byte)
            assert torch.equal(got[int(table[0, 0]), :, t].float().cpu().double(), c)
    k, v = ops.paged_kv_read(pool, table.cuda(), kv_len.cuda(), q_start.cuda(), 4, dtype=F32)
    assert torch.isfinite(k).all() and torch.equal(v, -k)
    assert k[0, 0, 3].item() == code * 2.0 ** e


@pytest.mark.parametrize("store", [E4M3, I8])
@pytest.mark.parametrize("n,past", [(1, 40), (90, 40), (90, 400)])
@pytest.mark.parametrize("kw", [{}, dict(causal=False), dict(window=3)])
def test_attention_agrees_on_the_largest_held_values(store, n, past, kw):
    """one value of bf16's largest among small ones, seen by some rows or by all, on few and on many rows: the same finite value for both"""
    from ralf_amd import ops

    L = past + n
    pool, table, q_start, kv_len = make([L], [L], 1, 64, 16, store, BF16, seed=3)
    k, v, q = rnd(L, 1, 64, seed=1, dtype=BF16), rnd(L, 1, 64, seed=2, dtype=BF16), rnd(n, 2, 64, seed=4, dtype=BF16)
    for t in (10, L - 20):
        v[t, 0, 7] = torch.finfo(BF16).max
    ops.paged_kv_write(pool, k.cuda(), v.cuda(), table.cuda(), q_start.cuda(), kv_len.cuda())
    start = torch.tensor([0, n], dtype=torch.int32)
    many = ops.paged_attention(q.cuda(), pool, table.cuda(), start.cuda(), kv_len.cuda(), **kw)
    want, e, _ = O.attention(q, *O.pool_values(pool), table, start, kv_len, 0.125, p_step=O.half_step(BF16), **kw)
    assert torch.isfinite(want).all()
    O.check(many, want, e + O.half_step(BF16) * (want.abs() + e), "rows together")
    if kw.get("causal", True):
        for i in (0, n // 2, n - 1):                       # the same rows alone
            at = torch.tensor([L - n + i + 1], dtype=torch.int32)
            one = ops.paged_attention(q[i:i + 1].cuda(), pool, table.cuda(), torch.tensor([0, 1], dtype=torch.int32).cuda(), at.cuda(), **kw)
            O.check(one, want[i:i + 1], (e + O.half_step(BF16) * (want.abs() + e))[i:i + 1], "a row alone")


# ---------------------------------------------------------------------------------------------- rotary positions
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("P,D", [(8, 20), (16, 32), (11, 22)])
def test_pairs_of_foreign_axes_stay_as_they_are(dtype, adjacent, P, D):
    """a pair whose axis has no positions keeps its bits, infinities, NaN and negative zeros included, forwards and backwards, out of and in place"""
    from ralf_amd import functional, ops

    freq, axis = torch.full((P,), 0.7, dtype=torch.float64), torch.arange(P, dtype=torch.int32) % 2
    away = [0, 1, P // 2, P - 1]
    axis[away] = torch.tensor([-1, 2, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)
    x, pos = rnd(5, 3, D, seed=1), torch.randint(1, 99, (2, 5), generator=gen(2))
    first, second = ([2 * j for j in away], [2 * j + 1 for j in away]) if adjacent else (away, [j + P for j in away])
    odd = torch.tensor([math.inf, -math.inf, math.nan, -0.0, 3.0, -5.0])
    for n, (a, b) in enumerate(zip(first, second)):
        x[..., a], x[..., b] = odd[torch.arange(15) % 6].view(5, 3), odd[(torch.arange(15) // 6 + n + 1) % 6].view(5, 3)
    x = x.to(dtype).cuda()
    args = (pos.cuda(), freq.cuda(), axis.cuda())
    for inverse in (False, True):
        y = ops.rope_axes(x, *args, adjacent=adjacent, inverse=inverse)
        assert torch.equal(bits(y[..., first + second]), bits(x[..., first + second]))
        rest = [i for i in range(D) if i not in first + second]
        want, e = O.rope(x.cpu(), pos, freq, axis, adjacent, -1 if inverse else 1)
        O.check(y[..., rest], want[..., rest], (e + O.half_step(dtype) * (want.abs() + e))[..., rest], "the others")
        z = x.clone()
        ops.rope_axes(z, *args, adjacent=adjacent, inverse=inverse, out=z)
        assert torch.equal(bits(z), bits(y))
    leaf = torch.zeros_like(x, requires_grad=True)
    g, = torch.autograd.grad(functional.rope_axes(leaf, *args, adjacent), leaf, x)
    assert torch.equal(bits(g[..., first + second]), bits(x[..., first + second]))


# ---------------------------------------------------------------------------------------------- attention: a scale of zero
@pytest.mark.parametrize("store,dtype", [(F32, F32), (BF16, BF16), (I8, BF16)])
@pytest.mark.parametrize("n", [1, 100])
def test_scale_of_zero_keeps_what_is_not_finite(store, dtype, n):
    """0 * inf is NaN, whichever number of rows; finite rows are the mean of what they see"""
    from ralf_amd import ops

    pool, table, q_start, kv_len = make([n + 30], [n], 1, 64, 16, store, dtype, seed=3)
    q, k, v = rnd(n, 2, 64, seed=4, dtype=dtype), rnd(n, 1, 64, seed=5, dtype=dtype), rnd(n, 1, 64, seed=6, dtype=dtype)
    q[n // 2, 0, 3], q[n // 2, 1, 5] = math.nan, math.inf
    ops.paged_kv_write(pool, k.cuda(), v.cuda(), table.cuda(), q_start.cuda(), kv_len.cuda())
    out = ops.paged_attention(q.cuda(), pool, table.cuda(), q_start.cuda(), kv_len.cuda(), scale=0.0)
    want, e, _ = O.attention(q, *O.pool_values(pool), table, q_start, kv_len, 0.0, p_step=O.half_step(dtype) if dtype == BF16 else 0.0)
    assert want[n // 2].isnan().all()
    O.check(out, want, e.nan_to_num() + O.half_step(dtype) * (want.abs() + e).nan_to_num(), "scale 0")


# ---------------------------------------------------------------------------------------------- outputs given by strides
def test_outputs_whose_rows_overlap_are_refused():
    from ralf_amd import _lib, ops

    pool, table, q_start, kv_len = make([20, 30], [3, 2], 2, 64, 16, BF16, BF16, seed=2)
    q = rnd(5, 4, 64, seed=3, dtype=BF16).cuda()
    args = (pool, table.cuda(), q_start.cuda(), kv_len.cuda())
    freq, axis = ops.rope_table((32,), device="cuda")
    pos = torch.arange(5).view(1, 5).cuda()
    flat = torch.full((5 * 4 * 64,), 7.0, dtype=BF16, device="cuda")
    for out in (flat[:256].view(1, 4, 64).expand(5, 4, 64), flat[:320].view(5, 1, 64).expand(5, 4, 64), flat.as_strided((5, 4, 64), (192, 64, 1))):
        with pytest.raises(_lib.RalfHipError, match="overlap"):
            ops.paged_attention(q, *args, out=out)
        with pytest.raises(_lib.RalfHipError, match="overlap"):
            ops.rope_axes(q, pos, freq, axis, out=out)
    assert bool((flat == 7.0).all())


def test_outputs_in_other_orders():
    """heads outermost, every second head or token of a wider tensor: the same bits"""
    from ralf_amd import ops

    pool, table, q_start, kv_len = make([90, 300, 40], [3, 100, 1], 2, 64, 16, BF16, BF16, seed=2)
    T = int(q_start[-1])
    q = rnd(T, 4, 64, seed=3, dtype=BF16).cuda()
    args = (pool, table.cuda(), q_start.cuda(), kv_len.cuda())
    freq, axis = ops.rope_table((32,), device="cuda")
    pos = torch.arange(T).view(1, T).cuda()
    for run in (lambda x, **kw: ops.paged_attention(x, *args, **kw), lambda x, **kw: ops.rope_axes(x, pos, freq, axis, **kw)):
        want = run(q)
        for wide, view in ((torch.full((4, T, 64), 7.0), lambda t: t.transpose(0, 1)), (torch.full((T, 8, 64), 7.0), lambda t: t[:, 1::2]), (torch.full((2 * T, 4, 64), 7.0), lambda t: t[::2])):
            wide = wide.to(BF16).cuda()
            run(q, out=view(wide))
            assert torch.equal(bits(view(wide)), bits(want))
            assert bool((wide == 7.0).any()) == (wide.numel() > want.numel())


def test_outputs_beside_and_in_place_of_their_inputs():
    """an output among the heads that its input leaves free in one buffer, or the input itself: the same bits, and the input or what lies around it unharmed"""
    from ralf_amd import ops

    pool, table, q_start, kv_len = make([90, 300, 40, 9000], [3, 100, 1, 1], 2, 64, 16, BF16, BF16, seed=2)
    T = int(q_start[-1])
    q = rnd(T, 4, 64, seed=3, dtype=BF16).cuda()
    args = (pool, table.cuda(), q_start.cuda(), kv_len.cuda())
    freq, axis = ops.rope_table((32,), device="cuda")
    pos = torch.arange(T).view(1, T).cuda()
    for run in (lambda x, **kw: ops.paged_attention(x, *args, **kw), lambda x, **kw: ops.rope_axes(x, pos, freq, axis, **kw)):
        want = run(q)
        for src, dst in ((slice(0, 4), slice(4, 8)), (slice(5, 9), slice(1, 5)), (slice(0, 8, 2), slice(1, 9, 2))):
            wide = torch.full((T, 9, 64), 7.0, dtype=BF16, device="cuda")
            wide[:, src] = q
            run(wide[:, src], out=wide[:, dst])
            assert torch.equal(bits(wide[:, dst]), bits(want)) and torch.equal(bits(wide[:, src]), bits(q))
        wide = torch.full((T, 6, 64), 7.0, dtype=BF16, device="cuda")
        wide[:, 1:5] = q
        run(wide[:, 1:5], out=wide[:, 1:5])
        assert torch.equal(bits(wide[:, 1:5]), bits(want)) and bool((wide[:, ::5] == 7.0).all())
        outer = torch.cat([q.transpose(0, 1), torch.full((4, T, 64), 7.0, dtype=BF16, device="cuda")])          # heads outermost
        run(outer[:4].transpose(0, 1), out=outer[4:].transpose(0, 1))
        assert torch.equal(bits(outer[4:].transpose(0, 1)), bits(want))
    x = rnd(6, 1000, seed=1).cuda()
    bias = rnd(1000, seed=2).cuda()
    both = torch.cat([x, torch.zeros_like(x)], 1)
    ops.logits_process(both[:, :1000], bias=bias, out=both[:, 1000:])
    assert torch.equal(both[:, 1000:], x + bias) and torch.equal(both[:, :1000], x)


# ---------------------------------------------------------------------------------------------- attention: chunks beside single tokens, both with their keys cut
@pytest.mark.parametrize("lens,new,Hq,heads,dim,kw", [
    ([5000, 9000], [100, 1], 2, 1, 64, dict(max_q=100, max_kv=9000)), ([9000, 300, 5000, 0, 40], [1, 200, 16, 0, 3], 4, 2, 64, {}), ([6000, 6000, 6000], [33, 16, 17], 4, 1, 128, dict(max_q=33, max_kv=6000)),
    ([3000, 4000], [70, 1], 4, 2, 256, dict(window=900)), ([3000, 5000, 2000], [70, 2, 65], 2, 2, 32, dict(causal=False)), ([2500, 2600], [150, 120], 2, 1, 64, dict(max_q=150, max_kv=2600)),
    ([2500, 2600], [150, 1], 2, 1, 64, dict(max_q=76, max_kv=2600)), ([3000] * 12, [70] + [1] * 11, 4, 2, 64, dict(max_q=70, max_kv=3000)), ([2000, 3000, 2500], [67, 1, 1], 1, 1, 32, {})])
@pytest.mark.parametrize("store", [BF16, E4M3, I8])
def test_mixed_batches_with_cut_keys(lens, new, Hq, heads, dim, kw, store):
    """rows of both kernels, each with splits of its own (their partial sums by token, or by sequence where that takes less); two rows behind the last sequence stay; in place of the queries the same bits"""
    from ralf_amd import ops

    pool, table, q_start, kv_len = make(lens, new, heads, dim, 64, store, BF16, seed=len(lens))
    T = int(q_start[-1])
    q, k, v = (rnd(T + 2, h, dim, seed=i, dtype=BF16) for i, h in ((1, Hq), (2, heads), (3, heads)))
    args = (pool, table.cuda(), q_start.cuda(), kv_len.cuda())
    ops.paged_kv_write(pool, k.cuda(), v.cuda(), *args[1:])
    out = torch.full_like(q, 3.0).cuda()
    ops.paged_attention(q.cuda(), *args, out=out, **kw)
    assert bool((out[T:] == 3.0).all())
    want, e, _ = O.attention(q[:T], *O.pool_values(pool), table, q_start, kv_len, dim ** -0.5, p_step=O.half_step(BF16), causal=kw.get("causal", True), window=kw.get("window", 0))
    O.check(out[:T], want, e + O.half_step(BF16) * (want.abs() + e) + 1e-37, "mixed")
    same = q.cuda()
    ops.paged_attention(same, *args, out=same, **kw)
    assert torch.equal(bits(same[:T]), bits(out[:T])) and torch.equal(bits(same[T:]), bits(q[T:]))


@pytest.mark.parametrize("q_starts", [([0, 100, 101, 101], [0, 3, 60, 101], [0, 0, 1, 101], [0, 33, 66, 99]), ([0, 1, 101, 101], [0, 50, 101, 101], [0, 101, 101, 101])])
def test_captured_mixed_call_follows_its_starts(q_starts):
    """a call of both kernels in a graph: replayed with other starts, sequences change sides and every replay has the eager call's bits; eager calls of the same kind in between"""
    from ralf_amd import ops

    lens, heads, dim = [3000, 5000, 2500], 2, 64
    pool, table, _, kv_len = make(lens, lens, heads, dim, 64, BF16, BF16, seed=9, garbage=False)
    k, v = (rnd(sum(lens), heads, dim, seed=i, dtype=BF16).cuda() for i in (1, 2))
    table, kv_len = table.cuda(), kv_len.cuda()
    ops.paged_kv_write(pool, k, v, table, torch.tensor([0] + lens).cumsum(0).int().cuda(), kv_len)
    q, start = rnd(101, 4, dim, seed=3, dtype=BF16).cuda(), torch.tensor(q_starts[0], dtype=torch.int32).cuda()
    call = lambda: ops.paged_attention(q, pool, table, start, kv_len, max_q=100, max_kv=5000)    # noqa: E731
    st = ops.own_stream("serving_edges_test")
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        out = call()
    for turn in range(2):
        for s in q_starts:
            start.copy_(torch.tensor(s, dtype=torch.int32))
            n = s[-1]
            want = call()[:n].clone()
            out.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(bits(out[:n]), bits(want)) and not out[n:].any()
            ref, e, _ = O.attention(q[:n].cpu(), *O.pool_values(pool), table.cpu(), s, kv_len.cpu(), dim ** -0.5, p_step=O.half_step(BF16))
            O.check(want, ref, e + O.half_step(BF16) * (ref.abs() + e) + 1e-37, "mixed")


# ---------------------------------------------------------------------------------------------- a packed projection
@pytest.mark.parametrize("store", [BF16, E4M3])
def test_decode_on_a_packed_projection(store):
    """query and key heads rotated where they lie in the projection, keys and values stored and queries taken as slices of it: the bits of separate tensors"""
    from ralf_amd import ops

    Hq, Hk, D = 8, 2, 64
    lens, new = [40, 7, 300], [1, 7, 100]
    T = sum(new)
    qkv = rnd(T, Hq + 2 * Hk, D, seed=1, dtype=BF16).cuda()
    freq, axis = ops.rope_table((8, 24), device="cuda")
    pos = torch.randint(0, 400, (2, T), generator=gen(2)).cuda()
    outs = []
    for packed in (True, False):
        pool, table, q_start, kv_len = make(lens, new, Hk, D, 16, store, BF16, seed=4)
        args = (table.cuda(), q_start.cuda(), kv_len.cuda())
        if packed:
            x = qkv.clone()
            ops.rope_axes(x[:, :Hq + Hk], pos, freq, axis, out=x[:, :Hq + Hk])
            q, k, v = x[:, :Hq], x[:, Hq:Hq + Hk], x[:, Hq + Hk:]
            assert torch.equal(v, qkv[:, Hq + Hk:])
        else:
            q, k, v = (t.contiguous() for t in (qkv[:, :Hq], qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:]))
            q, k = ops.rope_axes(q, pos, freq, axis), ops.rope_axes(k, pos, freq, axis)
        ops.paged_kv_write(pool, k, v, *args)
        outs.append(ops.paged_attention(q, pool, *args, max_q=100, max_kv=300))
    assert torch.equal(bits(outs[0]), bits(outs[1]))
