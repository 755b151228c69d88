"""Serving operators on the GPU against their definitions in 64 bits (tests/serving_oracle.py), with the bounds that their roundings allow."""
import math

import pytest
import torch

import serving_oracle as O

pytestmark = pytest.mark.gpu
F32, BF16, E4M3, I8 = torch.float32, torch.bfloat16, torch.float8_e4m3fn, torch.int8


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rnd(*shape, seed=0, dtype=F32):
    return torch.randn(*shape, generator=gen(seed)).to(dtype)


def bits(t):
    return t.cpu().view(torch.uint8) if t.dtype.itemsize == 1 else t.cpu().contiguous().view(torch.int16 if t.dtype.itemsize == 2 else torch.int32)


# ---------------------------------------------------------------------------------------------- rotary positions
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,H,D,sections,adjacent,far", [
    (1, 1, 2, (1,), False, 3), (1, 16, 32, (16,), False, 50), (5, 3, 80, (16, 16), True, 1000), (33, 2, 128, (16, 24, 24), False, 2 ** 31 - 40), (33, 2, 128, (16, 24, 24), True, 2 ** 20),
    (7, 5, 66, (33,), False, 7), (7, 5, 66, (30, 3), True, 7), (700, 1, 64, (3, 5, 4, 20), False, 100), (9, 40, 256, (64, 64), False, -2 ** 31 + 40), (257, 3, 98, (33,), False, 11), (6, 2, 71, (33,), True, 3), (6, 2, 135, (64,), False, 3)])
def test_rope(dtype, T, H, D, sections, adjacent, far):
    from ralf_amd import ops

    x = rnd(T, H, D, seed=T + D, dtype=dtype)
    pos = far + torch.randint(-20, 21, (len(sections), T), generator=gen(T))
    freq, axis = ops.rope_table(sections, theta=10000.0, order="round" if adjacent else "blocks")
    args = (pos.cuda(), freq.cuda(), axis.cuda())
    # freq * position is exact to 2^-53 relative on both sides: at 2^31 radians 5e-7 of angle, counted into the bound
    lost = abs(far) * 2.0 ** -52
    for inverse in (False, True):
        y = ops.rope_axes(x.cuda(), *args, adjacent=adjacent, inverse=inverse)
        assert y.dtype == dtype and y.is_contiguous()
        want, e = O.rope(x, pos, freq, axis, adjacent, -1 if inverse else 1)
        O.check(y, want, e + lost * 2 * x.double().abs().amax() + O.half_step(dtype) * (want.abs() + e), "rope")
        xi = x.cuda()
        assert ops.rope_axes(xi, *args, adjacent=adjacent, inverse=inverse, out=xi) is xi        # in place: the same bits
        assert torch.equal(bits(xi), bits(y))
        packed = torch.zeros(T, H + 3, D + 8, dtype=dtype, device="cuda")                             # heads 1 .. H of a wider projection, into one of another width
        packed[:, 1:H + 1, :D] = x.cuda()
        out = torch.full((T, 2 * H, D), 7.0, dtype=dtype, device="cuda")
        ops.rope_axes(packed[:, 1:H + 1, :D], *args, adjacent=adjacent, inverse=inverse, out=out[:, ::2])
        assert torch.equal(bits(out[:, ::2]), bits(y)) and bool((out[:, 1::2] == 7).all())


def test_rope_foreign_axis_and_empty():
    from ralf_amd import ops

    freq, axis = ops.rope_table((4, 4), device="cuda")
    axis[1], axis[6] = -1, 2                                       # pairs whose axis has no positions stay
    x, pos = rnd(6, 2, 20, seed=1), torch.randint(0, 99, (2, 6), generator=gen(2))
    y = ops.rope_axes(x.cuda(), pos.cuda(), freq, axis)
    want, e = O.rope(x, pos, freq.cpu(), axis.cpu(), False)
    O.check(y, want, e + O.U32 * want.abs(), "rope")
    for j in (1, 6):
        assert torch.equal(y[..., [j, j + 8]].cpu(), x[..., [j, j + 8]])
    assert ops.rope_axes(x[:0].cuda(), pos[:, :0].cuda(), freq, axis).shape == (0, 2, 20)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("adjacent", [False, True])
def test_rope_gradient(dtype, adjacent):
    from ralf_amd import functional, ops

    T, H, D = 19, 3, 48
    freq, axis = ops.rope_table((8, 12), device="cuda")
    pos = torch.randint(0, 5000, (2, T), generator=gen(1)).cuda()
    x = rnd(T, H, D, seed=3, dtype=dtype).cuda().requires_grad_(True)
    dy = rnd(T, H, D, seed=4, dtype=dtype).cuda()
    y = functional.rope_axes(x, pos, freq, axis, adjacent)
    y.backward(dy.transpose(0, 1).contiguous().transpose(0, 1))   # a gradient that is not contiguous
    want, e = O.rope(dy.cpu(), pos.cpu(), freq.cpu(), axis.cpu(), adjacent, -1)
    O.check(x.grad, want, e + O.half_step(dtype) * (want.abs() + e), "gradient")
    if dtype == F32:        # against differences: the map is linear, so a difference of any length is the derivative; sums of T H D products in 64 bits
        step = rnd(T, H, D, seed=5).cuda()
        diff = (functional.rope_axes((x + step).detach(), pos, freq, axis, adjacent).double() - y.detach().double())
        real = (x + step).detach().double() - x.detach().double()
        a, b = (diff * dy.double()).sum(), (real * x.grad.double()).sum()
        bound = 4 * (dy.double().abs() * (2 * x.detach().double().abs() + 2 * step.double().abs())).sum() * (2 * math.pi * 2.0 ** -26 + 2 * 2.0 ** -23 + 4 * O.U32)
        assert (a - b).abs() <= bound
        g, = torch.autograd.grad(functional.rope_axes(x, pos, freq, axis, adjacent)[:, :1].expand(-1, H, -1), x, dy)     # one head's output used by all: the heads' gradients add up before
        want, e = O.rope(dy.cpu().double().sum(1, keepdim=True), pos.cpu(), freq.cpu(), axis.cpu(), adjacent, -1)
        O.check(g[:, :1], want, e + 4 * O.U32 * dy.cpu().double().abs().sum(1, keepdim=True) * 2, "shared head")
        assert not g[:, 1:].any()


def test_rope_gradient_of_the_gradient():
    from ralf_amd import functional

    freq, axis = torch.full((4,), 0.3, dtype=torch.float64).cuda(), torch.zeros(4, dtype=torch.int32).cuda()
    pos = torch.arange(5).view(1, 5).cuda()
    x, dy = rnd(5, 2, 8, seed=1).cuda().requires_grad_(True), rnd(5, 2, 8, seed=2).cuda().requires_grad_(True)
    g, = torch.autograd.grad(functional.rope_axes(x, pos, freq, axis), x, dy, create_graph=True)
    gg, = torch.autograd.grad(g, dy, rnd(5, 2, 8, seed=3).cuda())
    want, e = O.rope(rnd(5, 2, 8, seed=3), pos.cpu(), freq.cpu(), axis.cpu(), False)
    O.check(gg, want, e + O.U32 * want.abs(), "second gradient")


# ---------------------------------------------------------------------------------------------- the cache
def make(lens, new, heads, dim, page, store, dtype, seed, spare=2, garbage=True):
    """a pool whose unwritten cells hold what must not be looked at, page tables in random order, sequences filled with values"""
    from ralf_amd import ops

    need = [-(-t // page) for t in lens]
    n = sum(need) + spare
    pool = ops.paged_kv_pool(n, page, heads, dim, store)
    if garbage:
        for p in (pool.k, pool.v):
            p.view(torch.uint8).fill_(0xFF)             # NaN in fp32, bf16 and e4m3
        if pool.k_exp is not None:
            pool.k_exp.fill_(255), pool.v_exp.fill_(255)
    order = torch.randperm(n, generator=gen(seed)).int()
    table = torch.full((len(lens), max(need + [0]) + 1), -1, dtype=torch.int32)
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = order[at:at + m]
        at += m
    old = [max(0, t - m) for t, m in zip(lens, new)]
    k, v = (rnd(sum(old), heads, dim, seed=seed + i, dtype=dtype).cuda() for i in (1, 2))
    starts = torch.tensor([0] + old).cumsum(0).int().cuda()
    ops.paged_kv_write(pool, k, v, table.cuda(), starts, torch.tensor(old).int().cuda())
    q_start = torch.tensor([0] + new).cumsum(0).int()
    return pool, table, q_start, torch.tensor(lens).int()


def cells(table, b, p, page):
    return int(table[b, p // page]), p % page


@pytest.mark.parametrize("store,dtype", [(F32, F32), (BF16, BF16), (E4M3, F32), (E4M3, BF16), (I8, F32), (I8, BF16)])
@pytest.mark.parametrize("heads,dim,page", [(1, 32, 16), (3, 64, 32), (2, 128, 256), (5, 256, 16), (8, 128, 64)])
def test_cache_write_read(store, dtype, heads, dim, page):
    from ralf_amd import ops

    lens, new = [1, page, 0, 2 * page + 3, 7, page - 1], [1, 3, 0, page + 5, 7, 0]
    pool, table, q_start, kv_len = make(lens, new, heads, dim, page, store, dtype, seed=heads)
    T = int(q_start[-1])
    rows = rnd(T + 2, 2 * heads + 1, dim, seed=9, dtype=dtype)                # slices of a projection, two rows behind the last sequence
    x = rows.clone()
    x[0, 0], x[1, 1, :] = 0.0, x[1, 1, :] * 1e-30
    x[2, 0, 3], x[3, heads, 5], x[4, 0, 0] = math.nan, math.inf, 3e38
    x[5] = torch.where(x[5] > 0, 1.0, -1.0) * torch.tensor(448.0 if store == E4M3 else 127.0)     # exactly the largest code
    x[6, :, 0] = 0.5 * 448.0
    x = x.to(dtype).cuda()
    k, v = x[:, :heads], x[:, heads:2 * heads]
    before = [bits(p) for p in pool if p is not None]
    ops.paged_kv_write(pool, k, v, table.cuda(), q_start.cuda(), kv_len.cuda())
    after = [bits(p) for p in pool if p is not None]
    touched = torch.zeros(pool.k.shape[:3], dtype=torch.bool)
    for b, (t, n) in enumerate(zip(lens, new)):
        for i in range(n):
            pg, r = cells(table, b, t - n + i, page)
            touched[pg, :, r] = True
            for src, got, exp in ((k, pool.k, pool.k_exp), (v, pool.v, pool.v_exp)):
                s = src[int(q_start[b]) + i].cpu()
                if exp is None:
                    assert torch.equal(bits(got[pg, :, r]), bits(s))
                else:
                    code, byte = O.quantise(s, store)
                    assert torch.equal(exp[pg, :, r].cpu(), byte)
                    assert torch.equal(got[pg, :, r].float().cpu().double(), code)
    for a, b in zip(before, after):                                  # everything else as it was
        assert torch.equal(a[~touched], b[~touched])
    # read back: ragged, longer than held for one, not at all for another; rows behind the last sequence stay
    take = [1, page - 2, 4, 2 * page + 3, 9, 0]
    start = torch.tensor([0] + take).cumsum(0).int()
    N = int(start[-1])
    for out_t in (F32, BF16):
        out = tuple(torch.full((N + 3, heads, dim), 5.0, dtype=out_t, device="cuda") for _ in range(2))
        got = ops.paged_kv_read(pool, table.cuda(), kv_len.cuda(), start.cuda(), N + 3, out=out)
        for g, held in zip(got, O.pool_values(pool)):
            assert bool((g[N:] == 5.0).all())
            want = torch.zeros(N, heads, dim, dtype=torch.float64)
            for b, m in enumerate(take):
                for p in range(min(m, lens[b])):
                    pg, r = cells(table, b, p, page)
                    want[int(start[b]) + p] = held[pg, :, r]
            w32 = want.float()
            assert torch.equal(g[:N].cpu().isnan(), w32.isnan()) and torch.equal(torch.nan_to_num(g[:N].cpu().float(), nan=1.5), torch.nan_to_num(w32.to(out_t).float(), nan=1.5))
    k2, v2 = ops.paged_kv_read(pool, table.cuda(), kv_len.cuda(), start.cuda(), N)
    assert k2.dtype == (store if store.itemsize > 1 else BF16) and k2.shape == (N, heads, dim)


@pytest.mark.parametrize("store", [BF16, E4M3])
def test_cache_bad_pages(store):
    """pages outside the pool, positions outside the table: nothing is written, zeros are read"""
    from ralf_amd import ops

    pool = ops.paged_kv_pool(3, 16, 2, 64, store)
    table = torch.tensor([[7, 1], [-5, 3], [2, 2 ** 31 - 1]], dtype=torch.int32).cuda()
    kv_len = torch.tensor([20, 30, 40], dtype=torch.int32).cuda()              # the last one longer than its table
    q_start = torch.tensor([0, 22, 52, 92], dtype=torch.int32).cuda()          # the first with more rows than tokens
    k = rnd(92, 2, 64, seed=1, dtype=BF16).cuda()
    ops.paged_kv_write(pool, k, 2 * k, table, q_start, kv_len)
    touched = torch.zeros(3, 16, dtype=torch.bool)
    touched[1, :4] = touched[2] = True
    held = O.pool_values(pool)
    want = torch.zeros(3, 2, 16, 64, dtype=torch.float64)
    for p in range(4):
        want[1, :, p] = k[2 + 16 + p].cpu().double()
    for p in range(16):
        want[2, :, p] = k[52 + p].cpu().double()
    if store == E4M3:
        assert ((held[0] != 0).flatten(3).any(-1).any(1) == touched).all()
    else:
        assert torch.equal(held[0], want) and torch.equal(held[1], 2 * want)
    got, _ = ops.paged_kv_read(pool, table, kv_len, q_start, 92)
    assert not got[:16].any() and got[16:20].any() and not got[20:52].any() and got[52:68].any() and not got[68:].any()


# ---------------------------------------------------------------------------------------------- attention
def run_attention(lens, new, Hq, heads, dim, page, store, dtype, seed=1, tail=0, scale=None, x=1.0, change=None, **kw):
    from ralf_amd import ops

    pool, table, q_start, kv_len = make(lens, new, heads, dim, page, store, dtype, seed)
    T = int(q_start[-1])
    q = (x * rnd(T + tail, Hq, dim, seed=seed + 5)).to(dtype)
    k, v = (rnd(T + tail, heads, dim, seed=seed + i, dtype=dtype) for i in (6, 7))
    if change is not None:
        change(q, k, v, pool, table)
    ops.paged_kv_write(pool, k.cuda(), v.cuda(), table.cuda(), q_start.cuda(), kv_len.cuda())
    wide = torch.full((T + tail, Hq + 1, dim), 3.0, dtype=dtype, device="cuda")
    qw = torch.zeros(T + tail, Hq + 2, dim, dtype=dtype, device="cuda")
    qw[:, 2:] = q.cuda()
    out = ops.paged_attention(qw[:, 2:], pool, table.cuda(), q_start.cuda(), kv_len.cuda(), scale=scale, out=wide[:, :Hq], **kw)
    assert bool((wide[:, Hq] == 3.0).all()) and bool((wide[T:] == 3.0).all())
    kw.pop("max_q", None), kw.pop("max_kv", None)
    want, e, done = O.attention(q, *O.pool_values(pool), table, q_start, kv_len, dim ** -0.5 if scale is None else scale,
                                p_step=O.half_step(dtype) if dtype == BF16 else 0.0, **kw)
    assert bool(done[:T].all())
    O.check(out[:T], want[:T], (e + O.half_step(dtype) * (want.abs() + e) + 1e-37)[:T], "attention")
    # without out=, without bounds: the same definition
    again = ops.paged_attention(q.cuda(), pool, table.cuda(), q_start.cuda(), kv_len.cuda(), scale=scale, **kw)
    O.check(again[:T], want[:T], (e + O.half_step(dtype) * (want.abs() + e) + 1e-37)[:T], "attention without bounds")
    return out[:T], want[:T]


TYPES = [(F32, F32), (BF16, BF16), (E4M3, F32), (E4M3, BF16), (I8, F32), (I8, BF16)]


@pytest.mark.parametrize("store,dtype", TYPES)
@pytest.mark.parametrize("dim", [32, 64, 128, 256])
def test_attention_types(store, dtype, dim):
    run_attention([37, 1, 70, 16], [5, 1, 33, 16], 6, 2, dim, 16, store, dtype, seed=dim, max_q=33, max_kv=70)


@pytest.mark.parametrize("Hq,heads,page", [(1, 1, 16), (8, 8, 32), (5, 1, 64), (40, 8, 16), (17, 1, 128), (12, 4, 256)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_heads(Hq, heads, page, dtype):
    run_attention([90, 33, 200], [1, 33, 7], Hq, heads, 64, page, dtype, dtype, seed=Hq, tail=3)


@pytest.mark.parametrize("kw", [dict(causal=False), dict(window=1), dict(window=13), dict(window=64, causal=False), dict(window=10 ** 6), dict(window=2 ** 31 - 1, causal=False), dict(scale=0.0),
                                dict(scale=-0.3), dict(x=30.0)])
@pytest.mark.parametrize("store,dtype", [(F32, F32), (BF16, BF16), (I8, BF16)])
def test_attention_masks(kw, store, dtype):
    run_attention([130, 64, 65, 1, 300], [40, 64, 1, 1, 3], 4, 2, 32, 32, store, dtype, seed=4, **kw)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_empty_rows(dtype):
    """sequences without tokens, without new ones, with more rows than tokens (the first rows see nothing), no keys at all"""
    out, want = run_attention([0, 5, 20, 3], [2, 9, 0, 3], 4, 2, 64, 16, dtype, dtype, seed=3, tail=2)
    assert not out[:2].any() and not out[2:6].any() and out[6:].any()
    from ralf_amd import ops

    pool = ops.paged_kv_pool(2, 16, 2, 64, dtype)
    none = torch.zeros(0, 3, dtype=torch.int32, device="cuda")
    q = rnd(4, 4, 64, dtype=dtype).cuda()
    ops.paged_attention(q, pool, none, torch.zeros(1, dtype=torch.int32, device="cuda"), none[:, 0].contiguous())
    ops.paged_attention(q[:0], pool, none, torch.zeros(1, dtype=torch.int32, device="cuda"), none[:, 0].contiguous())
    empty = torch.zeros(2, 0, dtype=torch.int32, device="cuda")                                   # a table without pages
    o = ops.paged_attention(q, pool, empty, torch.tensor([0, 1, 4], dtype=torch.int32, device="cuda"), torch.tensor([3, 9], dtype=torch.int32, device="cuda"))
    assert not o.any()


@pytest.mark.parametrize("lens,new,Hq,heads,dim,page,store", [
    ([70001], [1], 8, 2, 64, 64, BF16), ([9000, 17], [3, 2], 4, 1, 128, 16, E4M3), ([5000], [1], 32, 4, 128, 256, I8), ([30000], [2], 2, 2, 32, 128, BF16)])
def test_attention_long(lens, new, Hq, heads, dim, page, store):
    """few rows and many keys: the axis is split and joined"""
    run_attention(lens, new, Hq, heads, dim, page, store, BF16, seed=2, max_q=max(new), max_kv=max(lens))


@pytest.mark.parametrize("lens,new,Hq,heads,dim,page,store,kw", [
    ([400], [400], 8, 2, 128, 64, BF16, {}), ([700, 300, 40], [257, 1, 40], 4, 1, 64, 16, E4M3, {}), ([350], [130], 6, 2, 256, 32, I8, {}), ([500, 90], [300, 90], 3, 3, 32, 128, BF16, {}),
    ([600], [333], 4, 2, 128, 16, BF16, dict(window=100)), ([300], [200], 4, 4, 64, 64, E4M3, dict(causal=False)), ([2000], [129], 4, 1, 128, 64, BF16, dict(max_q=129, max_kv=2000)),
    ([257, 258, 1, 64], [257, 129, 1, 64], 5, 1, 128, 32, I8, dict(window=70))])
def test_attention_chunks(lens, new, Hq, heads, dim, page, store, kw):
    """many new tokens: tiles of rows that share their keys"""
    run_attention(lens, new, Hq, heads, dim, page, store, BF16, seed=7, tail=1, **kw)


@pytest.mark.parametrize("wrong", [dict(max_q=1, max_kv=1), dict(max_q=1), dict(max_kv=16), dict(max_q=10 ** 9, max_kv=10 ** 9)])
def test_attention_bounds_only_steer(wrong):
    run_attention([300, 200], [150, 3], 4, 2, 64, 16, BF16, BF16, seed=8, **wrong)


@pytest.mark.parametrize("n,past", [(1, 37), (6, 37), (70, 37), (300, 37), (3, 6000), (100, 6000)])
@pytest.mark.parametrize("store,dtype", [(F32, F32), (BF16, BF16), (E4M3, BF16), (E4M3, F32), (I8, BF16), (I8, F32)])
def test_attention_hidden_values_stay_hidden(store, dtype, n, past):
    """infinities and NaN in keys and values of tokens that a row does not see leave it alone; the rows that see them get them"""
    def change(q, k, v, pool, table):
        v[n // 2, 0, 3], v[n // 2, 1, 4], v[n - 1, 0, 5], v[n - 1, 0, 6] = math.nan, math.inf, -math.inf, math.nan
        k[n - 1, 1, 0] = math.nan

    out, want = run_attention([n + past], [n], 4, 2, 64, 16, store, dtype, seed=6, change=change)
    if n > 6:
        assert torch.isfinite(out[:n // 2]).all() and not torch.isfinite(out).all()
    run_attention([n + past], [n], 4, 2, 64, 16, store, dtype, seed=6, change=change, window=5)


def test_attention_infinite_scores():
    """scores of -inf throughout: no weight, zeros; one of them among others: left out"""
    def change(q, k, v, pool, table):
        q.zero_()
        q[:, :, 0] = 1.0
        k.zero_()
        k[:, 0, 0] = -math.inf

    out, _ = run_attention([3], [3], 2, 2, 32, 16, BF16, BF16, change=change)
    assert not out[:, 0].any() and out[:, 1].any()


@pytest.mark.parametrize("store", [BF16, I8])
def test_attention_bad_pages(store):
    from ralf_amd import ops

    pool, table, q_start, kv_len = make([100, 64], [1, 40], 2, 64, 16, store, BF16, seed=5)
    k, v, q = (rnd(41, h, 64, seed=h + i, dtype=BF16) for i, h in ((1, 2), (2, 2), (3, 4)))
    ops.paged_kv_write(pool, k.cuda(), v.cuda(), table.cuda(), q_start.cuda(), kv_len.cuda())
    table[0, 2], table[0, 5], table[1, 0], table[1, 3] = 10 ** 6, -1, pool.k.shape[0], -2 ** 31
    out = ops.paged_attention(q.cuda(), pool, table.cuda(), q_start.cuda(), kv_len.cuda())
    want, e, _ = O.attention(q, *O.pool_values(pool), table, q_start, kv_len, 0.125, p_step=O.half_step(BF16))
    O.check(out, want, e + O.half_step(BF16) * (want.abs() + e), "bad pages")


@pytest.mark.parametrize("store,dtype", [(BF16, BF16), (I8, F32)])
def test_empty_pool(store, dtype):
    """a cache without a page: nothing stored, zeros read, zeros attended"""
    from ralf_amd import ops

    pool = ops.paged_kv_pool(0, 16, 2, 32, store)
    table, one = torch.zeros(1, 2, dtype=torch.int32, device="cuda"), torch.tensor([5], dtype=torch.int32, device="cuda")
    start = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    k = rnd(3, 2, 32, dtype=dtype).cuda()
    ops.paged_kv_write(pool, k, k, table, start, one)
    assert not ops.paged_kv_read(pool, table, one, start, 3)[0].any()
    assert not ops.paged_attention(k, pool, table, start, one).any()


def test_strides_of_single_tokens_and_heads():
    """a dim of size 1 may have any stride"""
    from ralf_amd import ops

    pool, table, q_start, kv_len = make([20], [1], 1, 64, 16, BF16, BF16, seed=2)
    q = rnd(1, 3, 64, seed=3, dtype=BF16).cuda()
    k = rnd(1, 1, 64, seed=4, dtype=BF16).cuda()
    freq, axis = ops.rope_table((32,), device="cuda")
    pos = torch.tensor([[7]]).cuda()
    odd = lambda t: t.as_strided(t.shape, (193 if t.shape[0] == 1 else t.stride(0), 77 if t.shape[1] == 1 else t.stride(1), 1))    # noqa: E731
    assert torch.equal(ops.rope_axes(odd(q), pos, freq, axis), ops.rope_axes(q, pos, freq, axis))
    ops.paged_kv_write(pool, odd(k), odd(k), table.cuda(), q_start.cuda(), kv_len.cuda())
    pg, r = cells(table, 0, 19, 16)
    assert torch.equal(pool.k[pg, 0, r], k[0, 0])
    args = (pool, table.cuda(), q_start.cuda(), kv_len.cuda())
    assert torch.equal(ops.paged_attention(odd(q), *args, out=odd(torch.empty_like(q))), ops.paged_attention(q, *args))


@pytest.mark.parametrize("B", [65, 200, 4300])
@pytest.mark.parametrize("new", [0, 1, 40])
def test_many_sequences(B, new):
    """more sequences than a wave has lanes, and than its squares: new = 0: one or no new token each, otherwise one of them brings a chunk; page table rows of a wider pitch"""
    from ralf_amd import ops

    lens = [1 + b % 5 for b in range(B)]
    fresh = [min(t, (b * 7 % 3 > 0) * 1) for b, t in enumerate(lens)]
    if new:
        lens[B // 2], fresh[B // 2] = 70, new
    pool, table, q_start, kv_len = make(lens, fresh, 1, 32, 16, BF16, BF16, seed=B)
    wide = torch.full((B, table.shape[1] + 3), 2 ** 30, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table.cuda()
    strided = wide[:, :table.shape[1]]
    T = int(q_start[-1])
    q, k, v = rnd(T, 2, 32, seed=1, dtype=BF16), rnd(T, 1, 32, seed=2, dtype=BF16), rnd(T, 1, 32, seed=3, dtype=BF16)
    ops.paged_kv_write(pool, k.cuda(), v.cuda(), strided, q_start.cuda(), kv_len.cuda())
    start = torch.tensor([0] + lens).cumsum(0).int()
    rk, _ = ops.paged_kv_read(pool, strided, kv_len.cuda(), start.cuda(), int(start[-1]))
    held = O.pool_values(pool)
    rows = torch.tensor([(b, p) for b, t in enumerate(lens) for p in range(t)])
    assert torch.equal(rk.cpu().double(), held[0][table[rows[:, 0], rows[:, 1] // 16].long(), :, rows[:, 1] % 16])
    newest = torch.tensor([int(start[b]) + t - n + i for b, (t, n) in enumerate(zip(lens, fresh)) for i in range(n)])
    assert torch.equal(rk.cpu()[newest], k)
    for kw in (dict(), dict(max_q=max(fresh), max_kv=max(lens))):
        out = ops.paged_attention(q.cuda(), pool, strided, q_start.cuda(), kv_len.cuda(), **kw)
        want, e, _ = O.attention(q, *held, table, q_start, kv_len, 32 ** -0.5, p_step=O.half_step(BF16))
        O.check(out, want, e + O.half_step(BF16) * (want.abs() + e), "many sequences")


def test_attention_longer_than_the_table():
    """kv_len beyond what the table has room for: the keys that are there count, at their positions"""
    from ralf_amd import ops

    pool, table, q_start, kv_len = make([64], [8], 1, 32, 16, BF16, BF16, seed=5, garbage=False)
    table, kv_len = table[:, :4].contiguous(), torch.tensor([70], dtype=torch.int32)
    q = rnd(8, 2, 32, seed=3, dtype=BF16)
    for kw in (dict(), dict(window=9)):
        out = ops.paged_attention(q.cuda(), pool, table.cuda(), q_start.cuda(), kv_len.cuda(), **kw)
        want, e, _ = O.attention(q, *O.pool_values(pool), table, q_start, kv_len, 32 ** -0.5, p_step=O.half_step(BF16), **kw)
        O.check(out, want, e + O.half_step(BF16) * (want.abs() + e), "clamped")


def test_cache_beyond_32_bit_offsets():
    """a pool of 4.3 G elements a side: cells behind 2^32 bytes and 2^31 elements"""
    from ralf_amd import ops

    n, page, heads, dim = 66000, 256, 1, 256
    pool = ops.PagedKV(*(torch.empty(n, heads, page, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2)))
    assert pool.k.numel() > 2 ** 32
    table = torch.tensor([[n - 1, 3], [n - 2, n - 3]], dtype=torch.int32)
    q_start, kv_len = torch.tensor([0, 300, 600], dtype=torch.int32), torch.tensor([300, 300], dtype=torch.int32)
    k, v, q = (rnd(600, h, dim, seed=i, dtype=BF16) for i, h in ((1, 1), (2, 1), (3, 2)))
    ops.paged_kv_write(pool, k.cuda(), v.cuda(), table.cuda(), q_start.cuda(), kv_len.cuda())
    rk, rv = ops.paged_kv_read(pool, table.cuda(), kv_len.cuda(), q_start.cuda(), 600)
    assert torch.equal(rk.cpu(), k) and torch.equal(rv.cpu(), v)
    out = ops.paged_attention(q.cuda(), pool, table.cuda(), q_start.cuda(), kv_len.cuda())
    small = torch.stack([pool.k[p].cpu() for p in (n - 1, 3, n - 2, n - 3)]), torch.stack([pool.v[p].cpu() for p in (n - 1, 3, n - 2, n - 3)])
    want, e, _ = O.attention(q[290:310], small[0].double(), small[1].double(), torch.tensor([[0, 1], [2, 3]]), torch.tensor([0, 10, 20]), kv_len, 1 / 16, p_step=O.half_step(BF16))
    O.check(out[290:300], want[:10], (e + O.half_step(BF16) * (want.abs() + e))[:10], "far pages")
    tail = ops.paged_attention(q[590:].cuda(), pool, table[1:].cuda(), torch.tensor([0, 10], dtype=torch.int32).cuda(), kv_len[1:].cuda())
    want, e, _ = O.attention(q[590:], small[0].double(), small[1].double(), torch.tensor([[2, 3]]), torch.tensor([0, 10]), kv_len[1:], 1 / 16, p_step=O.half_step(BF16))
    O.check(tail, want, e + O.half_step(BF16) * (want.abs() + e), "far pages")
    del pool
    torch.cuda.empty_cache()


# ---------------------------------------------------------------------------------------------- logits
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,V,L", [(1, 1, 1), (3, 518, 51), (2, 519, 0), (5, 33, 200), (2, 40001, 300), (70, 2048, 9), (1, 20000, 700)])
def test_logits(dtype, B, V, L):
    from ralf_amd import ops

    g = gen(V)
    x = rnd(B, V, seed=V, dtype=dtype)
    x[:, 0], x[0, V // 2] = -math.inf, torch.finfo(dtype).min
    tokens = torch.randint(-2, V + 2, (B, L + 2), generator=g)[:, :L]            # ids outside the vocabulary, rows of another pitch
    lens = torch.randint(0, L + 1, (B,), generator=g).int()
    if L:
        lens[0] = L + 5                                                          # clamped
    prompt = (lens * torch.rand(B, generator=g)).int()
    r, p, f = 0.7 + torch.rand(B, generator=g), torch.rand(B, generator=g), torch.rand(B, generator=g)
    bias1, bias2 = rnd(V, seed=1), rnd(B, V + 3, seed=2)[:, :V]
    mask = torch.randint(-2 ** 31, 2 ** 31, (4, (V + 31) // 32 + 1), generator=g).int()
    mask[3] = 0
    row = torch.randint(-1, 5, (B,), generator=g).int()
    row[0] = 3 if B > 1 else 0
    c = lambda t: None if t is None else t.cuda()    # noqa: E731
    for kw in (dict(repetition=r, presence=p, frequency=f, prompt_lens=prompt, bias=bias1, mask=mask, mask_row=row), dict(repetition=r), dict(presence=p, bias=bias2), dict(frequency=f, prompt_lens=prompt),
               dict(mask=mask, mask_row=row), dict(bias=bias2), dict(mask=mask[torch.arange(B) % 4].contiguous()), dict()):
        want, e = O.logits(x, tokens, lens, kw.get("prompt_lens"), kw.get("repetition"), kw.get("presence"), kw.get("frequency"), kw.get("bias"), kw.get("mask"), kw.get("mask_row"))
        big = want.abs() > torch.finfo(dtype).max                                 # the lowest value made larger: -inf once rounded
        want = torch.where(big, want.sign() * math.inf, want)
        e = torch.where(big, 0.0, e)
        args = {n: c(t) for n, t in kw.items()}
        y = ops.logits_process(x.cuda(), tokens.cuda(), lens.cuda(), **args)
        O.check(y, want, e + O.half_step(dtype) * (want.abs().nan_to_num(posinf=0.0) + e), str(list(kw)))
        z = x.cuda()
        assert ops.logits_process(z, tokens.cuda(), lens.cuda(), out=z, **args) is z and torch.equal(bits(z), bits(y))
        wide = torch.full((B, V + 5), 9.0, dtype=dtype, device="cuda")
        src = torch.zeros(B, V + 4, dtype=dtype, device="cuda")
        src[:, :V] = x.cuda()
        ops.logits_process(src[:, :V], tokens.cuda(), lens.cuda(), out=wide[:, :V], **args)
        assert torch.equal(bits(wide[:, :V]), bits(y)) and bool((wide[:, V:] == 9.0).all())
    assert ops.logits_process(x[:0].cuda()).shape == (0, V)


# ---------------------------------------------------------------------------------------------- together
def step(ops, s):
    """one serving step as a program runs it: rotate q and k of the packed projection, store, attend, project, treat the logits, choose"""
    n = s["Hq"] + s["Hk"]
    qkv = s["qkv"]
    rot = ops.rope_axes(qkv[:, :n], s["pos"], s["freq"], s["axis"])
    ops.paged_kv_write(s["pool"], rot[:, s["Hq"]:], qkv[:, n:], s["table"], s["q_start"], s["kv_len"])
    o = ops.paged_attention(rot[:, :s["Hq"]], s["pool"], s["table"], s["q_start"], s["kv_len"], max_q=s["max_q"], max_kv=s["max_kv"])
    z = ops.gemm(o.view(o.shape[0], -1), s["W"], o.shape[0], s["W"].shape[0], s["W"].shape[1], out_dtype=F32)
    ops.logits_process(z, s["tokens"], s["lens"], repetition=s["rep"], mask=s["mask"], mask_row=s["mask_row"], out=z)
    return rot, o, z, ops.mask_sample(z)


def serving_state(ops, lens, new, store, dtype, seed):
    Hq, Hk, D, V = 8, 2, 32, 518
    pool, table, q_start, kv_len = make(lens, new, Hk, D, 16, store, dtype, seed)
    T = sum(new)
    freq, axis = ops.rope_table((8, 8))
    s = dict(Hq=Hq, Hk=Hk, pool=pool, table=table, q_start=q_start, kv_len=kv_len, max_q=max(new), max_kv=max(lens), qkv=rnd(T, Hq + 2 * Hk, D, seed=seed, dtype=dtype),
             pos=torch.randint(0, 60, (2, T), generator=gen(seed)), freq=freq, axis=axis, W=0.2 * rnd(V, Hq * D, seed=seed + 1, dtype=dtype),
             tokens=torch.randint(0, V, (T, 20), generator=gen(seed)), lens=torch.full((T,), 20, dtype=torch.int32), rep=1 + torch.rand(T, generator=gen(seed)),
             mask=torch.randint(-2 ** 31, 2 ** 31, (2, 17), generator=gen(seed)).int(), mask_row=(torch.arange(T) % 3 - 1).int())
    return {n: v.cuda() if torch.is_tensor(v) else v for n, v in s.items()}


def check_step(s, got):
    rot, o, z, choice = got
    cpu = {n: v.cpu() if torch.is_tensor(v) else v for n, v in s.items()}
    dtype, Hq = s["qkv"].dtype, s["Hq"]
    want, e = O.rope(cpu["qkv"][:, :Hq + s["Hk"]], cpu["pos"], cpu["freq"], cpu["axis"], False)
    O.check(rot, want, e + O.half_step(dtype) * (want.abs() + e), "rope")
    want, e, _ = O.attention(rot[:, :Hq].cpu(), *O.pool_values(s["pool"]), cpu["table"], cpu["q_start"], cpu["kv_len"], 32 ** -0.5, p_step=O.half_step(dtype) if dtype == BF16 else 0.0)
    O.check(o, want, e + O.half_step(dtype) * (want.abs() + e), "attention")
    a, w = o.cpu().double().flatten(1), cpu["W"].double()
    raw = a @ w.t()
    want, e = O.logits(raw, cpu["tokens"], cpu["lens"], None, cpu["rep"], None, None, None, cpu["mask"], cpu["mask_row"])
    e = e + 2 * (a.shape[1] + 4) * O.U32 * (a.abs() @ w.abs().t())            # the product's fp32 sums, times a repetition factor of at most 2
    O.check(z, want, e + O.U32 * want.abs().nan_to_num(posinf=0.0), "logits")
    assert torch.equal(choice, z.argmax(1))


@pytest.mark.parametrize("store,dtype", [(BF16, BF16), (E4M3, BF16), (F32, F32), (I8, F32)])
def test_serving_steps_together(store, dtype):
    """a prompt's chunk, then single tokens, on the same cache"""
    from ralf_amd import ops

    s = serving_state(ops, [40, 23, 64], [30, 23, 1], store, dtype, seed=11)
    check_step(s, step(ops, s))
    for i in range(3):
        T = 3
        s.update(kv_len=s["kv_len"] + 1, max_kv=s["max_kv"] + 1, max_q=1, q_start=torch.arange(4, dtype=torch.int32).cuda(), qkv=rnd(T, 12, 32, seed=50 + i, dtype=dtype).cuda(),
                 pos=torch.randint(0, 60, (2, T), generator=gen(i)).cuda())
        for n in ("tokens", "lens", "rep", "mask_row"):
            s[n] = s[n][:T].contiguous()
        if int(s["kv_len"][2]) > 64:                                          # the third sequence needs a page: one of the spare ones
            used = set(s["table"].flatten().tolist())
            if int(s["table"][2, 4]) < 0:
                s["table"][2, 4] = next(p for p in range(s["pool"].k.shape[0]) if p not in used)
        check_step(s, step(ops, s))


@pytest.mark.parametrize("lens,new", [([200, 90], [1, 1]), ([200, 90], [100, 60]), ([4000], [1])])
def test_captured_step_replays(lens, new):
    """the step in a graph, replayed on changed inputs, with eager work of the same operators and a second graph's replays in between: every replay is the eager step"""
    from ralf_amd import ops

    st = ops.own_stream("serving_test")
    states, graphs, outs = [], [], []
    for seed in (21, 22):
        s = serving_state(ops, lens, new, E4M3, BF16, seed)
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            step(ops, s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            out = step(ops, s)
        states.append(s), graphs.append(g), outs.append(out)
    eager = serving_state(ops, [50], [7], BF16, BF16, 30)
    for turn in range(3):
        want = []
        for i, s in enumerate(states):
            s["qkv"].copy_(rnd(*s["qkv"].shape, seed=100 + 10 * turn + i, dtype=BF16))
            s["kv_len"].copy_(torch.tensor([t - turn for t in lens], dtype=torch.int32))
            want.append([t.clone() for t in step(ops, s)])
        for i in (0, 1):
            graphs[i].replay()
        check_step(eager, step(ops, eager))
        torch.cuda.synchronize()
        for w, o in zip(want, outs):
            for a, b in zip(w, o):
                assert torch.equal(bits(a) if a.dtype != torch.int64 else a, bits(b) if b.dtype != torch.int64 else b)


def test_rope_gradient_captured_beside_an_eager_graph():
    """forward and gradient in a graph while an eager autograd graph of the same leaf is alive: by the opposite rotation, which needs no autograd graph (with one, a leaf
    is refused in a capture: tests/test_serving_cpu.py)"""
    from ralf_amd import functional, ops

    freq, axis = ops.rope_table((16,), device="cuda")
    pos = torch.arange(8).view(1, 8).cuda()
    x, dy = rnd(8, 2, 32, seed=1).cuda().requires_grad_(True), rnd(8, 2, 32, seed=2).cuda()
    alive = functional.rope_axes(x, pos, freq, axis)
    want, = torch.autograd.grad(functional.rope_axes(x, pos, freq, axis), x, dy)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(g, stream=ops.own_stream("serving_test")):
        y = functional.rope_axes(x, pos, freq, axis)
        got = ops.rope_axes(dy, pos, freq, axis, inverse=True)
    for k in range(3):
        got.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(y, alive)
    alive.backward(dy)
    assert torch.equal(x.grad, want)


def test_other_streams():
    """every operator on a stream of its own, ordered by it alone"""
    from ralf_amd import ops

    s = serving_state(ops, [300, 40, 7], [64, 1, 7], E4M3, BF16, 31)
    want = [t.clone() for t in step(ops, s)]
    torch.cuda.synchronize()
    st = ops.own_stream("serving_test_2")
    for k in range(4):
        with torch.cuda.stream(st):
            got = step(ops, s)
        st.synchronize()
        for a, b in zip(want, got):
            assert torch.equal(a, b)
