"""The serving operators in 64 bits on the CPU, token by token where that is the plainest, with the bounds that the kernels' roundings allow."""
import math

import torch

U32 = 2.0 ** -24                    # half a step of fp32, relative
LARGEST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rope(x, pos, freq, axis, adjacent, sign=1):
    """(y, bound without the output's rounding): sin / cos are off by 2 pi 2^-26 (the fraction of a turn in fp32) and 2 steps of 2^-23 at most; two products, a sum"""
    x = x.double()
    R = 2 * freq.numel()
    a = sign * pos.double()[axis.long().clamp(0, pos.shape[0] - 1)].t() * freq
    a = torch.where((axis >= 0) & (axis < pos.shape[0]), a, 0.0)
    c, s = a.cos()[:, None], a.sin()[:, None]
    i = torch.arange(0, R, 2) if adjacent else torch.arange(R // 2)
    j = i + (1 if adjacent else R // 2)
    y, e = x.clone(), torch.zeros_like(x)
    y[..., i] = x[..., i] * c - x[..., j] * s
    y[..., j] = x[..., j] * c + x[..., i] * s
    off = 2 * math.pi * 2.0 ** -26 + 2 * 2.0 ** -23 + 3 * U32
    e[..., i] = e[..., j] = (x[..., i].abs() + x[..., j].abs()) * off
    return y, e


def quantise(x, store):
    """(codes as float64, exponent bytes) of rows [..., dim]: the smallest e >= -100 with max|x| <= largest * 2^e, codes to the nearest (ties to even)"""
    x = x.double()
    top = x.abs().amax(-1)
    bad = ~torch.isfinite(x).all(-1)
    safe = torch.where(bad | (top == 0), torch.ones_like(top), top)
    e = torch.floor(torch.log2(safe / LARGEST[store])).long() - 1
    for _ in range(3):
        e = e + (safe > LARGEST[store] * torch.ldexp(torch.ones_like(safe), e)).long()
    e = torch.where(top == 0, torch.full_like(e, -100), e).clamp(min=-100)
    y = torch.ldexp(torch.where(bad[..., None], torch.zeros_like(x), x), -e[..., None])
    if store == torch.int8:
        code = torch.round(y)
    else:
        b = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
        hi = torch.searchsorted(b, y.abs().contiguous()).clamp(max=126)
        lo = (hi - 1).clamp(min=0)
        up, down = b[hi] - y.abs(), y.abs() - b[lo]
        code = torch.where((down < up) | ((down == up) & (lo % 2 == 0)), b[lo], b[hi]) * torch.where(y < 0, -1.0, 1.0)
    return code, torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)


def value(code, byte):
    v = torch.ldexp(code.double(), byte.long()[..., None] - 127)
    return torch.where(byte[..., None] == 255, torch.full_like(v, math.nan), v)


def pool_values(pool):
    """the cache's k, v in 64 bits on the CPU"""
    out = []
    for p, e in ((pool.k, pool.k_exp), (pool.v, pool.v_exp)):
        p = p.cpu()
        out.append(p.double() if e is None else value(p.float(), e.cpu()))
    return out


def attention(q, k_pages, v_pages, table, q_start, kv_len, scale, causal=True, window=0, p_step=0.0):
    """(o, bound without the output's rounding); k_pages, v_pages: pool_values.  p_step: half a step of the type that the probabilities are rounded to"""
    q = q.double()
    T, Hq, D = q.shape
    n_pages, Hk, page, _ = k_pages.shape
    o, e = torch.zeros_like(q), torch.zeros_like(q)
    done = torch.zeros(T, dtype=torch.bool)
    for b in range(table.shape[0]):
        s0, s1 = int(q_start[b]), min(int(q_start[b + 1]), T)
        n = int(q_start[b + 1]) - s0
        L = max(0, min(int(kv_len[b]), table.shape[1] * page))
        p = torch.arange(L)
        pg = table[b].long()[p // page]
        good = (pg >= 0) & (pg < n_pages)
        kk, vv = k_pages[pg.clamp(0, n_pages - 1), :, p % page], v_pages[pg.clamp(0, n_pages - 1), :, p % page]      # [L, Hk, D]
        for i in range(s1 - s0):
            at = int(kv_len[b]) - n + i
            see = good & ((p <= at) if causal else torch.ones_like(good)) & ((p > at - window) if window else torch.ones_like(good))
            done[s0 + i] = True
            if not see.any():
                continue
            ks, vs = kk[see], vv[see]
            for h in range(Hq):
                qk = ks[:, h // (Hq // Hk)] * q[s0 + i, h]
                z = qk.sum(-1) * scale
                # products exact in fp32's accumulation up to one rounding a term; the scale, the maximum's difference and exp2 (2 steps): relative error of a weight
                dz = (D + 6) * U32 * qk.abs().sum(-1) * abs(scale)
                m = z.max()
                if m == -math.inf:
                    continue
                w = torch.exp(z - m)
                w = w / w.sum()
                vh = vs[:, h // (Hq // Hk)]
                o[s0 + i, h] = (w[:, None] * vh).sum(0)
                mag = (w[:, None] * vh.abs()).sum(0)
                rel = 2 * (dz.max() if torch.isfinite(dz).all() else 0.0) + p_step + (ks.shape[0] + 16) * U32 + 8 * 2.0 ** -23
                e[s0 + i, h] = mag * rel
    return o, e, done


def logits(x, tokens, lens, prompt, r, p, f, bias, mask, mask_row):
    """(y, bound without the output's rounding)"""
    x = x.double().clone()
    e = torch.zeros_like(x)
    B, V = x.shape
    for b in range(B):
        if r is not None or p is not None or f is not None:
            n = max(0, min(int(lens[b]), tokens.shape[1]))
            m = 0 if prompt is None else int(prompt[b])
            for v in set(t for t in tokens[b, :n].tolist() if 0 <= t < V):
                c = sum(1 for i in range(n) if i >= m and int(tokens[b, i]) == v)
                if r is not None:
                    x[b, v] = x[b, v] / r[b].double() if x[b, v] > 0 else x[b, v] * r[b].double()
                fc = 0.0 if f is None else float(f[b]) * c
                pc = 0.0 if p is None or c == 0 else float(p[b])
                if math.isfinite(x[b, v]):
                    e[b, v] = 4 * U32 * (abs(float(x[b, v])) + abs(fc) + abs(pc))
                x[b, v] -= fc + pc
        if bias is not None:
            bb = (bias if bias.dim() == 1 else bias[b]).double()
            x[b] += bb
            e[b] += torch.where(torch.isfinite(x[b]), U32 * (x[b].abs() + bb.abs()), 0.0)
        if mask is not None:
            mr = b if mask_row is None else int(mask_row[b])
            if 0 <= mr < mask.shape[0]:
                v = torch.arange(V)
                x[b][((mask[mr].long()[v // 32] >> (v % 32)) & 1) == 0] = -math.inf
    return x, e


def check(got, want, bound, what=""):
    """every element within its bound; infinities and NaN in the same places"""
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN elsewhere"
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], want[inf]), f"{what}: infinities elsewhere"
    ok = torch.isfinite(want)
    over = ((got - want).abs() - bound)[ok]
    if over.numel():
        worst = over.max().item()
        assert worst <= 0, f"{what}: {worst:.3g} over the bound at {(over == over.max()).nonzero()[0].item()}"
