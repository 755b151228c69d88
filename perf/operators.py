"""Cases of the serving operators: rotary positions with several axes, the paged key/value cache (quantised as it is written, read back),
attention of new tokens over that cache, and the history-dependent treatment of logits in front of the token choice.

`own = False`: the operators in elementary torch operations; `own = True`: the framework's entry points (ralf_amd.ops, ralf_amd.functional)."""
import math

import torch

own = False

_STORES = {"same": None, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
_LARGEST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def listed():
    return [
        # one generated token of one small sequence, q and k heads of a packed projection: latency alone
        dict(name="rope_token", op="rope", tokens=1, heads=16, dim=32, sections="16", adjacent=False, dtype="float32", backward=False, far=50),
        # a training step over a video / image-grid sequence: time, height, width; forward and the gradient of x
        dict(name="rope_grid_train", op="rope", tokens=16384, heads=40, dim=128, sections="16,24,24", adjacent=False, dtype="bfloat16", backward=True, far=1000),
        # a decode step of 64 sequences into an unquantised cache
        dict(name="cache_step", op="cache", seqs=64, kv=2000, new=1, heads=8, dim=128, page=16, store="same", dtype="bfloat16", read=False, mixed=False),
        # prompts of up to 1024 tokens written in 8-bit floats, and the sequences read back whole (hand-over to another worker)
        dict(name="cache_e4m3", op="cache", seqs=16, kv=4100, new=1024, heads=8, dim=128, page=64, store="e4m3", dtype="bfloat16", read=True, mixed=False),
        # fp32 parity mode, 8-bit integers, short ragged sequences in pages of 16
        dict(name="cache_int8", op="cache", seqs=37, kv=517, new=129, heads=4, dim=64, page=16, store="int8", dtype="float32", read=True, mixed=False),
        # one token of one layout (8 heads of 32, at most 51 positions): the smallest attention call
        dict(name="attn_token", op="attention", seqs=1, kv=51, new=1, q_heads=8, heads=8, dim=32, page=16, store="same", dtype="bfloat16", window=0, mixed=False),
        # a decode step of 64 ragged sequences over an 8-bit cache, 4 query heads to a key head
        dict(name="attn_batch_e4m3", op="attention", seqs=64, kv=8192, new=1, q_heads=32, heads=8, dim=128, page=64, store="e4m3", dtype="bfloat16", window=0, mixed=False),
        # one sequence far out: few rows, all of the card has to come from the keys' axis
        dict(name="attn_long", op="attention", seqs=1, kv=131072, new=1, q_heads=32, heads=4, dim=128, page=256, store="same", dtype="bfloat16", window=0, mixed=False),
        # a chunk of a long prompt on top of what is cached: matrix products
        dict(name="attn_chunk", op="attention", seqs=1, kv=10240, new=2048, q_heads=32, heads=8, dim=128, page=64, store="same", dtype="bfloat16", window=0, mixed=False),
        # fp32 parity mode: prompts' chunks and single tokens in one call, 8-bit integers, sliding window
        dict(name="attn_mixed_int8", op="attention", seqs=9, kv=1500, new=200, q_heads=12, heads=4, dim=64, page=16, store="int8", dtype="float32", window=400, mixed=True),
        # the layout vocabulary, 51 positions of history, per-task grammar masks
        dict(name="logits_layout", op="logits", rows=64, vocab=518, history=51, dtype="float32", bias="shared", masks=4),
        # a large vocabulary and long histories, a mask per row
        dict(name="logits_wide", op="logits", rows=64, vocab=130001, history=4096, dtype="float32", bias="rows", masks=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "cache", "attention", "attention", "attention", "logits"])
    if op == "rope":
        half = rng.choice([8, 16, 20, 32, 33, 48, 64])
        a = rng.randint(1, 3)
        cut = sorted(rng.sample(range(1, half), a - 1))
        sections = [y - x for x, y in zip([0] + cut, cut + [half])]
        return dict(op=op, tokens=_log(rng, 1, 8000), heads=rng.choice([1, 2, 3, 8, 10, 16, 40]), dim=2 * half + rng.choice([0, 0, 0, 6, 32]), sections=",".join(map(str, sections)),
                    adjacent=rng.random() < 0.4, dtype=rng.choice(["bfloat16", "bfloat16", "float32"]), backward=rng.random() < 0.5, far=_log(rng, 10, 1000000))
    if op == "logits":
        rows = _log(rng, 1, 256)
        return dict(op=op, rows=rows, vocab=min(_log(rng, 500, 260000), 8000000 // rows), history=_log(rng, 1, 4000), dtype=rng.choice(["float32", "float32", "bfloat16"]),
                    bias=rng.choice(["none", "shared", "rows"]), masks=rng.choice([0, 1, 3, rows]))
    heads, dim, page = rng.choice([1, 2, 4, 8]), rng.choice([32, 64, 128, 128, 256]), rng.choice([16, 32, 64, 128, 256])
    store, dtype = rng.choice(["same", "e4m3", "int8"]), rng.choice(["bfloat16", "bfloat16", "float32"])
    if op == "cache":
        seqs, read = _log(rng, 1, 64), rng.random() < 0.6
        kv = _log(rng, 1, 60000 // seqs)
        return dict(op=op, seqs=seqs, kv=kv, new=_log(rng, 1, kv), heads=heads, dim=dim, page=page, store=store, dtype=dtype, read=read or store != "same", mixed=rng.random() < 0.4)
    seqs, q_heads = _log(rng, 1, 64), heads * rng.choice([1, 2, 4, 5, 8])
    kv = _log(rng, 1, max(2, min(60000, 200000 // (seqs * heads))))
    most = max(1, min(kv, 300000000 // (seqs * q_heads * kv), 16000 // seqs))
    new = rng.choice([1, _log(rng, 1, most)])
    return dict(op=op, seqs=seqs, kv=kv, new=new, q_heads=q_heads, heads=heads, dim=dim, page=page, store=store, dtype=dtype,
                window=rng.choice([0, 0, 0, _log(rng, 1, kv)]), mixed=rng.random() < 0.4)


def _lengths(case):
    """(new, total) tokens of each sequence: ragged by a fixed pattern from a quarter of the largest up; `mixed`: only every fourth brings a chunk"""
    B, kv, new = case["seqs"], case["kv"], case["new"]
    part = [1.0 - 0.75 * ((37 * b) % B) / B for b in range(B)]
    total = [max(1, round(kv * f)) for f in part]
    fresh = [max(1, round(new * f)) if not case["mixed"] or b % 4 == 0 else 1 for b, f in enumerate(part)]
    return [min(n, t) for n, t in zip(fresh, total)], total


def _sections(case):
    return [int(s) for s in case["sections"].split(",")]


def _power(e):
    """2^e in 32 bits, exactly"""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantised(x, store):
    """codes, and 127 + e of the power of two that they are multiples of: e is the smallest integer with max |x| <= largest code * 2^e, at least -100"""
    x = x.float()
    m, e = torch.frexp(x.abs().amax(-1))
    m0, e0 = math.frexp(_LARGEST[store])
    e = (e - e0 + (m > m0).int()).clamp(min=-100)
    y = x * _power(-e)[..., None]
    return (y.round().to(store) if store == torch.int8 else y.to(store)), (e + 127).to(torch.uint8)


def _value(code, exp):
    return code.float() * _power(exp.int() - 127)[..., None] if exp is not None else code.float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = torch.device("cuda")
    op, dtype = case["op"], getattr(torch, case["dtype"])

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    if op == "rope":
        T, H, D, sec = case["tokens"], case["heads"], case["dim"], _sections(case)
        R = 2 * sum(sec)
        s = dict(x=normal(T, H, D).to(dtype), adjacent=case["adjacent"], backward=case["backward"])
        # a grid of 24 columns read row by row, 20 rows to a picture; single tokens stand somewhere in it
        i = torch.arange(T, device=dev) + int(torch.randint(0, 480, (), generator=g, device=dev))
        s["pos"] = torch.stack([i // 480 + case["far"], i // 24 % 20, i % 24][:len(sec)] if len(sec) > 1 else [i + case["far"]])
        s["freq"] = 10000.0 ** (-2.0 * torch.arange(R // 2, device=dev, dtype=torch.float64) / R)
        s["axis"] = torch.repeat_interleave(torch.arange(len(sec), device=dev, dtype=torch.int32), torch.tensor(sec, device=dev))
        s["dy"] = normal(T, H, D).to(dtype)
        s["x"].requires_grad_(case["backward"])
        return s
    if op == "logits":
        B, V, N = case["rows"], case["vocab"], case["history"]
        s = dict(logits=(4 * normal(B, V)).to(dtype))
        # few ids come often, as in text
        s["tokens"] = (V * torch.rand(B, N, generator=g, device=dev, dtype=torch.float64) ** 4).long().clamp(max=V - 1)
        s["lens"] = torch.randint(max(1, N // 2), N + 1, (B,), generator=g, device=dev).int()
        s["prompt"] = (s["lens"] * torch.rand(B, generator=g, device=dev)).int()
        s["repetition"] = 1 + 0.3 * torch.rand(B, generator=g, device=dev)
        s["presence"], s["frequency"] = torch.rand(B, generator=g, device=dev), 0.2 * torch.rand(B, generator=g, device=dev)
        s["bias"] = None if case["bias"] == "none" else normal(V) if case["bias"] == "shared" else normal(B, V)
        M = case["masks"]
        words = torch.randint(-2 ** 31, 2 ** 31, (max(M, 1), (V + 31) // 32), generator=g, device=dev)
        s["mask"] = words.int() if M else None
        s["mask_row"] = torch.randint(-1, M, (B,), generator=g, device=dev).int() if M else None
        return s
    new, total = _lengths(case)
    H, D, page, store = case["heads"], case["dim"], case["page"], _STORES[case["store"]]
    T, need = sum(new), [-(-t // page) for t in total]
    n = sum(need) + 3
    order = torch.randperm(n, generator=g, device=dev).int()
    at = torch.arange(max(need), device=dev)
    need_t = torch.tensor(need, device=dev)
    first = need_t.cumsum(0) - need_t
    table = torch.where(at[None] < need_t[:, None], order[(first[:, None] + at[None]).clamp(max=n - 1)], -1)
    s = dict(table=table, q_start=torch.tensor([0] + new, device=dev).cumsum(0).int(), kv_len=torch.tensor(total, device=dev).int(), max_q=max(new), max_kv=max(total), page=page)
    for name in ("k", "v"):
        cached = normal(n, H, page, D).to(dtype)
        s[name + "_pages"], s[name + "_exp"] = _quantised(cached, store) if store is not None else (cached, None)
    if op == "cache":
        # keys and values as slices of one packed projection
        qkv = normal(T, 2 * H, D).to(dtype)
        s.update(k=qkv[:, :H], v=qkv[:, H:], read=case["read"], dtype=dtype)
        s["start"] = torch.tensor([0] + total, device=dev).cumsum(0).int()
        s["rows"] = sum(total)
        return s
    s.update(q=normal(T, case["q_heads"], D).to(dtype), window=case["window"])
    return s


def _rope_plain(x, pos, freq, axis, adjacent, sign):
    angle = sign * pos[axis.long()].t().double() * freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    h, R = x.float(), 2 * freq.numel()
    a, b = (h[..., 0:R:2], h[..., 1:R:2]) if adjacent else (h[..., :R // 2], h[..., R // 2:R])
    a, b = a * cos - b * sin, b * cos + a * sin
    y = torch.stack([a, b], -1).flatten(-2) if adjacent else torch.cat([a, b], -1)
    return torch.cat([y, h[..., R:]], -1).to(x.dtype)


def _places(s):
    """page and row in it of each new token"""
    T = s["k"].shape[0]
    t = torch.arange(T, device=s["k"].device)
    b = torch.searchsorted(s["q_start"][1:].long(), t, right=True)
    p = s["kv_len"].long()[b] - s["q_start"].long()[b + 1] + t
    return s["table"][b, p // s["page"]].long(), p % s["page"]


def _write_plain(s):
    page, row = _places(s)
    for name in ("k", "v"):
        pages, exp = s[name + "_pages"], s[name + "_exp"]
        if exp is None:
            pages[page, :, row] = s[name]
        else:
            code, e = _quantised(s[name], pages.dtype)
            pages.view(torch.uint8)[page, :, row] = code.view(torch.uint8)
            exp[page, :, row] = e


def _read_plain(s):
    n = torch.arange(s["rows"], device=s["table"].device)
    b = torch.searchsorted(s["start"][1:].long(), n, right=True)
    p = n - s["start"].long()[b]
    page, row = s["table"][b, p // s["page"]].long(), p % s["page"]
    return tuple(_value(s[x + "_pages"].view(torch.uint8)[page, :, row].view(s[x + "_pages"].dtype) if s[x + "_exp"] is not None else s[x + "_pages"][page, :, row],
                        s[x + "_exp"][page, :, row] if s[x + "_exp"] is not None else None).to(s["dtype"]) for x in ("k", "v"))


def _attention_plain(s):
    q, L = s["q"], s["max_kv"]
    T, Hq, D = q.shape
    table = s["table"].long().clamp(min=0)
    B, Hk = table.shape[0], s["k_pages"].shape[1]

    def rows(x):                                                        # [B, Hk, L, D]
        pages, exp = s[x + "_pages"], s[x + "_exp"]
        got = _value(pages.view(torch.uint8)[table].view(pages.dtype), exp[table]) if exp is not None else pages[table].float()
        return got.transpose(1, 2).reshape(B, Hk, -1, D)[:, :, :L].contiguous()

    k, v = rows("k"), rows("v")
    start, kv_len = s["q_start"].long(), s["kv_len"].long()
    i = torch.arange(s["max_q"], device=q.device)
    new = start[1:] - start[:-1]
    there = i[None] < new[:, None]
    token = torch.where(there, start[:-1, None] + i[None], 0)
    padded = q[token].float().reshape(B, -1, Hk, Hq // Hk, D).transpose(1, 2).reshape(B, Hk, -1, D)
    score = torch.matmul(padded, k.transpose(2, 3).contiguous()) * D ** -0.5
    at = (kv_len - new)[:, None] + i[None]
    p = torch.arange(L, device=q.device)
    seen = (p[None, None] <= at[..., None]) & there[..., None]
    if s["window"]:
        seen &= p[None, None] > at[..., None] - s["window"]
    seen = seen[:, None, :, None].expand(-1, -1, -1, Hq // Hk, -1).reshape(B, 1, -1, L)
    score = score.masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight, v) / torch.where(total > 0, total, 1.0)
    out = out.reshape(B, Hk, -1, Hq // Hk, D).transpose(1, 2).reshape(B, -1, Hq, D)
    t = torch.arange(T, device=q.device)
    b = torch.searchsorted(start[1:].contiguous(), t, right=True)
    return out[b, t - start[b]].to(q.dtype)


def _logits_plain(s):
    x = s["logits"].float()
    B, V = x.shape
    at = torch.arange(s["tokens"].shape[1], device=x.device)[None]
    live = at < s["lens"][:, None]
    seen = torch.zeros(B, V, device=x.device, dtype=torch.int32).scatter_add_(1, s["tokens"], live.int())
    out = torch.zeros(B, V, device=x.device, dtype=torch.int32).scatter_add_(1, s["tokens"], (live & (at >= s["prompt"][:, None])).int())
    r = s["repetition"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * out - s["presence"][:, None] * (out > 0)
    if s["bias"] is not None:
        x = x + s["bias"]
    if s["mask"] is not None:
        v = torch.arange(V, device=x.device)
        words = s["mask"][s["mask_row"].long().clamp(min=0)][:, v // 32]
        allowed = ((words >> (v % 32).int()) & 1).bool() | (s["mask_row"] < 0)[:, None]
        x = torch.where(allowed, x, -math.inf)
    return x.to(s["logits"].dtype)


def run(s):
    if own:
        from ralf_amd import functional, ops

        if "freq" in s:
            if not s["backward"]:
                return ops.rope_axes(s["x"], s["pos"], s["freq"], s["axis"], adjacent=s["adjacent"])
            y = functional.rope_axes(s["x"], s["pos"], s["freq"], s["axis"], adjacent=s["adjacent"])
            return (y.detach(), *torch.autograd.grad(y, s["x"], s["dy"]))
        if "logits" in s:
            return ops.logits_process(s["logits"], s["tokens"], s["lens"], prompt_lens=s["prompt"], repetition=s["repetition"], presence=s["presence"],
                                      frequency=s["frequency"], bias=s["bias"], mask=s["mask"], mask_row=s["mask_row"])
        pool = ops.PagedKV(s["k_pages"], s["v_pages"], s["k_exp"], s["v_exp"])
        if "q" in s:
            return ops.paged_attention(s["q"], pool, s["table"], s["q_start"], s["kv_len"], window=s["window"], max_q=s["max_q"], max_kv=s["max_kv"])
        ops.paged_kv_write(pool, s["k"], s["v"], s["table"], s["q_start"], s["kv_len"])
        if s["read"]:
            return ops.paged_kv_read(pool, s["table"], s["kv_len"], s["start"], s["rows"], dtype=s["dtype"])
        return pool.k, pool.v
    if "freq" in s:
        y = _rope_plain(s["x"].detach(), s["pos"], s["freq"], s["axis"], s["adjacent"], 1)
        return (y, _rope_plain(s["dy"], s["pos"], s["freq"], s["axis"], s["adjacent"], -1)) if s["backward"] else y
    if "logits" in s:
        return _logits_plain(s)
    if "q" in s:
        return _attention_plain(s)
    _write_plain(s)
    return _read_plain(s) if s["read"] else (s["k_pages"], s["v_pages"])


def work(case):
    size = {"bfloat16": 2, "float32": 4}[case["dtype"]]
    if case["op"] == "rope":
        n = case["tokens"] * case["heads"] * case["dim"]
        ways = 2 if case["backward"] else 1
        return {"bytes": ways * (2 * n * size + 8 * case["tokens"] * len(_sections(case))), "flops": ways * 3 * n}
    if case["op"] == "logits":
        B, V = case["rows"], case["vocab"]
        return {"bytes": 2 * B * V * size + 8 * B * case["history"] + {"none": 0, "shared": 4 * V, "rows": 4 * B * V}[case["bias"]] + min(case["masks"], B) * V // 8, "flops": 4 * B * V}
    new, total = _lengths(case)
    D, H = case["dim"], case["heads"]
    cell = D * size if case["store"] == "same" else D + 1                  # a key or value row of one head, as held
    if case["op"] == "cache":
        return {"bytes": 2 * H * (sum(new) * (D * size + cell) + (sum(total) * (D * size + cell) if case["read"] else 0)), "flops": 4 * H * D * sum(new)}
    w = case["window"]
    pairs = sum(sum(min(p + 1, w) if w else p + 1 for p in range(t - n, t)) for n, t in zip(new, total))
    keys = sum(min(t, w + n - 1) if w else t for n, t in zip(new, total))
    return {"bytes": 2 * sum(new) * case["q_heads"] * D * size + 2 * keys * H * cell, "flops": 4 * D * case["q_heads"] * pairs}


def exact(case, seed):
    """the operators' definitions in 64 bits, sequence by sequence"""
    s = prepare(case, seed)
    if case["op"] == "rope":
        R = 2 * s["freq"].numel()
        first = torch.arange(0, R, 2, device="cuda") if case["adjacent"] else torch.arange(R // 2, device="cuda")
        second = first + (1 if case["adjacent"] else R // 2)

        def turn(x, sign):
            z = torch.complex(x[..., first].double(), x[..., second].double())
            z = z * torch.polar(torch.ones((), device="cuda", dtype=torch.float64), sign * s["freq"] * s["pos"][s["axis"].long()].t())[:, None]
            y = x.detach().double().clone()
            y[..., first], y[..., second] = z.real.detach(), z.imag.detach()
            return y

        return (turn(s["x"], 1), turn(s["dy"], -1)) if case["backward"] else turn(s["x"], 1)
    if case["op"] == "logits":
        rows = []
        for b in range(case["rows"]):
            n, m, V = int(s["lens"][b]), int(s["prompt"][b]), case["vocab"]
            x = s["logits"][b].double()
            every, later = (torch.bincount(s["tokens"][b, i:n], minlength=V) for i in (0, m))
            r = s["repetition"][b].double()
            x = torch.where((every > 0) & (x > 0), x / r, torch.where(every > 0, x * r, x))
            x = x - later * s["frequency"][b].double() - later.clamp(max=1) * s["presence"][b].double()
            if s["bias"] is not None:
                x = x + (s["bias"] if s["bias"].dim() == 1 else s["bias"][b]).double()
            if s["mask"] is not None and int(s["mask_row"][b]) >= 0:
                word = s["mask"][int(s["mask_row"][b])].long() & 0xffffffff
                bits = (word[:, None] >> torch.arange(32, device="cuda")) & 1
                x[bits.flatten()[:V] == 0] = -math.inf
            rows.append(x)
        return torch.stack(rows)
    new, total = _lengths(case)
    page, grid = case["page"], None

    def two(e):
        return ((e.long() + 1023) << 52).view(torch.float64)

    def held(name):
        """the pool's values in 64 bits"""
        pages, exp = s[name + "_pages"], s[name + "_exp"]
        return pages.double() if exp is None else pages.float().double() * two(exp.long() - 127)[..., None]

    def cells(b, n):
        p = torch.arange(n, device="cuda")
        return s["table"][b, p // page].long(), p % page

    if case["op"] == "cache":
        store = _STORES[case["store"]]
        if store == torch.float8_e4m3fn:                                  # every non-negative code's value, from the format's definition
            c = torch.arange(127, device="cuda")
            grid = torch.where(c < 8, c.double() / 512, (8 + c % 8) * two(c // 8 - 10))
        pools = []
        for name in ("k", "v"):
            x = s[name].double()
            if store is not None:
                big = x.abs().amax(-1, keepdim=True)
                e = torch.ceil(torch.log2(big / _LARGEST[store])).clamp(min=-100)
                e = e + (big > _LARGEST[store] * two(e)).double()
                e = e - ((big <= _LARGEST[store] * two(e - 1)) & (e > -100)).double()
                y = x / two(e)
                if grid is None:
                    y = y.round()
                else:
                    a = y.abs()
                    hi = torch.searchsorted(grid, a).clamp(max=126)
                    lo = (hi - 1).clamp(min=0)
                    up, down = grid[hi] - a, a - grid[lo]
                    y = torch.where((down < up) | ((down == up) & (lo % 2 == 0)), grid[lo], grid[hi]) * y.sign()
                x = y * two(e)
            pool, at = held(name), 0
            for b, (n, t) in enumerate(zip(new, total)):
                pg, row = cells(b, t)
                pool[pg[t - n:], :, row[t - n:]] = x[at:at + n]
                at += n
            pools.append(pool)
        if not case["read"]:
            return tuple(pools)
        return tuple(torch.cat([p[cells(b, t)[0], :, cells(b, t)[1]] for b, t in enumerate(total)]) for p in pools)
    k, v, outs, at = held("k"), held("v"), [], 0
    G = case["q_heads"] // case["heads"]
    for b, (n, t) in enumerate(zip(new, total)):
        pg, row = cells(b, t)
        keys, values = k[pg, :, row].repeat_interleave(G, 1), v[pg, :, row].repeat_interleave(G, 1)
        d = torch.arange(t - n, t, device="cuda")[:, None] - torch.arange(t, device="cuda")[None]
        hidden = (d < 0) | (d >= case["window"]) if case["window"] else d < 0
        z = torch.bmm(s["q"][at:at + n].double().transpose(0, 1).contiguous(), keys.permute(1, 2, 0).contiguous()) / math.sqrt(case["dim"])
        outs.append(torch.bmm(torch.softmax(z.masked_fill_(hidden, -math.inf), -1), values.transpose(0, 1).contiguous()).transpose(0, 1))
        at += n
    return torch.cat(outs)
