"""The operators of the 8-bit serving step, measured: RMSNorm with the residual's addition and an e4m3 output, the e4m3
linear layer that consumes it, appending keys and values to a paged e4m3 cache, and attention over that cache.

``listed()`` and ``draw()`` give the cases, ``prepare()`` their inputs, ``run()`` one pass (the plain torch form, or with
``own`` the framework's operators), ``exact()`` the results in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
AMAX_FLOOR = 2.0 ** -100  # rows of zeros get this maximum, so that no scale is zero
SCALE_EXP = (-64, 120)    # range of the cache scales' exponents


def listed():
    return [
        # one decode step of eight sequences: the smallest call, its latency counts
        dict(name="norm decode", op="norm", rows=8, cols=1024, dtype="bf16", residual=True),
        # the 64 x 512 token forward of the benchmark
        dict(name="norm prompt", op="norm", rows=32768, cols=1024, dtype="bf16", residual=True),
        # fp32 rows of an odd length, no residual: nothing is aligned
        dict(name="norm odd f32", op="norm", rows=4099, cols=1001, dtype="f32", residual=False),
        # a single token through the layer of the linear benchmark
        dict(name="linear token", op="linear", M=1, N=6144, K=2048),
        # a decode batch through a QKV projection, rows that fill no tile
        dict(name="linear batch", op="linear", M=67, N=4096, K=1024),
        # the linear benchmark's shape
        dict(name="linear prompt", op="linear", M=4096, N=6144, K=2048),
        # one new token for each of 64 sequences
        dict(name="append decode", op="append", B=64, new_min=1, new_max=1, ctx_max=2000, Hkv=8, D=128, page=64),
        # prompts of mixed lengths behind cached ones
        dict(name="append prompts", op="append", B=24, new_min=0, new_max=2048, ctx_max=700, Hkv=8, D=128, page=64),
        # one sequence, one token: latency
        dict(name="attend token", op="attend", B=1, Sq=1, len_min=1500, len_max=1500, Hq=16, Hkv=8, D=128, page=64),
        # a decode batch of mixed lengths, one of them possibly empty
        dict(name="attend batch", op="attend", B=64, Sq=1, len_min=0, len_max=8192, Hq=16, Hkv=8, D=128, page=64),
        # few sequences with a long past: the work has to be split along it
        dict(name="attend long", op="attend", B=3, Sq=1, len_min=100001, len_max=131071, Hq=32, Hkv=8, D=128, page=128),
        # four draft tokens a sequence, small heads, small pages
        dict(name="attend drafts", op="attend", B=17, Sq=4, len_min=1, len_max=4097, Hq=32, Hkv=8, D=64, page=16),
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm; 0 is drawn now and then where lo is 0."""
    if lo == 0:
        return 0 if rng.random() < 0.1 else _log_int(rng, 1, hi)
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "linear", "append", "attend", "attend"])
    if op == "norm":
        cols = _log_int(rng, 64, 8192)
        if rng.random() < 0.7:
            cols = max(64, cols // 64 * 64)
        return dict(op="norm", rows=_log_int(rng, 1, 33_000_000 // cols), cols=cols, dtype=rng.choice(["bf16", "bf16", "f32"]),
                    residual=rng.random() < 0.7)
    if op == "linear":
        N, K = 8 * _log_int(rng, 16, 768), 16 * _log_int(rng, 8, 256)
        return dict(op="linear", M=_log_int(rng, 1, 4096), N=N, K=K)
    Hkv, D, page = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 128, 256])
    if op == "append":
        B = _log_int(rng, 1, 96)
        new_max = _log_int(rng, 1, max(1, 32768 // B))
        return dict(op="append", B=B, new_min=rng.choice([0, 1, new_max]) if new_max > 1 else 1, new_max=new_max,
                    ctx_max=_log_int(rng, 0, 3000), Hkv=Hkv, D=D, page=page)
    B, group, Sq = _log_int(rng, 1, 96), rng.choice([1, 2, 3, 4, 6, 8, 16]), rng.choice([1, 1, 1, 2, 3, 5, 8])
    # as much work as the longest listed one at most
    len_max = _log_int(rng, 1, max(1, min(131071, 8 * 393213 * 4 // (B * Hkv * max(4, group * Sq)))))
    return dict(op="attend", B=B, Sq=Sq, len_min=rng.choice([0, 1, len_max]), len_max=len_max, Hq=Hkv * group, Hkv=Hkv, D=D,
                page=page)


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _host_lens(seed, B, lo, hi):
    g = torch.Generator().manual_seed(seed * 7919 + 17)
    return torch.randint(lo, hi + 1, (B,), generator=g)


def _page_table(seed, B, max_pages):
    """Pages of a pool that has a quarter more than is used, in no order."""
    g = torch.Generator(device=DEV).manual_seed(seed + 5)
    pool = B * max_pages + max(1, B * max_pages // 4)
    return torch.randperm(pool, generator=g, device=DEV)[:B * max_pages].view(B, max_pages).to(torch.int32), pool


def _random_cache(g, pool, Hkv, page, D):
    """A cache as appending leaves it: normal values whose size differs by page and head, at power-of-two scales."""
    sigma_exp = torch.randint(-2, 3, (pool, Hkv), generator=g, device=DEV)
    codes = torch.empty(pool, Hkv, page, D, dtype=E4M3, device=DEV)
    step = max(1, (1 << 26) // (Hkv * page * D))
    for at in range(0, pool, step):  # in pieces: the values before rounding need no room for the whole cache
        n = min(step, pool - at)
        codes[at:at + n] = (torch.randn(n, Hkv, page, D, generator=g, device=DEV) * 64.0).clamp(-E4M3_MAX, E4M3_MAX).to(E4M3)
    return codes, torch.ldexp(torch.ones(pool, Hkv, device=DEV), sigma_exp - 6)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    op = case["op"]
    s = dict(op=op)
    if op == "norm":
        t = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        rows, cols = case["rows"], case["cols"]
        # a few channels carry most of a residual stream's size
        gain = torch.exp(1.2 * torch.randn(cols, generator=g, device=DEV))
        s["x"] = torch.randn(rows, cols, generator=g, device=DEV).to(t)
        s["residual"] = (torch.randn(rows, cols, generator=g, device=DEV) * gain).to(t) if case["residual"] else None
        s["weight"] = (1.0 + 0.2 * torch.randn(cols, generator=g, device=DEV)).to(t)
        s["eps"] = 1e-6
    elif op == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        x, w = torch.randn(M, K, generator=g, device=DEV), 0.02 * torch.randn(N, K, generator=g, device=DEV)
        s["x_scale"], s["w_scale"] = x.abs().amax(1) / E4M3_MAX, w.abs().amax(1) / E4M3_MAX
        s["x"], s["w"] = (x / s["x_scale"][:, None]).to(E4M3), (w / s["w_scale"][:, None]).to(E4M3)
    elif op == "append":
        B, Hkv, D, page = case["B"], case["Hkv"], case["D"], case["page"]
        new = _host_lens(seed, B, case["new_min"], case["new_max"])
        new[0] = max(1, int(new[0]))  # a call has a token at least
        ctx = _host_lens(seed + 1, B, 0, case["ctx_max"])
        max_pages = -(-(case["ctx_max"] + case["new_max"]) // page)
        s["table"], pool = _page_table(seed, B, max_pages)
        s["k_codes"], s["k_scale"] = _random_cache(g, pool, Hkv, page, D)
        s["v_codes"], s["v_scale"] = _random_cache(g, pool, Hkv, page, D)
        total = int(new.sum())
        size = torch.exp2(torch.randint(-2, 4, (total, 1, 1), generator=g, device=DEV).float())  # some tokens outgrow their page's scale
        qkv = torch.randn(total, 4 * Hkv, D, generator=g, device=DEV)
        qkv[:, 2 * Hkv:] *= size
        qkv = qkv.to(torch.bfloat16)  # a fused projection [T, Hq + 2 Hkv, D]: keys and values are strided views of it
        s["k"], s["v"] = qkv[:, 2 * Hkv:3 * Hkv], qkv[:, 3 * Hkv:]
        s["ctx"] = ctx.to(device=DEV, dtype=torch.int32)
        s["cu"] = torch.cat([torch.zeros(1, dtype=torch.int64), new.cumsum(0)]).to(device=DEV, dtype=torch.int32)
    else:
        B, Sq, Hq, Hkv, D, page = (case[k] for k in ("B", "Sq", "Hq", "Hkv", "D", "page"))
        lens = _host_lens(seed, B, case["len_min"], case["len_max"])
        max_pages = -(-case["len_max"] // page)
        s["table"], pool = _page_table(seed, B, max_pages)
        s["k_codes"], s["k_scale"] = _random_cache(g, pool, Hkv, page, D)
        s["v_codes"], s["v_scale"] = _random_cache(g, pool, Hkv, page, D)
        s["q"] = torch.randn(B, Sq, Hq, D, generator=g, device=DEV).to(torch.bfloat16)
        s["lens"] = lens.to(device=DEV, dtype=torch.int32)
        s["scale"] = 1.0 / math.sqrt(D)
    return s


# ---------------------------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------------------------
def _norm_plain(s):
    x, residual = s["x"], s["residual"]
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    f = h.float()
    y = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + s["eps"]) * s["weight"].float()
    scale = y.abs().amax(-1).clamp_min(AMAX_FLOOR) / E4M3_MAX
    q = (y / scale[:, None]).to(E4M3)
    return (q, scale) if residual is None else (q, scale, h)


def _linear_plain(s):
    y = (s["x"].float() @ s["w"].float().t()) * s["x_scale"][:, None] * s["w_scale"]
    return y.to(torch.bfloat16)


def _power_of_two_scale(amax):
    """The smallest 2^e with amax <= 448 * 2^e, e within SCALE_EXP (448 = 0.875 * 2^9)."""
    m, e = torch.frexp(amax)
    e = torch.where(m <= 0.875, e - 9, e - 8)
    e = torch.where(amax > 0, e, SCALE_EXP[0]).clamp(*SCALE_EXP)
    return torch.ldexp(torch.ones_like(amax), e)


def _append_one(x, codes, scale, pages, slots, first_page, kept):
    """New rows ``x [T, Hkv, D]`` into pages ``pages [T]`` at ``slots [T]``; ``kept [B]``: tokens that stay in each
    sequence's first touched page (0: none, or the sequence appends nothing)."""
    P, Hkv, page, D = codes.shape
    x = x.float()
    finite = torch.isfinite(x)
    amax = torch.zeros(P, Hkv, device=x.device).index_reduce_(0, pages, torch.where(finite, x.abs(), 0.0).amax(-1), "amax")
    mine = _power_of_two_scale(amax)
    old = scale[first_page]
    grown = torch.where(kept[:, None] > 0, torch.maximum(old, mine[first_page]), old)
    # the codes that stay, rounded again where their page's scale grew
    held = codes[first_page]
    stay = (torch.arange(page, device=x.device) < kept[:, None])[:, None, :, None]
    moved = (held.float() * (old / grown)[:, :, None, None]).to(E4M3)
    codes.view(torch.uint8)[first_page] = torch.where(stay, moved.view(torch.uint8), held.view(torch.uint8))
    mine[first_page] = torch.where(kept[:, None] > 0, grown, mine[first_page])
    scale[pages] = mine[pages]
    value = torch.where(finite, x / mine[pages][:, :, None], torch.nan).to(E4M3)
    codes.view(torch.uint8)[pages, :, slots] = value.view(torch.uint8)


def _append_plain(s):
    cu, ctx, table, page = s["cu"].long(), s["ctx"].long(), s["table"].long(), s["k_codes"].shape[2]
    t = torch.arange(s["k"].shape[0], device=cu.device)
    b = torch.searchsorted(cu, t, right=True) - 1
    pos = ctx[b] + t - cu[b]
    pages, slots = table[b, pos // page], pos % page
    kept = torch.where(cu[1:] > cu[:-1], ctx % page, 0)
    first_page = table.gather(1, (ctx // page).clamp_max(table.shape[1] - 1)[:, None])[:, 0]
    _append_one(s["k"], s["k_codes"], s["k_scale"], pages, slots, first_page, kept)
    _append_one(s["v"], s["v_codes"], s["v_scale"], pages, slots, first_page, kept)
    return s["k_codes"], s["k_scale"], s["v_codes"], s["v_scale"]


def _dense(codes, scale, table):
    """The pages of ``table [B, n]`` as values ``[B, Hkv, n * page, D]``."""
    B, n = table.shape
    _, Hkv, page, D = codes.shape
    x = codes.view(torch.uint8)[table].view(E4M3).to(scale.dtype) * scale[table][..., None, None]
    return x.transpose(1, 2).reshape(B, Hkv, n * page, D)


def _attend(q, k, v, lens, scale):
    """``q [B, Sq, Hq, D]`` over ``k, v [B, Hkv, L, D]`` of which ``lens [B]`` tokens count, in the type of ``k``."""
    B, Sq, Hq, D = q.shape
    Hkv, L = k.shape[1], k.shape[2]
    at = torch.arange(L, device=q.device)
    last = lens[:, None] - Sq + torch.arange(Sq, device=q.device)              # position of every query
    seen = (at <= last[:, :, None])[:, None, None]                             # [B, 1, 1, Sq, L]
    qg = q.to(k.dtype).view(B, Sq, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4)   # [B, Hkv, G, Sq, D]
    scores = (qg.reshape(B, Hkv, -1, D) @ k.transpose(2, 3)).view(B, Hkv, Hq // Hkv, Sq, L) * scale
    scores = scores.masked_fill(~seen, -torch.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(top), 0.0, top))
    total = p.sum(-1, keepdim=True)
    v = torch.where((at < lens[:, None])[:, None, :, None], v, 0.0)
    o = (p.view(B, Hkv, -1, L) @ v).view(B, Hkv, Hq // Hkv, Sq, D) / torch.where(total > 0, total, 1.0)
    return o.permute(0, 3, 1, 2, 4).reshape(B, Sq, Hq, D)


def _attend_plain(s):
    table = s["table"].long()
    k, v = _dense(s["k_codes"], s["k_scale"], table), _dense(s["v_codes"], s["v_scale"], table)
    return _attend(s["q"], k, v, s["lens"].long(), s["scale"]).to(s["q"].dtype)


def run(s):
    if own:
        from deplodock_b200 import ops

        if s["op"] == "norm":
            return ops.rmsnorm_e4m3(s["x"], s["weight"], s["eps"], residual=s["residual"])
        if s["op"] == "linear":
            return ops.linear_e4m3(s["x"], s["x_scale"], s["w"], s["w_scale"])
        cache = ops.KV8Cache(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"])
        if s["op"] == "append":
            ops.kv8_append_(cache, s["k"], s["v"], s["table"], s["ctx"], s["cu"])
            return s["k_codes"], s["k_scale"], s["v_codes"], s["v_scale"]
        return ops.sdpa_kv8(s["q"], cache, s["table"], s["lens"], scale=s["scale"])
    return {"norm": _norm_plain, "linear": _linear_plain, "append": _append_plain, "attend": _attend_plain}[s["op"]](s)


def _mean_len(lo, hi):
    return 0.5 * (lo + hi)


def work(case):
    op = case["op"]
    if op == "norm":
        n, t = case["rows"] * case["cols"], 2 if case["dtype"] == "bf16" else 4
        return {"bytes": n * (t * (3 if case["residual"] else 1) + 1) + case["rows"] * 4 + case["cols"] * t, "flops": 6.0 * n}
    if op == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": M * K + N * K + 2 * M * N + 4 * (M + N), "flops": 2.0 * M * N * K}
    if op == "append":
        tokens = case["B"] * _mean_len(case["new_min"], case["new_max"])
        return {"bytes": tokens * case["Hkv"] * case["D"] * 2 * (2 + 1), "flops": tokens * case["Hkv"] * case["D"] * 2 * 3.0}
    tokens = case["B"] * _mean_len(case["len_min"], case["len_max"])
    qo = case["B"] * case["Sq"] * case["Hq"] * case["D"] * 2 * 2
    pages = tokens / case["page"]
    return {"bytes": tokens * case["Hkv"] * case["D"] * 2 + qo + pages * (4 + 8 * case["Hkv"]),
            "flops": 4.0 * tokens * case["Hq"] * case["D"] * case["Sq"]}


# ---------------------------------------------------------------------------------------------------------------
# in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def _exact_norm(s):
    out = []
    for at in range(0, s["x"].shape[0], 4096):
        h = s["x"][at:at + 4096].double()
        if s["residual"] is not None:
            h = (h + s["residual"][at:at + 4096].double()).to(s["x"].dtype).double()  # the stored sum is what is normalised
        y = h / torch.sqrt(h.square().sum(1, keepdim=True) / h.shape[1] + s["eps"]) * s["weight"].double()
        scale = y.abs().max(1).values.clamp_min(AMAX_FLOOR) / E4M3_MAX
        out.append((y / scale[:, None], scale) + (() if s["residual"] is None else (h,)))
    return tuple(torch.cat(c) for c in zip(*out))


def _exact_linear(s):
    x, w = s["x"].double() * s["x_scale"].double()[:, None], s["w"].double() * s["w_scale"].double()[:, None]
    return torch.einsum("mk,nk->mn", x, w)


def _exact_append(s):
    page = s["k_codes"].shape[2]
    cu, ctx, table = s["cu"].tolist(), s["ctx"].tolist(), s["table"].tolist()
    out = []
    for name in ("k", "v"):
        codes, scale = s[name + "_codes"].double(), s[name + "_scale"].double()
        for b in range(len(ctx)):
            t, pos, end = cu[b], ctx[b], ctx[b] + cu[b + 1] - cu[b]
            while pos < end:  # a page at a time
                n, at, p = min(end - pos, page - pos % page), pos % page, table[b][pos // page]
                new = s[name][t:t + n].double()
                e = torch.ceil(torch.log2(new.abs().amax((0, 2)).clamp_min(2.0 ** -140) / E4M3_MAX)).clamp(*SCALE_EXP)
                to = torch.exp2(e)
                if at > 0:
                    to = torch.maximum(to, scale[p])
                    codes[p, :, :at] = (codes[p, :, :at] * (scale[p] / to)[:, None, None]).to(E4M3).double()
                codes[p, :, at:at + n] = (new / to[None, :, None]).to(E4M3).double().transpose(0, 1)
                scale[p] = to
                t, pos = t + n, pos + n
        out += [codes, scale]
    return tuple(out)


def _exact_attend(s):
    out = []
    for b in range(s["q"].shape[0]):
        n, page = int(s["lens"][b]), s["k_codes"].shape[2]
        Sq, Hq, D = s["q"].shape[1:]
        o = torch.zeros(Sq, Hq, D, dtype=torch.float64, device=DEV)
        at = s["table"][b, :-(-n // page)].long()
        Hkv = s["k_codes"].shape[1]
        for h in range(Hkv):
            k = (s["k_codes"].view(torch.uint8)[at, h].view(E4M3).double() * s["k_scale"][at, h].double()[:, None, None]).reshape(-1, D)[:n]
            v = (s["v_codes"].view(torch.uint8)[at, h].view(E4M3).double() * s["v_scale"][at, h].double()[:, None, None]).reshape(-1, D)[:n]
            mine = slice(h * (Hq // Hkv), (h + 1) * (Hq // Hkv))
            for i in range(Sq):
                m = n - Sq + i + 1
                if m > 0:
                    o[i, mine] = torch.softmax(s["q"][b, i, mine].double() @ k[:m].T * s["scale"], dim=-1) @ v[:m]
        out.append(o)
    return torch.stack(out)


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "linear": _exact_linear, "append": _exact_append, "attend": _exact_attend}[s["op"]](s)
