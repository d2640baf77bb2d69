"""The 8-bit operators as a decoder layer uses them: a prompt pass that fills the cache and single-token steps over it.

  h, x8 = rmsnorm_e4m3(...)  ->  linear_e4m3 (QKV)  ->  q/k-norm + RoPE in place  ->  kv8_append_  ->  sdpa_kv8
  -> linear_w8 (o_proj)  ->  rmsnorm_e4m3 with the residual  ->  linear_e4m3 (gate | up)  ->  silu(gate) * up  ->  linear_w8

Every stage is compared with 64 bits on the very inputs that the stage before gave it on the GPU, so that each tolerance is
its own operator's; and the captured step has to give the same bits as the eager one.
"""

from __future__ import annotations

import math

import pytest
import torch

from tests.test_gpu_serving8 import E4M3, _append_ref, _attend_check, _check_norm, _gen, _linear_check, _norm_ref, _same_codes, _to

pytestmark = pytest.mark.gpu

HIDDEN, HQ, HKV, D, INNER, PAGE = 256, 8, 2, 128, 512, 32


@pytest.fixture(scope="module")
def ops(libemk):
    from deplodock_b200 import ops as _ops

    assert torch.cuda.is_available()
    return _ops


def _weights(seed):
    from oracle.inputs import quantize_e4m3_per_channel

    g = _gen(seed)
    w = {name: quantize_e4m3_per_channel(0.06 * torch.randn(*shape, generator=g))
         for name, shape in dict(qkv=((HQ + 2 * HKV) * D, HIDDEN), o=(HIDDEN, HQ * D), gate_up=(2 * INNER, HIDDEN), down=(HIDDEN, INNER)).items()}
    for name, n in dict(n1=HIDDEN, n2=HIDDEN, qn=D, kn=D).items():
        w[name] = (1 + 0.1 * torch.randn(n, generator=g)).bfloat16()
    return {k: tuple(t.cuda() for t in v) if isinstance(v, tuple) else v.cuda() for k, v in w.items()}


def _layer(ops, w, x, residual, tables, cache, table, ctx, cu, lens, B, Sq, log=None):
    """One layer over ``x [T, HIDDEN]``; keeps what each stage got and gave in ``log``."""
    note = (lambda **kw: log.update({k: tuple(t.clone() for t in v) if isinstance(v, tuple) else v.clone() for k, v in kw.items()})) if log is not None else (lambda **kw: None)
    T = x.shape[0]
    n1 = ops.rmsnorm_e4m3(x, w["n1"], residual=residual)
    note(x=x, residual=residual, n1=n1)
    qkv = ops.linear_e4m3(n1[0], n1[1], *w["qkv"])
    note(qkv_raw=qkv)
    ops.qknorm_rope_(qkv, w["qn"], w["kn"], tables[0], tables[1], T, HQ, HKV)
    heads = qkv.view(T, HQ + 2 * HKV, D)
    note(qkv=heads)
    ops.kv8_append_(cache, heads[:, HQ:HQ + HKV], heads[:, HQ + HKV:], table, ctx, cu)
    o = ops.sdpa_kv8(heads.view(B, Sq, HQ + 2 * HKV, D)[:, :, :HQ], cache, table, lens)
    note(attn=o)
    y = ops.linear_w8(o.view(T, HQ * D), *w["o"])
    n2 = ops.rmsnorm_e4m3(y, w["n2"], residual=n1[2])
    note(y=y, n2=n2)
    gu = ops.linear_e4m3(n2[0], n2[1], *w["gate_up"])
    note(gate_up=gu)
    act = ops.elementwise("silu_multiply", gu[:, :INNER].contiguous(), gu[:, INNER:].contiguous())
    return ops.linear_w8(act, *w["down"]), n2[2]


def _rope(positions):
    from deplodock_b200.model import rope_tables

    cos, sin = rope_tables(512, D, 1e6, "cuda")
    return cos[positions].contiguous(), sin[positions].contiguous()


def test_prompt_then_single_token_steps(ops):
    B, Sq0, steps = 3, 5, 30
    w = _weights(1)
    g = _gen(2)
    max_pages = 3
    cache = ops.kv8_cache(B * max_pages + 1, HKV, PAGE, D)
    host = ops.kv8_cache(B * max_pages + 1, HKV, PAGE, D, device="cpu")
    table = torch.randperm(B * max_pages + 1, generator=g)[:B * max_pages].view(B, max_pages).int()
    td = table.cuda()
    at = 0
    for step in range(steps):
        Sq = Sq0 if step == 0 else 1
        T = B * Sq
        x, r = (torch.randn(T, HIDDEN, generator=g).bfloat16() for _ in "xr")
        ctx = torch.full((B,), at, dtype=torch.int32)
        cu = torch.arange(0, T + 1, Sq, dtype=torch.int32)
        pos = (at + torch.arange(Sq)).repeat(B)
        log = {}
        out, hidden = _layer(ops, w, x.cuda(), r.cuda(), _rope(pos.cuda()), cache, td, ctx.cuda(), cu.cuda(), (ctx + Sq).cuda(), B, Sq, log)
        ops.device_status()
        assert torch.isfinite(out.float()).all() and torch.equal(hidden, log["n2"][2])
        at += Sq
        heads = log["qkv"].cpu()
        _append_ref(host.k, host.k_scale, heads[:, HQ:HQ + HKV], table, ctx.tolist(), cu.tolist())
        _append_ref(host.v, host.v_scale, heads[:, HQ + HKV:], table, ctx.tolist(), cu.tolist())
        if step not in (0, 1, 26, 27, 28, steps - 1):  # the prompt, the first step, the steps over a page's end, the last
            continue
        cpu = {k: tuple(t.cpu() for t in v) if isinstance(v, tuple) else v.cpu() for k, v in log.items()}
        _check_norm(cpu["n1"], _norm_ref(cpu["x"], w["n1"].cpu(), 1e-6, cpu["residual"]), terms=HIDDEN)
        _linear_check(cpu["qkv_raw"], cpu["n1"][0], cpu["n1"][1], *(t.cpu() for t in w["qkv"]))
        assert torch.equal(cache.k_scale.cpu(), host.k_scale) and torch.equal(cache.v_scale.cpu(), host.v_scale)
        assert _same_codes(cache.k, host.k) and _same_codes(cache.v, host.v)
        _attend_check(ops, cpu["attn"], heads.view(B, Sq, -1, D)[:, :, :HQ], host, table, [at] * B, 1 / math.sqrt(D))
        _check_norm(cpu["n2"], _norm_ref(cpu["y"], w["n2"].cpu(), 1e-6, cpu["n1"][2]), terms=HIDDEN)
        _linear_check(cpu["gate_up"], cpu["n2"][0], cpu["n2"][1], *(t.cpu() for t in w["gate_up"]))


def test_captured_step_gives_the_eager_bits_with_padding_sequences(ops):
    """A batch of four slots of which two hold no sequence (no new token, length 0): their rows come out as zeros, and the
    step's graph, replayed as sequences come and go, gives what the eager step gives."""
    B, max_pages = 4, 2
    w = _weights(3)
    g = _gen(4)
    caches = [ops.kv8_cache(B * max_pages, HKV, PAGE, D) for _ in range(2)]
    table = torch.randperm(B * max_pages, generator=g).view(B, max_pages).int().cuda()
    x, r = (torch.empty(B, HIDDEN, dtype=torch.bfloat16, device="cuda") for _ in "xr")
    ctx, lens = (torch.zeros(B, dtype=torch.int32, device="cuda") for _ in "cl")
    cu = torch.zeros(B + 1, dtype=torch.int32, device="cuda")
    cos, sin = (torch.empty(B, D, dtype=torch.bfloat16, device="cuda") for _ in "cs")
    state = [0] * B

    def load(active):
        x.copy_(torch.randn(B, HIDDEN, generator=g).bfloat16())
        r.copy_(torch.randn(B, HIDDEN, generator=g).bfloat16())
        ctx.copy_(torch.tensor(state, dtype=torch.int32))
        new = torch.tensor([1 if b in active else 0 for b in range(B)], dtype=torch.int32)
        # rows of the step are by slot: an empty slot's row lies between its neighbours' and belongs to nobody's range, so
        # active slots come first
        cu.copy_(torch.cat([torch.zeros(1, dtype=torch.int32), new.cumsum(0).int()]))
        lens.copy_(torch.tensor([state[b] + 1 if b in active else 0 for b in range(B)], dtype=torch.int32))
        c, s = _rope(torch.tensor(state).cuda())
        cos.copy_(c)
        sin.copy_(s)
        for b in active:
            state[b] += 1

    def step(cache):
        log = {}
        out, hidden = _layer(ops, w, x, r, (cos, sin), cache, table, ctx, cu, lens, B, 1, None)
        return out, hidden

    warm = ops.kv8_cache(B * max_pages, HKV, PAGE, D)
    load([0, 1])
    state[:] = [0] * B
    step(warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(caches[0])
    for c in caches:
        for t in c:
            t.view(torch.uint8).zero_()
    for i in range(40):
        active = [0, 1] if i % 3 else [0, 1, 2]
        load(active)
        graph.replay()
        eager = step(caches[1])
        assert torch.equal(captured[0], eager[0]) and torch.equal(captured[1], eager[1])
    ops.device_status()
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(*caches))
    assert state[0] == 40 and state[2] == 14 and state[3] == 0
    o = ops.sdpa_kv8(torch.randn(B, 1, HQ, D, device="cuda").bfloat16(), caches[0], table, lens)
    assert (o[3] == 0).all() and (o[0] != 0).any()


def test_two_streams_at_once(ops):
    """Attention and linear layers of two requests on two streams, each with its own buffers, give what they give alone."""
    jobs = []
    for seed, lens in ((5, [3000, 10]), (6, [1, 2500, 700])):
        g = _gen(seed)
        B, max_pages = len(lens), 1 << 11
        cache = ops.kv8_cache(B * 100, HKV, PAGE, D)
        table = torch.zeros(B, max_pages, dtype=torch.int32, device="cuda")
        table[:, :100] = torch.arange(B * 100, dtype=torch.int32).view(B, 100).cuda()
        total = sum(lens)
        kv = torch.randn(total, 2 * HKV, D, generator=g).bfloat16().cuda()
        cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32).cuda()
        ops.kv8_append_(cache, kv[:, :HKV], kv[:, HKV:], table, torch.zeros(B, dtype=torch.int32).cuda(), cu)
        q = torch.randn(B, 1, HQ, D, generator=g).bfloat16().cuda()
        jobs.append((q, cache, table, torch.tensor(lens, dtype=torch.int32).cuda()))
    alone = [ops.sdpa_kv8(*j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    outs = [[], []]
    for _ in range(20):
        for j, s, o in zip(jobs, streams, outs):
            with torch.cuda.stream(s):
                o.append(ops.sdpa_kv8(*j))
    torch.cuda.synchronize()
    ops.device_status()
    for a, o in zip(alone, outs):
        assert all(torch.equal(a, x) for x in o)
