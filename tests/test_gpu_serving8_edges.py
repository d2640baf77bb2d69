"""Calls of the 8-bit serving operators that their documentation allows at its edges: pages that sequences share, an output
over the queries, tensors past 2^31 elements, two captured graphs in flight at once."""

import math

import pytest
import torch

from tests.test_gpu_serving8 import E4M3, ROOM, _attend_check, _check_norm, _codes, _gen, _linear_check, _norm_ref, _random_cache, _to, ops  # noqa: F401

pytestmark = pytest.mark.gpu


def _table(rows, room, page):
    t = torch.tensor(rows, dtype=torch.int32)
    return t if room == "tight" else torch.cat([t, torch.full((len(rows), room // page - t.shape[1]), -1, dtype=torch.int32)], 1)


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("Sq,Hq,D", [(1, 8, 128), (3, 8, 64), (3, 16, 128)])
def test_pages_may_be_shared_and_the_output_may_be_the_query(ops, room, Sq, Hq, D):  # noqa: F811
    page, Hkv, pages = 64, 2, 12
    rows = [[3, 7, 1, 9, 4, 0], [3, 7, 1, 2, 2, 2], [5, 5, 5, 5, 5, 5], [3, 0, 0, 0, 0, 0]]
    lens = [380, 301, 384, 64]
    cache = _random_cache(ops, pages, Hkv, page, D, 5)
    q = torch.randn(4, Sq, Hq, D, generator=_gen(6)).bfloat16()
    table = _table(rows, room, page).cuda()
    dev, lens_t, qd = _to(cache, "cuda"), torch.tensor(lens, dtype=torch.int32).cuda(), q.cuda()
    got = ops.sdpa_kv8(qd, dev, table, lens_t)
    _attend_check(ops, got, q, cache, torch.tensor(rows), lens, 1 / math.sqrt(D))
    over = qd.clone()
    assert ops.sdpa_kv8(over, dev, table, lens_t, out=over) is over
    assert torch.equal(over, got)
    ops.device_status()


def test_rmsnorm_e4m3_past_2_31_elements(ops):  # noqa: F811
    rows, cols = 140001, 16384
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    w = torch.randn(cols, generator=_gen(1)).bfloat16()
    tail = torch.randn(3, cols, generator=_gen(2)).bfloat16()
    x[-3:] = tail.cuda()
    q, scale, hidden = ops.rmsnorm_e4m3(x, w.cuda(), 1e-6, x, hidden_out=x)
    ops.device_status()
    doubled = (2 * tail.float()).bfloat16()  # exact
    _check_norm((q[-3:], scale[-3:], hidden[-3:]), _norm_ref(doubled, w, 1e-6, None), cols)
    # zeros, with the sign of their weight
    assert all(int((part.view(torch.uint8) & 0x7f).count_nonzero()) == 0 for part in q[:-3].split(10000)) and (scale[:-3] == scale[0]).all()


def test_linear_e4m3_past_2_31_outputs(ops):  # noqa: F811
    M, N, K = 270001, 8192, 16
    g = _gen(3)
    x, w = _codes(g, M, K), _codes(g, N, K)
    xs, ws = torch.rand(M, generator=g) + 0.5, torch.rand(N, generator=g) + 0.5
    y = ops.linear_e4m3(x.cuda(), xs.cuda(), w.cuda(), ws.cuda())
    ops.device_status()
    for part in (slice(0, 300), slice(131000, 131300), slice(M - 300, M)):
        _linear_check(y[part], x[part], xs[part], w, ws)


@pytest.mark.parametrize("room", ROOM)
def test_two_captured_graphs_in_flight_at_once(ops, room):  # noqa: F811
    page, Hkv, D, B = 64, 2, 128, 40
    states = []
    for seed in (1, 2):
        g = _gen(seed)
        lens = torch.randint(0, 700, (B,), generator=g)
        rows = torch.randperm(B * 11, generator=g).view(B, 11).tolist()
        cache = _to(_random_cache(ops, B * 11, Hkv, page, D, seed), "cuda")
        args = (torch.randn(B, 1, 8, D, generator=g).bfloat16().cuda(), cache, _table(rows, room, page).cuda(), lens.int().cuda())
        want = ops.sdpa_kv8(*args)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.sdpa_kv8(*args)
        states.append((graph, out, want, torch.cuda.Stream(), args))  # (a graph does not keep its inputs alive)
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, out, _, stream, _ in states:
            with torch.cuda.stream(stream):
                out.zero_()
                graph.replay()
        torch.cuda.synchronize()
        for _, out, want, *_ in states:
            assert torch.equal(out, want)
    ops.device_status()


@pytest.mark.parametrize("room", ROOM + ["short"])
@pytest.mark.parametrize("Sq,G,D", [(2, 1, 128), (4, 4, 64), (5, 2, 128), (4, 1, 64), (20, 1, 128)])
def test_nan_tokens_reach_only_the_queries_that_see_them(ops, room, Sq, G, D):  # noqa: F811
    """A draft token's NaN values spoil its channel for the queries at or behind it, and leave those before it alone."""
    page, Hkv = 16, 2
    lens = [70, 33, 16, Sq, 64, 3] * (200 if room == "short" else 1)
    B, max_pages = len(lens), 5
    g = _gen(Sq + D)
    cache = _random_cache(ops, B * max_pages, Hkv, page, D, 8)
    rows = torch.randperm(B * max_pages, generator=g).view(B, max_pages).tolist()
    bad = torch.zeros(B, Hkv, max_pages * page, D, dtype=torch.bool)  # NaN values, by token
    for b, n in enumerate(lens):
        for back, head, channels in ((1, 0, [0, 9]), (2, 0, [5, D - 1]), (1, 1, [D // 2]), (Sq, 1, [2, 3])):
            if back <= n:
                t = n - back
                bad[b, head, t, channels] = True
                cache.v.view(torch.uint8)[rows[b][t // page], head, t % page, channels] = 0x7f if back & 1 else 0xff
                cache.k.view(torch.uint8)[rows[b][(n - 1) // page], head, (n - 1) % page, 7] = 0x7f  # and the last key
    q = torch.randn(B, Sq, G * Hkv, D, generator=g).bfloat16()
    lens_t = torch.tensor(lens, dtype=torch.int32)
    table = _table(rows, "tight" if room == "short" else room, page).cuda()
    got = ops.sdpa_kv8(q.cuda(), _to(cache, "cuda"), table, lens_t.cuda())
    ops.device_status()
    got = got.cpu()
    for b, n in enumerate(lens[:6]):
        for i in range(Sq):
            m = n - Sq + i + 1
            want = bad[b, :, :max(m, 0)].any(1)  # [Hkv, D]
            if m == n:
                want = torch.ones_like(want)  # the last token's key is NaN
            assert torch.equal(torch.isnan(got[b, i].float()).view(Hkv, G, D), want[:, None].expand(-1, G, -1)), (b, i)
    # the finite values are right: the same cache with zeros for the NaN values gives them
    clean = type(cache)(*(x.clone() for x in cache))
    for codes in (clean.k.view(torch.uint8), clean.v.view(torch.uint8)):
        codes[(codes & 0x7f) == 0x7f] = 0
    ref = ops.sdpa_kv8(q.cuda(), _to(clean, "cuda"), table, lens_t.cuda()).cpu()
    # (to the tolerance, not to the bit: when one row's maximum moves, the others' roundings move with it)
    for some in (ref, torch.where(torch.isnan(got), ref, got)):
        _attend_check(ops, some[:6], q[:6], clean, torch.tensor(rows[:6]), lens[:6], 1 / math.sqrt(D))


def test_a_tensor_left_on_the_cpu_is_refused_wherever_it_stands(ops):  # noqa: F811
    cache = ops.kv8_cache(3, 2, 16, 64)
    i32 = dict(dtype=torch.int32, device="cuda")
    table, lens, cu = torch.zeros(1, 2, **i32), torch.ones(1, **i32), torch.tensor([0, 1], **i32)
    k = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device="cuda")
    q = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16, device="cuda")
    x = torch.zeros(2, 16, device="cuda")
    x8, w8, s2, s8 = x.to(E4M3), torch.zeros(8, 16, device="cuda").to(E4M3), torch.ones(2, device="cuda"), torch.ones(8, device="cuda")
    calls = [(ops.sdpa_kv8, [q, cache, table, lens]), (ops.kv8_append_, [cache, k, k, table, lens, cu]),
             (ops.linear_e4m3, [x8, s2, w8, s8]), (ops.rmsnorm_e4m3, [x, torch.ones(16, device="cuda"), 1e-6, x])]
    for f, args in calls:
        f(*args)
        for i, a in enumerate(args):
            for there in [a.cpu()] if torch.is_tensor(a) else [a._replace(**{n: getattr(a, n).cpu()}) for n in a._fields] if isinstance(a, tuple) else []:
                with pytest.raises(ValueError):
                    f(*args[:i], there, *args[i + 1:])
    ops.device_status()
