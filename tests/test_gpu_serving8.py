"""The 8-bit serving operators against plain implementations in 64 bits: RMSNorm with an e4m3 output, appending to the
paged e4m3 key/value cache, attention over it.

Tolerances. A rounding is off by half a step at most: 2^-8 relative for bf16, 2^-11 for fp16 (the attention's
probabilities), 2^-4 for e4m3 (2^-10 absolute below its normal range). fp32 sums of n terms carry n * 2^-24 relative to
the sum of the magnitudes; the tensor core truncates where the FMA pipe rounds, so its sums count 2^-23 a step.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops(libemk):
    from deplodock_b200 import ops as _ops

    assert torch.cuda.is_available()
    return _ops


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------------------------------------------------
# RMSNorm, e4m3 output
# ------------------------------------------------------------------------------------------------------------
def _norm_ref(x, w, eps, residual):
    h = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    f = h.double()
    y = f / torch.sqrt(f.square().mean(-1, keepdim=True) + eps) * w.double()
    return y, y.abs().amax(-1).clamp_min(2.0 ** -100) / 448.0, h


def _check_norm(got, ref, terms):
    y, scale, h = ref
    # the fp32 sum's error halves under the root; six more roundings (quotient, root, two products, scale)
    rel = (0.5 * terms + 6) * 2.0 ** -24
    q, s = got[0].cpu(), got[1].cpu()
    assert q.dtype == E4M3 and s.dtype == torch.float32 and s.shape == y.shape[:-1]
    assert ((s.double() - scale).abs() <= rel * scale).all()
    want = y / scale[..., None]
    err = (q.double() - want).abs()
    # a value next to a rounding border may fall to either side of it: rel of the value on top of the half step
    assert (err <= torch.maximum(want.abs() * 2.0 ** -4, torch.tensor(2.0 ** -10)) + 3 * rel * want.abs()).all()
    if len(got) > 2:
        assert torch.equal(got[2].cpu(), h)


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 7), (3, 64), (8, 1024), (5, 1001), (1300, 250), (1301, 256), (2000, 1024),
                                       (1200, 2056), (37, 4096), (9, 8192), (3, 16392), (2, 20011), (1500, 33)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("with_residual", [False, True])
def test_rmsnorm_e4m3(ops, rows, cols, dtype, with_residual):
    g = _gen(rows * 100003 + cols)
    x = torch.randn(rows, cols, generator=g).to(dtype)
    r = (3 * torch.randn(rows, cols, generator=g)).to(dtype) if with_residual else None
    w = (1 + 0.2 * torch.randn(cols, generator=g)).to(dtype)
    got = ops.rmsnorm_e4m3(x.cuda(), w.cuda(), 1e-6, residual=None if r is None else r.cuda())
    ops.device_status()
    _check_norm(got, _norm_ref(x, w, 1e-6, r), terms=cols)


@pytest.mark.parametrize("cols", [1024, 1023, 20000])
def test_rmsnorm_e4m3_special_rows(ops, cols):
    g = _gen(5)
    x = torch.randn(6, cols, generator=g)
    x[1] = 0.0
    x[2, cols // 2] = float("nan")
    x[3] *= 1e-30
    x[4] *= 1e15
    w = torch.ones(cols)
    q, s = ops.rmsnorm_e4m3(x.cuda(), w.cuda(), 1e-6)
    q, s = q.float().cpu(), s.cpu()
    assert (q[1] == 0).all() and 0 < s[1] < 1e-30
    assert torch.isnan(q[2]).all() and torch.isnan(s[2])
    keep = torch.tensor([0, 3, 4, 5])
    _check_norm((q[keep].to(E4M3), s[keep]), tuple(t[keep] for t in _norm_ref(x, w, 1e-6, None)), terms=cols)


@pytest.mark.parametrize("cols", [512, 513, 20000])
def test_rmsnorm_e4m3_in_place_and_given_outputs(ops, cols):
    g = _gen(6)
    x, r = (torch.randn(2, 11, cols, generator=g).bfloat16() for _ in "xr")
    w = torch.rand(cols, generator=g).bfloat16()
    ref = _norm_ref(x, w, 1e-5, r)
    for alias in ("x", "residual"):
        xc, rc = x.cuda(), r.cuda()
        out = torch.empty(2, 11, cols, dtype=E4M3, device="cuda")
        scale = torch.empty(2, 11, device="cuda")
        got = ops.rmsnorm_e4m3(xc, w.cuda(), 1e-5, residual=rc, out=out, scale_out=scale, hidden_out=xc if alias == "x" else rc)
        assert got[0] is out and got[1] is scale and got[2] is (xc if alias == "x" else rc)
        _check_norm(got, ref, terms=cols)


def test_rmsnorm_e4m3_unaligned_rows_and_empty(ops):
    g = _gen(7)
    flat = torch.randn(1 + 5 * 64, generator=g).bfloat16()
    x = flat.cuda()[1:].view(5, 64)  # 2-byte aligned only
    w = torch.ones(64).bfloat16()
    _check_norm(ops.rmsnorm_e4m3(x, w.cuda()), _norm_ref(flat[1:].view(5, 64), w, 1e-6, None), terms=64)
    q, s = ops.rmsnorm_e4m3(torch.empty(0, 64, device="cuda"), torch.ones(64, device="cuda"))
    assert q.shape == (0, 64) and s.shape == (0,)


def test_rmsnorm_e4m3_refusals(ops):
    x, w = torch.randn(4, 8, device="cuda"), torch.ones(8, device="cuda")
    with pytest.raises(ValueError):
        ops.rmsnorm_e4m3(x, w[:4].contiguous())
    with pytest.raises(ValueError):
        ops.rmsnorm_e4m3(x, w, residual=torch.randn(4, 4, device="cuda"))
    with pytest.raises(ValueError):
        ops.rmsnorm_e4m3(x, w, hidden_out=torch.empty_like(x))
    with pytest.raises(ValueError):
        ops.rmsnorm_e4m3(x.t(), torch.ones(4, device="cuda"))
    with pytest.raises(ValueError):
        ops.rmsnorm_e4m3(x, w.cpu())
    with pytest.raises(ValueError):
        ops.rmsnorm_e4m3(x, w, out=torch.empty(3, 8, dtype=E4M3, device="cuda"))
    with pytest.raises(TypeError):
        ops.rmsnorm_e4m3(x.half(), w.half())


# ------------------------------------------------------------------------------------------------------------
# e4m3 linear
# ------------------------------------------------------------------------------------------------------------
def _codes(g, rows, cols):
    return (torch.randn(rows, cols, generator=g) * 60).clamp(-448, 448).to(E4M3)


def _linear_check(got, x, xs, w, ws):
    a, b = x.double() * xs.double()[:, None], w.double() * ws.double()[:, None]
    want, mass = a @ b.T, a.abs() @ b.abs().T
    # fp32 sums of exact products: the tensor core adds 32 at a time, each addition truncating
    tol = want.abs() * 2.0 ** -8 + mass * (x.shape[1] / 32 + 40) * 2.0 ** -23
    err = (got.cpu().double() - want).abs()
    assert (err <= tol).all(), float((err / tol.clamp_min(1e-300)).max())


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 33, 64, 65, 128, 129, 200, 256, 257, 300, 511, 1000])
@pytest.mark.parametrize("N,K", [(8, 16), (136, 1040), (1000, 528), (520, 2048)])
def test_linear_e4m3(ops, M, N, K):
    g = _gen(M * 1000 + N + K)
    x, w = _codes(g, M, K), _codes(g, N, K)
    xs, ws = torch.rand(M, generator=g) * 0.01, torch.rand(N, generator=g) * 0.001
    got = ops.linear_e4m3(x.cuda(), xs.cuda(), w.cuda(), ws.cuda())
    ops.device_status()
    assert got.shape == (M, N) and got.dtype == torch.bfloat16
    _linear_check(got, x, xs, w, ws)


@pytest.mark.parametrize("M,N,K", [(1, 6144, 2048), (9, 40000, 256), (40, 256, 16384), (100, 4096, 1024), (513, 2048, 4096)])
def test_linear_e4m3_larger(ops, M, N, K):
    g = _gen(M + N + K)
    x, w = _codes(g, M, K), _codes(g, N, K)
    xs, ws = torch.rand(M, generator=g) * 0.01, torch.rand(N, generator=g) * 0.001
    args = [t.cuda() for t in (x, xs, w, ws)]
    got = ops.linear_e4m3(*args)
    _linear_check(got, x, xs, w, ws)
    for _ in range(3):
        assert torch.equal(ops.linear_e4m3(*args), got)  # the same bits every time


@pytest.mark.parametrize("M", [3, 100, 300])
def test_linear_e4m3_leaves_what_is_not_its_own(ops, M):
    N, K = 264, 144
    g = _gen(M)
    x, w = _codes(g, M, K), _codes(g, N, K)
    xs, ws = torch.rand(M, generator=g), torch.rand(N, generator=g)
    buf = torch.full((M * N + 4096,), 7.0, dtype=torch.bfloat16, device="cuda")
    assert ops.linear_e4m3(x.cuda(), xs.cuda(), w.cuda(), ws.cuda(), out=buf) is buf
    assert (buf[M * N:] == 7.0).all()
    _linear_check(buf[:M * N].view(M, N), x, xs, w, ws)


@pytest.mark.parametrize("M", [4, 130, 400])
def test_linear_e4m3_nan_codes_stay_in_their_row_and_column(ops, M):
    N, K = 256, 256
    g = _gen(M + 1)
    x, w = _codes(g, M, K), _codes(g, N, K)
    x.view(torch.uint8)[2, 100] = 0x7f
    w.view(torch.uint8)[9, 30] = 0xff
    ones = torch.ones(max(M, N)).cuda()
    nan = torch.isnan(ops.linear_e4m3(x.cuda(), ones[:M], w.cuda(), ones[:N])).cpu()
    want = torch.zeros(M, N, dtype=torch.bool)
    want[2], want[:, 9] = True, True
    assert torch.equal(nan, want)


def test_linear_e4m3_refusals_and_empty(ops):
    g = _gen(1)
    x, w = _codes(g, 4, 32).cuda(), _codes(g, 16, 32).cuda()
    xs, ws = torch.ones(4, device="cuda"), torch.ones(16, device="cuda")
    for f in (lambda: ops.linear_e4m3(x, xs[:3], w, ws), lambda: ops.linear_e4m3(x, xs, w, ws[:8]),
              lambda: ops.linear_e4m3(x, xs, w[:, :16].contiguous(), ws), lambda: ops.linear_e4m3(x, xs, w[:12], ws[:12]),
              lambda: ops.linear_e4m3(_codes(g, 4, 24).cuda(), xs, _codes(g, 16, 24).cuda(), ws),
              lambda: ops.linear_e4m3(x, xs, w, ws, out=torch.empty(4, 15, dtype=torch.bfloat16, device="cuda")),
              lambda: ops.linear_e4m3(x[:, ::2], xs, w[:, ::2], ws), lambda: ops.linear_e4m3(x.cpu(), xs, w, ws)):
        with pytest.raises(ValueError):
            f()
    for f in (lambda: ops.linear_e4m3(x.float(), xs, w, ws), lambda: ops.linear_e4m3(x, xs.double(), w, ws)):
        with pytest.raises(TypeError):
            f()
    assert ops.linear_e4m3(x[:0], xs[:0], w, ws).shape == (0, 16)
    assert ops.linear_e4m3(x.view(2, 2, 32), xs.view(2, 2), w, ws).shape == (2, 2, 16)


# ------------------------------------------------------------------------------------------------------------
# the paged 8-bit cache: append
# ------------------------------------------------------------------------------------------------------------
def _pow2_scale(amax: float) -> float:
    if amax == 0:
        return 2.0 ** -64
    m, e = math.frexp(amax)
    return 2.0 ** min(max(e - 9 if m <= 0.875 else e - 8, -64), 120)


def _append_ref(codes, scale, x, table, ctx, cu):
    """codes [P, Hkv, page, D] e4m3 and scale [P, Hkv] fp32 on the CPU, in place, page by page as the definition says."""
    Hkv, page = codes.shape[1], codes.shape[2]
    for b in range(len(ctx)):
        t, pos, end = cu[b], ctx[b], min(ctx[b] + cu[b + 1] - cu[b], table.shape[1] * page)
        while pos < end:
            at, n, p = pos % page, min(end - pos, page - pos % page), int(table[b, pos // page])
            for h in range(Hkv):
                new = x[t:t + n, h].double()
                fin = new[torch.isfinite(new)]
                s = _pow2_scale(float(fin.abs().max()) if fin.numel() else 0.0)
                if at > 0:
                    old = float(scale[p, h])
                    s = max(s, old)
                    if s != old:
                        codes[p, h, :at] = (codes[p, h, :at].double() * (old / s)).to(E4M3)
                new = torch.where(torch.isfinite(new), new / s, torch.nan)
                codes[p, h, at:at + n] = new.to(E4M3)
                scale[p, h] = s
            t, pos = t + n, pos + n


def _random_cache(ops, pages, Hkv, page, D, seed, sigma_exp=(-2, 3), fill=None):
    g = _gen(seed)
    out = []
    for _ in "kv":
        codes = (torch.randn(pages, Hkv, page, D, generator=g) * 64).clamp(-448, 448).to(E4M3)
        if fill is not None:
            codes.view(torch.uint8).fill_(fill)
        scale = torch.ldexp(torch.ones(pages, Hkv), torch.randint(*sigma_exp, (pages, Hkv), generator=g) - 6)
        out.append((codes, scale))
    return ops.KV8Cache(out[0][0], out[1][0], out[0][1], out[1][1])


def _to(cache, device):
    return type(cache)(*(t.to(device) for t in cache))


def _same_codes(a, b):
    a, b = a.float().cpu(), b.float().cpu()
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))


def _check_append(ops, Hkv, D, page, ctx, new, seed=0, max_pages=None, size=None, special=False):
    g = _gen(seed + 11)
    B = len(ctx)
    need = max(-(-(c + n) // page) for c, n in zip(ctx, new))
    max_pages = max(1, need) if max_pages is None else max_pages
    pages = B * max_pages + 3
    table = torch.randperm(pages, generator=g)[:B * max_pages].view(B, max_pages).int()
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    T = cu[-1] + 2  # two rows behind the last sequence: not read
    fused = torch.randn(T, 3 * Hkv, D, generator=g)
    if size is not None:
        fused *= torch.exp2(torch.randint(*size, (T, 1, 1), generator=g).float())
    fused = fused.bfloat16()
    if special:
        fused[:, :, 3] = torch.where(torch.rand(T, 3 * Hkv, generator=g) < 0.3, float("inf"), fused[:, :, 3].float()).bfloat16()
        fused[:, :, 5] = torch.where(torch.rand(T, 3 * Hkv, generator=g) < 0.3, float("nan"), fused[:, :, 5].float()).bfloat16()
        fused[cu[1]:cu[2]] = 0
    fused[cu[-1]:] = float("nan")
    cache = _random_cache(ops, pages, Hkv, page, D, seed)
    want = type(cache)(*(t.clone() for t in cache))
    k, v = fused[:, Hkv:2 * Hkv], fused[:, 2 * Hkv:]
    _append_ref(want.k, want.k_scale, k, table, ctx, cu)
    _append_ref(want.v, want.v_scale, v, table, ctx, cu)
    dev, fd = _to(cache, "cuda"), fused.cuda()
    args = (table.cuda(), torch.tensor(ctx, dtype=torch.int32).cuda(), torch.tensor(cu, dtype=torch.int32).cuda())
    for _ in range(2):  # appending the same tokens at the same place again changes nothing
        assert ops.kv8_append_(dev, fd[:, Hkv:2 * Hkv], fd[:, 2 * Hkv:], *args) is dev
        ops.device_status()
        assert torch.equal(dev.k_scale.cpu(), want.k_scale) and torch.equal(dev.v_scale.cpu(), want.v_scale)
        assert _same_codes(dev.k, want.k) and _same_codes(dev.v, want.v)


@pytest.mark.parametrize("Hkv,D", [(1, 64), (2, 128), (3, 64), (8, 128)])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_kv8_append_mixed(ops, Hkv, D, page):
    ctx = [0, 1, page - 1, page, page + 1, 3 * page - 1, 5, 0]
    new = [1, 0, 1, 2, 2 * page + 3, 1, page - 5, 3 * page]
    _check_append(ops, Hkv, D, page, ctx, new, seed=page + Hkv, size=(-2, 6))


@pytest.mark.parametrize("B", [1, 31, 33, 70])
def test_kv8_append_single_tokens(ops, B):
    ctx = [(37 * b) % 200 for b in range(B)]
    _check_append(ops, 2, 128, 32, ctx, [1] * B, seed=B, size=(-3, 9))


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("kind", ["even", "mixed", "prompt"])
def test_kv8_append_some_tokens_of_many_sequences(ops, page, kind):
    B = 70
    ctx = [(53 * b) % 300 for b in range(B)]
    new = {"even": [9] * B, "mixed": [(11 * b) % 31 for b in range(B)], "prompt": [1] * 30 + [700] + [2] * (B - 31)}[kind]
    _check_append(ops, 8, 128, page, ctx, new, seed=page, size=(-3, 6))


def test_kv8_append_extreme_sizes_and_non_finite(ops):
    _check_append(ops, 2, 64, 16, [3, 20, 0], [20, 5, 9], seed=1, size=(-120, 126))
    _check_append(ops, 2, 128, 16, [3, 20, 0], [20, 5, 9], seed=2, size=(-140, -60))
    _check_append(ops, 4, 128, 32, [3, 20, 40, 0], [20, 5, 9, 70], seed=3, special=True)


def test_kv8_append_drops_what_the_table_cannot_hold(ops):
    _check_append(ops, 2, 64, 16, [30, 3, 32], [10, 40, 4], seed=4, max_pages=2)


def test_kv8_append_scale_borders(ops):
    # 448 fits a scale of one, the next bf16 above it does not
    for value, scale in ((448.0, 1.0), (450.0, 2.0), (224.0, 0.5), (1.0, 2.0 ** -8), (1.75, 2.0 ** -8), (1.7578125, 2.0 ** -7)):
        cache = ops.kv8_cache(1, 1, 16, 64)
        x = torch.full((1, 1, 64), value, dtype=torch.bfloat16, device="cuda")
        one = torch.zeros(1, dtype=torch.int32, device="cuda")
        ops.kv8_append_(cache, x, -x, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), one,
                        torch.tensor([0, 1], dtype=torch.int32, device="cuda"))
        assert float(cache.k_scale) == scale and float(cache.v_scale) == scale
        want = float((torch.tensor(value) / scale).to(E4M3))
        assert (cache.k[0, 0, 0].float() == want).all() and (cache.v[0, 0, 0].float() == -want).all()
        assert (cache.k[0, 0, 1:].view(torch.uint8) == 0).all()


# ------------------------------------------------------------------------------------------------------------
# attention over the cache
# ------------------------------------------------------------------------------------------------------------
def _attend_check(ops, got, q, cache, table, lens, scale):
    """Every output row against 64 bits, with a bound made from the row's own probabilities."""
    B, Sq, Hq, D = q.shape
    Hkv, page = cache.k.shape[1], cache.k.shape[2]
    G = Hq // Hkv
    got = got.cpu().double()
    for b in range(B):
        n = int(lens[b])
        at = table[b, :-(-n // page)].long()
        for h in range(Hkv):
            k = (cache.k.view(torch.uint8)[at, h].view(E4M3).double() * cache.k_scale[at, h].double()[:, None, None]).reshape(-1, D)[:n]
            v = (cache.v.view(torch.uint8)[at, h].view(E4M3).double() * cache.v_scale[at, h].double()[:, None, None]).reshape(-1, D)[:n]
            for i in range(Sq):
                o = got[b, i, h * G:(h + 1) * G]
                m = n - Sq + i + 1
                if m <= 0:
                    assert (o == 0).all(), (b, i)
                    continue
                qd = q[b, i, h * G:(h + 1) * G].double()
                s = qd @ k[:m].T * scale
                p = torch.softmax(s, -1)
                want, mass = p @ v[:m], p @ v[:m].abs()
                # logits: fp32 sums of D products, and roundings of the scaled logit next to log2 of the value scale
                ds = D * 2.0 ** -23 * (qd.abs() @ k[:m].abs().T * abs(scale)).amax(-1, keepdim=True) + 2.0 ** -22 * (s.abs().amax(-1, keepdim=True) + 100)
                # probabilities: fp16; sums over the tokens: one step in 16 tokens
                rel = 2.0 ** -11 + 2 * ds + 2.0 ** -20 + (m / 16 + 16) * 2.0 ** -23
                tol = want.abs() * 2.0 ** -8 + rel * mass
                bad = (o - want).abs() > tol
                assert not bad.any(), (b, h, i, m, float(((o - want).abs() / tol).max()))


#: tokens a page table has room for: as many as the longest sequence (a kernel of one launch where that is short), or so
#: many that the sequences' lengths may lie far apart (the list of tiles and its join). The rest of the table is never read.
ROOM = ["tight", 1 << 20]


def _attend_case(ops, Sq, Hq, Hkv, D, page, lens, seed=0, q_scale=1.0, sigma_exp=(-2, 3), fused=False, check=True, room="tight"):
    g = _gen(seed + 31)
    B = len(lens)
    max_pages = max(1, -(-max(lens) // page))
    pages = B * max_pages + 2
    table = torch.randperm(pages, generator=g)[:B * max_pages].view(B, max_pages).int()
    if room != "tight":
        table = torch.cat([table, torch.full((B, room // page - max_pages), -1, dtype=torch.int32)], 1)
    cache = _random_cache(ops, pages, Hkv, page, D, seed, sigma_exp)
    # whatever is behind a sequence's last token must not matter: NaN codes there, NaN scales on pages nobody uses
    used = torch.zeros(pages, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for i in range(-(-n // page)):
            used[table[b, i], :min(page, n - i * page)] = True
    for codes, sc in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        codes.view(torch.uint8)[(~used)[:, None].expand(-1, Hkv, -1)] = 0x7f
        sc[~used.any(1)] = float("nan")
    q = (q_scale * torch.randn(B, Sq, Hq, D, generator=g)).bfloat16()
    qd = q.cuda()
    if fused:  # a view of a fused projection [B, Sq, (Hq + 2 Hkv) * D]
        buf = torch.full((B, Sq, Hq + 2 * Hkv, D), float("nan"), dtype=torch.bfloat16, device="cuda")
        buf[:, :, :Hq] = qd
        qd = buf[:, :, :Hq]
    dev = _to(cache, "cuda")
    lens_t = torch.tensor(lens, dtype=torch.int32)
    scale = 1.0 / math.sqrt(D)
    got = ops.sdpa_kv8(qd, dev, table.cuda(), lens_t.cuda())
    ops.device_status()
    assert got.shape == q.shape and got.dtype == torch.bfloat16
    if check:
        _attend_check(ops, got, q, cache, table, lens, scale)
    return got, qd, dev, table.cuda(), lens_t.cuda()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (4, 2), (16, 1), (10, 2)])
@pytest.mark.parametrize("room", ROOM)
def test_sdpa_kv8_single_token(ops, D, page, Hq, Hkv, room):
    lens = [1, 0, 2, 15, 16, 17, 63, 64, 65, page, page + 1, 127, 129, 0, 1000, 3]
    _attend_case(ops, 1, Hq, Hkv, D, page, lens, seed=D + page + Hq, room=room)


@pytest.mark.parametrize("Sq", [2, 3, 4, 9])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (3, 1, 64), (32, 1, 64)])
@pytest.mark.parametrize("room", ROOM)
def test_sdpa_kv8_several_tokens(ops, Sq, Hq, Hkv, D, room):
    lens = [0, 1, Sq - 1, Sq, Sq + 1, 16, 70, 333]  # the first queries of a sequence shorter than Sq see nothing
    _attend_case(ops, Sq, Hq, Hkv, D, 32, lens, seed=Sq + Hq, fused=True, room=room)


@pytest.mark.parametrize("room", ROOM)
def test_sdpa_kv8_long_and_ragged(ops, room):
    # few sequences: every row is cut over many CTAs; the longest next to the shortest
    _attend_case(ops, 1, 4, 1, 128, 128, [40000], seed=1, room=room)
    _attend_case(ops, 1, 4, 2, 128, 64, [1, 20000, 0, 300, 64], seed=2, room=room)
    _attend_case(ops, 2, 8, 4, 64, 16, [5, 9000, 1], seed=3, fused=True, room=room)


@pytest.mark.parametrize("room", ROOM)
def test_sdpa_kv8_many_sequences(ops, room):
    lens = [(b * 7919) % 130 for b in range(300)]
    _attend_case(ops, 1, 2, 1, 64, 16, lens, seed=4, room=room)
    _attend_case(ops, 1, 9, 1, 128, 16, [17] * 700, seed=5, room=room)


@pytest.mark.parametrize("B,longest", [(130, 33), (301, 130), (600, 500)])
@pytest.mark.parametrize("G,Sq,D,Hkv", [(2, 1, 128, 8), (1, 3, 64, 7), (4, 3, 64, 5), (2, 5, 128, 7)])
def test_sdpa_kv8_many_short_rows(ops, B, longest, G, Sq, D, Hkv):
    """A warp may take a row to itself; empty rows, and rows that are no multiple of the block's warps."""
    lens = _mixed_lengths(B, longest)
    if longest == 500:  # not short rows for every head count: the others' kernels see the same lengths
        got, q, cache, table, lens_t = _attend_case(ops, Sq, G * Hkv, Hkv, D, 16, lens, seed=B + D, check=False)
        rows = torch.tensor([0, 1, 5, 300, 598, 599])
        _attend_check(ops, got[rows.cuda()], q[rows.cuda()].cpu(), _to(cache, "cpu"), table.cpu()[rows], [lens[i] for i in rows], 1 / math.sqrt(D))
    else:
        _attend_case(ops, Sq, G * Hkv, Hkv, D, 16, lens, seed=B + D)
    ops.device_status()


@pytest.mark.parametrize("B", [1, 3, 6, 12, 16, 17])
@pytest.mark.parametrize("G,Sq,D", [(2, 1, 128), (1, 3, 64), (4, 3, 64), (2, 5, 128)])
def test_sdpa_kv8_few_rows(ops, B, G, Sq, D):
    """A row's warps lie in 8, 4, 2 or 1 CTAs; sequences shorter than their number of warps, and empty ones."""
    lens = [1500, 0, 17, 640, 1, 1499, 16, 33, 512, 0, 1024, 250, 3, 1500, 90, 47, 1211][:B]
    got, *args = _attend_case(ops, Sq, 8 * G, 8, D, 64, lens, seed=B + G + D)
    for _ in range(3):
        assert torch.equal(ops.sdpa_kv8(*args), got)
    ops.device_status()


def _mixed_lengths(B, longest):
    g = _gen(B)
    lens = (torch.rand(B, generator=g) ** 2 * (longest + 1)).long().clamp(max=longest).tolist()
    lens[:6] = [0, longest, 1, longest, 0, 16]
    return lens


@pytest.mark.parametrize("B,Hq,Hkv,D,Sq", [(150, 4, 2, 128, 1), (256, 2, 1, 64, 1), (257, 2, 1, 128, 1), (150, 8, 2, 64, 3), (150, 8, 2, 128, 3)])
@pytest.mark.parametrize("kind", ["mixed", "equal", "one"])
def test_sdpa_kv8_more_rows_than_the_machine_takes_at_once(ops, B, Hq, Hkv, D, Sq, kind):
    """Up to 256 sequences are taken longest first: every one of them exactly once, whatever their lengths."""
    longest = 1300
    lens = {"mixed": _mixed_lengths(B, longest), "equal": [longest] * B, "one": [0] * (B - 1) + [longest]}[kind]
    got, q, cache, table, lens_t = _attend_case(ops, Sq, Hq, Hkv, D, 64, lens, seed=B + D, check=kind == "mixed" and Sq == 1)
    # every sequence by itself: other kernels' sums in another order, so a rounding of the output apart
    for b in {0, 1, B // 2, B - 2, B - 1}:
        alone = ops.sdpa_kv8(q[b:b + 1], cache, table[b:b + 1], lens_t[b:b + 1])
        assert torch.isfinite(alone).all()
        # both lie within 2^-9 of the value (half a step) and twice 2^-11 of the probabilities' mass, which the values' largest bounds
        vmax = float((cache.v[table[b].long()].float().nan_to_num().abs().amax((1, 2, 3)) * cache.v_scale[table[b].long()].amax(1).nan_to_num()).max())
        tol = got[b].float().abs() * 2.0 ** -7 + 2.0 ** -9 * vmax
        assert ((got[b].float() - alone[0].float()).abs() <= tol).all(), b


@pytest.mark.parametrize("q_scale,sigma_exp", [(30.0, (-2, 3)), (1.0, (-58, -40)), (1e-25, (60, 110)), (1.0, (-20, 4)), (0.0, (-2, 3))])
@pytest.mark.parametrize("room", ROOM)
def test_sdpa_kv8_extreme_scales(ops, q_scale, sigma_exp, room):
    # peaked rows; pages whose scales lie far apart (a small-scale page may carry all the probability); zero queries
    _attend_case(ops, 1, 4, 2, 128, 16, [200, 33, 1], seed=5, q_scale=q_scale, sigma_exp=sigma_exp, room=room)


@pytest.mark.parametrize("room", ROOM)
def test_sdpa_kv8_zero_scale_pages(ops, room):
    got, q, cache, table, lens = _attend_case(ops, 1, 4, 2, 128, 16, [100, 40], seed=6, check=False, room=room)
    cache.v_scale[table[0, 2]] = 0.0
    cache.k_scale[table[0, 3]] = 0.0
    cache.v_scale[table[1, :3]] = 0.0
    out = ops.sdpa_kv8(q, cache, table, lens)
    _attend_check(ops, out, q.cpu(), _to(cache, "cpu"), table.cpu(), lens.tolist(), 1 / math.sqrt(128))


@pytest.mark.parametrize("room", ROOM)
def test_sdpa_kv8_non_finite_inputs_reach_their_rows_only(ops, room):
    got, q, cache, table, lens = _attend_case(ops, 1, 4, 2, 128, 16, [100, 40, 70], seed=7, check=False, room=room)
    q = q.clone()
    q[1, 0, 0, 5] = float("inf")
    cache.v.view(torch.uint8)[table[2, 1], 1, 3, 9] = 0x7f  # one value of sequence 2, KV head 1, channel 9
    out = ops.sdpa_kv8(q, cache, table, lens)
    nan = torch.isnan(out.float())
    assert nan[1, 0, 0].all() and not nan[1, 0, 1:].any() and not nan[0].any()
    assert nan[2, 0, 2:, 9].all() and nan[2].sum() == 2
    cache.k.view(torch.uint8)[table[0, 0], 0, 2, 1] = 0xff  # one key: every head that reads it
    nan = torch.isnan(ops.sdpa_kv8(q, cache, table, lens).float())
    assert nan[0, 0, :2].all() and not nan[0, 0, 2:].any()


@pytest.mark.parametrize("room", ROOM)
def test_sdpa_kv8_same_bits_every_time_and_given_buffers(ops, room):
    got, q, cache, table, lens = _attend_case(ops, 1, 8, 2, 128, 64, [5000, 0, 77], seed=8, check=False, room=room)
    ws = ops.sdpa_kv8_workspace(3, 1, 8, cache, table.shape[1])
    ws.fill_(255)  # holds nothing between calls
    out = torch.full_like(got, float("nan"))
    assert ops.sdpa_kv8(q, cache, table, lens, out=out, workspace=ws) is out
    assert torch.equal(out, got)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = ops.sdpa_kv8(q, cache, table, lens)
    side.synchronize()
    assert torch.equal(again, got)


def test_sdpa_kv8_offsets_past_32_bits(ops):
    page, Hkv, D = 256, 8, 128
    pages = 17000  # 17000 * 262144 bytes > 2^32 of codes each
    cache = ops.kv8_cache(pages, Hkv, page, D)
    table = torch.tensor([[16999, 0, 16500]], dtype=torch.int32, device="cuda")
    g = _gen(9)
    kv = torch.randn(600, 2 * Hkv, D, generator=g).bfloat16().cuda()
    lens = torch.tensor([600], dtype=torch.int32, device="cuda")
    ops.kv8_append_(cache, kv[:, :Hkv], kv[:, Hkv:], table, torch.zeros_like(lens), torch.tensor([0, 600], dtype=torch.int32, device="cuda"))
    q = torch.randn(1, 1, 16, D, generator=g).bfloat16()
    out = ops.sdpa_kv8(q.cuda(), cache, table, lens)
    ids = table[0].long()
    small = ops.KV8Cache(cache.k.view(torch.uint8)[ids].view(E4M3).cpu(), cache.v.view(torch.uint8)[ids].view(E4M3).cpu(),
                         cache.k_scale[ids].cpu(), cache.v_scale[ids].cpu())
    assert (small.k.float().abs().amax((2, 3)) > 0).all()
    _attend_check(ops, out, q, small, torch.tensor([[0, 1, 2]]), [600], 1 / math.sqrt(D))


@pytest.mark.parametrize("max_pages", [4, 1 << 16])
def test_kv8_captured_step_replays_with_new_lengths(ops, max_pages):
    """Append and attention in one captured graph; tokens, lengths and page table are device data."""
    B, Hq, Hkv, D, page, used = 3, 8, 2, 128, 16, 4
    g = _gen(10)
    cache = ops.kv8_cache(B * used, Hkv, page, D)
    table = torch.full((B, max_pages), -1, dtype=torch.int32, device="cuda")
    table[:, :used] = torch.randperm(B * used, generator=g).view(B, used).int().cuda()
    cu = torch.arange(B + 1, dtype=torch.int32, device="cuda")
    ctx = torch.zeros(B, dtype=torch.int32, device="cuda")
    qkv = torch.empty(B, Hq + 2 * Hkv, D, dtype=torch.bfloat16, device="cuda")
    out = torch.empty(B, 1, Hq, D, dtype=torch.bfloat16, device="cuda")
    ws = ops.sdpa_kv8_workspace(B, 1, Hq, cache, max_pages)

    def step():
        ops.kv8_append_(cache, qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:], table, ctx, cu)
        ctx.add_(1)
        ops.sdpa_kv8(qkv[:, :Hq].unsqueeze(1), cache, table, ctx, out=out, workspace=ws)

    qkv.zero_()
    step()  # the first call sets kernel attributes
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    ctx.copy_(torch.tensor([0, 0, 0], dtype=torch.int32))
    keys = []
    for i in range(40):
        keys.append(torch.randn(B, Hq + 2 * Hkv, D, generator=g).bfloat16())
        qkv.copy_(keys[-1])
        graph.replay()
    ops.device_status()
    assert ctx.tolist() == [40] * B
    _attend_check(ops, out, keys[-1][:, :Hq].unsqueeze(1), _to(cache, "cpu"), table.cpu(), [40] * B, 1 / math.sqrt(D))
    want = ops.kv8_cache(B * used, Hkv, page, D, device="cpu")
    for i, x in enumerate(keys):
        _append_ref(want.k, want.k_scale, x[:, Hq:Hq + Hkv], table.cpu(), [i] * B, list(range(B + 1)))
        _append_ref(want.v, want.v_scale, x[:, Hq + Hkv:], table.cpu(), [i] * B, list(range(B + 1)))
    assert torch.equal(cache.k_scale.cpu(), want.k_scale) and _same_codes(cache.k, want.k)
    assert torch.equal(cache.v_scale.cpu(), want.v_scale) and _same_codes(cache.v, want.v)


def test_kv8_refusals(ops):
    cache = ops.kv8_cache(4, 2, 16, 64)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    table, lens, cu = i32([0, 1], [2, 3]), i32(1, 2), i32(0, 1, 2)
    x = torch.randn(2, 2, 64, device="cuda").bfloat16()
    q = torch.randn(2, 1, 4, 64, device="cuda").bfloat16()
    bad_values = [
        lambda: ops.kv8_append_(cache, x[:, :1], x, table, lens, cu),
        lambda: ops.kv8_append_(cache, x, x, table, lens, cu[:2].contiguous()),
        lambda: ops.kv8_append_(cache, x, x, table, lens[:1].contiguous(), cu),
        lambda: ops.kv8_append_(cache, x.transpose(1, 2).contiguous().transpose(1, 2), x, table, lens, cu),
        lambda: ops.kv8_append_(cache, x[:1].expand(2, 2, 64), x, table, lens, cu),
        lambda: ops.kv8_append_(cache, x.cpu(), x, table, lens, cu),
        lambda: ops.kv8_append_(cache._replace(k_scale=cache.k_scale[:2]), x, x, table, lens, cu),
        lambda: ops.kv8_append_(ops.kv8_cache(4, 2, 24, 64), x, x, table, lens, cu),
        lambda: ops.sdpa_kv8(q, ops.kv8_cache(4, 2, 24, 64), table, lens),
        lambda: ops.sdpa_kv8(q[:, :, :3].contiguous(), cache, table, lens),
        lambda: ops.sdpa_kv8(q[:1], cache, table, lens),
        lambda: ops.sdpa_kv8(q, cache, table[:, :0].contiguous(), lens),
        lambda: ops.sdpa_kv8(q, cache, table.repeat(1, 1 << 16), lens, workspace=torch.empty(16, dtype=torch.uint8, device="cuda")),
        lambda: ops.sdpa_kv8(q, cache, table, lens, out=torch.empty(2, 1, 4, 32, dtype=torch.bfloat16, device="cuda")),
        lambda: ops.sdpa_kv8(torch.randn(2, 1, 4, 96, device="cuda").bfloat16(), ops.kv8_cache(4, 2, 16, 96), table, lens),
        lambda: ops.sdpa_kv8(torch.randn(2, 1, 4, 68, device="cuda").bfloat16()[..., 4:], cache, table, lens),
    ]
    for f in bad_values:
        with pytest.raises(ValueError):
            f()
    for f in (lambda: ops.sdpa_kv8(q.float(), cache, table, lens), lambda: ops.sdpa_kv8(q, cache, table.long(), lens),
              lambda: ops.kv8_append_(cache, x.float(), x, table, lens, cu),
              lambda: ops.kv8_append_(cache._replace(k=cache.k.view(torch.uint8)), x, x, table, lens, cu)):
        with pytest.raises(TypeError):
            f()
    assert ops.sdpa_kv8(q[:0], cache, table[:0], lens[:0]).shape == (0, 1, 4, 64)
    assert ops.kv8_append_(cache, x[:0], x[:0], table, lens, cu) is cache
    ops.device_status()
    assert (cache.k.view(torch.uint8) == 0).all()
