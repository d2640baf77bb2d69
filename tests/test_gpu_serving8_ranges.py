"""Ranges of values that the 8-bit serving operators have to hold over: eps far below and rows far above what fp32's squares
carry, value scales that lie as far apart as appending can leave them. Tolerances are those of ``test_gpu_serving8``."""

from __future__ import annotations

import math

import pytest
import torch

from tests.test_gpu_serving8 import _attend_check, _check_norm, _gen, _norm_ref, _random_cache, _to, ops  # noqa: F401

pytestmark = pytest.mark.gpu

#: rows x columns that reach every form of the norm's kernel: threads per row, packs per thread, odd lengths, long rows
NORM_SIZES = [(9, 64), (7, 1024), (7, 1023), (5, 4096), (3, 16384), (4, 20000), (4, 20011), (1300, 32), (1301, 250), (1290, 256),
              (1290, 1024), (1290, 2048)]


def _norm_case(ops, rows, cols, dtype, eps, with_residual, kinds, seed):  # noqa: F811
    """Rows of every kind in turn (neighbours share a warp or a CTA); weights of one, so that f * w is exact."""
    g = _gen(seed + cols)
    x = torch.randn(rows, cols, generator=g)
    for i, kind in enumerate(kinds):
        x[i::len(kinds)] = kind(x[i::len(kinds)])
    x = x.to(dtype)
    r = torch.zeros_like(x)
    if with_residual:
        r[::len(kinds)] = torch.randn(r[::len(kinds)].shape, generator=g).to(dtype)
    w = torch.ones(cols, dtype=dtype)
    args = (x.cuda(), w.cuda(), eps)
    got = ops.rmsnorm_e4m3(*args, residual=r.cuda()) if with_residual else ops.rmsnorm_e4m3(*args)
    ops.device_status()
    return got, _norm_ref(x, w, eps, r if with_residual else None)


@pytest.mark.parametrize("rows,cols", NORM_SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("eps", [1e-12, 1e-30])
def test_rmsnorm_e4m3_rows_of_zeros_and_small_eps(ops, rows, cols, dtype, with_residual, eps):  # noqa: F811
    """A row of zeros gives zeros, however large 1 / sqrt(eps) is; so small a row that its scale is at the floor keeps its
    codes."""
    kinds = [lambda v: v, lambda v: 0 * v, lambda v: v * 2.0 ** -121, lambda v: v * 2.0 ** -135]
    got, ref = _norm_case(ops, rows, cols, dtype, eps, with_residual, kinds, 1)
    assert (got[0][1::4].view(torch.uint8) & 0x7f == 0).all()
    _check_norm(got, ref, terms=cols)


@pytest.mark.parametrize("rows,cols", NORM_SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("with_residual", [False, True])
def test_rmsnorm_e4m3_rows_whose_squares_pass_fp32(ops, rows, cols, dtype, with_residual):  # noqa: F811
    def one_huge(v):
        v[:, v.shape[1] // 2] = 3e38
        return v

    kinds = [lambda v: v, lambda v: v * 1e25, one_huge, lambda v: v * 1e18, lambda v: v * 1e37]
    got, ref = _norm_case(ops, rows, cols, dtype, 1e-6, with_residual, kinds, 2)
    _check_norm(got, ref, terms=cols)


@pytest.mark.parametrize("rows,cols", NORM_SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("eps", [0.0, 1e-38])
def test_rmsnorm_e4m3_rows_whose_squares_vanish(ops, rows, cols, dtype, with_residual, eps):  # noqa: F811
    kinds = [lambda v: v, lambda v: v * 1e-25, lambda v: v * 1e-30, lambda v: v * 1e-20, lambda v: v * 1e-36]
    got, ref = _norm_case(ops, rows, cols, dtype, eps, with_residual, kinds, 3)
    _check_norm(got, ref, terms=cols)


@pytest.mark.parametrize("cols", [64, 1023, 1024, 20000])
def test_rmsnorm_e4m3_non_finite_rows_stay_nan(ops, cols):  # noqa: F811
    x = torch.randn(1300, cols, generator=_gen(4))
    x[1::4, cols // 3] = float("inf")
    x[2::4, 0] = float("nan")
    x[3::4, :2] = torch.tensor([float("-inf"), 3e38])
    q, scale = ops.rmsnorm_e4m3(x.cuda(), torch.ones(cols).cuda(), 1e-6)
    bad = torch.isnan(q.float()).all(1).cpu()
    assert bad[1::4].all() and bad[2::4].all() and bad[3::4].all() and not bad[::4].any()
    assert torch.equal(torch.isnan(scale).cpu(), bad)
    assert torch.isfinite(q[::4].float()).all()


@pytest.mark.parametrize("rows,cols", NORM_SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rmsnorm_e4m3_products_past_fp32_are_nan_rows(ops, rows, cols, dtype):  # noqa: F811
    """Where f * w, or the normalised value itself, passes fp32's range: NaN codes and a NaN scale, and its neighbours are right."""
    x = torch.randn(rows, cols, generator=_gen(8)).to(dtype)
    w = torch.ones(cols, dtype=dtype)
    w[cols // 2] = 1e30
    x[:, cols // 2] = 1e-30
    x[1::3, cols // 2] = 1e12  # f * w
    x[2::3] *= 1e-20
    x[2::3, cols // 2] = 1e-3  # 1e30 sqrt(cols) once normalised
    q, scale = ops.rmsnorm_e4m3(x.cuda(), w.cuda(), 1e-30)
    far = torch.tensor([i % 3 == 1 for i in range(rows)])
    assert torch.equal(torch.isnan(scale).cpu(), far) and torch.isnan(q[far.cuda()].float()).all()
    ok = ~far
    y, s, _ = _norm_ref(x, w, 1e-30, None)
    _check_norm((q.cpu()[ok], scale.cpu()[ok]), (y[ok], s[ok], None), terms=cols)
    # weights so large that a normalised value of more than one passes the range: a lone element's is sqrt(cols)
    w[:] = 3e38
    v = torch.zeros(rows, cols, dtype=dtype)
    v[:, 0] = 1e-3
    v[::2, 1:] = 1e-3
    q, scale = ops.rmsnorm_e4m3(v.cuda(), w.cuda(), 1e-12)
    assert torch.equal(torch.isnan(scale).cpu(), torch.tensor([i % 2 == 1 for i in range(rows)]))
    assert torch.isnan(q[1::2].float()).all() and not torch.isnan(q[::2].float()).any()


#: batch, longest sequence and room of the page table for the ways to share the work: a warp a row, clusters of small CTAs,
#: clusters of SM-sized CTAs, the list of tiles
WAYS = [(300, 80, "tight"), (40, 300, "tight"), (2, 900, "tight"), (3, 900, 1 << 20)]


def _spread(ops, B, longest, room, Sq, G, D, exponents, order, seed, Hkv=2, page=16):  # noqa: F811
    """Sequences whose pages have value scales 2^e, e of ``exponents`` in the given order; queries so small that all pages weigh
    alike in the sum. Returns the output and what ``_attend_check`` takes, of the first sequences."""
    g = _gen(seed)
    max_pages = -(-longest // page)
    lens = torch.randint(Sq, longest + 1, (B,), generator=g).int()
    lens[0] = longest
    table = torch.randperm(B * max_pages, generator=g).view(B, max_pages).int()
    cache = _random_cache(ops, B * max_pages, Hkv, page, D, seed)
    e = torch.tensor(exponents)[torch.randint(len(exponents), (B, max_pages, Hkv), generator=g)]
    if order != "mixed":
        e = e.sort(1, descending=order == "falling").values
    cache.v_scale[table.long()] = torch.exp2(e.double()).float()
    q = (0.05 * torch.randn(B, Sq, G * Hkv, D, generator=g)).bfloat16()
    wide = table if room == "tight" else torch.cat([table, torch.full((B, room // page - max_pages), -1, dtype=torch.int32)], 1)
    out = ops.sdpa_kv8(q.cuda(), _to(cache, "cuda"), wide.cuda(), lens.cuda())
    ops.device_status()
    n = min(B, 6)
    return out[:n], q[:n], cache, table[:n], lens[:n].tolist()


@pytest.mark.parametrize("B,longest,room", WAYS)
@pytest.mark.parametrize("Sq,G,D", [(1, 2, 128), (1, 4, 64), (4, 4, 128), (3, 2, 64)])
def test_value_scales_too_small_to_matter_count_as_zero(ops, B, longest, room, Sq, G, D):  # noqa: F811
    out, q, cache, table, lens = _spread(ops, B, longest, room, Sq, G, D, [-120], "mixed", 5)
    assert (out == 0).all()
    # beside others they weigh in the sum as pages of zeros do
    out, q, cache, table, lens = _spread(ops, B, longest, room, Sq, G, D, [-120, -3], "mixed", 6)
    cache.v_scale[cache.v_scale < 2.0 ** -100] = 0.0
    _attend_check(ops, out, q, cache, table, lens, 1 / math.sqrt(D))


@pytest.mark.parametrize("order", ["rising", "falling", "mixed"])
@pytest.mark.parametrize("B,longest,room", WAYS)
@pytest.mark.parametrize("Sq,G,D", [(1, 2, 128), (1, 4, 64), (4, 4, 128), (3, 2, 64)])
@pytest.mark.parametrize("exponents", [(-64, 110), (-64, -20, 40, 100), (70, 110)])
def test_pages_of_any_value_scale_weigh_in_the_sum(ops, order, B, longest, room, Sq, G, D, exponents):  # noqa: F811
    """A page whose values are too small to be seen beside another's still takes its share of the probability."""
    _attend_check(ops, *_spread(ops, B, longest, room, Sq, G, D, list(exponents), order, 7), 1 / math.sqrt(D))
