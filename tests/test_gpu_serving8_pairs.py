"""The many-rows kernel of the 8-bit linear layer at each of its tile widths: several tiles a CTA pair, so that the ring wraps from one
tile into the next and both accumulators change hands; ragged rows and columns; odd numbers of K slices."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_serving8 import _codes, _gen, _linear_check, ops  # noqa: F401
from tests.test_serving8_pairs_host import PAIR_SHAPES, SMS

pytestmark = pytest.mark.gpu


def _inputs(M, N, K):
    g = _gen(M + N + K)
    return _codes(g, M, K), torch.rand(M, generator=g) * 0.01, _codes(g, N, K), torch.rand(N, generator=g) * 0.001


@pytest.mark.parametrize("shape", PAIR_SHAPES)
def test_linear_e4m3_several_tiles_a_pair(ops, shape):  # noqa: F811
    M, N, K = shape
    assert torch.cuda.get_device_properties(0).multi_processor_count == SMS  # (the widths are those of this many)
    x, xs, w, ws = _inputs(M, N, K)
    args = [t.cuda() for t in (x, xs, w, ws)]
    guard = torch.full((M * N + 4096,), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.linear_e4m3(*args, out=guard)
    ops.device_status()
    assert (guard[M * N:] == 7.0).all()
    got = guard[:M * N].view(M, N)
    # every row tile's first, middle and last rows against 64 bits, and all columns of them
    rows = sorted({min(m, M - 1) for m0 in range(0, M, 256) for m in (m0, m0 + 31, m0 + 32, m0 + 127, m0 + 128, m0 + 255)} | {M - 1})
    rows = torch.tensor(rows)
    _linear_check(got[rows.cuda()], x[rows], xs[rows], w, ws)
    # and all rows: the other kernel's sums of the same products
    few = torch.cat([ops.linear_e4m3(args[0][m:m + 64], args[1][m:m + 64], args[2], args[3]) for m in range(0, M, 64)])
    mass = (x.float().abs() * xs[:, None]).cuda() @ (w.float().abs() * ws[:, None]).cuda().T
    tol = few.float().abs() * 2.0 ** -7 + mass * (1 + 2.0 ** -6) * 2 * (K / 32 + 40) * 2.0 ** -23
    assert ((got.float() - few.float()).abs() <= tol).all()


def test_linear_e4m3_pairs_back_to_back(ops):  # noqa: F811
    """Calls of one to six tiles a pair right behind one another (the next one's CTAs start as this one's leave): the same bits each
    time."""
    shapes = [(300, 512, 144), (1024, 6144, 2048), (1024, 4736, 1024), (3999, 6136, 1040), (300, 2048, 528), (5000, 9992, 400)]
    calls = [[t.cuda() for t in _inputs(*s)] for s in shapes]
    want = []
    for c in calls:
        want.append(ops.linear_e4m3(*c))
        torch.cuda.synchronize()
    for turn in range(30):
        got = [ops.linear_e4m3(*calls[(i * (turn % 5 + 1)) % 6]) for i in range(6)]
        for i, y in enumerate(got):
            assert torch.equal(y, want[(i * (turn % 5 + 1)) % 6])
    ops.device_status()
