"""Sizes of the 8-bit serving operators that a step does not have: as many queries as a prompt over the cache, the weights of large
layers under few rows."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_serving8 import ROOM, _attend_case, _codes, _gen, _linear_check, ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("Sq,Hq,Hkv,D", [(200, 4, 1, 128), (131, 6, 2, 64), (64, 2, 2, 128)])
def test_sdpa_kv8_prompt_sized_queries(ops, room, Sq, Hq, Hkv, D):  # noqa: F811
    lens = [0, 1, Sq - 1, Sq, Sq + 17, 700, 64]
    _attend_case(ops, Sq, Hq, Hkv, D, 64, lens, seed=Sq, fused=True, room=room)


@pytest.mark.parametrize("M", [1, 16, 64, 128])
@pytest.mark.parametrize("N,K", [(28672, 4096), (8192, 8192), (4096, 14336)])
def test_linear_e4m3_few_rows_of_large_weights(ops, M, N, K):  # noqa: F811
    g = _gen(N + K)
    x, w = _codes(g, M, K), _codes(g, 256, K).repeat(N // 256, 1)
    xs, ws = torch.rand(M, generator=g) * 0.01, torch.rand(N, generator=g) * 0.001
    w[N - 8:] = _codes(g, 8, K)
    args = [t.cuda() for t in (x, xs, w, ws)]
    got = ops.linear_e4m3(*args)
    ops.device_status()
    # the first and the last columns against 64 bits; the others repeat the first 256 rows of w under scales of their own
    ends = torch.cat([torch.arange(256), torch.arange(N - 256, N)])
    _linear_check(got[:, ends.cuda()], x, xs, w[ends], ws[ends])
    bare = ops.linear_e4m3(args[0], torch.ones_like(args[1]), args[2], torch.ones_like(args[3])).view(M, N // 256, 256)
    assert torch.equal(bare[:, 1:-1], bare[:, :1].expand(-1, N // 256 - 2, -1))
    assert torch.equal(ops.linear_e4m3(*args), got)
