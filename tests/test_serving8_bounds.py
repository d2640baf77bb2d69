"""Indices that come from data, in the 8-bit cache operators: page ids, cached lengths and cu_seqlens that point outside.
Both builds make the access safe (drop, clamp or cut); the bounds-check build reports it through ``device_status``. Nothing
here faults: every bad index is caught before it reaches memory."""

from __future__ import annotations

import os
import subprocess
import sys
import textwrap
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent

SCRIPT = textwrap.dedent('''
    import sys
    sys.path.insert(0, %r)
    import torch
    from deplodock_b200 import cabi, ops
    checked = bool(cabi.load_library().emk_bounds_check_enabled())
    assert checked == cabi.BOUNDS_CHECK

    def expect(kind, fn):
        r = fn()
        if checked:
            try:
                ops.device_status()
            except IndexError as e:
                assert kind in str(e), str(e)
            else:
                raise AssertionError(kind + ": violation not reported")
        else:
            ops.device_status()
        ops.device_status()              # the word is cleared, the context is fine
        return r

    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    torch.manual_seed(1)
    PAGES, HKV, PAGE, D = 12, 2, 16, 64
    guard = 5
    def fresh():
        # the pool proper is the middle of a larger buffer, so that a write just outside it would be seen
        big = [torch.full((PAGES + 2 * guard, HKV, PAGE, D), 0x11, dtype=torch.uint8, device="cuda") for _ in "kv"]
        scales = [torch.full((PAGES + 2 * guard, HKV), 0.25, device="cuda") for _ in "kv"]
        cut = lambda t: t[guard:guard + PAGES]
        return ops.KV8Cache(*(cut(t).view(torch.float8_e4m3fn) for t in big), *(cut(t) for t in scales)), big, scales
    def guards_intact(big, scales):
        for t in big:
            assert (t[:guard] == 0x11).all() and (t[guard + PAGES:] == 0x11).all()
        for t in scales:
            assert (t[:guard] == 0.25).all() and (t[guard + PAGES:] == 0.25).all()

    kv = torch.randn(40, 2 * HKV, D, device="cuda").bfloat16()
    k, v = kv[:, :HKV], kv[:, HKV:]
    table = i32([0, 1, 2], [3, 4, 5], [6, 7, 8])
    ctx, cu = i32(3, 0, 20), i32(0, 10, 30, 40)
    for few in (False, True):            # the two append kernels: many tokens, a few per sequence
        kk, vv, c = (k, v, cu) if not few else (k[:3], v[:3], i32(0, 1, 2, 3))
        good, big, scales = fresh()
        ops.kv8_append_(good, kk, vv, table, ctx, c)
        ops.device_status()
        guards_intact(big, scales)
        # a page id outside the pool: that page's tokens are dropped, all others are written
        for bad in (PAGES, -1, 2 ** 31 - 1, -2 ** 31):
            t = table.clone()
            t[1, 0] = bad
            cache, big, scales = fresh()
            expect("page id", lambda: ops.kv8_append_(cache, kk, vv, t, ctx, c))
            guards_intact(big, scales)
            same = [p for p in range(PAGES) if p != 3]
            assert torch.equal(cache.k.view(torch.uint8)[same], good.k.view(torch.uint8)[same])
            assert (cache.k.view(torch.uint8)[3] == 0x11).all() and (cache.k_scale[3] == 0.25).all()
        # lengths that the table cannot hold, negative ones: cut
        for bad in (2 ** 31 - 1, 48, -7):
            cache, big, scales = fresh()
            expect("length of a cached", lambda: ops.kv8_append_(cache, kk, vv, table, i32(3, bad, 20), c))
            guards_intact(big, scales)
            assert torch.equal(cache.k.view(torch.uint8)[:3], good.k.view(torch.uint8)[:3])
        # cu_seqlens past the rows, falling, negative: no row outside k and v is read, nothing outside the pool written
        for bad in (i32(0, 10, 30, 4000), i32(0, 30, 10, 40), i32(-5, 10, 30, 40), i32(0, 2 ** 31 - 1, -2 ** 31, 3)):
            cache, big, scales = fresh()
            expect("cu_seqlens", lambda: ops.kv8_append_(cache, kk, vv, table, i32(3, 0, 5), bad))
            guards_intact(big, scales)

    # attention
    cache, _, _ = fresh()
    ops.kv8_append_(cache, k, v, table, i32(0, 0, 0), cu)
    q = torch.randn(3, 1, 4, D, device="cuda").bfloat16()
    lens = i32(10, 20, 10)
    for wide in (1, 1 << 14):            # the kernel for short sequences, the one for any length
        t0 = torch.cat([table, table.new_full((3, wide), -1)], 1)
        good = ops.sdpa_kv8(q, cache, t0, lens)
        ops.device_status()              # ids behind a sequence's pages are not looked at
        for bad in (PAGES, -1, 2 ** 31 - 1, -2 ** 31):
            t = t0.clone()
            t[1, 1] = bad
            out = expect("page id", lambda: ops.sdpa_kv8(q, cache, t, lens))
            assert torch.equal(out[0], good[0]) and torch.equal(out[2], good[2]) and torch.isfinite(out.float()).all()
        out = expect("length of a cached", lambda: ops.sdpa_kv8(q, cache, t0, i32(10, -3, 10)))
        assert torch.equal(out[0], good[0]) and (out[1] == 0).all() and torch.equal(out[2], good[2])
    tight = table[:, :2].contiguous()
    out = expect("length of a cached", lambda: ops.sdpa_kv8(q, cache, tight, i32(10, 2 ** 31 - 1, 10)))
    assert torch.equal(out[1], ops.sdpa_kv8(q, cache, tight, i32(10, 32, 10))[1])
    print("BOUNDS_OK", checked)
''') % str(ROOT)


@pytest.mark.gpu
@pytest.mark.parametrize("checked", [True, False])
def test_bad_indices_of_the_cache_are_made_safe_and_reported_by_the_checked_build(libemk, checked):
    from deplodock_b200 import build

    if checked:
        build.build(bounds_check=True)
    env = dict(os.environ, EMK_BOUNDS_CHECK="1" if checked else "0")
    res = subprocess.run([sys.executable, "-c", SCRIPT], capture_output=True, text=True, env=env, timeout=600)
    assert res.returncode == 0, res.stdout[-2000:] + res.stderr[-3000:]
    assert f"BOUNDS_OK {checked}" in res.stdout
