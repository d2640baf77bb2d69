"""What the 8-bit serving operators refuse, without a GPU: the C entry points check sizes, alignment and workspaces before
any CUDA call, the Python front end checks tensors before it looks for a device."""

from __future__ import annotations

import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib(libemk):
    from deplodock_b200 import cabi

    return cabi.load_library()


@pytest.fixture(scope="module")
def fake_handle():
    """Zeroed memory in a handle's place: enough for the checks that come before any CUDA call."""
    return ctypes.cast(ctypes.create_string_buffer(8192), ctypes.c_void_p)


P = 1 << 20  # an aligned address that is never followed


def _append(lib, h, **kw):
    a = dict(k=P, v=P, ld_k=256, ld_v=256, kc=P, vc=P, ks=P, vs=P, table=P, ctx=P, cu=P, B=2, T=4, max_pages=2, num_pages=8,
             Hkv=2, page=16, D=128)
    a.update(kw)
    return lib.emk_kv8_append(h, a["k"], a["v"], a["ld_k"], a["ld_v"], a["kc"], a["vc"], a["ks"], a["vs"], a["table"], a["ctx"],
                              a["cu"], a["B"], a["T"], a["max_pages"], a["num_pages"], a["Hkv"], a["page"], a["D"], None)


@pytest.mark.parametrize("kw,want", [
    (dict(k=0), "ARG"), (dict(cu=0), "ARG"), (dict(B=0), "SHAPE"), (dict(T=0), "SHAPE"), (dict(Hkv=0), "SHAPE"),
    (dict(num_pages=1 << 40), "SHAPE"), (dict(page=0), "SHAPE"), (dict(page=24), "SHAPE"), (dict(page=512), "SHAPE"),
    (dict(D=96), "SHAPE"), (dict(D=0), "SHAPE"), (dict(ld_k=248), "SHAPE"), (dict(ld_v=0), "SHAPE"), (dict(ld_k=260), "ALIGN"),
    (dict(k=P + 2), "ALIGN"), (dict(vc=P + 8), "ALIGN"), (dict(ks=P + 2), "ALIGN"), (dict(table=P + 1), "ALIGN")])
def test_append_refuses(lib, fake_handle, kw, want):
    from deplodock_b200 import cabi

    assert _append(lib, fake_handle, **kw) == getattr(cabi, f"EMK_ERR_{want}")
    assert _append(lib, None) == cabi.EMK_ERR_ARG


def _attend(lib, h, **kw):
    a = dict(q=P, ld_q=1024, kc=P, vc=P, ks=P, vs=P, table=P, lens=P, o=P, B=2, Sq=1, Hq=8, Hkv=2, D=128, page=16, max_pages=4,
             num_pages=8, ws=P, ws_bytes=0)
    a.update(kw)
    return lib.emk_sdpa_kv8(h, a["q"], a["ld_q"], a["kc"], a["vc"], a["ks"], a["vs"], a["table"], a["lens"], a["o"], a["B"],
                            a["Sq"], a["Hq"], a["Hkv"], a["D"], a["page"], a["max_pages"], a["num_pages"], 0.1, a["ws"],
                            a["ws_bytes"], None)


@pytest.mark.parametrize("kw,want", [
    (dict(q=0), "ARG"), (dict(ws=0, max_pages=1 << 20), "ARG"), (dict(B=0), "SHAPE"), (dict(Sq=0), "SHAPE"), (dict(Hq=7), "SHAPE"),
    (dict(Hkv=0), "SHAPE"), (dict(page=0), "SHAPE"), (dict(page=48), "SHAPE"), (dict(D=256), "SHAPE"), (dict(D=0), "SHAPE"),
    (dict(max_pages=0), "SHAPE"), (dict(max_pages=1 << 28), "SHAPE"), (dict(ld_q=1016), "SHAPE"), (dict(ld_q=1028), "ALIGN"),
    (dict(q=P + 4), "ALIGN"), (dict(o=P + 8), "ALIGN"), (dict(ws=P + 8), "ALIGN"), (dict(lens=P + 2), "ALIGN"),
    (dict(B=1 << 40), "LIMIT"), (dict(Sq=1 << 31), "LIMIT"), (dict(B=1 << 30, Hkv=8), "LIMIT"), (dict(num_pages=1 << 28), "LIMIT"),
    (dict(max_pages=1 << 26, Hq=256, Hkv=256, ld_q=1 << 15), "LIMIT"), (dict(max_pages=1 << 20), "WORKSPACE")])
def test_attention_refuses(lib, fake_handle, kw, want):
    from deplodock_b200 import cabi

    assert _attend(lib, fake_handle, **kw) == getattr(cabi, f"EMK_ERR_{want}")
    assert _attend(lib, None) == cabi.EMK_ERR_ARG


def test_workspace_of_bad_sizes_is_zero(lib, fake_handle):
    f = lib.emk_sdpa_kv8_workspace_bytes
    assert f(None, 1, 1, 8, 2, 64, 128) == 0
    for sizes in ((0, 1, 8, 2, 64, 128), (1, 1, 7, 2, 64, 128), (1, 1, 8, 0, 64, 128), (1, 1, 8, 2, 0, 128), (1, 1, 8, 2, 64, 96),
                  (1 << 62, 1, 8, 2, 64, 128), (1, 1 << 62, 8, 2, 64, 128)):
        assert f(fake_handle, *sizes) == 0
    assert f(fake_handle, 2, 1, 8, 2, 64, 128) == 0  # short sequences need none
    assert f(fake_handle, 2, 1, 8, 2, 1 << 20, 128) >= 2 * 2 * 8


def _norm(lib, h, **kw):
    a = dict(x=P, r=0, w=P, q=P, s=P, hid=0, rows=2, cols=8, dtype=0)
    a.update(kw)
    return lib.emk_rmsnorm_e4m3(h, a["x"], a["r"], a["w"], a["q"], a["s"], a["hid"], a["rows"], a["cols"], 1e-6, a["dtype"], None)


@pytest.mark.parametrize("kw,want", [
    (dict(x=0), "ARG"), (dict(s=0), "ARG"), (dict(r=P), "ARG"), (dict(hid=P), "ARG"), (dict(rows=0), "SHAPE"), (dict(cols=0), "SHAPE"),
    (dict(cols=1 << 40), "SHAPE"), (dict(dtype=2), "DTYPE"), (dict(x=P + 2), "ALIGN"), (dict(x=P + 1, dtype=1), "ALIGN"),
    (dict(s=P + 2), "ALIGN")])
def test_rmsnorm_refuses(lib, fake_handle, kw, want):
    from deplodock_b200 import cabi

    assert _norm(lib, fake_handle, **kw) == getattr(cabi, f"EMK_ERR_{want}")
    assert _norm(lib, None) == cabi.EMK_ERR_ARG


@pytest.mark.parametrize("kw,want", [
    (dict(x=0), "ARG"), (dict(xs=0), "ARG"), (dict(M=0), "SHAPE"), (dict(N=0), "SHAPE"), (dict(K=0), "SHAPE"),
    (dict(M=1 << 31), "SHAPE"), (dict(K=24), "ALIGN"), (dict(N=12), "ALIGN"), (dict(x=P + 8), "ALIGN"), (dict(ws=P + 4), "ALIGN"),
    (dict(xs=P + 2), "ALIGN"), (dict(M=1 << 30, N=1 << 30), "LIMIT")])
def test_linear_refuses(lib, fake_handle, kw, want):
    from deplodock_b200 import cabi

    a = dict(x=P, xs=P, w=P, ws=P, y=P, M=2, N=16, K=32)
    a.update(kw)
    args = (a["x"], a["xs"], a["w"], a["ws"], a["y"], a["M"], a["N"], a["K"], None)
    assert lib.emk_linear_e4m3(fake_handle, *args) == getattr(cabi, f"EMK_ERR_{want}")
    assert lib.emk_linear_e4m3(None, *args) == cabi.EMK_ERR_ARG


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the message of a machine without a GPU")
def test_no_cpu_fallback():
    from deplodock_b200 import ops

    x = torch.randn(2, 8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.rmsnorm_e4m3(x, torch.ones(8))
    cache = ops.kv8_cache(2, 1, 16, 64, device="cpu")
    lens = torch.zeros(1, dtype=torch.int32)
    table = torch.zeros(1, 1, dtype=torch.int32)
    q = torch.randn(1, 1, 1, 64).bfloat16()
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.sdpa_kv8(q, cache, table, lens)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.kv8_append_(cache, q[0], q[0], table, lens, torch.zeros(2, dtype=torch.int32))


class _On:
    """Stands for a tensor on a device."""

    def __init__(self, device):
        self.device = device

    def get_device(self):
        return self.device


@pytest.mark.parametrize("devices,want", [((0, 0), 0), ((3, None, 3), 3), ((-1, 0), ValueError), ((0, -1), ValueError), ((-1, -1), ValueError),
                                          ((0, 1), ValueError), ((0, 0, 0, -1), ValueError)])
def test_all_tensors_lie_on_one_device(monkeypatch, devices, want):
    from deplodock_b200 import ops

    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    tensors = [None if d is None else _On(d) for d in devices]
    if want is ValueError:
        with pytest.raises(ValueError):
            ops._cuda_index(*tensors)
    else:
        assert ops._cuda_index(*tensors) == want


@pytest.mark.parametrize("devices,dense,want", [((0, 0), (1, 1), 0), ((3, None, 3), (1, 1, 1), 3), ((0, 1), (1, 1), ValueError),
                                                ((-1, 0), (1, 1), ValueError), ((0, 0, -1), (1, 1, 1), ValueError),
                                                ((0, 0), (1, 0), ValueError), ((2, 2, 2), (0, 1, 1), ValueError)])
def test_contiguous_tensors_lie_on_one_device(monkeypatch, devices, dense, want):
    from deplodock_b200 import ops

    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    tensors = [None if d is None else _On(d) for d in devices]
    for t, c in zip(tensors, dense):
        if t is not None:
            t.is_contiguous = lambda c=c: bool(c)
    if want is ValueError:
        with pytest.raises(ValueError):
            ops._contiguous_index(*tensors)
    else:
        assert ops._contiguous_index(*tensors) == want


def test_call_runs_on_the_tensors_device_and_its_stream(monkeypatch):
    """The tensors' device need not be the current one; the stream is that device's."""
    import contextlib

    from deplodock_b200 import cabi, ops

    seen, current = [], [0]

    @contextlib.contextmanager
    def device(idx):
        before, current[0] = current[0], idx
        yield
        current[0] = before

    class Lib:
        @staticmethod
        def emk_thing(*args):
            seen.append((current[0], args))
            return cabi.EMK_OK if args[1] == 7 else cabi.EMK_ERR_SHAPE

    class Handle:
        lib, ptr = Lib, "ptr"

        @staticmethod
        def check(rc, what):
            raise ValueError(f"{what}: {rc}")

    monkeypatch.setattr(ops, "_handles", {2: Handle, 0: Handle})
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda idx: 100 + idx, raising=False)
    ops._call_on(2, "emk_thing", 7)
    ops._call_on(0, "emk_thing", 7)
    assert seen == [(2, ("ptr", 7, 102)), (0, ("ptr", 7, 100))] and current[0] == 0
    with pytest.raises(ValueError, match="emk_thing"):
        ops._call_on(0, "emk_thing", 8)


def test_cache_shapes_are_checked():
    from deplodock_b200 import ops

    cache = ops.kv8_cache(3, 2, 16, 64, device="cpu")
    table, lens = torch.zeros(4, 5, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    assert ops._kv8_sizes(cache, table, lens) == (3, 2, 16, 64, 4, 5)
    with pytest.raises(ValueError):
        ops._kv8_sizes(cache._replace(v=cache.v[:2]), table, lens)
    with pytest.raises(ValueError):
        ops._kv8_sizes(cache._replace(v_scale=cache.v_scale[:, :1]), table, lens)
    with pytest.raises(ValueError):
        ops._kv8_sizes(cache, table[:3], lens)
    with pytest.raises(TypeError):
        ops._kv8_sizes(cache, table, lens.long())
    with pytest.raises(TypeError):
        ops._kv8_sizes(cache._replace(k=cache.k.view(torch.uint8)), table, lens)
