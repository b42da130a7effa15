"""Pointers that the 4-bit cache's calls and the batch sampler are given: alignment without a GPU, and whose memory it is with one."""
import ctypes as C

import numpy as np
import pytest

ONE = C.c_void_p(1 << 20)       # a pointer that no refused call reads


def off(n):
    return C.c_void_p((1 << 20) + n)


def append(L, q=ONE, out=ONE, k=ONE, v=ONE, tab=ONE, rope=64, caches=ONE, pos=ONE):
    return L.wl_kv4_append(q, out, k, v, 4, 8, 2, 64, tab, rope, 0, caches, pos, 100, None)


def read(L, caches=ONE, pos=ONE, k=ONE, v=ONE):
    return L.wl_kv4_read(caches, pos, 4, 2, 64, 100, k, v, None)


def attend(L, q=ONE, caches=ONE, pos=ONE, out=ONE, ws=ONE):
    return L.wl_kv4_attention(q, 4, 1, 8, 2, 64, 1.0, caches, pos, 100, 0, 0, out, ws, 1 << 30, None)


def sample(L, x=ONE, opts=ONE, ids=ONE):
    return L.wl_sample_rows(x, 10, 10, 1, opts, ids, None)


def init(L, ws=ONE):
    return L.wl_kv4_workspace_init(ws, 1 << 30, None)


MISALIGNED = [(append, dict(q=8)), (append, dict(out=4)), (append, dict(k=8)), (append, dict(v=8)), (append, dict(tab=2)),
              (append, dict(caches=4)), (append, dict(pos=2)), (read, dict(caches=4)), (read, dict(pos=2)), (read, dict(k=8)),
              (read, dict(v=2)), (attend, dict(q=4)), (attend, dict(caches=4)), (attend, dict(pos=1)), (attend, dict(out=8)),
              (attend, dict(ws=8)), (sample, dict(x=2)), (sample, dict(opts=4)), (sample, dict(ids=2)), (init, dict(ws=4))]


@pytest.mark.parametrize("call,bad", MISALIGNED, ids=lambda x: x.__name__ if callable(x) else next(iter(x)))
def test_misaligned_pointers_are_refused_before_any_device_work(wl, call, bad):
    assert call(wl.lib(), **{k: off(n) for k, n in bad.items()}) == wl.WL_EINVAL
    assert b"aligned" in wl.lib().wl_last_error()


@pytest.mark.gpu
def test_host_memory_is_refused(wl):
    """Every pointer in turn is pageable host memory; the call returns before anything is launched."""
    from gpu_util import empty, ptr
    buf = empty(1 << 16)
    L, there = wl.lib(), ptr(buf)
    page = np.zeros(1 << 12, np.uint8)
    here = C.c_void_p((page.ctypes.data + 255) & ~255)
    for call, names in ((append, ("q", "out", "k", "v", "tab", "caches", "pos")), (read, ("caches", "pos", "k", "v")),
                        (attend, ("q", "caches", "pos", "out", "ws")), (sample, ("x", "opts", "ids")), (init, ("ws",))):
        args = call.__code__.co_varnames[1:call.__code__.co_argcount]
        for n in names:
            st = call(L, **{a: (here if a == n else there) for a in args if a != "rope"})
            assert st == wl.WL_EINVAL and b"not device memory" in L.wl_last_error(), (call.__name__, n)


@pytest.mark.gpu
def test_pinned_tables_and_any_aligned_rope_table_serve(wl):
    """Positions and cache pointers in pinned host memory, ids written to it, and a rope table aligned to 4 bytes only."""
    import kv4_ref as R
    from gpu_util import dev, empty, host, ptr, torch_cuda
    from test_gpu_kv4 import Cache, check, table, workspace
    torch = torch_cuda()
    rng = np.random.default_rng(4)
    L, heads, kv_heads, hd, cap = wl.lib(), 8, 2, 64, 32
    c = Cache(1, kv_heads, hd, cap, fill=0)
    tab = table(cap, hd)
    q, k, v = (rng.standard_normal((20, n, hd)).astype(np.float32) for n in (heads, kv_heads, kv_heads))
    rows = torch.full((20,), c.t.data_ptr(), dtype=torch.int64).pin_memory()
    pos = torch.arange(20, dtype=torch.int32).pin_memory()
    room = dev(np.concatenate((np.zeros(1, np.float32), tab.reshape(-1))))
    out, dq, dk, dv = empty((20, heads, hd)), dev(q), dev(k), dev(v)
    wl.check(L.wl_kv4_append(ptr(dq), ptr(out), ptr(dk), ptr(dv), 20, heads, kv_heads, hd, C.c_void_p(room.data_ptr() + 4), hd, 1,
                             ptr(rows), ptr(pos), cap, None))
    raw = c.host()
    kc, kd = R.quantise(R.rotate(k, tab, range(20), hd, True))
    vc, vd = R.quantise(v)
    want = np.zeros_like(raw)
    for p in range(20):
        R.write(want[0], kv_heads, hd, p, kc[p], kd[p], False)
        R.write(want[0], kv_heads, hd, p, vc[p], vd[p], True)
    assert np.array_equal(raw, want)
    ws = workspace(wl, 20, 1, heads, kv_heads, hd, cap)
    o = empty((20, heads, hd))
    wl.check(L.wl_kv4_attention(ptr(out), 20, 1, heads, kv_heads, hd, hd ** -0.5, ptr(rows), ptr(pos), cap, 0, 0, ptr(o), ptr(ws), ws.numel(), None))
    check(host(o), host(out), raw, kv_heads, hd, [0] * 20, list(range(20)))
    x = dev(np.array([[0, 3, 1]], np.float32))
    opts = dev(np.frombuffer(wl.SampleOpts(0.0, 1.0, 0.0, 0.5, 0), np.uint8).copy())
    ids = torch.full((1,), -7, dtype=torch.int32).pin_memory()
    wl.check(L.wl_sample_rows(ptr(x), 3, 3, 1, ptr(opts), ptr(ids), None))
    torch.cuda.synchronize()
    assert ids.item() == 1
