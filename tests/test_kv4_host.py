"""The 4-bit KV cache's host side without a GPU: sizes, refusals, and the test reference against itself."""
import ctypes as C

import numpy as np
import pytest

import kv4_ref as R

ONE = C.c_void_p(16)        # a pointer that no refused call reads


def test_sizes(wl):
    n = C.c_int64()
    for kv_heads, hd, p in ((8, 128, 1), (8, 128, 16), (8, 128, 17), (1, 64, 100), (3, 96, 40), (2, 256, 2 ** 31 - 1)):
        wl.check(wl.lib().wl_kv4_bytes(kv_heads, hd, p, C.byref(n)))
        assert n.value == R.cache_bytes(kv_heads, hd, p)
    for bad in ((0, 128, 16), (8, 0, 16), (8, 128, 0), (8, 128, -1), (8, 128, 2 ** 31)):
        with pytest.raises(wl.ArgumentError):
            wl.check(wl.lib().wl_kv4_bytes(*bad, C.byref(n)))
    for hd in (32, 80, 120, 192, 512):
        with pytest.raises(wl.NotSupportedError):
            wl.check(wl.lib().wl_kv4_bytes(8, hd, 16, C.byref(n)))
    assert wl.lib().wl_kv4_bytes(8, 128, 16, None) == wl.WL_EINVAL


def test_workspace_grows_with_the_ranges_only(wl):
    n = C.c_int64()

    def need(*a):
        wl.check(wl.lib().wl_kv4_workspace_bytes(*a, C.byref(n)))
        return n.value
    small = need(1, 1, 8, 8, 64, 16, 0, 0)
    assert need(0, 1, 8, 8, 64, 16, 0, 0) == small == need(64, 1, 8, 8, 64, 256, 0, 0)
    assert need(1, 1, 8, 8, 64, 100000, 0, 0) > small
    assert need(1, 1, 8, 8, 64, 100000, 64, 4) == small             # a window of a few tiles: one range
    assert need(65, 1, 8, 8, 64, 100000, 0, 0) == small             # many rows: one range each
    assert need(64, 1, 64, 8, 128, 2 ** 31 - 1, 0, 0) < 2 ** 28


def test_refusals(wl):
    L = wl.lib()
    ok = dict(T=4, runs=1, heads=8, kv=2, hd=64, cap=100, window=0, sinks=0, ws=1 << 30)

    def attend(q=ONE, caches=ONE, pos=ONE, out=ONE, ws_ptr=ONE, **kw):
        a = {**ok, **kw}
        return L.wl_kv4_attention(q, a["T"], a["runs"], a["heads"], a["kv"], a["hd"], 1.0, caches, pos, a["cap"], a["window"],
                                  a["sinks"], out, ws_ptr, a["ws"], None)
    for kw in (dict(T=-1), dict(runs=0), dict(runs=3), dict(heads=0), dict(kv=0), dict(cap=0), dict(cap=2 ** 31), dict(window=-1),
               dict(sinks=-1), dict(ws=1024), dict(q=None), dict(caches=None), dict(pos=None), dict(out=None), dict(ws_ptr=None)):
        assert attend(**kw) == wl.WL_EINVAL, kw
        assert b"wl_kv4_attention" in L.wl_last_error()
    for kw in (dict(heads=9), dict(hd=80), dict(hd=32)):
        assert attend(**kw) == wl.WL_EUNSUPPORTED, kw
    assert attend(T=0) == wl.WL_OK

    def append(q=ONE, out=ONE, k=ONE, v=ONE, T=4, heads=8, kv=2, hd=64, tab=ONE, rope=64, caches=ONE, pos=ONE, cap=100):
        return L.wl_kv4_append(q, out, k, v, T, heads, kv, hd, tab, rope, 0, caches, pos, cap, None)
    for kw in (dict(T=-1), dict(rope=-2), dict(rope=3), dict(rope=66), dict(q=None), dict(out=None), dict(k=None), dict(v=None),
               dict(tab=None), dict(caches=None), dict(pos=None), dict(cap=0)):
        assert append(**kw) == wl.WL_EINVAL, kw
    assert append(hd=48) == wl.WL_EUNSUPPORTED
    assert append(T=0) == wl.WL_OK and append(T=0, rope=0, tab=None) == wl.WL_OK
    for kw in (dict(T=-1), dict(k=None), dict(v=None)):
        a = {**dict(T=4, k=ONE, v=ONE), **kw}
        assert L.wl_kv4_read(ONE, ONE, a["T"], 2, 64, 100, a["k"], a["v"], None) == wl.WL_EINVAL
    assert L.wl_kv4_workspace_init(None, 1 << 30, None) == wl.WL_EINVAL
    assert L.wl_kv4_workspace_init(ONE, 100, None) == wl.WL_EINVAL


def test_the_reference_reads_what_it_writes():
    rng = np.random.default_rng(0)
    for kv_heads, hd in ((2, 64), (1, 96), (2, 128), (1, 256)):
        raw = np.zeros(R.cache_bytes(kv_heads, hd, 20), np.uint8)
        x = [rng.standard_normal((20, kv_heads, hd)) for _ in range(2)]
        for is_v in (False, True):
            c, d = R.quantise(x[is_v])
            for p in range(20):
                R.write(raw, kv_heads, hd, p, c[p], d[p], is_v)
        used = np.zeros(raw.size, bool)
        for is_v in (False, True):
            y = R.read(raw, kv_heads, hd, 20, is_v)
            # half a step of the block's scale (an eighth of its largest value), a whole one at the end that 15 cuts off
            step = np.repeat(np.abs(x[is_v]).reshape(20, kv_heads, -1, 32).max(-1), 32, -1) / 8
            assert (np.abs(y - x[is_v]) <= step * (1 + 2 ** -9)).all()
            for p in range(16):
                code, shift, sc = R._places(hd, p, is_v)
                used[code] = used[sc] = used[sc + 1] = True
        assert used[:R.tile_bytes(hd)].all()


def test_sampler_refusals(wl):
    L = wl.lib()
    for a in ((None, 10, 10, 1, ONE, ONE), (ONE, 10, 10, 1, None, ONE), (ONE, 10, 10, 1, ONE, None), (ONE, 9, 10, 1, ONE, ONE),
              (ONE, 10, 0, 1, ONE, ONE), (ONE, 10, 10, -1, ONE, ONE)):
        assert L.wl_sample_rows(*a, None) == wl.WL_EINVAL, a
    assert L.wl_sample_rows(ONE, 10, 10, 0, ONE, ONE, None) == wl.WL_OK
    assert L.wl_forward_sample_opts(None, None, None, 1, 0, None, None, None, wl.PROGRESS(), None) == wl.WL_EINVAL
    assert L.wl_forward_batch_sample_opts(None, None, None, 1, None, None, None, wl.PROGRESS(), None) == wl.WL_EINVAL
    o = wl.SampleOpts(1.0, 1.0, 0.0, 1.0, 0)
    out = (C.c_int32 * 1)()
    assert L.wl_forward_sample_opts(None, None, None, 1, 0, C.byref(o), out, None, wl.PROGRESS(), None) == wl.WL_EINVAL
    assert b"draw" in L.wl_last_error()


def test_model_options_are_refused_before_any_device_work(wl):
    from windlass_b200.transformer import config0_spec, synth_spec
    L = wl.lib()

    def open_(spec=None, **kw):
        h = C.c_void_p()
        return L.wl_open_synthetic(C.byref(spec or config0_spec()), C.byref(wl.options(**kw)), C.byref(h))
    assert open_(kv_type=3) == wl.WL_EUNSUPPORTED and b"kv_type" in L.wl_last_error()
    assert open_(attn_window=64) == wl.WL_EUNSUPPORTED and b"attn_window" in L.wl_last_error()
    assert open_(kv_type=2, attn_window=-1) == wl.WL_EINVAL
    assert open_(kv_type=2, attn_window=64, attn_sinks=-1) == wl.WL_EINVAL
    assert open_(kv_type=2, attn_sinks=4) == wl.WL_EINVAL
    spec = synth_spec("llama", 1, 320, 4, 4, 80, 256, 512, 512)
    assert open_(spec, kv_type=2) == wl.WL_EUNSUPPORTED and b"head_dim" in L.wl_last_error()
