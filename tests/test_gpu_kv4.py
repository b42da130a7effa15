"""The 4-bit KV cache (wl_kv4_append, wl_kv4_read, wl_kv4_attention) against numpy in 64 bits (kv4_ref.py)."""
import ctypes as C

import numpy as np
import pytest

import kv4_ref as R
from gpu_util import dev, empty, host, ptr, torch_cuda

pytestmark = pytest.mark.gpu

SHAPES = [(8, 8, 64), (8, 2, 64), (6, 3, 96), (16, 2, 128), (10, 2, 128), (8, 1, 256), (32, 2, 64)]


class Cache:
    """n caches of `positions` positions, filled with `fill` bytes, and the pointer table of rows over them."""

    def __init__(self, n, kv_heads, hd, positions, fill=0xFF):
        torch = torch_cuda()
        self.kv_heads, self.hd, self.positions = kv_heads, hd, positions
        self.bytes = R.cache_bytes(kv_heads, hd, positions)
        self.t = torch.full((n, self.bytes), fill, dtype=torch.uint8, device="cuda")

    def rows(self, seq):
        return dev(np.array([self.t[s].data_ptr() if s >= 0 else 0 for s in seq], dtype=np.int64))

    def host(self):
        return host(self.t)


def table(positions, rope, seed=0):
    i = np.arange(rope // 2)
    a = np.arange(positions)[:, None] * 0.5 * 10000.0 ** (-2 * i / max(1, rope))
    return np.stack((np.cos(a), np.sin(a)), -1).astype(np.float32)


def append(wl, cache, seq, pos, q, k, v, tab, rope, neox, in_place=False, stream=None):
    T, heads, hd = q.shape
    dq, dk, dv, dt = dev(q), dev(k), dev(v), dev(tab if tab.size else np.zeros((1, 1, 2), np.float32))
    out = dq if in_place else empty((T, heads, hd))
    rows, dp = cache.rows(seq), dev(np.array(pos, np.int32))
    wl.check(wl.lib().wl_kv4_append(ptr(dq), ptr(out), ptr(dk), ptr(dv), T, heads, cache.kv_heads, hd, ptr(dt), rope, int(neox),
                                    ptr(rows), ptr(dp), cache.positions, stream))
    return host(out)


def workspace(wl, T, runs, heads, kv_heads, hd, capacity, window=0, sinks=0):
    n = C.c_int64()
    wl.check(wl.lib().wl_kv4_workspace_bytes(T, runs, heads, kv_heads, hd, capacity, window, sinks, C.byref(n)))
    ws = empty(n.value, "uint8")
    ws.fill_(0x7F)
    wl.check(wl.lib().wl_kv4_workspace_init(ptr(ws), n.value, None))
    return ws


def attend(wl, cache, seq, pos, q, window=0, sinks=0, runs=1, scale=None, ws=None):
    T, heads, hd = q.shape
    dq, out = dev(q), empty((T, heads, hd))
    rows, dp = cache.rows(seq), dev(np.array(pos, np.int32))
    ws = workspace(wl, T, runs, heads, cache.kv_heads, hd, cache.positions, window, sinks) if ws is None else ws
    wl.check(wl.lib().wl_kv4_attention(ptr(dq), T, runs, heads, cache.kv_heads, hd, hd ** -0.5 if scale is None else scale, ptr(rows),
                                       ptr(dp), cache.positions, window, sinks, ptr(out), ptr(ws), ws.numel(), None))
    return host(out)


def filled(rng, n, kv_heads, hd, positions, lengths, vscale=1.0):
    """Caches whose first lengths[i] positions hold random values; what lies behind reads as NaN (0xFF bytes)."""
    c = Cache(n, kv_heads, hd, positions)
    raw = c.host().copy()
    for i, ln in enumerate(lengths):
        kc, kd = R.quantise(rng.standard_normal((ln, kv_heads, hd)) * (1 + 3 * (rng.random(hd) > 0.95)))
        vc, vd = R.quantise(rng.standard_normal((ln, kv_heads, hd)) * vscale)
        for p in range(ln):
            R.write(raw[i], kv_heads, hd, p, kc[p], kd[p], False)
            R.write(raw[i], kv_heads, hd, p, vc[p], vd[p], True)
    c.t.copy_(dev(raw))
    return c, raw


def check(out, q, raw, kv_heads, hd, seq, pos, window=0, sinks=0, scale=None):
    kv = {}
    for t, (s, p) in enumerate(zip(seq, pos)):
        if p < 0:
            assert (out[t] == 0).all(), t
            continue
        if s not in kv:
            n = max(pp for ss, pp in zip(seq, pos) if ss == s) + 1
            kv[s] = [R.read(raw[s], kv_heads, hd, n, e) for e in (False, True)]
        want, bound = R.attention(q[t], *kv[s], p, hd ** -0.5 if scale is None else scale, window, sinks)
        off = np.abs(out[t] - want).max(-1)
        assert (off <= bound).all(), (t, p, float((off / bound).max()))


@pytest.mark.parametrize("heads,kv_heads,hd", SHAPES)
@pytest.mark.parametrize("neox", [False, True])
def test_append_writes_the_codes_of_64_bits(wl, heads, kv_heads, hd, neox):
    rng = np.random.default_rng(hd + neox)
    cap = 50
    for rope, in_place in ((hd, True), (hd // 2, False), (18, True), (0, False)):
        seq, pos = [0, 0, 1, 2, 1, 0, 2], [0, 33, 17, 49, 16, 15, -1]
        T = len(seq)
        q, k, v = (rng.standard_normal((T, n, hd)).astype(np.float32) for n in (heads, kv_heads, kv_heads))
        k[1, 0, :32] = 0                                  # a block of zeros
        k[2, 0, 5], k[2, 0, 7] = 9.0, -9.0                # a pair of largest values
        v[3, 0, 32:64] *= 1e-9                            # a scale below fp16's smallest
        v[4, 0, 0] = np.inf
        v[5, 0, 40] = np.nan
        v[0, 0, 3] = 1e7                                  # a scale past fp16's largest
        tab = table(cap, rope)
        c = Cache(3, kv_heads, hd, cap, fill=0x5A)
        want = c.host().copy()
        got_q = append(wl, c, seq, pos, q, k, v, tab, rope, neox, in_place)
        kr = R.rotate(k, tab, [max(p, 0) for p in pos], rope, neox)
        kc, kd = R.quantise(kr)
        vc, vd = R.quantise(v)
        for t in range(T):
            if pos[t] >= 0:
                R.write(want[seq[t]], kv_heads, hd, pos[t], kc[t], kd[t], False)
                R.write(want[seq[t]], kv_heads, hd, pos[t], vc[t], vd[t], True)
        assert np.array_equal(c.host(), want), (rope, int((c.host() != want).sum()))
        qr = R.rotate(q, tab, [max(p, 0) for p in pos], rope, neox)
        # two products and a sum in fp32: three half steps of at most |x0| + |x1|
        for t in range(T - 1):
            assert np.abs(got_q[t] - qr[t]).max() <= 3 * 2.0 ** -24 * 2 * np.abs(q[t]).max()
        if in_place:
            assert np.array_equal(got_q[T - 1], q[T - 1])       # padding: left as it was


def test_read_gives_the_held_values_and_append_refuses_rows_past_the_cache(wl):
    rng = np.random.default_rng(3)
    for heads, kv_heads, hd in SHAPES:
        cap = 40
        c, raw = filled(rng, 2, kv_heads, hd, cap, [40, 23])
        seq, pos = [0, 1, 0, 1, -1, 0], [39, 22, 0, -1, 3, 40]
        rows, dp = c.rows(seq), dev(np.array(pos, np.int32))
        k, v = empty((6, kv_heads, hd), "float16"), empty((6, kv_heads, hd), "float16")
        wl.check(wl.lib().wl_kv4_read(ptr(rows), ptr(dp), 6, kv_heads, hd, cap, ptr(k), ptr(v), None))
        for got, is_v in ((host(k), False), (host(v), True)):
            for t in range(3):
                assert np.array_equal(got[t], R.read(raw[seq[t]], kv_heads, hd, 40, is_v)[pos[t]].astype(np.float16))
            assert (got[3] == 0).all() and np.isnan(got[4:]).all()
        x = rng.standard_normal((3, heads, hd)).astype(np.float32)
        y = x[:, :kv_heads].copy()
        append(wl, c, [0, -1, 1], [40, 3, 2 ** 31 - 1], x, y, y, table(cap, hd), hd, True)
        assert np.array_equal(c.host(), raw)


@pytest.mark.parametrize("heads,kv_heads,hd", SHAPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (20, 0), (16, 3), (33, 40), (100, 1)])
def test_attention_of_single_rows(wl, heads, kv_heads, hd, window, sinks):
    rng = np.random.default_rng(heads * hd + window)
    lengths = [1, 2, 15, 16, 17, 33, 64, 301, 700]
    c, raw = filled(rng, len(lengths), kv_heads, hd, 712, lengths)
    seq = list(range(len(lengths))) + [0]
    pos = [n - 1 for n in lengths] + [-1]
    q = rng.standard_normal((len(seq), heads, hd)).astype(np.float32) * 2
    out = attend(wl, c, seq, pos, q, window, sinks)
    check(out, q, raw, kv_heads, hd, seq, pos, window, sinks)
    # alone: the same bits
    for t in (0, 5, 8):
        one = attend(wl, c, seq[t:t + 1], pos[t:t + 1], q[t:t + 1], window, sinks)
        assert np.array_equal(one[0].view(np.uint32), out[t].view(np.uint32)), t
    assert wl.lib().wl_kernel_status(0) == 0


@pytest.mark.parametrize("heads,kv_heads,hd", SHAPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (7, 0), (40, 5)])
def test_attention_of_runs(wl, heads, kv_heads, hd, window, sinks):
    rng = np.random.default_rng(heads + hd + window)
    for rows, start, cap in ((9, 0, 9), (37, 0, 64), (70, 333, 403)):
        lengths = [start + rows, max(rows, start + rows - 5)]
        c, raw = filled(rng, 2, kv_heads, hd, cap, lengths)
        seq = [0] * rows + [1] * rows
        pos = [start + r for r in range(rows)] + [lengths[1] - rows + r for r in range(rows)]
        pos[3] = -1                                        # padding in the middle of a run
        q = rng.standard_normal((2 * rows, heads, hd)).astype(np.float32) * 2
        out = attend(wl, c, seq, pos, q, window, sinks, runs=rows)
        check(out, q, raw, kv_heads, hd, seq, pos, window, sinks)
    assert wl.lib().wl_kernel_status(0) == 0


@pytest.mark.parametrize("rows", [16, 17, 31, 64, 129, 257])
@pytest.mark.parametrize("heads,kv_heads,hd,window", [(4, 4, 64, 0), (8, 1, 128, 0), (3, 3, 128, 130), (12, 2, 64, 50), (4, 2, 96, 0),
                                                      (2, 2, 256, 90)])
def test_attention_of_runs_of_every_kernel(wl, rows, heads, kv_heads, hd, window):
    """Rows by themselves, one block of queries, blocks in pairs with and without a last one of its own; no, one and many steps."""
    rng = np.random.default_rng(rows * 7 + hd + heads)
    for start in (0, 700):
        c, raw = filled(rng, 2, kv_heads, hd, 1024, [start + rows, 1000])
        seq = [0] * rows + [1] * rows
        pos = [start + r for r in range(rows)] + [int(p) for p in rng.integers(0, 1000, rows)]
        pos[rows + 1] = -1
        q = rng.standard_normal((2 * rows, heads, hd)).astype(np.float32) * 2
        out = attend(wl, c, seq, pos, q, window, 3, runs=rows)
        check(out, q, raw, kv_heads, hd, seq, pos, window, 3)
    assert wl.lib().wl_kernel_status(0) == 0


@pytest.mark.parametrize("heads,kv_heads,hd", [(16, 2, 128), (8, 2, 64), (20, 4, 128), (7, 7, 64)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 17)])
def test_attention_of_long_runs(wl, heads, kv_heads, hd, window, sinks):
    """Several CTAs of queries a run, several steps of positions, ranges of a long cache joined, positions in any order."""
    rng = np.random.default_rng(heads + window)
    for rows, start, shuffle in ((130, 0, False), (130, 1000, True), (97, 2611, False)):
        c, raw = filled(rng, 1, kv_heads, hd, start + rows + 5, [start + rows])
        pos = [start + r for r in range(rows)]
        if shuffle:
            rng.shuffle(pos)
            pos[17] = -1
        q = rng.standard_normal((rows, heads, hd)).astype(np.float32) * 2
        out = attend(wl, c, [0] * rows, pos, q, window, sinks, runs=rows)
        check(out, q, raw, kv_heads, hd, [0] * rows, pos, window, sinks)
        again = attend(wl, c, [0] * rows, pos, q, window, sinks, runs=rows)
        assert np.array_equal(out.view(np.uint32), again.view(np.uint32))
    assert wl.lib().wl_kernel_status(0) == 0


def test_refused_rows_give_nan_and_leave_the_others(wl):
    rng = np.random.default_rng(8)
    heads, kv_heads, hd = 8, 2, 128
    c, raw = filled(rng, 2, kv_heads, hd, 100, [100, 100])
    q = rng.standard_normal((4, heads, hd)).astype(np.float32)
    out = attend(wl, c, [0, 1, -1, 1], [99, 100, 5, 50], q)
    check(out[[0, 3]], q[[0, 3]], raw, kv_heads, hd, [0, 1], [99, 50])
    assert np.isnan(out[1]).all() and np.isnan(out[2]).all()
    q = rng.standard_normal((12, heads, hd)).astype(np.float32)
    pos = list(range(88, 100))
    pos[4], pos[7] = 100, -3
    out = attend(wl, c, [0] * 12, pos, q, runs=12)
    keep = [t for t in range(12) if t not in (4, 7)]
    check(out[keep], q[keep], raw, kv_heads, hd, [0] * 10, [pos[t] for t in keep])
    assert np.isnan(out[4]).all() and (out[7] == 0).all()


@pytest.mark.parametrize("runs,heads,hd", [(1, 8, 64), (20, 8, 64), (20, 32, 64), (20, 16, 128)])
def test_a_nan_reaches_only_the_rows_that_see_it(wl, runs, heads, hd):
    rng = np.random.default_rng(runs)
    kv_heads = 2
    c, raw = filled(rng, 1, kv_heads, hd, 64, [60])
    bad = 47
    R.write(raw[0], kv_heads, hd, bad, np.zeros((kv_heads, hd), int), np.full((kv_heads, hd // 32), np.nan, np.float16), True)
    c.t.copy_(dev(raw))
    pos = list(range(40, 60))
    q = rng.standard_normal((20, heads, hd)).astype(np.float32)
    out = attend(wl, c, [0] * 20, pos, q, window=6, runs=runs)
    clean = [t for t in range(20) if not pos[t] - 6 < bad <= pos[t]]
    assert len(clean) == 14
    check(out[clean], q[clean], raw, kv_heads, hd, [0] * len(clean), [pos[t] for t in clean], window=6)
    hit = [t for t in range(20) if t not in clean]
    assert np.isnan(out[hit]).all()


@pytest.mark.parametrize("vscale", [1e-6, 1e-2, 300.0, 4e5])
@pytest.mark.parametrize("runs", [1, 24])
def test_values_of_any_scale(wl, vscale, runs):
    """The values' scales are brought into fp16's range by a power of two that follows the largest seen."""
    rng = np.random.default_rng(5)
    heads, kv_heads, hd = 8, 1, 128
    c, raw = filled(rng, 1, kv_heads, hd, 300, [300], vscale)
    tail, d = R.quantise(rng.standard_normal((40, kv_heads, hd)) * vscale * 30)     # larger ones late
    for i in range(40):
        R.write(raw[0], kv_heads, hd, 230 + i, tail[i], d[i], True)
    c.t.copy_(dev(raw))
    pos = list(range(300 - runs, 300))
    q = rng.standard_normal((runs, heads, hd)).astype(np.float32)
    out = attend(wl, c, [0] * runs, pos, q, runs=runs)
    check(out, q, raw, kv_heads, hd, [0] * runs, pos)


@pytest.mark.parametrize("qscale", [0.0, 1e-30, 1e-4, 40.0])
def test_queries_of_any_scale(wl, qscale):
    rng = np.random.default_rng(6)
    heads, kv_heads, hd = 16, 2, 128
    c, raw = filled(rng, 1, kv_heads, hd, 200, [200])
    q = (rng.standard_normal((1, heads, hd)) * qscale).astype(np.float32)
    check(attend(wl, c, [0], [199], q), q, raw, kv_heads, hd, [0], [199])
    q = (rng.standard_normal((30, heads, hd)) * qscale).astype(np.float32)
    pos = list(range(170, 200))
    check(attend(wl, c, [0] * 30, pos, q, runs=30), q, raw, kv_heads, hd, [0] * 30, pos)


def test_a_long_cache_past_32_bit_offsets(wl):
    """A row at the end of a cache of more than 2^31 bytes, its window and its sinks 2.4 GB apart."""
    torch = torch_cuda()
    rng = np.random.default_rng(9)
    heads, kv_heads, hd, n = 16, 8, 128, 2_100_003
    c = Cache(1, kv_heads, hd, n)
    assert c.bytes > 2 ** 31
    tab = np.zeros((1, 1, 2), np.float32)
    seen = list(range(4)) + list(range(n - 40, n))
    x = rng.standard_normal((len(seen), heads, hd)).astype(np.float32)
    y, z = x[:, :kv_heads].copy(), x[:, kv_heads:].copy()
    append(wl, c, [0] * len(seen), seen, x, y, z, tab, 0, False)
    q = rng.standard_normal((1, heads, hd)).astype(np.float32)
    out = attend(wl, c, [0], [n - 1], q, window=40, sinks=4)
    k, v = (np.float64(1) * (cc - 8) * np.repeat(d.astype(np.float64), 32, -1) for cc, d in (R.quantise(y), R.quantise(z)))
    want, bound = R.attention(q[0], k, v, len(seen) - 1, hd ** -0.5)
    assert (np.abs(out[0] - want).max(-1) <= bound).all()
    del c
    torch.cuda.empty_cache()


def test_captured_and_replayed_on_a_stream_of_its_own(wl):
    """Append and attention captured into a graph on a stream, replayed over moving positions; and two graphs with a
    workspace each on two streams at once."""
    torch = torch_cuda()
    rng = np.random.default_rng(12)
    heads, kv_heads, hd, cap = 16, 2, 128, 900
    lib = wl.lib()
    caches = [filled(rng, 1, kv_heads, hd, cap, [700]) for _ in range(2)]
    tab = table(cap, hd)
    dt = dev(tab)
    sets = []
    for c, raw in caches:
        st = torch.cuda.Stream()
        d = dict(q=empty((1, heads, hd)), o=empty((1, heads, hd)), qr=empty((1, heads, hd)), k=empty((1, kv_heads, hd)),
                 v=empty((1, kv_heads, hd)), pos=dev(np.zeros(1, np.int32)), rows=c.rows([0]), st=st,
                 ws=workspace(wl, 1, 1, heads, kv_heads, hd, cap))

        def call(d=d, c=c):
            s = C.c_void_p(d["st"].cuda_stream)
            wl.check(lib.wl_kv4_append(ptr(d["q"]), ptr(d["qr"]), ptr(d["k"]), ptr(d["v"]), 1, heads, kv_heads, hd, ptr(dt), hd, 1,
                                       ptr(d["rows"]), ptr(d["pos"]), cap, s))
            wl.check(lib.wl_kv4_attention(ptr(d["qr"]), 1, 1, heads, kv_heads, hd, hd ** -0.5, ptr(d["rows"]), ptr(d["pos"]), cap, 0, 0,
                                          ptr(d["o"]), ptr(d["ws"]), d["ws"].numel(), s))
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=st):
            call()
        d["g"] = g
        sets.append(d)
    for p in (700, 701, 702):
        x = []
        for d in sets:
            q, k, v = (rng.standard_normal((1, n, hd)).astype(np.float32) for n in (heads, kv_heads, kv_heads))
            x.append((q, k, v))
            for n, y in (("q", q), ("k", k), ("v", v), ("pos", np.array([p], np.int32))):
                d[n].copy_(dev(y))
        torch.cuda.synchronize()
        for d in sets:
            with torch.cuda.stream(d["st"]):
                d["g"].replay()
        torch.cuda.synchronize()
        for d, (c, raw), (q, k, v) in zip(sets, caches, x):
            kc, kd = R.quantise(R.rotate(k, tab, [p], hd, True))
            vc, vd = R.quantise(v)
            R.write(raw[0], kv_heads, hd, p, kc[0], kd[0], False)
            R.write(raw[0], kv_heads, hd, p, vc[0], vd[0], True)
            assert np.array_equal(c.host(), raw)
            check(host(d["o"]), host(d["qr"]), raw, kv_heads, hd, [0], [p])


@pytest.mark.parametrize("heads,kv_heads,hd", [(8, 2, 64), (8, 2, 128), (4, 2, 96), (4, 2, 256)])
@pytest.mark.parametrize("rows,start,cap", [(20, 200, 220), (40, 900, 1024), (80, 1900, 2000), (9, 50, 64)])
def test_padding_rows_that_hold_nan_give_zeros(wl, heads, kv_heads, hd, rows, start, cap):
    """The queries of padding rows may hold anything, whatever kernel and number of ranges; a refused row's stays NaN."""
    rng = np.random.default_rng(hd + rows)
    c, raw = filled(rng, 1, kv_heads, hd, cap, [start + rows])
    pos = [start + r for r in range(rows)]
    pos[0] = pos[5] = pos[rows - 1] = -1
    pos[7] = cap
    q = rng.standard_normal((rows, heads, hd)).astype(np.float32)
    q[[0, 7]], q[5], q[rows - 1] = np.nan, np.inf, 3e38
    out = attend(wl, c, [0] * rows, pos, q, runs=rows)
    keep = [t for t in range(rows) if t != 7]
    check(out[keep], q[keep], raw, kv_heads, hd, [0] * len(keep), [pos[t] for t in keep])
    assert np.isnan(out[7]).all()


def test_prompts_on_two_streams_and_replayed(wl):
    """Prompts of two shapes (pairs of CTAs and single ones, several ranges each) and a decode step captured on streams of their
    own and replayed at once, a workspace each: the bits of calls made alone."""
    torch = torch_cuda()
    rng = np.random.default_rng(21)
    lib, sets = wl.lib(), []
    for rows, heads, kv_heads, hd, start, window in ((130, 8, 2, 128, 1500, 0), (40, 2, 2, 64, 900, 300), (1, 8, 2, 128, 1700, 0)):
        c, raw = filled(rng, 1, kv_heads, hd, 1800, [start + rows])
        pos = [start + r for r in range(rows)]
        q = rng.standard_normal((rows, heads, hd)).astype(np.float32)
        want = attend(wl, c, [0] * rows, pos, q, window, 4, runs=rows)
        check(want, q, raw, kv_heads, hd, [0] * rows, pos, window, 4)
        st = torch.cuda.Stream()
        d = dict(c=c, q=dev(q), o=empty((rows, heads, hd)), rows=c.rows([0] * rows), pos=dev(np.array(pos, np.int32)), st=st, want=want,
                 ws=workspace(wl, rows, rows, heads, kv_heads, hd, 1800, window, 4), g=torch.cuda.CUDAGraph())
        torch.cuda.synchronize()
        with torch.cuda.graph(d["g"], stream=st):
            for _ in range(3):
                wl.check(lib.wl_kv4_attention(ptr(d["q"]), rows, rows, heads, kv_heads, hd, hd ** -0.5, ptr(d["rows"]), ptr(d["pos"]), 1800,
                                              window, 4, ptr(d["o"]), ptr(d["ws"]), d["ws"].numel(), C.c_void_p(st.cuda_stream)))
        sets.append(d)
    for _ in range(5):
        for d in sets:
            d["o"].zero_()
        torch.cuda.synchronize()
        for d in sets:
            with torch.cuda.stream(d["st"]):
                d["g"].replay()
        torch.cuda.synchronize()
        for d in sets:
            assert np.array_equal(host(d["o"]).view(np.uint32), d["want"].view(np.uint32))
    assert lib.wl_kernel_status(0) == 0


def test_one_workspace_serves_calls_of_different_shapes(wl):
    rng = np.random.default_rng(15)
    n = C.c_int64()
    shapes = [(16, 2, 128, 600, 1, 1), (8, 8, 64, 333, 5, 1), (8, 1, 256, 411, 40, 40), (16, 2, 128, 900, 64, 1), (16, 2, 128, 600, 1, 1)]
    need = 0
    for heads, kv_heads, hd, cap, T, runs in shapes:
        wl.check(wl.lib().wl_kv4_workspace_bytes(T, runs, heads, kv_heads, hd, cap, 0, 0, C.byref(n)))
        need = max(need, n.value)
    ws = empty(need, "uint8")
    ws.fill_(0xFF)
    wl.check(wl.lib().wl_kv4_workspace_init(ptr(ws), need, None))
    for heads, kv_heads, hd, cap, T, runs in shapes:
        c, raw = filled(rng, 1, kv_heads, hd, cap, [cap])
        pos = [cap - T + t for t in range(T)]
        q = rng.standard_normal((T, heads, hd)).astype(np.float32)
        check(attend(wl, c, [0] * T, pos, q, runs=runs, ws=ws), q, raw, kv_heads, hd, [0] * T, pos)


def test_buffers_that_are_not_the_devices_are_refused(wl):
    heads, kv_heads, hd, cap = 8, 2, 64, 32
    c = Cache(1, kv_heads, hd, cap)
    rows, dp = c.rows([0]), dev(np.zeros(1, np.int32))
    q, out, ws = empty((2, heads, hd)), empty((1, heads, hd)), workspace(wl, 1, 1, heads, kv_heads, hd, cap)
    on_host = np.zeros((1, heads, hd), np.float32)

    def call(qp, wsp=None):
        wl.check(wl.lib().wl_kv4_attention(qp, 1, 1, heads, kv_heads, hd, 1.0, ptr(rows), ptr(dp), cap, 0, 0, ptr(out),
                                           wsp or ptr(ws), ws.numel(), None))
    with pytest.raises(wl.ArgumentError, match="not device memory"):
        call(C.c_void_p(on_host.ctypes.data))
    with pytest.raises(wl.ArgumentError, match="aligned"):
        call(C.c_void_p(q.data_ptr() + 4))
    with pytest.raises(wl.ArgumentError, match="aligned"):
        call(ptr(q), C.c_void_p(ws.data_ptr() + 16 + 4))
    call(ptr(q))
