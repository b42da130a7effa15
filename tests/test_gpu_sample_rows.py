"""wl_sample_rows and the forward calls that use it (temperature, top-k, top-p, min-p) against the definition in numpy. A
choice may differ only where the draw, or the nucleus's end, lies within the sums' rounding of a boundary between two
ids: the reference reports that distance, and such draws (about one in a million) are left out."""
import ctypes as C

import numpy as np
import pytest

from gpu_util import dev, host, ptr, torch_cuda
from windlass_b200.transformer import CudaTransformer, config0_spec

pytestmark = pytest.mark.gpu

DT = np.dtype([("temperature", "f8"), ("top_p", "f8"), ("min_p", "f8"), ("draw", "f8"), ("top_k", "i8")])


def reference(x, o):
    """(id, distance of the nearest boundary in shares of the sum)."""
    x = np.asarray(x, dtype=np.float32)
    if not o["temperature"] > 0:
        return (0 if np.isnan(x[0]) or not (x > -np.inf).any() else int(np.nanargmax(x))), 1.0
    ok = x > -np.inf
    if not ok.any():
        return 0, 1.0
    top = x[ok].max()
    with np.errstate(invalid="ignore", over="ignore"):
        p = np.where(x == top, 1.0, np.exp((x - top).astype(np.float64) / o["temperature"]))
    p[~ok] = 0
    order = np.lexsort((np.arange(x.size), -np.where(ok, x, -np.inf).astype(np.float64)))
    order = order[ok[order]]
    margin = 1.0
    k = int(o["top_k"])
    if (k <= 0 or k >= x.size) and not o["top_p"] < 1 and not o["min_p"] > 0:
        order = np.flatnonzero(ok)
    if k > 0:
        order = order[:k]
    c = np.cumsum(p[order])
    keep = len(order)
    if o["top_p"] < 1:
        keep = min(keep, 1 + int(np.searchsorted(c, o["top_p"] * c[-1])))
        margin = np.abs(c - o["top_p"] * c[-1]).min() / c[-1]
    if o["min_p"] > 0:
        keep = min(keep, int((p[order] >= o["min_p"]).sum()))
    keep = max(1, keep)
    at = int(np.searchsorted(c[:keep], max(o["draw"] * c[keep - 1], 1e-300)))
    if o["draw"] > 0:
        margin = min(margin, np.abs(c[:keep] - o["draw"] * c[keep - 1]).min() / c[keep - 1])
    return int(order[min(at, keep - 1)]), margin


def sample(wl, x, opts, ld=None, stream=None):
    torch = torch_cuda()
    rows, v = x.shape
    d = torch.full((rows, ld or v), 1e30, device="cuda")
    d[:, :v] = dev(np.ascontiguousarray(x, dtype=np.float32))
    o = dev(np.ascontiguousarray(opts).view(np.uint8))
    ids = torch.full((rows + 1,), -7, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    wl.check(wl.lib().wl_sample_rows(ptr(d), ld or v, v, rows, ptr(o), ptr(ids), stream))
    out = host(ids)
    assert out[-1] == -7
    return out[:-1]


def check(wl, x, opts, ld=None):
    got = sample(wl, x, opts, ld)
    # rounding p to multiples of 2^-F moves a sum by at most V / 2 of them (F = 62 - log2 V, 51 at most); the reference's
    # running sum by V of its own half steps
    tol = 2 * x.shape[1] * (2.0 ** -min(51, 62 - int(np.ceil(np.log2(max(2, x.shape[1]))))) + 2.0 ** -53)
    near = 0
    for r in range(x.shape[0]):
        want, margin = reference(x[r], opts[r])
        if margin > tol:
            assert got[r] == want, (r, opts[r], int(got[r]), want, margin)
        else:
            near += 1
    return near


def mixed(rng, rows, v):
    o = np.zeros(rows, DT)
    o["temperature"] = np.where(rng.random(rows) < 0.1, 0.0, rng.uniform(0.3, 1.6, rows))
    o["top_p"] = np.where(rng.random(rows) < 0.4, 1.0, rng.uniform(0.02, 0.999, rows))
    o["min_p"] = np.where(rng.random(rows) < 0.6, 0.0, 10.0 ** rng.uniform(-6, 0, rows))
    o["top_k"] = np.where(rng.random(rows) < 0.5, 0, (v ** rng.random(rows)).astype(int))
    o["draw"] = rng.random(rows)
    return o


@pytest.mark.parametrize("V", [1, 2, 3, 31, 255, 4097, 8193, 20011, 32000, 65537, 128256, 151936])
def test_rows_of_every_kind(wl, V):
    rng = np.random.default_rng(V)
    rows = 40 if V < 50000 else 24
    x = (rng.standard_normal((rows, V)) * rng.uniform(0.3, 4, (rows, 1))).astype(np.float32)
    for r in range(0, rows, 3):
        x[r, rng.integers(0, V, 6)] += 9
    for r in range(1, rows, 4):
        x[r, rng.random(V) < 0.97] = -np.inf
    near = check(wl, x, mixed(rng, rows, V)) + check(wl, x, mixed(rng, rows, V), ld=V + 3)
    assert near <= 2


@pytest.mark.parametrize("V", [5, 700, 128256])
def test_ties_and_crowded_bins(wl, V):
    """Rows whose values are far from evenly spread: all equal, a few levels, one far outlier, subnormal differences."""
    rng = np.random.default_rng(V)
    base = [np.zeros(V), rng.integers(-2, 3, V), np.where(np.arange(V) == V // 2, 1e30, rng.standard_normal(V)),
            rng.standard_normal(V) * 1e-42, -rng.random(V) * 1e-6 + 5, np.where(rng.random(V) < 0.5, -1e38, 3e38),
            np.exp(rng.uniform(-80, 80, V)), -np.exp(rng.uniform(-80, 80, V)), np.where(rng.random(V) < 0.5, 0.0, -0.0)]
    for b in base:
        x = np.repeat(b[None].astype(np.float32), 12, 0)
        o = mixed(rng, 12, V)
        check(wl, x, o)


def test_infinite_and_nan_logits(wl):
    rng = np.random.default_rng(4)
    V = 9001
    x = rng.standard_normal((8, V)).astype(np.float32)
    x[0, :] = -np.inf                                   # nothing left
    x[1, :] = np.nan
    x[2, [7, 4000, 9000]] = np.inf                      # +inf takes all the mass, shared
    x[3, rng.random(V) < 0.9] = np.nan
    x[4, 0] = np.nan
    x[5, :] = -np.inf
    x[5, 8123] = -5.0                                   # one id left
    x[6, :] = -3.4028235e38
    x[6, 17] = -3.4e38
    x[7, rng.random(V) < 0.5] = -3.4028235e38           # a mask of the type's lowest value
    for kw in (dict(), dict(top_k=5), dict(top_p=0.9), dict(min_p=0.05), dict(top_k=300, top_p=0.7, min_p=1e-4), dict(temperature=0.0),
               dict(temperature=1e-300), dict(temperature=1e300), dict(top_p=-1.0), dict(min_p=7.0), dict(top_k=2 ** 62), dict(top_k=-3)):
        for draw in (0.0, 0.37, 0.999999):
            o = np.zeros(8, DT)
            o["temperature"], o["top_p"], o["draw"] = 0.8, 1.0, draw
            for k, v in kw.items():
                o[k] = v
            check(wl, x, o)


def test_a_draw_outside_its_range_gives_minus_one(wl):
    x = np.zeros((5, 100), np.float32)
    o = np.zeros(5, DT)
    o["temperature"], o["top_p"] = 1.0, 1.0
    o["draw"] = [1.0, -0.1, np.nan, 0.5, 7.0]
    o["temperature"][4] = 0.0
    got = sample(wl, x, o)
    assert list(got[:3]) == [-1, -1, -1] and got[3] == 49 and got[4] == 0


def test_agrees_with_wl_sample(wl):
    """Without top-k and min-p the choice is wl_sample's."""
    rng = np.random.default_rng(2)
    for V in (1000, 128256):
        x = (rng.standard_normal((6, V)) * 3).astype(np.float32)
        o = mixed(rng, 6, V)
        o["top_k"] = 0
        o["min_p"] = 0
        got = sample(wl, x, o)
        d, one = dev(x), dev(np.zeros(1, np.int32))
        for r in range(6):
            wl.check(wl.lib().wl_sample(C.c_void_p(d[r].data_ptr()), V, o["temperature"][r], o["top_p"][r], o["draw"][r], ptr(one), None))
            assert host(one)[0] == got[r]


def test_many_rows_and_repeats_on_two_streams_at_once(wl):
    torch = torch_cuda()
    rng = np.random.default_rng(7)
    V, rows = 5003, 3000
    x = (rng.standard_normal((rows, V)) * 2).astype(np.float32)
    o = mixed(rng, rows, V)
    first = sample(wl, x, o)
    for r in range(0, rows, 97):
        want, margin = reference(x[r], o[r])
        assert first[r] == want or margin < 1e-11
    d, do = dev(x), dev(o.view(np.uint8))
    outs, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for i in range(6):
        out = torch.empty(rows, dtype=torch.int32, device="cuda")
        wl.check(wl.lib().wl_sample_rows(ptr(d), V, V, rows, ptr(do), ptr(out), C.c_void_p(streams[i % 2].cuda_stream)))
        outs.append(out)
    for out in outs:
        assert np.array_equal(host(out), first)


def test_captured_rows_read_new_options_on_replay(wl):
    torch = torch_cuda()
    rng = np.random.default_rng(19)
    V = 32000
    x = (rng.standard_normal((4, V)) * 2).astype(np.float32)
    d, do, out = dev(x), dev(np.zeros(4, DT).view(np.uint8)), dev(np.zeros(4, np.int32))
    st, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=st):
        wl.check(wl.lib().wl_sample_rows(ptr(d), V, V, 4, ptr(do), ptr(out), C.c_void_p(st.cuda_stream)))
    for _ in range(4):
        o = mixed(rng, 4, V)
        do.copy_(dev(o.view(np.uint8)))
        torch.cuda.synchronize()
        g.replay()
        for r in range(4):
            want, margin = reference(x[r], o[r])
            assert host(out)[r] == want or margin < 1e-11


def test_a_vocabulary_past_shared_memory(wl):
    rng = np.random.default_rng(23)
    x = (rng.standard_normal((3, 700_001)) * 2).astype(np.float32)
    o = np.zeros(3, DT)
    o["temperature"], o["top_p"], o["top_k"], o["draw"] = 1.0, [1.0, 0.8, 1.0], [0, 0, 5000], [0.7, 0.3, 0.5]
    check(wl, x, o)


def test_forward_calls_sample_their_logits(wl):
    rng = np.random.default_rng(31)
    prompt = rng.integers(0, 4096, 16).astype(np.int32)
    with CudaTransformer(synthetic=config0_spec(), max_context=128) as m:
        a, b = m.new_sequence(), m.new_sequence()
        toks = prompt
        for i in range(4):
            lg = m.forward(toks, seq=a, pos0=a.length)
            kw = [dict(top_k=20), dict(top_p=0.8, min_p=0.01), dict(temperature=0.0), dict()][i]
            draw = float(rng.random())
            got = m.forward_sample_opts(toks, draw, seq=b, pos0=b.length, **kw)
            o = np.zeros(1, DT)
            o["temperature"], o["top_p"], o["draw"] = 1.0, 1.0, draw
            for k, v in kw.items():
                o[k] = v
            want, margin = reference(lg, o[0])
            assert got == want or margin < 1e-11
            toks = [want]
        with pytest.raises(wl.ArgumentError):
            m.forward_sample_opts([1], 1.0, seq=b, pos0=b.length)
        seqs = [m.new_sequence() for _ in range(5)]
        for j, s in enumerate(seqs):
            m.forward(prompt[: 2 + j], seq=s)
        toks = np.array([7, 70, 700, 3000, 1], dtype=np.int32)
        lb = m.forward_batch(seqs, toks)
        for s in seqs:
            s.truncate(s.length - 1)
        o = np.zeros(5, DT)
        o["temperature"], o["top_k"], o["top_p"], o["min_p"], o["draw"] = [1, 0, 0.5, 2, 1], [0, 0, 9, 0, 400], [1, 1, 0.9, 0.5, 1], [0, 0, 0, 0.01, 0], rng.random(5)
        got = m.forward_batch_sample_opts(seqs, toks, o["draw"], o["temperature"], o["top_k"], o["top_p"], o["min_p"])
        for r in range(5):
            want, margin = reference(lb[r], o[r])
            assert got[r] == want or margin < 1e-11
        assert [s.length for s in seqs] == [3, 4, 5, 6, 7]
        with pytest.raises(wl.ArgumentError):
            m.forward_batch_sample_opts(seqs, toks, 1.5)
