"""wl_sample_rows of different vocabularies next to one another: in one graph, and from two host threads at once."""
import ctypes as C
import threading

import numpy as np
import pytest

from gpu_util import dev, host, ptr, torch_cuda
from test_gpu_sample_rows import DT, mixed, reference

pytestmark = pytest.mark.gpu


def case(rng, rows, v):
    x = (rng.standard_normal((rows, v)) * 2).astype(np.float32)
    o = mixed(rng, rows, v)
    d, do, out = dev(x), dev(o.view(np.uint8)), dev(np.full(rows, -7, np.int32))
    want = [reference(x[r], o[r]) for r in range(rows)]
    return d, do, out, want


def right(ids, want):
    return all(i == w or margin < 1e-11 for i, (w, margin) in zip(ids, want))


def test_large_and_small_vocabularies_in_one_graph(wl):
    torch = torch_cuda()
    rng = np.random.default_rng(1)
    cases = [case(rng, 3, v) for v in (300_000, 151_936, 900, 40_000)]
    st, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=st):
        for d, do, out, _ in cases:
            wl.check(wl.lib().wl_sample_rows(ptr(d), d.shape[1], d.shape[1], 3, ptr(do), ptr(out), C.c_void_p(st.cuda_stream)))
    g.replay()
    for d, do, out, want in cases:
        assert right(host(out), want), d.shape


def test_vocabularies_of_many_sizes_on_host_threads(wl):
    torch = torch_cuda()
    rng = np.random.default_rng(2)
    cases = [case(rng, 2, v) for v in (128_256, 1000, 151_936, 40_000, 500, 2000)]
    failed = []

    def work(d, do, out, want):
        st = torch.cuda.Stream()
        for _ in range(20000):
            status = wl.lib().wl_sample_rows(ptr(d), d.shape[1], d.shape[1], 2, ptr(do), ptr(out), C.c_void_p(st.cuda_stream))
            if status:
                failed.append((d.shape[1], status, wl.lib().wl_last_error()))
                break
        st.synchronize()

    threads = [threading.Thread(target=work, args=c) for c in cases]
    torch.cuda.synchronize()
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for d, do, out, want in cases:
        assert right(host(out), want), d.shape
