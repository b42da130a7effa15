"""Batches of more than 64 rows on the 4-bit cache: a row's bits are those it has alone."""
import numpy as np
import pytest

import kv4_ref as R
from test_gpu_kv4 import append, attend, Cache
from windlass_b200 import _lib
from windlass_b200.transformer import CudaTransformer, synth_spec

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv_heads,hd", [(8, 8, 64), (8, 2, 64), (6, 3, 96), (16, 2, 128), (20, 1, 128), (4, 1, 256)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1500, 5)])
def test_rows_of_a_large_call_have_their_bits_alone(wl, heads, kv_heads, hd, window, sinks):
    rng = np.random.default_rng(heads + hd)
    n = 3000
    c = Cache(2, kv_heads, hd, n)
    raw = []
    for s in range(2):
        k, v = (rng.standard_normal((n, kv_heads, hd)).astype(np.float32) for _ in range(2))
        append(wl, c, [s] * n, range(n), k, k, v, np.zeros((1, 1, 2), np.float32), 0, False)
    raw = c.host()
    for T in (64, 65, 150):
        seq = [int(s) for s in rng.integers(0, 2, T)]
        pos = [int(p) for p in rng.integers(0, n, T)]
        pos[:6] = [n - 1, 767, 768, 783, 0, -1]
        pos[T - 1] = n - 2
        q = rng.standard_normal((T, heads, hd)).astype(np.float32)
        out = attend(wl, c, seq, pos, q, window, sinks)
        for t in [0, 1, 2, 3, 4, 5, T - 1] + [int(x) for x in rng.integers(6, T, 6)]:
            one = attend(wl, c, seq[t:t + 1], pos[t:t + 1], q[t:t + 1], window, sinks)
            assert np.array_equal(one[0].view(np.uint32), out[t].view(np.uint32)), (T, t, pos[t])
        for t in (0, T - 1):
            k, v = (R.read(raw[seq[t]], kv_heads, hd, pos[t] + 1, e) for e in (False, True))
            want, bound = R.attention(q[t], k, v, pos[t], hd ** -0.5, window, sinks)
            assert (np.abs(out[t] - want).max(-1) <= bound).all()
    assert wl.lib().wl_kernel_status(0) == 0


def test_model_steps_of_more_than_64_sequences_are_bit_identical_to_single_steps(wl):
    rng = np.random.default_rng(17)
    spec = synth_spec("llama", 2, 256, 8, 2, 64, 256, 1024, 4096, rope_base=10000.0, type_ffn_down=8, seed=1)
    kw = dict(synthetic=spec, max_context=4096, max_batch=80, kv_type=_lib.TYPES["q4_0"])
    lengths = [900, 1, 2500, 17] + [int(x) for x in rng.integers(1, 30, 61)] + [1300]
    with CudaTransformer(**kw) as m, CudaTransformer(**kw) as solo:
        seqs, ref = [m.new_sequence() for _ in lengths], [solo.new_sequence() for _ in lengths]
        for s, r, n in zip(seqs, ref, lengths):
            prompt = rng.integers(0, 1024, n).astype(np.int32)
            m.forward(prompt, seq=s)
            solo.forward(prompt, seq=r)
        toks = rng.integers(0, 1024, len(lengths)).astype(np.int32)
        for step in range(2):
            rows = m.forward_batch(seqs, toks)
            for i in (0, 1, 2, 3, 30, len(lengths) - 1):
                one = solo.forward([toks[i]], pos0=ref[i].length, seq=ref[i])
                assert np.array_equal(rows[i].view(np.uint32), one.view(np.uint32)), (step, i)
            for i in set(range(len(lengths))) - {0, 1, 2, 3, 30, len(lengths) - 1}:
                solo.forward([toks[i]], pos0=ref[i].length, seq=ref[i])
            toks = rows.argmax(1).astype(np.int32)
