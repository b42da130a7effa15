"""A model on the 4-bit cache split over several GPUs (one process for all of them) against the same model on one: each rank
keeps its own KV heads. Needs at least 2 GPUs; WL_TP_TEST_GPUS picks how many (default 2)."""
import os

import numpy as np
import pytest

from test_gpu_tp import _gpus
from tp_worker import spec_of
from windlass_b200 import _lib
from windlass_b200.transformer import CudaTransformer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("spec", ["gqa", "moe"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 2)])
def test_split_heads_give_the_whole_models_logits(wl, spec, window, sinks):
    n = int(os.environ.get("WL_TP_TEST_GPUS", "2"))
    if _gpus() < n:
        pytest.skip(f"needs {n} GPUs")
    rng = np.random.default_rng(5)
    prompt = rng.integers(0, 8192, 40).astype(np.int32)
    kw = dict(synthetic=spec_of(spec), max_context=256, kv_type=_lib.TYPES["q4_0"], attn_window=window, attn_sinks=sinks)
    with CudaTransformer(**kw) as one, CudaTransformer(**kw, tp_size=n, tp_rank=-1) as split:
        for m in (one, split):
            m.seqs = [m.new_sequence() for _ in range(3)]
        for t in range(3):
            a, b = (m.forward(prompt[t:30 + 5 * t], seq=m.seqs[t]) for m in (one, split))
            # sums of n partials: other roundings, so codes at a border may flip (1 % of the size each side, the largest of 8192
            # logits lies sqrt(2 ln 8192) = 4.2 of that out: sqrt(2) * 1 % * 4.2)
            assert np.abs(a - b).max() < 0.06 * a.std()
        toks = rng.integers(0, 8192, 3).astype(np.int32)
        a, b = (m.forward_batch(m.seqs, toks) for m in (one, split))
        assert np.abs(a - b).max() < 0.06 * a.std()
        ids = split.forward_batch_sample_opts(split.seqs, toks, 0.5, 1.0, 1, 1.0, 0.0)      # top-k of 1: the largest
        assert all(0 <= i < 8192 for i in ids)
        for m in (one, split):
            for s in m.seqs:
                s.close()
