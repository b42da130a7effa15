"""Models opened from a GGUF file in processes of their own: what is uploaded is there when the first kernels read it, streamed
or resident, however cold the process is."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = """
import sys
import numpy as np
sys.path[:0] = [{root!r}, {tests!r}]
from test_oracle_arch import PROBE
from windlass_b200.transformer import CudaTransformer
want = np.load({want!r})
for resident in {order}:
    with CudaTransformer({path!r}, resident=resident, prefill_path=2) as m:
        got = m.forward(PROBE, all_logits=True)
    assert np.abs(got - want).max() <= 1e-3 * want.std(), (resident, float(np.abs(got - want).max()))
"""


@pytest.mark.parametrize("order", [(0, 1), (1, 0)])
@pytest.mark.parametrize("i", [0, 2, 4, 5])
def test_a_fresh_process_reads_whole_weights(wl, oracle, tmp_path, i, order):
    import numpy as np
    from test_oracle_arch import PROBE, SPECS, write
    p = write(oracle, tmp_path, SPECS[i])
    want = str(tmp_path / "want.npy")
    np.save(want, oracle.Model(p).forward(PROBE, all_logits=True))
    code = CHILD.format(root=ROOT, tests=os.path.join(ROOT, "tests"), want=want, path=p, order=order)
    for _ in range(2):
        r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=120)
        assert r.returncode == 0, r.stderr[-800:]
