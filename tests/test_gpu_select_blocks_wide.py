"""select_blocks on wide rows, up to the widest it takes, against its CPU restatement."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

WIDE = """
import sys
sys.path[:0] = {paths!r}
import numpy as np, torch, hcu_ops
from oracle import sparse as O
from test_gpu_select_blocks import _make, _mask_words
dev = torch.device("cuda", 0)
for nb in {blocks}:
    width = 64 * nb - 5
    lens = np.array([width, width - 700], np.int32)
    s, bits = _make(2, width, lens, "normal", nb)
    buf = torch.full((2, (width + 3) // 4 * 4), float("nan"), device=dev)
    buf[:, :width] = torch.from_numpy(np.where(bits, s, np.float32(np.nan)))
    got = hcu_ops.select_blocks(buf[:, :width], torch.from_numpy(_mask_words(bits)).to(dev), torch.from_numpy(lens).to(dev),
                                64, n_sink=1, n_local=2).cpu().numpy()
    for r in range(2):
        assert np.array_equal(got[r], O.select_blocks(s[r], bits[r], int(lens[r]), 64, 1, 2)), (nb, r)
    print("ok", nb)
"""


@pytest.mark.parametrize("blocks", [(10000, 10200), (10208, 10209), (10240, 10241), (16384, 49152)])
def test_wide_rows_in_a_fresh_process(hcu, dev, blocks):
    """Widths around the one at which the keys of a row no longer fit the shared memory that a kernel has without
    asking, and the widest: in a process of its own, where no wider call came before."""
    here = os.path.dirname(os.path.abspath(__file__))
    repo = os.path.dirname(here)
    code = WIDE.format(paths=[repo, here, os.path.join(repo, "sglang0.5.18-opt_b200")], blocks=list(blocks))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=600, cwd=repo)
    assert r.returncode == 0, r.stderr[-2000:]
