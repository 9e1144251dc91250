"""GPU: bounded waits of the attention kernel for prompt chunks that run out.  In a process of its own: it counts them."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

CHECK = """
import sys
import numpy as np
import torch
from test_kv8_gpu import D, filled
from prime_kernels_b200 import _cabi, kv8

dev, lib = torch.device("cuda:0"), _cabi.library()
g = torch.Generator().manual_seed(1)
for new in ([300, 300, 0, 260], [800] + [30] * 49):          # the second: tiles taken in turns
    heads = 10
    cache, scales, table, lens = filled(g, [n + 250 for n in new], heads, 16, False, dev)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device=dev)
    q = torch.randn(sum(new), 3 * heads, D, generator=g).bfloat16().to(dev)
    table, lens = table.to(dev), lens.to(dev)

    def run():
        return kv8.attention(q, cache, scales, table, lens, cu, return_lse=True)

    out, lse = run()
    kv8.check_status(dev)
    assert torch.isfinite(out).all()
    for limit in (0, 0, 1, 2, 8, 64, 1000):
        lib.pk_kv8_set_wait_limit(limit)
        a, b = run()
        expired = True
        try:
            kv8.check_status(dev)
            expired = False
        except RuntimeError as e:
            assert "gave up" in str(e)
        lost = torch.isnan(a).any(-1)
        assert torch.equal(lost, torch.isnan(a).all(-1)) and torch.equal(lost, torch.isnan(b))
        assert torch.equal(a[~lost], out[~lost]) and torch.equal(b[~lost], lse[~lost])
        assert expired == bool(lost.any()), limit
        assert limit or lost.all()
        print(len(new), limit, expired, float(lost.float().mean()))
    lib.pk_kv8_set_wait_limit(-1)
    for _ in range(3):                                       # nothing is left behind: tensor memory, barriers, the counter
        a, b = run()
        assert torch.equal(a, out) and torch.equal(b, lse)
    kv8.check_status(dev)
print("done")
"""


def test_expired_waits_give_nan_and_an_error(cuda_device):
    """Limits from none to a thousand polls: rows are whole or NaN, the check raises exactly where some are, and the next
    launch is right again."""
    here = Path(__file__).resolve().parent
    proc = subprocess.run([sys.executable, "-c", CHECK], cwd=here, env={**os.environ, "PYTHONPATH": f"{here}:{here.parent}"},
                          capture_output=True, text=True, timeout=300)
    assert proc.returncode == 0 and proc.stdout.strip().endswith("done"), proc.stdout[-2000:] + proc.stderr[-3000:]
