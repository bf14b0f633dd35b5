"""Top-k, sampling and distillation at the ends of their ranges: workspaces of exactly the size that is asked for, borders within a rounding of what decides,
logits that lie anywhere, rows by many millions.

Tolerances count half steps of f32, as beside each test."""
import numpy as np
import pytest

from block_util import Guarded, Kind, up
from vocab_util import order

pytestmark = pytest.mark.gpu


# ---- scratch ------------------------------------------------------------------------------------


@pytest.mark.parametrize("name,rows,cols", [("bf16", 8192, 128256), ("f32", 4096, 128256), ("f32", 4096, 152000), ("f32", 16384, 50257), ("bf16", 32768, 32000),
                                            ("bf16", 4096, 256000), ("f32", 16384, 32000)])
def test_a_workspace_of_the_size_that_is_asked_for(hpt, dev, name, rows, cols):
    """Rows beyond one run, with the sum and without it. The same eight rows again and again."""
    kind, rng, k = Kind(hpt, name), np.random.default_rng(cols), 3
    t, x = kind.up(rng.standard_normal((8, cols)))
    v = hpt.Tensor.from_raw(t.ptr, [rows // 8, 8, cols], kind.dtype, 0, [0, cols, 1])
    ws = Guarded(hpt, [hpt.topk_workspace(v, k)], hpt.u8)
    want = np.broadcast_to(order(x)[:, :k], (rows // 8, 8, k))
    for lse in (False, True):
        got = v.topk(k, lse=lse, workspace=ws.t)
        ws.numpy()
        assert np.array_equal(got[1].numpy(), want)
