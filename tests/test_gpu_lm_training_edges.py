"""The output layer with its loss and the orthogonalised updates where their sizes, magnitudes and masks end, against their
definitions in 64 bits; the bars are those of test_gpu_lm_training."""
import ctypes
import math

import numpy as np
import pytest
import torch

from test_gpu_lm_training import COEF, check, definition, gen, make, muon64, run, schulz64, schulz_bar

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def capi():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    from origindl_amd import capi
    return capi


@pytest.mark.parametrize("count,rows,cols", [(63, 384, 1920), (61, 512, 3072), (35, 2000, 130), (33, 90, 5000)])
def test_a_batch_stays_inside_the_workspace_it_asks_for(capi, count, rows, cols):
    """What lies right behind the workspace keeps its bytes, whatever the last group's products are cut into."""
    from origindl_amd._lib import lib
    g = torch.randn(count, rows, cols, device="cuda", generator=gen(rows)) * 1e-2
    out = torch.empty_like(g)
    nb, guard = lib().query("odl_hip_newton_schulz_workspace_bytes", count, rows, cols), 64 << 20
    ws = torch.full((nb + guard,), 0x5A, dtype=torch.uint8, device="cuda")
    lib().call("odl_hip_newton_schulz", g.data_ptr(), count, rows, cols, 5, *COEF, 1e-7, out.data_ptr(), ws.data_ptr(), nb, capi._stream())
    assert bool((ws[nb:] == 0x5A).all())
    for i in (0, 31, 32, count - 1):
        want = schulz64(g[i])
        assert float((out[i].double() - want).norm()) <= schulz_bar(5) * max(1.0, float(want.norm())), i
