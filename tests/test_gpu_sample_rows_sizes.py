"""GPU tests of neon_sample_rows at the sizes of its documented range: workspaces
shared by batches of different sizes, vocabularies past 2^18 tokens."""
import numpy as np
import pytest

import neonengine_amd as ne
from tests.gpu_util import to_dev, to_host, torch_cuda

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [32003, 4097])
def test_one_workspace_for_all_batches(V):
    """Sized for 300 rows, used by fewer; flat rows, whose draw is floor(u V)."""
    torch = torch_cuda()
    ws = torch.empty(max(ne.sample_rows_workspace(300, V), 1), dtype=torch.uint8, device="cuda")
    rng = np.random.default_rng(V)
    for B in (300, 257, 256, 100, 17, 1):
        u = rng.random(B).astype(np.float32)
        out = torch.full((B,), -5, dtype=torch.int32, device="cuda")
        ws.fill_(0xA5)
        ne.sample_rows(torch.full((B, V), 1.5, device="cuda"), to_dev(u), out, workspace=ws)
        # u V is a multiple of 2^-24: exact in 64 bits
        assert np.array_equal(to_host(out), np.floor(u.astype(np.float64) * V).astype(np.int32)), B
    ne.device_check()
