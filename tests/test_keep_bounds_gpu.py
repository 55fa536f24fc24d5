"""Keeping rows whose places no table reaches."""
import pytest
import torch

import test_keep_rows_gpu as keeping

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("start", [1 << 14, (1 << 31) - 1000, (1 << 31) - 3])
def test_keeping_beyond_the_tables(start):
    """Places whose sum passes 2^31 are missing pages like others."""
    b = keeping.batch(torch.bfloat16, 2, 2, 64, 64, 16, [(20, 9, 4), (40, 4, 2)], 3)
    want_k, want_v = keeping.plain(dict(b, accepted=[0, 2]))
    b["path"][:4] = [0, 2, 4, 8]
    k, v, status = keeping.run(dict(b, starts=[start, 40]))
    assert status != 0 and torch.equal(k, want_k) and torch.equal(v, want_v)
