"""What requests of a batch say of themselves that cannot be: it is reported, nothing of theirs is read or written, the others come out as ever."""
import pytest
import torch

from test_tree_attention_gpu import BF, F32, FAR, Batch

pytestmark = pytest.mark.gpu


def others(b, out, bad, status):
    """Checks all requests but ``bad``, whose rows stay as they were."""
    assert int(b.status.item()) == status
    b.status.zero_()
    for i in bad:
        rows = out[b.firsts[i]:b.firsts[i + 1]]
        assert (rows == 7.0).all()
        rows.zero_()                                      # (what ``check`` expects of a padding request)
        b.shapes[i] = (-1, b.shapes[i][1])
    b.check(out)


@pytest.mark.parametrize("dtype,nh,nkv,hd,shapes,most,reach", [
    (F32, 4, 2, 64, [(1200, 9), (900, 40), (30, 4)], 9, None),                                 # shares and their sum
    (F32, 4, 2, 64, [(3, 9), (2, 40), (30, 4)], 9, 1),
    (BF, 4, 2, 64, [(1200, 9), (900, 40), (30, 4)], 9, None),                                  # clusters
    (BF, 4, 4, 64, [(2000, 20)] * 20 + [(1500, 150)] + [(2000, 20)] * 19, 20, None),           # keys cut evenly
    (BF, 6, 6, 96, [(700, 33)] * 20 + [(700, 100)] * 3, 33, None),
    (BF, 4, 2, 64, [(600, 40), (513, 300), (40, 33)], 40, FAR),                                # tcgen05
    (BF, 4, 2, 128, [(600, 40), (513, 300), (2000, 65)], 65, FAR),
    (BF, 4, 1, 128, [(600, 40), (513, 300), (2000, 65)], 65, FAR),
    (BF, 4, 1, 128, [(513, 1000), (600, 40), (2000, 65)], 65, None)])
def test_more_rows_than_said(dtype, nh, nkv, hd, shapes, most, reach):
    b = Batch(dtype, nh, nkv, hd, list(shapes), seed=31)
    bad = [i for i, (_, rows) in enumerate(shapes) if rows > most]
    b.most = most
    others(b, b.run(reach=reach), bad, 2)


@pytest.mark.parametrize("dtype,reach", [(F32, None), (BF, None), (BF, FAR)])
def test_rows_outside_the_batch(dtype, reach):
    b = Batch(dtype, 4, 2, 64, [(1200, 40), (900, 33), (1500, 20)], seed=32, behind=0)
    b.dev["first"][3] = b.n + 7
    others(b, b.run(reach=reach), [2], 2)


@pytest.mark.parametrize("start", [1 << 14, (1 << 31) - 1000, (1 << 31) - 30])
@pytest.mark.parametrize("dtype,hd,reach,rows", [(F32, 64, None, 9), (BF, 64, None, 9), (BF, 64, None, 60), (BF, 128, FAR, 40)])
def test_beyond_the_tables(start, dtype, hd, reach, rows):
    """Positions that the tables do not reach, the last ones with sums that pass 2^31."""
    b = Batch(dtype, 4, 2, hd, [(1200, rows), (900, rows), (30, 4)], seed=33)
    b.dev["start"][1] = start
    others(b, b.run(reach=reach), [1], 4)
