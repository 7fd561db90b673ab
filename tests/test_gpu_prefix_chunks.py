"""What prompt chunks share does not count for qg_prefix_least_saving; what the sequences of few rows beside them do does."""
import numpy as np
import pytest

from prefix_oracle import prefixes
from spec_oracle import BF16, F16, F32
from test_gpu_prefix import build

pytestmark = pytest.mark.gpu
FAMILY = [(-1, 0, 600), (0, 600, 3), (0, 560, 60), (2, 570, 0), (0, 530, 4)]


@pytest.mark.parametrize("typ,size", [(F32, 4), (F16, 2), (BF16, 2)])
@pytest.mark.parametrize("counts", [[70, 1, 90, 5, 65], [70, 64, 90, 100, 1], [1, 65, 65, 65, 65], [65, 64, 64, 64, 64]])
def test_chunks_do_not_count(qgl, typ, size, counts):
    rng = np.random.default_rng(sum(counts))
    a = build(rng, FAMILY, counts, heads=4, typ=typ)
    saves = prefixes(a.cache.table, a.cache.pages, a.cache.P, a.cache.length, [1] * 5)[1] // 256 * 256
    few = int(sum(s for s, n in zip(saves, counts) if n <= 64)) * 2 * size * a.cache.H * a.cache.D
    assert (saves[1:] == 512).all()
    before = qgl.qg_prefix_least_saving(0)
    try:
        outs, heads = [], []
        for least in (0, few, few + 1):
            qgl.qg_prefix_least_saving(least)
            outs.append(a.check())
            a.plan.check()
            heads.append(a.plan.buffer.get()[:8].view(np.int32).tolist())  # segments, and those that are shared
        assert heads[0] == heads[1] and heads[0][1] > 0
        assert heads[2] == [5, 0]
        assert np.array_equal(outs[0], outs[1])
    finally:
        qgl.qg_prefix_least_saving(before)
