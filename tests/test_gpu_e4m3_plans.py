"""Attention over the e4m3 cache on every path that a plan can take: several
items in a workgroup, unlike ones after each other, cut tiles of every height,
merges whose bases and sums outgrow the LDS."""
import numpy as np
import pytest

import _e4m3_steps as S
from test_gpu_e4m3 import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", S.STEPS)
def test_step(gpu, name):
    step = S.Step(name)
    got = step.run()
    assert np.isfinite(got).all()
    many = len(step.sessions) > 8
    for s, row, cols, want, bound in step.checks(rows=1 if many else 12):
        check(got[row, cols], want, bound, step.type)
    # the same bits again, through the same plan's merge records
    assert np.array_equal(step.run(), got)
    step.close()
